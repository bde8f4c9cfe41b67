"""8-bit moments of scenes without higher-order SH, and of scenes whose rows are all gone."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def strategy(pkg, kind, K):
    gen = torch.Generator().manual_seed(K)
    model = pkg.trainer.SplatData(200, K, torch.device("cuda"), 260)
    for name in pkg.trainer.PARAM_NAMES:
        model.tensor(name).copy_(torch.randn(model.tensor(name).shape, generator=gen))
    s = getattr(pkg.strategy, kind)(model)
    params = dict(optimizer="adamw", state_bits=8, max_cap=260, sh_degree=0 if K == 1 else 1)
    s.initialize(pkg.strategy.DefaultStrategy.Parameters(**params) if kind == "DefaultStrategy" else pkg.strategy.OptimizationParameters(**params))
    s.grads.flat.normal_(generator=torch.Generator("cuda").manual_seed(1))
    s.step(2000)
    return s


def check(pkg, s, size):
    model = s.get_model()
    assert model.size == size
    for x in (s._optimizer.exp_avg, s._optimizer.exp_avg_sq):
        x.size = size
        for name in pkg.trainer.PARAM_NAMES:
            assert x.tensor(name).shape == model.tensor(name).shape
    before = s._optimizer.step_count
    s._grads_valid = True
    s.step(2001)
    assert s._optimizer.step_count == before + 1 and all(torch.isfinite(t).all() for t in model.tensors().values())


@pytest.mark.parametrize("K", [1, 4])
def test_default_strategy(pkg, K):
    s = strategy(pkg, "DefaultStrategy", K)
    some = torch.arange(200, device="cuda") % 10 == 0
    s.duplicate(some)
    check(pkg, s, 220)
    s.split(torch.cat([some, some[:20]]))
    check(pkg, s, 242)
    s.remove(torch.arange(242, device="cuda") % 2 == 0)
    check(pkg, s, 121)
    s.reset_opacity()
    check(pkg, s, 121)
    s.remove(torch.ones(121, dtype=torch.bool, device="cuda"))
    check(pkg, s, 0)


@pytest.mark.parametrize("K", [1, 4])
def test_mcmc_and_its_checkpoint(pkg, tmp_path, K):
    s = strategy(pkg, "MCMC", K)
    s.get_model().tensor("opacity_raw")[::10] = -20.0
    assert s.relocate_gs() == 20
    check(pkg, s, 200)
    assert s.add_new_gs() > 0
    size = s.get_model().size
    check(pkg, s, size)
    path = pkg.formats.save_checkpoint(s, str(tmp_path / "a.ckpt"), 2002)
    other = strategy(pkg, "MCMC", K)
    assert pkg.formats.load_checkpoint(other, path) == 2002
    for x, y in ((s._optimizer.exp_avg, other._optimizer.exp_avg), (s._optimizer.exp_avg_sq, other._optimizer.exp_avg_sq)):
        assert all(torch.equal(x.tensor(k), y.tensor(k)) for k in pkg.trainer.PARAM_NAMES)
    mask = torch.arange(size, device="cuda") % 3 == 0
    s.remove_gaussians(mask)
    check(pkg, s, int((~mask).sum()))
    s.remove_gaussians(torch.ones(s.get_model().size, dtype=torch.bool, device="cuda"))
    check(pkg, s, 0)
