"""What the AdamW and embedding entry points refuse and keep, without a GPU."""
import ctypes as C

import pytest
import torch

P = 1 << 20   # an address that is never read: every call here is refused before a launch


def adamw(pkg, eps=1e-8, step=1, **fields):
    T = pkg._capi.AdamWTensor
    t = dict(param=P, grad=P, exp_avg=P, exp_avg_sq=P, exp_avg_scale=None, exp_avg_sq_scale=None, n=10, lr=1e-3, weight_decay=0.0, grad_dtype=0)
    t.update(fields)
    arr = (T * 1)(T(**t))
    return pkg._capi.lib().lfs_adamw_step_tensors(1, C.addressof(arr), 0.9, 0.999, eps, step, 1.0, None)


@pytest.mark.parametrize("eps", [1e-39, 1e-300, 2.0 ** -127, 1e38, float("inf"), float("nan")])
def test_eps_that_the_step_cannot_serve_is_refused(pkg, eps):
    """Below 2^-126 (and not zero) the reciprocal takes it as zero, and an element without a gradient would become 0 / 0; above 2^126 its reciprocal is not a normal number."""
    st = pkg.strategy
    assert adamw(pkg, eps=eps) == pkg._capi.LFS_EINVAL and "eps" in pkg._capi.lib().lfs_last_error().decode()
    model = pkg.trainer.SplatData(10, 4, torch.device("cpu"))
    with pytest.raises(RuntimeError, match="eps"):
        st.FusedAdamW(model, [1e-3] * 6, eps=eps)
    with pytest.raises(RuntimeError, match="eps"):
        st.AdamW([torch.zeros(4)], [torch.zeros(4)], eps=eps)


def test_eps_of_zero_and_of_the_smallest_normal_number_are_served(pkg):
    model = pkg.trainer.SplatData(10, 4, torch.device("cpu"))
    for eps in (0.0, 2.0 ** -126, 1e-15, 1.0):
        assert pkg.strategy.FusedAdamW(model, [1e-3] * 6, eps=eps).eps == eps
        assert adamw(pkg, eps=eps, n=0) == 0


def test_a_step_number_below_one_is_refused(pkg):
    for step, missed in ((5, 5), (5, 9), (5, -1), (1, 1)):
        assert adamw(pkg, step=step, missed=missed) == pkg._capi.LFS_EINVAL and "missed" in pkg._capi.lib().lfs_last_error().decode()
    assert adamw(pkg, step=5, missed=9, n=0) == 0     # a tensor that takes no part


def test_gradients_of_another_scene_are_refused(pkg):
    """FusedAdamW reads as many gradient rows as the model has."""
    st, tr = pkg.strategy, pkg.trainer
    cpu = torch.device("cpu")
    opt = st.FusedAdamW(tr.SplatData(10, 4, cpu), [1e-3] * 6, state_bits=8)
    for grads in (tr.SplatData(4, 4, cpu), tr.SplatData(10, 9, cpu), tr.SplatData(10, 4, torch.device("meta"))):
        size = grads.size
        with pytest.raises(RuntimeError, match="gradients"):
            opt.step(2000, grads)
        assert grads.size == size and opt.step_count == 0


def test_weight_decay_may_be_any_number(pkg):
    """numpy's scalars too, as one value for all groups."""
    import numpy as np
    st = pkg.strategy
    model = pkg.trainer.SplatData(10, 4, torch.device("cpu"))
    for zero in (0, 0.0, np.float32(0), np.float64(0)):
        assert type(st.make_optimizer(model, [1e-3] * 6, st.OptimizationParameters(weight_decay=zero))) is st.FusedAdam
    for some in (1, 0.5, np.float32(0.5), np.float64(0.5)):
        assert st.make_optimizer(model, [1e-3] * 6, st.OptimizationParameters(optimizer="adamw", weight_decay=some)).weight_decay == [float(some)] * 6
        with pytest.raises(RuntimeError, match="adamw"):
            st.make_optimizer(model, [1e-3] * 6, st.OptimizationParameters(weight_decay=some))


# ---- checkpoints ----------------------------------------------------------------------------------------------------
def strategy(pkg, kind="MCMC", **kw):
    st, tr = pkg.strategy, pkg.trainer
    model = tr.SplatData(9, 4, "cpu", capacity=16)
    params = dict(max_cap=16, sh_degree=1)
    params.update(kw)
    s = getattr(st, kind)(model)
    s.initialize(st.DefaultStrategy.Parameters(**params) if kind == "DefaultStrategy" else st.OptimizationParameters(**params))
    return s


@pytest.mark.parametrize("kind", ["MCMC", "DefaultStrategy"])
@pytest.mark.parametrize("bits", [32, 8])
def test_a_checkpoint_keeps_the_weight_decay(pkg, tmp_path, kind, bits):
    a = strategy(pkg, kind, optimizer="adamw", weight_decay=(0.0, 0.1, 0.2, 0.0, 0.3, 0.0), state_bits=bits)
    a._optimizer.weight_decay[5] = 0.7      # changed during the run, like a learning rate
    path = pkg.formats.save_checkpoint(a, str(tmp_path / "a.ckpt"), 100)
    b = strategy(pkg, kind, optimizer="adamw", weight_decay=0.05, state_bits=bits)
    assert pkg.formats.load_checkpoint(b, path) == 100
    assert b._optimizer.weight_decay == [0.0, 0.1, 0.2, 0.0, 0.3, 0.7]


def test_a_checkpoint_of_another_optimizer_is_refused(pkg, tmp_path):
    fm = pkg.formats
    path = fm.save_checkpoint(strategy(pkg, optimizer="adamw", weight_decay=0.1), str(tmp_path / "a.ckpt"), 1)
    with pytest.raises(RuntimeError, match="optimizer"):
        fm.load_checkpoint(strategy(pkg), path)
    path = fm.save_checkpoint(strategy(pkg), str(tmp_path / "b.ckpt"), 1)
    with pytest.raises(RuntimeError, match="optimizer"):
        fm.load_checkpoint(strategy(pkg, optimizer="adamw"), path)


def test_a_refused_checkpoint_changes_nothing(pkg, tmp_path):
    fm = pkg.formats
    path = fm.save_checkpoint(strategy(pkg, optimizer="adamw"), str(tmp_path / "a.ckpt"), 1)
    b = strategy(pkg)
    b.get_model().size = 5
    before = b.get_model().flat.clone()
    with pytest.raises(RuntimeError):
        fm.load_checkpoint(b, path)
    assert b.get_model().size == 5 and torch.equal(b.get_model().flat, before)


def test_a_checkpoint_without_these_fields_is_still_read(pkg, tmp_path):
    """As written before they were there: plain Adam's, and AdamW's with the caller's weight decay."""
    import json
    import struct
    fm = pkg.formats
    for kw in ({}, dict(optimizer="adamw", weight_decay=0.25)):
        path = fm.save_checkpoint(strategy(pkg, **kw), str(tmp_path / "a.ckpt"), 7)
        raw = open(path, "rb").read()
        (length,) = struct.unpack("<Q", raw[8:16])
        header = json.loads(raw[16:16 + length])
        header.pop("optimizer", None), header.pop("weight_decay", None)
        head = json.dumps(header).encode()
        with open(path, "wb") as f:
            f.write(raw[:8] + struct.pack("<Q", len(head)) + head + raw[16 + length:])
        b = strategy(pkg, **kw)
        assert fm.load_checkpoint(b, path) == 7
        if kw:
            assert b._optimizer.weight_decay == [0.25] * 6
