"""Scenes whose moments are in 8 bits: rows that are duplicated, split, removed and reset, and the steps that follow."""
import pytest
import torch

pytestmark = pytest.mark.gpu
TOPS = {"exp_avg": (448.0, 3, -6), "exp_avg_sq": (57344.0, 2, -14)}


def scene(pkg, n, K=4, capacity=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    model = pkg.trainer.SplatData(n, K, torch.device("cuda"), capacity)
    for name in pkg.trainer.PARAM_NAMES:
        model.tensor(name).copy_(torch.randn(model.tensor(name).shape, generator=gen))
    return model


def held(s):
    return {x: {k: getattr(s._optimizer, x).tensor(k) for k in s.get_model().tensors()} for x in TOPS}


def check_kept(before, after, rows, count):
    """`after`'s first `count` rows are `before`'s at `rows`, encoded again to the nearest code: half a place of the value's binade, or of the lowest one of the largest value (a second moment that is
    not zero is held as that one place at least)."""
    for x, (top, fraction, lowest) in TOPS.items():
        for k, b in before[x].items():
            a, b = after[x][k][:count], b[rows]
            if a.numel() == 0:
                continue
            place = torch.maximum(b.abs() * 2.0 ** -fraction, before[x][k].abs().max() / top * 2.0 ** (lowest - fraction))
            whole = x == "exp_avg_sq"
            assert ((a - b).abs() <= (1.0 if whole else 0.5) * place * (1 + 1e-5)).all(), (x, k)
            assert torch.equal(a == 0, b == 0) or not whole, (x, k)


def check_step(pkg, s, iteration, seed):
    """A step of the strategy is that of AdamW over copies of the live rows with the moments that are held."""
    st, opt, model, names = pkg.strategy, s._optimizer, s.get_model(), pkg.trainer.PARAM_NAMES
    s.grads.size = model.size
    s.grads.flat.copy_(scene(pkg, model.size, model.K, model.capacity, seed).flat)
    copies = [model.tensor(k).clone() for k in names]
    moments = []
    for k in names:
        (c, cs), (d, ds) = opt.exp_avg.live(k), opt.exp_avg_sq.live(k)
        moments.append(st.Moments(c.clone(), d.clone(), cs.clone(), ds.clone()))
    one = st.AdamW(copies, [s.grads.tensor(k).clone() for k in names], lr=list(opt.lr), eps=1e-15, weight_decay=opt.weight_decay, moments=moments)
    one.step_count = opt.step_count
    before = opt.step_count
    s._grads_valid = True
    s.step(iteration)
    assert opt.step_count == before + 1
    one.step()
    for i, k in enumerate(names):
        assert torch.isfinite(model.tensor(k)).all() and torch.equal(model.tensor(k), copies[i]), k
        for x, m, ms in ((opt.exp_avg, moments[i].exp_avg, moments[i].exp_avg_scale), (opt.exp_avg_sq, moments[i].exp_avg_sq, moments[i].exp_avg_sq_scale)):
            c, cs = x.live(k)
            assert torch.equal(c.view(torch.uint8), m.view(torch.uint8)) and torch.equal(cs, ms), k


def test_default_strategy_steps_after_each_kind_of_surgery(pkg):
    n = 300
    s = pkg.strategy.DefaultStrategy(scene(pkg, n, capacity=402))
    s.initialize(pkg.strategy.DefaultStrategy.Parameters(optimizer="adamw", state_bits=8, weight_decay=0.01, sh_degree=1))
    for it in (2000, 2001):
        check_step(pkg, s, it, it)
    # duplicate
    before, chosen = held(s), torch.zeros(n, dtype=torch.bool, device="cuda")
    chosen[::10] = True
    s.duplicate(chosen)
    assert s.get_model().size == 330 and not s._grads_valid
    after = held(s)
    check_kept(before, after, slice(None), n)
    assert all(after[x][k][n:].eq(0).all() for x in after for k in after[x])
    check_step(pkg, s, 2002, 5)
    # split
    before, chosen = held(s), torch.zeros(330, dtype=torch.bool, device="cuda")
    chosen[3:200:7] = True
    k = int(chosen.sum())
    s.split(chosen)
    assert s.get_model().size == 330 + k
    after = held(s)
    check_kept(before, after, ~chosen, 330 - k)
    assert all(after[x][name][330 - k:].eq(0).all() for x in after for name in after[x])
    check_step(pkg, s, 2003, 6)
    # remove
    before, gone = held(s), torch.arange(330 + k, device="cuda") % 3 == 0
    s.remove(gone)
    check_kept(before, held(s), ~gone, int((~gone).sum()))
    check_step(pkg, s, 2004, 7)
    # reset of the opacities: theirs alone
    before = held(s)
    s.reset_opacity()
    after = held(s)
    for x in after:
        for name in after[x]:
            assert after[x][name].eq(0).all() if name == "opacity_raw" else torch.equal(after[x][name], before[x][name])
    check_step(pkg, s, 2005, 8)


def test_mcmc_steps_after_each_kind_of_surgery(pkg):
    n = 400
    model = scene(pkg, n, capacity=500)
    model.tensor("opacity_raw")[::10] = -20.0     # dead
    s = pkg.strategy.MCMC(model)
    s.initialize(pkg.strategy.OptimizationParameters(max_cap=500, optimizer="adamw", state_bits=8, sh_degree=1))
    check_step(pkg, s, 2000, 1)
    assert s.relocate_gs() == 40
    check_step(pkg, s, 2001, 2)
    mask = torch.zeros(n, dtype=torch.bool, device="cuda")
    mask[5::7] = True
    before = held(s)
    s.remove_gaussians(mask)
    check_kept(before, held(s), ~mask, int((~mask).sum()))
    check_step(pkg, s, 2002, 3)
    # rows behind the last one that were in use before come back as zeros
    size = model.size
    assert s.add_new_gs() > 0
    after = held(s)
    assert all(after[x][k][size:].eq(0).all() for x in after for k in after[x])
    check_step(pkg, s, 2003, 4)


def test_surgery_needs_the_memory_of_one_group(pkg):
    """Largest group: 45 floats a row at SH degree 3. Duplicating holds its rows decoded and once more with the new ones behind them (180 bytes a row each), and their new codes (45 and a little); removing
    and splitting the same or less."""
    n = 200_000
    model = scene(pkg, n, 16, capacity=n + n // 10)
    s = pkg.strategy.DefaultStrategy(model)
    s.initialize(pkg.strategy.DefaultStrategy.Parameters(optimizer="adamw", state_bits=8))
    chosen = torch.zeros(n, dtype=torch.bool, device="cuda")
    chosen[::20] = True
    for f in (lambda: s.duplicate(chosen), lambda: s.remove(torch.arange(model.size, device="cuda") % 20 == 0), lambda: s.split(torch.arange(model.size, device="cuda") % 25 == 0)):
        torch.cuda.synchronize()
        torch.cuda.reset_peak_memory_stats()
        start, rows = torch.cuda.memory_allocated(), model.size
        f()
        torch.cuda.synchronize()
        assert torch.cuda.max_memory_allocated() - start <= (180 + 190 + 60 + 20 + 60) * rows, f"{(torch.cuda.max_memory_allocated() - start) / rows:.0f} bytes a row"
