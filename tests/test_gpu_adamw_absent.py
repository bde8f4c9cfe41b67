"""AdamW over tensors that do not all take part in every step: each has its own step number t in the bias corrections and in the thresholds of its 8-bit codes, so that it is trained as
by an optimizer of its own."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def st(pkg):
    return pkg.strategy


def values(n, seed, scale=1.0):
    return (torch.randn(n, generator=torch.Generator().manual_seed(seed)) * scale).cuda()


def state(opt, i):
    m = opt.moments[i]
    return [x.view(torch.uint8) for x in (opt.params[i], m.exp_avg, m.exp_avg_sq, m.exp_avg_scale, m.exp_avg_sq_scale) if x is not None]


@pytest.mark.parametrize("bits", [32, 8])
def test_a_first_gradient_late_in_a_run(st, bits):
    """A tensor left out of 40 steps and then trained for 3 has the bits of one that a fresh optimizer trains for 3, and its first step is lr: 0.1 g / (1 - 0.9) over the root of 0.001 g^2 / (1 - 0.999).
    Had it the common number t, the first step would be 0.1 / (1 - 0.9^t) / sqrt(0.001 / (1 - 0.999^t)) lr: 0.64 lr at t = 41, 2.5 lr at 1,000, 3.2 lr in the end. A gradient above 1e-3 makes
    eps = 1e-8 change the step by 1e-5 of lr, parameters of up to 5 are rounded by 2^-22, so 1e-5 = 0.001 lr is asked for."""
    for n in (12, 1000, 5000):
        always, late = values(300, 1), values(n, 2)
        g_always, g_late = values(300, 3), values(n, 4, 0.01)
        opt = st.AdamW([always, late], [g_always, None], lr=1e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(40):
            opt.step()
        assert torch.equal(late, values(n, 2))
        opt.set_grads([g_always, g_late])
        fresh = st.AdamW([values(n, 2)], [g_late], lr=1e-2, weight_decay=0.0, state_bits=bits)
        start = late.clone()
        for k in range(3):
            opt.step(), fresh.step()
            assert all(torch.equal(a, b) for a, b in zip(state(opt, 1), state(fresh, 0)))
            if k == 0:
                used = g_late.abs() > 1e-3
                assert ((late - start).abs() - 1e-2).abs()[used].max() < 1e-5
        whole = st.AdamW([values(300, 1)], [g_always], lr=1e-2, weight_decay=0.0, state_bits=bits)
        for _ in range(43):
            whole.step()
        assert all(torch.equal(a, b) for a, b in zip(state(opt, 0), state(whole, 0)))


@pytest.mark.parametrize("bits", [32, 8])
def test_tensors_that_come_and_go(st, bits):
    """Every tensor of a list takes part in some of the steps; each has the bits of its own optimizer that made those steps alone. Then the run goes on in a new optimizer from moments, step_count and missed."""
    sizes = [1, 12, 127, 130, 3000, 5001] + [20 + i for i in range(60)]
    G = [values(n, 100 + i, 0.1) for i, n in enumerate(sizes)]
    opt = st.AdamW([values(n, i) for i, n in enumerate(sizes)], [None] * len(sizes), lr=1e-2, state_bits=bits)
    alone = [st.AdamW([values(n, i)], [G[i]], lr=1e-2, state_bits=bits) for i, n in enumerate(sizes)]
    for step in range(7):
        if step == 4:
            opt2 = st.AdamW(opt.params, [None] * len(sizes), lr=1e-2, moments=opt.moments)
            opt2.step_count = opt.step_count
            opt2.missed[:] = opt.missed
            opt = opt2
        here = [(i * 7 + step * 3) % 4 != 0 for i in range(len(sizes))]
        opt.set_grads([g if h else None for g, h in zip(G, here)])
        opt.step()
        for i, h in enumerate(here):
            if h:
                alone[i].step()
    assert opt.step_count == 7
    for i in range(len(sizes)):
        assert 7 - opt.missed[i] == alone[i].step_count
        assert all(torch.equal(a, b) for a, b in zip(state(opt, i), state(alone[i], 0))), i


def test_missed_is_set_like_step_count(pkg, st):
    """Setting the counts sets what the steps go by, from a list or from another optimizer's, which stay apart from then on."""
    def make():
        return st.AdamW([values(40, 1), values(50, 2)], [values(40, 3), values(50, 4)], lr=1e-2)
    a, b = make(), make()
    a.step_count, a.missed = 10, [0, 7]
    b.step_count, b.missed = 10, a.missed
    a.set_grads([a.grads[0], None])
    a.step()
    assert a.missed.tolist() == [0, 8] and b.missed.tolist() == [0, 7]
    b.step()
    one = st.AdamW([values(50, 2)], [values(50, 4)], lr=1e-2)
    one.step_count = 3
    one.step()
    assert torch.equal(b.params[1], one.params[0]) and torch.equal(a.params[0], b.params[0]) and torch.equal(a.params[1], values(50, 2))
    for bad in ([1], [0, -1], 3, [0, 1 << 31], [[0, 0]]):
        with pytest.raises(RuntimeError, match="missed"):
            b.missed = bad
    assert b.missed.tolist() == [0, 7]
    b.missed[:] = 11                      # as many as there were steps: the next one is the first
    b.step()
    b.missed[1] = 13
    with pytest.raises(Exception, match="missed"):
        b.step()
    assert b.step_count == 12
