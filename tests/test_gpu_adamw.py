"""AdamW over many tensors (lfs_adamw_step_tensors) and its 8-bit moments against the formula in 64 bits, and the optimizers built on it.

Tolerances. U = 2^-24 is the most that one rounding to float32 is off, relative to the value. With b1 m and (1 - b1) g of any signs the first moment has three
products, one sum and the rounded constants, so it is off by at most 6 U (|b1 m| + |(1 - b1) g|); the second moment has no cancellation: 8 U. The step
lr mh / (sqrt(vh) + eps) adds a square root, two products, a sum, a quotient and the rounded constants: 10 U of the step besides the error of m over the same
denominator and half of v's. The parameter is rounded three times.

8-bit codes follow the definition exactly: x = |value| top / most, its last place p, floor(x / p + threshold) p. In 32 bits x / p (at most 16) is off by
16 times the relative error of the value and of three roundings, so a code may differ from the one computed in 64 bits only where x / p + threshold is that near a
whole number."""
import importlib

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
B1, B2 = 0.9, 0.999
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def st(pkg):
    return pkg.strategy


def tensor(n, offset=0, dtype=torch.float32, scale=1.0, seed=0, device="cuda"):
    """n random elements, `offset` elements behind an aligned address."""
    gen = torch.Generator().manual_seed(seed * 1000 + n % 1000 + offset)
    whole = torch.randn(n + offset, generator=gen) * scale
    return whole.to(dtype).to(device)[offset:]


def thresholds(n, t, bits):
    i = np.arange(n, dtype=np.uint64)
    first, second = (0x91E10DA5, 0x9E3779B9) if bits == 20 else (0x9E3779B9, 0xC13FA9A9)
    h = (i * np.uint64(first) + np.uint64(t * second % 2 ** 32)) % np.uint64(2 ** 32)
    return (h >> np.uint64(32 - bits)).astype(np.float64) / 2.0 ** bits


def f64(t):
    return t.detach().cpu().double().numpy()


def decode(codes, scales):
    s = np.repeat(f64(scales), 128)[: codes.numel()]
    return f64(codes.float()) * s


def check_codes(codes, scales, value, error, t, second):
    """Codes and scales against the definition. value: the moment in 64 bits; error: how far the kernel's may be from it."""
    n = value.size
    top, bits, lowest, fraction = (57344.0, 21, -14, 2) if second else (448.0, 20, -6, 3)
    pad = -n % 128
    most = np.pad(np.abs(value), (0, pad)).reshape(-1, 128).max(1)
    most_error = np.pad(error, (0, pad)).reshape(-1, 128).max(1)
    got = f64(scales)
    held = most >= 2.0 ** -110
    assert np.all(np.abs(got - np.where(held, most / top, 0)) <= (most_error + 3 * U * most) / top + 1e-45)
    assert np.all(got[~held] == 0)
    most, most_error, held = (np.repeat(x, 128)[:n] for x in (most, most_error, held))
    safe = np.where(held, most, 1.0)
    x = np.abs(value) * top / safe
    place = 2.0 ** (np.maximum(np.floor(np.log2(np.maximum(x, 1e-300))), lowest) - fraction)
    q = x / place + thresholds(n, t, bits)
    want = np.minimum(np.floor(q) * place, top)
    if second:
        want = np.where((value > 0) & held, np.maximum(want, 2.0 ** (lowest - fraction)), want)
    want = np.where(held, want, 0)
    have = np.abs(f64(codes.float()))
    off = (error * top / safe + x * (most_error / safe + 4 * U)) / place + 2.0 ** -20   # the lowest codes: one more rounding of 2^-24 of their start
    near = np.abs(q - np.round(q)) <= off
    wrong = (have != want) & ~near
    assert not wrong.any(), (np.flatnonzero(wrong)[:5], have[wrong][:5], want[wrong][:5])
    assert np.all(np.abs(have - want)[near] <= 2 * place[near])     # next code at the most (the place doubles at a binade)
    if not second:
        assert np.all(np.sign(f64(codes.float()))[have > 0] == np.sign(value)[have > 0])
    return near


class Model:
    """One tensor's AdamW in 64 bits, from the moments that the 8-bit form holds."""

    def __init__(self, p, lr, wd, eps):
        self.p, self.lr, self.wd, self.eps = f64(p), lr, wd, eps
        self.m = np.zeros_like(self.p)
        self.v = np.zeros_like(self.p)

    def step(self, g, t):
        lr, wd = np.float64(np.float32(self.lr)), np.float64(np.float32(self.wd))
        em = 6 * U * (np.abs(B1 * self.m) + np.abs((1 - B1) * g))
        self.m = B1 * self.m + (1 - B1) * g
        self.v = B2 * self.v + (1 - B2) * g * g
        ev = 8 * U * self.v + 1e-44
        with np.errstate(over="ignore", invalid="ignore", divide="ignore"):
            denominator = np.sqrt(self.v / (1 - B2 ** t)) + self.eps
            step = lr / (1 - B1 ** t) * self.m / denominator
            # products and sums below the smallest normal number are off by its last place instead
            ep = 4 * U * np.abs(self.p) + 10 * U * np.abs(step) + lr / (1 - B1 ** t) * (em + 1e-44) / denominator + 8 * U * np.abs(step) + 1e-44
        self.p = self.p * (1 - lr * wd) - step
        return em + 1e-44, ev, ep


SIZES = [1, 3, 31, 127, 128, 129, 1000, 20011]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("grad", list(DTYPES))
@pytest.mark.parametrize("offset", [0, 1])
def test_step_against_the_formula(st, bits, grad, offset):
    lrs = [1e-3 * (1 + i) for i in range(len(SIZES))]
    wds = [0.0 if i % 2 else 0.1 for i in range(len(SIZES))]
    P = [tensor(n, offset, seed=1) for n in SIZES]
    G = [tensor(n, offset, DTYPES[grad], 0.01, seed=2) for n in SIZES]
    models = [Model(p, lr, wd, 1e-8) for p, lr, wd in zip(P, lrs, wds)]
    opt = st.AdamW(P, G, lr=lrs, eps=1e-8, weight_decay=wds, state_bits=bits)
    for t in range(1, 5):
        for k, g in enumerate(G):
            g.copy_(tensor(SIZES[k], 0, DTYPES[grad], 0.01 * 10.0 ** (-t), seed=10 * t + k))
            g[: SIZES[k] // 3] = 0
        opt.step(grad_scale=0.5)
        for k, (p, g, model, held) in enumerate(zip(P, G, models, opt.moments)):
            em, ev, ep = model.step(f64(g) * 0.5, t)
            assert np.all(np.abs(f64(p) - model.p) <= ep), (k, t)
            if bits == 32:
                assert np.all(np.abs(f64(held.exp_avg) - model.m) <= em) and np.all(np.abs(f64(held.exp_avg_sq) - model.v) <= ev)
                model.m, model.v = f64(held.exp_avg), f64(held.exp_avg_sq)
            else:
                check_codes(held.exp_avg, held.exp_avg_scale, model.m, em, t, False)
                check_codes(held.exp_avg_sq, held.exp_avg_sq_scale, model.v, ev, t, True)
                model.m, model.v = decode(held.exp_avg, held.exp_avg_scale), decode(held.exp_avg_sq, held.exp_avg_sq_scale)
            model.p = f64(p)


def test_nothing_outside_the_tensors_is_touched(st):
    """Tensors that end inside a block, inside a vector, with other data right behind them."""
    for n in (1, 2, 5, 127, 130, 1021):
        flat = [torch.full((n + 8,), 7.0, device="cuda") for _ in range(2)]
        codes = [torch.full((n + 8,), 0x55, dtype=torch.uint8, device="cuda") for _ in range(2)]
        scales = [torch.full((-(-n // 128) + 1,), 3.0, device="cuda") for _ in range(2)]
        m = st.Moments(codes[0][:n].view(torch.float8_e4m3fn), codes[1][:n].view(torch.float8_e5m2), scales[0][:-1], scales[1][:-1])
        opt = st.AdamW([flat[0][:n]], [flat[1][:n]], moments=[m], lr=0.1)
        opt.step()
        assert flat[0][n:].eq(7).all() and flat[1].eq(7).all() and not flat[0][:n].eq(7).any()
        assert all(c[n:].eq(0x55).all() for c in codes) and all(float(s[-1]) == 3 for s in scales)


@pytest.mark.parametrize("bits", [32, 8])
def test_many_tensors_are_as_one_by_one(st, bits):
    """More tensors than one launch takes, empty ones and ones without a gradient among them: bit for bit what single steps give."""
    sizes = [(7 * i) % 41 for i in range(900)] + [5000]
    def make():
        P = [tensor(n, 0, seed=i) for i, n in enumerate(sizes)]
        G = [None if i % 13 == 5 else tensor(n, 0, scale=0.1, seed=i + 5000) for i, n in enumerate(sizes)]
        return P, G
    P, G = make()
    opt = st.AdamW(P, G, lr=[1e-3 * (1 + i % 5) for i in range(len(sizes))], state_bits=bits)
    opt.step(), opt.step()
    Q, H = make()
    for i in range(len(sizes)):
        one = st.AdamW([Q[i]], [H[i]], lr=1e-3 * (1 + i % 5), state_bits=bits)
        one.step(), one.step()
        assert torch.equal(P[i], Q[i])
        for a, b in ((opt.moments[i].exp_avg, one.moments[0].exp_avg), (opt.moments[i].exp_avg_sq, one.moments[0].exp_avg_sq)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))
    before = [p for p, g, n in zip(make()[0], G, sizes) if g is None and n]
    after = [p for p, g, n in zip(P, G, sizes) if g is None and n]
    assert all(torch.equal(a, b) for a, b in zip(before, after))


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [32, 33, 100, 128, 129, 424, 425])
def test_each_length_of_list_is_as_one_by_one(st, bits, count):
    """The lengths at which a launch takes other arguments: bit for bit what single steps give."""
    sizes = [1 + (13 * i) % 331 + (4096 if i % 50 == 31 else 0) for i in range(count)]
    def make():
        return [tensor(n, 0, seed=i) for i, n in enumerate(sizes)], [tensor(n, 0, scale=0.1, seed=i + 5000) for i, n in enumerate(sizes)]
    P, G = make()
    opt = st.AdamW(P, G, lr=[1e-3 * (1 + i % 5) for i in range(count)], weight_decay=0.01, state_bits=bits)
    opt.step(), opt.step()
    Q, H = make()
    for i in range(count):
        one = st.AdamW([Q[i]], [H[i]], lr=1e-3 * (1 + i % 5), weight_decay=0.01, state_bits=bits)
        one.step(), one.step()
        assert torch.equal(P[i], Q[i])
        for a, b in ((opt.moments[i].exp_avg, one.moments[0].exp_avg), (opt.moments[i].exp_avg_sq, one.moments[0].exp_avg_sq)):
            assert torch.equal(a.view(torch.uint8), b.view(torch.uint8))


def test_gradients_that_are_not_finite_stay_with_their_elements(st):
    n = 1000
    for bits in (32, 8):
        P, G = tensor(n, seed=3), tensor(n, seed=4)
        clean, grads = P.clone(), G.clone()
        bad = {0: float("nan"), 200: float("inf"), 999: float("-inf")}
        for i, x in bad.items():
            G[i] = x
            grads[i] = 0.0
        a, b = st.AdamW([P], [G], lr=0.1, state_bits=bits), st.AdamW([clean], [grads], lr=0.1, state_bits=bits)
        a.step(), b.step()
        rest = torch.ones(n, dtype=torch.bool, device="cuda")
        rest[list(bad)] = False
        assert torch.equal(P[rest], clean[rest]) and not torch.isfinite(P[~rest]).any()
        if bits == 8:
            ma, mb = a.moments[0], b.moments[0]
            assert torch.equal(ma.exp_avg.view(torch.uint8)[rest], mb.exp_avg.view(torch.uint8)[rest]) and torch.equal(ma.exp_avg_scale, mb.exp_avg_scale)
            assert torch.equal(ma.exp_avg_sq.view(torch.uint8)[rest], mb.exp_avg_sq.view(torch.uint8)[rest]) and torch.equal(ma.exp_avg_sq_scale, mb.exp_avg_sq_scale)
            assert ma.exp_avg[~rest].float().isnan().all()
            held = ma.exp_avg_sq.float()
            assert held[0].isnan() and held[200].isinf() and held[999].isinf()


def test_no_gradient_no_step(st):
    """Zero gradients from a fresh state: the parameters only decay, and the moments stay zero."""
    for bits in (32, 8):
        P = tensor(300, seed=5)
        want = (P * np.float32(1 - float(np.float32(0.1)) * float(np.float32(0.5)))).clone()
        opt = st.AdamW([P], [torch.zeros_like(P)], lr=0.1, weight_decay=0.5, state_bits=bits)
        opt.step()
        assert torch.equal(P, want)
        assert not opt.moments[0].exp_avg.view(torch.uint8).any() and not opt.moments[0].exp_avg_sq.view(torch.uint8).any()


def test_small_and_large_blocks(st):
    """A block below the smallest scale is held as zeros, one far above it next to it is not touched by that; no second moment above zero becomes zero."""
    n = 512
    G = torch.full((n,), 1e-30, device="cuda")     # second moments of 1e-63: zero in 32 bits
    G[128:256] = 1e-13                             # 1e-29, above 2^-110
    G[128] = 1e3                                   # and its block's largest 1e3: the others are 2^-106 of it
    G[256:] = 1.0
    P = torch.zeros(n, device="cuda")
    opt = st.AdamW([P], [G], lr=1.0, eps=1e-15, weight_decay=0.0, state_bits=8)
    opt.step()
    m = opt.moments[0]
    scales = m.exp_avg_sq_scale.cpu()
    assert scales[0] == 0 and scales[1] > 0 and scales[2] == scales[3] > 0
    codes = m.exp_avg_sq.view(torch.uint8)
    assert codes[:128].eq(0).all() and codes[129:256].eq(1).all() and codes[256:].eq(0x7B).all()
    for _ in range(20):
        opt.step()
    assert torch.isfinite(P).all() and P.abs().max() < 25      # a step is at most about lr


@pytest.mark.parametrize("start", [0.25, 4.0])
def test_moments_in_8_bits_follow_slow_changes(st, start):
    """A constant gradient and a second moment of a quarter (four times) its square: each step moves it by at most 0.3 % while the codes are 12 to 25 %
    apart. After 2000 steps the moment in 64 bits is within 0.135 of (1, start) of its end. Held values lie up to a code's distance (25 %) to either side; over 4096 elements
    with spread thresholds the mean is off by 25 % / sqrt(4096) = 0.4 % if they were independent; 10 % is asked for. Nearest codes would stay where they are."""
    n = 4096
    gen = torch.Generator().manual_seed(11)
    g = (torch.rand(n, generator=gen) + 0.5).cuda()
    v0 = (g * g * start)
    codes, scales = importlib.import_module("lichtfeld-studio_b200").ops.adamw_state_encode(v0, True)
    m = st.Moments.zeros(n, 8, "cuda")
    m.exp_avg_sq, m.exp_avg_sq_scale = codes, scales
    first = decode(codes, scales)
    opt = st.AdamW([torch.zeros(n, device="cuda")], [g], lr=1e-3, weight_decay=0.0, moments=[m])
    for _ in range(2000):
        opt.step()
    want = f64(g) ** 2 + (first - f64(g) ** 2) * B2 ** 2000
    ratio = decode(codes, scales) / want
    assert abs(ratio.mean() - 1) < 0.1 and np.abs(ratio - 1).max() < 0.8
    assert abs(decode(m.exp_avg, m.exp_avg_scale).mean() / f64(g).mean() - 1) < 0.02


def test_encode_and_decode(pkg):
    ops = pkg.ops
    for n in (1, 127, 129, 5000):
        x = tensor(n, seed=6) * torch.exp(tensor(n, seed=7) * 3)
        for second in (False, True):
            y = x.abs() if second else x
            codes, scales = ops.adamw_state_encode(y, second)
            back = ops.adamw_state_decode(codes, scales)
            want = decode(codes, scales)
            assert np.all(np.abs(f64(back) - want) <= U * np.abs(want))
            # nearest: half a place of the binade (2^-3 or 2^-2 of the value), or of the lowest one, of the block's largest over the top
            top, fraction, lowest = (57344.0, 2, -14) if second else (448.0, 3, -6)
            most = np.repeat(np.pad(np.abs(f64(y)), (0, -n % 128)).reshape(-1, 128).max(1), 128)[:n]
            place = np.maximum(np.abs(f64(y)) * 2.0 ** -fraction, most / top * 2.0 ** (lowest - fraction))
            floor = most / top * 2.0 ** (lowest - fraction) if second else 0   # what is not zero is not held as zero
            assert np.all(np.abs(f64(back) - f64(y)) <= np.maximum(0.5 * place, floor) * (1 + 1e-5))
            again, scales2 = ops.adamw_state_encode(back, second)
            assert torch.equal(again.view(torch.uint8), codes.view(torch.uint8))
    empty = torch.empty(0, device="cuda")
    assert ops.adamw_state_decode(*ops.adamw_state_encode(empty)).numel() == 0


@pytest.mark.parametrize("bits", [32, 8])
def test_repeats_bit_for_bit_on_other_streams_and_in_graphs(st, bits):
    n = 70001
    def make():
        return st.AdamW([tensor(n, seed=1), tensor(33, 1, seed=2)], [tensor(n, seed=3), tensor(33, 1, seed=4)], lr=0.01, state_bits=bits)
    def state(o):
        return [x.view(torch.uint8) for p, m in zip(o.params, o.moments) for x in (p, m.exp_avg, m.exp_avg_sq, m.exp_avg_scale, m.exp_avg_sq_scale) if x is not None]
    a, b, c = make(), make(), make()
    for _ in range(3):
        a.step()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(3):
            b.step()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(x, y) for x, y in zip(state(a), state(b)))
    # a captured step repeats its own step number
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.step()
    graph.replay(), graph.replay()
    d = make()
    d.step()
    d.step_count = 0
    d.step()
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(state(c), state(d)))


# ---- the six groups ---------------------------------------------------------------------------------
def scene(pkg, n, K=16, capacity=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    model = pkg.trainer.SplatData(n, K, torch.device("cuda"), capacity)
    for name in pkg.trainer.PARAM_NAMES:
        model.tensor(name).copy_(torch.randn(model.tensor(name).shape, generator=gen))
    return model


def test_fused_adamw_without_decay_is_fused_adam(pkg, st):
    """32 bits and no decay: FusedAdam's update up to roundings (a few U of the values and of the step)."""
    n, lrs = 1003, [1e-3 * (i + 1) for i in range(6)]
    out = []
    for kind in (st.FusedAdam, st.FusedAdamW):
        model, grads = scene(pkg, n), scene(pkg, n, seed=1)
        opt = kind(model, lrs)
        for it in (5, 1500, 1501):
            opt.step(it, grads, 0.3)
        out.append((model, opt))
    (a, oa), (b, ob) = out
    for name in pkg.trainer.PARAM_NAMES:
        assert (a.tensor(name) - b.tensor(name)).abs().max() <= 3 * 8 * U * (a.tensor(name).abs().max() + 6e-3)
        for x, y in ((oa.exp_avg, ob.exp_avg), (oa.exp_avg_sq, ob.exp_avg_sq)):
            # FusedAdam forms 1 - beta from the rounded beta: 2^-25 / (1 - beta2) = 3e-5 of the second moment
            assert (x.tensor(name) - y.tensor(name)).abs().max() <= 4e-5 * x.tensor(name).abs().max()
    assert oa.step_count == ob.step_count == 3


def test_fused_adamw_8_bits_is_adamw_of_the_groups(pkg, st):
    n, lrs, wds = 1003, [1e-3 * (i + 1) for i in range(6)], [0.0, 0.1, 0.2, 0.0, 0.0, 0.3]
    model, grads = scene(pkg, n, 4, capacity=1200), scene(pkg, n, 4, capacity=1200, seed=1)
    copy, names = scene(pkg, n, 4), pkg.trainer.PARAM_NAMES
    opt = st.FusedAdamW(model, lrs, weight_decay=wds, state_bits=8)
    one = st.AdamW([copy.tensor(x) for x in names], [grads.tensor(x) for x in names], lr=lrs, eps=1e-15, weight_decay=wds, state_bits=8)
    for _ in range(3):
        opt.step(2000, grads)
        one.step()
    for i, name in enumerate(names):
        assert torch.equal(model.tensor(name), copy.tensor(name))
        assert torch.equal(opt.exp_avg.live(name)[0].view(torch.uint8), one.moments[i].exp_avg.view(torch.uint8).view(-1))
        assert torch.equal(opt.exp_avg_sq.live(name)[1], one.moments[i].exp_avg_sq_scale)
    before = model.tensor("shN").clone()
    opt.step(1000, grads)          # the reference leaves shN out up to iteration 1000
    assert torch.equal(model.tensor("shN"), before)
    with pytest.raises(RuntimeError, match="all rows"):
        opt.step(2000, grads, first_row=5)


def test_mcmc_with_8_bit_moments(pkg, st):
    """Relocation clears the moments at the sampled rows, adding clears those of the new rows, removal keeps the others' values to a rounding."""
    n = 400
    model = scene(pkg, n, 4, capacity=500)
    model.tensor("opacity_raw")[::10] = -20.0     # dead
    s = st.MCMC(model)
    s.initialize(st.OptimizationParameters(max_cap=500, optimizer="adamw", weight_decay=(0, 0, 0.1, 0, 0, 0), state_bits=8, sh_degree=1))
    opt = s._optimizer
    s.grads.flat.copy_(scene(pkg, n, 4, capacity=500, seed=2).flat)
    s.step(2000)
    before = {k: opt.exp_avg.tensor(k) for k in pkg.trainer.PARAM_NAMES}
    sampled = torch.tensor([3, 7, 7, 100] * 10, device="cuda")
    assert s.relocate_gs(sampled) == 40
    rows = s._sampled[:40].unique()
    keep = torch.ones(n, dtype=torch.bool, device="cuda")
    keep[rows] = False
    for k in before:
        now = opt.exp_avg.tensor(k)
        assert now[rows].eq(0).all() and torch.equal(now[keep], before[k][keep]), k
        assert opt.exp_avg_sq.tensor(k)[rows].eq(0).all()
    new = s.add_new_gs(torch.arange(20, device="cuda"))
    more = int(np.float32(1.05) * np.float32(n))   # 419: 1.05 in float32 lies below 1.05
    assert new == more - n == 19 and opt.exp_avg.tensor("means").shape[0] == more and opt.exp_avg.size == more
    for k in before:
        assert opt.exp_avg.tensor(k)[400:].eq(0).all() and opt.exp_avg_sq.tensor(k)[400:].eq(0).all()
    held = {k: opt.exp_avg.tensor(k).clone() for k in before}
    mask = torch.zeros(more, dtype=torch.bool, device="cuda")
    mask[5::7] = True
    s.remove_gaussians(mask)
    for k in held:
        a, b = opt.exp_avg.tensor(k), held[k][~mask]
        # rows change blocks: nearest codes of another scale, half of 2^-3 of the value, and half the lowest place of the largest
        assert ((a - b).abs() <= b.abs() / 16 + held[k].abs().max() / 448 * 2.0 ** -10 + 1e-30).all(), k
    s._grads_valid = True
    s.grads.size = model.size
    s.step(2001)
    assert torch.isfinite(model.flat).all()
    with pytest.raises(RuntimeError, match="all rows"):
        s._optimizer.step(2001, s.grads, rasterizer=object())


def test_default_strategy_with_8_bit_moments(pkg, st):
    n = 300
    model = scene(pkg, n, 4, capacity=400)
    s = st.DefaultStrategy(model)
    p = st.DefaultStrategy.Parameters(optimizer="adamw", state_bits=8, sh_degree=1)
    s.initialize(p)
    s.grads.flat.copy_(scene(pkg, n, 4, capacity=400, seed=2).flat)
    s.step(2000)
    chosen = torch.zeros(n, dtype=torch.bool, device="cuda")
    chosen[::10] = True
    held = s._optimizer.exp_avg.tensor("scaling_raw")
    s.duplicate(chosen)
    m = s._optimizer.exp_avg.tensor("scaling_raw")
    assert model.size == 330 and m.shape == (330, 3) and m[300:].eq(0).all()
    assert ((m[:300] - held).abs() <= held.abs() / 16 + held.abs().max() / 448 * 2.0 ** -10).all()
    chosen = torch.zeros(330, dtype=torch.bool, device="cuda")
    chosen[:5] = True
    s.split(chosen)
    s.remove(torch.arange(model.size, device="cuda") % 3 == 0)
    s.reset_opacity()
    assert s._optimizer.exp_avg.tensor("opacity_raw").eq(0).all() and s._optimizer.exp_avg_sq.tensor("opacity_raw").eq(0).all()
    s.step(2001)
    assert torch.isfinite(model.flat[: 1]).all()


def test_checkpoint_of_8_bit_moments_resumes_bit_for_bit(pkg, st, tmp_path):
    fm = pkg.formats
    def make(bits=8):
        model = scene(pkg, 200, 4, capacity=260)
        s = st.MCMC(model)
        s.initialize(st.OptimizationParameters(max_cap=260, optimizer="adamw", state_bits=bits, sh_degree=1))
        return s
    a, b = make(), make()
    grads = scene(pkg, 200, 4, capacity=260, seed=3)
    for it in range(2000, 2003):
        a.grads.flat.copy_(grads.flat)
        a.step(it)
    path = str(tmp_path / "run.ckpt")
    fm.save_checkpoint(a, path, 2003)
    assert fm.load_checkpoint(b, path) == 2003
    for s in (a, b):
        s.grads.flat.copy_(grads.flat)
        s.step(2003)
    assert torch.equal(a.get_model().flat, b.get_model().flat)
    for name in pkg.trainer.PARAM_NAMES:
        assert torch.equal(a._optimizer.exp_avg_sq.live(name)[0].view(torch.uint8), b._optimizer.exp_avg_sq.live(name)[0].view(torch.uint8))
    with pytest.raises(RuntimeError, match="moments in 8 bits"):
        fm.load_checkpoint(make(32), path)


@pytest.mark.parametrize("grad", list(DTYPES))
@pytest.mark.parametrize("bits", [32, 8])
def test_many_tiles_are_as_separate_tensors(st, bits, grad):
    """A tensor of several tiles for every CTA of the GPU, next to small ones: the same bits as its pieces of 128 k elements each as a tensor of its own, but for the thresholds, which go by the
    element's index in its tensor (so the comparison in 8 bits is of the parameters after the first step, which the rounding of the moments does not enter)."""
    n = (1 << 17) * 30 + 77
    P, G = tensor(n, seed=1), tensor(n, 0, DTYPES[grad], 0.1, seed=2)
    Q = P.clone()
    small = [tensor(100, seed=k) for k in range(3)]
    one = st.AdamW([small[0], P, small[1]], [small[2], G, small[2]], lr=0.01, state_bits=bits)
    one.step()
    pieces = st.AdamW(list(Q.split(1 << 17)), list(G.split(1 << 17)), lr=0.01, state_bits=bits)
    pieces.step()
    assert torch.equal(P, Q)
    if bits == 32:
        one.step(), pieces.step()
        assert torch.equal(P, Q) and torch.equal(one.moments[1].exp_avg_sq, torch.cat([m.exp_avg_sq for m in pieces.moments]))
    else:
        m = one.moments[1]
        b1m, v = 0.1 * f64(G), 0.001 * f64(G) ** 2
        check_codes(m.exp_avg, m.exp_avg_scale, b1m, 6 * U * np.abs(b1m) + 1e-44, 1, False)
        check_codes(m.exp_avg_sq, m.exp_avg_sq_scale, v, 8 * U * v + 1e-44, 1, True)


def test_two_optimizers_at_once(st):
    """Steps of different tensors on two streams, and through two captured graphs, at the same time: nothing is shared."""
    n = 300_000
    def make(seed):
        return st.AdamW([tensor(n, seed=seed)], [tensor(n, seed=seed + 1)], lr=0.01, state_bits=8)
    a, b, c, d = make(1), make(5), make(1), make(5)
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(5):
        for opt, stream in ((a, streams[0]), (b, streams[1])):
            with torch.cuda.stream(stream):
                opt.step()
    torch.cuda.synchronize()
    for _ in range(5):
        c.step(), d.step()
    for x, y in ((a, c), (b, d)):
        assert torch.equal(x.params[0], y.params[0]) and torch.equal(x.moments[0].exp_avg.view(torch.uint8), y.moments[0].exp_avg.view(torch.uint8))


def test_binding_and_refusals(st):
    P, G = tensor(50), tensor(50, seed=1)
    with pytest.raises(RuntimeError, match="overlap"):
        st.AdamW([P, P[10:]], [G, G[10:]])
    with pytest.raises(RuntimeError, match="elements"):
        st.AdamW([P], [G[:40]])
    with pytest.raises(RuntimeError, match="contiguous"):
        st.AdamW([tensor(50).view(5, 10).t()], [G])
    with pytest.raises(RuntimeError, match="grads"):
        st.AdamW([P], [G.double()])
    with pytest.raises(RuntimeError, match="for 1 tensors"):
        st.AdamW([P], [G], lr=[0.1, 0.2])
    with pytest.raises(RuntimeError, match="elements"):
        st.AdamW([P], [G], moments=[st.Moments.zeros(40, 8, P.device)])
    opt = st.AdamW([P], [None], lr=0.1)
    before = P.clone()
    opt.step()
    assert torch.equal(P, before)
    opt.set_grads([G])
    opt.step()
    assert not torch.equal(P, before) and opt.step_count == 2
    # a rate changed by a scheduler counts from the next step on
    opt.lr[0] = 0.0
    before = P.clone()
    opt.step()
    assert torch.equal(P, before)
    # the parameter's memory stays where the optimizer writes it
    q = torch.nn.Parameter(tensor(30, seed=3))
    opt = st.AdamW([q], [tensor(30, seed=4)])
    q.data = torch.zeros(30, device="cuda")
    opt.step()
    torch.cuda.synchronize()
    assert q.eq(0).all()


@pytest.mark.parametrize("grad", list(DTYPES))
def test_moments_are_rounded_operation_by_operation(st, pkg, grad):
    """m = beta1 m + (1 - beta1) g and v = beta2 v + ((1 - beta2) g) g with every product and sum rounded to float32 (no fused ones), which decides the 8-bit codes: the same bits as torch's elementary
    operations, in 32 bits and as scales and codes."""
    n = 300_000
    g = tensor(n, 0, DTYPES[grad], 0.1, seed=3)
    p32, p8 = tensor(n, seed=1), tensor(n, seed=1)
    a, b = st.AdamW([p32], [g], lr=0.01), st.AdamW([p8], [g], lr=0.01, state_bits=8)
    m = v = torch.zeros(n, device="cuda")
    m8, v8 = m.clone(), v.clone()
    for t in range(1, 4):
        gs = g.float() * 0.3
        m, v = m * 0.9 + gs * (1 - 0.9), v * 0.999 + (gs * (1 - 0.999)) * gs
        m8, v8 = m8 * 0.9 + gs * (1 - 0.9), v8 * 0.999 + (gs * (1 - 0.999)) * gs
        a.step(0.3), b.step(0.3)
        assert torch.equal(a.moments[0].exp_avg, m) and torch.equal(a.moments[0].exp_avg_sq, v)
        held = b.moments[0]
        for scale, x, top in ((held.exp_avg_scale, m8, 448.0), (held.exp_avg_sq_scale, v8, 57344.0)):
            most = torch.nn.functional.pad(x.abs(), (0, -n % 128)).view(-1, 128).amax(1)
            assert torch.equal(scale, most * torch.full_like(most, 1.0 / top))
        # without an error of the value only the quotient and the product before the threshold's sum are rounded
        check_codes(held.exp_avg, held.exp_avg_scale, f64(m8), np.zeros(n), t, False)
        check_codes(held.exp_avg_sq, held.exp_avg_sq_scale, f64(v8), np.zeros(n), t, True)
        m8, v8 = pkg.ops.adamw_state_decode(held.exp_avg, held.exp_avg_scale), pkg.ops.adamw_state_decode(held.exp_avg_sq, held.exp_avg_sq_scale)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [1e-15, 1e-8, 0.0])
def test_steps_of_very_small_second_moments(st, pkg, bits, eps):
    """Second moments of zero and below the smallest normal number next to first moments that are not zero, and very large gradients: the denominator is the formula's (2^-126 has the root 1.1e-19, which counts
    beside an eps of 1e-15)."""
    n = 512
    v0 = torch.full((n,), 1e-40, device="cuda")
    v0[:128] = 0.0
    v0[256:384] = 1.2e-38
    v0[384:] = 1e25
    if bits == 8:
        v0[128:256] = 1e-33        # just above 2^-110, below which 8 bits hold zeros
    m0 = torch.linspace(0.5, 1.0, n, device="cuda") * 1e-16
    m0[384:] = 1e11
    g = torch.zeros(n, device="cuda")
    P = torch.zeros(n, device="cuda")
    if bits == 8:
        codes = [pkg.ops.adamw_state_encode(m0), pkg.ops.adamw_state_encode(v0, True)]
        m = st.Moments(codes[0][0], codes[1][0], codes[0][1], codes[1][1])
        m0, v0 = (pkg.ops.adamw_state_decode(*c) for c in codes)
    else:
        m = st.Moments(m0.clone(), v0.clone())
    opt = st.AdamW([P], [g], lr=1e-3, eps=eps, weight_decay=0.0, moments=[m])
    opt.step_count = 99
    opt.step()
    m1, v1 = (m0 * 0.9).double(), (v0 * 0.999).double()
    v1 = v1.float().double()                       # below the normal numbers a rounding is to a whole 2^-149
    step = 1e-3 / (1 - B1 ** 100) * m1 / (torch.sqrt(v1 / (1 - B2 ** 100)) + eps)
    got, want = P.double(), -step
    held = torch.isfinite(want)
    assert torch.equal(held, torch.isfinite(got)) and held[384:].all()
    assert ((got - want).abs() <= 40 * U * want.abs())[held].all()
