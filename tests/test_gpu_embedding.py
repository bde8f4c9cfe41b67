"""Embedding lookup, the order of its lookups, its gradient, and a palette trained with them.

The lookup is one product per element rounded once to float32 and once more to the output's type: elementary torch operations give the same bits. The gradient's sums have
twice float32's bits; how exact they are is tested in test_gpu_embedding_sums.py, and the gradients here are held to what sums in float32 keep: with U = 2^-24, an error of some U for every addition of the
sum of magnitudes."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


@pytest.fixture(scope="module")
def ops(pkg):
    return pkg.ops


def randn(*shape, dtype=torch.float32, seed=0, offset=0):
    gen = torch.Generator().manual_seed(seed)
    n = int(np.prod(shape))
    return torch.randn(n + offset, generator=gen).to(dtype).cuda()[offset:].view(shape)


def indices(n, rows, dtype=torch.int32, seed=0, kind="any"):
    gen = torch.Generator().manual_seed(seed + 77)
    i = torch.randint(rows, (n,), generator=gen)
    if kind == "outside" and n:
        i[torch.rand(n, generator=gen) < 0.3] = -1
        i[torch.rand(n, generator=gen) < 0.1] = rows
        i[0] = -5 if dtype == torch.int32 else -(1 << 40)
        i[-1] = 2 ** 31 - 1 if dtype == torch.int32 else 1 << 40
    if kind == "one":
        i[:] = rows // 2
    if kind == "few":
        i = torch.randint(rows, (3,), generator=gen)[torch.randint(3, (n,), generator=gen)]
    return i.to(dtype).cuda()


def lookup(table, i, scale, dtype):
    inside = (i >= 0) & (i < table.shape[0])
    rows = table.float()[torch.where(inside, i, 0).long()] * scale
    return torch.where(inside[..., None], rows, torch.zeros_like(rows)).to(dtype)


WIDTHS = [1, 3, 4, 9, 24, 45, 64, 300]


@pytest.mark.parametrize("width", WIDTHS + [4099, 8192])
@pytest.mark.parametrize("table,out", [("f32", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f16", "f16"), ("f16", "f32")])
def test_lookup(ops, width, table, out):
    for n, rows, kind in ((1, 1, "any"), (2, 5, "outside"), (257, 3, "outside"), (3001, 700, "any"), (1000, 70000 // width + 1, "few")):
        for index in (torch.int32, torch.int64):
            for offset in (0, 1):
                t = randn(rows, width, dtype=DTYPES[table], seed=n, offset=offset)
                i = indices(n, rows, index, seed=n, kind=kind)
                got = ops.embedding_fwd(t, i, 0.37, out_dtype=DTYPES[out])
                assert got.dtype == DTYPES[out] and got.shape == (n, width)
                assert torch.equal(got, lookup(t, i, np.float32(0.37), DTYPES[out]))


def test_lookup_shapes_out_and_values_that_are_not_finite(ops):
    t = randn(6, 5)
    t[2, 3], t[4, 0] = float("nan"), float("inf")
    i = torch.tensor([[0, 2], [4, -1], [7, 5]], device="cuda")
    got = ops.embedding_fwd(t, i)
    assert got.shape == (3, 2, 5) and got[0, 1, 3].isnan() and got[1, 0, 0].isinf() and got[1, 1].eq(0).all() and got[2, 0].eq(0).all()
    keep = torch.full((40,), 9.0, device="cuda")
    out = ops.embedding_fwd(t, i, out=keep[5:35])
    assert out.data_ptr() == keep[5:].data_ptr() and torch.equal(out.view(3, 2, 5)[0, 0], t[0]) and keep[:5].eq(9).all() and keep[35:].eq(9).all()
    assert ops.embedding_fwd(t, i[:0]).shape == (0, 2, 5)


def test_lookup_past_2_to_the_31_elements(ops):
    """Rows behind element 2^31 of the output."""
    t = randn(5, 1021, dtype=torch.float16, seed=3)
    n = (1 << 31) // 1021 + 1000
    i = (torch.arange(n, device="cuda", dtype=torch.int32) * 7) % 5
    got = ops.embedding_fwd(t, i)
    assert torch.equal(got[-2000:], t[i[-2000:].long()]) and torch.equal(got[:10], t[i[:10].long()])


ROWS = [1, 2, 511, 512, 513, 65536, (1 << 18) - 1, 1 << 18, 1 << 27, (1 << 31) - 2]


@pytest.mark.parametrize("rows", ROWS)
@pytest.mark.parametrize("n", [1, 31, 33, 4095, 4096, 4097, 100003])
def test_order(ops, rows, n):
    for kind in ("any", "outside", "one", "few"):
        for dtype in (torch.int32, torch.int64):
            i = indices(n, rows, dtype, seed=n, kind=kind)
            order = ops.embedding_sort(i, rows)
            key = i.long().cpu()
            key = torch.where((key >= 0) & (key < rows), key, rows)
            want, at = torch.sort(key, stable=True)
            assert torch.equal(order.sorted_rows.cpu().long(), want) and torch.equal(order.order.cpu().long(), at), (kind, dtype)


def check_gradient(v, i, rows, scale, got, base=None):
    key = i.reshape(-1).long().cpu().numpy()
    x = v.reshape(-1, v.shape[-1]).double().cpu().numpy()
    inside = (key >= 0) & (key < rows)
    want, size, count = np.zeros((rows, x.shape[1])), np.zeros((rows, x.shape[1])), np.zeros((rows, 1))
    np.add.at(want, key[inside], x[inside])
    np.add.at(size, key[inside], np.abs(x[inside]))
    np.add.at(count, key[inside], 1)
    scale = float(np.float32(scale))
    off = (64 + count / 64 + 4) * U * size * abs(scale)
    if base is not None:
        want, off = want + base.double().cpu().numpy() / scale, off + U * (np.abs(base.double().cpu().numpy()) + np.abs(want * scale))
    assert np.all(np.abs(got.double().cpu().numpy() - want * scale) <= off + 1e-44)


@pytest.mark.parametrize("width", WIDTHS + [513])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_gradient(ops, width, dtype):
    for n, rows, kind in ((1, 1, "any"), (1, 300, "any"), (63, 4, "outside"), (64, 2, "one"), (65, 90, "outside"), (128, 1, "one"), (129, 5, "few"),
                          (5000, 37, "any"), (5000, 3000, "outside"), (20011, 200, "few"), (20011, 7, "one")):
        for offset in (0, 1):
            v = randn(n, width, dtype=DTYPES[dtype], seed=n, offset=offset)
            i = indices(n, rows, torch.int64 if offset else torch.int32, seed=n + 1, kind=kind)
            order = ops.embedding_sort(i, rows)
            got = ops.embedding_bwd(v, order, 1.7)
            assert got.dtype == torch.float32 and got.shape == (rows, width)
            check_gradient(v, i, rows, 1.7, got)
            again = ops.embedding_bwd(v, order, 1.7)
            assert torch.equal(got, again)
            base = randn(rows, width, seed=5)
            added = ops.embedding_bwd(v, order, 1.7, out=base.clone(), accumulate=True)
            check_gradient(v, i, rows, 1.7, added, base)


def test_gradient_of_nothing(ops):
    i = torch.full((50,), -1, device="cuda")
    order = ops.embedding_sort(i, 9)
    out = torch.full((9, 6), 3.0, device="cuda")
    v = torch.full((50, 6), float("nan"), device="cuda")      # of lookups that name no row
    assert ops.embedding_bwd(v, order, out=out.clone(), accumulate=True).eq(3).all()
    assert ops.embedding_bwd(v, order, out=out).eq(0).all()
    empty = ops.embedding_sort(i[:0], 9)
    assert ops.embedding_bwd(v[:0], empty).eq(0).all()
    two = ops.embedding_sort(i.view(5, 10), 9)
    assert ops.embedding_bwd(v.view(5, 10, 6), two).shape == (9, 6)


def test_gradient_past_2_to_the_31_elements(ops):
    """Rows of v_out behind element 2^31."""
    width = 1021
    n = (1 << 31) // width + 64
    v = torch.zeros(n, width, dtype=torch.float16, device="cuda")
    v[-100:] = randn(100, width, dtype=torch.float16, seed=1)
    i = torch.zeros(n, dtype=torch.int32, device="cuda")
    i[-100:] = torch.arange(100, device="cuda", dtype=torch.int32) + 1
    got = ops.embedding_bwd(v, ops.embedding_sort(i, 101))
    assert torch.equal(got[1:], v[-100:].float()) and got[0].eq(0).all()


def test_gradient_against_differences(ops):
    """The lookup is linear in the table: <v, f(t + d) - f(t)> = <gradient, d>, to the roundings of its products (2 U a value) and sums."""
    t, d, v = randn(40, 45, seed=1), randn(40, 45, seed=2), randn(900, 45, seed=3)
    i = indices(900, 40, kind="outside")
    g = ops.embedding_bwd(v, ops.embedding_sort(i, 40), 0.6)
    up, down = ops.embedding_fwd(t + d, i, 0.6), ops.embedding_fwd(t, i, 0.6)
    left = (v.double() * (up.double() - down.double())).sum().item()
    right = (g.double() * d.double()).sum().item()
    size = (v.double().abs() * (up.double().abs() + down.double().abs())).sum().item() + 100 * (g.double().abs() * d.double().abs()).sum().item()
    assert abs(left - right) <= 4 * U * size


def test_streams_and_graphs(ops):
    """The same calls on another stream, captured and replayed on new values, and two graphs of their own."""
    t, i, v = randn(300, 45, seed=1), indices(20000, 300, kind="few"), randn(20000, 45, seed=2)
    def run():
        order = ops.embedding_sort(i, 300)
        return ops.embedding_fwd(t, i, 2.0), ops.embedding_bwd(v, order, 2.0)
    want = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    outs = []
    for graph in graphs:
        with torch.cuda.graph(graph):
            outs.append(run())
    t.copy_(randn(300, 45, seed=5)), v.copy_(randn(20000, 45, seed=6)), i.copy_(indices(20000, 300, seed=8))
    want = run()
    for graph in graphs:
        graph.replay()
    torch.cuda.synchronize()
    for out in outs:
        assert all(torch.equal(a, b) for a, b in zip(want, out))


def test_long_gradient(ops):
    """More lookups than a wave of CTAs takes in one round each: a row that spans many stretches next to short ones, rows without lookups, lookups that name no row at the end."""
    n, rows = 1_200_003, 70_000
    for width in (3, 16, 45):
        gen = torch.Generator(device="cuda").manual_seed(width)
        i = torch.randint(rows, (n,), device="cuda", generator=gen, dtype=torch.int32)
        i[: n // 3] = 777
        i[n // 3: n // 3 + 1000] = -1
        v = torch.randn(n, width, device="cuda", generator=gen)
        got = ops.embedding_bwd(v, ops.embedding_sort(i, rows), 1.0)
        inside = i >= 0
        want = torch.zeros(rows, width, device="cuda", dtype=torch.float64).index_add_(0, i[inside].long(), v[inside].double())
        size = torch.zeros(rows, width, device="cuda", dtype=torch.float64).index_add_(0, i[inside].long(), v[inside].double().abs())
        # two-float sums: U of the sum for its rounding, and n^2 U^2 < 0.006 U n of the magnitudes' mean is far below U / 1000 of their sum
        assert ((got.double() - want).abs() <= U * want.abs() + U / 1000 * size + 1e-44).all()


def test_infinite_gradients_stay_with_their_rows(ops):
    v = randn(1000, 9, seed=2)
    i = indices(1000, 20, kind="any")
    v[100, 3], v[200, 4] = float("inf"), float("nan")
    got = ops.embedding_bwd(v, ops.embedding_sort(i, 20), 0.5)
    bad = torch.zeros(20, 9, dtype=torch.bool, device="cuda")
    bad[i[100].long(), 3] = bad[i[200].long(), 4] = True
    assert got[i[100].long(), 3].isinf() and got[i[200].long(), 4].isnan() and torch.isfinite(got[~bad]).all()


def test_refusals(ops):
    t, i = randn(6, 5), indices(10, 6)
    for kw, message in ((dict(out=torch.empty(10, 4, device="cuda")), "hold 10 rows"), (dict(out=torch.empty(5, 10, device="cuda").t()), "contiguous"),
                        (dict(out_dtype=torch.float16), "float32"), (dict(out=torch.empty(10, 5, device="cuda"), out_dtype=torch.float16), "out")):
        with pytest.raises(RuntimeError, match=message):
            ops.embedding_fwd(t, i, **kw)
    order = ops.embedding_sort(i, 6)
    for v, kw, message in ((randn(9, 5), {}, "v_out must be"), (randn(10, 5).double(), {}, "v_out must be"), (randn(5, 10).t(), {}, "contiguous"), (randn(10, 5), dict(accumulate=True), "out"),
                           (randn(10, 5), dict(out=torch.empty(6, 4, device="cuda")), "6 rows"), (randn(10, 5), dict(out=torch.empty(6, 5, device="cuda").half()), "out must be")):
        with pytest.raises(RuntimeError, match=message):
            ops.embedding_bwd(v, order, **kw)
    for rows in (0, -3, 1 << 31):
        with pytest.raises(RuntimeError, match="bad sizes"):
            ops.embedding_sort(i, rows)


def test_palette_is_trained_with_the_scene(pkg, synth):
    """A palette of SH rows through render, loss and backward, its table and the scene's other groups updated by AdamW with 8-bit moments: the table's gradient is the
    sum of the shN gradients of each label, the run repeats bit for bit in what follows the render's atomic sums, and gradients agree with differences of the loss."""
    tr, st = pkg.trainer, pkg.strategy
    cfg = dict(synth.CONFIGS["tiny"], n=4000, W=96, H=80, fx=110.0)
    P = synth.make_gaussians(4000, 0, "cube", 1)
    poses, K = synth.make_cameras(cfg)
    dev = torch.device("cuda")
    model = tr.SplatData(4000, 4, dev).load(P)
    grads = model.like()
    gen = torch.Generator().manual_seed(4)
    labels = torch.randint(-1, 20, (4000,), generator=gen, dtype=torch.int32).cuda()
    palette = tr.ShPalette((torch.randn(20, 3, 3, generator=gen) * 0.2).cuda(), labels)
    rast, loss = tr.Rasterizer(model, 96, 80, 1), tr.PhotometricLoss(96, 80, dev)
    cam = tr.Camera(torch.from_numpy(poses[0]).to(dev), torch.from_numpy(K).to(dev), 96, 80)
    target = torch.rand(3, 80, 96, generator=gen).cuda()

    def value():
        palette.expand(model)
        return loss(rast.forward(cam, None).image, target)

    def backward():
        _, v = value()
        rast.backward(v, grads)
        return palette.backward(grads)

    g = backward().clone()
    shN = model.tensor("shN")
    inside = labels >= 0
    assert torch.equal(shN[inside], palette.table[labels[inside].long()]) and shN[~inside].eq(0).all()
    want = torch.zeros(20, 3, 3, dtype=torch.float64, device=dev).index_add_(0, labels[inside].long(), grads.tensor("shN")[inside].double())
    size = torch.zeros(20, 3, 3, dtype=torch.float64, device=dev).index_add_(0, labels[inside].long(), grads.tensor("shN")[inside].double().abs())
    assert ((g.double() - want).abs() <= 80 * U * size).all()
    # central difference of the loss along a direction; the loss is a float32 of about 0.3 (off by some U), the step changes it by about 1e-3
    d = torch.randn(20, 3, 3, generator=gen).cuda() * 0.02
    start = palette.table.clone()
    found = []
    for sign in (1, -1):
        palette.table.copy_(start + sign * d)
        found.append(float(value()[0][0]))
    palette.table.copy_(start)
    slope = (g.double() * d.double()).sum().item()
    assert abs((found[0] - found[1]) / 2 - slope) <= 0.1 * abs(slope) + 1e-6, (found, slope)

    scene = st.FusedAdamW(model, [1e-4] * 6, state_bits=8)
    table = st.AdamW([palette.table], [palette.grad], lr=1e-2, weight_decay=0.0, state_bits=8)
    for it in range(1, 6):
        backward()
        scene.step(it, grads)      # up to iteration 1000 without shN, which the palette holds
        table.step()
    assert torch.isfinite(model.flat).all() and not torch.equal(palette.table, start)
    with pytest.raises(RuntimeError, match="4000 Gaussians"):
        palette.expand(tr.SplatData(10, 4, dev))
