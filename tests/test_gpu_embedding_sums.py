"""How exact the sums of the embedding's gradient are.

A row's sum is held in two floats: every addition to the first is followed by what it rounded off (Knuth's two-sum, exact), which is added to the second in float32. With U = 2^-24, S the sum of
the magnitudes of a row's addends and K the most additions that one of them goes through, the roundings that the second float gathers are at most K U S together, and D additions in float32 lose
at most D U of that: D K U^2 S. The result (first + second) * scale is then rounded once, and its products lose U^2 (K + 3) S more (the scale is in two floats as well).

Here n <= 20,011: a group of lanes adds at most 128 lookups one after the other, its sum is joined with those of at most 128 groups by halves (7) and of one neighbour (1), and the stretches, at
most 20 of 1,024 lookups, one after the other: K <= 156. A join adds to the second float twice: D <= 128 + 2 * 28 = 184. D K + K + 3 < 3e4. With `accumulate` one more addition of the same kind, whose
addend is the old value. So the result is off by U of itself and 3e4 U^2 = 0.0018 U of the magnitudes' sum; sums in plain float32 are off by hundreds of U of the magnitudes' sum here."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu
U = 2.0 ** -24
SECOND = 3e4 * U * U
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}


def allowed(want, size):
    return U * want.abs() + SECOND * size + 2.0 ** -147   # and whole multiples of 2^-149 below the normal numbers


def sums(v, index, rows, scale, base=None):
    """Sum times scale and sum of magnitudes in 64 bits (off by 20,011 * 2^-53 of the magnitudes, a thousandth of SECOND)."""
    inside = (index >= 0) & (index < rows)
    x = v.reshape(-1, v.shape[-1])[inside].double()
    want = torch.zeros(rows, v.shape[-1], device="cuda", dtype=torch.float64).index_add_(0, index[inside].long(), x) * scale
    size = torch.zeros_like(want).index_add_(0, index[inside].long(), x.abs()) * abs(scale)
    if base is not None:
        want, size = want + base.double(), size + base.double().abs()
    return want, size


def lookups(n, rows, kind, seed):
    gen = torch.Generator().manual_seed(seed)
    i = torch.randint(rows, (n,), generator=gen)
    if kind == "one":
        i[:] = rows // 2
    if kind == "outside":
        i[torch.rand(n, generator=gen) < 0.3] = -1
        i[torch.rand(n, generator=gen) < 0.1] = rows
    return i.to(torch.int32).cuda()


def gradients(n, width, dtype, kind, seed, offset):
    """normal: of one size. large: one in 500 is 2^13 times the others (what plain sums lose is then the others' last places). cancel: those come in pairs of opposite sign, first and last."""
    gen = torch.Generator().manual_seed(seed)
    x = torch.randn(n, width, generator=gen)
    if kind != "normal":
        x[::500] = x[::500].sign() * 2.0 ** 13
    if kind == "cancel":
        x[::500] = 2.0 ** 13
        x[n - 1 - torch.arange(0, n, 500)] = -2.0 ** 13
    flat = torch.empty(n * width + offset, dtype=dtype, device="cuda")[offset:]
    flat.copy_(x.reshape(-1).to(dtype))
    return flat.view(n, width)


@pytest.mark.parametrize("width", [1, 3, 4, 9, 24, 45, 64, 113, 300, 388, 513])
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_sums_are_those_of_twice_the_bits(pkg, dtype, width):
    ops = pkg.ops
    for n, rows, where in ((1, 1, "any"), (65, 90, "outside"), (129, 5, "any"), (1500, 1, "one"), (5000, 37, "any"), (5000, 3000, "outside"), (20011, 3, "any"), (20011, 7, "one")):
        index = lookups(n, rows, where, n)
        order = ops.embedding_sort(index, rows)
        for kind in ("normal", "large", "cancel"):
            for offset in (0, 1):
                v = gradients(n, width, DTYPES[dtype], kind, n + width, offset)
                for scale in (1.0, 1.7):
                    got = ops.embedding_bwd(v, order, scale)
                    want, size = sums(v, index, rows, scale)
                    assert ((got.double() - want).abs() <= allowed(want, size)).all(), (n, kind, offset, scale)
                    base = torch.randn(rows, width, generator=torch.Generator().manual_seed(3)).cuda()
                    added = ops.embedding_bwd(v, order, scale, out=base.clone(), accumulate=True)
                    want, size = sums(v, index, rows, scale, base)
                    assert ((added.double() - want).abs() <= allowed(want, size)).all(), (n, kind, offset, scale, "accumulate")
                    assert torch.equal(got, ops.embedding_bwd(v, order, scale))


@pytest.mark.parametrize("big", [1e6, 1e9])
def test_large_gradients_that_cancel(pkg, big):
    """[B, 1000 normals, -B]: what is left is the sum of the normals, as exact as twice the bits beside B allow."""
    for width in (1, 16, 45):
        v = torch.randn(1002, width, generator=torch.Generator().manual_seed(1)).cuda()
        v[0], v[-1] = big, -big
        index = torch.zeros(1002, dtype=torch.int32, device="cuda")
        got = pkg.ops.embedding_bwd(v, pkg.ops.embedding_sort(index, 1))
        want, size = sums(v, index, 1, 1.0)
        assert ((got.double() - want).abs() <= allowed(want, size)).all()
        # of the two floats the first alone would be off by the last place of B: 2^-24 B for every lookup
        assert ((got.double() - want).abs().max() < U * big)


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("scale", [1.0, 1.7, -0.3, 0.5 * 45 ** 0.5, 1e-3, 2.0 ** 40 / 3])
def test_scale_and_sum_are_rounded_once(pkg, dtype, scale):
    """Rows of one to four lookups against the product of their exact sum with the scale as given: half a last place, and 2^-10 of one for what two floats cut off (2^-48 of sum and scale each, against a last
    place of 2^-24 at the least)."""
    ops = pkg.ops
    n, rows = 5000, 2000
    index = torch.cat([torch.arange(rows), torch.randint(rows, (n - rows,), generator=torch.Generator().manual_seed(1))]).to(torch.int32).cuda()
    v = gradients(n, 45, DTYPES[dtype], "normal", 2, 0)
    v.abs_()                                     # nothing cancels
    got = ops.embedding_bwd(v, ops.embedding_sort(index, rows), scale).cpu().numpy()
    want = sums(v, index, rows, scale)[0].cpu().numpy()
    place = np.spacing(np.abs(want).astype(np.float32)).astype(np.float64)
    assert (np.abs(got - want) <= (0.5 + 2.0 ** -10) * place).all()
