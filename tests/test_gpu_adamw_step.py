"""The step of AdamW with 32-bit moments: root and division are those of float32, each rounded once."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("eps", [0.0, 1e-8, 1e-15])
def test_root_and_division_are_rounded_once(pkg, eps):
    """With beta1 = 0.5, beta2 = 0.75, t = 1 and lr = 0.5 the constants are powers of two (1 / (1 - beta1) = 2, lr times it = 1, 1 / sqrt(1 - beta2) = 2), so that from parameters of zero
    nothing but the root, the sum with eps and the quotient is rounded: -(m / (2 sqrt(v) + eps)) has the same bits as in numpy, whose float32 operations are rounded once."""
    n = 300_007
    gen = torch.Generator().manual_seed(5)
    m0 = torch.randn(n, generator=gen) * torch.exp(torch.randn(n, generator=gen) * 4)
    v0 = torch.rand(n, generator=gen) * torch.exp(torch.randn(n, generator=gen) * 8) + 1e-30
    P = torch.zeros(n, device="cuda")
    opt = pkg.strategy.AdamW([P], [torch.zeros(n, device="cuda")], lr=0.5, betas=(0.5, 0.75), eps=eps, weight_decay=0.0,
                             moments=[pkg.strategy.Moments(m0.cuda(), v0.cuda())])
    opt.step()
    m, v = opt.moments[0].exp_avg.cpu().numpy(), opt.moments[0].exp_avg_sq.cpu().numpy()
    assert np.array_equal(m, m0.numpy() * np.float32(0.5)) and np.array_equal(v, v0.numpy() * np.float32(0.75))
    want = -(m / (np.sqrt(v) * np.float32(2) + np.float32(eps)))
    assert want.dtype == np.float32 and np.array_equal(P.cpu().numpy(), want)


def nearest(x, top, dtype):
    """Values as 8-bit floats with a scale per 128 of them, rounded to the nearest."""
    scale = (x.view(-1, 128).abs().amax(1) / top).clamp_min(1e-38).repeat_interleave(128)
    return (x / scale).clamp(-top, top).to(dtype).float() * scale


def long_run(pkg, n, steps, gradient):
    """`steps` steps of AdamW with 8-bit moments from parameters of zero, the same in 64 bits, and with moments rounded to the nearest code: second moments and paths of the parameters."""
    P, G = torch.zeros(n, device="cuda"), torch.zeros(n, device="cuda")
    opt = pkg.strategy.AdamW([P], [G], lr=1.0, eps=1e-15, weight_decay=0.0, state_bits=8)
    m = torch.zeros(n, device="cuda", dtype=torch.float64)
    v, path, near_path = m.clone(), m.clone(), m.clone()
    near_m, near_v = m.float(), v.float()
    for t in range(1, steps + 1):
        G.copy_(gradient(t))
        opt.step()
        g, b1, b2 = G.double(), 1 - 0.9 ** t, 1 - 0.999 ** t
        m, v = 0.9 * m + 0.1 * g, 0.999 * v + 0.001 * g * g
        path += (m / b1) / (torch.sqrt(v / b2) + 1e-15)
        near_m, near_v = near_m * 0.9 + G * 0.1, near_v * 0.999 + (G * 0.001) * G
        near_path += ((near_m / b1) / (torch.sqrt(near_v / b2) + 1e-15)).double()
        near_m, near_v = nearest(near_m, 448.0, torch.float8_e4m3fn), nearest(near_v, 57344.0, torch.float8_e5m2)
    held = pkg.ops.adamw_state_decode(opt.moments[0].exp_avg_sq, opt.moments[0].exp_avg_sq_scale)
    off, near_off = (float((x - path).norm() / path.norm()) for x in (-P.double(), near_path))
    return (held.double() / v), (near_v.double() / v), off, near_off


def test_8_bit_moments_over_a_long_run(pkg):
    """Gradients of a signal and noise that are there in half of the steps and become five times smaller half way, over 6000 steps: the second moments in 8 bits stay where those in 64 bits are, and so does the
    parameters' path.

    A step moves a second moment by about d = 0.001 of itself, codes are s = 12 to 25 % apart, and a threshold makes it move by a whole code in d / s of the steps: a variance of d s a step, of which the
    average keeps d s / (2 * 0.001) = 0.09: +-30 % for an element whose thresholds were independent, 0.7 % for the mean of 2048 of them (10 % is asked for, which also holds what is kept above zero).
    A step goes with the inverse root: 15 % each, in the same direction for about 1000 steps (30 % is asked for)."""
    n, steps = 128 * 16, 6000
    gen = torch.Generator("cuda").manual_seed(0)
    size = torch.exp(torch.randn(n // 16, 1, device="cuda", generator=gen) * 1.5 - 9).expand(-1, 16).reshape(-1)

    def gradient(t):
        seen = torch.rand(n, device="cuda", generator=gen) < 0.5
        return (torch.randn(n, device="cuda", generator=gen) + 0.3) * size * seen * (1.0 if t < steps // 2 else 0.2)

    ratio, near, off, near_off = long_run(pkg, n, steps, gradient)
    print(f"second moment {ratio.mean():.3f} of its own (nearest codes {near.mean():.3f}), path off by {off:.3f} (nearest codes {near_off:.3g})")
    assert abs(ratio.mean() - 1) < 0.1 and off < 0.3


def test_8_bit_moments_fall_beside_a_steady_largest_one(pkg):
    """A block whose largest second moment stays where it is has a constant scale. Gradients beside it halve after 1500 steps, so their second moments should fall to a quarter: after 4500 more steps to
    (1 + 3 * 0.999^4500) / 4 = 0.26 of what they were. Each step takes 0.1 % off them at the most and codes are 12 % apart: rounded to the nearest they stay near where they were, at 3 times their values and more
    (half a code, 12 %, below 1 / 0.26 = 3.8). With the thresholds the mean over 2032 elements has the error of the test above."""
    n, steps = 128 * 16, 6000
    gen = torch.Generator("cuda").manual_seed(1)
    top = torch.arange(n, device="cuda") % 128 == 0

    def gradient(t):
        return torch.where(top, 10.0, (torch.randn(n, device="cuda", generator=gen) * 0.3 + 1) * (1.0 if t < 1500 else 0.5))

    ratio, near, off, near_off = long_run(pkg, n, steps, gradient)
    print(f"second moment {ratio[~top].mean():.3f} of its own (nearest codes {near[~top].mean():.3f}), path off by {off:.3f} (nearest codes {near_off:.3g})")
    assert abs(ratio[~top].mean() - 1) < 0.1 and off < 0.3 and near[~top].mean() > 3


def test_rows_that_have_not_been_seen_for_long(pkg):
    """First moments that 1500 steps without a gradient made smaller than any normal number (0.9^1500 = 2^-228), and second moments that never had one, next to rows that are seen: the former stay where they are,
    the latter have the bits of a tensor of their own."""
    st = pkg.strategy
    n, seen = 4096, torch.arange(4096, device="cuda") % 2 == 0
    gen = torch.Generator("cuda").manual_seed(2)
    P = torch.randn(n, device="cuda", generator=gen)
    G = torch.randn(n, device="cuda", generator=gen)
    G[1::4] = 0.0                                   # of the rows that are not seen later, half never had a gradient
    opt = st.AdamW([P], [G], lr=1e-3, eps=1e-15, weight_decay=0.0)
    opt.step()
    G[~seen] = 0.0
    for _ in range(1500):
        opt.step()
    m = opt.moments[0].exp_avg
    assert m[3::4].abs().max() < 2.0 ** -126 and m[1::4].eq(0).all() and opt.moments[0].exp_avg_sq[1::4].eq(0).all()
    one = st.AdamW([P[seen].clone()], [G[seen].clone()], lr=1e-3, eps=1e-15, weight_decay=0.0, moments=[st.Moments(m[seen].clone(), opt.moments[0].exp_avg_sq[seen].clone())])
    one.step_count = opt.step_count
    before = P.clone()
    opt.step(), one.step()
    assert torch.equal(P[~seen], before[~seen]) and torch.equal(P[seen], one.params[0])
