"""Infinite second moments in 8 bits: held as infinite in every block, those whose finite numbers are held as zeros among them."""
import pytest
import torch

pytestmark = pytest.mark.gpu
INF = float("inf")


@pytest.mark.parametrize("n", [1, 128, 300])
@pytest.mark.parametrize("rest", [0.0, 1e-37, 1e-20, 3.0])
def test_an_infinite_moment_is_decoded_as_infinite(pkg, n, rest):
    ops = pkg.ops
    x = torch.full((n,), rest, device="cuda")
    x[n // 2] = INF
    back = ops.adamw_state_decode(*ops.adamw_state_encode(x, True))
    assert back[n // 2] == INF
    others = torch.ones(n, dtype=torch.bool, device="cuda")
    others[n // 2] = False
    # the largest finite number of a block is its scale times the top code: the constant 1 / 57344, the scale's product and that of the value are rounded, 2^-24 each; below 2^-110 it is held as zero
    want = 0.0 if rest < 2.0 ** -110 else rest
    assert ((back[others] - want).abs() <= 3 * 2.0 ** -24 * want).all()
    again = ops.adamw_state_decode(*ops.adamw_state_encode(back, True))
    assert again[n // 2] == INF and ((again - back).abs()[others] <= 3 * 2.0 ** -24 * back[others]).all()


def test_an_infinite_moment_stays_infinite_over_steps(pkg):
    """A gradient whose square is infinite, alone in its block: from the next step on the denominator is infinite and the element stays where it is, as with 32-bit moments."""
    st = pkg.strategy
    found = []
    for bits in (32, 8):
        P, G = torch.ones(128, device="cuda"), torch.zeros(128, device="cuda")
        opt = st.AdamW([P], [G], lr=0.1, weight_decay=0.0, state_bits=bits)
        G[5] = 1e25
        opt.step()
        G[5] = 0.0
        for _ in range(3):
            opt.step()
        v = opt.moments[0].exp_avg_sq
        v = v if bits == 32 else pkg.ops.adamw_state_decode(v, opt.moments[0].exp_avg_sq_scale)
        assert v[5] == INF and v[:5].eq(0).all() and v[6:].eq(0).all()
        found.append(P)
    assert torch.equal(found[0], found[1]) and found[0].eq(1).all()
