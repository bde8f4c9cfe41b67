"""What an AdamW step writes is written by one launch in no order: the same memory twice is refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_moments_that_overlap_are_refused(pkg):
    st = pkg.strategy
    P, G = [torch.zeros(300, device="cuda") for _ in range(2)], [torch.ones(300, device="cuda") for _ in range(2)]
    one = st.Moments.zeros(300, 32, P[0].device)
    for bits in (32, 8):
        m = st.Moments.zeros(300, bits, P[0].device)
        with pytest.raises(RuntimeError, match="overlap"):
            st.AdamW(P, G, moments=[m, m])          # one tensor's twice
    with pytest.raises(RuntimeError, match="overlap"):
        st.AdamW(P, G, moments=[one, st.Moments(torch.zeros(300, device="cuda"), one.exp_avg_sq)])
    with pytest.raises(RuntimeError, match="overlap"):
        st.AdamW(P, G, moments=[st.Moments(one.exp_avg, one.exp_avg), st.Moments.zeros(300, 32, P[0].device)])
    with pytest.raises(RuntimeError, match="overlap"):
        st.AdamW(P, G, moments=[st.Moments(P[0], one.exp_avg), st.Moments.zeros(300, 32, P[0].device)])
    with pytest.raises(RuntimeError, match="overlap"):
        st.AdamW([P[0], P[0][100:200]], [G[0], G[1][:100]])
    a, b = st.Moments.zeros(300, 8, P[0].device), st.Moments.zeros(300, 8, P[0].device)
    b.exp_avg_sq_scale = a.exp_avg_scale
    with pytest.raises(RuntimeError, match="overlap"):
        st.AdamW(P, G, moments=[a, b])
    assert all(p.eq(0).all() for p in P)


def test_neighbours_do_not_overlap(pkg):
    """Everything as pieces of one buffer, one behind the other, with an empty tensor at the address of another; one gradient for two parameters is only read."""
    st = pkg.strategy
    flat, g = torch.zeros(4096, device="cuda"), torch.ones(100, device="cuda")
    p = [flat[:100], flat[100:200], flat[100:100]]
    m = [st.Moments(flat[200:300], flat[300:400]), st.Moments(flat[400:500], flat[500:600]), st.Moments(flat[:0], flat[:0])]
    opt = st.AdamW(p, [g, g, flat[:0]], lr=0.1, weight_decay=0.0, moments=m)
    opt.step()
    assert (flat[:200] + 0.1).abs().max() < 1e-6 and flat[200:300].eq(flat[200]).all() and flat[600:].eq(0).all() and flat[200:600].gt(0).all()
