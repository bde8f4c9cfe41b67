"""A tensor of more than 2^31 elements: a launch takes it in pieces of 2^30, and an element's place in the whole tensor decides its threshold."""
import pytest
import torch

pytestmark = pytest.mark.gpu
PIECE, END = 1 << 30, (3 << 30) + 300
WINDOWS = [(0, 512), (PIECE - 512, PIECE + 512), (2 * PIECE - 512, 2 * PIECE + 512), (3 * PIECE - 512, END)]


def codes(x, start, t, second):
    """The definition in float32, whose operations round as the kernel's do: magnitude times top / largest of the block, rounded by adding the threshold to the bits of the fraction that go."""
    top, dropped, least, first, step = (57344.0, 21, 2.0 ** -14, 0x9E3779B9, 0xC13FA9A9) if second else (448.0, 20, 2.0 ** -6, 0x91E10DA5, 0x9E3779B9)
    n = x.numel()
    most = torch.nn.functional.pad(x.abs(), (0, -n % 128)).view(-1, 128).amax(1)
    inverse = torch.where(most > 0, torch.full_like(most, top) / most, most).repeat_interleave(128)[:n]
    y = (x.abs() * inverse).clamp(max=top)
    i = torch.arange(start, start + n, dtype=torch.int64)
    threshold = ((((i * first) % 2 ** 32 + (t * step) % 2 ** 32) % 2 ** 32) >> (32 - dropped)).to(torch.int32)
    small = y < least
    bits = (torch.where(small, y + least, y).view(torch.int32) + threshold) >> dropped << dropped
    y = torch.where(small, bits.view(torch.float32) - least, bits.view(torch.float32))
    if second:
        y = torch.where(x > 0, y.clamp(min=least * 0.25), y)
    return torch.copysign(y, x), most * torch.full_like(most, 1.0 / top)


@pytest.mark.parametrize("bits", [8, 32])
def test_each_piece_goes_on_where_the_one_before_ends(pkg, bits):
    st = pkg.strategy
    P = torch.zeros(END, device="cuda")
    G = torch.zeros(END, dtype=torch.bfloat16, device="cuda")
    gen = torch.Generator().manual_seed(3)
    parts = [torch.randn(b - a, generator=gen).to(torch.bfloat16) for a, b in WINDOWS]
    for (a, b), g in zip(WINDOWS, parts):
        G[a:b] = g.cuda()
    opt = st.AdamW([P], [G], lr=0.1, weight_decay=0.0, state_bits=bits)
    opt.step_count = 6
    opt.step()
    m = opt.moments[0]
    for (a, b), g in zip(WINDOWS, parts):
        one = torch.zeros(b - a, device="cuda")
        alone = st.AdamW([one], [g.cuda()], lr=0.1, weight_decay=0.0, state_bits=32)
        alone.step_count = 6
        alone.step()
        held = alone.moments[0]
        if bits == 32:
            assert torch.equal(P[a:b], one) and torch.equal(m.exp_avg[a:b], held.exp_avg) and torch.equal(m.exp_avg_sq[a:b], held.exp_avg_sq)
            continue
        # the step of 8-bit moments takes the approximate root and reciprocal, 2^-23 of it each, and a product more
        assert ((P[a:b] - one).abs() <= 8 * 2.0 ** -24 * one.abs()).all()
        for x, c, s, second in ((held.exp_avg, m.exp_avg, m.exp_avg_scale, False), (held.exp_avg_sq, m.exp_avg_sq, m.exp_avg_sq_scale, True)):
            want, scale = codes(x.cpu(), a, 7, second)
            assert torch.equal(c[a:b].cpu().float(), want) and torch.equal(s[a // 128: -(-b // 128)].cpu(), scale), (a, second)
    # between the windows nothing has a gradient: parameters and moments stay zero
    for a, b in ((512, PIECE - 512), (PIECE + 512, 2 * PIECE - 512), (2 * PIECE + 512, 3 * PIECE - 512)):
        assert not P[a:b].any() and not m.exp_avg[a:b].view(torch.uint8).any() and not m.exp_avg_sq[a:b].view(torch.uint8).any()
