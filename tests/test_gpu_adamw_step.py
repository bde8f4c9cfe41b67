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
