"""Scenes whose moments are in 8 bits: what duplicating, splitting and removing rows needs."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def scene(pkg, n, K=4, capacity=None, seed=0):
    gen = torch.Generator().manual_seed(seed)
    model = pkg.trainer.SplatData(n, K, torch.device("cuda"), capacity)
    for name in pkg.trainer.PARAM_NAMES:
        model.tensor(name).copy_(torch.randn(model.tensor(name).shape, generator=gen))
    return model


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
