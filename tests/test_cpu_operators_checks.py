"""What the AdamW and embedding entry points refuse and keep, without a GPU."""
import ctypes as C

import pytest
import torch

P = 1 << 20   # an address that is never read: every call here is refused before a launch


def adamw(pkg, eps=1e-8, step=1, **fields):
    T = pkg._capi.AdamWTensor
    t = dict(param=P, grad=P, exp_avg=P, exp_avg_sq=P, exp_avg_scale=None, exp_avg_sq_scale=None, n=10, lr=1e-3, weight_decay=0.0, grad_dtype=0)
    t.update(fields)
    arr = (T * 1)(T(**t))
    return pkg._capi.lib().lfs_adamw_step_tensors(1, C.addressof(arr), 0.9, 0.999, eps, step, 1.0, None)


@pytest.mark.parametrize("eps", [1e-39, 1e-300, 2.0 ** -127, 1e38, float("inf"), float("nan")])
def test_eps_that_the_step_cannot_serve_is_refused(pkg, eps):
    """Below 2^-126 (and not zero) the reciprocal takes it as zero, and an element without a gradient would become 0 / 0; above 2^126 its reciprocal is not a normal number."""
    st = pkg.strategy
    assert adamw(pkg, eps=eps) == pkg._capi.LFS_EINVAL and "eps" in pkg._capi.lib().lfs_last_error().decode()
    model = pkg.trainer.SplatData(10, 4, torch.device("cpu"))
    with pytest.raises(RuntimeError, match="eps"):
        st.FusedAdamW(model, [1e-3] * 6, eps=eps)
    with pytest.raises(RuntimeError, match="eps"):
        st.AdamW([torch.zeros(4)], [torch.zeros(4)], eps=eps)


def test_eps_of_zero_and_of_the_smallest_normal_number_are_served(pkg):
    model = pkg.trainer.SplatData(10, 4, torch.device("cpu"))
    for eps in (0.0, 2.0 ** -126, 1e-15, 1.0):
        assert pkg.strategy.FusedAdamW(model, [1e-3] * 6, eps=eps).eps == eps
        assert adamw(pkg, eps=eps, n=0) == 0


def test_a_step_number_below_one_is_refused(pkg):
    for step, missed in ((5, 5), (5, 9), (5, -1), (1, 1)):
        assert adamw(pkg, step=step, missed=missed) == pkg._capi.LFS_EINVAL and "missed" in pkg._capi.lib().lfs_last_error().decode()
    assert adamw(pkg, step=5, missed=9, n=0) == 0     # a tensor that takes no part


def test_gradients_of_another_scene_are_refused(pkg):
    """FusedAdamW reads as many gradient rows as the model has."""
    st, tr = pkg.strategy, pkg.trainer
    cpu = torch.device("cpu")
    opt = st.FusedAdamW(tr.SplatData(10, 4, cpu), [1e-3] * 6, state_bits=8)
    for grads in (tr.SplatData(4, 4, cpu), tr.SplatData(10, 9, cpu), tr.SplatData(10, 4, torch.device("meta"))):
        size = grads.size
        with pytest.raises(RuntimeError, match="gradients"):
            opt.step(2000, grads)
        assert grads.size == size and opt.step_count == 0
