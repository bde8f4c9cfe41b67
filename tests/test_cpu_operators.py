"""Refusals of the AdamW and embedding entry points: none of them needs a GPU, so none of them reaches a kernel."""
import ctypes as C

import numpy as np
import pytest
import torch


def lib(pkg):
    return pkg._capi.lib()


def error(pkg):
    return lib(pkg).lfs_last_error().decode()


P = 1 << 20   # an address that is never read: every call here is refused before a launch


def adamw(pkg, n_tensors=1, tensors="one", beta1=0.9, beta2=0.999, eps=1e-8, step=1, **fields):
    T = pkg._capi.AdamWTensor
    t = dict(param=P, grad=P, exp_avg=P, exp_avg_sq=P, exp_avg_scale=None, exp_avg_sq_scale=None, n=10, lr=1e-3, weight_decay=0.0, grad_dtype=0, reserved=0)
    t.update(fields)
    arr = (T * 1)(T(**t))
    return lib(pkg).lfs_adamw_step_tensors(n_tensors, C.addressof(arr) if tensors else None, beta1, beta2, eps, step, 1.0, None)


@pytest.mark.parametrize("kw,message", [
    (dict(n_tensors=-1), "tensor list"), (dict(tensors=None), "tensor list"), (dict(step=0), "step_count"), (dict(beta1=1.0), "betas"), (dict(beta2=-0.1), "betas"),
    (dict(beta1=float("nan")), "betas"), (dict(eps=-1.0), "eps"), (dict(n=-1), "size"), (dict(n=1 << 40), "size"), (dict(param=None), "null"), (dict(grad=None), "null"),
    (dict(exp_avg=None), "null"), (dict(exp_avg_sq=None), "null"), (dict(grad_dtype=3), "grad_dtype"), (dict(exp_avg_scale=P), "both"), (dict(exp_avg_sq_scale=P), "both"),
    (dict(param=P + 2), "misaligned"), (dict(grad=P + 1, grad_dtype=1), "misaligned"), (dict(exp_avg=P + 1), "misaligned"),
    (dict(exp_avg_scale=P + 1, exp_avg_sq_scale=P), "misaligned")])
def test_adamw_step_refuses(pkg, kw, message):
    assert adamw(pkg, **kw) == pkg._capi.LFS_EINVAL
    assert message in error(pkg)


def test_adamw_step_of_nothing(pkg):
    assert adamw(pkg, n_tensors=0, tensors=None) == 0
    assert adamw(pkg, n=0, param=None, grad=None, exp_avg=None, exp_avg_sq=None) == 0


def test_struct_has_the_layout_of_the_header(pkg):
    T = pkg._capi.AdamWTensor
    assert C.sizeof(T) == pkg.strategy._TABLE.itemsize == 72
    for name, _ in T._fields_:
        assert getattr(T, name).offset == pkg.strategy._TABLE.fields[name][1]


@pytest.mark.parametrize("name", ["encode", "decode"])
def test_state_codes_refuse(pkg, name):
    f = getattr(lib(pkg), f"lfs_adamw_state_{name}")
    args = (lambda n, a, b, c: (n, a, 0, b, c, None)) if name == "encode" else (lambda n, a, b, c: (n, a, b, 0, c, None))
    for bad in (args(-1, P, P, P), args(5, None, P, P), args(5, P, None, P), args(5, P, P, None), args(1 << 37, P, P, P)):
        assert f(*bad) == pkg._capi.LFS_EINVAL
    assert f(*args(0, None, None, None)) == 0


def test_embedding_calls_refuse(pkg):
    l, einval, ecap = lib(pkg), pkg._capi.LFS_EINVAL, pkg._capi.LFS_ECAPACITY
    ok = dict(n=5, rows=3, width=4, table=P, tt=0, idx=P, bits=32, out=P, ot=0)
    def fwd(**kw):
        a = {**ok, **kw}
        return l.lfs_embedding_fwd(a["n"], a["rows"], a["width"], a["table"], a["tt"], a["idx"], a["bits"], 1.0, a["out"], a["ot"], None)
    for bad in (dict(n=-1), dict(n=2 ** 31 - 1), dict(rows=0), dict(rows=2 ** 31 - 1), dict(width=0), dict(width=(1 << 20) + 1), dict(table=None), dict(idx=None), dict(out=None),
                dict(tt=3), dict(tt=0, ot=1), dict(tt=1, ot=2), dict(bits=16), dict(table=P + 2), dict(idx=P + 4, bits=64), dict(out=P + 1)):
        assert fwd(**bad) == einval, bad
    assert fwd(n=0, table=None, idx=None, out=None) == 0
    many = 100_000    # a few lookups need no workspace
    size = l.lfs_embedding_sort_workspace_bytes(many, 3)
    assert size > 0 and l.lfs_embedding_sort_workspace_bytes(5, 3) == l.lfs_embedding_sort_workspace_bytes(5, 0) == 0
    def sort(n=many, rows=3, idx=P, bits=32, order=P, srt=P, ws=P, size=size):
        return l.lfs_embedding_sort(n, rows, idx, bits, order, srt, ws, size, None)
    for bad in (dict(n=-1), dict(rows=0), dict(idx=None), dict(bits=8), dict(order=None), dict(srt=None), dict(ws=None), dict(ws=P + 64), dict(order=P + 1)):
        assert sort(**bad) == einval, bad
    assert sort(size=size - 1) == ecap and sort(n=0, idx=None, order=None, srt=None, ws=None, size=0) == 0
    size_b = l.lfs_embedding_bwd_workspace_bytes(many, 4)
    assert size_b > 0 and l.lfs_embedding_bwd_workspace_bytes(5, 4) == 0
    def bwd(n=many, rows=3, width=4, v=P, t=0, order=P, srt=P, out=P, ws=P, size=size_b):
        return l.lfs_embedding_bwd(n, rows, width, v, t, order, srt, 1.0, 1, out, ws, size, None)
    for bad in (dict(n=-1), dict(rows=0), dict(width=0), dict(v=None), dict(t=5), dict(order=None), dict(srt=None), dict(out=None), dict(ws=None), dict(ws=P + 4), dict(out=P + 2),
                dict(v=P + 1, t=2), dict(order=P + 4), dict(srt=P + 8)):
        assert bwd(**bad) == einval, bad
    assert bwd(size=size_b - 1) == ecap and bwd(n=0, v=None, order=None, srt=None, ws=None) == 0


def test_python_embedding_refuses(pkg):
    ops = pkg.ops
    t, i = torch.zeros(4, 3), torch.zeros(5, dtype=torch.int32)
    for args, kw, message in (((t, i), {}, "CUDA"), ((t.double(), i), {}, "table must be"), ((t.t(), i), {}, "contiguous"), ((t[0], i), {}, "table must be|CUDA"),
                              ((None, i), {}, "tensor")):
        with pytest.raises(RuntimeError, match=message):
            ops.embedding_fwd(*args, **kw)
    with pytest.raises(RuntimeError, match="indices must be"):
        ops.embedding_sort(t, 4)
    with pytest.raises(RuntimeError, match="CUDA"):
        ops.embedding_sort(i, 4)
    with pytest.raises(RuntimeError, match="embedding_sort"):
        ops.embedding_bwd(t, i)
    with pytest.raises(RuntimeError, match="values must be"):
        ops.adamw_state_encode(t.half())
    with pytest.raises(RuntimeError, match="codes must be"):
        ops.adamw_state_decode(t, t)


def test_python_optimizers_refuse(pkg):
    st, tr = pkg.strategy, pkg.trainer
    t = torch.zeros(4)
    for args, kw, message in ((([], []), {}, "at least one"), (([t], [t]), {}, "CUDA"), (([t.half()], [t]), {}, "params"), (([t], [t]), dict(betas=(1.0, 0.9)), "betas"),
                              (([t], [t]), dict(eps=-1), "eps")):
        with pytest.raises(RuntimeError, match=message):
            st.AdamW(*args, **kw)
    with pytest.raises(RuntimeError, match="state_bits"):
        st.Moments.zeros(5, 16, "cpu")
    m8, m32 = st.Moments.zeros(200, 8, "cpu"), st.Moments.zeros(200, 32, "cpu")
    assert m8.exp_avg.dtype == torch.float8_e4m3fn and m8.exp_avg_sq.dtype == torch.float8_e5m2 and m8.exp_avg_scale.numel() == 2
    m8.exp_avg_sq_scale = None
    with pytest.raises(RuntimeError, match="both"):
        m8.check(200, torch.device("cpu"), "m")
    with pytest.raises(RuntimeError, match="CUDA"):
        m32.check(200, torch.device("cpu"), "m")
    model = tr.SplatData(10, 4, torch.device("cpu"))
    lrs = [1e-3] * 6
    with pytest.raises(RuntimeError, match="state_bits"):
        st.FusedAdamW(model, lrs, state_bits=4)
    with pytest.raises(RuntimeError, match="values for 6"):
        st.FusedAdamW(model, lrs, weight_decay=[0.1] * 5)
    P_ = st.OptimizationParameters
    assert type(st.make_optimizer(model, lrs, P_())) is st.FusedAdam
    assert type(st.make_optimizer(model, lrs, P_(optimizer="adamw", state_bits=8))) is st.FusedAdamW
    for bad, message in ((P_(optimizer="sgd"), "adam or adamw"), (P_(weight_decay=0.1), "adamw"), (P_(state_bits=8), "adamw"), (P_(weight_decay=(0, 0, 0, 0, 0, 0.1)), "adamw")):
        with pytest.raises(RuntimeError, match=message):
            st.make_optimizer(model, lrs, bad)
    opt = st.FusedAdamW(model, lrs, state_bits=8)
    for kw in (dict(rasterizer=object()), dict(first_row=1), dict(n_rows=5)):
        with pytest.raises(RuntimeError, match="all rows"):
            opt.step(2000, model.like(), **kw)
    assert opt.step_count == 0
    with pytest.raises(RuntimeError, match="CUDA"):
        tr.ShPalette(torch.zeros(4, 3, 3), torch.zeros(10, dtype=torch.int32))
    with pytest.raises(RuntimeError, match="K-1"):
        tr.ShPalette(torch.zeros(4, 9), torch.zeros(10, dtype=torch.int32))


def test_8_bit_moments_take_a_quarter(pkg):
    model = pkg.trainer.SplatData(1000, 16, torch.device("cpu"))
    opt = pkg.strategy.FusedAdamW(model, [1e-3] * 6, state_bits=8)
    held = sum(x.codes[n].numel() + 4 * x.scales[n].numel() for x in (opt.exp_avg, opt.exp_avg_sq) for n in x.codes)
    assert 118 * 1000 <= held <= 122 * 1000    # 59 codes twice, and a scale for 128
    rows = torch.tensor([3, 3, 999])
    for name, codes in opt.exp_avg.codes.items():
        codes.view(torch.uint8).fill_(5)
    opt.exp_avg.zero_rows(rows)
    opt.exp_avg.zero_rows(slice(10, 20))
    for name, codes in opt.exp_avg.codes.items():
        c = codes.view(torch.uint8).view(1000, -1)
        gone = torch.zeros(1000, dtype=torch.bool)
        gone[[3, 999] + list(range(10, 20))] = True
        assert c[gone].eq(0).all() and c[~gone].eq(5).all()
