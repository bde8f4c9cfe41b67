"""Training-strategy interface of the reference over the C ABI.

Mirrors src/training/strategies/istrategy.hpp:13-32 (IStrategy), src/training/strategies/mcmc.{hpp,cpp}
(MCMC: relocate / add / noise / Adam step / LR decay), src/training/optimizers/fused_adam.{hpp,cpp}
(FusedAdam) and src/training/optimizers/scheduler.cpp (ExponentialLR) with the same method names,
argument meaning and defaults (include/core/parameters.hpp:16-40).

Differences that follow from the buffer design: parameters, gradients and Adam moments live in
capacity-reserved flat buffers (trainer.SplatData), so add_new_gs appends rows in place instead of
six torch::cat re-allocations and a re-keying of the optimizer state, and gradients are passed to
step() explicitly because there is no autograd .grad slot."""
from __future__ import annotations

import ctypes as C
import numbers
from dataclasses import dataclass

import numpy as np
import torch

from . import _capi as capi, ops
from ._capi import call, ptr
from .trainer import PARAM_NAMES, SplatData, adam_step_splats


def _stream():
    return capi.vp(torch.cuda.current_stream().cuda_stream)


@dataclass
class OptimizationParameters:
    """Subset of gs::param::OptimizationParameters used on this path (include/core/parameters.hpp:16-40)."""
    iterations: int = 30_000
    sh_degree_interval: int = 1_000
    means_lr: float = 0.00016
    shs_lr: float = 0.0025
    opacity_lr: float = 0.05
    scaling_lr: float = 0.005
    rotation_lr: float = 0.001
    lambda_dssim: float = 0.2
    min_opacity: float = 0.005
    refine_every: int = 100
    start_refine: int = 500
    stop_refine: int = 25_000
    max_cap: int = 1_000_000
    sh_degree: int = 3
    scene_scale: float = 1.0
    # no counterpart in the reference
    optimizer: str = "adam"                        # "adam" (FusedAdam) or "adamw" (FusedAdamW)
    weight_decay: float | tuple[float, ...] = 0.0  # adamw: one value, or one per parameter group
    state_bits: int = 32                           # adamw: moments in 32 or 8 bits


class FusedAdam:
    """torch::optim-style Adam over the six parameter groups with one fused launch per step
    (fused_adam.cpp:22-95). Group order: means, sh0, shN, scaling, rotation, opacity."""

    def __init__(self, model: SplatData, lrs, betas=(0.9, 0.999), eps=1e-15):
        self.model = model
        self.lr = [float(x) for x in lrs]
        self.betas, self.eps = (float(betas[0]), float(betas[1])), float(eps)
        self.exp_avg, self.exp_avg_sq = model.like(), model.like()
        self.step_count = 0

    def step(self, iteration: int, grads: SplatData, grad_scale: float = 1.0, first_row: int = 0, n_rows=None,
             rasterizer=None):
        """rasterizer: the Rasterizer whose backward(write_shN=False) of ONE camera produced `grads`; the shN rows are then
        updated from gradient rows rebuilt inside the optimizer kernel (lfs_adam_step_splats_rank1_sh)."""
        self.step_count += 1  # advances for the skipped shN group as well (fused_adam.cpp:66-70)
        self.exp_avg.size = self.exp_avg_sq.size = grads.size = self.model.size
        if rasterizer is not None:
            if first_row != 0 or n_rows not in (None, self.model.size):
                raise RuntimeError("the rank-1 shN update covers all rows")
            rasterizer.adam_step_rank1_sh(self.exp_avg, self.exp_avg_sq, grads, self.lr, self.step_count, self.betas[0],
                                          self.betas[1], self.eps, skip_shN=(iteration <= 1000), grad_scale=grad_scale)
            return
        adam_step_splats(self.model, self.exp_avg, self.exp_avg_sq, grads, self.lr, self.step_count, self.betas[0], self.betas[1],
                         self.eps, skip_shN=(iteration <= 1000), first_row=first_row, n_rows=n_rows, grad_scale=grad_scale)

    def zero_grad(self, set_to_none=True, iteration=0):
        """No-op: the next backward overwrites every gradient row."""


@dataclass
class Moments:
    """The moments of one tensor: float32, or 8-bit codes (e4m3, e5m2) with the scales of their blocks of 128 elements."""
    exp_avg: torch.Tensor
    exp_avg_sq: torch.Tensor
    exp_avg_scale: torch.Tensor | None = None
    exp_avg_sq_scale: torch.Tensor | None = None

    @staticmethod
    def zeros(n: int, state_bits: int, device) -> "Moments":
        if state_bits == 32:
            return Moments(*(torch.zeros(n, dtype=torch.float32, device=device) for _ in range(2)))
        if state_bits != 8:
            raise RuntimeError(f"state_bits must be 32 or 8, got {state_bits}")
        codes = [torch.zeros(n, dtype=torch.uint8, device=device).view(t) for t in (torch.float8_e4m3fn, torch.float8_e5m2)]
        return Moments(*codes, *(torch.zeros(-(-n // capi.LFS_ADAMW_BLOCK), dtype=torch.float32, device=device) for _ in range(2)))

    def check(self, n: int, device, what: str):
        bits = 32 if self.exp_avg_scale is None and self.exp_avg_sq_scale is None else 8
        if bits == 8 and (self.exp_avg_scale is None or self.exp_avg_sq_scale is None):
            raise RuntimeError(f"{what}: both moments have scales, or neither")
        types = (torch.float32, torch.float32) if bits == 32 else (torch.float8_e4m3fn, torch.float8_e5m2)
        for t, name, dtype in zip((self.exp_avg, self.exp_avg_sq), ("exp_avg", "exp_avg_sq"), types):
            ops._check_typed(t, f"{what}.{name}", (dtype,), device)
            if t.numel() != n:
                raise RuntimeError(f"{what}.{name} must have {n} elements, got {t.numel()}")
        for t, name in zip((self.exp_avg_scale, self.exp_avg_sq_scale), ("exp_avg_scale", "exp_avg_sq_scale")):
            if bits == 8:
                ops._check_typed(t, f"{what}.{name}", (torch.float32,), device)
                if t.numel() != -(-n // capi.LFS_ADAMW_BLOCK):
                    raise RuntimeError(f"{what}.{name} must have {-(-n // capi.LFS_ADAMW_BLOCK)} elements, got {t.numel()}")


_TABLE = np.dtype([("param", "u8"), ("grad", "u8"), ("exp_avg", "u8"), ("exp_avg_sq", "u8"), ("exp_avg_scale", "u8"), ("exp_avg_sq_scale", "u8"),
                   ("n", "i8"), ("lr", "f4"), ("weight_decay", "f4"), ("grad_dtype", "i4"), ("missed", "i4")])   # lfs_adamw_tensor


def _each(value, n: int, name: str) -> list:
    """One float per tensor from one for all or a list."""
    values = [float(value)] * n if isinstance(value, numbers.Real) else [float(x) for x in value]
    if len(values) != n:
        raise RuntimeError(f"{name}: {len(values)} values for {n} tensors")
    return values


def _check_betas(betas, eps):
    if not all(0.0 <= b < 1.0 for b in betas) or len(betas) != 2 or not (eps == 0.0 or 2.0 ** -126 <= eps <= 2.0 ** 126):
        raise RuntimeError(f"betas must be two numbers in [0, 1) and eps zero or in [2^-126, 2^126], got {betas}, {eps}")


class AdamW:
    """AdamW over a list of tensors, one launch per 424 of them (lfs_adamw_step_tensors): per-image codes, exposure matrices, grids,
    palettes, small networks. Parameters are contiguous float32, gradients contiguous float32, bfloat16 or float16 of the same number of elements, on one device.

    Parameters, gradients and moments are bound here and stay bound: a step reads the gradients that are in those buffers by then (torch: zero_grad(set_to_none=False)),
    and set_grads binds others. None in the place of a gradient leaves its parameter out, and the step does not count for it: `missed` [tensors] is how many of the step_count steps so far each one took no
    part in, and step_count - missed is the number that its bias corrections go by. `lr` and `weight_decay` (one value or one per tensor) are
    read at every step, so a scheduler may change one entry or set the whole again (one value or one per tensor). moments: those of a run to continue, with its step_count and missed to be set as well; else zeros, in state_bits (32 or 8) bits.

    A step costs little because everything is checked before: binding the gradients of 400 tensors takes 0.5 ms, a step over them 14 us. Tensors that begin on 16 bytes are read in whole vectors.
    A captured step repeats its own step number, so 8-bit moments, whose rounding goes by it, are for steps that are launched one by one."""

    def __init__(self, params, grads, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, state_bits=32, moments=None):
        params = list(params)
        if not params:
            raise RuntimeError("AdamW needs at least one tensor")
        n = len(params)
        self.betas, self.eps = tuple(float(b) for b in betas), float(eps)
        _check_betas(self.betas, self.eps)
        self.device = params[0].device
        for i, p in enumerate(params):
            ops._check_typed(p, f"params[{i}]", (torch.float32,), self.device)
        self.params = [p.detach() for p in params]   # keeps the memory that the kernel writes to
        if moments is None:
            moments = [Moments.zeros(p.numel(), b, self.device) for p, b in zip(self.params, self._bits(state_bits, n))]
        self.moments = list(moments)
        if len(self.moments) != n:
            raise RuntimeError(f"moments: {len(self.moments)} for {n} tensors")
        for i, (p, m) in enumerate(zip(self.params, self.moments)):
            m.check(p.numel(), self.device, f"moments[{i}]")
        self.lr, self.weight_decay = lr, weight_decay
        self.step_count = 0
        self._table, self._rates = np.zeros(n, _TABLE), None
        self._address = self._table.ctypes.data
        self._table["param"] = [p.data_ptr() for p in self.params]
        for name in ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale"):
            self._table[name] = [0 if getattr(m, name) is None else getattr(m, name).data_ptr() for m in self.moments]
        self._check_written([p.numel() for p in self.params])
        self.set_grads(grads)

    @property
    def missed(self) -> np.ndarray:
        return self._table["missed"]

    @missed.setter
    def missed(self, value):
        counts = np.asarray(value, dtype=np.int64)
        if counts.shape != (len(self.params),) or (counts < 0).any() or (counts >= 1 << 31).any():
            raise RuntimeError(f"missed: one count for each of {len(self.params)} tensors, got {value}")
        self._table["missed"] = counts

    @property
    def lr(self) -> list:
        return self._lr

    @lr.setter
    def lr(self, value):
        self._lr = _each(value, len(self.params), "lr")

    @property
    def weight_decay(self) -> list:
        return self._weight_decay

    @weight_decay.setter
    def weight_decay(self, value):
        self._weight_decay = _each(value, len(self.params), "weight_decay")

    @staticmethod
    def _bits(state_bits, n):
        bits = [state_bits] * n if isinstance(state_bits, int) else list(state_bits)
        if len(bits) != n:
            raise RuntimeError(f"state_bits: {len(bits)} values for {n} tensors")
        return bits

    def _check_written(self, sizes):
        """A step writes parameters, moments and scales in one launch, in no order."""
        t, n = self._table, np.array(sizes, dtype=np.int64)
        one = np.where(t["exp_avg_scale"] == 0, 4, 1)
        starts = np.concatenate([t[x].astype(np.int64) for x in ("param", "exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")])
        scales = np.where(t["exp_avg_scale"] == 0, 0, -(-n // capi.LFS_ADAMW_BLOCK) * 4)
        ends = starts + np.concatenate([4 * n, one * n, one * n, scales, scales])
        some = ends > starts
        order = np.argsort(starts[some])
        if (ends[some][order][:-1] > starts[some][order][1:]).any():
            raise RuntimeError("params and moments must not overlap")

    def set_grads(self, grads):
        grads = list(grads)
        if len(grads) != len(self.params):
            raise RuntimeError(f"grads: {len(grads)} for {len(self.params)} tensors")
        for i, (p, g) in enumerate(zip(self.params, grads)):
            if g is None:
                continue
            ops._check_typed(g, f"grads[{i}]", ops._DTYPES, self.device)
            if g.numel() != p.numel():
                raise RuntimeError(f"grads[{i}] must have {p.numel()} elements, got {g.numel()}")
        self.grads = [None if g is None else g.detach() for g in grads]
        absent = np.array([g is None for g in grads])
        self._absent = absent if absent.any() else None
        self._table["n"] = [0 if g is None else g.numel() for g in grads]
        self._table["grad"] = [0 if g is None else g.data_ptr() for g in grads]
        self._table["grad_dtype"] = [0 if g is None else ops._DTYPES[g.dtype] for g in grads]

    def step(self, grad_scale: float = 1.0):
        """One update from the bound gradients, which grad_scale multiplies."""
        rates = (list(self._lr), list(self._weight_decay))
        if rates != self._rates:
            for name, values in zip(("lr", "weight_decay"), rates):
                self._table[name] = _each(values, len(self.params), name)
            self._rates = rates
        ops._call_on(self.device, "lfs_adamw_step_tensors", len(self._table), self._address, self.betas[0], self.betas[1], self.eps,
                     self.step_count + 1, float(grad_scale))
        self.step_count += 1
        if self._absent is not None:
            self.missed[self._absent] += 1


class PackedMoments:
    """One Adam moment of all six groups in 8 bits: what SplatData is for 32-bit moments. tensor() gives the values that the codes of the live rows stand for (a copy),
    put() encodes new ones. Rows at and above `size` are cleared when they come into use (zero_rows)."""

    def __init__(self, model: SplatData, second: bool):
        self.capacity, self.size, self.device, self.K, self._w = model.capacity, model.size, model.device, model.K, model._w
        self.second = second
        self.codes, self.scales = {}, {}
        for name in PARAM_NAMES:
            m = Moments.zeros(self.capacity * self._w[name], 8, self.device)
            self.codes[name], self.scales[name] = (m.exp_avg_sq, m.exp_avg_sq_scale) if second else (m.exp_avg, m.exp_avg_scale)

    def live(self, name: str):
        """Codes and scales of the live rows."""
        n = self.size * self._w[name]
        return self.codes[name][:n], self.scales[name][:-(-n // capi.LFS_ADAMW_BLOCK)]

    def tensor(self, name: str) -> torch.Tensor:
        t = ops.adamw_state_decode(*self.live(name))
        return t.view(self.size, self._w[name] // 3, 3) if name in ("sh0", "shN") else t.view(self.size, self._w[name])

    def put(self, name: str, rows: torch.Tensor):
        codes, scales = self.live(name)
        c, s = ops.adamw_state_encode(rows.reshape(-1).contiguous(), self.second)
        codes.view(torch.uint8).copy_(c.view(torch.uint8))
        scales.copy_(s)

    def zero_rows(self, rows):
        """rows: an int64 tensor, or a slice."""
        for name in PARAM_NAMES:
            if self._w[name] == 0:
                continue
            codes = self.codes[name].view(torch.uint8).view(self.capacity, self._w[name])
            if isinstance(rows, slice):
                codes[rows] = 0
            else:
                codes.index_fill_(0, rows, 0)


class FusedAdamW(FusedAdam):
    """FusedAdam's interface with decoupled weight decay (one value or one per group) and moments in 32 or 8 bits, one launch per step. With 8 bits the
    moments of a scene take 118 bytes per Gaussian at SH degree 3 instead of 472; exp_avg and exp_avg_sq are PackedMoments."""

    def __init__(self, model: SplatData, lrs, betas=(0.9, 0.999), eps=1e-15, weight_decay=0.0, state_bits: int = 32):
        if state_bits not in (32, 8):
            raise RuntimeError(f"state_bits must be 32 or 8, got {state_bits}")
        _check_betas(betas, eps)
        self.model = model
        self.lr = _each(lrs, 6, "lrs")
        self.weight_decay = _each(weight_decay, 6, "weight_decay")
        self.betas, self.eps = (float(betas[0]), float(betas[1])), float(eps)
        self.state_bits = state_bits
        if state_bits == 32:
            self.exp_avg, self.exp_avg_sq = model.like(), model.like()
        else:
            self.exp_avg, self.exp_avg_sq = PackedMoments(model, False), PackedMoments(model, True)
        self.step_count = 0
        self._table = np.zeros(6, _TABLE)

    def step(self, iteration: int, grads: SplatData, grad_scale: float = 1.0, first_row: int = 0, n_rows=None, rasterizer=None):
        if rasterizer is not None or first_row != 0 or n_rows not in (None, self.model.size):
            raise RuntimeError("FusedAdamW updates all rows from materialised gradients")
        if grads.K != self.model.K or grads.capacity < self.model.size or grads.flat.device != self.model.flat.device:
            raise RuntimeError(f"gradients of {grads.capacity} rows with {grads.K} SH bases on {grads.flat.device} for {self.model.size} with {self.model.K} on {self.model.flat.device}")
        self.exp_avg.size = self.exp_avg_sq.size = grads.size = self.model.size
        packed = self.state_bits == 8
        for i, name in enumerate(PARAM_NAMES):
            n = 0 if name == "shN" and iteration <= 1000 else self.model.size * self.model._w[name]   # fused_adam.cpp:66-70
            moments = [x.codes[name] if packed else x._full[name] for x in (self.exp_avg, self.exp_avg_sq)]
            scales = [x.scales[name].data_ptr() if packed else 0 for x in (self.exp_avg, self.exp_avg_sq)]
            self._table[i] = (self.model._full[name].data_ptr(), grads._full[name].data_ptr(), moments[0].data_ptr(), moments[1].data_ptr(), *scales,
                              n, self.lr[i], self.weight_decay[i], capi.LFS_F32, 0)
        ops._call_on(self.model.flat.device, "lfs_adamw_step_tensors", 6, self._table.ctypes.data, self.betas[0], self.betas[1], self.eps,
                     self.step_count + 1, float(grad_scale))
        self.step_count += 1


def make_optimizer(model: SplatData, lrs, params) -> FusedAdam:
    """The optimizer that OptimizationParameters names."""
    kind, decay, bits = getattr(params, "optimizer", "adam"), getattr(params, "weight_decay", 0.0), getattr(params, "state_bits", 32)
    if kind == "adamw":
        return FusedAdamW(model, lrs, (0.9, 0.999), 1e-15, decay, bits)
    if kind != "adam":
        raise RuntimeError(f"optimizer must be adam or adamw, got {kind}")
    if bits != 32 or (decay if isinstance(decay, numbers.Real) else any(decay)):
        raise RuntimeError("weight_decay and state_bits need optimizer=\"adamw\"")
    return FusedAdam(model, lrs, (0.9, 0.999), 1e-15)


class ExponentialLR:
    """scheduler.cpp:10 / mcmc.cpp:20: lr *= gamma for one group (or all when index < 0)."""

    def __init__(self, optimizer: FusedAdam, gamma: float, param_group_index: int = -1):
        self.opt, self.gamma, self.idx = optimizer, float(gamma), int(param_group_index)

    def step(self):
        if self.idx >= 0:
            self.opt.lr[self.idx] *= self.gamma
        else:
            self.opt.lr = [x * self.gamma for x in self.opt.lr]


class IStrategy:
    def initialize(self, optim_params): raise NotImplementedError
    def post_backward(self, iter, render_output): raise NotImplementedError
    def step(self, iter): raise NotImplementedError
    def is_refining(self, iter) -> bool: raise NotImplementedError
    def get_model(self): raise NotImplementedError
    def remove_gaussians(self, mask): raise NotImplementedError


def binoms_table(n_max: int = 51) -> np.ndarray:
    """mcmc.cpp:459-472: running float32 product of (n - i) / (i + 1)."""
    b = np.zeros((n_max, n_max), np.float32)
    for n in range(n_max):
        for k in range(n + 1):
            v = np.float32(1.0)
            for i in range(k):
                v = np.float32(v * (np.float32(n - i) / np.float32(i + 1)))
            b[n, k] = v
    return b


class MCMC(IStrategy):
    """"3D Gaussian Splatting as Markov Chain Monte Carlo" strategy (mcmc.cpp)."""

    _noise_lr = 5e5  # mcmc.hpp:79

    def __init__(self, splat_data: SplatData):
        self._splat_data = splat_data
        self._params = None
        self._optimizer = None
        self._scheduler = None
        self.grads = splat_data.like()
        self.active_sh_degree = 0
        # False once a refinement has replaced the parameter rows of this iteration: the reference's new leaf tensors
        # have no .grad, so FusedAdam::step skips them before it counts the step (fused_adam.cpp:46-48)
        self._grads_valid = True

    # ------------------------------------------------------------------ IStrategy
    def initialize(self, optim_params: OptimizationParameters):
        p = self._params = optim_params
        dev = self._splat_data.device
        self._binoms = torch.from_numpy(binoms_table(51)).to(dev)
        lrs = [p.means_lr * p.scene_scale, p.shs_lr, p.shs_lr / 20.0, p.scaling_lr, p.rotation_lr, p.opacity_lr]  # mcmc.cpp:487-492
        self._optimizer = make_optimizer(self._splat_data, lrs, p)
        self._scheduler = ExponentialLR(self._optimizer, 0.01 ** (1.0 / p.iterations), 0)
        cap = self._splat_data.capacity
        i64 = lambda n: torch.empty(n, dtype=torch.int64, device=dev)
        self._dead, self._alive, self._sampled = i64(cap), i64(cap), i64(cap)
        self._alive_opac = torch.empty(cap, dtype=torch.float32, device=dev)
        self._counts2 = torch.zeros(2, dtype=torch.int32, device=dev)
        self._counts = torch.empty(cap, dtype=torch.int32, device=dev)
        self._ratios = torch.empty(cap, dtype=torch.int32, device=dev)
        self._s_opac = torch.empty(cap, dtype=torch.float32, device=dev)
        self._s_scales = torch.empty((cap, 3), dtype=torch.float32, device=dev)
        self._new_opac = torch.empty(cap, dtype=torch.float32, device=dev)
        self._new_scales = torch.empty((cap, 3), dtype=torch.float32, device=dev)
        self._noise = torch.empty((cap, 3), dtype=torch.float32, device=dev)
        self._ws = torch.empty(capi.lib().lfs_mcmc_workspace_bytes(cap), dtype=torch.uint8, device=dev)

    def is_refining(self, iter: int) -> bool:
        p = self._params
        return iter < p.stop_refine and iter > p.start_refine and iter % p.refine_every == 0

    def get_model(self) -> SplatData:
        return self._splat_data

    def post_backward(self, iter: int, render_output=None):
        if iter % self._params.sh_degree_interval == 0:
            self.active_sh_degree = min(self.active_sh_degree + 1, self._params.sh_degree)  # increment_sh_degree
        if self.is_refining(iter):
            self.relocate_gs()
            self.add_new_gs()
        self.inject_noise()
        self._means_moved_iter = iter     # the noise moved every mean; relocation rewrote rows

    def step(self, iter: int, grad_scale: float = 1.0, rasterizer=None):
        """mcmc.cpp:395-402. On an iteration whose post_backward appended or removed rows the optimizer does nothing and
        does not count the step (the gradients belong to the old rows); the scheduler still runs. The next backward
        writes every gradient row again.
        rasterizer (FusedAdam.step): the rank-1 shN update rebuilds each gradient row from the CURRENT means and the camera
        of the forward, so it is only equal to the materialised gradient while the means are those the forward saw. It is
        refused after this iteration's post_backward (which moved them); leave rasterizer=None in the reference's order
        backward -> post_backward -> step."""
        if rasterizer is not None and getattr(self, "_means_moved_iter", None) == iter:
            raise RuntimeError("MCMC.step(rasterizer=...): post_backward of this iteration moved the means; the rank-1 shN "
                               "update would rebuild its gradient rows from other view directions than the forward's. "
                               "Call step() without a rasterizer (backward must then write the shN gradient).")
        if iter < self._params.iterations:
            if self._grads_valid:
                self._optimizer.step(iter, self.grads, grad_scale, rasterizer=rasterizer)
            self._grads_valid = True
            self._optimizer.zero_grad(True, iter)
            self._scheduler.step()

    def remove_gaussians(self, mask: torch.Tensor):
        """mcmc.cpp:406-444: keep rows where mask is False (parameters and Adam moments)."""
        old_n = self._splat_data.size
        if mask.numel() != old_n:
            raise RuntimeError(f"mask must have {old_n} elements, got {mask.numel()}")
        keep = (~mask.bool()).nonzero().squeeze(-1)
        new_n = int(keep.numel())
        if new_n == old_n:
            return
        _rewrite_rows((self._splat_data, self._optimizer.exp_avg, self._optimizer.exp_avg_sq), old_n, new_n,
                      lambda _, name, rows: rows.index_select(0, keep))
        self.grads.size = new_n
        self._grads_valid = False

    # ------------------------------------------------------------------ pieces
    @staticmethod
    def multinomial_sample(weights: torch.Tensor, n: int, replacement: bool = True) -> torch.Tensor:
        """mcmc.cpp:43-84. torch.multinomial is the same libtorch call the reference makes, so for the same
        generator state and bit-identical weights the sampled indices are those of the reference."""
        if weights.numel() <= (1 << 24):
            return torch.multinomial(weights, n, replacement)
        w = (weights / weights.sum()).cpu()
        cdf = w.cumsum(0).numpy()
        # drawn from torch's generator so that ranks seeded alike stay replicated
        u = torch.rand(n, dtype=torch.float32, device=weights.device).cpu().numpy()
        return torch.from_numpy(np.minimum(np.searchsorted(cdf, u, side="left"), weights.numel() - 1)).to(weights.device)

    def _relocate_with(self, sampled: torch.Tensor, dst, n: int):
        """Everything after the draw: ratios, eq. (9), write-back, row copies, moment reset."""
        sd, opt = self._splat_data, self._optimizer
        N = sd.size
        st = _stream()
        call("lfs_mcmc_gather_ratios", N, n, ptr(sampled), ptr(sd._full["opacity_raw"]), ptr(sd._full["scaling_raw"]), 51,
             ptr(self._counts), ptr(self._ratios), ptr(self._s_opac), ptr(self._s_scales), st)
        call("lfs_relocation", n, ptr(self._s_opac), ptr(self._s_scales), ptr(self._ratios), ptr(self._binoms), 51,
             ptr(self._new_opac), ptr(self._new_scales), st)
        p = sd.struct()
        packed = isinstance(opt.exp_avg, PackedMoments)
        m, v = (None, None) if packed else (C.byref(opt.exp_avg.struct()), C.byref(opt.exp_avg_sq.struct()))
        call("lfs_mcmc_apply", N, sd.K, n, ptr(sampled), ptr(dst), ptr(self._new_opac), ptr(self._new_scales),
             float(self._params.min_opacity), C.byref(p), m, v, st)
        if packed:
            for x in (opt.exp_avg, opt.exp_avg_sq):
                x.zero_rows(slice(N, N + n) if dst is None else sampled[:n])

    def relocate_gs(self, sampled_local: torch.Tensor | None = None) -> int:
        """mcmc.cpp:112-190. `sampled_local` (indices into the alive list) may be injected for tests."""
        sd = self._splat_data
        N = sd.size
        call("lfs_mcmc_classify", N, ptr(sd._full["opacity_raw"]), ptr(sd._full["rotation_raw"]), float(self._params.min_opacity),
             ptr(self._dead), ptr(self._alive), ptr(self._alive_opac), ptr(self._counts2), ptr(self._ws), self._ws.numel(), _stream())
        n_dead, n_alive = (int(x) for x in self._counts2.tolist())  # host read, like dead_indices.numel()
        if n_dead == 0 or n_alive == 0:
            return 0
        if sampled_local is None:
            sampled_local = self.multinomial_sample(self._alive_opac[:n_alive], n_dead, True)
        call("lfs_mcmc_map_indices", n_dead, ptr(sampled_local), ptr(self._alive), ptr(self._sampled), _stream())
        self._relocate_with(self._sampled, self._dead, n_dead)
        return n_dead

    def add_new_gs(self, sampled: torch.Tensor | None = None) -> int:
        """mcmc.cpp:192-347."""
        sd, opt = self._splat_data, self._optimizer
        current_n = sd.size
        n_target = min(self._params.max_cap, int(np.float32(1.05) * np.float32(current_n)))
        n_new = max(0, n_target - current_n)
        if n_new == 0:
            return 0
        if current_n + n_new > sd.capacity:
            raise RuntimeError("SplatData capacity exhausted: reserve max_cap rows")
        if sampled is None:
            probs = torch.sigmoid(sd.tensor("opacity_raw")).flatten()
            sampled = self.multinomial_sample(probs, n_new, True)
        self._relocate_with(sampled, None, n_new)
        for s in (sd, opt.exp_avg, opt.exp_avg_sq, self.grads):
            s.size = current_n + n_new
        self._grads_valid = False   # the reference concatenates into new leaves without .grad (mcmc.cpp:254-259)
        return n_new

    def inject_noise(self, noise: torch.Tensor | None = None):
        """mcmc.cpp:349-367."""
        sd = self._splat_data
        current_lr = float(np.float32(self._optimizer.lr[0])) * self._noise_lr
        if noise is None:
            noise = self._noise[: sd.size]
            noise.normal_()  # torch::randn_like
        call("lfs_add_noise", sd.size, ptr(sd._full["opacity_raw"]), ptr(sd._full["scaling_raw"]), ptr(sd._full["rotation_raw"]),
             ptr(noise), ptr(sd._full["means"]), current_lr, _stream())


def _rewrite_rows(buffers, old_n: int, new_n: int, new_rows):
    """Replace the live rows of several buffers (parameters, moments) by new_rows(index of the buffer, group, its old rows), one
    group at a time: besides the buffers there are never more than the old and the new rows of one group (moments in 8 bits are
    decoded for this). Counterpart of update_param_with_optimizer (src/training/strategies/strategy_utils.cpp:57) on
    capacity-reserved storage. new_rows reads nothing but the rows that it is given."""
    for sd in buffers:
        if new_n > sd.capacity:
            raise RuntimeError("SplatData capacity exhausted: reserve more rows")
    for i, sd in enumerate(buffers):
        for name in PARAM_NAMES:
            sd.size = old_n
            rows = new_rows(i, name, sd.tensor(name))
            sd.size = new_n
            sd.put(name, rows)


class DefaultStrategy(IStrategy):
    """Adaptive density control of the original 3DGS (src/training/strategies/default_strategy.cpp):
    duplicate small / split large Gaussians with a high image-plane gradient, prune transparent or huge
    ones, reset opacities periodically. `densification_info` [2, N] (visibility count, accumulated
    image-plane gradient norm) is an input: the reference's gsplat path does not fill it either; its
    default EWA rasterizer does."""

    def __init__(self, splat_data: SplatData):
        self._splat_data = splat_data
        self._params = None
        self._optimizer = None
        self._scheduler = None
        self.grads = splat_data.like()
        self.active_sh_degree = 0
        self.densification_info = None
        self._grads_valid = True   # see MCMC: row surgery invalidates this iteration's gradients

    @dataclass
    class Parameters(OptimizationParameters):
        grad_threshold: float = 0.0002
        prune_opacity: float = 0.005
        grow_scale3d: float = 0.01
        prune_scale3d: float = 0.1
        reset_every: int = 3_000
        pause_refine_after_reset: int = 0
        revised_opacity: bool = False

    # ------------------------------------------------------------------ IStrategy
    def initialize(self, optim_params):
        p = self._params = optim_params
        sd = self._splat_data
        self.densification_info = torch.zeros((2, sd.size), dtype=torch.float32, device=sd.device)
        lrs = [p.means_lr * p.scene_scale, p.shs_lr, p.shs_lr / 20.0, p.scaling_lr, p.rotation_lr, p.opacity_lr]
        self._optimizer = make_optimizer(sd, lrs, p)
        self._scheduler = ExponentialLR(self._optimizer, 0.01 ** (1.0 / p.iterations), 0)

    def is_refining(self, iter: int) -> bool:
        p = self._params
        return iter > p.start_refine and iter % p.refine_every == 0 and iter % p.reset_every >= p.pause_refine_after_reset

    def get_model(self) -> SplatData:
        return self._splat_data

    def remove_gaussians(self, mask: torch.Tensor):
        if int(mask.sum()) == 0:
            return
        self.remove(mask)

    def post_backward(self, iter: int, render_output=None):
        p = self._params
        if iter % p.sh_degree_interval == 0:
            self.active_sh_degree = min(self.active_sh_degree + 1, p.sh_degree)
        if iter == p.stop_refine:
            self.densification_info = torch.empty(0)
        if iter >= p.stop_refine:
            return
        if self.is_refining(iter):
            self.grow_gs(iter)
            self.prune_gs(iter)
            self.densification_info = torch.zeros((2, self._splat_data.size), dtype=torch.float32, device=self._splat_data.device)
        if iter % p.reset_every == 0 and iter > 0:
            self.reset_opacity()

    def step(self, iter: int, grad_scale: float = 1.0):
        """default_strategy.cpp step(): duplicate / split / remove go through update_param_with_optimizer
        (strategy_utils.cpp:57), whose new leaf tensors have no .grad, so on those iterations FusedAdam::step skips every
        group before counting the step; the scheduler still runs."""
        if iter < self._params.iterations:
            if self._grads_valid:
                self._optimizer.step(iter, self.grads, grad_scale)
            self._grads_valid = True
            self._optimizer.zero_grad(True, iter)
            self._scheduler.step()

    # ------------------------------------------------------------------ pieces
    def _buffers(self):
        return (self._splat_data, self._optimizer.exp_avg, self._optimizer.exp_avg_sq)

    def _sync_sizes(self):
        n = self._splat_data.size
        for sd in (self._optimizer.exp_avg, self._optimizer.exp_avg_sq, self.grads):
            sd.size = n

    def _activated(self):
        sd = self._splat_data
        return torch.sigmoid(sd.tensor("opacity_raw")).squeeze(-1), torch.exp(sd.tensor("scaling_raw")), \
            torch.nn.functional.normalize(sd.tensor("rotation_raw"), dim=-1)

    def duplicate(self, is_duplicated: torch.Tensor):
        """default_strategy.cpp:49-87: append copies of the selected rows; their moments start at zero."""
        self._sync_sizes()
        idx = is_duplicated.nonzero().squeeze(-1)
        n, k = self._splat_data.size, int(idx.numel())

        def rows(buffer, name, old):
            extra = old.index_select(0, idx) if buffer == 0 else torch.zeros((k,) + tuple(old.shape[1:]), dtype=old.dtype, device=old.device)
            return torch.cat([old, extra], 0)

        _rewrite_rows(self._buffers(), n, n + k, rows)
        self._sync_sizes()
        self._grads_valid = False

    def split(self, is_split: torch.Tensor, noise: torch.Tensor | None = None):
        """default_strategy.cpp:89-159: each selected Gaussian is replaced by two samples of itself with scale / 1.6;
        the rest keep their order, the new rows are appended, their moments start at zero."""
        from . import ops
        self._sync_sizes()
        sd = self._splat_data
        idx = is_split.nonzero().squeeze(-1)
        rest = (~is_split.bool()).nonzero().squeeze(-1)
        k = int(idx.numel())
        _, scales, quats = self._activated()
        s_scales, s_quats = scales.index_select(0, idx), quats.index_select(0, idx).contiguous()
        rotmats = ops.quats_to_rotmats(s_quats)  # [k, 3, 3]
        if noise is None:
            noise = torch.randn((2, k, 3), dtype=torch.float32, device=sd.device)
        samples = torch.einsum("nij,nj,bnj->bni", rotmats, s_scales, noise)  # [2, k, 3]

        def rows(buffer, name, old):
            kept = old.index_select(0, rest)
            if buffer > 0:
                new = torch.zeros((2 * k,) + tuple(old.shape[1:]), dtype=old.dtype, device=old.device)
            else:
                sel = old.index_select(0, idx)
                if name == "means":
                    new = (sel.unsqueeze(0) + samples).reshape(-1, 3)
                elif name == "scaling_raw":
                    new = torch.log(s_scales / 1.6).repeat(2, 1)
                elif name == "opacity_raw" and self._params.revised_opacity:
                    new = torch.logit(1.0 - torch.sqrt(1.0 - torch.sigmoid(sel))).repeat(2, 1)
                else:
                    new = sel.repeat((2,) + (1,) * (sel.dim() - 1))
            del old
            return torch.cat([kept, new], 0)

        _rewrite_rows(self._buffers(), sd.size, int(rest.numel()) + 2 * k, rows)
        self._sync_sizes()
        self._grads_valid = False

    def grow_gs(self, iter: int):
        """default_strategy.cpp:161-189."""
        p, sd = self._params, self._splat_data
        info = self.densification_info
        grads = info[1] / torch.clamp_min(info[0], 1.0)
        _, scales, _ = self._activated()
        is_grad_high = grads > p.grad_threshold
        is_small = scales.max(-1).values <= p.grow_scale3d * p.scene_scale
        is_duplicated = is_grad_high & is_small
        num_dup = int(is_duplicated.sum())
        is_split = is_grad_high & ~is_small
        num_split = int(is_split.sum())
        if num_dup > 0:
            self.duplicate(is_duplicated)
        is_split = torch.cat([is_split, torch.zeros(num_dup, dtype=torch.bool, device=sd.device)])
        if num_split > 0:
            self.split(is_split)

    def remove(self, is_prune: torch.Tensor):
        """default_strategy.cpp:191-219."""
        self._sync_sizes()
        keep = (~is_prune.bool()).nonzero().squeeze(-1)
        _rewrite_rows(self._buffers(), self._splat_data.size, int(keep.numel()), lambda _, name, rows: rows.index_select(0, keep))
        self._sync_sizes()
        self._grads_valid = False

    def prune_gs(self, iter: int):
        """default_strategy.cpp:221-241."""
        p, sd = self._params, self._splat_data
        opac, scales, _ = self._activated()
        is_prune = opac < p.prune_opacity
        rot = sd.tensor("rotation_raw")
        is_prune |= (rot * rot).sum(-1) < 1e-8
        if iter > p.reset_every:
            is_prune |= scales.max(-1).values > p.prune_scale3d * p.scene_scale
        if int(is_prune.sum()) > 0:
            self.remove(is_prune)

    def reset_opacity(self):
        """default_strategy.cpp:243-282: clamp the logits at logit(2 prune_opacity), zero the opacity moments."""
        thr = torch.logit(torch.tensor(2.0 * self._params.prune_opacity)).item()
        self._sync_sizes()
        self._splat_data.tensor("opacity_raw").clamp_(max=thr)
        for moment in (self._optimizer.exp_avg, self._optimizer.exp_avg_sq):
            moment.put("opacity_raw", torch.zeros_like(moment.tensor("opacity_raw")))
