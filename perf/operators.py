"""The optimizer and embedding operators of a training run, as cases that can be timed one by one.

A case is a dict of plain values; its "op" says which operators it goes through:

  adamw     one AdamW step over a list of tensors. Decoupled weight decay, moments in 32 bits, or in 8 bits with one 32-bit
            scale per block of 128 elements (e4m3 for the first moment, e5m2 for the second, rounded up or down by a threshold
            that depends on the element and the step). "set" names the tensors: "splats" the six parameter groups of a
            Gaussian scene, "images" per-image codes and exposure matrices, "grids" per-image bilateral grids, codes and a
            small colour network
  lookup    out[i] = scale * table[indices[i]], zeros where an index names no row of the table
  gradient  its gradient: v_table[r] = scale * sum of v_out[i] over the i with indices[i] = r, from the indices' sorted order.
            That order is made in the pass ("order": "made") or kept where the indices stay the same from step to step
  palette   one step of fine-tuning a palette of spherical-harmonics rows: lookup, gradient and AdamW together

`own` false: elementary torch operations. `own` true: the calls of this framework."""
from __future__ import annotations

import importlib
import math

import torch

own = False

BLOCK = 128                     # elements that share a scale
TINY = 2.0 ** -110              # a block whose largest magnitude is below it is held as zeros
BETAS, EPS = (0.9, 0.999), 1e-15
DTYPES = {"f32": torch.float32, "bf16": torch.bfloat16, "f16": torch.float16}
SIZES = {"f32": 4, "bf16": 2, "f16": 2}
SPLAT_LRS = [1.6e-6, 2.5e-5, 1.25e-6, 5e-5, 1e-5, 5e-4]   # the end of the schedule: a scene stays what it is over many passes


def _package():
    return importlib.import_module("lichtfeld-studio_b200")


# ---------------------------------------------------------------------------------------------- cases
def _adamw(name, set, n, bits, grad="f32", K=16, decay=0.0):
    c = dict(op="adamw", set=set, n=n, bits=bits, grad=grad, K=K, decay=decay)
    return dict(c, name=name) if name else c


def _rows(name, op, n, rows, width, table="f32", out="f32", index_bits=32, spread="clusters", order="made"):
    c = dict(op=op, n=n, rows=rows, width=width, table=table, out=out, index_bits=index_bits, spread=spread, order=order)
    return dict(c, name=name) if name else c


def listed():
    return [
        # codes and exposure matrices of a capture's 200 images, every one a tensor of its own: the time of one launch
        _adamw("adamw32_images_200", "images", 200, 32, decay=1e-2),
        # the benchmark's scene, moments in 32 bits
        _adamw("adamw32_splats_1m", "splats", 1_000_000, 32, decay=1e-3),
        # a scene soon after its structure-from-motion start, SH degree 2, groups of odd length that end inside a block
        _adamw("adamw8_splats_120k", "splats", 120_003, 8, K=9),
        # bilateral grids, codes and a colour network whose gradients come out of torch in bfloat16
        _adamw("adamw8_grids_400_bf16", "grids", 400, 8, grad="bf16", decay=1e-2),
        # the large scene, where 8-bit moments save a gigabyte
        _adamw("adamw8_splats_3m", "splats", 3_000_000, 8, decay=1e-3),
        # codes of the 64 views of a batch
        _rows("lookup_codes_64", "lookup", 64, 200, 32, index_bits=64, spread="images"),
        # SH rows of degree 3 from the largest palette a compressed scene has
        _rows("lookup_palette_1m", "lookup", 1_000_000, 65_536, 45),
        # a palette kept in half precision, SH degree 2, a large scene
        _rows("lookup_half_3m", "lookup", 3_000_000, 32_768, 24, table="f16"),
        # the gradient of the batch's codes: the indices are new in every step
        _rows("gradient_codes_64", "gradient", 64, 200, 32, index_bits=64, spread="images"),
        # every Gaussian reads the code of one of the four cameras of a step, and a network returns the gradient in bfloat16
        _rows("gradient_cameras_400k_bf16", "gradient", 400_003, 200, 16, out="bf16", index_bits=64, spread="cameras"),
        # the palette's gradient; labels stay the same, so the order is kept
        _rows("gradient_palette_1m", "gradient", 1_000_000, 65_536, 45, order="kept"),
        # a step of palette fine-tuning on the large scene
        _rows("palette_step_3m", "palette", 3_000_000, 65_536, 45, order="kept"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["adamw", "adamw", "lookup", "gradient", "palette"])
    if op == "adamw":
        kind = rng.choice(["splats", "splats", "images", "grids"])
        n = _log(rng, 1, 2_000_000) if kind == "splats" else _log(rng, 1, 400)
        return _adamw(None, kind, n, rng.choice([8, 32]), grad=rng.choice(["f32", "f32", "bf16", "f16"]), K=rng.choice([1, 4, 9, 16]),
                      decay=rng.choice([0.0, 1e-3, 1e-2]))
    width = rng.choice([9, 24, 45, rng.randint(1, 64), rng.randint(65, 300)])
    n = max(1, _log(rng, 1, 2_000_000) * 45 // max(45, width))
    rows = _log(rng, 1, 65_536)
    spread = rng.choice(["clusters", "images", "cameras"])
    bits = rng.choice([32, 64])
    if op == "palette":
        return _rows(None, op, n, rows, width, index_bits=bits, spread=spread, order="kept")
    if op == "lookup":
        table = rng.choice(["f32", "f32", "bf16", "f16"])
        return _rows(None, op, n, rows, width, table=table, out=rng.choice(["f32", table]), index_bits=bits, spread=spread)
    return _rows(None, op, n, rows, width, out=rng.choice(["f32", "f32", "bf16", "f16"]), index_bits=bits, spread=spread,
                 order=rng.choice(["made", "kept"]))


def _tensors(case):
    """[(tensors of this kind, elements of each, row width, learning rate)] of an AdamW case."""
    n, K = case["n"], case["K"]
    if case["set"] == "splats":
        groups = [(1, n * w, w, lr) for w, lr in zip((3, 3, (K - 1) * 3, 3, 4, 1), SPLAT_LRS)]
        return [g for g in groups if g[1]]
    if case["set"] == "images":
        return [(n, 32, 32, 1e-5), (n, 12, 12, 1e-6)]
    layers = [(64 * 77, 77), (64, 64), (64 * 64, 64), (64, 64), (3 * 64, 64), (3, 3)]
    return [(1, n * 12 * 8 * 16 * 16, 256, 2e-5), (1, n * 32, 32, 1e-5)] + [(1, m, w, 1e-5) for m, w in layers]


def work(case):
    if case["op"] == "adamw":
        n = sum(t[0] * t[1] for t in _tensors(case))
        moments = 16 if case["bits"] == 32 else 4 + 16 / BLOCK
        return {"bytes": n * (8 + SIZES[case["grad"]] + moments), "flops": 16 * n}
    n, rows, width = case["n"], case["rows"], case["width"]
    index, read = n * case["index_bits"] // 8, min(n, rows) * width * SIZES[case["table"]]
    lookup = index + read + n * width * SIZES[case["out"]]
    gradient = index + n * width * SIZES[case["out"]] + rows * width * 4
    if case["op"] == "lookup":
        return {"bytes": lookup, "flops": n * width}
    if case["op"] == "gradient":
        return {"bytes": gradient, "flops": n * width + rows * width}
    step = rows * width * (8 + 4 + 4 + 16 / BLOCK)
    return {"bytes": lookup + gradient + step, "flops": 2 * n * width + 17 * rows * width}


# ---------------------------------------------------------------------------------------------- inputs
def _gradients(gen, n, width, dtype):
    """Gradients of rows: a third of the rows did not take part, the others differ in size by orders of magnitude."""
    rows = -(-n // width)
    size = torch.exp(torch.randn(rows, 1, device="cuda", generator=gen) * 1.5 - 9.0)
    size *= torch.rand(rows, 1, device="cuda", generator=gen) > 1 / 3
    g = torch.randn(rows, width, device="cuda", generator=gen) * size
    return g.reshape(-1)[:n].contiguous().to(dtype), size


def _moments(gen, n, width, size):
    """Moments of a run under way: the first a tenth of the gradients' size, the second their mean square."""
    rows = -(-n // width)
    m = torch.randn(rows, width, device="cuda", generator=gen) * (0.3 * size + 1e-6)
    v = (0.5 + torch.rand(rows, width, device="cuda", generator=gen)) * (size + 1e-6).square()
    return m.reshape(-1)[:n].contiguous(), v.reshape(-1)[:n].contiguous()


def _blocks(x):
    """[tensors, elements] -> [tensors, blocks, BLOCK], zeros behind the last element."""
    return torch.nn.functional.pad(x, (0, -x.shape[1] % BLOCK)).unflatten(1, (-1, BLOCK))


def _over(scale, n):
    """One value per block -> one per element."""
    return scale[:, :, None].expand(-1, -1, BLOCK).flatten(1)[:, :n]


def _hold(x, top, dtype):
    """Values as 8-bit floats of `dtype`, rounded to the nearest, with a scale per block (the state that a run starts from)."""
    scale = _blocks(x).abs().amax(2) * torch.tensor(1.0 / top, dtype=torch.float32, device=x.device)
    return (x / _over(torch.clamp_min(scale, 1e-38), x.shape[1])).clamp(-top, top).to(dtype), scale


def _optimizer_state(gen, shape, width, lr, bits, decay, gradient):
    g, size = gradient
    t = dict(p=torch.randn(shape, device="cuda", generator=gen), g=g.view(shape), lr=lr, decay=decay)
    m, v = (x.view(shape) for x in _moments(gen, shape[0] * shape[1], width, size))
    if bits == 8:
        t["m"], t["ms"] = _hold(m, 448.0, torch.float8_e4m3fn)
        t["v"], t["vs"] = _hold(v, 57344.0, torch.float8_e5m2)
    else:
        t["m"], t["v"], t["ms"], t["vs"] = m, v, None, None
    return t


def _state(tensors):
    return [{k: t[k] for k in ("p", "m", "v", "ms", "vs") if t[k] is not None} for t in tensors]


def _indices(case, gen):
    n, rows = case["n"], case["rows"]
    u = torch.rand(n, device="cuda", generator=gen, dtype=torch.float64)
    if case["spread"] == "clusters":      # clusters of a scene differ in size
        index = (u * u * rows).long()
        mix = torch.randperm(rows, device="cuda", generator=gen)
        index = mix[index.clamp(max=rows - 1)]
    elif case["spread"] == "cameras":     # everything reads one of four rows
        some = torch.randint(rows, (4,), device="cuda", generator=gen)
        index = some[(u * 4).long()]
    else:                                 # any image; some views have no code
        index = (u * rows).long()
        index[torch.rand(n, device="cuda", generator=gen) < 0.05] = -1
    return index.to(torch.int32 if case["index_bits"] == 32 else torch.int64)


def _handle(pkg, kinds):
    """The optimizer over all tensors; the tensors of a kind lie behind one another in memory."""
    parts = [{k: None if t[k] is None else t[k][i] for k in ("p", "g", "m", "v", "ms", "vs")} | dict(lr=t["lr"], decay=t["decay"])
             for t in kinds for i in range(t["p"].shape[0])]
    opt = pkg.strategy.AdamW([t["p"] for t in parts], [t["g"] for t in parts], lr=[t["lr"] for t in parts], betas=BETAS, eps=EPS,
                             weight_decay=[t["decay"] for t in parts],
                             moments=[pkg.strategy.Moments(t["m"], t["v"], t["ms"], t["vs"]) for t in parts])
    opt.step_count = 1000
    return opt


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(int(seed) * 7919 + 17)
    s = dict(case=dict(case), step=1000)
    if case["op"] == "adamw":
        s["tensors"] = [_optimizer_state(gen, (many, n), w, lr, case["bits"], case["decay"], _gradients(gen, many * n, w, DTYPES[case["grad"]]))
                        for many, n, w, lr in _tensors(case)]
        s["learned"] = _state(s["tensors"])
        if own:
            s["opt"] = _handle(_package(), s["tensors"])
        return s
    n, rows, width = case["n"], case["rows"], case["width"]
    s["scale"] = 1.0 if case["op"] == "palette" else 0.5 * math.sqrt(width)
    s["indices"] = _indices(case, gen)
    if case["op"] in ("lookup", "palette"):
        s["table"] = (torch.randn(rows, width, device="cuda", generator=gen) * 0.05).to(DTYPES[case["table"]])
    if case["op"] in ("gradient", "palette"):
        s["v_out"] = _gradients(gen, n * width, width, DTYPES[case["out"]])[0].reshape(n, width)
    if case["op"] == "palette":
        size = torch.full((rows, 1), 1e-3, device="cuda")
        s["v_table"] = torch.zeros(rows, width, device="cuda")
        t = _optimizer_state(gen, (1, rows * width), width, 1e-6, 8, 0.0, (s["v_table"], size))
        s["tensors"] = [dict(t, p=s["table"].view(1, -1))]
        s["learned"] = _state(s["tensors"])
    if own and case["order"] == "kept":   # labels that stay the same: their order is made once
        s["order"] = _package().ops.embedding_sort(s["indices"], rows)
    if own and case["op"] == "palette":
        s["opt"] = _handle(_package(), s["tensors"])
    return s


# ---------------------------------------------------------------------------------------------- plain forms
def _threshold(n, step, first, second, bits, device):
    """`bits` bits per element: the upper ones of element * first + step * second modulo 2^32."""
    h = torch.arange(n, device=device) * first + (step * second) % 2 ** 32
    return ((h & 0xFFFFFFFF) >> (32 - bits)).to(torch.int32)


def _float8(x, threshold, dropped, least):
    """|x| with `dropped` bits of its fraction rounded off (in 2^dropped-ths, up where the threshold carries), evenly spaced below `least`."""
    small = x < least
    t = torch.where(small, x + least, x)
    bits = (t.view(torch.int32) + threshold) >> dropped << dropped
    y = bits.view(torch.float32)
    return torch.where(small, y - least, y)


def _held(x, top, step, first, second, dropped, least, dtype, positive):
    """32-bit values -> 8-bit values and the scale of every block."""
    n = x.shape[1]
    a = x.abs()
    finite = torch.isfinite(x)
    most = _blocks(torch.where(finite, a, torch.zeros_like(a))).amax(2)
    flushed = most < TINY
    inverse = torch.where(flushed, torch.zeros_like(most), torch.full_like(most, top) / torch.where(flushed, torch.ones_like(most), most))
    scale = torch.where(flushed, torch.zeros_like(most), most * torch.full_like(most, 1.0 / top))
    inverse = _over(inverse, n)
    y = _float8((a * inverse).clamp(max=top), _threshold(n, step, first, second, dropped, x.device), dropped, least)
    if positive:   # what is not zero is not held as zero
        y = torch.where((x > 0) & (inverse > 0), y.clamp(min=least / 2.0 ** (23 - dropped)), y)
    y = torch.copysign(y, x)
    y = torch.where(finite, y, x if positive else torch.full_like(x, math.nan))
    return y.to(dtype), scale


def _adamw_plain(t, step):
    n = t["p"].shape[1]
    b1, b2 = BETAS
    g = t["g"].float()
    m, v = t["m"], t["v"]
    if t["ms"] is not None:
        m, v = m.float() * _over(t["ms"], n), v.float() * _over(t["vs"], n)
    m = m * b1 + g * (1 - b1)
    v = v * b2 + (g * (1 - b2)) * g
    size = t["lr"] * (1 / (1 - b1 ** step))
    p = t["p"] * (1 - t["lr"] * t["decay"])
    t["p"].copy_(p - (m * size) / (torch.sqrt(v) * (1 / math.sqrt(1 - b2 ** step)) + EPS))
    if t["ms"] is None:
        t["m"].copy_(m), t["v"].copy_(v)
        return
    m, ms = _held(m, 448.0, step, 0x91E10DA5, 0x9E3779B9, 20, 2.0 ** -6, torch.float8_e4m3fn, False)
    v, vs = _held(v, 57344.0, step, 0x9E3779B9, 0xC13FA9A9, 21, 2.0 ** -14, torch.float8_e5m2, True)
    t["m"].copy_(m), t["v"].copy_(v), t["ms"].copy_(ms), t["vs"].copy_(vs)


def _lookup_plain(table, indices, scale, dtype):
    valid = (indices >= 0) & (indices < table.shape[0])
    rows = table.float()[torch.where(valid, indices, torch.zeros_like(indices)).long()]
    return torch.where(valid[:, None], rows * scale, torch.zeros_like(rows)).to(dtype)


def _gradient_plain(v_out, indices, rows, scale):
    valid = (indices >= 0) & (indices < rows)
    total = torch.zeros(rows + 1, v_out.shape[1], device=v_out.device, dtype=torch.float64)   # one row more for indices of no row
    total.index_add_(0, torch.where(valid, indices, torch.full_like(indices, rows)).long(), v_out.double())
    return (total[:rows] * scale).float()


# ---------------------------------------------------------------------------------------------- a pass
def run(s):
    case = s["case"]
    s["step"] += 1
    if own:
        ops = _package().ops
        if case["op"] == "adamw":
            s["opt"].step()
            return s["learned"]
        if case["op"] == "lookup":
            return ops.embedding_fwd(s["table"], s["indices"], s["scale"], out_dtype=DTYPES[case["out"]])
        if case["op"] == "gradient":
            order = s["order"] if case["order"] == "kept" else ops.embedding_sort(s["indices"], case["rows"])
            return ops.embedding_bwd(s["v_out"], order, s["scale"])
        out = ops.embedding_fwd(s["table"], s["indices"], s["scale"])
        ops.embedding_bwd(s["v_out"], s["order"], s["scale"], out=s["v_table"])
        s["opt"].step()
        return [out, s["learned"]]
    if case["op"] == "adamw":
        for t in s["tensors"]:
            _adamw_plain(t, s["step"])
        return s["learned"]
    if case["op"] == "lookup":
        return _lookup_plain(s["table"], s["indices"], s["scale"], DTYPES[case["out"]])
    if case["op"] == "gradient":
        return _gradient_plain(s["v_out"], s["indices"], case["rows"], s["scale"])
    out = _lookup_plain(s["table"], s["indices"], s["scale"], torch.float32)
    s["v_table"].copy_(_gradient_plain(s["v_out"], s["indices"], case["rows"], s["scale"]))
    _adamw_plain(s["tensors"][0], s["step"])
    return [out, s["learned"]]


# ---------------------------------------------------------------------------------------------- the definition in 64 bits
def _exact_held(x, top, fraction_bits, lowest, thresholds, keep_positive):
    """x[i] times top / (largest of its block), as a float of `fraction_bits` whose lowest binade is 2^lowest, rounded down where the
    fraction of a last place plus thresholds[i] stays below one and up where it does not."""
    n = x.shape[-1]
    block = torch.arange(n, device=x.device) // BLOCK
    most = torch.stack([torch.zeros(n // BLOCK + 1, dtype=x.dtype, device=x.device).scatter_reduce(0, block, row.abs(), "amax")
                        for row in x])[:, :-(-n // BLOCK)]
    scale = torch.where(most >= TINY, most / top, torch.zeros_like(most))
    each = scale[:, block]
    y = torch.where(each > 0, x.abs() / each, torch.zeros_like(x))
    _, exponent = torch.frexp(y)                                    # y = [0.5, 1) * 2^exponent
    place = torch.ldexp(torch.ones_like(y), (exponent - 1).clamp(min=lowest) - fraction_bits)
    y = (torch.floor(y / place + thresholds) * place).clamp(max=top)
    if keep_positive:
        y = torch.where((x > 0) & (each > 0), y.clamp(min=2.0 ** (lowest - fraction_bits)), y)
    return torch.where(x < 0, -y, y), scale


def _exact_adamw(t, step):
    n, (b1, b2) = t["p"].shape[1], BETAS
    p, g, m, v = (t[k].double() for k in ("p", "g", "m", "v"))
    i = torch.arange(n, device=p.device)
    if t["ms"] is not None:
        m, v = m * t["ms"].double()[:, i // BLOCK], v * t["vs"].double()[:, i // BLOCK]
    m, v = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
    p = p - t["lr"] * t["decay"] * p - t["lr"] * (m / (1 - b1 ** step)) / (torch.sqrt(v / (1 - b2 ** step)) + EPS)
    if t["ms"] is None:
        return dict(p=p, m=m, v=v)
    first = (i * 0x91E10DA5 + step * 0x9E3779B9) % 2 ** 32 // 2 ** 12 / 2.0 ** 20
    second = (i * 0x9E3779B9 + step * 0xC13FA9A9) % 2 ** 32 // 2 ** 11 / 2.0 ** 21
    m, ms = _exact_held(m, 448.0, 3, -6, first, False)
    v, vs = _exact_held(v, 57344.0, 2, -14, second, True)
    return dict(p=p, m=m, v=v, ms=ms, vs=vs)


def _exact_gradient(v_out, indices, rows, scale):
    """Differences of running sums over the lookups in the order of their rows."""
    keep = (indices >= 0) & (indices < rows)
    row, at = torch.sort(indices[keep].long(), stable=True)
    total = torch.nn.functional.pad(v_out[keep][at].double().cumsum(0), (0, 0, 1, 0))
    ends = torch.searchsorted(row, torch.arange(rows + 1, device=row.device))
    return scale * (total[ends[1:]] - total[ends[:-1]])


def exact(case, seed):
    s = prepare(case, seed)
    step = s["step"] + 1
    if case["op"] == "adamw":
        return [_exact_adamw(t, step) for t in s["tensors"]]
    if case["op"] in ("lookup", "palette"):
        out = torch.zeros(case["n"], case["width"], device="cuda", dtype=torch.float64)
        keep = (s["indices"] >= 0) & (s["indices"] < case["rows"])
        out[keep] = s["table"].double()[s["indices"][keep].long()] * s["scale"]
        if case["op"] == "lookup":
            return out
    gradient = _exact_gradient(s["v_out"], s["indices"], case["rows"], s["scale"])
    if case["op"] == "gradient":
        return gradient
    return [out, [_exact_adamw(dict(s["tensors"][0], g=gradient.view(1, -1)), step)]]
