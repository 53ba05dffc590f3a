"""Workloads of the routed (mixture of experts) MLP operators and of the 4-bit
products: the calls a user's program makes, the same results in elementary
torch operations, and each result's definition in 64 bits.

Operators (case["op"]):
  sort      slots (token, choice) sorted by expert: counts, offsets, both maps
  exchange  one training pass of the rows' way to the experts and back:
            dispatch, weighted combine, and the gradients of both
  quantize  blocks of a matrix to 4-bit elements with a scale per block, and
            the values they stand for
  gemm      product of two 4-bit matrices, dense or by expert
  swiglu    gate and up products of 4-bit matrices with silu(g) * u, dense or
            by expert

`own` false: plain torch; true: this package's kernels.
"""
from __future__ import annotations

import functools
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "f16": torch.float16, "f32": torch.float32}
BLOCK = {"mx": 32, "nv": 16}
VALUES = (0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0)
DEVICE = "cuda"


# ---- cases ---------------------------------------------------------------------------

def listed():
    return [
        # A decode step of 64 sequences: the smallest call, latency only.
        dict(name="sort_decode", op="sort", tokens=64, topk=8, experts=128, first=0, total=128,
             align=128, ids="i32"),
        # A long prompt batch over many experts; ids as torch's topk gives them.
        dict(name="sort_prefill", op="sort", tokens=32768, topk=8, experts=256, first=0, total=256,
             align=128, ids="i64"),
        # A training micro-batch at the MLP chain's hidden size.
        dict(name="exchange_train", op="exchange", tokens=8192, topk=8, hidden=4096, experts=64,
             first=0, total=64, align=1, dtype="bf16"),
        # A ragged small batch whose experts are partly elsewhere, an odd hidden size, fp32.
        dict(name="exchange_odd", op="exchange", tokens=61, topk=4, hidden=1001, experts=12,
             first=4, total=20, align=8, dtype="f32"),
        # Activations of a prompt at the hidden size of the GEMM benchmarks.
        dict(name="quantize_acts", op="quantize", rows=8192, cols=8192, format="mx", dtype="bf16",
             transpose=False, scale=1.0, topk=0),
        # A down projection's weights [k, n] of one of eight GPUs, once per load or training step.
        dict(name="quantize_weight", op="quantize", rows=8192, cols=3584, format="nv",
             dtype="bf16", transpose=True, scale=256.0, topk=0),
        # The rows of a decode batch gathered to their experts while they are quantised.
        dict(name="quantize_routed", op="quantize", rows=256, cols=4096, format="nv", dtype="f16",
             transpose=False, scale=16.0, topk=8, experts=64, first=0, total=64),
        # A prompt through a square projection of the GEMM benchmarks' size.
        dict(name="gemm_prefill", op="gemm", m=4096, n=8192, k=8192, format="mx", dtype="bf16",
             experts=0),
        # A decode step through one of eight GPUs' slice of the down projection.
        dict(name="gemm_decode", op="gemm", m=16, n=8192, k=3584, format="nv", dtype="bf16",
             experts=0),
        # Experts' products over ragged groups, odd widths, fp32 out (a gradient's accumulation).
        dict(name="gemm_experts_ragged", op="gemm", m=1500, topk=2, n=1001, k=1120, format="mx",
             dtype="f32", experts=16),
        # One tensor-parallel MLP block's gate and up projection (one of eight GPUs).
        dict(name="swiglu_block", op="swiglu", m=2048, n=1792, k=4096, format="nv", dtype="bf16",
             experts=0),
        # A decode batch through every expert's gate and up weights: weight bound.
        dict(name="swiglu_experts_decode", op="swiglu", m=64, topk=8, n=1024, k=4096, format="mx",
             dtype="bf16", experts=64),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    limit = {op: max(_cost(c) for c in listed() if c["op"] == op)
             for op in ("sort", "exchange", "quantize", "gemm", "swiglu")}
    while True:
        case = _draw(rng)
        if _cost(case) <= limit[case["op"]]:
            return case


def _cost(case):
    w = work(case)
    return w["bytes"] / 6.5e12 + w["flops"] / 6.5e15


def _draw(rng):
    op = rng.choice(("sort", "exchange", "quantize", "gemm", "swiglu"))
    total = _log(rng, 4, 256)
    experts = total if rng.random() < 0.6 else max(1, total // rng.choice((2, 4)))
    first = rng.choice((0, total - experts))
    topk = min(total, rng.randint(1, 8))
    if op == "sort":
        return dict(op=op, tokens=_log(rng, 1, 32768), topk=topk, experts=experts, first=first,
                    total=total, align=rng.choice((1, 8, 128)), ids=rng.choice(("i32", "i64")))
    if op == "exchange":
        return dict(op=op, tokens=_log(rng, 1, 8192), topk=topk, hidden=_log(rng, 64, 8192),
                    experts=experts, first=first, total=total, align=rng.choice((1, 8, 128)),
                    dtype=rng.choice(tuple(DTYPES)))
    fmt = rng.choice(tuple(BLOCK))
    if op == "quantize":
        kind = rng.choice(("rows", "transposed", "routed"))
        case = dict(op=op, rows=_log(rng, 1, 8192), cols=32 * _log(rng, 1, 256), format=fmt,
                    dtype=rng.choice(tuple(DTYPES)), transpose=kind == "transposed",
                    scale=2.0 ** rng.randint(0, 8), topk=0)
        if kind == "routed":
            case.update(rows=_log(rng, 1, 2048), topk=topk, experts=experts, first=first,
                        total=total)
        return case
    grouped = rng.random() < 0.5
    case = dict(op=op, m=_log(rng, 1, 4096), n=_log(rng, 64, 8192 if not grouped else 2048),
                k=32 * _log(rng, 2, 256), format=fmt, dtype=rng.choice(tuple(DTYPES)), experts=0)
    if grouped:
        case.update(m=_log(rng, 1, 2048), experts=_log(rng, 2, 64))
        case["topk"] = min(case["experts"], rng.randint(1, 8))
    return case


def _rows(case):
    """Rows at most of the sorted order (the package's own rule is the same):
    every slot, and the padding of the experts that can have any."""
    slots = case["tokens"] * case["topk"]
    most = slots + min(case["experts"], slots) * (case["align"] - 1)
    return most // case["align"] * case["align"]


def _local(case):
    """Expected rows that have an expert here."""
    return case["tokens"] * case["topk"] * case["experts"] / case["total"]


def work(case):
    op = case["op"]
    if op == "sort":
        slots = case["tokens"] * case["topk"]
        ids = 4 if case["ids"] == "i32" else 8
        return {"bytes": slots * (ids + 4) + 4 * (_rows(case) + 2 * case["experts"] + 1),
                "flops": slots}
    if op == "exchange":
        size = 4 if case["dtype"] == "f32" else 2
        slots, rows = case["tokens"] * case["topk"], _local(case)
        return {"bytes": 4 * case["hidden"] * size * (case["tokens"] + rows) + 12 * slots,
                "flops": 6 * rows * case["hidden"]}
    block = BLOCK[case["format"]]
    if op == "quantize":
        size = 4 if case["dtype"] == "f32" else 2
        rows = case["rows"] if not case["topk"] else \
            case["rows"] * case["topk"] * case["experts"] / case["total"]
        return {"bytes": case["cols"] * (case["rows"] * size + rows * (2 + 0.5 + 1.0 / block)),
                "flops": 4 * rows * case["cols"]}
    weights = (2 if op == "swiglu" else 1) * case["n"]
    rows = case["m"] * case.get("topk", 1)
    used = min(case["experts"], rows) if case["experts"] else 1
    size = 4 if case["dtype"] == "f32" else 2
    return {"bytes": (0.5 + 1.0 / block) * case["k"] * (rows + used * weights)
            + size * rows * case["n"],
            "flops": 2 * rows * weights * case["k"]}


# ---- inputs --------------------------------------------------------------------------

@functools.lru_cache(None)
def _table(values, dtype):
    return torch.tensor(values, dtype=dtype, device=DEVICE)


def _pow2(e, dtype):
    """2 ** e exactly, -149 <= e <= 127."""
    return _table(tuple(2.0 ** i for i in range(-149, 128)), dtype)[e.to(torch.int64) + 149]


def _gen(seed):
    return torch.Generator(device=DEVICE).manual_seed(seed)


def _randn(gen, shape, dtype=torch.float32, spread=0.0):
    """Normal values; with `spread`, rows of unequal size and a few outliers, as
    activations have them."""
    x = torch.randn(shape, generator=gen, device=DEVICE)
    if spread:
        x *= torch.exp(spread * torch.randn((shape[0], 1), generator=gen, device=DEVICE))
        x *= 1 + 15 * (torch.rand((1, shape[-1]), generator=gen, device=DEVICE) < 0.004)
    return x.to(dtype)


def _experts_of(gen, tokens, topk, total):
    """Distinct experts per token, some of them much more popular."""
    logits = torch.randn((tokens, total), generator=gen, device=DEVICE)
    logits += 0.7 * torch.randn((1, total), generator=gen, device=DEVICE)
    return logits.topk(topk, dim=1).indices


def _plain_quantize(x, fmt, g):
    """(codes as signed values, scales as values) of [rows, cols] blocks of g * x."""
    wide = torch.float64 if x.dtype == torch.float32 else torch.float32
    rows, cols = x.shape
    z = (x.to(wide) * g).reshape(rows, cols // BLOCK[fmt], BLOCK[fmt])
    amax = z.abs().amax(-1)
    one = torch.ones_like(amax)
    if fmt == "mx":
        e = torch.where(amax > 0, torch.frexp(amax).exponent - 3, -127).clamp(-127, 127)
        scale = _pow2(e, wide)
    else:
        v = (amax / 6).clamp(max=448)
        step = _pow2((torch.frexp(v).exponent - 1).clamp(min=-6) - 3, wide)
        scale = torch.round(v / step) * step
    safe = torch.where(scale > 0, scale, one)
    y = torch.where(scale[..., None] > 0, z / safe[..., None], torch.zeros_like(z))
    a = y.abs()
    q = torch.where(a < 2, torch.round(a * 2) / 2,
                    torch.where(a < 4, torch.round(a), torch.round(a / 2) * 2)).clamp(max=6)
    return torch.where(y < 0, -q, q), scale


def _pack(q, scale, fmt):
    """Two elements a byte, the lower nibble first; scales as bytes in tiles of
    128 rows x 4 blocks, row r of a tile at (r % 32) * 16 + (r // 32) * 4."""
    rows, nblk = scale.shape
    a = q.abs().reshape(rows, -1)
    code = torch.zeros_like(a, dtype=torch.uint8)
    for v in VALUES[1:]:
        code += (a >= v).to(torch.uint8)
    code += 8 * (q.reshape(rows, -1) < 0).to(torch.uint8)
    data = code[:, 0::2] | (code[:, 1::2] << 4)
    exponent = torch.frexp(scale).exponent - 1
    if fmt == "mx":
        byte = (exponent + 127).to(torch.uint8)
    else:
        e = exponent.clamp(min=-6)
        mant = scale * _pow2(3 - e, scale.dtype)               # 8..15, below 8 subnormal
        byte = torch.where(mant >= 8, (e + 7) * 8 + mant - 8, mant).to(torch.uint8)
    return data.contiguous(), _tile_scales(byte)


def _tile_scales(byte):
    rows, nblk = byte.shape
    rt, kt = -(-rows // 128), -(-nblk // 4)
    full = torch.zeros((rt * 128, kt * 4), dtype=torch.uint8, device=byte.device)
    full[:rows, :nblk] = byte
    return full.view(rt, 4, 32, kt, 4).permute(0, 3, 2, 1, 4).contiguous().view(-1)


def _untile_scales(tiled, rows, nblk):
    rt, kt = -(-rows // 128), -(-nblk // 4)
    full = tiled.view(rt, kt, 32, 4, 4).permute(0, 3, 2, 1, 4).reshape(rt * 128, kt * 4)
    return full[:rows, :nblk]


def _scale_values(byte, fmt, wide):
    b = byte.to(torch.int32)
    if fmt == "mx":
        return _pow2(b - 127, wide)
    e, mant = b >> 3, b & 7
    return torch.where(e > 0, (mant + 8).to(wide) * _pow2(e - 10, wide),
                       mant.to(wide) * 2.0 ** -9)


def _decode(data, scales, rows, cols, fmt, wide=torch.float32):
    """The values of a packed matrix (g not applied)."""
    table = _table(VALUES + tuple(-v for v in VALUES), wide)
    d = data.to(torch.int64)
    q = torch.stack((table[d & 15], table[d >> 4]), -1).view(rows, cols)
    s = _scale_values(_untile_scales(scales, rows, cols // BLOCK[fmt]), fmt, wide)
    return (q.view(rows, -1, BLOCK[fmt]) * s[..., None]).view(rows, cols)


def _operand(gen, rows, cols, fmt, std):
    """A quantised matrix as a user's program holds it, made in pieces."""
    x = _randn(gen, (rows, cols), torch.bfloat16, 0.3) * std
    return _pack(*_plain_quantize(x, fmt, 1.0), fmt)


def _sorted(ids, experts, first, align, capacity):
    """Plain form of the sort."""
    tokens, topk = ids.shape
    local = (ids.reshape(-1) - first).to(torch.int64)
    here = (local >= 0) & (local < experts)
    hot = (local[:, None] == torch.arange(experts, device=ids.device)).to(torch.int32)
    upto = torch.cumsum(hot, 0, dtype=torch.int32)
    counts = upto[-1].clone()
    padded = (counts + (align - 1)) // align * align
    offsets = torch.zeros(experts + 1, dtype=torch.int32, device=ids.device)
    offsets[1:] = torch.cumsum(padded, 0)
    at = local.clamp(0, experts - 1)
    rank = upto.gather(1, at[:, None])[:, 0] - 1
    row = torch.where(here, offsets[at] + rank, -1).to(torch.int32)
    slot = torch.arange(tokens * topk, dtype=torch.int32, device=ids.device)
    back = torch.full((capacity + 1,), -1, dtype=torch.int32, device=ids.device)
    back[torch.where(here, row, capacity).to(torch.int64)] = slot
    return counts, offsets, row.view(tokens, topk), back[:capacity]


def _routing(gen, tokens, topk, experts, first, total, align):
    case = dict(tokens=tokens, topk=topk, experts=experts, align=align)
    ids = _experts_of(gen, tokens, topk, total)
    return _sorted(ids, experts, first, align, _rows(case))


def prepare(case, seed):
    gen = _gen(seed)
    op = case["op"]
    st = dict(case=case)
    if op == "sort":
        ids = _experts_of(gen, case["tokens"], case["topk"], case["total"])
        st["ids"] = ids.to(torch.int32 if case["ids"] == "i32" else torch.int64)
        new = lambda *shape: torch.empty(shape, dtype=torch.int32, device=DEVICE)
        st["out"] = (new(case["experts"]), new(case["experts"] + 1),
                     new(case["tokens"], case["topk"]), new(_rows(case)))
    elif op == "exchange":
        dtype, hidden = DTYPES[case["dtype"]], case["hidden"]
        rows, tokens = _rows(case), case["tokens"]
        _, _, st["row_of_slot"], st["slot_of_row"] = _routing(
            gen, tokens, case["topk"], case["experts"], case["first"], case["total"],
            case["align"])
        st["x"] = _randn(gen, (tokens, hidden), dtype)
        st["h"] = _randn(gen, (rows, hidden), dtype)
        st["dy"] = _randn(gen, (tokens, hidden), dtype)
        st["drows"] = _randn(gen, (rows, hidden), dtype)
        st["w"] = torch.softmax(_randn(gen, (tokens, case["topk"])), -1)
        zero = lambda *shape, t=dtype: torch.zeros(shape, dtype=t, device=DEVICE)
        st["out"] = (zero(rows, hidden), zero(tokens, hidden), zero(rows, hidden),
                     zero(tokens, case["topk"], t=torch.float32), zero(tokens, hidden))
    elif op == "quantize":
        rows, cols = case["rows"], case["cols"]
        shape = (cols, rows) if case["transpose"] else (rows, cols)
        st["x"] = (_randn(gen, shape, torch.float32, 0.5) / case["scale"]).to(
            DTYPES[case["dtype"]])
        st["rows"] = rows
        if case["topk"]:
            align = 128
            _, _, _, st["slot_of_row"] = _routing(gen, rows, case["topk"], case["experts"],
                                                  case["first"], case["total"], align)
            st["rows"] = st["slot_of_row"].numel()
        st["values"] = torch.zeros((st["rows"], cols), dtype=torch.bfloat16, device=DEVICE)
    else:
        fmt, n, k = case["format"], case["n"], case["k"]
        experts = case["experts"]
        if experts:
            counts, offsets, _, _ = _routing(gen, case["m"], case["topk"], experts, 0, experts,
                                             128)
            st["counts"], st["offsets"] = counts, offsets
            st["groups"] = list(zip(offsets.tolist(), counts.tolist()))
            rows = _rows(dict(tokens=case["m"], topk=case["topk"], experts=experts, align=128))
            st["alphas"] = torch.exp2(torch.randint(-2, 3, (experts,), generator=gen,
                                                    device=DEVICE).float()) * 0.75
        else:
            rows = case["m"]
        st["rows"] = rows
        st["a"] = _operand(gen, rows, k, fmt, 1.0)
        std = 1.0 / math.sqrt(k)
        names = ("gate", "up") if op == "swiglu" else ("b",)
        for name in names:
            parts = [_operand(gen, n, k, fmt, std) for _ in range(max(1, experts))]
            st[name] = (torch.cat([p[0] for p in parts]), torch.cat([p[1] for p in parts]))
        st["out"] = torch.zeros((rows, n), dtype=DTYPES[case["dtype"]], device=DEVICE)
    if own:
        _prepare_own(st, case)
    return st


def _prepare_own(st, case):
    import megacu_b200 as mb
    op = case["op"]
    code = {"bf16": mb.DTYPE_BF16, "f16": mb.DTYPE_F16, "f32": mb.DTYPE_F32}
    if op in ("sort", "exchange"):
        st["problem"] = mb.MoeProblem(
            case["tokens"], case["topk"], case["experts"], hidden=case.get("hidden", 0),
            first_expert=case["first"], align=case["align"],
            dtype=code[case.get("dtype", "bf16")])
        st["workspace"] = torch.empty(mb.moe_workspace_bytes(st["problem"]), dtype=torch.uint8,
                                      device=DEVICE)
        return
    fmt = mb.FP4_MX if case["format"] == "mx" else mb.FP4_NV
    if op == "quantize":
        st["problem"] = mb.Fp4Matrix(st["rows"], case["cols"], format=fmt,
                                     dtype=code[case["dtype"]], transpose=case["transpose"],
                                     scale=case["scale"])
        st["decode"] = mb.Fp4Matrix(st["rows"], case["cols"], format=fmt, dtype=mb.DTYPE_BF16,
                                    scale=case["scale"])
        data, scales = mb.fp4_sizes(st["problem"])
        # Rows of padding are left as they were by both calls.
        st["data"] = torch.zeros(data, dtype=torch.uint8, device=DEVICE)
        st["scales"] = torch.zeros(scales, dtype=torch.uint8, device=DEVICE)
        return
    st["problem"] = mb.Fp4Gemm(st["rows"], case["n"], case["k"], format=fmt,
                               out_dtype=code[case["dtype"]], experts=case["experts"])
    st["events"] = torch.zeros(mb.fp4_events_bytes(), dtype=torch.uint8, device=DEVICE)


# ---- one pass ------------------------------------------------------------------------

def run(state):
    if own:
        return _run_own(state)
    case = state["case"]
    op = case["op"]
    if op == "sort":
        return _sorted(state["ids"], case["experts"], case["first"], case["align"], _rows(case))
    if op == "exchange":
        return _plain_exchange(state)
    if op == "quantize":
        x = state["x"].t() if case["transpose"] else state["x"]
        q, s = _plain_quantize(x, case["format"], case["scale"])
        v = (q * s[..., None] / case["scale"]).reshape(x.shape).to(torch.bfloat16)
        return _place(v, state)
    return _plain_product(state)


def _place(v, state):
    """Values of the quantised rows, gathered to their experts' rows if routed."""
    case = state["case"]
    if not case["topk"]:
        return v
    slot = state["slot_of_row"].to(torch.int64)
    out = v[slot.clamp(min=0) // case["topk"]]
    return torch.where(slot[:, None] >= 0, out, torch.zeros_like(out))


def _plain_exchange(st):
    row = st["row_of_slot"].to(torch.int64)
    here = (row >= 0)[..., None]
    at = row.clamp(min=0)
    slot = st["slot_of_row"].to(torch.int64)
    used = (slot >= 0)[:, None]
    token = slot.clamp(min=0) // row.shape[1]
    zero = torch.zeros((), device=row.device)
    x, h, dy, drows, w = (st[n].float() for n in ("x", "h", "dy", "drows", "w"))
    dtype = st["x"].dtype
    rows = torch.where(used, x[token], zero).to(dtype)
    y, dx = torch.zeros_like(x), torch.zeros_like(x)
    dw = torch.zeros_like(w)
    for j in range(row.shape[1]):
        part = torch.where(here[:, j], h[at[:, j]], zero)
        y += w[:, j, None] * part
        dw[:, j] = (dy * part).sum(-1)
        dx += torch.where(here[:, j], drows[at[:, j]], zero)
    weight = w.reshape(-1)[slot.clamp(min=0)]
    dh = torch.where(used, weight[:, None] * dy[token], zero).to(dtype)
    return rows, y.to(dtype), dh, dw, dx.to(dtype)


def _plain_product(st):
    case = st["case"]
    fmt, n, k, dtype = case["format"], case["n"], case["k"], DTYPES[case["dtype"]]
    names = ("gate", "up") if case["op"] == "swiglu" else ("b",)
    a = _decode(*st["a"], st["rows"], k, fmt)
    if not case["experts"]:
        parts = [a @ _decode(*st[name], n, k, fmt).t() for name in names]
        return _finish(parts).to(dtype)
    out = torch.zeros((st["rows"], n), device=a.device)
    size = st[names[0]][1].numel() // case["experts"]
    for e, (start, count) in enumerate(st["groups"]):
        if count:
            parts = [a[start:start + count] @ _decode(
                st[name][0][e * n:(e + 1) * n], st[name][1][e * size:(e + 1) * size], n, k,
                fmt).t() * st["alphas"][e] for name in names]
            out[start:start + count] = _finish(parts)
    return out.to(dtype)


def _finish(parts):
    if len(parts) == 1:
        return parts[0]
    gate, up = parts
    return gate / (1 + torch.exp(-gate)) * up


def _run_own(st):
    import megacu_b200 as mb
    case = st["case"]
    op = case["op"]
    kw = dict(problem=st["problem"], stream=torch.cuda.current_stream())
    if op == "sort":
        counts, offsets, row_of_slot, slot_of_row = st["out"]
        mb.moe_sort(st["ids"], counts=counts, offsets=offsets, row_of_slot=row_of_slot,
                    slot_of_row=slot_of_row, workspace=st["workspace"], **kw)
        return st["out"]
    if op == "exchange":
        rows, y, dh, dw, dx = st["out"]
        at = st["row_of_slot"]
        mb.moe_dispatch(st["x"], rows, row_of_slot=at, **kw)
        mb.moe_combine(st["h"], y, weights=st["w"], row_of_slot=at, **kw)
        mb.moe_combine_grad(st["dy"], st["h"], dh, dw, weights=st["w"], row_of_slot=at, **kw)
        mb.moe_combine(st["drows"], dx, row_of_slot=at, **kw)
        return st["out"]
    if op == "quantize":
        slots = dict(slot_of_row=st["slot_of_row"], topk=case["topk"]) if case["topk"] else {}
        mb.fp4_quantize(st["x"], st["data"], st["scales"], **slots, **kw)
        kw["problem"] = st["decode"]
        mb.fp4_dequantize(st["data"], st["scales"], st["values"], **kw)
        return st["values"]
    kw.update(events=st["events"])
    if case["experts"]:
        kw.update(offsets=st["offsets"], counts=st["counts"], alphas=st["alphas"])
    if op == "gemm":
        mb.fp4_gemm(*st["a"], *st["b"], st["out"], **kw)
    else:
        mb.fp4_gemm_swiglu(*st["a"], *st["gate"], *st["up"], st["out"], **kw)
    return st["out"]


# ---- definitions in 64 bits ----------------------------------------------------------

def exact(case, seed):
    st = prepare(case, seed)
    op = case["op"]
    if op == "sort":
        return _exact_sort(case, st["ids"])
    if op == "exchange":
        return _exact_exchange(st)
    if op == "quantize":
        return _exact_quantize(case, st)
    return _exact_product(case, st)


def _exact_sort(case, ids):
    """By a stable sort of the keys."""
    key = ids.reshape(-1).to(torch.int64) - case["first"]
    key = torch.where((key < 0) | (key >= case["experts"]), case["experts"], key)
    order = torch.sort(key, stable=True).indices
    counts = torch.bincount(key, minlength=case["experts"] + 1)[:case["experts"]]
    align = case["align"]
    ends = torch.cumsum((counts + align - 1) // align, 0) * align
    offsets = torch.cat((ends.new_zeros(1), ends))
    starts = torch.cumsum(counts, 0) - counts
    here = int(counts.sum())
    slots = order[:here]
    expert = key[slots]
    row = offsets[expert] + torch.arange(here, device=ids.device) - starts[expert]
    row_of_slot = torch.full((key.numel(),), -1, dtype=torch.int64, device=ids.device)
    row_of_slot[slots] = row
    slot_of_row = torch.full((_rows(case),), -1, dtype=torch.int64, device=ids.device)
    slot_of_row[row] = slots
    return tuple(t.to(torch.int32) for t in
                 (counts, offsets, row_of_slot.view(ids.shape), slot_of_row))


def _exact_exchange(st):
    """By products with each choice's rows, accumulated by row index, in 64 bits."""
    row = st["row_of_slot"].to(torch.int64)
    tokens, topk = row.shape
    token = torch.arange(tokens, device=row.device)
    hidden = st["x"].shape[1]
    full = lambda n: torch.zeros((n, hidden), dtype=torch.float64, device=row.device)
    rows, dh = full(st["h"].shape[0]), full(st["h"].shape[0])
    y, dx = full(tokens), full(tokens)
    dw = torch.zeros((tokens, topk), dtype=torch.float64, device=row.device)
    w = st["w"].double()
    for j in range(topk):
        here = row[:, j] >= 0
        t, r = token[here], row[here, j]
        rows[r] = st["x"][t].double()
        h, dy = st["h"][r].double(), st["dy"][t].double()
        y.index_add_(0, t, h * w[t, j, None])
        dh[r] = dy * w[t, j, None]
        dw[t, j] = torch.einsum("rh,rh->r", h, dy)
        dx.index_add_(0, t, st["drows"][r].double())
    return rows, y, dh, dw, dx


def _exact_quantize(case, st):
    """Codes by counting the borders below |z|, scales by the formats' grids."""
    x = st["x"].double()
    if case["transpose"]:
        x = x.t()
    block = BLOCK[case["format"]]
    z = x.reshape(x.shape[0], -1, block) * case["scale"]
    top = z.abs().amax(-1, keepdim=True)
    if case["format"] == "mx":
        grid = torch.tensor([2.0 ** e for e in range(-127, 128)], dtype=torch.float64,
                            device=x.device)
        at = torch.searchsorted(grid, top / 4, right=True) - 1      # the last one <= top / 4
        s = grid[at.clamp(min=0)]
    else:
        grid = [m * 2.0 ** -9 for m in range(8)]
        grid += [(8 + m) * 2.0 ** (e - 3) for e in range(-6, 9) for m in range(8)]
        grid = torch.tensor(grid[:-1], dtype=torch.float64, device=x.device)  # up to 448
        mid = (grid[1:] + grid[:-1]) / 2
        low = torch.searchsorted(6 * mid, top.contiguous())          # borders below top
        up = torch.searchsorted(6 * mid, top.contiguous(), right=True)
        s = grid[torch.where(low % 2 == 0, low, up)]
    a = z.abs()
    code = torch.zeros_like(a, dtype=torch.int64)
    for border, tie_up in ((0.25, 0), (0.75, 1), (1.25, 0), (1.75, 1), (2.5, 0), (3.5, 1),
                           (5.0, 0)):
        code += (a > border * s) | ((a == border * s) & bool(tie_up))
    value = torch.tensor(VALUES, dtype=torch.float64, device=x.device)[code] * torch.sign(z)
    value = torch.where(s > 0, value * s / case["scale"], torch.zeros_like(value))
    return _place(value.reshape(x.shape), st)


def _exact_product(case, st):
    fmt, n, k = case["format"], case["n"], case["k"]
    block = BLOCK[fmt]
    names = ("gate", "up") if case["op"] == "swiglu" else ("b",)

    def values(pair, first, rows):
        """Rows [first, first + rows) of a packed matrix, byte by byte."""
        data, scales = pair
        byte = data[first:first + rows].to(torch.int64)
        nib = torch.empty((rows, k), dtype=torch.int64, device=byte.device)
        nib[:, 0::2], nib[:, 1::2] = byte % 16, byte // 16
        mag = nib % 8
        v = torch.where(mag < 2, mag * 0.5, (1 << (mag // 2)) * (0.5 + (mag % 2) * 0.25))
        v = torch.where(nib >= 8, -v, v)
        return v, scales

    def scaled(pair, first, rows, base):
        v, scales = values(pair, first, rows)
        r = torch.arange(rows, device=v.device)[:, None]
        b = torch.arange(k // block, device=v.device)[None, :]
        tiles = -(-(k // block) // 4)
        at = base + ((r // 128) * tiles + b // 4) * 512 + (r % 32) * 16 + (r % 128 // 32) * 4 \
            + b % 4
        byte = scales[at].long()
        if fmt == "mx":
            grid = [2.0 ** (i - 127) for i in range(255)] + [math.nan]
        else:
            grid = [m * 2.0 ** -9 for m in range(8)]
            grid += [(1 + m / 8) * 2.0 ** (e - 7) for e in range(1, 16) for m in range(8)]
            grid += [math.nan] * 128
        s = torch.tensor(grid, dtype=torch.float64, device=v.device)[byte]
        return v * s.repeat_interleave(block, 1)

    a = scaled(st["a"], 0, st["rows"], 0)
    groups = st.get("groups", [(0, st["rows"])])
    out = torch.zeros((st["rows"], n), dtype=torch.float64, device=a.device)
    for e, (start, count) in enumerate(groups):
        if not count:
            continue
        alpha = float(st["alphas"][e]) if case["experts"] else 1.0
        parts = []
        for name in names:
            base = e * (st[name][1].numel() // len(groups))
            parts.append(alpha * torch.matmul(a[start:start + count],
                                              scaled(st[name], e * n, n, base).T))
        if len(parts) == 2:
            parts = [parts[0] * torch.sigmoid(parts[0]) * parts[1]]
        out[start:start + count] = parts[0]
    return out
