"""4-bit quantisation and products on a B200 against plain 64-bit
implementations.

Quantisation and the values back are decided exactly: codes, scale bytes and
values are compared for equality. A product's fp32 accumulation of k terms,
each addition off by at most one step (2^-23) of a partial sum, is within
k 2^-23 M of the exact one, M = alpha * sum |a| |b|; its rounding by half a
step of the type.
"""
from __future__ import annotations

import math

import pytest
import torch

import megacu_b200 as mb
import moe_fp4_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = {mb.DTYPE_F16: torch.float16, mb.DTYPE_BF16: torch.bfloat16, mb.DTYPE_F32: torch.float32}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}
FORMATS = [mb.FP4_MX, mb.FP4_NV]


def _stream():
    return torch.cuda.current_stream()


def _buffers(m):
    data, scales = mb.fp4_sizes(m)
    return (torch.full((max(data, 1),), 0xEE, dtype=torch.uint8, device="cuda"),
            torch.full((max(scales, 1),), 0xEE, dtype=torch.uint8, device="cuda"))


def _check_quantized(data, scales, x, fmt, g):
    code, byte = ref.quantize(x, fmt, g)
    want_data, want_scales = ref.pack(code, byte)
    assert torch.equal(scales.cpu(), want_scales)
    # the sign of an element that rounds to zero carries no value
    got = data.cpu().view(want_data.shape)
    zero = lambda d: torch.stack((d & 15, d >> 4), -1).long().flatten(1)
    a, b = zero(got), zero(want_data)
    assert torch.equal(torch.where(a == 8, 0, a), torch.where(b == 8, 0, b))


def _matrix(rows, cols, dtype, gen):
    """Values of very different sizes per row and column, zeros, whole blocks
    of zeros, subnormals."""
    x = torch.randn(rows, cols, generator=gen) * torch.exp(
        3 * torch.randn(rows, 1, generator=gen)) * torch.exp(torch.randn(1, cols, generator=gen))
    x[torch.rand(rows, cols, generator=gen) < 0.1] = 0
    x[0, :32] = 0
    if rows > 2:
        x[1] *= 1e-38
        x[2, ::3] *= 1e-6
    return x.to(dtype)


SHAPES = [(1, 32), (3, 64), (128, 128), (129, 160), (255, 544), (16, 4096), (70, 256), (300, 96)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,cols", SHAPES)
def test_quantize(rows, cols, dtype, fmt):
    gen = torch.Generator().manual_seed(rows * cols)
    x = _matrix(rows, cols, DTYPES[dtype], gen)
    for g in (1.0, 2.0 ** 9, 2.0 ** -7):
        m = mb.Fp4Matrix(rows, cols, format=fmt, dtype=dtype, scale=g)
        data, scales = _buffers(m)
        mb.fp4_quantize(x.cuda(), data, scales, problem=m, stream=_stream())
        _check_quantized(data, scales, x, fmt, g)
        m.transpose = True
        data, scales = _buffers(m)
        mb.fp4_quantize(x.t().contiguous().cuda(), data, scales, problem=m, stream=_stream())
        _check_quantized(data, scales, x, fmt, g)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
def test_quantize_ties_and_grid(dtype, fmt):
    """Every border between two elements and between two scales, exactly on it
    and one step of the type beside it."""
    t = DTYPES[dtype]
    borders = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], dtype=torch.float64)
    tops = torch.cat([6 * ref.NV_SCALES[8:127], 3 * (ref.NV_SCALES[8:126] + ref.NV_SCALES[9:127]),
                      2.0 ** torch.arange(-12, 12, dtype=torch.float64)]).to(t)
    lift = lambda v, k: (v.view(torch.int32 if t == torch.float32 else torch.int16) + k).view(t)
    tops = torch.cat([lift(tops, k) for k in (-1, 0, 1)])
    rows = []
    for top in tops[torch.isfinite(tops)]:
        s = ref.SCALES[fmt][ref.quantize(top.view(1, 1).expand(1, 32), fmt)[1]][0, 0]
        near = (borders * s).to(t)
        near = torch.cat([lift(near, k) for k in (-1, 0, 1)])
        near = torch.where(near <= top, near, torch.zeros_like(near))[:15]
        block = torch.cat([top.view(1), near])
        rows.append(torch.cat([block, -block]))
    x = torch.stack(rows)
    m = mb.Fp4Matrix(x.shape[0], 32, format=fmt, dtype=dtype)
    data, scales = _buffers(m)
    mb.fp4_quantize(x.cuda(), data, scales, problem=m, stream=_stream())
    _check_quantized(data, scales, x, fmt, 1.0)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("transpose", [False, True])
def test_quantize_infinities_and_nan(transpose, dtype, fmt):
    """A block with an infinity or NaN is NaN; its neighbours are not touched.
    The largest finite values saturate."""
    t = DTYPES[dtype]
    x = torch.ones(4, 128, dtype=t)
    x[0, 5], x[1, 40], x[2, 100] = math.inf, -math.inf, math.nan
    x[3] = torch.finfo(t).max
    for g in (1.0, 2.0 ** 60, 2.0 ** -60):
        m = mb.Fp4Matrix(4, 128, format=fmt, dtype=dtype, transpose=transpose, scale=g)
        data, scales = _buffers(m)
        mb.fp4_quantize((x.t().contiguous() if transpose else x).cuda(), data, scales, problem=m,
                        stream=_stream())
        _check_quantized(data, scales, x, fmt, g)
        back = torch.empty(4, 128, device="cuda")
        mb.fp4_dequantize(data, scales, back, problem=mb.Fp4Matrix(
            4, 128, format=fmt, dtype=mb.DTYPE_F32, scale=g), stream=_stream())
        block = ref.BLOCK[fmt]
        bad = ~torch.isfinite(x).view(4, -1, block).all(-1)
        assert torch.equal(torch.isnan(back).cpu().view(4, -1, block).all(-1), bad)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("rows,cols,pad,shift", [(5, 64, 8, 0), (33, 96, 3, 0), (130, 160, 0, 1),
                                                 (9, 288, 5, 3)])
def test_strides_and_alignment(rows, cols, pad, shift, dtype, fmt):
    t = DTYPES[dtype]
    gen = torch.Generator().manual_seed(cols)
    x = _matrix(rows, cols, t, gen)

    def dev(mat):
        buf = torch.full((shift + mat.shape[0] * (mat.shape[1] + pad),), float("nan"), dtype=t,
                         device="cuda")
        view = buf[shift:].view(mat.shape[0], mat.shape[1] + pad)[:, :mat.shape[1]]
        view.copy_(mat)
        return view

    for transpose in (False, True):
        src = dev(x.t() if transpose else x)
        m = mb.Fp4Matrix(rows, cols, format=fmt, dtype=dtype, transpose=transpose,
                         stride=src.stride(0) if pad else 0)
        data, scales = _buffers(m)
        mb.fp4_quantize(src, data, scales, problem=m, stream=_stream())
        _check_quantized(data, scales, x, fmt, 1.0)
    out = dev(torch.zeros(rows, cols))
    m = mb.Fp4Matrix(rows, cols, format=fmt, dtype=dtype, stride=out.stride(0) if pad else 0)
    mb.fp4_dequantize(data, scales, out, problem=m, stream=_stream())
    code, byte = ref.quantize(x, fmt)
    want = ref.values(*ref.pack(code, byte), fmt).to(torch.float32).to(t)
    assert torch.equal(out.cpu(), want)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("g", [1.0, 2.0 ** 12, 2.0 ** -60, 2.0 ** 60])
def test_dequantize_every_code(g, dtype, fmt):
    """Every element with every scale byte, rounded once to the type."""
    rows = 256 if fmt == mb.FP4_MX else 128
    code = torch.arange(32).remainder(16).repeat(rows, 1)
    byte = torch.arange(rows).view(-1, 1).repeat(1, 32 // ref.BLOCK[fmt])
    data, tiled = ref.pack(code, byte)
    out = torch.empty(rows, 32, dtype=DTYPES[dtype], device="cuda")
    mb.fp4_dequantize(data.cuda(), tiled.cuda(), out,
                      problem=mb.Fp4Matrix(rows, 32, format=fmt, dtype=dtype, scale=g),
                      stream=_stream())
    want = ref.values(data, tiled, fmt, g)
    # fp32 holds the value exactly or is below half its smallest step
    want = want.to(torch.float32).to(DTYPES[dtype])
    assert torch.equal(torch.nan_to_num(out.cpu().float(), nan=-1.5),
                       torch.nan_to_num(want.float(), nan=-1.5))


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("align", [1, 128])
def test_quantize_gathered(align, fmt):
    """Rows gathered to their experts; rows without a slot stay as they were,
    scales included. The same mask without a gather."""
    gen = torch.Generator().manual_seed(align)
    tokens, topk, experts, cols = 50, 3, 6, 288
    p = mb.MoeProblem(tokens, topk, experts, align=align)
    ids = torch.randint(0, experts + 1, (tokens, topk), generator=gen)
    _, _, row_of_slot, slots = ref.sort(ids, experts, 0, align, mb.moe_rows(p))
    x = _matrix(tokens, cols, torch.bfloat16, gen)
    m = mb.Fp4Matrix(mb.moe_rows(p), cols, format=fmt)
    used = slots >= 0
    rows = x[(slots.clamp(min=0) // topk).long()]
    want_data, want_scales = ref.pack(*ref.quantize(rows, fmt))
    r, b = torch.meshgrid(torch.arange(m.rows), torch.arange(-(-cols // ref.BLOCK[fmt] // 4) * 4),
                          indexing="ij")
    at = ref.scale_index(r, b, -(-cols // ref.BLOCK[fmt] // 4))
    for way in ("gather", "mask", "scatter"):
        data, scales = _buffers(m)
        index = dict(row_of_slot=row_of_slot.cuda()) if way == "scatter" else \
            dict(slot_of_row=slots.cuda())
        mb.fp4_quantize((rows if way == "mask" else x).cuda(), data, scales, problem=m,
                        topk=0 if way == "mask" else topk, stream=_stream(), **index)
        data, scales = data.cpu().view(m.rows, -1), scales.cpu()
        assert torch.equal(data[used] & 0x77, want_data[used] & 0x77)
        assert (data[~used] == 0xEE).all()
        assert torch.equal(scales[at[used]], want_scales[at[used]])
        assert (scales[at[~used]] == 0xEE).all()


def test_gathered_entries_that_name_no_row_are_skipped():
    x = torch.randn(6, 64).to(torch.bfloat16)
    good = torch.tensor([0, -1, 11, -1, 5, -1], dtype=torch.int32)
    bad = torch.tensor([0, 12, 11, 2 ** 31 - 1, 5, -2 ** 31], dtype=torch.int32)
    m = mb.Fp4Matrix(6, 64)
    got = []
    for slots in (good, bad):
        got.append(_buffers(m))
        mb.fp4_quantize(x.cuda(), *got[-1], problem=m, slot_of_row=slots.cuda(), topk=2,
                        stream=_stream())
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    for rows in ([[0, -1], [4, 2], [-1, -1], [5, 3], [1, -1], [-1, -1]],
                 [[0, 6], [4, 2], [-7, 2 ** 31 - 1], [5, 3], [1, 600], [-1, -2 ** 31]]):
        got.append(_buffers(m))
        mb.fp4_quantize(x.cuda(), *got[-1], problem=m, topk=2, stream=_stream(),
                        row_of_slot=torch.tensor(rows, dtype=torch.int32).cuda())
    assert torch.equal(got[2][0], got[3][0]) and torch.equal(got[2][1], got[3][1])


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,topk,cols,pad", [(1, 1, 32, 0), (33, 8, 96, 0), (70, 5, 544, 3),
                                                  (300, 2, 4096, 16)])
def test_scattered_rows_are_the_gathered_ones(tokens, topk, cols, pad, dtype, fmt):
    gen = torch.Generator().manual_seed(cols)
    p = mb.MoeProblem(tokens, topk, 9, first_expert=1, align=128)
    ids = torch.randint(0, 11, (tokens, topk), generator=gen)
    _, _, row_of_slot, slots = ref.sort(ids, 9, 1, 128, mb.moe_rows(p))
    x = torch.zeros(tokens, cols + pad, dtype=DTYPES[dtype])
    x[:, :cols] = _matrix(tokens, cols, DTYPES[dtype], gen)
    x[tokens // 2, 7] = math.inf
    x = x.cuda()[:, :cols]
    m = mb.Fp4Matrix(mb.moe_rows(p), cols, format=fmt, dtype=dtype, scale=4.0,
                     stride=cols + pad if pad else 0)
    got = [_buffers(m) for _ in range(2)]
    mb.fp4_quantize(x, *got[0], problem=m, slot_of_row=slots.cuda(), topk=topk, stream=_stream())
    mb.fp4_quantize(x, *got[1], problem=m, row_of_slot=row_of_slot.cuda(), topk=topk,
                    stream=_stream())
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


# ---- products ------------------------------------------------------------------------

def _run(fn, *args, problem, **kw):
    events = torch.zeros(mb.fp4_events_bytes(), dtype=torch.uint8, device="cuda")
    fn(*args, events=events, problem=problem, stream=_stream(), **kw)
    mb.events_status(events, _stream())


def _gpu(pair):
    return pair[0].cuda(), pair[1].cuda()


def _assert_close(got, want, err, t, what=""):
    """|got - want| <= err, then one rounding to t."""
    err = err + HALF_STEP[t] * (want.abs() + err) * (1 + 2.0 ** -10) + SMALLEST[t]
    bad = (got.double() - want).abs() > err
    assert not bad.any(), (what, int(bad.sum()), got[bad][:4], want[bad][:4])


PRODUCTS = [(1, 1, 32), (1, 128, 256), (16, 256, 288), (33, 40, 64), (128, 128, 512),
            (129, 257, 544), (200, 130, 1024), (257, 600, 96), (64, 1000, 4096), (300, 512, 1120)]


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", PRODUCTS)
def test_gemm(m, n, k, fmt):
    gen = torch.Generator().manual_seed(m * n + k)
    a, b = ref.random_operand(gen, m, k, fmt), ref.random_operand(gen, n, k, fmt)
    want, mag = ref.product(ref.values(*a, fmt), ref.values(*b, fmt), 0.375)
    ag, bg = _gpu(a), _gpu(b)
    for dtype, t in DTYPES.items():
        for tile_n, split in ((0, 0), (128, 1), (256, 1), (128, 2), (256, 4), (128, 8), (256, 8),
                              (64, 1), (64, 2), (64, 4)):
            if split > -(-k // 256):
                continue
            p = mb.Fp4Gemm(m, n, k, format=fmt, out_dtype=dtype, alpha=0.375, tile_n=tile_n,
                           split=split)
            out = torch.full((m, n), float("nan"), dtype=t, device="cuda")
            _run(mb.fp4_gemm, *ag, *bg, out, problem=p)
            _assert_close(out.cpu(), want, k * 2.0 ** -23 * mag, t, (dtype, tile_n, split))


@pytest.mark.parametrize("fmt", FORMATS)
def test_gemm_many_tiles_per_sm(fmt):
    """More tiles than SMs: both accumulators and the ring's phases wrap."""
    gen = torch.Generator().manual_seed(2)
    m, n, k = 1500, 4300, 1312
    a, b = ref.random_operand(gen, m, k, fmt), ref.random_operand(gen, n, k, fmt)
    want, mag = ref.product(ref.values(*a, fmt), ref.values(*b, fmt))
    for tile_n in (64, 128, 256):
        p = mb.Fp4Gemm(m, n, k, format=fmt, out_dtype=mb.DTYPE_F32, tile_n=tile_n, split=1)
        out = torch.empty(m, n, device="cuda")
        _run(mb.fp4_gemm, *_gpu(a), *_gpu(b), out, problem=p)
        _assert_close(out.cpu(), want, k * 2.0 ** -23 * mag, torch.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m", [1, 31, 32, 33])
def test_gemm_few_rows_many_tiles(m, fmt):
    """Several tiles per SM around the 32 rows that a small stage holds."""
    gen = torch.Generator().manual_seed(m)
    n, k = 12000, 800
    a, b = ref.random_operand(gen, m, k, fmt), ref.random_operand(gen, n, k, fmt)
    want, mag = ref.product(ref.values(*a, fmt), ref.values(*b, fmt))
    out = torch.empty(m, n, device="cuda")
    _run(mb.fp4_gemm, *_gpu(a), *_gpu(b), out, problem=mb.Fp4Gemm(
        m, n, k, format=fmt, out_dtype=mb.DTYPE_F32, tile_n=64, split=1))
    _assert_close(out.cpu(), want, k * 2.0 ** -23 * mag, torch.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("pad,shift", [(0, 1), (5, 0), (16, 0)])
def test_gemm_output_strides(pad, shift, dtype, fmt):
    """Rows apart and off the 16-byte boundary; nothing is written between."""
    t = DTYPES[dtype]
    gen = torch.Generator().manual_seed(pad)
    m, n, k = 70, 200, 320
    a, b = ref.random_operand(gen, m, k, fmt), ref.random_operand(gen, n, k, fmt)
    want, mag = ref.product(ref.values(*a, fmt), ref.values(*b, fmt))
    for split in (1, 2):
        buf = torch.full((shift + m * (n + pad) + 64,), 7.0, dtype=t, device="cuda")
        view = buf[shift:shift + m * (n + pad)].view(m, n + pad)
        p = mb.Fp4Gemm(m, n, k, format=fmt, out_dtype=dtype, out_stride=n + pad, split=split)
        _run(mb.fp4_gemm, *_gpu(a), *_gpu(b), view[:, :n] if pad else view, problem=p)
        _assert_close(view[:, :n].cpu(), want, k * 2.0 ** -23 * mag, t)
        view[:, :n] = 7.0
        assert (buf == 7.0).all()


@pytest.mark.parametrize("fmt", FORMATS)
def test_gemm_nan_scale_stays_in_its_row_and_column(fmt):
    gen = torch.Generator().manual_seed(4)
    m, n, k = 140, 300, 512
    a, b = ref.random_operand(gen, m, k, fmt), ref.random_operand(gen, n, k, fmt)
    nan, tiles = (255, 4) if fmt == mb.FP4_MX else (127, 8)
    a[1][ref.scale_index(torch.tensor(131), torch.tensor(3), tiles)] = nan
    b[1][ref.scale_index(torch.tensor(290), torch.tensor(9), tiles)] = nan
    for split in (1, 2):
        out = torch.empty(m, n, device="cuda")
        _run(mb.fp4_gemm, *_gpu(a), *_gpu(b), out,
             problem=mb.Fp4Gemm(m, n, k, format=fmt, out_dtype=mb.DTYPE_F32, split=split))
        want = torch.zeros(m, n, dtype=torch.bool)
        want[131], want[:, 290] = True, True
        assert torch.equal(torch.isnan(out).cpu(), want)


def _swiglu_want(a, gate, up, alpha, k):
    g, gm = ref.product(a, gate, alpha)
    u, um = ref.product(a, up, alpha)
    want, err = ref.swiglu(g, u, k * 2.0 ** -23 * gm, k * 2.0 ** -23 * um)
    # exp, the division and two products: |g| 2^-22 from the exponent's
    # rounding (its argument is scaled by log2 e in fp32) and 8 steps more
    return want, err + (g.abs() * 2.0 ** -22 + 2.0 ** -20) * want.abs()


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("m,n,k", [(1, 1, 32), (16, 128, 512), (130, 200, 288), (70, 129, 1024),
                                   (400, 3001, 544)])
def test_swiglu(m, n, k, fmt):
    gen = torch.Generator().manual_seed(m + n + k)
    a, gate, up = (ref.random_operand(gen, r, k, fmt) for r in (m, n, n))
    want, err = _swiglu_want(*(ref.values(*x, fmt) for x in (a, gate, up)), 2.0 ** -4, k)
    for dtype, t in DTYPES.items():
        for split in (0, 1, 2, 4):
            if split > -(-k // 256):
                continue
            p = mb.Fp4Gemm(m, n, k, format=fmt, out_dtype=dtype, alpha=2.0 ** -4, split=split)
            out = torch.full((m, n), float("nan"), dtype=t, device="cuda")
            _run(mb.fp4_gemm_swiglu, *_gpu(a), *_gpu(gate), *_gpu(up), out, problem=p)
            if t == torch.float16:
                keep = want.abs() < 6e4  # beyond it fp16 has infinities
                _assert_close(out.cpu()[keep], want[keep], err[keep], t, split)
            else:
                _assert_close(out.cpu(), want, err, t, split)


@pytest.mark.parametrize("split", [1, 2])
def test_swiglu_of_large_gates(split):
    """Gates far from zero, both ways: alpha puts them between -90 and 90, where
    exp(-g) nears the type's ends; the up products are ones."""
    k, n = 512, 128
    gen = torch.Generator().manual_seed(1)
    gate = torch.randint(-3, 4, (n, k), generator=gen).double()
    a = torch.zeros(40, k, dtype=torch.float64)
    a[:, 0] = 1
    a[:, 1] = torch.arange(40) % 7
    up = torch.zeros(n, k, dtype=torch.float64)
    up[:, 0] = 1
    ops = [ref.pack(*ref.quantize(x, mb.FP4_MX)) for x in (a, gate, up)]
    va, vg, vu = (ref.values(*x, mb.FP4_MX) for x in ops)
    alpha = 4.0
    g, u = alpha * va @ vg.T, alpha * va @ vu.T
    assert g.min() < -80 and g.max() > 80
    want = g * torch.where(g < 0, torch.exp(g), torch.ones_like(g)) / (1 + torch.exp(-g.abs())) * u
    out = torch.empty(40, n, device="cuda")
    _run(mb.fp4_gemm_swiglu, *(t for x in ops for t in _gpu(x)), out, problem=mb.Fp4Gemm(
        40, n, k, out_dtype=mb.DTYPE_F32, alpha=alpha, split=split))
    # the products are whole numbers: exact; then as _swiglu_want's last line
    err = (g.abs() * 2.0 ** -22 + 2.0 ** -20) * want.abs()
    _assert_close(out.cpu(), want, err, torch.float32)


GROUPS = [  # counts per expert
    [1], [0, 5, 0, 0, 130, 1, 128, 0], [300, 0, 2], [0, 0, 0], [3] * 40,
    [0] * 70 + [129] + [0] * 29 + [1],
    [1300, 129, 1700, 0, 2000], [0, 900, 128, 2500],   # pairs of tiles, odd numbers of them
    [1] * 299 + [130]]                                 # more than are kept on chip


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("counts", GROUPS, ids=lambda c: f"{len(c)}x{sum(c)}")
def test_by_expert(counts, fmt):
    """Experts without rows, one row, whole tiles and more; rows of padding
    and behind the last stay as they were although A and its scales hold
    garbage (NaN scales) there."""
    gen = torch.Generator().manual_seed(len(counts))
    experts, n, k = len(counts), 150, 576
    padded = [-(-c // 128) * 128 for c in counts]
    offsets = [sum(padded[:i]) for i in range(experts + 1)]
    m = offsets[-1] + 256
    a = ref.random_operand(gen, m, k, fmt)
    used = torch.zeros(m, dtype=torch.bool)
    for o, c in zip(offsets, counts):
        used[o:o + c] = True
    av = ref.values(*a, fmt)
    blocks = k // ref.BLOCK[fmt]
    r, b = torch.meshgrid(torch.arange(m)[~used], torch.arange(blocks), indexing="ij")
    a[1][ref.scale_index(r, b, -(-blocks // 4))] = 255 if fmt == mb.FP4_MX else 127
    weights = {name: [ref.random_operand(gen, n, k, fmt) for _ in counts] for name in ("g", "u")}
    packed = {name: tuple(torch.cat([w[i] for w in ws]).cuda() for i in (0, 1))
              for name, ws in weights.items()}
    alphas = torch.rand(experts, generator=gen) * 0.1
    kw = dict(offsets=torch.tensor(offsets, dtype=torch.int32).cuda(),
              counts=torch.tensor(counts, dtype=torch.int32).cuda())
    for use_alphas in (True, False):
        for split, tile_n in ((0, 0), (1, 256), (2, 0)):
            p = mb.Fp4Gemm(m, n, k, format=fmt, out_dtype=mb.DTYPE_F32, experts=experts,
                           alpha=0.5, split=split, tile_n=tile_n)
            al = dict(alphas=alphas.cuda()) if use_alphas else {}
            out = torch.full((m, n), -3.0, device="cuda")
            act = torch.full((m, n), -3.0, device="cuda")
            _run(mb.fp4_gemm, *_gpu(a), *packed["g"], out, problem=p, **kw, **al)
            _run(mb.fp4_gemm_swiglu, *_gpu(a), *packed["g"], *packed["u"], act, problem=p, **kw,
                 **al)
            out, act = out.cpu(), act.cpu()
            assert (out[~used] == -3.0).all() and (act[~used] == -3.0).all()
            for e, (o, c) in enumerate(zip(offsets, counts)):
                if not c:
                    continue
                alpha = 0.5 * float(alphas[e]) if use_alphas else 0.5
                gv, uv = (ref.values(*weights[x][e], fmt) for x in ("g", "u"))
                rows = av[o:o + c]
                want, mag = ref.product(rows, gv, alpha)
                # two more roundings: alpha * alphas[e] and the product with it
                _assert_close(out[o:o + c], want, (k + 2) * 2.0 ** -23 * mag, torch.float32)
                want, err = _swiglu_want(rows, gv, uv, alpha, k + 2)
                _assert_close(act[o:o + c], want, err, torch.float32)


def test_gemm_repeats_bit_for_bit_and_replays():
    """No order of execution changes a bit; two captured graphs share events."""
    gen = torch.Generator().manual_seed(8)
    m, n, k = 100, 520, 2048
    a, b = _gpu(ref.random_operand(gen, m, k, 0)), _gpu(ref.random_operand(gen, n, k, 0))
    events = torch.zeros(mb.fp4_events_bytes(), dtype=torch.uint8, device="cuda")
    p = mb.Fp4Gemm(m, n, k, out_dtype=mb.DTYPE_F32, split=4)
    first = torch.empty(m, n, device="cuda")
    mb.fp4_gemm(*a, *b, first, events=events, problem=p, stream=_stream())
    out = torch.empty_like(first)
    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            mb.fp4_gemm(*a, *b, out, events=events, problem=p, stream=_stream())
        graphs.append(g)
    for i in range(6):
        out.zero_()
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
    mb.events_status(events, _stream())


def test_products_on_two_streams_at_once():
    gen = torch.Generator().manual_seed(10)
    fmt, m, n, k = mb.FP4_NV, 256, 2048, 1024
    a = ref.random_operand(gen, m, k, fmt)
    bs = [ref.random_operand(gen, n, k, fmt) for _ in range(2)]
    outs = [torch.empty(m, n, device="cuda") for _ in bs]
    dev = [(_gpu(a), _gpu(b), torch.zeros(256, dtype=torch.uint8, device="cuda")) for b in bs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in bs]
    p = mb.Fp4Gemm(m, n, k, format=fmt, out_dtype=mb.DTYPE_F32)
    for _ in range(5):
        for s, (ag, bg, ev), out in zip(streams, dev, outs):
            mb.fp4_gemm(*ag, *bg, out, events=ev, problem=p, stream=s)
    torch.cuda.synchronize()
    for b, out, (_, _, ev) in zip(bs, outs, dev):
        want, mag = ref.product(ref.values(*a, fmt), ref.values(*b, fmt))
        _assert_close(out.cpu(), want, k * 2.0 ** -23 * mag, torch.float32)
        mb.events_status(ev, _stream())


def test_linear_layer_and_its_gradients():
    """y = x w, dx = dy w^T, dw = x^T dy with every operand quantised along the
    sum's dimension, by rows or transposed, against the products of the
    quantised values."""
    gen = torch.Generator().manual_seed(6)
    tokens, fan_in, fan_out = 160, 96, 224
    fmt = mb.FP4_MX
    x = torch.randn(tokens, fan_in, generator=gen).to(torch.bfloat16)
    w = torch.randn(fan_in, fan_out, generator=gen).to(torch.bfloat16)
    dy = torch.randn(tokens, fan_out, generator=gen).to(torch.bfloat16)

    def quantized(plain, transpose):
        rows, cols = reversed(plain.shape) if transpose else plain.shape
        m = mb.Fp4Matrix(rows, cols, format=fmt, transpose=transpose)
        data, scales = _buffers(m)
        mb.fp4_quantize(plain.cuda(), data, scales, problem=m, stream=_stream())
        src = plain.t().contiguous() if transpose else plain
        return (data, scales), ref.values(*ref.pack(*ref.quantize(src, fmt)), fmt)

    for left, lt, right, rt in ((x, False, w, True), (dy, False, w, False), (x, True, dy, True)):
        (qa, va), (qb, vb) = quantized(left, lt), quantized(right, rt)
        m, k = va.shape
        out = torch.empty(m, vb.shape[0], device="cuda")
        _run(mb.fp4_gemm, *qa, *qb, out,
             problem=mb.Fp4Gemm(m, vb.shape[0], k, format=fmt, out_dtype=mb.DTYPE_F32))
        want, mag = ref.product(va, vb)
        _assert_close(out.cpu(), want, k * 2.0 ** -23 * mag, torch.float32)


@pytest.mark.parametrize("fmt", FORMATS)
@pytest.mark.parametrize("tokens", [1, 40, 300])
def test_routed_mlp(tokens, fmt):
    """The operators together: a routed 4-bit MLP block. Each stage is checked
    against the definition applied to the stage before it."""
    gen = torch.Generator().manual_seed(tokens)
    topk, experts, first, hidden, inter = 4, 10, 3, 256, 192
    p = mb.MoeProblem(tokens, topk, experts, hidden=hidden, first_expert=first, align=128)
    rows = mb.moe_rows(p)
    ids = torch.rand(tokens, experts + first, generator=gen).topk(topk, 1).indices
    x = torch.randn(tokens, hidden, generator=gen).to(torch.bfloat16)
    w = torch.softmax(torch.randn(tokens, topk, generator=gen), -1)
    new = lambda *shape, t=torch.int32: torch.zeros(shape, dtype=t, device="cuda")
    counts, offsets, at, slots = new(experts), new(experts + 1), new(tokens, topk), new(rows)
    kw = dict(stream=_stream())
    mb.moe_sort(ids.cuda(), counts=counts, offsets=offsets, row_of_slot=at, slot_of_row=slots,
                problem=p, **kw)
    want = ref.sort(ids, experts, first, 128, rows)
    for g, e in zip((counts, offsets, at, slots), want):
        assert torch.equal(g.cpu(), e)
    slot, used = slots.cpu().long(), slots.cpu() >= 0

    def weights(n, k):
        parts = [ref.random_operand(gen, n, k, fmt) for _ in range(experts)]
        return parts, tuple(torch.cat([q[i] for q in parts]).cuda() for i in (0, 1))

    (gate, gate_d), (up, up_d), (down, down_d) = (weights(inter, hidden), weights(inter, hidden),
                                                  weights(hidden, inter))
    kw.update(events=new(256, t=torch.uint8))
    group = dict(offsets=offsets, counts=counts)
    # rows to their experts, quantised
    m1 = mb.Fp4Matrix(rows, hidden, format=fmt)
    q1 = _buffers(m1)
    mb.fp4_quantize(x.cuda(), *q1, problem=m1, slot_of_row=slots, topk=topk, stream=_stream())
    xv = ref.values(*ref.pack(*ref.quantize(x[slot.clamp(min=0) // topk], fmt)), fmt)
    # gate and up
    act = new(rows, inter, t=torch.bfloat16)
    mb.fp4_gemm_swiglu(*q1, *gate_d, *up_d, act, **group, **kw, problem=mb.Fp4Gemm(
        rows, inter, hidden, format=fmt, experts=experts, alpha=2.0 ** -4))
    act_h = act.cpu()
    for e in range(experts):
        o, c = int(want[1][e]), int(want[0][e])
        if c:
            gv, uv = ref.values(*gate[e], fmt), ref.values(*up[e], fmt)
            res, err = _swiglu_want(xv[o:o + c], gv, uv, 2.0 ** -4, hidden)
            _assert_close(act_h[o:o + c], res, err, torch.bfloat16)
    # down
    m2 = mb.Fp4Matrix(rows, inter, format=fmt, scale=0.25)
    q2 = _buffers(m2)
    mb.fp4_quantize(act, *q2, problem=m2, slot_of_row=slots, stream=_stream())
    av = ref.values(*ref.pack(*ref.quantize(act_h, fmt, 0.25)), fmt)
    out = new(rows, hidden, t=torch.bfloat16)
    mb.fp4_gemm(*q2, *down_d, out, **group, **kw, problem=mb.Fp4Gemm(
        rows, hidden, inter, format=fmt, experts=experts, alpha=4.0))
    out_h = out.cpu()
    for e in range(experts):
        o, c = int(want[1][e]), int(want[0][e])
        if c:
            res, mag = ref.product(av[o:o + c], ref.values(*down[e], fmt), 4.0)
            _assert_close(out_h[o:o + c], res, inter * 2.0 ** -23 * mag, torch.bfloat16)
    # and back
    y = new(tokens, hidden, t=torch.bfloat16)
    mb.moe_combine(out, y, weights=w.cuda(), row_of_slot=at, problem=p, stream=_stream())
    res, mag = ref.combine(out_h, w, at.cpu())
    _assert_close(y.cpu(), res, topk * 2.0 ** -24 * mag, torch.bfloat16)
    mb.events_status(kw["events"], _stream())


@pytest.mark.parametrize("ids_type", [torch.int32, torch.int64])
@pytest.mark.parametrize("tokens,fmt,dtype", [(1, mb.FP4_MX, mb.DTYPE_BF16),
                                              (37, mb.FP4_NV, mb.DTYPE_F16),
                                              (700, mb.FP4_MX, mb.DTYPE_BF16)])
def test_routed_mlp_block_is_its_calls(tokens, fmt, dtype, ids_type):
    """moe_mlp_fp4 gives bit for bit what its calls give one by one, directly
    and replayed from a graph, whatever its workspace holds before."""
    gen = torch.Generator().manual_seed(tokens)
    t = DTYPES[dtype]
    topk, experts, first, hidden, inter = 3, 6, 2, 320, 160
    ids = torch.randint(0, experts + 3, (tokens, topk), generator=gen).to(ids_type).cuda()
    x = torch.randn(tokens, hidden, generator=gen).to(t).cuda()
    w = torch.rand(tokens, topk, generator=gen).cuda()

    def weights(n, k):
        parts = [ref.random_operand(gen, n, k, fmt) for _ in range(experts)]
        return tuple(torch.cat([q[i] for q in parts]).cuda() for i in (0, 1))

    gate, up, down = weights(inter, hidden), weights(inter, hidden), weights(hidden, inter)
    alphas = (torch.rand(experts, generator=gen) + 0.5).cuda()
    p = mb.MoeMlp(tokens, hidden, inter, topk, experts, first_expert=first, dtype=dtype,
                  format=fmt, x_scale=2.0, act_scale=0.5, up_alpha=2.0 ** -5,
                  down_alpha=2.0 ** -6)
    events = torch.zeros(256, dtype=torch.uint8, device="cuda")
    ws = torch.full((mb.moe_mlp_workspace_bytes(p),), 0xA5, dtype=torch.uint8, device="cuda")
    y = torch.empty(tokens, hidden, dtype=t, device="cuda")

    def block():
        mb.moe_mlp_fp4(x, ids, w, *gate, *up, *down, y, workspace=ws, events=events, problem=p,
                       up_alphas=alphas, down_alphas=None, stream=_stream())

    block()
    direct = y.clone()

    route = mb.MoeProblem(tokens, topk, experts, hidden=hidden, first_expert=first, align=128,
                          dtype=dtype)
    rows = mb.moe_rows(route)
    new = lambda *shape, u=torch.int32: torch.zeros(shape, dtype=u, device="cuda")
    counts, offsets, at, slots = new(experts), new(experts + 1), new(tokens, topk), new(rows)
    sort_ws = new(max(mb.moe_workspace_bytes(route), 1), u=torch.uint8)
    kw = dict(stream=_stream())
    mb.moe_sort(ids, counts=counts, offsets=offsets, row_of_slot=at, slot_of_row=slots,
                workspace=sort_ws, problem=route, **kw)
    xm = mb.Fp4Matrix(rows, hidden, format=fmt, dtype=dtype, scale=2.0)
    am = mb.Fp4Matrix(rows, inter, format=fmt, dtype=dtype, scale=0.5)
    xq, aq = _buffers(xm), _buffers(am)
    mb.fp4_quantize(x, *xq, problem=xm, slot_of_row=slots, topk=topk, **kw)
    act, out = new(rows, inter, u=t), new(rows, hidden, u=t)
    group = dict(offsets=offsets, counts=counts, events=events, **kw)
    mb.fp4_gemm_swiglu(*xq, *gate, *up, act, alphas=alphas, problem=mb.Fp4Gemm(
        rows, inter, hidden, format=fmt, out_dtype=dtype, experts=experts, alpha=2.0 ** -6),
        **group)
    mb.fp4_quantize(act, *aq, problem=am, slot_of_row=slots, **kw)
    mb.fp4_gemm(*aq, *down, out, problem=mb.Fp4Gemm(
        rows, hidden, inter, format=fmt, out_dtype=dtype, experts=experts, alpha=2.0 ** -5),
        **group)
    want = torch.empty_like(y)
    mb.moe_combine(out, want, weights=w, row_of_slot=at, problem=route, **kw)
    assert torch.equal(direct, want) and direct.float().abs().max() > 0

    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        block()
    for _ in range(2):
        ws.fill_(0x3C)
        y.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(y, want)
    mb.events_status(events, _stream())


def test_calls_in_a_row_wait_for_one_another():
    """Launches overlap their set-up with the kernel before them; their work
    must not. Blocks that feed one another in place, with nothing between them,
    give what they give with a synchronisation after every one."""
    gen = torch.Generator().manual_seed(12)
    tokens, topk, experts, hidden, inter, steps = 600, 4, 8, 256, 192, 12
    ids = torch.rand(steps, tokens, experts, generator=gen).topk(topk, -1).indices.cuda()
    start = torch.randn(tokens, hidden, generator=gen).to(torch.bfloat16).cuda()
    w = torch.softmax(torch.randn(tokens, topk, generator=gen), -1).cuda()

    def weights(n, k):
        parts = [ref.random_operand(gen, n, k, 0) for _ in range(experts)]
        return tuple(torch.cat([q[i] for q in parts]).cuda() for i in (0, 1))

    gate, up, down = weights(inter, hidden), weights(inter, hidden), weights(hidden, inter)
    p = mb.MoeMlp(tokens, hidden, inter, topk, experts, up_alpha=2.0 ** -5, down_alpha=2.0 ** -5)
    dense = mb.Fp4Gemm(tokens, hidden, hidden, alpha=2.0 ** -5)
    m = mb.Fp4Matrix(tokens, hidden)
    square = _gpu(ref.random_operand(gen, hidden, hidden, 0))

    def run(sync):
        x, events = start.clone(), torch.zeros(256, dtype=torch.uint8, device="cuda")
        ws = torch.empty(mb.moe_mlp_workspace_bytes(p), dtype=torch.uint8, device="cuda")
        data, scales = _buffers(m)
        torch.cuda.synchronize()
        for i in range(steps):
            mb.moe_mlp_fp4(x, ids[i], w, *gate, *up, *down, x, workspace=ws, events=events,
                           problem=p, stream=_stream())
            if sync:
                torch.cuda.synchronize()
            mb.fp4_quantize(x, data, scales, problem=m, stream=_stream())
            if sync:
                torch.cuda.synchronize()
            mb.fp4_gemm(data, scales, *square, x, events=events, problem=dense, stream=_stream())
            # Another library's kernels between them. Without a norm x would
            # overflow in both runs: the operands' elements are about 10, so a
            # block multiplies x^2 by about 50.
            x /= x.abs().amax()
            if sync:
                torch.cuda.synchronize()
        mb.events_status(events, _stream())
        return x.clone()

    want = run(True)
    assert torch.isfinite(want.float()).all() and want.float().abs().max() > 0
    for _ in range(5):
        assert torch.equal(run(False), want)


@pytest.mark.parametrize("swiglu", [False, True])
@pytest.mark.parametrize("m,n,k,experts,tile_n,split", [
    (16, 2048, 8192, 0, 64, 1), (100, 1000, 4096, 0, 256, 8), (100, 2000, 8192, 0, 256, 4),
    (1000, 4000, 8192, 0, 256, 1), (300, 9000, 2048, 0, 128, 1), (1024, 512, 4096, 8, 256, 1),
    (1024, 512, 4096, 8, 256, 2)])
def test_given_up_waits_end_the_call_and_spare_the_next(m, n, k, experts, tile_n, split, swiglu):
    """A call on events that still hold an error, and one whose waits may last
    no time at all, return (which of their waits give up is a matter of
    timing), report it, and the next calls compute what they always do."""
    if swiglu and tile_n != 256:
        tile_n, split = 256, 1
    gen = torch.Generator().manual_seed(n)
    a = _gpu(ref.random_operand(gen, m, k, 0))
    parts = [_gpu(ref.random_operand(gen, max(experts, 1) * n, k, 0)) for _ in range(1 + swiglu)]
    kw = {}
    if experts:
        rows = torch.full((experts,), m // experts, dtype=torch.int32)
        kw = dict(offsets=torch.arange(experts + 1, dtype=torch.int32).mul(m // experts).cuda(),
                  counts=rows.cuda())
    operands = [t for part in parts for t in part]
    fn = mb.fp4_gemm_swiglu if swiglu else mb.fp4_gemm
    events = torch.zeros(mb.fp4_events_bytes(), dtype=torch.uint8, device="cuda")

    def run(timeout_ns=0):
        p = mb.Fp4Gemm(m, n, k, alpha=2.0 ** -8, experts=experts, tile_n=tile_n, split=split,
                       timeout_ns=timeout_ns)
        out = torch.zeros(m, n, dtype=torch.bfloat16, device="cuda")
        fn(*a, *operands, out, events=events, problem=p, stream=_stream(), **kw)
        return out

    want = run()
    mb.events_status(events, _stream())
    for _ in range(3):
        events.view(torch.int32)[4] = 41  # the error word
        run()
        run(1)
        with pytest.raises(mb.MegacuError):
            mb.events_status(events, _stream())
        assert torch.equal(run(), want)
        mb.events_status(events, _stream())
        out = run(1)
        try:
            mb.events_status(events, _stream())
            assert torch.equal(out, want)
        except mb.MegacuError:
            pass
        assert torch.equal(run(), want)
        mb.events_status(events, _stream())


@pytest.mark.parametrize("tokens,fmt,dtype", [(3000, mb.FP4_MX, mb.DTYPE_F32),
                                              (4097, mb.FP4_NV, mb.DTYPE_BF16),
                                              (40, mb.FP4_NV, mb.DTYPE_F32)])
def test_routed_mlp_block_of_long_batches_and_in_f32(tokens, fmt, dtype):
    """The same where the block's sort takes two launches and a workspace (more
    than 8192 slots), and in 32 bits."""
    p = mb.MoeMlp(tokens, 320, 160, 3, 6)
    assert (mb.moe_workspace_bytes(mb.MoeProblem(tokens, p.topk, p.experts, align=128)) > 0) == (
        tokens * p.topk > 8192)
    test_routed_mlp_block_is_its_calls(tokens, fmt, dtype, torch.int64)
