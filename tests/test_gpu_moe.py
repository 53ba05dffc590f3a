"""Routing kernels on a B200 against plain 64-bit implementations.

Tolerances (u = half a step of the output type: bf16 2^-8, f16 2^-11, f32
2^-24; M = the sum of the terms' magnitudes): a sum of n products in fp32 by
fused multiply-adds is off by at most n 2^-24 M, its rounding by u |sum|; one
product w * dy rounded twice (fp32, then the type) by (2^-24 + u) |w dy|.
"""
from __future__ import annotations

import pytest
import torch

import megacu_b200 as mb
import moe_fp4_ref as ref

pytestmark = pytest.mark.gpu
DTYPES = {mb.DTYPE_F16: torch.float16, mb.DTYPE_BF16: torch.bfloat16, mb.DTYPE_F32: torch.float32}
HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2.0 ** -24}
SMALLEST = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float32: 2.0 ** -150}


def _new(*shape, dtype=torch.int32, fill=-77):
    return torch.full(shape, fill, dtype=dtype, device="cuda")


def _sort(ids, p, stream=None):
    out = (_new(p.experts), _new(p.experts + 1), _new(*ids.shape), _new(mb.moe_rows(p)))
    # any content: the workspace need not be initialised
    ws = _new(max(mb.moe_workspace_bytes(p), 1), dtype=torch.uint8, fill=0x5a)
    mb.moe_sort(ids, counts=out[0], offsets=out[1], row_of_slot=out[2], slot_of_row=out[3],
                workspace=ws, problem=p, stream=stream or torch.cuda.current_stream())
    return out


def _ids(kind, tokens, topk, total, seed):
    gen = torch.Generator().manual_seed(seed)
    if kind == "one":       # every slot to one expert
        return torch.full((tokens, topk), total - 1)
    if kind == "none":      # ids of other PEs only, and nonsense
        return torch.randint(0, 2, (tokens, topk), generator=gen) * 10 ** 6 - 5
    if kind == "edges":     # ids around the local range
        return torch.randint(-1, total + 1, (tokens, topk), generator=gen)
    return torch.randint(0, total, (tokens, topk), generator=gen)


SORTS = [(1, 1, 1, 0, 1), (1, 8, 8, 0, 128), (64, 8, 128, 0, 128), (37, 3, 5, 2, 8),
         (1024, 1, 1024, 0, 1), (1025, 1, 33, 1, 16), (1023, 8, 64, 0, 128), (1024, 8, 7, 0, 1),
         (4097, 2, 256, 0, 128), (4096, 8, 1000, 100, 128), (5001, 7, 16, 3, 5),
         (32768, 8, 3, 0, 1), (70001, 4, 300, 0, 1024), (200003, 4, 1024, 7, 16)]


@pytest.mark.parametrize("kind", ["random", "one", "none", "edges"])
@pytest.mark.parametrize("tokens,topk,experts,first,align", SORTS)
def test_sort(tokens, topk, experts, first, align, kind):
    p = mb.MoeProblem(tokens, topk, experts, first_expert=first, align=align)
    ids = _ids(kind, tokens, topk, experts + first, tokens)
    want = ref.sort(ids, experts, first, align, mb.moe_rows(p))
    for dtype in (torch.int32, torch.int64):
        got = _sort(ids.to(dtype).cuda(), p)
        for g, w, name in zip(got, want, ("counts", "offsets", "row_of_slot", "slot_of_row")):
            assert torch.equal(g.cpu(), w), (name, dtype)


def test_sort_ids_of_64_bits_do_not_wrap():
    p = mb.MoeProblem(2, 2, 4)
    ids = torch.tensor([[2 ** 32, 1], [-(2 ** 32), 2 ** 40 + 3]])
    got = _sort(ids.cuda(), p)
    for g, w in zip(got, ref.sort(ids, 4, 0, 1, mb.moe_rows(p))):
        assert torch.equal(g.cpu(), w)


def test_sort_empty_batch():
    p = mb.MoeProblem(0, 8, 5, align=128)
    counts, offsets = _new(5), _new(6)
    mb.moe_sort(None, counts=counts, offsets=offsets, row_of_slot=None, slot_of_row=None,
                problem=p, stream=torch.cuda.current_stream())
    assert counts.tolist() == [0] * 5 and offsets.tolist() == [0] * 6


ROWS = [  # tokens, topk, experts, hidden, align, token stride - hidden, row stride - hidden, offset
    (1, 1, 1, 8, 1, 0, 0, 0), (3, 2, 4, 64, 8, 0, 0, 0), (61, 4, 12, 1001, 8, 0, 0, 0),
    (40, 8, 16, 520, 1, 8, 16, 0), (17, 3, 5, 136, 128, 3, 0, 0), (33, 9, 20, 4104, 1, 0, 8, 0),
    (9, 32, 40, 72, 1, 0, 0, 1), (300, 2, 8, 2048, 16, 0, 0, 0)]


@pytest.mark.parametrize("dtype", list(DTYPES))
@pytest.mark.parametrize("tokens,topk,experts,hidden,align,ts,rs,shift", ROWS)
def test_rows_there_and_back(tokens, topk, experts, hidden, align, ts, rs, shift, dtype):
    t, u = DTYPES[dtype], HALF_STEP[DTYPES[dtype]]
    gen = torch.Generator().manual_seed(hidden)
    p = mb.MoeProblem(tokens, topk, experts, hidden=hidden, first_expert=1, align=align,
                      dtype=dtype, token_stride=hidden + ts if ts else 0,
                      row_stride=hidden + rs if rs else 0)
    ids = torch.randint(0, experts + 2, (tokens, topk), generator=gen)
    cap = mb.moe_rows(p)
    _, _, at, _ = ref.sort(ids, experts, 1, align, cap)
    assert (at < 0).any() or tokens < 4

    def host(rows):
        return torch.randn(rows, hidden, generator=gen).to(t)

    def dev(x, pad):
        # rows `pad` elements apart more than dense, the first element shifted
        # off the 16-byte boundary by `shift` elements
        buf = torch.full((shift + x.shape[0] * (hidden + pad),), float("nan"), dtype=t,
                         device="cuda")
        view = buf[shift:].view(x.shape[0], hidden + pad)[:, :hidden]
        view.copy_(x)
        return view

    x, dy, h, before = host(tokens), host(tokens), host(cap), host(cap)
    w = torch.rand(tokens, topk, generator=gen) - 0.3
    kw = dict(row_of_slot=at.cuda(), problem=p, stream=torch.cuda.current_stream())
    used = torch.zeros(cap, dtype=torch.bool)
    used[at[at >= 0].long()] = True
    h[~used] = float("nan")  # padding rows are never read

    rows = dev(before, rs)
    mb.moe_dispatch(dev(x, ts), rows, **kw)
    assert torch.equal(rows.cpu(), ref.dispatch(x, at, before))

    for weights in (w, None):
        y = dev(torch.zeros_like(x), ts)
        mb.moe_combine(dev(h, rs), y, weights=None if weights is None else weights.cuda(), **kw)
        want, mag = ref.combine(h, weights, at)
        tol = topk * 2.0 ** -24 * mag + u * want.abs() * (1 + 2.0 ** -10) + SMALLEST[t]
        assert ((y.cpu().double() - want).abs() <= tol).all()

    want_rows, want_dw, mag = ref.combine_grad(dy, h, w, at, before)
    for inplace in (False, True):
        drows = dev(h if inplace else before, rs)
        dw = _new(tokens, topk, dtype=torch.float32)
        mb.moe_combine_grad(dev(dy, ts), drows if inplace else dev(h, rs), drows, dw,
                            weights=w.cuda(), **kw)
        got = drows.cpu()
        tol = (2.0 ** -24 + u) * (1 + 2.0 ** -10) * want_rows.abs() + SMALLEST[t]
        assert ((got.double() - want_rows).abs() <= tol)[used].all()
        if not inplace:
            assert torch.equal(got[~used], before[~used])
        assert ((dw.cpu().double() - want_dw).abs() <= hidden * 2.0 ** -24 * mag).all()
        assert (dw.cpu()[at < 0] == 0).all()


def test_gradients_against_differences():
    """dw and the rows' gradient of L = <dy, combine(rows, w)>, and dispatch's
    gradient, against differences of the kernels' own forward. L is linear in
    each argument, so a difference of step 1 is exact up to the two forwards'
    rounding: 64 elements of y, each a sum of 3 terms below 2 * 4 and so off by
    3 * 2^-24 * 24, times |dy| < 4; the gradients' own rounding is below that."""
    p = mb.MoeProblem(6, 3, 4, hidden=64, dtype=mb.DTYPE_F32)
    gen = torch.Generator().manual_seed(3)
    ids = torch.randint(0, 5, (6, 3), generator=gen)
    _, _, at, _ = ref.sort(ids, 4, 0, 1, mb.moe_rows(p))
    x, dy = (torch.randn(6, 64, generator=gen).cuda() for _ in range(2))
    h = torch.randn(mb.moe_rows(p), 64, generator=gen).cuda()
    w = torch.rand(6, 3, generator=gen).cuda()
    kw = dict(row_of_slot=at.cuda(), problem=p, stream=torch.cuda.current_stream())

    def loss(rows, weights):
        y = torch.empty_like(dy)
        mb.moe_combine(rows, y, weights=weights, **kw)
        return (y.double() * dy.double()).sum().item()

    drows, dw = torch.zeros_like(h), torch.empty_like(w)
    mb.moe_combine_grad(dy, h, drows, dw, weights=w, **kw)
    base = loss(h, w)
    tol = 2 * 64 * 3 * 2.0 ** -24 * 24 * 4
    for t, j in ((0, 0), (2, 1), (5, 2), (3, 0)):
        step = torch.zeros_like(w)
        step[t, j] = 1
        assert abs(loss(h, w + step) - base - dw[t, j].item()) < tol
    for r, c in ((0, 0), (3, 17), (int(at.max()), 63)):
        step = torch.zeros_like(h)
        step[r, c] = 1
        assert abs(loss(h + step, w) - base - drows[r, c].item()) < tol

    def moved(inp):
        rows = torch.zeros_like(h)
        mb.moe_dispatch(inp, rows, **kw)
        return (rows.double() * h.double()).sum().item()

    dx = torch.empty_like(x)
    mb.moe_combine(h, dx, **kw)
    step = torch.zeros_like(x)
    step[4, 9] = 1
    assert abs(moved(x + step) - moved(x) - dx[4, 9].item()) < tol


def test_captured_and_replayed_on_another_stream():
    """The whole pass captured on a side stream, replayed with new inputs in
    the same buffers; two graphs share the buffers, one after the other."""
    tokens, topk, experts, hidden = 3000, 4, 32, 256
    p = mb.MoeProblem(tokens, topk, experts, hidden=hidden)
    ids, x = _new(tokens, topk), torch.empty(tokens, hidden, dtype=torch.bfloat16, device="cuda")
    w = torch.ones(tokens, topk, device="cuda")
    out = (_new(experts), _new(experts + 1), _new(tokens, topk), _new(mb.moe_rows(p)))
    ws = torch.empty(mb.moe_workspace_bytes(p), dtype=torch.uint8, device="cuda")
    rows = torch.empty(mb.moe_rows(p), hidden, dtype=torch.bfloat16, device="cuda")
    y = torch.empty_like(x)

    def one_pass():
        kw = dict(problem=p, stream=torch.cuda.current_stream())
        mb.moe_sort(ids, counts=out[0], offsets=out[1], row_of_slot=out[2], slot_of_row=out[3],
                    workspace=ws, **kw)
        mb.moe_dispatch(x, rows, row_of_slot=out[2], **kw)
        mb.moe_combine(rows, y, weights=w, row_of_slot=out[2], **kw)

    graphs = []
    for _ in range(2):
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            one_pass()
        graphs.append(g)
    gen = torch.Generator().manual_seed(9)
    for i in range(4):
        new = torch.randint(0, experts, (tokens, topk), generator=gen)
        ids.copy_(new)
        x.copy_(torch.randint(-8, 9, (tokens, hidden), generator=gen))
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        want = ref.sort(new, experts, 0, 1, mb.moe_rows(p))
        for g, e in zip(out, want):
            assert torch.equal(g.cpu(), e)
        assert torch.equal(y, x * topk)  # whole numbers up to 32: exact in bf16


def test_rows_beyond_2_31_elements():
    """Row offsets pass 2^31 elements."""
    hidden, tokens = 1 << 20, 2200
    free, _ = torch.cuda.mem_get_info()
    if free < 16 << 30:
        pytest.skip("needs 16 GB")
    p = mb.MoeProblem(tokens, 1, 1, hidden=hidden, dtype=mb.DTYPE_F16)
    at = torch.arange(tokens - 1, -1, -1, dtype=torch.int32, device="cuda").view(-1, 1)
    x = torch.zeros(tokens, hidden, dtype=torch.float16, device="cuda")
    x[:, -1] = torch.arange(tokens, device="cuda")
    rows = torch.zeros_like(x)
    mb.moe_dispatch(x, rows, row_of_slot=at, problem=p, stream=torch.cuda.current_stream())
    assert torch.equal(rows[:, -1], x[:, -1].flip(0))
    y = torch.zeros_like(x)
    mb.moe_combine(rows, y, row_of_slot=at, problem=p, stream=torch.cuda.current_stream())
    assert torch.equal(y[:, -1], x[:, -1])


def test_entries_that_name_no_row_are_skipped():
    """Entries outside the sorted order's capacity count as slots without a row."""
    p = mb.MoeProblem(4, 2, 3, hidden=32, dtype=mb.DTYPE_F32)
    cap = mb.moe_rows(p)
    good = torch.tensor([[0, 1], [2, -1], [-1, -1], [5, 7]], dtype=torch.int32)
    bad = torch.tensor([[0, 1], [2, cap], [2 ** 31 - 1, -2 ** 31], [5, 7]], dtype=torch.int32)
    x, w = torch.randn(4, 32), torch.rand(4, 2)
    got = []
    for at in (good, bad):
        kw = dict(row_of_slot=at.cuda(), problem=p, stream=torch.cuda.current_stream())
        rows, y, drows = (torch.zeros(n, 32, device="cuda") for n in (cap, 4, cap))
        dw = torch.empty(4, 2, device="cuda")
        mb.moe_dispatch(x.cuda(), rows, **kw)
        mb.moe_combine(rows, y, weights=w.cuda(), **kw)
        mb.moe_combine_grad(x.cuda(), rows, drows, dw, weights=w.cuda(), **kw)
        got.append((rows, y, drows, dw))
    for a, b in zip(*got):
        assert torch.equal(a, b)


def test_long_sorts_in_a_row_wait_for_their_ids():
    """Sorts of two launches whose ids the kernel before them has just written,
    with nothing between them, give what they give with a synchronisation
    before each: no launch reads the ids before its own wait."""
    tokens, topk, experts, steps = 20000, 4, 64, 16
    p = mb.MoeProblem(tokens, topk, experts)
    gen = torch.Generator().manual_seed(4)
    order = torch.randperm(tokens, generator=gen).to(torch.int32).view(-1, 1).cuda()
    move = mb.MoeProblem(tokens, 1, 1, hidden=topk, dtype=mb.DTYPE_F32)
    first = torch.randint(0, experts, (tokens, topk), generator=gen, dtype=torch.int32).cuda()

    def run(sync):
        ids = [first.clone(), torch.empty_like(first)]
        got = []
        for i in range(steps):
            # permutes the ids' rows: their 32 bits as a row's elements
            mb.moe_dispatch(ids[0].view(torch.float32), ids[1].view(torch.float32),
                            row_of_slot=order, problem=move, stream=torch.cuda.current_stream())
            if sync:
                torch.cuda.synchronize()
            got.append(outs[i])
            mb.moe_sort(ids[1], counts=outs[i][0], offsets=outs[i][1], row_of_slot=outs[i][2],
                        slot_of_row=outs[i][3], workspace=ws, problem=p,
                        stream=torch.cuda.current_stream())
            ids.reverse()
        return [t.clone() for out in got for t in out]

    ws = _new(mb.moe_workspace_bytes(p), dtype=torch.uint8)
    assert ws.numel() > 0
    outs = [(_new(experts), _new(experts + 1), _new(tokens, topk), _new(mb.moe_rows(p)))
            for _ in range(steps)]
    want = run(True)
    ids = first.cpu()[torch.argsort(order.view(-1).long().cpu())]
    for g, w in zip(want[:4], ref.sort(ids, experts, 0, 1, mb.moe_rows(p))):
        assert torch.equal(g.cpu(), w)
    for _ in range(5):
        assert all(torch.equal(a, b) for a, b in zip(run(False), want))
