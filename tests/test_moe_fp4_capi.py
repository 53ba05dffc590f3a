"""Routing and 4-bit entry points without a GPU: what they refuse (a null
stream only validates), their sizes, and the layout of their structs."""
from __future__ import annotations

import ctypes
import os
import shutil
import subprocess

import pytest
import torch

import megacu_b200 as mb
import moe_fp4_ref as ref
from megacu_b200 import _capi

FAKE = 0x100000  # never dereferenced
ODD = FAKE + 2


def _status(fn, *args):
    st = fn(mb.driver_view(None, 0), *args)
    return st.code, st.detail


def _moe(**kw):
    base = dict(tokens=5, topk=2, experts=4, hidden=64)
    base.update(kw)
    return mb.MoeProblem(**base).to_c()


@pytest.mark.parametrize("bad,want", [
    (dict(tokens=-1), (1, 1)), (dict(topk=0), (1, 1)), (dict(experts=0), (1, 1)),
    (dict(align=0), (1, 1)), (dict(topk=33), (2, 22)), (dict(experts=1025), (2, 22)),
    (dict(align=2048), (2, 22)), (dict(tokens=1 << 30, topk=2), (2, 22)),
    (dict(tokens=1 << 62, topk=4), (2, 22)),
    (dict(), (0, 0)), (dict(tokens=0), (0, 0)), (dict(align=128), (0, 0))])
def test_sort_refuses(bad, want):
    lib = _capi.load()
    p = _moe(**bad)
    args = [FAKE] * 6
    assert _status(lib.megacu_cuda_moe_sort, *args, ctypes.byref(p)) == want
    assert _status(lib.megacu_cuda_moe_sort, *args, None) == (1, 2)
    sizes = (ctypes.c_int64 * 2)()
    st = lib.megacu_b200_moe_sizes(ctypes.byref(p), sizes)
    assert (st.code, st.detail) == want
    assert lib.megacu_b200_moe_sizes(ctypes.byref(_moe()), None).detail == 2


@pytest.mark.parametrize("i", range(5))
def test_sort_refuses_missing_and_misaligned_storage(i):
    lib = _capi.load()
    p = _moe()
    args = [FAKE] * 5
    args[i] = None
    assert _status(lib.megacu_cuda_moe_sort, *args, None, ctypes.byref(p)) == (1, 2)
    args[i] = ODD + 1
    assert _status(lib.megacu_cuda_moe_sort, *args, None, ctypes.byref(p)) == (1, 21)
    # many slots need a workspace, few do not
    big = _moe(tokens=1 << 20)
    assert _status(lib.megacu_cuda_moe_sort, *[FAKE] * 5, None, ctypes.byref(big)) == (1, 2)
    p.id_bytes = 2
    assert _status(lib.megacu_cuda_moe_sort, *[FAKE] * 6, ctypes.byref(p)) == (2, 20)


@pytest.mark.parametrize("bad,want", [
    (dict(hidden=0), (1, 1)), (dict(dtype=7), (2, 20)), (dict(token_stride=63), (1, 1)),
    (dict(row_stride=63), (1, 1)), (dict(topk=0), (1, 1)), (dict(), (0, 0)),
    (dict(row_stride=65, dtype=mb.DTYPE_F32), (0, 0))])
def test_row_moves_refuse(bad, want):
    lib = _capi.load()
    p = ctypes.byref(_moe(**bad))
    assert _status(lib.megacu_cuda_moe_dispatch, FAKE, FAKE, FAKE, p) == want
    assert _status(lib.megacu_cuda_moe_combine, FAKE, None, FAKE, FAKE, p) == want
    assert _status(lib.megacu_cuda_moe_combine_grad, *[FAKE] * 6, p) == want


def test_row_moves_refuse_storage():
    lib = _capi.load()
    p = ctypes.byref(_moe())
    for i in range(3):
        args = [FAKE] * 3
        args[i] = None
        assert _status(lib.megacu_cuda_moe_dispatch, *args, p) == (1, 2)
        args[i] = FAKE + 1
        assert _status(lib.megacu_cuda_moe_dispatch, *args, p) == (1, 21)
    for i in range(6):
        args = [FAKE] * 6
        args[i] = None
        assert _status(lib.megacu_cuda_moe_combine_grad, *args, p) == (1, 2)
    # an empty batch needs no storage
    empty = ctypes.byref(_moe(tokens=0))
    assert _status(lib.megacu_cuda_moe_dispatch, None, None, None, empty) == (0, 0)
    assert _status(lib.megacu_cuda_moe_combine, None, None, None, None, empty) == (0, 0)


@pytest.mark.parametrize("tokens,topk,experts,align", [(0, 2, 4, 128), (1, 8, 64, 128),
                                                       (64, 8, 4, 128), (100, 3, 7, 1),
                                                       (33, 5, 9, 24)])
def test_sort_capacity_holds_the_worst_case(tokens, topk, experts, align):
    """The capacity is enough whatever the ids, and tight for the worst ones:
    every expert that can has one slot more than a multiple of align."""
    p = mb.MoeProblem(tokens, topk, experts, align=align)
    slots = tokens * topk
    used = min(experts, slots)
    spread = [0] * experts
    for e in range(used):
        spread[e] = 1
    left = slots - used
    for e in range(used):  # whole multiples keep the paddings
        take = left // align * align if e == used - 1 else 0
        spread[e] += take
        left -= take
    if used:
        spread[used - 1] += left
    rows = sum(-(-c // align) * align for c in spread)
    assert rows <= mb.moe_rows(p) <= slots + used * (align - 1)
    assert mb.moe_rows(p) % align == 0


def _matrix(**kw):
    base = dict(rows=10, cols=64)
    base.update(kw)
    return mb.Fp4Matrix(**base).to_c()


@pytest.mark.parametrize("bad,want", [
    (dict(rows=-1), (1, 1)), (dict(cols=0), (1, 1)), (dict(cols=48), (1, 21)),
    (dict(format=2), (1, 1)), (dict(dtype=0), (2, 20)), (dict(scale=3.0), (1, 1)),
    (dict(scale=0.0), (1, 1)), (dict(scale=-2.0), (1, 1)), (dict(scale=float("inf")), (1, 1)),
    (dict(scale=float("nan")), (1, 1)), (dict(scale=2.0 ** 61), (1, 1)),
    (dict(scale=2.0 ** -60), (0, 0)), (dict(stride=63), (1, 1)), (dict(stride=-1), (1, 1)),
    (dict(rows=(1 << 30) + 1), (2, 22)), (dict(rows=1 << 30, cols=1 << 30), (2, 22)),
    (dict(), (0, 0)), (dict(rows=0), (0, 0)), (dict(format=mb.FP4_NV, cols=32), (0, 0))])
def test_quantize_refuses(bad, want):
    lib = _capi.load()
    m = ctypes.byref(_matrix(**bad))
    assert _status(lib.megacu_cuda_fp4_quantize, FAKE, None, FAKE, FAKE, m) == want
    assert _status(lib.megacu_cuda_fp4_dequantize, FAKE, FAKE, FAKE, m) == want
    if "stride" not in bad:
        st = lib.megacu_b200_fp4_sizes(m, (ctypes.c_int64 * 2)())
        assert (st.code, st.detail) == want


def test_quantize_refuses_storage_and_options():
    lib = _capi.load()
    m = ctypes.byref(_matrix())
    q, d = lib.megacu_cuda_fp4_quantize, lib.megacu_cuda_fp4_dequantize
    for args in ((None, None, FAKE, FAKE), (FAKE, None, None, FAKE), (FAKE, None, FAKE, None)):
        assert _status(q, *args, m) == (1, 2)
    for args in ((FAKE + 1, None, FAKE, FAKE), (FAKE, None, FAKE + 8, FAKE),
                 (FAKE, None, FAKE, FAKE + 8), (FAKE, FAKE + 2, FAKE, FAKE)):
        assert _status(q, *args, m) == (1, 21)
    t = _matrix(transpose=True)
    assert _status(q, FAKE, FAKE, FAKE, FAKE, ctypes.byref(t)) == (2, 22)
    assert _status(d, FAKE, FAKE, FAKE, ctypes.byref(t)) == (2, 22)
    t = _matrix()
    t.topk = 2
    assert _status(q, FAKE, None, FAKE, FAKE, ctypes.byref(t)) == (1, 2)
    assert _status(q, FAKE, FAKE, FAKE, FAKE, ctypes.byref(t)) == (1, 1)
    t.x_rows = 5
    assert _status(q, FAKE, FAKE, FAKE, FAKE, ctypes.byref(t)) == (0, 0)
    t.scatter = 1
    assert _status(q, FAKE, FAKE, FAKE, FAKE, ctypes.byref(t)) == (0, 0)
    assert _status(q, FAKE, None, FAKE, FAKE, ctypes.byref(t)) == (1, 2)
    t.topk = 0
    assert _status(q, FAKE, FAKE, FAKE, FAKE, ctypes.byref(t)) == (1, 1)
    t.topk = 2
    assert _status(d, FAKE, FAKE, FAKE, ctypes.byref(t)) == (2, 22)
    # a transposed matrix's stride is between its stored rows
    t = _matrix(transpose=True, rows=10, cols=64, stride=12)
    assert _status(q, FAKE, None, FAKE, FAKE, ctypes.byref(t)) == (0, 0)


@pytest.mark.parametrize("rows,cols,fmt,data,scales", [
    (1, 32, mb.FP4_MX, 16, 512), (129, 160, mb.FP4_MX, 129 * 80, 2 * 2 * 512),
    (128, 160, mb.FP4_NV, 128 * 80, 3 * 512), (0, 64, mb.FP4_NV, 0, 0)])
def test_fp4_sizes(rows, cols, fmt, data, scales):
    assert mb.fp4_sizes(mb.Fp4Matrix(rows, cols, format=fmt)) == (data, scales)
    assert mb.fp4_events_bytes() == 256


def _gemm(**kw):
    base = dict(m=256, n=96, k=64)
    base.update(kw)
    return mb.Fp4Gemm(**base).to_c()


@pytest.mark.parametrize("bad,want", [
    (dict(m=-1), (1, 1)), (dict(n=0), (1, 1)), (dict(k=0), (1, 1)), (dict(k=40), (1, 21)),
    (dict(format=3), (1, 1)), (dict(out_dtype=0), (2, 20)), (dict(out_stride=95), (1, 1)),
    (dict(experts=-1), (1, 1)), (dict(experts=1025), (2, 22)), (dict(experts=4, m=130), (2, 22)),
    (dict(tile_n=32), (2, 22)), (dict(tile_n=64, split=8, k=4096), (2, 22)), (dict(split=3), (2, 22)), (dict(split=2), (2, 22)),
    (dict(split=2, k=512), (0, 0)), (dict(m=1 << 31), (2, 22)), (dict(n=1 << 29, experts=4), (2, 22)),
    (dict(), (0, 0)), (dict(m=0), (0, 0)), (dict(experts=4), (0, 0)), (dict(m=1, n=1, k=32), (0, 0))])
def test_products_refuse(bad, want):
    lib = _capi.load()
    p = ctypes.byref(_gemm(**bad))
    assert _status(lib.megacu_cuda_fp4_gemm, *[FAKE] * 9, p) == want
    assert _status(lib.megacu_cuda_fp4_gemm_swiglu, *[FAKE] * 11, p) == want


def test_products_refuse_storage():
    lib = _capi.load()
    fn = lib.megacu_cuda_fp4_gemm_swiglu
    names = ("a", "a_scales", "gate", "gate_scales", "up", "up_scales", "offsets", "counts",
             "alphas", "act", "events")
    for i, name in enumerate(names):
        for experts in (0, 2):
            p = ctypes.byref(_gemm(experts=experts))
            args = [FAKE] * 11
            args[i] = None
            optional = name == "alphas" or (experts == 0 and name in ("offsets", "counts"))
            assert _status(fn, *args, p) == ((0, 0) if optional else (1, 2)), name
            args[i] = FAKE + 1
            assert _status(fn, *args, p) == (1, 21), name
    assert _status(fn, *[FAKE] * 11, None) == (1, 2)
    p = ctypes.byref(_gemm(tile_n=128))
    assert _status(fn, *[FAKE] * 11, p) == (2, 22)  # SwiGLU tiles are 128 gate + 128 up


def _mlp(**kw):
    base = dict(tokens=5, hidden=64, inter=96, topk=2, experts=4)
    base.update(kw)
    return mb.MoeMlp(**base).to_c()


@pytest.mark.parametrize("bad,want", [
    (dict(tokens=-1), (1, 1)), (dict(hidden=40), (1, 21)), (dict(inter=0), (1, 1)),
    (dict(inter=33), (1, 21)), (dict(topk=0), (1, 1)), (dict(experts=1025), (2, 22)),
    (dict(dtype=0), (2, 20)), (dict(format=2), (1, 1)), (dict(x_scale=3.0), (1, 1)),
    (dict(act_scale=-1.0), (1, 1)), (dict(x_scale=0.0), (0, 0)), (dict(), (0, 0)),
    (dict(tokens=0), (0, 0))])
def test_routed_mlp_refuses(bad, want):
    lib = _capi.load()
    p = ctypes.byref(_mlp(**bad))
    assert _status(lib.megacu_cuda_moe_mlp_fp4, *[FAKE] * 14, p) == want
    st = lib.megacu_b200_moe_mlp_workspace_bytes(p, ctypes.byref(ctypes.c_int64()))
    assert (st.code, st.detail) == want


def test_routed_mlp_refuses_storage():
    lib = _capi.load()
    p = ctypes.byref(_mlp())
    names = ("x", "expert_ids", "weights", "gate", "gate_scales", "up", "up_scales", "down",
             "down_scales", "up_alphas", "down_alphas", "y", "workspace", "events")
    for i, name in enumerate(names):
        args = [FAKE] * 14
        args[i] = None
        want = (0, 0) if name.endswith("alphas") else (1, 2)
        assert _status(lib.megacu_cuda_moe_mlp_fp4, *args, p) == want, name
        args[i] = FAKE + 1
        assert _status(lib.megacu_cuda_moe_mlp_fp4, *args, p) == (1, 21), name
    empty = ctypes.byref(_mlp(tokens=0))
    assert _status(lib.megacu_cuda_moe_mlp_fp4, *[None] * 14, empty) == (0, 0)


def test_wrappers_check_tensors():
    """Shapes, types and strides of tensors are checked before the call."""
    p = mb.MoeProblem(4, 2, 3, hidden=8)
    x = torch.zeros(4, 8, dtype=torch.bfloat16)
    rows = torch.zeros(mb.moe_rows(p), 8, dtype=torch.bfloat16)
    at = torch.zeros(4, 2, dtype=torch.int32)
    mb.moe_dispatch(x, rows, row_of_slot=at, problem=p)  # no stream: validates only
    for bad in (x.float(), x[:3], x.t().contiguous().t()):
        with pytest.raises(ValueError):
            mb.moe_dispatch(bad, rows, row_of_slot=at, problem=p)
    with pytest.raises(ValueError):
        mb.moe_dispatch(x, rows, row_of_slot=at.long(), problem=p)
    wide = torch.zeros(4, 12, dtype=torch.bfloat16)
    strided = mb.MoeProblem(4, 2, 3, hidden=8, token_stride=12)
    mb.moe_dispatch(wide[:, :8], rows, row_of_slot=at, problem=strided)
    with pytest.raises(ValueError):
        mb.moe_dispatch(x, rows, row_of_slot=at, problem=strided)
    m = mb.Fp4Matrix(4, 32)
    data, scales = (torch.zeros(n, dtype=torch.uint8) for n in mb.fp4_sizes(m))
    plain = torch.zeros(4, 32, dtype=torch.bfloat16)
    mb.fp4_quantize(plain, data, scales, problem=m)
    with pytest.raises(ValueError):
        mb.fp4_quantize(plain, data[1:], scales, problem=m)
    m.cols = 64  # a changed field is seen by the next call
    with pytest.raises(ValueError):
        mb.fp4_quantize(plain, data, scales, problem=m)


def test_struct_layouts(tmp_path):
    cc = shutil.which("gcc")
    if cc is None:
        pytest.skip("no C compiler")
    from megacu_b200 import build
    structs = {"megacu_moe_problem": _capi.MoeProblem, "megacu_fp4_matrix": _capi.Fp4Matrix,
               "megacu_fp4_gemm_problem": _capi.Fp4GemmProblem,
               "megacu_moe_mlp_problem": _capi.MoeMlpProblem}
    lines, want = [], []
    for c_name, py in structs.items():
        lines.append(f'  printf("%zu\\n", sizeof({c_name}));')
        want.append(ctypes.sizeof(py))
        for field, _ in py._fields_:
            lines.append(f'  printf("%zu\\n", offsetof({c_name}, {field}));')
            want.append(getattr(py, field).offset)
    (tmp_path / "layout.c").write_text(
        "#include <stddef.h>\n#include <stdio.h>\n#include <megacu_b200.h>\n"
        "int main(void) {\n" + "\n".join(lines) + "\n  return 0;\n}\n")
    exe = str(tmp_path / "layout")
    subprocess.run([cc, "-std=c99", "-Wall", "-Werror", "-I" + os.path.join(build.ROOT, "include"),
                    str(tmp_path / "layout.c"), "-o", exe], check=True)
    got = [int(x) for x in subprocess.run([exe], capture_output=True, text=True,
                                          check=True).stdout.split()]
    assert got == want


@pytest.mark.parametrize("fmt", [mb.FP4_MX, mb.FP4_NV])
def test_reference_quantiser_against_every_element(fmt):
    """The tests' own quantiser picks the nearest element, the even code at a
    tie, by brute force over the sixteen values."""
    gen = torch.Generator().manual_seed(5)
    x = torch.randn(64, 64, generator=gen, dtype=torch.float64) * 3
    x[0, :32] = torch.arange(32) / 8.0      # every border, amax 3.875
    x[1, :32] = torch.arange(32) * 0.25
    code, byte = ref.quantize(x, fmt)
    s = ref.SCALES[fmt][byte].repeat_interleave(ref.BLOCK[fmt], 1)
    dist = (x.abs()[..., None] - ref.ELEMENTS[:8] * s[..., None]).abs()
    best = dist.amin(-1, keepdim=True)
    near = dist == best
    mag = code % 8
    assert near.gather(-1, mag[..., None]).all()
    tie = near.sum(-1) == 2
    assert (mag[tie] % 2 == 0).all() and tie.any()
    data, tiled = ref.pack(code, byte)
    assert torch.equal(ref.values(data, tiled, fmt), ref.ELEMENTS[code] * s)


def test_scattered_quantisation_needs_its_choices():
    """row_of_slot is a map of `topk` entries per row of x, never a mask of the
    matrix's rows: without topk, or with another one than the map's, the call
    is refused, whatever the map's length."""
    m = mb.Fp4Matrix(4, 32)
    data, scales = (torch.zeros(n, dtype=torch.uint8) for n in mb.fp4_sizes(m))
    x = torch.zeros(4, 32, dtype=torch.bfloat16)
    for at in (torch.tensor([2, 0, 3, 1], dtype=torch.int32), torch.zeros(1, dtype=torch.int32),
               torch.zeros(4, 1, dtype=torch.int32), FAKE):
        with pytest.raises(ValueError, match="topk"):
            mb.fp4_quantize(x, data, scales, problem=m, row_of_slot=at)
        with pytest.raises(ValueError, match="topk"):
            mb.fp4_quantize(x, data, scales, problem=m, row_of_slot=at, topk=-1)
    with pytest.raises(ValueError, match="topk"):
        mb.fp4_quantize(x[:2], data, scales, problem=m, topk=1,
                        row_of_slot=torch.zeros(2, 2, dtype=torch.int32))
    mb.fp4_quantize(x, data, scales, problem=m, topk=1,
                    row_of_slot=torch.zeros(4, 1, dtype=torch.int32))
    mb.fp4_quantize(x, data, scales, problem=m, topk=1,
                    row_of_slot=torch.zeros(4, dtype=torch.int32))


def test_problems_are_used_by_several_threads_at_once(monkeypatch):
    """Threads that meet on a new problem all get its C struct, whichever of
    them builds it, and a changed field's struct after the change."""
    import threading
    import time

    byref = ctypes.byref

    def slow_byref(c):  # holds the window open between a struct and its pointer
        time.sleep(0.002)
        return byref(c)

    monkeypatch.setattr(mb.api.ctypes, "byref", slow_byref)
    for i in range(10):
        p = mb.MoeProblem(i, 2, 4)
        gate = threading.Barrier(4)
        seen, errors = [], []

        def use(late):
            try:
                gate.wait()
                time.sleep(late * 0.001)
                seen.append(p._pointer()._obj.tokens)
                seen.append(p._wide_ids()._obj.tokens)
                mb.moe_rows(p)
            except Exception as e:  # a thread's error must reach the test
                errors.append(repr(e))

        threads = [threading.Thread(target=use, args=(n,)) for n in range(4)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert errors == [] and set(seen) == {i}
        p.tokens = i + 1
        assert p._pointer()._obj.tokens == p._wide_ids()._obj.tokens == i + 1


def test_used_problems_can_be_copied_and_pickled():
    """A problem's struct and pointers are its own: a copy of one that calls
    have used has the fields, builds its own and follows its own changes."""
    import copy
    import dataclasses
    import pickle

    problems = (mb.MoeProblem(5, 2, 4, hidden=64), mb.Fp4Matrix(10, 64), mb.Fp4Gemm(256, 96, 64),
                mb.MoeMlp(5, 64, 96, 2, 4))
    for p in problems:
        p._pointer()
        if hasattr(p, "_wide_ids"):
            p._wide_ids()
        for q in (copy.copy(p), copy.deepcopy(p), pickle.loads(pickle.dumps(p)),
                  dataclasses.replace(p)):
            assert q == p and q.to_c() is not p.to_c()
            first = dataclasses.fields(q)[0].name
            setattr(q, first, 7)
            assert getattr(q.to_c(), first) == 7 and getattr(p.to_c(), first) != 7


@pytest.mark.parametrize("block", [False, True])
def test_width_of_expert_ids(monkeypatch, block):
    """A tensor's type is its ids' width; an address has the problem's id_bytes
    (0: 32 bits), and a tensor of the other type than a given id_bytes is
    refused."""
    lib = _capi.load()
    seen = []

    class Spy:
        def __getattr__(self, name):
            fn = getattr(lib, name)
            if name not in ("megacu_cuda_moe_sort", "megacu_cuda_moe_mlp_fp4"):
                return fn

            def call(*args):
                seen.append(args[-1]._obj.id_bytes)
                return fn(*args)

            return call

    monkeypatch.setattr(mb.api, "lib", lambda: Spy())

    def call(ids, **kw):
        seen.clear()
        if block:
            p = mb.MoeMlp(5, 64, 96, 2, 4, **kw)
            mb.moe_mlp_fp4(FAKE, ids, *[FAKE] * 8, workspace=FAKE, events=FAKE, problem=p)
        else:
            p = mb.MoeProblem(5, 2, 4, **kw)
            mb.moe_sort(ids, counts=FAKE, offsets=FAKE, row_of_slot=FAKE, slot_of_row=FAKE,
                        problem=p)
        return seen[0]

    narrow, wide = (torch.zeros(5, 2, dtype=t) for t in (torch.int32, torch.int64))
    assert call(narrow) in (0, 4) and call(wide) == 8
    assert call(FAKE) in (0, 4) and call(FAKE, id_bytes=8) == 8 and call(FAKE, id_bytes=4) == 4
    assert call(wide, id_bytes=8) == 8 and call(narrow, id_bytes=4) == 4
    for ids, width in ((narrow, 8), (wide, 4)):
        with pytest.raises(ValueError, match="expert_ids"):
            call(ids, id_bytes=width)
    with pytest.raises(mb.MegacuError):
        call(FAKE, id_bytes=2)


def test_sizes_are_refused_without_a_stream():
    """A call that only validates refuses what a launch would: the composed
    block launches nothing before all its parts have passed."""
    lib = _capi.load()
    # B's scale tiles past 2^31: 1024 experts x 2^13 row tiles x 2^23 tiles of K
    huge = ctypes.byref(_gemm(m=128, n=1 << 20, k=1 << 30, experts=1024))
    assert _status(lib.megacu_cuda_fp4_gemm, *[FAKE] * 9, huge) == (2, 22)
    # A's: 2^16 row tiles x 2^23
    huge = ctypes.byref(_gemm(m=1 << 23, n=64, k=1 << 30))
    assert _status(lib.megacu_cuda_fp4_gemm, *[FAKE] * 9, huge) == (2, 22)
    # a scatter's CTAs, 32 rows of x x 256 columns each: 2^31 - 2^10, 2^31, and
    # more rows than a matrix may have
    for x_rows, want in (((1 << 26) - 32, (0, 0)), (1 << 26, (2, 22)), ((1 << 30) + 1, (2, 22)),
                         (1 << 62, (2, 22)), ((1 << 63) - 1, (2, 22))):
        m = _matrix(rows=128, cols=1 << 18)
        m.topk, m.x_rows, m.scatter = 1, x_rows, 1
        assert _status(lib.megacu_cuda_fp4_quantize, *[FAKE] * 4, ctypes.byref(m)) == want


def test_gathered_rows_of_a_batch_of_sequences(monkeypatch):
    """x of any dense shape is its rows of `cols` elements, as for the other
    calls: all of them are there to be gathered or scattered."""
    lib = _capi.load()
    seen = []

    class Spy:
        def __getattr__(self, name):
            fn = getattr(lib, name)
            if name != "megacu_cuda_fp4_quantize":
                return fn

            def call(*args):
                seen.append(args[-1]._obj.x_rows)
                return fn(*args)

            return call

    monkeypatch.setattr(mb.api, "lib", lambda: Spy())
    m = mb.Fp4Matrix(128, 32)
    data, scales = (torch.zeros(n, dtype=torch.uint8) for n in mb.fp4_sizes(m))
    for shape in ((2, 3, 32), (6, 32), (192,)):
        x = torch.zeros(shape, dtype=torch.bfloat16)
        mb.fp4_quantize(x, data, scales, problem=m, topk=2,
                        slot_of_row=torch.zeros(128, dtype=torch.int32))
        mb.fp4_quantize(x, data, scales, problem=m, topk=2,
                        row_of_slot=torch.zeros(6, 2, dtype=torch.int32))
        with pytest.raises(ValueError):
            mb.fp4_quantize(x, data, scales, problem=m, topk=2,
                            row_of_slot=torch.zeros(5, 2, dtype=torch.int32))
    assert seen == [6] * 6
    strided = mb.Fp4Matrix(128, 32, stride=40)
    wide = torch.zeros(6, 40, dtype=torch.bfloat16)
    mb.fp4_quantize(wide[:, :32], data, scales, problem=strided, topk=2,
                    slot_of_row=torch.zeros(128, dtype=torch.int32))
    assert seen[-1] == 6


def test_sort_refuses_more_slots_than_it_is_made_for():
    """Up to 2^26 slots: its second launch's work grows with the square. Calls
    on an order that another sort made have no such bound."""
    lib = _capi.load()
    for tokens, want in ((1 << 23, (0, 0)), ((1 << 23) + 1, (2, 22)), (1 << 27, (2, 22))):
        p = ctypes.byref(_moe(tokens=tokens, topk=8))
        assert _status(lib.megacu_cuda_moe_sort, *[FAKE] * 6, p) == want
        assert _status(lib.megacu_cuda_moe_dispatch, *[FAKE] * 3, p) == (0, 0)
        st = lib.megacu_b200_moe_sizes(p, (ctypes.c_int64 * 2)())
        assert (st.code, st.detail) == (0, 0)
