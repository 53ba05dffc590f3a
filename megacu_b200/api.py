"""Python host mirror of megacu's GEMM + allreduce entry points.

Thin wrappers over the C ABI (``include/megacu_b200.h``): torch tensors are
only device-memory holders here, every byte of work runs in
``libmegacu_b200.so``. Names and argument meaning follow megacu:

* :func:`cuda_nvshmem_gemm_allreduce_phased_orchestrate` — megacu's fp32
  orchestrate entry (phased/megacu/gemm_allreduce_phased_orchestrate.cc:3-20);
* :func:`megacu_cuda_gemm_allreduce_phased_f32` — its native launcher
  (megacu_gemm_allreduce_phased.cu:157-232);
* :func:`gemm_allreduce` / :func:`gemm_reduce_scatter` — the bf16 fused
  megakernel (B200 path), orchestrated through the same phase API;
* :class:`Team` — the symmetric heap that replaces NVSHMEM's.

Errors come back as :class:`MegacuError` carrying megacu's status code and
per-site detail number.
"""
from __future__ import annotations

import ctypes
import weakref
from dataclasses import dataclass, fields
from typing import Callable, Optional, Sequence

from . import _capi
from ._capi import DriverView, GemmArProblem, GemmArProblemV2, Status


class MegacuError(RuntimeError):
    def __init__(self, status: Status):
        self.code = int(status.code)
        self.detail = int(status.detail)
        self.message = status.message.decode() if status.message else ""
        super().__init__(f"megacu {_capi.STATUS_NAMES[self.code]} (detail {self.detail}): "
                         f"{self.message}")


def check(status: Status) -> Status:
    if status.code != _capi.OK:
        raise MegacuError(status)
    return status


def lib() -> ctypes.CDLL:
    return _capi.load()


def _ptr(x) -> Optional[int]:
    if x is None:
        return None
    if isinstance(x, int):
        return x
    return x.data_ptr()


CUDA_STREAM_LEGACY = 1  # cudaStreamLegacy: the legacy default stream, named explicitly


def _stream_handle(stream) -> Optional[int]:
    """Raw cudaStream_t of ``stream``. None stays None (megacu: validate only);
    torch's default stream (handle 0) is passed as cudaStreamLegacy so that it
    is not mistaken for "no stream"."""
    if stream is None:
        return None
    handle = stream if isinstance(stream, int) else stream.cuda_stream
    return handle if handle != 0 else CUDA_STREAM_LEGACY


# ---- team ----------------------------------------------------------------------

class Team:
    """This PE's symmetric heap, mapped by every peer of the team.

    ``exchange`` maps this PE's handle (bytes) to the list of every PE's
    handle in PE order — e.g. :func:`torch_exchange` over torch.distributed.
    Every PE must create the team and allocate from it in the same order
    (as with ``nvshmem_init`` / ``nvshmem_malloc``).

    ``multicast_bytes > 0`` also sets up a multicast (NVLS) region of at least
    that size (one process per PE; rounded up to the multicast granularity).
    Where the device, driver or team shape cannot have one, the team works
    without it (``self.multicast`` is False); every PE reaches the same
    decision, since all see every PE's set-up blob.
    """

    def __init__(self, my_pe: int, n_pes: int, device: int, heap_bytes: int,
                 exchange: Optional[Callable[[bytes], Sequence[bytes]]] = None,
                 multicast_bytes: int = 0):
        self.my_pe, self.n_pes, self.device = my_pe, n_pes, device
        handle = ctypes.c_void_p()
        check(lib().megacu_b200_team_create(my_pe, n_pes, device, heap_bytes,
                                            ctypes.byref(handle)))
        self.handle = handle.value
        # A team still open when the interpreter exits (an exception on the
        # way) is destroyed then: a process must not end with its memory bound
        # to a multicast object while the other PEs still use it.
        self._finalizer = weakref.finalize(self, _destroy_team, self.handle)
        if n_pes > 1:
            if exchange is None:
                raise ValueError("a team of more than one PE needs an exchange function")
            mine = ctypes.create_string_buffer(_capi.TEAM_HANDLE_BYTES)
            check(lib().megacu_b200_team_export(self.handle, mine))
            handles = list(exchange(mine.raw))
            if len(handles) != n_pes or any(len(h) != _capi.TEAM_HANDLE_BYTES for h in handles):
                raise ValueError("exchange must return one 128-byte handle per PE")
            blob = ctypes.create_string_buffer(b"".join(handles), n_pes * _capi.TEAM_HANDLE_BYTES)
            check(lib().megacu_b200_team_connect(self.handle, blob))
        base = ctypes.c_void_p()
        size = ctypes.c_int64()
        check(lib().megacu_b200_team_info(self.handle, None, None, ctypes.byref(base),
                                          ctypes.byref(size)))
        self.heap_base, self.heap_bytes = base.value, size.value
        self.multicast = False
        self.multicast_error = None
        if multicast_bytes > 0 and n_pes > 1:
            self._connect_multicast(multicast_bytes, exchange)

    def _connect_multicast(self, nbytes: int, exchange) -> None:
        mine = ctypes.create_string_buffer(_capi.TEAM_HANDLE_BYTES)
        st = lib().megacu_b200_team_multicast_export(self.handle, nbytes, mine)
        if st.code != _capi.OK:
            self.multicast_error = MegacuError(st)
        handles = list(exchange(mine.raw if st.code == _capi.OK else
                                bytes(_capi.TEAM_HANDLE_BYTES)))
        # A PE that could not export sends zeros: then nobody connects.
        if any(not any(h[:4]) for h in handles):
            if self.multicast_error is None:
                self.multicast_error = RuntimeError("a peer cannot set up a multicast region")
            return
        blob = ctypes.create_string_buffer(b"".join(handles), self.n_pes * _capi.TEAM_HANDLE_BYTES)
        st = lib().megacu_b200_team_multicast_connect(self.handle, blob)
        if st.code != _capi.OK:
            self.multicast_error = MegacuError(st)
            return
        base = ctypes.c_void_p()
        size = ctypes.c_int64()
        check(lib().megacu_b200_team_multicast_info(self.handle, ctypes.byref(base),
                                                    ctypes.byref(size)))
        self.multicast = size.value > 0
        self.multicast_base, self.multicast_bytes = base.value, size.value

    def malloc(self, nbytes: int) -> int:
        ptr = ctypes.c_void_p()
        check(lib().megacu_b200_team_malloc(self.handle, nbytes, ctypes.byref(ptr)))
        return ptr.value

    def multicast_malloc(self, nbytes: int) -> int:
        ptr = ctypes.c_void_p()
        check(lib().megacu_b200_team_multicast_malloc(self.handle, nbytes, ctypes.byref(ptr)))
        return ptr.value

    def tensor(self, shape, dtype, multicast: bool = False):
        """A torch tensor over a fresh symmetric allocation (zero-filled), in
        the heap or, with ``multicast=True``, in the multicast region."""
        import torch
        numel = 1
        for s in shape:
            numel *= s
        itemsize = torch.empty((), dtype=dtype).element_size()
        nbytes = max(numel * itemsize, 16)
        ptr = self.multicast_malloc(nbytes) if multicast else self.malloc(nbytes)
        return tensor_from_pointer(ptr, shape, dtype, self.device, owner=self)

    def barrier(self, stream=None) -> None:
        check(lib().megacu_b200_team_barrier(self.handle, _stream_handle(stream)))

    def close(self) -> None:
        """Destroys the team; collective when it has a multicast region."""
        if self.handle is not None:
            finalizer = getattr(self, "_finalizer", None)
            if finalizer is not None:
                finalizer.detach()
            check(lib().megacu_b200_team_destroy(self.handle))
            self.handle = None

    def __enter__(self) -> "Team":
        return self

    def __exit__(self, *exc) -> None:
        self.close()

    def view(self) -> _capi.TeamView:
        return _capi.TeamView(team=self.handle, team_my_pe=self.my_pe, team_n_pes=self.n_pes,
                              world_my_pe=self.my_pe, world_n_pes=self.n_pes,
                              cuda_device_ordinal=self.device)


def _destroy_team(handle) -> None:
    lib().megacu_b200_team_destroy(handle)


def torch_exchange(group=None) -> Callable[[bytes], Sequence[bytes]]:
    """Handle exchange over torch.distributed (any backend; gloo works)."""
    import torch.distributed as dist

    def exchange(mine: bytes) -> Sequence[bytes]:
        out = [None] * dist.get_world_size(group)
        dist.all_gather_object(out, mine, group=group)
        return out

    return exchange


def local_exchange(session: str, my_pe: int, n_pes: int,
                   timeout_ms: int = 60_000) -> Callable[[bytes], Sequence[bytes]]:
    """Handle exchange among the processes of one node without
    torch.distributed: every PE passes the same ``session`` string
    (megacu_b200_exchange_local, an abstract unix socket served by PE 0).
    Each call of the returned function is one collective exchange."""
    name = session.encode()

    def exchange(mine: bytes) -> Sequence[bytes]:
        size = len(mine)
        out = ctypes.create_string_buffer(size * n_pes)
        check(lib().megacu_b200_exchange_local(name, my_pe, n_pes, mine, size, out, timeout_ms))
        raw = out.raw
        return [raw[i * size:(i + 1) * size] for i in range(n_pes)]

    return exchange


def env_team(heap_bytes: int, multicast_bytes: int = 0, timeout_ms: int = 60_000) -> "Team":
    """A team of the processes torchrun (or any launcher setting LOCAL_RANK /
    LOCAL_WORLD_SIZE) started on this node, one per GPU, PE = local rank,
    built without torch.distributed. The session is MEGACU_B200_SESSION if
    set, else derived from MASTER_ADDR, MASTER_PORT and TORCHELASTIC_RUN_ID."""
    import os
    env = os.environ
    my_pe = int(env.get("LOCAL_RANK", env.get("RANK", "0")))
    n_pes = int(env.get("LOCAL_WORLD_SIZE", env.get("WORLD_SIZE", "1")))
    session = env.get("MEGACU_B200_SESSION") or "{}.{}.{}".format(
        env.get("MASTER_ADDR", "local"), env.get("MASTER_PORT", "0"),
        env.get("TORCHELASTIC_RUN_ID", "none"))
    return Team(my_pe, n_pes, my_pe, heap_bytes,
                local_exchange(session[:64], my_pe, n_pes, timeout_ms) if n_pes > 1 else None,
                multicast_bytes=multicast_bytes)


class _CudaArray:
    def __init__(self, ptr, shape, typestr, owner):
        self.__cuda_array_interface__ = {"shape": tuple(shape), "typestr": typestr,
                                         "data": (ptr, False), "version": 3, "strides": None}
        self._owner = owner


def tensor_from_pointer(ptr: int, shape, dtype, device: int, owner=None):
    """Wraps device memory at ``ptr`` as a torch tensor (no copy, no ownership)."""
    import torch
    codes = {torch.bfloat16: ("<i2", torch.bfloat16), torch.float16: ("<f2", None),
             torch.float32: ("<f4", None), torch.int32: ("<i4", None),
             torch.uint8: ("|u1", None), torch.int64: ("<i8", None)}
    typestr, view_as = codes[dtype]
    with torch.cuda.device(device):
        t = torch.as_tensor(_CudaArray(ptr, shape, typestr, owner), device=f"cuda:{device}")
    return t.view(view_as) if view_as is not None else t


# ---- driver views ------------------------------------------------------------------

_VIEWS: dict = {}  # (stream handle, device) -> DriverView of a one-PE call


def _launch_view(stream, device: int, team: Optional[Team]) -> DriverView:
    """driver_view() for the launch wrappers below, built once per (stream,
    device) and team: the struct is passed by value, so the cached object is
    never changed by a call. (driver_view itself returns a fresh struct, which
    callers may modify.)"""
    key = (_stream_handle(stream), device)
    cache = _VIEWS if team is None else team.__dict__.setdefault("_views", {})
    d = cache.get(key)
    if d is None:
        d = cache[key] = driver_view(stream, device, team)
    return d


def driver_view(stream=None, device: int = 0, team: Optional[Team] = None) -> DriverView:
    """megacu's driver_view{launch_view, team_view} for this PE."""
    d = DriverView()
    d.launch.stream = _stream_handle(stream)
    d.launch.device_ordinal = device
    if team is not None:
        d.team = team.view()
    else:
        d.team.team_my_pe, d.team.team_n_pes = 0, 1
        d.team.world_my_pe, d.team.world_n_pes = 0, 1
        d.team.cuda_device_ordinal = device
    return d


# ---- bf16 fused megakernel ---------------------------------------------------------

@dataclass
class Problem:
    """megacu_gemm_ar_problem_v2: out[m, n] = sum over PEs of a[m, k] @ b[k, n]."""
    m: int
    n: int
    k: int
    mode: int = _capi.MODE_ALLREDUCE
    algo: int = _capi.ALGO_AUTO
    deterministic: bool = False
    tile_n: int = 0
    num_ctas: int = 0
    timeout_ns: int = 0
    cta_pairs: int = _capi.CTA_PAIRS_AUTO

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        self.__dict__.pop("_c", None)  # a changed field rebuilds the C struct

    def to_c(self, trace_ptr: Optional[int] = None, trace_capacity: int = 0) -> GemmArProblemV2:
        """The C struct (passed by value). Without a trace it is built once and
        reused until a field changes."""
        if trace_ptr is None and trace_capacity == 0:
            c = self.__dict__.get("_c")
            if c is not None:
                return c
        c = GemmArProblemV2(m=self.m, n=self.n, k=self.k, tile_m=0, tile_n=self.tile_n,
                            mode=self.mode, algo=self.algo,
                            deterministic=1 if self.deterministic else 0,
                            dtype=_capi.DTYPE_BF16, num_ctas=self.num_ctas,
                            cta_pairs=self.cta_pairs,
                            timeout_ns=self.timeout_ns, trace=trace_ptr,
                            trace_capacity=trace_capacity)
        if trace_ptr is None and trace_capacity == 0:
            self.__dict__["_c"] = c
        return c


def workspace_bytes(problem: Problem, n_pes: int) -> int:
    out = ctypes.c_int64()
    check(lib().megacu_b200_workspace_bytes(problem.to_c(), n_pes, ctypes.byref(out)))
    return out.value


def events_bytes(problem: Problem, n_pes: int) -> int:
    out = ctypes.c_int64()
    check(lib().megacu_b200_events_bytes(problem.to_c(), n_pes, ctypes.byref(out)))
    return out.value


@dataclass
class Plan:
    tile_m: int
    tile_n: int
    m_tiles: int
    n_tiles: int
    one_shot: bool
    slots_per_src: int
    group_m: int
    wire_bytes: int
    cta_pairs: bool = False  # 2-CTA clusters compute 256-row pair tiles
    gemm_units: int = 0      # GEMM tickets per call

    @property
    def tiles(self) -> int:
        return self.m_tiles * self.n_tiles


def plan(problem: Problem, n_pes: int) -> Plan:
    info = (ctypes.c_int32 * 10)()
    check(lib().megacu_b200_plan_info(problem.to_c(), n_pes, info))
    return Plan(info[0], info[1], info[2], info[3], bool(info[4]), info[5], info[6], info[7],
                bool(info[8]), info[9])


def plan_tile(problem: Problem, n_pes: int, r: int, pe: int = 0) -> tuple[int, int, int, int]:
    """(tile_row, tile_col, owner, local index) of raster index ``r`` on PE
    ``pe`` (the all-gather raster starts with the PE's own shard; the other
    modes' rasters are the same on every PE)."""
    out = (ctypes.c_int32 * 4)()
    check(lib().megacu_b200_plan_tile_on(problem.to_c(), n_pes, pe, r, out))
    return tuple(out)


def plan_pair(problem: Problem, n_pes: int, q: int) -> tuple[int, int]:
    """Raster indices of the two tiles a CTA pair computes for GEMM ticket ``q``."""
    out = (ctypes.c_int32 * 2)()
    check(lib().megacu_b200_plan_pair(problem.to_c(), n_pes, q, out))
    return tuple(out)


def gemm_allreduce(a, b, out, *, workspace, events, problem: Problem, stream=None,
                   device: int = 0, team: Optional[Team] = None, trace=None,
                   orchestrate: bool = True) -> None:
    """Launches the fused bf16 GEMM + allreduce / reduce-scatter (async).

    ``orchestrate=True`` goes through megacu's phase API (dispatcher +
    scheduler validation, then the launcher), as megacu's orchestrate entry
    does; ``False`` calls the launcher directly.
    """
    trace_ptr = _ptr(trace)
    cap = trace.numel() // 4 if trace is not None else 0
    d = _launch_view(stream, device, team)
    p = problem.to_c(trace_ptr, cap)
    args = (d, _ptr(a), _ptr(b), _ptr(workspace), _ptr(out), _ptr(events), p)
    if orchestrate:
        check(lib().megacu_cuda_gemm_allreduce_bf16_orchestrate(*args))
    elif problem.mode == _capi.MODE_REDUCE_SCATTER:
        check(lib().megacu_cuda_gemm_reduce_scatter_bf16(*args))
    else:
        check(lib().megacu_cuda_gemm_allreduce_bf16(*args))


def gemm_reduce_scatter(a, b, out, *, workspace, events, problem: Problem, **kw) -> None:
    problem.mode = _capi.MODE_REDUCE_SCATTER
    gemm_allreduce(a, b, out, workspace=workspace, events=events, problem=problem, **kw)


def allgather_gemm(a_shard, b, gathered, out, *, events, problem: Problem, stream=None,
                   device: int = 0, team: Optional[Team] = None, trace=None) -> None:
    """Launches the all-gather + GEMM (async): ``gathered`` [m, k] receives
    every PE's ``a_shard`` [m / tp, k] in PE order and ``out`` [m, n] =
    gathered @ b. ``a_shard`` and ``events`` lie in the team's heap when the
    team has more than one PE; ``problem.mode`` is set to MODE_ALLGATHER."""
    problem.mode = _capi.MODE_ALLGATHER
    trace_ptr = _ptr(trace)
    cap = trace.numel() // 4 if trace is not None else 0
    d = _launch_view(stream, device, team)
    check(lib().megacu_cuda_allgather_gemm_bf16(d, _ptr(a_shard), _ptr(b), _ptr(gathered),
                                                 _ptr(out), _ptr(events),
                                                 problem.to_c(trace_ptr, cap)))


# ---- tensor-parallel MLP blocks (benchmark config 5) ----------------------------------

def swiglu_events_bytes(problem: Problem) -> int:
    out = ctypes.c_int64()
    check(lib().megacu_b200_swiglu_events_bytes(problem.to_c(), ctypes.byref(out)))
    return out.value


def gemm_swiglu(x, w_gate, w_up, act, *, events, problem: Problem, stream=None,
                device: int = 0, trace=None) -> None:
    """act = silu(x @ w_gate) * (x @ w_up) (one PE, async). ``problem``: m =
    tokens, n = act columns, k = hidden."""
    trace_ptr = _ptr(trace)
    cap = trace.numel() // 4 if trace is not None else 0
    check(lib().megacu_cuda_gemm_swiglu_bf16(_launch_view(stream, device, None), _ptr(x),
                                             _ptr(w_gate), _ptr(w_up), _ptr(act), _ptr(events),
                                             problem.to_c(trace_ptr, cap)))


@dataclass
class MlpChainProblem:
    """megacu_mlp_chain_problem: ``layers`` blocks x -> allreduce(swiglu(x) @ w_down)."""
    tokens: int
    hidden: int
    inter: int          # this PE's slice of the intermediate size
    layers: int = 1
    algo: int = _capi.ALGO_AUTO
    deterministic: bool = False
    num_ctas: int = 0
    cta_pairs: int = _capi.CTA_PAIRS_AUTO
    timeout_ns: int = 0
    single_launch: bool = False  # all blocks (at most 6) in one persistent launch

    def to_c(self) -> "_capi.MlpChainProblem":
        return _capi.MlpChainProblem(tokens=self.tokens, hidden=self.hidden, inter=self.inter,
                                     layers=self.layers, algo=self.algo,
                                     deterministic=1 if self.deterministic else 0,
                                     num_ctas=self.num_ctas, cta_pairs=self.cta_pairs,
                                     single_launch=1 if self.single_launch else 0,
                                     timeout_ns=self.timeout_ns)


def mlp_chain_sizes(problem: MlpChainProblem, n_pes: int) -> dict:
    """Bytes of each buffer megacu_cuda_mlp_chain_bf16 needs on ``n_pes`` PEs."""
    out = (ctypes.c_int64 * 5)()
    check(lib().megacu_b200_mlp_chain_sizes(problem.to_c(), n_pes, out))
    return {"act": out[0], "workspace": out[1], "events_swiglu": out[2],
            "events_down": out[3], "x_work": out[4]}


def mlp_chain(x, w_gate, w_up, w_down, out, *, act, workspace, x_work, events_swiglu,
              events_down, problem: MlpChainProblem, stream=None, device: int = 0,
              team: Optional[Team] = None) -> None:
    """Runs ``problem.layers`` tensor-parallel MLP blocks (async); the last
    block's output lands in ``out``. ``w_gate``, ``w_up``, ``w_down``: one
    tensor per layer (this PE's slices)."""
    n = problem.layers
    if not (len(w_gate) == len(w_up) == len(w_down) == n):
        raise ValueError("one gate, up and down weight per layer")
    arr = lambda ws: (ctypes.c_void_p * n)(*[_ptr(w) for w in ws])
    check(lib().megacu_cuda_mlp_chain_bf16(_launch_view(stream, device, team), _ptr(x),
                                           arr(w_gate), arr(w_up), arr(w_down), _ptr(act),
                                           _ptr(workspace), _ptr(x_work), _ptr(out),
                                           _ptr(events_swiglu), _ptr(events_down),
                                           problem.to_c()))


# ---- routing of tokens to experts, 4-bit products ---------------------------------------

class _CProblem:
    """Base of the problem dataclasses passed by pointer: the C struct, the
    pointer to it and what follows from it are built once and reused until a
    field changes. Struct and pointer are one entry, so that threads that meet
    on a new problem see both or neither."""

    def __setattr__(self, name, value):
        object.__setattr__(self, name, value)
        self.__dict__.pop("_c", None)
        self.__dict__.pop("_sizes", None)
        self.__dict__.pop("_need", None)

    def __getstate__(self):
        """Copies and pickles hold the fields alone: structs and pointers to them
        belong to one object."""
        return {f.name: getattr(self, f.name) for f in fields(self)}

    def _built(self):
        built = self.__dict__.get("_c")
        if built is None:
            c = self._build()
            built = self.__dict__["_c"] = (c, ctypes.byref(c))
        return built

    def to_c(self):
        return self._built()[0]

    def _pointer(self):
        return self._built()[1]


class _Types(dict):
    """torch types by their element type code; "u8", "i32" and "i64" too.
    Filled on first use (importing this package does not import torch)."""

    def __missing__(self, key):
        import torch
        self.update({_capi.DTYPE_F16: torch.float16, _capi.DTYPE_BF16: torch.bfloat16,
                     _capi.DTYPE_F32: torch.float32, "u8": torch.uint8, "i32": torch.int32,
                     "i64": torch.int64})
        return self[key]


_TYPES = _Types()


def _buffer(x, name: str, elements: int, dtype, device: Optional[int]) -> Optional[int]:
    """The address of ``x``: a contiguous tensor on ``device`` (None: anywhere,
    for calls that only validate) of the type with code ``dtype`` and at least
    ``elements`` elements. None and raw addresses (int) are taken as they are."""
    if x is None or x.__class__ is int:
        return x
    if (x.dtype is _TYPES[dtype] and x.numel() >= elements and x.is_contiguous()
            and (device is None or x.get_device() == device)):
        return x.data_ptr()
    if x.dtype is not _TYPES[dtype]:
        raise ValueError(f"{name} has dtype {x.dtype}")
    if x.numel() < elements or not x.is_contiguous():
        raise ValueError(f"{name} must be contiguous with at least {elements} elements")
    raise ValueError(f"{name} is on {x.device}, the call on device {device}")


def _matrix(x, name: str, rows: int, cols: int, stride: int, dtype: int,
            device: Optional[int]) -> Optional[int]:
    """The address of the row-major matrix ``x``, whose rows are ``stride``
    elements apart (0: dense)."""
    if stride == 0 or stride == cols or x is None or x.__class__ is int:
        return _buffer(x, name, rows * cols, dtype, device)
    if x.dtype is not _TYPES[dtype]:
        raise ValueError(f"{name} has dtype {x.dtype}")
    if (x.dim() != 2 or x.shape[0] < rows or x.shape[1] < cols or x.stride(1) != 1
            or (rows > 1 and x.stride(0) != stride)):
        raise ValueError(f"{name} must be [{rows}, {cols}] with rows {stride} elements apart")
    if device is not None and x.get_device() != device:
        raise ValueError(f"{name} is on {x.device}, the call on device {device}")
    return x.data_ptr()


@dataclass
class MoeProblem(_CProblem):
    """megacu_moe_problem: ``tokens`` tokens with ``topk`` expert ids each, on a
    PE that holds experts [first_expert, first_expert + experts). Strides are
    in elements, 0 = hidden."""
    tokens: int
    topk: int
    experts: int
    hidden: int = 0
    first_expert: int = 0
    align: int = 1       # 128 for products by expert
    dtype: int = _capi.DTYPE_BF16
    token_stride: int = 0
    row_stride: int = 0
    id_bytes: int = 0    # of ids given as an address: 4 (or 0) or 8; a tensor has its type

    def _build(self, id_bytes: int = 0):
        return _capi.MoeProblem(tokens=self.tokens, hidden=self.hidden, topk=self.topk,
                                experts=self.experts, first_expert=self.first_expert,
                                align=self.align, dtype=self.dtype,
                                id_bytes=id_bytes or self.id_bytes,
                                token_stride=self.token_stride, row_stride=self.row_stride)

    def _wide_ids(self):
        """The pointer for 64-bit ids."""
        c = self.to_c()
        wide = self.__dict__.get("_wide")
        if wide is None or wide[0] is not c:
            wide = self.__dict__["_wide"] = (c, ctypes.byref(self._build(8)))
        return wide[1]


def _expert_ids(ids, slots: int, problem, device: Optional[int]):
    """The address of ``ids`` and the problem's pointer for their width: a
    tensor's type, or problem.id_bytes for an address."""
    wide = getattr(ids, "dtype", None) is _TYPES["i64"]
    if problem.id_bytes and ids is not None and ids.__class__ is not int and (
            wide != (problem.id_bytes == 8)):
        raise ValueError(f"expert_ids has dtype {ids.dtype}, id_bytes is {problem.id_bytes}")
    return (_buffer(ids, "expert_ids", slots, "i64" if wide else "i32", device),
            problem._wide_ids() if wide else problem._pointer())


def _moe_sizes(problem: MoeProblem) -> tuple[int, int]:
    sizes = problem.__dict__.get("_sizes")
    if sizes is None:
        out = (ctypes.c_int64 * 2)()
        check(lib().megacu_b200_moe_sizes(problem._pointer(), out))
        sizes = problem.__dict__["_sizes"] = (out[0], out[1])
    return sizes


def moe_rows(problem: MoeProblem) -> int:
    """Rows the sorted order can need: entries of ``slot_of_row``, rows of ``rows``."""
    return _moe_sizes(problem)[0]


def moe_workspace_bytes(problem: MoeProblem) -> int:
    return _moe_sizes(problem)[1]


def moe_sort(expert_ids, *, counts, offsets, row_of_slot, slot_of_row, problem: MoeProblem,
             workspace=None, stream=None, device: int = 0) -> None:
    """Sorts the (token, choice) slots by expert, stably (async).
    ``expert_ids`` [tokens, topk] int32 or int64 (an address: problem.id_bytes
    each); writes int32 ``counts``
    [experts], ``offsets`` [experts + 1], ``row_of_slot`` [tokens, topk] and
    ``slot_of_row`` [moe_rows(problem)]; -1 marks slots whose expert is
    elsewhere and rows without a slot. At most 2^26 slots. ``workspace``: moe_workspace_bytes()."""
    where = None if stream is None else device
    rows, need = _moe_sizes(problem)
    slots, experts = problem.tokens * problem.topk, problem.experts
    ids, pointer = _expert_ids(expert_ids, slots, problem, where)
    check(lib().megacu_cuda_moe_sort(
        _launch_view(stream, device, None), ids,
        _buffer(counts, "counts", experts, "i32", where),
        _buffer(offsets, "offsets", experts + 1, "i32", where),
        _buffer(row_of_slot, "row_of_slot", slots, "i32", where),
        _buffer(slot_of_row, "slot_of_row", rows, "i32", where),
        _buffer(workspace, "workspace", need, "u8", where) if need else None, pointer))


def _token_rows(x, name: str, p: MoeProblem, where: Optional[int]) -> Optional[int]:
    return _matrix(x, name, p.tokens, p.hidden, p.token_stride, p.dtype, where)


def _expert_rows(x, name: str, p: MoeProblem, where: Optional[int]) -> Optional[int]:
    return _matrix(x, name, moe_rows(p), p.hidden, p.row_stride, p.dtype, where)


def moe_dispatch(x, rows, *, row_of_slot, problem: MoeProblem, stream=None,
                 device: int = 0) -> None:
    """rows[row_of_slot[t, j]] = x[t] (async); other rows are left as they
    were. The gradient is :func:`moe_combine` of the rows' gradient without
    weights."""
    p, where = problem, None if stream is None else device
    check(lib().megacu_cuda_moe_dispatch(
        _launch_view(stream, device, None), _token_rows(x, "x", p, where),
        _buffer(row_of_slot, "row_of_slot", p.tokens * p.topk, "i32", where),
        _expert_rows(rows, "rows", p, where), p._pointer()))


def moe_combine(rows, y, *, row_of_slot, problem: MoeProblem, weights=None, stream=None,
                device: int = 0) -> None:
    """y[t] = sum over j of weights[t, j] * rows[row_of_slot[t, j]] (async), fp32
    sums in the order of j, one rounding; ``weights`` fp32, None = 1."""
    p, slots = problem, problem.tokens * problem.topk
    where = None if stream is None else device
    check(lib().megacu_cuda_moe_combine(
        _launch_view(stream, device, None), _expert_rows(rows, "rows", p, where),
        _buffer(weights, "weights", slots, _capi.DTYPE_F32, where),
        _buffer(row_of_slot, "row_of_slot", slots, "i32", where), _token_rows(y, "y", p, where),
        p._pointer()))


def moe_combine_grad(dy, rows, drows, dweights, *, weights, row_of_slot, problem: MoeProblem,
                     stream=None, device: int = 0) -> None:
    """Gradient of the weighted :func:`moe_combine` (async): drows = weights *
    dy at the rows of each token (other rows are left as they were), dweights
    [tokens, topk] fp32 = <dy[t], rows[...]>, 0 for a slot without a row."""
    p, slots = problem, problem.tokens * problem.topk
    where = None if stream is None else device
    check(lib().megacu_cuda_moe_combine_grad(
        _launch_view(stream, device, None), _token_rows(dy, "dy", p, where),
        _expert_rows(rows, "rows", p, where),
        _buffer(weights, "weights", slots, _capi.DTYPE_F32, where),
        _buffer(row_of_slot, "row_of_slot", slots, "i32", where),
        _expert_rows(drows, "drows", p, where),
        _buffer(dweights, "dweights", slots, _capi.DTYPE_F32, where),
        p._pointer()))


@dataclass
class Fp4Matrix(_CProblem):
    """megacu_fp4_matrix: a quantised matrix [rows, cols] of FP4_MX or FP4_NV
    blocks along its rows, and the plain matrix of ``dtype`` it comes from
    (stored [cols, rows] with ``transpose``). ``scale``: a power of two that
    multiplies the values before they are quantised."""
    rows: int
    cols: int
    format: int = _capi.FP4_MX
    dtype: int = _capi.DTYPE_BF16
    transpose: bool = False
    scale: float = 1.0
    stride: int = 0

    def _build(self, topk: int = 0, x_rows: int = 0, scatter: int = 0):
        return _capi.Fp4Matrix(rows=self.rows, cols=self.cols, stride=self.stride, x_rows=x_rows,
                               format=self.format, dtype=self.dtype,
                               transpose=1 if self.transpose else 0, topk=topk,
                               scale=self.scale, scatter=scatter)


def fp4_sizes(problem: Fp4Matrix) -> tuple[int, int]:
    """Bytes of the data and of the scales of a quantised matrix."""
    sizes = problem.__dict__.get("_sizes")
    if sizes is None:
        out = (ctypes.c_int64 * 2)()
        check(lib().megacu_b200_fp4_sizes(problem._pointer(), out))
        sizes = problem.__dict__["_sizes"] = (out[0], out[1])
    return sizes


def fp4_quantize(x, data, scales, *, problem: Fp4Matrix, slot_of_row=None, row_of_slot=None,
                 topk: int = 0, x_rows: int = 0, stream=None, device: int = 0) -> None:
    """Quantises ``x`` into ``data`` and ``scales`` (async). With
    ``slot_of_row`` (of :func:`moe_sort`, int32 [rows]) rows whose entry is
    negative are left as they were; with ``topk`` too, row r is taken from
    x[slot_of_row[r] // topk]. With ``row_of_slot`` ([x rows, topk]) and its
    ``topk`` instead, each row of ``x`` is quantised once and written to the
    rows of its choices: the same bytes, sooner when topk > 1. ``x_rows``: the
    rows of ``x``, needed only when ``x`` is a raw address and topk > 0."""
    if slot_of_row is not None and row_of_slot is not None:
        raise ValueError("slot_of_row or row_of_slot, not both")
    if row_of_slot is not None and (topk < 1 or (getattr(row_of_slot, "ndim", 1) == 2
                                                 and row_of_slot.shape[1] != topk)):
        raise ValueError(f"row_of_slot holds topk entries per row of x, topk is {topk}")
    p, where = problem, None if stream is None else device
    nbytes, sbytes = fp4_sizes(p)
    if topk:
        if x_rows == 0 and x is not None and x.__class__ is not int:
            dense = p.stride == 0 or p.stride == p.cols
            x_rows = x.numel() // p.cols if dense else x.shape[0]
        x_ptr = _matrix(x, "x", x_rows, p.cols, p.stride, p.dtype, where)
        key = (topk, x_rows, 0 if row_of_slot is None else 1)
        gathered = p.__dict__.get("_gathered")
        if gathered is None or gathered[0] is not p.to_c() or gathered[1] != key:
            gathered = p.__dict__["_gathered"] = (p.to_c(), key, ctypes.byref(p._build(*key)))
        pointer = gathered[2]
    else:
        rows, cols = (p.cols, p.rows) if p.transpose else (p.rows, p.cols)
        x_ptr = _matrix(x, "x", rows, cols, p.stride, p.dtype, where)
        pointer = p._pointer()
    check(lib().megacu_cuda_fp4_quantize(
        _launch_view(stream, device, None), x_ptr,
        _buffer(slot_of_row, "slot_of_row", p.rows, "i32", where) if row_of_slot is None else
        _buffer(row_of_slot, "row_of_slot", x_rows * topk, "i32", where),
        _buffer(data, "data", nbytes, "u8", where),
        _buffer(scales, "scales", sbytes, "u8", where), pointer))


def fp4_dequantize(data, scales, out, *, problem: Fp4Matrix, stream=None,
                   device: int = 0) -> None:
    """The values of a quantised matrix (async): out [rows, cols] = element *
    scale / problem.scale, rounded once to problem.dtype."""
    p, where = problem, None if stream is None else device
    nbytes, sbytes = fp4_sizes(p)
    check(lib().megacu_cuda_fp4_dequantize(
        _launch_view(stream, device, None), _buffer(data, "data", nbytes, "u8", where),
        _buffer(scales, "scales", sbytes, "u8", where),
        _matrix(out, "out", p.rows, p.cols, p.stride, p.dtype, where), p._pointer()))


@dataclass
class Fp4Gemm(_CProblem):
    """megacu_fp4_gemm_problem: out [m, n] = alpha * A [m, k] @ B [n, k]^T of
    quantised matrices; ``experts`` > 0: B is [experts, n, k] and A's rows are
    sorted by expert."""
    m: int
    n: int
    k: int
    format: int = _capi.FP4_MX
    out_dtype: int = _capi.DTYPE_BF16
    experts: int = 0
    alpha: float = 1.0
    out_stride: int = 0
    tile_n: int = 0
    split: int = 0
    timeout_ns: int = 0

    def _build(self):
        return _capi.Fp4GemmProblem(m=self.m, n=self.n, k=self.k, out_stride=self.out_stride,
                                    format=self.format, out_dtype=self.out_dtype,
                                    experts=self.experts, tile_n=self.tile_n, split=self.split,
                                    alpha=self.alpha, timeout_ns=self.timeout_ns)


def fp4_events_bytes() -> int:
    """Bytes of the products' ``events`` (zero-filled once, then reused)."""
    out = ctypes.c_int64()
    check(lib().megacu_b200_fp4_events_bytes(ctypes.byref(out)))
    return out.value


def _operand_bytes(matrices: int, rows: int, k: int, fmt: int) -> tuple[int, int]:
    """Bytes of the data and scales of ``matrices`` quantised matrices [rows, k]."""
    tiles = -(-k // (128 if fmt == _capi.FP4_MX else 64))
    return matrices * rows * (k // 2), matrices * -(-rows // 128) * tiles * 512


def _product_needs(p: Fp4Gemm) -> tuple[int, int, int, int]:
    """Bytes of A, of its scales, of one B operand and of its scales."""
    need = p.__dict__.get("_need")
    if need is None:
        need = p.__dict__["_need"] = (*_operand_bytes(1, p.m, p.k, p.format),
                                      *_operand_bytes(max(p.experts, 1), p.n, p.k, p.format))
    return need


def fp4_gemm(a, a_scales, b, b_scales, out, *, events, problem: Fp4Gemm, offsets=None,
             counts=None, alphas=None, stream=None, device: int = 0) -> None:
    """out = alpha * A @ B^T of two quantised matrices (async), fp32
    accumulation and one rounding. By expert: ``offsets`` and ``counts`` of
    :func:`moe_sort` (align 128), ``alphas`` fp32 [experts] factors; rows
    without a slot are left as they were."""
    p, where = problem, None if stream is None else device
    need = _product_needs(p)
    check(lib().megacu_cuda_fp4_gemm(
        _launch_view(stream, device, None), _buffer(a, "a", need[0], "u8", where),
        _buffer(a_scales, "a_scales", need[1], "u8", where),
        _buffer(b, "b", need[2], "u8", where),
        _buffer(b_scales, "b_scales", need[3], "u8", where),
        _buffer(offsets, "offsets", p.experts + 1, "i32", where),
        _buffer(counts, "counts", p.experts, "i32", where),
        _buffer(alphas, "alphas", p.experts, _capi.DTYPE_F32, where),
        _matrix(out, "out", p.m, p.n, p.out_stride, p.out_dtype, where),
        _buffer(events, "events", 256, "u8", where), p._pointer()))


def fp4_gemm_swiglu(a, a_scales, gate, gate_scales, up, up_scales, act, *, events,
                    problem: Fp4Gemm, offsets=None, counts=None, alphas=None, stream=None,
                    device: int = 0) -> None:
    """act = silu(alpha * A @ gate^T) * (alpha * A @ up^T) of quantised
    matrices (async); ``problem.n`` = act columns. By expert as
    :func:`fp4_gemm`."""
    p, where = problem, None if stream is None else device
    need = _product_needs(p)
    check(lib().megacu_cuda_fp4_gemm_swiglu(
        _launch_view(stream, device, None), _buffer(a, "a", need[0], "u8", where),
        _buffer(a_scales, "a_scales", need[1], "u8", where),
        _buffer(gate, "gate", need[2], "u8", where),
        _buffer(gate_scales, "gate_scales", need[3], "u8", where),
        _buffer(up, "up", need[2], "u8", where),
        _buffer(up_scales, "up_scales", need[3], "u8", where),
        _buffer(offsets, "offsets", p.experts + 1, "i32", where),
        _buffer(counts, "counts", p.experts, "i32", where),
        _buffer(alphas, "alphas", p.experts, _capi.DTYPE_F32, where),
        _matrix(act, "act", p.m, p.n, p.out_stride, p.out_dtype, where),
        _buffer(events, "events", 256, "u8", where), p._pointer()))


@dataclass
class MoeMlp(_CProblem):
    """megacu_moe_mlp_problem: a routed MLP block with 4-bit weights (see
    :func:`moe_mlp_fp4`)."""
    tokens: int
    hidden: int
    inter: int          # this PE's slice of the intermediate size
    topk: int
    experts: int
    first_expert: int = 0
    dtype: int = _capi.DTYPE_BF16
    format: int = _capi.FP4_MX
    x_scale: float = 1.0
    act_scale: float = 1.0
    up_alpha: float = 1.0
    down_alpha: float = 1.0
    timeout_ns: int = 0
    id_bytes: int = 0   # as MoeProblem's

    def _build(self, id_bytes: int = 0):
        return _capi.MoeMlpProblem(
            tokens=self.tokens, hidden=self.hidden, inter=self.inter, topk=self.topk,
            experts=self.experts, first_expert=self.first_expert, dtype=self.dtype,
            id_bytes=id_bytes or self.id_bytes, format=self.format, x_scale=self.x_scale,
            act_scale=self.act_scale, up_alpha=self.up_alpha, down_alpha=self.down_alpha,
            timeout_ns=self.timeout_ns)

    _wide_ids = MoeProblem._wide_ids


def moe_mlp_workspace_bytes(problem: MoeMlp) -> int:
    sizes = problem.__dict__.get("_sizes")
    if sizes is None:
        out = ctypes.c_int64()
        check(lib().megacu_b200_moe_mlp_workspace_bytes(problem._pointer(), ctypes.byref(out)))
        sizes = problem.__dict__["_sizes"] = (out.value,)
    return sizes[0]


def moe_mlp_fp4(x, expert_ids, weights, gate, gate_scales, up, up_scales, down, down_scales, y, *,
                workspace, events, problem: MoeMlp, up_alphas=None, down_alphas=None, stream=None,
                device: int = 0) -> None:
    """A routed MLP block (async): y[t] = sum over the choices j of token t whose
    expert e is here of weights[t, j] * down_e(silu(gate_e(x[t])) * up_e(x[t])),
    on weights quantised by :func:`fp4_quantize`: ``gate``, ``up`` [experts,
    inter, hidden], ``down`` [experts, hidden, inter]. The calls of this module
    in a row on one ``workspace`` (moe_mlp_workspace_bytes(), uint8, 256-byte
    aligned); with experts or inter spread over PEs, y is this PE's part of
    the sum."""
    p, where = problem, None if stream is None else device
    slots = p.tokens * p.topk
    ids, pointer = _expert_ids(expert_ids, slots, p, where)
    need = moe_mlp_workspace_bytes(p)
    up_need = _operand_bytes(p.experts, p.inter, p.hidden, p.format)
    down_need = _operand_bytes(p.experts, p.hidden, p.inter, p.format)
    check(lib().megacu_cuda_moe_mlp_fp4(
        _launch_view(stream, device, None),
        _matrix(x, "x", p.tokens, p.hidden, 0, p.dtype, where), ids,
        _buffer(weights, "weights", slots, _capi.DTYPE_F32, where),
        _buffer(gate, "gate", up_need[0], "u8", where),
        _buffer(gate_scales, "gate_scales", up_need[1], "u8", where),
        _buffer(up, "up", up_need[0], "u8", where),
        _buffer(up_scales, "up_scales", up_need[1], "u8", where),
        _buffer(down, "down", down_need[0], "u8", where),
        _buffer(down_scales, "down_scales", down_need[1], "u8", where),
        _buffer(up_alphas, "up_alphas", p.experts, _capi.DTYPE_F32, where),
        _buffer(down_alphas, "down_alphas", p.experts, _capi.DTYPE_F32, where),
        _matrix(y, "y", p.tokens, p.hidden, 0, p.dtype, where),
        _buffer(workspace, "workspace", need, "u8", where),
        _buffer(events, "events", 256, "u8", where), pointer))


def events_status(events, stream=None) -> list[int]:
    """Synchronises ``stream`` and raises MegacuError if a device wait failed."""
    info = (ctypes.c_int64 * 4)()
    check(lib().megacu_b200_events_status(_ptr(events), _stream_handle(stream), info))
    return list(info)


def events_counters(events, stream=None) -> list[int]:
    out = (ctypes.c_uint64 * 8)()
    check(lib().megacu_b200_events_counters(_ptr(events), _stream_handle(stream), out))
    return list(out)


# ---- megacu's fp32 phased entry points -------------------------------------------------

def megacu_cuda_gemm_allreduce_phased_f32(driver: DriverView, a, b, partial, out, events,
                                          m: int, n: int, k: int, tile_m: int,
                                          tile_n: int) -> Status:
    return lib().megacu_cuda_gemm_allreduce_phased_f32(
        driver, _ptr(a), _ptr(b), _ptr(partial), _ptr(out), _ptr(events),
        GemmArProblem(m=m, n=n, k=k, tile_m=tile_m, tile_n=tile_n))


def cuda_nvshmem_gemm_allreduce_phased_orchestrate(driver: DriverView, a, b, partial, out,
                                                   events, m: int, n: int, k: int,
                                                   tile_m: int, tile_n: int) -> Status:
    return lib().megacu_cuda_gemm_allreduce_f32_orchestrate(
        driver, _ptr(a), _ptr(b), _ptr(partial), _ptr(out), _ptr(events),
        GemmArProblem(m=m, n=n, k=k, tile_m=tile_m, tile_n=tile_n))


def co_resident_control_bytes() -> int:
    out = ctypes.c_int64()
    check(lib().megacu_b200_co_resident_control_bytes(ctypes.byref(out)))
    return out.value


def megacu_cuda_gemm_allreduce_f32_co_resident(driver: DriverView, a, b, partial, out, events,
                                               control, m: int, n: int, k: int, tile_m: int,
                                               tile_n: int) -> Status:
    """megacu's fp32 phase with co-resident persistent progress (one
    cooperative persistent launch; ``control`` holds
    :func:`co_resident_control_bytes` bytes of device memory)."""
    return lib().megacu_cuda_gemm_allreduce_f32_co_resident(
        driver, _ptr(a), _ptr(b), _ptr(partial), _ptr(out), _ptr(events), _ptr(control),
        GemmArProblem(m=m, n=n, k=k, tile_m=tile_m, tile_n=tile_n))


def co_resident_status(control, stream=None) -> list[int]:
    """Synchronises ``stream``; raises MegacuError (detail 40) if a wait of the
    last co-resident launch gave up; returns [node, tile] of that wait."""
    info = (ctypes.c_int64 * 2)()
    check(lib().megacu_b200_co_resident_status(_ptr(control), _stream_handle(stream), info))
    return list(info)
