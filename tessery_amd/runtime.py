"""HipRuntime: tessery's native-bridge runtime over libtessery_hip.so (HIP, gfx950).

The class is a drop-in for tessery's MetalRuntime (src/metal_inference/metal.py:169-801) on the
prefill-attention path and the layers around it. Callers see the same names, signatures, error
classes and route selection:
  * buffers: buffer / upload / read / write, Buffer.close;
  * commands: `with rt.command():` queues launches, leaving the block runs them and waits;
  * `_dispatch(name, buffers, *, threads, group_size, ...)` packs the 64-byte Params block;
  * the route selectors `_attention`, `_linear4`, `_gated4`, `_matmul_f32`, `_matmul_bias_f32`;
  * `_workspace`, `_execution_plan`, `profile_kernels`, `diagnostics`, `add`, `matmul`, `close`.
It is exported as `MetalRuntime` too, so code written against tessery's bridge runs unchanged.

Additions, all keyword-only with defaults that keep the reference behaviour:
  * `_attention(..., precision="f16", out_dtype=...)`: fp16 operands, fp32 accumulation on MFMA;
  * `_attention_norm_rope(...)`: the Qwen3 q/k RMSNorm + RoPE fused into the fp16 attention;
  * `_qkv4(...)`: the three uint4 QKV projections of fp16 activations in one launch;
  * `_attention_masked(...)`, `_rotary(...)`, `_rotary_table(...)`, `_linear_f16(...)`: attention with
    capped or biased scores and prefix, window and document masks, rotary positions of other layouts
    and lengths, and fp16 projections with their epilogue, for encoders other than the two here;
  * `read(..., dtype=...)` for fp16 buffers, `write` and `upload`.

Structure of the host side:
  * launch planners (pure functions): each route selector turns its shape into a list of Launch
    records - the reference's route names, thread formulas and row partitions - and the runtime
    dispatches them in order;
  * _DeviceMemory: the allocation ledger (live buffers, bytes in use, high-water mark);
  * _Retained: device memory kept between forwards under one byte budget - scratch buffers of
    finished workspaces, reused by exact size, and prepared plans, least recently used first out;
  * _Command: one open command - its launch records for profiling and its timing.
The library queues launches at dispatch and runs them at finish; a buffer released while a
command is open keeps its device memory until that command ends.

The product path has no CPU fallback: without the library or a gfx950 device construction fails
with NativeBuildError / HipUnavailableError.
"""

from __future__ import annotations

import ctypes as ct
import hashlib
import math
import struct
import threading
import time
from collections import Counter, OrderedDict
from collections.abc import Iterator, Sequence
from contextlib import contextmanager
from pathlib import Path
from typing import Any, NamedTuple
from weakref import WeakSet

import numpy as np
from numpy.typing import NDArray

from .errors import ClosedError, HipUnavailableError, InferenceError, NativeBuildError

ABI_VERSION = 2
LIBRARY_NAME = "libtessery_hip.so"

# ctypes signatures of the C ABI (include/tessery_hip.h). The mi_* entries tessery binds are the
# table of metal.py:42-83; mi_abi_version, mi_write, mi_graph_counts, mi_fusion_counts,
# mi_profile_fused and mi_attention_norm_rope_noalloc are this library's additions.
SIGNATURES: dict[str, tuple[list[Any], Any]] = {
    "mi_abi_version": ([], ct.c_int),
    "mi_create": ([ct.c_char_p], ct.c_void_p),
    "mi_destroy": ([ct.c_void_p], None),
    "mi_buffer": ([ct.c_void_p, ct.c_void_p, ct.c_uint64], ct.c_void_p),
    "mi_free": ([ct.c_void_p], None),
    "mi_read": ([ct.c_void_p, ct.c_void_p, ct.c_uint64], ct.c_int),
    "mi_write": ([ct.c_void_p, ct.c_void_p, ct.c_uint64], ct.c_int),
    "mi_begin": ([ct.c_void_p], ct.c_int),
    "mi_finish": ([ct.c_void_p], ct.c_int),
    "mi_gpu_seconds": ([ct.c_void_p], ct.c_double),
    "mi_abort": ([ct.c_void_p], None),
    "mi_profile_enable": ([ct.c_void_p, ct.c_int], ct.c_int),
    "mi_profile_read": ([ct.c_void_p, ct.POINTER(ct.c_double), ct.c_uint32], ct.c_int),
    "mi_profile_fused": ([ct.c_void_p, ct.POINTER(ct.c_uint8), ct.c_uint32], ct.c_int),
    "mi_plan_create": ([ct.c_void_p, ct.POINTER(ct.c_void_p), ct.c_uint32], ct.c_void_p),
    "mi_plan_add": (
        [
            ct.c_void_p,
            ct.c_char_p,
            ct.POINTER(ct.c_uint32),
            ct.c_uint32,
            ct.c_void_p,
            ct.c_uint64,
            ct.c_uint32,
        ],
        ct.c_int,
    ),
    "mi_plan_bytes": ([ct.c_void_p], ct.c_uint64),
    "mi_plan_free": ([ct.c_void_p], None),
    "mi_plan_run": ([ct.c_void_p, ct.c_void_p, ct.POINTER(ct.c_void_p), ct.c_uint32], ct.c_int),
    "mi_graph_counts": ([ct.c_void_p, ct.POINTER(ct.c_uint64), ct.POINTER(ct.c_uint64)], ct.c_int),
    "mi_fusion_counts": ([ct.c_void_p, ct.POINTER(ct.c_uint64), ct.POINTER(ct.c_uint64)], ct.c_int),
    "mi_dispatch": (
        [
            ct.c_void_p,
            ct.c_char_p,
            ct.POINTER(ct.c_void_p),
            ct.c_uint32,
            ct.c_void_p,
            ct.c_uint32,
            ct.c_uint64,
            ct.c_uint32,
        ],
        ct.c_int,
    ),
    "mi_attention_norm_rope_noalloc": (
        [ct.c_void_p] * 7 + [ct.c_uint32] * 5 + [ct.c_float, ct.c_float, ct.c_int, ct.c_int,
                                                 ct.c_void_p],
        ct.c_int,
    ),
}

# Params layout, kernels.metal:5-8 / metal.py:596-614.
PARAMS_FORMAT = "<12I4f"

# Head dimensions served by the pipelined MFMA kernel of the fp16 path (plain and fused q/k
# norm + RoPE); other head dimensions take the scalar fp16 route.
F16_TILE_DIMS = (64, 128)
F16_NORM_ROPE_DIMS = (64, 128)

# Prepared plans kept per runtime (metal.py keeps four as well).
MAX_PLANS = 4


def library_path() -> Path:
    return Path(__file__).resolve().parent / LIBRARY_NAME


def _library(path: Path | None = None) -> Any:
    """Open the native library and bind the C ABI. NativeBuildError when the file is missing,
    changes while it is loaded, lacks a symbol or reports another ABI version."""
    path = library_path() if path is None else path
    if not path.is_file():
        raise NativeBuildError()
    try:
        image = path.read_bytes()
        lib: Any = ct.CDLL(str(path))
        unchanged = path.read_bytes() == image
    except OSError:
        raise NativeBuildError() from None
    if not unchanged:
        raise NativeBuildError()
    lib._tessery_sha256 = hashlib.sha256(image).hexdigest()
    for name, (argtypes, restype) in SIGNATURES.items():
        function = getattr(lib, name, None)
        if function is None:
            raise NativeBuildError()
        function.argtypes, function.restype = argtypes, restype
    if lib.mi_abi_version() != ABI_VERSION:
        raise NativeBuildError()
    return lib


def pack_params(
    *,
    n: int = 0,
    rows: int = 0,
    cols: int = 0,
    k: int = 0,
    heads: int = 0,
    kv_heads: int = 0,
    seq: int = 0,
    batch: int = 0,
    dim: int = 0,
    group: int = 64,
    u0: int = 0,
    u1: int = 0,
    eps: float = 1e-6,
    theta: float = 1e6,
    scale: float = 1.0,
) -> bytes:
    """The 64-byte Params block (kernels.metal:5-8): twelve u32 fields, then eps, theta, scale and
    a reserved float."""
    words = (n, rows, cols, k, heads, kv_heads, seq, batch, dim, group, u0, u1)
    return struct.pack(PARAMS_FORMAT, *words, eps, theta, scale, 0.0)


# ---- launch planning: the reference's route tables as data ----------------------------------


class Launch(NamedTuple):
    """One kernel launch of a route: the kernel name, the reference's thread count and group size,
    the Params fields it sets, and which of the caller's buffers it binds (None: all, in order)."""

    name: str
    threads: int
    group_size: int
    fields: dict[str, Any]
    slots: tuple[int, ...] | None = None


# (cols, k) of the Qwen3-0.6B projections that the reference sends to its large uint4 tiles
# (metal.py:417-423).
QWEN_PROJECTIONS = frozenset({(1024, 1024), (2048, 1024), (3072, 1024), (1024, 2048), (1024, 3072)})
# (cols, k) of the BGE-small projections with a chunked dense route (metal.py:665, 704).
BGE_PROJECTIONS = frozenset({(384, 384), (1536, 384), (384, 1536)})


def attention_plan(*, tokens: int, seq: int, heads: int, kv_heads: int, dim: int,
                   bidirectional: int = 0, precision: str = "f32",
                   out_dtype: str | None = None) -> list[Launch]:
    """metal.py:532-569 for fp32: the bounded tail route for 64 <= seq <= 512 unaligned to 32
    (dim 32 / 128), the tiled route for aligned seq >= 64, the scalar route otherwise. fp16
    operands (this library's addition) take attention_f16, or its scalar form for head dims the
    MFMA kernel does not tile; out_dtype picks fp32 (default) or fp16 output there."""
    attn = dict(seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, scale=dim**-0.5,
                bidirectional=bidirectional)
    if precision == "f16":
        out_f16 = {None: 0, "f32": 0, "f16": 1}.get(out_dtype)
        if out_f16 is None:
            raise InferenceError()
        if dim in F16_TILE_DIMS:
            return [Launch("attention_f16", tokens, 256, {**attn, "out_f16": out_f16})]
        return [Launch("attention_f16_scalar", tokens, 64, {**attn, "out_f16": out_f16})]
    if precision != "f32" or out_dtype not in (None, "f32"):
        raise InferenceError()
    if dim in (32, 128) and 64 <= seq <= 512 and seq % 32:
        blocks = (tokens // seq) * ((seq + 7) // 8)
        return [Launch(f"attention_tail_{dim}", blocks * heads * 128, 128, attn)]
    if dim in (32, 128) and seq >= 64 and seq % 32 == 0:
        return [Launch("attention_tiled", tokens // 8 * heads * 128, 128, attn)]
    return [Launch("attention", tokens * heads * 32, 32, attn)]


def attention_norm_rope_plan(*, tokens: int, seq: int, heads: int, kv_heads: int, dim: int,
                             eps: float, theta: float, bidirectional: int,
                             out_dtype: str) -> list[Launch]:
    """The k prologue (norm_rope_f16 into hi/lo planes in k_work) then the fused attention, over
    buffers [q_pre, k_pre, v, lengths, out, q_norm, k_norm, k_work]."""
    out_f16 = {"f32": 0, "f16": 1}.get(out_dtype)
    if out_f16 is None or dim not in F16_NORM_ROPE_DIMS:
        raise InferenceError()
    return [
        Launch("norm_rope_f16", tokens, 256,
               dict(heads=kv_heads, seq=seq, dim=dim, eps=eps, theta=theta, flags=1),
               slots=(1, 6, 3, 7)),
        Launch("attention_f16_norm_rope", tokens, 256,
               dict(seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, scale=dim**-0.5, eps=eps,
                    theta=theta, bidirectional=bidirectional, out_f16=out_f16),
               slots=(0, 7, 2, 3, 4, 5)),
    ]


# Head dimensions of attention_masked: multiples of 8 up to this.
MASKED_MAX_DIM = 256
# The least cap of its scores: 2 * log2(e) / cap is a factor of the kernel's, in fp32.
MASKED_MIN_CAP = 1e-30
MASKS = {"causal": 0, "bidirectional": 1, "prefix": 2}
ACTIVATIONS = {"none": 0, "relu": 1, "gelu": 2, "gelu_tanh": 3, "silu": 4}
ROTARY_LAYOUTS = {"half": 0, "interleaved": 1}
_F16_FLAG = {"f32": 0, "f16": 1}


def _sized(*values: Any) -> bool:
    """Whether every value is a positive int."""
    return all(type(v) is int and v > 0 for v in values)


def attention_masked_plan(*, tokens: int, seq: int, heads: int, kv_heads: int, dim: int,
                          mask: str = "causal", window: int = 0, cap: float = 0.0,
                          radius: int = 0, scale: float | None = None, precision: str = "f16",
                          packed: bool | str = False, spans: bool = False, slopes: bool = False,
                          table: bool = False, prefix: bool = False) -> list[Launch]:
    """The one launch of _attention_masked over buffers [q, k, v, lengths, out, spans, bias,
    prefix]; spans, slopes, table and prefix say which of the last three are there, and lengths
    stands in for the others. Params: u0 the mask, u1 the flags, n the window, rows the table's
    radius, theta the cap."""
    if not _sized(tokens, seq, heads, kv_heads, dim) or tokens % seq or heads % kv_heads or \
            dim % 8 or dim > MASKED_MAX_DIM:
        raise InferenceError()
    if mask not in MASKS or precision not in _F16_FLAG or packed not in (False, True, "v") or \
            (mask == "prefix") != prefix or (slopes and table):
        raise InferenceError()
    if type(window) is not int or not 0 <= window < 2**32 or type(radius) is not int or \
            not 0 <= radius <= 2**20 or (radius and not table):
        raise InferenceError()
    scale = dim**-0.5 if scale is None else float(scale)
    cap = float(cap)
    if not math.isfinite(scale) or not (cap == 0.0 or MASKED_MIN_CAP <= cap < 3.4e38):
        raise InferenceError()
    flags = (_F16_FLAG[precision] | 2 * spans | 4 * slopes | 8 * table | 16 * (packed is True)
             | 32 * (packed is not False))
    here = [spans, slopes or table, prefix]
    slots = (0, 1, 2, 3, 4) + tuple(5 + i if there else 3 for i, there in enumerate(here))
    return [Launch("attention_masked", tokens, 256,
                   dict(seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, scale=scale, theta=cap,
                        n=window, rows=radius, bidirectional=MASKS[mask], flags=flags), slots)]


def rotary_plan(*, tokens: int, seq: int, heads: int, kv_heads: int, dim: int, rotary_dim: int,
                layout: str = "half", precision: str = "f16", eps: float = 1e-6,
                packed: bool = False, packed_out: bool = False, positions: bool = False,
                norm: bool = False) -> list[Launch]:
    """The one launch of _rotary over buffers [q, k, table, q_out, k_out, positions, q_norm,
    k_norm]; positions and norm say which of the last three are there, and the table stands in for
    the others (and for k and k_out where there are no key heads)."""
    if not _sized(tokens, seq, heads, dim, rotary_dim) or tokens % seq or \
            type(kv_heads) is not int or kv_heads < 0 or rotary_dim % 2 or rotary_dim > dim or \
            dim > 1024:
        raise InferenceError()
    if layout not in ROTARY_LAYOUTS or precision not in _F16_FLAG or not 0.0 <= eps < 3.4e38 or \
            ((packed or packed_out) and not kv_heads):
        raise InferenceError()
    flags = (_F16_FLAG[precision] | 2 * positions | 4 * norm | 8 * bool(packed)
             | 16 * bool(packed_out))
    k, k_out = (1, 4) if kv_heads else (2, 2)
    slots = (0, k, 5 if positions else 2, 2, 6 if norm else 2, 7 if norm and kv_heads else 2, 3,
             k_out)
    return [Launch("rotary", tokens, 256,
                   dict(seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, k=rotary_dim, eps=eps,
                        bidirectional=ROTARY_LAYOUTS[layout], flags=flags), slots)]


def linear_f16_plan(*, rows: int, cols: int, k: int, activation: str = "none",
                    out_dtype: str = "f16", bias: bool = False,
                    residual: bool = False) -> list[Launch]:
    """The one launch of _linear_f16 over buffers [x, w, out, bias, residual]; bias and residual
    say which of the last two are there, and x stands in for the others."""
    if not _sized(rows, cols, k) or activation not in ACTIVATIONS or out_dtype not in _F16_FLAG:
        raise InferenceError()
    flags = bias | 2 * residual | 4 * (out_dtype == "f32")
    return [Launch("linear_f16", rows, 256,
                   dict(rows=rows, cols=cols, k=k, bidirectional=ACTIVATIONS[activation],
                        flags=flags), (0, 1, 3 if bias else 0, 4 if residual else 0, 2))]


def linear4_plan(*, rows: int, cols: int, k: int) -> list[Launch]:
    """metal.py:416-499. Qwen3 projection shapes: 32-row tiles for the measured full-model heights,
    the three-row kernel for three rows, else complete 16-row tiles; the rows left over go to
    complete 8-row tiles and at most one partial tile (scalar for up to four rows). Shapes the
    tiled kernels cannot take run the scalar route over every row. Regions never overlap."""
    shape = dict(rows=rows, cols=cols, k=k)
    tiles = cols // 32
    qwen = (cols, k) in QWEN_PROJECTIONS
    if qwen and rows in (128, 160, 256, 512):
        return [Launch("linear4_32x32_k64", rows // 32 * tiles * 256, 256, shape)]
    if qwen and rows == 3:
        return [Launch("linear4_small3", cols * 32, 32, shape)]
    plan: list[Launch] = []
    done = 0
    if qwen and rows >= 16:
        plan.append(Launch("linear4_16x32_k64", rows // 16 * tiles * 256, 256, shape))
        done = rows // 16 * 16
        if done == rows:
            return plan
    if rows < 5 or cols % 32 or k % 64:
        return plan + [Launch("linear4", (rows + 3) // 4 * cols * 32, 32, shape)]
    complete = (rows - done) // 8
    if complete:
        plan.append(Launch("linear4_tiled", complete * tiles * 128, 128, {**shape, "n": done}))
    left = rows % 8
    if left:
        start = done + complete * 8
        if left <= 4:
            plan.append(Launch("linear4", cols * 32, 32, {**shape, "n": start}))
        else:
            plan.append(Launch("linear4_tail", tiles * 128, 128, {**shape, "n": start}))
    return plan


def gated4_fused_plan(*, rows: int, cols: int, k: int) -> list[Launch] | None:
    """metal.py:501-530, buffers [x, gate w/s/b, up w/s/b, gate out, up scratch]: the fused
    gate/up + SiLU routes for the measured Qwen3 MLP heights (a 24-row batch adds one 8-row tile
    after its 16-row prefix); None for every other shape, which runs linear4 for gate, linear4
    for up and silu_gate."""
    if rows not in (16, 24, 128, 160, 256, 512) or (cols, k) != (3072, 1024):
        return None
    shape = dict(rows=rows, cols=cols, k=k)
    fused = (0, 1, 2, 3, 4, 5, 6, 7)
    plan = [Launch("gated4_16x32_k64", rows // 16 * (cols // 32) * 256, 256, shape, fused)]
    if rows == 24:
        plan.append(Launch("gated4_8x32", cols // 32 * 128, 128, {**shape, "n": 16}, fused))
    return plan


def matmul_plan(*, rows: int, cols: int, k: int) -> list[Launch]:
    """metal.py:664-700, buffers [a, bt, out] with bt the [cols, k] weight: complete 8-row tiles on
    the chunked route for the BGE shapes and the scalar route for the rows after them; elsewhere
    the tiled route when aligned, else the scalar route."""
    shape = dict(rows=rows, cols=cols, k=k)
    if rows >= 8 and (cols, k) in BGE_PROJECTIONS:
        complete = rows // 8
        plan = [Launch("matmul_f32_chunk32", complete * (cols // 32) * 128, 128, shape)]
        if rows % 8:
            plan.append(Launch("matmul_f32", (rows % 8 + 3) // 4 * cols * 32, 32,
                               {**shape, "n": complete * 8}))
        return plan
    if rows >= 8 and rows % 8 == 0 and cols % 32 == 0 and k % 8 == 0 and k <= 512:
        return [Launch("matmul_f32_tiled", (rows + 7) // 8 * (cols // 32) * 128, 128, shape)]
    return [Launch("matmul_f32", (rows + 3) // 4 * cols * 32, 32, shape)]


def matmul_bias_plan(*, rows: int, cols: int, k: int) -> list[Launch] | None:
    """metal.py:702-731, buffers [a, bt, out, bias]: on the BGE shapes the bias is added after the
    same partial sums; None elsewhere, where the plain projection runs and then add_bias."""
    if rows < 8 or (cols, k) not in BGE_PROJECTIONS:
        return None
    shape = dict(rows=rows, cols=cols, k=k)
    complete = rows // 8
    plan = [Launch("matmul_bias_f32_chunk32", complete * (cols // 32) * 128, 128, shape)]
    if rows % 8:
        plan.append(Launch("matmul_bias_f32", (rows % 8 + 3) // 4 * cols * 32, 32,
                           {**shape, "n": complete * 8}))
    return plan


def _run_plan(target: Any, buffers: Sequence[Any], plan: list[Launch]) -> None:
    """Dispatch a route's launches in order through target._dispatch, each bound to its slots of
    `buffers`."""
    for launch in plan:
        bound = buffers if launch.slots is None else [buffers[i] for i in launch.slots]
        target._dispatch(launch.name, bound, threads=launch.threads,
                         group_size=launch.group_size, **launch.fields)


# ---- device memory ---------------------------------------------------------------------------


class Buffer:
    """A device allocation of `size` bytes owned by one HipRuntime. `pointer` is the library's
    opaque handle (None once released). Released by close() or when collected; released while a
    command is open, its device memory stays until that command has run."""

    __slots__ = ("runtime", "size", "pointer", "__weakref__")

    def __init__(self, runtime: "HipRuntime", size: int, data: NDArray[Any] | None) -> None:
        self.runtime = runtime
        self.size = size
        self.pointer: int | None = None
        self.pointer = runtime._memory.allocate(self, data)

    def close(self) -> None:
        runtime = getattr(self, "runtime", None)
        if runtime is None:
            return
        with runtime._lock:
            runtime._memory.release(self)

    def __del__(self) -> None:
        try:
            self.close()
        except Exception:  # interpreter shutdown: the library may already be gone
            pass


class _DeviceMemory:
    """Allocation ledger of one runtime: its live buffers, the bytes they hold, the high-water mark
    and cumulative allocation counts."""

    def __init__(self, lib: Any, handle: int) -> None:
        self.lib = lib
        self.handle = handle
        self.live: WeakSet[Buffer] = WeakSet()
        self.in_use = 0
        self.high_water = 0
        self.count = 0
        self.total = 0

    def allocate(self, buffer: Buffer, data: NDArray[Any] | None) -> int:
        pointer = self.lib.mi_buffer(self.handle, None if data is None else data.ctypes.data,
                                     buffer.size)
        if not pointer:
            raise InferenceError()
        self.in_use += buffer.size
        self.high_water = max(self.high_water, self.in_use)
        self.count += 1
        self.total += buffer.size
        self.live.add(buffer)
        return pointer

    def release(self, buffer: Buffer) -> None:
        pointer, buffer.pointer = buffer.pointer, None
        if pointer:
            self.lib.mi_free(pointer)
            self.in_use -= buffer.size
            self.live.discard(buffer)

    def release_all(self) -> None:
        for buffer in list(self.live):
            self.release(buffer)


class _Plan(NamedTuple):
    handle: int
    nbytes: int
    launches: Counter[str]


class _Retained:
    """Device memory kept between forwards under the runtime's workspace budget: scratch buffers
    returned by finished workspaces (handed out again to requests of the same size, oldest first)
    and prepared plans (at most MAX_PLANS; the least recently used goes first). Plans count
    against the budget with their host-side size, so neither kind can grow without bound."""

    def __init__(self, runtime: "HipRuntime") -> None:
        self.runtime = runtime
        self.scratch: OrderedDict[int, Buffer] = OrderedDict()  # id -> buffer, oldest first
        self.plans: OrderedDict[tuple[Any, ...], _Plan] = OrderedDict()
        self.scratch_bytes = 0
        self.plan_bytes = 0

    @property
    def limit(self) -> int:
        return self.runtime.workspace_limit_bytes

    def take(self, size: int) -> Buffer | None:
        for key, buffer in self.scratch.items():
            if buffer.size == size:
                del self.scratch[key]
                self.scratch_bytes -= size
                return buffer
        return None

    def keep(self, buffer: Buffer) -> bool:
        """Retain a released workspace buffer if the budget allows it, evicting older scratch."""
        if not buffer.pointer or self.plan_bytes + buffer.size > self.limit:
            return False
        self._shed_scratch(buffer.size)
        self.scratch[id(buffer)] = buffer
        self.scratch_bytes += buffer.size
        return True

    def _shed_scratch(self, incoming: int) -> None:
        while self.scratch and self.scratch_bytes + self.plan_bytes + incoming > self.limit:
            _, old = self.scratch.popitem(last=False)
            self.scratch_bytes -= old.size
            old.close()

    def plan(self, key: tuple[Any, ...]) -> _Plan | None:
        found = self.plans.get(key)
        if found is not None:
            self.plans.move_to_end(key)
        return found

    def add_plan(self, key: tuple[Any, ...], plan: _Plan) -> bool:
        if plan.nbytes > self.limit:
            return False
        while self.plans and (len(self.plans) >= MAX_PLANS
                              or self.plan_bytes + plan.nbytes > self.limit):
            _, old = self.plans.popitem(last=False)
            self._free_plan(old)
        self._shed_scratch(plan.nbytes)
        self.plans[key] = plan
        self.plan_bytes += plan.nbytes
        return True

    def _free_plan(self, plan: _Plan) -> None:
        self.runtime._lib.mi_plan_free(plan.handle)
        self.plan_bytes -= plan.nbytes

    def drop_plans(self) -> None:
        while self.plans:
            self._free_plan(self.plans.popitem()[1])

    def drop_scratch(self) -> None:
        while self.scratch:
            self.scratch.popitem()[1].close()
        self.scratch_bytes = 0


class _Lease:
    """The allocator a workspace hands out: requests without data reuse retained scratch of the same
    size; everything it handed out goes back (or is released) when the workspace closes."""

    def __init__(self, runtime: "HipRuntime") -> None:
        self.runtime = runtime
        self.handed: list[tuple[Buffer, bool]] = []
        self.open = True

    def __call__(self, size: int, data: NDArray[Any] | None = None) -> Buffer:
        if not self.open:
            raise InferenceError()
        buffer = self.runtime._retained.take(size) if data is None else None
        if buffer is None:
            buffer = self.runtime.buffer(size, data)
        self.handed.append((buffer, data is None))
        return buffer

    def close(self) -> None:
        self.open = False
        handed, self.handed = self.handed, []
        for buffer, reusable in handed:
            if not (reusable and self.runtime._retained.keep(buffer)):
                buffer.close()


class _Command:
    """One open command: the launch records kept for profiling and when recording started."""

    def __init__(self, profiled: bool) -> None:
        self.started = time.perf_counter()
        self.records: list[dict[str, Any]] | None = [] if profiled else None


class _PlanCapture(NamedTuple):
    handle: int
    slots: dict[Buffer, int]
    launches: Counter[str]


class _Stats:
    """Cumulative counters behind diagnostics()."""

    def __init__(self) -> None:
        self.commands = 0
        self.gpu_samples = 0
        self.gpu_seconds = 0.0
        self.encode_seconds = 0.0
        self.submit_wait_seconds = 0.0
        self.dispatches: Counter[str] = Counter()
        self.plan_hits = 0
        self.plan_builds = 0


# ---- the runtime ------------------------------------------------------------------------------


class HipRuntime:
    """Owner of one HIP stream and everything queued on it. Commands are serialized per instance:
    every public call takes the instance lock, and a command holds it until its launches ran."""

    def __init__(self, *, workspace_limit_bytes: int = 64 * 1024 * 1024) -> None:
        if type(workspace_limit_bytes) is not int or not 0 <= workspace_limit_bytes <= 2**30:
            raise InferenceError()
        self.workspace_limit_bytes = workspace_limit_bytes
        self._lib = _library()
        self._pointer: int | None = self._lib.mi_create(None)
        if not self._pointer:
            raise HipUnavailableError()
        self._lock = threading.RLock()
        self._memory = _DeviceMemory(self._lib, self._pointer)
        self._retained = _Retained(self)
        self._stats = _Stats()
        self._command: _Command | None = None
        self._capture: _PlanCapture | None = None
        self._workspace_open = False
        self._profile: list[dict[str, Any]] | None = None
        self._plans_enabled = True
        self.last_gpu_seconds = -1.0

    # ---- state ---------------------------------------------------------------------------------

    @property
    def active_bytes(self) -> int:
        return self._memory.in_use

    @property
    def peak_bytes(self) -> int:
        return self._memory.high_water

    @property
    def cache_bytes(self) -> int:
        return self._retained.scratch_bytes

    @property
    def _recording(self) -> bool:
        return self._command is not None

    def _check_open(self) -> None:
        if not self._pointer:
            raise ClosedError()

    def _owns(self, buffers: Sequence[Buffer]) -> bool:
        return all(b.pointer and b.runtime is self for b in buffers)

    def diagnostics(self) -> dict[str, Any]:
        """Cumulative counters under tessery's keys (metal.py:208-234), plus the library hash, the
        HIP-graph counts of plan replays and the launch-time fusions."""
        with self._lock:
            launches, builds = ct.c_uint64(0), ct.c_uint64(0)
            if not self._pointer or self._lib.mi_graph_counts(self._pointer, ct.byref(launches),
                                                              ct.byref(builds)):
                launches.value = builds.value = 0
            pairs, gated = ct.c_uint64(0), ct.c_uint64(0)
            if not self._pointer or self._lib.mi_fusion_counts(self._pointer, ct.byref(pairs),
                                                               ct.byref(gated)):
                pairs.value = gated.value = 0
            s = self._stats
            return {
                "native_library_sha256": self._lib._tessery_sha256,
                "allocations": self._memory.count,
                "allocated_bytes": self._memory.total,
                "completed_commands": s.commands,
                "gpu_timed_commands": s.gpu_samples,
                "gpu_seconds": s.gpu_seconds,
                "encode_seconds": s.encode_seconds,
                "submit_wait_seconds": s.submit_wait_seconds,
                "dispatches": dict(s.dispatches),
                "active_bytes": self.active_bytes,
                "cache_bytes": self.cache_bytes,
                "plan_cache_bytes": self._retained.plan_bytes,
                "plan_cache_entries": len(self._retained.plans),
                "plan_hits": s.plan_hits,
                "plan_builds": s.plan_builds,
                "graph_launches": int(launches.value),
                "graph_builds": int(builds.value),
                "fused_pairs": int(pairs.value),
                "fused_gated": int(gated.value),
                "peak_bytes": self.peak_bytes,
            }

    # ---- buffers -------------------------------------------------------------------------------

    def buffer(self, size: int, data: NDArray[Any] | None = None) -> Buffer:
        """A new device buffer of `size` bytes (1 <= size <= 2^31), zero-filled or holding `data`
        (C-contiguous, exactly `size` bytes)."""
        with self._lock:
            self._check_open()
            if type(size) is not int or size < 1 or size > 2**31:
                raise InferenceError()
            if data is not None and (not data.flags.c_contiguous or data.nbytes != size):
                raise InferenceError()
            return Buffer(self, size, data)

    def upload(self, data: NDArray[Any]) -> Buffer:
        """A buffer holding a copy of `data` (copied to C order first if needed)."""
        array = np.ascontiguousarray(data)
        return self.buffer(array.nbytes, array)

    def write(self, buffer: Buffer, data: NDArray[Any]) -> None:
        """Overwrite the start of `buffer` with host data, synchronously, outside commands."""
        array = np.ascontiguousarray(data)
        with self._lock:
            self._check_open()
            if self._recording or not self._owns([buffer]) or array.nbytes > buffer.size:
                raise InferenceError()
            if self._lib.mi_write(buffer.pointer, array.ctypes.data, array.nbytes):
                raise InferenceError()

    def read(self, buffer: Buffer, shape: tuple[int, ...],
             dtype: Any = np.float32) -> NDArray[Any]:
        """The whole buffer as a host array of `shape` and `dtype` (sizes must agree), outside
        commands."""
        dtype = np.dtype(dtype)
        with self._lock:
            self._check_open()
            if self._recording or not self._owns([buffer]):
                raise InferenceError()
            if int(np.prod(shape)) * dtype.itemsize != buffer.size:
                raise InferenceError()
            host = np.empty(shape, dtype=dtype)
            if self._lib.mi_read(buffer.pointer, host.ctypes.data, host.nbytes):
                raise InferenceError()
            return host

    # ---- commands ------------------------------------------------------------------------------

    @contextmanager
    def command(self) -> Iterator[None]:
        """Launches dispatched inside the block are queued; leaving it runs them in order and waits
        (metal.py:374-414). An exception inside, or a failed launch, discards what is queued and
        every prepared plan."""
        with self._lock:
            self._check_open()
            if self._recording:
                raise InferenceError()
            if self._lib.mi_begin(self._pointer):
                self._lib.mi_abort(self._pointer)
                raise InferenceError()
            command = _Command(self._profile is not None)
            self._command = command
            try:
                yield
                self._complete(command)
            except BaseException:
                self._retained.drop_plans()
                raise
            finally:
                self._lib.mi_abort(self._pointer)  # no-op after a finish; discards otherwise
                self._command = None

    def _complete(self, command: _Command) -> None:
        submitted = time.perf_counter()
        if self._lib.mi_finish(self._pointer):
            raise InferenceError()
        if command.records is not None:
            seconds = (ct.c_double * len(command.records))()
            fused = (ct.c_uint8 * len(command.records))()
            if self._lib.mi_profile_read(self._pointer, seconds, len(seconds)) or \
                    self._lib.mi_profile_fused(self._pointer, fused, len(fused)):
                raise InferenceError()
            carrier = None
            for record, value, inside in zip(command.records, seconds, fused, strict=True):
                record["gpu_seconds"] = float(value)
                # a dispatch that ran inside the kernel of the one before it: its events enclose
                # no work, its time is in the carrier's record
                if inside and carrier is not None:
                    record["fused_into"] = carrier["kernel"]
                else:
                    carrier = record
            assert self._profile is not None
            self._profile.extend(command.records)
        stats = self._stats
        stats.encode_seconds += submitted - command.started
        stats.submit_wait_seconds += time.perf_counter() - submitted
        stats.commands += 1
        self.last_gpu_seconds = float(self._lib.mi_gpu_seconds(self._pointer))
        if self.last_gpu_seconds >= 0:
            stats.gpu_seconds += self.last_gpu_seconds
            stats.gpu_samples += 1

    @contextmanager
    def profile_kernels(self) -> Iterator[list[dict[str, Any]]]:
        """Per-launch GPU seconds from HIP events around every launch of the commands run inside
        the block (at most 2048 launches per command); plans are not replayed meanwhile."""
        with self._lock:
            self._check_open()
            busy = self._recording or self._profile is not None
            if busy or self._lib.mi_profile_enable(self._pointer, 1):
                raise InferenceError()
            self._profile = []
            try:
                yield self._profile
            finally:
                self._profile = None
                self._lib.mi_profile_enable(self._pointer, 0)

    # ---- workspaces and prepared plans ---------------------------------------------------------

    @contextmanager
    def _workspace(self) -> Iterator[_Lease]:
        """A forward's allocator (see _Lease). Opened outside commands; what it handed out returns
        to the retained scratch (or is released) when the block ends, after its commands ran."""
        with self._lock:
            self._check_open()
            if self._recording or self._workspace_open:
                raise InferenceError()
            self._workspace_open = True
            lease = _Lease(self)
            try:
                yield lease
            finally:
                lease.close()
                self._workspace_open = False

    def trim_workspace(self) -> None:
        """Release every retained scratch buffer and prepared plan."""
        with self._lock:
            self._retained.drop_plans()
            self._retained.drop_scratch()

    def _clear_plans(self) -> None:
        self._retained.drop_plans()

    @contextmanager
    def _execution_plan(self, key: tuple[Any, ...], bindings: Sequence[Buffer]) -> Iterator[bool]:
        """Record (False) or replay (True) the launch sequence of `key` over `bindings`, inside a
        command and a workspace. A replay queues the recorded launches bound to these buffers, run
        by the library as one cached HIP graph; a recording keeps the launches dispatched in the
        block as a new plan. Profiling, a zero budget or disabled plans record nothing."""
        if not self._recording or not self._workspace_open or self._capture is not None:
            raise InferenceError()
        if not self._plans_enabled or self._profile is not None or not self.workspace_limit_bytes:
            yield False
            return
        if not self._owns(bindings):
            raise InferenceError()
        pointers = (ct.c_void_p * len(bindings))(*(b.pointer for b in bindings))
        plan = self._retained.plan(key)
        if plan is not None:
            if self._lib.mi_plan_run(self._pointer, plan.handle, pointers, len(bindings)):
                raise InferenceError()
            self._stats.dispatches.update(plan.launches)
            self._stats.plan_hits += 1
            yield True
            return
        handle = self._lib.mi_plan_create(self._pointer, pointers, len(bindings))
        if not handle:
            raise InferenceError()
        capture = _PlanCapture(handle, {b: i for i, b in enumerate(bindings)}, Counter())
        self._capture = capture
        kept = False
        try:
            yield False
            entry = _Plan(handle, int(self._lib.mi_plan_bytes(handle)), capture.launches)
            kept = self._retained.add_plan(key, entry)
            if kept:
                self._stats.plan_builds += 1
        finally:
            self._capture = None
            if not kept:
                self._lib.mi_plan_free(handle)

    # ---- dispatch ------------------------------------------------------------------------------

    def _dispatch(
        self,
        name: str,
        buffers: Sequence[Buffer],
        *,
        threads: int,
        group_size: int = 256,
        n: int = 0,
        rows: int = 0,
        cols: int = 0,
        k: int = 0,
        heads: int = 0,
        kv_heads: int = 0,
        seq: int = 0,
        batch: int = 0,
        dim: int = 0,
        group: int = 64,
        eps: float = 1e-6,
        theta: float = 1e6,
        scale: float = 1.0,
        bidirectional: int = 0,
        first_token: int = 0,
        out_f16: int = 0,
        flags: int = 0,
    ) -> None:
        """Queue one launch of kernel `name` on `buffers` (metal.py:571-648). Params u0 carries the
        bidirectional flag; u1 the reference's first_token flag, and in this library also the fp16
        output flag of the attention_f16 routes (out_f16) and route flags (norm_rope_f16: bit 0
        writes hi + lo planes; qkv4_f16: bit 0 selects bf16 scales)."""
        if self._command is None or not self._owns(buffers):
            raise InferenceError()
        params = pack_params(n=n, rows=rows, cols=cols, k=k, heads=heads, kv_heads=kv_heads,
                             seq=seq, batch=batch, dim=dim, group=group, u0=int(bidirectional),
                             u1=int(first_token) | int(out_f16) | int(flags), eps=eps,
                             theta=theta, scale=scale)
        kernel = name.encode("ascii")
        handles = (ct.c_void_p * len(buffers))(*(b.pointer for b in buffers))
        if self._lib.mi_dispatch(self._pointer, kernel, handles, len(buffers), params,
                                 len(params), threads, group_size):
            raise InferenceError()
        capture = self._capture
        if capture is not None:
            slots = (ct.c_uint32 * len(buffers))(*(capture.slots[b] for b in buffers))
            if self._lib.mi_plan_add(capture.handle, kernel, slots, len(buffers), params, threads,
                                     group_size):
                raise InferenceError()
            capture.launches[name] += 1
        self._stats.dispatches[name] += 1
        if self._command.records is not None:
            self._command.records.append(dict(kernel=name, rows=rows, cols=cols, k=k, seq=seq,
                                              heads=heads, threads=threads))

    # ---- routes --------------------------------------------------------------------------------

    def _attention(self, buffers: Sequence[Buffer], *, tokens: int, seq: int, heads: int,
                   kv_heads: int, dim: int, bidirectional: int = 0, precision: str = "f32",
                   out_dtype: str | None = None) -> None:
        """buffers = [q, k, v, lengths (u32), out]; the route selection of metal.py:532-569 (see
        attention_plan). precision="f16" takes fp16 q/k/v and accumulates in fp32 on MFMA;
        out_dtype ("f32" or "f16", default f32) selects the output element type there."""
        _run_plan(self, buffers, attention_plan(tokens=tokens, seq=seq, heads=heads, kv_heads=kv_heads,
                                          dim=dim, bidirectional=bidirectional,
                                          precision=precision, out_dtype=out_dtype))

    def _attention_norm_rope(self, buffers: Sequence[Buffer], *, tokens: int, seq: int,
                             heads: int, kv_heads: int, dim: int, eps: float = 1e-6,
                             theta: float = 1e6, bidirectional: int = 0,
                             out_dtype: str = "f32") -> None:
        """The Qwen3 attention block tail (qwen3.py:216-245) on fp16 activations:
        buffers = [q_pre, k_pre, v, lengths, out, q_norm(bf16 [dim]), k_norm(bf16 [dim]),
        k_work]. k_work (twice k_pre's size) receives the normalized, rotated keys of valid rows
        as two fp16 planes (hi, lo); q is normalized and rotated inside the attention kernel as it
        is loaded. Scores use the hi/lo pairs of both q and k, probabilities are split the same
        way, all accumulation is fp32; out_dtype "f32" (default) or "f16"."""
        if len(buffers) != 8:
            raise InferenceError()
        _run_plan(self, buffers, attention_norm_rope_plan(
            tokens=tokens, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, eps=eps,
            theta=theta, bidirectional=bidirectional, out_dtype=out_dtype))

    def _qkv4(self, buffers: Sequence[Buffer], *, rows: int, k: int, q_cols: int, kv_cols: int,
              scale_dtype: str = "bf16") -> None:
        """Fused uint4 group-64 Q/K/V projection of fp16 activations (the three _linear4 calls of
        qwen3.py:195-215 in one launch). buffers = [x fp16 [rows, k], w u32 [q_cols+2*kv_cols,
        k/8], scales, biases ([q_cols+2*kv_cols, k/64] words), yq, yk, yv fp16]: the q, k and v
        weight rows concatenated along N (tessery's dispatch holds at most 8 buffers).
        scale_dtype "bf16" (tessery's storage) or "f16"."""
        flag = {"bf16": 1, "f16": 0}.get(scale_dtype)
        if flag is None:
            raise InferenceError()
        self._dispatch("qkv4_f16", buffers, threads=rows, group_size=256, rows=rows, k=k,
                       cols=q_cols, n=kv_cols, flags=flag)

    def _attention_masked(self, buffers: Sequence[Buffer], *, tokens: int, seq: int, heads: int,
                          kv_heads: int, dim: int, mask: str = "causal", window: int = 0,
                          cap: float = 0.0, scale: float | None = None, precision: str = "f16",
                          packed: bool | str = False, prefix: Buffer | None = None,
                          spans: Buffer | None = None, slopes: Buffer | None = None,
                          table: Buffer | None = None, radius: int = 0) -> None:
        """Attention whose scores and keys depend on more than q and k; buffers = [q, k, v, lengths
        (u32 [batch]), out], fp16 or fp32 (`precision`) as _attention lays them out, out of the same
        type. dim is a multiple of 8 up to 256.

        Scores are scale * q.k (scale: dim^-0.5 unless given), then cap * tanh(score / cap) with a
        cap > 0, then less slopes[head] * |i - j| (fp32 [heads]) or plus
        table[head, clamp(j - i, -radius, radius) + radius] (fp32 [heads, 2 * radius + 1]).

        Token i of a batch row attends the keys j below the row's length that `mask` leaves -
        "causal" j <= i, "bidirectional" all, "prefix" j <= i or j < prefix[row] (u32 [batch]) -
        and that satisfy |i - j| < window (0: no window) and
        spans[row, i, 0] <= j < spans[row, i, 1] (u32 [batch, seq, 2], the documents of packed rows:
        batching.document_spans). A token that attends no key gets zeros. Rows at or past the length
        are outputs like any other. Infinities and NaN of keys and values reach only the tokens
        that attend them.

        packed: q, k and v are one buffer (given three times) whose rows hold the heads of q, k and
        v; "v": only v lies in such rows."""
        if len(buffers) != 5:
            raise InferenceError()
        plan = attention_masked_plan(
            tokens=tokens, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim, mask=mask,
            window=window, cap=cap, radius=radius, scale=scale, precision=precision,
            packed=packed, spans=spans is not None, slopes=slopes is not None,
            table=table is not None, prefix=prefix is not None)
        _run_plan(self, [*buffers, spans, slopes if slopes is not None else table, prefix], plan)

    def _rotary(self, buffers: Sequence[Buffer | None], *, tokens: int, seq: int, heads: int,
                kv_heads: int, dim: int, rotary_dim: int, layout: str = "half",
                precision: str = "f16", packed: bool = False, positions: Buffer | None = None,
                q_norm: Buffer | None = None, k_norm: Buffer | None = None,
                eps: float = 1e-6) -> None:
        """Rotation of q and k by position, after their per-head RMSNorm where q_norm and k_norm
        (bf16 [dim]) are given; buffers = [q [tokens, heads, dim], k [tokens, kv_heads, dim], table,
        q_out, k_out], fp16 or fp32 (`precision`), table as rotary.table makes it (fp32 [positions,
        rotary_dim]). The first rotary_dim channels of a head turn, in pairs (c, c + rotary_dim / 2)
        ("half") or (2c, 2c + 1) ("interleaved"); the others keep their normed values. q_out and
        k_out may be q and k. kv_heads = 0: only q (k and k_out None).

        positions: u32 [tokens] (documents of packed rows: batching.document_positions); without
        them a token's index in its row of seq tokens. A position behind the table gives zeros.

        packed: q and k are one buffer whose rows hold the heads of q, k and v (kv_heads of v); so
        are q_out and k_out when they are that buffer, else they hold q and k alone."""
        if len(buffers) != 5 or (q_norm is None) != (k_norm is None) and (kv_heads or k_norm):
            raise InferenceError()
        q, k, table, q_out, k_out = buffers
        same = packed and q_out is q and k_out is k
        plan = rotary_plan(tokens=tokens, seq=seq, heads=heads, kv_heads=kv_heads, dim=dim,
                           rotary_dim=rotary_dim, layout=layout, precision=precision, eps=eps,
                           packed=packed, packed_out=same, positions=positions is not None,
                           norm=q_norm is not None)
        _run_plan(self, [q, k, table, q_out, k_out, positions, q_norm, k_norm], plan)

    def _rotary_table(self, buffers: Sequence[Buffer], *, positions: int, rotary_dim: int,
                      factor: float = 1.0) -> None:
        """The table _rotary reads; buffers = [frequencies (float64 [rotary_dim / 2], radians a
        position), table (fp32 [positions, rotary_dim])]. The cosines and sines of
        position * frequency are taken in float64 and multiplied by `factor`."""
        if len(buffers) != 2 or not _sized(positions, rotary_dim) or rotary_dim % 2 or \
                not math.isfinite(factor):
            raise InferenceError()
        self._dispatch("rotary_table", buffers, threads=positions * (rotary_dim // 2),
                       group_size=256, n=positions, dim=rotary_dim, scale=factor)

    def _linear_f16(self, buffers: Sequence[Buffer], *, rows: int, cols: int, k: int,
                    bias: Buffer | None = None, residual: Buffer | None = None,
                    activation: str = "none", out_dtype: str = "f16") -> None:
        """out = act(x w^T + bias) + residual for fp16 activations and weights; buffers = [x [rows,
        k], w [cols, k], out [rows, cols]], bias fp32 [cols], residual fp16 [rows, cols], out fp16
        or fp32 (`out_dtype`). activation: "none", "relu", "gelu" (with erf), "gelu_tanh" or
        "silu". Sums and epilogue are fp32, rounded once. A fp16 out may be the residual."""
        if len(buffers) != 3:
            raise InferenceError()
        _run_plan(self, [*buffers, bias, residual], linear_f16_plan(
            rows=rows, cols=cols, k=k, activation=activation, out_dtype=out_dtype,
            bias=bias is not None, residual=residual is not None))

    def _linear4(self, buffers: Sequence[Buffer], *, rows: int, cols: int, k: int) -> None:
        """uint4 projection [x, w, scales, biases, out] over the route partition of
        metal.py:416-499 (see linear4_plan)."""
        _run_plan(self, buffers, linear4_plan(rows=rows, cols=cols, k=k))

    def _gated4(self, buffers: Sequence[Buffer], *, rows: int, cols: int, k: int) -> None:
        """Fused gate/up projection + SiLU (metal.py:501-530): buffers = [x, gate w/s/b,
        up w/s/b, gate output, up scratch]; identical results on the fused and unfused routes.
        The unfused form goes through _linear4 twice, as in the reference."""
        fused = gated4_fused_plan(rows=rows, cols=cols, k=k)
        if fused is not None:
            _run_plan(self, buffers, fused)
            return
        x, gate, up = buffers[0], buffers[7], buffers[8]
        self._linear4([x, *buffers[1:4], gate], rows=rows, cols=cols, k=k)
        self._linear4([x, *buffers[4:7], up], rows=rows, cols=cols, k=k)
        self._dispatch("silu_gate", [gate, up], threads=rows * cols, n=rows * cols)

    def _matmul_f32(self, buffers: Sequence[Buffer], *, rows: int, cols: int, k: int) -> None:
        """fp32 projection [a, bt, out] with bt the [cols, k] weight (metal.py:664-700)."""
        _run_plan(self, buffers, matmul_plan(rows=rows, cols=cols, k=k))

    def _matmul_bias_f32(self, buffers: Sequence[Buffer], *, rows: int, cols: int,
                         k: int) -> None:
        """BGE affine projection [a, bt, out, bias] (metal.py:702-731); outside the BGE shapes
        the plain projection (through _matmul_f32, as in the reference) then add_bias."""
        plan = matmul_bias_plan(rows=rows, cols=cols, k=k)
        if plan is not None:
            _run_plan(self, buffers, plan)
            return
        self._matmul_f32(buffers[:3], rows=rows, cols=cols, k=k)
        self._dispatch("add_bias", buffers[2:4], threads=rows * cols, n=rows * cols, cols=cols)

    # ---- one-shot operations -------------------------------------------------------------------

    def _one_shot(self, inputs: Sequence[NDArray[np.float32]], out_shape: tuple[int, ...],
                  launch: Any) -> NDArray[np.float32]:
        """Upload `inputs`, run `launch(buffers)` in one command with an output buffer appended,
        read the output back and release everything."""
        with self._lock:
            held: list[Buffer] = []
            try:
                held.extend(self.upload(array) for array in inputs)
                held.append(self.buffer(int(np.prod(out_shape)) * 4))
                with self.command():
                    launch(held)
                return self.read(held[-1], out_shape)
            finally:
                for buffer in held:
                    buffer.close()

    @staticmethod
    def _f32_operands(*arrays: Any) -> bool:
        return all(isinstance(a, np.ndarray) and a.dtype == np.float32 and a.size for a in arrays)

    def add(self, a: NDArray[np.float32], b: NDArray[np.float32]) -> NDArray[np.float32]:
        """Elementwise float32 a + b on the device (tessery's add kernel)."""
        if not self._f32_operands(a, b) or a.shape != b.shape:
            raise InferenceError()
        return self._one_shot([a, b], a.shape, lambda bufs: self._dispatch(
            "add", bufs, threads=a.size, n=a.size))

    def matmul(self, a: NDArray[np.float32], b: NDArray[np.float32]) -> NDArray[np.float32]:
        """float32 [M, K] @ [K, N] on the device: b goes up transposed, as projection weights are,
        and runs the _matmul_f32 route partition."""
        if not self._f32_operands(a, b) or a.ndim != 2 or b.ndim != 2 or a.shape[1] != b.shape[0]:
            raise InferenceError()
        (m, k), n = a.shape, b.shape[1]
        return self._one_shot([a, b.T], (m, n), lambda bufs: self._matmul_f32(
            bufs, rows=m, cols=n, k=k))

    # ---- lifetime ------------------------------------------------------------------------------

    def close(self) -> None:
        """Release every buffer, plan and the stream. Not allowed inside a command, a workspace or
        a profiling block."""
        with self._lock:
            if self._recording or self._workspace_open or self._profile is not None:
                raise InferenceError()
            if not self._pointer:
                return
            self.trim_workspace()
            self._memory.release_all()
            self._lib.mi_destroy(self._pointer)
            self._pointer = None

    def __enter__(self) -> "HipRuntime":
        return self

    def __exit__(self, *_: object) -> None:
        self.close()

    def __del__(self) -> None:
        if getattr(self, "_pointer", None) and hasattr(self, "_lock"):
            try:
                self.close()
            except Exception:
                pass


MetalRuntime = HipRuntime
