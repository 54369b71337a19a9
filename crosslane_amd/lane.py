"""ctypes binding of libcrosslane.so and the `Lane` class.

`Lane` keeps the reference lane's method names and meaning
(engine/strata/warm/runtime.hpp:10-16):

    warm_contains(layer, e)            -> bool
    warm_grouped()                     -> True (layer batches run in one call)
    warm_compute(layer, e, x)          -> y            (one expert)
    warm_compute_many(layer, ids, x)   -> [y_i ...]    (ids order)

plus `layer_forward`, which adds the caller's fixed-order combine
(warm_execute, engine/strata/warm/runtime.cpp:180-188), and device-resident
variants taking torch CUDA tensors. Errors raise `XLError`, as the reference
raises std::runtime_error from `require`.
"""
from __future__ import annotations

import ctypes as C
import os
import struct
import sys
from typing import Optional, Sequence

import numpy as np

IQ2_XXS, IQ2_XS, IQ1_M = 16, 17, 29
BLOCK_BYTES = {IQ2_XXS: 66, IQ2_XS: 74, IQ1_M: 56}
ABI_VERSION = 3
_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libcrosslane.so")


class XLError(RuntimeError):
    def __init__(self, code: int, message: str):
        super().__init__(f"[xl {code}] {message}")
        self.code = code


class _Err(C.Structure):
    _fields_ = [("code", C.c_int32), ("message", C.c_char * 512)]


class _Config(C.Structure):
    _fields_ = [("struct_bytes", C.c_uint32), ("device", C.c_int32), ("dim", C.c_int32), ("ff", C.c_int32),
                ("n_layers", C.c_int32), ("n_experts", C.c_int32), ("max_picks", C.c_int32),
                ("max_tokens", C.c_int32), ("swiglu_limit", C.c_float)]


class _BankInfo(C.Structure):
    _fields_ = [("payload_bytes", C.c_uint64), ("allocated_bytes", C.c_uint64), ("workspace_bytes", C.c_uint64),
                ("n_layers", C.c_int32), ("n_experts", C.c_int32), ("generated", C.c_int32),
                ("reserved", C.c_int32)]


_P = C.c_void_p
_I32 = C.c_int32
_f32p = np.ctypeslib.ndpointer(np.float32, flags="C_CONTIGUOUS")
_i32p = np.ctypeslib.ndpointer(np.int32, flags="C_CONTIGUOUS")
_u64p = np.ctypeslib.ndpointer(np.uint64, flags="C_CONTIGUOUS")
_ErrP = C.POINTER(_Err)


class _KVBatch(C.Structure):
    _fields_ = [("struct_bytes", C.c_uint32), ("head_dim", C.c_int32), ("kv_heads", C.c_int32), ("page_tokens", C.c_int32),
                ("n_pages", C.c_int32), ("max_pages", C.c_int32), ("n_seqs", C.c_int32), ("rows", C.c_int32),
                ("max_rows", C.c_int32), ("reserved", C.c_int32), ("page_stride", C.c_int64), ("table_stride", C.c_int64),
                ("pages", _P), ("table", _P), ("lens", _P), ("starts", _P)]


class _Rotary(C.Structure):
    _fields_ = [("struct_bytes", C.c_uint32), ("n_freqs", C.c_int32), ("n_axes", C.c_int32), ("interleaved", C.c_int32),
                ("section", C.c_int32 * 3), ("reserved", C.c_int32), ("positions_stride", C.c_int64), ("freqs", _P),
                ("positions", _P)]


_ROTARY_BYTES = C.sizeof(_Rotary)
_ROTARY = struct.Struct("=I7iqQQ")   # the same fields
assert _ROTARY.size == _ROTARY_BYTES


class _PackMeta(C.Structure):
    _fields_ = [("struct_bytes", C.c_uint32), ("dim", C.c_int32), ("ff", C.c_int32), ("n_layers", C.c_int32),
                ("n_experts", C.c_int32), ("top_k", C.c_int32), ("swiglu_limit", C.c_float)]


_SIGNATURES = {
    "xl_abi_version": (C.c_uint32, []),
    "xl_open": (_I32, [C.c_uint32, C.POINTER(_Config), C.POINTER(_P), _ErrP]),
    "xl_close": (None, [_P]),
    "xl_last_error": (_I32, [_P, _ErrP]),
    "xl_bank_create": (_I32, [_P, _i32p, _ErrP]),
    "xl_bank_generate": (_I32, [_P, C.c_uint64, _ErrP]),
    "xl_bank_upload": (_I32, [_P, _I32, _I32, _I32, _P, C.c_uint64, _ErrP]),
    "xl_bank_download": (_I32, [_P, _I32, _I32, _I32, _P, C.c_uint64, _ErrP]),
    "xl_bank_info_get": (_I32, [_P, C.POINTER(_BankInfo)]),
    "xl_contains": (_I32, [_P, _I32, _I32]),
    "xl_expert_forward": (_I32, [_P, _I32, _I32, _f32p, _f32p, _ErrP]),
    "xl_experts_forward": (_I32, [_P, _I32, _i32p, _I32, _f32p, _f32p, _ErrP]),
    "xl_layer_forward": (_I32, [_P, _I32, _i32p, _f32p, _I32, _f32p, _P, _f32p, _ErrP]),
    "xl_expert_trace": (_I32, [_P, _I32, _I32, _f32p, _P, _P, _P, _P, _P, _ErrP]),
    "xl_layer_forward_async": (_I32, [_P, _I32, _P, _P, _I32, _P, _P, _P, _P, _ErrP]),
    "xl_sync": (_I32, [_P, _P, _ErrP]),
    "xl_layer_trace_async": (_I32, [_P, _I32, _P, _P, _I32, _P, _P, _P, _P, _P, _P, _P, _P, C.POINTER(_I32), _P,
                                    _ErrP]),
    "xl_grouped_trace_async": (_I32, [_P, _I32, _I32, _I32, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _P, _ErrP]),
    "xl_combine_async": (_I32, [_P, _P, _P, _I32, _P, _I32, _P, _P, _P, _ErrP]),
    "xl_grouped_forward": (_I32, [_P, _I32, _I32, _I32, _i32p, _f32p, _f32p, _P, _f32p, _ErrP]),
    "xl_grouped_forward_async": (_I32, [_P, _I32, _I32, _I32, _P, _P, _P, _P, _P, _P, _ErrP]),
    "xl_route_async": (_I32, [_P, _P, _I32, _I32, _P, _I32, _I32, C.c_float, _P, _P, _P, _ErrP]),
    "xl_pack_meta_get": (_I32, [C.c_char_p, C.POINTER(_PackMeta), _ErrP]),
    "xl_pack_types": (_I32, [C.c_char_p, _I32, _I32, _I32, _i32p, _ErrP]),
    "xl_bank_load_pack": (_I32, [_P, C.c_char_p, _I32, _ErrP]),
    "xl_layer_forward_routed_async": (_I32, [_P, _I32, _P, _P, _I32, C.c_float, _P, _P, _P, _P, _ErrP]),
    "xl_grouped_forward_routed_async": (_I32, [_P, _I32, _I32, _P, _P, _I32, C.c_float, _P, _P, _P, _P, _ErrP]),
    "xl_quantize_q8k_async": (_I32, [_P, _P, _I32, _I32, _P, _P, _ErrP]),
    "xl_matvec_async": (_I32, [_P, _I32, _P, _I32, _I32, _P, _P, _P, _P, _ErrP]),
    "xl_swiglu_async": (_I32, [_P, _P, _P, _I32, C.c_float, _P, _P, _ErrP]),
    "xl_layer_forward_per32": (_I32, [_P, _I32, _i32p, _P, _I32, _f32p, _P, _P, _P, _ErrP]),
    "xl_layer_forward_per32_async": (_I32, [_P, _I32, _P, _P, _I32, _P, _P, _P, _P, _P, _ErrP]),
    "xl_quantize_per32_async": (_I32, [_P, _P, _I32, _I32, _P, _P, _P, _ErrP]),
    "xl_matvec_per32_async": (_I32, [_P, _I32, _P, _I32, _I32, _P, _P, _P, _P, _ErrP]),
    "xl_shared_work_bytes": (C.c_uint64, [_I32, _I32, _I32]),
    "xl_shared_forward_async": (_I32, [_P, _I32, _P, _I32, _P, _I32, _P, _I32, _I32, _P, _P, _P, C.c_uint64, _P,
                                       _ErrP]),
    "xl_shared_forward_noalloc": (_I32, [_P, _I32, _P, _I32, _P, _I32, _P, _I32, _I32, _P, _P, _P, _ErrP]),
    "xl_hc_post_async": (_I32, [_P, _P, _P, _P, _P, _I32, _I32, _I32, _P, _P, _ErrP]),
    "xl_hc_pre_norm_async": (_I32, [_P, _P, _P, _P, _I32, _I32, _I32, C.c_float, _P, _P, _ErrP]),
    "xl_layer_forward_prenorm_async": (_I32, [_P, _I32, _P, _P, _I32, _P, _I32, _P, _P, C.c_float, _P, _P, _P, _P,
                                              _ErrP]),
    "xl_layer_forward_post_async": (_I32, [_P, _I32, _P, _P, _I32, _P, _P, _P, _P, _P, _P, _I32, _P, _P, _ErrP]),
    "xl_moe_block_async": (_I32, [_P, _I32, _P, _P, _I32, _P, _I32, _P, _I32, _P, _I32, _P, _I32, _P, C.c_uint64,
                                  _P, _P, _P, _I32, _P, _P, _P, _ErrP]),
    "xl_route_scored_async": (_I32, [_P, _P, _I32, _I32, C.c_int64, _P, _I32, _I32, _I32, _I32, _I32, _I32, _I32,
                                     C.c_float, _P, _P, _P, _ErrP]),
    "xl_block_norm_async": (_I32, [_P, _P, C.c_int64, _P, C.c_int64, _P, C.c_int64, _P, _P, _I32, _I32, _I32, _I32,
                                   C.c_float, C.c_float, _P, C.c_int64, _P, C.c_int64, _P, C.c_int64, _P, _P, _ErrP]),
    "xl_quantize_rows_async": (_I32, [_P, _P, _I32, _I32, _I32, C.c_int64, _P, C.c_int64, _P, _P, _ErrP]),
    "xl_linear_i8_work_bytes": (C.c_uint64, [_I32, _I32, _I32, _I32]),
    "xl_linear_i8_async": (_I32, [_P, _P, _I32, _P, C.c_int64, _I32, _I32, _P, _P, _P, _P, C.c_int64, _I32, C.c_float,
                                  _P, _I32, C.c_int64, _P, C.c_uint64, _P, _ErrP]),
    "xl_kv_page_bytes": (C.c_uint64, [_I32, _I32]),
    "xl_kv_write_async": (_I32, [_P, _P, _P, C.c_int64, _P, C.c_int64, _I32, _P, _P, C.c_int64, _I32, _P, C.c_int64, _P, _ErrP]),
    "xl_kv_read_async": (_I32, [_P, _P, _P, C.c_int64, _P, C.c_int64, _I32, _P, _ErrP]),
    "xl_attention_work_bytes": (C.c_uint64, [_P, _I32]),
    "xl_attention_async": (_I32, [_P, _P, _P, C.c_int64, _I32, _I32, C.c_float, _I32, C.c_float, _P, C.c_int64, _P, C.c_uint64,
                                  _P, _ErrP]),
    "xl_profile_begin": (_I32, [_P, _I32, _ErrP]),
    "xl_profile_end": (_I32, [_P, _f32p, _I32, C.POINTER(_I32), C.POINTER(_I32), C.c_char_p, _I32, _ErrP]),
    "xl_profile_timeline": (_I32, [_P, _u64p, _I32, C.POINTER(_I32), _ErrP]),
    "xl_debug_set_launch_count": (_I32, [_P, C.c_uint32, _ErrP]),
    "xl_layer_forward_exact_async": (_I32, [_P, _I32, _P, _P, _I32, _P, _P, _P, _P, _ErrP]),
    "xl_debug_launch_counts": (_I32, [_P, np.ctypeslib.ndpointer(np.int64, flags="C_CONTIGUOUS"), _I32, _ErrP]),
    "xl_planar_bytes": (C.c_uint64, [_I32, _I32, _I32]),
    "xl_repack": (_I32, [_I32, _I32, _I32, _P, _P]),
    "xl_restore": (_I32, [_I32, _I32, _I32, _P, _P]),
    "xl_generate_host": (_I32, [_I32, C.c_uint64, _I32, _I32, _I32, _I32, _I32, _P]),
    "xl_codebook": (_I32, [_I32, _u64p]),
}

_lib: Optional[C.CDLL] = None


def lib() -> C.CDLL:
    """Loads libcrosslane.so from the package directory. No fallback."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise ImportError(f"{LIB_PATH} is missing: build it with `python -m crosslane_amd._build` "
                              "(or __graft_entry__.build()); there is no CPU fallback")
        L = C.CDLL(LIB_PATH)
        for name, (res, args) in _SIGNATURES.items():
            f = getattr(L, name)
            f.restype = res
            f.argtypes = args
        if L.xl_abi_version() != ABI_VERSION:
            raise ImportError("libcrosslane.so ABI version differs from this binding")
        _lib = L
    return _lib


def _check(rc: int, err: _Err) -> None:
    if rc != 0:
        raise XLError(int(err.code or rc), err.message.decode(errors="replace"))


def _ptr(t) -> Optional[int]:
    if t is None:
        return None
    return int(t.data_ptr())


# ---- host utilities (no GPU) -------------------------------------------------
def planar_bytes(t: int, n: int, k: int) -> int:
    return int(lib().xl_planar_bytes(t, n, k))


def repack(t: int, n: int, k: int, aos: np.ndarray) -> np.ndarray:
    aos = np.ascontiguousarray(aos, dtype=np.uint8)
    assert aos.size == n * (k // 256) * BLOCK_BYTES[t]
    out = np.zeros(planar_bytes(t, n, k), dtype=np.uint8)
    rc = lib().xl_repack(t, n, k, aos.ctypes.data, out.ctypes.data)
    if rc:
        raise XLError(rc, "repack rejected its arguments")
    return out


def restore(t: int, n: int, k: int, planar: np.ndarray) -> np.ndarray:
    planar = np.ascontiguousarray(planar, dtype=np.uint8)
    out = np.zeros(n * (k // 256) * BLOCK_BYTES[t], dtype=np.uint8)
    rc = lib().xl_restore(t, n, k, planar.ctypes.data, out.ctypes.data)
    if rc:
        raise XLError(rc, "restore rejected its arguments")
    return out


def generate_host(t: int, seed: int, layer: int, expert: int, role: int, n: int, k: int) -> np.ndarray:
    out = np.zeros(n * (k // 256) * BLOCK_BYTES[t], dtype=np.uint8)
    rc = lib().xl_generate_host(t, seed, layer, expert, role, n, k, out.ctypes.data)
    if rc:
        raise XLError(rc, "generate_host rejected its arguments")
    return out


def codebook(which: int) -> np.ndarray:
    out = np.zeros((256, 512, 2048, 128)[which], dtype=np.uint64)
    rc = lib().xl_codebook(which, out)
    if rc:
        raise XLError(rc, "codebook index")
    return out


def pack_meta(pack_dir: str) -> dict:
    """Shape of a weight pack (ds4.txt): dim, ff, n_layers, n_experts, top_k, swiglu_limit."""
    m = _PackMeta(C.sizeof(_PackMeta))
    err = _Err()
    _check(lib().xl_pack_meta_get(os.fsencode(pack_dir), C.byref(m), C.byref(err)), err)
    return {f: getattr(m, f) for f, _ in _PackMeta._fields_[1:]}


def shared_work_bytes(dim: int, ff: int, T: int = 1) -> int:
    """Workspace bytes xl_shared_forward_async needs for T tokens."""
    return int(lib().xl_shared_work_bytes(dim, ff, T))


def linear_i8_work_bytes(T: int, K: int, N: int, gated: bool = False) -> int:
    """Workspace bytes xl_linear_i8_async needs for T tokens of K values and N output channels."""
    return int(lib().xl_linear_i8_work_bytes(T, K, N, int(gated)))


SCORES = {"softmax": 0, "sigmoid": 1}


class _Kinds(dict):
    """Element types of the calls around a block (XL_F32 ..., 4: int32 vectors) by
    torch dtype; looked up by name once each, torch itself is not imported here."""
    NAMES = {"torch.float32": 0, "torch.float16": 1, "torch.bfloat16": 2, "torch.int8": 3, "torch.int32": 4}

    def __missing__(self, dtype) -> int:   # other types: -2 (-1 stands for a matrix that is not given)
        kind = self[dtype] = self.NAMES.get(str(dtype), -2)
        return kind


_KINDS = _Kinds()
_INT8, _INT32 = 3, 4


# The checks below run before every launch of a decode loop: no message is built
# and no attribute read that a passing call does not need.
def _refuse(message: str):
    raise XLError(1, message)


def _act(t, what: str) -> int:
    kind = _KINDS[t.dtype]
    if not 0 <= kind < _INT8:
        _refuse(f"{what}: element type {t.dtype} not taken here")
    return kind


def _mat(t, what: str, shape=None):
    """A [T, n] matrix of contiguous rows on the GPU: address, row stride, element type (None: null)."""
    if t is None:
        return None, 0, -1
    sh, st = t.shape, t.stride()
    if len(sh) != 2 or (st[1] != 1 and sh[1] != 1):
        _refuse(f"{what}: a matrix of contiguous rows is wanted")
    if not t.is_cuda:
        _refuse(f"{what}: not on the GPU")
    if shape is not None and sh != shape:
        _refuse(f"{what}: shape {tuple(sh)} where {tuple(shape)} is wanted")
    row = st[0]
    if sh[0] <= 1 and row < sh[1]:
        row = sh[1]
    return t.data_ptr(), row, _KINDS[t.dtype]


def _vec(t, n: int, what: str, kind: int = 0):
    """The address of a contiguous GPU vector of n values (None passes)."""
    if t is None:
        return None
    if not (t.is_cuda and t.is_contiguous() and t.numel() == n and _KINDS[t.dtype] == kind):
        _refuse(f"{what}: {n} contiguous values of the right type on the GPU are wanted")
    return t.data_ptr()


def _heads(t, what: str, shape):
    """[rows, heads, head_dim] on the GPU, a row's heads consecutive: address, row stride, element type."""
    rows, heads, dim = shape
    row, st1, st2 = t.stride() if t.shape == shape else (0, 0, 0)
    if st2 != 1 or (st1 != dim and heads != 1) or not t.is_cuda:
        if t.shape != shape:
            _refuse(f"{what}: shape {tuple(t.shape)} where {tuple(shape)} is wanted")
        if st2 != 1 or (st1 != dim and heads != 1):
            _refuse(f"{what}: a row's heads must be consecutive")
        _refuse(f"{what}: not on the GPU")
    if rows == 1 and row < heads * dim:
        row = heads * dim
    return t.data_ptr(), row, _KINDS[t.dtype]


def kv_page_bytes(page_tokens: int, head_dim: int) -> int:
    """Bytes of one kv head in a page of the 4-bit cache (0: not a size it takes)."""
    return int(lib().xl_kv_page_bytes(page_tokens, head_dim))


class KVBatch:
    """A batch of sequences over a 4-bit cache of keys and values, for `kv_write_async`,
    `kv_read_async` and `attention_async`.

    cache    uint8 [n_pages, kv_heads, kv_page_bytes(page_tokens, head_dim)], pages at any stride (a
             multiple of 16 bytes)
    table    int32 [n_seqs, max_pages]: the pages of each sequence's tokens, in order
    lens     int32 [n_seqs]: tokens of each sequence, those of the rows among them
    starts   int32 [n_seqs + 1]: where each sequence's rows begin among the `rows` rows of a
             call, and behind the last; a sequence's rows are its last tokens
    max_rows the most rows that a sequence has (default: `rows`)

    It holds addresses, checked once: their contents may change from call to call, and
    the tensors are kept alive with it. A layer with a cache of its own has a batch of its own."""

    def __init__(self, cache, table, lens, starts, rows: int, head_dim: int, max_rows: Optional[int] = None):
        if not (1 <= rows < 2 ** 31 and (max_rows is None or 1 <= max_rows < 2 ** 31)):   # (a field of the struct drops higher bits)
            _refuse("rows and max_rows: 1 to 2^31 - 1 is wanted")
        sh, st = cache.shape, cache.stride()
        if len(sh) != 3 or str(cache.dtype) != "torch.uint8" or st[2] != 1 or (st[1] != sh[2] and sh[1] != 1):
            _refuse("cache: uint8 [n_pages, kv_heads, bytes] with a page's heads consecutive is wanted")
        if not cache.is_cuda:
            _refuse("cache: not on the GPU")
        page = sh[2] * 4 // (5 * head_dim) if head_dim > 0 else 0
        if page < 1 or kv_page_bytes(page, head_dim) != sh[2]:
            _refuse(f"cache: {sh[2]} bytes are no page of head_dim {head_dim}")
        stride = st[0] if sh[0] > 1 else max(st[0], sh[1] * sh[2])
        tp, ts, tk = _mat(table, "table")
        if tk != _INT32:
            _refuse("table: int32 is wanted")
        n = int(table.shape[0])
        self.tensors = (cache, table, lens, starts)
        self.rows, self.kv_heads, self.head_dim, self.page_tokens = int(rows), int(sh[1]), int(head_dim), int(page)
        self.struct = _KVBatch(C.sizeof(_KVBatch), head_dim, sh[1], page, sh[0], table.shape[1], n, rows,
                               rows if max_rows is None else max_rows, 0, stride, ts, cache.data_ptr(), tp,
                               _vec(lens, n, "lens", _INT32), _vec(starts, n + 1, "starts", _INT32))
        self.ref = C.addressof(self.struct)
        self._kv_shape = (self.rows, self.kv_heads, self.head_dim)
        self.scale = self.head_dim ** -0.5


def attention_work_bytes(batch: KVBatch, q_heads: int) -> int:
    """Workspace bytes attention_async needs for the batch and q_heads heads of q."""
    need = int(lib().xl_attention_work_bytes(batch.ref, q_heads))
    if need == 2 ** 64 - 1:
        _refuse("a batch or a head count that attention does not take")
    return need


def pack_types(pack_dir: str, first_layer: int, n_layers: int, n_experts: int) -> np.ndarray:
    """Block types [n_layers, n_experts, 3] (gate, up, down) of a pack's layer window."""
    out = np.zeros((n_layers, n_experts, 3), np.int32)
    err = _Err()
    _check(lib().xl_pack_types(os.fsencode(pack_dir), first_layer, n_layers, n_experts, out.reshape(-1), C.byref(err)),
           err)
    return out


# ---- the lane ------------------------------------------------------------------
class Lane:
    """One context: a resident bank of n_layers x n_experts experts on one GPU.

    The *_async calls enqueue on `stream` (a raw HIP stream handle), by default
    on the context's own non-blocking stream, which does not wait for what PyTorch has
    enqueued on its streams (a fill of an output, say). Tensors passed to them must stay
    alive until that stream has run the call (`sync(stream)`): PyTorch's caching
    allocator hands a freed tensor's memory to the next allocation on its own
    current stream at once, so a temporary such as `torch.tensor(...).cuda()`
    passed inline and followed by another allocation before the sync can be
    overwritten while the kernel reads it. Passing
    `stream=torch.cuda.current_stream().cuda_stream` orders the call with
    PyTorch's own work and allocations on that stream."""

    def __init__(self, dim: int, ff: int, n_layers: int, n_experts: int, types: np.ndarray,
                 max_picks: int = 8, max_tokens: int = 0, device: int = 0, swiglu_limit: float = 0.0):
        L = lib()
        cfg = _Config(C.sizeof(_Config), device, dim, ff, n_layers, n_experts, max_picks, max_tokens,
                      float(swiglu_limit))
        ctx = _P()
        err = _Err()
        _check(L.xl_open(ABI_VERSION, C.byref(cfg), C.byref(ctx), C.byref(err)), err)
        self._ctx = ctx
        self._err = _Err()   # of the calls that a decode loop makes many of (a context has one caller at a time)
        self._errp = C.byref(self._err)
        self._rotary = (C.c_uint64 * (_ROTARY_BYTES // 8))()
        self.dim, self.ff, self.n_layers, self.n_experts, self.max_picks = dim, ff, n_layers, n_experts, max_picks
        types = np.ascontiguousarray(types, dtype=np.int32).reshape(n_layers, n_experts, 3)
        self.types = types
        self._call("xl_bank_create", types.reshape(-1))

    # -- plumbing
    def _call(self, name: str, *args) -> None:
        err = _Err()
        _check(getattr(lib(), name)(self._ctx, *args, C.byref(err)), err)

    def close(self) -> None:
        if getattr(self, "_ctx", None):
            lib().xl_close(self._ctx)
            self._ctx = None

    def __del__(self):
        # At interpreter shutdown the HIP runtime (and torch's hold on it) may
        # already be torn down; process exit releases the device memory anyway,
        # so the context is left to it rather than closed into a dead runtime.
        if sys.is_finalizing():
            return
        try:
            self.close()
        except Exception:
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    # -- bank
    def generate(self, seed: int) -> None:
        self._call("xl_bank_generate", C.c_uint64(seed))

    def load_pack(self, pack_dir: str, first_layer: int = 0) -> None:
        """Uploads every expert of pack layers first_layer .. + n_layers - 1."""
        self._call("xl_bank_load_pack", os.fsencode(pack_dir), first_layer)

    def upload(self, layer: int, expert: int, role: int, aos: np.ndarray) -> None:
        aos = np.ascontiguousarray(aos, dtype=np.uint8)
        self._call("xl_bank_upload", layer, expert, role, aos.ctypes.data, C.c_uint64(aos.size))

    def download(self, layer: int, expert: int, role: int) -> np.ndarray:
        t = int(self.types[layer, expert, role])
        n, k = (self.ff, self.dim) if role < 2 else (self.dim, self.ff)
        out = np.zeros(n * (k // 256) * BLOCK_BYTES[t], dtype=np.uint8)
        self._call("xl_bank_download", layer, expert, role, out.ctypes.data, C.c_uint64(out.size))
        return out

    def info(self) -> dict:
        bi = _BankInfo()
        lib().xl_bank_info_get(self._ctx, C.byref(bi))
        return {f: getattr(bi, f) for f, _ in _BankInfo._fields_}

    # -- WarmRedirect surface
    def warm_contains(self, layer: int, e: int) -> bool:
        return bool(lib().xl_contains(self._ctx, layer, e))

    def warm_grouped(self) -> bool:
        return True

    def warm_compute(self, layer: int, e: int, x: np.ndarray) -> np.ndarray:
        y = np.zeros(self.dim, dtype=np.float32)
        self._call("xl_expert_forward", layer, e, np.ascontiguousarray(x, dtype=np.float32), y)
        return y

    def warm_compute_many(self, layer: int, ids: Sequence[int], x: np.ndarray) -> list:
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        ys = np.zeros((ids.size, self.dim), dtype=np.float32)
        self._call("xl_experts_forward", layer, ids, ids.size, np.ascontiguousarray(x, dtype=np.float32),
                   ys.reshape(-1))
        return [ys[i] for i in range(ids.size)]

    def layer_forward(self, layer: int, ids: Sequence[int], weights: Sequence[float], x: np.ndarray,
                      shared: Optional[np.ndarray] = None) -> np.ndarray:
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        w = np.ascontiguousarray(weights, dtype=np.float32)
        out = np.zeros(self.dim, dtype=np.float32)
        sh = None if shared is None else np.ascontiguousarray(shared, dtype=np.float32)
        self._call("xl_layer_forward", layer, ids, w, ids.size, np.ascontiguousarray(x, dtype=np.float32),
                   None if sh is None else sh.ctypes.data, out)
        return out

    def grouped_forward(self, layer: int, ids: np.ndarray, weights: np.ndarray, x: np.ndarray,
                        shared: Optional[np.ndarray] = None) -> np.ndarray:
        """T tokens at once: ids, weights [T, k]; x, shared [T, dim] -> out [T, dim]."""
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        T, k = ids.shape
        w = np.ascontiguousarray(weights, dtype=np.float32).reshape(T, k)
        x = np.ascontiguousarray(x, dtype=np.float32).reshape(T, self.dim)
        sh = None if shared is None else np.ascontiguousarray(shared, dtype=np.float32).reshape(T, self.dim)
        out = np.zeros((T, self.dim), dtype=np.float32)
        self._call("xl_grouped_forward", layer, T, k, ids.reshape(-1), w.reshape(-1), x.reshape(-1),
                   None if sh is None else sh.ctypes.data, out.reshape(-1))
        return out

    def layer_forward_per32(self, layer: int, ids: Sequence[int], x: np.ndarray,
                            weights: Optional[Sequence[float]] = None, shared: Optional[np.ndarray] = None):
        """per32 layer (the reference's HIP lane arithmetic): returns (y [k, dim]
        per-pick down outputs, out [dim] their combine, or None without weights)."""
        ids = np.ascontiguousarray(ids, dtype=np.int32)
        y = np.zeros((ids.size, self.dim), dtype=np.float32)
        out = None if weights is None else np.zeros(self.dim, dtype=np.float32)
        w = None if weights is None else np.ascontiguousarray(weights, dtype=np.float32)
        sh = None if shared is None else np.ascontiguousarray(shared, dtype=np.float32)
        self._call("xl_layer_forward_per32", layer, ids, None if w is None else w.ctypes.data, ids.size,
                   np.ascontiguousarray(x, dtype=np.float32), None if sh is None else sh.ctypes.data, y.ctypes.data,
                   None if out is None else out.ctypes.data)
        return y, out

    def expert_trace(self, layer: int, e: int, x: np.ndarray) -> dict:
        ff, dim = self.ff, self.dim
        g = np.zeros(ff, np.float32); u = np.zeros(ff, np.float32); h = np.zeros(ff, np.float32)
        q8h = np.zeros((ff // 256) * 292, np.uint8); y = np.zeros(dim, np.float32)
        self._call("xl_expert_trace", layer, e, np.ascontiguousarray(x, dtype=np.float32), g.ctypes.data,
                   u.ctypes.data, h.ctypes.data, q8h.ctypes.data, y.ctypes.data)
        return {"g": g, "u": u, "h": h, "q8h": q8h, "y": y}

    # -- device-resident (torch CUDA tensors)
    def layer_forward_async(self, layer: int, ids, w, x, out, shared=None, stream=None) -> None:
        self._call("xl_layer_forward_async", layer, _ptr(ids), _ptr(w), int(ids.numel()), _ptr(x), _ptr(shared),
                   _ptr(out), None if stream is None else int(stream))

    def layer_forward_exact_async(self, layer: int, ids, w, x, out, shared=None, stream=None) -> None:
        """xl_layer_forward_async with every float in the reference CPU lane's
        order (q8k_core.hpp:76-95): the reference's output bit for bit."""
        self._call("xl_layer_forward_exact_async", layer, _ptr(ids), _ptr(w), int(ids.numel()), _ptr(x), _ptr(shared),
                   _ptr(out), None if stream is None else int(stream))

    def layer_forward_prenorm_async(self, layer: int, ids, w, h, mix, norm_w, x, out, eps: float = 1e-6, shared=None,
                                    stream=None) -> None:
        """The layer on x = hc_pre_norm(h, mix, norm_w) of one token: h [H, dim]
        (or [1, H, dim]), mix [8], norm_w [dim] or None; x [dim] receives the
        normalized input (one launch when H == 1 and the layer has a streaming
        instance: the norm runs in its prologue)."""
        H = int(h.shape[-2]) if h.dim() >= 2 else 1
        self._call("xl_layer_forward_prenorm_async", layer, _ptr(ids), _ptr(w), int(ids.numel()), _ptr(h), H,
                   _ptr(mix), _ptr(norm_w), float(eps), _ptr(x), _ptr(shared), _ptr(out),
                   None if stream is None else int(stream))

    def layer_forward_post_async(self, layer: int, ids, w, x, out, res, post, comb, post_out, shared=None,
                                 stream=None) -> None:
        """The layer (out [dim], with shared added last) and hc_post of its output
        for one token: res and post_out [H, dim] (or [1, H, dim]; post_out may be
        res), post [8], comb [64]. One launch when the layer has a streaming
        instance: each workgroup applies hc_post to the rows it combines."""
        H = int(res.shape[-2]) if res.dim() >= 2 else 1
        self._call("xl_layer_forward_post_async", layer, _ptr(ids), _ptr(w), int(ids.numel()), _ptr(x), _ptr(shared),
                   _ptr(out), _ptr(res), _ptr(post), _ptr(comb), H, _ptr(post_out),
                   None if stream is None else int(stream))

    def moe_block_async(self, layer: int, ids, w, x, types, gate, up, down, ff: int, work, res, post, comb, out,
                        post_out, stream=None) -> None:
        """The MoE block of one token: the routed layer, the shared-expert FFN
        (types, gate, up, down, ff as shared_forward_async) added last, and
        hc_post of the sum: out [dim], res and post_out [H, dim] (post_out may be
        res), post [8], comb [64]; work >= shared_work_bytes(dim, ff, 1). The same
        bits as shared_forward_async then layer_forward_post_async with that row."""
        H = int(res.shape[-2]) if res.dim() >= 2 else 1
        self._call("xl_moe_block_async", layer, _ptr(ids), _ptr(w), int(ids.numel()), _ptr(x), int(types[0]),
                   _ptr(gate), int(types[1]), _ptr(up), int(types[2]), _ptr(down), ff, _ptr(work),
                   int(work.numel() * work.element_size()), _ptr(res), _ptr(post), _ptr(comb), H, _ptr(out),
                   _ptr(post_out), None if stream is None else int(stream))

    def layer_trace_async(self, layer: int, ids, w, x, out, q8x=None, q8h=None, h=None, ints=None, shared=None,
                          stream=None, y=None) -> int:
        """The single-launch layer call with its own Q8_K(x) / Q8_K(h) blocks (uint8
        tensors of 292-byte blocks), h, block integers and per-pick rows (y, k x dim,
        as its combine read them) written out; returns the kernel that ran (1
        streaming, 3 all-types)."""
        kern = _I32()
        self._call("xl_layer_trace_async", layer, _ptr(ids), _ptr(w), int(ids.numel()), _ptr(x), _ptr(shared),
                   _ptr(out), _ptr(q8x), _ptr(q8h), _ptr(h), _ptr(ints), _ptr(y), C.byref(kern),
                   None if stream is None else int(stream))
        return kern.value

    def grouped_trace_async(self, layer: int, ids, w, x, out, q8x=None, q8h=None, h=None, ints=None, shared=None,
                            stream=None, y=None) -> None:
        T, k = int(ids.shape[0]), int(ids.shape[1])
        self._call("xl_grouped_trace_async", layer, T, k, _ptr(ids), _ptr(w), _ptr(x), _ptr(shared), _ptr(out),
                   _ptr(q8x), _ptr(q8h), _ptr(h), _ptr(ints), _ptr(y), None if stream is None else int(stream))

    def combine_async(self, ids, w, rows, out, shared=None, stream=None) -> None:
        """xl_combine_async: out = fixed-order combine of rows [k, dim] (device tensors)."""
        k, dim = int(rows.shape[0]), int(rows.shape[1])
        self._call("xl_combine_async", _ptr(ids), _ptr(w), k, _ptr(rows), dim, _ptr(shared), _ptr(out),
                   None if stream is None else int(stream))

    def grouped_forward_async(self, layer: int, ids, w, x, out, shared=None, stream=None) -> None:
        """ids, w: [T, k] device tensors; x, out (and shared): [T, dim]."""
        T, k = int(ids.shape[0]), int(ids.shape[1])
        self._call("xl_grouped_forward_async", layer, T, k, _ptr(ids), _ptr(w), _ptr(x), _ptr(shared), _ptr(out),
                   None if stream is None else int(stream))

    def route_async(self, logits, k: int, ids, w, scale: float = 1.0, bias=None, stream=None) -> None:
        """logits: [T, n] device tensor; ids (int32), w: [T, k] device tensors."""
        T, n = int(logits.shape[0]), int(logits.shape[1])
        self._call("xl_route_async", _ptr(logits), T, int(logits.stride(0)), _ptr(bias), n, k, float(scale), _ptr(ids),
                   _ptr(w), None if stream is None else int(stream))

    def layer_forward_routed_async(self, layer: int, logits, k: int, x, out, scale: float = 1.0, bias=None,
                                   shared=None, stream=None) -> None:
        self._call("xl_layer_forward_routed_async", layer, _ptr(logits), _ptr(bias), k, float(scale), _ptr(x),
                   _ptr(shared), _ptr(out), None if stream is None else int(stream))

    def grouped_forward_routed_async(self, layer: int, logits, k: int, x, out, scale: float = 1.0, bias=None,
                                     shared=None, stream=None) -> None:
        self._call("xl_grouped_forward_routed_async", layer, int(logits.shape[0]), _ptr(logits), _ptr(bias), k,
                   float(scale), _ptr(x), _ptr(shared), _ptr(out), None if stream is None else int(stream))

    def sync(self, stream=None) -> None:
        self._call("xl_sync", None if stream is None else int(stream))

    def profile_begin(self, max_calls: int) -> None:
        self._call("xl_profile_begin", max_calls)

    def profile_end(self) -> dict:
        """Per-stage total milliseconds over the profiled calls: {name: ms}, calls."""
        ms = np.zeros(8, np.float32)
        ns, nc = _I32(), _I32()
        names = C.create_string_buffer(256)
        self._call("xl_profile_end", ms, 8, C.byref(ns), C.byref(nc), names, 256)
        keys = names.value.decode().split(",") if ns.value else []
        return {"calls": nc.value, "stages": {k: float(ms[i]) for i, k in enumerate(keys)}}

    def profile_timeline(self) -> np.ndarray:
        """Per-wave phase stamps (100 MHz) of the last profiled single-launch call: [waves, 32]."""
        out = np.zeros(1 << 16, np.uint64)
        n = _I32()
        self._call("xl_profile_timeline", out, out.size, C.byref(n))
        return out[: n.value].reshape(-1, 32)

    def debug_set_launch_count(self, launches: int) -> None:
        """Sets the single-launch kernels' launch counters (epoch / parity) as if
        `launches` launches had run: for testing their wrap at 2^32."""
        self._call("xl_debug_set_launch_count", C.c_uint32(launches & 0xFFFFFFFF))

    LAUNCH_KINDS = ("stream", "alltypes", "separate", "routed", "prenorm", "exact", "post", "block")   # XL_LAUNCH_* order

    def launch_counts(self) -> dict:
        """Layer calls so far by how they ran ({kind: count}, XL_LAUNCH_* kinds):
        which launch served a call (e.g. a routed call routed inside its launch)."""
        out = np.zeros(len(self.LAUNCH_KINDS), np.int64)
        self._call("xl_debug_launch_counts", out, out.size)
        return dict(zip(self.LAUNCH_KINDS, (int(v) for v in out)))

    def quantize_q8k_async(self, x, rows: int, k: int, q8k_out, stream=None) -> None:
        self._call("xl_quantize_q8k_async", _ptr(x), rows, k, _ptr(q8k_out), None if stream is None else int(stream))

    def layer_forward_per32_async(self, layer: int, ids, x, y, w=None, out=None, shared=None, stream=None) -> None:
        self._call("xl_layer_forward_per32_async", layer, _ptr(ids), _ptr(w), int(ids.numel()), _ptr(x), _ptr(shared),
                   _ptr(y), _ptr(out), None if stream is None else int(stream))

    def quantize_per32_async(self, x, rows: int, k: int, q, d, stream=None) -> None:
        self._call("xl_quantize_per32_async", _ptr(x), rows, k, _ptr(q), _ptr(d), None if stream is None else int(stream))

    def matvec_per32_async(self, t: int, planar, n: int, k: int, q, d, y, stream=None) -> None:
        self._call("xl_matvec_per32_async", t, _ptr(planar), n, k, _ptr(q), _ptr(d), _ptr(y),
                   None if stream is None else int(stream))

    def shared_forward_async(self, types, gate, up, down, ff: int, x, out, work, stream=None) -> None:
        """Shared-expert FFN of T tokens: x, out [T, dim] device tensors; gate, up,
        down raw ggml (dense) or planar (IQ) device bytes; work >= shared_work_bytes."""
        T = int(x.numel()) // self.dim
        self._call("xl_shared_forward_async", int(types[0]), _ptr(gate), int(types[1]), _ptr(up), int(types[2]),
                   _ptr(down), ff, T, _ptr(x), _ptr(out), _ptr(work), int(work.numel() * work.element_size()),
                   None if stream is None else int(stream))

    def shared_forward_noalloc(self, types, gate, up, down, ff: int, x, out, stream=None) -> None:
        """The shared-expert FFN with its intermediates in the library's static
        device scratch (no workspace, no allocation): x, out [T, dim]."""
        T = int(x.numel()) // self.dim
        self._call("xl_shared_forward_noalloc", int(types[0]), _ptr(gate), int(types[1]), _ptr(up), int(types[2]),
                   _ptr(down), ff, T, _ptr(x), _ptr(out), None if stream is None else int(stream))

    def hc_pre_norm_async(self, h, mix, w, x, eps: float = 1e-6, stream=None) -> None:
        """h [T, H, D], mix [T, 8], w [D] or None, x [T, D] device tensors."""
        T, H, D = (int(v) for v in h.shape)
        self._call("xl_hc_pre_norm_async", _ptr(h), _ptr(mix), _ptr(w), D, H, T, float(eps), _ptr(x),
                   None if stream is None else int(stream))

    def hc_post_async(self, y, res, post, comb, out, stream=None) -> None:
        """y [T, D], res / out [T, H, D], post [T, 8], comb [T, 64] device tensors."""
        T, H, D = (int(v) for v in res.shape)
        self._call("xl_hc_post_async", _ptr(y), _ptr(res), _ptr(post), _ptr(comb), D, H, T, _ptr(out),
                   None if stream is None else int(stream))

    def route_scored_async(self, logits, k: int, ids, w, score: str = "softmax", bias=None, groups: int = 1,
                           top_groups: int = 1, group_keys: int = 1, renorm: bool = True, scale: float = 1.0,
                           stream=None) -> None:
        """Router over softmax or sigmoid scores: logits [T, n] (f32, f16 or bf16; -inf
        masks an expert), bias [n] float32 added to the scores for the choice only,
        `top_groups` of `groups` expert groups by the sum of their `group_keys`
        largest keys; ids (int32) and w [T, k]."""
        if score not in SCORES:
            _refuse(f"score must be one of {sorted(SCORES)}")
        lp, stride, _ = _mat(logits, "logits")
        T, n = logits.shape
        _check(lib().xl_route_scored_async(
            self._ctx, lp, _act(logits, "logits"), T, stride, _vec(bias, n, "bias"), n, SCORES[score], groups, top_groups,
            group_keys, int(k), bool(renorm), float(scale), _vec(ids, T * k, "ids", _INT32), _vec(w, T * k, "w"),
            None if stream is None else int(stream), self._errp), self._err)

    def block_norm_async(self, res, y=None, post_w=None, gate=None, alpha: float = 1.0, pre_w=None, eps: float = 1e-6,
                         res_out=None, x=None, q=None, q_scale=None, stream=None) -> None:
        """Between two blocks: a = y (RMS-normed with post_w [D]); r = alpha * res +
        gate * a; x = RMS norm of r with pre_w [D]. res, y [T, D] (one may be None),
        gate [T, D], [D] or None; outputs res_out (r, as res), x (as y) [T, D], and q
        int8 [T, D] with q_scale [T]: x quantized, for linear_i8_async."""
        some = y if res is None else res
        if some is None:
            _refuse("res or y is wanted")
        shape = some.shape
        yp, ys, yk = _mat(y, "y", shape)
        rp, rs, rk = _mat(res, "res", shape)
        op, os_, ok = _mat(res_out, "res_out", shape)
        xp, xs, xk = _mat(x, "x", shape)
        qp, qs, qk = _mat(q, "q", shape)
        T, D = shape
        gp, gs, gk = None, 0, -1
        if gate is not None:
            if gate.dim() == 1:
                gk = _KINDS[gate.dtype]
                gp = _vec(gate, D, "gate", gk)
            else:
                gp, gs, gk = _mat(gate, "gate", shape)
        # -1: not given
        kind = yk if yk >= 0 else xk if xk >= 0 else gk
        rkind = rk if rk >= 0 else ok
        if kind not in (yk, xk, gk) or (yk >= 0 and yk != kind) or (xk >= 0 and xk != kind) or (gk >= 0 and gk != kind) \
                or (ok >= 0 and ok != rkind):
            _refuse("y, x and gate have one element type, res and res_out one")
        if kind >= _INT8 or rkind >= _INT8 or min(yk, xk, gk, rk, ok) < -1:
            _refuse("y, x, gate, res and res_out: element type not taken here")
        if q is not None and qk != _INT8:
            _refuse("q must be int8")
        if rkind < 0:
            rkind = 0
        _check(lib().xl_block_norm_async(
            self._ctx, yp, ys, rp, rs, gp, gs, _vec(post_w, D, "post_w"), _vec(pre_w, D, "pre_w"), T, D,
            kind if kind >= 0 else rkind, rkind, float(alpha), float(eps), op, os_, xp, xs, qp, qs,
            _vec(q_scale, T, "q_scale"), None if stream is None else int(stream), self._errp), self._err)

    def quantize_rows_async(self, x, q, scale, stream=None) -> None:
        """x [T, K] (f32, f16 or bf16) to int8 q [T, K] (16-byte aligned rows) with scale [T]."""
        xp, xs, _ = _mat(x, "x")
        T, K = shape = x.shape
        qp, qs, qk = _mat(q, "q", shape)
        if qk != _INT8:
            _refuse("q must be int8")
        _check(lib().xl_quantize_rows_async(self._ctx, xp, _act(x, "x"), T, K, xs, qp, qs, _vec(scale, T, "scale"),
                                            None if stream is None else int(stream), self._errp), self._err)

    def linear_i8_async(self, x, w, w_scale, out, x_scale=None, up=None, up_scale=None, limit: float = 0.0, work=None,
                        stream=None) -> None:
        """out [T, N] = x [T, K] times int8 w [N, K] (16-byte aligned rows) with a scale
        for each token and channel; x int8 with x_scale [T], or float (quantized by
        the call). With up, up_scale: SwiGLU of the products with w (gate) and up.
        work: linear_i8_work_bytes(T, K, N, gated) bytes."""
        xp, xs, kind = _mat(x, "x")
        wp, ws, wk = _mat(w, "w")
        T, K = x.shape
        shape = w.shape
        N = shape[0]
        if shape[1] != K or wk != _INT8:
            _refuse("w: int8 [N, K] is wanted")
        op, os_, _ = _mat(out, "out", (T, N))
        up_, us, uk = _mat(up, "up", shape)
        if up is not None and (uk != _INT8 or us != ws):
            _refuse("up: int8 with w's shape and stride is wanted")
        if work is None or not (work.is_cuda and work.is_contiguous()):
            _refuse("work: a contiguous GPU buffer is wanted")
        if not 0 <= kind <= _INT8:
            _refuse(f"x: element type {x.dtype} not taken here")
        _check(lib().xl_linear_i8_async(
            self._ctx, xp, kind, _vec(x_scale, T, "x_scale"), xs, T, K, wp, _vec(w_scale, N, "w_scale"), up_,
            _vec(up_scale, N, "up_scale"), ws, N, float(limit), op, _act(out, "out"), os_, work.data_ptr(), work.nbytes,
            None if stream is None else int(stream), self._errp), self._err)

    def kv_write_async(self, batch: KVBatch, k, v, q=None, q_out=None, freqs=None, positions=None, sections=None,
                       interleaved: bool = False, stream=None) -> None:
        """Rows of k and v [rows, kv_heads, head_dim] into the batch's cache; with freqs
        [n] (float32, angles a position), k and q [rows, q_heads, head_dim] are turned first, q
        into q_out. positions: int32 [axes, rows] or [rows] (None: positions in the sequences);
        sections: how many of the frequencies go by each axis."""
        kp, ks, kind = _heads(k, "k", batch._kv_shape)
        vp, vs, vk = _heads(v, "v", batch._kv_shape)
        if not 0 <= kind < _INT8 or vk != kind:
            _refuse("k and v must have one element type, f32, f16 or bf16")
        qp, qs, heads, op, os_ = None, 0, 0, None, 0
        if q is not None:
            if q_out is None:
                _refuse("q needs q_out")
            shape = q.shape
            if len(shape) != 3 or shape[0] != batch.rows or shape[2] != batch.head_dim:
                _refuse(f"q: shape {tuple(shape)} where [{batch.rows}, q_heads, {batch.head_dim}] is wanted")
            heads = shape[1]
            qp, qs, qk = _heads(q, "q", shape)
            op, os_, ok = _heads(q_out, "q_out", shape)
            if qk != kind or ok != kind:
                _refuse("q and q_out must have k's element type")
        elif q_out is not None:
            _refuse("q_out without q")
        rotary = None
        if freqs is not None:
            n = freqs.numel()
            pp, pstride, axes = None, 0, 1
            if positions is not None:
                if positions.dim() == 1:
                    pp, pstride = _vec(positions, batch.rows, "positions", _INT32), batch.rows
                else:
                    axes = positions.shape[0]
                    pp, pstride, pk = _mat(positions, "positions", (axes, batch.rows))
                    if pk != _INT32:
                        _refuse("positions: int32 is wanted")
            parts = (n,) if sections is None else sections
            if len(parts) != axes or not 1 <= axes <= 3:
                _refuse("a section for each of one to three axes is wanted")
            fp = _vec(freqs, n, "freqs")
            t, h, w = (*parts, 0, 0)[:3]
            try:   # (0.4 us less than a new _Rotary)
                _ROTARY.pack_into(self._rotary, 0, _ROTARY_BYTES, n, axes, bool(interleaved), t, h, w, 0, pstride, fp, pp or 0)
            except struct.error:
                _refuse("sections: whole numbers of 32 bits are wanted")
            rotary = C.addressof(self._rotary)
        elif q is not None or positions is not None or sections is not None:
            _refuse("q, positions and sections go with freqs")
        rc = lib().xl_kv_write_async(self._ctx, batch.ref, kp, ks, vp, vs, kind, rotary,
                                     qp, qs, heads, op, os_, None if stream is None else int(stream), self._errp)
        if rc:
            _check(rc, self._err)

    def kv_read_async(self, batch: KVBatch, k, v, stream=None) -> None:
        """What the batch's cache holds at its rows' positions, into k and v [rows, kv_heads, head_dim]."""
        kp, ks, kind = _heads(k, "k", batch._kv_shape)
        vp, vs, vk = _heads(v, "v", batch._kv_shape)
        if not 0 <= kind < _INT8 or vk != kind:
            _refuse("k and v must have one element type, f32, f16 or bf16")
        rc = lib().xl_kv_read_async(self._ctx, batch.ref, kp, ks, vp, vs, kind, None if stream is None else int(stream), self._errp)
        if rc:
            _check(rc, self._err)

    def attention_async(self, batch: KVBatch, q, out, scale: Optional[float] = None, window: int = 0, softcap: float = 0.0,
                        work=None, stream=None) -> None:
        """out [rows, q_heads, head_dim] = attention of the rows of q over the batch's cache (f16 or
        bf16): tokens up to each row's own, with window > 0 the last `window` of them (pages below every
        row's window may be gone, their entries of the table anything), softcap > 0 (up to 16384): scores
        through softcap * tanh(score / softcap). scale: 1 / sqrt(head_dim) by default. work:
        attention_work_bytes(batch, q_heads) bytes (None where that is 0)."""
        shape = q.shape
        if len(shape) != 3 or shape[0] != batch.rows or shape[2] != batch.head_dim:
            _refuse(f"q: shape {tuple(shape)} where [{batch.rows}, q_heads, {batch.head_dim}] is wanted")
        heads = shape[1]
        qp, qs, kind = _heads(q, "q", shape)
        op, os_, ok = _heads(out, "out", shape)
        if kind not in (1, 2) or ok != kind:
            _refuse("q and out must have one element type, f16 or bf16")
        wp, wb = None, 0
        if work is not None:
            if not (work.is_cuda and work.is_contiguous()):
                _refuse("work: a contiguous GPU buffer is wanted")
            wb = work.nbytes
            wp = work.data_ptr() if wb else None
        if not 0 <= window < 2 ** 31:
            _refuse("window: 0 to 2^31 - 1 is wanted")
        rc = lib().xl_attention_async(self._ctx, batch.ref, qp, qs, heads, kind, batch.scale if scale is None else scale, window,
                                      softcap, op, os_, wp, wb, None if stream is None else int(stream), self._errp)
        if rc:
            _check(rc, self._err)

    def swiglu_async(self, g, u, h, limit: float = 0.0, stream=None) -> None:
        self._call("xl_swiglu_async", _ptr(g), _ptr(u), int(g.numel()), float(limit), _ptr(h),
                   None if stream is None else int(stream))

    def matvec_async(self, t: int, planar, n: int, k: int, x, y, partials=None, stream=None) -> None:
        self._call("xl_matvec_async", t, _ptr(planar), n, k, _ptr(x), _ptr(y), _ptr(partials),
                   None if stream is None else int(stream))
