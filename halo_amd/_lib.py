"""ctypes bindings of libhalo_mi355x.so (the C ABI in include/halo_mi355x.h).

Pointer arguments are plain integers (device addresses, e.g. ``tensor.data_ptr()``) and
``stream`` is a hipStream_t as an integer (0 = null stream). Functions taking torch tensors
validate dtype/device and pass ``torch.cuda.current_stream()`` unless a stream is given.
"""
from __future__ import annotations

import ctypes
import enum
import functools
import struct
import typing
from pathlib import Path

_PKG = Path(__file__).resolve().parent
_LIB_PATH = _PKG / "libhalo_mi355x.so"

SLAB_ROWS = 64


class DType(enum.IntEnum):
    """ggml type ids (include/halo/tensor/dtype.h:18-49 of the reference)."""

    F32 = 0
    F16 = 1
    Q4_0 = 2
    Q4_1 = 3
    Q5_0 = 6
    Q5_1 = 7
    Q8_0 = 8
    Q2_K = 10
    Q3_K = 11
    Q4_K = 12
    Q5_K = 13
    Q6_K = 14
    IQ4_NL = 20
    IQ3_S = 21
    IQ4_XS = 23
    BF16 = 30


class Layout(enum.IntEnum):
    GGUF = 0
    SLAB = 1


class Variant(enum.IntEnum):
    DEFAULT = 0
    GGUF_REF = 1
    SLAB_GEMV = 2
    SLAB_GEMM_BF16 = 3
    SLAB_AUTO = 4
    SLAB_GEMM_BF16_M512 = 5
    SLAB_GEMV_VALU = 6
    SLAB_GEMM_BF16_SMALL_M = 7
    SLAB_GEMM_EXACT_SMALL_M = 8
    SLAB_GEMM_EXACT_INVARIANT = 9


class ErrorCode(enum.IntEnum):
    """Status codes; names follow halo::ErrorCode (include/halo/core/error.h:13-24)."""

    Ok = 0
    Kernel = 1
    Unsupported = 2
    Config = 3
    Memory = 4
    Device = 5


class HaloError(RuntimeError):
    def __init__(self, code: int, message: str):
        self.code = ErrorCode(code)
        super().__init__(f"{self.code.name.upper()}_ERROR: {message}")


_BLOCK = {DType.F32: (1, 4), DType.F16: (1, 2), DType.BF16: (1, 2), DType.Q4_0: (32, 18), DType.Q4_1: (32, 20),
          DType.Q5_0: (32, 22), DType.Q5_1: (32, 24), DType.Q8_0: (32, 34), DType.Q2_K: (256, 84),
          DType.Q3_K: (256, 110), DType.Q4_K: (256, 144), DType.Q5_K: (256, 176), DType.Q6_K: (256, 210),
          DType.IQ4_NL: (32, 18), DType.IQ3_S: (256, 110), DType.IQ4_XS: (256, 136)}


def block_elems(t: int) -> int:
    """Weights per block; 0 for a type this backend does not handle."""
    return _BLOCK.get(int(t), (0, 0))[0]


def block_bytes(t: int) -> int:
    return _BLOCK.get(int(t), (0, 0))[1]


class _GemvParams(ctypes.Structure):
    _fields_ = [
        ("type", ctypes.c_uint32),
        ("layout", ctypes.c_uint32),
        ("w", ctypes.c_void_p),
        ("w_stride", ctypes.c_uint64),
        ("x", ctypes.c_void_p),
        ("x_stride", ctypes.c_uint64),
        ("y", ctypes.c_void_p),
        ("y_stride", ctypes.c_uint64),
        ("rows", ctypes.c_uint32),
        ("cols", ctypes.c_uint32),
        ("n_vec", ctypes.c_uint32),
        ("variant", ctypes.c_uint32),
        ("norm_w", ctypes.c_void_p),
        ("norm_eps", ctypes.c_float),
    ]


class _GateUpParams(ctypes.Structure):
    _fields_ = [
        ("type", ctypes.c_uint32),
        ("layout", ctypes.c_uint32),
        ("w_gate", ctypes.c_void_p),
        ("w_up", ctypes.c_void_p),
        ("x", ctypes.c_void_p),
        ("x_stride", ctypes.c_uint64),
        ("out", ctypes.c_void_p),
        ("out_stride", ctypes.c_uint64),
        ("rows", ctypes.c_uint32),
        ("cols", ctypes.c_uint32),
        ("n_vec", ctypes.c_uint32),
        ("variant", ctypes.c_uint32),
        ("norm_w", ctypes.c_void_p),
        ("norm_eps", ctypes.c_float),
    ]


class _GemvSegment(ctypes.Structure):
    _fields_ = [("type", ctypes.c_uint32), ("w", ctypes.c_void_p), ("rows", ctypes.c_uint32), ("y", ctypes.c_void_p),
                ("y_stride", ctypes.c_uint64)]


class _GemvGroupParams(ctypes.Structure):
    _fields_ = [
        ("segs", ctypes.POINTER(_GemvSegment)),
        ("n_segs", ctypes.c_uint32),
        ("x", ctypes.c_void_p),
        ("x_stride", ctypes.c_uint64),
        ("cols", ctypes.c_uint32),
        ("n_vec", ctypes.c_uint32),
        ("norm_w", ctypes.c_void_p),
        ("norm_eps", ctypes.c_float),
    ]


class _LmHeadParams(ctypes.Structure):
    _fields_ = [
        ("gemv", _GemvParams),
        ("result", ctypes.c_void_p),
        ("valid_rows", ctypes.c_uint32),
        ("ids", ctypes.c_void_p),
        ("ids_slots", ctypes.c_void_p),
        ("ids_scatter", ctypes.c_void_p),
        ("ids_scatter_len", ctypes.c_uint64),
    ]


class _UploadPart(ctypes.Structure):
    _fields_ = [("src", ctypes.c_void_p), ("src_stride", ctypes.c_uint64), ("rows", ctypes.c_uint32)]


class _UploadTensor(ctypes.Structure):
    _fields_ = [
        ("type", ctypes.c_uint32),
        ("cols", ctypes.c_uint32),
        ("parts", ctypes.POINTER(_UploadPart)),
        ("n_parts", ctypes.c_uint32),
        ("dst", ctypes.c_void_p),
    ]


class _GetRowsParams(ctypes.Structure):
    _fields_ = [
        ("type", ctypes.c_uint32),
        ("layout", ctypes.c_uint32),
        ("table", ctypes.c_void_p),
        ("table_stride", ctypes.c_uint64),
        ("n_rows", ctypes.c_uint32),
        ("cols", ctypes.c_uint32),
        ("ids", ctypes.c_void_p),
        ("n_ids", ctypes.c_uint32),
        ("out", ctypes.c_void_p),
        ("out_stride", ctypes.c_uint64),
        ("status", ctypes.c_void_p),
        ("status_keep", ctypes.c_uint32),
    ]


class _RopeScaling(ctypes.Structure):
    _fields_ = [("kind", ctypes.c_uint32), ("scale", ctypes.c_double), ("context", ctypes.c_double),
                ("beta_fast", ctypes.c_double), ("beta_slow", ctypes.c_double)]


class _Layout:
    """A parameter block of the C ABI as one struct.pack: these calls are made hundreds of times a step, and a decode step's
    kernels take less time than filling a ctypes.Structure field by field (a rope call of one token: 7.0 us, packed 5.6)."""

    def __init__(self, *parts: str):
        packer = struct.Struct("@" + "".join(parts))
        self.pack_into, self.buffer = packer.pack_into, ctypes.c_char * packer.size

    def __call__(self, *values):
        out = self.buffer()
        try:
            self.pack_into(out, 0, *values)
        except (struct.error, OverflowError) as e:
            raise HaloError(ErrorCode.Kernel, f"an argument is out of range or of the wrong kind: {e}") from None
        return out


# Members in the order of halo_mi355x.h, padded as C pads them (P: pointer, Q: uint64, I: uint32, f: float).
_ROWS = "PQQ"  # data, stride, head stride
_CACHE = "P5I4x"  # pool, n_pages, n_layers, n_kv_heads, head_dim, block_tokens
_BATCH = "PQI4xPP4I"  # tables, stride, width, kv_lens, row_starts, n_seqs, n_rows, max_rows, max_kv
_STATUS = "PI4x"  # status, status_keep
_ROPE_PART = _ROWS + _ROWS + "I4x"  # in, out, n_heads
_rope_params = _Layout(_ROPE_PART, _ROPE_PART, "IIPIIIIPPf4x")  # the two parts, then halo_mi_rope_params
_POINTER = struct.Struct("@P")
_ROPE_PARAMS_AT = 2 * struct.calcsize("@" + _ROPE_PART)
_kv_write_params = _Layout("I4x", _CACHE, "I4x", _BATCH, _ROWS, _ROWS, _STATUS)
_kv_read_params = _Layout(_CACHE, "I4x", _BATCH, _ROWS, _ROWS, _STATUS)
_attention_block = _Layout("I4x", _CACHE, "I4x", _BATCH, _ROWS, _ROWS, "IfI4xPQ", _STATUS)
_cache_block = _Layout(_CACHE)
_norm_rope_params = _Layout(_ROPE_PART, _ROPE_PART, "IIPIIIIPPf4x", "PPf4x")  # the two parts, then halo_mi_norm_rope_params
_gemm_i8_params = _Layout("I4xPQPPQPPQIII4x")
_linear_attention_params = _Layout("5I4xPPI4xPPP3I4x", _ROWS, _ROWS, _ROWS, _ROWS, "PQIfPQ", _STATUS)
_state_block = _Layout("PPPQII")


ARGMAX_RESULT_BYTES = 12  # HALO_MI_ARGMAX_RESULT_BYTES: {index, value bits, poisoned} per vector
STATUS_BAD_INDEX = 8  # HALO_MI_STATUS_BAD_INDEX: a GET_ROWS id outside the table
STATUS_SPLITK_TIMEOUT = 0x100  # HALO_MI_STATUS_SPLITK_TIMEOUT: a split-K reduction gave up waiting
STATUS_KV_FULL = 16  # HALO_MI_STATUS_KV_FULL: no free page, or no column in a sequence's table
KV_LIST_MAX = 1024  # HALO_MI_KV_LIST_MAX: entries of one kv_resize or kv_fork call


# Every symbol include/halo_mi355x.h declares, with its ctypes signature.
_U32, _U64, _VP, _INT = ctypes.c_uint32, ctypes.c_uint64, ctypes.c_void_p, ctypes.c_int
SIGNATURES = {
    "halo_mi_last_error": (ctypes.c_char_p, []),
    "halo_mi_gemv": (_INT, [ctypes.POINTER(_GemvParams), _VP]),
    "halo_mi_gemv_noalloc": (_INT, [ctypes.POINTER(_GemvParams), _VP]),
    "halo_mi_gemv_group": (_INT, [ctypes.POINTER(_GemvGroupParams), _VP]),
    "halo_mi_gemm_group": (_INT, [ctypes.POINTER(_GemvGroupParams), _VP]),
    "halo_mi_gate_up_swiglu": (_INT, [ctypes.POINTER(_GateUpParams), _VP]),
    "halo_mi_lm_head": (_INT, [ctypes.POINTER(_LmHeadParams), _VP]),
    "halo_mi_argmax": (_INT, [_VP, _U64, _U32, _U32, _VP, _VP]),
    "halo_mi_swiglu": (_INT, [_VP, _U64, _VP, _U64, _VP, _U64, _U32, _U32, _VP]),
    "halo_mi_dequant_rows": (_INT, [_U32, _U32, _VP, _U64, _U32, _U32, _U32, _U32, _VP, _U64, _VP]),
    "halo_mi_get_rows": (_INT, [ctypes.POINTER(_GetRowsParams), _VP]),
    "halo_mi_rms_norm": (_INT, [_VP, _U64, _VP, _VP, _U64, _U32, _U32, ctypes.c_float, _VP]),
    "halo_mi_rope_freqs": (_INT, [_U32, ctypes.c_double, ctypes.POINTER(_RopeScaling), _VP, ctypes.POINTER(ctypes.c_float)]),
    "halo_mi_rope": (_INT, [_VP, _VP]),
    "halo_mi_norm_rope": (_INT, [_VP, _VP]),
    "halo_mi_kv_page_bytes": (_U64, [_U32, _U32, _U32, _U32]),
    "halo_mi_kv_write": (_INT, [_VP, _VP]),
    "halo_mi_kv_read": (_INT, [_VP, _VP]),
    "halo_mi_attention": (_INT, [_VP, _VP]),
    "halo_mi_attention_workspace": (_U64, [_VP]),
    "halo_mi_kv_resize": (_INT, [_VP, _VP, _VP, _VP, _U32, _VP, _U32, _VP]),
    "halo_mi_kv_fork": (_INT, [_VP, _VP, _VP, _VP, _U32, _VP, _U32, _VP]),
    "halo_mi_kv_compact": (_INT, [_VP, _VP, _VP, _VP]),
    "halo_mi_kv_copy_pages": (_INT, [_VP, _VP, _VP, _U32, _VP, _U32, _VP]),
    "halo_mi_quantize_rows": (_INT, [_U32, _VP, _U64, _VP, _U64, _VP, _U32, _U32, _VP]),
    "halo_mi_gemm_i8": (_INT, [_VP, _VP]),
    "halo_mi_linear_attention": (_INT, [_VP, _VP]),
    "halo_mi_linear_attention_workspace": (_U64, [_VP]),
    "halo_mi_stream_read": (_INT, [_VP, _U64, _U32, _U32, _VP, _VP]),
    "halo_mi_stream_check": (_INT, [_VP]),
    "halo_mi_stream_release": (_INT, [_VP]),
    "halo_mi_test_splitk_timeout": (_INT, [_U32, _INT]),
    "halo_mi_row_bytes": (_U64, [_U32, _U32]),
    "halo_mi_slab_bytes": (_U64, [_U32, _U32, _U32]),
    "halo_mi_repack_slab": (_INT, [_U32, _VP, _U64, _U32, _U32, _VP, _VP]),
    "halo_mi_unpack_slab": (_INT, [_U32, _VP, _U32, _U32, _VP, _U64, _VP]),
    "halo_mi_repack_slab_host": (_INT, [_U32, _VP, _U64, _U32, _U32, _VP]),
    "halo_mi_unpack_slab_host": (_INT, [_U32, _VP, _U32, _U32, _VP, _U64]),
    "halo_mi_upload_slab": (_INT, [_U32, _VP, _U64, _U32, _U32, _VP, _U64, _VP]),
    "halo_mi_upload_tensors": (_INT, [ctypes.POINTER(_UploadTensor), _U32, _U64, _U32, _VP]),
    "halo_mi_fill_normal": (None, [_U64, _VP, _U64, ctypes.c_float, ctypes.c_float]),
    "halo_mi_quantize": (_INT, [_U32, _VP, _U64, _VP, _U32]),
}


def hip_runtimes() -> list[str]:
    """Paths of the HIP runtime libraries mapped into this process."""
    with open("/proc/self/maps") as f:
        return sorted({line.split()[-1] for line in f if "libamdhip64" in line})


@functools.lru_cache(maxsize=None)
def lib() -> ctypes.CDLL:
    """The loaded library. Raises (never falls back) when it has not been built.

    The process must hold exactly one HIP runtime. torch bundles its own libamdhip64 (soname
    libamdhip64.so.7, but its own libraries ask for it as "libamdhip64.so"), so if this library
    were loaded first it would pull in /opt/rocm's copy and a later torch import would load a
    second one: torch's streams and allocations would then reach the wrong runtime. Importing
    torch first makes this library bind to torch's runtime by soname.
    """
    if not _LIB_PATH.exists():
        raise RuntimeError(f"{_LIB_PATH} is missing: build it with `python -m halo_amd.build` (hipcc, gfx950)")
    try:
        import torch  # noqa: F401
    except ImportError:
        pass
    so = ctypes.CDLL(str(_LIB_PATH))
    runtimes = hip_runtimes()
    if len(runtimes) > 1:
        raise RuntimeError(f"two HIP runtimes are loaded in this process: {runtimes}")
    for name, (res, args) in SIGNATURES.items():
        fn = getattr(so, name)
        fn.restype = res
        fn.argtypes = args
    return so


def _check(rc: int) -> None:
    if rc != 0:
        raise HaloError(rc, lib().halo_mi_last_error().decode())


def _ptr(t) -> int:
    if t is None:
        return 0
    if isinstance(t, int):
        return t
    return t.data_ptr()


def _stream(stream) -> int:
    if stream is not None:
        return int(stream)
    import torch

    return torch.cuda.current_stream().cuda_stream


# ---- geometry ---------------------------------------------------------------------------


def row_bytes(t: int, cols: int) -> int:
    return int(lib().halo_mi_row_bytes(int(t), int(cols)))


def slab_bytes(t: int, rows: int, cols: int) -> int:
    return int(lib().halo_mi_slab_bytes(int(t), int(rows), int(cols)))


# ---- host utilities ---------------------------------------------------------------------


def fill_normal(seed: int, n: int, mean: float = 0.0, std: float = 1.0):
    """SplitMix64 + Box-Muller normal fill (portable, seed-determined), as a float32 numpy array."""
    import numpy as np

    out = np.empty(int(n), dtype=np.float32)
    lib().halo_mi_fill_normal(int(seed), out.ctypes.data, int(n), float(mean), float(std))
    return out


def quantize(t: int, src, threads: int = 0):
    """fp32 numpy array (size a multiple of the block) -> GGUF block bytes (numpy uint8)."""
    import numpy as np

    src = np.ascontiguousarray(src, dtype=np.float32)
    be, bb = block_elems(t), block_bytes(t)
    out = np.empty(src.size // be * bb if be and src.size % be == 0 else 1, dtype=np.uint8)
    _check(lib().halo_mi_quantize(int(t), src.ctypes.data, src.size, out.ctypes.data, int(threads)))
    return out


def repack_slab_host(t: int, src, rows: int, cols: int, src_stride: int = 0):
    import numpy as np

    src = np.ascontiguousarray(src, dtype=np.uint8)
    out = np.empty(slab_bytes(t, rows, cols), dtype=np.uint8)
    _check(lib().halo_mi_repack_slab_host(int(t), src.ctypes.data, int(src_stride), int(rows), int(cols), out.ctypes.data))
    return out


def unpack_slab_host(t: int, src, rows: int, cols: int):
    import numpy as np

    src = np.ascontiguousarray(src, dtype=np.uint8)
    out = np.empty(rows * row_bytes(t, cols), dtype=np.uint8)
    _check(lib().halo_mi_unpack_slab_host(int(t), src.ctypes.data, int(rows), int(cols), out.ctypes.data, 0))
    return out


# ---- device entry points (torch tensors or raw device addresses) -------------------------


def gemv(t: int, w, x, y, rows: int, cols: int, n_vec: int, *, layout: int = Layout.SLAB, w_stride: int = 0,
         x_stride: int = 0, y_stride: int = 0, variant: int = Variant.DEFAULT, norm_w=None, norm_eps: float = 1e-6,
         stream=None) -> None:
    """y = W x (halo_mi_gemv); with norm_w, y = W (rms_norm(x) * norm_w), eps = norm_eps."""
    p = _GemvParams(int(t), int(layout), _ptr(w), int(w_stride), _ptr(x), int(x_stride), _ptr(y), int(y_stride),
                    int(rows), int(cols), int(n_vec), int(variant), _ptr(norm_w), float(norm_eps))
    _check(lib().halo_mi_gemv(ctypes.byref(p), _stream(stream)))


def gemv_noalloc(t: int, w, x, y, rows: int, cols: int, n_vec: int, *, x_stride: int = 0, y_stride: int = 0,
                 variant: int = Variant.DEFAULT, norm_w=None, norm_eps: float = 1e-6, stream=None) -> None:
    """halo_mi_gemv_noalloc: the SLAB GEMV over the library's device-resident scratch (no allocation)."""
    p = _GemvParams(int(t), int(Layout.SLAB), _ptr(w), 0, _ptr(x), int(x_stride), _ptr(y), int(y_stride), int(rows),
                    int(cols), int(n_vec), int(variant), _ptr(norm_w), float(norm_eps))
    _check(lib().halo_mi_gemv_noalloc(ctypes.byref(p), _stream(stream)))


def _group_params(segs, x, cols, n_vec, x_stride, norm_w, norm_eps):
    arr = (_GemvSegment * len(segs))()
    for i, seg in enumerate(segs):
        t, w, rows, y = seg[:4]
        arr[i] = _GemvSegment(int(t), _ptr(w), int(rows), _ptr(y), int(seg[4]) if len(seg) > 4 else 0)
    # the segment array is kept alive with the params (ctypes keeps the reference)
    return _GemvGroupParams(arr, len(segs), _ptr(x), int(x_stride), int(cols), int(n_vec), _ptr(norm_w), float(norm_eps))


def gemv_group(segs, x, cols: int, n_vec: int, *, x_stride: int = 0, norm_w=None, norm_eps: float = 1e-6,
               stream=None) -> None:
    """Grouped GEMV (halo_mi_gemv_group): segs is a list of (type, w, rows, y) or (type, w, rows, y,
    y_stride), SLAB matrices that share x; one launch per pair of weight types."""
    p = _group_params(segs, x, cols, n_vec, x_stride, norm_w, norm_eps)
    _check(lib().halo_mi_gemv_group(ctypes.byref(p), _stream(stream)))


def gemm_group(segs, x, cols: int, n_vec: int, *, x_stride: int = 0, norm_w=None, norm_eps: float = 1e-6,
               stream=None) -> None:
    """Grouped bf16 GEMM (halo_mi_gemm_group): the segments of gemv_group on the bf16 MFMA GEMM,
    x staged once, one launch per pair of weight types."""
    p = _group_params(segs, x, cols, n_vec, x_stride, norm_w, norm_eps)
    _check(lib().halo_mi_gemm_group(ctypes.byref(p), _stream(stream)))


def gate_up_swiglu(t: int, w_gate, w_up, x, out, rows: int, cols: int, n_vec: int, *, layout: int = Layout.SLAB,
                   x_stride: int = 0, out_stride: int = 0, variant: int = Variant.DEFAULT, norm_w=None,
                   norm_eps: float = 1e-6, stream=None) -> None:
    p = _GateUpParams(int(t), int(layout), _ptr(w_gate), _ptr(w_up), _ptr(x), int(x_stride), _ptr(out), int(out_stride),
                      int(rows), int(cols), int(n_vec), int(variant), _ptr(norm_w), float(norm_eps))
    _check(lib().halo_mi_gate_up_swiglu(ctypes.byref(p), _stream(stream)))


def lm_head(t: int, w, x, result, rows: int, cols: int, n_vec: int, *, logits=None, valid_rows: int = 0, ids=None,
            ids_slots=None, ids_scatter=None, ids_scatter_len: int = 0, layout: int = Layout.SLAB, w_stride: int = 0,
            x_stride: int = 0, y_stride: int = 0, variant: int = Variant.DEFAULT, norm_w=None, norm_eps: float = 1e-6,
            stream=None) -> None:
    """The gemv over the vocabulary and the fused argmax (halo_mi_lm_head): result receives
    n_vec triples {index, value bits, poisoned} as uint32; logits (optional) every row."""
    g = _GemvParams(int(t), int(layout), _ptr(w), int(w_stride), _ptr(x), int(x_stride), _ptr(logits), int(y_stride),
                    int(rows), int(cols), int(n_vec), int(variant), _ptr(norm_w), float(norm_eps))
    p = _LmHeadParams(g, _ptr(result), int(valid_rows), _ptr(ids), _ptr(ids_slots), _ptr(ids_scatter),
                      int(ids_scatter_len))
    _check(lib().halo_mi_lm_head(ctypes.byref(p), _stream(stream)))


def argmax(logits, result, n: int, n_vec: int, *, logits_stride: int = 0, stream=None) -> None:
    """ARGMAX (halo_mi_argmax): result receives n_vec triples {index, value bits, poisoned}."""
    _check(lib().halo_mi_argmax(_ptr(logits), int(logits_stride), int(n), int(n_vec), _ptr(result), _stream(stream)))


def swiglu(gate, up, out, rows: int, cols: int, *, gate_stride: int = 0, up_stride: int = 0, out_stride: int = 0,
           stream=None) -> None:
    _check(lib().halo_mi_swiglu(_ptr(gate), int(gate_stride), _ptr(up), int(up_stride), _ptr(out), int(out_stride),
                                int(rows), int(cols), _stream(stream)))


def dequant_rows(t: int, layout: int, w, rows: int, cols: int, out, *, first_row: int = 0, n_rows: int | None = None,
                 w_stride: int = 0, out_stride: int = 0, stream=None) -> None:
    n = rows - first_row if n_rows is None else n_rows
    _check(lib().halo_mi_dequant_rows(int(t), int(layout), _ptr(w), int(w_stride), int(rows), int(cols), int(first_row),
                                      int(n), _ptr(out), int(out_stride), _stream(stream)))


def get_rows(t: int, layout: int, table, n_rows: int, cols: int, ids, n_ids: int, out, *, table_stride: int = 0,
             out_stride: int = 0, status=None, status_keep: bool = False, stream=None) -> None:
    """GET_ROWS (halo_mi_get_rows): out[i] = dequant(table row ids[i]); ids int32 on the device."""
    p = _GetRowsParams(int(t), int(layout), _ptr(table), int(table_stride), int(n_rows), int(cols), _ptr(ids), int(n_ids),
                       _ptr(out), int(out_stride), _ptr(status), 1 if status_keep else 0)
    _check(lib().halo_mi_get_rows(ctypes.byref(p), _stream(stream)))


def rms_norm(x, w, out, rows: int, cols: int, *, eps: float = 1e-6, x_stride: int = 0, out_stride: int = 0,
             stream=None) -> None:
    """RMS_NORM (halo_mi_rms_norm), bitwise cpu::rms_norm."""
    _check(lib().halo_mi_rms_norm(_ptr(x), int(x_stride), _ptr(w), _ptr(out), int(out_stride), int(rows), int(cols),
                                  float(eps), _stream(stream)))


# ---- attention over an 8-bit paged cache -------------------------------------------------


class RopePairs(enum.IntEnum):
    """The two elements that a rotation takes together."""

    HALF = 0  # i and i + rot_dims / 2
    INTERLEAVED = 1  # 2 i and 2 i + 1


class RopeScaling(enum.IntEnum):
    PLAIN = 0
    LINEAR = 1
    NTK = 2
    YARN = 3


class KvCache(typing.NamedTuple):
    """The pool of an 8-bit paged cache (halo_mi_kv_cache): n_pages records of kv_page_bytes() bytes."""

    pool: object
    n_pages: int
    n_layers: int
    n_kv_heads: int
    head_dim: int
    block_tokens: int


class KvBatch(typing.NamedTuple):
    """The sequences of a call (halo_mi_kv_batch): rows row_starts[s] .. row_starts[s + 1] of the row operands are
    the last tokens of sequence s, which holds kv_lens[s] tokens; tables, kv_lens and row_starts are int32
    on the device."""

    tables: object
    table_width: int
    kv_lens: object
    row_starts: object
    n_seqs: int
    n_rows: int
    max_rows: int = 0
    max_kv: int = 0
    table_stride: int = 0


class KvState(typing.NamedTuple):
    """Who holds which page (halo_mi_kv_state), int32 on the device: refs [n_pages], lens [n_slots], tables
    [n_slots, table_width]."""

    refs: object
    lens: object
    tables: object
    n_slots: int
    table_width: int
    table_stride: int = 0


@functools.lru_cache(None)
def _torch():
    """torch; an import statement costs a call 0.1 us each time."""
    import torch

    return torch


def _current_device() -> int:
    """The current GPU, or -2 where nothing runs on one yet (no tensor is there then: a CPU tensor's is -1)."""
    torch = _torch()
    return torch._C._cuda_getDevice() if torch.cuda.is_initialized() else -2


def _raw_stream(stream, dev: int) -> int:
    """The given stream, or torch's current one on device dev."""
    if stream is not None:
        return int(stream)
    return _torch()._C._cuda_getCurrentRawStream(dev) if dev >= 0 else _stream(None)


@functools.lru_cache(None)
def _kinds() -> tuple:
    """The torch types that operands have: lists, status words (either), fp32 rows, frequencies, and rows by their element type."""
    torch = _torch()
    return (torch.int32, (torch.int32, torch.uint32), torch.float32, torch.float64,
            {int(DType.F32): torch.float32, int(DType.F16): torch.float16, int(DType.BF16): torch.bfloat16})


@functools.lru_cache(None)
def _int8():
    return _torch().int8


def _range(values, bits: int):
    for v in values:
        if not 0 <= int(v) < 1 << bits:
            raise HaloError(ErrorCode.Kernel, f"an argument is out of range: {v}")
    return values


def _uints(*values):
    """Arguments that are passed as uint32: ctypes would cut them to 32 bits without a word."""
    return _range(values, 32)


def _sizes(*values):
    return _range(values, 64)


def _dev(t, dev: int) -> int:
    """Device address of an operand; a tensor has to be on the current device."""
    if t is None:
        return 0
    if t.__class__ is int:
        return t
    if t.get_device() != dev:
        raise HaloError(ErrorCode.Kernel, f"an operand is on {t.device}, not on the current GPU")
    return t.data_ptr()


def _dev_of(t, dev: int, kind) -> int:
    """... and of the type `kind` (several: one of them; None: a type that the call itself refuses)."""
    if t is None:
        return 0
    if t.__class__ is int:
        return t
    if t.dtype is not kind:
        kinds = kind if kind.__class__ is tuple else (kind,)
        if kind is not None and t.dtype not in kinds:
            raise HaloError(ErrorCode.Kernel, f"an operand is {t.dtype}, not {' or '.join(map(str, kinds))}")
    if t.get_device() != dev:
        raise HaloError(ErrorCode.Kernel, f"an operand is on {t.device}, not on the current GPU")
    return t.data_ptr()


def _cache(c: KvCache, dev: int) -> tuple:
    return (_dev(c[0], dev), *c[1:])


def _batch(b: KvBatch, dev: int, ints) -> tuple:
    tables, width, kv_lens, row_starts, n_seqs, n_rows, max_rows, max_kv, stride = b
    return _dev_of(tables, dev, ints), stride, width, _dev_of(kv_lens, dev, ints), _dev_of(row_starts, dev, ints), n_seqs, n_rows, max_rows, max_kv


def _state(s: KvState, dev: int, ints):
    refs, lens, tables, n_slots, width, stride = s
    return _state_block(_dev_of(refs, dev, ints), _dev_of(lens, dev, ints), _dev_of(tables, dev, ints), stride, width, n_slots)


def rope_freqs(rot_dims: int, theta: float = 10000.0, *, scaling: int = RopeScaling.PLAIN, scale: float = 1.0,
               context: float = 0.0, beta_fast: float = 32.0, beta_slow: float = 1.0):
    """The rot_dims / 2 frequencies in radians per position (float64 numpy array) and the factor on the rotated
    values (halo_mi_rope_freqs)."""
    import numpy as np

    out = np.empty(max(int(rot_dims) // 2, 1), dtype=np.float64)
    factor = ctypes.c_float(1.0)
    sc = _RopeScaling(int(scaling), float(scale), float(context), float(beta_fast), float(beta_slow))
    _check(lib().halo_mi_rope_freqs(int(rot_dims), float(theta), ctypes.byref(sc), out.ctypes.data, ctypes.byref(factor)))
    return out, float(factor.value)


def rope(t: int, positions, freqs, n_tokens: int, head_dim: int, rot_dims: int, q, q_out, n_heads: int, *, k=None,
         k_out=None, n_kv_heads: int = 0, pairs: int = RopePairs.HALF, factor: float = 1.0, q_stride: int = 0,
         q_head_stride: int = 0, q_out_stride: int = 0, q_out_head_stride: int = 0, k_stride: int = 0,
         k_head_stride: int = 0, k_out_stride: int = 0, k_out_head_stride: int = 0, stream=None) -> None:
    """PARTIAL_ROPE of q and, with k, of k in one launch (halo_mi_rope). q_out may be q, k_out may be k. positions:
    int32, freqs: float64 radians per position (rope_freqs), both on the device; strides in elements."""
    dev = _current_device()
    ints, _, _, doubles, values = _kinds()
    x = values.get(t)
    p = _rope_params(_dev_of(q, dev, x), q_stride, q_head_stride, _dev_of(q_out, dev, x), q_out_stride, q_out_head_stride, n_heads,
                     _dev_of(k, dev, x), k_stride, k_head_stride, _dev_of(k_out, dev, x), k_out_stride, k_out_head_stride, n_kv_heads,
                     t, pairs, 0, 1 if k is None else 2, n_tokens, head_dim, rot_dims, _dev_of(positions, dev, ints),
                     _dev_of(freqs, dev, doubles), factor)
    at = ctypes.addressof(p)
    _POINTER.pack_into(p, _ROPE_PARAMS_AT + 8, at)  # halo_mi_rope_params.parts
    _check(lib().halo_mi_rope(at + _ROPE_PARAMS_AT, _raw_stream(stream, dev)))


def norm_rope(t: int, positions, freqs, n_tokens: int, head_dim: int, rot_dims: int, q, q_out, n_heads: int, *, q_norm=None, k=None,
              k_out=None, n_kv_heads: int = 0, k_norm=None, eps: float = 1e-6, pairs: int = RopePairs.HALF, factor: float = 1.0,
              q_stride: int = 0, q_head_stride: int = 0, q_out_stride: int = 0, q_out_head_stride: int = 0, k_stride: int = 0,
              k_head_stride: int = 0, k_out_stride: int = 0, k_out_head_stride: int = 0, stream=None) -> None:
    """rope with the RMS norm of each head before it, in one pass (halo_mi_norm_rope): q_norm and k_norm are head_dim fp32 weights, or
    None where the heads are rotated only."""
    dev = _current_device()
    ints, _, singles, doubles, values = _kinds()
    x = values.get(t)
    p = _norm_rope_params(_dev_of(q, dev, x), q_stride, q_head_stride, _dev_of(q_out, dev, x), q_out_stride, q_out_head_stride, n_heads,
                          _dev_of(k, dev, x), k_stride, k_head_stride, _dev_of(k_out, dev, x), k_out_stride, k_out_head_stride, n_kv_heads,
                          t, pairs, 0, 1 if k is None else 2, n_tokens, head_dim, rot_dims, _dev_of(positions, dev, ints),
                          _dev_of(freqs, dev, doubles), factor, _dev_of(q_norm, dev, singles), _dev_of(k_norm, dev, singles), eps)
    at = ctypes.addressof(p)
    _POINTER.pack_into(p, _ROPE_PARAMS_AT + 8, at)  # halo_mi_rope_params.parts
    _check(lib().halo_mi_norm_rope(at + _ROPE_PARAMS_AT, _raw_stream(stream, dev)))


def kv_page_bytes(n_layers: int, n_kv_heads: int, head_dim: int, block_tokens: int) -> int:
    """Bytes of a page of the 8-bit cache; 0 for a geometry that it does not have."""
    return int(lib().halo_mi_kv_page_bytes(n_layers, n_kv_heads, head_dim, block_tokens))


def kv_write(t: int, cache: KvCache, layer: int, batch: KvBatch, k, v, *, k_stride: int = 0, k_head_stride: int = 0,
             v_stride: int = 0, v_head_stride: int = 0, status=None, status_keep: bool = False, stream=None) -> None:
    """KV_WRITE: the batch's rows of k and v into their sequences' pages (halo_mi_kv_write)."""
    dev = _current_device()
    ints, words, _, _, values = _kinds()
    x = values.get(t)
    p = _kv_write_params(t, *_cache(cache, dev), layer, *_batch(batch, dev, ints), _dev_of(k, dev, x), k_stride, k_head_stride,
                         _dev_of(v, dev, x), v_stride, v_head_stride, _dev_of(status, dev, words), 1 if status_keep else 0)
    _check(lib().halo_mi_kv_write(p, _raw_stream(stream, dev)))


def kv_read(cache: KvCache, layer: int, batch: KvBatch, k_out=None, v_out=None, *, k_stride: int = 0, k_head_stride: int = 0,
            v_stride: int = 0, v_head_stride: int = 0, status=None, status_keep: bool = False, stream=None) -> None:
    """The values that the cache holds for the batch's rows, in fp32 (halo_mi_kv_read)."""
    dev = _current_device()
    ints, words, singles, _, _ = _kinds()
    p = _kv_read_params(*_cache(cache, dev), layer, *_batch(batch, dev, ints), _dev_of(k_out, dev, singles), k_stride, k_head_stride,
                        _dev_of(v_out, dev, singles), v_stride, v_head_stride, _dev_of(status, dev, words), 1 if status_keep else 0)
    _check(lib().halo_mi_kv_read(p, _raw_stream(stream, dev)))


def _attention_params(t, cache, layer, batch, q, out, n_heads, scale, window, q_stride, q_head_stride, out_stride, out_head_stride,
                      workspace, workspace_bytes, status, status_keep, dev):
    if workspace is not None and not isinstance(workspace, int) and not workspace_bytes:
        workspace_bytes = workspace.numel() * workspace.element_size()
    ints, words, _, _, values = _kinds()
    x = values.get(t)
    return _attention_block(t, *_cache(cache, dev), layer, *_batch(batch, dev, ints), _dev_of(q, dev, x), q_stride, q_head_stride,
                            _dev_of(out, dev, x), out_stride, out_head_stride, n_heads, scale, window, _dev(workspace, dev), workspace_bytes,
                            _dev_of(status, dev, words), 1 if status_keep else 0)


def attention(t: int, cache: KvCache, layer: int, batch: KvBatch, q, out, n_heads: int, *, scale: float = 0.0, window: int = 0,
              q_stride: int = 0, q_head_stride: int = 0, out_stride: int = 0, out_head_stride: int = 0, workspace=None,
              workspace_bytes: int = 0, status=None, status_keep: bool = False, stream=None) -> None:
    """ATTENTION of the batch's rows over their sequences' cached tokens, causal, over the last `window` tokens where it
    is not 0 (halo_mi_attention). scale 0: 1 / sqrt(head_dim)."""
    dev = _current_device()
    p = _attention_params(t, cache, layer, batch, q, out, n_heads, scale, window, q_stride, q_head_stride, out_stride, out_head_stride,
                          workspace, workspace_bytes, status, status_keep, dev)
    _check(lib().halo_mi_attention(p, _raw_stream(stream, dev)))


def attention_workspace(t: int, cache: KvCache, layer: int, batch: KvBatch, q, out, n_heads: int, *, window: int = 0,
                        q_stride: int = 0, q_head_stride: int = 0, out_stride: int = 0, out_head_stride: int = 0) -> int:
    """Workspace bytes that the same attention call makes use of (halo_mi_attention_workspace)."""
    dev = _current_device()
    p = _attention_params(t, cache, layer, batch, q, out, n_heads, 0.0, window, q_stride, q_head_stride, out_stride, out_head_stride,
                          None, 0, None, False, dev)
    return int(lib().halo_mi_attention_workspace(p))


def kv_resize(cache: KvCache, state: KvState, slots, new_lens, n: int, *, status=None, status_keep: bool = False, stream=None) -> None:
    """Gives slots their new lengths, with pages taken and released (halo_mi_kv_resize); length 0 frees a slot."""
    dev = _current_device()
    ints, words = _kinds()[:2]
    c, s = _cache_block(*_cache(cache, dev)), _state(state, dev, ints)
    _check(lib().halo_mi_kv_resize(c, s, _dev_of(slots, dev, ints), _dev_of(new_lens, dev, ints), n, _dev_of(status, dev, words),
                                   1 if status_keep else 0, _raw_stream(stream, dev)))


def kv_fork(cache: KvCache, state: KvState, src, dst, n: int, *, status=None, status_keep: bool = False, stream=None) -> None:
    """Empty slots dst become copies of src: whole pages shared, a last one that is not full copied (halo_mi_kv_fork)."""
    dev = _current_device()
    ints, words = _kinds()[:2]
    c, s = _cache_block(*_cache(cache, dev)), _state(state, dev, ints)
    _check(lib().halo_mi_kv_fork(c, s, _dev_of(src, dev, ints), _dev_of(dst, dev, ints), n, _dev_of(status, dev, words),
                                 1 if status_keep else 0, _raw_stream(stream, dev)))


def kv_compact(cache: KvCache, state: KvState, *, live=None, stream=None) -> None:
    """Moves the live pages to the front of the pool (halo_mi_kv_compact); live (uint32 or int32) receives their number."""
    dev = _current_device()
    ints, words = _kinds()[:2]
    c, s = _cache_block(*_cache(cache, dev)), _state(state, dev, ints)
    _check(lib().halo_mi_kv_compact(c, s, _dev_of(live, dev, words), _raw_stream(stream, dev)))


def kv_copy_pages(cache: KvCache, src, dst, n: int, *, status=None, status_keep: bool = False, stream=None) -> None:
    """Copies whole pages (halo_mi_kv_copy_pages)."""
    dev = _current_device()
    ints, words = _kinds()[:2]
    c = _cache_block(*_cache(cache, dev))
    _check(lib().halo_mi_kv_copy_pages(c, _dev_of(src, dev, ints), _dev_of(dst, dev, ints), n, _dev_of(status, dev, words), 1 if status_keep else 0,
                                       _raw_stream(stream, dev)))


# ---- products of 8-bit integers ----------------------------------------------------------


def quantize_rows(t: int, x, codes, scales, rows: int, cols: int, *, x_stride: int = 0, codes_stride: int = 0, stream=None) -> None:
    """Rows of x as int8 codes and one fp32 scale each (halo_mi_quantize_rows). codes: int8 rows codes_stride bytes apart, a multiple of
    16 (0: cols rounded up to 16), with zeros behind a row's codes."""
    dev = _current_device()
    _, _, singles, _, values = _kinds()
    _check(lib().halo_mi_quantize_rows(*_uints(t), _dev_of(x, dev, values.get(t)), *_sizes(x_stride), _dev_of(codes, dev, _int8()), *_sizes(codes_stride),
                                       _dev_of(scales, dev, singles), *_uints(rows, cols), _raw_stream(stream, dev)))


def gemm_i8(t: int, w, w_scales, x, x_scales, y, rows: int, cols: int, n_vec: int, *, w_stride: int = 0, x_stride: int = 0, y_stride: int = 0,
            stream=None) -> None:
    """y[v][n] = x_scales[v] * w_scales[n] * sum_i x[v][i] w[n][i] over int8 codes as quantize_rows writes them, y of type t
    (halo_mi_gemm_i8)."""
    dev = _current_device()
    _, _, singles, _, values = _kinds()
    codes = _int8()
    p = _gemm_i8_params(t, _dev_of(w, dev, codes), w_stride, _dev_of(w_scales, dev, singles), _dev_of(x, dev, codes), x_stride,
                        _dev_of(x_scales, dev, singles), _dev_of(y, dev, values.get(t)), y_stride, rows, cols, n_vec)
    _check(lib().halo_mi_gemm_i8(p, _raw_stream(stream, dev)))


# ---- linear attention --------------------------------------------------------------------


class LinearState(typing.NamedTuple):
    """The states of linear attention's heads: n_slots slots of n_heads x k_dim x v_dim fp32, and where the new ones go (None: into the
    same)."""

    data: object
    n_slots: int
    n_heads: int
    k_dim: int
    v_dim: int
    out: object = None


class LinearBatch(typing.NamedTuple):
    """The sequences of a call: rows row_starts[s] .. row_starts[s + 1] of the row operands are the next tokens of the sequence in slot
    slots[s]; seq_lens (optional) its tokens with them. int32 on the device."""

    slots: object
    row_starts: object
    n_seqs: int
    n_rows: int
    max_rows: int = 0
    seq_lens: object = None


def _linear_block(t, state, batch, q, k, v, out, decay, n_k_heads, decay_per_head, scale, decay_stride, q_stride, q_head_stride, k_stride,
                  k_head_stride, v_stride, v_head_stride, out_stride, out_head_stride, workspace, workspace_bytes, status, status_keep, dev):
    if workspace is not None and not isinstance(workspace, int) and not workspace_bytes:
        workspace_bytes = workspace.numel() * workspace.element_size()
    ints, words, singles, _, values = _kinds()
    x = values.get(t)
    data, n_slots, n_heads, k_dim, v_dim, new = state
    slots, row_starts, n_seqs, n_rows, max_rows, seq_lens = batch
    before = _dev_of(data, dev, singles)
    return _linear_attention_params(
        t, n_heads, n_k_heads, k_dim, v_dim, before, before if new is None else _dev_of(new, dev, singles), n_slots, _dev_of(slots, dev, ints),
        _dev_of(row_starts, dev, ints), _dev_of(seq_lens, dev, ints), n_seqs, n_rows, max_rows, _dev_of(q, dev, x), q_stride, q_head_stride,
        _dev_of(k, dev, x), k_stride, k_head_stride, _dev_of(v, dev, x), v_stride, v_head_stride, _dev_of(out, dev, x), out_stride,
        out_head_stride, _dev_of(decay, dev, singles), decay_stride, 1 if decay_per_head else 0, scale, _dev(workspace, dev), workspace_bytes,
        _dev_of(status, dev, words), 1 if status_keep else 0)


def linear_attention(t: int, state: LinearState, batch: LinearBatch, q, k, v, out, decay, n_k_heads: int, *, decay_per_head: bool = False,
                     scale: float = 0.0, decay_stride: int = 0, q_stride: int = 0, q_head_stride: int = 0, k_stride: int = 0,
                     k_head_stride: int = 0, v_stride: int = 0, v_head_stride: int = 0, out_stride: int = 0, out_head_stride: int = 0,
                     workspace=None, workspace_bytes: int = 0, status=None, status_keep: bool = False, stream=None) -> None:
    """S <- exp(decay) S + k v^T, out = scale S^T q for each sequence's rows in order, S its heads' states (halo_mi_linear_attention).
    decay: fp32 logarithms, [n_rows, n_heads], or [n_heads] with decay_per_head. scale 0: 1 / sqrt(k_dim)."""
    dev = _current_device()
    p = _linear_block(t, state, batch, q, k, v, out, decay, n_k_heads, decay_per_head, scale, decay_stride, q_stride, q_head_stride, k_stride,
                      k_head_stride, v_stride, v_head_stride, out_stride, out_head_stride, workspace, workspace_bytes, status, status_keep, dev)
    _check(lib().halo_mi_linear_attention(p, _raw_stream(stream, dev)))


def linear_attention_workspace(t: int, state: LinearState, batch: LinearBatch, q, k, v, out, decay, n_k_heads: int, *,
                               decay_per_head: bool = False, decay_stride: int = 0, q_stride: int = 0, q_head_stride: int = 0,
                               k_stride: int = 0, k_head_stride: int = 0, v_stride: int = 0, v_head_stride: int = 0, out_stride: int = 0,
                               out_head_stride: int = 0) -> int:
    """Workspace bytes that the same linear_attention call makes use of (halo_mi_linear_attention_workspace)."""
    dev = _current_device()
    p = _linear_block(t, state, batch, q, k, v, out, decay, n_k_heads, decay_per_head, 0.0, decay_stride, q_stride, q_head_stride, k_stride,
                      k_head_stride, v_stride, v_head_stride, out_stride, out_head_stride, None, 0, None, False, dev)
    return int(lib().halo_mi_linear_attention_workspace(p))


def stream_read(p, nbytes: int, workgroups: int, unroll: int, sink, stream=None) -> None:
    """One read-only stream over nbytes at p (halo_mi_stream_read): the read floor's kernel."""
    _check(lib().halo_mi_stream_read(_ptr(p), int(nbytes), int(workgroups), int(unroll), _ptr(sink), _stream(stream)))


def stream_check(stream=None) -> None:
    """Synchronizes the stream and raises HaloError(Device) when a kernel marked its status word
    (a split-K reduction that gave up waiting) since the last check (halo_mi_stream_check)."""
    _check(lib().halo_mi_stream_check(_stream(stream)))


def stream_release(stream=None) -> None:
    """Frees the stream's workspace on the current device (halo_mi_stream_release)."""
    _check(lib().halo_mi_stream_release(_stream(stream)))


def force_splitk_timeout(spin_limit: int, force: bool) -> None:
    """Failure-path test hook (halo_mi_test_splitk_timeout): force every split-K reduction to give
    up after spin_limit rounds; force=False restores normal operation."""
    _check(lib().halo_mi_test_splitk_timeout(int(spin_limit), 1 if force else 0))


def repack_slab(t: int, src, rows: int, cols: int, dst, *, src_stride: int = 0, stream=None) -> None:
    _check(lib().halo_mi_repack_slab(int(t), _ptr(src), int(src_stride), int(rows), int(cols), _ptr(dst), _stream(stream)))


def unpack_slab(t: int, src, rows: int, cols: int, dst, *, dst_stride: int = 0, stream=None) -> None:
    _check(lib().halo_mi_unpack_slab(int(t), _ptr(src), int(rows), int(cols), _ptr(dst), int(dst_stride), _stream(stream)))


def upload_tensors(tensors, *, chunk_bytes: int = 0, host_threads: int = 0, stream=None) -> None:
    """Model-scale upload (halo_mi_upload_tensors). tensors: a list of (type, cols, parts, dst)
    with parts a list of (host rows, rows) or (host rows, rows, src_stride); host rows are numpy
    uint8 arrays (e.g. memmaps of the GGUF tensors) or host addresses. The parts' rows are
    concatenated into one SLAB matrix at dst (a row-fused projection when there are several)."""
    keep = []
    arr = (_UploadTensor * len(tensors))()
    for i, (t, cols, parts, dst) in enumerate(tensors):
        pa = (_UploadPart * len(parts))()
        for j, part in enumerate(parts):
            src, rows = part[0], part[1]
            stride = part[2] if len(part) > 2 else 0
            pa[j] = _UploadPart(src if isinstance(src, int) else src.ctypes.data, int(stride), int(rows))
        keep.append(pa)
        arr[i] = _UploadTensor(int(t), int(cols), pa, len(parts), _ptr(dst))
    _check(lib().halo_mi_upload_tensors(arr, len(tensors), int(chunk_bytes), int(host_threads), _stream(stream)))


def upload_slab(t: int, host_src, rows: int, cols: int, dst, *, src_stride: int = 0, chunk_bytes: int = 0,
                stream=None) -> None:
    """host_src: a numpy uint8 array (e.g. a memmap of the GGUF tensor) or a host address."""
    addr = host_src if isinstance(host_src, int) else host_src.ctypes.data
    _check(lib().halo_mi_upload_slab(int(t), addr, int(src_stride), int(rows), int(cols), _ptr(dst), int(chunk_bytes),
                                     _stream(stream)))
