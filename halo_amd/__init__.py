"""halo_amd: MI355X-native quantized matrix-multiply backend (GGUF Q4_0 / Q8_0 / Q4_K / Q5_K / Q6_K /
IQ4_XS).

The compute path is hand-written HIP for gfx950 in ``libhalo_mi355x.so``, reached through the
C ABI declared in ``include/halo_mi355x.h``. This package loads that library with ctypes and
mirrors the reference's operator interface for the path (``Backend::gemv`` over
``GemvArgs``; include/halo/backend/backend.h:283-314, :562). Beside it stand rotary positions, an
8-bit paged cache and the attention over it (``rope``, ``norm_rope``, ``kv_*``, ``attention``), products of 8-bit integers
(``quantize_rows``, ``gemm_i8``) and linear attention with a state (``linear_attention``). There is no CPU
fallback: if the library is missing every entry point raises.
"""
from __future__ import annotations

from ._lib import (  # noqa: F401
    DType,
    ErrorCode,
    HaloError,
    KvBatch,
    KvCache,
    KvState,
    Layout,
    LinearBatch,
    LinearState,
    RopePairs,
    RopeScaling,
    Variant,
    ARGMAX_RESULT_BYTES,
    KV_LIST_MAX,
    SLAB_ROWS,
    STATUS_BAD_INDEX,
    STATUS_KV_FULL,
    STATUS_SPLITK_TIMEOUT,
    argmax,
    attention,
    attention_workspace,
    block_bytes,
    block_elems,
    dequant_rows,
    fill_normal,
    force_splitk_timeout,
    gate_up_swiglu,
    gemv,
    gemm_group,
    gemm_i8,
    gemv_group,
    gemv_noalloc,
    get_rows,
    kv_compact,
    kv_copy_pages,
    kv_fork,
    kv_page_bytes,
    kv_read,
    kv_resize,
    kv_write,
    lib,
    linear_attention,
    linear_attention_workspace,
    lm_head,
    norm_rope,
    quantize,
    quantize_rows,
    repack_slab,
    repack_slab_host,
    rms_norm,
    rope,
    rope_freqs,
    row_bytes,
    slab_bytes,
    stream_check,
    stream_read,
    stream_release,
    swiglu,
    unpack_slab,
    unpack_slab_host,
    upload_slab,
    upload_tensors,
)
