/*
 * halo_mi355x: MI355X (gfx950) quantized matrix-multiply backend, C ABI.
 *
 * This is the seam between host code and the hand-written HIP kernels. It replaces the HIP
 * backend's launcher seam of the reference (backends/hip/src/launch.h:16-37:
 * `int launch_gemv_*(const kern::GemvParams&, const kern::Launch&, void* stream)`, returning
 * the hipError_t as an int). Every entry point takes plain pointers, sizes and a hipStream_t
 * passed as `void*`, validates its arguments on the host, enqueues work, and returns a status
 * code; no exception crosses the ABI. halo_mi_last_error() gives the message of the last
 * failing call on the calling thread.
 *
 * Device pointers are HIP device memory on the current device. `stream` may be NULL (the
 * null stream). Work is asynchronous: outputs are valid after the stream is synchronized.
 *
 * Status codes follow the reference's error mapping (include/halo/backend/backend.h:24-26):
 * shape / alias / range / alignment -> HALO_MI_E_KERNEL, dtype or limit -> HALO_MI_E_UNSUPPORTED,
 * unknown variant id -> HALO_MI_E_CONFIG, allocation -> HALO_MI_E_MEMORY, a HIP runtime error
 * -> HALO_MI_E_DEVICE.
 */
#ifndef HALO_MI355X_H
#define HALO_MI355X_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* ---- status codes ---------------------------------------------------------------------- */
enum {
    HALO_MI_OK = 0,
    HALO_MI_E_KERNEL = 1,      /* shape, alias, range or alignment problem */
    HALO_MI_E_UNSUPPORTED = 2, /* weight type or limit not supported */
    HALO_MI_E_CONFIG = 3,      /* unknown variant id */
    HALO_MI_E_MEMORY = 4,      /* allocation failure */
    HALO_MI_E_DEVICE = 5       /* HIP runtime / launch failure */
};

/* Message of the last failing call on this thread ("" when none). */
const char* halo_mi_last_error(void);

/* ---- weight types (ggml ids, include/halo/tensor/dtype.h:18-49) ------------------------- */
/*
 * Every type of the reference's CPU dequantizer (src/tensor/quant.cpp:386-407) is decoded on
 * the GGUF layout by halo_mi_dequant_rows, halo_mi_get_rows and the reference-order GEMV
 * (HALO_MI_GEMV_GGUF_REF), bitwise as dequantize_row and cpu::matmul. The SLAB layout, and with
 * it every fast kernel, takes Q4_0, Q8_0, Q4_K, Q5_K, Q6_K and IQ4_XS. The reference's HIP
 * backend has kernels for eleven of them (backends/hip/src/ops.cpp:531-549: not BF16, Q4_1,
 * Q5_0, Q5_1, Q2_K); the C++ backend of this library refuses the same five.
 */
enum {
    HALO_MI_F32 = 0,
    HALO_MI_F16 = 1,
    HALO_MI_Q4_0 = 2,
    HALO_MI_Q4_1 = 3,
    HALO_MI_Q5_0 = 6,
    HALO_MI_Q5_1 = 7,
    HALO_MI_Q8_0 = 8,
    HALO_MI_Q2_K = 10,
    HALO_MI_Q3_K = 11,
    HALO_MI_Q4_K = 12,
    HALO_MI_Q5_K = 13,
    HALO_MI_Q6_K = 14,
    HALO_MI_IQ4_NL = 20,
    HALO_MI_IQ3_S = 21,
    HALO_MI_IQ4_XS = 23,
    HALO_MI_BF16 = 30
};

/* ---- weight layouts ---------------------------------------------------------------------- */
/*
 * HALO_MI_LAYOUT_GGUF: rows of GGUF blocks exactly as in the file (w_stride bytes apart, any
 *   alignment). What the reference imports (src/backend/hip_adapter.cpp:502-515).
 * HALO_MI_LAYOUT_SLAB: the device layout written by halo_mi_repack_slab(). Rows are grouped
 *   in slabs of 64; inside a slab every plane is slot-major and row-minor, so one wave's
 *   load of a slot covers 64 rows contiguously. A slab has exactly 64 * row_bytes bytes; the
 *   last slab of a matrix is zero-padded to 64 rows. The GGUF bytes are recoverable with
 *   halo_mi_unpack_slab().
 */
enum { HALO_MI_LAYOUT_GGUF = 0, HALO_MI_LAYOUT_SLAB = 1 };

/* Rows per slab. */
#define HALO_MI_SLAB_ROWS 64u

/* ---- gemv variants (append-only ids; 0 = default for the layout) ------------------------ */
/*
 * Counterpart of the reference's KernelChoice registry (backend.h:173-176, ids pinned by
 * tests/unit/backend/test_hip_backend.cpp:925-981). These are this library's own ids; the
 * reference registry ids they take behind its HIP backend are listed with the C++ backend
 * (include/halo_mi355x_backend.hpp).
 *   0 HALO_MI_GEMV_DEFAULT   GGUF layout -> gemv_gguf_ref; SLAB layout -> gemv_slab_auto.
 *   1 HALO_MI_GEMV_GGUF_REF  GGUF layout, 8 lanes per output in cpu::detail::dot's order:
 *                            bit-identical to the CPU backend.
 *   2 HALO_MI_GEMV_SLAB      SLAB layout, wave64 row-per-lane weight stream, split-K inside
 *                            the workgroup and across workgroups (fixed-order fix-up); any
 *                            n_vec (4 per pass over the weights). Within the summation bound;
 *                            every row is bitwise independent of n_vec.
 *   3 HALO_MI_GEMM_SLAB_BF16 SLAB layout, bf16 MFMA GEMM (dequantized W and x rounded to
 *                            bf16, fp32 accumulate) on M tiles of 64 / 128 / 256 rows by n_vec;
 *                            any n_vec.
 *   4 HALO_MI_GEMV_SLAB_AUTO SLAB layout: 2 for n_vec <= 2 (Q6_K: <= 4); 8 for the rest up to
 *                            n_vec <= 8 (2 when cols is not a multiple of 256); so up to 8
 *                            vectors the result is within 2's bound.
 *                            Above 8, the small-M bf16 GEMM (same numerics as 3) for n_vec <= 32
 *                            when cols is a multiple of 256; else 5 when n_vec > 256 and its
 *                            tiles fill the GPU, else 3.
 *   5 HALO_MI_GEMM_SLAB_BF16_M512  the bf16 MFMA GEMM on 512-row M tiles (every wave both
 *                            dequantizes and multiplies; same numerics as 3); any n_vec.
 *   6 HALO_MI_GEMV_SLAB_VALU the SLAB GEMV with its multiply-adds on the VALU instead of the
 *                            matrix core (Q4_0, Q8_0, Q4_K, Q6_K; no fused norm); the same
 *                            split and bound as 2.
 *   7 HALO_MI_GEMM_SLAB_BF16_SMALL_M  the bf16 MFMA GEMM's small-M kernel (no LDS stage; waves
 *                            dequantize their own MFMA operands): n_vec <= 32, cols a multiple
 *                            of 256; same numerics as 3.
 *   8 HALO_MI_GEMM_SLAB_EXACT_SMALL_M  the exact-product small-M GEMM: the slab GEMV's
 *                            arithmetic (integer codes times x split exactly into three bf16
 *                            pieces, fp32 sums, scales applied per slot) on 32x32 MFMA tiles;
 *                            n_vec <= 8, cols a multiple of 256; within the bound of 2. Its K
 *                            split is the one planned for 8 vectors whatever n_vec is, so rows do
 *                            not depend on n_vec.
 *   9 HALO_MI_GEMM_SLAB_EXACT_INVARIANT  8's kernel for any n_vec, in passes of 8 vectors:
 *                            every row of y is bitwise the row an n_vec = 1 call
 *                            gives (the batch-invariance contract of GemvArgs::allow_gemm =
 *                            false, backend.h:298-304). Where that split does not fit the shape
 *                            (cols not a multiple of 256, or more partial sums than the stream's
 *                            workspace holds) it runs 2, which is batch-invariant too: the
 *                            choice follows the shape only. Within the bound of 2. Faster than
 *                            2 from 3 vectors (one pass over the weights up to 8), slower at 1.
 */
enum {
    HALO_MI_GEMV_DEFAULT = 0,
    HALO_MI_GEMV_GGUF_REF = 1,
    HALO_MI_GEMV_SLAB = 2,
    HALO_MI_GEMM_SLAB_BF16 = 3,
    HALO_MI_GEMV_SLAB_AUTO = 4,
    HALO_MI_GEMM_SLAB_BF16_M512 = 5,
    HALO_MI_GEMV_SLAB_VALU = 6,
    HALO_MI_GEMM_SLAB_BF16_SMALL_M = 7,
    HALO_MI_GEMM_SLAB_EXACT_SMALL_M = 8,
    HALO_MI_GEMM_SLAB_EXACT_INVARIANT = 9,
    HALO_MI_GEMV_VARIANT_LAST = 9
};

/*
 * y[t][n] = sum_i x[t][i] * W[n][i] for t < n_vec, n < rows, i < cols.
 * Replaces backend::GemvArgs + Backend::gemv (include/halo/backend/backend.h:283-314, :562)
 * at the launcher level, as kern::GemvParams does (backends/hip/kernels/gemv.h:267-281).
 *   w: device weights in `layout`; for GGUF, w_stride = bytes between rows (0 = row_bytes);
 *      for SLAB, w_stride must be 0.
 *   x: n_vec rows of cols fp32, x_stride floats apart (0 = cols).
 *   y: n_vec rows of rows fp32, y_stride floats apart (0 = rows). y must not overlap x or w.
 *   norm_w (optional, cols fp32): the fused input norm of GemvArgs::norm_w / norm_eps
 *      (backend.h:292-299): y = W (rms_norm(x) * norm_w) with eps = norm_eps, x the raw rows;
 *      rms_norm as cpu::rms_norm (backends/cpu/ops_basic.cpp:18-33). Every variant, layout and
 *      n_vec (the reference accepts it on one Vulkan path only):
 *        - GGUF reference variant: x is normalized first exactly as cpu::rms_norm, so y is
 *          bitwise rms_norm then matmul;
 *        - bf16 GEMM variants: the same normalized x, rounded to bf16 while it is staged;
 *        - SLAB GEMV (2 and the GEMV legs of the auto variants), one vector: inside the MFMA
 *          GEMV's launch, one dispatch: every workgroup computes 1 / rms in cpu::rms_norm's
 *          order and normalizes its own x elements as cpu::rms_norm rounds them (cols <= 8192;
 *          matrices of up to 256 slabs or 1024 columns, or whose launch splits K over workgroups);
 *        - otherwise (more vectors, wider rows, more slabs than that with K unsplit, variant 6): x
 *          is normalized into the stream's workspace by the RMS_NORM kernel, then the GEMV runs on it.
 *      So y is bitwise halo_mi_rms_norm then the same variant without the norm, at any n_vec
 *      (the reference's Limits::max_fused_norm_cols contract, backend.h:236-242).
 *      norm_w must not overlap y.
 */
typedef struct halo_mi_gemv_params {
    uint32_t type;
    uint32_t layout;
    const void* w;
    uint64_t w_stride;
    const float* x;
    uint64_t x_stride;
    float* y;
    uint64_t y_stride;
    uint32_t rows;
    uint32_t cols;
    uint32_t n_vec;
    uint32_t variant;
    const float* norm_w;
    float norm_eps;
} halo_mi_gemv_params;

int halo_mi_gemv(const halo_mi_gemv_params* p, void* stream);

/*
 * halo_mi_gemv without any allocation. No counterpart in the reference: it is for callers that
 * cannot allocate device memory (code under HIP graph capture, tight serving loops, harnesses
 * that forbid hipMalloc). Same operands, checks and results as halo_mi_gemv (bitwise) for the
 * calls that run the SLAB GEMV: variants 2 and 6 at any n_vec, and 0 and 4 where their auto
 * choice is the SLAB GEMV (up to 2 vectors; up to 4 for Q6_K and for Q4_K, Q5_K and IQ4_XS
 * matrices of at most 128 slabs; up to 8 where the exact small-M GEMM's plan does not fit).
 * Where 0 or 4 would run a GEMM kernel, and for the GEMM variants, it returns
 * HALO_MI_E_UNSUPPORTED. The split-K words, slab counters and status word live in a fixed
 * device array of this library (about 8.3 MiB per GPU, held until the process ends), not in a
 * per-stream workspace: a shape whose split needs more than 65536 slabs of counters or 2^20
 * words (e.g. the 17408 x 5120 headline needs 2^17.7) returns HALO_MI_E_UNSUPPORTED. Every call
 * on one GPU shares that array, so calls that overlap in time on one GPU (other streams, other
 * threads) race and give wrong results: order them. halo_mi_stream_check also reports this
 * array's status word.
 */
int halo_mi_gemv_noalloc(const halo_mi_gemv_params* p, void* stream);

/*
 * Grouped GEMV: several SLAB matrices that share x, in one launch per pair of weight types,
 * e.g. a layer's q, k and v projections (Q4_K q and k, Q6_K v) after the same input norm. The
 * reference issues them one by one on one stream (Qwen35::Impl::gemv,
 * src/models/qwen35.cpp:486-498), and each small projection then pays a whole launch's ramp and
 * drain; row-fusing them into one matrix (halo_mi_upload_tensors) needs equal types.
 *   segs[i]: the segment's weight type, SLAB image (16-byte aligned), rows, and output y_i
 *            (n_vec rows of rows floats, y_stride apart, 0 = rows): y_i = W_i x (with the fused
 *            norm: W_i (rms_norm(x) * norm_w), as halo_mi_gemv).
 *   x, x_stride, cols, n_vec, norm_w, norm_eps: shared, with halo_mi_gemv's meaning.
 * Numerics: halo_mi_gemv's SLAB GEMV bound per output (the K split follows the group's total
 * slabs, so a row may round differently from a call of its own; rows stay independent of n_vec).
 * No output may overlap x, norm_w, any segment's weights or another output.
 * n_segs <= HALO_MI_GEMV_GROUP_MAX; more than two weight types take one launch per pair.
 */
#define HALO_MI_GEMV_GROUP_MAX 4u

typedef struct halo_mi_gemv_segment {
    uint32_t type;
    const void* w;
    uint32_t rows;
    float* y;
    uint64_t y_stride;
} halo_mi_gemv_segment;

typedef struct halo_mi_gemv_group_params {
    const halo_mi_gemv_segment* segs;
    uint32_t n_segs;
    const float* x;
    uint64_t x_stride;
    uint32_t cols;
    uint32_t n_vec;
    const float* norm_w;
    float norm_eps;
} halo_mi_gemv_group_params;

int halo_mi_gemv_group(const halo_mi_gemv_group_params* p, void* stream);

/*
 * Grouped bf16 GEMM: the same segments and operands as halo_mi_gemv_group, computed by the bf16
 * MFMA GEMM (the prefill path, GemvArgs::allow_gemm: halo_mi_gemv's numerics for more than 8
 * vectors), with x staged once for all segments and one launch per pair of weight types (M
 * tiles of 64 / 128 / 256 rows by n_vec; when a launch's tiles fill less than half the GPU,
 * every tile is split over the same K chunks and one reduce adds them in chunk order). The
 * reference issues the projections one by one (Qwen35::Impl::gemv, src/models/qwen35.cpp:
 * 486-498); a layer's q, k and v at M = 512 then pay three x stagings, three under-filled
 * launches and three reduces. Numerics per output: halo_mi_gemv's bf16 GEMM bound; x rows
 * 16-byte aligned (x_stride a multiple of 4 floats), as the single-matrix GEMM.
 */
int halo_mi_gemm_group(const halo_mi_gemv_group_params* p, void* stream);

/*
 * Fused FFN gate/up: out[t][n] = silu((Wg x_t)[n]) * (Wu x_t)[n], silu(v) = v / (1 + exp(-v)).
 * The reference composes it as gemv(gate), gemv(up), swiglu (src/models/qwen35.cpp:789-805;
 * backends/cpu/ops_basic.cpp:165-167); here both matmuls and the epilogue are one launch.
 * Wg and Wu share type, layout and shape (rows x cols). SLAB layout only; variant 0/4 = auto
 * (the gemv pair for n_vec <= 2, the exact small-M GEMM (8) for 3 and 4 when cols is a multiple
 * of 256, else the gemv pair up to 4; above 4 the bf16 GEMM, its M
 * tiles chosen as for halo_mi_gemv), 2 = gemv kernel (any n_vec, 4 vectors per pass over the
 * weights), 3 / 5 / 7 = bf16 MFMA GEMM on 64..256 / 512-row / small-M tiles, 8 = the exact
 * small-M GEMM (n_vec <= 8). The GEMMs' SiLU is the fast form (relative error at most
 * (1.5 |v| + 8) 2^-24), the gemv pair's the IEEE one. out may not overlap x, Wg or Wu.
 * norm_w / norm_eps (optional): the fused input norm as for halo_mi_gemv (the FFN's
 * post-attention norm folded into the pair).
 */
typedef struct halo_mi_gate_up_params {
    uint32_t type;
    uint32_t layout;
    const void* w_gate;
    const void* w_up;
    const float* x;
    uint64_t x_stride;
    float* out;
    uint64_t out_stride;
    uint32_t rows;
    uint32_t cols;
    uint32_t n_vec;
    uint32_t variant;
    const float* norm_w;
    float norm_eps;
} halo_mi_gate_up_params;

int halo_mi_gate_up_swiglu(const halo_mi_gate_up_params* p, void* stream);

/*
 * LM head: the gemv over the vocabulary plus the fused argmax. Replaces Backend::lm_head and
 * LmHeadArgs (include/halo/backend/backend.h:433-460, :572); the semantics are
 * CpuBackend::lm_head's (src/backend/cpu_backend.cpp:669-770):
 *   - the argmax is taken over exactly the values the gemv produces: higher value first, ties
 *     to the lowest index;
 *   - a NaN logit poisons only its own vector: its result is {0xFFFFFFFF, quiet NaN, 1};
 *   - rows at or past valid_rows (when not 0) are not ranked (GGUF LM-head padding), but a NaN
 *     in them still poisons; the logits of every row are still written;
 *   - a vector with no ranked row reports {0xFFFFFFFF, 0.0f, 0}.
 * gemv: the operands and variant as for halo_mi_gemv, except that y may be NULL (the logits are
 *   not kept). With the SLAB layout and variant 0, 2 or 4 the argmax is fused into the slab
 *   GEMV (any n_vec); the GGUF reference kernel and the MFMA GEMM variants (1, 3, 5) rank the
 *   logits afterwards and need y.
 * result: n_vec triples of uint32 {index, value bits, poisoned} (HALO_MI_ARGMAX_RESULT_BYTES
 *   each, 4-byte aligned), as kArgmaxResultBytes (backend.h:430-431).
 * ids (optional): n_vec int32 winning indices, 0 for a poisoned vector or one with no ranked row.
 * ids_slots / ids_scatter (optional, both or neither, only with ids): vector t's id is also
 *   written to ids_scatter[ids_slots[t]]; a slot at or past ids_scatter_len is not written.
 * None of result, ids, ids_scatter may overlap x, w, y or each other.
 */
#define HALO_MI_ARGMAX_RESULT_BYTES 12u

typedef struct halo_mi_lm_head_params {
    halo_mi_gemv_params gemv;
    void* result;
    uint32_t valid_rows;
    int32_t* ids;
    const uint32_t* ids_slots;
    int32_t* ids_scatter;
    uint64_t ids_scatter_len;
} halo_mi_lm_head_params;

int halo_mi_lm_head(const halo_mi_lm_head_params* p, void* stream);

/*
 * ARGMAX (ArgmaxArgs, backend.h:463-468; CpuBackend::argmax, src/backend/cpu_backend.cpp:772-783):
 * for each of n_vec rows of n fp32 logits (logits_stride floats apart, 0 = n) the result words
 * {index, value bits, poisoned} of halo_mi_lm_head: the highest value, ties to the lowest index;
 * a NaN poisons its row's words (the CPU backend's Error(Kernel) for it). n >= 1. result may not
 * overlap logits.
 */
int halo_mi_argmax(const float* logits, uint64_t logits_stride, uint32_t n, uint32_t n_vec, void* result, void* stream);

/*
 * SWIGLU: out[r][c] = silu(gate[r][c]) * up[r][c] for rows x cols fp32 (strides in floats,
 * 0 = cols). The reference's op (backends/cpu/ops_basic.cpp:165-167, EltwiseArgs at
 * include/halo/backend/backend.h:420-427). out may not overlap gate or up.
 */
int halo_mi_swiglu(const float* gate, uint64_t gate_stride, const float* up, uint64_t up_stride, float* out,
                   uint64_t out_stride, uint32_t rows, uint32_t cols, void* stream);

/*
 * Dequantize rows [first_row, first_row + n_rows) of W to fp32 (out rows out_stride floats
 * apart, 0 = cols), bit-identical to tensor::dequantize_row (src/tensor/quant.cpp:430-435).
 * Works on both layouts; it shares its unpacking code with the gemv/gemm kernels.
 * The reference counterpart at the backend level is GET_ROWS (backend.h:254-263).
 */
int halo_mi_dequant_rows(uint32_t type, uint32_t layout, const void* w, uint64_t w_stride,
                         uint32_t rows, uint32_t cols, uint32_t first_row, uint32_t n_rows,
                         float* out, uint64_t out_stride, void* stream);

/*
 * GET_ROWS (GetRowsArgs, include/halo/backend/backend.h:254-263; CPU at
 * src/backend/cpu_backend.cpp:284-303; the HIP status word at backends/hip/src/ops.cpp:982-1012):
 * out[i] = dequant(table row ids[i]) for i < n_ids, bit-identical to tensor::dequantize_row.
 *   table: n_rows rows of cols weights in `layout` (GGUF: table_stride bytes apart, 0 =
 *          row_bytes; SLAB: table_stride 0). ids: n_ids int32 on the device.
 *   out: n_ids rows of cols fp32, out_stride floats apart (0 = cols); must not overlap table,
 *        ids or status.
 *   status (optional, one uint32 on the device): an id outside [0, n_rows) leaves its output
 *        row unwritten and sets HALO_MI_STATUS_BAD_INDEX (the reference's kStatusBadIndex,
 *        backends/hip/kernels/hd.h:156) in it. Ids live on the device, so this is where the CPU
 *        backend's Error(Kernel) shows: read the word after the stream is done.
 *   status_keep: 0 = the call clears the word first (it reports this call only); otherwise the
 *        bits accumulate over calls until the caller clears the word (a stream's report up to
 *        its next wait).
 */
#define HALO_MI_STATUS_BAD_INDEX 8u

typedef struct halo_mi_get_rows_params {
    uint32_t type;
    uint32_t layout;
    const void* table;
    uint64_t table_stride;
    uint32_t n_rows;
    uint32_t cols;
    const int32_t* ids;
    uint32_t n_ids;
    float* out;
    uint64_t out_stride;
    uint32_t* status;
    uint32_t status_keep;
} halo_mi_get_rows_params;

int halo_mi_get_rows(const halo_mi_get_rows_params* p, void* stream);

/*
 * RMS_NORM (RmsNormArgs, backend.h:267-272; cpu::rms_norm, backends/cpu/ops_basic.cpp:18-33):
 * out[r] = (x[r] * inv) * w with inv = 1 / sqrt(dot(x[r], x[r]) / cols + eps), bitwise equal to
 * the CPU (the sum of squares in cpu::detail::dot's order). rows x cols fp32, strides in floats
 * (0 = cols); out may be x itself with the same stride, or must not overlap x or w. This is the
 * normalization halo_mi_gemv's fused norm applies for the reference and GEMM variants.
 */
int halo_mi_rms_norm(const float* x, uint64_t x_stride, const float* w, float* out, uint64_t out_stride,
                     uint32_t rows, uint32_t cols, float eps, void* stream);

/* ---- attention over an 8-bit paged cache ---------------------------------------------------- */
/*
 * What a layer runs between its q / k / v projections and its output projection, and what a server
 * runs between steps: PARTIAL_ROPE (RopeArgs), KV_WRITE (KvWriteArgs) and ATTENTION (AttentionArgs)
 * of the reference's interface (backend.h:369-418) over batches of sequences, with the cache held in
 * 8 bits (KvType::Q8, backend.h:68-75) in a layout of this library's own.
 *
 * Element types (`type`) of q, k, v and out: HALO_MI_F32, HALO_MI_F16, HALO_MI_BF16. Strides count
 * elements; a stride of 0 is the dense one.
 *
 * Device lists (positions, tables, lengths, row starts, slots) are read when the kernel runs, so a
 * captured call follows their values at each replay. What they hold is checked on the device: an
 * entry out of range is never followed; it sets a bit of the optional status word (as in
 * halo_mi_get_rows: cleared by the call unless status_keep).
 */
#define HALO_MI_STATUS_KV_FULL 16u /* a sequence found no free page, or its table no column */

/* The two elements that a rotation takes together, of the first rot_dims of a head. */
enum {
    HALO_MI_ROPE_HALF = 0,       /* i and i + rot_dims / 2 */
    HALO_MI_ROPE_INTERLEAVED = 1 /* 2 i and 2 i + 1 */
};

enum {
    HALO_MI_ROPE_PLAIN = 0,  /* f_i = theta^(-2 i / rot_dims) radians per position */
    HALO_MI_ROPE_LINEAR = 1, /* f_i / scale */
    HALO_MI_ROPE_NTK = 2,    /* theta times scale^(rot_dims / (rot_dims - 2)) */
    HALO_MI_ROPE_YARN = 3    /* f_i / scale for pairs that turn less than beta_slow times over `context` positions, f_i for
                                pairs that turn more than beta_fast times, a linear ramp between; factor 0.1 ln(scale) + 1 */
};

typedef struct halo_mi_rope_scaling {
    uint32_t kind;
    double scale;     /* >= 1 */
    double context;   /* YARN: the positions that the model was trained on */
    double beta_fast; /* YARN: 32 in the usual models */
    double beta_slow; /* YARN: 1 */
} halo_mi_rope_scaling;

/*
 * Host: the rot_dims / 2 frequencies in radians per position, in 64 bits, and the factor that the
 * rotated values are multiplied by (1 but for YARN). A program computes them once per model and keeps
 * the table on the device. scaling may be NULL (PLAIN).
 */
int halo_mi_rope_freqs(uint32_t rot_dims, double theta, const halo_mi_rope_scaling* scaling, double* freqs, float* factor);

/*
 * Rotary positions of q and, in the same launch, k: with a = positions[t] * freqs[i], the pair (x, y)
 * becomes factor * (x cos a - y sin a, y cos a + x sin a); elements from rot_dims on are copied. The
 * angle is reduced in 64 bits, so far positions keep their precision; products are in 32 bits.
 *   parts[0..n_parts): in, out: n_tokens rows of n_heads heads of head_dim elements (n_heads may be 0); out may be in
 *          (same strides), or must not overlap it or any other operand.
 *   rot_dims: even, 2..min(head_dim, 512). freqs: rot_dims / 2 doubles on the device (8-byte aligned).
 *   positions: n_tokens int32 on the device, any value.
 */
typedef struct halo_mi_rope_part {
    const void* in;
    uint64_t in_stride, in_head_stride;
    void* out;
    uint64_t out_stride, out_head_stride;
    uint32_t n_heads;
} halo_mi_rope_part;

typedef struct halo_mi_rope_params {
    uint32_t type;
    uint32_t pairs;
    const halo_mi_rope_part* parts;
    uint32_t n_parts; /* 1 or 2 */
    uint32_t n_tokens, head_dim, rot_dims;
    const int32_t* positions;
    const double* freqs;
    float factor;
} halo_mi_rope_params;

int halo_mi_rope(const halo_mi_rope_params* p, void* stream);

/*
 * The norm of each head of q and k and the rotary positions in one pass over them: every head x becomes
 *   (x_j / sqrt(sum_j x_j^2 / head_dim + eps)) * norm_w[i][j],
 * which is then rotated as halo_mi_rope does; elements from rot_dims on are normed only. Sums and products are in 32 bits (a head
 * whose squares sum past 2^128 becomes zeros), rounded once to `type` at the end.
 *   rope: as halo_mi_rope takes it, with its checks.
 *   norm_w[i]: head_dim fp32 of part i, or NULL (its heads are rotated only); no output may overlap it.
 *   eps: finite, not negative.
 */
typedef struct halo_mi_norm_rope_params {
    halo_mi_rope_params rope;
    const float* norm_w[2];
    float eps;
} halo_mi_norm_rope_params;

int halo_mi_norm_rope(const halo_mi_norm_rope_params* p, void* stream);

/*
 * The cache: n_pages records of halo_mi_kv_page_bytes() bytes each (pool 16-byte aligned). A page holds
 * block_tokens tokens of every layer:
 *   int8 codes, for each layer: K [head][token][dim], then V [head][dim][token];
 *   then fp32 scales, for each layer: K [head], then V [head]; then padding to a multiple of 128 bytes.
 * A code c stands for c * scale. A scale is 0 (all codes 0) or at least 2^-80; NaN marks a block that
 * was given a value that is not finite, and everything read from it is NaN.
 * head_dim: 64, 96, 128, 192 or 256. block_tokens: 16, 32, 64 or 128.
 */
typedef struct halo_mi_kv_cache {
    void* pool;
    uint32_t n_pages, n_layers, n_kv_heads, head_dim, block_tokens;
} halo_mi_kv_cache;

/* Bytes of a page; 0 on error. */
uint64_t halo_mi_kv_page_bytes(uint32_t n_layers, uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_tokens);

/*
 * A batch of sequences. Rows [row_starts[s], row_starts[s + 1]) of the call's row operands are the LAST
 * tokens of sequence s, which holds kv_lens[s] tokens with them: row i of n stands at position
 * kv_lens[s] - n + i. Rows below row_starts[0] or from row_starts[n_seqs] on belong to no sequence:
 * they are neither read nor written. Token t of s lives in page tables[s * table_stride + t / block_tokens].
 *   tables: n_seqs rows of table_width int32, table_stride apart (0 = table_width).
 *   kv_lens: n_seqs int32. row_starts: n_seqs + 1 int32, not decreasing, at most n_rows. They are cut to [0, n_rows];
 *     where they fall, nothing outside the operands is touched, but rows are several sequences', and hold one's results.
 *   max_rows, max_kv: the most rows and tokens of a sequence, as the host knows them (0: n_rows, and
 *     table_width * block_tokens). They shape the launch; larger values than these on the device are still
 *     computed whole, only slower. Attention of a decode batch needs max_rows to be fast: as the rows of one sequence, which 0 takes
 *     them for, they go the way of prompts (48 sequences of one row: 276 us, with max_rows 1 86).
 */
typedef struct halo_mi_kv_batch {
    const int32_t* tables;
    uint64_t table_stride;
    uint32_t table_width;
    const int32_t* kv_lens;
    const int32_t* row_starts;
    uint32_t n_seqs, n_rows;
    uint32_t max_rows, max_kv;
} halo_mi_kv_batch;

/*
 * KV_WRITE: the batch's rows of k and v (n_rows rows of n_kv_heads heads of head_dim) into the sequences'
 * pages of `layer`. Per (page, K or V, head), with amax over the rows that fall into the page:
 *   scale' = max(scale, amax / 127), rounded to fp32; scale counts as 0 where the first row is the
 *            page's first token; an amax / 127 below 2^-80 counts as 0;
 *   code   = x / scale' rounded to the nearest integer, ties to even (0 where scale' is 0);
 *   codes of the page's earlier tokens become code * scale / scale', rounded the same way, where the scale grew.
 * A value that is not finite makes the scale NaN. Tokens of the page behind the last row keep their
 * bytes. Every page that a call writes must belong to one sequence of the batch, in one place of its table.
 * Rows at negative positions (more rows than kv_lens) are not written. A page id outside [0, n_pages), or a
 * token past the table's columns, is not written and sets HALO_MI_STATUS_BAD_INDEX.
 */
typedef struct halo_mi_kv_write_params {
    uint32_t type;
    halo_mi_kv_cache cache;
    uint32_t layer;
    halo_mi_kv_batch batch;
    const void* k;
    uint64_t k_stride, k_head_stride;
    const void* v;
    uint64_t v_stride, v_head_stride;
    uint32_t* status;
    uint32_t status_keep;
} halo_mi_kv_write_params;

int halo_mi_kv_write(const halo_mi_kv_write_params* p, void* stream);

/*
 * The values that the cache holds for the batch's rows: code * scale in fp32, k_out and v_out n_rows
 * rows of n_kv_heads heads of head_dim floats (either may be NULL). Rows at negative positions are zeros; rows in a
 * page out of range are NaN and set HALO_MI_STATUS_BAD_INDEX. k_out and v_out may lie side by side in rows of one stride.
 */
typedef struct halo_mi_kv_read_params {
    halo_mi_kv_cache cache;
    uint32_t layer;
    halo_mi_kv_batch batch;
    float* k_out;
    uint64_t k_stride, k_head_stride;
    float* v_out;
    uint64_t v_stride, v_head_stride;
    uint32_t* status;
    uint32_t status_keep;
} halo_mi_kv_read_params;

int halo_mi_kv_read(const halo_mi_kv_read_params* p, void* stream);

/*
 * ATTENTION of the batch's rows over their sequences' cached tokens:
 *   out[r][h] = sum_t p_t V_t / sum_t p_t, p_t = exp(scale * q[r][h] . K_t), K and V of head h / (n_heads / n_kv_heads),
 * over the tokens t <= position (causal), and t > position - window where window is not 0. A row that sees
 * no token (a negative position) is zeros. q and out are n_rows rows of n_heads heads of head_dim; n_heads is
 * a multiple of n_kv_heads. A row of q that is not finite, and a row that sees a NaN block or a page out of
 * range, is NaN; tokens that a row does not see never reach it, whatever their bytes are. Pages that no row sees, as those behind
 * a window, may be out of range.
 * Numerics: the codes are exact in the products. q is rounded to 11 bits for 16-bit types (exactly q, but for elements under
 * 2^-28 of their row's largest and for rows all under 2^-112) and carried in two pieces, to within 2^-22, for fp32. The softmax
 * weights are two pieces for fp32, and for F16 where rows are few (decode and verify steps: 16 and fewer rows of q a kv head, and up to
 * four times as many for some shapes), else rounded to 11 bits. Sums and the softmax are in fp32.
 *   scale: 0 = 1 / sqrt(head_dim).
 *   workspace (optional, 16-byte aligned): workspace_bytes of device memory for the partial results of long
 *     sequences, in place of the stream's own workspace. Graphs captured on one stream share that stream's
 *     workspace: give each its own if their replays may overlap. halo_mi_attention_workspace() says what a
 *     call makes use of; with less (or on a capturing stream that has none yet) sequences are split less.
 * out may not overlap q (they may lie side by side in rows of one stride), the pool, the batch's lists or the workspace.
 */
typedef struct halo_mi_attention_params {
    uint32_t type;
    halo_mi_kv_cache cache;
    uint32_t layer;
    halo_mi_kv_batch batch;
    const void* q;
    uint64_t q_stride, q_head_stride;
    void* out;
    uint64_t out_stride, out_head_stride;
    uint32_t n_heads;
    float scale;
    uint32_t window;
    void* workspace;
    uint64_t workspace_bytes;
    uint32_t* status;
    uint32_t status_keep;
} halo_mi_attention_params;

int halo_mi_attention(const halo_mi_attention_params* p, void* stream);
/* The workspace bytes that the call splits as it likes best with (0: none, or an argument out of range). */
uint64_t halo_mi_attention_workspace(const halo_mi_attention_params* p);

/*
 * The pages' owner, kept on the device: how often each page is held (refs, n_pages int32), and each
 * slot's tokens and pages (lens n_slots int32, tables n_slots rows of table_width int32, table_stride apart, 0 =
 * table_width; entries past ceil(len / block_tokens) are not read). A slot is a sequence or is empty (length 0).
 * The calls read and change this state in stream order, with no word from the host: a free page is one with refs
 * 0, and the lowest free ones are given first, in the order of the call's list. A listed slot outside [0,
 * n_slots), one that the list names before, and an id out of range in the place of a page that would be copied or written
 * further (the last one, not full, of a fork's source or of a slot that grows) leave their entry's slot as it is and set
 * HALO_MI_STATUS_BAD_INDEX. An id out of range among whole pages that a fork shares stays what it is in the new slot's table
 * (what reads it gets NaN there, as from the source), one among pages given back becomes -1; both set the bit and are not
 * counted. Where the pages run out, that entry and every later one that needs pages are left as they
 * are and HALO_MI_STATUS_KV_FULL is set; so is an entry whose length does not fit the table's columns.
 * At most HALO_MI_KV_LIST_MAX entries a call, and fewer than 2^32 columns of the entries' tables (or pages of the pool,
 * if it has fewer) together. The calls work in the stream's workspace: replays of graphs captured on one stream must not
 * overlap, and a capturing stream needs its workspace already (E_MEMORY; any earlier call that takes one makes it).
 * It has room for lists and pools of 1 + 5 n + n_pages <= 2^23 (resize, fork) and 2 + 3 n_pages <= 2^23 (compact:
 * 2 796 202 pages); larger ones are E_UNSUPPORTED. A refused call leaves the status word as it is.
 */
#define HALO_MI_KV_LIST_MAX 1024u

typedef struct halo_mi_kv_state {
    int32_t* refs;
    int32_t* lens;
    int32_t* tables;
    uint64_t table_stride;
    uint32_t table_width, n_slots;
} halo_mi_kv_state;

/*
 * Gives slots[i] the length new_lens[i], i < n: grown, it gets pages (their bytes are whatever they were);
 * shrunk, the pages that it no longer needs are released (length 0 frees the slot); their table entries become -1. Where a slot
 * grows behind tokens in a page that another slot holds too, it gets a copy of that page. Pages released by a
 * call are free from the next call on. A negative length is out of range.
 */
int halo_mi_kv_resize(const halo_mi_kv_cache* cache, const halo_mi_kv_state* state, const int32_t* slots,
                      const int32_t* new_lens, uint32_t n, uint32_t* status, uint32_t status_keep, void* stream);

/*
 * dst[i] becomes a copy of src[i], i < n: whole pages are shared (refs + 1), a last page that is not full is
 * copied. dst[i] must be an empty slot (otherwise it is left as it is, HALO_MI_STATUS_BAD_INDEX); sources are
 * read as they were before the call.
 */
int halo_mi_kv_fork(const halo_mi_kv_cache* cache, const halo_mi_kv_state* state, const int32_t* src, const int32_t* dst,
                    uint32_t n, uint32_t* status, uint32_t status_keep, void* stream);

/*
 * Moves the live pages (refs > 0) to the front of the pool: with L of them, the k-th live page at or past L goes
 * to the k-th free place below L, its table entries and its count with it. live (optional, one uint32 on the device) receives L.
 */
int halo_mi_kv_compact(const halo_mi_kv_cache* cache, const halo_mi_kv_state* state, uint32_t* live, void* stream);

/*
 * Copies page src[i] to page dst[i], i < n, all layers. No destination may be named twice or be a source.
 * A pair with an id out of range is skipped and sets HALO_MI_STATUS_BAD_INDEX.
 */
int halo_mi_kv_copy_pages(const halo_mi_kv_cache* cache, const int32_t* src, const int32_t* dst, uint32_t n, uint32_t* status,
                          uint32_t status_keep, void* stream);

/* ---- products of 8-bit integers --------------------------------------------------------------- */
/*
 * Rows held in 8 bits: codes (int8, a row of cols codes and zeros up to the next multiple of 16, rows codes_stride
 * bytes apart, 16-byte aligned) and one fp32 scale each; a code c stands for c * scale. Both operands of halo_mi_gemm_i8 are
 * such rows: x has a row for each token, w one for each output channel.
 */

/*
 * Quantizes rows of x (rows x cols of `type` F32, F16 or BF16, x_stride elements apart, 0 = cols):
 *   scale = max_i |x_i| / 127, rounded to fp32; one below 2^-80 counts as 0;
 *   code  = x / scale rounded to the nearest integer, ties to even (0 where scale is 0).
 * A row with a value that is not finite has scale NaN and codes 0. codes_stride: a multiple of 16, 0 = cols rounded
 * up to 16; the zeros behind a row's codes are written too, what lies between them and the next row is not. codes and
 * scales may not overlap x or each other. cols <= 131071, rows < 2^31.
 */
int halo_mi_quantize_rows(uint32_t type, const void* x, uint64_t x_stride, int8_t* codes, uint64_t codes_stride, float* scales,
                          uint32_t rows, uint32_t cols, void* stream);

/*
 * y[t][n] = x_scales[t] * w_scales[n] * sum_i x[t][i] * w[n][i] for t < n_vec, n < rows, i < cols.
 * The sum is exact (32-bit integers), so a row of y does not depend on the call's other rows; the scales are multiplied in fp32
 * (x_scales[t] * w_scales[n] first, then with the sum rounded to fp32), and the result is rounded once to `type` (F32, F16, BF16).
 *   w, x: int8 codes in rows of cols, as halo_mi_quantize_rows writes them (16-byte aligned; strides in bytes, multiples of 16,
 *     0 = cols rounded up to 16, at most 2^20). The bytes from cols up to the next multiple of 16 are read, and are zeros in x or in
 *     w. Codes of -128 are allowed.
 *   w_scales: rows fp32, x_scales: n_vec fp32, any values.
 *   y: n_vec rows of rows elements, y_stride elements apart (0 = rows); may not overlap the other operands.
 *   cols <= 131071 (the sum fits 32 bits), rows and n_vec < 2^31.
 */
typedef struct halo_mi_gemm_i8_params {
    uint32_t type;
    const int8_t* w;
    uint64_t w_stride;
    const float* w_scales;
    const int8_t* x;
    uint64_t x_stride;
    const float* x_scales;
    void* y;
    uint64_t y_stride;
    uint32_t rows, cols, n_vec;
} halo_mi_gemm_i8_params;

int halo_mi_gemm_i8(const halo_mi_gemm_i8_params* p, void* stream);

/* ---- linear attention ---------------------------------------------------------------------------- */
/*
 * Attention without a softmax over tokens that fade, for batches of sequences. Head h has a state S of k_dim x v_dim
 * fp32 numbers, which holds all of a sequence's past; for a sequence's rows t in order
 *   S <- exp(decay[t][h]) S + k[t][h'] v[t][h]^T,   out[t][h] = scale * S^T q[t][h'],   h' = h / (n_heads / n_k_heads).
 * Prompts run in chunks on the matrix cores, few rows one after another; both follow the same formula.
 *
 * Rows [row_starts[s], row_starts[s + 1]) of the row operands are the next tokens of sequence s, whose state is slot slots[s]
 * of the pool. A sequence without rows is left alone: its slot is not looked at. Rows below row_starts[0] or from row_starts[n_seqs] on are
 * neither read nor written; row_starts that fall are cut as in halo_mi_kv_batch. The lists are read when the kernel runs, so a captured
 * call follows their values at each replay. A slot outside [0, n_slots), or one that an earlier sequence with rows has, gives NaN rows, leaves the
 * state alone and sets HALO_MI_STATUS_BAD_INDEX.
 *   type: F32, F16 or BF16, of q, k, v and out. q, k: n_rows rows of n_k_heads heads of k_dim; v, out: of n_heads heads of v_dim; n_heads
 *     is a multiple of n_k_heads, 4096 at most. Strides in elements, 0 = dense; rows of q, k and v at most 2^24 apart. n_seqs <= 65535.
 *   decay: the logarithm of the factor on the state, fp32: n_rows rows of n_heads, decay_stride elements apart (0 = n_heads), or with
 *     decay_per_head n_heads values that hold for every row. -infinity empties the state; values above 0 are taken as they are.
 *   state: n_slots slots of n_heads x k_dim x v_dim fp32 (16-byte aligned, dense); state_out: where the new states go, of the same
 *     shape; it is state itself, or does not overlap it (the states before the call are kept, as for a verify step that may be
 *     taken back). Slots of state_out that no sequence with rows has keep their bytes.
 *   seq_lens (optional): n_seqs int32, the tokens of each sequence with these rows. Where it is no more than the sequence's rows, the
 *     sequence begins here, and its state is taken as zeros, whatever the slot holds.
 *   k_dim, v_dim: 64, 96, 128, 192 or 256. scale: 0 = 1 / sqrt(k_dim).
 *   max_rows: the most rows of a sequence, as the host knows it (0: n_rows). It chooses how the call runs; more rows on the device are
 *     still computed whole, only slower.
 *   workspace (optional, 16-byte aligned): device memory for the states inside long sequences, in place of the stream's own
 *     workspace. Graphs captured on one stream share that stream's workspace: give each its own if their replays may overlap.
 *     halo_mi_linear_attention_workspace() says what a call makes use of; with less (or on a capturing stream that has none
 *     yet) sequences are split less: the results are as right, and slower.
 * Attention of models whose state only fades and adds; the gated delta rule, whose state takes k times (v - S^T k), is another recurrence.
 * Numerics: the state, the sums and the decays are in 32 bits, the decays' running sums in 64; an output is rounded to its type once. A chunk's state
 * is held with a factor of up to 2^40 either way: k, the state and its products with q are to stay below 2^80, and what lies under
 * 2^-80 may be lost. Where a value of v is not finite, that column of out from its row on, and of the state, has no finite numbers (infinities
 * or NaN); one of k, or a decay of NaN: all columns of the heads that read it, from its row on; one of q: its own row's.
 * out may not overlap any other operand (it may lie beside q, k and v in rows of one stride), state_out none but state.
 */
typedef struct halo_mi_linear_attention_params {
    uint32_t type;
    uint32_t n_heads, n_k_heads, k_dim, v_dim;
    const float* state;
    float* state_out;
    uint32_t n_slots;
    const int32_t* slots;
    const int32_t* row_starts;
    const int32_t* seq_lens;
    uint32_t n_seqs, n_rows, max_rows;
    const void* q;
    uint64_t q_stride, q_head_stride;
    const void* k;
    uint64_t k_stride, k_head_stride;
    const void* v;
    uint64_t v_stride, v_head_stride;
    void* out;
    uint64_t out_stride, out_head_stride;
    const float* decay;
    uint64_t decay_stride;
    uint32_t decay_per_head;
    float scale;
    void* workspace;
    uint64_t workspace_bytes;
    uint32_t* status;
    uint32_t status_keep;
} halo_mi_linear_attention_params;

int halo_mi_linear_attention(const halo_mi_linear_attention_params* p, void* stream);
/* The workspace bytes that the call splits as it likes best with (0: none, or an argument out of range). */
uint64_t halo_mi_linear_attention_workspace(const halo_mi_linear_attention_params* p);

/* ---- stream state --------------------------------------------------------------------------- */
/*
 * The kernels' own failures cannot be returned by the call that enqueued them. A split-K
 * reduction of the SLAB GEMV waits for the partial sums of the slab's other workgroups for a
 * bounded time; if it gives up, the output holds NaN and the stream's status word gets
 * HALO_MI_STATUS_SPLITK_TIMEOUT. halo_mi_stream_check() synchronizes `stream`, reads and clears
 * the word and returns HALO_MI_E_DEVICE when it was set (the reference's device-loss path,
 * Stream::wait() -> Error(Device), backend.h:495-506); the workspace is then reset.
 */
#define HALO_MI_STATUS_SPLITK_TIMEOUT 0x100u
int halo_mi_stream_check(void* stream);

/*
 * Every (device, stream) pair that runs a gemv-family call gets a workspace of device memory
 * (split-K words, GEMM partials and staging, argmax parts, normalized x: about 136 MiB), allocated on the
 * first call. halo_mi_stream_release() synchronizes `stream` and frees its workspace on the
 * current device; call it before destroying the stream. A later call on the stream allocates
 * a new one.
 */
int halo_mi_stream_release(void* stream);

/*
 * Test hook, no counterpart in the reference: with force != 0 every split-K reduction of the
 * SLAB GEMV waits for a tag no partial carries, for spin_limit rounds (0 = the default bound),
 * then gives up as above; force = 0 restores normal operation. The kernels still exit
 * normally. Process-wide; for the failure-path tests only.
 */
int halo_mi_test_splitk_timeout(uint32_t spin_limit, int force);

/*
 * Measurement helper, no reference counterpart: one launch that only reads `bytes` of device
 * memory at p (16 B per load, `unroll` loads of 2/4/8/16 in flight per thread, `workgroups` of
 * 256 threads, grid-stride) and writes nothing (sink, workgroups * 256 uint32, is written only
 * for an input no benchmark uses). Its duration is the single-launch read floor of that many
 * bytes, the bound a GEMV streaming the same bytes cannot beat.
 */
int halo_mi_stream_read(const void* p, uint64_t bytes, uint32_t workgroups, uint32_t unroll, uint32_t* sink, void* stream);

/* ---- geometry ------------------------------------------------------------------------------ */
/* Bytes of one GGUF row of `cols` elements (src/tensor/quant.cpp:411-418); 0 on error. */
uint64_t halo_mi_row_bytes(uint32_t type, uint32_t cols);
/* Bytes of the SLAB image of a rows x cols matrix (rows rounded up to 64); 0 on error. */
uint64_t halo_mi_slab_bytes(uint32_t type, uint32_t rows, uint32_t cols);

/* ---- upload and repack (north-star part (c)) ------------------------------------------------ */
/*
 * Device-side repack: GGUF rows (src_stride bytes apart, any alignment) -> SLAB image.
 * Replaces the reference's load-time repack (src/tensor/repack.cpp:100-124, called from
 * src/models/qwen35.cpp:324-346) with a layout for this backend's kernels.
 */
int halo_mi_repack_slab(uint32_t type, const void* src, uint64_t src_stride, uint32_t rows,
                        uint32_t cols, void* dst, void* stream);
/* Exact inverse on the device: SLAB image -> GGUF rows (dst_stride bytes apart, 0 = dense). */
int halo_mi_unpack_slab(uint32_t type, const void* src, uint32_t rows, uint32_t cols, void* dst,
                        uint64_t dst_stride, void* stream);
/* Host versions of the same two maps (identical bytes). */
int halo_mi_repack_slab_host(uint32_t type, const void* src, uint64_t src_stride, uint32_t rows,
                             uint32_t cols, void* dst);
int halo_mi_unpack_slab_host(uint32_t type, const void* src, uint32_t rows, uint32_t cols,
                             void* dst, uint64_t dst_stride);
/*
 * Model-scale upload: host GGUF rows (e.g. the mmap'd file, GgufFile::tensor_data,
 * src/model/gguf.cpp:540-549) -> SLAB images in device memory, for many tensors in one call.
 * Replaces Backend::import_host_readonly's device copy (src/backend/hip_adapter.cpp:502-515)
 * plus the loader's repack, and builds the row-fused projections of try_make_fused
 * (src/models/qwen35.cpp:253-288; gate|up, q|k|v, beta|alpha) on the way: a tensor's parts are
 * matrices of its type and cols whose rows are concatenated, in order, into one matrix.
 *   parts[i].src: host rows, src_stride bytes apart (0 = row_bytes); any host memory.
 *   dst: device memory of halo_mi_slab_bytes(type, sum of the parts' rows, cols) bytes,
 *        16-byte aligned; destinations must not overlap.
 *   chunk_bytes: rows move in chunks of about this size (0 = 24 MiB for a load of up to 512 MiB
 *     that is not all dense pinned memory, else 64 MiB), whole slabs of one tensor;
 *   host_threads: threads that gather a chunk into pinned memory (0 = up to 8).
 * A three-stage pipeline over 4 chunk slots: the host gathers chunk i + 2 into pinned memory
 * while the copy engine moves chunk i + 1 (on a stream of its own) and `stream` repacks chunk i.
 * Returns after the last chunk has been repacked. The GGUF bytes remain recoverable
 * (halo_mi_unpack_slab).
 */
typedef struct halo_mi_upload_part {
    const void* src;
    uint64_t src_stride;
    uint32_t rows;
} halo_mi_upload_part;

typedef struct halo_mi_upload_tensor {
    uint32_t type;
    uint32_t cols;
    const halo_mi_upload_part* parts;
    uint32_t n_parts;
    void* dst;
} halo_mi_upload_tensor;

int halo_mi_upload_tensors(const halo_mi_upload_tensor* tensors, uint32_t n, uint64_t chunk_bytes,
                           uint32_t host_threads, void* stream);

/*
 * One tensor, one part: halo_mi_upload_tensors with host_threads = 0.
 */
int halo_mi_upload_slab(uint32_t type, const void* host_src, uint64_t src_stride, uint32_t rows,
                        uint32_t cols, void* dst, uint64_t chunk_bytes, void* stream);

/* ---- synthetic inputs (no reference counterpart: the reference has no quantizer) ----------- */
/* Portable SplitMix64 + Box-Muller normal fill: out[i] = mean + std * N(0, 1), seed-determined. */
void halo_mi_fill_normal(uint64_t seed, float* out, uint64_t n, float mean, float std);
/* fp32 -> GGUF blocks for Q4_0 / Q8_0 / Q4_K / Q5_K / Q6_K / IQ4_XS; n must be a multiple of the block size.
 * `threads` = 0 uses all host threads. Deterministic for any thread count. */
int halo_mi_quantize(uint32_t type, const float* src, uint64_t n, void* dst, uint32_t threads);

#ifdef __cplusplus
}
#endif

#endif
