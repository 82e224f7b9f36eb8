// The extern "C" entry points of the 8-bit integer products and of linear attention (include/halo_mi355x.h): argument
// validation with the library's error mapping and the dispatch to the launchers of k_quantize.hip, k_gemm_i8.hip and k_linear.hip.
#include <hip/hip_runtime.h>

#include <cmath>
#include <cstdint>

#include "checks.h"
#include "layer.h"
#include "launch.h"

namespace halo_mi {
namespace {

constexpr uint32_t kMaxI8Cols = 131071;  // 128 * 128 * cols < 2^31

// Rows of 8-bit codes: resolves the dense stride; bytes receives the operand's extent, padding included.
int check_codes(const char* op, const char* name, const int8_t* codes, uint64_t* stride, uint32_t rows, uint32_t cols, uint64_t* bytes) {
    const uint64_t row = (cols + 15ull) / 16 * 16;
    if (*stride == 0) *stride = row;
    if (*stride % 16 || *stride < row || *stride > 1u << 20) return set_error(HALO_MI_E_KERNEL, "%s: %s stride %llu is no multiple of 16 in %llu..2^20", op, name, (unsigned long long)*stride, (unsigned long long)row);
    *bytes = extent(rows, *stride, row);
    return rows ? check_aligned(op, name, codes, 16) : HALO_MI_OK;
}

int check_dim(const char* op, const char* name, uint32_t dim) {
    if (dim != 64 && dim != 96 && dim != 128 && dim != 192 && dim != 256)
        return set_error(HALO_MI_E_UNSUPPORTED, "%s: %s %u is not 64, 96, 128, 192 or 256", op, name, dim);
    return HALO_MI_OK;
}

// The checks of a linear attention call; *nothing: valid, but without rows.
int check_linear(const halo_mi_linear_attention_params* p, LinearArgs* a, bool* nothing) {
    const char* op = "linear_attention";
    if (!p) return set_error(HALO_MI_E_KERNEL, "%s: null params", op);
    int rc;
    if ((rc = check_type(op, p->type)) || (rc = check_dim(op, "k_dim", p->k_dim)) || (rc = check_dim(op, "v_dim", p->v_dim))) return rc;
    if (p->n_k_heads == 0 || p->n_heads == 0 || p->n_heads % p->n_k_heads || p->n_heads > 4096)
        return set_error(HALO_MI_E_KERNEL, "%s: %u heads over %u heads of q and k", op, p->n_heads, p->n_k_heads);
    if (p->n_seqs > 65535) return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u sequences in one call (65535 at most)", op, p->n_seqs);
    if (p->n_rows > 0x7FFFFFFFu) return set_error(HALO_MI_E_KERNEL, "%s: n_rows %u is out of range", op, p->n_rows);
    if (!(std::fabs(p->scale) < INFINITY)) return set_error(HALO_MI_E_KERNEL, "%s: scale is not finite", op);
    const uint32_t size = elem_bytes(p->type);
    a->q = {p->q, p->q_stride, p->q_head_stride};
    a->k = {p->k, p->k_stride, p->k_head_stride};
    a->v = {p->v, p->v_stride, p->v_head_stride};
    a->out = {p->out, p->out_stride, p->out_head_stride};
    Range q{p->q, 0, "q"}, k{p->k, 0, "k"}, v{p->v, 0, "v"}, out{p->out, 0, "out"};
    if ((rc = check_rows(op, "q", a->q, p->n_rows, p->n_k_heads, p->k_dim, size, &q.bytes)) ||
        (rc = check_rows(op, "k", a->k, p->n_rows, p->n_k_heads, p->k_dim, size, &k.bytes)) ||
        (rc = check_rows(op, "v", a->v, p->n_rows, p->n_heads, p->v_dim, size, &v.bytes)) ||
        (rc = check_rows(op, "out", a->out, p->n_rows, p->n_heads, p->v_dim, size, &out.bytes)))
        return rc;
    // the rows of a chunk are addressed with 32 bits
    for (const HeadRows* r : {&a->q, &a->k, &a->v})
        if (p->n_rows > 1 && r->stride > 1u << 24) return set_error(HALO_MI_E_UNSUPPORTED, "%s: a row stride over 2^24 elements", op);
    uint64_t decay_stride = p->decay_per_head ? 0 : p->decay_stride ? p->decay_stride : p->n_heads;
    if (p->decay_per_head && p->decay_stride) return set_error(HALO_MI_E_KERNEL, "%s: a decay stride with one decay per head", op);
    if (!p->decay_per_head && p->n_rows > 1 && (decay_stride < p->n_heads || decay_stride > 1ull << 40))
        return set_error(HALO_MI_E_KERNEL, "%s: decay stride %llu is out of range", op, (unsigned long long)decay_stride);
    if (p->workspace && reinterpret_cast<uintptr_t>(p->workspace) % 16) return set_error(HALO_MI_E_KERNEL, "%s: workspace must be 16-byte aligned", op);
    *nothing = p->n_seqs == 0 || p->n_rows == 0;
    a->decay = p->decay;
    a->decay_stride = decay_stride;
    a->state = p->state;
    a->state_out = p->state_out;
    a->slots = p->slots;
    a->row_starts = p->row_starts;
    a->seq_lens = p->seq_lens;
    a->n_slots = p->n_slots;
    a->n_seqs = p->n_seqs;
    a->n_rows = p->n_rows;
    a->max_rows = p->max_rows == 0 || p->max_rows > p->n_rows ? p->n_rows : p->max_rows;
    a->heads = p->n_heads;
    a->group = p->n_heads / p->n_k_heads;
    a->k_dim = p->k_dim;
    a->v_dim = p->v_dim;
    a->scale = p->scale == 0.0f ? 1.0f / std::sqrt((float)p->k_dim) : p->scale;
    a->status = p->status;
    const uint64_t slot = 4ull * p->n_heads * p->k_dim * p->v_dim, pool = (uint64_t)p->n_slots * slot;
    if (p->n_slots > 0x7FFFFFFFu || pool > 1ull << 56) return set_error(HALO_MI_E_KERNEL, "%s: n_slots %u is out of range", op, p->n_slots);
    const Range state{p->state, pool, "state"}, state_out{p->state_out, pool, "state_out"}, ws{p->workspace, p->workspace ? p->workspace_bytes : 0, "the workspace"},
        slots{p->slots, 4ull * p->n_seqs, "slots"}, starts{p->row_starts, 4ull * p->n_seqs + 4, "row_starts"},
        lens{p->seq_lens, p->seq_lens ? 4ull * p->n_seqs : 0, "seq_lens"},
        decay{p->decay, p->decay_per_head ? 4ull * p->n_heads : extent(p->n_rows, decay_stride * 4, 4ull * p->n_heads), "decay"};
    if (!*nothing) {
        if ((rc = check_aligned(op, "state", p->state, 16)) || (rc = check_aligned(op, "state_out", p->state_out, 16)) ||
            (rc = check_aligned(op, "slots", p->slots, 4)) || (rc = check_aligned(op, "row_starts", p->row_starts, 4)) ||
            (rc = check_aligned(op, "decay", p->decay, 4)))
            return rc;
        if (p->seq_lens && (rc = check_aligned(op, "seq_lens", p->seq_lens, 4))) return rc;
        if (p->n_slots == 0) return set_error(HALO_MI_E_KERNEL, "%s: no slots", op);
        if (!apart_in_rows(a->out, p->n_heads, a->q, p->n_k_heads, p->v_dim, p->k_dim, size, out, q) ||
            !apart_in_rows(a->out, p->n_heads, a->k, p->n_k_heads, p->v_dim, p->k_dim, size, out, k) ||
            !apart_in_rows(a->out, p->n_heads, a->v, p->n_heads, p->v_dim, p->v_dim, size, out, v))
            return set_error(HALO_MI_E_KERNEL, "%s: out overlaps q, k or v", op);
        if ((rc = check_apart(op, out, {state, state_out, ws, slots, starts, lens, decay}))) return rc;
        if ((rc = check_apart(op, state_out, {q, k, v, ws, slots, starts, lens, decay}))) return rc;
        if (p->state_out != p->state && (rc = check_apart(op, state_out, {state}))) return rc;
        if ((rc = check_apart(op, ws, {q, k, v, state, slots, starts, lens, decay}))) return rc;
    }
    return check_status(op, p->status, {q, k, v, out, state, state_out, ws, slots, starts, lens, decay});
}

}  // namespace
}  // namespace halo_mi

using namespace halo_mi;

extern "C" {

int halo_mi_quantize_rows(uint32_t type, const void* x, uint64_t x_stride, int8_t* codes, uint64_t codes_stride, float* scales, uint32_t rows,
                          uint32_t cols, void* stream) {
    clear_error();
    const char* op = "quantize_rows";
    int rc;
    if ((rc = check_type(op, type))) return rc;
    if (cols == 0 || cols > kMaxI8Cols) return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u columns (1..%u)", op, cols, kMaxI8Cols);
    if (rows > 0x7FFFFFFFu) return set_error(HALO_MI_E_KERNEL, "%s: rows %u is out of range", op, rows);
    const uint32_t size = elem_bytes(type);
    QuantizeArgs a{x, x_stride ? x_stride : cols, codes, codes_stride, scales, rows, cols};
    Range out{codes, 0, "codes"};
    if ((rc = check_codes(op, "codes", codes, &a.codes_stride, rows, cols, &out.bytes))) return rc;
    if (rows == 0) return HALO_MI_OK;
    if ((rc = check_aligned(op, "x", x, size)) || (rc = check_aligned(op, "scales", scales, 4))) return rc;
    if (rows > 1 && (a.x_stride < cols || a.x_stride > 1ull << 28)) return set_error(HALO_MI_E_KERNEL, "%s: x stride %llu is out of range", op, (unsigned long long)a.x_stride);
    const Range in{x, extent(rows, a.x_stride * size, (uint64_t)cols * size), "x"}, sc{scales, 4ull * rows, "scales"};
    if ((rc = check_apart(op, out, {in, sc})) || (rc = check_apart(op, sc, {in}))) return rc;
    return launch_quantize_rows(type, a, static_cast<hipStream_t>(stream));
}

int halo_mi_gemm_i8(const halo_mi_gemm_i8_params* p, void* stream) {
    clear_error();
    const char* op = "gemm_i8";
    int rc;
    if (!p) return set_error(HALO_MI_E_KERNEL, "%s: null params", op);
    if ((rc = check_type(op, p->type))) return rc;
    if (p->cols == 0 || p->cols > kMaxI8Cols) return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u columns (1..%u)", op, p->cols, kMaxI8Cols);
    if (p->rows > 0x7FFFFFFFu || p->n_vec > 0x7FFFFFFFu) return set_error(HALO_MI_E_KERNEL, "%s: %u rows, %u vectors", op, p->rows, p->n_vec);
    uint64_t ws = p->w_stride, xs = p->x_stride;
    Range w{p->w, 0, "w"}, x{p->x, 0, "x"};
    if ((rc = check_codes(op, "w", p->w, &ws, p->rows, p->cols, &w.bytes)) || (rc = check_codes(op, "x", p->x, &xs, p->n_vec, p->cols, &x.bytes))) return rc;
    const uint32_t size = elem_bytes(p->type);
    const uint64_t ys = p->y_stride ? p->y_stride : p->rows;
    if (p->rows == 0 || p->n_vec == 0) return HALO_MI_OK;
    if ((rc = check_aligned(op, "y", p->y, size)) || (rc = check_aligned(op, "w_scales", p->w_scales, 4)) || (rc = check_aligned(op, "x_scales", p->x_scales, 4)))
        return rc;
    if (p->n_vec > 1 && (ys < p->rows || ys > 1ull << 32)) return set_error(HALO_MI_E_KERNEL, "%s: y stride %llu is out of range", op, (unsigned long long)ys);
    const Range y{p->y, extent(p->n_vec, ys * size, (uint64_t)p->rows * size), "y"};
    if ((rc = check_apart(op, y, {w, x, {p->w_scales, 4ull * p->rows, "w_scales"}, {p->x_scales, 4ull * p->n_vec, "x_scales"}}))) return rc;
    const GemmI8Args a{p->w, p->x, p->w_scales, p->x_scales, p->y, ys, (uint32_t)ws, (uint32_t)xs, p->rows, p->cols, p->n_vec};
    return launch_gemm_i8(p->type, a, static_cast<hipStream_t>(stream));
}

int halo_mi_linear_attention(const halo_mi_linear_attention_params* p, void* stream) {
    clear_error();
    LinearArgs a{};
    bool nothing = false;
    int rc;
    if ((rc = check_linear(p, &a, &nothing))) return rc;
    auto st = static_cast<hipStream_t>(stream);
    float* part = static_cast<float*>(p->workspace);
    uint64_t bytes = p->workspace ? p->workspace_bytes : 0;
    if (!part && !nothing && plan_linear(a, ~0ull)) {
        Workspace* w = nullptr;
        if ((rc = workspace_for(st, &w))) return rc;
        if (w) part = w->partials, bytes = kPartialFloats * sizeof(float);
    }
    if ((rc = clear_status(p->status, p->status_keep, st))) return rc;
    return nothing ? HALO_MI_OK : launch_linear(p->type, a, part, bytes, st);
}

uint64_t halo_mi_linear_attention_workspace(const halo_mi_linear_attention_params* p) {
    clear_error();
    LinearArgs a{};
    bool nothing = false;
    if (check_linear(p, &a, &nothing) || nothing) return 0;
    return plan_linear(a, ~0ull);
}

}  // extern "C"
