// The extern "C" entry points of attention over the 8-bit paged cache (include/halo_mi355x.h): argument
// validation with the library's error mapping, geometry, the rotary frequencies, and the dispatch to
// the launchers of k_rope.hip, k_kv.hip, k_kv_pages.hip and k_attention.hip.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>

#include "kv.h"
#include "launch.h"

namespace halo_mi {
namespace {

// A range of an operand, for the overlap checks.
struct Range {
    const void* p;
    uint64_t bytes;
    const char* name;
};

int check_apart(const char* op, const Range& out, std::initializer_list<Range> others) {
    for (const Range& r : others)
        if (ranges_overlap(out.p, out.bytes, r.p, r.bytes)) return set_error(HALO_MI_E_KERNEL, "%s: %s overlaps %s", op, out.name, r.name);
    return HALO_MI_OK;
}

uint32_t elem_bytes(uint32_t type) { return type == HALO_MI_F32 ? 4 : type == HALO_MI_F16 || type == HALO_MI_BF16 ? 2 : 0; }

int check_type(const char* op, uint32_t type) {
    if (elem_bytes(type) == 0) return set_error(HALO_MI_E_UNSUPPORTED, "%s: element type %u is not F32, F16 or BF16", op, type);
    return HALO_MI_OK;
}

// Rows of heads: resolves the dense strides, checks alignment and that heads and rows do not overlap.
// bytes receives the operand's extent.
int check_rows(const char* op, const char* name, HeadRows& r, uint64_t rows, uint32_t heads, uint32_t dim, uint32_t size, uint64_t* bytes) {
    if (r.head_stride == 0) r.head_stride = dim;
    const uint64_t row = (uint64_t)(heads ? heads - 1 : 0) * r.head_stride + dim;
    if (r.stride == 0) r.stride = (uint64_t)heads * r.head_stride;
    *bytes = 0;
    if (rows == 0 || heads == 0) return HALO_MI_OK;
    if (!r.data) return set_error(HALO_MI_E_KERNEL, "%s: operand %s is empty", op, name);
    if (r.head_stride > 1ull << 40 || r.stride > 1ull << 40 || (rows > 1 && r.stride > (1ull << 58) / rows)) return set_error(HALO_MI_E_KERNEL, "%s: a stride of %s is out of range", op, name);
    if (heads > 1 && r.head_stride < dim) return set_error(HALO_MI_E_KERNEL, "%s: %s head stride < %u elements", op, name, dim);
    // rows may lie inside the heads' stride (a layout [head][row][dim]) or around them
    if (rows > 1 && r.stride < row && !(r.stride >= dim && (heads == 1 || r.head_stride >= (rows - 1) * r.stride + dim)))
        return set_error(HALO_MI_E_KERNEL, "%s: %s row stride %llu lets rows overlap", op, name, (unsigned long long)r.stride);
    if (reinterpret_cast<uintptr_t>(r.data) % size) return set_error(HALO_MI_E_KERNEL, "%s: %s must be %u-byte aligned", op, name, size);
    *bytes = ((rows - 1) * r.stride + row) * size;
    return HALO_MI_OK;
}

// Whether two operands share no element: their ranges are apart, or they lie side by side in rows of one
// stride (q and k of a row-fused projection).
bool apart_in_rows(const HeadRows& x, uint32_t x_heads, const HeadRows& y, uint32_t y_heads, uint32_t dim, uint32_t size, const Range& xr,
                   const Range& yr) {
    if (!ranges_overlap(xr.p, xr.bytes, yr.p, yr.bytes)) return true;
    const uint64_t row = x.stride * size;
    const uint64_t x_row = ((uint64_t)(x_heads - 1) * x.head_stride + dim) * size, y_row = ((uint64_t)(y_heads - 1) * y.head_stride + dim) * size;
    if (x.stride != y.stride || x_row > row || y_row > row) return false;
    const auto px = reinterpret_cast<uintptr_t>(x.data), py = reinterpret_cast<uintptr_t>(y.data);
    const uint64_t off = py >= px ? (py - px) % row : (row - (px - py) % row) % row;  // of y's rows behind x's
    return off >= x_row && off + y_row <= row;
}

int check_aligned(const char* op, const char* name, const void* p, uint32_t to) {
    if (!p) return set_error(HALO_MI_E_KERNEL, "%s: operand %s is empty", op, name);
    if (reinterpret_cast<uintptr_t>(p) % to) return set_error(HALO_MI_E_KERNEL, "%s: %s must be %u-byte aligned", op, name, to);
    return HALO_MI_OK;
}

uint64_t page_bytes_of(uint32_t layers, uint32_t heads, uint32_t dim, uint32_t block) {
    if (dim != 64 && dim != 96 && dim != 128 && dim != 192 && dim != 256) return 0;
    if (block != 16 && block != 32 && block != 64 && block != 128) return 0;
    if (layers == 0 || layers > 4096 || heads == 0 || heads > 1024) return 0;
    const uint64_t units = 2ull * layers * heads, bytes = units * block * dim + 4 * units;
    return bytes > 0x40000000u ? 0 : (bytes + 127) / 128 * 128;  // offsets inside a page fit 32 bits
}

int check_cache(const char* op, const halo_mi_kv_cache& c, uint64_t* page_bytes) {
    *page_bytes = page_bytes_of(c.n_layers, c.n_kv_heads, c.head_dim, c.block_tokens);
    if (*page_bytes == 0)
        return set_error(HALO_MI_E_UNSUPPORTED, "%s: no cache of %u layers, %u heads of %u, %u tokens a page", op, c.n_layers,
                         c.n_kv_heads, c.head_dim, c.block_tokens);
    if (c.n_pages == 0 || c.n_pages > 0x7FFFFFFFu) return set_error(HALO_MI_E_KERNEL, "%s: n_pages %u is out of range", op, c.n_pages);
    return check_aligned(op, "the pool", c.pool, 16);
}

int check_layer(const char* op, const halo_mi_kv_cache& c, uint32_t layer, KvLayer* out) {
    if (int rc = check_cache(op, c, &out->page_bytes)) return rc;
    if (layer >= c.n_layers) return set_error(HALO_MI_E_KERNEL, "%s: layer %u of %u", op, layer, c.n_layers);
    out->pool = static_cast<uint8_t*>(c.pool);
    out->n_pages = c.n_pages;
    out->heads = c.n_kv_heads;
    out->dim = c.head_dim;
    out->block = c.block_tokens;
    out->block_log2 = (uint32_t)__builtin_ctz(c.block_tokens);
    out->plane = c.block_tokens * c.head_dim;
    out->codes = layer * 2 * c.n_kv_heads * out->plane;
    out->scales = c.n_layers * 2 * c.n_kv_heads * out->plane + layer * 2 * c.n_kv_heads * 4;
    return HALO_MI_OK;
}

uint64_t pool_bytes(const KvLayer& c) { return (uint64_t)c.n_pages * c.page_bytes; }

int check_batch(const char* op, const halo_mi_kv_batch& b, const KvLayer& c, KvBatch* out) {
    const uint64_t stride = b.table_stride ? b.table_stride : b.table_width;
    if (b.n_seqs > 65535) return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u sequences in one call (65535 at most)", op, b.n_seqs);
    if (b.n_rows > 0x7FFFFFFFu) return set_error(HALO_MI_E_KERNEL, "%s: n_rows %u is out of range", op, b.n_rows);
    if (b.n_seqs > 1 && stride < b.table_width) return set_error(HALO_MI_E_KERNEL, "%s: table stride < table width", op);
    if (stride > 1ull << 40) return set_error(HALO_MI_E_KERNEL, "%s: the table stride is out of range", op);
    if (b.table_width == 0 || (uint64_t)b.table_width * c.block > 0x7FFFFF00u)
        return set_error(HALO_MI_E_KERNEL, "%s: table width %u is out of range", op, b.table_width);
    *out = {b.tables, stride, b.kv_lens, b.row_starts, b.table_width, b.n_seqs, b.n_rows, b.max_rows, b.max_kv};
    if (out->max_rows == 0 || out->max_rows > b.n_rows) out->max_rows = b.n_rows;
    const uint32_t cap = b.table_width * c.block;
    if (out->max_kv == 0 || out->max_kv > cap) out->max_kv = cap;
    if (b.n_seqs == 0 || b.n_rows == 0) return HALO_MI_OK;
    if (int rc = check_aligned(op, "tables", b.tables, 4)) return rc;
    if (int rc = check_aligned(op, "kv_lens", b.kv_lens, 4)) return rc;
    return check_aligned(op, "row_starts", b.row_starts, 4);
}

Range tables_range(const KvBatch& b) { return {b.tables, extent(b.n_seqs, b.table_stride * 4, (uint64_t)b.table_width * 4), "tables"}; }
Range lens_range(const KvBatch& b) { return {b.kv_lens, (uint64_t)b.n_seqs * 4, "kv_lens"}; }
Range starts_range(const KvBatch& b) { return {b.row_starts, ((uint64_t)b.n_seqs + 1) * 4, "row_starts"}; }

// The optional status word is no operand of the call. It is cleared, unless the caller keeps it, once nothing else can refuse the
// call.
int check_status(const char* op, uint32_t* status, std::initializer_list<Range> others) {
    if (!status) return HALO_MI_OK;
    if (reinterpret_cast<uintptr_t>(status) % 4) return set_error(HALO_MI_E_KERNEL, "%s: status must be 4-byte aligned", op);
    return check_apart(op, {status, 4, "status"}, others);
}
int clear_status(uint32_t* status, uint32_t keep, hipStream_t st) { return status && !keep ? launch_fill_u32(status, 1, 0u, st) : HALO_MI_OK; }

// The checks of an attention call; *nothing: valid, but without rows.
int check_attention(const halo_mi_attention_params* p, AttnArgs* a, std::initializer_list<Range*> ranges) {
    const char* op = "ATTENTION";
    if (!p) return set_error(HALO_MI_E_KERNEL, "%s: null params", op);
    int rc;
    if ((rc = check_type(op, p->type))) return rc;
    if ((rc = check_layer(op, p->cache, p->layer, &a->c))) return rc;
    if ((rc = check_batch(op, p->batch, a->c, &a->b))) return rc;
    if (p->n_heads == 0 || p->n_heads % p->cache.n_kv_heads || p->n_heads > 65536)
        return set_error(HALO_MI_E_KERNEL, "%s: %u heads over %u kv heads", op, p->n_heads, p->cache.n_kv_heads);
    if (!(std::fabs(p->scale) < INFINITY)) return set_error(HALO_MI_E_KERNEL, "%s: scale is not finite", op);
    a->q = {p->q, p->q_stride, p->q_head_stride};
    a->out = {p->out, p->out_stride, p->out_head_stride};
    const uint32_t size = elem_bytes(p->type);
    Range q{p->q, 0, "q"}, out{p->out, 0, "out"};
    if ((rc = check_rows(op, "q", a->q, p->batch.n_rows, p->n_heads, p->cache.head_dim, size, &q.bytes))) return rc;
    if ((rc = check_rows(op, "out", a->out, p->batch.n_rows, p->n_heads, p->cache.head_dim, size, &out.bytes))) return rc;
    if ((uint64_t)p->batch.n_rows * p->n_heads > 0x7FFFFFFFull)
        return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u rows of %u heads in one call", op, p->batch.n_rows, p->n_heads);
    if (p->workspace && reinterpret_cast<uintptr_t>(p->workspace) % 16)
        return set_error(HALO_MI_E_KERNEL, "%s: workspace must be 16-byte aligned", op);
    a->type = p->type;
    a->heads = p->n_heads;
    a->group = p->n_heads / p->cache.n_kv_heads;
    if ((uint64_t)p->batch.n_seqs * p->cache.n_kv_heads > 1u << 22)
        return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u sequences of %u kv heads in one call", op, p->batch.n_seqs, p->cache.n_kv_heads);
    a->window = p->window < 0x7FFFFFFFu ? p->window : 0;  // more than any table holds
    const float scale = p->scale == 0.0f ? 1.0f / std::sqrt((float)p->cache.head_dim) : p->scale;
    a->scale_log2 = (float)(scale * 1.4426950408889634);
    a->part = nullptr;
    a->status = p->status;
    const Range* found[] = {&q, &out};
    size_t i = 0;
    for (Range* r : ranges) *r = *found[i++];
    return HALO_MI_OK;
}

int check_state(const char* op, const halo_mi_kv_cache* cache, const halo_mi_kv_state* s, KvPagesArgs* a) {
    if (!cache || !s) return set_error(HALO_MI_E_KERNEL, "%s: null params", op);
    int rc;
    if ((rc = check_cache(op, *cache, &a->page_bytes))) return rc;
    const uint64_t stride = s->table_stride ? s->table_stride : s->table_width;
    if (s->n_slots == 0 || s->n_slots > 0x7FFFFFFFu) return set_error(HALO_MI_E_KERNEL, "%s: n_slots %u is out of range", op, s->n_slots);
    if (s->table_width == 0 || (uint64_t)s->table_width * cache->block_tokens > 0x7FFFFF00u || stride > (1ull << 58) / s->n_slots ||
        (s->n_slots > 1 && stride < s->table_width))
        return set_error(HALO_MI_E_KERNEL, "%s: table width %u or its stride is out of range", op, s->table_width);
    if ((rc = check_aligned(op, "refs", s->refs, 4)) || (rc = check_aligned(op, "lens", s->lens, 4)) ||
        (rc = check_aligned(op, "tables", s->tables, 4)))
        return rc;
    a->pool = static_cast<uint8_t*>(cache->pool);
    a->n_pages = cache->n_pages;
    a->block = cache->block_tokens;
    a->refs = s->refs;
    a->lens = s->lens;
    a->tables = s->tables;
    a->table_stride = stride;
    a->table_width = s->table_width;
    a->n_slots = s->n_slots;
    const Range pool{a->pool, a->n_pages * a->page_bytes, "the pool"}, refs{a->refs, 4ull * a->n_pages, "refs"},
        lens{a->lens, 4ull * a->n_slots, "lens"},
        tables{a->tables, extent(a->n_slots, stride * 4, (uint64_t)a->table_width * 4), "tables"};
    if ((rc = check_apart(op, refs, {pool, lens, tables})) || (rc = check_apart(op, lens, {pool, tables}))) return rc;
    return check_apart(op, tables, {pool});
}

Range tables_range(const KvPagesArgs& a) {
    return {a.tables, extent(a.n_slots, a.table_stride * 4, (uint64_t)a.table_width * 4), "tables"};
}

// A listed call's lists: n int32 each, apart from what the call changes.
int check_lists(const char* op, const KvPagesArgs& a, const int32_t* x, const int32_t* y, uint32_t n) {
    int rc;
    if (n > HALO_MI_KV_LIST_MAX) return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u entries in one call (%u at most)", op, n, HALO_MI_KV_LIST_MAX);
    // what the entries ask for together is summed in 32 bits
    if ((uint64_t)n * (std::min(a.table_width, a.n_pages) + 2ull) > 0xFFFFFFFFull)
        return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u entries of %u columns in one call", op, n, a.table_width);
    if (n == 0) return HALO_MI_OK;
    if ((rc = check_aligned(op, "a list", x, 4)) || (rc = check_aligned(op, "a list", y, 4))) return rc;
    for (const int32_t* l : {x, y})
        if ((rc = check_apart(op, {l, 4ull * n, "a list"},
                              {{a.pool, a.n_pages * a.page_bytes, "the pool"},
                               {a.refs, 4ull * a.n_pages, "refs"},
                               {a.lens, 4ull * a.n_slots, "lens"},
                               tables_range(a)})))
            return rc;
    return HALO_MI_OK;
}

// `words` of scratch from the stream's workspace.
int scratch_for(const char* op, hipStream_t st, uint64_t words, uint32_t** out) {
    if (words > kPartialFloats) return set_error(HALO_MI_E_UNSUPPORTED, "%s: the pool has too many pages for the scratch memory", op);
    Workspace* w = nullptr;
    if (int rc = workspace_for(st, &w)) return rc;
    if (!w) return set_error(HALO_MI_E_MEMORY, "%s: needs this stream's workspace (make one call on it before capturing)", op);
    *out = reinterpret_cast<uint32_t*>(w->partials);
    return HALO_MI_OK;
}

}  // namespace
}  // namespace halo_mi

using namespace halo_mi;

extern "C" {

int halo_mi_rope_freqs(uint32_t rot_dims, double theta, const halo_mi_rope_scaling* scaling, double* freqs, float* factor) {
    clear_error();
    const char* op = "rope_freqs";
    if (!freqs || !factor) return set_error(HALO_MI_E_KERNEL, "%s: empty operand", op);
    if (rot_dims < 2 || rot_dims % 2 || rot_dims > 512) return set_error(HALO_MI_E_UNSUPPORTED, "%s: rot_dims %u is not even or not in 2..512", op, rot_dims);
    if (!(theta > 1.0) || !std::isfinite(theta)) return set_error(HALO_MI_E_KERNEL, "%s: theta must be finite and above 1", op);
    const halo_mi_rope_scaling none{HALO_MI_ROPE_PLAIN, 1.0, 0.0, 0.0, 0.0}, &s = scaling ? *scaling : none;
    if (s.kind > HALO_MI_ROPE_YARN) return set_error(HALO_MI_E_CONFIG, "%s: unknown scaling %u", op, s.kind);
    if (s.kind != HALO_MI_ROPE_PLAIN && (!(s.scale >= 1.0) || !std::isfinite(s.scale)))
        return set_error(HALO_MI_E_KERNEL, "%s: a scale must be finite and at least 1", op);
    const double rot = rot_dims, pi = 3.14159265358979323846;
    *factor = 1.0f;
    double base = theta, low = 0.0, high = 0.0;
    if (s.kind == HALO_MI_ROPE_NTK && rot_dims > 2) base *= std::pow(s.scale, rot / (rot - 2.0));
    const bool yarn = s.kind == HALO_MI_ROPE_YARN && s.scale > 1.0;
    if (s.kind == HALO_MI_ROPE_YARN) {
        if (!(s.context > 0.0) || !(s.beta_slow > 0.0) || !(s.beta_fast > s.beta_slow) || !std::isfinite(s.context) || !std::isfinite(s.beta_fast))
            return set_error(HALO_MI_E_KERNEL, "%s: YARN needs a context and 0 < beta_slow < beta_fast", op);
        // the pair index that turns `turns` times over the context
        const auto at = [&](double turns) { return rot * std::log(s.context / (turns * 2.0 * pi)) / (2.0 * std::log(theta)); };
        low = std::max(std::floor(at(s.beta_fast)), 0.0);
        high = std::min(std::ceil(at(s.beta_slow)), rot - 1.0);
        if (yarn) *factor = (float)(0.1 * std::log(s.scale) + 1.0);
    }
    for (uint32_t i = 0; i < rot_dims / 2; ++i) {
        const double f = std::pow(base, -2.0 * i / rot);
        if (yarn) {
            const double ramp = std::min(std::max((i - low) / std::max(high - low, 0.001), 0.0), 1.0);
            freqs[i] = f / s.scale * ramp + f * (1.0 - ramp);
        } else {
            freqs[i] = s.kind == HALO_MI_ROPE_LINEAR ? f / s.scale : f;
        }
    }
    return HALO_MI_OK;
}

int halo_mi_rope(const halo_mi_rope_params* p, void* stream) {
    clear_error();
    const char* op = "PARTIAL_ROPE";
    int rc;
    if (!p || !p->parts) return set_error(HALO_MI_E_KERNEL, "%s: null params", op);
    if ((rc = check_type(op, p->type))) return rc;
    if (p->pairs > HALO_MI_ROPE_INTERLEAVED) return set_error(HALO_MI_E_CONFIG, "%s: unknown pairs %u", op, p->pairs);
    if (p->n_parts == 0 || p->n_parts > 2) return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u parts (1 or 2)", op, p->n_parts);
    if (p->head_dim == 0 || p->head_dim > 65536) return set_error(HALO_MI_E_UNSUPPORTED, "%s: head_dim %u", op, p->head_dim);
    if (p->rot_dims < 2 || p->rot_dims % 2 || p->rot_dims > 512 || p->rot_dims > p->head_dim)
        return set_error(HALO_MI_E_KERNEL, "%s: rot_dims %u of %u is not even or not in 2..512", op, p->rot_dims, p->head_dim);
    if (p->n_tokens > 0x7FFFFFFFu) return set_error(HALO_MI_E_KERNEL, "%s: n_tokens %u is out of range", op, p->n_tokens);
    if (!std::isfinite(p->factor)) return set_error(HALO_MI_E_KERNEL, "%s: factor is not finite", op);
    const uint32_t size = elem_bytes(p->type);
    RopeArgs a{};
    Range in[2] = {}, out[2] = {};
    for (uint32_t i = 0; i < p->n_parts; ++i) {
        const halo_mi_rope_part& s = p->parts[i];
        RopePart& d = a.part[i];
        d.heads = s.n_heads;
        if (s.n_heads > 65535) return set_error(HALO_MI_E_UNSUPPORTED, "%s: %u heads", op, s.n_heads);
        d.in = {s.in, s.in_stride, s.in_head_stride};
        d.out = {s.out, s.out_stride, s.out_head_stride};
        in[i] = {s.in, 0, "an input"};
        out[i] = {s.out, 0, "an output"};
        if ((rc = check_rows(op, "in", d.in, p->n_tokens, s.n_heads, p->head_dim, size, &in[i].bytes))) return rc;
        if ((rc = check_rows(op, "out", d.out, p->n_tokens, s.n_heads, p->head_dim, size, &out[i].bytes))) return rc;
        d.in_place = s.in == s.out && d.in.stride == d.out.stride && d.in.head_stride == d.out.head_stride;
        if (!d.in_place && ranges_overlap(in[i].p, in[i].bytes, out[i].p, out[i].bytes))
            return set_error(HALO_MI_E_KERNEL, "%s: out overlaps in", op);
        a.heads += s.n_heads;
    }
    a.n_tokens = p->n_tokens;
    a.dim = p->head_dim;
    a.rot = p->rot_dims;
    a.positions = p->positions;
    a.freqs = p->freqs;
    a.factor = p->factor;
    if (a.n_tokens == 0 || a.heads == 0) return HALO_MI_OK;
    if ((rc = check_aligned(op, "positions", p->positions, 4)) || (rc = check_aligned(op, "freqs", p->freqs, 8))) return rc;
    for (int i = 0; i < 2; ++i) {
        if ((rc = check_apart(op, out[i], {{p->positions, 4ull * a.n_tokens, "positions"}, {p->freqs, 4ull * a.rot, "freqs"}}))) return rc;
        const RopePart &x = a.part[i], &y = a.part[1 - i];
        if (!apart_in_rows(x.out, x.heads, y.in, y.heads, a.dim, size, out[i], in[1 - i]) ||
            !apart_in_rows(x.out, x.heads, y.out, y.heads, a.dim, size, out[i], out[1 - i]))
            return set_error(HALO_MI_E_KERNEL, "%s: an output overlaps the other part", op);
    }
    return launch_rope(p->type, p->pairs, a, static_cast<hipStream_t>(stream));
}

uint64_t halo_mi_kv_page_bytes(uint32_t n_layers, uint32_t n_kv_heads, uint32_t head_dim, uint32_t block_tokens) {
    return page_bytes_of(n_layers, n_kv_heads, head_dim, block_tokens);
}

int halo_mi_kv_write(const halo_mi_kv_write_params* p, void* stream) {
    clear_error();
    const char* op = "KV_WRITE";
    int rc;
    if (!p) return set_error(HALO_MI_E_KERNEL, "%s: null params", op);
    KvWriteArgs a{};
    if ((rc = check_type(op, p->type)) || (rc = check_layer(op, p->cache, p->layer, &a.c)) || (rc = check_batch(op, p->batch, a.c, &a.b))) return rc;
    a.x[0] = {p->k, p->k_stride, p->k_head_stride};
    a.x[1] = {p->v, p->v_stride, p->v_head_stride};
    Range k{p->k, 0, "k"}, v{p->v, 0, "v"};
    const uint32_t size = elem_bytes(p->type);
    if ((rc = check_rows(op, "k", a.x[0], a.b.n_rows, a.c.heads, a.c.dim, size, &k.bytes))) return rc;
    if ((rc = check_rows(op, "v", a.x[1], a.b.n_rows, a.c.heads, a.c.dim, size, &v.bytes))) return rc;
    const Range pool{a.c.pool, pool_bytes(a.c), "the pool"};
    if ((rc = check_apart(op, pool, {k, v, tables_range(a.b), lens_range(a.b), starts_range(a.b)}))) return rc;
    a.status = p->status;
    auto st = static_cast<hipStream_t>(stream);
    if ((rc = check_status(op, p->status, {pool, k, v, tables_range(a.b), lens_range(a.b), starts_range(a.b)}))) return rc;
    if ((rc = clear_status(p->status, p->status_keep, st))) return rc;
    if (a.b.n_seqs == 0 || a.b.n_rows == 0) return HALO_MI_OK;
    return launch_kv_write(p->type, a, st);
}

int halo_mi_kv_read(const halo_mi_kv_read_params* p, void* stream) {
    clear_error();
    const char* op = "kv_read";
    int rc;
    if (!p) return set_error(HALO_MI_E_KERNEL, "%s: null params", op);
    KvReadArgs a{};
    if ((rc = check_layer(op, p->cache, p->layer, &a.c)) || (rc = check_batch(op, p->batch, a.c, &a.b))) return rc;
    a.out[0] = {p->k_out, p->k_stride, p->k_head_stride};
    a.out[1] = {p->v_out, p->v_stride, p->v_head_stride};
    const Range pool{a.c.pool, pool_bytes(a.c), "the pool"};
    Range out[2] = {{p->k_out, 0, "k_out"}, {p->v_out, 0, "v_out"}};
    for (int i = 0; i < 2; ++i)
        if (out[i].p) {
            if ((rc = check_rows(op, out[i].name, a.out[i], a.b.n_rows, a.c.heads, a.c.dim, 4, &out[i].bytes))) return rc;
            if ((rc = check_apart(op, out[i], {pool, tables_range(a.b), lens_range(a.b), starts_range(a.b)}))) return rc;
        }
    if (!apart_in_rows(a.out[0], a.c.heads, a.out[1], a.c.heads, a.c.dim, 4, out[0], out[1]))
        return set_error(HALO_MI_E_KERNEL, "%s: k_out overlaps v_out", op);
    a.status = p->status;
    auto st = static_cast<hipStream_t>(stream);
    if ((rc = check_status(op, p->status, {pool, out[0], out[1], tables_range(a.b), lens_range(a.b), starts_range(a.b)}))) return rc;
    if ((rc = clear_status(p->status, p->status_keep, st))) return rc;
    if (a.b.n_seqs == 0 || a.b.n_rows == 0 || (!p->k_out && !p->v_out)) return HALO_MI_OK;
    return launch_kv_read(a, st);
}

int halo_mi_attention(const halo_mi_attention_params* p, void* stream) {
    clear_error();
    const char* op = "ATTENTION";
    int rc;
    AttnArgs a{};
    Range q, out;
    if ((rc = check_attention(p, &a, {&q, &out}))) return rc;
    const Range pool{a.c.pool, pool_bytes(a.c), "the pool"}, ws{p->workspace, p->workspace ? p->workspace_bytes : 0, "the workspace"};
    if (!apart_in_rows(a.out, a.heads, a.q, a.heads, a.c.dim, elem_bytes(a.type), out, q)) return set_error(HALO_MI_E_KERNEL, "%s: out overlaps q", op);
    if ((rc = check_apart(op, out, {pool, ws, tables_range(a.b), lens_range(a.b), starts_range(a.b)}))) return rc;
    if ((rc = check_apart(op, ws, {q, pool, tables_range(a.b), lens_range(a.b), starts_range(a.b)}))) return rc;
    auto st = static_cast<hipStream_t>(stream);
    if ((rc = check_status(op, p->status, {q, out, pool, ws, tables_range(a.b), lens_range(a.b), starts_range(a.b)}))) return rc;
    const bool nothing = a.b.n_seqs == 0 || a.b.n_rows == 0;
    float* part = static_cast<float*>(p->workspace);
    uint64_t bytes = ws.bytes;
    if (!part && !nothing) {
        Workspace* w = nullptr;
        if ((rc = workspace_for(st, &w))) return rc;
        if (w) part = w->partials, bytes = kPartialFloats * sizeof(float);
    }
    if ((rc = clear_status(p->status, p->status_keep, st))) return rc;
    if (nothing) return HALO_MI_OK;
    if (plan_attention(a, bytes)) a.part = part;
    return launch_attention(a, st);
}

uint64_t halo_mi_attention_workspace(const halo_mi_attention_params* p) {
    clear_error();
    AttnArgs a{};
    Range q, out;
    if (check_attention(p, &a, {&q, &out}) || a.b.n_seqs == 0 || a.b.n_rows == 0) return 0;
    return plan_attention(a, ~0ull);
}

int halo_mi_kv_resize(const halo_mi_kv_cache* cache, const halo_mi_kv_state* state, const int32_t* slots, const int32_t* new_lens, uint32_t n,
                      uint32_t* status, uint32_t status_keep, void* stream) {
    clear_error();
    const char* op = "kv_resize";
    KvPagesArgs a{};
    int rc;
    uint32_t* scratch = nullptr;
    auto st = static_cast<hipStream_t>(stream);
    if ((rc = check_state(op, cache, state, &a)) || (rc = check_lists(op, a, slots, new_lens, n))) return rc;
    if ((rc = check_status(op, status, {{a.refs, 4ull * a.n_pages, "refs"}, {a.lens, 4ull * a.n_slots, "lens"}, tables_range(a), {slots, 4ull * n, "slots"}, {new_lens, 4ull * n, "new_lens"}, {a.pool, a.n_pages * a.page_bytes, "the pool"}}))) return rc;
    if (n && (rc = scratch_for(op, st, 1 + 5ull * n + a.n_pages, &scratch))) return rc;
    if ((rc = clear_status(status, status_keep, st))) return rc;
    return n ? launch_kv_resize(a, slots, new_lens, n, scratch, status, st) : HALO_MI_OK;
}

int halo_mi_kv_fork(const halo_mi_kv_cache* cache, const halo_mi_kv_state* state, const int32_t* src, const int32_t* dst, uint32_t n,
                    uint32_t* status, uint32_t status_keep, void* stream) {
    clear_error();
    const char* op = "kv_fork";
    KvPagesArgs a{};
    int rc;
    uint32_t* scratch = nullptr;
    auto st = static_cast<hipStream_t>(stream);
    if ((rc = check_state(op, cache, state, &a)) || (rc = check_lists(op, a, src, dst, n))) return rc;
    if ((rc = check_status(op, status, {{a.refs, 4ull * a.n_pages, "refs"}, {a.lens, 4ull * a.n_slots, "lens"}, tables_range(a), {src, 4ull * n, "src"}, {dst, 4ull * n, "dst"}, {a.pool, a.n_pages * a.page_bytes, "the pool"}}))) return rc;
    if (n && (rc = scratch_for(op, st, 1 + 5ull * n + a.n_pages, &scratch))) return rc;
    if ((rc = clear_status(status, status_keep, st))) return rc;
    return n ? launch_kv_fork(a, src, dst, n, scratch, status, st) : HALO_MI_OK;
}

int halo_mi_kv_compact(const halo_mi_kv_cache* cache, const halo_mi_kv_state* state, uint32_t* live, void* stream) {
    clear_error();
    const char* op = "kv_compact";
    KvPagesArgs a{};
    int rc;
    uint32_t* scratch = nullptr;
    auto st = static_cast<hipStream_t>(stream);
    if ((rc = check_state(op, cache, state, &a))) return rc;
    if (live) {
        if ((rc = check_aligned(op, "live", live, 4))) return rc;
        if ((rc = check_apart(op, {live, 4, "live"}, {{a.refs, 4ull * a.n_pages, "refs"}, {a.lens, 4ull * a.n_slots, "lens"}, tables_range(a), {a.pool, a.n_pages * a.page_bytes, "the pool"}}))) return rc;
    }
    if ((rc = scratch_for(op, st, 2 + 3ull * a.n_pages, &scratch))) return rc;
    return launch_kv_compact(a, scratch, live, st);
}

int halo_mi_kv_copy_pages(const halo_mi_kv_cache* cache, const int32_t* src, const int32_t* dst, uint32_t n, uint32_t* status, uint32_t status_keep,
                          void* stream) {
    clear_error();
    const char* op = "kv_copy_pages";
    if (!cache) return set_error(HALO_MI_E_KERNEL, "%s: null params", op);
    KvPagesArgs a{};
    int rc;
    auto st = static_cast<hipStream_t>(stream);
    if ((rc = check_cache(op, *cache, &a.page_bytes))) return rc;
    a.pool = static_cast<uint8_t*>(cache->pool);
    a.n_pages = cache->n_pages;
    const Range pool{a.pool, a.n_pages * a.page_bytes, "the pool"};
    if (n) {
        if ((rc = check_aligned(op, "src", src, 4)) || (rc = check_aligned(op, "dst", dst, 4))) return rc;
        if ((rc = check_apart(op, pool, {{src, 4ull * n, "src"}, {dst, 4ull * n, "dst"}}))) return rc;
    }
    if ((rc = check_status(op, status, {pool, {src, 4ull * n, "src"}, {dst, 4ull * n, "dst"}}))) return rc;
    if ((rc = clear_status(status, status_keep, st))) return rc;
    return n ? launch_kv_copy_pages(a, src, dst, n, status, st) : HALO_MI_OK;
}

}  // extern "C"
