// The 8-bit paged cache between its C ABI (kv_api.cpp) and its kernels (k_rope.hip, k_kv.hip,
// k_kv_pages.hip, k_attention.hip): geometry, argument blocks and launchers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "common.h"

namespace halo_mi {

constexpr uint32_t kStatusKvBadIndex = HALO_MI_STATUS_BAD_INDEX;
constexpr uint32_t kStatusKvFull = HALO_MI_STATUS_KV_FULL;
// A scale below this counts as 0: the attention takes the scales' logarithms and reciprocals in fp32.
constexpr float kKvMinScale = 0x1p-80f;

// One layer of the pool, by value in the kernels' arguments. Offsets inside a page fit 32 bits (checked).
struct KvLayer {
    uint8_t* pool;
    uint64_t page_bytes;
    uint32_t n_pages, heads, dim, block, block_log2;
    uint32_t codes;   // byte offset of the layer's K codes in a page; V's follow at codes + heads * plane
    uint32_t scales;  // byte offset of the layer's K scales; V's follow at scales + 4 * heads
    uint32_t plane;   // bytes of one head's K or V codes: block * dim
};

struct KvBatch {
    const int32_t* tables;
    uint64_t table_stride;
    const int32_t* kv_lens;
    const int32_t* row_starts;
    uint32_t table_width, n_seqs, n_rows, max_rows, max_kv;
};

// Rows of heads: element (row, head, i) at row * stride + head * head_stride + i.
struct HeadRows {
    const void* data;
    uint64_t stride, head_stride;
};

struct RopePart {
    HeadRows in;
    HeadRows out;  // data is written
    uint32_t heads;
    bool in_place;
};

struct RopeArgs {
    RopePart part[2];
    uint32_t heads;  // of both parts
    uint32_t n_tokens, dim, rot;
    const int32_t* positions;
    const double* freqs;
    float factor;
};

struct KvWriteArgs {
    KvLayer c;
    KvBatch b;
    HeadRows x[2];  // k, v
    uint32_t* status;
};

struct KvReadArgs {
    KvLayer c;
    KvBatch b;
    HeadRows out[2];  // fp32; data null: not asked for
    uint32_t* status;
};

struct AttnArgs {
    KvLayer c;
    KvBatch b;
    HeadRows q, out;
    uint32_t type, heads, group;  // group: q heads per kv head
    uint32_t window;
    float scale_log2;  // scale * log2(e)
    // How the work is dealt out (plan_attention): workgroups, row tiles of the longest sequence, tokens of a unit;
    // the parts of what several workgroups have meet in `part` (null: nothing is split).
    bool few;
    uint32_t splits, tiles, unit, unit_log2;
    float* part;
    uint32_t* status;
};

struct KvPagesArgs {
    uint8_t* pool;
    uint64_t page_bytes;
    uint32_t n_pages, block;
    int32_t* refs;
    int32_t* lens;
    int32_t* tables;
    uint64_t table_stride;
    uint32_t table_width, n_slots;
};

int launch_rope(uint32_t type, uint32_t pairs, const RopeArgs& a, hipStream_t st);
int launch_kv_write(uint32_t type, const KvWriteArgs& a, hipStream_t st);
int launch_kv_read(const KvReadArgs& a, hipStream_t st);
// How the work is dealt out with part_bytes of partial results; returns the bytes made use of (0: nothing is split). Sets a.few,
// a.splits and a.tiles, and where rows are few a.unit and a.unit_log2.
uint64_t plan_attention(AttnArgs& a, uint64_t part_bytes);
int launch_attention(const AttnArgs& a, hipStream_t st);
// scratch: 1 + 5 n + n_pages words (resize, fork); 2 + 3 n_pages words (compact)
int launch_kv_resize(const KvPagesArgs& a, const int32_t* slots, const int32_t* new_lens, uint32_t n, uint32_t* scratch,
                     uint32_t* status, hipStream_t st);
int launch_kv_fork(const KvPagesArgs& a, const int32_t* src, const int32_t* dst, uint32_t n, uint32_t* scratch, uint32_t* status,
                   hipStream_t st);
int launch_kv_compact(const KvPagesArgs& a, uint32_t* scratch, uint32_t* live, hipStream_t st);
int launch_kv_copy_pages(const KvPagesArgs& a, const int32_t* src, const int32_t* dst, uint32_t n, uint32_t* status, hipStream_t st);

}  // namespace halo_mi
