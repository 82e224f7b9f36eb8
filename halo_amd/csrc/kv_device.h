// Device helpers of the paged cache's kernels: element types, the pages of a sequence, the codes.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kv.h"

namespace halo_mi::dev {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float float4v __attribute__((ext_vector_type(4)));

// N consecutive elements of type T as one load or store (16 bytes for N = 16 / sizeof(T)).
template <typename T, int N>
struct alignas(sizeof(T) * N) Vec {
    T v[N];
};

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
    return (T)v;
}

// |v| as a word that orders like it: infinities above every number, NaN above infinities.
__device__ __forceinline__ uint32_t abs_bits(float v) { return __float_as_uint(v) & 0x7FFFFFFFu; }
constexpr uint32_t kLargestFinite = 0x7F7FFFFFu;

// A batch's rows of one sequence: its first row, row count and cached tokens. Row starts that fall or that
// pass n_rows are cut to what the row operands hold.
struct SeqRows {
    uint32_t row0;
    int32_t rows, len;
};
__device__ __forceinline__ SeqRows seq_rows(const KvBatch& b, uint32_t s) {
    const int32_t last = (int32_t)min(b.n_rows, 0x7FFFFFFFu);
    const int32_t r0 = min(max(b.row_starts[s], 0), last), r1 = min(max(b.row_starts[s + 1], r0), last);
    return {(uint32_t)r0, r1 - r0, max(b.kv_lens[s], 0)};
}

// The page of a sequence's token block j, or -1 (past the table, or an id that is no page).
__device__ __forceinline__ int32_t page_at(const KvBatch& b, const KvLayer& c, uint32_t s, uint32_t j) {
    const int32_t id = j < b.table_width ? b.tables[(uint64_t)s * b.table_stride + j] : -1;
    return (uint32_t)id < c.n_pages ? id : -1;
}

__device__ __forceinline__ const uint8_t* page_ptr(const KvLayer& c, int32_t page) {
    return c.pool + (uint64_t)(uint32_t)page * c.page_bytes;
}

// Four int8 codes as two pairs of f16: 1024 + (code + 128) has the code in its low byte, and 1152 comes off exactly.
__device__ __forceinline__ void codes_f16(uint32_t codes, half2v& lo, half2v& hi) {
    const uint32_t u = codes ^ 0x80808080u;
    const half2v off = {(_Float16)1152.0f, (_Float16)1152.0f};
    lo = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - off;
    hi = __builtin_bit_cast(half2v, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - off;
}
__device__ __forceinline__ half8v codes_f16(uint32_t a, uint32_t b) {
    half2v x[4];
    codes_f16(a, x[0], x[1]);
    codes_f16(b, x[2], x[3]);
    return half8v{x[0][0], x[0][1], x[1][0], x[1][1], x[2][0], x[2][1], x[3][0], x[3][1]};
}

__device__ __forceinline__ void set_status(uint32_t* status, uint32_t bit) {
    if (status) atomicOr(status, bit);
}

}  // namespace halo_mi::dev
