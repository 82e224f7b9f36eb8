// Device helpers of the paged cache's kernels and those beside them: element types, the pages of a sequence, the codes.
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

// The integer nearest to x / s (ties to even) as the low byte of the result's bits, for |x| <= 127 s (1 + 2^-23), s normal; inv =
// 1 / s rounded. The multiply-add rounds x inv to an integer r, the quotient's or its neighbour (1.5 2^23 is where
// fp32 has steps of 1), and e = x - r s decides: for r even and not 0, x >= 1.5 s is a multiple of s's last bit and e
// fits 24 bits; for r = 0 e is x; for r = +-1 e is exact from x = s / 2 on, and below, where it may round to s / 2,
// the tie moves an odd r the same way. Without EXACT only `unsure` is set where r may have to move.
template <bool EXACT>
__device__ __forceinline__ uint32_t nearest(float x, float s, float inv, bool& unsure) {
    constexpr float kStepsOfOne = 12582912.0f;
    const float t = fmaf(x, inv, kStepsOfOne), r = t - kStepsOfOne;
    const float e = fmaf(-r, s, x), half = 0.5f * s;
    if constexpr (EXACT) {
        const bool move = fabsf(e) > half || (fabsf(e) == half && (__float_as_uint(t) & 1));
        return __float_as_uint(move ? t + copysignf(1.0f, e) : t);
    } else {
        unsure = unsure || fabsf(e) >= half;
        return __float_as_uint(t);
    }
}
// The low bytes of four words.
__device__ __forceinline__ uint32_t low_bytes(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    return __builtin_amdgcn_perm(__builtin_amdgcn_perm(d, c, 0x0C0C0400u), __builtin_amdgcn_perm(b, a, 0x0C0C0400u), 0x05040100u);
}

// Sums across lanes by moves of the vector unit. lanes<CTRL>: another lane's value of the same 16, by the move's control.
template <int CTRL>
__device__ __forceinline__ float lanes(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), CTRL, 0xF, 0xF, true));
}
// The sum of a's two halves of 32 lanes in the lower half, of b's in the upper; both16: of a's two 16 in each even 16, of b's in the odd.
__device__ __forceinline__ float both32(float a, float b) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float both16(float a, float b) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

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
