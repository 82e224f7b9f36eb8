// gfx950 kernels of attention over the 8-bit paged cache (ATTENTION, AttentionArgs at
// include/halo/backend/backend.h:392-408 of the reference):
//   out = sum_t p_t V_t / sum_t p_t, p_t = exp(scale q . K_t), K_t = ks c_t, V_t = vs c'_t with int8 codes c, c'.
//
// Products run on v_mfma_f32_16x16x32_f16. An int8 code is exact in f16, so K and V lose nothing; q, scaled per
// row by a power of two to the top of f16's range, is one f16 piece (16-bit types) or two (fp32); the weights are two for fp32, and
// for F16 over few rows, else one.
// The scales stay out of the products: with x_t = s_t ks scale log2(e) + log2(vs), s_t = q . c_t, the weight of V's
// codes is w_t = 2^(x_t - m), m a reference that follows the maximum of x_t, and the sum that divides is sum_t w_t / vs (where
// scales lie very far apart taken from the scores instead: sum_apart). One multiply-add per score applies both scales, and w_t fits f16
// whatever the blocks' scales are.
//
// Layout of a step of 64 tokens (4 groups of 16, each inside one page since block_tokens is a multiple of 16). The
// scores are computed transposed, S^T = K Q^T, 16 tokens a tile: tile a holds tokens 4 a .. 4 a + 3 of every
// group, so lane (q, g) = (lane % 16, lane / 16) ends up with all 16 scores of q against group g, one scale each
// for K and V. These are in place as the B operand of O^T = V^T P^T: no weight crosses a lane. V's codes lie as
// [dim][token] in the page, so the A operand of 16 tokens is one 16-byte load per lane, as K's is per 16 dims.
//
// What bounds it, as measured: few rows are a stream of the cache (48 bf16 rows over 405 MB in 88 us, 200 rows over 1.6 GB in
// 300: 4.7 and 5.5 TB/s with the join; a plain read of 405 MB runs at 6.9), or, when short, its chain of reads (one row over 777 tokens 15.7 us);
// many rows are the vector unit's work and the products, which overlap in part (three bf16 prompts of up to 5000 tokens, 321 GFLOP, in
// 377 to 402 us: 799 to 852 TFLOP/s where a large bf16 library product reaches 1300; vector unit 51 % busy, matrix cores 35 %; 256 fp32 rows
// over 16300 tokens in 185 to 196 us, 1040 to 1100 with the second pieces, 40 % and 44 %).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kv.h"
#include "kv_device.h"
#include "launch.h"

namespace halo_mi {
namespace {

using namespace dev;

constexpr uint32_t kAttnWaves = 4;
constexpr uint32_t kStep = 64;                     // tokens a wave takes at a time
constexpr uint32_t kChunk = kAttnWaves * kStep;    // tokens a workgroup takes at a time
constexpr uint32_t kChunkLog2 = 8;
static_assert(kChunk == 1u << kChunkLog2);
// Weights are carried times 2^kShift, and the reference that they are taken against follows the maximum only where it would
// take them past 2^15.5 (largest f16: 65504), so that most steps leave the outputs as they are. One piece: 2^8, which
// leaves f16 all of its 11 bits for weights down to 2^-22 of the largest and an absolute 2^-33; two pieces: 2^14, 2^-39.
template <int NP>
constexpr float kShift = NP == 1 ? 8.0f : 14.0f;
template <int NP>
constexpr float kSlack = NP == 1 ? 7.5f : 1.5f;
constexpr uint32_t kFewGrid = 768;  // workgroups of a call with few rows at most: three per CU
// Once the largest weights are of blocks of V with a scale over 2^this, a wave takes its sums apart from its weights (sum_apart).
constexpr float kFarLog2 = 10.0f;

__device__ __forceinline__ float quiet_nan() { return __uint_as_float(0x7FC00000u); }

// A value that the whole wave shares, as the scalar that the compiler cannot see it is; lane l's, l itself shared. Loop
// bounds, pages' places and the mask's limits then stay out of the vector registers (36 bytes of scratch a lane, then none).
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return (uint32_t)__builtin_amdgcn_readfirstlane((int)v); }
__device__ __forceinline__ uint32_t of_lane(uint32_t v, uint32_t l) { return (uint32_t)__builtin_amdgcn_readlane((int)v, (int)l); }

// max over the lanes of a column: lane, lane ^ 16, lane ^ 32, lane ^ 48
__device__ __forceinline__ float column_max(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    return fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
}
__device__ __forceinline__ float column_sum(float v) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v), false, false);
    v = __int_as_float(r[0]) + __int_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v), false, false);
    return __int_as_float(r[0]) + __int_as_float(r[1]);
}

// l * 2^d, d <= 0 (NaN, of two references that are both -inf, counts as 0): the sums that divide span more powers of two
// than one factor has.
__device__ __forceinline__ float lowered(float l, float d) {
    return l * __builtin_amdgcn_exp2f(fmaxf(d, -126.0f)) * __builtin_amdgcn_exp2f(fminf(d + 126.0f, 0.0f));
}

__device__ __forceinline__ void store_any(void* p, uint32_t type, uint64_t i, float v) {
    if (type == HALO_MI_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
    else if (type == HALO_MI_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
    else static_cast<float*>(p)[i] = v;
}
// Whether rows can be read and written 16 bytes at a time (uniform).
__device__ __forceinline__ bool wide_rows(const HeadRows& r, uint32_t type) {
    const uint32_t mask = type == HALO_MI_F32 ? 3 : 7;
    return reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && ((r.stride | r.head_stride) & mask) == 0;
}
// Four consecutive outputs, of any alignment.
__device__ __forceinline__ void store4(const HeadRows& r, uint32_t type, uint64_t i, float4v v) {
    void* p = const_cast<void*>(r.data);
    if (wide_rows(r, type)) {
        if (type == HALO_MI_F32) *reinterpret_cast<float4v*>(static_cast<float*>(p) + i) = v;
        else if (type == HALO_MI_F16) *reinterpret_cast<Vec<_Float16, 4>*>(static_cast<_Float16*>(p) + i) = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
        else *reinterpret_cast<Vec<__bf16, 4>*>(static_cast<__bf16*>(p) + i) = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
        return;
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) store_any(p, type, i + j, v[j]);
}

// The first token that a row at `pos` sees. Past the table's room every row sees the group there, which is out of range.
__device__ __forceinline__ int32_t first_seen(const AttnArgs& a, int32_t pos, int32_t cap) {
    return a.window && pos >= (int32_t)a.window ? min(pos - (int32_t)a.window + 1, cap) : 0;
}

// A lane's row of a tile of 16: its tokens [lo, hi), q as f16 fragments scaled to the top of f16's range, and what
// takes a score to the exponent's base 2: scale * log2(e) / (what q was scaled by), NaN where the row is not
// finite. A negative scale turns q's sign, so that `c` is never negative.
// GROUPS lane groups share a row: 4 (16 x 16 tiles) or 2 (32 x 32).
template <int D, int NP, int GROUPS = 4>
struct QRow {
    static constexpr int F = D / (8 * GROUPS);  // fragments of 8 elements a lane
    half8v f[F][NP];
    float c;
    int32_t lo, hi;

    // dim of element 0 of fragment i in lane group g: 16 bytes of codes hold two fragments' elements
    static __device__ __forceinline__ uint32_t dim(int i, uint32_t g) {
        return i / 2 * 2 + 1 < F ? i / 2 * 16 * GROUPS + 16 * g + i % 2 * 8 : i * 8 * GROUPS + 8 * g;
    }

    // Packed row r of `packed`: token r / group, head r % group of kv head kvh. fetch only loads, every word before the
    // first is used, one round trip (a tile of 16 rows of a verify step: 26.1 us against 27.6); finish converts. Rows past
    // the last are not read: lanes that all ask for one row wait for each other (one row of 6 heads at 256 dims: 17.0 us
    // against 20.1 with row 0 read in their place). Two pieces: fp32, a word an element; one: 16 bits, two a word.
    static constexpr int W = NP == 2 ? 8 : 4;
    __device__ __forceinline__ void fetch(const AttnArgs& a, const SeqRows& sr, uint32_t kvh, uint32_t r, uint32_t packed, uint32_t g,
                                          int32_t cap, uint32_t (&raw)[F][W]) {
        const bool live = r < packed;
        const uint32_t token = live ? r / a.group : 0, head = kvh * a.group + (live ? r % a.group : 0);
        const uint64_t at = (uint64_t)(sr.row0 + token) * a.q.stride + head * a.q.head_stride;
        const int32_t pos = sr.len - sr.rows + (int32_t)token;
        hi = live ? max(pos + 1, 0) : 0;
        lo = first_seen(a, pos, cap);
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < W; ++j) raw[i][j] = 0;
        if (!live) return;
        if (wide_rows(a.q, a.type)) {
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int h = 0; h < W; h += 4) {
                    const Vec<uint32_t, 4> x = *reinterpret_cast<const Vec<uint32_t, 4>*>(
                        static_cast<const uint8_t*>(a.q.data) + (at + dim(i, g)) * (NP == 2 ? 4 : 2) + h * 4);
#pragma unroll
                    for (int j = 0; j < 4; ++j) raw[i][h + j] = x.v[j];
                }
        } else if constexpr (NP == 2) {
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < 8; ++j) raw[i][j] = (static_cast<const uint32_t*>(a.q.data) + at)[dim(i, g) + j];
        } else {
            const uint16_t* p = static_cast<const uint16_t*>(a.q.data) + at;
#pragma unroll
            for (int i = 0; i < F; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) raw[i][j] = (uint32_t)p[dim(i, g) + 2 * j] | (uint32_t)p[dim(i, g) + 2 * j + 1] << 16;
        }
    }
    __device__ __forceinline__ void finish(const AttnArgs& a, const uint32_t (&raw)[F][W]) {
        const bool half = a.type == HALO_MI_F16;
        const auto element = [&](int i, int j) {
            if constexpr (NP == 2) {
                return __uint_as_float(raw[i][j]);
            } else {
                const uint32_t w = raw[i][j / 2];
                const float b = __uint_as_float(j % 2 ? w & 0xFFFF0000u : w << 16);
                return half ? (float)__builtin_bit_cast(half2v, w)[j % 2] : b;
            }
        };
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) top = max(top, abs_bits(element(i, j)));
        if constexpr (GROUPS == 4) top = max(top, (uint32_t)__shfl_xor((int)top, 16));
        top = max(top, (uint32_t)__shfl_xor((int)top, 32));
        const bool bad = top > kLargestFinite;
        // 2^up takes the row's largest to [2^14, 2^15); rows under 2^-112, whose scores are nothing, go up by 2^126
        const int32_t e = (int32_t)(top >> 23) - 127, up = min(14 - e, 126);
        c = bad ? quiet_nan() : ldexpf(fabsf(a.scale_log2), -up);
        const float times = __uint_as_float((uint32_t)(up + 127) << 23) * (a.scale_log2 < 0.0f ? -1.0f : 1.0f);
#pragma unroll
        for (int i = 0; i < F; ++i)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float x = bad ? 0.0f : element(i, j) * times;
                f[i][0][j] = (_Float16)x;
                if constexpr (NP == 2) f[i][1][j] = (_Float16)(x - (float)f[i][0][j]);
            }
    }
};

// What a lane group has of a step: K's and V's scales of its 16 tokens' block.
struct Scales {
    float k, lv, rv;  // K's; log2 of V's and its reciprocal
};
__device__ __forceinline__ Scales make_scales(float ks, float vs, bool page) {
    vs = vs == 0.0f ? kKvMinScale : vs;  // an all-zero block of V counts with the smallest scale
    return {page ? ks : quiet_nan(), __builtin_amdgcn_logf(vs), __builtin_amdgcn_rcpf(vs)};
}

// Bit i: token tg + i is in [lo, hi), i < 16.
__device__ __forceinline__ uint32_t seen_tokens(uint32_t tg, int32_t lo, int32_t hi) {
    const int32_t from = min(max(lo - (int32_t)tg, 0), 16), to = min(max(hi - (int32_t)tg, 0), 16);
    return ((1u << to) - 1u) & ~((1u << from) - 1u);
}

// The sum that divides is of 2^(s k - m + shift): the weights' over V's scale, as long as no weight that it needs lies under fp32's
// 2^-126. Scales are 2^-80 at least and the row's largest weight has 2^(shift - log2 vs) in the sum, so while its scale is under
// 2^kFarLog2 what is lost is under 2^-44 of the sum a token. Else a lane sums its scores against their own largest and moves
// the sum to the reference m (a block of V = 1.3e16 beside zeros, all scores alike: half of it, and not all). k is not negative.
template <int NP, class Rows>
__device__ __forceinline__ float sum_apart(const Rows& score, float k, float m, uint32_t seen) {
    __asm__ volatile("" : "+v"(seen));  // masks are made where they are used: kept, they fill the scalar registers
    float top = -INFINITY, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < 16; ++i) top = fmaxf(top, seen >> i & 1 ? score(i) : -INFINITY);
    const float base = top * k;
    __asm__ volatile("" : "+v"(seen));
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += __builtin_amdgcn_exp2f(seen >> i & 1 ? fmaf(score(i), k, -base) : -INFINITY);
    const float half = __builtin_amdgcn_exp2f(0.5f * (base - m + kShift<NP>));
    return seen ? sum * half * half : 0.0f;
}

// The running maximum and sum of a row, and its outputs: O^T as DT tiles of 16 dims.
template <int DT>
struct Running {
    float m, l;
    bool far;  // of the wave: a scale over 2^kFarLog2 was met
    float4v o[DT];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
        far = false;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[t] = float4v{0, 0, 0, 0};
    }

    // A step's scores become weights w = 2^(s k + lv - m + kShift) as f16 fragments; m, l and o follow. The maximum is
    // taken over the scores (k is not negative), so a score costs half a max3, one multiply-add, one exp2, one add and
    // half a conversion. Four parts; in all: weigh().

    // The largest exponent of the lane's scores, of all 16 tokens of its group or of those that are `seen`.
    __device__ __forceinline__ static float peak(const float4v (&s)[4], const Scales& sc, float c) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, s[i / 4][i % 4]);
        return fmaf(top, sc.k * c, sc.lv);
    }
    __device__ __forceinline__ static float peak_seen(const float4v (&s)[4], const Scales& sc, float c, uint32_t seen) {
        float top = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) top = fmaxf(top, seen >> i & 1 ? s[i / 4][i % 4] : -INFINITY);
        return seen ? fmaf(top, sc.k * c, sc.lv) : -INFINITY;
    }
    // `top`, over the column's lanes, joins the maximum.
    template <int NP>
    __device__ __forceinline__ void raise(float top) {
        top = column_max(top);
        if (__ballot(top > m + kSlack<NP>)) {
            const float m_new = fmaxf(m, top), f = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            l = lowered(l, m - m_new);
#pragma unroll
            for (int t = 0; t < DT; ++t) o[t] *= f;
            m = m_new;
        }
    }
    // The exponents; with `seen`, -inf for the others.
    template <int NP>
    __device__ __forceinline__ void exponents(const float4v (&s)[4], const Scales& sc, float c, bool all, uint32_t seen, float (&x)[16]) const {
        const float k = sc.k * c, shift = sc.lv - (m == -INFINITY ? 0.0f : m - kShift<NP>);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = fmaf(s[i / 4][i % 4], k, shift);
        if (!all) {
            __asm__ volatile("");  // a branch: most steps see everything
#pragma unroll
            for (int i = 0; i < 16; ++i) x[i] = seen >> i & 1 ? x[i] : -INFINITY;
        }
    }
    template <int NP>
    __device__ __forceinline__ void weights(const float (&x)[16], const Scales& sc, half8v (&w)[2][NP]) {
        float sum = 0.0f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float v = __builtin_amdgcn_exp2f(x[i]);
            w[i / 8][0][i % 8] = (_Float16)v;
            // in fp32: where V's scale is far below the others', f16 would lose weights that 1 / vs makes count
            sum += v;
            if constexpr (NP == 2) w[i / 8][1][i % 8] = (_Float16)(v - (float)w[i / 8][0][i % 8]);
        }
        l += sum == 0.0f || far ? 0.0f : sum * sc.rv;
    }
    template <int NP>
    __device__ __forceinline__ void weigh(const float4v (&s)[4], const Scales& sc, float c, uint32_t tg, int32_t lo, int32_t hi, bool all,
                                          half8v (&w)[2][NP]) {
        uint32_t seen = 0xFFFFu;
        if (all) {
            raise<NP>(peak(s, sc, c));
        } else {
            __asm__ volatile("");
            seen = seen_tokens(tg, lo, hi);
            raise<NP>(peak_seen(s, sc, c, seen));
        }
        far = far || __ballot(sc.lv > kFarLog2);  // inside raise's branch the rest is compiled twice and spills
        if (far) l += sum_apart<NP>([&](int i) { return s[i / 4][i % 4]; }, sc.k * c, m, seen);
        float x[16];
        exponents<NP>(s, sc, c, all, seen, x);
        weights<NP>(x, sc, w);
    }
};

__device__ __forceinline__ float4v mfma(half8v a, half8v b, float4v c) { return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0); }

// ---- few rows: the cache is streamed once ---------------------------------------------------------------------
//
// Work is cut into units: a unit is a.unit tokens (a multiple of kChunk) of one (sequence, kv head, row tile). All
// units of the call, in that order, are dealt out evenly to the workgroups, each a run of `per`, so a batch
// of ragged lengths loads every CU alike and no length is needed on the host. Where a run ends inside a
// (sequence, kv head, tile), the parts meet in the workspace: slot 0 of a workgroup holds its first
// segment, slot 1 its last. A segment that is whole writes out itself. Inside a unit a wave takes every fourth step.

// A sequence in units.
struct SeqUnits {
    SeqRows r;
    int32_t begin, end;  // tokens that its rows see: from a multiple of kStep
    uint32_t chunks, tiles;
    uint32_t units;
};

template <int ROWS>
__device__ __forceinline__ SeqUnits seq_units(const AttnArgs& a, const SeqRows& rows) {
    SeqUnits u;
    u.r = rows;
    const int32_t cap = (int32_t)(a.b.table_width * a.c.block);
    u.begin = first_seen(a, u.r.len - u.r.rows, cap) / (int32_t)kStep * (int32_t)kStep;
    u.end = min(u.r.len, cap + 16);  // past the table: one group out of range, which makes its rows NaN
    // without memory for parts a unit is all of its tokens
    u.chunks = a.part && u.end > u.begin ? ((uint32_t)(u.end - u.begin) + a.unit - 1) >> a.unit_log2 : 1;
    u.tiles = ((uint32_t)u.r.rows * a.group + ROWS - 1) / ROWS;
    u.units = a.c.heads * u.tiles * u.chunks;
    return u;
}

template <int ROWS>
__device__ __forceinline__ SeqUnits seq_units(const AttnArgs& a, uint32_t seq) {
    return seq_units<ROWS>(a, seq_rows(a.b, seq));
}

// The call's units are under 2^31 where the row starts do not fall (plan_attention), and a sequence's always are; where starts fall,
// rows count for several sequences. Sums stop at kMostUnits, so that they order as they should all the same, and units from there on
// are nobody's: a wrapped sum would send the search for a unit's sequence past the last one, and the join past the workspace.
constexpr uint32_t kMostUnits = 0x7FFFFFFFu;
__device__ __forceinline__ uint32_t add_units(uint32_t a, uint32_t b) { return min(a + b, kMostUnits); }

// Sums of lanes 0..lane, right for the lanes under n; and of the lanes below lane l.
__device__ __forceinline__ uint32_t wave_scan(uint32_t v, uint32_t lane, uint32_t n) {
    for (uint32_t off = 1; off < min(n, 64u); off <<= 1) {
        const uint32_t below = (uint32_t)__shfl_up((int)v, off);
        if (lane >= off) v = add_units(v, below);
    }
    return v;
}
__device__ __forceinline__ uint32_t below_lane(uint32_t sum, uint32_t l) { return l ? of_lane(sum, l - 1) : 0; }

// The run of units of a workgroup (of `workgroups`), and the sequence that the run's first unit lies in, with the
// units before that sequence. Every wave finds them for itself, 64 sequences at a time.
struct Run {
    uint32_t first, last;  // [first, last)
    uint32_t seq, before;
    SeqRows rows;  // of seq
};
template <int ROWS>
__device__ __forceinline__ Run find_run(const AttnArgs& a, uint32_t lane, uint32_t workgroups, uint32_t id) {
    Run r{};
    const uint32_t n = a.b.n_seqs;
    SeqRows rows = seq_rows(a.b, min(lane, n - 1));
    uint32_t v = lane < n ? seq_units<ROWS>(a, rows).units : 0, sum = wave_scan(v, lane, n), total = of_lane(sum, min(n, 64u) - 1);
    for (uint32_t s0 = 64; s0 < n; s0 += 64) {
        const uint32_t w = s0 + lane < n ? seq_units<ROWS>(a, s0 + lane).units : 0;
        total = add_units(total, of_lane(wave_scan(w, lane, n - s0), min(n - s0, 64u) - 1));
    }
    const uint32_t per = max(1u, (total + workgroups - 1) / workgroups);
    r.first = min(id * per, total);
    r.last = min(r.first + per, total);
    for (uint32_t s0 = 0; s0 < n; s0 += 64) {
        if (s0) {
            rows = seq_rows(a.b, min(s0 + lane, n - 1));
            v = s0 + lane < n ? seq_units<ROWS>(a, rows).units : 0;
            sum = wave_scan(v, lane, n - s0);
        }
        const uint64_t hit = __ballot(s0 + lane < n && r.before + sum > r.first);
        if (hit) {
            const uint32_t l = (uint32_t)__ffsll((long long)hit) - 1;
            r.before += below_lane(sum, l);
            r.seq = s0 + l;
            r.rows = {of_lane(rows.row0, l), (int32_t)of_lane((uint32_t)rows.rows, l), (int32_t)of_lane((uint32_t)rows.len, l)};
            break;
        }
        r.before += of_lane(sum, min(n - s0, 64u) - 1);
    }
    return r;
}

// Partial results of workgroup w's segment `slot`: ROWS rows of D outputs (unnormalised), the maximum and the sum.
template <int ROWS>
__device__ __forceinline__ float* part_of(const AttnArgs& a, uint64_t w, uint32_t slot, uint32_t row) {
    return a.part + ((w * 2 + slot) * ROWS + row) * (a.c.dim + 4);
}

// The same of (row, head) r and split s of a call with many rows.
__device__ __forceinline__ float* many_part(const AttnArgs& a, uint64_t r, uint32_t s) { return a.part + (r * a.splits + s) * (a.c.dim + 4); }

// 16 bytes of the cache. ONCE: nothing else reads them soon (48 ragged sequences of bf16, 405 MB: 97 us against 104; one
// sequence of 131000 tokens 59 against 63; 33 MB that two row tiles read 30 against 27).
template <bool ONCE>
__device__ __forceinline__ uint4 stream16(const uint8_t* p) {
    typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
    if constexpr (ONCE) {
        const uint4v v = __builtin_nontemporal_load(reinterpret_cast<const uint4v*>(p));
        return {v[0], v[1], v[2], v[3]};
    } else {
        return *reinterpret_cast<const uint4*>(p);
    }
}

// Workgroups of k_attention_few that a CU's registers hold (4 waves each, one per SIMD). With two row tiles one, though two
// fit up to head_dim 96: 60 sequences of 2000 tokens, 24 bf16 rows of head_dim 64 each, 31.7 us against 39, with as many more parts to join.
template <int D, int NQ>
constexpr int kFewPerCu = D == 64 && NQ == 1 ? 3 : D <= 128 && NQ == 1 ? 2 : 1;

// D: head_dim. NP: f16 pieces of q. WP: of the weights: two for F16, whose outputs have as many bits as one piece has (8 verify steps
// of 4 rows, 24 heads of 256: an rms error of 2.1e-4, the outputs' rounding, against 2.4e-4, for 25.6 us against 24.6); one for
// BF16, 1/16 of whose rounding it is off by. NQ: row tiles of 16 that share K and V.
template <int D, int NP, int WP, int NQ, bool ONCE>
__global__ __launch_bounds__(kAttnWaves * 64, (kFewPerCu<D, NQ>)) void k_attention_few(AttnArgs a) {
    constexpr int C = D / 64, TAIL = D % 64 / 32;  // 64-dim chunks of a K row, and a last one of 32
    constexpr int DT = D / 16;                     // tiles of 16 dims
    constexpr int ROWS = 16 * NQ;
    const uint32_t lane = threadIdx.x % 64, wave = uniform(threadIdx.x / 64), col = lane % 16, g = lane / 16;
    constexpr int kWide = D < 128 ? D : 128;  // outputs that meet in LDS at a time
    __shared__ __align__(16) float lds_o[kAttnWaves][16][kWide + 4];
    __shared__ float lds_m[kAttnWaves][ROWS], lds_l[kAttnWaves][ROWS];

    const Run mine = find_run<ROWS>(a, lane, gridDim.x, blockIdx.x);
    uint32_t u = mine.first, before = mine.before, seq = mine.seq;
    if (u >= mine.last) return;
    SeqUnits su = seq_units<ROWS>(a, mine.rows);
    const int32_t cap = (int32_t)(a.b.table_width * a.c.block);

    for (bool first = true; u < mine.last; first = false) {
        while (u >= before + su.units) {
            before += su.units;
            su = seq_units<ROWS>(a, ++seq);
        }
        // the segment: chunks [chunk, chunk + n) of (seq, kvh, tile)
        const uint32_t in_seq = (u - before) / su.chunks, chunk = (u - before) - in_seq * su.chunks;
        const uint32_t kvh = in_seq / su.tiles, tile = in_seq % su.tiles;
        const uint32_t n_chunks = min(su.chunks - chunk, mine.last - u);
        const bool whole = n_chunks == su.chunks;
        u += n_chunks;
        const uint32_t packed = (uint32_t)su.r.rows * a.group;

        // tokens that every row of the tile sees
        const int32_t pos0 = su.r.len - su.r.rows + (int32_t)(tile * ROWS / a.group);
        const int32_t pos1 = su.r.len - su.r.rows + (int32_t)((min(tile * ROWS + ROWS, packed) - 1) / a.group);
        const uint32_t all_hi = (uint32_t)max(pos0 + 1, 0), all_lo = (uint32_t)first_seen(a, pos1, cap), any_lo = (uint32_t)first_seen(a, pos0, cap);
        const uint32_t end = (uint32_t)max(min(pos1 + 1, su.end), 0);
        const uint32_t t_first = (uint32_t)su.begin + (chunk << a.unit_log2) + wave * kStep;
        const uint32_t t_end = whole ? end : min((uint32_t)su.begin + ((chunk + n_chunks) << a.unit_log2), end);

        const int32_t* table = a.b.tables + (uint64_t)seq * a.b.table_stride;
        const uint32_t head_codes = a.c.codes + kvh * a.c.plane;
        // the table entry of this lane group's 16 tokens of the step at t
        const auto entry = [&](uint32_t t) { return table[min((t + 16 * g) >> a.c.block_log2, a.b.table_width - 1)]; };
        // ... and what it says: the page, or page 0 and `ok` false
        const auto page_of = [&](uint32_t t, int32_t id, bool& ok) {
            const uint32_t tg = t + 16 * g;
            ok = (uint32_t)id < a.c.n_pages && (tg >> a.c.block_log2) < a.b.table_width;
            return page_ptr(a.c, ok ? id : 0);
        };
        uint4 kb[4][C > 0 ? C : 1];
        uint2 kt[4];
        float ks = 0.0f, vs = 0.0f;
        bool ok = true;
        const uint8_t* page = a.c.pool;
        // K of the step at t: the K row of tile i in this lane is token 4 i + col % 4 of group col / 4
        const auto load_k = [&](uint32_t t, int32_t id) {
            page = page_of(t, id, ok);
            // a page's number crosses the lanes, not its address: loads stay global ones (flat ones would hold up LDS)
            const uint32_t row = (t + 16 * (col / 4)) % a.c.block + col % 4;
            const uint8_t* k = page_ptr(a.c, __shfl(ok ? id : 0, 16 * (col / 4))) + head_codes + row * D;
            const float* sc = reinterpret_cast<const float*>(page + a.c.scales) + kvh;
            ks = sc[0];
            vs = sc[a.c.heads];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
#pragma unroll
                for (int c = 0; c < C; ++c) kb[i][c] = stream16<ONCE>(k + 4 * i * D + c * 64 + 16 * g);
                if constexpr (TAIL) kt[i] = *reinterpret_cast<const uint2*>(k + 4 * i * D + C * 64 + 8 * g);
            }
        };
        int32_t id_next = 0;
        QRow<D, NP> q[NQ];
        Running<DT> run[NQ];
        {
            const int32_t id = t_first < t_end ? entry(t_first) : 0;
            uint32_t raw[NQ][QRow<D, NP>::F][QRow<D, NP>::W];
#pragma unroll
            for (int n = 0; n < NQ; ++n) q[n].fetch(a, su.r, kvh, tile * ROWS + 16 * n + col, packed, g, cap, raw[n]);
            if (t_first < t_end) {
                load_k(t_first, id);
                id_next = entry(t_first + kChunk);
            }
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                q[n].finish(a, raw[n]);
                run[n].clear();
            }
        }
        for (uint32_t t0 = t_first; t0 < t_end; t0 += kChunk) {
            const uint32_t tg = t0 + 16 * g;
            // V of this step: 16 tokens of dim 16 i + col of group g
            uint4 vb[DT];
            {
                const uint8_t* v = page + head_codes + a.c.heads * a.c.plane + col * a.c.block + (tg & (a.c.block - 1));
#pragma unroll
                for (int i = 0; i < DT; ++i) vb[i] = stream16<ONCE>(v + i * 16 * a.c.block);
            }
            __builtin_amdgcn_sched_barrier(0);
            const Scales sc = make_scales(ks, vs, ok || tg >= end);
            if (!ok && tg < end && tg + 16 > any_lo) set_status(a.status, kStatusKvBadIndex);  // some row sees the group
            // dims outside, tiles inside: consecutive products have accumulators of their own
            float4v s[NQ][4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[n][i] = float4v{0, 0, 0, 0};
#pragma unroll
            for (int c = 0; c < C; ++c) {
                half8v k[2][4];
#pragma unroll
                for (int i = 0; i < 4; ++i) k[0][i] = codes_f16(kb[i][c].x, kb[i][c].y), k[1][i] = codes_f16(kb[i][c].z, kb[i][c].w);
#pragma unroll
                for (int h = 0; h < 2; ++h)
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int n = 0; n < NQ; ++n)
#pragma unroll
                            for (int i = 0; i < 4; ++i) s[n][i] = mfma(k[h][i], q[n].f[2 * c + h][p], s[n][i]);
            }
            if constexpr (TAIL) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const half8v k0 = codes_f16(kt[i].x, kt[i].y);
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int n = 0; n < NQ; ++n) s[n][i] = mfma(k0, q[n].f[2 * C][p], s[n][i]);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
            if (t0 + kChunk < t_end) {
                load_k(t0 + kChunk, id_next);
                id_next = entry(t0 + 2 * kChunk);
            }
            __builtin_amdgcn_sched_barrier(0);
            const bool all = t0 >= all_lo && t0 + kStep <= all_hi;
            half8v w[NQ][2][WP];
#pragma unroll
            for (int n = 0; n < NQ; ++n) run[n].template weigh<WP>(s[n], sc, q[n].c, tg, q[n].lo, q[n].hi, all, w[n]);
#pragma unroll
            for (int i = 0; i < DT; ++i) {
                const half8v v0 = codes_f16(vb[i].x, vb[i].y), v1 = codes_f16(vb[i].z, vb[i].w);
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int p = 0; p < WP; ++p) {
                        run[n].o[i] = mfma(v0, w[n][0][p], run[n].o[i]);
                        run[n].o[i] = mfma(v1, w[n][1][p], run[n].o[i]);
                    }
            }
        }
        // the waves' results, added in wave order
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const float l = column_sum(run[n].l);
            if (g == 0) {
                lds_m[wave][16 * n + col] = run[n].m;
                lds_l[wave][16 * n + col] = l;
            }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float m[kAttnWaves], peak = -INFINITY, sum = 0.0f;
#pragma unroll
            for (uint32_t w = 0; w < kAttnWaves; ++w) peak = fmaxf(peak, m[w] = lds_m[w][16 * n + col]);
#pragma unroll
            for (uint32_t w = 0; w < kAttnWaves; ++w) {
                // a wave without a maximum has no weights, or only NaN
                const float l = lds_l[w][16 * n + col];
                sum += m[w] == -INFINITY ? l : lowered(l, m[w] - peak);
            }
            const float part_f = run[n].m == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(run[n].m - peak);
            const float f = !whole ? part_f : sum == 0.0f ? 0.0f : part_f / sum;
            if (!whole && wave == 0 && g == 0) {
                float* part = part_of<ROWS>(a, blockIdx.x, first ? 0 : 1, 16 * n + col);
                part[D] = peak;
                part[D + 1] = sum;
            }
#pragma unroll
            for (int d0 = 0; d0 < D; d0 += kWide) {
#pragma unroll
                for (int t = 0; t < kWide / 16 && d0 / 16 + t < DT; ++t)
                    *reinterpret_cast<float4v*>(&lds_o[wave][col][16 * t + 4 * g]) = run[n].o[d0 / 16 + t] * f;
                __syncthreads();
#pragma unroll
                for (uint32_t i = threadIdx.x; i < 16 * kWide / 4; i += kAttnWaves * 64) {
                    const uint32_t row = i / (kWide / 4), d = d0 + i % (kWide / 4) * 4, r = tile * ROWS + 16 * n + row;
                    if (r >= packed || d >= D) continue;
                    float4v acc = {0, 0, 0, 0};
#pragma unroll
                    for (uint32_t w = 0; w < kAttnWaves; ++w) acc += *reinterpret_cast<const float4v*>(&lds_o[w][row][d - d0]);
                    if (!whole) {
                        *reinterpret_cast<float4v*>(part_of<ROWS>(a, blockIdx.x, first ? 0 : 1, 16 * n + row) + d) = acc;
                    } else {
                        const uint32_t token = r / a.group, head = kvh * a.group + r % a.group;
                        store4(a.out, a.type, (uint64_t)(su.r.row0 + token) * a.out.stride + head * a.out.head_stride + d, acc);
                    }
                }
                __syncthreads();
            }
        }
    }
}

// Joins the parts of the (sequence, kv head, tile)s that several workgroups of k_attention_few had, in unit order: a
// workgroup has one row. Its threads take the parts' maxima and sums side by side, then, as 256 / (D / 4) groups,
// every so many-th part's outputs, and the groups are added in order. What it waits for is memory, so the first outputs are
// asked for together with the maxima.
template <int ROWS>
__global__ __launch_bounds__(256) void k_attention_few_join(AttnArgs a, uint32_t workgroups) {
    constexpr int kEach = kFewGrid / 256, kEarly = 4, kBatch = 8;
    __shared__ float factor[kFewGrid], red[2][4];
    __shared__ uint32_t found[2];
    __shared__ float4v acc_of[256];
    const uint32_t tid = threadIdx.x, lane = tid % 64, D = a.c.dim, quads = D / 4;
    const uint32_t groups = 256 / quads, group = tid / quads, d = tid % quads * 4;
    // blockIdx.x counts (sequence, kv head, tile) by their sequences' most tiles
    const uint32_t seq = blockIdx.x / (a.c.heads * a.tiles), kvh = blockIdx.x / a.tiles % a.c.heads;
    const SeqUnits su = seq_units<ROWS>(a, seq);
    if (tid < 64) {  // one wave looks the sequences up: every workgroup of the call reads the same lines
        uint32_t total = 0, before = 0;
        for (uint32_t s0 = 0; s0 < a.b.n_seqs; s0 += 64) {
            const uint32_t n = min(a.b.n_seqs - s0, 64u), v = lane < n ? seq_units<ROWS>(a, s0 + lane).units : 0, sum = wave_scan(v, lane, n);
            if (seq - s0 < 64) before = add_units(total, below_lane(sum, seq - s0));
            total = add_units(total, of_lane(sum, n - 1));
        }
        if (lane == 0) found[0] = max(1u, (total + workgroups - 1) / workgroups), found[1] = before;
    }
    __syncthreads();
    const uint32_t per = uniform(found[0]), before = uniform(found[1]);
    const uint32_t packed = (uint32_t)su.r.rows * a.group;
    // of its rows, gridDim.y at a time
    for (uint32_t tile = blockIdx.x % a.tiles, row = blockIdx.y; tile < su.tiles; row += gridDim.y) {
        const uint32_t u0 = before + (kvh * su.tiles + tile) * su.chunks, r = tile * ROWS + row;
        const uint32_t w0 = u0 / per, w1 = (u0 + su.chunks - 1) / per, n = w1 - w0 + 1;
        if (n == 1 || w1 >= workgroups || row >= ROWS || r >= packed) {
            tile += a.tiles;
            row = blockIdx.y - gridDim.y;
            continue;
        }
        // a workgroup that began before u0 has this as its last segment
        const auto part = [&](uint32_t i) { return part_of<ROWS>(a, w0 + i, (w0 + i) * per < u0 ? 1 : 0, row); };
        float m[kEach], l[kEach];
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const uint32_t i = tid + k * 256;
            m[k] = -INFINITY, l[k] = 0.0f;
            if (i < n) m[k] = part(i)[D], l[k] = part(i)[D + 1];
        }
        float4v early[kEarly];
#pragma unroll
        for (int k = 0; k < kEarly; ++k) early[k] = *reinterpret_cast<const float4v*>(part(min(group + k * groups, n - 1)) + d);
        float top = m[0];
#pragma unroll
        for (int k = 1; k < kEach; ++k) top = fmaxf(top, m[k]);
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) top = fmaxf(top, __shfl_xor(top, off));
        if (lane == 0) red[0][tid / 64] = top;
        __syncthreads();
        top = fmaxf(fmaxf(red[0][0], red[0][1]), fmaxf(red[0][2], red[0][3]));
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < kEach; ++k) {
            const uint32_t i = tid + k * 256;
            const float f = m[k] == -INFINITY ? (l[k] == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m[k] - top);
            if (i < n) factor[i] = f;
            sum += m[k] == -INFINITY ? l[k] : lowered(l[k], m[k] - top);
        }
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) sum += __shfl_xor(sum, off);
        if (lane == 0) red[1][tid / 64] = sum;
        __syncthreads();
        sum = (red[1][0] + red[1][1]) + (red[1][2] + red[1][3]);
        float4v acc = {0, 0, 0, 0};
        if (group < groups) {
#pragma unroll
            for (int k = 0; k < kEarly; ++k)
                if (group + k * groups < n) acc += early[k] * factor[group + k * groups];
            // whole batches, the last one's too: a loop's remainder would wait for one part after another
            for (uint32_t i = group + kEarly * groups; i < n; i += kBatch * groups) {
                float4v v[kBatch];
#pragma unroll
                for (int k = 0; k < kBatch; ++k) v[k] = *reinterpret_cast<const float4v*>(part(min(i + k * groups, n - 1)) + d);
#pragma unroll
                for (int k = 0; k < kBatch; ++k)
                    if (i + k * groups < n) acc += v[k] * factor[i + k * groups];
            }
        }
        acc_of[tid] = acc;
        __syncthreads();
        if (group == 0) {
            for (uint32_t k = 1; k < groups; ++k) acc += acc_of[k * quads + tid];
            const uint32_t token = r / a.group, head = kvh * a.group + r % a.group;
            store4(a.out, a.type, (uint64_t)(su.r.row0 + token) * a.out.stride + head * a.out.head_stride + d, sum == 0.0f ? float4v{0, 0, 0, 0} : acc / sum);
        }
        __syncthreads();
    }
}

// Rows of a tile: a wider one reads K and V once for twice the rows, where the registers hold its outputs.
uint32_t few_rows(const AttnArgs& a) { return (uint64_t)a.b.max_rows * a.group <= 16 || a.c.dim > 128 ? 16 : 32; }

template <int D, int NP, int WP>
void run_few(const AttnArgs& a, hipStream_t st) {
    const uint32_t rows = few_rows(a);
    const dim3 join(a.b.n_seqs * a.c.heads * a.tiles, std::min<uint32_t>(rows, std::max<uint64_t>(1, (uint64_t)a.b.max_rows * a.group)));
    // one row tile, and more bytes than the L2 caches hold: read once
    const bool once = a.tiles == 1 && 2ull * a.b.n_seqs * a.b.max_kv * a.c.heads * D > 32ull << 20;
    if constexpr (D <= 128) {
        if (rows == 32) {
            hipLaunchKernelGGL((k_attention_few<D, NP, WP, 2, false>), dim3(a.splits), dim3(kAttnWaves * 64), 0, st, a);
            if (a.part) hipLaunchKernelGGL(k_attention_few_join<32>, join, dim3(256), 0, st, a, a.splits);
            return;
        }
    }
    auto* k = once ? k_attention_few<D, NP, WP, 1, true> : k_attention_few<D, NP, WP, 1, false>;
    hipLaunchKernelGGL(k, dim3(a.splits), dim3(kAttnWaves * 64), 0, st, a);
    if (a.part) hipLaunchKernelGGL(k_attention_few_join<16>, join, dim3(256), 0, st, a, a.splits);
}

template <int D>
void run_few_of(const AttnArgs& a, hipStream_t st) {
    a.type == HALO_MI_F32 ? run_few<D, 2, 2>(a, st) : a.type == HALO_MI_F16 ? run_few<D, 1, 2>(a, st) : run_few<D, 1, 1>(a, st);
}

// ---- many rows: prompts and chunks ----------------------------------------------------------------------------
//
// A workgroup has a tile of WAVES * 32 rows (tokens x the heads of a kv head) and goes over the tokens they see, 64 at a
// time. The codes of a step are widened to f16 once for all its waves and laid in LDS as the MFMA's A fragments, lane by
// lane, so that every write and read of LDS is 16 bytes per lane without a bank conflict; two buffers, so that the next step's
// codes are loaded, widened and stored while this one's are used: one barrier per step. A wave reads kAhead fragments
// ahead of the products that take them, V's first ones before the softmax.
//
// v_mfma_f32_32x32x16_f16: half the instructions of the 16 x 16 form for the same work, and the vector unit runs beside it
// (16 cycles of either form side by side with a v_exp_f32 stream: 1.01 against 1.13 times the stream alone). A
// step is two tiles u of 32 tokens; lane (r, h) = (lane % 32, lane / 32) has the scores of row r with the 16 tokens of
// group 2 u + h, as K's row r of tile u is token 4 (r / 8) + r % 4 of group 2 u + r / 4 % 2.
//
// The weights are one piece for both 16-bit types: V's products are half of the work here, and F16 prompts (16 heads of 256, up to
// 3000 rows) in two pieces take 252 us against 204, for an rms error of 2.1e-4 against 2.6e-4; fp32 is for callers who need it.
//
// The tiles of the latest rows, which see most, start first. With fewer tiles than CUs the tokens of each are split, and
// k_attention_many_join adds the parts.

typedef float float16v __attribute__((ext_vector_type(16)));

__device__ __forceinline__ float16v mfma32(half8v a, half8v b, float16v c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }

template <int D>
struct StepLds {
    half8v k[2][D / 16][64];  // [tile of 32 tokens][16 dims][lane]
    half8v v[4][D / 32][64];  // [2 u + half of a group's tokens][tile of 32 dims][lane]
    Scales scale[4];
};

// The maximum and sum of a lane's row, and its outputs: O^T as tiles of 32 dims.
template <int D>
struct Running32 {
    float m, l;
    bool far;
    float16v o[D / 32];
    __device__ __forceinline__ void clear() {
        m = -INFINITY;
        l = 0.0f;
        far = false;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[t][i] = 0.0f;
    }
    // As Running::weigh, over both tiles of a step. tg: the position of this lane's first token of tile 0.
    template <int NP>
    __device__ __forceinline__ void weigh(const float16v (&s)[2], const Scales (&sc)[2], float c, uint32_t tg, int32_t lo, int32_t hi, bool all,
                                          half8v (&w)[2][2][NP]) {
        const float k[2] = {sc[0].k * c, sc[1].k * c};
        uint32_t seen[2] = {0xFFFFu, 0xFFFFu};
        float top[2] = {-INFINITY, -INFINITY};
        if (all) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int i = 0; i < 16; ++i) top[u] = fmaxf(top[u], s[u][i]);
                top[u] = fmaf(top[u], k[u], sc[u].lv);
            }
        } else {
            __asm__ volatile("");  // a branch: most steps see everything
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                seen[u] = seen_tokens(tg + 32 * u, lo, hi);
#pragma unroll
                for (int i = 0; i < 16; ++i) top[u] = fmaxf(top[u], seen[u] >> i & 1 ? s[u][i] : -INFINITY);
                top[u] = seen[u] ? fmaf(top[u], k[u], sc[u].lv) : -INFINITY;
            }
        }
        float peak = fmaxf(top[0], top[1]);
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(peak), __float_as_int(peak), false, false);
        peak = fmaxf(__int_as_float(r[0]), __int_as_float(r[1]));
        if (__ballot(peak > m + kSlack<NP>) || far) {
            const float m_new = fmaxf(m, peak), f = m_new == m ? 1.0f : __builtin_amdgcn_exp2f(m - m_new);
            l = lowered(l, m - m_new);
#pragma unroll
            for (int t = 0; t < D / 32; ++t) o[t] *= f;
            m = m_new;
            // the row's largest weight is of a step that raised m, so its scale is looked at here only (1 % of a call of prompts; 2 % with
            // a look every step)
            far = far || __ballot(fmaxf(sc[0].lv, sc[1].lv) > kFarLog2);
            if (far) {
#pragma unroll
                for (int u = 0; u < 2; ++u) l += sum_apart<NP>([&](int i) { return s[u][i]; }, k[u], m, seen[u]);
            }
        }
        const float base = m == -INFINITY ? 0.0f : m - kShift<NP>;
        float x[2][16];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < 16; ++i) x[u][i] = fmaf(s[u][i], k[u], sc[u].lv - base);
        if (!all) {
            __asm__ volatile("");
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 16; ++i) x[u][i] = seen[u] >> i & 1 ? x[u][i] : -INFINITY;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float v = __builtin_amdgcn_exp2f(x[u][i]);
                sum += v;
                w[u][i / 8][0][i % 8] = (_Float16)v;
                if constexpr (NP == 2) w[u][i / 8][1][i % 8] = (_Float16)(v - (float)w[u][i / 8][0][i % 8]);
            }
            l += sum == 0.0f || far ? 0.0f : sum * sc[u].rv;
        }
    }
};

template <int D, int NP, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void k_attention_many(AttnArgs a) {
    constexpr int F = D / 16, C = D / 32, ROWS = 32 * WAVES;
    constexpr int UW = (C + WAVES / 2 - 1) / (WAVES / 2);  // 16-byte loads of K, and of V, per wave and step
    constexpr int kAhead = NP == 2 ? 4 : 8;                // fragments read ahead (8 spill at two pieces)
    extern __shared__ __align__(16) uint8_t lds_raw[];
    StepLds<D>* lds = reinterpret_cast<StepLds<D>*>(lds_raw);
    const uint32_t lane = threadIdx.x % 64, wave = uniform(threadIdx.x / 64), row = lane % 32, h = lane / 32;
    const uint32_t pairs = a.b.n_seqs * a.c.heads;
    uint32_t id = blockIdx.x;
    const uint32_t kvh = id % a.c.heads, seq = id % pairs / a.c.heads;
    id /= pairs;
    const uint32_t split = id % a.splits;
    const SeqRows sr = seq_rows(a.b, seq);
    const uint32_t packed = (uint32_t)sr.rows * a.group, tiles = (packed + ROWS - 1) / ROWS;
    const int32_t cap = (int32_t)(a.b.table_width * a.c.block), first = sr.len - sr.rows;
    const int32_t* table = a.b.tables + (uint64_t)seq * a.b.table_stride;
    const uint32_t head_codes = a.c.codes + kvh * a.c.plane;

    for (uint32_t back = id / a.splits; back < tiles; back += a.tiles) {
        const uint32_t row0 = (tiles - 1 - back) * ROWS, row_n = min(row0 + ROWS, packed);
        const uint32_t my0 = row0 + wave * 32, my_n = min(my0 + 32, row_n);  // this wave's rows: [my0, my_n)
        // tokens that the tile sees, and this split's share of them
        const int32_t tile_lo = first + (int32_t)(row0 / a.group), tile_hi = first + (int32_t)((row_n - 1) / a.group);
        const uint32_t lo = (uint32_t)first_seen(a, tile_lo, cap), begin = lo / kStep * kStep;
        const uint32_t end = (uint32_t)max(min(tile_hi + 1, cap + 16), 0);
        const uint32_t steps = end > begin ? (end - begin + kStep - 1) / kStep : 0, share = (steps + a.splits - 1) / a.splits;
        const uint32_t t_first = begin + min(split * share, steps) * kStep, t_end = min(begin + min((split + 1) * share, steps) * kStep, end);
        // tokens that some row of this wave sees, and that all of them see
        const int32_t my_lo = first + (int32_t)(my0 / a.group), my_hi = my0 < my_n ? first + (int32_t)((my_n - 1) / a.group) : -1;
        const uint32_t any_hi = (uint32_t)max(my_hi + 1, 0), all_hi = (uint32_t)max(my_lo + 1, 0);
        const uint32_t any_lo = (uint32_t)first_seen(a, my_lo, cap), all_lo = (uint32_t)first_seen(a, my_hi, cap);

        QRow<D, NP, 2> q;
        Running32<D> run;
        {
            uint32_t raw[F][QRow<D, NP, 2>::W];
            q.fetch(a, sr, kvh, my0 + row, packed, h, cap, raw);
            q.finish(a, raw);
            run.clear();
        }

        // The codes of a step on their way from the cache to LDS: this wave's are of tile wave % 2. A lane has the
        // table entry of group lane % 4; numbers of pages cross the lanes, not addresses: loads stay global ones (flat ones
        // would hold up LDS).
        uint4 kb[UW], vb[UW];
        float ks = 0.0f, vs = 0.0f;
        bool ok = true;
        const uint32_t u0 = wave % 2, c0 = wave / 2;
        const auto entry = [&](uint32_t t) { return table[min((t + 16 * (lane % 4)) >> a.c.block_log2, a.b.table_width - 1)]; };
        const auto load = [&](uint32_t t, int32_t page_id) {
            const uint32_t tg = t + 16 * (lane % 4);
            ok = (uint32_t)page_id < a.c.n_pages && (tg >> a.c.block_log2) < a.b.table_width;
            const int32_t number = ok ? page_id : 0;
            ok = ok || tg >= end || tg + 16 <= lo;  // no row sees the group
            const uint32_t kg = 2 * u0 + row / 4 % 2, vg = 2 * u0 + h;
            const uint8_t* k = page_ptr(a.c, __shfl(number, kg)) + head_codes + ((t + 16 * kg) % a.c.block + 4 * (row / 8) + row % 4) * D + 16 * h;
            const uint8_t* v = page_ptr(a.c, __shfl(number, vg)) + head_codes + a.c.heads * a.c.plane + row * a.c.block + (t + 16 * vg) % a.c.block;
#pragma unroll
            for (int j = 0; j < UW; ++j) {
                const uint32_t c = c0 + j * (WAVES / 2);
                if (C % (WAVES / 2) && c >= C) break;
                kb[j] = *reinterpret_cast<const uint4*>(k + c * 32);
                vb[j] = *reinterpret_cast<const uint4*>(v + c * 32 * a.c.block);
            }
            if (wave == 0) {
                const float* sc = reinterpret_cast<const float*>(page_ptr(a.c, number) + a.c.scales) + kvh;
                ks = sc[0];
                vs = sc[a.c.heads];
            }
        };
        const auto store = [&](StepLds<D>& to) {
#pragma unroll
            for (int j = 0; j < UW; ++j) {
                const uint32_t c = c0 + j * (WAVES / 2);
                if (C % (WAVES / 2) && c >= C) break;
                to.k[u0][2 * c][lane] = codes_f16(kb[j].x, kb[j].y);
                to.k[u0][2 * c + 1][lane] = codes_f16(kb[j].z, kb[j].w);
                to.v[2 * u0][c][lane] = codes_f16(vb[j].x, vb[j].y);
                to.v[2 * u0 + 1][c][lane] = codes_f16(vb[j].z, vb[j].w);
            }
            if (wave == 0) {
                if (!ok) set_status(a.status, kStatusKvBadIndex);
                if (lane < 4) to.scale[lane] = make_scales(ks, vs, ok);
            }
        };

        int32_t id_next = 0;
        if (t_first < t_end) {
            load(t_first, entry(t_first));
            id_next = entry(t_first + kStep);
            store(lds[0]);
        }
        __syncthreads();
        uint32_t buf = 0;
        for (uint32_t t0 = t_first; t0 < t_end; t0 += kStep, buf ^= 1) {
            const bool more = t0 + kStep < t_end;
            if (more) {
                load(t0 + kStep, id_next);
                id_next = entry(t0 + 2 * kStep);
            }
            if (t0 < any_hi && t0 + kStep > any_lo) {
                const StepLds<D>& from = lds[buf];
                // the fragments in the order of their use: K's of both tiles, dims by dims, then V's
                const auto fragment = [&](int i) { return i < 2 * F ? from.k[i % 2][i / 2][lane] : from.v[(i - 2 * F) / C][(i - 2 * F) % C][lane]; };
                half8v ring[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) ring[i] = fragment(i);
                const Scales sc[2] = {from.scale[h], from.scale[2 + h]};
                float16v s[2];
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 16; ++i) s[u][i] = 0.0f;
#pragma unroll
                for (int i = 0; i < 2 * F; i += 4) {
#pragma unroll
                    for (int j = i; j < i + 4; ++j)
#pragma unroll
                        for (int p = 0; p < NP; ++p) s[j % 2] = mfma32(ring[j % kAhead], q.f[j / 2][p], s[j % 2]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = i; j < i + 4; ++j) ring[j % kAhead] = fragment(j + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
                const bool all = t0 >= all_lo && t0 + kStep <= all_hi;
                half8v w[2][2][NP];
                run.template weigh<NP>(s, sc, q.c, t0 + 16 * h, q.lo, q.hi, all, w);
#pragma unroll
                for (int i = 0; i < 4 * C; i += 4) {
#pragma unroll
                    for (int j = i; j < i + 4; ++j)
#pragma unroll
                        for (int p = 0; p < NP; ++p)
                            run.o[j % C] = mfma32(ring[(2 * F + j) % kAhead], w[j / C / 2][j / C % 2][p], run.o[j % C]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = i; j < i + 4; ++j)
                        if (j + kAhead < 4 * C) ring[(2 * F + j) % kAhead] = fragment(2 * F + j + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (more) store(lds[buf ^ 1]);
            __syncthreads();
        }
        const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(run.l), __float_as_int(run.l), false, false);
        const float l = __int_as_float(r[0]) + __int_as_float(r[1]), f = l == 0.0f ? 0.0f : 1.0f / l;
        if (my0 + row >= packed) continue;
        const uint32_t token = sr.row0 + (my0 + row) / a.group, head = kvh * a.group + (my0 + row) % a.group;
        if (a.splits > 1) {
            float* part = many_part(a, (uint64_t)token * a.heads + head, split);
#pragma unroll
            for (int t = 0; t < C; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    *reinterpret_cast<float4v*>(part + 32 * t + 8 * i + 4 * h) = float4v{run.o[t][4 * i], run.o[t][4 * i + 1], run.o[t][4 * i + 2], run.o[t][4 * i + 3]};
            if (h == 0) {
                part[D] = run.m;
                part[D + 1] = l;
            }
        } else {
            const uint64_t at = (uint64_t)token * a.out.stride + head * a.out.head_stride;
#pragma unroll
            for (int t = 0; t < C; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    store4(a.out, a.type, at + 32 * t + 8 * i + 4 * h, float4v{run.o[t][4 * i], run.o[t][4 * i + 1], run.o[t][4 * i + 2], run.o[t][4 * i + 3]} * f);
        }
    }
}

// The same on v_mfma_f32_16x16x32_f16, 16 rows a wave, for the head_dims whose outputs would not leave 32-row tiles two
// waves per SIMD. Each wave reads all of K and V from LDS for half the rows, so LDS bounds it beside the
// products; one wave per SIMD with 32 rows was slower all the same (fp32, 24 heads of 256, 256 rows over 16300 tokens: 338 us).
template <int D>
struct StepLds16 {
    half8v k[4][D / 32][64];  // [tile of 16 tokens][32 dims][lane]
    half8v v[2][D / 16][64];  // [half of a group's tokens][tile of 16 dims][lane]
    Scales scale[4];
};

template <int D, int NP, int WAVES>
__global__ __launch_bounds__(WAVES * 64, 2) void k_attention_many16(AttnArgs a) {
    static_assert(D % 64 == 0 && WAVES == 8);
    constexpr int F = D / 32, C = D / 64, DT = D / 16, ROWS = 16 * WAVES;
    constexpr int KW = (C + 1) / 2, VW = (DT + WAVES - 1) / WAVES;  // 16-byte loads of K and V per wave and step
    constexpr int kAhead = 4;                                       // fragments read ahead (8 spill: 195 against 188 us)
    extern __shared__ __align__(16) uint8_t lds_raw[];
    StepLds16<D>* lds = reinterpret_cast<StepLds16<D>*>(lds_raw);
    const uint32_t lane = threadIdx.x % 64, wave = uniform(threadIdx.x / 64), col = lane % 16, g = lane / 16;
    const uint32_t pairs = a.b.n_seqs * a.c.heads;
    uint32_t id = blockIdx.x;
    const uint32_t kvh = id % a.c.heads, seq = id % pairs / a.c.heads;
    id /= pairs;
    const uint32_t split = id % a.splits;
    const SeqRows sr = seq_rows(a.b, seq);
    const uint32_t packed = (uint32_t)sr.rows * a.group, tiles = (packed + ROWS - 1) / ROWS;
    const int32_t cap = (int32_t)(a.b.table_width * a.c.block), first = sr.len - sr.rows;
    const int32_t* table = a.b.tables + (uint64_t)seq * a.b.table_stride;
    const uint32_t head_codes = a.c.codes + kvh * a.c.plane;

    for (uint32_t back = id / a.splits; back < tiles; back += a.tiles) {
        const uint32_t row0 = (tiles - 1 - back) * ROWS, row_n = min(row0 + ROWS, packed);
        const uint32_t my0 = row0 + wave * 16, my_n = min(my0 + 16, row_n);
        const int32_t tile_lo = first + (int32_t)(row0 / a.group), tile_hi = first + (int32_t)((row_n - 1) / a.group);
        const uint32_t lo = (uint32_t)first_seen(a, tile_lo, cap), begin = lo / kStep * kStep;
        const uint32_t end = (uint32_t)max(min(tile_hi + 1, cap + 16), 0);
        const uint32_t steps = end > begin ? (end - begin + kStep - 1) / kStep : 0, share = (steps + a.splits - 1) / a.splits;
        const uint32_t t_first = begin + min(split * share, steps) * kStep, t_end = min(begin + min((split + 1) * share, steps) * kStep, end);
        const int32_t my_lo = first + (int32_t)(my0 / a.group), my_hi = my0 < my_n ? first + (int32_t)((my_n - 1) / a.group) : -1;
        const uint32_t any_hi = (uint32_t)max(my_hi + 1, 0), all_hi = (uint32_t)max(my_lo + 1, 0);
        const uint32_t any_lo = (uint32_t)first_seen(a, my_lo, cap), all_lo = (uint32_t)first_seen(a, my_hi, cap);

        QRow<D, NP> q;
        Running<DT> run;
        {
            uint32_t raw[F][QRow<D, NP>::W];
            q.fetch(a, sr, kvh, my0 + col, packed, g, cap, raw);
            q.finish(a, raw);
            run.clear();
        }

        uint4 kb[KW], vb[VW];
        float ks = 0.0f, vs = 0.0f;
        bool ok = true;
        const uint32_t tile = wave % 4, c0 = wave / 4;  // this wave's loads of K: of one tile of 16 tokens
        const auto entry = [&](uint32_t t) { return table[min((t + 16 * (lane % 4)) >> a.c.block_log2, a.b.table_width - 1)]; };
        const auto load = [&](uint32_t t, int32_t page_id) {
            const uint32_t tg = t + 16 * (lane % 4);
            ok = (uint32_t)page_id < a.c.n_pages && (tg >> a.c.block_log2) < a.b.table_width;
            const int32_t number = ok ? page_id : 0;
            ok = ok || tg >= end || tg + 16 <= lo;  // no row sees the group
            const uint32_t kg = col / 4;
            const uint8_t* k = page_ptr(a.c, __shfl(number, kg)) + head_codes + ((t + 16 * kg) % a.c.block + 4 * tile + col % 4) * D + 16 * g;
            const uint8_t* v = page_ptr(a.c, __shfl(number, g)) + head_codes + a.c.heads * a.c.plane + col * a.c.block + (t + 16 * g) % a.c.block;
#pragma unroll
            for (int j = 0; j < KW; ++j)
                if (C % 2 == 0 || c0 + 2 * j < C) kb[j] = *reinterpret_cast<const uint4*>(k + (c0 + 2 * j) * 64);
#pragma unroll
            for (int j = 0; j < VW; ++j)
                if (DT % WAVES == 0 || wave + WAVES * j < DT) vb[j] = *reinterpret_cast<const uint4*>(v + (wave + WAVES * j) * 16 * a.c.block);
            if (wave == 0) {
                const float* sc = reinterpret_cast<const float*>(page_ptr(a.c, number) + a.c.scales) + kvh;
                ks = sc[0];
                vs = sc[a.c.heads];
            }
        };
        const auto store = [&](StepLds16<D>& to) {
#pragma unroll
            for (int j = 0; j < KW; ++j)
                if (C % 2 == 0 || c0 + 2 * j < C) {
                    to.k[tile][2 * (c0 + 2 * j)][lane] = codes_f16(kb[j].x, kb[j].y);
                    to.k[tile][2 * (c0 + 2 * j) + 1][lane] = codes_f16(kb[j].z, kb[j].w);
                }
#pragma unroll
            for (int j = 0; j < VW; ++j)
                if (DT % WAVES == 0 || wave + WAVES * j < DT) {
                    to.v[0][wave + WAVES * j][lane] = codes_f16(vb[j].x, vb[j].y);
                    to.v[1][wave + WAVES * j][lane] = codes_f16(vb[j].z, vb[j].w);
                }
            if (wave == 0) {
                if (!ok) set_status(a.status, kStatusKvBadIndex);
                if (lane < 4) to.scale[lane] = make_scales(ks, vs, ok);
            }
        };

        int32_t id_next = 0;
        if (t_first < t_end) {
            load(t_first, entry(t_first));
            id_next = entry(t_first + kStep);
            store(lds[0]);
        }
        __syncthreads();
        uint32_t buf = 0;
        for (uint32_t t0 = t_first; t0 < t_end; t0 += kStep, buf ^= 1) {
            const bool more = t0 + kStep < t_end;
            if (more) {
                load(t0 + kStep, id_next);
                id_next = entry(t0 + 2 * kStep);
            }
            if (t0 < any_hi && t0 + kStep > any_lo) {
                const StepLds16<D>& from = lds[buf];
                const auto fragment = [&](int i) { return i < 4 * F ? from.k[i % 4][i / 4][lane] : from.v[(i - 4 * F) / DT][(i - 4 * F) % DT][lane]; };
                half8v ring[kAhead];
#pragma unroll
                for (int i = 0; i < kAhead; ++i) ring[i] = fragment(i);
                const Scales sc = from.scale[g];
                float4v s[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) s[i] = float4v{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 4 * F; i += 4) {
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int j = i; j < i + 4; ++j) s[j % 4] = mfma(ring[j % kAhead], q.f[j / 4][p], s[j % 4]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = i; j < i + 4; ++j) ring[j % kAhead] = fragment(j + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
                const bool all = t0 >= all_lo && t0 + kStep <= all_hi;
                half8v w[2][NP];
                run.template weigh<NP>(s, sc, q.c, t0 + 16 * g, q.lo, q.hi, all, w);
#pragma unroll
                for (int i = 0; i < 2 * DT; i += 4) {
#pragma unroll
                    for (int p = 0; p < NP; ++p)
#pragma unroll
                        for (int j = i; j < i + 4; ++j) run.o[j % DT] = mfma(ring[(4 * F + j) % kAhead], w[j / DT][p], run.o[j % DT]);
                    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                    for (int j = i; j < i + 4; ++j)
                        if (j + kAhead < 2 * DT) ring[(4 * F + j) % kAhead] = fragment(4 * F + j + kAhead);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (more) store(lds[buf ^ 1]);
            __syncthreads();
        }
        const float l = column_sum(run.l), f = l == 0.0f ? 0.0f : 1.0f / l;
        if (my0 + col >= packed) continue;
        const uint32_t token = sr.row0 + (my0 + col) / a.group, head = kvh * a.group + (my0 + col) % a.group;
        if (a.splits > 1) {
            float* part = many_part(a, (uint64_t)token * a.heads + head, split);
#pragma unroll
            for (int t = 0; t < DT; ++t) *reinterpret_cast<float4v*>(part + 16 * t + 4 * g) = run.o[t];
            if (g == 0) {
                part[D] = run.m;
                part[D + 1] = l;
            }
        } else {
            const uint64_t at = (uint64_t)token * a.out.stride + head * a.out.head_stride;
#pragma unroll
            for (int t = 0; t < DT; ++t) store4(a.out, a.type, at + 16 * t + 4 * g, run.o[t] * f);
        }
    }
}

// Joins the splits of each (row, head), in order: D / 4 lanes a row. Eight splits are asked for at once and the sums moved to
// the new maximum after them: 94 rows of 16 heads over 10000 tokens, 32 splits, 7 us against 22 with a pass for the
// maximum and then one split after another.
__global__ __launch_bounds__(256) void k_attention_many_join(AttnArgs a) {
    constexpr uint32_t kBatch = 8;
    const uint32_t D = a.c.dim, quads = D / 4, at_once = 256 / quads, d = threadIdx.x % quads * 4;
    const uint64_t r = (uint64_t)blockIdx.x * at_once + threadIdx.x / quads;
    if (threadIdx.x / quads >= at_once || r >= (uint64_t)a.b.n_rows * a.heads) return;
    const uint32_t row = (uint32_t)(r / a.heads), head = (uint32_t)(r % a.heads);
    if ((int32_t)row < max(a.b.row_starts[0], 0) || (int32_t)row >= a.b.row_starts[a.b.n_seqs]) return;  // of no sequence
    float top = -INFINITY, sum = 0.0f;
    float4v acc = {0, 0, 0, 0};
    for (uint32_t s0 = 0; s0 < a.splits; s0 += kBatch) {
        float m[kBatch], l[kBatch], peak = top;
        float4v o[kBatch];
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) {
            const float* p = many_part(a, r, min(s0 + k, a.splits - 1));  // the last one again: its maximum changes nothing
            m[k] = p[D], l[k] = p[D + 1], o[k] = *reinterpret_cast<const float4v*>(p + d);
        }
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) peak = fmaxf(peak, m[k]);
        const float moved = top == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(top - peak);
        sum = top == -INFINITY ? sum : lowered(sum, top - peak);
        acc *= moved;
        top = peak;
#pragma unroll
        for (uint32_t k = 0; k < kBatch; ++k) {
            if (s0 + k >= a.splits) continue;
            const float f = m[k] == -INFINITY ? (l[k] == 0.0f ? 0.0f : 1.0f) : __builtin_amdgcn_exp2f(m[k] - top);
            sum += m[k] == -INFINITY ? l[k] : lowered(l[k], m[k] - top);
            acc += o[k] * f;
        }
    }
    store4(a.out, a.type, row * a.out.stride + head * a.out.head_stride + d, sum == 0.0f ? float4v{0, 0, 0, 0} : acc / sum);
}

constexpr int kManyWaves = 8;  // of a workgroup: of 32 rows each, or of 16 where the outputs of 32 would leave one wave per SIMD
template <int D>
constexpr bool kHalfTiles = D > 128;

template <int D, int NP>
int run_many(const AttnArgs& a, hipStream_t st) {
    constexpr int W = kManyWaves;
    void (*k)(AttnArgs);
    size_t lds;
    if constexpr (kHalfTiles<D>) {
        k = k_attention_many16<D, NP, W>;
        lds = 2 * sizeof(StepLds16<D>);
    } else {
        k = k_attention_many<D, NP, W>;
        lds = 2 * sizeof(StepLds<D>);
    }
    // more than 64 KiB of LDS has to be asked for, once per device and kernel; cheap enough to ask every time
    if (lds > 65536)
        if (int rc = hip_status(hipFuncSetAttribute(reinterpret_cast<const void*>(k), hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds), "ATTENTION")) return rc;
    hipLaunchKernelGGL(k, dim3(a.splits * a.tiles * a.c.heads * a.b.n_seqs), dim3(W * 64), lds, st, a);
    if (a.splits > 1) {
        const uint64_t at_once = 256 / (a.c.dim / 4), rows = (uint64_t)a.b.n_rows * a.heads;
        hipLaunchKernelGGL(k_attention_many_join, dim3((uint32_t)((rows + at_once - 1) / at_once)), dim3(256), 0, st, a);
    }
    return HALO_MI_OK;
}

constexpr uint64_t kMaxGrid = 1u << 22;  // workgroups of a launch (up to 512 threads each; n_seqs * kv heads is at most this)
constexpr uint32_t many_rows(uint32_t dim) { return dim > 128 ? 128 : 256; }

}  // namespace

namespace {

// Tiles of a call with many rows, and the splits that bring a workgroup to every CU.
uint64_t plan_many(AttnArgs& a, uint64_t part_bytes) {
    const uint32_t rows = many_rows(a.c.dim);
    const uint64_t pairs = (uint64_t)a.c.heads * a.b.n_seqs;
    a.tiles = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(((uint64_t)a.b.max_rows * a.group + rows - 1) / rows, kMaxGrid / pairs));
    const uint64_t groups = a.tiles * pairs, want = 256;
    uint64_t span = a.b.max_kv;
    if (a.window) span = std::min<uint64_t>(span, (uint64_t)a.window + rows / a.group + kStep);
    const uint64_t each = (uint64_t)a.b.n_rows * a.heads * (a.c.dim + 4) * sizeof(float);
    // a split has three steps at least: with two, 94 rows of 16 heads over 2500 tokens take 18.9 us against 18.0, with four 60 rows
    // of 12 heads over 600 tokens 25.6 against 24.4
    a.splits = (uint32_t)std::max<uint64_t>(1, std::min({want / groups, (span + 3 * kStep - 1) / (3 * kStep), part_bytes / each}));
    if ((uint64_t)a.b.n_rows * a.heads > 4 * kMaxGrid) a.splits = 1;  // the join's grid (rows behind the last sequence count)
    return a.splits > 1 ? a.splits * each : 0;
}

}  // namespace

// As many workgroups as the registers let run at once, one to three per CU, or fewer where there are not as many units. With memory for fewer parts than there are
// (sequence, kv head, tile)s, each of these is one unit.
uint64_t plan_attention(AttnArgs& a, uint64_t part_bytes) {
    // Few rows per kv head: what counts is the cache's stream. More: the products, on tiles that share K and V. A second tile
    // of few rows streams the cache again, which pays while the streams are too few to fill the GPU: 64 rows over 4000 tokens
    // (bf16, head_dim 128), 4 sequences of 4 kv heads: 23.5 us against 29.1 with many, 10 sequences of fp32 47 against 40; 24
    // rows (head_dim 256, two tiles) 2 sequences 21 against 27, 32 sequences 95 against 73.
    const uint64_t all = (uint64_t)a.b.max_rows * a.group, tile = few_rows(a);
    a.few = all <= tile || (all <= 2 * tile && (uint64_t)a.b.n_seqs * a.c.heads <= 32);
    if (!a.few) return plan_many(a, part_bytes);
    const uint32_t rows = few_rows(a);
    const uint64_t pairs = (uint64_t)a.b.n_seqs * a.c.heads;
    a.tiles = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(((uint64_t)a.b.max_rows * a.group + rows - 1) / rows, kMaxGrid / pairs));
    // units of a call at most: sequences' tiles, by the table's tokens; a unit grows until they fit 31 bits
    const uint64_t cap = (uint64_t)a.b.table_width * a.c.block + 16;
    const uint64_t most = ((uint64_t)a.b.n_rows * a.group / rows + a.b.n_seqs) * a.c.heads;
    a.unit_log2 = kChunkLog2;
    while (a.unit_log2 < 31 && most * ((cap >> a.unit_log2) + 2) > 0x7FFFFFFFull) ++a.unit_log2;
    a.unit = 1u << a.unit_log2;
    const uint64_t per_wg = 2ull * rows * (a.c.dim + 4) * sizeof(float);
    const uint64_t chunks = std::max<uint64_t>(1, ((uint64_t)a.b.max_kv + a.unit - 1) / a.unit);
    const uint32_t per_cu = rows == 32 ? kFewPerCu<128, 2> : a.c.dim == 64 ? kFewPerCu<64, 1> : a.c.dim <= 128 ? kFewPerCu<128, 1> : kFewPerCu<256, 1>;
    a.splits = (uint32_t)std::min<uint64_t>(256 * per_cu, pairs * a.tiles * chunks);
    const uint64_t fit = part_bytes / per_wg;
    const bool split = chunks > 1 && fit >= std::min<uint64_t>(a.splits, pairs * a.tiles);
    if (split) a.splits = (uint32_t)std::min<uint64_t>(a.splits, fit);
    return split ? a.splits * per_wg : 0;
}

int launch_attention(const AttnArgs& a, hipStream_t st) {
    const bool two = a.type == HALO_MI_F32;
    if (!a.few) {
        int rc;
        switch (a.c.dim) {
            case 64: rc = two ? run_many<64, 2>(a, st) : run_many<64, 1>(a, st); break;
            case 96: rc = two ? run_many<96, 2>(a, st) : run_many<96, 1>(a, st); break;
            case 128: rc = two ? run_many<128, 2>(a, st) : run_many<128, 1>(a, st); break;
            case 192: rc = two ? run_many<192, 2>(a, st) : run_many<192, 1>(a, st); break;
            default: rc = two ? run_many<256, 2>(a, st) : run_many<256, 1>(a, st); break;
        }
        return rc ? rc : hip_status(hipGetLastError(), "ATTENTION");
    }
    switch (a.c.dim) {
        case 64: run_few_of<64>(a, st); break;
        case 96: run_few_of<96>(a, st); break;
        case 128: run_few_of<128>(a, st); break;
        case 192: run_few_of<192>(a, st); break;
        default: run_few_of<256>(a, st); break;
    }
    return hip_status(hipGetLastError(), "ATTENTION");
}

}  // namespace halo_mi
