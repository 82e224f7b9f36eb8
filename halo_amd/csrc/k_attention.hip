// gfx950 kernels of attention over the 8-bit paged cache (ATTENTION, AttentionArgs at
// include/halo/backend/backend.h:392-408 of the reference):
//   out = sum_t p_t V_t / sum_t p_t, p_t = exp(scale q . K_t), K_t = ks c_t, V_t = vs c'_t with int8 codes c, c'.
//
// Products run on v_mfma_f32_16x16x32_f16. An int8 code is exact in f16, so K and V lose nothing; q, scaled per
// row by a power of two to the top of f16's range, and the weights are one f16 piece (16-bit types) or two (fp32).
// The scales stay out of the products: with x_t = s_t ks scale log2(e) + log2(vs), s_t = q . c_t, the weight of V's
// codes is w_t = 2^(x_t - m), m the running maximum of x_t, and the sum that divides is sum_t w_t / vs. One
// multiply-add per score applies both scales, and w_t <= 1 always fits f16 whatever the blocks' scales are.
//
// Layout of a step of 64 tokens (4 groups of 16, each inside one page since block_tokens is a multiple of 16). The
// scores are computed transposed, S^T = K Q^T, 16 tokens a tile: tile a holds tokens 4 a .. 4 a + 3 of every
// group, so lane (q, g) = (lane % 16, lane / 16) ends up with all 16 scores of q against group g, one scale each
// for K and V. These are in place as the B operand of O^T = V^T P^T: no weight crosses a lane. V's codes lie as
// [dim][token] in the page, so the A operand of 16 tokens is one 16-byte load per lane, as K's is per 16 dims.
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
constexpr uint32_t kStep = 64;  // tokens a wave takes at a time
// Weights are carried times 2^14, which leaves f16 all of its 11 bits for weights down to 2^-28.
constexpr float kWeightShift = 14.0f;
constexpr float kLog2Tiny = -80.0f;  // log2 of the scale that an all-zero block of V counts with

__device__ __forceinline__ float load_any(const void* p, uint32_t type, uint64_t i) {
    if (type == HALO_MI_F16) return (float)static_cast<const _Float16*>(p)[i];
    if (type == HALO_MI_BF16) return (float)static_cast<const __bf16*>(p)[i];
    return static_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_any(void* p, uint32_t type, uint64_t i, float v) {
    if (type == HALO_MI_F16) static_cast<_Float16*>(p)[i] = (_Float16)v;
    else if (type == HALO_MI_BF16) static_cast<__bf16*>(p)[i] = (__bf16)v;
    else static_cast<float*>(p)[i] = v;
}

// Partial results of (row, head) r and split s: D outputs (unnormalised), then the maximum and the sum.
__device__ __forceinline__ float* part_of(const AttnArgs& a, uint64_t r, uint32_t s) {
    return a.part + (r * a.splits + s) * (a.c.dim + 4);
}

// D: head_dim. NP: f16 pieces of q and of the weights. NQ: row tiles of 16 that share K and V.
template <int D, int NP, int NQ>
__global__ __launch_bounds__(kAttnWaves * 64) void k_attention(AttnArgs a) {
    constexpr int C = D / 64, TAIL = D % 64 / 32;  // 64-dim chunks of a K row, and a last one of 32
    constexpr int DT = D / 16;                     // tiles of 16 dims
    constexpr int ROWS = 16 * NQ;
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64, col = lane % 16, g = lane / 16;
    uint32_t id = blockIdx.x;
    const uint32_t split = id % a.splits;
    id /= a.splits;
    const uint32_t tile0 = id % a.tiles;
    id /= a.tiles;
    const uint32_t kvh = id % a.c.heads, seq = id / a.c.heads;
    const SeqRows sr = seq_rows(a.b, seq);
    const int32_t first = sr.len - sr.rows;  // position of the sequence's first row
    const uint32_t packed = (uint32_t)sr.rows * a.group;
    // tokens that the table has room for; what a length claims beyond is one group out of range (NaN)
    const int32_t cap = (int32_t)(a.b.table_width * a.c.block);

    __shared__ float lds_o[kAttnWaves][16][64 + 4];
    __shared__ float lds_m[kAttnWaves][ROWS], lds_l[kAttnWaves][ROWS];

    for (uint32_t tile = tile0; tile * ROWS < packed; tile += a.tiles) {
        // rows of this tile: packed row r is token r / group, head r % group of the kv head's
        half8v qf[NQ][2 * C + TAIL][NP];
        float c_log2[NQ];      // scale * log2(e) * 2^-(what q was scaled by)
        int32_t lo[NQ], hi[NQ];  // tokens that this lane's row sees: [lo, hi)
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            const uint32_t r = tile * ROWS + 16 * n + col;
            const bool live = r < packed;
            const uint32_t token = live ? r / a.group : 0, head = kvh * a.group + (live ? r % a.group : 0);
            const uint64_t at = (uint64_t)(sr.row0 + token) * a.q.stride + head * a.q.head_stride;
            const int32_t pos = first + (int32_t)token;
            hi[n] = live ? max(pos + 1, 0) : 0;
            lo[n] = a.window ? min(max(pos - (int32_t)a.window + 1, 0), cap) : 0;
            uint32_t top = 0;
#pragma unroll
            for (int f = 0; f < 2 * C + TAIL; ++f)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t d = f < 2 * C ? f / 2 * 64 + 16 * g + f % 2 * 8 + j : C * 64 + 8 * g + j;
                    top = max(top, live ? abs_bits(load_any(a.q.data, a.type, at + d)) : 0u);
                }
            top = max(top, (uint32_t)__shfl_xor((int)top, 16));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            const int e = top ? ilogbf(__uint_as_float(min(top, kLargestFinite))) : 0;
            const bool bad = top > kLargestFinite;
            c_log2[n] = bad ? __uint_as_float(0x7FC00000u) : ldexpf(a.scale_log2, e - 14);
#pragma unroll
            for (int f = 0; f < 2 * C + TAIL; ++f)
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    const uint32_t d = f < 2 * C ? f / 2 * 64 + 16 * g + f % 2 * 8 + j : C * 64 + 8 * g + j;
                    const float v = live && !bad ? ldexpf(load_any(a.q.data, a.type, at + d), 14 - e) : 0.0f;
                    qf[n][f][0][j] = (_Float16)v;
                    if constexpr (NP == 2) qf[n][f][1][j] = (_Float16)(v - (float)(_Float16)v);
                }
        }
        // the tile's tokens, and this workgroup's share of them
        const int32_t pos_min = first + (int32_t)(tile * ROWS / a.group);
        const int32_t pos_max = first + (int32_t)((min(tile * ROWS + ROWS, packed) - 1) / a.group);
        const int32_t begin = a.window ? min(max(pos_min - (int32_t)a.window + 1, 0), cap) / (int32_t)kStep * (int32_t)kStep : 0;
        const int32_t end = min(max(pos_max + 1, 0), cap + 16);
        const int64_t from = begin + (int64_t)split * a.chunk;
        const int64_t to = split + 1 == a.splits ? end : min((int64_t)end, from + a.chunk);

        float4v o[NQ][DT];
        float m[NQ], l[NQ];
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            m[n] = -INFINITY;
            l[n] = 0.0f;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[n][t] = float4v{0, 0, 0, 0};
        }
        for (int64_t t64 = from + wave * kStep; t64 < to; t64 += kAttnWaves * kStep) {
            const uint32_t t0 = (uint32_t)t64;
            // the page of group g; a page out of range reads page 0 and counts as NaN
            const uint32_t tg = t0 + 16 * g;
            int32_t page = 0;
            bool no_page = false;
            if (tg < (uint32_t)end) {
                page = page_at(a.b, a.c, seq, tg >> a.c.block_log2);
                no_page = page < 0;
                page = max(page, 0);
            }
            const uint8_t* base = page_ptr(a.c, page) + a.c.codes + kvh * a.c.plane;
            const float* scales = reinterpret_cast<const float*>(page_ptr(a.c, page) + a.c.scales) + kvh;
            float ks = scales[0], vs = scales[a.c.heads];
            if (no_page) {
                ks = __uint_as_float(0x7FC00000u);
                set_status(a.status, kStatusKvBadIndex);
            }
            const float lv = vs == 0.0f ? kLog2Tiny : log2f(vs);
            const float rv = vs == 0.0f ? 0x1p80f : 1.0f / vs;
            // S^T: the K row of tile a in this lane is token 4 a + col % 4 of group col / 4
            const uint32_t row_off = (t0 + 16 * (col / 4)) % a.c.block + col % 4;
            const uint8_t* krow = reinterpret_cast<const uint8_t*>(__shfl((long long)base, 16 * (col / 4))) + row_off * D;
            float4v s[NQ][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                const uint8_t* k = krow + 4 * t * D;
#pragma unroll
                for (int n = 0; n < NQ; ++n) s[n][t] = float4v{0, 0, 0, 0};
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const uint4 w = *reinterpret_cast<const uint4*>(k + c * 64 + 16 * g);
                    const half8v k0 = codes_f16(w.x, w.y), k1 = codes_f16(w.z, w.w);
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int p = 0; p < NP; ++p) {
                            s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[n][2 * c][p], s[n][t], 0, 0, 0);
                            s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[n][2 * c + 1][p], s[n][t], 0, 0, 0);
                        }
                }
                if constexpr (TAIL) {
                    const uint2 w = *reinterpret_cast<const uint2*>(k + C * 64 + 8 * g);
                    const half8v k0 = codes_f16(w.x, w.y);
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int p = 0; p < NP; ++p)
                            s[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[n][2 * C][p], s[n][t], 0, 0, 0);
                }
            }
            half8v wf[NQ][2][NP];
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
                const float k = ks * c_log2[n];
                float x[16], top = -INFINITY;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int32_t token = (int32_t)(tg + i);
                    const bool seen = token >= lo[n] && token < hi[n];
                    x[i] = seen ? fmaf(s[n][i / 4][i % 4], k, lv) : -INFINITY;
                    top = fmaxf(top, x[i]);
                }
                top = fmaxf(top, __shfl_xor(top, 16));
                top = fmaxf(top, __shfl_xor(top, 32));
                const float m_new = fmaxf(m[n], top);
                if (__ballot(m_new > m[n])) {
                    const float f = m_new == m[n] ? 1.0f : exp2f(m[n] - m_new);
                    l[n] *= f;
#pragma unroll
                    for (int t = 0; t < DT; ++t) o[n][t] *= f;
                }
                m[n] = m_new;
                const float shift = m_new == -INFINITY ? 0.0f : m_new - kWeightShift;
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const float w = exp2f(x[i] - shift);
                    sum += w;
                    wf[n][i / 8][0][i % 8] = (_Float16)w;
                    if constexpr (NP == 2) wf[n][i / 8][1][i % 8] = (_Float16)(w - (float)(_Float16)w);
                }
                l[n] += sum == 0.0f ? 0.0f : sum * rv;
            }
            // O^T: 16 tokens of dim 16 t + col of group g
            const uint8_t* vrow = base + a.c.heads * a.c.plane + col * a.c.block + (tg & (a.c.block - 1));
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                const uint4 w = *reinterpret_cast<const uint4*>(vrow + t * 16 * a.c.block);
                const half8v v0 = codes_f16(w.x, w.y), v1 = codes_f16(w.z, w.w);
#pragma unroll
                for (int n = 0; n < NQ; ++n)
#pragma unroll
                    for (int p = 0; p < NP; ++p) {
                        o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, wf[n][0][p], o[n][t], 0, 0, 0);
                        o[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, wf[n][1][p], o[n][t], 0, 0, 0);
                    }
            }
        }
        // the waves' results: l over the groups, then the waves in order
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            l[n] += __shfl_xor(l[n], 16);
            l[n] += __shfl_xor(l[n], 32);
            if (g == 0) {
                lds_m[wave][16 * n + col] = m[n];
                lds_l[wave][16 * n + col] = l[n];
            }
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
            float top = -INFINITY;
#pragma unroll
            for (uint32_t w = 0; w < kAttnWaves; ++w) top = fmaxf(top, lds_m[w][16 * n + col]);
            const float mine = m[n] == -INFINITY ? (l[n] == 0.0f ? 0.0f : 1.0f) : exp2f(m[n] - top);
#pragma unroll
            for (int d0 = 0; d0 < D; d0 += 64) {
#pragma unroll
                for (int t = 0; t < 4 && d0 / 16 + t < DT; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) lds_o[wave][col][16 * t + 4 * g + i] = o[n][d0 / 16 + t][i] * mine;
                __syncthreads();
                constexpr int WIDE = D < 64 ? D : 64;
                for (uint32_t i = threadIdx.x; i < 16 * WIDE; i += kAttnWaves * 64) {
                    const uint32_t q = i / WIDE, d = d0 + i % WIDE, r = tile * ROWS + 16 * n + q;
                    if (r >= packed || d >= D) continue;
                    float peak = -INFINITY, sum = 0.0f, acc = 0.0f;
#pragma unroll
                    for (uint32_t w = 0; w < kAttnWaves; ++w) peak = fmaxf(peak, lds_m[w][16 * n + q]);
#pragma unroll
                    for (uint32_t w = 0; w < kAttnWaves; ++w) {
                        const float mw = lds_m[w][16 * n + q], lw = lds_l[w][16 * n + q];
                        sum += lw == 0.0f ? 0.0f : lw * (mw == -INFINITY ? 1.0f : exp2f(mw - peak));
                        acc += lds_o[w][q][i % WIDE];
                    }
                    const uint32_t token = r / a.group, head = kvh * a.group + r % a.group;
                    if (a.splits > 1) {
                        float* part = part_of(a, (uint64_t)(sr.row0 + token) * a.heads + head, split);
                        part[d] = acc;
                        if (d == 0) {
                            part[D] = peak;
                            part[D + 1] = sum;
                        }
                    } else {
                        store_any(const_cast<void*>(a.out.data), a.type,
                                  (uint64_t)(sr.row0 + token) * a.out.stride + head * a.out.head_stride + d, sum == 0.0f ? 0.0f : acc / sum);
                    }
                }
                __syncthreads();
            }
        }
    }
}

// One wave per (row, head): the splits' results, in order.
__global__ __launch_bounds__(256) void k_attention_join(AttnArgs a) {
    const uint32_t lane = threadIdx.x % 64, D = a.c.dim;
    const uint64_t r = (uint64_t)blockIdx.x * 4 + threadIdx.x / 64;
    if (r >= (uint64_t)a.b.n_rows * a.heads) return;
    const uint32_t row = (uint32_t)(r / a.heads), head = (uint32_t)(r % a.heads);
    const int32_t r0 = max(a.b.row_starts[0], 0), r1 = a.b.row_starts[a.b.n_seqs];
    if ((int32_t)row < r0 || (int32_t)row >= r1) return;  // of no sequence
    float peak = -INFINITY;
    for (uint32_t s = 0; s < a.splits; ++s) peak = fmaxf(peak, part_of(a, r, s)[D]);
    float sum = 0.0f, acc[4] = {};
    for (uint32_t s = 0; s < a.splits; ++s) {
        const float* p = part_of(a, r, s);
        if (p[D + 1] == 0.0f) continue;
        const float f = p[D] == -INFINITY ? 1.0f : exp2f(p[D] - peak);
        sum += p[D + 1] * f;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            if (lane + 64 * i < D) acc[i] += p[lane + 64 * i] * f;
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
        if (lane + 64 * i < D)
            store_any(const_cast<void*>(a.out.data), a.type, row * a.out.stride + head * a.out.head_stride + lane + 64 * i,
                      sum == 0.0f ? 0.0f : acc[i] / sum);
}

uint32_t rows_per_tile(const AttnArgs& a) { return (uint64_t)a.b.max_rows * a.group <= 16 ? 16 : 32; }

template <int D>
void run_attention(const AttnArgs& a, uint32_t grid, hipStream_t st) {
    const bool two = a.type == HALO_MI_F32, small = rows_per_tile(a) == 16;
    auto* k = two ? (small ? k_attention<D, 2, 1> : k_attention<D, 2, 2>) : (small ? k_attention<D, 1, 1> : k_attention<D, 1, 2>);
    hipLaunchKernelGGL(k, dim3(grid), dim3(kAttnWaves * 64), 0, st, a);
}

}  // namespace

uint64_t plan_attention(AttnArgs& a, uint64_t part_bytes) {
    const uint64_t rows = rows_per_tile(a);
    a.tiles = (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(((uint64_t)a.b.max_rows * a.group + rows - 1) / rows, 1u << 16));
    const uint64_t groups = (uint64_t)a.tiles * a.c.heads * a.b.n_seqs;
    uint64_t span = a.b.max_kv;
    if (a.window) span = std::min<uint64_t>(span, (uint64_t)a.window + a.b.max_rows + kStep);
    // two workgroups per CU, of at least one step per wave
    const uint64_t most = std::max<uint64_t>(1, (span + kAttnWaves * kStep - 1) / (kAttnWaves * kStep));
    uint64_t splits = std::max<uint64_t>(1, std::min(most, 1024 / groups));
    const uint64_t each = (uint64_t)a.b.n_rows * a.heads * (a.c.dim + 4) * sizeof(float);
    splits = std::max<uint64_t>(1, std::min(splits, part_bytes / each));
    const uint64_t steps = (span + kStep - 1) / kStep;
    a.chunk = (uint32_t)((steps + splits - 1) / splits * kStep);
    a.splits = (uint32_t)std::max<uint64_t>(1, (span + a.chunk - 1) / std::max(a.chunk, 1u));
    if (a.chunk == 0) a.chunk = kStep;
    return a.splits > 1 ? each * a.splits : 0;
}

int launch_attention(const AttnArgs& a, hipStream_t st) {
    const uint32_t grid = a.splits * a.tiles * a.c.heads * a.b.n_seqs;
    switch (a.c.dim) {
        case 64: run_attention<64>(a, grid, st); break;
        case 96: run_attention<96>(a, grid, st); break;
        case 128: run_attention<128>(a, grid, st); break;
        case 192: run_attention<192>(a, grid, st); break;
        default: run_attention<256>(a, grid, st); break;
    }
    if (a.splits > 1)
        hipLaunchKernelGGL(k_attention_join, dim3((uint32_t)(((uint64_t)a.b.n_rows * a.heads + 3) / 4)), dim3(256), 0, st, a);
    return hip_status(hipGetLastError(), "ATTENTION");
}

}  // namespace halo_mi
