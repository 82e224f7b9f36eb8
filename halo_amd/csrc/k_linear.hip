// gfx950 kernels of linear attention with a decay for each head: S <- e^g S + k v^T, out = scale S^T q for a sequence's rows in order,
// S a k_dim x v_dim matrix of fp32 numbers per head that goes from call to call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "kv_device.h"
#include "launch.h"
#include "layer.h"

namespace halo_mi {
namespace {

using namespace dev;

constexpr uint32_t kBlock = 256;
constexpr uint32_t kColumns = 32;  // of S in a workgroup

struct LinearRows {
    uint32_t row0, rows;
};
__device__ __forceinline__ LinearRows linear_rows(const LinearArgs& a, uint32_t s) {
    const int32_t last = (int32_t)a.n_rows;
    const int32_t r0 = min(max(a.row_starts[s], 0), last), r1 = min(max(a.row_starts[s + 1], r0), last);
    return {(uint32_t)r0, (uint32_t)(r1 - r0)};
}

// Whether this thread finds an earlier sequence with rows that has the slot; tid of `threads` look through them.
__device__ __forceinline__ bool slot_taken(const LinearArgs& a, uint32_t s, int32_t slot, uint32_t tid, uint32_t threads) {
    bool taken = false;
    for (uint32_t i = tid; i < s; i += threads)
        if (a.slots[i] == slot) taken = taken || linear_rows(a, i).rows > 0;
    return taken;
}

// Row after row. One workgroup: columns 32 blockIdx.x and on of head blockIdx.y's state in sequence blockIdx.z, in its registers: a
// thread has 4 columns of rows tid / 8 + 32 j.
template <typename T, int RK>
__global__ __launch_bounds__(kBlock) void k_linear_rows(LinearArgs a) {
    __shared__ float parts[2][4][kColumns];
    const uint32_t tid = threadIdx.x, head = blockIdx.y, s = blockIdx.z;
    const uint32_t col = blockIdx.x * kColumns + tid % 8 * 4, row = tid / 8;
    const LinearRows r = linear_rows(a, s);
    if (r.rows == 0) return;
    const int32_t slot = a.slots[s];
    const bool in_pool = (uint32_t)slot < a.n_slots, begins = a.seq_lens && a.seq_lens[s] <= (int32_t)r.rows;
    const uint64_t at = ((uint64_t)(in_pool ? slot : 0) * a.heads + head) * a.k_dim * a.v_dim + row * a.v_dim + col;
    float4v S[RK];
#pragma unroll
    for (int j = 0; j < RK; ++j) S[j] = begins ? float4v{} : *reinterpret_cast<const float4v*>(a.state + at + j * 32 * a.v_dim);
    const bool bad = __syncthreads_or(!in_pool || slot_taken(a, s, slot, tid, kBlock));
    const uint32_t hk = head / a.group;
    const T* q = static_cast<const T*>(a.q.data) + r.row0 * a.q.stride + hk * a.q.head_stride + row;
    const T* k = static_cast<const T*>(a.k.data) + r.row0 * a.k.stride + hk * a.k.head_stride + row;
    const T* v = static_cast<const T*>(a.v.data) + r.row0 * a.v.stride + head * a.v.head_stride + col;
    const float* g = a.decay + (uint64_t)r.row0 * a.decay_stride + head;
    T* out = const_cast<T*>(static_cast<const T*>(a.out.data)) + r.row0 * a.out.stride + head * a.out.head_stride + blockIdx.x * kColumns;
    if (bad) {
        if (tid == 0 && blockIdx.x == 0 && head == 0) set_status(a.status, HALO_MI_STATUS_BAD_INDEX);
        for (uint32_t i = tid; i < r.rows * kColumns; i += kBlock) out[i / kColumns * a.out.stride + i % kColumns] = from_f32<T>(__uint_as_float(0x7FC00000u));
        return;
    }
    for (uint32_t t = 0; t < r.rows; ++t) {
        const float fade = __expf(g[t * a.decay_stride]);
        float4v vv, o{};
#pragma unroll
        for (int i = 0; i < 4; ++i) vv[i] = to_f32(v[t * a.v.stride + i]);
#pragma unroll
        for (int j = 0; j < RK; ++j) {
            const float kk = to_f32(k[t * a.k.stride + j * 32]), qq = to_f32(q[t * a.q.stride + j * 32]);
            S[j] = S[j] * fade + kk * vv;
            o += qq * S[j];
        }
#pragma unroll
        for (int i = 8; i < 64; i *= 2)
#pragma unroll
            for (int c = 0; c < 4; ++c) o[c] += __shfl_xor(o[c], i);
        if (tid % 64 < 8) *reinterpret_cast<float4v*>(&parts[t & 1][tid / 64][tid * 4 % kColumns]) = o;
        __syncthreads();
        if (tid < kColumns) {
            const float sum = (parts[t & 1][0][tid] + parts[t & 1][1][tid]) + (parts[t & 1][2][tid] + parts[t & 1][3][tid]);
            out[t * a.out.stride + tid] = from_f32<T>(sum * a.scale);
        }
    }
#pragma unroll
    for (int j = 0; j < RK; ++j) *reinterpret_cast<float4v*>(a.state_out + at + j * 32 * a.v_dim) = S[j];
}

// ---- prompts: chunks on the matrix cores -------------------------------------------------------------------------------

typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kChunk = 32;

// Elements that need not begin on more than an element: rows of any stride are read and written with whole accesses.
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[N];
};

// What a type is in pieces of bf16, exactly: the first has its leading 8 bits, the next the 8 after them.
template <typename T>
constexpr int kPieces = sizeof(T) == 4 ? 3 : 2;
template <>
constexpr int kPieces<__bf16> = 1;
// Pieces that a 32-bit weight or state is cut to on its way to an output of type T.
template <typename T>
constexpr int kOutPieces = sizeof(T) == 4 ? 3 : 2;

__device__ __forceinline__ uint32_t high_halves(float a, float b) { return __builtin_amdgcn_perm(__float_as_uint(b), __float_as_uint(a), 0x07060302u); }
__device__ __forceinline__ float without_high(float a) { return a - __uint_as_float(__float_as_uint(a) & 0xFFFF0000u); }

// Four values in N pieces; all but the last are cut, the last is rounded.
template <int N>
__device__ __forceinline__ void pieces_of(const float* x, uint2* out) {
    float r[4] = {x[0], x[1], x[2], x[3]};
#pragma unroll
    for (int p = 0; p < N; ++p) {
        if (p == N - 1 && N > 1) {
            const bf16x4 v = {(__bf16)r[0], (__bf16)r[1], (__bf16)r[2], (__bf16)r[3]};
            out[p] = __builtin_bit_cast(uint2, v);
        } else {
            out[p] = {high_halves(r[0], r[1]), high_halves(r[2], r[3])};
            if (p + 1 < N)
#pragma unroll
                for (int i = 0; i < 4; ++i) r[i] = without_high(r[i]);
        }
    }
}

__device__ __forceinline__ float4v mfma(uint4 a, uint4 b, float4v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// A thread's patch of q, k or v: 4 tokens by 4 dims.
template <typename T>
struct Patch {
    Vec<T, 4> row[4];
};

// Whether one of a patch's elements is not a finite number.
template <typename T>
__device__ __forceinline__ bool not_finite(const Patch<T>& p) {
    uint32_t top = 0;
    if constexpr (sizeof(T) == 2) {
        typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
        ushort2v most = {0, 0};
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint2 w = __builtin_bit_cast(uint2, p.row[t]);
            most = __builtin_elementwise_max(most, __builtin_bit_cast(ushort2v, w.x & 0x7FFF7FFFu));
            most = __builtin_elementwise_max(most, __builtin_bit_cast(ushort2v, w.y & 0x7FFF7FFFu));
        }
        top = max(most[0], most[1]);
        return top >= (std::is_same_v<T, __bf16> ? 0x7F80u : 0x7C00u);
    } else {
#pragma unroll
        for (int t = 0; t < 4; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, abs_bits(p.row[t].v[i]));
        return top > kLargestFinite;
    }
}

// The chunked form. With b_i the sum of a chunk's decays up to its row i, S the state before the chunk and P_ij = e^(b_i - b_j) q_i . k_j for
// j <= i:
//   out_i = scale (e^(b_i) S^T q_i + sum_j P_ij v_j),     S <- e^(b_last) S + sum_j (e^(b_last - b_j) k_j) v_j^T.
// One workgroup: 32 WAVES columns of a head's state, for a sequence or a segment of it. A wave keeps its 32 columns of S in its registers as
// the products leave them (rows 4 (lane / 16) + i, column lane % 16), which is also how the next product takes S^T: its order of k_dim is
// that of the registers, and q and k lie in LDS in the same order. Products are of bf16 pieces, summed in 32 bits: q, k and v exactly (one
// piece for BF16, two for F16, three for F32), the faded k in three, P and S in two where the output has 16 bits, else in three; of pairs of
// pieces those that matter in the result are multiplied.
// Chunks of 32 tokens keep LDS at 52 KB for BF16 and k_dim 128, three workgroups a CU.
// STATES: only the state that a segment adds is made (from zeros), for the segments after it.
// Sequences are cut into segments where there are too few for the GPU.
struct Segments {
    uint32_t length, most;  // rows of a segment; segments of a sequence at most
    uint32_t room;          // boundaries that `states` holds
    float* states;          // what a segment but the last of its sequence adds, then the state before the next one; [boundary][head][k_dim][v_dim]
    float* fades;           // ... and its decays' sum (log2): [boundary][head]
};

// Which pieces of a row of q or k change places, so that 16 rows' pieces of one place lie in 16 different sixteenths of the banks.
template <int KD>
__device__ __forceinline__ uint32_t row_swap(uint32_t token) {
    return KD % 128 == 0 ? token & 15 : KD == 96 ? token / 4 & 3 : token / 2 & 7;
}

// A sequence's boundaries between segments: their number, and how many lie before it. Where the room for their states ends (row starts that
// fall count rows twice), a sequence is not cut. For all of a workgroup.
struct Cuts {
    uint32_t parts, base;
};
__device__ __forceinline__ uint32_t cuts_of(const Segments& seg, uint32_t rows) { return rows ? min((rows - 1) / seg.length, seg.most - 1) : 0; }

// ... and whether the sequence has its slot to itself, in the pool.
__device__ __forceinline__ bool look_up(const LinearArgs& a, const Segments& seg, uint32_t s, int32_t slot, uint32_t rows, uint32_t threads, Cuts& cuts) {
    __shared__ uint32_t count;
    if (threadIdx.x == 0) count = 0;
    bool good = (uint32_t)slot < a.n_slots;
    uint32_t before = 0;
    for (uint32_t i = threadIdx.x; i < s; i += threads) {
        const LinearRows other = linear_rows(a, i);
        good = good && !(other.rows > 0 && a.slots[i] == slot);
        before += cuts_of(seg, other.rows);
    }
    good = !__syncthreads_or(!good);
    if (before) atomicAdd(&count, before);
    __syncthreads();
    cuts = {cuts_of(seg, rows), count};
    if (cuts.base > seg.room || seg.room - cuts.base < cuts.parts) cuts.parts = 0;
    return good;
}

template <typename T, int KD, int WAVES, bool STATES>
__global__ __launch_bounds__(WAVES * 64) void k_linear_chunks(LinearArgs a, Segments seg) {
    constexpr int NP = kPieces<T>, NO = kOutPieces<T>, KT = KD / 16, KS = KD / 32, THREADS = WAVES * 64;
    constexpr int QP = (KD / 4 * 8 + THREADS - 1) / THREADS;  // patches of q and k per thread
    constexpr int kColumnsHere = 32 * WAVES;
    constexpr bool K_ROWS = NP * KD < 768;  // k's rows lie in LDS too, where they fit
    // Rows of q and k: KD codes of 2 bytes, 16-byte pieces swapped by the row; of k^T, v^T and P: 32 tokens, pieces swapped by a quarter of the row.
    __shared__ uint4 q_lds[STATES ? 1 : NP * kChunk * KD / 8], k_lds[STATES || !K_ROWS ? 1 : NP * kChunk * KD / 8], kt_lds[3 * KD * 4], vt_lds[NP * kColumnsHere * 4],
        p_lds[STATES ? 1 : NO * kChunk * 4];
    __shared__ double sums_lds[kChunk];
    __shared__ int32_t bad_at[kColumnsHere];
    __shared__ int32_t bad_chunk;
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), m = lane % 16, g = lane / 16;
    const uint32_t v_blocks = a.v_dim / kColumnsHere, head = blockIdx.x / v_blocks, v0 = blockIdx.x % v_blocks * kColumnsHere;
    const uint32_t s = blockIdx.z, part = blockIdx.y;
    const LinearRows r = linear_rows(a, s);
    // the segment's rows; the last segment has all that are left
    const uint32_t first = part * seg.length;
    if (first >= r.rows) return;
    const int32_t slot = a.slots[s];
    Cuts cuts;
    const bool bad = !look_up(a, seg, s, slot, r.rows, THREADS, cuts);
    if (part > cuts.parts || (STATES && part == cuts.parts)) return;
    const bool last_part = part == cuts.parts, begins = a.seq_lens && a.seq_lens[s] <= (int32_t)r.rows;
    const uint32_t rows = last_part ? r.rows - first : seg.length, row0 = r.row0 + first, boundary = cuts.base + part;
    const uint32_t hk = head / a.group;
    T* out = const_cast<T*>(static_cast<const T*>(a.out.data)) + row0 * a.out.stride + head * a.out.head_stride + v0;
    if (bad) {
        if (STATES) return;
        if (tid == 0 && blockIdx.x == 0 && part == 0) set_status(a.status, HALO_MI_STATUS_BAD_INDEX);
        for (uint64_t i = tid; i < (uint64_t)rows * kColumnsHere; i += THREADS)
            out[i / kColumnsHere * a.out.stride + i % kColumnsHere] = from_f32<T>(__uint_as_float(0x7FC00000u));
        return;
    }
    const T* qg = static_cast<const T*>(a.q.data) + row0 * a.q.stride + hk * a.q.head_stride;
    const T* kg = static_cast<const T*>(a.k.data) + row0 * a.k.stride + hk * a.k.head_stride;
    const T* vg = static_cast<const T*>(a.v.data) + row0 * a.v.stride + head * a.v.head_stride + v0;
    const float* dg = a.decay + (uint64_t)row0 * a.decay_stride + head;

    // ---- the state: tile (t, u) has rows 16 t .. and columns 32 wave + 16 u ..
    const uint64_t plane = (uint64_t)KD * a.v_dim, mine = v0 + wave * 32 + m + (uint64_t)(4 * g) * a.v_dim;
    float4v S[KT][2] = {};
    const float* before = nullptr;
    if (!STATES) {
        if (part > 0) before = seg.states + ((uint64_t)(boundary - 1) * a.heads + head) * plane;
        else if (!begins) before = a.state + ((uint64_t)slot * a.heads + head) * plane;
    }
    if (before)
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[t][u][i] = before[mine + (uint64_t)(16 * t + i) * a.v_dim + 16 * u];

    // ---- a chunk's way into the registers, one chunk ahead
    Patch<T> qn[QP], kn[QP], vn;
    float dn = 0.0f;
    const auto patch = [&](const T* base, uint64_t stride, uint32_t row, uint32_t dim) {
        Patch<T> p;
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            p.row[t] = Vec<T, 4>{};
            if (row + t < rows) p.row[t] = __builtin_bit_cast(Vec<T, 4>, *reinterpret_cast<const Loose<T, 4>*>(base + (row + t) * stride + dim));
        }
        return p;
    };
    const auto fetch = [&](uint32_t at) {
#pragma unroll
        for (int j = 0; j < QP; ++j) {
            const uint32_t i = tid + j * THREADS;
            if (KD / 4 * 8 % THREADS != 0 && i >= KD / 4 * 8) continue;
            const uint32_t dim = i % (KD / 4) * 4, row = at + i / (KD / 4) * 4;
            if (!STATES) qn[j] = patch(qg, a.q.stride, row, dim);
            kn[j] = patch(kg, a.k.stride, row, dim);
        }
        vn = patch(vg, a.v.stride, at + tid / (kColumnsHere / 4) * 4, tid % (kColumnsHere / 4) * 4);
        // a decay of -infinity, or far under the smallest exponential, empties the state; NaN stays
        const uint32_t t = at + lane % kChunk;
        dn = t < rows ? dg[t * a.decay_stride] : 0.0f;
    };
    // q and k in the order of S's registers: dims 4 g .. + 3 and 16 + 4 g .. + 3 of 32 side by side
    const auto put_row = [](uint4* lds, int np, uint32_t token, uint32_t dim, uint2 v) {
        reinterpret_cast<uint2*>(lds)[((np * kChunk + token) * (KD / 8) + ((dim / 32 * 4 + dim % 16 / 4) ^ row_swap<KD>(token))) * 2 + dim % 32 / 16] = v;
    };
    const auto row_at = [&](int np, uint32_t token, uint32_t ks) { return (np * kChunk + token) * (KD / 8) + ((ks * 4 + g) ^ row_swap<KD>(token)); };
    const auto column_at = [](uint32_t row, uint32_t piece) { return row * 4 + (piece ^ (row / 4 & 3)); };

    for (uint32_t i = tid; i < kColumnsHere; i += THREADS) bad_at[i] = kChunk;
    if (tid == 0) bad_chunk = -1;
    double total = 0.0;
    fetch(0);
    __syncthreads();
    for (uint32_t at = 0; at < rows; at += kChunk) {
        // ---- the decays' running sums, in 64 bits and turns of log2
        double b = (double)(dn < -1e4f ? -1e4f : dn) * 1.4426950408889634;
#pragma unroll
        for (int i = 1; i < kChunk; i *= 2) {
            const double o = __shfl_up(b, i, kChunk);
            if ((int)(lane % kChunk) >= i) b += o;
        }
        const double b_last = __shfl(b, kChunk - 1, kChunk);
        if (STATES) total += b_last;
        if (tid < kChunk) sums_lds[tid] = b;
        // ---- to LDS, in pieces
#pragma unroll
        for (int j = 0; j < QP; ++j) {
            const uint32_t i = tid + j * THREADS;
            const uint32_t dim = i % (KD / 4) * 4, token = i / (KD / 4) * 4;
            // every lane takes part in the cross-lane reads
            float fade[4];
#pragma unroll
            for (int t = 0; t < 4; ++t) fade[t] = __builtin_amdgcn_exp2f((float)(b_last - __shfl(b, (token + t) % kChunk, kChunk)));
            if (KD / 4 * 8 % THREADS != 0 && i >= KD / 4 * 8) continue;
            float kf[4][4];
#pragma unroll
            for (int t = 0; t < 4; ++t) {
                uint2 w[NP > 3 ? NP : 3];
                float qf[4];
#pragma unroll
                for (int d = 0; d < 4; ++d) kf[t][d] = to_f32(kn[j].row[t].v[d]);
                if constexpr (!STATES) {
#pragma unroll
                    for (int d = 0; d < 4; ++d) qf[d] = to_f32(qn[j].row[t].v[d]);
                    pieces_of<NP>(qf, w);
#pragma unroll
                    for (int p = 0; p < NP; ++p) put_row(q_lds, p, token + t, dim, w[p]);
                    if constexpr (K_ROWS) {
                        pieces_of<NP>(kf[t], w);
#pragma unroll
                        for (int p = 0; p < NP; ++p) put_row(k_lds, p, token + t, dim, w[p]);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint2 w[3];
                float f[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) f[t] = kf[t][d] * fade[t];
                pieces_of<3>(f, w);
#pragma unroll
                for (int p = 0; p < 3; ++p) reinterpret_cast<uint2*>(kt_lds)[column_at(p * KD + dim + d, token / 8) * 2 + token / 4 % 2] = w[p];
            }
        }
        {
            const uint32_t col = tid % (kColumnsHere / 4) * 4, token = tid / (kColumnsHere / 4) * 4;
            const bool odd = not_finite(vn);
            if (odd) bad_chunk = (int32_t)(at / kChunk);
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint2 w[NP];
                float f[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    f[t] = to_f32(vn.row[t].v[d]);
                    if (odd && abs_bits(f[t]) > kLargestFinite) {
                        atomicMin(&bad_at[col + d], (int32_t)(token + t));
                        f[t] = 0.0f;
                    }
                }
                pieces_of<NP>(f, w);
#pragma unroll
                for (int p = 0; p < NP; ++p) reinterpret_cast<uint2*>(vt_lds)[column_at(p * kColumnsHere + col + d, token / 8) * 2 + token / 4 % 2] = w[p];
            }
        }
        if (at + kChunk < rows) fetch(at + kChunk);
        __syncthreads();
        const bool some_bad = bad_chunk == (int32_t)(at / kChunk);
        // ---- P^T = K Q^T: tiles (tokens 16 jt .., rows 16 it ..) on and under the diagonal
        if constexpr (!STATES) {
            for (uint32_t tile = wave; tile < 3; tile += WAVES) {
                const uint32_t jt = tile == 2, it = tile > 0;
                float4v p{};
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    uint4 kf[NP];
                    if constexpr (K_ROWS) {
#pragma unroll
                        for (int x = 0; x < NP; ++x) kf[x] = k_lds[row_at(x, 16 * jt + m, ks)];
                    } else {
                        const uint32_t row = at + 16 * jt + m;
                        float f[2][4] = {};
                        if (row < rows)
#pragma unroll
                            for (int h = 0; h < 2; ++h) {
                                const Loose<T, 4> v = *reinterpret_cast<const Loose<T, 4>*>(kg + row * a.k.stride + 32 * ks + 16 * h + 4 * g);
#pragma unroll
                                for (int i = 0; i < 4; ++i) f[h][i] = to_f32(v.v[i]);
                            }
                        uint2 lo[NP], hi[NP];
                        pieces_of<NP>(f[0], lo);
                        pieces_of<NP>(f[1], hi);
#pragma unroll
                        for (int x = 0; x < NP; ++x) kf[x] = uint4{lo[x].x, lo[x].y, hi[x].x, hi[x].y};
                    }
#pragma unroll
                    for (int x = 0; x < NP; ++x)
#pragma unroll
                        for (int y = 0; y < NP && x + y < NO; ++y) p = mfma(kf[x], q_lds[row_at(y, 16 * it + m, ks)], p);
                }
                const double bi = sums_lds[16 * it + m];
                float f[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float w = p[i] * __builtin_amdgcn_exp2f((float)(bi - sums_lds[16 * jt + 4 * g + i]));
                    f[i] = it > jt || m >= 4 * g + i ? w : 0.0f;
                }
                uint2 w[NO];
                pieces_of<NO>(f, w);
#pragma unroll
                for (int x = 0; x < NO; ++x) reinterpret_cast<uint2*>(p_lds)[column_at(x * kChunk + 16 * it + m, 2 * jt + g / 2) * 2 + g % 2] = w[x];
                if (tile == 0)  // tokens 16 .. 31 of rows 0 .. 15
#pragma unroll
                    for (int x = 0; x < NO; ++x) reinterpret_cast<uint2*>(p_lds)[column_at(x * kChunk + m, 2 + g / 2) * 2 + g % 2] = uint2{0, 0};
            }
            // ---- out^T = S^T q^T, faded
            float4v o[2][2] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint4 qf[NP][2];
#pragma unroll
                for (int x = 0; x < NP; ++x)
#pragma unroll
                    for (int it = 0; it < 2; ++it) qf[x][it] = q_lds[row_at(x, 16 * it + m, ks)];
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint2 lo[NO], hi[NO];
                    pieces_of<NO>(reinterpret_cast<const float*>(&S[2 * ks][u]), lo);
                    pieces_of<NO>(reinterpret_cast<const float*>(&S[2 * ks + 1][u]), hi);
#pragma unroll
                    for (int x = 0; x < NO; ++x)
#pragma unroll
                        for (int y = 0; y < NP && x + y < NO; ++y)
#pragma unroll
                            for (int it = 0; it < 2; ++it) o[u][it] = mfma(uint4{lo[x].x, lo[x].y, hi[x].x, hi[x].y}, qf[y][it], o[u][it]);
                }
            }
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const float fade = __builtin_amdgcn_exp2f((float)sums_lds[16 * it + m]);
#pragma unroll
                for (int u = 0; u < 2; ++u) o[u][it] *= fade;
            }
            __syncthreads();
            // ---- ... and V^T P^T
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int x = 0; x < NP; ++x) {
                    const uint4 vf = vt_lds[column_at(x * kColumnsHere + wave * 32 + 16 * u + m, g)];
#pragma unroll
                    for (int y = 0; y < NO && x + y < NO; ++y)
#pragma unroll
                        for (int it = 0; it < 2; ++it) o[u][it] = mfma(vf, p_lds[column_at(y * kChunk + 16 * it + m, g)], o[u][it]);
                }
#pragma unroll
            for (int it = 0; it < 2; ++it) {
                const uint32_t row = 16 * it + m;
                if (at + row >= rows) continue;
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const uint32_t col = wave * 32 + 16 * u + 4 * g;
                    Loose<T, 4> y;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float v = o[u][it][i] * a.scale;
                        if (some_bad && bad_at[col + i] <= (int32_t)row) v = __uint_as_float(0x7FC00000u);
                        y.v[i] = from_f32<T>(v);
                    }
                    *reinterpret_cast<Loose<T, 4>*>(out + (uint64_t)(at + row) * a.out.stride + col) = y;
                }
            }
        }
        // ---- S <- e^(b_last) S + k^T v
        const float fade = __builtin_amdgcn_exp2f((float)b_last);
        uint4 vf[NP][2];
#pragma unroll
        for (int x = 0; x < NP; ++x)
#pragma unroll
            for (int u = 0; u < 2; ++u) vf[x][u] = vt_lds[column_at(x * kColumnsHere + wave * 32 + 16 * u + m, g)];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
#pragma unroll
            for (int u = 0; u < 2; ++u) S[t][u] *= fade;
#pragma unroll
            for (int x = 0; x < 3; ++x) {
                const uint4 kf = kt_lds[column_at(x * KD + 16 * t + m, g)];
#pragma unroll
                for (int y = 0; y < NP && x + y < 3; ++y)
#pragma unroll
                    for (int u = 0; u < 2; ++u) S[t][u] = mfma(kf, vf[y][u], S[t][u]);
            }
        }
        if (some_bad) {
#pragma unroll
            for (int u = 0; u < 2; ++u)
                if (bad_at[wave * 32 + 16 * u + m] < kChunk)
#pragma unroll
                    for (int t = 0; t < KT; ++t) S[t][u] = float4v{} + __uint_as_float(0x7FC00000u);
            if (lane < 32) bad_at[wave * 32 + lane] = kChunk;  // these columns are this wave's alone
        }
        __syncthreads();
    }
    float* after = nullptr;
    if (STATES) after = seg.states + ((uint64_t)boundary * a.heads + head) * plane;
    else if (last_part) after = a.state_out + ((uint64_t)slot * a.heads + head) * plane;
    if (after)
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) after[mine + (uint64_t)(16 * t + i) * a.v_dim + 16 * u] = S[t][u][i];
    if (STATES && tid == 0 && v0 == 0) seg.fades[(uint64_t)boundary * a.heads + head] = (float)total;
}

// What a segment adds becomes the state before the next one: S_(p+1) = e^(fade_p) S_p + added_p, from the sequence's own state on.
__global__ __launch_bounds__(kBlock) void k_linear_join(LinearArgs a, Segments seg) {
    const uint32_t tid = threadIdx.x, head = blockIdx.y, s = blockIdx.z, at = (blockIdx.x * kBlock + tid) * 4, plane = a.k_dim * a.v_dim;
    const LinearRows r = linear_rows(a, s);
    if (cuts_of(seg, r.rows) == 0) return;
    const int32_t slot = a.slots[s];
    Cuts cuts;
    if (!look_up(a, seg, s, slot, r.rows, kBlock, cuts)) return;
    if (at >= plane) return;
    const bool begins = a.seq_lens && a.seq_lens[s] <= (int32_t)r.rows;
    float4v S = begins ? float4v{} : *reinterpret_cast<const float4v*>(a.state + ((uint64_t)slot * a.heads + head) * plane + at);
    for (uint32_t p = 0; p < cuts.parts; ++p) {
        const uint64_t i = (uint64_t)(cuts.base + p) * a.heads + head;
        float4v* x = reinterpret_cast<float4v*>(seg.states + i * plane + at);
        S = S * __builtin_amdgcn_exp2f(seg.fades[i]) + *x;
        *x = S;
    }
}

constexpr uint32_t kCus = 256;
constexpr uint32_t kFewRows = 12;  // up to this many rows of a sequence go one after another

// Columns of a workgroup: a whole head's where they are 64, 96 or 128.
uint32_t waves_of(const LinearArgs& a) { return a.v_dim == 64 ? 2 : a.v_dim % 128 == 0 ? 4 : 3; }

// How sequences are cut into segments with part_bytes of workspace, and the bytes made use of.
Segments plan_segments(const LinearArgs& a, uint64_t part_bytes, uint64_t* bytes) {
    Segments seg{std::max(a.max_rows, 1u), 1, 0, nullptr, nullptr};
    *bytes = 0;
    if (a.max_rows <= kFewRows) return seg;
    const uint64_t per = (uint64_t)a.heads * (a.k_dim * a.v_dim + 1) * 4;  // of a boundary
    const uint64_t blocks = (uint64_t)a.heads * (a.v_dim / (32 * waves_of(a)));
    // about three workgroups a CU, and no segment under 256 rows
    uint64_t length = std::max<uint64_t>(256, (a.n_rows * blocks / (3 * kCus) + kChunk - 1) / kChunk * kChunk);
    // boundaries: one behind every whole segment of a sequence but its last
    const auto boundaries = [&](uint64_t l) { return std::min<uint64_t>(a.n_rows / l, (uint64_t)a.n_seqs * ((a.max_rows + l - 1) / l - 1)); };
    while (length < a.max_rows && boundaries(length) * per > part_bytes) length += std::max<uint64_t>(kChunk, length / 16 / kChunk * kChunk);
    if (length >= a.max_rows) return seg;
    seg.length = (uint32_t)length;
    seg.most = (uint32_t)((a.max_rows + length - 1) / length);
    seg.room = (uint32_t)boundaries(length);
    *bytes = seg.room * per;
    return seg;
}

template <typename T, int KD>
int launch_chunks(const LinearArgs& a, const Segments& seg, hipStream_t st) {
    const uint32_t waves = waves_of(a), blocks = a.heads * (a.v_dim / (32 * waves));
    const auto run = [&](auto states) {
        constexpr bool S = decltype(states)::value;
        auto* k = waves == 2 ? k_linear_chunks<T, KD, 2, S> : waves == 3 ? k_linear_chunks<T, KD, 3, S> : k_linear_chunks<T, KD, 4, S>;
        hipLaunchKernelGGL(k, dim3(blocks, S ? seg.most - 1 : seg.most, a.n_seqs), dim3(waves * 64), 0, st, a, seg);
    };
    if (seg.most > 1) {
        run(std::true_type{});
        hipLaunchKernelGGL(k_linear_join, dim3((a.k_dim * a.v_dim / 4 + kBlock - 1) / kBlock, a.heads, a.n_seqs), dim3(kBlock), 0, st, a, seg);
    }
    run(std::false_type{});
    return hip_status(hipGetLastError(), "linear_attention");
}

template <typename T>
int launch_typed(const LinearArgs& a, float* part, uint64_t part_bytes, hipStream_t st) {
    if (a.max_rows > kFewRows) {
        uint64_t bytes;
        Segments seg = plan_segments(a, part ? part_bytes : 0, &bytes);
        if (seg.most > 1) {
            seg.states = part;
            seg.fades = part + (uint64_t)seg.room * a.heads * a.k_dim * a.v_dim;
        }
        switch (a.k_dim) {
            case 64: return launch_chunks<T, 64>(a, seg, st);
            case 96: return launch_chunks<T, 96>(a, seg, st);
            case 128: return launch_chunks<T, 128>(a, seg, st);
            case 192: return launch_chunks<T, 192>(a, seg, st);
            default: return launch_chunks<T, 256>(a, seg, st);
        }
    }
    auto* k = a.k_dim == 64 ? k_linear_rows<T, 2> : a.k_dim == 96 ? k_linear_rows<T, 3> : a.k_dim == 128 ? k_linear_rows<T, 4> : a.k_dim == 192 ? k_linear_rows<T, 6> : k_linear_rows<T, 8>;
    hipLaunchKernelGGL(k, dim3(a.v_dim / kColumns, a.heads, a.n_seqs), dim3(kBlock), 0, st, a);
    return hip_status(hipGetLastError(), "linear_attention");
}

}  // namespace

uint64_t plan_linear(const LinearArgs& a, uint64_t part_bytes) {
    uint64_t bytes;
    plan_segments(a, part_bytes, &bytes);
    return bytes;
}

int launch_linear(uint32_t type, const LinearArgs& a, float* part, uint64_t part_bytes, hipStream_t st) {
    switch (type) {
        case HALO_MI_F16: return launch_typed<_Float16>(a, part, part_bytes, st);
        case HALO_MI_BF16: return launch_typed<__bf16>(a, part, part_bytes, st);
        default: return launch_typed<float>(a, part, part_bytes, st);
    }
}

}  // namespace halo_mi
