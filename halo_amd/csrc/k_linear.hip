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
// thread has 4 columns of rows tid / 8 + 32 j. Rows of q, k and v after the first come by way of LDS, one row ahead: loaded where they are used, each element
// by eight lanes, rows of 61 sequences took 9 us each, and so 6.
//
// The states bound one row a sequence: 61 sequences of 48 heads of 128 x 128 in 78.5 us (4.9 TB/s read and written).
template <typename T, int RK>
__global__ __launch_bounds__(kBlock) void k_linear_rows(LinearArgs a) {
    constexpr uint32_t KD = 32 * RK, kElements = (2 * KD + kColumns + kBlock - 1) / kBlock;  // of a row, per thread: q, k, then v
    __shared__ float parts[2][4][kColumns];
    __shared__ alignas(16) float qk_lds[2][2][KD], v_lds[2][kColumns];  // q and k: the RK elements of a thread side by side
    const uint32_t tid = threadIdx.x, head = blockIdx.y, s = blockIdx.z;
    const uint32_t col = blockIdx.x * kColumns + tid % 8 * 4, row = tid / 8;
    const LinearRows r = linear_rows(a, s);
    if (r.rows == 0) return;
    const int32_t slot = a.slots[s];
    const bool in_pool = (uint32_t)slot < a.n_slots, begins = a.seq_lens && a.seq_lens[s] <= (int32_t)r.rows;
    const uint64_t at = ((uint64_t)(in_pool ? slot : 0) * a.heads + head) * a.k_dim * a.v_dim + row * a.v_dim + col;
    const uint32_t hk = head / a.group;
    const T* q = static_cast<const T*>(a.q.data) + r.row0 * a.q.stride + hk * a.q.head_stride;
    const T* k = static_cast<const T*>(a.k.data) + r.row0 * a.k.stride + hk * a.k.head_stride;
    const T* v = static_cast<const T*>(a.v.data) + r.row0 * a.v.stride + head * a.v.head_stride + blockIdx.x * kColumns;
    const float* g = a.decay + (uint64_t)r.row0 * a.decay_stride + head;
    T* out = const_cast<T*>(static_cast<const T*>(a.out.data)) + r.row0 * a.out.stride + head * a.out.head_stride + blockIdx.x * kColumns;
    T element[kElements];
    const auto fetch = [&](uint32_t t) {
#pragma unroll
        for (uint32_t e = 0; e < kElements; ++e) {
            const uint32_t i = tid + e * kBlock;
            if (i < KD) element[e] = q[t * a.q.stride + i];
            else if (i < 2 * KD) element[e] = k[t * a.k.stride + (i - KD)];
            else if (i < 2 * KD + kColumns) element[e] = v[t * a.v.stride + (i - 2 * KD)];
        }
    };
    const auto put = [&](uint32_t t) {
#pragma unroll
        for (uint32_t e = 0; e < kElements; ++e) {
            const uint32_t i = tid + e * kBlock, d = i % KD;
            if (i < 2 * KD) qk_lds[t & 1][i / KD][d % 32 * RK + d / 32] = to_f32(element[e]);
            else if (i < 2 * KD + kColumns) v_lds[t & 1][i - 2 * KD] = to_f32(element[e]);
        }
    };
    float4v S[RK];
#pragma unroll
    for (int j = 0; j < RK; ++j) S[j] = begins ? float4v{} : *reinterpret_cast<const float4v*>(a.state + at + j * 32 * a.v_dim);
    // the first row as it is used: a single one is on its way with S
    float kk[RK], qq[RK];
    float4v vv;
#pragma unroll
    for (int j = 0; j < RK; ++j) kk[j] = to_f32(k[row + 32 * j]), qq[j] = to_f32(q[row + 32 * j]);
#pragma unroll
    for (int i = 0; i < 4; ++i) vv[i] = to_f32(v[tid % 8 * 4 + i]);
    const bool bad = __syncthreads_or(!in_pool || slot_taken(a, s, slot, tid, kBlock));
    if (bad) {
        if (tid == 0 && blockIdx.x == 0 && head == 0) set_status(a.status, HALO_MI_STATUS_BAD_INDEX);
        for (uint64_t i = tid; i < (uint64_t)r.rows * kColumns; i += kBlock) out[i / kColumns * a.out.stride + i % kColumns] = from_f32<T>(__uint_as_float(0x7FC00000u));
        return;
    }
    for (uint32_t t = 0; t < r.rows; ++t) {
        if (t + 1 < r.rows) fetch(t + 1);
        const float fade = __expf(g[t * a.decay_stride]);
        float4v o{};
#pragma unroll
        for (int j = 0; j < RK; ++j) {
            S[j] = S[j] * fade + kk[j] * vv;
            o += qq[j] * S[j];
        }
        // the four columns' sums over the wave's rows: each step leaves a lane half of the columns
        const float sum = both16(both32(o[0], o[1]), both32(o[2], o[3]));
        const float all = sum + lanes<0x128>(sum);
        if (tid % 16 < 8) parts[t & 1][tid / 64][tid % 8 * 4 + tid / 32 % 2 + tid / 16 % 2 * 2] = all;
        if (t + 1 < r.rows) put(t + 1);
        __syncthreads();
        if (tid < kColumns) {
            const float sum = (parts[t & 1][0][tid] + parts[t & 1][1][tid]) + (parts[t & 1][2][tid] + parts[t & 1][3][tid]);
            out[t * a.out.stride + tid] = from_f32<T>(sum * a.scale);
        }
        if (t + 1 < r.rows) {
#pragma unroll
            for (int j = 0; j < RK; ++j) qq[j] = qk_lds[~t & 1][0][row * RK + j], kk[j] = qk_lds[~t & 1][1][row * RK + j];
            vv = *reinterpret_cast<const float4v*>(&v_lds[~t & 1][tid % 8 * 4]);
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

// A value from the lanes before, 0 where there is none: CTRL 0x110 + n, from n lanes before in the same 16; 0x142 with rows 0xA, the last of the
// 16 before to lanes 16 .. 31 of 32.
template <int CTRL, int ROWS>
__device__ __forceinline__ double lanes_before(double v) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)bits, CTRL, ROWS, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(bits >> 32), CTRL, ROWS, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double lane_of(double v, int lane) {
    const uint64_t bits = __builtin_bit_cast(uint64_t, v);
    return __builtin_bit_cast(double, (uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)(bits >> 32), lane) << 32 | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)bits, lane));
}

// What a type is in pieces of bf16, exactly: the first has its leading 8 bits, the next the 8 after them.
template <typename T>
constexpr int kPieces = sizeof(T) == 4 ? 3 : 2;
template <>
constexpr int kPieces<__bf16> = 1;
// Pieces that a 32-bit weight or state is cut to on its way to an output: all of its 24 bits, so that the output's rounding is the only one to fewer. With
// two, 16 bits, outputs of 16 bits were up to a tenth of a step further off.
constexpr int kOutPieces = 3;

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

// A row of a patch in its type's pieces.
template <typename T>
__device__ __forceinline__ void to_pieces(const Vec<T, 4>& x, uint2* w) {
    if constexpr (kPieces<T> == 1) {
        w[0] = __builtin_bit_cast(uint2, x);
    } else {
        const float f[4] = {to_f32(x.v[0]), to_f32(x.v[1]), to_f32(x.v[2]), to_f32(x.v[3])};
        pieces_of<kPieces<T>>(f, w);
    }
}

// The columns of a patch of 16-bit values.
template <typename T>
__device__ __forceinline__ void turned(const Patch<T>& p, uint2* w) {
    uint2 r[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) r[t] = __builtin_bit_cast(uint2, p.row[t]);
    w[0] = {__builtin_amdgcn_perm(r[1].x, r[0].x, 0x05040100u), __builtin_amdgcn_perm(r[3].x, r[2].x, 0x05040100u)};
    w[1] = {__builtin_amdgcn_perm(r[1].x, r[0].x, 0x07060302u), __builtin_amdgcn_perm(r[3].x, r[2].x, 0x07060302u)};
    w[2] = {__builtin_amdgcn_perm(r[1].y, r[0].y, 0x05040100u), __builtin_amdgcn_perm(r[3].y, r[2].y, 0x05040100u)};
    w[3] = {__builtin_amdgcn_perm(r[1].y, r[0].y, 0x07060302u), __builtin_amdgcn_perm(r[3].y, r[2].y, 0x07060302u)};
}

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
// One workgroup: 16 UT WAVES columns of a head's state, for a sequence or a segment of it. A wave keeps its 16 UT columns of S in its registers as
// the products leave them (rows 4 (lane / 16) + i, column lane % 16), which is also how the next product takes S^T: its order of k_dim is
// that of the registers, and q and k lie in LDS in the same order. Products are of bf16 pieces, summed in 32 bits: q, k and v exactly (one
// piece for BF16, two for F16, three for F32), the faded k, P and S in three; of pairs of pieces those that matter in 24 bits are multiplied.
//
// What bounds it (BF16, 48 heads of 128, four prompts of 1639 to 5000 rows, 351 to 357 us): two workgroups a CU, by their registers (236; LDS 67 KB),
// whose waves issue vector instructions half of the time (835 a wave and chunk, 112 matrix products and 352 for S's pieces among them) and feed the
// matrix cores a quarter of it; segments of unequal length leave a quarter of the places empty. An earlier state of it, which cut S to two pieces for 16-bit
// types, took 399 us: its stores, which a branch could skip, made every chunk wait for all loads in flight. With stores that every lane makes, and k^T's
// pieces read one product ahead, it took 380. Tried on that state, and slower: the fade on v in place of k (405), loads a whole chunk ahead (386), the
// segments' pass with half the columns a workgroup (403).
// STATES: only the state that a segment adds is made (from zeros), for the segments after it.
// Sequences are cut into segments where there are too few for the GPU.
struct Segments {
    uint32_t length, most;  // rows of a segment; segments of a sequence at most
    uint32_t room;          // boundaries that `states` holds
    float* states;          // what a segment but the last of its sequence adds, then the state before the next one; [boundary][head][k_dim][v_dim]
    float* fades;           // ... and its decays' sum (log2): [boundary][head]
};

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

// LDS serves a 16-byte read of 64 lanes in four parts, each with lanes 4 .. 11 of one quarter of the wave and the others of its neighbour. With rows
// an odd number of 16 bytes long, their pieces lie in different banks once rows 4 .. 11 of 16 have their pieces' pairs swapped.
__device__ __forceinline__ uint32_t beside(uint32_t row) { return (row + 4) / 8 & 1; }

// k^T and v^T: a row has a dim's 32 tokens, in 5 units of 16 bytes. Threads write four dims each, all lanes the same one of their four at a time, and
// the products read 16 dims side by side: rows of equal row % 4 lie together, in planes that begin a quarter of the banks apart; of every other 64 rows the
// halves of each 16 bytes have changed places. By these alone 32 lanes that write 8 bytes each would meet all banks; with the swap of the 16-byte reads
// (`beside`) they share them two by two, and a write takes twice its cycles.
constexpr int plane_of(int rows) { return rows / 4 * 5 + (20 - rows / 4 * 5 % 16) % 16; }
template <int ROWS>
__device__ __forceinline__ uint32_t turned_row(uint32_t row) { return row % 4 * plane_of(ROWS) + row / 4 * 5; }

// LDS of a workgroup in units of 16 bytes: rows of q (which out passes through on its way), rows of k, k^T, v^T, and P by its rows.
template <typename T, int KD>
struct ChunkLds {
    static constexpr int R = KD / 8 + 1;  // of a row of q or k
    static constexpr int rows = kPieces<T> * kChunk * R, kt = 4 * plane_of(KD), p = kOutPieces * kChunk * 5;
    static constexpr int q(int columns) { return rows > kChunk * columns * (int)sizeof(T) / 16 ? rows : kChunk * columns * (int)sizeof(T) / 16; }
    static constexpr int vt(int columns) { return 4 * plane_of(columns); }
    static constexpr int bytes(int columns, bool k_rows) { return 16 * (q(columns) + (k_rows ? rows : 0) + 3 * kt + kPieces<T> * vt(columns) + p) + 2048; }
};
constexpr int kLds = 160 * 1024;
// k's rows lie in LDS too, unless they keep a second workgroup from the CU, or do not fit; then they are read from memory again.
template <typename T, int KD>
constexpr bool k_in_lds(int columns) {
    return ChunkLds<T, KD>::bytes(columns, true) <= (ChunkLds<T, KD>::bytes(columns, false) <= kLds / 2 ? kLds / 2 : kLds);
}

// The waves of a SIMD that a workgroup's registers leave room for: two, where LDS takes two workgroups or a workgroup is that many.
template <typename T, int KD, int WAVES, int UT, bool STATES>
constexpr int waves_at_least() {
    typedef ChunkLds<T, KD> L;
    constexpr int columns = 16 * UT * WAVES;
    constexpr int bytes = STATES ? 16 * (3 * L::kt + kPieces<T> * L::vt(columns)) + 2048 : L::bytes(columns, k_in_lds<T, KD>(columns));
    return bytes <= kLds / 2 && WAVES > 2 ? 2 : (WAVES + 3) / 4;
}

template <typename T, int KD, int WAVES, int UT, bool STATES>
__global__ __launch_bounds__(WAVES * 64, (waves_at_least<T, KD, WAVES, UT, STATES>())) void k_linear_chunks(LinearArgs a, Segments seg) {
    constexpr int NP = kPieces<T>, NO = kOutPieces, KT = KD / 16, KS = KD / 32, THREADS = WAVES * 64;
    constexpr int QP = (KD / 4 + THREADS / 8 - 1) / (THREADS / 8);  // patches of q and k per thread
    constexpr int kColumnsHere = 16 * UT * WAVES;
    constexpr bool K_ROWS = k_in_lds<T, KD>(kColumnsHere);
    typedef ChunkLds<T, KD> L;
    constexpr int R = L::R, KT_SIZE = L::kt, VT_SIZE = L::vt(kColumnsHere);
    __shared__ uint4 q_lds[STATES ? 1 : L::q(kColumnsHere)], k_lds[STATES || !K_ROWS ? 1 : L::rows], kt_lds[3 * KT_SIZE], vt_lds[NP * VT_SIZE], p_lds[STATES ? 1 : L::p];
    __shared__ double sums_lds[kChunk];
    __shared__ float fades_lds[kChunk];
    __shared__ int32_t bad_at[kColumnsHere];
    __shared__ int32_t bad_chunk;
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64), m = lane % 16, g = lane / 16;
    // workgroups go to the eight XCDs in turn: each takes heads side by side, whose q and k are the same
    const uint32_t block = gridDim.x % 8 ? blockIdx.x : blockIdx.x % 8 * (gridDim.x / 8) + blockIdx.x / 8;
    const uint32_t v_blocks = a.v_dim / kColumnsHere, head = block / v_blocks, v0 = block % v_blocks * kColumnsHere;
    const uint32_t s = blockIdx.z, part = blockIdx.y;
    const LinearRows r = linear_rows(a, s);
    if (part > cuts_of(seg, r.rows) || r.rows == 0) return;
    const int32_t slot = a.slots[s];
    Cuts cuts;
    const bool bad = !look_up(a, seg, s, slot, r.rows, THREADS, cuts);
    if (part > cuts.parts || (STATES && part == cuts.parts)) return;
    const bool last_part = part == cuts.parts, begins = a.seq_lens && a.seq_lens[s] <= (int32_t)r.rows;
    // segments of whole chunks, one more than the mean length has (512 rows in two: 288 and 224); the last one has what is left, which may be nothing
    const uint32_t each = (r.rows / (cuts.parts + 1) + kChunk) / kChunk * kChunk, first = part * each;
    const uint32_t rows = last_part ? r.rows - min(first, r.rows) : min(each, r.rows - min(first, r.rows)), row0 = r.row0 + first, boundary = cuts.base + part;
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
    const uint64_t plane = (uint64_t)KD * a.v_dim, mine = v0 + wave * (16 * UT) + m + (uint64_t)(4 * g) * a.v_dim;
    float4v S[KT][UT] = {};
    const float* before = nullptr;
    if (!STATES) {
        if (part > 0) before = seg.states + ((uint64_t)(boundary - 1) * a.heads + head) * plane;
        else if (!begins) before = a.state + ((uint64_t)slot * a.heads + head) * plane;
    }
    if (before)
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int u = 0; u < UT; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) S[t][u][i] = before[mine + (uint64_t)(16 * t + i) * a.v_dim + 16 * u];

    // ---- a chunk's way into the registers, one chunk ahead. This thread's patches: 4 tokens by 4 dims, lanes along
    // the dims, so that a load covers whole lines. Rows behind the last are read as the last one, and put to zero on the way to LDS.
    const uint32_t my_token = tid / (THREADS / 8) * 4, my_dim = tid % (THREADS / 8) * 4;
    Patch<T> qn[QP], kn[QP], vn;
    const T *q_from = qg, *k_from = kg, *v_from = vg;
    const float* d_from = dg + lane % kChunk * a.decay_stride;
    uint32_t q_off[4], k_off[4], v_off[4];
    const auto place = [&](uint32_t left) {
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            const uint32_t token = min(my_token + t, left - 1);
            q_off[t] = (token * (uint32_t)a.q.stride + my_dim) * sizeof(T);
            k_off[t] = (token * (uint32_t)a.k.stride + my_dim) * sizeof(T);
            v_off[t] = (token * (uint32_t)a.v.stride + my_dim) * sizeof(T);
        }
    };
    const auto fetch = [&](uint32_t left) {
        if (left < kChunk) place(left);
        const auto patch = [&](Patch<T>& p, const T* from, const uint32_t* off, int more) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                p.row[t] = __builtin_bit_cast(Vec<T, 4>, *reinterpret_cast<const Loose<T, 4>*>(reinterpret_cast<const uint8_t*>(from + more) + off[t]));
        };
#pragma unroll
        for (int j = 0; j < QP; ++j) {
            if (KD % (THREADS / 2) != 0 && my_dim + j * (THREADS / 2) >= KD) continue;
            if (!STATES) patch(qn[j], q_from, q_off, j * (THREADS / 2));
            patch(kn[j], k_from, k_off, j * (THREADS / 2));
        }
        if (my_dim < kColumnsHere) patch(vn, v_from, v_off, 0);
        q_from += kChunk * a.q.stride;
        k_from += kChunk * a.k.stride;
        v_from += kChunk * a.v.stride;
    };
    // q and k in the order of S's registers: dims 4 g .. + 3 and 16 + 4 g .. + 3 of 32 side by side
    const auto put_row = [](uint4* lds, int np, uint32_t token, uint32_t dim, uint2 v) {
        reinterpret_cast<uint2*>(lds)[((np * kChunk + token) * R + ((dim / 32 * 4 + dim % 16 / 4) ^ beside(token))) * 2 + dim % 32 / 16] = v;
    };
    const auto row_at = [&](int np, uint32_t token, uint32_t ks) { return (np * kChunk + token) * R + ((ks * 4 + g) ^ beside(token)); };
    // four tokens of a row that begins at `from`
    const auto put_tokens = [](uint4* lds, uint32_t from, uint32_t row, uint32_t token, uint2 v) {
        reinterpret_cast<uint2*>(lds)[(from + (token / 8 ^ beside(row))) * 2 + (token / 4 + row / 64) % 2] = v;
    };
    const auto halves = [](uint4 v, bool swapped) { return swapped ? uint4{v.z, v.w, v.x, v.y} : v; };
    const auto p_row = [](int x, uint32_t row) { return (x * kChunk + row) * 5; };

    for (uint32_t i = tid; i < kColumnsHere; i += THREADS) bad_at[i] = kChunk;
    if (tid == 0) bad_chunk = -1;
    // The decays' running sums of a chunk, in 64 bits and turns of log2: lane % 32 has its row's. A decay of -infinity, or far under the
    // smallest exponential, empties the state; NaN stays.
    const auto next_decay = [&](uint32_t at) {
        const float d = at + lane % kChunk < rows ? *d_from : 0.0f;
        d_from += kChunk * a.decay_stride;
        return d;
    };
    const auto running = [&](float d) {
        double b = (double)(d < -1e4f ? -1e4f : d) * 1.4426950408889634;
        b += lanes_before<0x111, 0xF>(b);
        b += lanes_before<0x112, 0xF>(b);
        b += lanes_before<0x114, 0xF>(b);
        b += lanes_before<0x118, 0xF>(b);
        return b + lanes_before<0x142, 0xA>(b);
    };
    // S is 2^held times what the registers hold: they take the decays only when those have grown large
    double held = 0.0, total = 0.0;
    if (rows) {
        place(kChunk);
        fetch(rows);
    }
    double b = running(next_decay(0));
    float decay_ahead = next_decay(kChunk);
    asm volatile("" : "+v"(decay_ahead));  // waited for here, or the loop would wait for it, and for all that is in flight, every time
    __syncthreads();
    for (uint32_t at = 0; at < rows; at += kChunk) {
        const double b_last = lane_of(b, kChunk - 1), grown = held + b_last;
        const bool settle = !(fabs(grown) < 40.0);
        const float row_fade = __builtin_amdgcn_exp2f((float)(b + held)) * a.scale;                      // on S^T q of row lane % 32
        const float k_fade = __builtin_amdgcn_exp2f((float)(settle ? b_last - b : b_last - b - grown));  // on k of token lane % 32
        if (STATES) total += b_last;
        if (tid < kChunk) sums_lds[tid] = b, fades_lds[tid] = row_fade;
        // ---- to LDS, in pieces
        if (rows - at < kChunk) {
#pragma unroll
            for (int t = 0; t < 4; ++t)
                if (my_token + t >= rows - at) {
#pragma unroll
                    for (int j = 0; j < QP; ++j) qn[j].row[t] = kn[j].row[t] = Vec<T, 4>{};
                    vn.row[t] = Vec<T, 4>{};
                }
        }
        float fade[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) fade[t] = __shfl(k_fade, my_token + t, kChunk);
#pragma unroll
        for (int j = 0; j < QP; ++j) {
            const uint32_t dim = my_dim + j * (THREADS / 2);
            if (KD % (THREADS / 2) != 0 && dim >= KD) continue;
            if constexpr (!STATES) {
#pragma unroll
                for (int t = 0; t < 4; ++t) {
                    uint2 w[NP];
                    to_pieces(qn[j].row[t], w);
#pragma unroll
                    for (int p = 0; p < NP; ++p) put_row(q_lds, p, my_token + t, dim, w[p]);
                    if constexpr (K_ROWS) {
                        to_pieces(kn[j].row[t], w);
#pragma unroll
                        for (int p = 0; p < NP; ++p) put_row(k_lds, p, my_token + t, dim, w[p]);
                    }
                }
            }
#pragma unroll
            for (int d = 0; d < 4; ++d) {
                uint2 w[3];
                float f[4];
#pragma unroll
                for (int t = 0; t < 4; ++t) f[t] = to_f32(kn[j].row[t].v[d]) * fade[t];
                pieces_of<3>(f, w);
#pragma unroll
                for (int p = 0; p < 3; ++p) put_tokens(kt_lds, p * KT_SIZE + turned_row<KD>(dim + d), dim + d, my_token, w[p]);
            }
        }
        if (my_dim < kColumnsHere) {
            if (not_finite(vn)) {
                bad_chunk = (int32_t)(at / kChunk);
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int d = 0; d < 4; ++d)
                        if (abs_bits(to_f32(vn.row[t].v[d])) > kLargestFinite) {
                            atomicMin(&bad_at[my_dim + d], (int32_t)(my_token + t));
                            vn.row[t].v[d] = from_f32<T>(0.0f);
                        }
            }
            if constexpr (NP == 1) {
                uint2 w[4];
                turned(vn, w);
#pragma unroll
                for (int d = 0; d < 4; ++d) put_tokens(vt_lds, turned_row<kColumnsHere>(my_dim + d), my_dim + d, my_token, w[d]);
            } else {
#pragma unroll
                for (int d = 0; d < 4; ++d) {
                    uint2 w[NP];
                    const float f[4] = {to_f32(vn.row[0].v[d]), to_f32(vn.row[1].v[d]), to_f32(vn.row[2].v[d]), to_f32(vn.row[3].v[d])};
                    pieces_of<NP>(f, w);
#pragma unroll
                    for (int p = 0; p < NP; ++p) put_tokens(vt_lds, p * VT_SIZE + turned_row<kColumnsHere>(my_dim + d), my_dim + d, my_token, w[p]);
                }
            }
        }
        const float decays = decay_ahead;  // the next chunk's, asked for a chunk ago
        decay_ahead = next_decay(at + 2 * kChunk);
        if (at + kChunk < rows) fetch(rows - at - kChunk);
        __syncthreads();
        const bool some_bad = __builtin_amdgcn_readfirstlane(bad_chunk) == (int32_t)(at / kChunk);
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
                    const float w = p[i] * (__builtin_amdgcn_exp2f((float)(bi - sums_lds[16 * jt + 4 * g + i])) * a.scale);
                    f[i] = it > jt || m >= 4 * g + i ? w : 0.0f;
                }
                uint2 w[NO];
                pieces_of<NO>(f, w);
#pragma unroll
                for (int x = 0; x < NO; ++x) put_tokens(p_lds, p_row(x, 16 * it + m), m, 16 * jt + 4 * g, w[x]);
                if (tile == 0)  // tokens 16 .. 31 of rows 0 .. 15
#pragma unroll
                    for (int x = 0; x < NO; ++x) put_tokens(p_lds, p_row(x, m), m, 16 + 4 * g, uint2{0, 0});
            }
            // ---- out^T = S^T q^T, faded
            float4v o[UT][2] = {};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                uint4 qf[NP][2];
#pragma unroll
                for (int x = 0; x < NP; ++x)
#pragma unroll
                    for (int it = 0; it < 2; ++it) qf[x][it] = q_lds[row_at(x, 16 * it + m, ks)];
#pragma unroll
                for (int u = 0; u < UT; ++u) {
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
                const float f = fades_lds[16 * it + m];
#pragma unroll
                for (int u = 0; u < UT; ++u) o[u][it] *= f;
            }
            __syncthreads();
            // ---- ... and V^T P^T
#pragma unroll
            for (int u = 0; u < UT; ++u)
#pragma unroll
                for (int x = 0; x < NP; ++x) {
                    const uint4 vf = halves(vt_lds[x * VT_SIZE + turned_row<kColumnsHere>(wave * (16 * UT) + 16 * u + m) + (g ^ beside(m))], (wave * (16 * UT) + 16 * u) / 64 % 2);
#pragma unroll
                    for (int y = 0; y < NO && x + y < NO; ++y)
#pragma unroll
                        for (int it = 0; it < 2; ++it) o[u][it] = mfma(vf, p_lds[p_row(y, 16 * it + m) + (g ^ beside(m))], o[u][it]);
                }
            // ---- out, by way of this wave's part of LDS: lanes side by side in a row
            constexpr int OP = 16 * UT * sizeof(T) / 16;  // pieces of a row
            uint8_t* const o_lds = reinterpret_cast<uint8_t*>(q_lds) + wave * (kChunk * OP * 16);
            const auto o_at = [](uint32_t row, uint32_t piece) { return (row * OP + (piece ^ (OP == 8 ? row / 2 & 7 : OP == 4 ? row / 4 & 3 : row / 8 & 1))) * 16; };
            if (some_bad) {
#pragma unroll
                for (int it = 0; it < 2; ++it)
#pragma unroll
                    for (int u = 0; u < UT; ++u)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (bad_at[wave * (16 * UT) + 16 * u + 4 * g + i] <= (int32_t)(16 * it + m)) o[u][it][i] = __uint_as_float(0x7FC00000u);
            }
#pragma unroll
            for (int it = 0; it < 2; ++it)
#pragma unroll
                for (int u = 0; u < UT; ++u) {
                    const uint32_t col = 16 * u + 4 * g, row = 16 * it + m;
                    Vec<T, 4> y;
#pragma unroll
                    for (int i = 0; i < 4; ++i) y.v[i] = from_f32<T>(o[u][it][i]);
                    *reinterpret_cast<Vec<T, 4>*>(o_lds + o_at(row, col * sizeof(T) / 16) + col * sizeof(T) % 16) = y;
                }
            // the wave reads what its own lanes wrote: LDS serves a wave in order
            __builtin_amdgcn_wave_barrier();
#pragma unroll
            for (int j = 0; j < kChunk * OP / 64; ++j) {
                // rows behind the last are the last one once more: stores that all lanes make are counted, and the loads in flight are not waited for
                const uint32_t row = min((j * 64 + lane) / OP, rows - at - 1), piece = (j * 64 + lane) % OP;
                typedef Loose<T, 16 / sizeof(T)> Piece;
                const uint4 y = *reinterpret_cast<const uint4*>(o_lds + o_at(row, piece));
                *reinterpret_cast<Piece*>(out + (uint64_t)(at + row) * a.out.stride + wave * (16 * UT) + piece * (16 / sizeof(T))) = __builtin_bit_cast(Piece, y);
            }
        }
        b = running(decays);
        // ---- S <- e^(b_last) S + k^T v
        held = settle ? 0.0 : grown;
        if (settle) {
            const float f = __builtin_amdgcn_exp2f((float)grown);
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int u = 0; u < UT; ++u) S[t][u] *= f;
        }
        uint4 vf[NP][UT], kf[2][3];  // k^T's tile and the next one's
#pragma unroll
        for (int x = 0; x < 3; ++x) kf[0][x] = kt_lds[x * KT_SIZE + turned_row<KD>(m) + (g ^ beside(m))];
#pragma unroll
        for (int x = 0; x < NP; ++x)
#pragma unroll
            for (int u = 0; u < UT; ++u) vf[x][u] = halves(vt_lds[x * VT_SIZE + turned_row<kColumnsHere>(wave * (16 * UT) + 16 * u + m) + (g ^ beside(m))], (wave * (16 * UT) + 16 * u) / 64 % 2);
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            if (t + 1 < KT)
#pragma unroll
                for (int x = 0; x < 3; ++x) kf[(t + 1) % 2][x] = kt_lds[x * KT_SIZE + turned_row<KD>(16 * (t + 1) + m) + (g ^ beside(m))];
#pragma unroll
            for (int x = 0; x < 3; ++x) {
                const uint4 k = halves(kf[t % 2][x], t / 4 % 2);
#pragma unroll
                for (int y = 0; y < NP && x + y < 3; ++y)
#pragma unroll
                    for (int u = 0; u < UT; ++u) S[t][u] = mfma(k, vf[y][u], S[t][u]);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (some_bad) {
#pragma unroll
            for (int u = 0; u < UT; ++u)
                if (bad_at[wave * (16 * UT) + 16 * u + m] < kChunk)
#pragma unroll
                    for (int t = 0; t < KT; ++t) S[t][u] = float4v{} + __uint_as_float(0x7FC00000u);
            if (lane < 16 * UT) bad_at[wave * (16 * UT) + lane] = kChunk;  // these columns are this wave's alone
        }
        __syncthreads();
    }
    float* after = nullptr;
    if (STATES) after = seg.states + ((uint64_t)boundary * a.heads + head) * plane;
    else if (last_part && part > 0 && a.state == a.state_out) after = seg.states + ((uint64_t)(boundary - 1) * a.heads + head) * plane;  // for k_linear_settle
    else if (last_part) after = a.state_out + ((uint64_t)slot * a.heads + head) * plane;
    const float settled = __builtin_amdgcn_exp2f((float)held);
    if (after)
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int u = 0; u < UT; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) after[mine + (uint64_t)(16 * t + i) * a.v_dim + 16 * u] = S[t][u][i] * settled;
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

// In place, the last segment of a sequence leaves its state where the one before it was: the first segment may not have read the pool's yet. Then
// it goes to the pool.
__global__ __launch_bounds__(kBlock) void k_linear_settle(LinearArgs a, Segments seg) {
    const uint32_t tid = threadIdx.x, head = blockIdx.y, s = blockIdx.z, at = (blockIdx.x * kBlock + tid) * 4, plane = a.k_dim * a.v_dim;
    const LinearRows r = linear_rows(a, s);
    if (cuts_of(seg, r.rows) == 0) return;
    const int32_t slot = a.slots[s];
    Cuts cuts;
    if (!look_up(a, seg, s, slot, r.rows, kBlock, cuts) || cuts.parts == 0 || at >= plane) return;
    *reinterpret_cast<float4v*>(a.state_out + ((uint64_t)slot * a.heads + head) * plane + at) =
        *reinterpret_cast<const float4v*>(seg.states + ((uint64_t)(cuts.base + cuts.parts - 1) * a.heads + head) * plane + at);
}

constexpr uint32_t kCus = 256;
// Up to this many rows of a sequence go one after another: a chunk costs the same for one row as for 32, and more the more pieces its type has (48 heads
// of 128; 8 and 61 sequences: 6 rows of BF16 in 16.3 and 86.0 us, a chunk in 17.0 and 97 to 100; 8 of F16 in 18.8 and 93.6, a chunk in 19.2 and 111 to 115; 16
// of F32 in 25.5 and 142, a chunk in 26.2 and 163).
template <typename T>
constexpr uint32_t kFewRows = kPieces<T> == 1 ? 6 : kPieces<T> == 2 ? 8 : 16;

// Columns of a workgroup: a whole head's where they are 64, 96 or 128.
uint32_t columns_of(const LinearArgs& a) { return a.v_dim == 64 ? 64 : a.v_dim % 128 == 0 ? 128 : 96; }

// How sequences are cut into segments with part_bytes of workspace, and the bytes made use of.
Segments plan_segments(const LinearArgs& a, uint64_t part_bytes, uint64_t* bytes) {
    Segments seg{std::max(a.max_rows, 1u), 1, 0, nullptr, nullptr};
    *bytes = 0;
    const uint64_t per = (uint64_t)a.heads * (a.k_dim * a.v_dim + 1) * 4;  // of a boundary
    const uint64_t blocks = (uint64_t)a.heads * (a.v_dim / columns_of(a));
    // two workgroups a CU, as many as run at once, where a sequence's last segment is half one (four prompts of 1639 to 5000 rows, 48 heads: BF16 351 us, with
    // three 405; F32 746, with three 796); no segment under 256 rows. Every sequence counts here, those of one row too: a prompt of 5000 rows beside 16 of one
    // row is cut into three, beside 20 not at all (134, 267 and 501 us)
    const uint64_t target = 2 * kCus, ends = a.n_seqs * blocks / 2;
    uint64_t length = a.max_rows;
    if (ends < target) length = std::max<uint64_t>(256, (a.n_rows * blocks / (target - ends) + kChunk - 1) / kChunk * kChunk);
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
    uint32_t columns = columns_of(a);
    // few workgroups: of half the columns each (fp32, 48 heads of 128, 256 rows: 42.4 us against 51.8)
    if (columns == 128 && (uint64_t)a.heads * (a.v_dim / 128) * a.n_seqs * seg.most <= kCus / 2) columns = 64;
    const uint32_t blocks = a.heads * (a.v_dim / columns);
    const auto run = [&](auto states) {
        constexpr bool S = decltype(states)::value;
        // 16 columns a wave where q and k take most of the registers and one workgroup the CU (fp32, k_dim 256: a seventh less time)
        constexpr int UT = kPieces<T> * KD >= 768 ? 1 : 2;
        auto* k = columns == 64 ? k_linear_chunks<T, KD, 4, 1, S> : columns == 96 ? k_linear_chunks<T, KD, 6 / UT, UT, S> : k_linear_chunks<T, KD, 8 / UT, UT, S>;
        hipLaunchKernelGGL(k, dim3(blocks, S ? seg.most - 1 : seg.most, a.n_seqs), dim3(columns == 64 ? 256 : columns / 16 / UT * 64), 0, st, a, seg);
    };
    const dim3 planes((a.k_dim * a.v_dim / 4 + kBlock - 1) / kBlock, a.heads, a.n_seqs);
    if (seg.most > 1) {
        run(std::true_type{});
        hipLaunchKernelGGL(k_linear_join, planes, dim3(kBlock), 0, st, a, seg);
    }
    run(std::false_type{});
    if (seg.most > 1 && a.state == a.state_out) hipLaunchKernelGGL(k_linear_settle, planes, dim3(kBlock), 0, st, a, seg);
    return hip_status(hipGetLastError(), "linear_attention");
}

template <typename T>
int launch_typed(const LinearArgs& a, float* part, uint64_t part_bytes, hipStream_t st) {
    if (a.max_rows > kFewRows<T>) {
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
