// gfx950 kernels that write rows into the 8-bit paged cache and read them back (KV_WRITE, KvWriteArgs at
// include/halo/backend/backend.h:379-390 of the reference).
//
// A page holds block tokens of a layer as int8 codes with one scale for K and one for V per head. Rows that
// fall into a page widen its scale to max(scale, amax / 127); where it grew, the codes of the tokens that the
// page holds already move to the new scale. Codes are the nearest integers to x / scale exactly (ties to even):
// the fp32 product with the reciprocal is within 2^-22 of the quotient, and only a value that close to a border
// between two codes is decided in 64 bits, where both sides of the comparison are exact.
//
// One workgroup owns one (page, K or V, head): nobody else touches its codes and scale. K rows are [token][dim];
// V is [dim][token], so a thread takes 16 tokens of one dim and stores them as 16 bytes.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kv.h"
#include "kv_device.h"
#include "launch.h"

namespace halo_mi {
namespace {

using namespace dev;

constexpr uint32_t kKvBlock = 256;

// The integer nearest to x / s (ties to even) for |x| <= 127.5 s, s > 0; inv = 1 / s rounded.
__device__ __forceinline__ int32_t nearest(float x, float s, float inv) {
    const float q = x * inv;
    int32_t r = (int32_t)rintf(q);
    const float from_border = 0.5f - fabsf(q - (float)r);
    if (from_border < 0x1p-14f) {  // 2^-22 * 127 at most is lost in q
        // 2 x against (2 r + 1) s and (2 r - 1) s: 24 + 9 bits, exact in 64
        const double x2 = 2.0 * x, up = (double)(2 * r + 1) * s, down = (double)(2 * r - 1) * s;
        if (x2 > up || (x2 == up && (r & 1))) ++r;
        else if (x2 < down || (x2 == down && (r & 1))) --r;
    }
    return min(max(r, -127), 127);
}

// The code c of a block of scale s0 in scale s1 > s0: the integer nearest to c * s0 / s1, exactly.
__device__ __forceinline__ int32_t rescaled(int32_t c, float s0, float s1) {
    const double x2 = 2.0 * c * s0;
    int32_t r = (int32_t)rint(x2 / (2.0 * s1));
    const double up = (double)(2 * r + 1) * s1, down = (double)(2 * r - 1) * s1;
    if (x2 > up || (x2 == up && (r & 1))) ++r;
    else if (x2 < down || (x2 == down && (r & 1))) --r;
    return r;
}

__device__ __forceinline__ uint32_t rescaled4(uint32_t codes, float s0, float s1) {
    uint32_t out = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) out |= (uint32_t)(uint8_t)rescaled((int8_t)(codes >> (8 * i)), s0, s1) << (8 * i);
    return out;
}

// What one workgroup of a write or read has: tokens [lo, hi) of a sequence, in one page.
struct PagePart {
    int32_t page;      // -1: out of range
    uint32_t row;      // of token lo
    uint32_t off, n;   // lo's place in the page, tokens
};

// The j-th page that a sequence's rows touch; false when there is none. Rows before position 0 belong to no page.
__device__ __forceinline__ bool page_part(const KvBatch& b, const KvLayer& c, uint32_t s, const SeqRows& r, uint32_t j, PagePart& p) {
    const int32_t first = r.len - r.rows;  // position of the first row
    const uint32_t a = max(first, 0), index = (a >> c.block_log2) + j;
    const uint32_t begin = index << c.block_log2;
    const uint32_t lo = max(a, begin), hi = min((uint32_t)r.len, begin + c.block);
    if (lo >= hi || r.rows == 0) return false;
    p.row = r.row0 + (uint32_t)((int32_t)lo - first);
    p.off = lo - begin;
    p.n = hi - lo;
    p.page = page_at(b, c, s, index);
    return true;
}

// V: elements per load of a K or V row.
template <typename T, int V>
__device__ void write_part(const KvWriteArgs& a, const PagePart& p, uint32_t which, uint32_t head, uint32_t* lds) {
    const KvLayer& c = a.c;
    const uint32_t tid = threadIdx.x, dim = c.dim;
    uint8_t* page = c.pool + (uint64_t)(uint32_t)p.page * c.page_bytes;
    uint8_t* codes = page + c.codes + (which * c.heads + head) * c.plane;
    float* scale = reinterpret_cast<float*>(page + c.scales) + which * c.heads + head;
    const T* x = static_cast<const T*>(a.x[which].data) + (uint64_t)p.row * a.x[which].stride + head * a.x[which].head_stride;
    const uint64_t stride = a.x[which].stride;
    const float s0 = p.off ? *scale : 0.0f;

    uint32_t top = 0;
    const uint32_t vecs = dim / V;
    for (uint32_t i = tid; i < p.n * vecs; i += kKvBlock) {
        const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(x + (i / vecs) * stride + i % vecs * V);
#pragma unroll
        for (int k = 0; k < V; ++k) top = max(top, abs_bits(to_f32(v.v[k])));
    }
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
    if (tid % 64 == 0) lds[tid / 64] = top;
    __syncthreads();
    top = max(max(lds[0], lds[1]), max(lds[2], lds[3]));
    const float fit = __uint_as_float(top) / 127.0f;
    float s1 = fit < kKvMinScale ? s0 : fmaxf(s0, fit);
    if (top > kLargestFinite || s0 != s0) s1 = __uint_as_float(0x7FC00000u);
    __syncthreads();  // every thread has s0 and the partial maxima
    if (tid == 0) *scale = s1;
    if (s1 != s1) return;  // the codes of a NaN block mean nothing
    const bool grew = p.off && s1 > s0 && s0 > 0.0f;
    const float inv = s1 > 0.0f ? 1.0f / s1 : 0.0f;
    auto code = [&](float v) { return s1 > 0.0f ? (uint32_t)(uint8_t)nearest(v, s1, inv) : 0u; };

    if (which == 0) {
        uint32_t* rows = reinterpret_cast<uint32_t*>(codes);
        if (grew)
            for (uint32_t i = tid; i < p.off * dim / 4; i += kKvBlock) rows[i] = rescaled4(rows[i], s0, s1);
        constexpr int W = V < 4 ? 4 : V;  // codes per store
        for (uint32_t i = tid; i < p.n * (dim / W); i += kKvBlock) {
            const uint32_t t = i / (dim / W), d = i % (dim / W) * W;
            uint32_t word[W / 4] = {};
#pragma unroll
            for (int k = 0; k < W; k += V) {
                const Vec<T, V> v = *reinterpret_cast<const Vec<T, V>*>(x + t * stride + d + k);
#pragma unroll
                for (int j = 0; j < V; ++j) word[(k + j) / 4] |= code(to_f32(v.v[j])) << (8 * ((k + j) % 4));
            }
#pragma unroll
            for (int k = 0; k < W / 4; ++k) rows[((p.off + t) * dim + d) / 4 + k] = word[k];
        }
        return;
    }
    // V: 16 tokens of one dim at a time; from the page's first one where the earlier codes change
    const uint32_t g0 = grew ? 0 : p.off / 16, g1 = (p.off + p.n + 15) / 16;
    for (uint32_t i = tid; i < (g1 - g0) * dim; i += kKvBlock) {
        const uint32_t d = i % dim, t0 = (g0 + i / dim) * 16;
        uint4* at = reinterpret_cast<uint4*>(codes + d * c.block + t0);
        uint4 old = {};
        if (t0 < p.off || t0 + 16 > p.off + p.n) old = *at;
        uint32_t word[4] = {old.x, old.y, old.z, old.w};
#pragma unroll
        for (uint32_t k = 0; k < 16; ++k) {
            const uint32_t t = t0 + k, shift = 8 * (k % 4), have = word[k / 4];
            uint32_t v;
            if (t >= p.off && t < p.off + p.n) v = code(to_f32(x[(t - p.off) * stride + d]));
            else if (t < p.off && grew) v = (uint8_t)rescaled((int8_t)(have >> shift), s0, s1);
            else continue;
            word[k / 4] = (have & ~(0xFFu << shift)) | v << shift;
        }
        *at = {word[0], word[1], word[2], word[3]};
    }
}

template <typename T, int V>
__global__ __launch_bounds__(kKvBlock) void k_kv_write(KvWriteArgs a) {
    __shared__ uint32_t lds[kKvBlock / 64];
    const uint32_t s = blockIdx.z, head = blockIdx.y >> 1, which = blockIdx.y & 1;
    const SeqRows r = seq_rows(a.b, s);
    PagePart p;
    for (uint32_t j = blockIdx.x; page_part(a.b, a.c, s, r, j, p); j += gridDim.x) {
        if (p.page < 0) {
            if (threadIdx.x == 0) set_status(a.status, kStatusKvBadIndex);
            continue;
        }
        write_part<T, V>(a, p, which, head, lds);
        __syncthreads();
    }
}

__global__ __launch_bounds__(kKvBlock) void k_kv_read(KvReadArgs a) {
    const uint32_t s = blockIdx.z, head = blockIdx.y >> 1, which = blockIdx.y & 1, dim = a.c.dim;
    if (!a.out[which].data) return;
    const SeqRows r = seq_rows(a.b, s);
    float* out = const_cast<float*>(static_cast<const float*>(a.out[which].data)) + head * a.out[which].head_stride;
    const uint64_t stride = a.out[which].stride;
    if (r.len < r.rows)  // rows before position 0
        for (uint64_t i = blockIdx.x * kKvBlock + threadIdx.x; i < (uint64_t)(r.rows - r.len) * dim; i += gridDim.x * kKvBlock)
            out[(r.row0 + i / dim) * stride + i % dim] = 0.0f;
    PagePart p;
    for (uint32_t j = blockIdx.x; page_part(a.b, a.c, s, r, j, p); j += gridDim.x) {
        float* o = out + (uint64_t)p.row * stride;
        if (p.page < 0) {
            if (threadIdx.x == 0) set_status(a.status, kStatusKvBadIndex);
            for (uint32_t i = threadIdx.x; i < p.n * dim; i += kKvBlock) o[i / dim * stride + i % dim] = __uint_as_float(0x7FC00000u);
            continue;
        }
        const uint8_t* page = page_ptr(a.c, p.page);
        const uint8_t* codes = page + a.c.codes + (which * a.c.heads + head) * a.c.plane;
        const float scale = reinterpret_cast<const float*>(page + a.c.scales)[which * a.c.heads + head];
        if (which == 0) {
            for (uint32_t i = threadIdx.x; i < p.n * dim / 4; i += kKvBlock) {
                const uint32_t word = reinterpret_cast<const uint32_t*>(codes + p.off * dim)[i];
                float* to = o + i / (dim / 4) * stride + i % (dim / 4) * 4;
#pragma unroll
                for (int k = 0; k < 4; ++k) to[k] = (float)(int8_t)(word >> (8 * k)) * scale;
            }
            continue;
        }
        const uint32_t g0 = p.off / 16, g1 = (p.off + p.n + 15) / 16;
        for (uint32_t i = threadIdx.x; i < (g1 - g0) * dim; i += kKvBlock) {
            const uint32_t d = i % dim, t0 = (g0 + i / dim) * 16;
            const uint4 w = *reinterpret_cast<const uint4*>(codes + d * a.c.block + t0);
            const uint32_t word[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (uint32_t k = 0; k < 16; ++k)
                if (t0 + k >= p.off && t0 + k < p.off + p.n)
                    o[(t0 + k - p.off) * stride + d] = (float)(int8_t)(word[k / 4] >> (8 * (k % 4))) * scale;
        }
    }
}

// Pages that a sequence's rows touch at most: rows begin inside a page.
dim3 page_grid(const KvLayer& c, const KvBatch& b) {
    const uint64_t pages = ((uint64_t)b.max_rows + 2 * c.block - 2) / c.block;
    return dim3((uint32_t)std::min<uint64_t>(pages, 65535), 2 * c.heads, b.n_seqs);
}

template <typename T>
int launch_write_typed(const KvWriteArgs& a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    bool wide = true;
    for (const HeadRows& r : a.x)
        wide = wide && reinterpret_cast<uintptr_t>(r.data) % 16 == 0 && r.stride % V == 0 && r.head_stride % V == 0;
    hipLaunchKernelGGL((wide ? k_kv_write<T, V> : k_kv_write<T, 1>), page_grid(a.c, a.b), dim3(kKvBlock), 0, st, a);
    return hip_status(hipGetLastError(), "KV_WRITE");
}

}  // namespace

int launch_kv_write(uint32_t type, const KvWriteArgs& a, hipStream_t st) {
    switch (type) {
        case HALO_MI_F16: return launch_write_typed<_Float16>(a, st);
        case HALO_MI_BF16: return launch_write_typed<__bf16>(a, st);
        default: return launch_write_typed<float>(a, st);
    }
}

int launch_kv_read(const KvReadArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(k_kv_read, page_grid(a.c, a.b), dim3(kKvBlock), 0, st, a);
    return hip_status(hipGetLastError(), "kv_read");
}

}  // namespace halo_mi
