// gfx950 kernels that write rows into the 8-bit paged cache and read them back (KV_WRITE, KvWriteArgs at
// include/halo/backend/backend.h:379-390 of the reference).
//
// A page holds block tokens of a layer as int8 codes with one scale for K and one for V per head. Rows that
// fall into a page widen its scale to max(scale, amax / 127); where it grew, the codes of the tokens that the
// page holds already move to the new scale. Codes are the nearest integers to x / scale exactly (ties to even).
//
// One workgroup owns one (page, K or V, head): nobody else touches its codes and scale. K rows are [token][dim], V
// [dim][token]: a thread takes patches of 4 tokens by 4 elements of a row, which are whole words of V's codes, and keeps
// them in registers from the maximum to the codes, so that x is read once. V's threads lie along the tokens, so that
// their words join into whole lines (17.6 us against 18.7 with threads along the dims).
//
// Bound by memory: 7 bf16 prompts of 201 to 2100 rows, 8 heads of 128, written in 17.6 us (56 MB, 3.2 TB/s: the chain of
// lengths, rows, maximum and codes of a workgroup shows, as 2300 workgroups are not much more than fit at once) and read
// back in 18.2 (94 MB, 5.2 TB/s); 61 sequences' single tokens 5.4 and 5.8 us, one launch each.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <type_traits>

#include "kv.h"
#include "kv_device.h"
#include "launch.h"

namespace halo_mi {
namespace {

using namespace dev;

constexpr uint32_t kKvBlock = 256;

// The code c of a block of scale s0 in scale s1 > s0: the integer nearest to c * s0 / s1, exactly.
__device__ __forceinline__ int32_t rescaled(int32_t c, float s0, float s1) {
    const double x2 = 2.0 * c * s0;
    int32_t r = (int32_t)rint(x2 / (2.0 * s1));
    const double up = (double)(2 * r + 1) * s1, down = (double)(2 * r - 1) * s1;
    if (x2 > up || (x2 == up && (r & 1))) ++r;
    else if (x2 < down || (x2 == down && (r & 1))) --r;
    return r;
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

// A thread's patch: 4 tokens that share a word of V's codes, V consecutive dims of each.
template <typename T, int V>
struct Patch {
    Vec<T, V> row[4];
};

// The largest |element| of a patch as a word that orders like it (abs_bits, or the type's own 16 bits twice).
template <typename T, int V>
__device__ __forceinline__ uint32_t patch_peak(const Patch<T, V>& q, uint32_t top) {
    if constexpr (sizeof(T) == 2 && V > 1) {
        typedef uint16_t ushort2v __attribute__((ext_vector_type(2)));
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const uint32_t w = (uint32_t)__builtin_bit_cast(uint16_t, q.row[k].v[j]) | (uint32_t)__builtin_bit_cast(uint16_t, q.row[k].v[j + 1]) << 16;
                top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(ushort2v, top), __builtin_bit_cast(ushort2v, w & 0x7FFF7FFFu)));
            }
    } else {
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
            for (int j = 0; j < V; ++j) top = max(top, abs_bits(to_f32(q.row[k].v[j])));
    }
    return top;
}
// ... and what it stands for, as abs_bits.
template <typename T, int V>
__device__ __forceinline__ uint32_t peak_bits(uint32_t top) {
    if constexpr (sizeof(T) == 2 && V > 1) {
        const uint16_t h = (uint16_t)max(top & 0xFFFFu, top >> 16);
        return abs_bits(to_f32(__builtin_bit_cast(T, h)));
    } else {
        return top;
    }
}

// V: elements per load of a K or V row, 4 or 1. KEEP: patches per thread that stay in registers between the maximum and
// the codes; a part with more is read again. THREADS: of the workgroup, as few as have a whole page's patches between them,
// so that more pages of 16 tokens are under way at once. A thread has one place of `vecs` in a row and every `at_once`-th
// group of 4 tokens.
template <typename T, int V, int KEEP, uint32_t THREADS>
__device__ void write_part(const KvWriteArgs& a, const PagePart& p, uint32_t which, uint32_t head, uint32_t* lds) {
    typedef std::conditional_t<V == 1, uint64_t, uint32_t> Offset;  // wide rows are at most 2^22 elements apart
    const KvLayer& c = a.c;
    const uint32_t tid = threadIdx.x, dim = c.dim, vecs = dim / V, at_once = min(THREADS / vecs, c.block / 4);
    // V's words of 4 tokens lie side by side along the tokens: 8 lanes along a row, then up to 8 groups of tokens
    const uint32_t beside = which ? min(at_once & -at_once, 8u) : 1, rest = tid / 8 / beside;
    const uint32_t d = (rest % (vecs / 8) * 8 + tid % 8) * V, mine_first = rest / (vecs / 8) * beside + tid / 8 % beside;
    const T* x = static_cast<const T*>(a.x[which].data) + (uint64_t)p.row * a.x[which].stride + head * a.x[which].head_stride;
    const Offset stride = (Offset)a.x[which].stride;
    // groups of 4 tokens, aligned in the page, that the part touches
    const uint32_t g0 = p.off / 4, groups = (p.off + p.n + 3) / 4 - g0, my_groups = mine_first < at_once ? groups : 0;
    const bool kept = groups <= KEEP * at_once;
    const auto load = [&](uint32_t g, Patch<T, V>& q) {
        const uint32_t t0 = (g0 + g) * 4;
        // tokens outside the part repeat its nearest row: no branch, the same maximum; their codes are not stored
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            q.row[k] = *reinterpret_cast<const Vec<T, V>*>(x + ((Offset)(min(max(t0 + k, p.off), p.off + p.n - 1) - p.off) * stride + d));
    };
    uint32_t top = 0;
    Patch<T, V> mine[KEEP];
    if (kept) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) load(min(mine_first + j * at_once, groups - 1), mine[j]);  // past the end: not used
    }
    if (p.page < 0) {  // the rows are on their way while the table's entry is
        if (tid == 0) set_status(a.status, kStatusKvBadIndex);
        return;
    }
    uint8_t* page = c.pool + (uint64_t)(uint32_t)p.page * c.page_bytes;
    uint8_t* codes = page + c.codes + (which * c.heads + head) * c.plane;
    uint32_t* words = reinterpret_cast<uint32_t*>(codes);
    float* scale = reinterpret_cast<float*>(page + c.scales) + which * c.heads + head;
    const float s0 = p.off ? *scale : 0.0f;
    if (kept) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) top = patch_peak(mine[j], top);
    } else {
        for (uint32_t g = mine_first; g < my_groups; g += at_once) {
            load(g, mine[0]);
            top = patch_peak(mine[0], top);
        }
    }
    top = peak_bits<T, V>(top);
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, off));
    if (tid % 64 == 0) lds[tid / 64] = top;
    __syncthreads();  // every thread has s0, too
    top = lds[0];
#pragma unroll
    for (uint32_t w = 1; w < THREADS / 64; ++w) top = max(top, lds[w]);
    const float fit = __uint_as_float(top) / 127.0f;
    float s1 = fit < kKvMinScale ? s0 : fmaxf(s0, fit);
    if (top > kLargestFinite || s0 != s0) s1 = __uint_as_float(0x7FC00000u);
    if (tid == 0) *scale = s1;
    if (s1 != s1) return;  // the codes of a NaN block mean nothing

    if (p.off && s1 > s0 && s0 > 0.0f) {  // the scale grew: the earlier tokens' codes follow
        const uint32_t per = which ? (p.off + 3) / 4 : p.off * dim / 4;  // words of a dim of V; of K
        const uint32_t rows = which ? dim : 1;
        for (uint32_t i = tid; i < per * rows; i += THREADS) {
            uint32_t* w = words + i / per * (c.block / 4) + i % per;
            const uint32_t keep = !which || i % per * 4 + 4 <= p.off ? 0u : 0xFFFFFFFFu << 8 * (p.off % 4);
            uint32_t word = *w & keep;
            for (uint32_t k = 0; k < 32; k += 8)
                if (!(keep >> k & 1)) word |= (uint32_t)(uint8_t)rescaled((int8_t)(*w >> k), s0, s1) << k;
            *w = word;
        }
        __syncthreads();
    }
    const float inv = s1 > 0.0f ? 1.0f / s1 : 0.0f;
    // The patch's codes; exactly where an element is too near a border to be sure. code[k][j]: token k, dim j.
    const auto codes_of = [&](const Patch<T, V>& q, uint32_t (&code)[4][V]) {
        const auto all = [&](auto exact, float by, float times) {
            bool unsure = false;
#pragma unroll
            for (int k = 0; k < 4; ++k)
#pragma unroll
                for (int j = 0; j < V; ++j) code[k][j] = nearest<decltype(exact)::value>(to_f32(q.row[k].v[j]), by, times, unsure);
            return unsure;
        };
        if (all(std::false_type{}, s1, inv)) {
            float by = s1, again = inv;
            __asm__ volatile("" : "+v"(by), "+v"(again));  // nothing of the first pass is kept in registers for this one
            all(std::true_type{}, by, again);
        }
    };
    const auto store = [&](uint32_t g, const Patch<T, V>& q) {
        const uint32_t t0 = (g0 + g) * 4;
        uint32_t code[4][V] = {};
        if (s1 > 0.0f) codes_of(q, code);
        const bool whole = t0 >= p.off && t0 + 4 <= p.off + p.n;
        const auto mine_too = [&](uint32_t k) { return whole || (t0 + k >= p.off && t0 + k < p.off + p.n); };
        if (which == 0) {
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k) {
                if (!mine_too(k)) continue;
                if constexpr (V == 4) words[((t0 + k) * dim + d) / 4] = low_bytes(code[k][0], code[k][1], code[k][2], code[k][3]);
                else codes[(t0 + k) * dim + d] = (uint8_t)code[k][0];
            }
            return;
        }
#pragma unroll
        for (int j = 0; j < V; ++j) {
            uint32_t* w = words + ((d + j) * c.block + t0) / 4;
            uint32_t word = low_bytes(code[0][j], code[1][j], code[2][j], code[3][j]);
            if (!whole) {  // the word's other tokens keep their bytes
                uint32_t cover = 0;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k) cover |= mine_too(k) ? 0xFFu << 8 * k : 0u;
                word = (*w & ~cover) | (word & cover);
            }
            *w = word;
        }
    };
    if (kept) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j)
            if (mine_first + j * at_once < my_groups) store(mine_first + j * at_once, mine[j]);
    } else {
        for (uint32_t g = mine_first; g < my_groups; g += at_once) {
            load(g, mine[0]);
            store(g, mine[0]);
        }
    }
}

template <typename T, int V, int KEEP, uint32_t THREADS>
__global__ __launch_bounds__(THREADS) void k_kv_write(KvWriteArgs a) {
    __shared__ uint32_t lds[THREADS / 64];
    const uint32_t s = blockIdx.z, head = blockIdx.y >> 1, which = blockIdx.y & 1;
    const SeqRows r = seq_rows(a.b, s);
    PagePart p;
    for (uint32_t j = blockIdx.x; page_part(a.b, a.c, s, r, j, p); j += gridDim.x) {
        write_part<T, V, KEEP, THREADS>(a, p, which, head, lds);
        __syncthreads();
    }
}

__global__ __launch_bounds__(kKvBlock) void k_kv_read(KvReadArgs a) {
    const uint32_t threads = blockDim.x;  // a page's 16 tokens of a dim each, up to kKvBlock
    const uint32_t s = blockIdx.z, head = blockIdx.y >> 1, which = blockIdx.y & 1, dim = a.c.dim;
    if (!a.out[which].data) return;
    const SeqRows r = seq_rows(a.b, s);
    float* out = const_cast<float*>(static_cast<const float*>(a.out[which].data)) + head * a.out[which].head_stride;
    const uint64_t stride = a.out[which].stride;
    if (r.len < r.rows)  // rows before position 0
        for (uint64_t i = blockIdx.x * threads + threadIdx.x; i < (uint64_t)(r.rows - r.len) * dim; i += gridDim.x * threads)
            out[(r.row0 + i / dim) * stride + i % dim] = 0.0f;
    PagePart p;
    for (uint32_t j = blockIdx.x; page_part(a.b, a.c, s, r, j, p); j += gridDim.x) {
        float* o = out + (uint64_t)p.row * stride;
        if (p.page < 0) {
            if (threadIdx.x == 0) set_status(a.status, kStatusKvBadIndex);
            for (uint32_t i = threadIdx.x; i < p.n * dim; i += threads) o[i / dim * stride + i % dim] = __uint_as_float(0x7FC00000u);
            continue;
        }
        const uint8_t* page = page_ptr(a.c, p.page);
        const uint8_t* codes = page + a.c.codes + (which * a.c.heads + head) * a.c.plane;
        const float scale = reinterpret_cast<const float*>(page + a.c.scales)[which * a.c.heads + head];
        if (which == 0) {
            for (uint32_t i = threadIdx.x; i < p.n * dim / 4; i += threads) {
                const uint32_t word = reinterpret_cast<const uint32_t*>(codes + p.off * dim)[i];
                float* to = o + i / (dim / 4) * stride + i % (dim / 4) * 4;
#pragma unroll
                for (int k = 0; k < 4; ++k) to[k] = (float)(int8_t)(word >> (8 * k)) * scale;
            }
            continue;
        }
        const uint32_t g0 = p.off / 16, g1 = (p.off + p.n + 15) / 16;
        for (uint32_t i = threadIdx.x; i < (g1 - g0) * dim; i += threads) {
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
    constexpr int V = 4;
    bool wide = true;
    for (const HeadRows& r : a.x)
        wide = wide && reinterpret_cast<uintptr_t>(r.data) % (V * sizeof(T)) == 0 && r.stride % V == 0 && r.head_stride % V == 0 && r.stride <= 1u << 22;
    // Up to two patches of a page per thread in small workgroups: 7 bf16 prompts of 200 to 2000 rows, 8 heads, pages of 16 tokens,
    // written and read back at 64 / 128 / 256 dims in 24 / 32.7 / 56 us, against 32 / 39 / 62 with 256 threads (the reads
    // alike). Larger pages are written faster by 256: pages of 64 tokens at 128 dims 35.9 against 37.4 with 128.
    const uint32_t patches = a.c.block / 4 * (a.c.dim / V), at_once = kKvBlock / (a.c.dim / V);
    const uint32_t each = (a.c.block / 4 + at_once - 1) / at_once;  // patches of a page per thread of 256
    uint32_t threads = kKvBlock;
    void (*k)(KvWriteArgs);
    if (!wide) k = k_kv_write<T, 1, 4, kKvBlock>;
    else if (patches <= 64) k = k_kv_write<T, V, 1, 64>, threads = 64;
    else if (patches <= 128) k = k_kv_write<T, V, 2, 64>, threads = 64;
    else if (patches <= 256) k = k_kv_write<T, V, 2, 128>, threads = 128;
    else k = each <= 2 ? k_kv_write<T, V, 2, kKvBlock> : each <= 4 ? k_kv_write<T, V, 4, kKvBlock> : k_kv_write<T, V, 8, kKvBlock>;
    hipLaunchKernelGGL(k, page_grid(a.c, a.b), dim3(threads), 0, st, a);
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
    const uint32_t threads = std::min(kKvBlock, (a.c.dim * a.c.block / 16 + 63) / 64 * 64);
    hipLaunchKernelGGL(k_kv_read, page_grid(a.c, a.b), dim3(threads), 0, st, a);
    return hip_status(hipGetLastError(), "kv_read");
}

}  // namespace halo_mi
