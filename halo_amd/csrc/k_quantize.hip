// gfx950 kernel that holds rows in 8 bits: scale = max |x| / 127 of the row, code = the integer nearest to x / scale (exactly, ties to
// even). One workgroup has a row; what a thread has of it stays in its registers between the maximum and the codes, so that x is read
// once (rows too wide for that are read again).
//
// Memory bounds it: 3990 rows of 5120 in bfloat16 take 14.5 us (4.2 TB/s read and written), 17408 rows 49.7 (5.4). Each code is rounded by one
// multiply-add and checked by another; only where the check cannot tell is the exact step taken (taken always: 17.8 and 61.5).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kv_device.h"
#include "launch.h"
#include "layer.h"

namespace halo_mi {
namespace {

using namespace dev;

// V elements that need not begin on more than an element: rows of any stride are read with whole 16-byte loads.
template <typename T, int V>
struct __attribute__((packed, aligned(sizeof(T)))) Loose {
    T v[V];
};

// KEEP: units of V elements per thread that stay in registers; 0: rows of any width, read twice.
template <typename T, uint32_t THREADS, int KEEP>
__global__ __launch_bounds__(THREADS) void k_quantize_rows(QuantizeArgs a) {
    constexpr int V = 16 / sizeof(T);
    constexpr uint32_t kWaves = THREADS / 64;
    __shared__ uint32_t tops[kWaves];
    const uint32_t tid = threadIdx.x, units = (a.cols + 15) / 16 * (16 / V);
    const T* x = static_cast<const T*>(a.x) + (uint64_t)blockIdx.x * a.x_stride;
    const auto fetch = [&](uint32_t u) {
        Vec<T, V> r{};
        const uint32_t e = u * V;
        if (e + V <= a.cols) {
            r = __builtin_bit_cast(Vec<T, V>, *reinterpret_cast<const Loose<T, V>*>(x + e));
        } else {
#pragma unroll
            for (int i = 0; i < V; ++i)
                if (e + i < a.cols) r.v[i] = x[e + i];
        }
        return r;
    };
    uint32_t top = 0;
    const auto peak = [&](const Vec<T, V>& r) {
#pragma unroll
        for (int i = 0; i < V; ++i) top = max(top, abs_bits(to_f32(r.v[i])));
    };
    Vec<T, V> kept[KEEP ? KEEP : 1];
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j) kept[j] = tid + j * THREADS < units ? fetch(tid + j * THREADS) : Vec<T, V>{};
#pragma unroll
        for (int j = 0; j < KEEP; ++j) peak(kept[j]);
    } else {
        for (uint32_t u = tid; u < units; u += THREADS) peak(fetch(u));
    }
#pragma unroll
    for (int i = 1; i < 64; i *= 2) top = max(top, (uint32_t)__shfl_xor((int)top, i));
    if constexpr (kWaves > 1) {
        if (tid % 64 == 0) tops[tid / 64] = top;
        __syncthreads();
#pragma unroll
        for (uint32_t w = 0; w < kWaves; ++w) top = max(top, tops[w]);
    }
    const bool finite = top <= kLargestFinite;
    float scale = __uint_as_float(top) / 127.0f;
    if (scale < kKvMinScale) scale = 0.0f;
    const float inv = finite && scale > 0.0f ? 1.0f / scale : 0.0f;
    if (tid == 0) a.scales[blockIdx.x] = finite ? scale : __uint_as_float(0x7FC00000u);
    int8_t* codes = a.codes + (uint64_t)blockIdx.x * a.codes_stride;
    const auto put = [&](uint32_t u, const Vec<T, V>& r) {
        uint32_t c[V] = {}, words[V / 4];
        if (inv > 0.0f) {
            bool unsure = false;
#pragma unroll
            for (int i = 0; i < V; ++i) c[i] = nearest<false>(to_f32(r.v[i]), scale, inv, unsure);
            if (unsure)  // one value in a hundred thousand
#pragma unroll
                for (int i = 0; i < V; ++i) c[i] = nearest<true>(to_f32(r.v[i]), scale, inv, unsure);
        }
#pragma unroll
        for (int i = 0; i < V / 4; ++i) words[i] = low_bytes(c[4 * i], c[4 * i + 1], c[4 * i + 2], c[4 * i + 3]);
        *reinterpret_cast<Vec<uint32_t, V / 4>*>(codes + u * V) = __builtin_bit_cast(Vec<uint32_t, V / 4>, words);
    };
    if constexpr (KEEP > 0) {
#pragma unroll
        for (int j = 0; j < KEEP; ++j)
            if (tid + j * THREADS < units) put(tid + j * THREADS, kept[j]);
    } else {
        for (uint32_t u = tid; u < units; u += THREADS) put(u, fetch(u));
    }
}

template <typename T, uint32_t THREADS>
auto* kernel_of(uint32_t each) {
    return each <= 1 ? k_quantize_rows<T, THREADS, 1> : each <= 2 ? k_quantize_rows<T, THREADS, 2> : each <= 4 ? k_quantize_rows<T, THREADS, 4> : each <= 8 ? k_quantize_rows<T, THREADS, 8> : k_quantize_rows<T, THREADS, 0>;
}

template <typename T>
int launch_typed(const QuantizeArgs& a, hipStream_t st) {
    const uint32_t units = (a.cols + 15) / 16 * sizeof(T);
    // few rows: as many threads as a row has units; many: two to four units each, a wave of its own for narrow ones (20000 rows of 1024 in
    // bfloat16: 13.5 us against 21.2 with 256 threads; of 4096: 41.7 with 256, 47.8 with a wave)
    const uint32_t threads = units <= (a.rows > 512 ? 256 : 64) ? 64 : units <= 512 || (units <= 2048 && a.rows > 512) ? 256 : 1024;
    const uint32_t each = (units + threads - 1) / threads;
    auto* k = threads == 64 ? kernel_of<T, 64>(each) : threads == 256 ? kernel_of<T, 256>(each) : kernel_of<T, 1024>(each);
    hipLaunchKernelGGL(k, dim3(a.rows), dim3(threads), 0, st, a);
    return hip_status(hipGetLastError(), "quantize_rows");
}

}  // namespace

int launch_quantize_rows(uint32_t type, const QuantizeArgs& a, hipStream_t st) {
    // a grid has fewer than 2^32 threads along x
    constexpr uint32_t kRows = 1u << 21;
    for (uint32_t r = 0; r < a.rows; r += kRows) {
        QuantizeArgs some = a;
        some.rows = std::min(a.rows - r, kRows);
        some.x = static_cast<const uint8_t*>(a.x) + (uint64_t)r * a.x_stride * (type == HALO_MI_F32 ? 4 : 2);
        some.codes += (uint64_t)r * a.codes_stride;
        some.scales += r;
        const int rc = type == HALO_MI_F16 ? launch_typed<_Float16>(some, st) : type == HALO_MI_BF16 ? launch_typed<__bf16>(some, st) : launch_typed<float>(some, st);
        if (rc) return rc;
    }
    return HALO_MI_OK;
}

}  // namespace halo_mi
