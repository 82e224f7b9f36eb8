// gfx950 kernels of the product of 8-bit integers with a scale for each token and each output channel,
//   y[t][n] = sx[t] sw[n] sum_i x[t][i] w[n][i],
// on the integer matrix cores: the sums are exact in 32 bits, whatever their order, so how K is split is free.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kv_device.h"
#include "launch.h"
#include "layer.h"

namespace halo_mi {
namespace {

using namespace dev;

typedef int32_t int4v __attribute__((ext_vector_type(4)));

constexpr uint32_t kFewWaves = 8;

template <typename T>
__device__ __forceinline__ T scaled(int32_t sum, float xs, float ws) {
    return from_f32<T>(xs * ws * (float)sum);
}

// Few vectors. One workgroup: 16 AT channels and up to 16 NT vectors, K over its waves in pieces of 256 codes; the waves' sums meet in
// LDS. On v_mfma_i32_16x16x64_i8 a lane has 16 codes of row lane % 16; the products come as channel 4 (lane / 16) + i, vector lane % 16.
template <typename T, int AT, int NT>
__global__ __launch_bounds__(kFewWaves * 64) void k_gemm_i8_few(GemmI8Args a) {
    __shared__ int32_t sums[kFewWaves][AT * NT * 4][64];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t n0 = blockIdx.x * (16 * AT), t0 = blockIdx.y * (16 * NT), at_k = lane / 16 * 16;
    const int8_t *w[AT], *x[NT];
#pragma unroll
    for (int i = 0; i < AT; ++i) w[i] = a.w + (uint64_t)min(n0 + i * 16 + lane % 16, a.rows - 1) * a.w_stride;
#pragma unroll
    for (int i = 0; i < NT; ++i) x[i] = a.x + (uint64_t)min(t0 + i * 16 + lane % 16, a.n_vec - 1) * a.x_stride;
    int4v acc[AT][NT] = {};
    const uint32_t cols = (a.cols + 15) / 16 * 16, whole = cols / 256;
    for (uint32_t c = wave; c < whole; c += kFewWaves) {
        int4v wf[4][AT], xf[4][NT];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const uint32_t k = c * 256 + u * 64 + at_k;
#pragma unroll
            for (int i = 0; i < AT; ++i) wf[u][i] = *reinterpret_cast<const int4v*>(w[i] + k);
#pragma unroll
            for (int i = 0; i < NT; ++i) xf[u][i] = *reinterpret_cast<const int4v*>(x[i] + k);
        }
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int i = 0; i < AT; ++i)
#pragma unroll
                for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u][i], xf[u][j], acc[i][j], 0, 0, 0);
    }
    // what is left: up to 4 steps of 64 codes, one a wave
    if (const uint32_t k0 = whole * 256 + wave * 64; wave < 4 && k0 < cols) {
        const uint32_t k = k0 + at_k;
        const bool in = k < cols;
        int4v wf[AT], xf[NT];
#pragma unroll
        for (int i = 0; i < AT; ++i) wf[i] = in ? *reinterpret_cast<const int4v*>(w[i] + k) : int4v{};
#pragma unroll
        for (int i = 0; i < NT; ++i) xf[i] = in ? *reinterpret_cast<const int4v*>(x[i] + k) : int4v{};
#pragma unroll
        for (int i = 0; i < AT; ++i)
#pragma unroll
            for (int j = 0; j < NT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[i], xf[j], acc[i][j], 0, 0, 0);
    }
#pragma unroll
    for (int i = 0; i < AT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[wave][(i * NT + j) * 4 + r][lane] = acc[i][j][r];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < AT * NT * 256; e += kFewWaves * 64) {
        // channels vary fastest
        const uint32_t ch = e % (16 * AT), v = e / (16 * AT), n = n0 + ch, t = t0 + v;
        if (n >= a.rows || t >= a.n_vec) continue;
        const uint32_t reg = (ch / 16 * NT + v / 16) * 4 + ch % 4, from = ch % 16 / 4 * 16 + v % 16;
        int32_t sum = 0;
#pragma unroll
        for (uint32_t s = 0; s < kFewWaves; ++s) sum += sums[s][reg][from];
        static_cast<T*>(a.y)[t * a.y_stride + n] = scaled<T>(sum, a.x_scales[t], a.w_scales[n]);
    }
}

template <typename T>
int launch_typed(const GemmI8Args& a, hipStream_t st) {
    const uint32_t nt = a.n_vec <= 16 ? 1 : a.n_vec <= 32 ? 2 : 4;
    auto* k = nt == 1 ? k_gemm_i8_few<T, 1, 1> : nt == 2 ? k_gemm_i8_few<T, 1, 2> : k_gemm_i8_few<T, 1, 4>;
    const uint32_t at_once = 65535 * 16 * nt;
    for (uint32_t t = 0; t < a.n_vec; t += at_once) {
        GemmI8Args some = a;
        some.n_vec = std::min(a.n_vec - t, at_once);
        some.x += (uint64_t)t * a.x_stride;
        some.x_scales += t;
        some.y = static_cast<T*>(a.y) + t * a.y_stride;
        hipLaunchKernelGGL(k, dim3((a.rows + 15) / 16, (some.n_vec + 16 * nt - 1) / (16 * nt)), dim3(kFewWaves * 64), 0, st, some);
        if (const int rc = hip_status(hipGetLastError(), "gemm_i8")) return rc;
    }
    return HALO_MI_OK;
}

}  // namespace

int launch_gemm_i8(uint32_t type, const GemmI8Args& a, hipStream_t st) {
    switch (type) {
        case HALO_MI_F16: return launch_typed<_Float16>(a, st);
        case HALO_MI_BF16: return launch_typed<__bf16>(a, st);
        default: return launch_typed<float>(a, st);
    }
}

}  // namespace halo_mi
