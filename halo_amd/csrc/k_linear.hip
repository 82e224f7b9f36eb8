// gfx950 kernels of linear attention with a decay for each head: S <- e^g S + k v^T, out = scale S^T q for a sequence's rows in order,
// S a k_dim x v_dim matrix of fp32 numbers per head that goes from call to call.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

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

template <typename T>
int launch_typed(const LinearArgs& a, hipStream_t st) {
    auto* k = a.k_dim == 64 ? k_linear_rows<T, 2> : a.k_dim == 96 ? k_linear_rows<T, 3> : a.k_dim == 128 ? k_linear_rows<T, 4> : a.k_dim == 192 ? k_linear_rows<T, 6> : k_linear_rows<T, 8>;
    hipLaunchKernelGGL(k, dim3(a.v_dim / kColumns, a.heads, a.n_seqs), dim3(kBlock), 0, st, a);
    return hip_status(hipGetLastError(), "linear_attention");
}

}  // namespace

uint64_t plan_linear(const LinearArgs&, uint64_t) { return 0; }

int launch_linear(uint32_t type, const LinearArgs& a, float*, uint64_t, hipStream_t st) {
    switch (type) {
        case HALO_MI_F16: return launch_typed<_Float16>(a, st);
        case HALO_MI_BF16: return launch_typed<__bf16>(a, st);
        default: return launch_typed<float>(a, st);
    }
}

}  // namespace halo_mi
