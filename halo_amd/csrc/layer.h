// 8-bit integer products and linear attention between their C ABI (layer_api.cpp) and their kernels (k_quantize.hip, k_gemm_i8.hip,
// k_linear.hip): argument blocks and launchers.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

#include "kv.h"

namespace halo_mi {

struct QuantizeArgs {
    const void* x;
    uint64_t x_stride;  // elements
    int8_t* codes;
    uint64_t codes_stride;
    float* scales;
    uint32_t rows, cols;
};

struct GemmI8Args {
    const int8_t* w;
    const int8_t* x;
    const float* w_scales;
    const float* x_scales;
    void* y;
    uint64_t y_stride;            // elements
    uint32_t w_stride, x_stride;  // bytes, multiples of 16
    uint32_t rows, cols, n_vec;
};

struct LinearArgs {
    HeadRows q, k, v, out;
    const float* decay;
    uint64_t decay_stride;  // elements between rows; 0: one value per head
    const float* state;
    float* state_out;
    const int32_t* slots;
    const int32_t* row_starts;
    const int32_t* seq_lens;  // or null
    uint32_t n_slots, n_seqs, n_rows, max_rows;
    uint32_t heads, group;  // group: heads per head of q and k
    uint32_t k_dim, v_dim;
    float scale;
    uint32_t* status;
};

int launch_quantize_rows(uint32_t type, const QuantizeArgs& a, hipStream_t st);
int launch_gemm_i8(uint32_t type, const GemmI8Args& a, hipStream_t st);
// The bytes of workspace that the call makes use of when it has part_bytes of them.
uint64_t plan_linear(const LinearArgs& a, uint64_t part_bytes);
int launch_linear(uint32_t type, const LinearArgs& a, float* part, uint64_t part_bytes, hipStream_t st);

}  // namespace halo_mi
