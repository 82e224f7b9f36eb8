// The angle of a rotary position on the device, as the kernels with rotations share it (k_rope.hip, k_norm_rope.hip).
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>

namespace halo_mi::dev {

// cos and sin of `angle` radians: the nearest quarter turn comes off in 64 bits.
__device__ __forceinline__ float2 turn(double angle) {
    const double quarters = angle * 0.63661977236758134308;  // 2 / pi
    const double n = rint(quarters);
    float s, c;
    sincospif((float)(quarters - n) * 0.5f, &s, &c);
    const int32_t q = (int32_t)(int64_t)n & 3;
    if (q & 1) {
        const float t = s;
        s = c;
        c = -t;
    }
    return (q & 2) ? float2{-c, -s} : float2{c, s};
}

}  // namespace halo_mi::dev
