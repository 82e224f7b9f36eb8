// gfx950 kernel of the rotary positions (PARTIAL_ROPE, RopeArgs at include/halo/backend/backend.h:369-377 of
// the reference): for a = positions[t] * freqs[i],
//   (x, y) -> factor * (x cos a - y sin a, y cos a + x sin a)
// of the pairs (i, i + rot / 2) or (2 i, 2 i + 1); elements from rot on are copied.
//
// The angle a is taken in 64 bits and reduced there to a quarter turn (a rotation by a position of 2^20 would
// otherwise lose 4 decimal digits), its sine and cosine in 32. They are the same for every head, so a
// workgroup makes a token's table once, in LDS, and streams the token's heads with 16-byte accesses.
//
// Bound by memory: 6133 tokens of 40 bf16 heads of 128, 126 MB, in 27.4 us (4.6 TB/s, a large copy's rate); one token is
// one launch (3.4 us).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kv.h"
#include "kv_device.h"
#include "launch.h"
#include "rope_device.h"

namespace halo_mi {
namespace {

using namespace dev;

constexpr uint32_t kRopeBlock = 256;
constexpr uint32_t kRopeTokens = 1u << 23;  // of a launch: a grid has fewer than 2^32 threads along x
constexpr uint32_t kRopePairs = HALO_MI_ROPE_INTERLEAVED;

// One workgroup: token blockIdx.x, the heads from blockIdx.y * heads_per on. V elements per access.
template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(kRopeBlock) void k_rope(RopeArgs a, uint32_t heads_per) {
    __shared__ float2 table[256];
    const uint32_t t = blockIdx.x, half = a.rot / 2;
    const double pos = (double)a.positions[t];
    for (uint32_t i = threadIdx.x; i < half; i += kRopeBlock) {
        const float2 cs = turn(pos * a.freqs[i]);
        table[i] = {cs.x * a.factor, cs.y * a.factor};
    }
    __syncthreads();
    // items of a head: its rotated pairs, V at a time (half layout: V firsts and V seconds; adjacent pairs: 2 V
    // elements), then the copied elements
    const uint32_t turned = half / V, items = turned + (a.dim - a.rot) / V;
    const uint32_t per = max(1u, kRopeBlock / items), sub = threadIdx.x / items;
    if (items <= kRopeBlock && sub >= per) return;
    const uint32_t h_end = min(a.heads, (blockIdx.y + 1) * heads_per);
    for (uint32_t h = blockIdx.y * heads_per + (items <= kRopeBlock ? sub : 0); h < h_end; h += per) {
        const bool second = h >= a.part[0].heads;
        const RopePart& p = a.part[second];
        const uint32_t head = second ? h - a.part[0].heads : h;
        const T* in = static_cast<const T*>(p.in.data) + t * p.in.stride + head * p.in.head_stride;
        T* out = const_cast<T*>(static_cast<const T*>(p.out.data)) + t * p.out.stride + head * p.out.head_stride;
        for (uint32_t c = items <= kRopeBlock ? threadIdx.x % items : threadIdx.x; c < items; c += items <= kRopeBlock ? items : kRopeBlock) {
            if (c >= turned) {
                if (p.in_place) continue;
                const uint32_t e = a.rot + (c - turned) * V;
                *reinterpret_cast<Vec<T, V>*>(out + e) = *reinterpret_cast<const Vec<T, V>*>(in + e);
                continue;
            }
            // INTERLEAVED: x holds the first V of the item's 2 V elements, y the others
            const uint32_t ex = c * V * (INTERLEAVED ? 2 : 1), ey = INTERLEAVED ? ex + V : ex + half;
            Vec<T, V> x = *reinterpret_cast<const Vec<T, V>*>(in + ex), y = *reinterpret_cast<const Vec<T, V>*>(in + ey);
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 cs = table[c * V + i];
                if constexpr (INTERLEAVED && V > 1) {
                    T* e = i < V / 2 ? &x.v[2 * i] : &y.v[2 * i - V];
                    const float u = to_f32(e[0]), w = to_f32(e[1]);
                    e[0] = from_f32<T>(u * cs.x - w * cs.y);
                    e[1] = from_f32<T>(w * cs.x + u * cs.y);
                } else {
                    const float u = to_f32(x.v[i]), w = to_f32(y.v[i]);
                    x.v[i] = from_f32<T>(u * cs.x - w * cs.y);
                    y.v[i] = from_f32<T>(w * cs.x + u * cs.y);
                }
            }
            *reinterpret_cast<Vec<T, V>*>(out + ex) = x;
            *reinterpret_cast<Vec<T, V>*>(out + ey) = y;
        }
    }
}

template <typename T>
int launch_typed(uint32_t pairs, const RopeArgs& a, hipStream_t st) {
    constexpr int V = 16 / sizeof(T);
    // whole 16-byte accesses where every row and every part of a head begins on 16 bytes
    bool wide = a.rot / 2 % V == 0 && a.dim % V == 0;
    for (const RopePart& p : a.part)
        if (p.heads)
            for (const HeadRows* r : {&p.in, &p.out})
                wide = wide && reinterpret_cast<uintptr_t>(r->data) % 16 == 0 && r->stride % V == 0 && r->head_stride % V == 0;
    const uint32_t vec = wide ? V : 1, items = (a.rot / 2 + a.dim - a.rot) / vec;
    const uint32_t at_once = std::max(1u, kRopeBlock / items);
    // few tokens: their heads over several workgroups, one pass each
    const uint32_t passes = std::max<uint64_t>(1, std::min<uint64_t>(a.heads, (uint64_t)a.n_tokens * ((a.heads + at_once - 1) / at_once) / 2048));
    // at most 2^15 workgroups along y
    const uint32_t heads_per = std::min(a.heads, std::max(passes * at_once, a.heads / 32768 + 1));
    const bool inter = pairs == kRopePairs;
    auto* k = wide ? (inter ? k_rope<T, V, true> : k_rope<T, V, false>) : (inter ? k_rope<T, 1, true> : k_rope<T, 1, false>);
    for (uint32_t t = 0; t < a.n_tokens; t += kRopeTokens) {
        RopeArgs some = a;
        some.n_tokens = std::min(a.n_tokens - t, kRopeTokens);
        some.positions += t;
        for (RopePart& p : some.part)
            for (HeadRows* r : {&p.in, &p.out}) r->data = static_cast<const T*>(r->data) + t * r->stride;
        hipLaunchKernelGGL(k, dim3(some.n_tokens, (a.heads + heads_per - 1) / heads_per), dim3(kRopeBlock), 0, st, some, heads_per);
    }
    return hip_status(hipGetLastError(), "PARTIAL_ROPE");
}

}  // namespace

int launch_rope(uint32_t type, uint32_t pairs, const RopeArgs& a, hipStream_t st) {
    switch (type) {
        case HALO_MI_F16: return launch_typed<_Float16>(pairs, a, st);
        case HALO_MI_BF16: return launch_typed<__bf16>(pairs, a, st);
        default: return launch_typed<float>(pairs, a, st);
    }
}

}  // namespace halo_mi
