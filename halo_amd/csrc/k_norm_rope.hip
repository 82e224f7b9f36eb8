// gfx950 kernels of the heads' norms with the rotary positions: for a head x of head_dim elements
//   y_j = x_j / sqrt(sum_j x_j^2 / head_dim + eps) * w_j,
// then the rotation of k_rope.hip on y. The head is read once: the lanes that hold it add their squares with
// cross-lane moves and turn what they have in their registers. A token's table of sines and cosines and both parts'
// weights are made once per workgroup, in LDS, while the first heads are on their way.
//
// Memory bounds it: 6133 tokens of 40 heads of 128 in bfloat16 take 27.6 us (4.5 TB/s read and written), of 256 with 64 turned 63.4 us (4.0). One
// token a workgroup took 33.2: 40 heads are two and a half rounds of its lanes, and every one waits for its table. A wave per token, with its table and
// weights in registers, took 34 to 48, a head loaded ahead 32 to 37: fewer waves fit. Sums by way of LDS took 28.2 and 80.7, adjacent
// pairs loaded 32 bytes a lane 31.3.
//
// Sums, products and the root are in 32 bits, one rounding to the type at the end: rounding the normed head to 16 bits before the
// rotation, as two launches do, is left out.
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

constexpr uint32_t kBlock = 256;
constexpr uint32_t kTokensHere = 4;  // of a workgroup, at most
constexpr uint32_t kTokens = 1u << 23;  // of a launch: a grid has fewer than 2^32 threads along x

// The turned pair, rounded as k_rope.hip rounds it: a part without weights is bitwise what rope gives.
__device__ __forceinline__ float first_of(float x, float y, float2 cs) { return fmaf(x, cs.x, -(y * cs.y)); }
__device__ __forceinline__ float second_of(float x, float y, float2 cs) { return fmaf(x, cs.y, y * cs.x); }

// The sum over G lanes, in all of them.
template <int G>
__device__ __forceinline__ float group_sum(float v) {
    v += lanes<0xB1>(v);   // the neighbour
    v += lanes<0x4E>(v);   // the other pair of 4
    v += lanes<0x141>(v);  // 8 lanes mirrored: the other 4
    if (G >= 16) v += lanes<0x140>(v);
    if (G >= 32) v = both16(v, v);
    if (G == 64) v = both32(v, v);
    return v;
}

// Both parts' rows, chosen lane by lane. They are kept in scalar registers by force: the compiler would choose the arguments' address instead, and
// load them in front of every head.
struct BothRows {
    uint64_t data[2], stride[2], head_stride[2];
    __device__ __forceinline__ BothRows(const HeadRows& a, const HeadRows& b, uint32_t heads, uint32_t size)
        : data{reinterpret_cast<uint64_t>(a.data), reinterpret_cast<uint64_t>(b.data) - heads * b.head_stride * size},
          stride{a.stride * size, b.stride * size},
          head_stride{a.head_stride * size, b.head_stride * size} {
#pragma unroll
        for (int i = 0; i < 2; ++i) asm volatile("" : "+s"(data[i]), "+s"(stride[i]), "+s"(head_stride[i]));
    }
    // head h of both parts' in a row, of token t
    template <typename T>
    __device__ __forceinline__ T* at(bool second, uint32_t t, uint32_t h) const {
        return reinterpret_cast<T*>((second ? data[1] : data[0]) + t * (second ? stride[1] : stride[0]) + h * (second ? head_stride[1] : head_stride[0]));
    }
};

// One workgroup: tokens blockIdx.x * tokens .. + tokens - 1, of each the heads from blockIdx.y * heads_per on, side by side. G lanes have a head between
// them, an item each: V pairs (2 V elements), or V elements that are not turned.
template <typename T, int V, bool INTERLEAVED, int G>
__global__ __launch_bounds__(kBlock) void k_norm_rope(NormRopeArgs n, uint32_t heads_per, uint32_t tokens) {
    const RopeArgs& a = n.rope;
    __shared__ alignas(16) float2 table[kTokensHere][V * G];
    __shared__ alignas(16) float weight[2][2 * V * G];
    const uint32_t t0 = blockIdx.x * tokens, here = min(tokens, a.n_tokens - t0), half = a.rot / 2, c = threadIdx.x % G, turned = half / V, items = turned + (a.dim - a.rot) / V;
    const uint32_t h0 = blockIdx.y * heads_per, h_count = min(a.heads - h0, heads_per);
    // the item's elements: V of the head from ex on, and for a turned one V from ey on: its pairs' others, or other pairs
    const bool turns = c < turned, has = c < items;
    const uint32_t ex = turns ? c * V : a.rot + (c - turned) * V, ey = ex + half;
    Vec<T, V> x{}, y{};
    const bool normed[2] = {n.norm_w[0] != nullptr, n.norm_w[1] != nullptr};
    const BothRows in_rows(a.part[0].in, a.part[1].in, a.part[0].heads, sizeof(T)), out_rows(a.part[0].out, a.part[1].out, a.part[0].heads, sizeof(T));
    // head h0 + h of token t0 + t
    const auto fetch = [&](uint32_t t, uint32_t h) {
        h += h0;
        const T* in = in_rows.template at<const T>(h >= a.part[0].heads, t0 + t, h);
        if (has) x = *reinterpret_cast<const Vec<T, V>*>(in + ex);
        if (turns) y = *reinterpret_cast<const Vec<T, V>*>(in + ey);
    };
    uint32_t t = threadIdx.x / G / h_count, h = threadIdx.x / G % h_count;
    const uint32_t t_step = kBlock / G / h_count, h_step = kBlock / G % h_count;
    if (t < here) fetch(t, h);
    for (uint32_t i = threadIdx.x; i < a.dim; i += kBlock)
        for (int p = 0; p < 2; ++p) weight[p][i] = n.norm_w[p] ? n.norm_w[p][i] : 1.0f;
    for (uint32_t i = threadIdx.x; i < half * here; i += kBlock) {
        const float2 cs = turn((double)a.positions[t0 + i / half] * a.freqs[i % half]);
        table[i / half][i % half] = {cs.x * a.factor, cs.y * a.factor};
    }
    __syncthreads();
    const float over_dim = 1.0f / (float)a.dim;
    while (t < here) {
        const uint32_t head = h0 + h;
        const bool second = head >= a.part[0].heads;
        float u[V], w[V], sum = 0.0f;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            u[i] = to_f32(x.v[i]);
            sum = fmaf(u[i], u[i], sum);
        }
#pragma unroll
        for (int i = 0; i < V; ++i) {
            w[i] = to_f32(y.v[i]);
            sum = fmaf(w[i], w[i], sum);
        }
        sum = group_sum<G>(sum);
        const float inv = (second ? normed[1] : normed[0]) ? 1.0f / sqrtf(fmaf(sum, over_dim, n.eps)) : 1.0f;
        T* out = out_rows.template at<T>(second, t0 + t, head);
        const float* wx = weight[second] + ex;
        if (turns) {
            const float* wy = weight[second] + ey;
            Vec<T, V> ox, oy;
#pragma unroll
            for (int i = 0; i < V; ++i) u[i] = u[i] * inv * wx[i], w[i] = w[i] * inv * wy[i];
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float2 cs = table[t][INTERLEAVED ? (i < V / 2 ? ex : ey) / 2 + i % (V / 2) : ex + i];
                if constexpr (INTERLEAVED) {
                    const float f = i < V / 2 ? u[2 * i] : w[2 * i - V], g = i < V / 2 ? u[2 * i + 1] : w[2 * i + 1 - V];
                    T* e = i < V / 2 ? &ox.v[2 * i] : &oy.v[2 * i - V];
                    e[0] = from_f32<T>(first_of(f, g, cs));
                    e[1] = from_f32<T>(second_of(f, g, cs));
                } else {
                    ox.v[i] = from_f32<T>(first_of(u[i], w[i], cs));
                    oy.v[i] = from_f32<T>(second_of(u[i], w[i], cs));
                }
            }
            *reinterpret_cast<Vec<T, V>*>(out + ex) = ox;
            *reinterpret_cast<Vec<T, V>*>(out + ey) = oy;
        } else if (has) {
            Vec<T, V> ox;
#pragma unroll
            for (int i = 0; i < V; ++i) ox.v[i] = from_f32<T>(u[i] * inv * wx[i]);
            *reinterpret_cast<Vec<T, V>*>(out + ex) = ox;
        }
        t += t_step, h += h_step;
        if (h >= h_count) h -= h_count, ++t;
        if (t < here) fetch(t, h);
    }
}

// Heads of any size and alignment: a wave has one, and reads it twice.
template <typename T, bool INTERLEAVED>
__global__ __launch_bounds__(kBlock) void k_norm_rope_any(NormRopeArgs n, uint32_t heads_per, uint32_t) {
    const RopeArgs& a = n.rope;
    __shared__ float2 table[256];
    const uint32_t t = blockIdx.x, half = a.rot / 2, lane = threadIdx.x % 64;
    const double pos = (double)a.positions[t];
    for (uint32_t i = threadIdx.x; i < half; i += kBlock) {
        const float2 cs = turn(pos * a.freqs[i]);
        table[i] = {cs.x * a.factor, cs.y * a.factor};
    }
    __syncthreads();
    const uint32_t h_end = min(a.heads, (blockIdx.y + 1) * heads_per);
    for (uint32_t h = blockIdx.y * heads_per + threadIdx.x / 64; h < h_end; h += kBlock / 64) {
        const bool second = h >= a.part[0].heads;
        const RopePart& p = a.part[second];
        const uint32_t head = second ? h - a.part[0].heads : h;
        const T* in = static_cast<const T*>(p.in.data) + t * p.in.stride + head * p.in.head_stride;
        T* out = const_cast<T*>(static_cast<const T*>(p.out.data)) + t * p.out.stride + head * p.out.head_stride;
        const float* norm = n.norm_w[second];
        float inv = 1.0f;
        if (norm) {
            float sum = 0.0f;
            for (uint32_t i = lane; i < a.dim; i += 64) {
                const float v = to_f32(in[i]);
                sum = fmaf(v, v, sum);
            }
#pragma unroll
            for (int i = 1; i < 64; i *= 2) sum += __shfl_xor(sum, i);
            inv = 1.0f / sqrtf(fmaf(sum, 1.0f / (float)a.dim, n.eps));
        }
        const auto normed = [&](uint32_t i) { return norm ? to_f32(in[i]) * inv * norm[i] : to_f32(in[i]); };
        for (uint32_t i = lane; i < half; i += 64) {
            const uint32_t ex = INTERLEAVED ? 2 * i : i, ey = INTERLEAVED ? 2 * i + 1 : i + half;
            const float u = normed(ex), w = normed(ey);
            const float2 cs = table[i];
            out[ex] = from_f32<T>(first_of(u, w, cs));
            out[ey] = from_f32<T>(second_of(u, w, cs));
        }
        for (uint32_t i = a.rot + lane; i < a.dim; i += 64) out[i] = from_f32<T>(normed(i));
    }
}

template <typename T, int V, int G>
auto* kernel_of(bool inter) {
    return inter ? k_norm_rope<T, V, true, G> : k_norm_rope<T, V, false, G>;
}

template <typename T>
int launch_typed(uint32_t pairs, const NormRopeArgs& n, hipStream_t st) {
    const RopeArgs& a = n.rope;
    const bool inter = pairs == HALO_MI_ROPE_INTERLEAVED;
    // the widest accesses that divide a head's parts and on which every row and head begins
    const auto fits = [&](uint32_t v) {
        bool ok = a.rot / 2 % v == 0 && a.dim % v == 0;
        for (const RopePart& p : a.part)
            if (p.heads)
                for (const HeadRows* r : {&p.in, &p.out})
                    ok = ok && reinterpret_cast<uintptr_t>(r->data) % (v * sizeof(T)) == 0 && r->stride % v == 0 && r->head_stride % v == 0;
        return ok && a.rot / 2 / v + (a.dim - a.rot) / v <= 64;
    };
    uint32_t v = 16 / sizeof(T);
    while (v > 1 && !fits(v)) v /= 2;
    void (*k)(NormRopeArgs, uint32_t, uint32_t) = inter ? k_norm_rope_any<T, true> : k_norm_rope_any<T, false>;
    uint32_t at_once = kBlock / 64;
    if (v > 1) {
        const uint32_t items = a.rot / 2 / v + (a.dim - a.rot) / v, g = items <= 8 ? 8 : items <= 16 ? 16 : items <= 32 ? 32 : 64;
        at_once = kBlock / g;
        const auto pick = [&](auto wide) {
            constexpr int V = decltype(wide)::value;
            return g == 8 ? kernel_of<T, V, 8>(inter) : g == 16 ? kernel_of<T, V, 16>(inter) : g == 32 ? kernel_of<T, V, 32>(inter) : kernel_of<T, V, 64>(inter);
        };
        if constexpr (sizeof(T) == 2) k = v == 8 ? pick(std::integral_constant<int, 8>{}) : v == 4 ? pick(std::integral_constant<int, 4>{}) : pick(std::integral_constant<int, 2>{});
        else k = v == 4 ? pick(std::integral_constant<int, 4>{}) : pick(std::integral_constant<int, 2>{});
    }
    // many tokens: several a workgroup; few: their heads over several workgroups
    const uint32_t tokens = v > 1 ? std::min(std::max(a.n_tokens / 1024, 1u), kTokensHere) : 1;
    const uint32_t passes = std::max<uint64_t>(1, std::min<uint64_t>(a.heads, (uint64_t)a.n_tokens * ((a.heads + at_once - 1) / at_once) / 2048));
    // at most 2^15 workgroups along y
    const uint32_t heads_per = std::min(a.heads, std::max(passes * at_once, a.heads / 32768 + 1));
    for (uint32_t t = 0; t < a.n_tokens; t += kTokens) {
        NormRopeArgs some = n;
        some.rope.n_tokens = std::min(a.n_tokens - t, kTokens);
        some.rope.positions += t;
        for (RopePart& p : some.rope.part)
            for (HeadRows* r : {&p.in, &p.out}) r->data = static_cast<const T*>(r->data) + t * r->stride;
        hipLaunchKernelGGL(k, dim3((some.rope.n_tokens + tokens - 1) / tokens, (a.heads + heads_per - 1) / heads_per), dim3(kBlock), 0, st, some, heads_per, tokens);
    }
    return hip_status(hipGetLastError(), "norm_rope");
}

}  // namespace

int launch_norm_rope(uint32_t type, uint32_t pairs, const NormRopeArgs& a, hipStream_t st) {
    switch (type) {
        case HALO_MI_F16: return launch_typed<_Float16>(pairs, a, st);
        case HALO_MI_BF16: return launch_typed<__bf16>(pairs, a, st);
        default: return launch_typed<float>(pairs, a, st);
    }
}

}  // namespace halo_mi
