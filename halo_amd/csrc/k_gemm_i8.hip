// gfx950 kernels of the product of 8-bit integers with a scale for each token and each output channel,
//   y[t][n] = sx[t] sw[n] sum_i x[t][i] w[n][i],
// on the integer matrix cores: the sums are exact in 32 bits, whatever their order, so how K is split is free.
//
// Few vectors read w once, and its stream bounds them: 17408 channels of 5120 codes for one vector take 16.4 us (89 MB, 5.4 TB/s). Many are bound by
// the products: 3990 vectors take 355 to 375 us (1.9 to 2.0 POP/s; a large library product of these sizes reaches 2.0), 44 % of the matrix cores'
// cycles at the 2.1 GHz that the card then keeps; 4096 vectors of 8192 codes by 8192 channels 2.3 POP/s. In between, 61 vectors by 6144
// channels take 12.7 us and 509 by 17408 62 (1.5 POP/s; 218 tiles on 256 CUs, whose loads take as long as their products).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <iterator>
#include <utility>

#include "kv_device.h"
#include "launch.h"
#include "layer.h"

namespace halo_mi {
namespace {

using namespace dev;

typedef int32_t int4v __attribute__((ext_vector_type(4)));

// The product of the scales, then with the sum, then to the type: the compiler may not take two of these roundings together, so that every
// kernel gives the same bits.
template <typename T>
__device__ __forceinline__ T scaled(int32_t sum, float xs, float ws) {
    float v = xs * ws * (float)sum;
    __asm__("" : "+v"(v));
    return from_f32<T>(v);
}

// Few vectors. One workgroup: 16 channels and up to 16 NT vectors, K over its waves in pieces of 64 U codes; the waves' sums meet in
// LDS. On v_mfma_i32_16x16x64_i8 a lane has 16 codes of row lane % 16; the products come as channel 4 (lane / 16) + i, vector lane % 16.
template <typename T, int AT, int NT, int WAVES, int U>
__global__ __launch_bounds__(WAVES * 64) void k_gemm_i8_few(GemmI8Args a, uint32_t each) {
    __shared__ int32_t sums[WAVES][AT * NT * 4][64];
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    const uint32_t n0 = blockIdx.x * each, n1 = min(n0 + each, a.rows), at_k = lane / 16 * 16;
    const int8_t *w[AT], *x[NT];
#pragma unroll
    for (int i = 0; i < AT; ++i) w[i] = a.w + (uint64_t)min(n0 + i * 16 + lane % 16, n1 - 1) * a.w_stride + at_k;
#pragma unroll
    for (int i = 0; i < NT; ++i) x[i] = a.x + (uint64_t)min(i * 16 + lane % 16, a.n_vec - 1) * a.x_stride + at_k;
    int4v acc[AT][NT] = {};
    const uint32_t cols = (a.cols + 15) / 16 * 16, whole = cols / (64 * U);
    struct Piece {
        int4v w[AT][U], x[NT][U];
    };
    const auto fetch = [&](Piece& p, uint32_t c) {
#pragma unroll
        for (int i = 0; i < AT; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) p.w[i][u] = *reinterpret_cast<const int4v*>(w[i] + c * (64 * U) + u * 64);
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int u = 0; u < U; ++u) p.x[i][u] = *reinterpret_cast<const int4v*>(x[i] + c * (64 * U) + u * 64);
    };
    const auto multiply = [&](const Piece& p) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int j = 0; j < AT; ++j)
#pragma unroll
                for (int i = 0; i < NT; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(p.w[j][u], p.x[i][u], acc[j][i], 0, 0, 0);
    };
    // a piece ahead
    Piece p, q;
    uint32_t c = wave;
    if (c < whole) fetch(p, c);
    while (c < whole) {
        if (c + WAVES < whole) fetch(q, c + WAVES);
        multiply(p);
        c += WAVES;
        if (c >= whole) break;
        if (c + WAVES < whole) fetch(p, c + WAVES);
        multiply(q);
        c += WAVES;
    }
    // what is left: up to U steps of 64 codes, one a wave
    if (const uint32_t k0 = whole * (64 * U) + wave * 64; wave < U && k0 < cols) {
        const bool in = k0 + at_k < cols;
        int4v wf[AT];
#pragma unroll
        for (int j = 0; j < AT; ++j) wf[j] = in ? *reinterpret_cast<const int4v*>(w[j] + k0) : int4v{};
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int4v xf = in ? *reinterpret_cast<const int4v*>(x[i] + k0) : int4v{};
#pragma unroll
            for (int j = 0; j < AT; ++j) acc[j][i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf, acc[j][i], 0, 0, 0);
        }
    }
#pragma unroll
    for (int j = 0; j < AT; ++j)
#pragma unroll
        for (int i = 0; i < NT; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) sums[wave][(j * NT + i) * 4 + r][lane] = acc[j][i][r];
    __syncthreads();
    for (uint32_t e = threadIdx.x; e < AT * NT * 256; e += WAVES * 64) {
        // channels vary fastest
        const uint32_t ch = e % (16 * AT), v = e / (16 * AT), n = n0 + ch;
        if (n >= n1 || v >= a.n_vec) continue;
        const uint32_t reg = (ch / 16 * NT + v / 16) * 4 + ch % 4, from = ch % 16 / 4 * 16 + v % 16;
        int32_t sum = 0;
#pragma unroll
        for (uint32_t s = 0; s < WAVES; ++s) sum += sums[s][reg][from];
        static_cast<T*>(a.y)[v * a.y_stride + n] = scaled<T>(sum, a.x_scales[v], a.w_scales[n]);
    }
}

// ---- many vectors --------------------------------------------------------------------------------------------------------

constexpr uint32_t kTileK = 128;         // codes of a row in a step
constexpr uint32_t kNone = 0x80000000u;  // an offset past every buffer: what is loaded there is 0

typedef __attribute__((address_space(3))) uint8_t lds_u8;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t rows_of(const int8_t* base, uint64_t bytes) {
    return __builtin_amdgcn_make_buffer_rsrc(const_cast<int8_t*>(base), 0, (uint32_t)bytes, 0x00020000);
}

// What this wave has read from LDS is in its registers, and of its loads all but the last N have arrived; then the workgroup meets.
template <int N>
__device__ __forceinline__ void meet() {
    __asm__ __volatile__("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The place of tile p: workgroups go to the eight XCDs in turn, so that each XCD takes a stretch of the tiles; in a stretch, bands of four
// tiles of vectors keep what the XCD reads at one time small.
__device__ __forceinline__ void place_of(uint32_t p, uint32_t tiles_n, uint32_t tiles_t, uint32_t& tn, uint32_t& tt) {
    const uint32_t all = tiles_n * tiles_t, each = all / 8, more = all % 8, xcd = p % 8;
    p = xcd * each + min(xcd, more) + p / 8;
    const uint32_t band = p / (4 * tiles_n), in_band = p - band * 4 * tiles_n, high = min(tiles_t - band * 4, 4u);
    tn = in_band / high;
    tt = band * 4 + in_band % high;
}

// One workgroup of 8 waves, 2 along the channels and 4 along the vectors; a wave has FN x FT products of 16 x 16. Steps of 128 codes go from
// memory to LDS with no register between, one step ahead, in two buffers; a wave reads the fragments of a half step while it multiplies the
// half before.
//
// Rows of a tile lie in LDS 128 bytes apart, their 16-byte pieces swapped by the row, so that eight lanes that read one piece of the rows of a
// fragment read eight different sixteenths of the banks. x's fragments are rows side by side; w's row m is channel 4 FN (m / 4) + 4 i + m % 4 of the
// wave's, so that a lane's products are channels side by side.
template <typename T, int FN, int FT, int S>
__global__ __launch_bounds__(512, 2) void k_gemm_i8_tiles(GemmI8Args a, uint32_t tiles_n, uint32_t tiles_t, uint32_t each_n, uint32_t each_t) {
    constexpr uint32_t TN = 32 * FN, TT = 64 * FT;
    constexpr uint32_t kW = (TN + 63) / 64 * 64;       // rows of w's part of a buffer: whole loads of the workgroup
    constexpr int LOADS = (kW + TT) / 64;              // of a wave and step: 8 rows, 1 KiB each
    constexpr uint32_t kStage = (kW + TT) * kTileK;
    extern __shared__ uint8_t lds[];
    const uint32_t tid = threadIdx.x, lane = tid % 64, wave = __builtin_amdgcn_readfirstlane(tid / 64);
    uint32_t tn, tt;
    place_of(blockIdx.x, tiles_n, tiles_t, tn, tt);
    const uint32_t n0 = tn * each_n, t0 = tt * each_t, cols = (a.cols + 15) / 16 * 16;
    const uint32_t nrows = min(a.rows - n0, each_n), trows = min(a.n_vec - t0, each_t);
    const int8_t *w = a.w + (uint64_t)n0 * a.w_stride, *x = a.x + (uint64_t)t0 * a.x_stride;
    const __amdgpu_buffer_rsrc_t wbuf = rows_of(w, (uint64_t)(nrows - 1) * a.w_stride + cols), xbuf = rows_of(x, (uint64_t)(trows - 1) * a.x_stride + cols);
    const auto swap_w = [](uint32_t row) { return (row & 3) | (row / (4 * FN) & 1) << 2; };
    const auto swap_x = [](uint32_t row) { return row & 7; };
    // this lane's part of the wave's loads: rows 8 (wave + 8 j) + lane / 8 of w's and then x's, piece lane % 8 as swapped; rows past the
    // tile's are zeros
    uint32_t from[LOADS], piece[LOADS];
#pragma unroll
    for (int j = 0; j < LOADS; ++j) {
        const bool is_w = 64 * j < kW;
        const uint32_t r = (wave + 8 * j) * 8 + lane / 8 - (is_w ? 0 : kW);
        piece[j] = (lane % 8 ^ (is_w ? swap_w(r) : swap_x(r))) * 16;
        from[j] = r * (is_w ? a.w_stride : a.x_stride) + piece[j];
        if (r >= (is_w ? nrows : trows)) piece[j] = kNone;
    }
    const auto fetch = [&](uint32_t step) {
        const uint32_t k = step * kTileK;
        uint8_t* stage = lds + step % S * kStage;
#pragma unroll
        for (int j = 0; j < LOADS; ++j) {
            const uint32_t at = k + piece[j] < cols ? from[j] + k : kNone;
            lds_u8* to = (lds_u8*)(stage + (wave + 8 * j) * 1024);
            __builtin_amdgcn_raw_ptr_buffer_load_lds(64 * j < kW ? wbuf : xbuf, to, 16, at, 0, 0, 0);
        }
    };
    const uint32_t wn = wave % 2 * (TN / 2), wt = wave / 2 * (TT / 4), m = lane % 16, g = lane / 16;
    const auto x_row = [&](int j) { return wt + 16 * j + m; };
    const uint32_t w_row0 = wn + m / 4 * (4 * FN) + m % 4;
    // the fragments' places in a buffer: both halves' pieces differ in one bit
    const uint32_t w_at = w_row0 * kTileK + (g ^ swap_w(w_row0)) * 16, x_at = kW * kTileK + x_row(0) * kTileK + (g ^ swap_x(m)) * 16;
    struct Half {
        int4v w[FN], x[FT];
    };
    const auto read = [&](Half& f, uint32_t step, uint32_t h) {
        const uint8_t* b = lds + step % S * kStage;
#pragma unroll
        for (int i = 0; i < FN; ++i) f.w[i] = *reinterpret_cast<const int4v*>(b + (w_at ^ h * 64) + i * 4 * kTileK);
#pragma unroll
        for (int j = 0; j < FT; ++j) f.x[j] = *reinterpret_cast<const int4v*>(b + (x_at ^ h * 64) + j * 16 * kTileK);
    };
    int4v acc[FN][FT] = {};
    const auto multiply = [&](const Half& f) {
#pragma unroll
        for (int i = 0; i < FN; ++i)
#pragma unroll
            for (int j = 0; j < FT; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(f.w[i], f.x[j], acc[i][j], 0, 0, 0);
    };
    const uint32_t steps = (cols + kTileK - 1) / kTileK;
    // reads and loads spread between the products
    const auto interleave = [&](bool loads) {
        constexpr int all = FN * FT, reads = FN + FT, per = all / reads ? all / reads : 1;
        if (loads) __builtin_amdgcn_sched_group_barrier(0x020, LOADS, 0);  // loads
#pragma unroll
        for (int i = 0; i < reads; ++i) {
            __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                          // a read of LDS
            __builtin_amdgcn_sched_group_barrier(0x008, per, 0);                        // products
        }
        __builtin_amdgcn_sched_group_barrier(0x008, all, 0);
        __builtin_amdgcn_sched_barrier(0);
    };
#pragma unroll
    for (int i = 0; i + 1 < S; ++i) fetch(i);
    meet<(S - 2) * LOADS>();
    fetch(S - 1);
    // what is loaded and read past the last step is zeros, or is not used
    Half f0, f1;
    read(f0, 0, 0);
    for (uint32_t step = 0; step < steps; ++step) {
        read(f1, step, 1);
        multiply(f0);
        interleave(false);
        meet<(S - 2) * LOADS>();
        fetch(step + S);
        read(f0, step + 1, 0);
        multiply(f1);
        interleave(true);
    }
    __syncthreads();  // no load is under way when the workgroup ends
    // a lane has channels c0 .. c0 + 4 FN of vectors x_row(j)
    constexpr int C = FN * 4, V = C % (16 / sizeof(T)) == 0 ? 16 / sizeof(T) : 4;
    const uint32_t c0 = n0 + wn + g * C, n1 = n0 + nrows;
    float ws[C];
#pragma unroll
    for (int i = 0; i < C; ++i) ws[i] = a.w_scales[min(c0 + i, n1 - 1)];
    const bool wide = c0 + C <= n1 && reinterpret_cast<uintptr_t>(a.y) % (V * sizeof(T)) == 0 && a.y_stride % V == 0 && c0 % V == 0;
#pragma unroll
    for (int j = 0; j < FT; ++j) {
        const uint32_t t = t0 + x_row(j);
        if (x_row(j) >= trows) continue;
        const float xs = a.x_scales[t];
        T* y = static_cast<T*>(a.y) + t * a.y_stride + c0;
        if (wide) {
#pragma unroll
            for (int i = 0; i < C; i += V) {
                Vec<T, V> out;
#pragma unroll
                for (int e = 0; e < V; ++e) out.v[e] = scaled<T>(acc[(i + e) / 4][j][(i + e) % 4], xs, ws[i + e]);
                *reinterpret_cast<Vec<T, V>*>(y + i) = out;
            }
        } else {
#pragma unroll
            for (int i = 0; i < C; ++i)
                if (c0 + i < n1) y[i] = scaled<T>(acc[i / 4][j][i % 4], xs, ws[i]);
        }
    }
}

// The kernels for many vectors by their fragments, stages and the workgroups of each that a CU's LDS takes.
struct TileShape {
    uint32_t fn, ft, stages;
};
constexpr TileShape kShapes[] = {{8, 4, 2}, {7, 4, 2}, {6, 4, 2}, {5, 4, 2}, {8, 3, 2}, {7, 3, 2}, {6, 3, 2}, {4, 3, 2}, {4, 2, 3}, {3, 2, 4}, {2, 2, 4}, {4, 1, 4}, {3, 1, 4}, {2, 1, 4}, {1, 1, 4}};
constexpr uint32_t kCus = 256;

uint32_t stage_bytes(const TileShape& s) { return ((32 * s.fn + 63) / 64 * 64 + 64 * s.ft) * kTileK; }

struct TilePlan {
    TileShape shape;
    uint32_t tiles_n, tiles_t, each_n, each_t;
};

// The shape whose rounds of tiles take the least time, in us, by what steps of 128 codes measured: products 0.056 for each 16 x 16 of a
// wave, or the way to them, 0.015 a KiB loaded and 0.04 a fragment read. Where the loads bound a shape, the channels are dealt out evenly over all
// the tiles that its rounds have room for (61 vectors, 17408 channels of 5120: 242 tiles of 72 channels 19.3 us, 182 of 96 23.7).
TilePlan plan_tiles(uint32_t rows, uint32_t cols, uint32_t n_vec) {
    const double steps = (cols + kTileK - 1) / kTileK;
    TilePlan best{};
    double least = 1e300;
    for (const TileShape& s : kShapes) {
        TilePlan p{s};
        p.tiles_t = (n_vec + 64 * s.ft - 1) / (64 * s.ft);
        p.each_t = (n_vec + p.tiles_t - 1) / p.tiles_t;
        p.tiles_t = (n_vec + p.each_t - 1) / p.each_t;
        const uint64_t few = (rows + 32ull * s.fn - 1) / (32 * s.fn), tiles = few * p.tiles_t;
        const uint64_t fit = std::max(1u, 160 * 1024 / (s.stages * stage_bytes(s))), beside = std::min(fit, (tiles + kCus - 1) / kCus);
        const uint64_t slots = kCus * beside, rounds = (tiles + slots - 1) / slots;
        const double products = 0.056 * s.fn * s.ft;
        const auto share = [&](uint64_t n) { return (uint32_t)(((rows + n - 1) / n + 7) / 8 * 8); };
        const auto loads = [&] { return 0.015 / 8 * (p.each_n + p.each_t) + 0.04 * (s.fn + s.ft) - 0.05; };
        p.each_n = share(few);
        if (loads() > products) p.each_n = share(std::max<uint64_t>(few, std::min<uint64_t>(slots * rounds / p.tiles_t, (rows + 7) / 8)));
        p.tiles_n = (rows + p.each_n - 1) / p.each_n;
        const double time = (double)rounds * (2.0 + steps * (double)beside * std::max(products, loads()));
        if (time < least) least = time, best = p;
    }
    return best;
}

template <typename T>
auto* kernel_of(const TileShape& s) {
    void (*k)(GemmI8Args, uint32_t, uint32_t, uint32_t, uint32_t) = nullptr;
    const auto pick = [&]<size_t... I>(std::index_sequence<I...>) {
        ((kShapes[I].fn == s.fn && kShapes[I].ft == s.ft ? (void)(k = k_gemm_i8_tiles<T, kShapes[I].fn, kShapes[I].ft, kShapes[I].stages>) : (void)0), ...);
    };
    pick(std::make_index_sequence<std::size(kShapes)>{});
    return k;
}

template <typename T>
int launch_few(const GemmI8Args& a, hipStream_t st) {
    // a CU's channels in as few workgroups as take them: 5120 of 17408 codes as 256 workgroups of 20 channels 15.3 us, as 320 of 16 22.2
    const uint32_t beside = (a.rows + 32 * kCus - 1) / (32 * kCus), each = (a.rows + beside * kCus - 1) / (beside * kCus);
    auto* k = a.n_vec <= 16 ? (each > 16 ? k_gemm_i8_few<T, 2, 1, 8, 2> : k_gemm_i8_few<T, 1, 1, 8, 4>) : k_gemm_i8_few<T, 1, 2, 8, 4>;
    hipLaunchKernelGGL(k, dim3((a.rows + each - 1) / each), dim3(512), 0, st, a, each);
    return hip_status(hipGetLastError(), "gemm_i8");
}

// A part of y: channels n0.. and vectors t0.. of a.
template <typename T>
GemmI8Args part_of(const GemmI8Args& a, uint32_t n0, uint32_t rows, uint32_t t0, uint32_t n_vec) {
    GemmI8Args p = a;
    p.w += (uint64_t)n0 * a.w_stride;
    p.w_scales += n0;
    p.rows = rows;
    p.x += (uint64_t)t0 * a.x_stride;
    p.x_scales += t0;
    p.n_vec = n_vec;
    p.y = static_cast<T*>(a.y) + t0 * a.y_stride + n0;
    return p;
}

template <typename T>
int launch_typed(const GemmI8Args& a, hipStream_t st) {
    // a grid has fewer than 2^32 threads
    constexpr uint32_t kRows = 1u << 21, kVectors = 1u << 16;
    if (a.rows > kRows || a.n_vec > kVectors) {
        for (uint32_t t = 0; t < a.n_vec; t += kVectors)
            for (uint32_t n = 0; n < a.rows; n += kRows)
                if (const int rc = launch_typed<T>(part_of<T>(a, n, std::min(a.rows - n, kRows), t, std::min(a.n_vec - t, kVectors)), st)) return rc;
        return HALO_MI_OK;
    }
    // up to 16 vectors are one fragment; up to 32, where a CU has no more channels than one fragment takes (20 vectors by 1024 channels of 5120:
    // 6.5 us, on tiles 10.1)
    if (a.n_vec <= 16 || (a.n_vec <= 32 && a.rows <= 16 * kCus)) return launch_few<T>(a, st);
    const TilePlan p = plan_tiles(a.rows, a.cols, a.n_vec);
    hipLaunchKernelGGL(kernel_of<T>(p.shape), dim3(p.tiles_n * p.tiles_t), dim3(512), p.shape.stages * stage_bytes(p.shape), st, a, p.tiles_n, p.tiles_t, p.each_n, p.each_t);
    return hip_status(hipGetLastError(), "gemm_i8");
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
