// gfx950 kernels of the pages' owner: giving slots pages, releasing them, forking slots, packing the pool, and
// copying pages. The state (reference counts, lengths, tables) lives on the device and is changed there, so a
// serving loop needs no word from the host between steps and can be captured whole.
//
// Who gets which page is one order (the list's) over another (the free pages by number), so one workgroup of 1024
// threads decides: prefix sums over the list and over the counts, 4096 counts a step (1024 where pages move). What costs time is the
// pages' bytes (hundreds of KB each with all layers) and long tables: a second kernel copies them with the whole GPU,
// from lists that the first one leaves in scratch memory.
//
// Measured: 8 sequences forked 8 ways over 1300 pages, deciding 7.4 us (a chain of scans and reads) and copying 6.1; grown
// 5.4 and 2.0; a pool of 1500 pages packed, 186 MB of pages read and written, 5.0 and 33.7 (5.5 TB/s).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>

#include "kv.h"
#include "kv_device.h"
#include "launch.h"

namespace halo_mi {
namespace {

using namespace dev;

constexpr uint32_t kOwnerBlock = 1024;   // threads of the deciding workgroup; >= HALO_MI_KV_LIST_MAX
constexpr uint32_t kOwnerWaves = kOwnerBlock / 64;
constexpr uint32_t kCopyBlock = 256;
constexpr uint32_t kCopyBytes = 16384;   // of a page per workgroup and step: 4 accesses of 16 bytes per thread
constexpr uint32_t kCopyGrid = 2048;     // 8 workgroups per CU
// Words of scratch before the free pages' list: the copies (their number, then source and destination), then
// what the second kernel does to each entry's table.
constexpr uint32_t entry_words(uint32_t n) { return 1 + 2 * n; }
constexpr uint32_t list_words(uint32_t n) { return entry_words(n) + 3 * n; }
static_assert(kOwnerBlock >= HALO_MI_KV_LIST_MAX);

// Exclusive prefix sum over the workgroup; total receives the sum. lds: kOwnerWaves words.
__device__ __forceinline__ uint32_t block_scan(uint32_t v, uint32_t* lds, uint32_t& total) {
    const uint32_t lane = threadIdx.x % 64, wave = threadIdx.x / 64;
    uint32_t sum = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t below = (uint32_t)__shfl_up((int)sum, off);
        if (lane >= (uint32_t)off) sum += below;
    }
    __syncthreads();  // lds may still be read from the last scan
    if (lane == 63) lds[wave] = sum;
    __syncthreads();
    uint32_t before = 0;
    total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kOwnerWaves; ++w) {
        before += w < wave ? lds[w] : 0u;
        total += lds[w];
    }
    return before + sum - v;
}

struct OwnerLds {
    uint32_t scan[kOwnerWaves];
    __align__(16) int32_t slots[kOwnerBlock];
    uint32_t first[kOwnerBlock + 1];  // prefix sums of the entries' pages
    uint32_t column[kOwnerBlock];     // where an entry's first new page goes in its table
};

// Whether entry i is the first that names `slot` (every thread calls it). Four names a read and no way out of the loop, so
// that the reads follow each other without a wait.
__device__ __forceinline__ bool first_of_its_name(OwnerLds& l, int32_t slot, uint32_t i, uint32_t n) {
    typedef int32_t int4v __attribute__((ext_vector_type(4)));
    l.slots[i] = slot;
    __syncthreads();
    bool seen = false;
#pragma unroll 4
    for (uint32_t j = 0; j < n; j += 4) {
        const int4v name = *reinterpret_cast<const int4v*>(&l.slots[j]);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) seen |= (name[k] == slot) & (j + k < i);
    }
    return !seen;
}

// The lowest min(want, all) free pages, in order, to `list`; returns how many.
__device__ uint32_t free_pages(const KvPagesArgs& a, uint32_t want, uint32_t* list, OwnerLds& l) {
    uint32_t found = 0;
    for (uint32_t p0 = 0; p0 < a.n_pages && found < want; p0 += 4 * kOwnerBlock) {
        const uint32_t p = p0 + 4 * threadIdx.x;
        bool is_free[4];
        uint32_t mine = 0;
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k) {
            is_free[k] = p + k < a.n_pages && a.refs[p + k] <= 0;
            mine += is_free[k];
        }
        uint32_t total, at = found + block_scan(mine, l.scan, total);
#pragma unroll
        for (uint32_t k = 0; k < 4; ++k)
            if (is_free[k] && at < want) list[at++] = p + k;
        found += total;
    }
    __syncthreads();
    return min(found, want);
}

// Entry i of a call (thread i): `need` pages from `column` of its slot's table on, of which the first becomes a
// copy of page `copy` (-1: none). Returns whether the pages reach; they are then in the table, held once, and the
// copies in `pairs` (count, then source and destination).
__device__ bool take_pages(const KvPagesArgs& a, int32_t slot, uint32_t need, uint32_t column, int32_t copy, uint32_t* list,
                           uint32_t* pairs, uint32_t* status, OwnerLds& l) {
    const uint32_t i = threadIdx.x;
    uint32_t total;
    const uint32_t before = block_scan(need, l.scan, total);
    l.first[i] = before;
    l.column[i] = column;
    l.slots[i] = slot;
    if (i == 0) l.first[kOwnerBlock] = total;
    const uint32_t found = free_pages(a, total, list, l);
    const bool granted = need == 0 || before + need <= found;
    if (!granted) set_status(status, kStatusKvFull);
    for (uint32_t r = i; r < found; r += kOwnerBlock) {
        uint32_t lo = 0, hi = kOwnerBlock;  // the entry that rank r belongs to: the last one with first <= r
        while (hi - lo > 1) {
            const uint32_t mid = (lo + hi) / 2;
            (l.first[mid] <= r ? lo : hi) = mid;
        }
        if (l.first[lo + 1] > found) continue;  // not all of its pages are there
        const uint32_t page = list[r];
        a.tables[(uint64_t)l.slots[lo] * a.table_stride + l.column[lo] + (r - l.first[lo])] = (int32_t)page;
        a.refs[page] = 1;
    }
    const bool copies = granted && need && copy >= 0;
    const uint32_t at = block_scan(copies, l.scan, total);
    if (copies) {
        pairs[1 + 2 * at] = (uint32_t)copy;
        pairs[2 + 2 * at] = list[before];
    }
    if (i == 0) pairs[0] = total;
    return granted;
}

__device__ __forceinline__ uint32_t pages_of(int32_t len, uint32_t block) { return len > 0 ? ((uint32_t)len + block - 1) / block : 0; }

__global__ __launch_bounds__(kOwnerBlock) void k_kv_resize(KvPagesArgs a, const int32_t* slots, const int32_t* new_lens, uint32_t n,
                                                            uint32_t* scratch, uint32_t* status) {
    __shared__ OwnerLds l;
    const uint32_t i = threadIdx.x;
    const int32_t slot = i < n ? slots[i] : -1, want = i < n ? new_lens[i] : 0;
    bool ok = first_of_its_name(l, slot, i, n) && i < n && (uint32_t)slot < a.n_slots && want >= 0;
    if (i < n && !ok) set_status(status, kStatusKvBadIndex);
    uint32_t have = 0, take = 0, column = 0;
    int32_t len = 0, tail = -1;
    const uint32_t goal = pages_of(want, a.block);
    if (ok && goal > a.table_width) {
        ok = false;
        set_status(status, kStatusKvFull);
    }
    if (ok) {
        len = max(a.lens[slot], 0);
        have = min(pages_of(len, a.block), a.table_width);
        column = have;
        take = goal > have ? min(goal - have, a.n_pages + 1) : 0;  // more than all pages is as much as any: sums stay in 32 bits
        if (want > len && len % a.block && have) {
            // tokens go behind others in a page: if it is held twice, into a copy
            const int32_t id = a.tables[(uint64_t)slot * a.table_stride + have - 1];
            if ((uint32_t)id >= a.n_pages) {  // the new tokens would share a page that is none: the slot stays as it is
                ok = false;
                take = 0;
                set_status(status, kStatusKvBadIndex);
            } else if (a.refs[id] > 1) {
                tail = id;
                ++take;
                --column;
            }
        }
    }
    __syncthreads();  // every count, length and table entry has been read
    const bool granted = take_pages(a, slot, take, column, tail, scratch + list_words(n), scratch, status, l);
    ok = ok && granted;
    if (ok && tail >= 0) atomicSub(a.refs + tail, 1);
    if (ok) a.lens[slot] = want;
    if (i < n) {  // the columns that the slot gives back
        uint32_t* e = scratch + entry_words(n) + 3 * i;
        e[0] = (uint32_t)slot;
        e[1] = ok ? goal : 0;
        e[2] = ok ? have : 0;
    }
}

__global__ __launch_bounds__(kOwnerBlock) void k_kv_fork(KvPagesArgs a, const int32_t* src, const int32_t* dst, uint32_t n,
                                                          uint32_t* scratch, uint32_t* status) {
    __shared__ OwnerLds l;
    const uint32_t i = threadIdx.x;
    const int32_t s = i < n ? src[i] : -1, d = i < n ? dst[i] : -1;
    bool ok = first_of_its_name(l, d, i, n) && i < n && (uint32_t)s < a.n_slots && (uint32_t)d < a.n_slots && s != d;
    if (ok) ok = a.lens[d] == 0;
    if (i < n && !ok) set_status(status, kStatusKvBadIndex);
    int32_t len = 0, tail = -1;
    uint32_t full = 0, part = 0;
    if (ok) {
        len = max(a.lens[s], 0);
        full = (uint32_t)len / a.block;
        part = (uint32_t)len % a.block != 0;
        if (full + part > a.table_width) {
            ok = false;
            set_status(status, kStatusKvBadIndex);
        } else if (part) {
            tail = a.tables[(uint64_t)s * a.table_stride + full];
            if ((uint32_t)tail >= a.n_pages) {  // a fresh page in its place would hold another sequence's tokens
                ok = false;
                tail = -1;
                set_status(status, kStatusKvBadIndex);
            }
        }
    }
    __syncthreads();
    const bool granted = take_pages(a, d, ok ? part : 0, full, tail, scratch + list_words(n), scratch, status, l);
    ok = ok && granted;
    if (ok) a.lens[d] = len;
    if (i < n) {  // the columns that the two slots share
        uint32_t* e = scratch + entry_words(n) + 3 * i;
        e[0] = (uint32_t)s;
        e[1] = (uint32_t)d;
        e[2] = ok ? full : 0;
    }
}

// Bytes [at, at + kCopyBytes) of a page, or what there is of them (page_bytes is a multiple of 128).
__device__ __forceinline__ void copy_part(const KvPagesArgs& a, uint32_t from, uint32_t to, uint64_t at) {
    typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
    const uint4v* s = reinterpret_cast<const uint4v*>(a.pool + from * a.page_bytes + at);
    uint4v* d = reinterpret_cast<uint4v*>(a.pool + to * a.page_bytes + at);
    const uint32_t n = (uint32_t)(min(a.page_bytes - at, (uint64_t)kCopyBytes) / 16);
    if (n < kCopyBytes / 16) {  // a page's end
        for (uint32_t k = threadIdx.x; k < n; k += kCopyBlock) d[k] = s[k];
        return;
    }
    constexpr uint32_t U = kCopyBytes / 16 / kCopyBlock;
    uint4v v[U];
#pragma unroll
    for (uint32_t k = 0; k < U; ++k) v[k] = s[threadIdx.x + k * kCopyBlock];
#pragma unroll
    for (uint32_t k = 0; k < U; ++k) d[threadIdx.x + k * kCopyBlock] = v[k];
}

// The pages' bytes and the whole tables' entries, after the deciding kernel. FORK: entries share columns [0, full) of the
// source's table; otherwise they give back columns [goal, have).
template <bool FORK>
__global__ __launch_bounds__(kCopyBlock) void k_kv_apply(KvPagesArgs a, const uint32_t* scratch, uint32_t n, uint32_t* status) {
    const uint32_t parts = (uint32_t)((a.page_bytes + kCopyBytes - 1) / kCopyBytes);
    const uint64_t units = (uint64_t)scratch[0] * parts;
    for (uint32_t e = blockIdx.x; e < n; e += gridDim.x) {
        const uint32_t* w = scratch + entry_words(n) + 3 * e;
        const uint32_t s = w[0], from = FORK ? 0 : w[1], to = w[2];
        for (uint32_t c = from + threadIdx.x; c < to; c += kCopyBlock) {
            int32_t* entry = a.tables + (uint64_t)s * a.table_stride + c;
            const int32_t id = *entry;
            if ((uint32_t)id < a.n_pages) atomicAdd(a.refs + id, FORK ? 1 : -1);
            else set_status(status, kStatusKvBadIndex);
            if (FORK) a.tables[(uint64_t)w[1] * a.table_stride + c] = id;
            else *entry = -1;
        }
    }
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t i = (uint32_t)(u / parts);
        copy_part(a, scratch[1 + 2 * i], scratch[2 + 2 * i], u % parts * kCopyBytes);
    }
}

__global__ __launch_bounds__(kCopyBlock) void k_kv_copy_listed(KvPagesArgs a, const int32_t* src, const int32_t* dst, uint32_t n,
                                                                uint32_t* status) {
    const uint32_t parts = (uint32_t)((a.page_bytes + kCopyBytes - 1) / kCopyBytes);
    const uint64_t units = (uint64_t)n * parts;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int32_t s = src[u / parts], d = dst[u / parts];
        if ((uint32_t)s < a.n_pages && (uint32_t)d < a.n_pages) copy_part(a, (uint32_t)s, (uint32_t)d, u % parts * kCopyBytes);
        else if (threadIdx.x == 0) set_status(status, kStatusKvBadIndex);
    }
}

// scratch: live pages, moves, then the moved pages, their new places, and every page's new place (n_pages words each)
__global__ __launch_bounds__(kOwnerBlock) void k_kv_compact(KvPagesArgs a, uint32_t* scratch, uint32_t* live_out) {
    __shared__ OwnerLds l;
    uint32_t *moved = scratch + 2, *place = moved + a.n_pages, *where = place + a.n_pages;
    uint32_t live = 0, total;
    for (uint32_t p = threadIdx.x; p < a.n_pages; p += kOwnerBlock) live += a.refs[p] > 0;
    block_scan(live, l.scan, total);
    live = total;
    uint32_t n_moved = 0, n_holes = 0;
    for (uint32_t p0 = 0; p0 < a.n_pages; p0 += kOwnerBlock) {
        const uint32_t p = p0 + threadIdx.x;
        const bool in = p < a.n_pages, alive = in && a.refs[p] > 0, moves = alive && p >= live, hole = in && !alive && p < live;
        if (in) where[p] = p;
        // at most one of the two: one scan counts both (2 * 1024 fits 16 bits)
        uint32_t both;
        const uint32_t at = block_scan(moves | (uint32_t)hole << 16, l.scan, both);
        if (moves) moved[n_moved + (at & 0xFFFFu)] = p;
        if (hole) place[n_holes + (at >> 16)] = p;
        n_moved += both & 0xFFFFu;
        n_holes += both >> 16;
    }
    __threadfence_block();
    __syncthreads();
    for (uint32_t k = threadIdx.x; k < n_moved; k += kOwnerBlock) {
        where[moved[k]] = place[k];
        a.refs[place[k]] = a.refs[moved[k]];
        a.refs[moved[k]] = 0;
    }
    if (threadIdx.x == 0) {
        scratch[0] = live;
        scratch[1] = n_moved;
        if (live_out) *live_out = live;
    }
}

__global__ __launch_bounds__(kCopyBlock) void k_kv_move(KvPagesArgs a, const uint32_t* scratch) {
    const uint32_t live = scratch[0];
    const uint32_t *moved = scratch + 2, *place = moved + a.n_pages, *where = place + a.n_pages;
    const uint32_t parts = (uint32_t)((a.page_bytes + kCopyBytes - 1) / kCopyBytes);
    const uint64_t units = (uint64_t)scratch[1] * parts;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t i = (uint32_t)(u / parts);
        copy_part(a, moved[i], place[i], u % parts * kCopyBytes);
    }
    for (uint64_t e = (uint64_t)blockIdx.x * kCopyBlock + threadIdx.x; e < (uint64_t)a.n_slots * a.table_width;
         e += (uint64_t)gridDim.x * kCopyBlock) {
        const uint32_t slot = (uint32_t)(e / a.table_width), c = (uint32_t)(e % a.table_width);
        int32_t* entry = a.tables + slot * a.table_stride + c;
        if (c >= pages_of(a.lens[slot], a.block)) continue;
        const uint32_t id = (uint32_t)*entry;
        if (id >= live && id < a.n_pages) *entry = (int32_t)where[id];
    }
}

uint32_t copy_grid(const KvPagesArgs& a, uint64_t pages) {
    const uint64_t units = pages * ((a.page_bytes + kCopyBytes - 1) / kCopyBytes);
    return (uint32_t)std::max<uint64_t>(1, std::min<uint64_t>(units, kCopyGrid));
}

}  // namespace

int launch_kv_resize(const KvPagesArgs& a, const int32_t* slots, const int32_t* new_lens, uint32_t n, uint32_t* scratch,
                     uint32_t* status, hipStream_t st) {
    hipLaunchKernelGGL(k_kv_resize, dim3(1), dim3(kOwnerBlock), 0, st, a, slots, new_lens, n, scratch, status);
    hipLaunchKernelGGL(k_kv_apply<false>, dim3(copy_grid(a, n)), dim3(kCopyBlock), 0, st, a, scratch, n, status);
    return hip_status(hipGetLastError(), "kv_resize");
}

int launch_kv_fork(const KvPagesArgs& a, const int32_t* src, const int32_t* dst, uint32_t n, uint32_t* scratch, uint32_t* status,
                   hipStream_t st) {
    hipLaunchKernelGGL(k_kv_fork, dim3(1), dim3(kOwnerBlock), 0, st, a, src, dst, n, scratch, status);
    hipLaunchKernelGGL(k_kv_apply<true>, dim3(copy_grid(a, n)), dim3(kCopyBlock), 0, st, a, scratch, n, status);
    return hip_status(hipGetLastError(), "kv_fork");
}

int launch_kv_compact(const KvPagesArgs& a, uint32_t* scratch, uint32_t* live, hipStream_t st) {
    hipLaunchKernelGGL(k_kv_compact, dim3(1), dim3(kOwnerBlock), 0, st, a, scratch, live);
    hipLaunchKernelGGL(k_kv_move, dim3(copy_grid(a, a.n_pages)), dim3(kCopyBlock), 0, st, a, scratch);
    return hip_status(hipGetLastError(), "kv_compact");
}

int launch_kv_copy_pages(const KvPagesArgs& a, const int32_t* src, const int32_t* dst, uint32_t n, uint32_t* status, hipStream_t st) {
    hipLaunchKernelGGL(k_kv_copy_listed, dim3(copy_grid(a, n)), dim3(kCopyBlock), 0, st, a, src, dst, n, status);
    return hip_status(hipGetLastError(), "kv_copy_pages");
}

}  // namespace halo_mi
