// Checks of operands that the entry points with rows of heads, lists and status words share (kv_api.cpp, layer_api.cpp): types,
// strides, alignment, overlap.
#pragma once

#include <cstdint>
#include <initializer_list>

#include "kv.h"
#include "launch.h"

namespace halo_mi {

// A range of an operand, for the overlap checks.
struct Range {
    const void* p;
    uint64_t bytes;
    const char* name;
};

inline int check_apart(const char* op, const Range& out, std::initializer_list<Range> others) {
    for (const Range& r : others)
        if (ranges_overlap(out.p, out.bytes, r.p, r.bytes)) return set_error(HALO_MI_E_KERNEL, "%s: %s overlaps %s", op, out.name, r.name);
    return HALO_MI_OK;
}

inline uint32_t elem_bytes(uint32_t type) { return type == HALO_MI_F32 ? 4 : type == HALO_MI_F16 || type == HALO_MI_BF16 ? 2 : 0; }

inline int check_type(const char* op, uint32_t type) {
    if (elem_bytes(type) == 0) return set_error(HALO_MI_E_UNSUPPORTED, "%s: element type %u is not F32, F16 or BF16", op, type);
    return HALO_MI_OK;
}

// Rows of heads: resolves the dense strides, checks alignment and that heads and rows do not overlap.
// bytes receives the operand's extent.
inline int check_rows(const char* op, const char* name, HeadRows& r, uint64_t rows, uint32_t heads, uint32_t dim, uint32_t size, uint64_t* bytes) {
    if (r.head_stride == 0) r.head_stride = dim;
    const uint64_t row = (uint64_t)(heads ? heads - 1 : 0) * r.head_stride + dim;
    if (r.stride == 0) r.stride = (uint64_t)heads * r.head_stride;
    *bytes = 0;
    if (rows == 0 || heads == 0) return HALO_MI_OK;
    if (!r.data) return set_error(HALO_MI_E_KERNEL, "%s: operand %s is empty", op, name);
    if (r.head_stride > 1ull << 40 || r.stride > 1ull << 40 || (rows > 1 && r.stride > (1ull << 58) / rows)) return set_error(HALO_MI_E_KERNEL, "%s: a stride of %s is out of range", op, name);
    if (heads > 1 && r.head_stride < dim) return set_error(HALO_MI_E_KERNEL, "%s: %s head stride < %u elements", op, name, dim);
    // rows may lie inside the heads' stride (a layout [head][row][dim]) or around them
    if (rows > 1 && r.stride < row && !(r.stride >= dim && (heads == 1 || r.head_stride >= (rows - 1) * r.stride + dim)))
        return set_error(HALO_MI_E_KERNEL, "%s: %s row stride %llu lets rows overlap", op, name, (unsigned long long)r.stride);
    if (reinterpret_cast<uintptr_t>(r.data) % size) return set_error(HALO_MI_E_KERNEL, "%s: %s must be %u-byte aligned", op, name, size);
    *bytes = ((rows - 1) * r.stride + row) * size;
    return HALO_MI_OK;
}

// Whether two operands share no element: their ranges are apart, or they lie side by side in rows of one
// stride (q and k of a row-fused projection).
inline bool apart_in_rows(const HeadRows& x, uint32_t x_heads, const HeadRows& y, uint32_t y_heads, uint32_t x_dim, uint32_t y_dim,
                          uint32_t size, const Range& xr, const Range& yr) {
    if (!ranges_overlap(xr.p, xr.bytes, yr.p, yr.bytes)) return true;
    const uint64_t row = x.stride * size;
    const uint64_t x_row = ((uint64_t)(x_heads - 1) * x.head_stride + x_dim) * size, y_row = ((uint64_t)(y_heads - 1) * y.head_stride + y_dim) * size;
    if (x.stride != y.stride || x_row > row || y_row > row) return false;
    const auto px = reinterpret_cast<uintptr_t>(x.data), py = reinterpret_cast<uintptr_t>(y.data);
    const uint64_t off = py >= px ? (py - px) % row : (row - (px - py) % row) % row;  // of y's rows behind x's
    return off >= x_row && off + y_row <= row;
}
inline bool apart_in_rows(const HeadRows& x, uint32_t x_heads, const HeadRows& y, uint32_t y_heads, uint32_t dim, uint32_t size,
                          const Range& xr, const Range& yr) {
    return apart_in_rows(x, x_heads, y, y_heads, dim, dim, size, xr, yr);
}

inline int check_aligned(const char* op, const char* name, const void* p, uint32_t to) {
    if (!p) return set_error(HALO_MI_E_KERNEL, "%s: operand %s is empty", op, name);
    if (reinterpret_cast<uintptr_t>(p) % to) return set_error(HALO_MI_E_KERNEL, "%s: %s must be %u-byte aligned", op, name, to);
    return HALO_MI_OK;
}

// The optional status word is no operand of the call. It is cleared, unless the caller keeps it, once nothing else can refuse the
// call.
inline int check_status(const char* op, uint32_t* status, std::initializer_list<Range> others) {
    if (!status) return HALO_MI_OK;
    if (reinterpret_cast<uintptr_t>(status) % 4) return set_error(HALO_MI_E_KERNEL, "%s: status must be 4-byte aligned", op);
    return check_apart(op, {status, 4, "status"}, others);
}
inline int clear_status(uint32_t* status, uint32_t keep, hipStream_t st) { return status && !keep ? launch_fill_u32(status, 1, 0u, st) : HALO_MI_OK; }

}  // namespace halo_mi
