// Argument checks that the C ABI's calls on caches share.
#pragma once

#include <hip/hip_runtime_api.h>
#include <stddef.h>
#include <stdint.h>

#include "api_internal.h"
#include "paged_launch.h"

namespace afhip {

constexpr size_t kInt32Max = 0x7fffffff;

inline bool aligned(afhip_buffer b, size_t to) { return b.ptr != 0 && b.ptr % to == 0; }

// count elements of `size` bytes, aligned to their size
inline bool holds(afhip_buffer b, size_t count, size_t size) {
    size_t bytes;
    return checked_mul(count, size, &bytes) && bytes <= b.len && (count == 0 || aligned(b, size));
}

inline bool add(size_t* sum, size_t count, size_t stride) {
    size_t more;
    return checked_mul(count, stride, &more) && !__builtin_add_overflow(*sum, more, sum);
}

// The elements from the first of [n0][n1][n2] to the last, the last dimension contiguous.
inline bool span(size_t n0, size_t s0, size_t n1, size_t s1, size_t n2, size_t* out) {
    *out = n2;
    return n0 != 0 && n1 != 0 && n2 != 0 && add(out, n0 - 1, s0) && add(out, n1 - 1, s1);
}

inline afhip_status view_of(const afhip_paged_cache& c, CacheView* view) {
    if (c.type != AFHIP_TYPE_F16 && c.type != AFHIP_TYPE_BF16) return AFHIP_ERR_UNSUPPORTED_TENSOR_TYPE;
    size_t slots, elements, bytes;
    if (c.blocks == 0 || c.block_size == 0 || c.kv_heads == 0 || c.head_dim == 0 || !checked_mul(c.blocks, c.block_size, &slots) ||
        slots > kInt32Max || c.kv_heads > kInt32Max || c.head_dim > kInt32Max || c.head_dim % 8 != 0 || c.block_stride % 8 != 0 ||
        c.slot_stride % 8 != 0 || c.head_stride % 8 != 0)
        return AFHIP_ERR_INVALID_STATE;
    if (!span(c.blocks, c.block_stride, c.block_size, c.slot_stride, c.head_dim, &elements) ||
        !add(&elements, c.kv_heads - 1, c.head_stride) || !checked_mul(elements, 2, &bytes) || bytes >= (size_t{1} << 36) ||
        c.block_stride / 8 > 0xffffffffu || c.slot_stride / 8 > 0xffffffffu || c.head_stride / 8 > 0xffffffffu)
        return AFHIP_ERR_INVALID_STATE;
    if (bytes > c.keys.len || bytes > c.values.len || !aligned(c.keys, 16) || !aligned(c.values, 16)) return AFHIP_ERR_INVALID_STATE;
    *view = CacheView{reinterpret_cast<uint4*>(c.keys.ptr),
                      reinterpret_cast<uint4*>(c.values.ptr),
                      static_cast<uint32_t>(c.blocks),
                      static_cast<uint32_t>(c.block_size),
                      static_cast<uint32_t>(c.kv_heads),
                      static_cast<uint32_t>(c.head_dim),
                      static_cast<uint32_t>(c.block_stride / 8),
                      static_cast<uint32_t>(c.slot_stride / 8),
                      static_cast<uint32_t>(c.head_stride / 8)};
    return AFHIP_OK;
}

inline afhip_status status_of(hipError_t e) { return e == hipSuccess ? AFHIP_OK : static_cast<afhip_status>(e); }

}  // namespace afhip
