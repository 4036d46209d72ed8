// What the entry points check of a tensor's layout.
#pragma once
#include <stdint.h>

#include <algorithm>

#include "../../include/flame_attn.h"

namespace fattn {

// element strides of n axes: the last 1, the others multiples of 8 (16-byte rows)
inline int check_view(const void* base, const int64_t* st, int axes) {
    if (!base || !st) return FLAME_ATTN_ERR_INVALID;
    if (st[axes - 1] != 1 || (reinterpret_cast<uintptr_t>(base) & 15u)) return FLAME_ATTN_ERR_UNSUPPORTED;
    for (int i = 0; i < axes - 1; ++i)
        if (st[i] < 0 || (st[i] & 7)) return FLAME_ATTN_ERR_UNSUPPORTED;
    return st[axes - 2] < (int64_t(1) << 24) ? FLAME_ATTN_OK : FLAME_ATTN_ERR_UNSUPPORTED;   // row offsets inside a tile are kept in 32 bits
}

// the same of a tensor of bytes: multiples of 16
inline int check_byte_view(const void* base, const int64_t* st, int axes) {
    if (const int rc = check_view(base, st, axes)) return rc;
    for (int i = 0; i < axes - 1; ++i)
        if (st[i] & 15) return FLAME_ATTN_ERR_UNSUPPORTED;
    return FLAME_ATTN_OK;
}
// fp32 scales, any strides; the offset of the last axis (of `size` elements) is kept in 32 bits
inline int check_scales(const void* base, const int64_t* st, int axes, int64_t size) {
    if (!base || !st) return FLAME_ATTN_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(base) & 3u) return FLAME_ATTN_ERR_UNSUPPORTED;
    for (int i = 0; i < axes; ++i)
        if (st[i] < 0) return FLAME_ATTN_ERR_UNSUPPORTED;
    return st[axes - 1] <= INT32_MAX && size * st[axes - 1] <= INT32_MAX ? FLAME_ATTN_OK : FLAME_ATTN_ERR_UNSUPPORTED;
}

// whether two elements of a written tensor share their memory: axes sorted by stride must not reach
// into each other
inline bool overlaps(const int64_t* st, const int64_t* size, int axes) {
    int order[5];
    for (int i = 0; i < axes; ++i) order[i] = i;
    std::sort(order, order + axes, [&](int a, int b) { return st[a] < st[b]; });
    int64_t reach = 1;             // elements that the axes so far span
    for (int j = 0; j < axes; ++j) {
        const int i = order[j];
        if (size[i] == 1) continue;
        if (st[i] < reach) return true;
        reach += (size[i] - 1) * st[i];
    }
    return false;
}

// A launch has fewer than 2^32 threads.
inline bool grid_fits(int64_t groups) { return groups * 256 <= (int64_t)UINT32_MAX; }

}  // namespace fattn
