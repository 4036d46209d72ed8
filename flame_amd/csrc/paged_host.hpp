// What the entry points of the paged cache check and plan on the host, and how the attention is launched.
#pragma once
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "attn_paged.hpp"
#include "launch_lds.hpp"
#include "view_checks.hpp"
#include "../../include/flame_attn.h"

namespace fattn {

// log2 of a page size that is built, or -1
inline int page_shift(int page) {
    for (int s = 4; s <= 16; ++s)
        if (page == 1 << s) return s;
    return -1;
}
// log2 of the tokens that share a scale, a power of two up to 128 and to the page, or -1
inline int block_shift(int block, int page) {
    for (int s = 0; s <= 7; ++s)
        if (block == 1 << s) return block <= page ? s : -1;
    return -1;
}
inline bool head_dim_ok(int D) { return D % 8 == 0 && D <= 128; }

// Most units that PagedCut makes of `tiles` tiles that `groups` walks (sequences, heads, row tiles) have together at most.
inline int64_t most_units(int64_t tiles, int64_t groups) {
    if (tiles <= 0) return 0;
    return std::min<int64_t>(PagedCut::places((int)groups), (tiles + PagedCut::least((int)groups) - 1) / PagedCut::least((int)groups)) + groups;
}
inline int64_t most_shared_units(int64_t tiles, int64_t groups) {
    return tiles <= 0 ? 0 : std::min<int64_t>(PagedCut::kShared, (tiles + PagedCut::kLeast - 1) / PagedCut::kLeast) + groups;
}

struct PagedSizes {
    int64_t prefix_units, own_units, prefix_rows, own_rows;        // bounds of the units and of their rows
    bool direct;                                                   // one workgroup takes all keys
    size_t plan_bytes, ml_bytes, bytes;                            // of the workspace
};
// Up to so many keys of a table one workgroup takes all of a sequence's, in one launch and without the summing of the batch; with as many walks as
// the cut leaves whole, up to as many keys as it leaves whole.  (In two launches -> in one, us, D = 128, 8 key heads: one sequence of 500 12.0 -> 8.2, 4 of
// 1000 13.0 -> 11.4, 64 of 1000 48 -> 42, 64 of 2000 97 -> 92, 64 of 200 to 2000 57 -> 52.  4 of 2000 15.4, one workgroup each 17.9.)
constexpr int64_t kDirectKeys = 1024;

constexpr int64_t kMostRanges = 1024;          // workgroups that run at once at most

// false: too large; `ranges`: without a prefix the tiles are cut into ranges
inline bool paged_sizes(int B, int H, int H_kv, int N, int D, int page, int pages, int prefix_pages, bool ranges, PagedSizes* z) {
    const int64_t rows = (int64_t)N * (H / H_kv), rt = (rows + 31) / 32;
    if (rows > INT32_MAX / 2 || B * rows > INT32_MAX / 2) return false;
    const int64_t prefix_rt = PagedCut::prefix_row_tiles((int)(B * rows));
    const double own = (double)(((int64_t)pages * page + 31) / 32) * B * H_kv * rt, prefix = (double)(((int64_t)prefix_pages * page + 31) / 32) * H_kv * prefix_rt;
    if (own > INT32_MAX / 2 || prefix > INT32_MAX / 2 || (double)pages * page > INT32_MAX / 2 || (double)prefix_pages * page > INT32_MAX / 2) return false;
    const bool shared = PagedCut::shared((int)(B * rows));
    z->direct = prefix_pages == 0 && (int64_t)pages * page <= (B * H_kv * rt < PagedCut::kFill / 2 ? kDirectKeys : PagedCut::kLong * PagedCut::kTile);
    if (!grid_fits(z->direct ? B * H_kv * rt : ((int64_t)B * H * N + 3) / 4)) return false;          // as launch_paged launches
    z->own_units = most_units((int64_t)own, B * H_kv * rt);
    if (ranges && prefix_pages == 0) z->own_units = 2 * std::min<int64_t>(kMostRanges, ((int64_t)own + PagedCut::kLeast - 1) / PagedCut::kLeast);
    z->prefix_units = shared ? most_shared_units((int64_t)prefix, H_kv * prefix_rt) : most_units((int64_t)prefix, H_kv * prefix_rt);
    z->prefix_rows = z->prefix_units * (shared ? 128 : 32);
    z->own_rows = z->own_units * std::min<int64_t>(32, rows);
    z->plan_bytes = ((size_t)(B + 1) * sizeof(int2) + 255) / 256 * 256;
    z->ml_bytes = ((size_t)(z->prefix_rows + z->own_rows) * sizeof(f32x2) + 255) / 256 * 256;
    z->bytes = z->direct ? 0 : z->plan_bytes + z->ml_bytes + (size_t)(z->prefix_rows + z->own_rows) * D * sizeof(float);
    return true;
}

template <int D, class P>
int launch_paged(const P& p, const PagedSizes& z, hipStream_t s) {
    static std::atomic<uint64_t> done{0}, done4{0}, done8{0};
    const int rows = p.N * (p.H / p.Hkv);
    if (z.direct) {
        const int64_t grid = (int64_t)p.B * p.Hkv * PagedCut::row_tiles(rows);
        // a workgroup of eight wavefronts has its compute unit to itself, of four there are two (four -> eight, us, D = 128, keys 1000: 8
        // workgroups 14.1 -> 11.1, 64 15.1 -> 11.9, 256 22.6 -> 23.1, D = 64 13.8 -> 13.2, 504 40.4 -> 42.2)
        const bool wide = grid <= 256;
        const auto kern = wide ? paged_direct_kernel<D, 8, P> : paged_direct_kernel<D, 4, P>;
        const int lds = paged_lds_bytes<D>(&p, wide ? 8 : 4);
        if (const int rc = set_lds_of_device(reinterpret_cast<const void*>(kern), lds, wide ? done8 : done4)) return rc;
        hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(wide ? 512 : 256), lds, s, p);
        return (int)hipGetLastError();
    }
    const int lds = paged_lds_bytes<D>(&p, 4);
    const auto kern = paged_fwd_kernel<D, P>;
    if (const int rc = set_lds_of_device(reinterpret_cast<const void*>(kern), lds, done)) return rc;
    const int64_t room = D <= 64 ? 768 : 512;          // workgroups that the card holds (D = 64, 64 sequences of 4000: 512 of them 105.4 us, 768 102.8)
    hipLaunchKernelGGL(kern, dim3((unsigned)std::min(room, z.prefix_units + z.own_units)), dim3(256), lds, s, p);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    return launch_paged_merge(p, false, s);
}

}  // namespace fattn
