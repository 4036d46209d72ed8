// Entry points of the paged cache: attention of new tokens (attn_paged.hpp), stores and page copies (kv_pages.hpp).
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>
#include <new>
#include <vector>

#include "attn_paged.hpp"
#include "kv_pages.hpp"
#include "launch_lds.hpp"
#include "../../include/flame_attn.h"

using namespace fattn;

namespace {

// element strides of n axes: the last 1, the others multiples of 8 (16-byte rows)
int check_view(const void* base, const int64_t* st, int axes) {
    if (!base || !st) return FLAME_ATTN_ERR_INVALID;
    if (st[axes - 1] != 1 || (reinterpret_cast<uintptr_t>(base) & 15u)) return FLAME_ATTN_ERR_UNSUPPORTED;
    for (int i = 0; i < axes - 1; ++i)
        if (st[i] < 0 || (st[i] & 7)) return FLAME_ATTN_ERR_UNSUPPORTED;
    return st[axes - 2] < (int64_t(1) << 24) ? FLAME_ATTN_OK : FLAME_ATTN_ERR_UNSUPPORTED;   // row offsets inside a tile are kept in 32 bits
}

// whether two elements of a written tensor share their memory (the last axis is contiguous): axes sorted by stride must not reach
// into each other
bool overlaps(const int64_t* st, const int64_t* size, int axes) {
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

// log2 of a page size that is built, or -1
int page_shift(int page) {
    for (int s = 4; s <= 16; ++s)
        if (page == 1 << s) return s;
    return -1;
}
bool head_dim_ok(int D) { return D % 8 == 0 && D <= 128; }

// Most units that PagedCut makes of `tiles` tiles that `groups` walks (sequences, heads, row tiles) have together at most.
int64_t most_units(int64_t tiles, int64_t groups) {
    if (tiles <= 0) return 0;
    return std::min<int64_t>(PagedCut::places((int)groups), (tiles + PagedCut::least((int)groups) - 1) / PagedCut::least((int)groups)) + groups;
}
int64_t most_shared_units(int64_t tiles, int64_t groups) {
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

// A launch has fewer than 2^32 threads.
bool grid_fits(int64_t groups) { return groups * 256 <= (int64_t)UINT32_MAX; }

// false: too large
bool paged_sizes(int B, int H, int H_kv, int N, int D, int page, int pages, int prefix_pages, PagedSizes* z) {
    const int64_t rows = (int64_t)N * (H / H_kv), rt = (rows + 31) / 32;
    if (rows > INT32_MAX / 2 || B * rows > INT32_MAX / 2) return false;
    const int64_t prefix_rt = PagedCut::prefix_row_tiles((int)(B * rows));
    const double own = (double)(((int64_t)pages * page + 31) / 32) * B * H_kv * rt, prefix = (double)(((int64_t)prefix_pages * page + 31) / 32) * H_kv * prefix_rt;
    if (own > INT32_MAX / 2 || prefix > INT32_MAX / 2 || (double)pages * page > INT32_MAX / 2 || (double)prefix_pages * page > INT32_MAX / 2) return false;
    const bool shared = PagedCut::shared((int)(B * rows));
    z->direct = prefix_pages == 0 && (int64_t)pages * page <= (B * H_kv * rt < PagedCut::kFill / 2 ? kDirectKeys : PagedCut::kLong * PagedCut::kTile);
    if (!grid_fits(z->direct ? B * H_kv * rt : ((int64_t)B * H * N + 3) / 4)) return false;          // as launch_paged launches
    z->own_units = most_units((int64_t)own, B * H_kv * rt);
    z->prefix_units = shared ? most_shared_units((int64_t)prefix, H_kv * prefix_rt) : most_units((int64_t)prefix, H_kv * prefix_rt);
    z->prefix_rows = z->prefix_units * (shared ? 128 : 32);
    z->own_rows = z->own_units * std::min<int64_t>(32, rows);
    z->plan_bytes = ((size_t)(B + 1) * sizeof(int2) + 255) / 256 * 256;
    z->ml_bytes = ((size_t)(z->prefix_rows + z->own_rows) * sizeof(f32x2) + 255) / 256 * 256;
    z->bytes = z->direct ? 0 : z->plan_bytes + z->ml_bytes + (size_t)(z->prefix_rows + z->own_rows) * D * sizeof(float);
    return true;
}

template <int D>
int launch_paged(const PagedParams& p, const PagedSizes& z, hipStream_t s) {
    static std::atomic<uint64_t> done{0}, done4{0}, done8{0};
    const int rows = p.N * (p.H / p.Hkv);
    if (z.direct) {
        const int64_t grid = (int64_t)p.B * p.Hkv * PagedCut::row_tiles(rows);
        // a workgroup of eight wavefronts has its compute unit to itself, of four there are two (four -> eight, us, D = 128, keys 1000: 8
        // workgroups 14.1 -> 11.1, 64 15.1 -> 11.9, 256 22.6 -> 23.1, D = 64 13.8 -> 13.2, 504 40.4 -> 42.2)
        const bool wide = grid <= 256;
        const auto kern = wide ? paged_direct_kernel<D, 8> : paged_direct_kernel<D, 4>;
        const int lds = PagedTile<D>::lds_bytes(wide ? 8 : 4);
        if (const int rc = set_lds_of_device(reinterpret_cast<const void*>(kern), lds, wide ? done8 : done4)) return rc;
        hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(wide ? 512 : 256), lds, s, p);
        return (int)hipGetLastError();
    }
    constexpr int lds = PagedTile<D>::lds_bytes(4);
    if (const int rc = set_lds_of_device(reinterpret_cast<const void*>(paged_fwd_kernel<D>), lds, done)) return rc;
    const int64_t room = D <= 64 ? 768 : 512;          // workgroups that the card holds (D = 64, 64 sequences of 4000: 512 of them 105.4 us, 768 102.8)
    hipLaunchKernelGGL(paged_fwd_kernel<D>, dim3((unsigned)std::min(room, z.prefix_units + z.own_units)), dim3(256), lds, s, p);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    // (a workgroup for four rows -> per row, us: 32 rows of 500 units 101 -> 92, 256 rows 21.1 -> 20.4, 992 46.9 -> 47.5, 2048 101.6 -> 104.4)
    const int all = p.B * p.H * p.N;                   // rows
    if (all >= 1024) hipLaunchKernelGGL(paged_merge_kernel<1>, dim3((unsigned)((all + 3) / 4)), dim3(256), 0, s, p);
    else hipLaunchKernelGGL(paged_merge_kernel<4>, dim3((unsigned)all), dim3(256), 0, s, p);
    return (int)hipGetLastError();
}

}  // namespace

extern "C" {

size_t flame_attn_paged_workspace_bytes(int B, int H, int H_kv, int N, int D, int page, int table_pages, int prefix_pages) {
    if (B <= 0 || H <= 0 || H_kv <= 0 || N <= 0 || D <= 0 || table_pages <= 0 || prefix_pages < 0 || H % H_kv != 0 || !head_dim_ok(D) || page_shift(page) < 0) return 0;
    PagedSizes z;
    return paged_sizes(B, H, H_kv, N, D, page, table_pages, prefix_pages, &z) ? z.bytes : 0;
}

int flame_attn_paged_fwd_bf16(const void* Q, const void* K_cache, const void* V_cache, void* O, void* LSE, const int32_t* page_table,
                              int64_t table_stride, int table_pages, const int32_t* kv_len, const int32_t* prefix_table, int prefix_pages,
                              const int32_t* prefix_len, int B, int H, int H_kv, int N, int D, int n_pages, int page, float scale,
                              const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides, void* workspace,
                              size_t workspace_bytes, void* stream) {
    if (B <= 0 || H <= 0 || H_kv <= 0 || N <= 0 || D <= 0 || n_pages <= 0 || page <= 0 || table_pages <= 0 || prefix_pages < 0) return FLAME_ATTN_ERR_INVALID;
    if (!page_table || !kv_len || table_stride < 0 || H % H_kv != 0 || !(scale > 0.f) || !std::isfinite(scale)) return FLAME_ATTN_ERR_INVALID;
    if ((prefix_pages > 0) != (prefix_table != nullptr) || (prefix_table != nullptr) != (prefix_len != nullptr)) return FLAME_ATTN_ERR_INVALID;
    if (!head_dim_ok(D) || page_shift(page) < 0) return FLAME_ATTN_ERR_UNSUPPORTED;
    int rc;
    if ((rc = check_view(Q, q_strides, 4)) || (rc = check_view(K_cache, k_strides, 4)) || (rc = check_view(V_cache, v_strides, 4)) ||
        (rc = check_view(O, o_strides, 4)))
        return rc;
    const int64_t o_size[4] = {B, H, N, D};
    if (overlaps(o_strides, o_size, 4)) return FLAME_ATTN_ERR_UNSUPPORTED;
    PagedSizes z;
    if (!paged_sizes(B, H, H_kv, N, D, page, table_pages, prefix_pages, &z) || (int64_t)B * H * N > INT32_MAX / 2) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (z.bytes && (!workspace || workspace_bytes < z.bytes)) return FLAME_ATTN_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return FLAME_ATTN_ERR_UNSUPPORTED;
    PagedParams p{};
    p.q = static_cast<const uint16_t*>(Q);
    p.k = static_cast<const uint16_t*>(K_cache);
    p.v = static_cast<const uint16_t*>(V_cache);
    p.o = static_cast<uint16_t*>(O);
    p.lse = static_cast<float*>(LSE);
    p.table = page_table;
    p.table_stride = table_stride;
    p.table_pages = table_pages;
    p.kv_len = kv_len;
    p.prefix_table = prefix_table;
    p.prefix_len = prefix_len;
    p.prefix_pages = prefix_pages;
    p.qs = Strides{q_strides[0], q_strides[1], q_strides[2]};
    p.ks = Strides{k_strides[0], k_strides[1], k_strides[2]};
    p.vs = Strides{v_strides[0], v_strides[1], v_strides[2]};
    p.os = Strides{o_strides[0], o_strides[1], o_strides[2]};
    p.B = B;
    p.H = H;
    p.Hkv = H_kv;
    p.N = N;
    p.n_pages = n_pages;
    p.page_shift = page_shift(page);
    p.d = D;
    p.scale = scale;
    p.own_slot = z.prefix_rows;
    p.plan = static_cast<int2*>(workspace);
    p.part_ml = reinterpret_cast<f32x2*>(static_cast<char*>(workspace) + z.plan_bytes);
    p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + z.plan_bytes + z.ml_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return D <= 64 ? launch_paged<64>(p, z, s) : D <= 96 ? launch_paged<96>(p, z, s) : launch_paged<128>(p, z, s);
}

int flame_kv_store_bf16(const void* K, const void* V, void* K_cache, void* V_cache, const int32_t* page_table, int64_t table_stride, int table_pages,
                        const int32_t* cu, const int32_t* start, int n_seqs, int T, int H_kv, int D, int n_pages, int page, const int64_t* k_strides,
                        const int64_t* v_strides, const int64_t* kc_strides, const int64_t* vc_strides, void* stream) {
    if (!page_table || !cu || !start || n_seqs <= 0 || T <= 0 || H_kv <= 0 || D <= 0 || n_pages <= 0 || page <= 0 || table_pages <= 0 || table_stride < 0)
        return FLAME_ATTN_ERR_INVALID;
    if (D % 8 != 0 || (int64_t)H_kv * D > INT32_MAX / 2 || page_shift(page) < 0) return FLAME_ATTN_ERR_UNSUPPORTED;
    // (a workgroup's rows are counted in 32 bits, also those past T)
    const int rows_per_wave = std::max(1, 64 / (H_kv * (D / 8)));
    const int64_t grid = ((int64_t)T + 4 * rows_per_wave - 1) / (4 * rows_per_wave);
    if (T > INT32_MAX - 1023 || !grid_fits(grid)) return FLAME_ATTN_ERR_UNSUPPORTED;
    int rc;
    if ((rc = check_view(K, k_strides, 3)) || (rc = check_view(V, v_strides, 3)) || (rc = check_view(K_cache, kc_strides, 4)) || (rc = check_view(V_cache, vc_strides, 4)))
        return rc;
    const int64_t size[4] = {n_pages, H_kv, page, D};
    if (overlaps(kc_strides, size, 4) || overlaps(vc_strides, size, 4)) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (K_cache == V_cache) return FLAME_ATTN_ERR_INVALID;             // both would be written to the same places
    KvStoreParams p{};
    p.k = static_cast<const uint16_t*>(K);
    p.v = static_cast<const uint16_t*>(V);
    p.kc = static_cast<uint16_t*>(K_cache);
    p.vc = static_cast<uint16_t*>(V_cache);
    p.table = page_table;
    p.table_stride = table_stride;
    p.table_pages = table_pages;
    p.cu = cu;
    p.start = start;
    p.ks = Strides{0, k_strides[1], k_strides[0]};
    p.vs = Strides{0, v_strides[1], v_strides[0]};
    p.kcs = Strides{kc_strides[0], kc_strides[1], kc_strides[2]};
    p.vcs = Strides{vc_strides[0], vc_strides[1], vc_strides[2]};
    p.n = n_seqs;
    p.rows = T;
    p.Hkv = H_kv;
    p.d = D;
    p.n_pages = n_pages;
    p.page_shift = page_shift(page);
    p.rows_per_wave = rows_per_wave;
    hipLaunchKernelGGL(kv_store_kernel, dim3((unsigned)grid), dim3(256), 0, static_cast<hipStream_t>(stream), p);
    return (int)hipGetLastError();
}

int flame_kv_copy_pages_bf16(void* K_cache, void* V_cache, int layers, int n_pages, int H_kv, int page, int D, const int64_t* k_strides,
                             const int64_t* v_strides, const int32_t* src, const int32_t* dst, int n, void* stream) {
    if (layers <= 0 || n_pages <= 0 || H_kv <= 0 || page <= 0 || D <= 0 || n < 0 || (n > 0 && (!src || !dst))) return FLAME_ATTN_ERR_INVALID;
    if (D % 8 != 0 || (double)H_kv * page * D > INT32_MAX / 2 || layers > 65535) return FLAME_ATTN_ERR_UNSUPPORTED;
    int rc;
    if ((rc = check_view(K_cache, k_strides, 5)) || (rc = check_view(V_cache, v_strides, 5))) return rc;
    const int64_t size[5] = {layers, n_pages, H_kv, page, D};
    if (overlaps(k_strides, size, 5) || overlaps(v_strides, size, 5)) return FLAME_ATTN_ERR_UNSUPPORTED;
    try {
        std::vector<int32_t> to(dst, dst + n);
        std::sort(to.begin(), to.end());
        if (std::adjacent_find(to.begin(), to.end()) != to.end()) return FLAME_ATTN_ERR_INVALID;          // two sources for one page
        for (int i = 0; i < n; ++i) {
            if (src[i] < 0 || src[i] >= n_pages || dst[i] < 0 || dst[i] >= n_pages) return FLAME_ATTN_ERR_INVALID;
            if (std::binary_search(to.begin(), to.end(), src[i])) return FLAME_ATTN_ERR_INVALID;             // read and written in one call
        }
    } catch (const std::bad_alloc&) {
        return (int)hipErrorOutOfMemory;
    }
    KvCopyParams p{};
    const int64_t* const st[2] = {k_strides, v_strides};
    p.c[0] = static_cast<uint16_t*>(K_cache);
    p.c[1] = static_cast<uint16_t*>(V_cache);
    p.contiguous = 1;
    for (int w = 0; w < 2; ++w) {
        p.layer[w] = st[w][0];
        p.page[w] = st[w][1];
        p.head[w] = st[w][2];
        p.token[w] = st[w][3];
        if (st[w][3] != D || (H_kv > 1 && st[w][2] != (int64_t)page * D)) p.contiguous = 0;
    }
    p.layers = layers;
    p.Hkv = H_kv;
    p.page_size = page;
    p.d = D;
    p.granules = H_kv * page * (D / 8);
    p.chunks = (p.granules + 256 * kKvCopyPerThread - 1) / (256 * kKvCopyPerThread);
    for (int first = 0; first < n; first += KvCopyPairs::kMost) {
        KvCopyPairs pairs{};
        const int count = std::min(n - first, KvCopyPairs::kMost);
        std::copy(src + first, src + first + count, pairs.src);
        std::copy(dst + first, dst + first + count, pairs.dst);
        hipLaunchKernelGGL(kv_copy_kernel, dim3((unsigned)(2 * p.chunks), (unsigned)layers, (unsigned)count), dim3(256), 0, static_cast<hipStream_t>(stream), p, pairs);
        if (const hipError_t e = hipGetLastError()) return (int)e;
    }
    return FLAME_ATTN_OK;
}

}  // extern "C"
