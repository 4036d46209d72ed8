// Entry points of the paged cache: attention of new tokens (attn_paged.hpp), stores and page copies (kv_pages.hpp).
#include <new>
#include <vector>

#include "kv_pages.hpp"
#include "paged_host.hpp"

using namespace fattn;

__attribute__((visibility("hidden"))) int fattn::launch_paged_merge(const PagedParams& p, bool ranges, hipStream_t s) {
    // (a workgroup for four rows -> per row, us: 32 rows of 500 units 101 -> 92, 256 rows 21.1 -> 20.4, 992 46.9 -> 47.5, 2048 101.6 -> 104.4)
    const int all = p.B * p.H * p.N;                   // rows
    const bool four = all >= 1024;
    const auto kern = ranges ? (four ? paged_merge_kernel<1, true> : paged_merge_kernel<4, true>) : four ? paged_merge_kernel<1, false> : paged_merge_kernel<4, false>;
    hipLaunchKernelGGL(kern, dim3((unsigned)(four ? (all + 3) / 4 : all)), dim3(256), 0, s, p);
    return (int)hipGetLastError();
}

namespace {

// `p`: the scales, if any
template <bool SCALES>
int copy_pages(void* K_cache, void* V_cache, int layers, int n_pages, int H_kv, int page, int D, const int64_t* k_strides, const int64_t* v_strides,
               const int32_t* src, const int32_t* dst, int n, KvCopyParams p, void* stream) {
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
        hipLaunchKernelGGL(kv_copy_kernel<SCALES>, dim3((unsigned)(2 * p.chunks), (unsigned)layers, (unsigned)count), dim3(256), 0, static_cast<hipStream_t>(stream), p, pairs);
        if (const hipError_t e = hipGetLastError()) return (int)e;
    }
    return FLAME_ATTN_OK;
}

}  // namespace

extern "C" {

size_t flame_attn_paged_workspace_bytes(int B, int H, int H_kv, int N, int D, int page, int table_pages, int prefix_pages) {
    if (B <= 0 || H <= 0 || H_kv <= 0 || N <= 0 || D <= 0 || table_pages <= 0 || prefix_pages < 0 || H % H_kv != 0 || !head_dim_ok(D) || page_shift(page) < 0) return 0;
    PagedSizes z;
    return paged_sizes(B, H, H_kv, N, D, page, table_pages, prefix_pages, false, &z) ? z.bytes : 0;
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
    if (!paged_sizes(B, H, H_kv, N, D, page, table_pages, prefix_pages, false, &z) || (int64_t)B * H * N > INT32_MAX / 2) return FLAME_ATTN_ERR_UNSUPPORTED;
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
    return copy_pages<false>(K_cache, V_cache, layers, n_pages, H_kv, page, D, k_strides, v_strides, src, dst, n, KvCopyParams{}, stream);
}

int flame_kv_copy_pages_q8(void* K_cache, void* V_cache, float* K_scale, float* V_scale, int layers, int n_pages, int H_kv, int page, int D, int block,
                           const int64_t* k_strides, const int64_t* v_strides, const int64_t* ks_strides, const int64_t* vs_strides, const int32_t* src,
                           const int32_t* dst, int n, void* stream) {
    if (layers <= 0 || n_pages <= 0 || H_kv <= 0 || page <= 0 || D <= 0 || block <= 0) return FLAME_ATTN_ERR_INVALID;
    if (D % 16 != 0 || page_shift(page) < 0 || block_shift(block, page) < 0) return FLAME_ATTN_ERR_UNSUPPORTED;
    const int blocks = page / block;
    int rc;
    if ((rc = check_byte_view(K_cache, k_strides, 5)) || (rc = check_byte_view(V_cache, v_strides, 5)) || (rc = check_scales(K_scale, ks_strides, 4, blocks)) ||
        (rc = check_scales(V_scale, vs_strides, 4, blocks)))
        return rc;
    const int64_t size[4] = {layers, n_pages, H_kv, blocks};
    if (overlaps(ks_strides, size, 4) || overlaps(vs_strides, size, 4)) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (K_scale == V_scale) return FLAME_ATTN_ERR_INVALID;
    KvCopyParams p{};
    float* const scales[2] = {K_scale, V_scale};
    const int64_t* const st[2] = {ks_strides, vs_strides};
    for (int w = 0; w < 2; ++w) {
        p.s[w] = scales[w];
        p.s_layer[w] = st[w][0];
        p.s_page[w] = st[w][1];
        p.s_head[w] = st[w][2];
        p.s_block[w] = st[w][3];
    }
    p.blocks = blocks;
    // two codes travel as one number of 16 bits
    int64_t half[2][5];
    for (int i = 0; i < 5; ++i) {
        half[0][i] = i < 4 ? k_strides[i] / 2 : 1;
        half[1][i] = i < 4 ? v_strides[i] / 2 : 1;
    }
    return copy_pages<true>(K_cache, V_cache, layers, n_pages, H_kv, page, D / 2, half[0], half[1], src, dst, n, p, stream);
}

}  // extern "C"
