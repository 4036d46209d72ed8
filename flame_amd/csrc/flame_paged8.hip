// Entry points of the paged cache in 8 bits: attention of new tokens (attn_paged8.hpp), stores and read-backs (kv_pages8.hpp; of bf16 caches, too).
#include "attn_paged8.hpp"
#include "kv_pages8.hpp"
#include "paged_host.hpp"

using namespace fattn;

namespace {

bool is_codes(int dtype) { return dtype == FLAME_ATTN_DTYPE_I8 || dtype == FLAME_ATTN_DTYPE_E4M3; }

template <int CODE, int LANES, int E>
int launch_store(KvStore8Params p, int64_t slots, hipStream_t s) {
    constexpr int PER = 256 / LANES;                   // groups per workgroup
    // A group for every unit, as long as the card has room for them; with more of them a group takes several (us, 7759 rows, 8 heads, D = 128, blocks of 1:
    // 20.3 -> 17.3, 32768 rows 69.6 -> 55.9).
    int per = 1;
    while (LANES <= 64 && per < 8 && slots * 2 * p.Hkv * LANES / per > (1 << 19)) per *= 2;
    p.slot_groups = (2 * p.Hkv + per - 1) / per;
    p.groups = (uint32_t)slots * (uint32_t)p.slot_groups;
    const int64_t grid = ((int64_t)p.groups + PER - 1) / PER;
    if (!grid_fits(grid)) return FLAME_ATTN_ERR_UNSUPPORTED;
    hipLaunchKernelGGL((kv_store8_kernel<CODE, LANES, E>), dim3((unsigned)grid), dim3(256), 0, s, p);
    return (int)hipGetLastError();
}
template <int CODE>
int launch_store(const KvStore8Params& p, int64_t slots, hipStream_t s) {
    const int granules = (p.d / 8) << p.block_shift;   // of a block's head
    if (granules <= 16) return launch_store<CODE, 16, 1>(p, slots, s);
    if (granules <= 32) return launch_store<CODE, 32, 1>(p, slots, s);
    if (granules <= 64) return launch_store<CODE, 64, 1>(p, slots, s);
    if (granules <= 256) return launch_store<CODE, 64, 4>(p, slots, s);
    if (granules <= 512) return launch_store<CODE, 64, 8>(p, slots, s);
    return launch_store<CODE, 256, 8>(p, slots, s);    // up to 128 tokens of 128 numbers
}

template <int D, int CODE, int R>
int attend(const Paged8Params<CODE, R>& p, const PagedSizes& z, hipStream_t s) {
    if (z.direct || p.prefix_pages) return launch_paged<D>(p, z, s);
    static std::atomic<uint64_t> done{0};
    const auto kern = paged_ranges_kernel<D, Paged8Params<CODE, R>>;
    constexpr int lds = Paged8Tile<D>::lds_bytes(4);
    if (const int rc = set_lds_of_device(reinterpret_cast<const void*>(kern), lds, done)) return rc;
    const int64_t room = 256 * kPaged8Groups<D>;       // workgroups that the card holds
    hipLaunchKernelGGL(kern, dim3((unsigned)std::max<int64_t>(1, std::min(room, z.own_units / 2))), dim3(256), lds, s, p);
    if (const hipError_t e = hipGetLastError()) return (int)e;
    return launch_paged_merge(p, true, s);
}
template <int CODE, int R>
int attend(const Paged8Params<CODE, R>& p, const PagedSizes& z, hipStream_t s) {
    return p.d <= 64 ? attend<64>(p, z, s) : attend<128>(p, z, s);
}

}  // namespace

extern "C" {

size_t flame_attn_paged_q8_workspace_bytes(int B, int H, int H_kv, int N, int D, int page, int table_pages, int prefix_pages) {
    if (B <= 0 || H <= 0 || H_kv <= 0 || N <= 0 || D <= 0 || table_pages <= 0 || prefix_pages < 0 || H % H_kv != 0 || D % 16 != 0 || D > 128 || page_shift(page) < 0) return 0;
    PagedSizes z;
    return paged_sizes(B, H, H_kv, N, D, page, table_pages, prefix_pages, true, &z) ? z.bytes : 0;
}

int flame_attn_paged_fwd_q8(const void* Q, const void* K_cache, const void* V_cache, int cache_dtype, const float* K_scale, const float* V_scale, int block,
                            void* O, void* LSE, const int32_t* page_table, int64_t table_stride, int table_pages, const int32_t* kv_len,
                            const int32_t* prefix_table, int prefix_pages, const int32_t* prefix_len, int B, int H, int H_kv, int N, int D, int n_pages,
                            int page, float scale, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides, const int64_t* ks_strides,
                            const int64_t* vs_strides, const int64_t* o_strides, void* workspace, size_t workspace_bytes, void* stream) {
    if (B <= 0 || H <= 0 || H_kv <= 0 || N <= 0 || D <= 0 || n_pages <= 0 || page <= 0 || table_pages <= 0 || prefix_pages < 0 || block <= 0) return FLAME_ATTN_ERR_INVALID;
    if (!page_table || !kv_len || table_stride < 0 || H % H_kv != 0 || !(scale > 0.f) || !std::isfinite(scale)) return FLAME_ATTN_ERR_INVALID;
    if ((prefix_pages > 0) != (prefix_table != nullptr) || (prefix_table != nullptr) != (prefix_len != nullptr)) return FLAME_ATTN_ERR_INVALID;
    if (!is_codes(cache_dtype) || D % 16 != 0 || D > 128 || page_shift(page) < 0 || block_shift(block, page) < 0) return FLAME_ATTN_ERR_UNSUPPORTED;
    int rc;
    if ((rc = check_view(Q, q_strides, 4)) || (rc = check_byte_view(K_cache, k_strides, 4)) || (rc = check_byte_view(V_cache, v_strides, 4)) ||
        (rc = check_scales(K_scale, ks_strides, 3, page / block)) || (rc = check_scales(V_scale, vs_strides, 3, page / block)) || (rc = check_view(O, o_strides, 4)))
        return rc;
    for (const int64_t* st : {ks_strides, vs_strides})             // kept in bytes and 32 bits
        if (st[0] > INT32_MAX / 4 || st[2] > INT32_MAX / 4) return FLAME_ATTN_ERR_UNSUPPORTED;
    const int64_t o_size[4] = {B, H, N, D};
    if (overlaps(o_strides, o_size, 4)) return FLAME_ATTN_ERR_UNSUPPORTED;
    PagedSizes z;
    if (!paged_sizes(B, H, H_kv, N, D, page, table_pages, prefix_pages, true, &z) || (int64_t)B * H * N > INT32_MAX / 2) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (z.bytes && (!workspace || workspace_bytes < z.bytes)) return FLAME_ATTN_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return FLAME_ATTN_ERR_UNSUPPORTED;
    auto call = [&](auto p) {
        p.q = static_cast<const uint16_t*>(Q);
        p.k8 = static_cast<const uint8_t*>(K_cache);
        p.v8 = static_cast<const uint8_t*>(V_cache);
        p.k_scale = K_scale;
        p.v_scale = V_scale;
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
        p.kss = Strides{4 * ks_strides[0], 4 * ks_strides[1], 4 * ks_strides[2]};
        p.vss = Strides{4 * vs_strides[0], 4 * vs_strides[1], 4 * vs_strides[2]};
        p.os = Strides{o_strides[0], o_strides[1], o_strides[2]};
        p.B = B;
        p.H = H;
        p.Hkv = H_kv;
        p.N = N;
        p.n_pages = n_pages;
        p.page_shift = page_shift(page);
        p.block_shift = block_shift(block, page);
        p.d = D;
        p.scale = scale;
        p.own_slot = z.prefix_rows;
        p.plan = static_cast<int2*>(workspace);
        p.part_ml = reinterpret_cast<f32x2*>(static_cast<char*>(workspace) + z.plan_bytes);
        p.part_o = reinterpret_cast<float*>(static_cast<char*>(workspace) + z.plan_bytes + z.ml_bytes);
        return attend(p, z, static_cast<hipStream_t>(stream));
    };
    if (N * (H / H_kv) <= 16) return cache_dtype == FLAME_ATTN_DTYPE_I8 ? call(Paged8Params<kI8, 1>{}) : call(Paged8Params<kE4m3, 1>{});
    return cache_dtype == FLAME_ATTN_DTYPE_I8 ? call(Paged8Params<kI8, 2>{}) : call(Paged8Params<kE4m3, 2>{});
}

int flame_kv_store_q8(const void* K, const void* V, void* K_cache, void* V_cache, int cache_dtype, float* K_scale, float* V_scale, int block,
                      const int32_t* page_table, int64_t table_stride, int table_pages, const int32_t* cu, const int32_t* start, int n_seqs, int T, int H_kv,
                      int D, int n_pages, int page, const int64_t* k_strides, const int64_t* v_strides, const int64_t* kc_strides, const int64_t* vc_strides,
                      const int64_t* ks_strides, const int64_t* vs_strides, void* stream) {
    if (!page_table || !cu || !start || n_seqs <= 0 || T <= 0 || H_kv <= 0 || D <= 0 || n_pages <= 0 || page <= 0 || table_pages <= 0 || table_stride < 0 || block <= 0)
        return FLAME_ATTN_ERR_INVALID;
    if (!is_codes(cache_dtype) || D % 16 != 0 || D > 128 || page_shift(page) < 0 || block_shift(block, page) < 0) return FLAME_ATTN_ERR_UNSUPPORTED;
    const int blocks = page / block, shift = block_shift(block, page);
    int rc;
    if ((rc = check_view(K, k_strides, 3)) || (rc = check_view(V, v_strides, 3)) || (rc = check_byte_view(K_cache, kc_strides, 4)) ||
        (rc = check_byte_view(V_cache, vc_strides, 4)) || (rc = check_scales(K_scale, ks_strides, 3, blocks)) || (rc = check_scales(V_scale, vs_strides, 3, blocks)))
        return rc;
    const int64_t size[4] = {n_pages, H_kv, page, D}, s_size[3] = {n_pages, H_kv, blocks};
    if (overlaps(kc_strides, size, 4) || overlaps(vc_strides, size, 4) || overlaps(ks_strides, s_size, 3) || overlaps(vs_strides, s_size, 3)) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (K_cache == V_cache || K_scale == V_scale) return FLAME_ATTN_ERR_INVALID;
    const double units = ((double)kv_store8_slot(T, n_seqs, shift) + 1) * 2 * H_kv;
    if (units > INT32_MAX / 2) return FLAME_ATTN_ERR_UNSUPPORTED;
    KvStore8Params p{};
    p.x[0] = static_cast<const uint16_t*>(K);
    p.x[1] = static_cast<const uint16_t*>(V);
    p.c[0] = static_cast<uint8_t*>(K_cache);
    p.c[1] = static_cast<uint8_t*>(V_cache);
    p.s[0] = K_scale;
    p.s[1] = V_scale;
    p.xs[0] = Strides{0, k_strides[1], k_strides[0]};
    p.xs[1] = Strides{0, v_strides[1], v_strides[0]};
    p.cs[0] = Strides{kc_strides[0], kc_strides[1], kc_strides[2]};
    p.cs[1] = Strides{vc_strides[0], vc_strides[1], vc_strides[2]};
    p.ss[0] = Strides{ks_strides[0], ks_strides[1], ks_strides[2]};
    p.ss[1] = Strides{vs_strides[0], vs_strides[1], vs_strides[2]};
    p.table = page_table;
    p.table_stride = table_stride;
    p.table_pages = table_pages;
    p.cu = cu;
    p.start = start;
    p.n = n_seqs;
    p.rows = T;
    p.Hkv = H_kv;
    p.d = D;
    p.n_pages = n_pages;
    p.page_shift = page_shift(page);
    p.block_shift = shift;
    const int64_t slots = kv_store8_slot(T, n_seqs, shift);
    hipStream_t s = static_cast<hipStream_t>(stream);
    return cache_dtype == FLAME_ATTN_DTYPE_I8 ? launch_store<kI8>(p, slots, s) : launch_store<kE4m3>(p, slots, s);
}

int flame_kv_load(const void* K_cache, const void* V_cache, int cache_dtype, const float* K_scale, const float* V_scale, int block, void* K, void* V,
                  const int32_t* page_table, int64_t table_stride, int table_pages, const int32_t* cu, const int32_t* start, int n_seqs, int T, int H_kv, int D,
                  int n_pages, int page, const int64_t* kc_strides, const int64_t* vc_strides, const int64_t* ks_strides, const int64_t* vs_strides,
                  const int64_t* k_strides, const int64_t* v_strides, void* stream) {
    const bool codes = is_codes(cache_dtype);
    if (!page_table || !cu || !start || n_seqs <= 0 || T <= 0 || H_kv <= 0 || D <= 0 || n_pages <= 0 || page <= 0 || table_pages <= 0 || table_stride < 0 ||
        (codes && block <= 0) || codes != (K_scale != nullptr) || codes != (V_scale != nullptr))
        return FLAME_ATTN_ERR_INVALID;
    if ((!codes && cache_dtype != FLAME_ATTN_DTYPE_BF16) || D % (codes ? 16 : 8) != 0 || (int64_t)H_kv * D > INT32_MAX / 2 || page_shift(page) < 0 ||
        (codes && block_shift(block, page) < 0))
        return FLAME_ATTN_ERR_UNSUPPORTED;
    const int rows_per_wave = std::max(1, 64 / (H_kv * (D / (codes ? 16 : 8))));
    const int64_t grid = ((int64_t)T + 4 * rows_per_wave - 1) / (4 * rows_per_wave);
    if (T > INT32_MAX - 1023 || !grid_fits(grid)) return FLAME_ATTN_ERR_UNSUPPORTED;
    int rc;
    if ((rc = check_view(K, k_strides, 3)) || (rc = check_view(V, v_strides, 3)) ||
        (rc = codes ? check_byte_view(K_cache, kc_strides, 4) : check_view(K_cache, kc_strides, 4)) ||
        (rc = codes ? check_byte_view(V_cache, vc_strides, 4) : check_view(V_cache, vc_strides, 4)))
        return rc;
    if (codes && ((rc = check_scales(K_scale, ks_strides, 3, page / block)) || (rc = check_scales(V_scale, vs_strides, 3, page / block)))) return rc;
    const int64_t size[3] = {T, H_kv, D};
    if (overlaps(k_strides, size, 3) || overlaps(v_strides, size, 3)) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (K == V) return FLAME_ATTN_ERR_INVALID;
    KvLoadParams p{};
    p.c[0] = K_cache;
    p.c[1] = V_cache;
    p.s[0] = K_scale;
    p.s[1] = V_scale;
    p.y[0] = static_cast<uint16_t*>(K);
    p.y[1] = static_cast<uint16_t*>(V);
    p.cs[0] = Strides{kc_strides[0], kc_strides[1], kc_strides[2]};
    p.cs[1] = Strides{vc_strides[0], vc_strides[1], vc_strides[2]};
    if (codes) {
        p.ss[0] = Strides{ks_strides[0], ks_strides[1], ks_strides[2]};
        p.ss[1] = Strides{vs_strides[0], vs_strides[1], vs_strides[2]};
        p.block_shift = block_shift(block, page);
    }
    p.ys[0] = Strides{0, k_strides[1], k_strides[0]};
    p.ys[1] = Strides{0, v_strides[1], v_strides[0]};
    p.table = page_table;
    p.table_stride = table_stride;
    p.table_pages = table_pages;
    p.cu = cu;
    p.start = start;
    p.n = n_seqs;
    p.rows = T;
    p.Hkv = H_kv;
    p.d = D;
    p.n_pages = n_pages;
    p.page_shift = page_shift(page);
    p.rows_per_wave = rows_per_wave;
    hipStream_t s = static_cast<hipStream_t>(stream);
    const auto kern = !codes ? kv_load_kernel<-1> : cache_dtype == FLAME_ATTN_DTYPE_I8 ? kv_load_kernel<kI8> : kv_load_kernel<kE4m3>;
    hipLaunchKernelGGL(kern, dim3((unsigned)grid), dim3(256), 0, s, p);
    return (int)hipGetLastError();
}

}  // extern "C"
