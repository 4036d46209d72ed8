// Entry points of the attention of packed sequences (attn_packed.hpp): argument checks and launches.
#include <algorithm>
#include <atomic>
#include <climits>
#include <cmath>

#include "attn_packed.hpp"
#include "launch_lds.hpp"
#include "../../include/flame_attn.h"

using namespace fattn;

namespace {

// [rows, heads, D] element strides: D stride 1, the others multiples of 8 (16-byte rows)
int check_rows(const void* base, const int64_t* st) {
    if (!base || !st) return FLAME_ATTN_ERR_INVALID;
    if (st[2] != 1) return FLAME_ATTN_ERR_UNSUPPORTED;
    if ((st[0] | st[1]) & 7) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (st[0] < 0 || st[1] < 0 || st[0] >= (int64_t(1) << 24)) return FLAME_ATTN_ERR_UNSUPPORTED;   // row offsets inside a tile are kept in 32 bits
    if (reinterpret_cast<uintptr_t>(base) & 15u) return FLAME_ATTN_ERR_UNSUPPORTED;
    return FLAME_ATTN_OK;
}
Strides rows_of(const int64_t* st) { return Strides{0, st[1], st[0]}; }

// an output whose rows or heads lie on each other would be written by several workgroups at once
bool overlaps(const int64_t* st, int rows, int heads, int D) {
    const int64_t n = st[0], h = st[1];
    if ((rows > 1 && n < D) || (heads > 1 && h < D)) return true;
    if (rows == 1 || heads == 1) return false;
    return n >= h ? n < h * (heads - 1) + D : h < n * (rows - 1) + D;
}

template <class P>
int launch(void (*kern)(P, PackedArgs), int lds, std::atomic<uint64_t>& done, int64_t units, int heads, const P& p, const PackedArgs& a, hipStream_t s, int threads = 256) {
    if (const int rc = set_lds_of_device(reinterpret_cast<const void*>(kern), lds, done)) return rc;
    hipLaunchKernelGGL(kern, dim3((unsigned)(units * heads)), dim3(threads), (size_t)lds, s, p, a);
    return (int)hipGetLastError();
}
template <class P>
int launch_merge(void (*kern)(P, PackedArgs), int64_t tiles, int heads, int blocks, const P& p, const PackedArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(kern, dim3((unsigned)(tiles * heads), (unsigned)blocks), dim3(256), 0, s, p, a);
    return (int)hipGetLastError();
}

int padded(int D) { return D <= 64 ? 64 : D <= 96 ? 96 : 128; }
size_t align256(size_t x) { return (x + 255) / 256 * 256; }

// Rows of a tensor.  The kernels and the rules here count tiles and steps of up to 128 rows in 32 bits, from sums such as T + 127 and, under the
// causal flag, Sk + 255: a number of tiles that has become negative would be a place in front of the tensor.
constexpr int kMostRows = INT32_MAX - 1023;
// ... and a launch has fewer than 2^32 threads: 256 for every tile of every head
bool grid_fits(int rows, int n_seqs, int heads) { return (double)packed_slots(rows, n_seqs, 128) * heads * 256.0 <= (double)UINT32_MAX; }

// Two workgroups of queries per compute unit, one of keys (at D = 64 a second one fits).  The backward's steps are longer, so shorter parts pay
// there (at least 16 steps each -> 8, us: 8 heads on 2 of 612 65 -> 51, 4 of 2000 72 -> 58, D = 64, 4 of 2000 50 -> 42; forward, 8 of 100 rows on 30000 keys
// 37 -> 46).
constexpr PackedCut kCutFwd{9, 16, 16, 1.6f}, kCutDq{9, 8, 12, 1.6f};
PackedCut cut_dkdv(int D) { return PackedCut{8, 8, 12, D <= 64 ? 0.65f : 1.6f}; }
// Whether a problem gets room for walks in parts, which the device then cuts or not by the lengths (PackedCut): not where whole walks fill the
// 256 compute units one and a half times, nor where the mean walk is short, nor where no lengths of these sums would be cut (the fewest
// steps: a causal self-attention's), nor of more than 64 sequences.  The mean stands for the longest walk, which the host does not know: one
// long sequence among many short ones stays whole (us, D = 128, causal; 4 heads of 8192: forward 88, with 8 of 50 rows 117; on 2 key heads, backward 265,
// with 8 of 50 267, with 31 of 50 439; one head of 8000, backward 112, with 15 of 10 285).
// (Whole -> in parts, us, D = 128.  Forward: 4 heads of 8192 117 -> 88, 32 of 128 rows on 8192 keys 115 -> 32, 8 of 100 rows on 30000 400 -> 37.  Backward: 4 of
// 1024 53 -> 48, 8 on 2 of 612 67 -> 52, of 2000 207 -> 82, 4 on 2 of 8192 439 -> 263.  Left whole: 24 of 1200 23 and 64, in parts 35 and 94.)
bool parts_pay(const PackedCut& cut, int64_t slots, int heads, int n_seqs, int walked_rows) {
    if (n_seqs > 64 || walked_rows / n_seqs < 64 * cut.gain || slots * heads * 2 >= 3 << PackedCut::kUnits_log2) return false;
    return cut.pays((walked_rows + 63) / 64, (slots - n_seqs) * heads * (walked_rows / n_seqs / 128));
}

struct Parts {
    int64_t slots, units;          // per head: tiles, and units at most
    PackedCut cut;
    size_t bytes;                  // of the units' sums
};
Parts whole(int64_t slots) { return Parts{slots, slots, PackedCut{0, 0, 0, 0.f}, 0}; }
Parts parts_of(const PackedCut& cut, int tile_rows, int walked_rows, int n_seqs, int heads, size_t unit_bytes) {
    Parts z = whole(packed_slots(tile_rows, n_seqs, 128));
    if (parts_pay(cut, z.slots, heads, n_seqs, walked_rows)) {
        z.cut = cut;
        z.units = cut.most(z.slots, heads);
        z.bytes = align256((size_t)z.units * heads * unit_bytes);
    }
    return z;
}
// Workgroups of 32 queries whose wavefronts share the keys, in place of 128 queries per workgroup: where two fit a compute unit, or four at D = 64, all
// at once, the second half of them for walks that are not the shortest; and where walks are not so long that parts of them (above) are better, for
// which all keys stand up to three sequences and four times the mean beyond: one long walk among many short ones passes, too (one head of 8000 43 us, with
// 15 of 10 rows 61).
// (128 queries -> 32, us.  D = 128: 24 heads of 77 7.7 -> 6.5, 4 of 1024 19.7 -> 12.8, 4 of 2000 25.6 -> 18.5, 8 of 1200 24.5 -> 17.6, 16 of four pieces of 100 on
// 900 keys 19.5 -> 14.9; beyond: 24 of 1024 21.5 -> 26.1, 32 of 700 15.7 -> 21.0, 8 of 4000 53.5 -> 60; short: 24 of eight times 32 6.9 -> 7.4.  D = 64: 8 of 612 11.3 -> 7.8, 12 of
// 2000 24.3 -> 18.4, 16 of 2000 26.9 -> 20.2; beyond: 24 of 2000 25.6 -> 29.7.  8 heads of 100 on 4000 keys: 23.6 -> 25.5, D = 64 18.6 -> 17.9.)
bool keyshare_pays(int n_seqs, int T_q, int T_kv, int H, int D) {
    const int64_t grid = packed_slots(T_q, n_seqs, 32) * H, most = D <= 64 ? 1024 : 512;
    return grid <= (T_kv / n_seqs >= 256 ? most : most / 2) && (n_seqs < 4 ? T_kv : 4 * (int64_t)T_kv / n_seqs) <= 4096;
}
// ... eight wavefronts while a compute unit gets one workgroup at most (two at D = 64 with long walks), else four
bool keyshare_wide(int n_seqs, int T_q, int T_kv, int H, int D) {
    const int64_t grid = packed_slots(T_q, n_seqs, 32) * H;
    return grid <= 256 || (D <= 64 && grid <= 512 && T_kv / n_seqs >= 2048);
}
Parts fwd_parts(int n_seqs, int T_q, int T_kv, int H, int D) {
    if (keyshare_pays(n_seqs, T_q, T_kv, H, D)) return whole(packed_slots(T_q, n_seqs, 32));
    return parts_of(kCutFwd, T_q, T_kv, n_seqs, H, (size_t)128 * (padded(D) * sizeof(float) + sizeof(f32x2)));
}
Parts dq_parts(int n_seqs, int T_q, int T_kv, int H, int D) { return parts_of(kCutDq, T_q, T_kv, n_seqs, H, (size_t)128 * padded(D) * sizeof(float)); }
Parts dkdv_parts(int n_seqs, int T_q, int T_kv, int H, int H_kv, int D) {
    return parts_of(cut_dkdv(D), T_kv, (int)std::min<int64_t>((int64_t)T_q * (H / H_kv), kMostRows), n_seqs, H_kv, (size_t)2 * 128 * padded(D) * sizeof(float));
}

// One launch for the sums of the parts: with few tiles a workgroup per eight columns, with more one per 32.  (Per 32 -> per eight, us: 8 tiles of 30
// parts each 45.8 -> 37.0, backward, D = 64, 8 heads on 2 of 1024 47.5 -> 43.8; 192 tiles of two or three parts 39.9 -> 44.7.)
template <class P>
int merge_parts_of(const Parts& z, int heads, int D, void (*eight)(P, PackedArgs), void (*wide)(P, PackedArgs), const P& p, const PackedArgs& a, hipStream_t s) {
    if (!z.cut.room_log2) return FLAME_ATTN_OK;
    return z.slots * heads <= 96 ? launch_merge(eight, z.slots, heads, D / 8, p, a, s) : launch_merge(wide, z.slots, heads, D / 32, p, a, s);
}

template <int D>
int launch_fwd(FwdParams p, PackedArgs a, void* workspace, size_t bytes, hipStream_t s) {
    static std::atomic<uint64_t> done{0}, done4{0}, done8{0};
    if (keyshare_pays(a.n, a.total_q, a.total_k, a.H, D)) {
        const int64_t slots = packed_slots(a.total_q, a.n, 32);
        return keyshare_wide(a.n, a.total_q, a.total_k, a.H, D)
                   ? launch(fwd_packed_keyshare_kernel<D, 8>, FwdKeyShareTile<D, 8>::LDS_BYTES, done8, slots, a.H, p, a, s, 512)
                   : launch(fwd_packed_keyshare_kernel<D, 4>, FwdKeyShareTile<D, 4>::LDS_BYTES, done4, slots, a.H, p, a, s);
    }
    Parts z = fwd_parts(a.n, a.total_q, a.total_k, a.H, D);
    if (!workspace || bytes < z.bytes) z = whole(z.slots);
    a.cut = z.cut;
    p.part_o = static_cast<float*>(workspace);
    p.part_lse = p.part_o + z.units * a.H * 128 * D;
    if (const int rc = launch(fwd_packed_kernel<D>, FwdTile<D>::LDS_BYTES + FwdTile<D>::q_pass_bytes(4), done, z.units, a.H, p, a, s)) return rc;
    return merge_parts_of(z, a.H, D, fwd_packed_merge_kernel<D, 1>, fwd_packed_merge_kernel<D, 4>, p, a, s);
}

template <int D>
int launch_bwd(BwdParams p, PackedArgs a, size_t part_bytes, hipStream_t s) {
    static std::atomic<uint64_t> done_q{0}, done_kv{0};
    Parts q = dq_parts(a.n, a.total_q, a.total_k, a.H, D), kv = dkdv_parts(a.n, a.total_q, a.total_k, a.H, a.Hkv, D);
    if (part_bytes < std::max(q.bytes, kv.bytes)) q = whole(q.slots), kv = whole(kv.slots);
    a.cut = q.cut;
    if (const int rc = launch(bwd_dq_packed_kernel<D>, BwdDqTile<D>::LDS_BYTES, done_q, q.units, a.H, p, a, s)) return rc;
    if (const int rc = merge_parts_of(q, a.H, D, bwd_dq_packed_merge_kernel<D, 1>, bwd_dq_packed_merge_kernel<D, 4>, p, a, s)) return rc;
    a.cut = kv.cut;
    if (const int rc = launch(bwd_dkdv_packed_kernel<D>, BwdTile<D>::LDS_BYTES, done_kv, kv.units, a.Hkv, p, a, s)) return rc;
    return merge_parts_of(kv, a.Hkv, D, bwd_dkdv_packed_merge_kernel<D, 1>, bwd_dkdv_packed_merge_kernel<D, 4>, p, a, s);
}

bool head_dim_ok(int D) { return D > 0 && D % 8 == 0 && D <= 128; }
size_t bwd_rows_bytes(int H, int T_q) { return 2 * align256((size_t)H * T_q * sizeof(float)); }

int check_sizes(const void* cu_q, const void* cu_k, int n_seqs, int T_q, int T_kv, int H, int H_kv, int D, float scale) {
    if (!cu_q || !cu_k || n_seqs <= 0 || T_q <= 0 || T_kv <= 0 || H <= 0 || H_kv <= 0 || D <= 0) return FLAME_ATTN_ERR_INVALID;
    if (H % H_kv != 0 || !(scale > 0.f) || !std::isfinite(scale)) return FLAME_ATTN_ERR_INVALID;
    return head_dim_ok(D) && T_q <= kMostRows && T_kv <= kMostRows && grid_fits(T_q, n_seqs, H) ? FLAME_ATTN_OK : FLAME_ATTN_ERR_UNSUPPORTED;
}

}  // namespace

extern "C" {

size_t flame_attn_packed_fwd_workspace_bytes(int n_seqs, int T_q, int T_kv, int H, int D) {
    if (n_seqs <= 0 || T_q <= 0 || T_kv <= 0 || T_q > kMostRows || T_kv > kMostRows || H <= 0 || !head_dim_ok(D)) return 0;
    return fwd_parts(n_seqs, T_q, T_kv, H, D).bytes;
}

int flame_attn_packed_fwd_bf16(const void* Q, const void* K, const void* V, void* O, void* LSE, const int32_t* cu_q, const int32_t* cu_k,
                               int n_seqs, int T_q, int T_kv, int H, int H_kv, int D, float scale, const int64_t* q_strides,
                               const int64_t* k_strides, const int64_t* v_strides, const int64_t* o_strides, int causal, void* workspace,
                               size_t workspace_bytes, void* stream) {
    int rc;
    if ((rc = check_sizes(cu_q, cu_k, n_seqs, T_q, T_kv, H, H_kv, D, scale))) return rc;
    if ((rc = check_rows(Q, q_strides)) || (rc = check_rows(K, k_strides)) || (rc = check_rows(V, v_strides)) || (rc = check_rows(O, o_strides))) return rc;
    if (overlaps(o_strides, T_q, H, D) || (reinterpret_cast<uintptr_t>(workspace) & 15u)) return FLAME_ATTN_ERR_UNSUPPORTED;
    FwdParams p{};
    p.q = static_cast<const uint16_t*>(Q);
    p.k = static_cast<const uint16_t*>(K);
    p.v = static_cast<const uint16_t*>(V);
    p.o = static_cast<uint16_t*>(O);
    p.lse = static_cast<float*>(LSE);
    p.qs = rows_of(q_strides); p.ks = rows_of(k_strides); p.vs = rows_of(v_strides); p.os = rows_of(o_strides);
    p.d = p.dv = D;
    p.scale = scale;
    p.m.causal = causal ? 1 : 0;
    const PackedArgs a{cu_q, cu_k, n_seqs, T_q, T_kv, H, H_kv, p.m.causal, PackedCut{0, 0, 0, 0.f}};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return D <= 64 ? launch_fwd<64>(p, a, workspace, workspace_bytes, s)
                   : D <= 96 ? launch_fwd<96>(p, a, workspace, workspace_bytes, s) : launch_fwd<128>(p, a, workspace, workspace_bytes, s);
}

size_t flame_attn_packed_bwd_workspace_bytes(int n_seqs, int T_q, int T_kv, int H, int H_kv, int D) {
    if (n_seqs <= 0 || T_q <= 0 || T_kv <= 0 || T_q > kMostRows || T_kv > kMostRows || H <= 0 || H_kv <= 0 || H % H_kv != 0 || !head_dim_ok(D)) return 0;
    return bwd_rows_bytes(H, T_q) + std::max(dq_parts(n_seqs, T_q, T_kv, H, D).bytes, dkdv_parts(n_seqs, T_q, T_kv, H, H_kv, D).bytes);
}

int flame_attn_packed_bwd_bf16(const void* Q, const void* K, const void* V, const void* O, const void* dO, const void* LSE, void* dQ, void* dK,
                               void* dV, const int32_t* cu_q, const int32_t* cu_k, int n_seqs, int T_q, int T_kv, int H, int H_kv, int D,
                               float scale, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                               const int64_t* o_strides, const int64_t* do_strides, const int64_t* dq_strides, const int64_t* dk_strides,
                               const int64_t* dv_strides, int causal, void* workspace, size_t workspace_bytes, void* stream) {
    int rc;
    if ((rc = check_sizes(cu_q, cu_k, n_seqs, T_q, T_kv, H, H_kv, D, scale))) return rc;
    if (!grid_fits(T_kv, n_seqs, H_kv)) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (!LSE || !workspace || workspace_bytes < bwd_rows_bytes(H, T_q)) return FLAME_ATTN_ERR_INVALID;
    if (reinterpret_cast<uintptr_t>(workspace) & 15u) return FLAME_ATTN_ERR_UNSUPPORTED;
    if ((rc = check_rows(Q, q_strides)) || (rc = check_rows(K, k_strides)) || (rc = check_rows(V, v_strides)) || (rc = check_rows(O, o_strides)) ||
        (rc = check_rows(dO, do_strides)) || (rc = check_rows(dQ, dq_strides)) || (rc = check_rows(dK, dk_strides)) || (rc = check_rows(dV, dv_strides)))
        return rc;
    if (overlaps(dq_strides, T_q, H, D) || overlaps(dk_strides, T_kv, H_kv, D) || overlaps(dv_strides, T_kv, H_kv, D)) return FLAME_ATTN_ERR_UNSUPPORTED;
    BwdParams p{};
    p.q = static_cast<const uint16_t*>(Q);
    p.k = static_cast<const uint16_t*>(K);
    p.v = static_cast<const uint16_t*>(V);
    p.o = static_cast<const uint16_t*>(O);
    p.dout = static_cast<const uint16_t*>(dO);
    p.lse = static_cast<const float*>(LSE);
    p.dq = static_cast<uint16_t*>(dQ);
    p.dk = static_cast<uint16_t*>(dK);
    p.dv = static_cast<uint16_t*>(dV);
    p.ndelta = static_cast<float*>(workspace);
    p.lse2 = reinterpret_cast<float*>(static_cast<char*>(workspace) + bwd_rows_bytes(H, T_q) / 2);
    p.split_ws = reinterpret_cast<float*>(static_cast<char*>(workspace) + bwd_rows_bytes(H, T_q));
    const size_t part_bytes = workspace_bytes - bwd_rows_bytes(H, T_q);
    p.qs = rows_of(q_strides); p.ks = rows_of(k_strides); p.vs = rows_of(v_strides); p.os = rows_of(o_strides);
    p.dos = rows_of(do_strides); p.dqs = rows_of(dq_strides); p.dks = rows_of(dk_strides); p.dvs = rows_of(dv_strides);
    p.d = D;
    p.scale = scale;
    p.m.causal = causal ? 1 : 0;
    const PackedArgs a{cu_q, cu_k, n_seqs, T_q, T_kv, H, H_kv, p.m.causal, PackedCut{0, 0, 0, 0.f}};
    hipStream_t s = static_cast<hipStream_t>(stream);
    return D <= 64 ? launch_bwd<64>(p, a, part_bytes, s) : D <= 96 ? launch_bwd<96>(p, a, part_bytes, s) : launch_bwd<128>(p, a, part_bytes, s);
}

}  // extern "C"
