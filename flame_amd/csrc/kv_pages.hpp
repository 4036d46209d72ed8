// Moves of keys and values between rows and the pages of a cache: nothing but memory traffic, 16 bytes per lane and access.
#pragma once
#include "attn_common.hpp"
#include "packed_units.hpp"

namespace fattn {

struct KvStoreParams {
    const uint16_t* k;             // [rows][Hkv][d] through ks, vs (n: row, h: head)
    const uint16_t* v;
    uint16_t* kc;                  // [pages][Hkv][page][d] through kcs, vcs (b: page, h: head, n: token)
    uint16_t* vc;
    const int32_t* table;
    int64_t table_stride;
    int table_pages;
    const int32_t* cu;             // [n + 1]: rows of the sequences
    const int32_t* start;          // [n]: place of a sequence's first row in its pages
    Strides ks, vs, kcs, vcs;
    int n, rows, Hkv, d, n_pages, page_shift;
    int rows_per_wave;
};

// A wavefront takes one row, all heads of K and V, or as many rows as make 64 granules of 16 bytes.  A row whose place lies outside its
// sequence's pages, or on a page outside the cache, is left out.
// Bound by memory: 32768 rows of 8 heads, D = 128, 41 us, 6.5 TB/s of what is read and written (with eight rows one behind the other in
// a wavefront 48: the search is short against the latency of a row's chain of table and copy); 65536 rows of one
// head, D = 64, 6.7 us, 5.0 TB/s (with a row per wavefront 28).
static __global__ __launch_bounds__(256) void kv_store_kernel(const KvStoreParams p) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int r0 = ((int)blockIdx.x * 4 + wave) * p.rows_per_wave;
    if (r0 >= p.rows) return;
    const int last = packed_find(p.n, r0, [&](int at) { return packed_bound(p.cu, at, p.rows); });      // sequence that begins at or before r0
    const int per_row = p.d / 8, n = p.Hkv * per_row, together = min(n, 64), sub = lane / together, r = r0 + sub;
    if (sub >= p.rows_per_wave || r >= p.rows) return;
    int b = last;
    while (b < p.n && packed_bound(p.cu, b + 1, p.rows) <= r) ++b;
    if (b >= p.n) return;                              // behind the last sequence
    const int64_t pos = (int64_t)p.start[b] + (r - packed_bound(p.cu, b, p.rows));
    if (pos < 0 || (pos >> p.page_shift) >= p.table_pages) return;
    const int page = p.table[b * p.table_stride + (pos >> p.page_shift)];
    if (page < 0 || page >= p.n_pages) return;
    const int64_t token = pos & ((1 << p.page_shift) - 1);
    uint16_t* const kd = p.kc + page * p.kcs.b + token * p.kcs.n;
    uint16_t* const vd = p.vc + page * p.vcs.b + token * p.vcs.n;
    const uint16_t* const ks = p.k + r * p.ks.n;
    const uint16_t* const vs = p.v + r * p.vs.n;
    for (int e = lane - sub * together; e < n; e += together) {
        const int h = e / per_row, c = 8 * (e - h * per_row);
        const u32x4 a = *reinterpret_cast<const u32x4*>(ks + h * p.ks.h + c);
        const u32x4 w = *reinterpret_cast<const u32x4*>(vs + h * p.vs.h + c);
        *reinterpret_cast<u32x4*>(kd + h * p.kcs.h + c) = a;
        *reinterpret_cast<u32x4*>(vd + h * p.vcs.h + c) = w;
    }
}

// Pairs of pages travel in the launch's own arguments: the host has checked them, and nothing has to be copied to the device first.
struct KvCopyPairs {
    static constexpr int kMost = 400;
    int32_t src[kMost], dst[kMost];
};
struct KvCopyParams {
    uint16_t* c[2];                // K and V: [layers][pages][Hkv][page][d]
    int64_t layer[2], page[2], head[2], token[2];      // element strides
    int layers, Hkv, page_size, d;
    int granules;                  // of 16 bytes in a page
    int chunks;                    // workgroups per page and tensor
    int contiguous;                // a page is one piece of memory in both tensors
};

constexpr int kKvCopyPerThread = 4;

// blockIdx.x: chunk of a page, of K or V; y: layer; z: pair.  Bound by memory: 600 pages of 16 tokens, 8 heads, D = 128 in 24 layers 386 us,
// 4.9 TB/s of what is read and written, as fast as a large copy.  Four granules per thread are requested before the first is stored.
static __global__ __launch_bounds__(256) void kv_copy_kernel(const KvCopyParams p, const KvCopyPairs pairs) {
    const int which = (int)blockIdx.x / p.chunks, chunk = (int)blockIdx.x - which * p.chunks;
    uint16_t* const layer = p.c[which] + (int)blockIdx.y * p.layer[which];
    const uint16_t* const from = layer + pairs.src[blockIdx.z] * p.page[which];
    uint16_t* const to = layer + pairs.dst[blockIdx.z] * p.page[which];
    const int g0 = chunk * 256 * kKvCopyPerThread + (int)threadIdx.x;
    int64_t at[kKvCopyPerThread];
    u32x4 w[kKvCopyPerThread];
#pragma unroll
    for (int i = 0; i < kKvCopyPerThread; ++i) {
        const int g = g0 + 256 * i;
        if (p.contiguous) {
            at[i] = (int64_t)g * 8;
        } else {
            const int per_row = p.d / 8, row = g / per_row, h = row / p.page_size;
            at[i] = h * p.head[which] + (row - h * p.page_size) * p.token[which] + 8 * (g - row * per_row);
        }
        if (g < p.granules) w[i] = *reinterpret_cast<const u32x4*>(from + at[i]);
    }
#pragma unroll
    for (int i = 0; i < kKvCopyPerThread; ++i)
        if (g0 + 256 * i < p.granules) *reinterpret_cast<u32x4*>(to + at[i]) = w[i];
}

}  // namespace fattn
