// Attention of one or a few new tokens per sequence over a paged cache of keys and values, with a prefix that all sequences of the
// batch share or without.
//
// A sequence's keys are the prefix's and its own; the softmax is taken over both.  The keys are cut into units of a few tiles each:
// a unit of the prefix serves 128 rows (sequence, new token, head) of one key head at a time, whichever sequences they are of, so
// that the prefix is read once for the batch and not once per sequence; a unit of a sequence's own keys serves the rows of that
// sequence.  Every unit leaves O' = sum_j exp2(s_j - m) v_j, m = max_j s_j and l = sum_j exp2(s_j - m) of its keys (s in units of
// log 2, all in fp32), and the merge kernel joins them:  M = max m,  O = sum exp2(m - M) O' / sum exp2(m - M) l.
//
// What bounds the own keys is memory: each key and value is read once and meets a row of at most 32 queries, 4 * 32 operations per 4
// bytes.  So the four wavefronts of a workgroup each walk keys of their own: no barrier in the walk, no wavefront waits for another's
// copies; two workgroups per compute unit.  A wavefront owns one K and one V tile of 32 keys in LDS and requests the next K tile as
// soon as the fragments of the present one are in registers, V likewise, so that one of the two is always on its way.
// What bounds the prefix of a large batch is the way from L2: read by every 32 rows for themselves (as the own keys are) it moved at
// 13 TB/s and no faster.  So there the four wavefronts have 32 rows each and share the tiles, of which four are in LDS; what is left is
// the issue of one wavefront per SIMD, 0.75 us a tile.
// Measured, D = 128, 32 heads on 8: 64 sequences of 4000 keys 189 us, 5.5 TB/s, 256 of 4000 700 us, 6.0 TB/s, one of 131072 104 us, 5.2 TB/s, 8 of 32000
// 187 us, 5.6 TB/s; 64 of 1 to 509 keys on a prefix of 8192 38.5 us.  (Reads alone reach 5.7 TB/s on this card, more from its last level of cache.)
//
// The number of keys is known on the device only.  The units are therefore cut there: every workgroup sums the tiles of the batch
// and takes the unit length that gives about as many units as the device holds workgroups.
// Short tables (paged_direct_kernel) need none of this: one workgroup per sequence, key head and 32 rows takes all keys and writes O itself.
#pragma once
#include "attn_common.hpp"
#include "packed_units.hpp"

namespace fattn {

struct PagedParams {
    const uint16_t* q;
    const uint16_t* k;             // cache: [pages][Hkv][page][D] through ks, vs (b: page, h: head, n: token)
    const uint16_t* v;
    uint16_t* o;
    float* lse;                    // [B * H, N] or null
    const int32_t* table;          // pages of every sequence's own keys
    int64_t table_stride;
    int table_pages;               // entries of a row
    const int32_t* kv_len;         // [B]: own keys
    const int32_t* prefix_table;   // or null
    const int32_t* prefix_len;     // one number, or null
    int prefix_pages;
    Strides qs, ks, vs, os;
    int B, H, Hkv, N;
    int n_pages;                   // of the cache
    int page_shift;                // log2 of the tokens in a page (at least 4)
    int d;                         // head dim: a multiple of 8, at most the compiled D
    float scale;
    int64_t own_slot;              // rows of the partial results that the prefix has (a host bound); the own ones follow
    float* part_o;                 // [row][d]
    f32x2* part_ml;                // m and l of every row
    // [B] first unit and units per (head, row tile) of a sequence, then the splits of the prefix; with ranges of tiles: [B] first tile and
    // tiles per (head, row tile), then the tiles of a range
    int2* plan;
};

// How the keys are cut.  A walk (one sequence, key head and tile of rows, or the prefix in place of the sequence) has a tile for every 32 keys; a
// unit of fewer than kLeast tiles would leave wavefronts without work.
//   Fewer walks than half of the kFill workgroups that run at once: units so long that all of them run at once, the last one of every walk
//   taking a place whatever is left for it.  (Against units of 32 tiles, some to a second round, us: 8 sequences of 16k to 40k keys,
//   4 key heads, D = 128 105 -> 97; 16 of 500 to 5000, 8 key heads 46 -> 40.)
//   More: whole walks up to kLong tiles, as a unit's start costs what about ten tiles do; longer ones in even units, kMany in all.
//   (64 sequences of 2000 101 -> 97, 256 of 400 to 4000 439 -> 402, 64 of 1600 to 16000 416 -> 404; 48 of 1500 to 3000 91 -> 104.)
// The prefix of more than 64 rows has units of 128 rows, up to kShared of them, with at least kSharedMost tiles each once there are half as
// many: the partial results of a unit's rows weigh as much as two tiles.  (One key head with 512 rows on 4096 keys, D = 64, at kSharedMost
// tiles throughout 21.8 us, so 16.5.  Rows or keys apart, 8 key heads, prefix of 8192: 96 rows each 29.5 and 35.2 us, 48 rows 28.2 and 24.8.)
struct PagedCut {
    static constexpr int kTile = 32, kLeast = 4, kFill = 512, kMany = 2048, kLong = 64, kShared = 256, kSharedMost = 16;
    // tiles per unit for `total` tiles of `walks` walks
    static __host__ __device__ int places(int walks) { return walks < kFill / 2 ? kFill - walks : walks < kMany - kFill / 2 ? kMany - walks : kFill / 2; }
    static __host__ __device__ int least(int walks) { return walks < kFill / 2 ? kLeast : kLong; }
    static __host__ __device__ int unit(int total, int walks) {
        const int n = (total + places(walks) - 1) / places(walks);
        return n < least(walks) ? least(walks) : (n + kLeast - 1) / kLeast * kLeast;       // (no tiles: a divisor all the same)
    }
    // tiles per unit of a walk of `tiles` tiles, at most `unit`, and how many units that makes
    static __host__ __device__ int even(int tiles, int unit, int walks) {
        if (walks < kFill / 2 || tiles <= unit) return unit;
        const int n = (tiles + unit - 1) / unit, each = (tiles + n - 1) / n;
        return (each + kLeast - 1) / kLeast * kLeast;
    }
    static __host__ __device__ int splits(int tiles, int unit, int walks) { return (tiles + even(tiles, unit, walks) - 1) / even(tiles, unit, walks); }
    static __host__ __device__ int shared_unit(int total) {
        const int n = (total + kShared - 1) / kShared, half = 2 * n < kSharedMost ? 2 * n : kSharedMost;
        return n > half ? n : half < kLeast ? kLeast : half;
    }
    // rows of a prefix unit: of up to 64 rows the wavefronts take the keys apart, not the rows
    static __host__ __device__ bool shared(int rows) { return rows > 64; }
    static __host__ __device__ int row_tiles(int rows) { return (rows + kTile - 1) / kTile; }
    static __host__ __device__ int prefix_row_tiles(int rows) { return shared(rows) ? (rows + 127) / 128 : row_tiles(rows); }
    static __host__ __device__ int prefix_tile_rows(int rows) { return shared(rows) ? 128 : 32; }
};

template <int D>
struct PagedTile {
    static constexpr int BN = 32;
    static constexpr int RS = kRowPitch<D>;
    static constexpr int TILE_ELEMS = BN * RS;
    static constexpr int WAVE_ELEMS = 2 * TILE_ELEMS;              // one K and one V tile, or the 32 x D fp32 sums at the end
    static constexpr int lds_bytes(int nw) { return nw * WAVE_ELEMS * 2; }
    static constexpr int NDMA = BN * RS * 2 / 1024;                // copies per tile
    static constexpr int RPD = 1024 / (RS * 2);                    // rows per copy
};

// dynamic LDS of a workgroup of nw wavefronts
template <int D>
constexpr int paged_lds_bytes(const PagedParams*, int nw) { return PagedTile<D>::lds_bytes(nw); }

// This wavefront's reads of LDS have returned and none moves to behind this: a copy may overwrite what they read.
__device__ __forceinline__ void lds_reads_done() {
    asm volatile("" ::: "memory");
    wait_lds_reads<0>();
    asm volatile("" ::: "memory");
}

// keys of sequence b, none where its number is negative; more than its pages hold is reported by `bad`
__device__ __forceinline__ int paged_len(const PagedParams& p, int b, bool& bad) {
    const int n = max(p.kv_len[b], 0), most = p.table_pages << p.page_shift;
    bad = n > most;
    return min(n, most);
}
__device__ __forceinline__ int paged_prefix_len(const PagedParams& p, bool& bad) {
    bad = false;
    if (!p.prefix_len) return 0;
    const int n = max(p.prefix_len[0], 0), most = p.prefix_pages << p.page_shift;
    bad = n > most;
    return min(n, most);
}
__device__ __forceinline__ int paged_tiles(int keys) { return (keys + PagedCut::kTile - 1) / PagedCut::kTile; }

// The cut of the whole batch.  Own units are numbered sequence by sequence: first + (head, row tile) * splits + split.
struct PagedPlan {
    int prefix_keys, prefix_tiles, prefix_unit, prefix_splits, prefix_units;   // keys, tiles, tiles per unit, units per row tile and head, all units
    bool prefix_bad;
    int own_tiles, own_unit;       // of all walks together, tiles per unit
    int len;                       // raw number of keys of sequence `tid`
};
// Every thread of the workgroup (256) calls this; `sums` is 4 ints of LDS.
__device__ __forceinline__ PagedPlan paged_plan(const PagedParams& p, int* sums) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, most = p.table_pages << p.page_shift;
    PagedPlan c;
    c.len = tid < p.B ? p.kv_len[tid] : 0;
    c.prefix_keys = packed_uniform(paged_prefix_len(p, c.prefix_bad));
    int tiles = paged_tiles(min(max(c.len, 0), most));
    for (int b = tid + 256; b < p.B; b += 256) {
        bool bad;
        tiles += paged_tiles(paged_len(p, b, bad));
    }
    tiles = wave_scan(tiles);
    if (lane == 63) sums[wave] = tiles;
    __syncthreads();
    const int rows = p.N * (p.H / p.Hkv);
    const int heads = p.Hkv * PagedCut::row_tiles(rows), own = packed_uniform(sums[0] + sums[1] + sums[2] + sums[3]) * heads;
    c.own_tiles = own;
    c.own_unit = packed_uniform(PagedCut::unit(own, p.B * heads));
    c.prefix_tiles = paged_tiles(c.prefix_keys);
    const int all = p.B * rows, per_split = p.Hkv * PagedCut::prefix_row_tiles(all), total = c.prefix_tiles * per_split;
    c.prefix_unit = PagedCut::shared(all) ? PagedCut::shared_unit(total) : PagedCut::unit(total, per_split);
    c.prefix_splits = packed_uniform((c.prefix_tiles + c.prefix_unit - 1) / c.prefix_unit);
    c.prefix_units = c.prefix_splits * per_split;
    return c;
}

// Walks the sequences in the order of their units, units_of(tiles) for every row tile and head, and calls take(b, raw keys, first unit, units per row
// tile and head) in the one thread that has sequence b, for every b (the threads of a workgroup take 256 sequences at a time).  `sums`: 4 ints
// of LDS.
template <class N, class F>
__device__ __forceinline__ void paged_own_units(const PagedParams& p, const PagedPlan& c, int* sums, N&& units_of, F&& take) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, most = p.table_pages << p.page_shift;
    const int per_split = p.Hkv * PagedCut::row_tiles(p.N * (p.H / p.Hkv));
    int before = 0;
    for (int b0 = 0; b0 < p.B; b0 += 256) {
        const int b = b0 + tid;
        const int len = b0 == 0 ? c.len : b < p.B ? p.kv_len[b] : 0;
        const int splits = units_of(paged_tiles(min(max(len, 0), most)));
        const int through = wave_scan(splits * per_split);
        __syncthreads();                               // the sums are free
        if (lane == 63) sums[wave] = through;
        __syncthreads();
        int first = before + through - splits * per_split;
        for (int w = 0; w < wave; ++w) first += sums[w];
        if (b < p.B) take(b, len, first, splits);
        before += sums[0] + sums[1] + sums[2] + sums[3];
    }
}

struct PagedUnit {
    const int32_t* table;      // of the keys' pages
    int entries;               // of the table
    int rows;                  // of this unit's row tile, at most 32 (a prefix unit of shared tiles: 128)
    int row0;                  // its first row: (sequence in the batch for the prefix, new token, head) of the key head
    int kv_head;
    int b0;                    // sequence of row 0 of the key head
    int keys;                  // all keys of the walk's sequence (or the prefix)
    int tile0, tiles;          // this unit's share
    int lag;                   // row (token i) attends to keys j < keys - lag + i, at least none; the prefix: to all
    bool own;
};

struct PagedRow {              // of a unit: sequence, token and head
    int b, i, h;
};
__device__ __forceinline__ PagedRow paged_row(const PagedParams& p, const PagedUnit& u, int r) {
    const int G = p.H / p.Hkv, per_b = p.N * G, row = u.row0 + r;
    const int b = row / per_b, rest = row - b * per_b, i = rest / G;
    return {u.b0 + b, i, u.kv_head * G + rest - i * G};
}

// This thread's number in its workgroup, not known to be the same from unit to unit: what follows from it is formed for every unit, where
// the compiler would keep what all kinds of units need in registers through the loop over them (19 registers went to scratch memory).
__device__ __forceinline__ int paged_thread() {
    int t = threadIdx.x;
    asm volatile("" : "+v"(t));
    return t;
}

// The pages of a walk: a lane holds the page of 1 << page_shift keys, 64 pages at a time.
struct PagedPages {
    int first = 0, mine = 0;
    bool bad = false;          // a page that the walk needs lies outside the cache
    __device__ __forceinline__ void load(const PagedParams& p, const PagedUnit& u, int lane, int from) {
        const int at = from + lane;
        int e = at < u.entries ? u.table[at] : 0;
        const bool outside = e < 0 || e >= p.n_pages;
        bad |= outside && at <= ((u.keys - 1) >> p.page_shift);
        first = from;
        mine = outside ? 0 : e;
    }
    __device__ __forceinline__ bool holds(const PagedParams& p, int key) const { return (key >> p.page_shift) - first < 64; }
    // first of the 16 rows (tokens) from `key` on, a multiple of 16: these always lie in one page
    __device__ __forceinline__ int64_t rows16(const PagedParams& p, int key, const Strides& st) const {
        return __builtin_amdgcn_readlane(mine, (key >> p.page_shift) - first) * st.b + (key & ((1 << p.page_shift) - 1)) * st.n;
    }
};

// N of a tile's NDMA copies of 1 KiB to LDS: all, or those from i0 on, a wavefront's share, which lie in one half of 16 rows.  `off`: bytes of
// a lane within 16 rows, of every copy of 16 rows or of the share's.  Rows past the last key (`most` of the tile) re-read it.
template <int D, int N>
__device__ __forceinline__ void paged_copy(const PagedParams& p, const PagedPages& pages, const uint16_t* base, const Strides& st,
                                           const uint32_t (&off)[N > PagedTile<D>::NDMA / 2 ? PagedTile<D>::NDMA / 2 : N], int lane, int key0, int most, int i0,
                                           uint32_t dst) {
    using T = PagedTile<D>;
    constexpr int HALF = T::NDMA / 2, GPR = T::RS / 8, EACH = N > HALF ? HALF : N;
#pragma unroll
    for (int g = 0; g < N / EACH; ++g) {
        const int half = N > HALF ? g : i0 / HALF, first = N > HALF ? 0 : i0 % HALF;
        const int from = 16 * half <= most ? half : 0;               // a half without a key: the last key is in the other one
        const uint16_t* const rows = base + pages.rows16(p, key0 + 16 * from, st);
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            uint32_t o = off[j];
            if (16 * half + 15 > most) {
                const int row = (first + j) * T::RPD + lane / GPR;
                o += 2u * (uint32_t)((min(16 * half + row, most) - 16 * from - row) * (int)st.n);
            }
            dma16u(rows, o, dst + 1024u * (uint32_t)(half * HALF + first + j));
        }
    }
}
// ... and `off`, for the copies of 16 rows from `first` on
template <int D, int EACH>
__device__ __forceinline__ void paged_offsets(const PagedParams& p, const Strides& st, int lane, int first, uint32_t (&off)[EACH]) {
    using T = PagedTile<D>;
    constexpr int GPR = T::RS / 8;
#pragma unroll
    for (int j = 0; j < EACH; ++j) {
        const int row = (first + j) * T::RPD + lane / GPR;           // (the swizzle of row + 16 is the same)
        off[j] = 2u * (uint32_t)(row * (int)st.n + src_granule(lane % GPR ^ swz<D>(row), p.d) * 8);
    }
}

// What a wavefront holds of 32 rows: their queries as MFMA fragments and the running softmax over the keys it has seen.
template <int D>
struct PagedRows {
    using T = PagedTile<D>;
    static constexpr int DC = D / 16, DB = D / 32, RS = T::RS;
    bf16x8 qf[DC];
    f32x16 oacc[DB];
    float m_run = -INFINITY, l_run = 0.f, c_log2, stale_ok;
    int koff[DC];              // K fragment: row n, logical granule 2 dc + h
    int voff[2][DB];           // V^T fragment halves: rows 4 h + r / 4 (+ 8), logical granule 4 db + 2 g16 + (r & 3) / 2

    // `at`: this lane's row, there: whether it exists
    __device__ __forceinline__ void begin(const PagedParams& p, int lane, const PagedRow& at, bool there) {
        const int n = lane & 31, h = lane >> 5, tr_r = lane & 15, tr_g16 = (lane >> 4) & 1;
        const uint16_t* const qrow = p.q + at.b * p.qs.b + at.h * p.qs.h + at.i * p.qs.n;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            qf[dc] = __builtin_bit_cast(bf16x8, ldg16(qrow + 16 * dc + 8 * h, there && 16 * dc + 8 * h < p.d));
            koff[dc] = n * RS + (((2 * dc + h) ^ swz<D>(n)) << 3);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int row = 4 * h + (tr_r >> 2) + 8 * half;
#pragma unroll
            for (int db = 0; db < DB; ++db) voff[half][db] = row * RS + (((4 * db + 2 * tr_g16 + ((tr_r & 3) >> 1)) ^ swz<D>(row)) << 3) + 4 * (tr_r & 1);
        }
        c_log2 = p.scale * kLog2e;
        stale_ok = stale_scope(c_log2);        // the reference maximum may lag the true one by 2^8
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[db][r] = 0.f;
    }
    __device__ __forceinline__ void read_k(bf16x8 (&kf)[DC], const uint16_t* tile) const {
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) kf[dc] = *reinterpret_cast<const bf16x8*>(tile + koff[dc]);
    }
    __device__ __forceinline__ void read_v(bf16x8 (&vf)[2 * DB], const uint16_t* tile) const {
#pragma unroll
        for (int i = 0; i < 2 * DB; ++i) {
            const int cc = i / DB, db = i % DB;
            const u32x2 lo = lds_read_tr16(tile + voff[0][db] + 16 * cc * RS), hi = lds_read_tr16(tile + voff[1][db] + 16 * cc * RS);
            const u32x4 w = {lo[0], lo[1], hi[0], hi[1]};
            vf[i] = __builtin_bit_cast(bf16x8, w);
        }
    }
    // S^T = K Q^T: a lane's row, 16 keys
    __device__ __forceinline__ f32x16 scores(const bf16x8 (&kf)[DC]) const {
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) s = mfma32(kf[dc], qf[dc], s);
        return s;
    }
    // keys of the tile from `limit` on are excluded
    static __device__ __forceinline__ void exclude(f32x16& s, int lane, int limit) {
        const int lim = limit - 4 * (lane >> 5);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 8 * (r >> 2) + (r & 3) >= lim ? -INFINITY : s[r];
    }
    // the maximum of a tile's scores joins the running one, which moves (and the sums are rescaled) only when it lags by more than 2^8
    __device__ __forceinline__ void fold(const f32x16& s) {
        float top = s[0];
#pragma unroll
        for (int r = 1; r < 16; ++r) top = fmaxf(top, s[r]);
        if (__any(top > m_run + stale_ok)) {
            top = max_of_halves(top);
            const float m_new = fmaxf(m_run, top), m_to = m_new == -INFINITY ? 0.f : m_new;
            const float alpha = exp2_fast((m_run - m_to) * c_log2);
            m_run = m_new;
            l_run *= alpha;
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int r = 0; r < 16; ++r) oacc[db][r] *= alpha;
        }
    }
    // exp2 of the scores against the running maximum; the weights meet V rounded to bf16 (the sum l is of the unrounded ones): the matrix
    // instructions take no wider operand
    __device__ __forceinline__ void weights(f32x16& s, bf16x8 (&pf)[2]) {
        const float shift = (m_run == -INFINITY ? 0.f : m_run) * c_log2;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(fmaf(s[r], c_log2, -shift));
            sum[r & 1] += s[r];
        }
        l_run += sum[0] + sum[1];
        pf[0] = pack8(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]);
        pf[1] = pack8(s[8], s[9], s[10], s[11], s[12], s[13], s[14], s[15]);
    }
    // 16 keys of a V tile straight from LDS
    __device__ __forceinline__ void add16(const uint16_t* tile, int cc, bf16x8 pf) {
        bf16x8 vf[DB];
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const u32x2 lo = lds_read_tr16(tile + voff[0][db] + 16 * cc * RS), hi = lds_read_tr16(tile + voff[1][db] + 16 * cc * RS);
            const u32x4 x = {lo[0], lo[1], hi[0], hi[1]};
            vf[db] = __builtin_bit_cast(bf16x8, x);
        }
#pragma unroll
        for (int db = 0; db < DB; ++db) oacc[db] = mfma32(vf[db], pf, oacc[db]);
    }
    __device__ __forceinline__ void add(const bf16x8 (&vf)[2 * DB], const bf16x8 (&pf)[2]) {
#pragma unroll
        for (int i = 0; i < 2 * DB; ++i) oacc[i % DB] = mfma32(vf[i], pf[i / DB], oacc[i % DB]);
    }
};

// The end of a unit whose wavefronts have walked keys of their own: their states become one, which is the result (direct) or goes to the
// merge.  `lds`: the tiles of the wavefronts, into which no copy is under way; `bad`: the rows are NaN.
template <int D, int NW>
__device__ __forceinline__ void paged_unit_join(const PagedParams& p, const PagedUnit& u, PagedRows<D>& w, float* lds, int tid, bool bad, bool direct,
                                                float* out_o, f32x2* out_ml) {
    constexpr int DB = D / 32, WAVE_FLOATS = PagedTile<D>::WAVE_ELEMS / 2;
    const int lane = tid & 63, wave = packed_uniform(tid >> 6), n = lane & 31, h = lane >> 5;
    w.l_run += xhalf(w.l_run);
    if (__any(bad)) w.l_run = __builtin_nanf("");    // a page outside the cache, or more keys than pages: NaN
    __shared__ f32x2 state[NW][32];
    if (h == 0) state[wave][n] = f32x2{w.m_run, w.l_run};
    __syncthreads();                                   // (no copy is under way: every wavefront has waited for its last one)
    float M = -INFINITY, L = 0.f;
#pragma unroll
    for (int i = 0; i < NW; ++i) M = fmaxf(M, state[i][n][0]);
    const float M_to = M == -INFINITY ? 0.f : M;
#pragma unroll
    for (int i = 0; i < NW; ++i) L += state[i][n][1] * exp2_fast((state[i][n][0] - M_to) * w.c_log2);
    const float f = exp2_fast((w.m_run - M_to) * w.c_log2);
    float* const sums = lds + wave * WAVE_FLOATS;       // [32][D], granules of four swizzled by the row
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x16& a = w.oacc[db];
            *reinterpret_cast<f32x4*>(sums + n * D + (((8 * db + 2 * g + h) ^ (n & 7)) << 2)) = f32x4{a[4 * g] * f, a[4 * g + 1] * f, a[4 * g + 2] * f, a[4 * g + 3] * f};
        }
    __shared__ f32x2 joined[32];
    if (wave == 0 && h == 0) joined[n] = f32x2{M * w.c_log2, L};
    __syncthreads();
    for (int e = tid; e < u.rows * (D / 4); e += 64 * NW) {
        const int r = e / (D / 4), g = e % (D / 4);
        if (4 * g >= p.d) continue;
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) a += *reinterpret_cast<const f32x4*>(lds + i * WAVE_FLOATS + r * D + ((g ^ (r & 7)) << 2));
        if (direct) {
            const float l = joined[r][1], inv = l == 0.f ? 0.f : 1.0f / l;
            const PagedRow at = paged_row(p, u, r);
            *reinterpret_cast<u32x2*>(p.o + at.b * p.os.b + at.h * p.os.h + at.i * p.os.n + 4 * g) = u32x2{pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[2] * inv, a[3] * inv)};
        } else {
            *reinterpret_cast<f32x4*>(out_o + (int64_t)r * p.d + 4 * g) = a;
        }
    }
    if (tid < u.rows) {
        const f32x2 ml = joined[tid];
        if (!direct) out_ml[tid] = ml;
        else if (p.lse) {
            const PagedRow at = paged_row(p, u, tid);
            p.lse[((int64_t)at.b * p.H + at.h) * p.N + at.i] = ml[1] == 0.f ? -INFINITY : (ml[0] + log2_fast(ml[1])) * kLn2;
        }
    }
}

// A unit whose wavefronts walk keys of their own: wavefront w the tiles from tile0 + w * `run` on, STRIDED: tile0 + w, tile0 + w + NW, ...
template <int D, int NW, bool STRIDED>
__device__ __forceinline__ void paged_unit_body(const PagedParams& p, const PagedUnit& u, uint16_t* lds, bool bad, bool direct, float* out_o, f32x2* out_ml) {
    using T = PagedTile<D>;
    constexpr int DC = D / 16, DB = D / 32, NDMA = T::NDMA;
    const int tid = paged_thread(), lane = tid & 63, wave = packed_uniform(tid >> 6), n = lane & 31;
    uint16_t* const mine = lds + wave * T::WAVE_ELEMS;
    const uint32_t lds_k = lds_addr(mine), lds_v = lds_k + 2u * T::TILE_ELEMS;
    const uint16_t* const kbase = p.k + u.kv_head * p.ks.h;
    const uint16_t* const vbase = p.v + u.kv_head * p.vs.h;
    constexpr int STEP = STRIDED ? NW : 1;
    const int run = (u.tiles + NW - 1) / NW;
    const int t_lo = u.tile0 + (STRIDED ? wave : wave * run), t_hi = STRIDED ? u.tile0 + u.tiles : min(t_lo + run, u.tile0 + u.tiles);
    const int last_key = u.keys - 1;

    PagedPages pages;
    uint32_t k_off[NDMA / 2], v_off[NDMA / 2];
    paged_offsets<D>(p, p.ks, lane, 0, k_off);
    paged_offsets<D>(p, p.vs, lane, 0, v_off);
    auto copy = [&](const uint16_t* base, const Strides& st, const uint32_t (&off)[NDMA / 2], int t, uint32_t dst) {
        paged_copy<D, NDMA>(p, pages, base, st, off, lane, t * T::BN, last_key - t * T::BN, 0, dst);
    };
    if (STRIDED || t_lo < t_hi) pages.load(p, u, lane, (t_lo * T::BN) >> p.page_shift);
    if (t_lo < t_hi) {
        copy(kbase, p.ks, k_off, t_lo, lds_k);
        copy(vbase, p.vs, v_off, t_lo, lds_v);
    }
    const PagedRow me = paged_row(p, u, min(n, u.rows - 1));
    PagedRows<D> w;
    w.begin(p, lane, me, n < u.rows);
    const int limit = u.own ? max(u.keys - u.lag + me.i, 0) : u.keys;             // this lane's row attends to the keys below it
    const int clean = u.own ? max(u.keys - u.lag, 0) : u.keys;                    // ... and every row to those below this

    for (int t = t_lo; t < t_hi; t += STEP) {
        const bool more = t + STEP < t_hi;
        if (more && !pages.holds(p, (t + STEP + 1) * T::BN - 1)) pages.load(p, u, lane, ((t + STEP) * T::BN) >> p.page_shift);
        wait_vm<NDMA>();                               // K(t) has landed (V(t) may be on its way)
        bf16x8 kf[DC];
        w.read_k(kf, mine);
        lds_reads_done();
        if (more) copy(kbase, p.ks, k_off, t + STEP, lds_k);
        f32x16 s = w.scores(kf);
        if ((t + 1) * T::BN > clean) w.exclude(s, lane, limit - t * T::BN);
        w.fold(s);
        bf16x8 pf[2];
        w.weights(s, pf);
        if (more) wait_vm<NDMA>();                     // V(t) has landed (the next K may be on its way)
        else wait_vm<0>();
        bf16x8 vf[2 * DB];
        w.read_v(vf, mine + T::TILE_ELEMS);
        lds_reads_done();
        if (more) copy(vbase, p.vs, v_off, t + STEP, lds_v);
        w.add(vf, pf);
    }

    paged_unit_join<D, NW>(p, u, w, reinterpret_cast<float*>(lds), tid, bad | (pages.bad && t_lo < t_hi), direct, out_o, out_ml);
}

// A unit of the prefix with 128 rows: the wavefronts have 32 each and share the tiles, a quarter of each copied by every wavefront.
// Four stages: tile t is in stage t % 4, the copies run three tiles ahead, one barrier per tile, behind which tile t + 1 is there and
// the stage of the tile before free.  Copies past the last tile re-read it, so that the number under way is always the same.
template <int D>
__device__ __forceinline__ void paged_shared_body(const PagedParams& p, const PagedUnit& u, uint16_t* lds, bool bad, float* out_o, f32x2* out_ml) {
    using T = PagedTile<D>;
    constexpr int DC = D / 16, DB = D / 32, PER = T::NDMA / 4, NSTAGE = 4;
    static_assert(NSTAGE == 4, "three tiles under way, one read");
    const int tid = paged_thread(), lane = tid & 63, wave = packed_uniform(tid >> 6), n = lane & 31, h = lane >> 5;
    const uint16_t* const kbase = p.k + u.kv_head * p.ks.h;
    const uint16_t* const vbase = p.v + u.kv_head * p.vs.h;
    const uint32_t lds0 = lds_addr(lds);
    const int rows = min(32, u.rows - 32 * wave), last_key = u.keys - 1, t_hi = u.tile0 + u.tiles;      // rows: of this wavefront, not positive: none
    PagedPages pages;
    uint32_t k_off[PER], v_off[PER];
    paged_offsets<D>(p, p.ks, lane, wave * PER % (T::NDMA / 2), k_off);
    paged_offsets<D>(p, p.vs, lane, wave * PER % (T::NDMA / 2), v_off);
    auto copy = [&](int t) {
        const int at = min(t, t_hi - 1), key0 = at * T::BN;
        if (!pages.holds(p, key0 + T::BN - 1)) pages.load(p, u, lane, key0 >> p.page_shift);
        const uint32_t dst = lds0 + (uint32_t)((t - u.tile0) % NSTAGE) * (4u * T::TILE_ELEMS);
        paged_copy<D, PER>(p, pages, kbase, p.ks, k_off, lane, key0, last_key - key0, wave * PER, dst);
        paged_copy<D, PER>(p, pages, vbase, p.vs, v_off, lane, key0, last_key - key0, wave * PER, dst + 2u * T::TILE_ELEMS);
    };
    pages.load(p, u, lane, (u.tile0 * T::BN) >> p.page_shift);
#pragma unroll
    for (int i = 0; i < NSTAGE - 1; ++i) copy(u.tile0 + i);
    const PagedRow me = paged_row(p, u, min(32 * wave + n, u.rows - 1));
    PagedRows<D> w;
    w.begin(p, lane, me, n < rows);
    auto stage_of = [&](int t) { return lds + ((t - u.tile0) % NSTAGE) * (2 * T::TILE_ELEMS); };
    auto scores_of = [&](int t) {
        bf16x8 kf[DC];
        w.read_k(kf, stage_of(t));
        return w.scores(kf);
    };
    auto landed = [&]() {                              // everyone's copies are, and nobody reads the tile before any more
        lds_reads_done();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    wait_vm<2 * (NSTAGE - 2) * PER>();                 // this wavefront's copies of the first tile
    landed();
    f32x16 s = scores_of(u.tile0);
    if (T::BN > u.keys - u.tile0 * T::BN) w.exclude(s, lane, u.keys - u.tile0 * T::BN);
    w.fold(s);
    // The exponentials of tile t run between the matrix instructions that form the scores of tile t + 1 (after the last tile: of what
    // the copies past the end have left there, which nobody uses).
    for (int t = u.tile0; t < t_hi; ++t) {
        wait_vm<2 * (NSTAGE - 3) * PER>();             // this wavefront's copies of tile t + 1 have landed
        landed();
        copy(t + NSTAGE - 1);
        f32x16 next = scores_of(t + 1);
        bf16x8 pf[2];
        w.weights(s, pf);
#pragma unroll
        for (int c = 0; c < 2; ++c) w.add16(stage_of(t) + T::TILE_ELEMS, c, pf[c]);
        s = next;
        if (t + 1 < t_hi) {
            if ((t + 2) * T::BN > u.keys) w.exclude(s, lane, u.keys - (t + 1) * T::BN);
            w.fold(s);
        }
    }
    wait_vm<0>();                                      // (the next unit's copies take the same stages)
    w.l_run += xhalf(w.l_run);
    if (__any(bad | pages.bad)) w.l_run = __builtin_nanf("");
    if (n >= rows) return;
    float* const out = out_o + (int64_t)(32 * wave + n) * p.d + 4 * h;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x16& a = w.oacc[db];
            if (32 * db + 8 * g + 4 * h < p.d) *reinterpret_cast<f32x4*>(out + 32 * db + 8 * g) = f32x4{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
        }
    if (h == 0) out_ml[32 * wave + n] = f32x2{w.m_run * w.c_log2, w.l_run};
}

// The units are dealt to the workgroups in turn, as the host does not know how many there are and a workgroup without one would cost as
// much as the summing of the batch: those of the prefix first, then the own ones, of which the first go to the workgroups that have
// none of the prefix, a few each while the others are at theirs (24 sequences on a prefix of 8192 34.5 -> 29.8 us, D = 64 35.5 -> 27.0).
template <int D, class P>
__global__ __launch_bounds__(256, D <= 64 ? 3 : 2) void paged_fwd_kernel(const P p) {
    extern __shared__ __attribute__((aligned(1024))) uint16_t lds[];
    __shared__ int sums[4], found[4];
    const int G = p.H / p.Hkv, rows = p.N * G, rt = PagedCut::row_tiles(rows), slot_rows = min(32, rows);
    const int all = p.B * rows, prefix_rt = PagedCut::prefix_row_tiles(all), prefix_rows = PagedCut::prefix_tile_rows(all);
    const PagedPlan c = paged_plan(p, sums);
    const int free = max((int)gridDim.x - c.prefix_units, 0), ahead = c.prefix_units && free ? 1 + c.prefix_unit / 16 : 0;      // units of such a workgroup ahead of the common deal
    const int spare = (int)blockIdx.x - c.prefix_units;             // which of these workgroups this is, if not negative
    int taken = spare < 0 ? ahead : 0;
    for (int at = (int)blockIdx.x;;) {
        __syncthreads();                               // the last unit's LDS is free
        PagedUnit u;
        if (at < c.prefix_units) {
            // the row tiles of the same keys one behind the other on one XCD
            const int unit = xcd_remap(at, c.prefix_units), part = packed_uniform(unit / prefix_rt);
            const int tile = unit - part * prefix_rt, split = packed_uniform(part / p.Hkv);
            u.own = false;
            u.table = p.prefix_table;
            u.entries = p.prefix_pages;
            u.keys = c.prefix_keys;
            u.row0 = prefix_rows * tile;
            u.rows = min(prefix_rows, all - u.row0);
            u.kv_head = part - split * p.Hkv;
            u.b0 = 0;
            u.lag = 0;
            u.tile0 = split * c.prefix_unit;
            u.tiles = min(c.prefix_unit, c.prefix_tiles - u.tile0);
            const int64_t slot = (int64_t)unit * prefix_rows;
            if (PagedCut::shared(all)) paged_shared_body<D>(p, u, lds, c.prefix_bad, p.part_o + slot * p.d, p.part_ml + slot);
            else paged_unit_body<D, 4, false>(p, u, lds, c.prefix_bad, false, p.part_o + slot * p.d, p.part_ml + slot);
            at += (int)gridDim.x;
        } else {
            const int number = taken < ahead ? spare + taken * free : ahead * free + (int)blockIdx.x + (taken - ahead) * (int)gridDim.x;
            ++taken;
            if (threadIdx.x == 0) found[0] = -1;
            auto units_of = [&](int tiles) { return PagedCut::splits(tiles, c.own_unit, p.B * p.Hkv * rt); };
            paged_own_units(p, c, sums, units_of, [&](int b, int len, int first, int splits) {
                if (number >= first && number < first + splits * p.Hkv * rt) {
                    found[0] = b;
                    found[1] = first;
                    found[2] = splits;
                    found[3] = len;
                }
                if (blockIdx.x == 0) p.plan[b] = int2{first, splits};
            });
            if (blockIdx.x == 0 && threadIdx.x == 0) p.plan[p.B] = int2{c.prefix_splits, 0};
            __syncthreads();
            const int b = packed_uniform(found[0]);
            if (b < 0) return;                         // past the last unit: nobody has one any more
            const int in_b = number - packed_uniform(found[1]), splits = packed_uniform(found[2]), len = packed_uniform(found[3]);
            const int pair = packed_uniform(in_b / splits), split = in_b - pair * splits, most = p.table_pages << p.page_shift;
            u.own = true;
            u.table = p.table + b * p.table_stride;
            u.entries = p.table_pages;
            u.keys = min(max(len, 0), most);
            u.kv_head = packed_uniform(pair / rt);
            u.row0 = 32 * (pair - u.kv_head * rt);
            u.rows = min(32, rows - u.row0);
            u.b0 = b;
            u.lag = p.N - 1;
            const int unit = packed_uniform(PagedCut::even(paged_tiles(u.keys), c.own_unit, p.B * p.Hkv * rt));
            u.tile0 = split * unit;
            u.tiles = min(unit, paged_tiles(u.keys) - u.tile0);
            const int64_t slot = p.own_slot + (int64_t)number * slot_rows;
            paged_unit_body<D, 4, false>(p, u, lds, len > most, splits == 1 && c.prefix_tiles == 0, p.part_o + slot * p.d, p.part_ml + slot);
        }
    }
}

// Short tables, no prefix: blockIdx.x = (sequence, key head, 32 rows).  The first pages are requested before the number of keys is known.
template <int D, int NW, class P>
__global__ __launch_bounds__(64 * NW, NW == 4 ? (D <= 64 ? 3 : 2) : 2) void paged_direct_kernel(const P p) {
    extern __shared__ __attribute__((aligned(1024))) uint16_t lds[];
    const int rows = p.N * (p.H / p.Hkv), rt = PagedCut::row_tiles(rows);
    const int pair = packed_uniform((int)blockIdx.x / rt), b = packed_uniform(pair / p.Hkv);
    PagedUnit u;
    u.own = true;
    u.table = p.table + b * p.table_stride;
    u.entries = p.table_pages;
    u.kv_head = pair - b * p.Hkv;
    u.row0 = 32 * ((int)blockIdx.x - pair * rt);
    u.rows = min(32, rows - u.row0);
    u.b0 = b;
    u.lag = p.N - 1;
    u.tile0 = 0;
    bool bad;
    u.keys = packed_uniform(paged_len(p, b, bad));
    u.tiles = paged_tiles(u.keys);
    paged_unit_body<D, NW, true>(p, u, lds, bad, true, nullptr, nullptr);
}

int launch_paged_merge(const PagedParams& p, bool ranges, hipStream_t s);        // compiled in flame_paged.hip

// Joins the units of a row: SHARE wavefronts take a share of the units each (4: a workgroup per row, 1: a workgroup for four rows).  Bound by the
// latency of plan, maxima and sums one behind the other, about 6 us with its launch.  RANGES: the keys were cut into ranges of tiles.  (One kernel that
// asks the plan -> one for each, us, bf16: one sequence of 2000 13.3 -> 13.0, of 8000 19.9 -> 19.4, 12 answers on a prefix of 4096 18.2 -> 17.8.)
template <int SHARE, bool RANGES>
__global__ __launch_bounds__(256) void paged_merge_kernel(const PagedParams p) {
    __shared__ f32x2 quarter[4][64];
    const int lane = threadIdx.x & 63, wave = SHARE == 1 ? 0 : packed_uniform(threadIdx.x >> 6);
    const int at_row = SHARE == 1 ? (int)blockIdx.x * 4 + packed_uniform(threadIdx.x >> 6) : (int)blockIdx.x;
    if (SHARE == 1 && at_row >= p.B * p.H * p.N) return;
    const int G = p.H / p.Hkv, rows = p.N * G, rt = PagedCut::row_tiles(rows), all = p.B * rows, slot_rows = min(32, rows);
    const int pair = packed_uniform(at_row / rows), r = at_row - pair * rows, b = packed_uniform(pair / p.Hkv), kv_head = pair - b * p.Hkv;
    const int2 mine = p.plan[b];
    const int first = packed_uniform(mine.x), each = packed_uniform(mine.y), all_of = packed_uniform(p.plan[p.B].x);
    int own = each, prefix = RANGES ? 0 : all_of, range = 0;
    if constexpr (RANGES) {
        const int at_tile = first + (kv_head * rt + r / 32) * each;
        range = at_tile / all_of;                          // that the walk begins in
        own = each == 0 ? 0 : (at_tile + each - 1) / all_of - range + 1;
    }
    const int parts = own + prefix;
    if (own == 1 && prefix == 0) return;                   // written by the unit itself
    // rows of the partial results: unit s of the prefix, unit s of the own keys
    const int64_t prefix_pad = (int64_t)PagedCut::prefix_row_tiles(all) * PagedCut::prefix_tile_rows(all);
    const int64_t prefix_at = kv_head * prefix_pad + b * rows + r, prefix_step = p.Hkv * prefix_pad;
    const int64_t own_at = p.own_slot + (int64_t)(first + (kv_head * rt + r / 32) * own) * slot_rows + r % 32;
    auto slot_of = [&](int s) {
        // a range has two places, for a walk that it ends or goes on with and for one that it begins
        if (RANGES) return p.own_slot + (int64_t)(s == 0 ? 2 * range + 1 : 2 * (range + s)) * slot_rows + r % 32;
        return s < prefix ? prefix_at + s * prefix_step : own_at + (int64_t)(s - prefix) * slot_rows;
    };
    float M = -INFINITY, L = 0.f, a0 = 0.f, a1 = 0.f;
    bool nan = false;
    const bool col = 2 * lane < p.d;
    for (int s0 = 0; s0 < parts; s0 += 64) {
        const f32x2 ml = s0 + lane < parts ? p.part_ml[slot_of(s0 + lane)] : f32x2{-INFINITY, 0.f};
        nan |= __any(ml[1] != ml[1] || ml[0] != ml[0]);
        float m = ml[0];
#pragma unroll
        for (int d = 1; d < 64; d *= 2) m = fmaxf(m, __shfl_xor(m, d, 64));
        const float M_new = fmaxf(M, m), M_to = M_new == -INFINITY ? 0.f : M_new, old = exp2_fast(M - M_to);
        const float w = ml[1] == 0.f ? 0.f : exp2_fast(ml[0] - M_to);
        float l = w * ml[1];
#pragma unroll
        for (int d = 1; d < 64; d *= 2) l += __shfl_xor(l, d, 64);
        L = L * old + l;
        a0 *= old;
        a1 *= old;
        M = M_new;
        const int count = min(64, parts - s0);
        constexpr int AHEAD = SHARE == 1 ? 8 : 4;          // units of this wavefront on their way before the first is used
        for (int s = wave; s < count; s += AHEAD * SHARE) {
            f32x2 v[AHEAD];
            float ws[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int at = s + SHARE * i;
                ws[i] = at < count ? __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, w), at)) : 0.f;
                v[i] = f32x2{0.f, 0.f};
                if (at < count && col) v[i] = *reinterpret_cast<const f32x2*>(p.part_o + slot_of(s0 + at) * p.d + 2 * lane);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                a0 = fmaf(ws[i], v[i][0], a0);
                a1 = fmaf(ws[i], v[i][1], a1);
            }
        }
    }
    f32x2 sum = {a0, a1};
    if constexpr (SHARE > 1) {
        quarter[wave][lane] = sum;
        __syncthreads();
        if (wave != 0) return;
#pragma unroll
        for (int i = 1; i < SHARE; ++i) sum += quarter[i][lane];
    }
    const int i = r / G, hh = kv_head * G + r % G;
    const float inv = nan ? __builtin_nanf("") : L == 0.f ? 0.f : 1.0f / L;
    if (col) *reinterpret_cast<uint32_t*>(p.o + b * p.os.b + hh * p.os.h + i * p.os.n + 2 * lane) = pack_bf16(sum[0] * inv, sum[1] * inv);
    if (p.lse && lane == 0) p.lse[((int64_t)b * p.H + hh) * p.N + i] = nan ? __builtin_nanf("") : L == 0.f ? -INFINITY : (M + log2_fast(L)) * kLn2;
}

}  // namespace fattn
