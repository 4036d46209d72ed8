// Attention over a paged cache held in 8 bits (kv_codes.hpp): what attn_paged.hpp does, with tiles of codes.
//
//   s_j = scale k_scale[j] sum_d q_d k_code[j][d],   O = sum_j p_j v_scale[j] v_code[j] / sum_j p_j
// The scales of a key and a value are factors of its score and its weight: a multiplication each for every pair of row and key, where
// numbers out of codes and scales would take one for every element and a rounding.  The codes become bf16 (exactly) on their way from LDS to the
// matrix instructions: a value's column comes through the transposing read of 8 bits, eight tokens at a time, in the order of the weights.
//
// The way of units, plan and merge is that of the bf16 cache.  A wavefront has two tiles of K, V and scales in LDS, as many bytes as one of bf16,
// and requests a tile two steps ahead.
#pragma once
#include "attn_paged.hpp"
#include "kv_codes.hpp"

namespace fattn {

template <int CODE>
struct Paged8Params : PagedParams {        // k, v unused; ks, vs in bytes
    const uint8_t* k8;
    const uint8_t* v8;
    const float* k_scale;          // [pages][Hkv][page / block] through kss, vss (b: page, h: head, n: block)
    const float* v_scale;
    Strides kss, vss;
    int block_shift;               // log2 of the tokens that share a scale
};

template <int D>
struct Paged8Tile {
    static_assert(D == 64 || D == 128, "rows of 64 or 128 bytes");
    static constexpr int BN = 32, RB = D;                          // keys, bytes of a row
    static constexpr int TILE = BN * RB, SCALES = 2 * BN * 4;      // bytes: of K or V, of both scales
    static constexpr int STAGE = 2 * TILE + SCALES;
    static constexpr int WAVE = 2 * STAGE;
    static_assert(WAVE >= 32 * D * 4, "the 32 x D fp32 sums at the end");
    static constexpr int NDMA = TILE / 1024, RPD = 1024 / RB, GPR = RB / 16;       // copies per tile, rows per copy, granules per row
    static constexpr int lds_bytes(int nw) { return nw * WAVE; }
    // Swizzle of the 16-byte granules of a row.  Free of bank conflicts: 16-byte reads of one granule of 16 rows one behind the other, and the transposing
    // reads, whose half wavefront takes two neighbouring granules of rows 4 h .. 4 h + 3 and 8 + 4 h .. 8 + 4 h + 3.  Rows 16 apart have the same.
    static __device__ __forceinline__ constexpr int swz(int row) {
        if (RB == 64) return (row >> 2) & 3;
        const int pair = row >> 1;
        return (pair & 4) | ((pair & 1) << 1) | ((pair >> 1) & 1);
    }
};
template <int D, int CODE>
constexpr int paged_lds_bytes(const Paged8Params<CODE>*, int nw) { return Paged8Tile<D>::lds_bytes(nw); }

// ds_read_b64_tr_b8: a group of 16 lanes reads 8 rows of 16 bytes, lane r the half r % 2 of row r / 2; lane i receives byte i of each row.
__device__ __forceinline__ u32x2 lds_read_tr8(const uint8_t* p) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(p)));
}

// Copies of a tile (NDMA of 1 KiB) and of its scales to LDS.  Rows past the last key (`most` of the tile) re-read it.
template <int D, int CODE>
struct Paged8Copy {
    using T = Paged8Tile<D>;
    static constexpr int EACH = T::NDMA / 2;           // per 16 rows, which lie in one page
    const Paged8Params<CODE>& p;
    const PagedUnit& u;
    PagedPages& pages;
    int lane;
    uint32_t k_off[EACH], v_off[EACH];                 // bytes of this lane within 16 rows

    __device__ __forceinline__ Paged8Copy(const Paged8Params<CODE>& p, const PagedUnit& u, PagedPages& pages, int lane) : p(p), u(u), pages(pages), lane(lane) {
#pragma unroll
        for (int j = 0; j < EACH; ++j) {
            const int row = j * T::RPD + lane / T::GPR, g = lane % T::GPR ^ T::swz(row), from = 16 * g < p.d ? 16 * g : 0;
            k_off[j] = (uint32_t)(row * (int)p.ks.n + from);
            v_off[j] = (uint32_t)(row * (int)p.vs.n + from);
        }
    }
    // the pages that tile t needs are there
    __device__ __forceinline__ void find(int t) {
        if (!pages.holds(p, (t + 1) * T::BN - 1)) pages.load(p, u, lane, (t * T::BN) >> p.page_shift);
    }
    __device__ __forceinline__ void tile(const uint8_t* base, const Strides& st, const uint32_t (&off)[EACH], int t, uint32_t dst) const {
        const int key0 = t * T::BN, most = u.keys - 1 - key0;
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int from = 16 * half <= most ? half : 0;         // a half without a key: the last key is in the other one
            const uint8_t* const rows = base + pages.rows16(p, key0 + 16 * from, st);
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                uint32_t o = off[j];
                if (16 * half + 15 > most) {
                    const int row = j * T::RPD + lane / T::GPR;
                    o += (uint32_t)((min(16 * half + row, most) - 16 * from - row) * (int)st.n);
                }
                dma16u(rows, o, dst + 1024u * (uint32_t)(half * EACH + j));
            }
        }
    }
    __device__ __forceinline__ void k(int t, uint32_t dst) const { tile(p.k8 + u.kv_head * p.ks.h, p.ks, k_off, t, dst); }
    __device__ __forceinline__ void v(int t, uint32_t dst) const { tile(p.v8 + u.kv_head * p.vs.h, p.vs, v_off, t, dst); }
    // lanes 0 .. 31: K, 32 .. 63: V
    __device__ __forceinline__ void scales(int t, uint32_t dst) const {
        const int key0 = t * T::BN, most = u.keys - 1 - key0, at = min(lane & 31, most), token = (key0 + at) & ((1 << p.page_shift) - 1);
        const int e0 = __builtin_amdgcn_readlane(pages.mine, (key0 >> p.page_shift) - pages.first);
        const int e1 = most >= 16 ? __builtin_amdgcn_readlane(pages.mine, ((key0 + 16) >> p.page_shift) - pages.first) : e0;
        const int64_t k0 = e0 * p.kss.b + u.kv_head * p.kss.h, k1 = e1 * p.kss.b + u.kv_head * p.kss.h;
        const int64_t v0 = e0 * p.vss.b + u.kv_head * p.vss.h, v1 = e1 * p.vss.b + u.kv_head * p.vss.h;
        const float* const from = lane < 32 ? p.k_scale + (at < 16 ? k0 : k1) : p.v_scale + (at < 16 ? v0 : v1);
        dma4(from + (token >> p.block_shift) * (int)(lane < 32 ? p.kss.n : p.vss.n), dst);
    }
};

template <int D, int CODE>
struct Paged8Rows : PagedRows<D> {
    using T = Paged8Tile<D>;
    using PagedRows<D>::qf;
    static constexpr int DC = D / 16, DB = D / 32;
    int k_at[DB];              // K: row n, granule 2 c + h, which are the contraction's steps 2 c and 2 c + 1
    int v_at;                  // V: rows 4 h + 0 .. 3, 8 + 4 h + 0 .. 3
    int v_granule[DB];         // (swizzled)

    __device__ __forceinline__ void begin(const PagedParams& p, int lane, const PagedRow& at, bool there) {
        const int n = lane & 31, h = lane >> 5, r = (lane & 15) >> 1, row = 4 * h + (r & 3) + 8 * (r >> 2);
        const uint16_t* const qrow = p.q + at.b * p.qs.b + at.h * p.qs.h + at.i * p.qs.n;
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            const int d0 = 32 * (dc >> 1) + 16 * h + 8 * (dc & 1);
            qf[dc] = __builtin_bit_cast(bf16x8, ldg16(qrow + d0, there && d0 < p.d));
        }
        v_at = row * T::RB + 8 * (lane & 1);
#pragma unroll
        for (int c = 0; c < DB; ++c) {
            k_at[c] = n * T::RB + (((2 * c + h) ^ T::swz(n)) << 4);
            v_granule[c] = ((2 * c + ((lane >> 4) & 1)) ^ T::swz(row)) << 4;
        }
        this->c_log2 = p.scale * kLog2e;
        this->stale_ok = stale_scope(this->c_log2);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int i = 0; i < 16; ++i) this->oacc[db][i] = 0.f;
    }
    __device__ __forceinline__ void read_k(u32x4 (&k)[DB], const uint8_t* tile) const {
#pragma unroll
        for (int c = 0; c < DB; ++c) k[c] = *reinterpret_cast<const u32x4*>(tile + k_at[c]);
    }
    __device__ __forceinline__ void read_v(u32x2 (&v)[2 * DB], const uint8_t* tile) const {
#pragma unroll
        for (int i = 0; i < 2 * DB; ++i) v[i] = lds_read_tr8(tile + v_at + v_granule[i % DB] + 16 * (i / DB) * T::RB);
    }
    // of the keys 8 g + 4 h .. + 3, the rows that this lane's scores and weights are of
    static __device__ __forceinline__ void read_scales(f32x4 (&s)[4], const float* scales, int lane) {
#pragma unroll
        for (int g = 0; g < 4; ++g) s[g] = *reinterpret_cast<const f32x4*>(scales + 8 * g + 4 * (lane >> 5));
    }
    __device__ __forceinline__ f32x16 scores(const u32x4 (&k)[DB], const f32x4 (&scale)[4]) const {
        f32x16 s;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 0.f;
#pragma unroll
        for (int c = 0; c < DB; ++c) {
            s = mfma32(codes_to_bf16<CODE>(k[c][0], k[c][1]), qf[2 * c], s);
            s = mfma32(codes_to_bf16<CODE>(k[c][2], k[c][3]), qf[2 * c + 1], s);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] *= scale[r >> 2][r & 3];
        return s;
    }
    // as PagedRows::weights; what meets V is the weight times V's scale, rounded to bf16
    __device__ __forceinline__ void weights(f32x16& s, const f32x4 (&scale)[4], bf16x8 (&pf)[2]) {
        const float shift = (this->m_run == -INFINITY ? 0.f : this->m_run) * this->c_log2;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            s[r] = exp2_fast(fmaf(s[r], this->c_log2, -shift));
            sum[r & 1] += s[r];
            s[r] *= scale[r >> 2][r & 3];
        }
        this->l_run += sum[0] + sum[1];
        pf[0] = pack8(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]);
        pf[1] = pack8(s[8], s[9], s[10], s[11], s[12], s[13], s[14], s[15]);
    }
    __device__ __forceinline__ void add(const u32x2 (&v)[2 * DB], const bf16x8 (&pf)[2]) {
#pragma unroll
        for (int i = 0; i < 2 * DB; ++i) this->oacc[i % DB] = mfma32(codes_to_bf16<CODE>(v[i][0], v[i][1]), pf[i / DB], this->oacc[i % DB]);
    }
};

// The walk of one wavefront over the tiles t_lo, t_lo + STEP, ... below t_hi.  `mine`: its Paged8Tile::WAVE bytes of LDS; limit: this lane's row
// attends to the keys below it, clean: every row to those below this.  Of the stage of tile t: K, V and the scales of tile t + 2 STEP follow as soon as
// those of t are in registers, in the order K, scales, V, which is what the numbers of copies under way below count.
template <int STEP, int D, int CODE>
__device__ __forceinline__ void paged8_walk(const PagedUnit& u, Paged8Copy<D, CODE>& copy, Paged8Rows<D, CODE>& w, const uint8_t* mine, int t_lo, int t_hi,
                                            int limit, int clean) {
    using T = Paged8Tile<D>;
    constexpr int DB = D / 32, N = T::NDMA;
    int at = 0;                                        // bytes: this tile's stage
    const uint32_t lds = lds_addr(mine);
    for (int t = t_lo; t < t_hi; t += STEP) {
        const bool one = t + STEP < t_hi, two = t + 2 * STEP < t_hi;
        if (two) copy.find(t + 2 * STEP);
        if (one) wait_vm<3 * N + 1>();                 // K and scales of t have landed (V of t, all of the next may be on their way)
        else wait_vm<N>();
        u32x4 k[DB];
        f32x4 ks[4], vs[4];
        w.read_k(k, mine + at);
        w.read_scales(ks, reinterpret_cast<const float*>(mine + at + 2 * T::TILE), copy.lane);
        w.read_scales(vs, reinterpret_cast<const float*>(mine + at + 2 * T::TILE) + 32, copy.lane);
        lds_reads_done();
        if (two) copy.k(t + 2 * STEP, lds + at);
        f32x16 s = w.scores(k, ks);
        if ((t + 1) * T::BN > clean) w.exclude(s, copy.lane, limit - t * T::BN);
        w.fold(s);
        bf16x8 pf[2];
        w.weights(s, vs, pf);
        if (two) wait_vm<3 * N + 1>();                 // V of t
        else if (one) wait_vm<2 * N + 1>();
        else wait_vm<0>();
        u32x2 v[2 * DB];
        w.read_v(v, mine + at + T::TILE);
        lds_reads_done();
        if (two) {
            copy.scales(t + 2 * STEP, lds + at + 2 * T::TILE);
            copy.v(t + 2 * STEP, lds + at + T::TILE);
        }
        w.add(v, pf);
        at = T::STAGE - at;
    }
}
// ... its first two tiles
template <int STEP, int D, int CODE>
__device__ __forceinline__ void paged8_start(Paged8Copy<D, CODE>& copy, const uint8_t* mine, int t_lo, int t_hi) {
    using T = Paged8Tile<D>;
    const uint32_t lds = lds_addr(mine);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int t = t_lo + i * STEP;
        if (t >= t_hi) break;
        if (i) copy.find(t);
        copy.k(t, lds + i * T::STAGE);
        copy.scales(t, lds + i * T::STAGE + 2 * T::TILE);
        copy.v(t, lds + i * T::STAGE + T::TILE);
    }
}

template <int D, int NW, bool STRIDED, int CODE>
__device__ __forceinline__ void paged_unit_body(const Paged8Params<CODE>& p, const PagedUnit& u, uint16_t* lds, bool bad, bool direct, float* out_o,
                                                f32x2* out_ml) {
    using T = Paged8Tile<D>;
    const int tid = paged_thread(), lane = tid & 63, wave = packed_uniform(tid >> 6), n = lane & 31;
    const uint8_t* const mine = reinterpret_cast<const uint8_t*>(lds) + wave * T::WAVE;
    constexpr int STEP = STRIDED ? NW : 1;
    const int run = (u.tiles + NW - 1) / NW;
    const int t_lo = u.tile0 + (STRIDED ? wave : wave * run), t_hi = STRIDED ? u.tile0 + u.tiles : min(t_lo + run, u.tile0 + u.tiles);
    PagedPages pages;
    Paged8Copy<D, CODE> copy(p, u, pages, lane);
    if (t_lo < t_hi) {
        pages.load(p, u, lane, (t_lo * T::BN) >> p.page_shift);
        paged8_start<STEP>(copy, mine, t_lo, t_hi);
    }
    const PagedRow me = paged_row(p, u, min(n, u.rows - 1));
    Paged8Rows<D, CODE> w;
    w.begin(p, lane, me, n < u.rows);
    const int limit = u.own ? max(u.keys - u.lag + me.i, 0) : u.keys, clean = u.own ? max(u.keys - u.lag, 0) : u.keys;
    paged8_walk<STEP>(u, copy, w, mine, t_lo, t_hi, limit, clean);
    paged_unit_join<D, NW, T::WAVE / 4>(p, u, w, reinterpret_cast<float*>(lds), tid, bad | pages.bad, direct, out_o, out_ml);
}

// A unit of the prefix with 128 rows: the wavefronts have 32 each.
template <int D, int CODE>
__device__ __forceinline__ void paged_shared_body(const Paged8Params<CODE>& p, const PagedUnit& u, uint16_t* lds, bool bad, float* out_o, f32x2* out_ml) {
    using T = Paged8Tile<D>;
    constexpr int DB = D / 32;
    const int tid = paged_thread(), lane = tid & 63, wave = packed_uniform(tid >> 6), n = lane & 31, h = lane >> 5;
    const uint8_t* const mine = reinterpret_cast<const uint8_t*>(lds) + wave * T::WAVE;
    const int rows = min(32, u.rows - 32 * wave), t_lo = u.tile0, t_hi = u.tile0 + u.tiles;
    if (rows <= 0) return;
    PagedPages pages;
    Paged8Copy<D, CODE> copy(p, u, pages, lane);
    pages.load(p, u, lane, (t_lo * T::BN) >> p.page_shift);
    paged8_start<1>(copy, mine, t_lo, t_hi);
    const PagedRow me = paged_row(p, u, min(32 * wave + n, u.rows - 1));
    Paged8Rows<D, CODE> w;
    w.begin(p, lane, me, n < rows);
    paged8_walk<1>(u, copy, w, mine, t_lo, t_hi, u.keys, u.keys);
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

}  // namespace fattn
