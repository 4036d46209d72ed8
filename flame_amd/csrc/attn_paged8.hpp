// Attention over a paged cache held in 8 bits (kv_codes.hpp): what attn_paged.hpp does, with tiles of codes.
//
//   s_j = scale k_scale[j] sum_d q_d k_code[j][d],   O = sum_j p_j v_scale[j] v_code[j] / sum_j p_j
// The scales of a key and a value are factors of its score and its weight: a multiplication each for every pair of row and key, where
// numbers out of codes and scales would take one for every element and a rounding.  The codes become bf16 (exactly) on their way from LDS to the
// matrix instructions: a value's column comes through the transposing read of 8 bits, eight tokens at a time, in the order of the weights.
//
// Units, partial results and merge are those of the bf16 cache; without a prefix the keys are cut otherwise (paged_ranges_kernel).  With half the bytes a tile's arithmetic weighs twice as much, so rows come in blocks of 16
// (v_mfma_f32_16x16x32_bf16), one block where a sequence has no more rows than that: half of the exponentials and of what goes with them.  A
// wavefront has two tiles of K, V and scales in LDS and requests a tile two steps ahead.
#pragma once
#include "attn_paged.hpp"
#include "kv_codes.hpp"

namespace fattn {

// R: blocks of 16 rows that a unit of own keys has, 1 or 2.
template <int CODE, int R>
struct Paged8Params : PagedParams {        // k, v unused; ks, vs in bytes
    const uint8_t* k8;
    const uint8_t* v8;
    const float* k_scale;          // [pages][Hkv][page / block] through kss, vss (b: page, h: head, n: block; bytes, b and n below 2^31)
    const float* v_scale;
    Strides kss, vss;
    int block_shift;               // log2 of the tokens that share a scale
};

template <int D>
struct Paged8Tile {
    static_assert(D == 64 || D == 128, "rows of 64 or 128 bytes");
    static constexpr int BN = 32, RB = D;                          // keys, bytes of a row
    static constexpr int TILE = BN * RB, SCALES = 2 * BN * 4;      // bytes: of K or V, of both scales
    static constexpr int V = TILE, S = 2 * TILE, STAGE = 2 * TILE + SCALES;
    static constexpr int WAVE = 2 * STAGE;
    static_assert(WAVE >= 32 * D * 4, "the 32 x D fp32 sums at the end");
    static constexpr int NDMA = TILE / 1024, RPD = 1024 / RB, GPR = RB / 16;       // copies per tile, rows per copy, granules per row
    static constexpr int lds_bytes(int nw) { return nw * WAVE; }
    // Swizzle of the 16-byte granules of a row.  Free of bank conflicts: 16-byte reads of one granule of the 16 rows of either half, and the transposing
    // reads, whose half wavefront takes one granule of rows 8 x .. 8 x + 7 and 16 + 8 x .. 16 + 8 x + 7.
    static __device__ __forceinline__ constexpr int swz(int row) {
        return RB == 64 ? ((row >> 2) & 3) ^ ((row >> 4) << 1) : ((row >> 1) & 3) | ((((row >> 3) ^ (row >> 4)) & 1) << 2);
    }
};
template <int D, int CODE, int R>
constexpr int paged_lds_bytes(const Paged8Params<CODE, R>*, int nw) { return Paged8Tile<D>::lds_bytes(nw); }

// ds_read_b64_tr_b8: a group of 16 lanes reads 8 rows of 16 bytes, lane r the half r % 2 of row r / 2; lane i receives byte i of each row.
__device__ __forceinline__ u32x2 lds_read_tr8(const uint8_t* p) {
    typedef int i32x2 __attribute__((ext_vector_type(2)));
    typedef __attribute__((address_space(3))) i32x2 lds_i32x2;
    return __builtin_bit_cast(u32x2, __builtin_amdgcn_ds_read_tr8_b64_v2i32((lds_i32x2*)(p)));
}
// v_mfma_f32_16x16x32_bf16: lane l, g = l / 16, n = l % 16: A[n][8 g .. 8 g + 7], B[8 g .. 8 g + 7][n], D[4 g + r][n]
__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }

// Copies of a tile (NDMA of 1 KiB) and of its scales to LDS.  Rows past the last key (`most` of the tile) re-read it.
template <int D, class P>
struct Paged8Copy {
    using T = Paged8Tile<D>;
    static constexpr int EACH = T::NDMA / 2;           // per 16 rows, which lie in one page
    const P& p;
    const PagedUnit& u;
    PagedPages& pages;
    const int lane;
    const uint8_t* const k_base;
    const uint8_t* const v_base;
    uint32_t k_off[T::NDMA], v_off[T::NDMA];           // bytes of this lane within 16 rows
    const char* s_base;                                // lanes 0 .. 31: K's scales, 32 .. 63: V's
    int s_page, s_block;                               // bytes from page to page, from block to block
    int key0, most, e0, e1;                            // of the tile that is aimed at: first key, last key of it, the pages of its halves

    __device__ __forceinline__ Paged8Copy(const P& p, const PagedUnit& u, PagedPages& pages, int lane)
        : p(p), u(u), pages(pages), lane(lane), k_base(p.k8 + u.kv_head * p.ks.h), v_base(p.v8 + u.kv_head * p.vs.h) {
#pragma unroll
        for (int i = 0; i < T::NDMA; ++i) {
            const int row = i % EACH * T::RPD + lane / T::GPR, g = lane % T::GPR ^ T::swz(row + 16 * (i / EACH)), from = 16 * g < p.d ? 16 * g : 0;
            k_off[i] = (uint32_t)(row * (int)p.ks.n + from);
            v_off[i] = (uint32_t)(row * (int)p.vs.n + from);
        }
        s_base = lane < 32 ? reinterpret_cast<const char*>(p.k_scale) + u.kv_head * p.kss.h : reinterpret_cast<const char*>(p.v_scale) + u.kv_head * p.vss.h;
        s_page = (int)(lane < 32 ? p.kss.b : p.vss.b);
        s_block = (int)(lane < 32 ? p.kss.n : p.vss.n);
    }
    __device__ __forceinline__ void aim(int t) {
        key0 = t * T::BN;
        most = u.keys - 1 - key0;
        if (!pages.holds(p, key0 + T::BN - 1)) pages.load(p, u, lane, key0 >> p.page_shift);
        e0 = __builtin_amdgcn_readlane(pages.mine, (key0 >> p.page_shift) - pages.first);
        e1 = most >= 16 ? __builtin_amdgcn_readlane(pages.mine, ((key0 + 16) >> p.page_shift) - pages.first) : e0;
    }
    __device__ __forceinline__ void tile(const uint8_t* base, const Strides& st, const uint32_t (&off)[T::NDMA], uint32_t dst) const {
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int from = 16 * half <= most ? half : 0;         // a half without a key: the last key is in the other one
            const uint8_t* const rows = base + (half ? e1 : e0) * st.b + ((key0 + 16 * from) & ((1 << p.page_shift) - 1)) * st.n;
#pragma unroll
            for (int j = 0; j < EACH; ++j) {
                uint32_t o = off[half * EACH + j];
                if (16 * half + 15 > most) {
                    const int row = j * T::RPD + lane / T::GPR;
                    o += (uint32_t)((min(16 * half + row, most) - 16 * from - row) * (int)st.n);
                }
                dma16u(rows, o, dst + 1024u * (uint32_t)(half * EACH + j));
            }
        }
    }
    __device__ __forceinline__ void k(uint32_t dst) const { tile(k_base, p.ks, k_off, dst); }
    __device__ __forceinline__ void v(uint32_t dst) const { tile(v_base, p.vs, v_off, dst); }
    __device__ __forceinline__ void scales(uint32_t dst) const {
        const int at = min(lane & 31, most), token = (key0 + at) & ((1 << p.page_shift) - 1), e = at < 16 ? e0 : e1;
        dma4(s_base + (int64_t)e * s_page + (int64_t)(token >> p.block_shift) * s_block, dst);
    }
};

// What a wavefront holds of 16 R rows: their queries as MFMA fragments and the running softmax over the keys it has seen.  Lane (n, g): row n of
// every block; of a tile the keys 16 k + 4 g .. + 3, k = 0, 1, which are the contraction's steps of the second product in this order.
template <int D, int CODE, int R>
struct Paged8Rows {
    using T = Paged8Tile<D>;
    static constexpr int DC = D / 64, DB = D / 16;
    bf16x8 qf[R][2 * DC];
    f32x4 oacc[R][DB];
    float m_run[R], l_run[R], c_log2, stale_ok;
    int k_at[2][DC];           // K: row 16 k + n, granule 4 c + g, which are the contraction's steps 2 c and 2 c + 1
    int v_at[DB];              // V: rows 4 g + 0 .. 3, 16 + 4 g + 0 .. 3, granule db
    int s_at;

    __device__ __forceinline__ void begin(const PagedParams& p, const PagedUnit& u, int lane, int row0) {
        const int n = lane & 15, g = lane >> 4, j = n >> 1, row = 4 * g + (j & 3) + 16 * (j >> 2);
#pragma unroll
        for (int b = 0; b < R; ++b) {
            const int r = row0 + 16 * b + n;
            const PagedRow at = paged_row(p, u, min(r, u.rows - 1));
            const uint16_t* const qrow = p.q + at.b * p.qs.b + at.h * p.qs.h + at.i * p.qs.n;
#pragma unroll
            for (int dc = 0; dc < 2 * DC; ++dc) {
                const int d0 = 64 * (dc >> 1) + 16 * g + 8 * (dc & 1);
                qf[b][dc] = __builtin_bit_cast(bf16x8, ldg16(qrow + d0, r < u.rows && d0 < p.d));
            }
#pragma unroll
            for (int db = 0; db < DB; ++db) oacc[b][db] = f32x4{0.f, 0.f, 0.f, 0.f};
            m_run[b] = -INFINITY;
            l_run[b] = 0.f;
        }
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int c = 0; c < DC; ++c) k_at[k][c] = (16 * k + n) * T::RB + (((4 * c + g) ^ T::swz(16 * k + n)) << 4);
#pragma unroll
        for (int db = 0; db < DB; ++db) v_at[db] = T::V + row * T::RB + ((db ^ T::swz(row)) << 4) + 8 * (lane & 1);
        s_at = T::S + 16 * g;
        c_log2 = p.scale * kLog2e;
        stale_ok = stale_scope(c_log2);        // the reference maximum may lag the true one by 2^8
    }
    // (stage: bytes of the tile's stage)
    __device__ __forceinline__ void read_k(u32x4 (&k)[2][DC], const uint8_t* mine, int stage) const {
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int c = 0; c < DC; ++c) k[i][c] = *reinterpret_cast<const u32x4*>(mine + stage + k_at[i][c]);
    }
    __device__ __forceinline__ void read_v(u32x2 (&v)[DB], const uint8_t* mine, int stage) const {
#pragma unroll
        for (int db = 0; db < DB; ++db) v[db] = lds_read_tr8(mine + stage + v_at[db]);
    }
    __device__ __forceinline__ void read_scales(f32x4 (&s)[2], const uint8_t* mine, int stage) const {
#pragma unroll
        for (int k = 0; k < 2; ++k) s[k] = *reinterpret_cast<const f32x4*>(mine + stage + s_at + 64 * k);
    }
    __device__ __forceinline__ void scores(f32x4 (&s)[R][2], const u32x4 (&k)[2][DC], const f32x4 (&scale)[2]) const {
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int b = 0; b < R; ++b) s[b][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int c = 0; c < DC; ++c) {
                const bf16x8 lo = codes_to_bf16<CODE>(k[i][c][0], k[i][c][1]), hi = codes_to_bf16<CODE>(k[i][c][2], k[i][c][3]);
#pragma unroll
                for (int b = 0; b < R; ++b) {
                    s[b][i] = mfma16(lo, qf[b][2 * c], s[b][i]);
                    s[b][i] = mfma16(hi, qf[b][2 * c + 1], s[b][i]);
                }
            }
#pragma unroll
            for (int b = 0; b < R; ++b) s[b][i] *= scale[i];
        }
    }
    // keys of the tile from `limit` (of block b) on are excluded
    __device__ __forceinline__ static void exclude(f32x4 (&s)[2], int lane, int limit) {
        const int lim = limit - 4 * (lane >> 4);
#pragma unroll
        for (int k = 0; k < 2; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) s[k][r] = 16 * k + r >= lim ? -INFINITY : s[k][r];
    }
    static __device__ __forceinline__ float over_groups_max(float x) {
        x = fmaxf(x, __shfl_xor(x, 16, 64));
        return max_of_halves(x);
    }
    static __device__ __forceinline__ float over_groups_sum(float x) {
        x += __shfl_xor(x, 16, 64);
        return x + xhalf(x);
    }
    // the maximum of a tile's scores joins the running one, which moves (and the sums are rescaled) only when it lags by more than 2^8
    __device__ __forceinline__ void fold(const f32x4 (&s)[R][2]) {
        float top[R];
        bool behind = false;
#pragma unroll
        for (int b = 0; b < R; ++b) {
            top[b] = s[b][0][0];
#pragma unroll
            for (int r = 1; r < 8; ++r) top[b] = fmaxf(top[b], s[b][r >> 2][r & 3]);
            behind |= top[b] > m_run[b] + stale_ok;
        }
        if (__any(behind)) {
#pragma unroll
            for (int b = 0; b < R; ++b) {
                const float m_new = fmaxf(m_run[b], over_groups_max(top[b])), m_to = m_new == -INFINITY ? 0.f : m_new;
                const float alpha = exp2_fast((m_run[b] - m_to) * c_log2);
                m_run[b] = m_new;
                l_run[b] *= alpha;
#pragma unroll
                for (int db = 0; db < DB; ++db) oacc[b][db] *= alpha;
            }
        }
    }
    // exp2 of the scores against the running maximum.  What meets V is the weight times V's scale, rounded to bf16 (the sum l is of the unrounded
    // weights): the matrix instructions take no wider operand
    __device__ __forceinline__ void weights(f32x4 (&s)[R][2], const f32x4 (&scale)[2], bf16x8 (&pf)[R]) {
#pragma unroll
        for (int b = 0; b < R; ++b) {
            const float shift = (m_run[b] == -INFINITY ? 0.f : m_run[b]) * c_log2;
            float sum[2] = {0.f, 0.f};
#pragma unroll
            for (int k = 0; k < 2; ++k)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float e = exp2_fast(fmaf(s[b][k][r], c_log2, -shift));
                    sum[r & 1] += e;
                    s[b][k][r] = e * scale[k][r];
                }
            l_run[b] += sum[0] + sum[1];
            pf[b] = pack8(s[b][0][0], s[b][0][1], s[b][0][2], s[b][0][3], s[b][1][0], s[b][1][1], s[b][1][2], s[b][1][3]);
        }
    }
    __device__ __forceinline__ void add(const u32x2 (&v)[DB], const bf16x8 (&pf)[R]) {
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            const bf16x8 vf = codes_to_bf16<CODE>(v[db][0], v[db][1]);
#pragma unroll
            for (int b = 0; b < R; ++b) oacc[b][db] = mfma16(vf, pf[b], oacc[b][db]);
        }
    }
};

// The walk of one wavefront over the tiles t_lo, t_lo + STEP, ... below t_hi.  `mine`: its Paged8Tile::WAVE bytes of LDS; limit: this lane's row of a
// block attends to the keys below it, clean: every row to those below this.  Of the stage of tile t: K, V and the scales of tile t + 2 STEP follow as soon as
// those of t are in registers, in the order K, scales, V, which is what the numbers of copies under way below count.
template <int STEP, int D, int CODE, int R, class P>
__device__ __forceinline__ void paged8_walk(Paged8Copy<D, P>& copy, Paged8Rows<D, CODE, R>& w, const uint8_t* mine, int t_lo, int t_hi, const int (&limit)[R],
                                            int clean) {
    using T = Paged8Tile<D>;
    constexpr int N = T::NDMA;
    const uint32_t lds = lds_addr(mine);
    auto step = [&](int t, auto stage_tag) {
        constexpr int stage = decltype(stage_tag)::value * T::STAGE;
        const bool one = t + STEP < t_hi, two = t + 2 * STEP < t_hi;
        if (two) copy.aim(t + 2 * STEP);
        if (one) wait_vm<3 * N + 1>();                 // K and scales of t have landed (V of t, all of the next may be on their way)
        else wait_vm<N>();
        u32x4 k[2][D / 64];
        f32x4 scale[2], s[R][2];
        w.read_k(k, mine, stage);
        w.read_scales(scale, mine, stage);
        f32x4 v_scale[2];
        w.read_scales(v_scale, mine, stage + 128);
        lds_reads_done();
        if (two) copy.k(lds + stage);
        w.scores(s, k, scale);
        if ((t + 1) * T::BN > clean) {
#pragma unroll
            for (int b = 0; b < R; ++b) w.exclude(s[b], copy.lane, limit[b] - t * T::BN);
        }
        w.fold(s);
        bf16x8 pf[R];
        w.weights(s, v_scale, pf);
        if (two) wait_vm<3 * N + 1>();                 // V of t
        else if (one) wait_vm<2 * N + 1>();
        else wait_vm<0>();
        u32x2 v[D / 16];
        w.read_v(v, mine, stage);
        lds_reads_done();
        if (two) {
            copy.scales(lds + stage + T::S);
            copy.v(lds + stage + T::V);
        }
        w.add(v, pf);
    };
    for (int t = t_lo; t < t_hi; t += 2 * STEP) {
        step(t, std::integral_constant<int, 0>{});
        if (t + STEP < t_hi) step(t + STEP, std::integral_constant<int, 1>{});
    }
}
// ... its first two tiles
template <int STEP, int D, class P>
__device__ __forceinline__ void paged8_start(Paged8Copy<D, P>& copy, const uint8_t* mine, int t_lo, int t_hi) {
    using T = Paged8Tile<D>;
    const uint32_t lds = lds_addr(mine);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if (t_lo + i * STEP >= t_hi) break;
        copy.aim(t_lo + i * STEP);
        copy.k(lds + i * T::STAGE);
        copy.scales(lds + i * T::STAGE + T::S);
        copy.v(lds + i * T::STAGE + T::V);
    }
}
// This lane's rows of the blocks from row0 on attend to the keys below `limit`; returns below which key all rows do.
template <int R>
__device__ __forceinline__ int paged8_limits(const PagedParams& p, const PagedUnit& u, int lane, int row0, int (&limit)[R]) {
#pragma unroll
    for (int b = 0; b < R; ++b) limit[b] = u.own ? max(u.keys - u.lag + paged_row(p, u, min(row0 + 16 * b + (lane & 15), u.rows - 1)).i, 0) : u.keys;
    return u.own ? max(u.keys - u.lag, 0) : u.keys;
}

// A unit whose wavefronts walk keys of their own: as in attn_paged.hpp.
template <int D, int NW, bool STRIDED, int R, int CODE, class P>
__device__ __forceinline__ void paged8_unit(const P& p, const PagedUnit& u, uint8_t* lds, bool bad, bool direct, float* out_o, f32x2* out_ml) {
    using T = Paged8Tile<D>;
    constexpr int DB = D / 16, ROWS = 16 * R;
    const int tid = paged_thread(), lane = tid & 63, wave = packed_uniform(tid >> 6), n = lane & 15, g = lane >> 4;
    const uint8_t* const mine = lds + wave * T::WAVE;
    constexpr int STEP = STRIDED ? NW : 1;
    const int run = (u.tiles + NW - 1) / NW;
    const int t_lo = u.tile0 + (STRIDED ? wave : wave * run), t_hi = STRIDED ? u.tile0 + u.tiles : min(t_lo + run, u.tile0 + u.tiles);
    PagedPages pages;
    if (STRIDED || t_lo < t_hi) pages.load(p, u, lane, (t_lo * T::BN) >> p.page_shift);
    Paged8Copy<D, P> copy(p, u, pages, lane);
    paged8_start<STEP>(copy, mine, t_lo, t_hi);
    Paged8Rows<D, CODE, R> w;
    w.begin(p, u, lane, 0);
    int limit[R];
    const int clean = paged8_limits<R>(p, u, lane, 0, limit);
    paged8_walk<STEP>(copy, w, mine, t_lo, t_hi, limit, clean);

    // ---- the wavefronts' states become one
    __shared__ f32x2 state[NW][ROWS], joined[ROWS];
    const bool lost = __any(bad | (pages.bad && t_lo < t_hi));                    // a page outside the cache, or more keys than pages: NaN
#pragma unroll
    for (int b = 0; b < R; ++b) {
        w.l_run[b] = lost ? __builtin_nanf("") : w.over_groups_sum(w.l_run[b]);
        if (g == 0) state[wave][16 * b + n] = f32x2{w.m_run[b], w.l_run[b]};
    }
    __syncthreads();                                   // (no copy is under way: every wavefront has waited for its last one)
    float* const sums = reinterpret_cast<float*>(lds + wave * T::WAVE);           // [rows][D], granules of four swizzled by the row
#pragma unroll
    for (int b = 0; b < R; ++b) {
        float M = -INFINITY, L = 0.f;
#pragma unroll
        for (int i = 0; i < NW; ++i) M = fmaxf(M, state[i][16 * b + n][0]);
        const float M_to = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int i = 0; i < NW; ++i) L += state[i][16 * b + n][1] * exp2_fast((state[i][16 * b + n][0] - M_to) * w.c_log2);
        const float f = exp2_fast((w.m_run[b] - M_to) * w.c_log2);
#pragma unroll
        for (int db = 0; db < DB; ++db) *reinterpret_cast<f32x4*>(sums + (16 * b + n) * D + (((4 * db + g) ^ (n & 7)) << 2)) = w.oacc[b][db] * f;
        if (wave == 0 && g == 0) joined[16 * b + n] = f32x2{M * w.c_log2, L};
    }
    __syncthreads();
    for (int e = tid; e < u.rows * (D / 4); e += 64 * NW) {
        const int r = e / (D / 4), q = e % (D / 4);
        if (4 * q >= p.d) continue;
        f32x4 a = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < NW; ++i) a += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds + i * T::WAVE) + r * D + ((q ^ (r & 7)) << 2));
        if (direct) {
            const float l = joined[r][1], inv = l == 0.f ? 0.f : 1.0f / l;
            const PagedRow at = paged_row(p, u, r);
            *reinterpret_cast<u32x2*>(p.o + at.b * p.os.b + at.h * p.os.h + at.i * p.os.n + 4 * q) = u32x2{pack_bf16(a[0] * inv, a[1] * inv), pack_bf16(a[2] * inv, a[3] * inv)};
        } else {
            *reinterpret_cast<f32x4*>(out_o + (int64_t)r * p.d + 4 * q) = a;
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
// Own keys: R blocks; a prefix, whose rows are those of several sequences: two.
template <int D, int NW, bool STRIDED, int CODE, int R>
__device__ __forceinline__ void paged_unit_body(const Paged8Params<CODE, R>& p, const PagedUnit& u, uint16_t* lds, bool bad, bool direct, float* out_o, f32x2* out_ml) {
    if (STRIDED || u.own || R == 2) paged8_unit<D, NW, STRIDED, R, CODE>(p, u, reinterpret_cast<uint8_t*>(lds), bad, direct, out_o, out_ml);
    else paged8_unit<D, NW, STRIDED, 2, CODE>(p, u, reinterpret_cast<uint8_t*>(lds), bad, direct, out_o, out_ml);
}

// A unit of the prefix with 128 rows: the wavefronts have 32 each and share the tiles, as those of the bf16 cache do (attn_paged.hpp), in blocks of 32 rows.
// Every wavefront converts a quarter of a tile, on the way from its registers to LDS: eight rows of K and of V, which it has requested two tiles ahead.
// Three stages: tile t is in stage t % 3; behind the barrier of tile t, tile t + 1 is there and the stage of tile t - 1 free for tile t + 2.  Loads past the
// last tile re-read it.
// (Each wavefront with tiles of its own -> shared, us, 64 answers on a prefix of 8192, D = 128: int8 41.8 -> 39.8, e4m3 38.6 -> 36.4.)
template <int D, int CODE, int R>
__device__ __forceinline__ void paged_shared_body(const Paged8Params<CODE, R>& p, const PagedUnit& u, uint16_t* lds, bool bad, float* out_o, f32x2* out_ml) {
    using B16 = PagedTile<D>;
    constexpr int DC = D / 16, DB = D / 32, PIECE = D / 8, TILE = B16::TILE_ELEMS, STAGE = 2 * TILE + 128;       // PIECE: bytes of a lane; 16-bit elements of a stage
    static_assert(3 * STAGE * 2 <= Paged8Tile<D>::lds_bytes(4), "three stages");
    const int tid = paged_thread(), lane = tid & 63, wave = packed_uniform(tid >> 6), n = lane & 31, h = lane >> 5;
    const uint8_t* const k_base = p.k8 + u.kv_head * p.ks.h;
    const uint8_t* const v_base = p.v8 + u.kv_head * p.vs.h;
    const int my_row = 8 * wave + (lane >> 3), column = (lane & 7) * PIECE, from_column = column < p.d ? column : 0;      // (columns past d meet zeros of Q or are not stored)
    const int t_hi = u.tile0 + u.tiles, rows = min(32, u.rows - 32 * wave);
    const float* const s_base = lane < 32 ? reinterpret_cast<const float*>(reinterpret_cast<const char*>(p.k_scale) + u.kv_head * p.kss.h)
                                          : reinterpret_cast<const float*>(reinterpret_cast<const char*>(p.v_scale) + u.kv_head * p.vss.h);
    const int s_page = (int)(lane < 32 ? p.kss.b : p.vss.b), s_block = (int)(lane < 32 ? p.kss.n : p.vss.n);
    PagedPages pages;
    pages.load(p, u, lane, (u.tile0 * 32) >> p.page_shift);
    uint32_t piece[2][2][PIECE / 4];                   // of tiles t and t + 1: K, V
    float scale[2];
    auto request = [&](int t, uint32_t (&w)[2][PIECE / 4], float& sc) {
        const int key0 = min(t, t_hi - 1) * 32, most = u.keys - 1 - key0, mask = (1 << p.page_shift) - 1;
        if (!pages.holds(p, key0 + 31)) pages.load(p, u, lane, key0 >> p.page_shift);
        const int e0 = __builtin_amdgcn_readlane(pages.mine, (key0 >> p.page_shift) - pages.first);
        const int e1 = most >= 16 ? __builtin_amdgcn_readlane(pages.mine, ((key0 + 16) >> p.page_shift) - pages.first) : e0;
        const int key = min(my_row, most), e = key < 16 ? e0 : e1, token = (key0 + key) & mask;
        const uint8_t* const k = k_base + e * p.ks.b + token * p.ks.n + from_column;
        const uint8_t* const v = v_base + e * p.vs.b + token * p.vs.n + from_column;
        if constexpr (PIECE == 16) {
            const u32x4 a = *reinterpret_cast<const u32x4*>(k), b = *reinterpret_cast<const u32x4*>(v);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[0][i] = a[i], w[1][i] = b[i];
        } else {
            const u32x2 a = *reinterpret_cast<const u32x2*>(k), b = *reinterpret_cast<const u32x2*>(v);
#pragma unroll
            for (int i = 0; i < 2; ++i) w[0][i] = a[i], w[1][i] = b[i];
        }
        if (wave == 0) {
            const int at = min(lane & 31, most), page = at < 16 ? e0 : e1;
            sc = *reinterpret_cast<const float*>(reinterpret_cast<const char*>(s_base) + (int64_t)page * s_page +
                                                 (int64_t)(((key0 + at) & mask) >> p.block_shift) * s_block);
        }
    };
    auto stage_of = [&](int t) { return lds + (t - u.tile0) % 3 * STAGE; };
    auto place = [&](int t, const uint32_t (&w)[2][PIECE / 4], float sc) {
        uint16_t* const to = stage_of(t);
#pragma unroll
        for (int x = 0; x < 2; ++x)
#pragma unroll
            for (int i = 0; i < PIECE / 8; ++i) {
                const int granule = column / 8 + i;
                *reinterpret_cast<bf16x8*>(to + x * TILE + my_row * B16::RS + ((granule ^ swz<D>(my_row)) << 3)) = codes_to_bf16<CODE>(w[x][2 * i], w[x][2 * i + 1]);
            }
        if (wave == 0) reinterpret_cast<float*>(to + 2 * TILE)[lane] = sc;
    };
    auto together = [&]() {                            // everyone has read and written what comes before
        lds_reads_done();
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
    };
    request(u.tile0, piece[0], scale[0]);
    request(u.tile0 + 1, piece[1], scale[1]);
    const PagedRow me = paged_row(p, u, min(32 * wave + n, u.rows - 1));
    PagedRows<D> w;
    w.begin(p, lane, me, n < rows);
    place(u.tile0, piece[0], scale[0]);
    request(u.tile0 + 2, piece[0], scale[0]);
    place(u.tile0 + 1, piece[1], scale[1]);
    request(u.tile0 + 3, piece[1], scale[1]);
    auto scores_of = [&](int t) {
        const uint16_t* const tile = stage_of(t);
        bf16x8 kf[DC];
        w.read_k(kf, tile);
        f32x16 s = w.scores(kf);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 of = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(tile + 2 * TILE) + 8 * i + 4 * h);
#pragma unroll
            for (int r = 0; r < 4; ++r) s[4 * i + r] *= of[r];
        }
        return s;
    };
    together();
    f32x16 s = scores_of(u.tile0);
    if (32 > u.keys - u.tile0 * 32) w.exclude(s, lane, u.keys - u.tile0 * 32);
    w.fold(s);
    auto step = [&](int t, uint32_t (&pc)[2][PIECE / 4], float& sc) {
        if (t != u.tile0) together();
        place(t + 2, pc, sc);
        request(t + 4, pc, sc);
        f32x16 next = scores_of(t + 1);                // (after the last tile: of the last one again, which nobody uses)
        const uint16_t* const tile = stage_of(t);
        // as PagedRows::weights, and V's scales
        const float shift = (w.m_run == -INFINITY ? 0.f : w.m_run) * w.c_log2;
        float sum[2] = {0.f, 0.f};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4 of = *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(tile + 2 * TILE) + 32 + 8 * i + 4 * h);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float e = exp2_fast(fmaf(s[4 * i + r], w.c_log2, -shift));
                sum[r & 1] += e;
                s[4 * i + r] = e * of[r];
            }
        }
        w.l_run += sum[0] + sum[1];
        w.add16(tile + TILE, 0, pack8(s[0], s[1], s[2], s[3], s[4], s[5], s[6], s[7]));
        w.add16(tile + TILE, 1, pack8(s[8], s[9], s[10], s[11], s[12], s[13], s[14], s[15]));
        s = next;
        if (t + 1 < t_hi) {
            if ((t + 2) * 32 > u.keys) w.exclude(s, lane, u.keys - (t + 1) * 32);
            w.fold(s);
        }
    };
    for (int t = u.tile0; t < t_hi; t += 2) {
        step(t, piece[0], scale[0]);
        if (t + 1 < t_hi) step(t + 1, piece[1], scale[1]);
    }
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

// Without a prefix: all tiles of all walks (sequence by sequence, key head by key head, one tile of rows after the other) are cut into ranges of the same
// length, one for every workgroup that runs at once, whatever the sequences' lengths.  A walk that lies in one range is written by its workgroup, the
// others' parts are joined by the merge; a range has at most one walk that began before it and one that goes on behind it.
// (In units of up to 64 tiles dealt in turn -> in ranges, us, D = 128, e4m3, 64 sequences of 2000 to 6000 114 -> 105, of 8000 194 -> 185 (5.7 TB/s), one of
// 131072 61 -> 58; in int8 117 -> 107, 197 -> 189, 63 -> 60.)
template <int D>
constexpr int kPaged8Groups = D <= 64 ? 3 : 2;         // workgroups on a compute unit
template <int D, class P>
__global__ __launch_bounds__(256, kPaged8Groups<D>) void paged_ranges_kernel(const P p) {
    extern __shared__ __attribute__((aligned(1024))) uint16_t lds[];
    __shared__ int sums[4], found[4];
    const int rows = p.N * (p.H / p.Hkv), rt = PagedCut::row_tiles(rows), heads = p.Hkv * rt, slot_rows = min(32, rows), most = p.table_pages << p.page_shift;
    const PagedPlan c = paged_plan(p, sums);
    const int share = packed_uniform(max(PagedCut::kLeast, (int)((c.own_tiles + gridDim.x - 1) / gridDim.x)));
    const int range = (int)blockIdx.x;                 // (ranges one behind the other on one XCD: no gain, also where its heads' rows share lines)
    int at = min(range * share, c.own_tiles);
    const int end = min(at + share, c.own_tiles);
    if (range != 0 && at >= end) return;
    if (threadIdx.x == 0) found[0] = -1;               // (what the lengths, read again, always replace unless somebody changes them meanwhile)
    paged_own_units(p, c, sums, [](int tiles) { return tiles; }, [&](int b, int len, int first, int tiles) {
        if (at >= first && at < first + tiles * heads) {
            found[0] = b;
            found[1] = first;
            found[2] = tiles;
            found[3] = len;
        }
        if (range == 0) p.plan[b] = int2{first, tiles};
    });
    if (range == 0 && threadIdx.x == 0) p.plan[p.B] = int2{share, 0};
    if (at >= end) return;
    __syncthreads();
    int b = packed_uniform(found[0]), tiles = packed_uniform(found[2]), len = packed_uniform(found[3]);
    if (b < 0) return;
    int pair = packed_uniform((at - found[1]) / tiles), tile0 = packed_uniform(at - found[1]) - pair * tiles;
    while (true) {
        PagedUnit u;
        u.own = true;
        u.table = p.table + b * p.table_stride;
        u.entries = p.table_pages;
        u.keys = min(max(len, 0), most);
        u.kv_head = packed_uniform(pair / rt);
        u.row0 = 32 * (pair - u.kv_head * rt);
        u.rows = min(32, rows - u.row0);
        u.b0 = b;
        u.lag = p.N - 1;
        u.tile0 = tile0;
        u.tiles = min(tiles - tile0, end - at);
        const int64_t slot = p.own_slot + (int64_t)(2 * range + (tile0 == 0)) * slot_rows;
        paged_unit_body<D, 4, false>(p, u, lds, len > most, u.tiles == tiles, p.part_o + slot * p.d, p.part_ml + slot);
        at += u.tiles;
        if (at >= end) return;
        tile0 = 0;
        if (++pair == heads) {
            pair = tiles = 0;
            while (tiles == 0 && ++b < p.B) {          // (there is another one with keys: the range goes on)
                len = packed_uniform(p.kv_len[b]);
                tiles = paged_tiles(min(max(len, 0), most));
            }
            if (tiles == 0) return;
        }
        __syncthreads();                               // the last unit's LDS is free
    }
}

}  // namespace fattn
