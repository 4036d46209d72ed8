// Backward of the tiled attention for gfx950: recomputes P tile by tile from Q, K and the saved
// log-sum-exp, never materialising the Sq x Sk matrix.
//
//   dq       one workgroup owns 128 queries (32 per wavefront, two wavefronts per SIMD) or, when the
//            problem fills them, 256 queries (64 per wavefront, one wavefront per SIMD), and walks over
//            the key tiles (64 keys), with the logits transposed (lane = query): S^T = K Q^T, dP^T = V dO^T,
//            dS^T = P^T (dP^T - delta) and dQ^T += K^T dS^T accumulated in fp32 registers for the whole
//            walk, dS^T going into the last MFMA straight from the accumulators.  Runs first and also
//            leaves -delta_i = -sum_d dO_id * O_id and LSE_i * log2(e) (fp32, one value per query row)
//            in the workspace for the next kernel.
//   dkdv     one workgroup owns 128 keys (32 per wavefront) of one (batch, head) and walks over the
//            query tiles (64 rows): S = Q K^T, dP = dO V^T, P = exp2(S*c - LSE*log2e),
//            dS = P * (dP - delta); dV^T += dO^T P and dK^T += Q^T dS stay in fp32 registers for the
//            whole walk (P and dS are used as MFMA operands straight from the accumulators), and so do
//            the wavefront's K and V fragments (in the accumulation registers).  When the
//            key blocks do not fill the last scheduling round, the blocks of that round are split
//            along the walk and their fp32 partial sums are combined by the merge kernel.
// Accumulating dQ from the dkdv walk with fp32 atomics was measured at about one lane-atomic per
// clock per CU, more than the whole MFMA time of the backward; recomputing S and dP in a second,
// query-major kernel costs 2 extra GEMMs out of 7 and no atomics, no fp32 scratch and no convert pass.
//
// Tiles are copied global -> LDS by asynchronous LDS-DMA loads (two stages where two wavefronts share a
// SIMD, three where one wavefront runs alone and nobody would cover a drained pipeline), row-major with an XOR swizzle of the 16-byte granules; their
// transposed MFMA operands (Q^T, dO^T) and the dS operand come from transposing LDS reads, so no tile
// is stored twice and no access pattern has bank conflicts.  One workgroup barrier per step.
#pragma once
#include <type_traits>

#include "attn_common.hpp"
#include "packed_units.hpp"

namespace fattn {

struct BwdParams {
    // dK/dV grid: workgroups [0, n_whole) walk every query tile of one key block; the remaining key
    // blocks are served by split_parts workgroups each, every one walking a slice of the query tiles
    // and leaving fp32 partial sums in split_ws for bwd_dkdv_merge_kernel.  n_whole < 0: no splitting.
    int n_whole = -1;
    int split_parts = 1;
    int rows_ready = 0;            // -delta and lse2 are in the workspace already (bwd_rows_kernel ran): read, do not form
    int dq_base = 0;               // the dQ launch covers the problem's workgroups from this one on (problems without exclusions only)
    int dq_parts = 1;              // workgroups that share the key walk of one 128-query tile, leaving fp32 partial sums in split_ws
    int joint_n_dq = 0;            // bwd_joint_kernel: the first joint_n_dq workgroups are dQ workgroups
    float* split_ws = nullptr;
    size_t split_ws_bytes = 0;     // host side only
    float dv_scale = 1.f;          // merge kernel: what the sums of dV are multiplied by (dropout: 1 / (1 - p))
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    const uint16_t* o;
    const uint16_t* dout;
    const float* lse;     // contiguous [B*H, Sq]
    uint16_t* dq;
    uint16_t* dk;
    uint16_t* dv;
    float* ndelta;        // workspace, [B*H, Sq]: -rowsum(dO * O)
    float* lse2;          // workspace, [B*H, Sq]: LSE * log2(e), +inf where LSE = -inf
    Strides qs, ks, vs, os, dos, dqs, dks, dvs;
    int B, H, Sq, Sk;
    int d;                // real head dim: a multiple of 8, at most the compiled D
    float scale;
    MaskArgs m;
    int key_mask = 0;     // m.mask is the same for every query: kernels without the general mask code serve it
    unsigned long long* phase_cycles;   // profiling aid: per-phase cycle sums of wave 0 of every workgroup, or null
};

// ------------------------------------------------------------------------------------------ dkdv
template <int D>
struct BwdTile {
    static constexpr int BM = 64;                   // query rows per step
    static constexpr int BN = 128;                  // keys per workgroup
    static constexpr int RS = kRowPitch<D>;         // LDS row stride of the Q / dO / K / V tiles (swizzled)
    static constexpr int Q_ELEMS = BM * RS;
    static constexpr int STAGE_ELEMS = 2 * Q_ELEMS;               // Q tile + dO tile (also one 128-row tile)
    static constexpr int ROW_FLOATS = 2 * BM;                     // lse2 and -delta of one step
    static constexpr int NSTAGE = 3;
    // [3 stages of Q,dO][3 x (lse2, -delta)]
    static constexpr int LDS_BYTES = NSTAGE * STAGE_ELEMS * 2 + NSTAGE * ROW_FLOATS * 4;
    // with a keep-mask staged through LDS: [3 x (64 queries x 128 keys) mask bytes] behind the rest
    static constexpr int MASK_STAGE_BYTES = BM * BN;
    static constexpr int LDS_BYTES_VECMASK = LDS_BYTES + NSTAGE * MASK_STAGE_BYTES;
    // kDropRows64: the generator's word of every query row at each wavefront's first key, behind the rest
    static constexpr int LDS_BYTES_DROP = LDS_BYTES + 4 * BM * 4;
    static constexpr int ROWS_PER_DMA = 1024 / (RS * 2);
    static constexpr int DMA_PER_WAVE = BM / ROWS_PER_DMA / 4;    // 1 KiB copies per wave and tensor
};

template <int D>
__device__ __forceinline__ void dkdv_store(const BwdParams& p, uint16_t* own, const f32x16 (&dkacc)[D / 32], const f32x16 (&dvacc)[D / 32],
                                           uint16_t* dkbase, uint16_t* dvbase, int Sk, int kw0, float dv_scale = 1.0f);

// VECMASK (with HASMASK): the keep-mask rows are contiguous and 16-byte aligned, Sq is a multiple of 64, Sk
// of 128, and there is no causal flag.  The 64 x 128 mask bytes of a step then travel to LDS with the step's other copies (two more
// 1 KiB copies per wavefront) and every lane reads the bytes of its key a few elements ahead of use,
// instead of fetching 32 bytes from global memory into 32 registers at the start of every step; with the
// registers back, the walk runs the same straight-line steps as the unmasked one.
// DROP (DropMode): dV takes the dropped and rescaled probabilities, dP = f (dO V^T) with the same factor f (drop_factor), and
// -delta is added per element instead of seeding the dP accumulators.
// BITS: a keep-mask as bits (mask_bits.hpp): the walk takes the query tiles of which anything attends to one of the 128 keys, the
// cut ones first, and a lane has one word of its key for every cut one.
// DEALT: the units come in the order of causal_order.hpp (deals_units, which the host asks).
// block / nblocks: this workgroup's index in the dK/dV grid and the size of that grid (the kernel's own launch, or
// the dK/dV part of bwd_joint_kernel's).
// PACKED: the unit is a key block of one of several sequences of different lengths (packed_units.hpp), `u`, and the walk goes
// through the query tiles of the u.rep heads that share the key head: the cut tiles of all heads, then the others head by head, all
// into the same sums.
template <int D, bool HASMASK, bool TIMING, bool VECMASK = false, int DROP = kDropNone, bool BITS = false, bool DEALT = false, bool PACKED = false>
__device__ __forceinline__ void bwd_dkdv_body(const BwdParams& p, const int block, const int nblocks, const PackedUnit& u = PackedUnit()) {
    static_assert(!PACKED || (!HASMASK && !BITS && !DEALT && !TIMING && DROP == kDropNone), "packed sequences: causal flag and lengths only");
    static_assert(!VECMASK || HASMASK, "VECMASK is a special case of HASMASK");
    static_assert(!BITS || (!HASMASK && DROP == kDropNone), "bits stand for the mask");
    constexpr bool DROPOUT = DROP != kDropNone;
    using T = BwdTile<D>;
    constexpr int BM = T::BM, BN = T::BN, RS = T::RS;
    constexpr int DC = D / 16;     // contraction chunks over the head dim
    constexpr int DB = D / 32;     // 32-row blocks of dK^T / dV^T
    constexpr int GPR = RS / 8;    // 16-byte granules per row in LDS
    constexpr int RPD = T::ROWS_PER_DMA, NDQ = T::DMA_PER_WAVE;

    extern __shared__ __attribute__((aligned(1024))) uint16_t lds[];
    uint16_t* stage0 = lds;                                        // [3][Q tile | dO tile]
    float* rows0 = reinterpret_cast<float*>(lds + T::NSTAGE * T::STAGE_ELEMS);   // [3][lse2 | -delta]
    const uint8_t* mask0 = reinterpret_cast<const uint8_t*>(lds) + T::LDS_BYTES;  // [3][64 x 128] mask bytes (VECMASK)

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;

    const int Sq = PACKED ? u.Sq : p.Sq, Sk = PACKED ? u.Sk : p.Sk;
    const int past = PACKED ? u.past : 0;             // under the causal flag query i attends to key j <= i + past
    const int n_kt = (Sk + BN - 1) / BN;
    int wg = 0, part = 0, nparts = 1;
    if constexpr (PACKED) {
        wg = u.unit;
        part = u.part;
    } else if (p.n_whole < 0) {
        wg = xcd_remap_heads(block, nblocks, n_kt, p.m.kv_len || p.key_mask, false);
    } else if (block < p.n_whole) {
        wg = xcd_remap(block, p.n_whole);
    } else {          // the split key blocks come last in dispatch order and fill the final, partial round (or are all there is)
        const int e = p.n_whole == 0 ? xcd_remap_split(block, nblocks) : block - p.n_whole;
        nparts = p.split_parts;
        wg = p.n_whole + e / nparts;
        part = e % nparts;
    }
    int kt = PACKED ? u.tile : wg % n_kt, bh = PACKED ? 0 : wg / n_kt;
    if constexpr (DEALT) {       // under the causal flag the first key blocks have the longest walks
        int t, s;
        dealt_unit(block, n_kt, p.B, p.H, p.m.kv_len || p.key_mask, t, s);
        kt = __builtin_amdgcn_readfirstlane(t);
        bh = __builtin_amdgcn_readfirstlane(s);
    }
    const int b = bh / p.H, hh = bh % p.H;
    const int k0 = kt * BN;
    const int kw0 = k0 + 32 * wave;

    // PACKED: of the first head that shares this key head
    const uint16_t* qbase = PACKED ? p.q + u.q_at(p.qs) : p.q + b * p.qs.b + hh * p.qs.h;
    const uint16_t* kbase = PACKED ? p.k + u.k_at(p.ks) : p.k + b * p.ks.b + hh * p.ks.h;
    const uint16_t* vbase = PACKED ? p.v + u.k_at(p.vs) : p.v + b * p.vs.b + hh * p.vs.h;
    const uint16_t* dobase = PACKED ? p.dout + u.q_at(p.dos) : p.dout + b * p.dos.b + hh * p.dos.h;
    const float* lsebase = p.lse2 + (PACKED ? u.stat_row() : (int64_t)bh * p.Sq);
    const float* ndeltabase = p.ndelta + (PACKED ? u.stat_row() : (int64_t)bh * p.Sq);
    auto store_rows = [&](const f32x16 (&dkacc)[D / 32], const f32x16 (&dvacc)[D / 32], float dv_scale) {
        uint16_t* const dkbase = PACKED ? p.dk + u.k_at(p.dks) : p.dk + b * p.dks.b + hh * p.dks.h;
        uint16_t* const dvbase = PACKED ? p.dv + u.k_at(p.dvs) : p.dv + b * p.dvs.b + hh * p.dvs.h;
        dkdv_store<D>(p, lds + wave * 32 * RS, dkacc, dvacc, dkbase, dvbase, Sk, kw0, dv_scale);
    };

    int klimit = Sk;
    if (!PACKED && p.m.kv_len) klimit = min(klimit, max(p.m.kv_len[b], 0));
    const uint8_t* mbase = HASMASK ? mask_head_base(p.m, b, hh) : nullptr;

    // A keep-mask of keys is a key length with holes: a lane owns one key, so its P and dS need no test, and the columns of
    // the excluded keys are zeroed before the store.  Two loads per wavefront tell whether any of the 128 keys is attended.
    bool dead = false;
    uint64_t any_alive = ~0ull;
    if (!HASMASK && !PACKED && p.key_mask) {
        const uint8_t* kmask = mask_head_base(p.m, b, hh);
        bool alive[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const int kk = k0 + 64 * u + lane;
            alive[u] = kk < klimit && mask_attends(p.m, kmask, (int64_t)min(kk, p.Sk - 1) * p.m.sk);
        }
        const uint64_t b0 = __ballot(alive[0]), b1 = __ballot(alive[1]);
        any_alive = b0 | b1;
        dead = ((((wave & 2) ? b1 : b0) >> (32 * (wave & 1) + n)) & 1ull) == 0;
    }
    const int n_qt = (Sq + BM - 1) / BM;
    int qt_begin = p.m.causal && !BITS ? (PACKED ? max(k0 - past, 0) : k0) / BM : 0;
    KeyTiles qtiles;                       // BITS: of queries
    const uint64_t* bcols = nullptr;       // this lane's key's word of query tile 0; tiles lie 64 bit_nkt words apart
    if constexpr (BITS) {
        const int plane = b * p.m.plane_b + hh * p.m.plane_h;
        const uint8_t* flags = p.m.tile_flags + (int64_t)plane * p.m.bit_nqt * p.m.bit_nkt + k0 / 64;
        qtiles.build_of_tiles(reinterpret_cast<char*>(lds) + T::LDS_BYTES, n_qt, [&](int u) {
            const int f0 = flags[(int64_t)u * p.m.bit_nkt], f1 = flags[(int64_t)u * p.m.bit_nkt + 1];
            return f0 & f1 & kTileAllRows ? 2 : (f0 | f1) & kTileAny ? 1 : 0;
        });
        bcols = p.m.bit_cols + (int64_t)plane * p.m.bit_nqt * (64 * p.m.bit_nkt) + kw0 + n;
        if (qtiles.n_tiles == 0) any_alive = 0;
    }
    if (k0 >= klimit || any_alive == 0 || (PACKED ? qt_begin >= n_qt : !BITS && p.m.causal && k0 >= p.Sq)) {
        // Nothing attends to these keys (past the key length, masked, or past the last query under the causal flag):
        // dK = dV = 0, written at once.  Padded batches launch many such workgroups; they must not cost a
        // prologue each.
        f32x16 zero[D / 32];
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) zero[db][r] = 0.f;
        if (!PACKED || part == 0) store_rows(zero, zero, 1.0f);
        return;
    }
    const int rep = PACKED ? u.rep : 1;
    const int n_it_head = BITS ? qtiles.n_tiles : n_qt - qt_begin, n_it = rep * n_it_head;
    if constexpr (PACKED) {
        nparts = packed_parts(u, n_it);
        if (part >= nparts) return;
    }
    // The walk visits the query tiles that need per-element exclusions first (all of them when an explicit
    // mask is given, else the causal diagonal tiles and a partial last tile) and the fully attended ones afterwards, so that each of the two loops runs one
    // specialised, branch-free body.  The order of the tiles does not matter to the sums.
    // (A key block that the key length cuts needs none: a lane owns one key, its column of dK^T / dV^T
    // depends on no other key's P or dS, and the columns of the keys past the length are zeroed before the store.)
    const bool all_masked = HASMASK;
    int lead_end = qt_begin;
    if (n_it > 0) {
        if (BITS) lead_end = n_it - qtiles.n_whole;
        else if (all_masked) lead_end = n_qt;
        else if (PACKED && p.m.causal) lead_end = max(qt_begin, min(n_qt, (max(k0 + BN - 1 - past, 0) + BM - 1) / BM));
        else if (p.m.causal) lead_end = max(qt_begin, min(n_qt, (k0 + BN - 2) / BM + 1));
    }
    const int n_lead = lead_end - qt_begin;
    const int tail_extra = (n_it > 0 && !BITS && !all_masked && (Sq % BM) != 0 && lead_end < n_qt) ? 1 : 0;
    const int n_masked_head = n_lead + tail_extra, n_masked = rep * n_masked_head;
    const int n_full_head = PACKED ? max(n_it_head - n_masked_head, 1) : 1;       // (divisors)
    const int n_cut_head = PACKED ? max(n_masked_head, 1) : 1;
    auto tile_of = [&](int it) {
        if constexpr (PACKED) {
            const int j = packed_uniform(it < n_masked ? it % n_cut_head : (it - n_masked) % n_full_head);
            const int full = lead_end + j, cut = qt_begin + j, last = n_qt - 1, lead = n_lead;       // (values: the compiler would choose among addresses)
            return it >= n_masked ? full : j < lead ? cut : last;
        }
        if constexpr (BITS) return qtiles.tile(it < n_masked ? qtiles.n_whole + it : it - n_masked);
        if (it < n_lead) return qt_begin + it;
        if (it < n_masked) return n_qt - 1;
        return lead_end + (it - n_masked);
    };
    auto head_of = [&](int it) {           // PACKED: of step `it`, counted from u.head
        if constexpr (PACKED) return packed_uniform(it < n_masked ? it / n_cut_head : (it - n_masked) / n_full_head);
        else return 0;
    };
    // ---- per-lane LDS offsets (elements), constant over the walk
    int roff[DC];          // 16-byte row reads: row (32*blk + n), logical granule 2*dc + h
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) roff[dc] = n * RS + (((2 * dc + h) ^ swz<D>(n)) << 3);
    const int tr_r = lane & 15, tr_g16 = (lane >> 4) & 1;
    int toff[2][DB];       // transposing reads of a D-wide tile: rows 4h + r/4 (+8), granule 4*db + 2*g16 + (r&3)/2
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int row = 4 * h + (tr_r >> 2) + 8 * half;
#pragma unroll
        for (int db = 0; db < DB; ++db)
            toff[half][db] = row * RS + (((4 * db + 2 * tr_g16 + ((tr_r & 3) >> 1)) ^ swz<D>(row)) << 3) + 4 * (tr_r & 1);
    }
    auto tr_frag = [&](const uint16_t* tile, int o0, int o1) {
        const u32x2 lo = lds_read_tr16(tile + o0);
        const u32x2 hi = lds_read_tr16(tile + o1);
        const u32x4 u = {lo[0], lo[1], hi[0], hi[1]};
        return __builtin_bit_cast(bf16x8, u);
    };

    const int dma_row_in = lane / GPR, dma_gran = lane % GPR;
    const uint32_t lds0 = lds_addr(lds);
    const uint32_t rows_lds0 = lds0 + 2u * T::NSTAGE * T::STAGE_ELEMS;   // byte address of rows0

    // ---- prologue: the K and V fragments of this wavefront's 32 keys are held in registers for the whole walk
    bf16x8 kf[DC], vf[DC];
    {
        constexpr int NDMA = BN / RPD / 4;     // 1 KiB copies per wave for a 128-row tile
#pragma unroll
        for (int i = 0; i < NDMA; ++i) {
            const int ji = wave * NDMA + i;
            const int row = ji * RPD + dma_row_in;
            const int key = max(min(k0 + row, klimit - 1), 0);   // rows past the attended range re-read a valid row
            const int c = src_granule(dma_gran ^ swz<D>(row), p.d);
            dma16(kbase + (int64_t)key * p.ks.n + c * 8, lds0 + 2u * (T::STAGE_ELEMS + ji * 512));
            dma16(vbase + (int64_t)key * p.vs.n + c * 8, lds0 + 2u * (ji * 512));
        }
        wait_vm0();
        __syncthreads();
        if (p.d < D) {      // padded head dim: S and dP must not see the copies' filler, so it is zeroed in LDS
            const u32x4 z = {0u, 0u, 0u, 0u};
            for (int idx = tid; idx < BN * GPR; idx += 256) {
                const int row = idx / GPR, gl = idx % GPR;
                if (gl * 8 >= p.d) {
                    const int off = row * RS + ((gl ^ swz<D>(row)) << 3);
                    *reinterpret_cast<u32x4*>(stage0 + off) = z;
                    *reinterpret_cast<u32x4*>(stage0 + T::STAGE_ELEMS + off) = z;
                }
            }
            __syncthreads();
        }
#pragma unroll
        for (int dc = 0; dc < DC; ++dc) {
            kf[dc] = *reinterpret_cast<const bf16x8*>(stage0 + T::STAGE_ELEMS + roff[dc] + 32 * wave * RS);
            vf[dc] = *reinterpret_cast<const bf16x8*>(stage0 + roff[dc] + 32 * wave * RS);
        }
        __syncthreads();
    }

    // ---- asynchronous staging of the 64-row Q / dO tiles and their lse2 / -delta rows, three stages.
    //      Address = uniform tile base + a per-lane 32-bit offset that never changes.
    uint32_t q_lane_off[NDQ], do_lane_off[NDQ];     // bytes
#pragma unroll
    for (int i = 0; i < NDQ; ++i) {
        const int row = (wave * NDQ + i) * RPD + dma_row_in;
        const int c = src_granule(dma_gran ^ swz<D>(row), p.d);
        q_lane_off[i] = 2u * (uint32_t)(row * (int)p.qs.n + c * 8);
        do_lane_off[i] = 2u * (uint32_t)(row * (int)p.dos.n + c * 8);
    }
    auto q_dst = [&](int stg, int which, int i) {    // LDS byte address of copy i of this wave (which: 0 = Q, 1 = dO)
        return lds0 + 2u * (uint32_t)(stg * T::STAGE_ELEMS + which * T::Q_ELEMS + (wave * NDQ + i) * 512);
    };
    auto rows_dst = [&](int stg) { return rows_lds0 + 4u * (uint32_t)(stg * T::ROW_FLOATS + wave * BM); };
    // keep-mask tile of a step: 8 copies of 8 rows x 128 bytes, two per wavefront
    uint32_t m_lane_off[2] = {0u, 0u};
    if (VECMASK) {
#pragma unroll
        for (int jm = 0; jm < 2; ++jm)
            m_lane_off[jm] = (uint32_t)(((wave * 2 + jm) * 8 + (lane >> 3)) * (int)p.m.sq + 16 * (lane & 7));
    }
    auto mask_dst = [&](int stg, int jm) {
        return lds0 + (uint32_t)(T::LDS_BYTES + stg * T::MASK_STAGE_BYTES + (wave * 2 + jm) * 1024);
    };
    auto mask_tile = [&](int qt) { return mbase + (int64_t)qt * BM * p.m.sq + k0; };
    auto issue_q_tile = [&](int qt, int head, int stg) {
        const int q0 = qt * BM;
        const uint16_t* const qhead = PACKED ? qbase + head * p.qs.h : qbase;
        const uint16_t* const dohead = PACKED ? dobase + head * p.dos.h : dobase;
        const float* const lsehead = PACKED ? lsebase + (int64_t)head * u.total_q : lsebase;
        const float* const ndeltahead = PACKED ? ndeltabase + (int64_t)head * u.total_q : ndeltabase;
        if (q0 + BM <= Sq) {
            const uint16_t* qt_base = qhead + (int64_t)q0 * p.qs.n;
            const uint16_t* dot_base = dohead + (int64_t)q0 * p.dos.n;
#pragma unroll
            for (int i = 0; i < NDQ; ++i) {
                dma16u(qt_base, q_lane_off[i], q_dst(stg, 0, i));
                dma16u(dot_base, do_lane_off[i], q_dst(stg, 1, i));
            }
            if (wave < 2) dma4((wave == 0 ? lsehead : ndeltahead) + q0 + lane, rows_dst(stg));
            if (VECMASK) {
#pragma unroll
                for (int jm = 0; jm < 2; ++jm) dma16u(mask_tile(qt), m_lane_off[jm], mask_dst(stg, jm));
            }
        } else {   // last, partial tile: rows past the end re-read the last valid row
#pragma unroll
            for (int i = 0; i < NDQ; ++i) {
                const int ji = wave * NDQ + i;
                const int row = ji * RPD + dma_row_in;
                const int qi = min(q0 + row, Sq - 1);
                const int c = src_granule(dma_gran ^ swz<D>(row), p.d);
                dma16(qhead + (int64_t)qi * p.qs.n + c * 8, q_dst(stg, 0, i));
                dma16(dohead + (int64_t)qi * p.dos.n + c * 8, q_dst(stg, 1, i));
            }
            if (wave < 2) {
                const int qi = min(q0 + lane, Sq - 1);
                dma4((wave == 0 ? lsehead : ndeltahead) + qi, rows_dst(stg));
            }
        }
    };

    f32x16 dkacc[DB], dvacc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
            dkacc[db][r] = 0.f;
            dvacc[db][r] = 0.f;
        }

    const float c_log2 = p.scale * kLog2e;
    const int key = kw0 + n;
    const uint32_t drop_lane = xorshift32((uint32_t)n);
    (void)drop_lane;
    // VECMASK: a mask byte excludes its element when it is <= this: 0 for an attended key, 255 for one past the key length
    const uint32_t dead_thr = key >= klimit ? 0xffu : 0u;

    unsigned long long ph[6] = {0, 0, 0, 0, 0, 0};
    unsigned long long tprev = TIMING ? __builtin_readcyclecounter() : 0ull;
    const unsigned long long wall0 = TIMING ? wall_clock64() : 0ull;
#define FATTN_PHASE(i)                                                  \
    if (TIMING) {                                                       \
        const unsigned long long tnow = __builtin_readcyclecounter();   \
        ph[i] += tnow - tprev;                                          \
        tprev = tnow;                                                   \
    }

    // One step of the walk handles one 64-query tile as two 32-query blocks in four phases of NS MFMAs:
    //   A0: S,dP(block 0)          | issue of the next tile's copies
    //   A1: S,dP(block 1)          | P,dS(block 0)
    //   B0: dV,dK += (block 0)     | P,dS(block 1)
    //   B1: dV,dK += (block 1)
    // written as an explicit software pipeline for a single wavefront per SIMD: the MFMA pipe and the
    // vector ALU run side by side only when their instructions alternate in the instruction stream, so
    // the per-element arithmetic of one block is threaded between the MFMAs of its neighbour, one
    // accumulator register per MFMA.  The G = 4 NS operand fragments of a step come from LDS through one
    // ring of PD registers that runs PD fragments ahead of the MFMAs, across the phases and on into the
    // next step; the scheduling barriers keep the compiler from undoing either interleave.
    //
    // Three LDS stages, one workgroup barrier per step, placed just before the ring first reads the next
    // stage: by then every wave's copies of the next tile have landed, and every wave has finished the
    // previous step, whose stage the next step's copies overwrite.  No wave ever drains its pipeline.
    //
    // dP accumulates on top of -delta (loaded from LDS straight into the accumulator registers), so
    // dS = P * dP' needs no subtraction.
    constexpr int NS = 2 * DC;      // MFMAs per phase
    constexpr int G = 4 * NS;       // MFMAs = operand fragments per step
    constexpr int PD = 4;           // read-ahead depth of the fragment ring
    static_assert(2 * DC == 4 * DB, "all phases must have the same number of MFMA slots");
    constexpr int NCOPY = 2 * NDQ + 1 + (VECMASK ? 2 : 0);     // copies per wavefront and step: Q, dO, a row, mask
    static_assert(NS % PD == 0 && 4 * (NCOPY - 1) + 1 < G - PD, "ring depth / copy slices do not fit");
    f32x16 dpacc[2];
    bf16x8 fb[PD];
    // fragment g of a step: [0, 2 NS) 16-byte row reads (block, dc, Q | dO); [2 NS, 4 NS) transposing
    // reads (block, 16-query chunk, db, dO^T | Q^T)
    auto frag = [&](const uint16_t* Qs, int g) {
        const uint16_t* dOs = Qs + T::Q_ELEMS;
        const int qb = (g / NS) & 1, i = g % NS;
        if (g < 2 * NS) {
            const int dc = i >> 1;
            return *reinterpret_cast<const bf16x8*>(((i & 1) ? dOs : Qs) + roff[dc] + 32 * qb * RS);
        }
        const int c = i / (2 * DB), db = (i >> 1) % DB, cc = 2 * qb + c;
        return tr_frag((i & 1) ? Qs : dOs, toff[0][db] + 16 * cc * RS, toff[1][db] + 16 * cc * RS);
    };
    // -delta of queries 8*g4 + 4h .. +3 of block qb -> the dP accumulator registers of those rows
    auto ndelta_rows = [&](const float* rows, int qb, int g4) {
        const f32x4 v = *reinterpret_cast<const f32x4*>(rows + BM + 32 * qb + 8 * g4 + 4 * h);
#pragma unroll
        for (int t = 0; t < 4; ++t) dpacc[qb][4 * g4 + t] = DROPOUT ? 0.f : v[t];
    };

    // this workgroup's slice [it_lo, it_hi) of the walk
    const int it_lo = (int)((int64_t)part * n_it / nparts);
    const int it_hi = (int)((int64_t)(part + 1) * n_it / nparts);
    // The stages are numbered so that the steps which need exclusions (they come first and take their
    // stage from a run-time counter) leave the counter at 0 for the main loop, whose three unrolled
    // steps have their stages fixed at compile time.
    const int n_masked_here = max(min(n_masked, it_hi) - it_lo, 0);
    // (VECMASK: every step needs exclusions and the straight-line loop comes first, so it starts in stage 0)
    int st = VECMASK ? 0 : (3 - n_masked_here % 3) % 3;        // LDS stage of the step about to run
    if (it_hi > it_lo) {
        issue_q_tile(tile_of(it_lo), head_of(it_lo), st);
        wait_vm0();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PD; ++i) fb[i] = frag(stage0 + st * T::STAGE_ELEMS, i);
#pragma unroll
        for (int g4 = 0; g4 < 4; ++g4) ndelta_rows(rows0 + st * T::ROW_FLOATS, 0, g4);
    }

    uint64_t word_ahead = 0;               // BITS: of the next cut tile
    if constexpr (BITS) {
        if (n_masked > 0) word_ahead = bcols[(int64_t)tile_of(0) * (64 * p.m.bit_nkt)];
    }
    // COPY: 0 = this is the last step, 1 = the next tile is a full one (straight-line copies),
    //       2 = decide at run time (used by the few steps that need exclusions)
    // STAGE: LDS stage that holds this step's tile (0 / 1 / 2), or -1 to take it from `st`.
    auto step = [&](auto masked_tag, auto copy_tag, auto stage_tag, int st, int it, int qt, int qt_next,
                    const uint16_t* nq_base, const uint16_t* ndo_base, const float* nrow_base) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        constexpr int COPY = decltype(copy_tag)::value;
        constexpr int STAGE = decltype(stage_tag)::value;
        const int cur = STAGE >= 0 ? STAGE : st;
        const int nxt = STAGE >= 0 ? (STAGE + 1) % 3 : (st == 2 ? 0 : st + 1);
        const int q0 = qt * BM;
        const bool have_next = COPY == 1 || (COPY == 2 && it + 1 < it_hi);

        const uint16_t* Qs = stage0 + cur * T::STAGE_ELEMS;
        const uint16_t* Qn = stage0 + nxt * T::STAGE_ELEMS;
        const float* rows_c = rows0 + cur * T::ROW_FLOATS;      // [lse2 | -delta] of this step's queries
        const float* rows_n = rows0 + nxt * T::ROW_FLOATS;

        f32x16 sacc[2];
        bf16x8 pf[2][2], dsf[2][2];
        f32x4 l4, l4n;
        uint32_t keep_bits[2] = {0u, 0u};       // BITS: of this lane's half, query block by query block
        if constexpr (BITS && MASKED) {
            keep_bits[0] = (uint32_t)word_ahead >> (4 * h);
            keep_bits[1] = (uint32_t)(word_ahead >> 32) >> (4 * h);
            if (it + 1 < n_masked) word_ahead = bcols[(int64_t)qt_next * (64 * p.m.bit_nkt)];
        }
        // keep-mask bytes of this lane's key for the 64 queries of the tile, fetched up front in one batch
        // (a load per element inside the pipelined slices would wait out a memory round trip each time)
        uint32_t mk[2][16];
        if (HASMASK && !VECMASK && MASKED) {
            const int64_t mkey = (int64_t)min(key, p.Sk - 1) * p.m.sk;
#pragma unroll
            for (int qb = 0; qb < 2; ++qb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    const int qi = q0 + 32 * qb + 8 * (r >> 2) + 4 * h + (r & 3);
                    mk[qb][r] = mask_attends(p.m, mbase, mkey + (int64_t)min(qi, p.Sq - 1) * p.m.sq) ? 1u : 0u;
                }
        }
        // lse2 is read one group of four queries ahead of its use, so that waiting for it never drains
        // the fragment reads that were issued in between
        // (VECMASK: and with it the four mask bytes of this lane's key for those queries)
        const uint8_t* mask_c = mask0 + cur * T::MASK_STAGE_BYTES + (4 * h) * BN + 32 * wave + n;
        const uint8_t* nm_base = VECMASK ? mask_tile(qt_next) : nullptr;
        uint32_t m4[4], m4n[4];
        f32x4 nd4, nd4n;                 // DROPOUT: -delta of the same four queries
        // kDropRows64: the index of (query, key) is the query's index at this wavefront's first key XOR the lane's n, so the 64
        // lanes evaluate the generator for the 64 queries of the step, once, and pass the words on through LDS (a wavefront
        // reads what it has written itself: no barrier)
        u32x4 dw4{}, dw4n{};
        // kDropFlat: index of the next element; the elements are visited in query order, four rows and then four of the other half
        uint32_t drop_idx = ((uint32_t)bh * (uint32_t)p.Sq + (uint32_t)(q0 + 4 * h)) * (uint32_t)p.Sk + (uint32_t)key;
        (void)drop_idx;
        uint32_t* const drop_words = reinterpret_cast<uint32_t*>(reinterpret_cast<uint8_t*>(lds) + T::LDS_BYTES) + wave * BM;
        if constexpr (DROP == kDropRows64)
            drop_words[lane] = xorshift32(p.m.drop_seed ^ (((uint32_t)bh * (uint32_t)p.Sq + (uint32_t)(q0 + lane)) * (uint32_t)p.Sk + (uint32_t)kw0));
        auto rows_ahead = [&](int qb, int g) {
            l4n = *reinterpret_cast<const f32x4*>(rows_c + 32 * qb + 8 * g + 4 * h);
            if (DROPOUT) nd4n = *reinterpret_cast<const f32x4*>(rows_c + BM + 32 * qb + 8 * g + 4 * h);
            if (DROP == kDropRows64) dw4n = *reinterpret_cast<const u32x4*>(drop_words + 32 * qb + 8 * g + 4 * h);
            if (VECMASK) {
#pragma unroll
                for (int t = 0; t < 4; ++t) m4n[t] = mask_c[(32 * qb + 8 * g + t) * BN];
            }
        };

        // element r of block qb: P = exp2(S*c - lse2), dS = P*(dP - delta); pack after 8 and 16.
        // The product for element r is issued with the exponential of element r + 1, so that no
        // instruction waits on the transcendental unit.
        auto ds_mul = [&](int qb, int r) {
            if (!DROPOUT) dpacc[qb][r] = sacc[qb][r] * dpacc[qb][r];       // DROPOUT: elem() has formed dS already
            if ((r & 7) == 7) {
                const int c = r >> 3, o8 = 8 * c;
                const f32x16& d = dpacc[qb];
                dsf[qb][c] = pack8(d[o8], d[o8 + 1], d[o8 + 2], d[o8 + 3], d[o8 + 4], d[o8 + 5], d[o8 + 6], d[o8 + 7]);
            }
        };
        auto elem = [&](int qb, int r) {
            const int g = r >> 2, t = r & 3;
            if (t == 0) {
                l4 = l4n;
                if (DROPOUT) nd4 = nd4n;
                if (DROP == kDropRows64) dw4 = dw4n;
                if (VECMASK) {
#pragma unroll
                    for (int u = 0; u < 4; ++u) m4[u] = m4n[u];
                }
                if (g < 3) rows_ahead(qb, g + 1);
                else if (qb == 0) rows_ahead(1, 0);
            }
            float pr = exp2_fast(fmaf(sacc[qb][r], c_log2, -l4[t]));
            if (r > 0) ds_mul(qb, r - 1);
            if (MASKED) {
                const int qi = q0 + 32 * qb + 8 * g + 4 * h + t;
                bool drop;
                if constexpr (VECMASK) {
                    drop = m4[t] <= dead_thr;       // whole tiles, no causal flag: the mask byte decides, one compare
                } else if constexpr (BITS) {
                    drop = (keep_bits[qb] & (1u << (8 * g + t))) == 0;
                } else {
                    // bitwise, not short-circuit: one select per element instead of a chain of branches
                    drop = (key >= klimit) | (qi >= Sq) | ((p.m.causal != 0) & (key > qi + past));
                    if (HASMASK) drop |= mk[qb][r] == 0;
                }
                pr = drop ? 0.f : pr;
            }
            if constexpr (DROP == kDropTiled) {
                const uint32_t qi = (uint32_t)(q0 + 32 * qb + 8 * g + 4 * h + t);
                const float f = drop_factor_at(p.m, (uint32_t)bh, qi, (uint32_t)key, (uint32_t)p.Sq, (uint32_t)p.Sk);
                dpacc[qb][r] = pr * fmaf(f, dpacc[qb][r], nd4[t]);       // dS = P (f dP - delta)
                pr *= f;                                                  // what multiplied V in the forward
            } else if constexpr (DROPOUT) {                               // the same, dV rescaled at the end
                uint32_t w;
                if constexpr (DROP == kDropRows64) {
                    w = dw4[t] ^ drop_lane;
                } else {
                    w = xorshift32(p.m.drop_seed ^ drop_idx);
                    drop_idx += (t == 3 ? 5u : 1u) * (uint32_t)p.Sk;
                    asm volatile("" : "+v"(drop_idx));       // stepped, not 32 multiples of Sk kept in registers
                }
                const bool kept = w >= p.m.drop_thr32;
                dpacc[qb][r] = pr * fmaf(kept ? dpacc[qb][r] : 0.f, p.m.drop_scale, nd4[t]);
                pr = kept ? pr : 0.f;
            }
            sacc[qb][r] = pr;
            if ((r & 7) == 7) {
                const int c = r >> 3, o8 = 8 * c;
                const f32x16& s = sacc[qb];
                pf[qb][c] = pack8(s[o8], s[o8 + 1], s[o8 + 2], s[o8 + 3], s[o8 + 4], s[o8 + 5], s[o8 + 6], s[o8 + 7]);
            }
        };
        // slice s (of NS per block) of the element-wise work: logit registers 16 s / NS to 16 (s + 1) / NS; slice NS is the
        // last product
        auto elem_slot = [&](int qb, int s) {
            if (s == NS) {
                ds_mul(qb, 15);
                return;
            }
#pragma unroll
            for (int e = 0; e < (16 + NS - 1) / NS; ++e)
                if (16 * s / NS + e < 16 * (s + 1) / NS) elem(qb, 16 * s / NS + e);
        };

        // copies of the next tile, one instruction at a time (full tiles: uniform base + lane offset), each
        // in two halves around an MFMA: destination into M0, then the copy.  nq_base / ndo_base / nrow_base
        // are the wave-uniform addresses of the next tile's Q rows, dO rows and lse2 (even waves) or
        // -delta (odd waves) rows; waves 2 and 3 repeat the row copies of waves 0 and 1.
        const bool next_full = COPY == 1 || (qt_next * BM + BM) <= Sq;
        const bool copying = COPY == 1 || (COPY == 2 && have_next && next_full);
        auto copy_dst_of = [&](int j) {
            return j < 2 * NDQ ? q_dst(nxt, j & 1, j >> 1) : rows_lds0 + 4u * (uint32_t)(nxt * T::ROW_FLOATS + (wave & 1) * BM);
        };
        // Copy j goes with MFMA slot 4j + 1.  In straight-line steps, while that MFMA is a hand-emitted one
        // (phases A0 and A1), the copy is split around it.
        auto copy_dst = [&](int g) {
            const int j = g / 4;
            if (COPY == 1 && g % 4 == 1 && j <= 2 * NDQ && g < 2 * NS) dma_set_dst(copy_dst_of(j));
        };
        auto copy_issue = [&](int g) {
            const int j = g / 4;
            if (COPY == 0 || g % 4 != 1 || j >= NCOPY) return;
            if (COPY == 1 && g < 2 * NS) {
                if (j == 2 * NDQ) dma4u_issue(nrow_base, 4u * (uint32_t)lane);
                else if (j & 1) dma16u_issue(ndo_base, do_lane_off[j >> 1]);
                else dma16u_issue(nq_base, q_lane_off[j >> 1]);
            } else if (copying) {          // destination and copy in one piece
                if (j > 2 * NDQ) dma16u(nm_base, m_lane_off[j - 2 * NDQ - 1], mask_dst(nxt, j - 2 * NDQ - 1));
                else if (j == 2 * NDQ) dma4(nrow_base + lane, copy_dst_of(j));
                else if (j & 1) dma16u(ndo_base, do_lane_off[j >> 1], copy_dst_of(j));
                else dma16u(nq_base, q_lane_off[j >> 1], copy_dst_of(j));
            }
        };
        if (COPY == 2 && have_next && !next_full) issue_q_tile(qt_next, head_of(it + 1), nxt);   // partial tile: slow path, all at once

        // The element-wise work of a block trails the hand-emitted MFMAs that produced its S and dP by
        // LAG MFMA slots (see mfma32_vgpr_bacc), so its last LAG slices run at the start of the phase after.
        constexpr int LAG = 2;
        auto side = [&](int g) {
            const int phase = g / NS, i = g % NS;
            copy_issue(g);
            if (phase == 0) {
                if (i >= NS - 4) ndelta_rows(rows_c, 1, i - (NS - 4));
                if (i == NS - 1) rows_ahead(0, 0);
            } else if (phase == 1) {
                if (i >= LAG) elem_slot(0, i - LAG);
            } else if (phase == 2) {
                if (i <= LAG) elem_slot(0, NS - LAG + i);
                if (i >= LAG) elem_slot(1, i - LAG);
            } else {
                if (i <= LAG) elem_slot(1, NS - LAG + i);
            }
        };
        auto refill = [&](int g) {
            const int ng = g + PD;
            if (ng < G) fb[g % PD] = frag(Qs, ng);
            else if (COPY == 1 || (COPY == 2 && have_next)) fb[g % PD] = frag(Qn, ng - G);
        };

        // fragments are consumed in pairs, the younger read first: one s_waitcnt serves two MFMAs
        auto run_phase = [&](auto phase_tag) {
            constexpr int PHASE = decltype(phase_tag)::value;
#pragma unroll
            for (int i = 0; i < NS; i += 2) {
                const int g = PHASE * NS + i;
                if constexpr (PHASE < 2) {      // S = Q K^T and dP = dO V^T - delta, rows = queries of block qb, columns = this wave's keys
                    const int qb = PHASE, dc = i >> 1;
                    // the dropout builds: the allocator splits the accumulators around the longer element arithmetic
                    // and moves parts of them back right before these statements
                    mfma32_vgpr_bacc<DROPOUT>(dpacc[qb], fb[(g + 1) % PD], vf[dc]);
                    side(g);
                    __builtin_amdgcn_sched_barrier(0);
                    copy_dst(g + 1);
                    if (i == 0) mfma32_vgpr_first_bacc<DROPOUT>(sacc[qb], fb[g % PD], kf[dc]);
                    else mfma32_vgpr_bacc<DROPOUT>(sacc[qb], fb[g % PD], kf[dc]);
                    side(g + 1);
                } else {              // dV^T += dO^T P, dK^T += Q^T dS: rows = d, columns = keys, contraction over queries
                    const int qb = PHASE - 2, c = i / (2 * DB), db = (i >> 1) % DB;
                    dkacc[db] = mfma32(fb[(g + 1) % PD], dsf[qb][c], dkacc[db]);
                    side(g);
                    __builtin_amdgcn_sched_barrier(0);
                    dvacc[db] = mfma32(fb[g % PD], pf[qb][c], dvacc[db]);
                    side(g + 1);
                }
                if (g == G - PD && COPY != 0) {
                    if (COPY == 1 || have_next) {
                        __builtin_amdgcn_sched_barrier(0);
                        FATTN_PHASE(3)
                        wait_vm0();                          // this wave's copies of the next tile have landed
                        __builtin_amdgcn_s_barrier();        // ... everyone's have, and everyone is past the previous step
                        FATTN_PHASE(4)
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int g4 = 0; g4 < 4; ++g4) ndelta_rows(rows_n, 0, g4);
                    }
                }
                refill(g);
                refill(g + 1);
                __builtin_amdgcn_sched_barrier(0);
            }
            if (PHASE < 3) { FATTN_PHASE(PHASE) }
        };
        run_phase(std::integral_constant<int, 0>{});
        run_phase(std::integral_constant<int, 1>{});
        run_phase(std::integral_constant<int, 2>{});
        run_phase(std::integral_constant<int, 3>{});
    };

    using IM = std::integral_constant<int, -1>;
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    const int64_t q_tile_stride = (int64_t)BM * p.qs.n, do_tile_stride = (int64_t)BM * p.dos.n;
    const float* rowbase = (wave & 1) ? ndeltabase : lsebase;
    int it_m = it_lo;
    if constexpr (VECMASK) {
        // Every tile needs exclusions, all are whole and consecutive: the same three straight-line steps
        // with fixed stages as the unmasked loop below.
        int qt = qt_begin + it_m;
        const uint16_t* nq = qbase + (qt + 1) * q_tile_stride;
        const uint16_t* ndo = dobase + (qt + 1) * do_tile_stride;
        const float* nrow = rowbase + (qt + 1) * BM;
        for (; it_m + 3 <= it_hi - 1; it_m += 3, qt += 3) {
            step(std::true_type{}, I1{}, I0{}, 0, it_m, qt, qt + 1, nq, ndo, nrow);
            nq += q_tile_stride, ndo += do_tile_stride, nrow += BM;
            step(std::true_type{}, I1{}, I1{}, 1, it_m + 1, qt + 1, qt + 2, nq, ndo, nrow);
            nq += q_tile_stride, ndo += do_tile_stride, nrow += BM;
            step(std::true_type{}, I1{}, I2{}, 2, it_m + 2, qt + 2, qt + 3, nq, ndo, nrow);
            nq += q_tile_stride, ndo += do_tile_stride, nrow += BM;
        }
    }
    if constexpr (BITS) {
        // Cut tiles in straight-line steps of three as well, once the stage counter is 0: every next tile of theirs is a cut one
        // that is not the last, which alone can be a partial one.
        int it = 0;
        auto one = [&]() {
            const int qn = it + 1 < it_hi ? tile_of(it + 1) : 0;
            step(std::true_type{}, I2{}, IM{}, st, it, 0, qn, qbase + qn * q_tile_stride, dobase + qn * do_tile_stride, rowbase + qn * BM);
            st = st == 2 ? 0 : st + 1;
            ++it;
        };
        while (it < n_masked && st != 0) one();
        if (it + 3 < n_masked - 1) {
            int at_tile = tile_of(it + 1);
            const uint16_t* nq = qbase + at_tile * q_tile_stride;
            const uint16_t* ndo = dobase + at_tile * do_tile_stride;
            const float* nrow = rowbase + at_tile * BM;
            auto advance = [&](int next) {
                const int d = tile_of(next) - at_tile;
                at_tile += d;
                nq += d * q_tile_stride;
                ndo += d * do_tile_stride;
                nrow += d * BM;
            };
            for (; it + 3 < n_masked - 1; it += 3) {
                step(std::true_type{}, I1{}, I0{}, 0, it, 0, at_tile, nq, ndo, nrow);
                advance(it + 2);
                step(std::true_type{}, I1{}, I1{}, 1, it + 1, 0, at_tile, nq, ndo, nrow);
                advance(it + 3);
                step(std::true_type{}, I1{}, I2{}, 2, it + 2, 0, at_tile, nq, ndo, nrow);
                advance(it + 4);
            }
        }
        while (it < n_masked) one();
        it_m = n_masked;
    }
    for (int it = it_m; it < n_masked_here + it_lo; ++it) {
        const int qn = it + 1 < it_hi ? tile_of(it + 1) : 0;
        const int hn = PACKED && it + 1 < it_hi ? head_of(it + 1) : 0;
        step(std::true_type{}, I2{}, IM{}, st, it, tile_of(it), qn, qbase + qn * q_tile_stride + hn * p.qs.h, dobase + qn * do_tile_stride + hn * p.dos.h,
             rowbase + qn * BM + (int64_t)hn * u.total_q);
        st = st == 2 ? 0 : st + 1;
    }
    // every tile after the first n_masked is a full, fully attended one, and they are consecutive;
    // the stage counter is 0 here
    {
        int it = max(n_masked, it_lo);
        int qt = lead_end + (it - n_masked);                       // (BITS: the list says which tile, and no step asks for its number)
        const uint16_t* nq = qbase + (qt + 1) * q_tile_stride;     // the tile after the current one
        const uint16_t* ndo = dobase + (qt + 1) * do_tile_stride;
        const float* nrow = rowbase + (qt + 1) * BM;
        // PACKED: the tile after the current one is tile `ahead` of the full ones of its head
        int ahead = 0;
        if constexpr (PACKED) {
            const int f = it + 1 - n_masked, head = packed_uniform(f / n_full_head);
            ahead = f - head * n_full_head;
            nq = qbase + (lead_end + ahead) * q_tile_stride + head * p.qs.h;
            ndo = dobase + (lead_end + ahead) * do_tile_stride + head * p.dos.h;
            nrow = rowbase + (lead_end + ahead) * BM + (int64_t)head * u.total_q;
        }
        // BITS: the list says how many tiles to go on (from the one the pointers are at; kept as steps, not as places: pointers
        // formed anew from the bases took so many scalar registers that 560 bytes per lane went to scratch)
        int listed = it + 1, at_tile = qt + 1;
        auto on_by_list = [&]() {
            if (listed < it_hi) {
                const int d = tile_of(listed) - at_tile;
                at_tile += d;
                ++listed;
                nq += d * q_tile_stride;
                ndo += d * do_tile_stride;
                nrow += d * BM;
            }
        };
        if constexpr (BITS) on_by_list();
        auto advance = [&]() {
            if constexpr (BITS) {
                on_by_list();
                return;
            }
            if constexpr (PACKED) {
                if (++ahead == n_full_head) {          // on to the next head
                    ahead = 0;
                    nq += p.qs.h - n_full_head * q_tile_stride;
                    ndo += p.dos.h - n_full_head * do_tile_stride;
                    nrow += u.total_q - n_full_head * BM;
                }
            }
            nq += q_tile_stride;
            ndo += do_tile_stride;
            nrow += BM;
        };
        for (; it + 3 <= it_hi - 1; it += 3, qt += 3) {
            step(std::false_type{}, I1{}, I0{}, 0, it, qt, qt + 1, nq, ndo, nrow);
            advance();
            step(std::false_type{}, I1{}, I1{}, 1, it + 1, qt + 1, qt + 2, nq, ndo, nrow);
            advance();
            step(std::false_type{}, I1{}, I2{}, 2, it + 2, qt + 2, qt + 3, nq, ndo, nrow);
            advance();
        }
        for (; it < it_hi - 1; ++it, ++qt) {
            step(std::false_type{}, I1{}, IM{}, st, it, qt, qt + 1, nq, ndo, nrow);
            advance();
            st = st == 2 ? 0 : st + 1;
        }
        if (it < it_hi) step(std::false_type{}, I0{}, IM{}, st, it, qt, qt, nq, ndo, nrow);
    }

    if (TIMING && p.phase_cycles && tid == 0) {
        ph[5] = wall_clock64() - wall0;      // 100 MHz
#pragma unroll
        for (int i = 0; i < 6; ++i) p.phase_cycles[(size_t)block * 6 + i] = ph[i];
    }
#undef FATTN_PHASE

    // ---- epilogue
    if (nparts > 1) {
        // fp32 partial sums of this slice, in accumulator order: [tensor][db][group of four][thread], so that the lanes of a
        // wavefront write, and the merge reads, 1 KiB at a time
        float* dst = p.split_ws + (PACKED ? (size_t)wg : (size_t)(wg - p.n_whole) * nparts + part) * (size_t)(2 * BN * D);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x16& a = dkacc[db];
                const f32x16& c = dvacc[db];
                const size_t at = ((size_t)(db * 4 + g) * 256 + tid) * 4;
                *reinterpret_cast<f32x4*>(dst + at) = f32x4{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
                *reinterpret_cast<f32x4*>(dst + (size_t)BN * D + at) = f32x4{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]};
            }
        return;
    }
    if (key >= klimit || dead) {  // nothing attends to this lane's key
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                dkacc[db][r] = 0.f;
                dvacc[db][r] = 0.f;
            }
    }
    __syncthreads();              // nobody reads a tile any more
    store_rows(dkacc, dvacc, DROP == kDropFlat || DROP == kDropRows64 ? p.m.drop_scale : 1.0f);
}

template <int D, bool HASMASK, bool TIMING, bool VECMASK = false, int DROP = kDropNone, bool BITS = false>
__global__ __launch_bounds__(256) void bwd_dkdv_kernel(const BwdParams p) {
    bwd_dkdv_body<D, HASMASK, TIMING, VECMASK, DROP, BITS>(p, (int)blockIdx.x, (int)gridDim.x);
}
template <int D, bool BITS>
__global__ __launch_bounds__(256) void bwd_dkdv_dealt_kernel(const BwdParams p) {
    bwd_dkdv_body<D, false, false, false, kDropNone, BITS, true>(p, (int)blockIdx.x, (int)gridDim.x);
}

// dK^T / dV^T accumulators (rows = d, column = a lane's key) of the 32 keys from kw0 on -> bf16 rows of dK (scaled) and dV, of which
// dkbase and dvbase are key 0
template <int D>
__device__ __forceinline__ void dkdv_store(const BwdParams& p, uint16_t* own, const f32x16 (&dkacc)[D / 32], const f32x16 (&dvacc)[D / 32],
                                           uint16_t* dkbase, uint16_t* dvbase, int Sk, int kw0, float dv_scale) {
    const auto rows_of = [&](const f32x16 (&acc)[D / 32], float s) {
        return [&acc, s](int db, int g) {
            const f32x16& a = acc[db];
            return u32x2{pack_bf16(a[4 * g] * s, a[4 * g + 1] * s), pack_bf16(a[4 * g + 2] * s, a[4 * g + 3] * s)};
        };
    };
    store_rows32<D>(own, dkbase + (int64_t)kw0 * p.dks.n, p.dks.n, Sk - kw0, p.d, rows_of(dkacc, p.scale));
    store_rows32<D>(own, dvbase + (int64_t)kw0 * p.dvs.n, p.dvs.n, Sk - kw0, p.d, rows_of(dvacc, dv_scale));
}

// Sums the fp32 partials that the split workgroups of one key block left behind and writes dK, dV; keys that nothing attends
// to (past the key length, masked, past the last query under the causal flag) get zeros.
// One workgroup per (split key block, 32-wide block of d); the thread layout mirrors the accumulators.
template <int D>
__global__ __launch_bounds__(256) void bwd_dkdv_merge_kernel(const BwdParams p) {
    constexpr int BN = BwdTile<D>::BN, DB = D / 32;
    const int tid = threadIdx.x;
    const int lane = tid & 63, wave = tid >> 6;
    const int n = lane & 31, h = lane >> 5;
    const int n_kt = (p.Sk + BN - 1) / BN;
    const int sb = (int)blockIdx.x / DB, db = (int)blockIdx.x % DB;
    const int wg = p.n_whole + sb;
    const int kt = wg % n_kt;
    const int bh = wg / n_kt;
    const int b = bh / p.H, hh = bh % p.H;
    f32x4 ak[4], av[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        ak[g] = f32x4{0.f, 0.f, 0.f, 0.f};
        av[g] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float* src = p.split_ws + (size_t)sb * p.split_parts * (size_t)(2 * BN * D) + ((size_t)db * 4 * 256 + tid) * 4;
#pragma unroll 2
    for (int part = 0; part < p.split_parts; ++part, src += (size_t)(2 * BN * D)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            ak[g] += *reinterpret_cast<const f32x4*>(src + g * 1024);
            av[g] += *reinterpret_cast<const f32x4*>(src + (size_t)BN * D + g * 1024);
        }
    }
    const int krow = kt * BN + 32 * wave + n;
    if (krow < p.Sk) {
        bool dead = p.m.kv_len && krow >= p.m.kv_len[b];
        if (p.key_mask && !dead) dead = !mask_attends(p.m, mask_head_base(p.m, b, hh), (int64_t)krow * p.m.sk);
        if (p.m.causal && kt * BN >= p.Sq) dead = true;
        uint16_t* dkrow = p.dk + b * p.dks.b + hh * p.dks.h + (int64_t)krow * p.dks.n;
        uint16_t* dvrow = p.dv + b * p.dvs.b + hh * p.dvs.h + (int64_t)krow * p.dvs.n;
        const float s = p.scale;
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            u32x2 wk = {pack_bf16(ak[g][0] * s, ak[g][1] * s), pack_bf16(ak[g][2] * s, ak[g][3] * s)};
            u32x2 wv = {pack_bf16(av[g][0] * p.dv_scale, av[g][1] * p.dv_scale), pack_bf16(av[g][2] * p.dv_scale, av[g][3] * p.dv_scale)};
            if (dead) wk = wv = u32x2{0u, 0u};
            if (32 * db + 8 * g + 4 * h < p.d) *reinterpret_cast<u32x2*>(dkrow + 32 * db + 8 * g + 4 * h) = wk;
            if (32 * db + 8 * g + 4 * h < p.d) *reinterpret_cast<u32x2*>(dvrow + 32 * db + 8 * g + 4 * h) = wv;
        }
    }
}

// -------------------------------------------------------------------------------------------- dq
template <int D>
struct BwdDqTile {
    static constexpr int BM = 128;                  // query rows per workgroup (32 per wavefront)
    static constexpr int BN = 64;                   // keys per tile
    static constexpr int RS = kRowPitch<D>;
    static constexpr int TILE_ELEMS = BN * RS;
    static constexpr int STAGE_ELEMS = 2 * TILE_ELEMS;            // K tile + V tile
    static constexpr int LDS_BYTES = 2 * STAGE_ELEMS * 2;
    static constexpr int ROWS_PER_DMA = 1024 / (RS * 2);
    static constexpr int DMA_PER_WAVE = BN / ROWS_PER_DMA / 4;
};

// NW wavefronts of 32 queries each per workgroup, two per SIMD (the library instantiates NW = 4; problems
// that fill 256-query workgroups go to bwd_dq_wide_kernel below).
// EXCL, DEALT: see there.  Only the general form compiles per-element mask loads in; the others fit two workgroups per unit.
// KG = 2: two groups of NW wavefronts share the workgroup's queries, each walks one half of the key tiles in LDS stages of its
// own, and the second adds its dQ to the first's through LDS: for grids that give a compute unit one workgroup at most.
// PACKED: the unit is a query tile of one of several sequences of different lengths (packed_units.hpp), `u`.
template <int D, int EXCL, int NW, int DROP, int KG, bool DEALT, bool PACKED = false>
__device__ __forceinline__ void bwd_dq_body(const BwdParams& p, const PackedUnit& u = PackedUnit()) {
    static_assert(!PACKED || (EXCL == kExNone && DROP == kDropNone && !DEALT), "packed sequences: causal flag and lengths only");
    static_assert(KG == 1 || (KG == 2 && EXCL == kExNone), "key groups: nothing excluded but by causal flag and key lengths");
    constexpr bool HASMASK = EXCL == kExRows16 || EXCL == kExGeneral, VECMASK = EXCL == kExRows16, BITS = EXCL == kExBits, KEYS = EXCL == kExKeys || BITS;
    using T = BwdDqTile<D>;
    constexpr int BM = 32 * NW, BN = T::BN, RS = T::RS;
    constexpr int DC = D / 16;
    constexpr int DB = D / 32;
    constexpr int GPR = RS / 8;

    extern __shared__ __attribute__((aligned(1024))) uint16_t lds_all[];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave_all = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wave = KG == 1 ? wave_all : wave_all % NW, group = KG == 1 ? 0 : wave_all / NW;
    uint16_t* lds = lds_all + (KG == 1 ? 0 : group * (T::LDS_BYTES / 2));
    const int n = lane & 31, h = lane >> 5;

    const int Sq = PACKED ? u.Sq : p.Sq, Sk = PACKED ? u.Sk : p.Sk;
    const int past = PACKED ? u.past : 0;             // under the causal flag query i attends to key j <= i + past
    const int n_qt = (Sq + BM - 1) / BM;
    const bool falling = !(EXCL == kExKeys) && p.m.causal && !p.m.kv_len;
    int wg = 0, part = 0;
    if constexpr (PACKED) {
        wg = u.unit;
        part = u.part;
    } else if (p.dq_parts > 1) {
        const int all = xcd_remap_split(blockIdx.x, gridDim.x);
        part = all % p.dq_parts;
        wg = all / p.dq_parts;
    } else {
        wg = p.dq_base + xcd_remap_heads<KG == 1 && !BITS>(blockIdx.x, gridDim.x, n_qt, p.m.kv_len || KEYS, falling);
    }
    int qt = PACKED ? u.tile : wg % n_qt, bh = PACKED ? 0 : wg / n_qt;
    if constexpr (PACKED) {
    } else if constexpr (DEALT) {
        int t, s;
        dealt_unit<!BITS>(blockIdx.x, n_qt, p.B, p.H, !falling, t, s);
        qt = __builtin_amdgcn_readfirstlane(falling ? n_qt - 1 - t : t);
        bh = __builtin_amdgcn_readfirstlane(s);
    } else if (falling && p.dq_parts == 1) {
        causal_longest_first<KG == 1>(wg, n_qt, gridDim.x, qt, bh);
    }
    if (!PACKED && !BITS && (KEYS || p.m.kv_len) && p.dq_parts == 1) bh = longest_batches_first<KEYS>(bh, p.B, p.H, p.Sk, p.m);
    const int b = bh / p.H, hh = bh % p.H;
    const int q0 = qt * BM;
    const int qw0 = q0 + wave * 32;

    const uint16_t* qbase = PACKED ? p.q + u.q_at(p.qs) : p.q + b * p.qs.b + hh * p.qs.h;
    const uint16_t* kbase = PACKED ? p.k + u.k_at(p.ks) : p.k + b * p.ks.b + hh * p.ks.h;
    const uint16_t* vbase = PACKED ? p.v + u.k_at(p.vs) : p.v + b * p.vs.b + hh * p.vs.h;
    const uint16_t* dobase = PACKED ? p.dout + u.q_at(p.dos) : p.dout + b * p.dos.b + hh * p.dos.h;
    auto obase = [&]() { return PACKED ? p.o + u.q_at(p.os) : p.o + b * p.os.b + hh * p.os.h; };
    auto stat_row = [&]() { return PACKED ? u.stat_row() : (int64_t)bh * p.Sq; };

    int klimit = Sk;
    if (!PACKED && p.m.kv_len) klimit = min(klimit, max(p.m.kv_len[b], 0));
    int kend = klimit;
    if (p.m.causal) kend = min(kend, q0 + BM + past);
    if constexpr (PACKED) kend = max(kend, 0);
    int n_tiles = (kend + BN - 1) / BN;
    const uint8_t* mbase = HASMASK || EXCL == kExKeys ? mask_head_base(p.m, b, hh) : nullptr;
    int t_lo = 0;             // first tile of this workgroup's share of the walk
    const int parts = PACKED ? packed_parts(u, n_tiles) : p.dq_parts;
    if (PACKED && part >= parts) return;
    if (parts > 1) {
        const int per = PACKED ? packed_uniform((n_tiles + parts - 1) / parts) : (n_tiles + parts - 1) / parts;
        t_lo = part * per;
        n_tiles = min(n_tiles, t_lo + per) - t_lo;      // not positive: nothing to do
    }
    const int n_first = (n_tiles + 1) / 2;              // KG: of group 0 (dq_parts is 1)
    if constexpr (KG == 2) {
        t_lo = group * n_first;
        n_tiles = group ? n_tiles - n_first : n_first;
    }
    // step t of the walk takes tile tile_of(t)
    KeyTiles kt;
    const uint64_t* brows = nullptr;       // BITS: this lane's query's word of key tile 0; tiles lie 64 bit_nqt words apart
    if constexpr (BITS) {
        const int plane = b * p.m.plane_b + hh * p.m.plane_h;
        const uint8_t* flags = p.m.tile_flags + ((int64_t)plane * p.m.bit_nqt + q0 / 64) * p.m.bit_nkt;       // of the first 64 queries, then of the others
        kt.build_of_tiles(reinterpret_cast<char*>(lds) + T::LDS_BYTES, (klimit + 63) / 64, [&](int t) {
            const int f0 = flags[t], f1 = flags[p.m.bit_nkt + t];
            return f0 & f1 & kTileAllKeys ? 2 : (f0 | f1) & kTileAny ? 1 : 0;
        });
        n_tiles = kt.n_tiles;
        brows = p.m.bit_rows + (int64_t)plane * p.m.bit_nkt * (64 * p.m.bit_nqt) + qw0 + n;
    } else if constexpr (KEYS) {
        kt.build(reinterpret_cast<char*>(lds) + T::LDS_BYTES, klimit, NW, [&](int key) {
            return key < klimit && mask_attends(p.m, mbase, (int64_t)min(key, p.Sk - 1) * p.m.sk);
        });
        n_tiles = kt.n_tiles;
    }
    auto tile_of = [&](int t) {
        if constexpr (KEYS) return kt.tile(t);
        else return t_lo + t;
    };

    const int dma_row_in = lane / GPR, dma_gran = lane % GPR;
    constexpr int NDMA = T::DMA_PER_WAVE * 4 / NW;
    const uint32_t lds0 = lds_addr(lds);
    uint32_t k_lane_off[NDMA], v_lane_off[NDMA];     // bytes
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
        const int row = (wave * NDMA + i) * T::ROWS_PER_DMA + dma_row_in;
        const int c = src_granule(dma_gran ^ swz<D>(row), p.d);
        k_lane_off[i] = 2u * (uint32_t)(row * (int)p.ks.n + c * 8);
        v_lane_off[i] = 2u * (uint32_t)(row * (int)p.vs.n + c * 8);
    }
    auto dst_of = [&](int buf, int which, int i) {    // LDS byte address of copy i of this wave (which: 0 = K, 1 = V)
        return lds0 + 2u * (uint32_t)(buf * T::STAGE_ELEMS + which * T::TILE_ELEMS + (wave * NDMA + i) * 512);
    };
    auto issue_tile = [&](int t, int buf) {
        const int tile = tile_of(t);
#pragma unroll
        for (int i = 0; i < NDMA; ++i) {
            const int row = (wave * NDMA + i) * T::ROWS_PER_DMA + dma_row_in;
            const int key = min(tile * BN + row, klimit - 1);   // tail rows re-read the last attended key
            const int c = src_granule(dma_gran ^ swz<D>(row), p.d);
            dma16(kbase + (int64_t)key * p.ks.n + c * 8, dst_of(buf, 0, i));
            dma16(vbase + (int64_t)key * p.vs.n + c * 8, dst_of(buf, 1, i));
        }
    };
    auto issue_full_tile = [&](int t, int buf) {
        const int tile = tile_of(t);
        const uint16_t* ktile = kbase + (int64_t)tile * BN * p.ks.n;
        const uint16_t* vtile = vbase + (int64_t)tile * BN * p.vs.n;
#pragma unroll
        for (int i = 0; i < NDMA; ++i) {
            dma16u(ktile, k_lane_off[i], dst_of(buf, 0, i));
            dma16u(vtile, v_lane_off[i], dst_of(buf, 1, i));
        }
    };

    // on its way before anything else is loaded: on short walks a second round trip to memory is a good part of the run time
    if (n_tiles > 0) issue_tile(0, 0);

    // ---- Q and dO fragments (B operands: column = query, 8 consecutive d), per-query scalars; through stage 1
    const int qrow = qw0 + n;
    const bool qok = qrow < Sq;
    bf16x8 qf[DC], dof[DC];
    // Per-query scalars, formed here and also left in the workspace for the dK/dV kernel that runs next:
    //   delta = rowsum(dO * O)   (the bf16 O that the forward saved)
    //   lse2  = LSE * log2(e), +inf for fully excluded rows and rows past the end (P = exp2(s - inf) = 0)
    float lse2 = INFINITY, delta = 0.f;
    {
        uint16_t* const pass = lds + T::STAGE_ELEMS + wave * 1024;
        u32x4 wq[DC], wd[DC], wo[DC];
        load_rows32<D>(wq, qbase + (int64_t)qw0 * p.qs.n, p.qs.n, Sq - qw0, p.d);
        load_rows32<D>(wd, dobase + (int64_t)qw0 * p.dos.n, p.dos.n, Sq - qw0, p.d);
        load_rows32<D>(wo, obase() + (int64_t)qw0 * p.os.n, p.os.n, Sq - qw0, p.d);
        const float l = qok ? p.lse[stat_row() + qrow] : 0.f;
        fragments_of_rows32<D>(pass, wq, [&](auto dc, u32x4 f) { qf[decltype(dc)::value] = __builtin_bit_cast(bf16x8, f); });
        fragments_of_rows32<D>(pass, wd, [&](auto dc, u32x4 f) { dof[decltype(dc)::value] = __builtin_bit_cast(bf16x8, f); });
        float part = 0.f;
        fragments_of_rows32<D>(pass, wo, [&](auto dc, u32x4 ov) {
            const u32x4 dv = __builtin_bit_cast(u32x4, dof[decltype(dc)::value]);
#pragma unroll
            for (int i = 0; i < 4; ++i) part += bf16_lo(dv[i]) * bf16_lo(ov[i]) + bf16_hi(dv[i]) * bf16_hi(ov[i]);
        });
        part += xhalf(part);
        if (qok) {
            lse2 = (l == -INFINITY) ? INFINITY : l * kLog2e;
            delta = part;
            if (h == 0 && group == 0) {
                p.ndelta[stat_row() + qrow] = -delta;
                p.lse2[stat_row() + qrow] = lse2;
            }
        }
    }

    int koff[DC];          // 16-byte row reads of K / V: row 32*kb + n, logical granule 2*dc + h
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) koff[dc] = n * RS + (((2 * dc + h) ^ swz<D>(n)) << 3);
    const int tr_r = lane & 15, tr_g16 = (lane >> 4) & 1;
    int toff[2][DB];       // transposing reads of K: rows 4h + r/4 (+8), logical granule 4*db + 2*g16 + (r&3)/2
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int row = 4 * h + (tr_r >> 2) + 8 * half;
#pragma unroll
        for (int db = 0; db < DB; ++db)
            toff[half][db] = row * RS + (((4 * db + 2 * tr_g16 + ((tr_r & 3) >> 1)) ^ swz<D>(row)) << 3) + 4 * (tr_r & 1);
    }

    const float c_log2 = p.scale * kLog2e;
    f32x16 dqacc[DB];      // dQ^T: rows = d, column = this lane's query
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) dqacc[db][r] = 0.f;

    MaskRow64 mnext;          // keep-mask bytes of this lane's query row for the next tile (vector-load layouts only)
#pragma unroll
    for (int j = 0; j < 4; ++j) mnext.w[j] = u32x4{0u, 0u, 0u, 0u};
    if (HASMASK && !VECMASK && p.m.rows16 && n_tiles > 0 && BN <= p.Sk) mnext.load(mbase + (int64_t)min(qrow, p.Sq - 1) * p.m.sq);
    wait_vm0();
    __syncthreads();

    uint64_t word_ahead = 0;               // BITS: of the next cut tile
    if constexpr (BITS) {
        if (kt.n_whole < n_tiles) word_ahead = brows[(int64_t)kt.tile(kt.n_whole) * (64 * p.m.bit_nqt)];
    }
    // One tile of 64 keys = two blocks of 32.  The phases of the two blocks are staggered so that the
    // element-wise work of one phase is threaded between the MFMAs of the next, two logits per MFMA:
    //   S(0) | dP(0) + P(0) | S(1) + dS(0) | dP(1) + P(1) | dQ(0) + dS(1) | dQ(1)
    // with one ring of LDS fragments, read PD ahead, running through all 48 operand fetches.
    // BUF: stage that holds this tile (0 / 1), or -1 to take it from the parity of t.
    auto tile_step = [&](auto masked_tag, auto copy_tag, auto buf_tag, int t) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        constexpr int COPY = decltype(copy_tag)::value;
        constexpr int BUF = decltype(buf_tag)::value;
        constexpr int PD = 4;
        const int buf = BUF >= 0 ? BUF : (t & 1);
        if (COPY == 1) issue_full_tile(t + 1, buf ^ 1);
        else if (t + 1 < n_tiles) issue_tile(t + 1, buf ^ 1);
        const uint16_t* ks = lds + buf * T::STAGE_ELEMS;
        const uint16_t* vs = ks + T::TILE_ELEMS;
        const int key0 = (t_lo + t) * BN;      // (not KEYS)
        const uint32_t drop_tile = ((uint32_t)bh * (uint32_t)p.Sq + (uint32_t)qrow) * (uint32_t)p.Sk + (uint32_t)(key0 + 4 * h);
        const uint32_t drop_word = DROP == kDropRows64 ? xorshift32(p.m.drop_seed ^ drop_tile) : 0u;
        (void)drop_tile;
        (void)drop_word;
        uint32_t keep_bits[2] = {0u, 0u};
        if constexpr (KEYS && MASKED) {
            const uint64_t w = BITS ? word_ahead : kt.bits[kt.tile(t)];
            if (BITS && t + 1 < n_tiles) word_ahead = brows[(int64_t)kt.tile(t + 1) * (64 * p.m.bit_nqt)];
            keep_bits[0] = (uint32_t)w >> (4 * h);
            keep_bits[1] = (uint32_t)(w >> 32) >> (4 * h);
        }

        // operand fetch f of the tile, in consumption order
        constexpr int NROW = 4 * DC;                // row-read fragments: S(0), dP(0), S(1), dP(1)
        constexpr int NALL = NROW + 4 * DB;         // + the transposed K fragments of dQ(0), dQ(1)
        auto fetch = [&](int f) {
            if (f < NROW) {
                const int phase = f / DC, dc = f % DC;            // phase: 0 S(0), 1 dP(0), 2 S(1), 3 dP(1)
                return *reinterpret_cast<const bf16x8*>(((phase & 1) ? vs : ks) + koff[dc] + 32 * (phase >> 1) * RS);
            }
            const int g = f - NROW, cc = g / DB, db = g % DB;      // cc = 16-key chunk of the tile
            const u32x2 lo = lds_read_tr16(ks + toff[0][db] + 16 * cc * RS);
            const u32x2 hi = lds_read_tr16(ks + toff[1][db] + 16 * cc * RS);
            const u32x4 u = {lo[0], lo[1], hi[0], hi[1]};
            return __builtin_bit_cast(bf16x8, u);
        };
        bf16x8 fb[PD];
#pragma unroll
        for (int i = 0; i < PD; ++i) {
            fb[i] = fetch(i);
            __builtin_amdgcn_sched_barrier(0);
        }

        f32x16 sacc[2], dpacc[2];
        bf16x8 dsf[2][2];
        // a lane's 64 keep-mask bytes of the tile in four 16-byte loads where the layout allows it, fetched
        // one tile ahead
        const bool vec_mask = HASMASK && MASKED && p.m.rows16 && key0 + BN <= p.Sk;
        MaskRow64 mrow = mnext;
        if constexpr (VECMASK) {
            // two workgroups per unit: the other wavefront of the SIMD covers the load, and a second row in
            // registers would spill
            mrow.load(mbase + (int64_t)min(qrow, p.Sq - 1) * p.m.sq + key0);
            // the key length and the causal diagonal cut few tiles: there they are folded into the mask bytes,
            // so that the per-element test is the mask byte alone
            const int lim = (p.m.causal ? min(klimit, qrow + 1) : klimit) - key0;
            if (__any(lim < BN)) mrow.restrict_to(lim);
        } else if (HASMASK && MASKED && p.m.rows16 && key0 + 2 * BN <= p.Sk && t + 1 < n_tiles) {
            mnext.load(mbase + (int64_t)min(qrow, p.Sq - 1) * p.m.sq + key0 + BN);
        }
        auto p_elem = [&](int kb, int r) {          // P^T: one query per lane, so LSE is a per-lane scalar
            float pr = exp2_fast(fmaf(sacc[kb][r], c_log2, -lse2));
            if constexpr (VECMASK) {
                pr = mrow.keep(kb, r, h) ? pr : 0.f;
            } else if constexpr (KEYS && MASKED) {
                pr = keep_bits[kb] & (1u << (8 * (r >> 2) + (r & 3))) ? pr : 0.f;
            } else if (MASKED) {
                const int key = key0 + 32 * kb + acc_row(r, h);
                bool drop = (key >= klimit) | ((p.m.causal != 0) & (key > qrow + past));     // bitwise: selects, not branches
                if (HASMASK) {
                    if (vec_mask) drop = drop || !mrow.keep(kb, r, h);
                    else if (!drop && qok) drop = !mask_attends(p.m, mbase, (int64_t)qrow * p.m.sq + (int64_t)key * p.m.sk);
                }
                pr = drop ? 0.f : pr;
            }
            sacc[kb][r] = pr;
        };
        auto ds_elem = [&](int kb, int r) {         // dS^T = P^T (dP^T - delta), packed after 8 and 16
            // O = (P f) V with f = 0 or 1 / (1 - p): dP = f (dO V^T), and rowsum(dP P) is still rowsum(dO O)
            const uint32_t off = 32 * kb + 8 * (r >> 2) + (r & 3);       // of the element, from drop_tile
            if constexpr (DROP == kDropTiled) {
                const float f = drop_factor_at(p.m, (uint32_t)bh, (uint32_t)qrow, (uint32_t)(key0 + 4 * h) + off, (uint32_t)p.Sq, (uint32_t)p.Sk);
                dpacc[kb][r] = sacc[kb][r] * fmaf(f, dpacc[kb][r], -delta);
            } else if constexpr (DROP != kDropNone) {
                const uint32_t w = DROP == kDropRows64 ? drop_word ^ xorshift32(off) : xorshift32(p.m.drop_seed ^ (drop_tile + off));
                dpacc[kb][r] = sacc[kb][r] * fmaf(w >= p.m.drop_thr32 ? dpacc[kb][r] : 0.f, p.m.drop_scale, -delta);
            } else {
                dpacc[kb][r] = sacc[kb][r] * (dpacc[kb][r] - delta);
            }
            if ((r & 7) == 7) {
                const int o8 = r - 7;
                const f32x16& d = dpacc[kb];
                dsf[kb][r >> 3] = pack8(d[o8], d[o8 + 1], d[o8 + 2], d[o8 + 3], d[o8 + 4], d[o8 + 5], d[o8 + 6], d[o8 + 7]);
            }
        };
        // logits per MFMA slot of a phase: slot s of n has 16 s / n to 16 (s + 1) / n
        static_assert(DC == 2 * DB, "the phases have the same number of slots");
        constexpr int EPM = (16 + DC - 1) / DC;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                sacc[kb][r] = 0.f;
                dpacc[kb][r] = 0.f;
            }
        auto row_phase = [&](auto phase_tag) {
            constexpr int PH = decltype(phase_tag)::value, KB = PH >> 1;
#pragma unroll
            for (int dc = 0; dc < DC; ++dc) {
                constexpr int F0 = PH * DC;
                const int f = F0 + dc;
                if (PH & 1) dpacc[KB] = mfma32(fb[f % PD], dof[dc], dpacc[KB]);
                else sacc[KB] = mfma32(fb[f % PD], qf[dc], sacc[KB]);
                fb[f % PD] = fetch(f + PD);
#pragma unroll
                for (int e = 0; e < EPM; ++e) {
                    const int r = 16 * dc / DC + e;
                    if (r >= 16 * (dc + 1) / DC) continue;
                    if (PH == 1) p_elem(0, r);
                    if (PH == 2) ds_elem(0, r);
                    if (PH == 3) p_elem(1, r);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto dq_phase = [&](auto kb_tag) {
            constexpr int KB = decltype(kb_tag)::value;
#pragma unroll
            for (int g = 0; g < 2 * DB; ++g) {
                const int f = NROW + 2 * DB * KB + g, c = g / DB, db = g % DB;
                dqacc[db] = mfma32(fb[f % PD], dsf[KB][c], dqacc[db]);
                if (f + PD < NALL) fb[f % PD] = fetch(f + PD);
                if (KB == 0) {
#pragma unroll
                    for (int e = 0; e < EPM; ++e)
                        if (16 * g / DC + e < 16 * (g + 1) / DC) ds_elem(1, 16 * g / DC + e);
                }
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        row_phase(std::integral_constant<int, 0>{});
        row_phase(std::integral_constant<int, 1>{});
        row_phase(std::integral_constant<int, 2>{});
        row_phase(std::integral_constant<int, 3>{});
        dq_phase(std::integral_constant<int, 0>{});
        dq_phase(std::integral_constant<int, 1>{});

        wait_vm0();
        __syncthreads();
    };

    int n_full = HASMASK ? 0 : KEYS ? kt.n_whole : klimit / BN;
    if (p.m.causal) n_full = min(n_full, PACKED ? max(q0 + 1 + past, 0) / BN : (q0 + 1) / BN);
    n_full = min(n_full - t_lo, n_tiles);
    using IM = std::integral_constant<int, -1>;
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    {
        int t = 0;
        for (; t + 2 < n_full; t += 2) {      // tiles t+1 and t+2 are full: straight-line copies, fixed stages
            tile_step(std::false_type{}, I1{}, I0{}, t);
            tile_step(std::false_type{}, I1{}, I1{}, t + 1);
        }
        for (; t < n_full; ++t) tile_step(std::false_type{}, I2{}, IM{}, t);
        for (; t < n_tiles; ++t) tile_step(std::true_type{}, I2{}, IM{}, t);
    }

    if constexpr (KG == 2) {
        for (int i = n_tiles; i < n_first; ++i) __syncthreads();        // one barrier per tile: the second group's walk may be one shorter
        static_assert(NW * 4 * DB * 64 * 16 <= T::LDS_BYTES, "the sums of a group fit in its own stages");
        f32x4* slot = reinterpret_cast<f32x4*>(lds_all + T::LDS_BYTES / 2) + wave * 4 * DB * 64 + lane;
        if (group == 1) {
#pragma unroll
            for (int i = 0; i < 4 * DB; ++i) {
                const f32x16& a = dqacc[i >> 2];
                slot[64 * i] = f32x4{a[4 * (i & 3)], a[4 * (i & 3) + 1], a[4 * (i & 3) + 2], a[4 * (i & 3) + 3]};
            }
        }
        __syncthreads();
        if (group == 1) return;
#pragma unroll
        for (int i = 0; i < 4 * DB; ++i) {
            const f32x4 v = slot[64 * i];
#pragma unroll
            for (int e = 0; e < 4; ++e) dqacc[i >> 2][4 * (i & 3) + e] += v[e];
        }
    }

    // ---- epilogue: fp32 partial sums for bwd_dq_merge_kernel, in accumulator order: [db][group of four][thread] ...
    if (parts > 1) {
        float* dst = p.split_ws + (PACKED ? (size_t)wg : (size_t)wg * parts + part) * (size_t)(BM * D);
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int g = 0; g < 4; ++g) {
                const f32x16& a = dqacc[db];
                *reinterpret_cast<f32x4*>(dst + ((size_t)(db * 4 + g) * 256 + tid) * 4) = f32x4{a[4 * g], a[4 * g + 1], a[4 * g + 2], a[4 * g + 3]};
            }
        return;
    }
    // ... or dQ = scale * dQ^T, bf16 (every walk ended with a barrier: the tiles are free)
    uint16_t* const dqbase = PACKED ? p.dq + u.q_at(p.dqs) : p.dq + b * p.dqs.b + hh * p.dqs.h;
    store_rows32<D>(lds_all + wave * 32 * RS, dqbase + (int64_t)qw0 * p.dqs.n, p.dqs.n, Sq - qw0, p.d, [&](int db, int g) {
        const f32x16& a = dqacc[db];
        return u32x2{pack_bf16(a[4 * g] * p.scale, a[4 * g + 1] * p.scale), pack_bf16(a[4 * g + 2] * p.scale, a[4 * g + 3] * p.scale)};
    });
}

template <int D, int EXCL, int NW, int DROP = kDropNone, int KG = 1>
__global__ __launch_bounds__(64 * NW * KG, (NW == 4 && EXCL != kExGeneral) ? 2 : 1) void bwd_dq_kernel(const BwdParams p) {
    bwd_dq_body<D, EXCL, NW, DROP, KG, false>(p);
}
template <int D, int EXCL, int NW>
__global__ __launch_bounds__(64 * NW, (NW == 4 && EXCL != kExGeneral) ? 2 : 1) void bwd_dq_dealt_kernel(const BwdParams p) {
    bwd_dq_body<D, EXCL, NW, kDropNone, 1, true>(p);
}

// Sums the fp32 partials of the workgroups that shared a 128-query tile and writes dQ.  One workgroup per (tile, 32-wide block
// of d); the thread layout mirrors the accumulators.
template <int D>
__global__ __launch_bounds__(256) void bwd_dq_merge_kernel(const BwdParams p) {
    constexpr int BM = BwdDqTile<D>::BM, DB = D / 32;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5;
    const int wg = (int)blockIdx.x / DB, db = (int)blockIdx.x % DB;
    const int n_qt = (p.Sq + BM - 1) / BM;
    const int bh = wg / n_qt, b = bh / p.H, hh = bh % p.H;
    f32x4 acc[4];
#pragma unroll
    for (int g = 0; g < 4; ++g) acc[g] = f32x4{0.f, 0.f, 0.f, 0.f};
    const float* src = p.split_ws + (size_t)wg * p.dq_parts * (size_t)(BM * D) + ((size_t)db * 4 * 256 + tid) * 4;
#pragma unroll 4
    for (int part = 0; part < p.dq_parts; ++part, src += (size_t)(BM * D)) {
#pragma unroll
        for (int g = 0; g < 4; ++g) acc[g] += *reinterpret_cast<const f32x4*>(src + g * 1024);
    }
    const int row = (wg % n_qt) * BM + 32 * wave + n;
    if (row >= p.Sq) return;
    uint16_t* dqrow = p.dq + b * p.dqs.b + hh * p.dqs.h + (int64_t)row * p.dqs.n;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        const u32x2 w = {pack_bf16(acc[g][0] * p.scale, acc[g][1] * p.scale), pack_bf16(acc[g][2] * p.scale, acc[g][3] * p.scale)};
        if (32 * db + 8 * g + 4 * h < p.d) *reinterpret_cast<u32x2*>(dqrow + 32 * db + 8 * g + 4 * h) = w;
    }
}

// ---------------------------------------------------------------------------- dq, 256-query workgroups
// The same computation as bwd_dq_kernel for workgroups of 256 queries, laid out for one wavefront per
// SIMD: 4 wavefronts of 64 queries (two 32-query blocks) each.  Every K / V fragment read from LDS then
// feeds two MFMAs (one per query block), which halves the LDS reads and waits per MFMA; the register
// file of a lone wavefront holds dQ^T of both blocks and the Q / dO fragments in the accumulation
// registers (Q / dO as MFMA B operands), and S^T / dP^T in architectural registers through hand-emitted
// MFMAs (see mfma32_vgpr_bacc).  dP^T starts from -delta, so dS^T = P^T * dP'^T is one multiply.
// Three LDS stages of K / V tiles, one barrier per tile, one ring of fragment reads that runs on into
// the next tile, copies split around MFMAs and spread over the tile: as in bwd_dkdv_kernel.
// No explicit keep-mask variant: such problems use bwd_dq_kernel.
template <int D>
struct BwdDqWideTile {
    static constexpr int BM = 256;                  // query rows per workgroup (64 per wavefront)
    static constexpr int BN = 64;                   // keys per tile
    static constexpr int RS = kRowPitch<D>;
    static constexpr int TILE_ELEMS = BN * RS;
    static constexpr int STAGE_ELEMS = 2 * TILE_ELEMS;            // K tile + V tile
    static constexpr int NSTAGE = 3;
    static constexpr int LDS_BYTES = NSTAGE * STAGE_ELEMS * 2;
    static constexpr int ROWS_PER_DMA = 1024 / (RS * 2);
    static constexpr int DMA_PER_WAVE = BN / ROWS_PER_DMA / 4;    // 1 KiB copies per wave and tensor
};

template <int D, bool DEALT = false>
__device__ __forceinline__ void bwd_dq_wide_body(const BwdParams& p, const int block, const int nblocks) {
    using T = BwdDqWideTile<D>;
    constexpr int BM = T::BM, BN = T::BN, RS = T::RS;
    constexpr int DC = D / 16;
    constexpr int DB = D / 32;
    constexpr int GPR = RS / 8;
    constexpr int NDMA = T::DMA_PER_WAVE;

    extern __shared__ __attribute__((aligned(1024))) uint16_t lds[];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 31, h = lane >> 5;

    const int n_qt = (p.Sq + BM - 1) / BM;
    const bool falling = p.m.causal && !p.m.kv_len;
    const int wg = xcd_remap_heads(block, nblocks, n_qt, p.m.kv_len != nullptr, falling);
    int qt = wg % n_qt, bh = wg / n_qt;
    if constexpr (DEALT) {
        int t, s;
        dealt_unit(block, n_qt, p.B, p.H, !falling, t, s);
        qt = __builtin_amdgcn_readfirstlane(falling ? n_qt - 1 - t : t);
        bh = __builtin_amdgcn_readfirstlane(s);
    } else if (falling) {
        causal_longest_first(wg, n_qt, nblocks, qt, bh);
    }
    const int b = bh / p.H, hh = bh % p.H;
    const int q0 = qt * BM;
    const int qw0 = q0 + wave * 64;

    const uint16_t* qbase = p.q + b * p.qs.b + hh * p.qs.h;
    const uint16_t* kbase = p.k + b * p.ks.b + hh * p.ks.h;
    const uint16_t* vbase = p.v + b * p.vs.b + hh * p.vs.h;
    const uint16_t* dobase = p.dout + b * p.dos.b + hh * p.dos.h;

    int klimit = p.Sk;
    if (p.m.kv_len) klimit = min(klimit, max(p.m.kv_len[b], 0));
    int kend = klimit;
    if (p.m.causal) kend = min(kend, q0 + BM);
    const int n_tiles = (kend + BN - 1) / BN;

    // ---- asynchronous staging of the K / V tiles
    const int dma_row_in = lane / GPR, dma_gran = lane % GPR;
    const uint32_t lds0 = lds_addr(lds);
    uint32_t k_lane_off[NDMA], v_lane_off[NDMA];     // bytes
#pragma unroll
    for (int i = 0; i < NDMA; ++i) {
        const int row = (wave * NDMA + i) * T::ROWS_PER_DMA + dma_row_in;
        const int c = src_granule(dma_gran ^ swz<D>(row), p.d);
        k_lane_off[i] = 2u * (uint32_t)(row * (int)p.ks.n + c * 8);
        v_lane_off[i] = 2u * (uint32_t)(row * (int)p.vs.n + c * 8);
    }
    auto dst_of = [&](int stg, int which, int i) {    // LDS byte address of copy i of this wave (which: 0 = K, 1 = V)
        return lds0 + 2u * (uint32_t)(stg * T::STAGE_ELEMS + which * T::TILE_ELEMS + (wave * NDMA + i) * 512);
    };
    auto issue_tile = [&](int t, int stg) {          // any tile: rows past the attended range re-read the last attended key
#pragma unroll
        for (int i = 0; i < NDMA; ++i) {
            const int row = (wave * NDMA + i) * T::ROWS_PER_DMA + dma_row_in;
            const int key = max(min(t * BN + row, klimit - 1), 0);
            const int c = src_granule(dma_gran ^ swz<D>(row), p.d);
            dma16(kbase + (int64_t)key * p.ks.n + c * 8, dst_of(stg, 0, i));
            dma16(vbase + (int64_t)key * p.vs.n + c * 8, dst_of(stg, 1, i));
        }
    };

    if (n_tiles > 0) issue_tile(0, 0);

    // ---- Q and dO fragments (B operands: column = query, 8 consecutive d) and the per-query scalars of
    //      both query blocks, through stage 2; -delta and lse2 are also left in the workspace for the dK/dV kernel
    bf16x8 qf[2][DC], dof[2][DC];          // pinned to accumulation registers: slots qb*DC + dc and 16 + qb*DC + dc
    float lse2[2];
    f32x16 ndelta16[2];
    int qrow[2];
    static_for<2>([&](auto qb_tag) {
        constexpr int qb = decltype(qb_tag)::value;
        const int row0 = qw0 + 32 * qb;
        qrow[qb] = row0 + n;
        const bool qok = qrow[qb] < p.Sq;
        uint16_t* const pass = lds + 2 * T::STAGE_ELEMS + wave * 1024;
        u32x4 wq[DC], wd[DC], wo[DC];
        load_rows32<D>(wq, qbase + (int64_t)row0 * p.qs.n, p.qs.n, p.Sq - row0, p.d);
        load_rows32<D>(wd, dobase + (int64_t)row0 * p.dos.n, p.dos.n, p.Sq - row0, p.d);
        if (!p.rows_ready) load_rows32<D>(wo, p.o + b * p.os.b + hh * p.os.h + (int64_t)row0 * p.os.n, p.os.n, p.Sq - row0, p.d);
        fragments_of_rows32<D>(pass, wq, [&](auto dc_tag, u32x4 f) {
            constexpr int dc = decltype(dc_tag)::value;
            qf[qb][dc] = pin_b_fragment<qb * DC + dc>(f);
        });
        u32x4 dvf[DC];
        fragments_of_rows32<D>(pass, wd, [&](auto dc_tag, u32x4 f) {
            constexpr int dc = decltype(dc_tag)::value;
            dvf[dc] = f;
            dof[qb][dc] = pin_b_fragment<16 + qb * DC + dc>(f);
        });
        lse2[qb] = INFINITY;
        float nd = 0.f;
        if (p.rows_ready) {       // bwd_rows_kernel has left both rows in the workspace
            if (qok) {
                nd = p.ndelta[(int64_t)bh * p.Sq + qrow[qb]];
                lse2[qb] = p.lse2[(int64_t)bh * p.Sq + qrow[qb]];
            }
        } else {
            float part = 0.f;
            fragments_of_rows32<D>(pass, wo, [&](auto dc_tag, u32x4 ov) {
                const u32x4 dv = dvf[decltype(dc_tag)::value];
#pragma unroll
                for (int i = 0; i < 4; ++i) part += bf16_lo(dv[i]) * bf16_lo(ov[i]) + bf16_hi(dv[i]) * bf16_hi(ov[i]);
            });
            part += xhalf(part);
            if (qok) {
                const float l = p.lse[(int64_t)bh * p.Sq + qrow[qb]];
                lse2[qb] = (l == -INFINITY) ? INFINITY : l * kLog2e;
                nd = -part;
                if (h == 0) {
                    p.ndelta[(int64_t)bh * p.Sq + qrow[qb]] = nd;
                    p.lse2[(int64_t)bh * p.Sq + qrow[qb]] = lse2[qb];
                }
            }
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) ndelta16[qb][r] = nd;
    });

    int koff[DC];          // 16-byte row reads of K / V: row 32*kb + n, logical granule 2*dc + h
#pragma unroll
    for (int dc = 0; dc < DC; ++dc) koff[dc] = n * RS + (((2 * dc + h) ^ swz<D>(n)) << 3);
    const int tr_r = lane & 15, tr_g16 = (lane >> 4) & 1;
    int toff[2][DB];       // transposing reads of K: rows 4h + r/4 (+8), logical granule 4*db + 2*g16 + (r&3)/2
#pragma unroll
    for (int half = 0; half < 2; ++half) {
        const int row = 4 * h + (tr_r >> 2) + 8 * half;
#pragma unroll
        for (int db = 0; db < DB; ++db)
            toff[half][db] = row * RS + (((4 * db + 2 * tr_g16 + ((tr_r & 3) >> 1)) ^ swz<D>(row)) << 3) + 4 * (tr_r & 1);
    }

    const float c_log2 = p.scale * kLog2e;
    f32x16 dqacc[2][DB];      // dQ^T: rows = d, column = this lane's query of block qb
#pragma unroll
    for (int qb = 0; qb < 2; ++qb)
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r = 0; r < 16; ++r) dqacc[qb][db][r] = 0.f;

    // Operand fragments of a tile, in consumption order; each feeds two MFMAs (query blocks 0 and 1):
    //   [0, DC) K rows of key block 0 (S), [DC, 2DC) V rows of block 0 (dP), then the same for block 1,
    //   [4DC, 4DC + 2DB) K^T of key block 0 by (16-key chunk, db) (dQ), then of block 1
    constexpr int NROW = 4 * DC, NF = NROW + 4 * DB;
    constexpr int PD = 4;                            // read-ahead depth of the fragment ring
    static_assert(NF % PD == 0, "read-ahead depth must divide the fragment count");
    auto fetch = [&](const uint16_t* ks, int f) {
        const uint16_t* vs = ks + T::TILE_ELEMS;
        if (f < NROW) {
            const int phase = f / DC, dc = f % DC;            // phase: 0 S(0), 1 dP(0), 2 S(1), 3 dP(1)
            return *reinterpret_cast<const bf16x8*>(((phase & 1) ? vs : ks) + koff[dc] + 32 * (phase >> 1) * RS);
        }
        const int g = f - NROW, cc = g / DB, db = g % DB;      // cc = 16-key chunk of the tile
        const u32x2 lo = lds_read_tr16(ks + toff[0][db] + 16 * cc * RS);
        const u32x2 hi = lds_read_tr16(ks + toff[1][db] + 16 * cc * RS);
        const u32x4 u = {lo[0], lo[1], hi[0], hi[1]};
        return __builtin_bit_cast(bf16x8, u);
    };
    bf16x8 fb[PD];
    if (n_tiles > 0) {
        wait_vm0();
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PD; ++i) fb[i] = fetch(lds, i);
    }

    // One tile of 64 keys = two key blocks of 32, six phases of 2 DC MFMAs (MFMA slot = 2 * fragment +
    // query block).  The element-wise work of a phase is threaded between the MFMAs of the next one:
    //   S(0) | dP(0) + P(0) | S(1) + dS(0) | dP(1) + P(1) | dQ(0) + dS(1) | dQ(1)
    // (16 slots:) element e of query block 0 goes with slot e of its phase, that of query block 1 with slot e + 1
    // (its S / dP are complete one MFMA later), the sixteenth spilling into the first slot of the
    // next phase: every hand-emitted MFMA result is first touched two MFMAs after it was issued.
    // COPY: 1 = the next tile is a full one (copies split around the MFMAs), 2 = decide at run time.
    // STAGE: LDS stage that holds this tile (0 / 1 / 2), or -1 to take it from st.
    auto tile_step = [&](auto masked_tag, auto copy_tag, auto stage_tag, int st, int t, const uint16_t* nk_base,
                         const uint16_t* nv_base) {
        constexpr bool MASKED = decltype(masked_tag)::value;
        constexpr int COPY = decltype(copy_tag)::value;
        constexpr int STAGE = decltype(stage_tag)::value;
        const int cur = STAGE >= 0 ? STAGE : st;
        const int nxt = STAGE >= 0 ? (STAGE + 1) % 3 : (st == 2 ? 0 : st + 1);
        const bool have_next = COPY == 1 || t + 1 < n_tiles;
        if (COPY == 2 && have_next) issue_tile(t + 1, nxt);
        const uint16_t* ks = lds + cur * T::STAGE_ELEMS;
        const uint16_t* kn = lds + nxt * T::STAGE_ELEMS;
        const int key0 = t * BN;

        f32x16 sacc[2][2], dpacc[2][2];             // [query block][key block]
        u32x4 dsw[2][2][2];                         // dS^T operands: [query block][key block][16-key chunk]

        auto p_elem = [&](int qb, int kb, int r) {  // P^T: one query per lane, so LSE is a per-lane scalar
            float pr = exp2_fast(fmaf(sacc[qb][kb][r], c_log2, -lse2[qb]));
            if (MASKED) {
                const int key = key0 + 32 * kb + acc_row(r, h);
                const bool drop = (key >= klimit) | ((p.m.causal != 0) & (key > qrow[qb]));     // bitwise: selects, not branches
                pr = drop ? 0.f : pr;
            }
            sacc[qb][kb][r] = pr;
        };
        auto ds_elem = [&](int qb, int kb, int r) { // dS^T = P^T * (dP^T - delta), packed in pairs
            f32x16& d = dpacc[qb][kb];
            d[r] = sacc[qb][kb][r] * d[r];
            if (r & 1) dsw[qb][kb][r >> 3][(r & 7) >> 1] = pack_bf16(d[r - 1], d[r]);
        };
        // element-wise work that goes with MFMA slot i of phase ph
        constexpr int NSL = 2 * DC;                 // MFMA slots per phase
        constexpr int EL = (16 + NSL - 1) / NSL;
        auto elems_at = [&](int qb, int i, auto fn) {      // elements 16 i / NSL to 16 (i + 1) / NSL
#pragma unroll
            for (int e = 0; e < EL; ++e)
                if (16 * i / NSL + e < 16 * (i + 1) / NSL) fn(qb, 16 * i / NSL + e);
        };
        auto elems_of = [&](int ph, int i, auto fn) {      // fn(qb, e) for the elements scheduled at (ph, i)
            elems_at(0, i, fn);
            if (i > 0) elems_at(1, i - 1, fn);             // query block 1: one slot later
        };
        auto spill_of = [&](auto fn) { elems_at(1, NSL - 1, fn); };     // its last elements, in slot 0 of the next phase
        // copies of the next tile: copy j goes with MFMA slot CS * j + 1 of the S / dP phases
        constexpr int NCOPY = 2 * NDMA;
        constexpr int CS = (4 * NSL - 2) / NCOPY;
        static_assert(CS >= 2, "copies do not fit the S / dP phases");
        auto copy_dst = [&](int g) {
            const int j = (g - 1) / CS;
            if (COPY == 1 && g >= 1 && (g - 1) % CS == 0 && j < NCOPY) dma_set_dst(dst_of(nxt, j & 1, j >> 1));
        };
        auto copy_issue = [&](int g) {
            const int j = (g - 1) / CS;
            if (COPY == 1 && g >= 1 && (g - 1) % CS == 0 && j < NCOPY) {
                if (j & 1) dma16u_issue(nv_base, v_lane_off[j >> 1]);
                else dma16u_issue(nk_base, k_lane_off[j >> 1]);
            }
        };
        auto refill = [&](int f) {
            const int nf = f + PD;
            if (nf < NF) fb[f % PD] = fetch(ks, nf);
            else if (have_next) fb[f % PD] = fetch(kn, nf - NF);
        };
        auto side = [&](int ph, int i) {
            if (ph == 1) elems_of(ph, i, [&](int qb, int e) { p_elem(qb, 0, e); });
            if (ph == 2) {
                if (i == 0) spill_of([&](int qb, int e) { p_elem(qb, 0, e); });
                elems_of(ph, i, [&](int qb, int e) { ds_elem(qb, 0, e); });
            }
            if (ph == 3) {
                if (i == 0) spill_of([&](int qb, int e) { ds_elem(qb, 0, e); });
                elems_of(ph, i, [&](int qb, int e) { p_elem(qb, 1, e); });
            }
            if (ph == 4) {
                if (i == 0) spill_of([&](int qb, int e) { p_elem(qb, 1, e); });
                elems_of(ph, i, [&](int qb, int e) { ds_elem(qb, 1, e); });
            }
            if (ph == 5 && i == 0) spill_of([&](int qb, int e) { ds_elem(qb, 1, e); });
        };

        auto row_phase = [&](auto phase_tag) {      // S^T(kb) = K Q^T or dP^T(kb) = V dO^T - delta
            constexpr int PH = decltype(phase_tag)::value, KB = PH >> 1;
            static_for<DC>([&](auto dc_tag) {
                constexpr int dc = decltype(dc_tag)::value;
                constexpr int f = PH * DC + dc;
                static_for<2>([&](auto qb_tag) {
                    constexpr int qb = decltype(qb_tag)::value;
                    constexpr int i = 2 * dc + qb, g = PH * NSL + i;
                    constexpr int SLOT = ((PH & 1) ? 16 : 0) + qb * DC + dc;      // Q fragments first, then dO
                    copy_dst(g);
                    if constexpr (PH & 1)
                        mfma32_vgpr_bpinned<SLOT, dc == 0 ? 2 : 1>(dpacc[qb][KB], fb[f % PD], dof[qb][dc], ndelta16[qb]);
                    else
                        mfma32_vgpr_bpinned<SLOT, dc == 0 ? 0 : 1>(sacc[qb][KB], fb[f % PD], qf[qb][dc], ndelta16[qb]);
                    __builtin_amdgcn_sched_barrier(0);      // the element-wise work below must not move above this MFMA
                    copy_issue(g);
                    side(PH, i);
                    if (qb == 1) refill(f);
                    __builtin_amdgcn_sched_barrier(0);
                });
            });
        };
        auto dq_phase = [&](auto kb_tag) {          // dQ^T += K^T(kb) dS^T(kb)
            constexpr int KB = decltype(kb_tag)::value;
#pragma unroll
            for (int g = 0; g < 2 * DB; ++g) {
                const int f = NROW + 2 * DB * KB + g, c = g / DB, db = g % DB;
#pragma unroll
                for (int qb = 0; qb < 2; ++qb) {
                    dqacc[qb][db] = mfma32(fb[f % PD], __builtin_bit_cast(bf16x8, dsw[qb][KB][c]), dqacc[qb][db]);
                    __builtin_amdgcn_sched_barrier(0);
                    side(4 + KB, 2 * g + qb);
                    if (qb == 1) {
                        if (f == NF - PD && have_next) {
                            __builtin_amdgcn_sched_barrier(0);
                            wait_vm0();                          // this wave's copies of the next tile have landed
                            __builtin_amdgcn_s_barrier();        // ... everyone's have, and everyone is past the previous tile
                            __builtin_amdgcn_sched_barrier(0);
                        }
                        refill(f);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
        };
        row_phase(std::integral_constant<int, 0>{});
        row_phase(std::integral_constant<int, 1>{});
        row_phase(std::integral_constant<int, 2>{});
        row_phase(std::integral_constant<int, 3>{});
        dq_phase(std::integral_constant<int, 0>{});
        dq_phase(std::integral_constant<int, 1>{});
    };

    int n_full = klimit / BN;
    if (p.m.causal) n_full = min(n_full, (q0 + 1) / BN);
    n_full = min(n_full, n_tiles);
    using IM = std::integral_constant<int, -1>;
    using I0 = std::integral_constant<int, 0>;
    using I1 = std::integral_constant<int, 1>;
    using I2 = std::integral_constant<int, 2>;
    {
        const int64_t k_tile_stride = (int64_t)BN * p.ks.n, v_tile_stride = (int64_t)BN * p.vs.n;
        const uint16_t* nk = kbase + k_tile_stride;      // the tile after the current one
        const uint16_t* nv = vbase + v_tile_stride;
        int t = 0, st = 0;
        for (; t + 3 < n_full; t += 3) {      // tiles t+1 .. t+3 are full: straight-line copies, fixed stages
            tile_step(std::false_type{}, I1{}, I0{}, 0, t, nk, nv);
            nk += k_tile_stride, nv += v_tile_stride;
            tile_step(std::false_type{}, I1{}, I1{}, 1, t + 1, nk, nv);
            nk += k_tile_stride, nv += v_tile_stride;
            tile_step(std::false_type{}, I1{}, I2{}, 2, t + 2, nk, nv);
            nk += k_tile_stride, nv += v_tile_stride;
        }
        for (; t < n_full; ++t) {
            tile_step(std::false_type{}, I2{}, IM{}, st, t, nk, nv);
            st = st == 2 ? 0 : st + 1;
        }
        for (; t < n_tiles; ++t) {
            tile_step(std::true_type{}, I2{}, IM{}, st, t, nk, nv);
            st = st == 2 ? 0 : st + 1;
        }
    }

    // ---- epilogue: dQ = scale * dQ^T, bf16
    __syncthreads();              // nobody reads a tile any more
#pragma unroll
    for (int qb = 0; qb < 2; ++qb) {
        const int row0 = qw0 + 32 * qb;
        store_rows32<D>(lds + wave * 32 * RS, p.dq + b * p.dqs.b + hh * p.dqs.h + (int64_t)row0 * p.dqs.n, p.dqs.n, p.Sq - row0, p.d, [&](int db, int g) {
            const f32x16& a = dqacc[qb][db];
            return u32x2{pack_bf16(a[4 * g] * p.scale, a[4 * g + 1] * p.scale), pack_bf16(a[4 * g + 2] * p.scale, a[4 * g + 3] * p.scale)};
        });
    }
}

template <int D>
__global__ __launch_bounds__(256) void bwd_dq_wide_kernel(const BwdParams p) {
    bwd_dq_wide_body<D>(p, (int)blockIdx.x, (int)gridDim.x);
}
template <int D>
__global__ __launch_bounds__(256) void bwd_dq_wide_dealt_kernel(const BwdParams p) {
    bwd_dq_wide_body<D, true>(p, (int)blockIdx.x, (int)gridDim.x);
}

// ------------------------------------------------------------------------------- per-query rows
// -delta_i = -sum_d dO_id * O_id and LSE_i * log2(e) (+inf where LSE = -inf) for every query row, as a pass of its
// own: with both rows in the workspace beforehand (BwdParams::rows_ready) the dQ and dK/dV walks no longer depend
// on each other and can share one grid.  D / 8 lanes per row, one 16-byte granule of O and of dO each.
template <int D>
__global__ __launch_bounds__(256) void bwd_rows_kernel(const BwdParams p) {
    constexpr int LPR = D / 8;                       // lanes per row
    constexpr int ROWS = 256 / LPR;                  // rows per workgroup
    const int tid = threadIdx.x;
    const int g = tid % LPR;
    const int64_t row = (int64_t)blockIdx.x * ROWS + tid / LPR;       // over [B*H, Sq]
    const int64_t n_rows = (int64_t)p.B * p.H * p.Sq;
    const bool ok = row < n_rows;
    const int64_t rr = ok ? row : 0;
    const int bh = (int)(rr / p.Sq), qi = (int)(rr % p.Sq);
    const int b = bh / p.H, hh = bh % p.H;
    const bool in_d = ok && 8 * g < p.d;
    const u32x4 ov = ldg16(p.o + b * p.os.b + hh * p.os.h + (int64_t)qi * p.os.n + 8 * g, in_d);
    const u32x4 dv = ldg16(p.dout + b * p.dos.b + hh * p.dos.h + (int64_t)qi * p.dos.n + 8 * g, in_d);
    float part = 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i) part += bf16_lo(dv[i]) * bf16_lo(ov[i]) + bf16_hi(dv[i]) * bf16_hi(ov[i]);
#pragma unroll
    for (int off = LPR / 2; off > 0; off >>= 1) part += __shfl_xor(part, off, 64);
    if (ok && g == 0) {
        const float l = p.lse[row];
        p.ndelta[row] = -part;
        p.lse2[row] = (l == -INFINITY) ? INFINITY : l * kLog2e;
    }
}

// ------------------------------------------------------------------------ dQ and dK/dV in one grid
// For problems whose walks are all equally long (no causal flag, key lengths or mask) and fill 256-query
// workgroups: the dQ workgroups (the longer ones) come first in dispatch order, the whole dK/dV key blocks next,
// the split ones last, so that compute units freed by one kind of workgroup go on with the next and only the
// short split pieces make up the tail.  Needs the per-query rows beforehand (bwd_rows_kernel).
template <int D>
__global__ __launch_bounds__(256) void bwd_joint_kernel(const BwdParams p) {
    const int block = (int)blockIdx.x;
    if (block < p.joint_n_dq) bwd_dq_wide_body<D>(p, block, p.joint_n_dq);
    else bwd_dkdv_body<D, false, false>(p, block - p.joint_n_dq, (int)gridDim.x - p.joint_n_dq);
}

}  // namespace fattn
