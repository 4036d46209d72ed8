// Attention of packed sequences of different lengths with grouped heads (packed_units.hpp), forward and backward: the loops are those
// of attn_fwd.hpp, attn_fwd_keyshare.hpp and attn_bwd.hpp, on one sequence of the packed tensors each.
//
//   forward   O_i = sum_j P_ij v_j,  P_ij = exp(scale q_i k_j - LSE_i),  j < Sk, and j <= i + Sk - Sq under the causal flag
//   backward  dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale sum over the heads of a key head of dS^T Q,  dV = the same of P^T dO
//
// The sums over the heads that share a key head are one walk, of one workgroup or in parts that are joined in their order: no atomics, no
// partial gradients per head.
//
// What bounds them is what bounds the dense kernels, at their rates: the matrix instructions and the exponentials between them.  Forward,
// eight prompts of 1 to 4096, 32 heads on 8, D = 128: 292 to 319 us by the card, 0.91 to 1.0 PFLOP/s (as much as the dense causal one on 4096); training on six
// documents of 333 to 4608, the same heads: forward 360 to 370, dQ 500 to 520, dK/dV 660 to 680 us.  Small batches: the longest walk, one step of 64 keys after the other at 0.6 to 1 us;
// a few heads of 1000 to 2000 rows: forward 13 to 18 us, backward 48 to 58.
// Roundings to 16 bits, which the matrix instructions' operands take: P before it meets V and dO, dS before it meets K and Q, O as it is saved,
// from which delta is formed; all sums are fp32.  dQ and dK are therefore off by 0.0025 of their root mean square against 0.0017 of one
// rounded result: 0.0017 from dS, 0.0013 from P and O in delta.
#pragma once
#include "attn_bwd.hpp"
#include "attn_fwd.hpp"
#include "attn_fwd_keyshare.hpp"

namespace fattn {

template <int D>
__global__ __launch_bounds__(256, 2) void fwd_packed_kernel(const FwdParams p, const PackedArgs a) {
    constexpr int BM = 128;
    PackedUnit u;
    const PackedWork work = packed_unit<BM, false>(a, (int)blockIdx.x, u);
    if (work == kPackedIdle) return;
    if (work == kPackedBehind) {
        packed_zero_rows<BM>(p.o + u.q_at(p.os), p.os.n, u.tile, u.Sq, p.dv);
        const int row = u.tile * BM + (int)threadIdx.x;
        if (p.lse && threadIdx.x < BM && row < u.Sq) p.lse[u.stat_row() + row] = -INFINITY;
        asm volatile("" ::: "memory");        // (else this store and the walk's become one, with what they need kept in scratch memory)
        return;
    }
    fwd_body<D, kExNone, 4, kDropNone, 1, false, false, true>(p, u);
}

// ... the same for few queries: 32 per workgroup, whose wavefronts share the keys
template <int D, int NW>
__global__ __launch_bounds__(64 * NW, D == 64 ? 4 : 2) void fwd_packed_keyshare_kernel(const FwdParams p, const PackedArgs a) {
    constexpr int BM = 32;
    PackedUnit u;
    const PackedWork work = packed_unit<BM, false>(a, (int)blockIdx.x, u);
    if (work == kPackedIdle) return;
    if (work == kPackedBehind) {
        packed_zero_rows<BM>(p.o + u.q_at(p.os), p.os.n, u.tile, u.Sq, p.dv);
        const int row = u.tile * BM + (int)threadIdx.x;
        if (p.lse && threadIdx.x < BM && row < u.Sq) p.lse[u.stat_row() + row] = -INFINITY;
        return;
    }
    FwdParams one = p;                 // the sequence and head as a problem of their own
    one.q += u.q_at(p.qs);
    one.k += u.k_at(p.ks);
    one.v += u.k_at(p.vs);
    one.o += u.q_at(p.os);
    if (p.lse) one.lse += u.stat_row();
    one.B = one.H = one.key_splits = 1;
    one.wg_base = 0;
    one.Sq = u.Sq;
    one.Sk = u.Sk;
    one.m.kv_len = nullptr;
    fwd_keyshare_body<D, NW, kDropNone>(one, u.tile, u.past);
}

template <int D>
__global__ __launch_bounds__(256, 2) void bwd_dq_packed_kernel(const BwdParams p, const PackedArgs a) {
    constexpr int BM = 128;
    PackedUnit u;
    const PackedWork work = packed_unit<BM, false>(a, (int)blockIdx.x, u);
    if (work == kPackedIdle) return;
    if (work == kPackedBehind) {
        packed_zero_rows<BM>(p.dq + u.q_at(p.dqs), p.dqs.n, u.tile, u.Sq, p.d);
        return;
    }
    bwd_dq_body<D, kExNone, 4, kDropNone, 1, false, true>(p, u);
}

template <int D>
__global__ __launch_bounds__(256) void bwd_dkdv_packed_kernel(const BwdParams p, const PackedArgs a) {
    constexpr int BN = BwdTile<D>::BN;
    PackedUnit u;
    const PackedWork work = packed_unit<BN, true>(a, (int)blockIdx.x, u);
    if (work == kPackedIdle) return;
    if (work == kPackedBehind) {
        packed_zero_rows<BN>(p.dk + u.k_at(p.dks), p.dks.n, u.tile, u.Sk, p.d);
        packed_zero_rows<BN>(p.dv + u.k_at(p.dvs), p.dvs.n, u.tile, u.Sk, p.d);
        return;
    }
    bwd_dkdv_body<D, false, false, false, kDropNone, false, false, true>(p, 0, 0, u);
}

// ---- the parts of a walk (PackedCut) are joined: a workgroup per tile and 8 * G columns of d, whose threads mirror the accumulators.
// Bound by latency, so the sums of eight parts are on their way at once (two with G = 4).

// calls add(part, i, four floats of the sums of columns 8 i + ...) for parts 0 .. n - 1; `next` floats from part to part
template <int G, class F>
__device__ __forceinline__ void merge_parts(const float* sums, int64_t next, int n, F&& add) {
    constexpr int AHEAD = 8 / G;
    for (int s0 = 0; s0 < n; s0 += AHEAD) {
        f32x4 v[AHEAD][G];
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
#pragma unroll
            for (int i = 0; i < G; ++i) v[j][i] = *reinterpret_cast<const f32x4*>(sums + min(s0 + j, n - 1) * next + i * 1024);
#pragma unroll
        for (int j = 0; j < AHEAD; ++j)
            if (s0 + j < n)
#pragma unroll
                for (int i = 0; i < G; ++i) add(s0 + j, i, v[j][i]);
    }
}

// O = sum exp2(m - M) O' / sum exp2(m - M) l over the parts, M = max m; LSE = (M + log2 of that sum) ln 2
template <int D, int G>
__global__ __launch_bounds__(256) void fwd_packed_merge_kernel(const FwdParams p, const PackedArgs a) {
    constexpr int BM = 128, BN = 64;
    PackedUnit u;
    if (packed_unit<BM, false, true>(a, (int)blockIdx.x, u) != kPackedTile || u.parts == 1) return;
    const int q0 = u.tile * BM, keys = max(a.causal ? min(u.Sk, q0 + BM + u.past) : u.Sk, 0);
    const int parts = packed_parts(u, (keys + BN - 1) / BN);
    if (parts == 1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5, g = G * (int)blockIdx.y;      // 8 g: the first column
    const f32x2* const ml = reinterpret_cast<const f32x2*>(p.part_lse) + (int64_t)u.unit * BM + 32 * wave + n;
    const int64_t next = a.H;          // parts of a tile are so many units apart
    float M = -INFINITY, L = 0.f;
#pragma unroll 8
    for (int s = 0; s < parts; ++s) M = fmaxf(M, ml[s * next * BM][0]);
    const float M_to = M == -INFINITY ? 0.f : M;
    f32x4 acc[G] = {};
    float w = 0.f;
    merge_parts<G>(p.part_o + (int64_t)u.unit * (BM * D) + (g * 256 + tid) * 4, next * (BM * D), parts, [&](int s, int i, const f32x4& v) {
        if (i == 0) {
            const f32x2 one = ml[s * next * BM];
            w = exp2_fast(one[0] - M_to);
            L = fmaf(w, one[1], L);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[i][e] = fmaf(w, v[e], acc[i][e]);
    });
    const int row = q0 + 32 * wave + n;
    if (row >= u.Sq) return;
    const float inv = L > 0.f ? 1.0f / L : 0.f;
    uint16_t* const out = p.o + u.q_at(p.os) + (int64_t)row * p.os.n + 8 * g + 4 * h;
#pragma unroll
    for (int i = 0; i < G; ++i)
        if (8 * (g + i) + 4 * h < p.dv) *reinterpret_cast<u32x2*>(out + 8 * i) = u32x2{pack_bf16(acc[i][0] * inv, acc[i][1] * inv), pack_bf16(acc[i][2] * inv, acc[i][3] * inv)};
    if (p.lse && g == 0 && h == 0) p.lse[u.stat_row() + row] = L > 0.f ? (M + log2_fast(L)) * kLn2 : -INFINITY;
}

template <int D, int G>
__global__ __launch_bounds__(256) void bwd_dq_packed_merge_kernel(const BwdParams p, const PackedArgs a) {
    constexpr int BM = 128, BN = 64;
    PackedUnit u;
    if (packed_unit<BM, false, true>(a, (int)blockIdx.x, u) != kPackedTile || u.parts == 1) return;
    const int q0 = u.tile * BM, keys = max(a.causal ? min(u.Sk, q0 + BM + u.past) : u.Sk, 0);
    const int parts = packed_parts(u, (keys + BN - 1) / BN);
    if (parts == 1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5, g = G * (int)blockIdx.y;
    f32x4 acc[G] = {};
    merge_parts<G>(p.split_ws + (int64_t)u.unit * (BM * D) + (g * 256 + tid) * 4, (int64_t)a.H * (BM * D), parts, [&](int, int i, const f32x4& v) { acc[i] += v; });
    const int row = q0 + 32 * wave + n;
    if (row >= u.Sq) return;
    uint16_t* const out = p.dq + u.q_at(p.dqs) + (int64_t)row * p.dqs.n + 8 * g + 4 * h;
#pragma unroll
    for (int i = 0; i < G; ++i)
        if (8 * (g + i) + 4 * h < p.d)
            *reinterpret_cast<u32x2*>(out + 8 * i) = u32x2{pack_bf16(acc[i][0] * p.scale, acc[i][1] * p.scale), pack_bf16(acc[i][2] * p.scale, acc[i][3] * p.scale)};
}

template <int D, int G>
__global__ __launch_bounds__(256) void bwd_dkdv_packed_merge_kernel(const BwdParams p, const PackedArgs a) {
    constexpr int BM = BwdTile<D>::BM, BN = BwdTile<D>::BN;
    PackedUnit u;
    if (packed_unit<BN, true, true>(a, (int)blockIdx.x, u) != kPackedTile || u.parts == 1) return;
    const int k0 = u.tile * BN, first = a.causal ? max(k0 - u.past, 0) / BM : 0, all = (u.Sq + BM - 1) / BM;
    if (first >= all) return;          // nothing attends to these keys: written by part 0
    const int parts = packed_parts(u, u.rep * (all - first));
    if (parts == 1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5, g = G * (int)blockIdx.y;
    const float* const sums = p.split_ws + (int64_t)u.unit * (2 * BN * D) + (g * 256 + tid) * 4;
    const int64_t next = (int64_t)a.Hkv * (2 * BN * D);
    f32x4 ak[G] = {}, av[G] = {};
    merge_parts<G>(sums, next, parts, [&](int, int i, const f32x4& v) { ak[i] += v; });
    merge_parts<G>(sums + BN * D, next, parts, [&](int, int i, const f32x4& v) { av[i] += v; });
    const int row = k0 + 32 * wave + n;
    if (row >= u.Sk) return;
    uint16_t* const dk = p.dk + u.k_at(p.dks) + (int64_t)row * p.dks.n + 8 * g + 4 * h;
    uint16_t* const dv = p.dv + u.k_at(p.dvs) + (int64_t)row * p.dvs.n + 8 * g + 4 * h;
#pragma unroll
    for (int i = 0; i < G; ++i) {
        if (8 * (g + i) + 4 * h >= p.d) continue;
        *reinterpret_cast<u32x2*>(dk + 8 * i) = u32x2{pack_bf16(ak[i][0] * p.scale, ak[i][1] * p.scale), pack_bf16(ak[i][2] * p.scale, ak[i][3] * p.scale)};
        *reinterpret_cast<u32x2*>(dv + 8 * i) = u32x2{pack_bf16(av[i][0], av[i][1]), pack_bf16(av[i][2], av[i][3])};
    }
}

}  // namespace fattn
