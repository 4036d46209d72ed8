// Attention of packed sequences of different lengths with grouped heads (packed_units.hpp), forward and backward: the loops are those
// of attn_fwd.hpp and attn_bwd.hpp, on one sequence of the packed tensors each.
//
//   forward   O_i = sum_j P_ij v_j,  P_ij = exp(scale q_i k_j - LSE_i),  j < Sk, and j <= i + Sk - Sq under the causal flag
//   backward  dS = P (dO V^T - delta),  dQ = scale dS K,  dK = scale sum over the heads of a key head of dS^T Q,  dV = the same of P^T dO
//
// The sums over the heads that share a key head are one walk of one workgroup: no atomics, no partial gradients per head.
//
// What bounds them is what bounds the dense kernels, at their rates: the matrix instructions and the exponentials between them.  Forward,
// eight prompts of 1 to 4096, 32 heads on 8, D = 128: 292 us, 1.0 PFLOP/s (as much as the dense causal one on 4096); training on six documents of
// 333 to 4608, the same heads: forward 370, dQ 520, dK/dV 680 us.  Small batches: the longest walk, one step of 64 keys after the other at 0.6 to 1 us.
// Roundings to 16 bits, which the matrix instructions' operands take: P before it meets V and dO, dS before it meets K and Q, O as it is saved,
// from which delta is formed; all sums are fp32.  dQ and dK are therefore off by 0.0025 of their root mean square against 0.0017 of one
// rounded result: 0.0017 from dS, 0.0013 from P and O in delta.
#pragma once
#include "attn_bwd.hpp"
#include "attn_fwd.hpp"

namespace fattn {

template <int D>
__global__ __launch_bounds__(256, 2) void fwd_packed_kernel(const FwdParams p, const PackedArgs a) {
    constexpr int BM = 128;
    PackedUnit u;
    const PackedWork work = packed_unit<BM, false, true>(a, (int)blockIdx.x, u);
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

template <int D>
__global__ __launch_bounds__(256, 2) void bwd_dq_packed_kernel(const BwdParams p, const PackedArgs a) {
    constexpr int BM = 128;
    PackedUnit u;
    const PackedWork work = packed_unit<BM, false, true>(a, (int)blockIdx.x, u);
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
    const PackedWork work = packed_unit<BN, true, false>(a, (int)blockIdx.x, u);
    if (work == kPackedIdle) return;
    if (work == kPackedBehind) {
        packed_zero_rows<BN>(p.dk + u.k_at(p.dks), p.dks.n, u.tile, u.Sk, p.d);
        packed_zero_rows<BN>(p.dv + u.k_at(p.dvs), p.dvs.n, u.tile, u.Sk, p.d);
        return;
    }
    bwd_dkdv_body<D, false, false, false, kDropNone, false, false, true>(p, 0, 0, u);
}

// ---- the parts of a walk (PackedCut) are joined: one workgroup per tile and 32-wide block of d, whose threads mirror the accumulators

// O = sum exp2(m - M) O' / sum exp2(m - M) l over the parts, M = max m; LSE = (M + log2 of that sum) ln 2
template <int D>
__global__ __launch_bounds__(256) void fwd_packed_merge_kernel(const FwdParams p, const PackedArgs a) {
    constexpr int BM = 128, BN = 64;
    PackedUnit u;
    if (packed_unit<BM, false, true, true>(a, (int)blockIdx.x, u) != kPackedTile || u.parts == 1) return;
    const int q0 = u.tile * BM, keys = max(a.causal ? min(u.Sk, q0 + BM + u.past) : u.Sk, 0);
    const int parts = packed_parts(u, (keys + BN - 1) / BN);
    if (parts == 1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5, db = (int)blockIdx.y;
    const f32x2* const ml = reinterpret_cast<const f32x2*>(p.part_lse) + (int64_t)u.unit * BM + 32 * wave + n;
    const float* const sums = p.part_o + (int64_t)u.unit * (BM * D) + (db * 4 * 256 + tid) * 4;
    const int64_t next = a.H;          // parts of a tile are so many units apart
    float M = -INFINITY, L = 0.f;
    for (int s = 0; s < parts; ++s) M = fmaxf(M, ml[s * next * BM][0]);
    const float M_to = M == -INFINITY ? 0.f : M;
    f32x4 acc[4] = {};
#pragma unroll 2
    for (int s = 0; s < parts; ++s) {
        const f32x2 one = ml[s * next * BM];
        const float w = exp2_fast(one[0] - M_to);
        L = fmaf(w, one[1], L);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const f32x4 v = *reinterpret_cast<const f32x4*>(sums + s * next * (BM * D) + g * 1024);
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[g][e] = fmaf(w, v[e], acc[g][e]);
        }
    }
    const int row = q0 + 32 * wave + n;
    if (row >= u.Sq) return;
    const float inv = L > 0.f ? 1.0f / L : 0.f;
    uint16_t* const out = p.o + u.q_at(p.os) + (int64_t)row * p.os.n + 32 * db + 4 * h;
#pragma unroll
    for (int g = 0; g < 4; ++g)
        if (32 * db + 8 * g + 4 * h < p.dv) *reinterpret_cast<u32x2*>(out + 8 * g) = u32x2{pack_bf16(acc[g][0] * inv, acc[g][1] * inv), pack_bf16(acc[g][2] * inv, acc[g][3] * inv)};
    if (p.lse && db == 0 && h == 0) p.lse[u.stat_row() + row] = L > 0.f ? (M + log2_fast(L)) * kLn2 : -INFINITY;
}

template <int D>
__global__ __launch_bounds__(256) void bwd_dq_packed_merge_kernel(const BwdParams p, const PackedArgs a) {
    constexpr int BM = 128, BN = 64;
    PackedUnit u;
    if (packed_unit<BM, false, true, true>(a, (int)blockIdx.x, u) != kPackedTile || u.parts == 1) return;
    const int q0 = u.tile * BM, keys = max(a.causal ? min(u.Sk, q0 + BM + u.past) : u.Sk, 0);
    const int parts = packed_parts(u, (keys + BN - 1) / BN);
    if (parts == 1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5, db = (int)blockIdx.y;
    const float* sums = p.split_ws + (int64_t)u.unit * (BM * D) + (db * 4 * 256 + tid) * 4;
    f32x4 acc[4] = {};
#pragma unroll 2
    for (int s = 0; s < parts; ++s, sums += (int64_t)a.H * (BM * D))
#pragma unroll
        for (int g = 0; g < 4; ++g) acc[g] += *reinterpret_cast<const f32x4*>(sums + g * 1024);
    const int row = q0 + 32 * wave + n;
    if (row >= u.Sq) return;
    uint16_t* const out = p.dq + u.q_at(p.dqs) + (int64_t)row * p.dqs.n + 32 * db + 4 * h;
#pragma unroll
    for (int g = 0; g < 4; ++g)
        if (32 * db + 8 * g + 4 * h < p.d) *reinterpret_cast<u32x2*>(out + 8 * g) = u32x2{pack_bf16(acc[g][0] * p.scale, acc[g][1] * p.scale), pack_bf16(acc[g][2] * p.scale, acc[g][3] * p.scale)};
}

template <int D>
__global__ __launch_bounds__(256) void bwd_dkdv_packed_merge_kernel(const BwdParams p, const PackedArgs a) {
    constexpr int BM = BwdTile<D>::BM, BN = BwdTile<D>::BN;
    PackedUnit u;
    if (packed_unit<BN, true, false, true>(a, (int)blockIdx.x, u) != kPackedTile || u.parts == 1) return;
    const int k0 = u.tile * BN, first = a.causal ? max(k0 - u.past, 0) / BM : 0, all = (u.Sq + BM - 1) / BM;
    if (first >= all) return;          // nothing attends to these keys: written by part 0
    const int parts = packed_parts(u, u.rep * (all - first));
    if (parts == 1) return;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, h = lane >> 5, db = (int)blockIdx.y;
    const float* sums = p.split_ws + (int64_t)u.unit * (2 * BN * D) + (db * 4 * 256 + tid) * 4;
    f32x4 ak[4] = {}, av[4] = {};
#pragma unroll 2
    for (int s = 0; s < parts; ++s, sums += (int64_t)a.Hkv * (2 * BN * D))
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            ak[g] += *reinterpret_cast<const f32x4*>(sums + g * 1024);
            av[g] += *reinterpret_cast<const f32x4*>(sums + BN * D + g * 1024);
        }
    const int row = k0 + 32 * wave + n;
    if (row >= u.Sk) return;
    uint16_t* const dk = p.dk + u.k_at(p.dks) + (int64_t)row * p.dks.n + 32 * db + 4 * h;
    uint16_t* const dv = p.dv + u.k_at(p.dvs) + (int64_t)row * p.dvs.n + 32 * db + 4 * h;
#pragma unroll
    for (int g = 0; g < 4; ++g) {
        if (32 * db + 8 * g + 4 * h >= p.d) continue;
        *reinterpret_cast<u32x2*>(dk + 8 * g) = u32x2{pack_bf16(ak[g][0] * p.scale, ak[g][1] * p.scale), pack_bf16(ak[g][2] * p.scale, ak[g][3] * p.scale)};
        *reinterpret_cast<u32x2*>(dv + 8 * g) = u32x2{pack_bf16(av[g][0], av[g][1]), pack_bf16(av[g][2], av[g][3])};
    }
}

}  // namespace fattn
