// The joining launch of a key split: a header of its own, for the one source that launches it.
#pragma once
#include "attn_fwd.hpp"

namespace fattn {

// Combines the partial outputs of a key split: LSE = log sum_s exp(LSE_s), O = sum_s exp(LSE_s - LSE) O_s.  A slice whose sum
// was NaN makes O NaN (and LSE -inf, as in a walk over all keys by one workgroup).  One lane per query row and 4 output columns.
static __global__ __launch_bounds__(256) void fwd_merge_kernel(const FwdParams p) {
    const int groups = p.dv >> 2;
    const int64_t rows = (int64_t)p.B * p.H * p.Sq;
    const int64_t idx = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (idx >= rows * groups) return;
    const int64_t row = idx / groups;
    const int g = (int)(idx % groups);
    float m = -INFINITY;
    bool nan = false;                  // fmaxf passes over a NaN
    for (int s = 0; s < p.key_splits; ++s) {
        const float l = p.part_lse[s * rows + row];
        m = fmaxf(m, l);
        nan |= l != l;
    }
    float sum = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    if (m != -INFINITY || nan) {
        for (int s = 0; s < p.key_splits; ++s) {
            const float w = expf(p.part_lse[s * rows + row] - m);
            const f32x4 v = *reinterpret_cast<const f32x4*>(p.part_o + (s * rows + row) * p.dv + 4 * g);
            sum += w;
            acc[0] = fmaf(w, v[0], acc[0]); acc[1] = fmaf(w, v[1], acc[1]);
            acc[2] = fmaf(w, v[2], acc[2]); acc[3] = fmaf(w, v[3], acc[3]);
        }
    }
    const float inv = sum > 0.f ? 1.0f / sum : 0.f;
    const int64_t bh = row / p.Sq, qi = row % p.Sq;
    uint16_t* orow = p.o + (bh / p.H) * p.os.b + (bh % p.H) * p.os.h + qi * p.os.n;
    const u32x2 w = {pack_bf16(acc[0] * inv, acc[1] * inv), pack_bf16(acc[2] * inv, acc[3] * inv)};
    *reinterpret_cast<u32x2*>(orow + 4 * g) = w;
    if (p.lse && g == 0) p.lse[row] = sum > 0.f ? m + logf(sum) : -INFINITY;
}

}  // namespace fattn
