// Entry point of the rotary positions (rotary.hpp).
#include <climits>
#include <cmath>

#include "rotary.hpp"
#include "rotary_rule.hpp"
#include "view_checks.hpp"
#include "../../include/flame_attn.h"

using namespace fattn;

namespace {

template <class T, bool WIDE, bool NEAR>
int launch(RotaryParams p, hipStream_t s) {
    p.chunks = rotary_chunks<T, WIDE, NEAR>(p.D, p.R);
    const int heads = p.H[0] + p.H[1];
    const double all = (double)p.B * p.S * p.chunks;
    const double most = (double)(UINT32_MAX - 256);    // threads of a launch
    const int per_thread = all * heads > most ? 4 : rotary_heads_per_thread(all * heads, WIDE, NEAR, sizeof(typename T::Raw) == 4, p.cu != nullptr);
    p.groups = (heads + per_thread - 1) / per_thread;
    if (all * p.groups > most) return FLAME_ATTN_ERR_UNSUPPORTED;
    p.items = (uint32_t)p.B * (uint32_t)p.S * (uint32_t)p.chunks * (uint32_t)p.groups;
    const unsigned grid = (p.items + 255u) / 256u;
    if (per_thread == 4) hipLaunchKernelGGL((rotary_kernel<T, WIDE, NEAR, 4>), dim3(grid), dim3(256), 0, s, p);
    else hipLaunchKernelGGL((rotary_kernel<T, WIDE, NEAR, 1>), dim3(grid), dim3(256), 0, s, p);
    return (int)hipGetLastError();
}
template <class T>
int launch(const RotaryParams& p, bool near, hipStream_t s) {
    bool wide = p.D % T::VEC == 0 && (near ? p.R : p.R / 2) % T::VEC == 0;
    for (int w = 0; w < (p.H[1] ? 2 : 1); ++w)
        for (const Strides* st : {&p.xs[w], &p.ys[w]}) wide = wide && (st->b | st->h | st->n) % T::VEC == 0;
    for (int w = 0; w < 2; ++w) wide = wide && ((reinterpret_cast<uintptr_t>(p.x[w]) | reinterpret_cast<uintptr_t>(p.y[w])) & 15u) == 0;
    if (near) return wide ? launch<T, true, true>(p, s) : launch<T, false, true>(p, s);
    return wide ? launch<T, true, false>(p, s) : launch<T, false, false>(p, s);
}

}  // namespace

extern "C" int flame_rotary(const void* Q, void* Q_out, int H, const int64_t* q_strides, const int64_t* qo_strides, const void* K, void* K_out, int H_kv,
                            const int64_t* k_strides, const int64_t* ko_strides, int dtype, const int64_t* turns, int rotary_dim, int interleaved,
                            float size, int inverse, const int32_t* positions, int64_t position_stride, const int32_t* cu, const int32_t* start, int n_seqs,
                            int B, int S, int D, void* stream) {
    if (!Q || !Q_out || H <= 0 || !q_strides || !qo_strides || H_kv < 0 || !turns || B <= 0 || S <= 0 || D <= 0 || rotary_dim <= 0 || !std::isfinite(size))
        return FLAME_ATTN_ERR_INVALID;
    if ((H_kv > 0) != (K != nullptr) || (K != nullptr) != (K_out != nullptr) || (H_kv > 0 && (!k_strides || !ko_strides))) return FLAME_ATTN_ERR_INVALID;
    if ((positions != nullptr) == (cu != nullptr) || (cu && (n_seqs <= 0 || B != 1)) || (start && !cu) || (positions && position_stride < 0)) return FLAME_ATTN_ERR_INVALID;
    if (rotary_dim % 2 != 0 || rotary_dim > D || (int64_t)H + H_kv > INT32_MAX / 2 || (int64_t)B * S > INT32_MAX) return FLAME_ATTN_ERR_UNSUPPORTED;
    if (dtype != FLAME_ATTN_DTYPE_BF16 && dtype != FLAME_ATTN_DTYPE_F16 && dtype != FLAME_ATTN_DTYPE_F32) return FLAME_ATTN_ERR_UNSUPPORTED;
    RotaryParams p{};
    const void* const x[2] = {Q, K};
    void* const y[2] = {Q_out, K_out};
    const int64_t* const xs[2] = {q_strides, k_strides};
    const int64_t* const ys[2] = {qo_strides, ko_strides};
    const int heads[2] = {H, H_kv}, unit = dtype == FLAME_ATTN_DTYPE_F32 ? 4 : 2;
    for (int w = 0; w < (H_kv ? 2 : 1); ++w) {
        if (xs[w][3] != 1 || ys[w][3] != 1 || (reinterpret_cast<uintptr_t>(x[w]) | reinterpret_cast<uintptr_t>(y[w])) % unit) return FLAME_ATTN_ERR_UNSUPPORTED;
        for (int i = 0; i < 3; ++i)
            if (xs[w][i] < 0 || ys[w][i] < 0) return FLAME_ATTN_ERR_UNSUPPORTED;
        const int64_t out[4] = {B, heads[w], S, D};
        if (overlaps(ys[w], out, 4)) return FLAME_ATTN_ERR_UNSUPPORTED;
        p.x[w] = x[w];
        p.y[w] = y[w];
        auto of = [&](const int64_t* st) { return Strides{B > 1 ? st[0] : 0, heads[w] > 1 ? st[1] : 0, S > 1 ? st[2] : 0}; };      // (axes of one element: no matter)
        p.xs[w] = of(xs[w]);
        p.ys[w] = of(ys[w]);
        p.H[w] = heads[w];
    }
    if (Q_out == K_out) return FLAME_ATTN_ERR_INVALID;
    p.turns = turns;
    p.positions = positions;
    p.position_step = position_stride;
    p.cu = cu;
    p.start = start;
    p.n = n_seqs;
    p.B = B;
    p.S = S;
    p.D = D;
    p.R = rotary_dim;
    p.size = size;
    p.back = inverse != 0;
    hipStream_t s = static_cast<hipStream_t>(stream);
    return dtype == FLAME_ATTN_DTYPE_BF16 ? launch<RotaryBf16>(p, interleaved != 0, s)
           : dtype == FLAME_ATTN_DTYPE_F16 ? launch<RotaryF16>(p, interleaved != 0, s) : launch<RotaryF32>(p, interleaved != 0, s);
}
