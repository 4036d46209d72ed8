// Rotary positions: the first R elements of a head are R / 2 pairs, and pair i of a token at position p is turned by the angle p f_i,
//   (a, b) -> size (a cos - b sin, b cos + a sin),
// the elements behind R are copied.  Pairs are neighbours (2 i, 2 i + 1) or halves (i, i + R / 2).  The gradient is the turn by the opposite angle.
//
// The angle: f_i / (2 pi) comes as a 64-bit fraction of a turn, so that p f_i modulo a turn is the low half of an integer product, exact for any
// position (in floating point the turns of a far position take the bits of the fraction).  Its upper 32 bits are reduced to an eighth of a turn
// either way, also exactly, and only then become fp32: sine and cosine are sums of their power series there, off by less than 2e-7.
//
// Bound by memory: every element is read and written once.  A thread serves a chunk of pairs (16 bytes of a head, halves: twice 16) for up to
// HPT heads (rotary_rule.hpp), which share the sines: 30 operations a pair, as much as three heads' loads and stores.  Queries and keys go in one launch.
#pragma once
#include "attn_common.hpp"
#include "packed_units.hpp"

namespace fattn {

struct RotaryParams {
    const void* x[2];              // queries and keys, [B][H][S][D] through xs
    void* y[2];
    Strides xs[2], ys[2];
    int H[2];                      // heads; 0: no keys
    const int64_t* turns;          // [R / 2]: 2^64 f / (2 pi)
    const int32_t* positions;      // [B or 1][S], or null:
    int64_t position_step;         //   from batch to batch
    const int32_t* cu;             // [n + 1]: rows of the sequences (B is 1), whose first positions are
    const int32_t* start;          // [n], or null: 0
    int n;
    int B, S, D, R;
    float size;
    int back;                      // turn by the opposite angle
    int chunks, groups;            // of a head, of the heads
    uint32_t items;
};

// The largest tables of a power series that 2^-29 of a turn needs: |a| <= pi / 4, the first term left out is below 2e-9 (sine) and 2e-10 (cosine).
__device__ __forceinline__ void rotary_sincos(uint32_t phase, float& s, float& c) {
    const uint32_t quarter = (phase + 0x20000000u) >> 30;
    const float a = (float)(int32_t)(phase - (quarter << 30)) * 1.4629180792671596e-9f;       // 2 pi / 2^32
    const float z = a * a;
    const float sn = fmaf(a * z, fmaf(z, fmaf(z, fmaf(z, 2.7557319e-6f, -1.9841270e-4f), 8.3333333e-3f), -1.6666667e-1f), a);
    const float cs = fmaf(z, fmaf(z, fmaf(z, fmaf(z, fmaf(z, -2.7557319e-7f, 2.4801587e-5f), -1.3888889e-3f), 4.1666667e-2f), -0.5f), 1.0f);
    const float u = quarter & 1 ? cs : sn, w = quarter & 1 ? sn : cs;
    s = quarter & 2 ? -u : u;                            // quarters: (sn, cs), (cs, -sn), (-sn, -cs), (-cs, sn)
    c = (quarter + 1) & 2 ? -w : w;
}

// One pair, with the same roundings in every variant, so that the result does not depend on a tensor's layout.
__device__ __forceinline__ void rotary_pair(float a, float b, float c, float s, float& y, float& z) {
    y = fmaf(a, c, -(b * s));
    z = fmaf(b, c, a * s);
}

// 16 bytes, or one number, of an element type
struct RotaryBf16 {
    typedef uint16_t Raw;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float one(uint16_t w) { return bf16_lo(w); }
    static __device__ __forceinline__ uint16_t raw(float v) { return (uint16_t)pack_bf16(v, 0.f); }
    static __device__ __forceinline__ void open(const u32x4& w, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = bf16_lo(w[i]);
            v[2 * i + 1] = bf16_hi(w[i]);
        }
    }
    static __device__ __forceinline__ u32x4 close(const float (&v)[8]) { return u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7])}; }
};
struct RotaryF16 {
    typedef uint16_t Raw;
    static constexpr int VEC = 8;
    static __device__ __forceinline__ float one(uint16_t w) { return (float)__builtin_bit_cast(_Float16, w); }
    static __device__ __forceinline__ uint16_t raw(float v) { return __builtin_bit_cast(uint16_t, (_Float16)v); }
    static __device__ __forceinline__ void open(const u32x4& w, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = one((uint16_t)w[i]);
            v[2 * i + 1] = one((uint16_t)(w[i] >> 16));
        }
    }
    static __device__ __forceinline__ u32x4 close(const float (&v)[8]) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = (uint32_t)raw(v[2 * i]) | (uint32_t)raw(v[2 * i + 1]) << 16;
        return w;
    }
};
struct RotaryF32 {
    typedef float Raw;
    static constexpr int VEC = 4;
    static __device__ __forceinline__ float one(float w) { return w; }
    static __device__ __forceinline__ float raw(float v) { return v; }
    static __device__ __forceinline__ void open(const u32x4& w, float (&v)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const uint32_t bits = w[i];                  // (a bit cast of the vector's element itself takes element 0)
            v[i] = __builtin_bit_cast(float, bits);
        }
    }
    static __device__ __forceinline__ u32x4 close(const float (&v)[4]) {
        u32x4 w;
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = __builtin_bit_cast(uint32_t, v[i]);
        return w;
    }
};

// Chunks of a head: pairs first, then what is copied.  WIDE: 16 bytes each (the halves' pairs: twice 16), else a pair or a number.
template <class T, bool WIDE, bool NEAR>
constexpr int kRotaryPairs = WIDE ? (NEAR ? T::VEC / 2 : T::VEC) : 1;
template <class T, bool WIDE, bool NEAR>
__host__ __device__ inline int rotary_turned_chunks(int R) { return R / 2 / kRotaryPairs<T, WIDE, NEAR>; }
template <class T, bool WIDE, bool NEAR>
__host__ __device__ inline int rotary_chunks(int D, int R) { return rotary_turned_chunks<T, WIDE, NEAR>(R) + (D - R) / (WIDE ? T::VEC : 1); }

template <class T, bool WIDE, bool NEAR, int HPT>
__global__ __launch_bounds__(256) void rotary_kernel(const RotaryParams p) {
    typedef typename T::Raw Raw;
    constexpr int P = kRotaryPairs<T, WIDE, NEAR>, VEC = T::VEC;
    const uint32_t item = blockIdx.x * 256u + threadIdx.x, wave0 = __builtin_amdgcn_readfirstlane(item);
    if (wave0 >= p.items) return;
    const uint32_t per_token = (uint32_t)(p.chunks * p.groups);
    const uint32_t at = min(item, p.items - 1u), token = at / per_token, rest = at - token * per_token;
    const int group = (int)(rest / (uint32_t)p.chunks), chunk = (int)(rest - (uint32_t)group * (uint32_t)p.chunks);
    int b = 0, s = (int)token;
    int32_t pos = 0;
    bool behind = false;
    if (p.cu) {
        const int first = packed_find(p.n, (int)(wave0 / per_token), [&](int i) { return packed_bound(p.cu, i, p.S); });
        int i = first;                                 // (every lane has taken part in the search)
        while (i < p.n && packed_bound(p.cu, i + 1, p.S) <= s) ++i;
        behind = i >= p.n;
        if (!behind) pos = (int32_t)((uint32_t)(p.start ? p.start[i] : 0) + (uint32_t)(s - packed_bound(p.cu, i, p.S)));
    } else {
        b = (int)(token / (uint32_t)p.S);
        s = (int)token - b * p.S;
        pos = p.positions[b * p.position_step + s];
    }
    if (item >= p.items) return;
    const int turned = rotary_turned_chunks<T, WIDE, NEAR>(p.R);
    const bool turns = chunk < turned;
    // first elements of the chunk's two pieces (the second: of the halves only)
    const int e0 = turns ? (NEAR ? 2 * P * chunk : P * chunk) : p.R + (WIDE ? VEC : 1) * (chunk - turned), e1 = p.R / 2 + P * chunk;
    float sn[P], cs[P];
    if (turns) {
#pragma unroll
        for (int i = 0; i < P; ++i) {
            const uint64_t f = (uint64_t)p.turns[P * chunk + i];
            // bits 32 .. 63 of pos f
            const uint32_t u = (uint32_t)pos;
            const uint32_t phase = __umulhi(u, (uint32_t)f) + u * (uint32_t)(f >> 32) - (pos < 0 ? (uint32_t)f : 0u);
            rotary_sincos(phase, sn[i], cs[i]);
            sn[i] *= p.back ? -p.size : p.size;
            cs[i] *= p.size;
        }
    }
    const int heads = p.H[0] + p.H[1];
    const Raw* from[HPT];
    Raw* to[HPT];
    bool there[HPT];
#pragma unroll
    for (int j = 0; j < HPT; ++j) {
        const int hh = group + j * p.groups;             // neighbouring threads: neighbouring heads
        there[j] = hh < heads;
        const int which = there[j] && hh >= p.H[0], h = there[j] ? hh - (which ? p.H[0] : 0) : 0;
        from[j] = static_cast<const Raw*>(which ? p.x[1] : p.x[0]) + b * (which ? p.xs[1].b : p.xs[0].b) + h * (which ? p.xs[1].h : p.xs[0].h) +
                  s * (which ? p.xs[1].n : p.xs[0].n);
        to[j] = static_cast<Raw*>(which ? p.y[1] : p.y[0]) + b * (which ? p.ys[1].b : p.ys[0].b) + h * (which ? p.ys[1].h : p.ys[0].h) +
                s * (which ? p.ys[1].n : p.ys[0].n);
    }
    if constexpr (WIDE) {
        u32x4 w0[HPT], w1[HPT];
#pragma unroll
        for (int j = 0; j < HPT; ++j) {
            w0[j] = w1[j] = u32x4{0u, 0u, 0u, 0u};
            if (there[j] && !behind) {
                w0[j] = *reinterpret_cast<const u32x4*>(from[j] + e0);
                if (!NEAR && turns) w1[j] = *reinterpret_cast<const u32x4*>(from[j] + e1);
            }
        }
#pragma unroll
        for (int j = 0; j < HPT; ++j) {
            if (turns && !behind) {
                float v[VEC], a[VEC], o[VEC], q[VEC];
                T::open(w0[j], v);
                if constexpr (NEAR) {
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        rotary_pair(v[2 * i], v[2 * i + 1], cs[i], sn[i], o[2 * i], o[2 * i + 1]);
                    }
                } else {
                    T::open(w1[j], a);
#pragma unroll
                    for (int i = 0; i < P; ++i) {
                        rotary_pair(v[i], a[i], cs[i], sn[i], o[i], q[i]);
                    }
                    w1[j] = T::close(q);
                }
                w0[j] = T::close(o);
            }
            if (there[j]) {
                *reinterpret_cast<u32x4*>(to[j] + e0) = w0[j];
                if (!NEAR && turns) *reinterpret_cast<u32x4*>(to[j] + e1) = w1[j];
            }
        }
    } else {
        const int second = NEAR ? e0 + 1 : e1;
#pragma unroll
        for (int j = 0; j < HPT; ++j) {
            if (!there[j]) continue;
            if (!turns) {
                to[j][e0] = behind ? T::raw(0.f) : from[j][e0];
                continue;
            }
            float o, q;
            rotary_pair(behind ? 0.f : T::one(from[j][e0]), behind ? 0.f : T::one(from[j][second]), cs[0], sn[0], o, q);
            to[j][e0] = T::raw(behind ? 0.f : o);
            to[j][second] = T::raw(behind ? 0.f : q);
        }
    }
}

}  // namespace fattn
