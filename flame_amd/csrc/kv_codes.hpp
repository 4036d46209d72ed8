// Numbers of a cache held in 8 bits: a code stands for code * scale, the scale that of its block of tokens and its head.
//   kI8:   whole numbers from -127 to 127
//   kE4m3: four bits of exponent, three of mantissa, largest 448, no infinities; 0x7f and 0xff are NaN
// Either is exact in bf16, so the products of the attention see the codes themselves and the scales join in fp32.
#pragma once
#include "attn_common.hpp"

namespace fattn {

enum KvCode : int { kI8 = 0, kE4m3 = 1 };

template <int CODE>
constexpr float kLargestCode = CODE == kI8 ? 127.f : 448.f;
// Of every scale the least: a block of zeros has it.  Its reciprocal and the codes' remainders are ordinary fp32 numbers.
constexpr float kLeastScale = 7.888609052210118e-31f;       // 2^-100

// four codes to fp32
template <int CODE>
__device__ __forceinline__ f32x4 codes_to_f32(uint32_t w) {
    if constexpr (CODE == kI8) {
        return f32x4{(float)(int8_t)w, (float)(int8_t)(w >> 8), (float)(int8_t)(w >> 16), (float)((int32_t)w >> 24)};
    } else {
        const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
        return f32x4{lo[0], lo[1], hi[0], hi[1]};
    }
}
// four numbers no larger than the largest code (or NaN: any code) to the nearest codes, the even one of two
template <int CODE>
__device__ __forceinline__ uint32_t f32_to_codes(float a, float b, float c, float d) {
    if constexpr (CODE == kI8) {
        // of a sum with 3 2^22 the last place is 1: the addition rounds, and the low byte is the code
        const uint32_t i = __builtin_bit_cast(uint32_t, a + 12582912.f), j = __builtin_bit_cast(uint32_t, b + 12582912.f);
        const uint32_t k = __builtin_bit_cast(uint32_t, c + 12582912.f), l = __builtin_bit_cast(uint32_t, d + 12582912.f);
        return __builtin_amdgcn_perm(__builtin_amdgcn_perm(l, k, 0x0c0c0400u), __builtin_amdgcn_perm(j, i, 0x0c0c0400u), 0x05040100u);
    } else {
        const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, lo, true);
    }
}
// Eight codes to bf16, exactly: a matrix operand.  Whole numbers go through fp32, of which the upper half is the bf16 number (three
// operations for two); e4m3 has an instruction for two.
template <int CODE>
__device__ __forceinline__ bf16x8 codes_to_bf16(uint32_t lo, uint32_t hi) {
    u32x4 r;
    const uint32_t w[2] = {lo, hi};
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        if constexpr (CODE == kI8) {
            const u32x4 f = __builtin_bit_cast(u32x4, codes_to_f32<kI8>(w[i]));
            r[2 * i] = __builtin_amdgcn_perm(f[1], f[0], 0x07060302u);
            r[2 * i + 1] = __builtin_amdgcn_perm(f[3], f[2], 0x07060302u);
        } else {
            r[2 * i] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], 1.0f, false));
            r[2 * i + 1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w[i], 1.0f, true));
        }
    }
    return __builtin_bit_cast(bf16x8, r);
}

}  // namespace fattn
