// The 8-bit activation tape: 32 consecutive values of a tensor (32 channels of one position in NHWC) are kept as one
// byte each and one exponent byte.
//     H    = the smallest power of two that the block's largest magnitude does not exceed by more than H / 256, at
//            least 2^-118
//     code = floor(128 v / H) + 128, held in 0 .. 255,  value = (code - 127.5) H / 128,  exponent byte e = log2(H) + 126
// Why this form:
//   - H is a power of two and a code an odd multiple of H / 256, so every value has 8 significant bits and is exact in
//     bf16: the weight gradient runs on bf16 matrix instructions without another rounding.  A free scale (max / 127)
//     would not gain anything where it matters: the outputs of tanh(v) + v / alpha reach up to 1, where H = 1; the
//     256th above H keeps it there when v / alpha carries a saturated float32 output past 1 (v up to alpha / 256).
//   - the code points lie half a step off zero, symmetrically: every value, the saturated +-1 included, comes back
//     within half a step (H / 256; bf16 itself is H / 512 off in the upper half of the range), one above H within a
//     whole one.  With a code point on zero
//     the 256 codes would reach -1 but only 127 / 128 on the other side, and the derivative 1 - y^2 recovered from the
//     two ends would differ.  The price: a zero in a block that is not all zeros comes back as half a step, and a saturated
//     unit's +-1 as +-255/256, so that no derivative recovered in a block that reaches 1 is under 1 - (255/256)^2 = 0.0078
//     where the unit's own is 1/alpha (0.00005): gradients through saturated units come out too large, by 0.0078 of the
//     arriving gradient.  A float32 layer keeps its derivative itself in this form: 0.0039 there.
//   - e = 0 is a block of zeros, which comes back as zeros; e = 255 a block that held an infinity or a NaN, which comes
//     back as NaN throughout (nothing non-finite is hidden from the gradients).
#pragma once
#include "bf16.h"

// (lane ^ 1) and (lane ^ 2) inside the groups of four lanes that share a block
__device__ __forceinline__ unsigned tape8_quad_max(unsigned m) {
    const unsigned a = (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xf, 0xf, true);   // quad_perm 1,0,3,2
    m = m > a ? m : a;
    const unsigned b = (unsigned)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xf, 0xf, true);   // quad_perm 2,3,0,1
    return m > b ? m : b;
}

// Exponent byte of a block from the float32 bits of its largest magnitude (as an integer the bits of an infinity or
// a NaN are above those of every finite value).
__device__ __forceinline__ unsigned tape8_exponent(unsigned maxbits) {
    unsigned e = (maxbits >> 23) + ((maxbits & 0x7fffffu) > 0x8000u ? 1u : 0u);      // 127 + log2 H (a subnormal maximum: 0 or 1)
    e = e < 9u ? 8u : e - 1u;
    e = maxbits == 0u ? 0u : e;
    return maxbits >= 0x7f800000u ? 255u : e;
}

// 128 / H; 0 for the two special bytes (codes 128, or 0 for the non-finite values themselves)
__device__ __forceinline__ float tape8_inverse(unsigned e) {
    return (e == 0u || e == 255u) ? 0.f : __builtin_bit_cast(float, (260u - e) << 23);
}

// H / 128
__device__ __forceinline__ float tape8_step(unsigned e) {
    const unsigned b = e == 0u ? 0u : (e - 6u) << 23;
    return __builtin_bit_cast(float, e == 255u ? 0x7fc00000u : b);
}

// byte k of `old` becomes the code of v; the product and the sum are exact
template <int K>
__device__ __forceinline__ unsigned tape8_code(float v, float inv, unsigned old) {
    const float f = __builtin_amdgcn_fmed3f(__builtin_floorf(v * inv) + 128.f, 0.f, 255.f);
    return __builtin_amdgcn_cvt_pk_u8_f32(f, K, old);
}

__device__ __forceinline__ unsigned tape8_code4(const float* v, float inv) {
    unsigned c = tape8_code<0>(v[0], inv, 0u);
    c = tape8_code<1>(v[1], inv, c);
    c = tape8_code<2>(v[2], inv, c);
    return tape8_code<3>(v[3], inv, c);
}

// the four values of a dword of codes; off = -127.5 step
__device__ __forceinline__ void tape8_value4(unsigned c, float step, float off, float* v) {
    v[0] = __builtin_fmaf((float)(c & 0xffu), step, off);
    v[1] = __builtin_fmaf((float)((c >> 8) & 0xffu), step, off);
    v[2] = __builtin_fmaf((float)((c >> 16) & 0xffu), step, off);
    v[3] = __builtin_fmaf((float)(c >> 24), step, off);
}

// Two float32 of 8 significant bits as one dword of bf16: the upper halves, nothing to round.
__device__ __forceinline__ unsigned tape8_bf16_pair(float lo, float hi) {
    return __builtin_amdgcn_perm(__builtin_bit_cast(unsigned, hi), __builtin_bit_cast(unsigned, lo), 0x07060302u);
}

// dact_from_y (bf16.h) that lets a NaN through, so that a non-finite block reaches the gradients.
__device__ __forceinline__ float tape8_dact(float y, float inv_alpha, float k1) {
    const float d = __builtin_fmaf(-y, y, k1);
    return d < inv_alpha ? inv_alpha : d;
}
