// Device functions of the wire quantizer (Q0) that more than one kernel uses: the scale rule, the E4M3 codes and the
// maximum over a block's lanes; and the BF16 rounding.
//
// Reference counterparts: crates/mimo26-coordinator/kernels/glue.cu:126-143 (quant_scales_kernel) and
// crates/mimo26-attn/kernels/include/mimo26_attn_device.cuh:33-55 (e4m3_encode).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace m26g {

// s = 0 for an all-zero block, else the smallest e with amax <= 448 * 2^e, plus 127, clamped to
// [0, 254]: with amax = m * 2^x, m in [0.5, 1), that is x - 9 for m <= 0.875 and x - 8 above
// (448 = 0.875 * 2^9). NaNs do not take part in amax; an infinite amax gives 254.
__device__ __forceinline__ uint32_t q0_scale_byte(float amax) {
    if (!(amax > 0.0f)) return 0;
    if (amax > 3.402823466e38f) return 254;
    int x;
    const float m = frexpf(amax, &x);  // exact, subnormals included
    int s = (m <= 0.875f ? x - 9 : x - 8) + 127;
    s = s < 0 ? 0 : s;
    return uint32_t(s > 254 ? 254 : s);
}

// E4M3FN code nearest to y = x * scale (scale a positive power of two), ties to the larger magnitude,
// saturating at 448, NaN -> 0. The sign bit is "the exact product is below zero", i.e. x < 0: -0.0
// gives 0x00 while a negative value that rounds to zero keeps 0x80, also where the binary32 product
// has already underflowed to -0 (the CPU rule multiplies in binary64). Integer arithmetic on the bit
// pattern: from 2^-6 up a code is the binary32 exponent and top three mantissa bits rebased, so
// round-half-up is one add and one shift and a mantissa that rounds over carries into the exponent by
// itself (448, the clamp, is code 0x7e exactly, so nothing larger can come out); below 2^-6 the
// quantum is 2^-9 whatever the exponent, and the significand is shifted down to it.
constexpr uint32_t kE4m3NormalFrom = 121u << 23;  // binary32 bits of 2^-6
__device__ __forceinline__ uint32_t e4m3_magnitude_bits(float y) { return __float_as_uint(fminf(fabsf(y), 448.0f)); }  // a NaN leaves as 448
__device__ __forceinline__ uint32_t e4m3_code_normal(uint32_t bits) { return ((bits + 0x80000u) >> 20) - ((127u - 7u) << 3); }
__device__ __forceinline__ uint32_t e4m3_code_small(uint32_t bits) {  // code = floor(value * 512 + 1/2)
    const uint32_t sig = (bits & 0x7fffffu) | 0x800000u, sh = 141u - (bits >> 23);  // value = sig * 2^(field - 150); sh >= 21
    return sh > 31u ? 0u : (sig + (1u << (sh - 1u))) >> sh;  // under 2^-11 (zero and binary32 subnormals too): nothing
}
__device__ __forceinline__ uint32_t e4m3_signed(float x, float y, uint32_t code) {
    return y != y ? 0u : (x < 0.0f ? 0x80u : 0u) | code;
}
__device__ __forceinline__ uint32_t e4m3_half_up(float x, float scale) {
    const float y = x * scale;
    const uint32_t bits = e4m3_magnitude_bits(y);
    return e4m3_signed(x, y, bits < kE4m3NormalFrom ? e4m3_code_small(bits) : e4m3_code_normal(bits));
}
// Four at once, packed low address first: the rule above, value by value.
__device__ __forceinline__ uint32_t e4m3_half_up4_any(const float4 v, float scale) {
    return e4m3_half_up(v.x, scale) | e4m3_half_up(v.y, scale) << 8 | e4m3_half_up(v.z, scale) << 16 | e4m3_half_up(v.w, scale) << 24;
}
// The same four codes in about a third of the instructions when the scale is positive and every scaled value is
// a number of at least 2^-6 in magnitude (a block's amax lands in (224, 448], so smaller ones are rare), which
// these kernels need: a wave64 vector instruction occupies its SIMD for four cycles, and at 16 bytes in per lane
// the budget for keeping up with HBM is about 85 of them per kilobyte. What is different: the sign bit is read
// off fma(x, scale, +0), which is x * scale except that -0 * scale + 0 is +0 (the rule's "x < 0") while a
// negative product that underflows still rounds to -0; the clamp is an integer minimum on the magnitude bits
// (an infinity saturates like any large value); and the rebasing constant rides in the rounding add.
__device__ __forceinline__ uint32_t e4m3_half_up4(const float4 v, float scale) {
    const float x[4] = {v.x, v.y, v.z, v.w};
    uint32_t bits[4], mag[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        bits[j] = __float_as_uint(__builtin_fmaf(x[j], scale, 0.0f));
        mag[j] = bits[j] & 0x7fffffffu;
    }
    auto lesser = [](uint32_t a, uint32_t b) { return a < b ? a : b; };
    auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    const uint32_t least = lesser(lesser(mag[0], mag[1]), lesser(mag[2], mag[3])), most = larger(larger(mag[0], mag[1]), larger(mag[2], mag[3]));
    if (least < kE4m3NormalFrom || most > 0x7f800000u || !(scale > 0.0f)) return e4m3_half_up4_any(v, scale);
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t code = (lesser(mag[j], 0x43e00000u /* 448 */) + (0x80000u - ((127u - 7u) << 23))) >> 20;
        word |= (((bits[j] >> 24) & 0x80u) | code) << (8 * j);
    }
    return word;
}

// Maximum over the eight lanes of a K32 block without leaving the vector unit: neighbours within a quad
// (lanes ^ 1, ^ 2), then the mirrored half-row, which pairs each quad with the other one of its eight.
constexpr int kQuadXor1 = 0xB1, kQuadXor2 = 0x4E, kHalfRowMirror = 0x141;  // DPP controls: quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror
__device__ __forceinline__ float max_over_eight(float v) {
    int b = __float_as_int(v);
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(b, b, kQuadXor1, 0xf, 0xf, false)));
    b = __float_as_int(v);
    v = fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(b, b, kQuadXor2, 0xf, 0xf, false)));
    b = __float_as_int(v);
    return fmaxf(v, __int_as_float(__builtin_amdgcn_update_dpp(b, b, kHalfRowMirror, 0xf, 0xf, false)));
}
__device__ __forceinline__ uint32_t max_bits_over_eight(uint32_t v) {
    auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = larger(v, uint32_t(__builtin_amdgcn_update_dpp(int(v), int(v), kQuadXor1, 0xf, 0xf, false)));
    v = larger(v, uint32_t(__builtin_amdgcn_update_dpp(int(v), int(v), kQuadXor2, 0xf, 0xf, false)));
    return larger(v, uint32_t(__builtin_amdgcn_update_dpp(int(v), int(v), kHalfRowMirror, 0xf, 0xf, false)));
}
// The same over a quad of lanes, for rows held eight values to a lane.
__device__ __forceinline__ uint32_t max_bits_over_four(uint32_t v) {
    auto larger = [](uint32_t a, uint32_t b) { return a > b ? a : b; };
    v = larger(v, uint32_t(__builtin_amdgcn_update_dpp(int(v), int(v), kQuadXor1, 0xf, 0xf, false)));
    return larger(v, uint32_t(__builtin_amdgcn_update_dpp(int(v), int(v), kQuadXor2, 0xf, 0xf, false)));
}

// FP32 -> BF16, nearest even; a NaN becomes 0x7fff, as the reference's conversion intrinsic gives.
__device__ __forceinline__ uint32_t bf16_rne_nan(float f) {
    const uint32_t b = __float_as_uint(f);
    return (b & 0x7fffffffu) > 0x7f800000u ? 0x7fffu : (b + 0x7fffu + ((b >> 16) & 1u)) >> 16;
}

}  // namespace m26g
