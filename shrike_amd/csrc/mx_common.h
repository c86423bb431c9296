// Microscaled (MX) blocks: 32 elements along a row share one E8M0 scale byte s, 2^(s - 127), 255 standing for NaN. Elements are E4M3
// (a byte, largest 448) or E2M1 (4 bits, two a byte, the even element in the low half; 0, 0.5, 1, 1.5, 2, 3, 4, 6).
#pragma once

#include "gemv_common.h"

namespace shrike {

constexpr uint32_t kMxBlock = 32;

// 8 bytes from any address (scales lie anywhere)
typedef uint32_t u32x2_by1 __attribute__((ext_vector_type(2), aligned(1)));

template <int FORMAT>
__host__ __device__ constexpr uint32_t mx_code_bytes(uint32_t elements) {
    return FORMAT == SHRIKE_MX_E4M3 ? elements : elements / 2u;
}

// The scale byte of a block whose largest magnitude has the fp32 bits `top`: the largest power of two in it over the format's own
// largest (2^8 of E4M3's 448, 2^2 of E2M1's 6), not below 2^-127. What then lies between the format's largest value and the next
// power of two saturates. An infinity or NaN anywhere makes the block NaN: E2M1 has no code for either.
template <int FORMAT>
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t top) {
    constexpr int kTop = FORMAT == SHRIKE_MX_E4M3 ? 8 : 2;
    return top >= 0x7f800000u ? 255u : uint32_t(max(int(top >> 23) - kTop, 0));
}
// 2^(127 - s), by which a block's values are multiplied: exactly, but for what becomes subnormal and rounds to a zero code anyway. (Not for
// the scale byte of a NaN block, whose codes are zero whatever its values.)
__device__ __forceinline__ float mx_inverse_scale(uint32_t s) { return __uint_as_float((254u - s) << 23); }

// 2^(s - 127)
__device__ __forceinline__ float mx_scale(uint32_t s) {
    return s == 255u ? __uint_as_float(0x7fc00000u) : s == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(s << 23);
}

// Four values, already scaled, to four E4M3 codes: round to nearest even. The conversion overflows to NaN, so it is handed no value past 448.
__device__ __forceinline__ uint32_t mx_e4m3_x4(float a, float b, float c, float d) {
    auto sat = [](float v) { return fminf(fmaxf(v, -448.0f), 448.0f); };
    const int lo = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a), sat(b), 0, false);
    return uint32_t(__builtin_amdgcn_cvt_pk_fp8_f32(sat(c), sat(d), lo, true));
}
// Eight values, already scaled, to eight E2M1 codes: round to nearest even, saturating (the conversion does both).
__device__ __forceinline__ uint32_t mx_e2m1_x8(const float (&v)[8]) {
    uint32_t w = 0;
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[0], v[1], 1.0f, 0);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[2], v[3], 1.0f, 1);
    w = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[4], v[5], 1.0f, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, v[6], v[7], 1.0f, 3);
}

__device__ __forceinline__ uint32_t magnitude_bits(float v) { return __float_as_uint(v) & 0x7fffffffu; }

// A block held by a quad of lanes, eight values each: the block's codes of this lane's values and its scale byte. All four lanes must be
// active. (Magnitudes compare as integers, NaN above infinity.)
template <int FORMAT>
struct MxEighths {
    uint32_t codes[FORMAT == SHRIKE_MX_E4M3 ? 2 : 1];
    uint32_t scale;
};
template <int FORMAT>
__device__ __forceinline__ MxEighths<FORMAT> mx_quantize_quad(const float (&v)[8]) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) top = max(top, magnitude_bits(v[i]));
    top = max(top, dpp_keep_u32<0xB1>(top));  // quad_perm [1,0,3,2]
    top = max(top, dpp_keep_u32<0x4E>(top));  // quad_perm [2,3,0,1]
    MxEighths<FORMAT> out;
    out.scale = mx_scale_byte<FORMAT>(top);
    const float inverse = mx_inverse_scale(out.scale);
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = out.scale == 255u ? 0.0f : __fmul_rn(v[i], inverse);
    if constexpr (FORMAT == SHRIKE_MX_E4M3) {
        out.codes[0] = mx_e4m3_x4(w[0], w[1], w[2], w[3]);
        out.codes[1] = mx_e4m3_x4(w[4], w[5], w[6], w[7]);
    } else {
        out.codes[0] = mx_e2m1_x8(w);
    }
    return out;
}

}  // namespace shrike
