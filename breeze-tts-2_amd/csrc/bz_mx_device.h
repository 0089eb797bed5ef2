// Microscaled (MX) blocks on gfx950: layouts and conversions shared by the
// kernels over them.
//
// A block is 32 consecutive k of a row: elements q of a narrow floating-point
// type and one scale 2^(code - 127), code 0..254; code 255 marks a block that
// holds a NaN or an infinity and reads as NaN.
//   e2m1  4 bits: 0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives;
//   e4m3  8 bits: OCP FP8, largest 448.
// Scale of a block with largest magnitude a: 2^(floor(log2 a) - emax), emax 2
// or 8, so a / scale lies in [2^emax, 2^(emax + 1)) and only values above the
// type's largest saturate; not below 2^-126, so that code << 23 is the scale
// as a normal float.
//
// Tiled rows (weights and, inside a call, activations): a row block is 16
// rows; a unit is 128 k of them, four blocks per row.  Per row block the NU
// unit tiles lie one after the other, then the scales.
//   e2m1 tile, 1 KiB: lane l = 16 g + r holds block g of row r at byte 16 l,
//     which is the operand placement of v_mfma_scale_f32_16x16x128_f8f6f4
//     for 4-bit types: one load per lane is one operand.
//   e4m3 tile, 2 KiB: the same instruction takes 8-bit k = 16 g .. 16 g + 15
//     and 64 + 16 g .. 64 + 16 g + 15 in lane row g, so bytes [16 l, +16) hold
//     the former and 1024 + [16 l, +16) the latter.
//   scales: per four units 256 bytes, byte u % 4 of dword l the code of block
//     g of row r in unit u.  The instruction takes the scale of block g from
//     lane row g for either type and picks the byte itself (its operand
//     selector), so one dword serves four units.
#pragma once

#include "bz_device.h"

namespace bz {

__host__ __device__ constexpr int64_t mx_scale_bytes(int NU) { return (int64_t)((NU + 3) >> 2) * 256; }
__host__ __device__ constexpr int64_t mx4_chunk_bytes(int NU) { return (int64_t)NU * 1024 + mx_scale_bytes(NU); }
__host__ __device__ constexpr int64_t mx8_chunk_bytes(int NU) { return (int64_t)NU * 2048 + mx_scale_bytes(NU); }
// from the start of the row block's scales; unit u is byte u % 4 of it
__host__ __device__ constexpr uint32_t mx_scale_offset(int u, int lane) {
    return (uint32_t)(u >> 2) * 256u + (uint32_t)lane * 4u;
}

// Unit u's scale as a float from its dword of codes.
__device__ __forceinline__ float mx_scale(uint32_t codes, int u) {
    return __uint_as_float(((codes >> (8 * (u & 3))) & 0xFFu) << 23);
}

// Eight e2m1 elements times their scale as bf16 pairs in natural order
// (exact; the conversion reads the scale's exponent field, 0 as 2^-127 and
// 255 as NaN).
__device__ __forceinline__ u32x4 mx4_weights(uint32_t v, float s) {
    return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, s, 0)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, s, 1)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, s, 2)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(v, s, 3))};
}

// Scale code of a block from the fp32 exponent field of its largest
// magnitude (255: a NaN or an infinity is among them).
template <int EMAX>
__device__ __forceinline__ uint32_t mx_code(uint32_t exponent) {
    return exponent == 255u ? 255u : (uint32_t)max((int)exponent - EMAX, 1);
}

// Eight values -> eight e2m1 elements (one dword), round to nearest even,
// magnitudes above 6 to 6: the hardware's scaled conversion.
__device__ __forceinline__ uint32_t mx4_pack_bf16(u32x4 v, float s) {
    auto p = [&](int i) { return as_bf16x2(v[i]); };
    uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(0u, p(0), s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, p(1), s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, p(2), s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, p(3), s, 3);
}
__device__ __forceinline__ uint32_t mx4_pack_f32(const float (&v)[8], float s) {
    uint32_t r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, v[0], v[1], s, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[2], v[3], s, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[4], v[5], s, 2);
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, v[6], v[7], s, 3);
}

// Four values -> four e4m3 elements.  The conversion turns magnitudes past
// 448 into NaN, so they are clamped first.
__device__ __forceinline__ uint32_t mx8_pack_f32(float a, float b, float c, float d, float s) {
    typedef short short2_t __attribute__((ext_vector_type(2)));
    const float top = 448.0f * s;
    auto clamp = [&](float v) { return __builtin_amdgcn_fmed3f(v, -top, top); };
    short2_t r = {0, 0};
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, clamp(a), clamp(b), s, false);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(r, clamp(c), clamp(d), s, true);
    return __builtin_bit_cast(uint32_t, r);
}

// The same of eight bf16 values (two dwords) without widening them: 448 times
// a scale code's power of two is a bf16, and magnitudes compare as integers.
typedef unsigned short us2_t __attribute__((ext_vector_type(2)));
__device__ __forceinline__ void mx8_pack_bf16(u32x4 v, uint32_t code, float s, uint32_t& lo, uint32_t& hi) {
    typedef short short2_t __attribute__((ext_vector_type(2)));
    const unsigned short t = (unsigned short)((code + 8u) << 7 | 0x60u);
    const us2_t top = {t, t};
    auto clamp = [&](uint32_t x) {
        const uint32_t m = __builtin_bit_cast(uint32_t, __builtin_elementwise_min(__builtin_bit_cast(us2_t, x & 0x7FFF7FFFu), top));
        return as_bf16x2(m | (x & 0x80008000u));
    };
    short2_t a = {0, 0}, b = {0, 0};
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, clamp(v[0]), s, false);
    a = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(a, clamp(v[1]), s, true);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(b, clamp(v[2]), s, false);
    b = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(b, clamp(v[3]), s, true);
    lo = __builtin_bit_cast(uint32_t, a);
    hi = __builtin_bit_cast(uint32_t, b);
}

}  // namespace bz
