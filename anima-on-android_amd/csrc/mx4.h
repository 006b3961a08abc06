// 4-bit rows in the OCP microscaling format (MX4): every 32 consecutive
// elements of a row share one scale byte s, an e8m0 number 2^(s - 127) with
// 255 for NaN; an element is an e2m1 code, sign in bit 3 and magnitude 0, 0.5,
// 1, 1.5, 2, 3, 4 or 6 in bits 0 to 2.  Byte i of a row's codes holds element
// 2i in its low half and element 2i + 1 in its high half; a row of K elements
// takes ceil(K / 32) * 16 bytes of codes, zero past K, and ceil(K / 32) scale
// bytes.
//
// A code times its scale has at most two significant bits, so every MX4 value
// is a bf16 number and a product of decoded values on the bf16 MFMA carries no
// rounding of the weights.  gfx950 decodes two codes per instruction, scale
// included (v_cvt_scalef32_pk_bf16_fp4; measured over all scale bytes: 255
// gives NaN, values past the bf16 range give infinity, subnormals are kept).
#pragma once

#include "flash_tile.h"

namespace anima_hip {
namespace mx4 {

using flash_tile::bf16x2;
using flash_tile::bf16x8;
using flash_tile::f32x2;
using flash_tile::f32x4;
using flash_tile::u32x4;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));

constexpr int kGroup = 32;     // elements per scale
constexpr int kNanScale = 255;  // scale byte of a group that held an infinity or a NaN
// Scale bytes the packer writes: 2^-125 keeps every magnitude a normal bf16
// number (0.5 * 2^-125), 2^125 keeps 6 finite (6 * 2^125 < 2^128).
constexpr int kMinScale = 2, kMaxScale = 252;

// The scale as the conversions take it: only the exponent field counts.
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// Codes 2 BYTE and 2 BYTE + 1 of a word as bf16 values.
template <int BYTE>
__device__ __forceinline__ unsigned decode2(unsigned word, float scale)
{
    const bf16x2 v = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, BYTE);
    return __builtin_bit_cast(unsigned, v);
}

// The same with the byte as an argument that folds to a constant.
__device__ __forceinline__ unsigned decode2_at(unsigned word, float scale, int byte)
{
    return byte == 0   ? decode2<0>(word, scale)
           : byte == 1 ? decode2<1>(word, scale)
           : byte == 2 ? decode2<2>(word, scale)
                       : decode2<3>(word, scale);
}

// The eight codes of a word as one bf16 MFMA operand.
__device__ __forceinline__ bf16x8 decode8(unsigned word, float scale)
{
    const u32x4 r = {decode2<0>(word, scale), decode2<1>(word, scale), decode2<2>(word, scale),
                     decode2<3>(word, scale)};
    return __builtin_bit_cast(bf16x8, r);
}

// Eight f32 values as codes.
__device__ __forceinline__ unsigned encode8(const float (&x)[8], float scale)
{
    unsigned r = 0;
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[0], x[1], scale, 0);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[2], x[3], scale, 1);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[4], x[5], scale, 2);
    r = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(r, x[6], x[7], scale, 3);
    return r;
}

// Scale byte of a group whose largest |x| has the bits `top` (as unsigned
// integers, magnitudes order like the numbers, NaN above infinity): with
// 2^E <= top < 2^(E+1) the largest code stands for 6 * 2^(E - 2), so values up
// to 1.75 * 2^E round to it with at most 2^(E-2), the largest rounding step below
// it; past that the next scale is nearer.
__device__ __forceinline__ int scale_byte(unsigned top)
{
    if (top >= 0x7F800000u)
        return kNanScale;
    const int e = int(top >> 23) - 2 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return min(max(e, kMinScale), kMaxScale);
}

// x as `N` bf16 terms whose sum is x exactly (three terms: 3 x 8 bits; below 2^-110,
// where the last bits lie under bf16's smallest number 2^-133, x cut off to a
// multiple of it): each term is the leading eight bits of what is left, by
// truncation.  An infinity is its own first term, with no NaN behind it (INF:
// there may be one).  Terms are packed in pairs.
template <int N, bool INF = true>
__device__ __forceinline__ void terms2(float x0, float x1, unsigned (&t)[N])
{
#pragma unroll
    for (int i = 0; i < N; ++i) {
        const unsigned u0 = __float_as_uint(x0), u1 = __float_as_uint(x1);
        t[i] = __builtin_amdgcn_perm(u1, u0, 0x07060302);
        if (i + 1 < N) {
            const float h0 = __uint_as_float(u0 & 0xFFFF0000u);
            const float h1 = __uint_as_float(u1 & 0xFFFF0000u);
            // What is left of an infinity is none.
            x0 = INF && i == 0 && x0 == h0 ? 0.0f : x0 - h0;
            x1 = INF && i == 0 && x1 == h1 ? 0.0f : x1 - h1;
        }
    }
}

__device__ __forceinline__ f32x4 mfma16(bf16x8 a, bf16x8 b, f32x4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

}  // namespace mx4
}  // namespace anima_hip
