// 8-bit rows (FP8): every 128 consecutive elements of a row share one scale
// byte s, an e8m0 number 2^(s - 127) with 255 for NaN; an element is an e4m3
// code (OCP: sign, four bits of exponent with bias 7, three of mantissa; no
// infinity, largest 448).  A row of K elements takes ceil(K / 128) * 128 bytes
// of codes, zero past K, and ceil(K / 512) * 4 scale bytes, zero past its
// groups, so that a dword holds four groups' scales at any row.
//
// The scale is the smallest power of two by which the group's largest magnitude
// is at most 448, so that an element is scaled exactly and rounded once.  A
// power of two rather than the quotient by 448: the MFMA takes e8m0 scales by
// itself, and what a scale between two powers of two would gain is none of an
// element's four significant bits, only half a power of two of range.
#pragma once

#include "flash_tile.h"

namespace anima_hip {
namespace fp8 {

using flash_tile::bf16x2;
using flash_tile::bf16x8;
using flash_tile::f32x2;
using flash_tile::f32x4;
using flash_tile::u32x4;
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef int i32x8 __attribute__((ext_vector_type(8)));
// Vectors at any element: the hardware takes vector accesses that are not aligned.
typedef f32x4 any_f32x4 __attribute__((aligned(4)));
typedef u32x4 any_u32x4 __attribute__((aligned(2)));
typedef u32x2 any_u32x2 __attribute__((aligned(2)));

constexpr int kGroup = 128;     // elements per scale
constexpr int kNanScale = 255;  // scale byte of a group that held an infinity or a NaN
// Scale bytes the packer writes: 2^-117 keeps the smallest element, 2^-9, a normal
// bf16 number, 2^119 keeps the largest, 448, finite (1.75 * 2^127).
constexpr int kMinScale = 10, kMaxScale = 246;

// Scale byte of a group whose largest |x| has the bits `top` (as unsigned
// integers, magnitudes order like the numbers, NaN above infinity).
__device__ __forceinline__ int scale_byte(unsigned top)
{
    if (top >= 0x7F800000u)
        return kNanScale;
    const int e = int(top >> 23) - 8 + ((top & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    return min(max(e, kMinScale), kMaxScale);
}

// 2^(127 - byte) for a byte the packer writes: what elements are multiplied by.
__device__ __forceinline__ float unscale_of(int byte) { return __uint_as_float((254u - byte) << 23); }

// The scale as the conversions take it: only the exponent field counts.
__device__ __forceinline__ float scale_of(unsigned byte) { return __uint_as_float(byte << 23); }

// Four values over their scale as codes, round to nearest even.  Only groups at
// the largest scale reach past 448; there elements saturate.
__device__ __forceinline__ unsigned encode4(float x0, float x1, float x2, float x3, float unscale)
{
    const auto in = [&](float x) { return __builtin_amdgcn_fmed3f(x * unscale, -448.0f, 448.0f); };
    int r = 0;
    r = __builtin_amdgcn_cvt_pk_fp8_f32(in(x0), in(x1), r, false);
    r = __builtin_amdgcn_cvt_pk_fp8_f32(in(x2), in(x3), r, true);
    return unsigned(r);
}

// Largest of v over the 16 lanes of a DPP row, in all of them.
__device__ __forceinline__ unsigned row16_max(unsigned v)
{
    v = max(v, unsigned(__builtin_amdgcn_update_dpp(0, int(v), 0x128, 0xF, 0xF, false)));  // row_ror:8
    v = max(v, unsigned(__builtin_amdgcn_update_dpp(0, int(v), 0x124, 0xF, 0xF, false)));
    v = max(v, unsigned(__builtin_amdgcn_update_dpp(0, int(v), 0x122, 0xF, 0xF, false)));
    v = max(v, unsigned(__builtin_amdgcn_update_dpp(0, int(v), 0x121, 0xF, 0xF, false)));
    return v;
}

// The eight elements of a group that one of 16 lanes has: two runs of four, kSecond apart.
// Rows in bf16: one 16-byte access; in f32: 64, so that each of a lane's two accesses
// follows its neighbour's.
template <typename T>
constexpr int kSecond = sizeof(T) == 4 ? 64 : 4;
// Where the first run of piece `piece` of a row begins, 16 pieces a group.
template <typename T>
__device__ __forceinline__ int run_of(int piece)
{
    return sizeof(T) == 4 ? (piece >> 4) * kGroup + (piece & 15) * 4 : 8 * piece;
}

// One group over the 16 lanes of a DPP row, eight elements each, group g of `groups`
// of its row.  All 16 lanes come here together.  Groups with an infinity or a NaN
// have zero codes, so that packing is a function of the values alone.  small(x) is called
// in groups of the smallest scale, the only one with a tie below f32's normal numbers.
template <typename T, typename Small>
__device__ __forceinline__ void pack_group(float (&x)[8], uint8_t *row_codes, uint8_t *row_scales,
                                           int g, int groups, int piece, Small &&small)
{
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = row16_max(top);
    const int s = scale_byte(top);
    if (s == kMinScale)
        small(x);
    u32x2 c = {0u, 0u};
    if (s != kNanScale) {
        const float u = unscale_of(s);
        c[0] = encode4(x[0], x[1], x[2], x[3], u);
        c[1] = encode4(x[4], x[5], x[6], x[7], u);
    }
    uint8_t *to = row_codes + int64_t(g) * kGroup + run_of<T>(piece);
    if constexpr (kSecond<T> == 4) {
        *reinterpret_cast<u32x2 *>(to) = c;
    } else {
        *reinterpret_cast<unsigned *>(to) = c[0];
        *reinterpret_cast<unsigned *>(to + kSecond<T>) = c[1];
    }
    // The last group's lanes write the zeros past it too.
    if (piece == 0 || (g == groups - 1 && piece < 4 - (g & 3)))
        row_scales[g + piece] = piece == 0 ? uint8_t(s) : uint8_t(0);
}

// Elements of a row of K from k0 and from k0 + SECOND on, four each; zero past its end.
template <int SECOND>
__device__ __forceinline__ void load8(const float *row, int k0, int K, float (&x)[8])
{
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = k0 + h * SECOND;
        if (k + 4 <= K) {
            const f32x4 a = *reinterpret_cast<const any_f32x4 *>(row + k);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[4 * h + i] = a[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                x[4 * h + i] = k + i < K ? row[k + i] : 0.0f;
        }
    }
}

template <int SECOND>
__device__ __forceinline__ void load8(const uint16_t *row, int k0, int K, float (&x)[8])
{
    static_assert(SECOND == 4);
    if (k0 + 8 <= K) {
        const u32x4 a = *reinterpret_cast<const any_u32x4 *>(row + k0);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[2 * i] = __uint_as_float(a[i] << 16);
            x[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u);
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = k0 + i < K ? __uint_as_float(unsigned(row[k0 + i]) << 16) : 0.0f;
}

// A vector stored past the caches (STREAM), or into them.
template <bool STREAM, typename V, typename T>
__device__ __forceinline__ void store_vector(T *p, const V &v)
{
    typedef V Anywhere __attribute__((aligned(sizeof(T))));
    if constexpr (STREAM)
        __builtin_nontemporal_store(v, reinterpret_cast<Anywhere *>(p));
    else
        *reinterpret_cast<Anywhere *>(p) = v;
}

// The same elements stored, rounded to the row's type.
template <int SECOND, bool STREAM>
__device__ __forceinline__ void store8(float *row, int k0, int K, const float (&x)[8])
{
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int k = k0 + h * SECOND;
        if (k + 4 <= K) {
            store_vector<STREAM>(row + k,
                                 f32x4{x[4 * h], x[4 * h + 1], x[4 * h + 2], x[4 * h + 3]});
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (k + i < K)
                    row[k + i] = x[4 * h + i];
        }
    }
}

__device__ __forceinline__ unsigned bf16_pair(float lo, float hi)
{
    return __builtin_bit_cast(unsigned, __builtin_convertvector(f32x2{lo, hi}, bf16x2));
}

template <int SECOND, bool STREAM>
__device__ __forceinline__ void store8(uint16_t *row, int k0, int K, const float (&x)[8])
{
    static_assert(SECOND == 4);
    u32x4 w;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        w[i] = bf16_pair(x[2 * i], x[2 * i + 1]);
    if (k0 + 8 <= K) {
        store_vector<STREAM>(row + k0, w);
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (k0 + i < K)
            row[k0 + i] = uint16_t(w[i >> 1] >> (16 * (i & 1)));
}

}  // namespace fp8
}  // namespace anima_hip
