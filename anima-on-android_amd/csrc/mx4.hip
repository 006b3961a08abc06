// MX4 rows (mx4.h): packing, unpacking and the append to a 4-bit K/V cache.
// All three only move data (about 3 operations per element), so they are bound
// by HBM, and by their launch where the rows are few: 268 M values pack in 147 us
// from bf16 (4.6 TB/s) and 244 from f32 (5.0), unpack to f32 in 240 (5.1) and to bf16
// in 129 (5.3), and are appended from f32 in 234 (5.2) and from bf16 in 183 (3.7: a
// thread's one load of 16 bytes waits for the start position and the count);
// 2048 x 2048 take 4.0 and 5.3 us.  A thread takes eight consecutive elements, 16 or
// 32 bytes of values against 4 bytes of codes, and four neighbouring lanes hold
// one group, whose largest magnitude they find with two lane exchanges.  Unpacking,
// a thread writes 16 bytes, so that a wave's stores are contiguous (32 bytes per
// thread in two stores: 6.6 us).
#include "mx4.h"

#include <algorithm>

namespace anima_hip {
namespace {

using namespace mx4;

// Elements k0 .. k0+7 of a row of K; zero past its end.  `vec`: 16-byte loads
// of a whole piece.
__device__ __forceinline__ void load8(const float *row, int k0, int K, bool vec, float (&x)[8])
{
    if (vec && k0 + 8 <= K) {
        const f32x4 a = *reinterpret_cast<const f32x4 *>(row + k0);
        const f32x4 b = *reinterpret_cast<const f32x4 *>(row + k0 + 4);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x[i] = a[i];
            x[4 + i] = b[i];
        }
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = k0 + i < K ? row[k0 + i] : 0.0f;
}

__device__ __forceinline__ void load8(const uint16_t *row, int k0, int K, bool vec, float (&x)[8])
{
    if (vec && k0 + 8 <= K) {
        const u32x4 a = *reinterpret_cast<const u32x4 *>(row + k0);
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

// One group over four neighbouring lanes, eight elements each.  Groups with an
// infinity or a NaN have zero codes, so that packing is a function of the
// values alone.
__device__ __forceinline__ void pack_group(const float (&x)[8], uint8_t *codes, uint8_t *scale,
                                           int piece)
{
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        top = max(top, __float_as_uint(x[i]) & 0x7FFFFFFFu);
    top = max(top, unsigned(__shfl_xor(int(top), 1)));
    top = max(top, unsigned(__shfl_xor(int(top), 2)));
    const int s = scale_byte(top);
    const unsigned c = s == kNanScale ? 0u : encode8(x, scale_of(s));
    reinterpret_cast<unsigned *>(codes)[piece] = c;
    if (piece == 0)
        *scale = uint8_t(s);
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_pack_kernel(const T *x, int64_t ldx, uint8_t *codes,
                                                       uint8_t *scales, unsigned groups,
                                                       unsigned total, int K, bool vec)
{
    const unsigned gi = blockIdx.x * 64u + (threadIdx.x >> 2);
    if (gi >= total)
        return;  // all four lanes of a group
    const int piece = threadIdx.x & 3;
    const unsigned row = gi / groups;
    float v[8];
    load8(x + int64_t(row) * ldx, int(gi - row * groups) * kGroup + 8 * piece, K, vec, v);
    pack_group(v, codes + int64_t(gi) * 16, scales + gi, piece);
}

// Values of a row from k0: as many as 16 bytes hold.
template <typename T, int E>
__device__ __forceinline__ void store16(T *row, int k0, int K, bool vec, const float (&x)[E])
{
    T v[E];
#pragma unroll
    for (int i = 0; i < E; ++i)
        if constexpr (sizeof(T) == 4)
            v[i] = x[i];
        else  // MX4 values are bf16 numbers: their upper halves are the values themselves
            v[i] = uint16_t(__float_as_uint(x[i]) >> 16);
    if (vec && k0 + E <= K) {
        u32x4 w;
        __builtin_memcpy(&w, v, 16);
        *reinterpret_cast<u32x4 *>(row + k0) = w;
        return;
    }
#pragma unroll
    for (int i = 0; i < E; ++i)
        if (k0 + i < K)
            row[k0 + i] = v[i];
}

template <typename T>
__global__ __launch_bounds__(256) void mx4_unpack_kernel(const uint8_t *codes,
                                                         const uint8_t *scales, T *x, int64_t ldx,
                                                         unsigned groups, unsigned total, int K,
                                                         bool vec)
{
    constexpr int E = 16 / int(sizeof(T)), LANES = kGroup / E;  // lanes of a group
    const unsigned gi = blockIdx.x * (256u / LANES) + threadIdx.x / LANES;
    if (gi >= total)
        return;
    const int piece = threadIdx.x % LANES;
    const unsigned row = gi / groups;
    const float s = scale_of(scales[gi]);
    const uint8_t *src = codes + int64_t(gi) * 16 + piece * (E / 2);
    float v[E];
    if constexpr (E == 8) {
        const unsigned w = *reinterpret_cast<const unsigned *>(src);
        const f32x2 p[4] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 2),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 3)};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            v[i] = p[i >> 1][i & 1];
    } else {
        const unsigned w = *reinterpret_cast<const uint16_t *>(src);
        const f32x2 p[2] = {__builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 0),
                            __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, s, 1)};
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = p[i >> 1][i & 1];
    }
    store16(x + int64_t(row) * ldx, int(gi - row * groups) * kGroup + E * piece, K, vec, v);
}

template <typename T>
__global__ __launch_bounds__(256) void kv4_append_kernel(const T *k, const T *v, Kv4Append p,
                                                         unsigned total, bool vec)
{
    const unsigned gi = blockIdx.x * 64u + (threadIdx.x >> 2);
    if (gi >= total)
        return;
    const int piece = threadIdx.x & 3;
    const bool is_v = blockIdx.y != 0;
    const unsigned groups = unsigned(p.D) / kGroup;
    unsigned r = gi / groups;
    const int g = int(gi - r * groups);
    const unsigned rest = r / unsigned(p.H_kv);
    const int h = int(r - rest * unsigned(p.H_kv));
    const int b = int(rest / unsigned(p.S_new));
    const int s = int(rest - unsigned(b) * unsigned(p.S_new));
    const int64_t at = int64_t(p.starts[b]) + s;
    // A row past its sequence's count, or with no place in the cache, is left out.
    if (s >= (p.counts ? p.counts[b] : p.S_new) || at < 0 || at >= p.S_max)
        return;
    const Strides &st = is_v ? p.vs : p.ks;
    const T *src = (is_v ? v : k) + b * st.b + h * st.h + s * st.s;
    float x[8];
    load8(src, g * kGroup + 8 * piece, p.D, vec, x);
    const int64_t dst = ((int64_t(b) * p.H_kv + h) * p.S_max + at) * groups + g;
    pack_group(x, (is_v ? p.cache.v : p.cache.k) + dst * 16,
               (is_v ? p.cache.v_scales : p.cache.k_scales) + dst, piece);
}

constexpr int64_t kMx4MaxGroups = (int64_t(1) << 29) - 64;

// Pieces of eight elements can move as 16-byte accesses: base, and every
// stride in elements.
bool wide(const void *p, int64_t ld, Mx4Type t)
{
    return flash_tile::aligned(p, 16) && ld % (t == kMx4F32 ? 4 : 8) == 0;
}

// Groups of a call, up to eight threads each, in one launch of at most 2^32 threads.
bool group_count(const char *who, int64_t rows, int64_t groups, unsigned &total)
{
    if (groups > 0 && rows > kMx4MaxGroups / groups)
        return fail(std::string(who) + ": too many elements");
    total = unsigned(rows * groups);
    return true;
}

}  // namespace

bool launch_mx4_pack(const void *x, int64_t ldx, Mx4Type type, uint8_t *codes, uint8_t *scales,
                     int64_t rows, int K, hipStream_t st)
{
    const unsigned groups = unsigned(mx4_groups(K));
    unsigned total = 0;
    if (!group_count("mx4_pack_dev", rows, groups, total))
        return false;
    if (total == 0)
        return true;
    const dim3 grid((total + 63) / 64), block(256);
    const bool vec = wide(x, ldx, type);
    if (type == kMx4F32)
        hipLaunchKernelGGL(mx4_pack_kernel<float>, grid, block, 0, st,
                           static_cast<const float *>(x), ldx, codes, scales, groups, total, K, vec);
    else
        hipLaunchKernelGGL(mx4_pack_kernel<uint16_t>, grid, block, 0, st,
                           static_cast<const uint16_t *>(x), ldx, codes, scales, groups, total, K,
                           vec);
    return hip_ok(hipGetLastError(), "mx4_pack_kernel launch");
}

bool launch_mx4_unpack(const uint8_t *codes, const uint8_t *scales, void *x, int64_t ldx,
                       Mx4Type type, int64_t rows, int K, hipStream_t st)
{
    const unsigned groups = unsigned(mx4_groups(K));
    unsigned total = 0;
    if (!group_count("mx4_unpack_dev", rows, groups, total))
        return false;
    if (total == 0)
        return true;
    const unsigned per = type == kMx4F32 ? 32 : 64;  // groups of a workgroup
    const dim3 grid((total + per - 1) / per), block(256);
    const bool vec = wide(x, ldx, type);
    if (type == kMx4F32)
        hipLaunchKernelGGL(mx4_unpack_kernel<float>, grid, block, 0, st, codes, scales,
                           static_cast<float *>(x), ldx, groups, total, K, vec);
    else
        hipLaunchKernelGGL(mx4_unpack_kernel<uint16_t>, grid, block, 0, st, codes, scales,
                           static_cast<uint16_t *>(x), ldx, groups, total, K, vec);
    return hip_ok(hipGetLastError(), "mx4_unpack_kernel launch");
}

bool launch_kv4_append(const void *k, const void *v, Mx4Type type, const Kv4Append &p,
                       hipStream_t st)
{
    unsigned total = 0;
    const int64_t rows = int64_t(p.B) * p.S_new;
    if (p.H_kv > 0 && rows > kMx4MaxGroups / p.H_kv)
        return fail("kv4_append_dev: too many elements");
    if (!group_count("kv4_append_dev", rows * p.H_kv, mx4_groups(p.D), total))
        return false;
    if (total == 0)
        return true;
    bool vec = true;
    for (const Strides *s : {&p.ks, &p.vs})
        for (int64_t ld : {s->b, s->h, s->s})
            vec = vec && wide(s == &p.ks ? k : v, ld, type);
    const dim3 grid((total + 63) / 64, 2), block(256);
    if (type == kMx4F32)
        hipLaunchKernelGGL(kv4_append_kernel<float>, grid, block, 0, st,
                           static_cast<const float *>(k), static_cast<const float *>(v), p, total,
                           vec);
    else
        hipLaunchKernelGGL(kv4_append_kernel<uint16_t>, grid, block, 0, st,
                           static_cast<const uint16_t *>(k), static_cast<const uint16_t *>(v), p,
                           total, vec);
    return hip_ok(hipGetLastError(), "kv4_append_kernel launch");
}

}  // namespace anima_hip
