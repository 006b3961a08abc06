// Rotary positions with several axes: token (b, s) stands at positions[b][s][a]
// on axis a, and pair p of every head of its query and key rows turns by
//   theta = positions[b][s][axis[p]] * freqs[p]:
//   (xa, xb) -> (xa cos - xb sin, xb cos + xa sin),
// or back by -theta (the gradient of the turn, and its inverse).  Pairs are
// (p, p + pairs) or neighbours (2p, 2p + 1) of a row's first 2 * pairs elements;
// the rest of a row is copied.
//
// Bound by HBM: every value is read and written once, against six operations a
// pair.  A workgroup takes the tokens that give each thread about two vector
// pairs, computes their angles' cosines and sines once for all heads into LDS, and turns
// 16 bytes of either half of a pair per thread.
#include "flash_tile.h"

#include <algorithm>

namespace anima_hip {
namespace {

using flash_tile::aligned;
using flash_tile::bf16x2;
using flash_tile::f32x2;
using flash_tile::f32x4;
using flash_tile::u32x4;

constexpr int kThreads = 256;
constexpr int kTable = 1024;  // angles of a workgroup, most

// n / d by a multiplication with m = ceil(2^32 / d): exact where n * d < 2^32.
struct Divisor {
    unsigned d = 1, m = 0;
    Divisor() = default;
    explicit Divisor(unsigned by) : d(by), m(unsigned(((uint64_t(1) << 32) + by - 1) / by)) {}
    __device__ __forceinline__ unsigned quotient(unsigned n) const
    {
        return d == 1 ? n : __umulhi(n, m);
    }
};

struct RopeArgs {
    const void *in[2];
    void *out[2];
    Strides is[2], os[2];
    const int32_t *pos, *counts;
    const double *freqs;
    const uint8_t *axis;
    int64_t pos_batch, tokens;  // tokens: B * S
    int S, axes, pairs, D, heads_q;
    int per_block;     // tokens of a workgroup
    Divisor items, chunks;  // of a token, of a head
    int turned;        // chunks of a head that turn; the rest are copied
    bool inverse;
};

template <typename T, int V>
struct Vec;
template <>
struct Vec<float, 4> {
    f32x4 v;
    __device__ __forceinline__ float get(int i) const { return v[i]; }
    __device__ __forceinline__ void set(const float (&x)[4]) { v = f32x4{x[0], x[1], x[2], x[3]}; }
};
template <>
struct Vec<uint16_t, 8> {
    u32x4 v;
    __device__ __forceinline__ float get(int i) const
    {
        return __uint_as_float(i & 1 ? v[i >> 1] & 0xFFFF0000u : v[i >> 1] << 16);
    }
    __device__ __forceinline__ void set(const float (&x)[8])
    {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            v[i] = __builtin_bit_cast(
                unsigned, __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, bf16x2));
    }
};
template <>
struct Vec<float, 1> {
    float v;
    __device__ __forceinline__ float get(int) const { return v; }
    __device__ __forceinline__ void set(const float (&x)[1]) { v = x[0]; }
};
template <>
struct Vec<uint16_t, 1> {
    uint16_t v;
    __device__ __forceinline__ float get(int) const { return __uint_as_float(unsigned(v) << 16); }
    __device__ __forceinline__ void set(const float (&x)[1])
    {
        v = __builtin_bit_cast(uint16_t, static_cast<__bf16>(x[0]));
    }
};

// A chunk is two vectors of V elements: V pairs of a head, or 2 V copied elements.
template <typename T, int V, bool NEIGHBOURS>
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(RopeArgs p)
{
    using X = Vec<T, V>;
    __shared__ float2 table[kTable];
    const int64_t token0 = int64_t(blockIdx.x) * p.per_block;
    const int n = int(min<int64_t>(p.per_block, p.tokens - token0));
    for (int i = threadIdx.x; i < n * p.pairs; i += kThreads) {
        const int t = i / p.pairs, pair = i - t * p.pairs;
        const int64_t token = token0 + t;
        const int64_t b = token / p.S;
        const int s = int(token - b * p.S);
        const int a = p.axis ? min(int(p.axis[pair]), p.axes - 1) : 0;
        // In turns, in 64 bits: a far position's angle keeps its place within the
        // turn to 2^-53 of itself.
        const double turns = double(p.pos[b * p.pos_batch + int64_t(s) * p.axes + a]) *
                             p.freqs[pair] * 0.15915494309189535;
        float sn, cs;
        sincospif(2.0f * float(turns - rint(turns)), &sn, &cs);
        table[i] = float2{cs, p.inverse ? -sn : sn};
    }
    __syncthreads();
    for (unsigned i = threadIdx.x; i < n * p.items.d; i += kThreads) {
        const unsigned t = p.per_block == 1 ? 0u : p.items.quotient(i);
        const unsigned item = i - t * p.items.d;
        int h = int(p.chunks.quotient(item));
        const int c = int(item - h * p.chunks.d);
        const int64_t token = token0 + t;
        const int64_t b = token / p.S;
        const int s = int(token - b * p.S);
        if (p.counts && s >= p.counts[b])
            continue;
        const int which = h >= p.heads_q;
        h -= which ? p.heads_q : 0;
        const T *src = static_cast<const T *>(p.in[which]) + b * p.is[which].b +
                       h * p.is[which].h + s * p.is[which].s;
        T *dst = static_cast<T *>(p.out[which]) + b * p.os[which].b + h * p.os[which].h +
                 s * p.os[which].s;
        if (c >= p.turned) {
            const int d = 2 * p.pairs + (c - p.turned) * 2 * V;
            *reinterpret_cast<X *>(dst + d) = *reinterpret_cast<const X *>(src + d);
            if (d + V < p.D)
                *reinterpret_cast<X *>(dst + d + V) = *reinterpret_cast<const X *>(src + d + V);
            continue;
        }
        const int d0 = NEIGHBOURS ? 2 * V * c : V * c, d1 = NEIGHBOURS ? d0 + V : d0 + p.pairs;
        const X x0 = *reinterpret_cast<const X *>(src + d0);
        const X x1 = *reinterpret_cast<const X *>(src + d1);
        const float2 *cs = table + t * p.pairs + c * V;
        float y0[V], y1[V];
        if constexpr (NEIGHBOURS && V > 1) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 u = cs[j / 2], w = cs[V / 2 + j / 2];
                y0[j] = x0.get(j) * u.x - x0.get(j + 1) * u.y;
                y0[j + 1] = x0.get(j + 1) * u.x + x0.get(j) * u.y;
                y1[j] = x1.get(j) * w.x - x1.get(j + 1) * w.y;
                y1[j + 1] = x1.get(j + 1) * w.x + x1.get(j) * w.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 u = cs[j];
                y0[j] = x0.get(j) * u.x - x1.get(j) * u.y;
                y1[j] = x1.get(j) * u.x + x0.get(j) * u.y;
            }
        }
        X z;
        z.set(y0);
        *reinterpret_cast<X *>(dst + d0) = z;
        z.set(y1);
        *reinterpret_cast<X *>(dst + d1) = z;
    }
}

template <typename T, int V>
bool run_rope(const RopeAxes &a, RopeArgs &p, bool copies, hipStream_t st)
{
    const int heads = a.H_q + a.H_k;
    p.turned = a.pairs / V;
    const int rest = copies ? (a.D - 2 * a.pairs + 2 * V - 1) / (2 * V) : 0;
    const int chunks = p.turned + rest;
    // At most 1024 chunks of a head and 2^12 heads: every quotient is exact.
    p.chunks = Divisor(unsigned(chunks));
    p.items = Divisor(unsigned(chunks * heads));
    // About two items a thread, and no more angles than the table holds.
    p.per_block = std::max(1, std::min(2 * kThreads / (chunks * heads), kTable / a.pairs));
    const int64_t blocks = (p.tokens + p.per_block - 1) / p.per_block;
    if (blocks > UINT32_MAX / kThreads)
        return fail("rope_axes_dev: too many tokens for one launch");
    const dim3 grid(static_cast<unsigned>(blocks));
    if (a.interleaved)
        hipLaunchKernelGGL((rope_axes_kernel<T, V, true>), grid, dim3(kThreads), 0, st, p);
    else
        hipLaunchKernelGGL((rope_axes_kernel<T, V, false>), grid, dim3(kThreads), 0, st, p);
    return hip_ok(hipGetLastError(), "rope_axes_kernel launch");
}

}  // namespace

bool launch_rope_axes(const RopeAxes &a, hipStream_t st)
{
    if (a.B <= 0 || a.S <= 0 || a.H_q + a.H_k <= 0)
        return true;
    RopeArgs p{};
    p.in[0] = a.q;
    p.in[1] = a.k;
    p.out[0] = a.q_out;
    p.out[1] = a.k_out;
    p.is[0] = a.qs;
    p.is[1] = a.ks;
    p.os[0] = a.qos;
    p.os[1] = a.kos;
    p.pos = a.positions;
    p.counts = a.counts;
    p.freqs = a.freqs;
    p.axis = a.pair_axis;
    p.pos_batch = a.pos_batch;
    p.tokens = int64_t(a.B) * a.S;
    p.S = a.S;
    p.axes = a.axes;
    p.pairs = a.pairs;
    p.D = a.D;
    p.heads_q = a.H_q;
    p.inverse = a.inverse;
    const int V = a.type == kMx4F32 ? 4 : 8;
    // 16-byte vectors where every piece starts and ends on one.
    bool vec = a.pairs % V == 0 && a.D % V == 0;
    bool copies = false;  // rows that are not turned in place have a rest to copy
    for (int i = 0; i < 2; ++i) {
        if ((i ? a.H_k : a.H_q) == 0)
            continue;
        for (int64_t s : {p.is[i].b, p.is[i].h, p.is[i].s, p.os[i].b, p.os[i].h, p.os[i].s})
            vec = vec && s % V == 0;
        vec = vec && aligned(p.in[i], 16) && aligned(p.out[i], 16);
        copies = copies || p.in[i] != p.out[i];
    }
    if (a.type == kMx4F32)
        return vec ? run_rope<float, 4>(a, p, copies, st) : run_rope<float, 1>(a, p, copies, st);
    return vec ? run_rope<uint16_t, 8>(a, p, copies, st)
               : run_rope<uint16_t, 1>(a, p, copies, st);
}

}  // namespace anima_hip
