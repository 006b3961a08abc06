// Rotary positions with several axes: token (b, s) stands at positions[b][s][a]
// on axis a, and pair p of every head of its query and key rows turns by
//   theta = positions[b][s][axis[p]] * freqs[p]:
//   (xa, xb) -> (xa cos - xb sin, xb cos + xa sin),
// or back by -theta (the gradient of the turn, and its inverse).  Pairs are
// (p, p + pairs) or neighbours (2p, 2p + 1) of a row's first 2 * pairs elements;
// the rest of a row is copied.
//
// Bound by HBM: every value is read and written once, against six operations a
// pair.  A workgroup takes the tokens that give each thread one chunk, up to 16 bytes of
// either member of its pairs, and computes their angles' cosines and sines once for all
// heads into LDS while the chunks are on their way.  From cold memory (calls in a captured
// graph over arrays in turn) 2 x 4096 tokens of 32 f32 heads of 128 take 49.2 us, 5.5 TB/s, and
// 30003 tokens of 14 bf16 heads of 64 25.7 us, 4.2 TB/s; over the same arrays again, which the
// last-level cache then holds in part or whole, 40.6 and 18.5 us.  Stores stay in the caches for
// the attention, which reads the rows next: 8192 tokens of 16 bf16 heads of 128 written and read
// back take 11.4 us, past the caches 14.1, though alone and from cold memory the store would gain
// a tenth.
#include "flash_tile.h"

#include <algorithm>

namespace anima_hip {
namespace {

using flash_tile::bf16x2;
using flash_tile::f32x2;

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
    Divisor pairs_by, sequence;  // by pairs, by S where a workgroup's tokens are more
    int turned;        // chunks of a head that turn; the rest are copied
    bool inverse;
};

// V elements, in words of 32 bits.
template <typename T, int V>
struct Vec {
    static constexpr int kEach = 4 / sizeof(T);
    typedef unsigned Words __attribute__((ext_vector_type(V / kEach)));
    typedef Words Anywhere __attribute__((aligned(sizeof(T))));  // as the hardware takes them
    Words v;
    // All of them, or with TAIL the first n.
    template <bool TAIL>
    __device__ __forceinline__ void load(const T *p, int n)
    {
        if (!TAIL || n >= V) {
            v = *reinterpret_cast<const Anywhere *>(p);
            return;
        }
        v = Words{};
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 4)
                    v[i] = __float_as_uint(p[i]);
                else
                    v[i / 2] |= unsigned(p[i]) << (i % 2 * 16);
            }
    }
    template <bool TAIL>
    __device__ __forceinline__ void store(T *p, int n) const
    {
        if (!TAIL || n >= V) {
            *reinterpret_cast<Anywhere *>(p) = v;
            return;
        }
#pragma unroll
        for (int i = 0; i < V; ++i)
            if (i < n) {
                if constexpr (sizeof(T) == 4)
                    p[i] = __uint_as_float(v[i]);
                else
                    p[i] = uint16_t(v[i / 2] >> (i % 2 * 16));
            }
    }
    __device__ __forceinline__ float get(int i) const
    {
        return __uint_as_float(sizeof(T) == 4 ? v[i]
                               : i % 2        ? v[i / kEach] & 0xFFFF0000u
                                              : v[i / kEach] << 16);
    }
    __device__ __forceinline__ void set(const float (&x)[V])
    {
#pragma unroll
        for (int i = 0; i < V / kEach; ++i)
            if constexpr (sizeof(T) == 4)
                v[i] = __float_as_uint(x[i]);
            else
                v[i] = __builtin_bit_cast(
                    unsigned, __builtin_convertvector(f32x2{x[2 * i], x[2 * i + 1]}, bf16x2));
    }
};

// A chunk is two vectors of V elements: V pairs of a head, or 2 V copied elements; the last
// of either may hold fewer (TAIL).  Whole chunks' vectors are half a turned row apart, also
// where pairs are neighbours, so that lanes' accesses follow one another (30003
// tokens of 14 heads of 64, arrays in the last-level cache: 19.5 us, so 18.9).
template <typename T, int V, bool NEIGHBOURS, bool TAIL>
__global__ __launch_bounds__(kThreads) void rope_axes_kernel(RopeArgs p)
{
    using X = Vec<T, V>;
    __shared__ float2 table[kTable + V];  // a head's last chunk reads past its angles
    const int64_t token0 = int64_t(blockIdx.x) * p.per_block;
    const int n = int(min<int64_t>(p.per_block, p.tokens - token0));
    // Uniform: the only 64-bit division.
    const int64_t b0 = token0 / p.S;
    const unsigned s0 = unsigned(token0 - b0 * p.S);
    struct Place {
        int64_t b;
        int s;
    };
    const auto place = [&](unsigned t) {
        const unsigned at = s0 + t;
        const unsigned on = p.S >= p.per_block ? unsigned(at >= unsigned(p.S))
                                               : p.sequence.quotient(at);
        return Place{b0 + on, int(at - on * unsigned(p.S))};
    };
    // Where an item's two vectors lie.
    struct Item {
        T *dst;
        const float2 *cs;
        X x0, x1;
        int d0, d1, n0, n1;  // places, elements
        bool turn;
    };
    const auto fetch = [&](unsigned i, Item &it) {
        const unsigned t = p.per_block == 1 ? 0u : p.items.quotient(i);
        const unsigned item = i - t * p.items.d;
        int h = int(p.chunks.quotient(item));
        const int c = int(item - h * p.chunks.d);
        const Place at = place(t);
        if (p.counts && at.s >= p.counts[at.b])
            return false;
        const int which = h >= p.heads_q;
        h -= which ? p.heads_q : 0;
        const T *src = static_cast<const T *>(p.in[which]) + at.b * p.is[which].b +
                       h * p.is[which].h + at.s * p.is[which].s;
        it.dst = static_cast<T *>(p.out[which]) + at.b * p.os[which].b + h * p.os[which].h +
                 at.s * p.os[which].s;
        it.turn = c < p.turned;
        if (it.turn) {
            it.d0 = NEIGHBOURS && TAIL ? 2 * V * c : V * c;
            it.d1 = NEIGHBOURS && TAIL ? it.d0 + V : it.d0 + p.pairs;
            it.n0 = NEIGHBOURS ? 2 * p.pairs - it.d0 : p.pairs - it.d0;
            it.n1 = NEIGHBOURS ? it.n0 - V : it.n0;
        } else {
            it.d0 = 2 * p.pairs + (c - p.turned) * 2 * V;
            it.d1 = it.d0 + V;
            it.n0 = p.D - it.d0;
            it.n1 = it.n0 - V;
        }
        it.cs = table + t * p.pairs + (NEIGHBOURS && !TAIL ? c * V / 2 : c * V);
        it.x0.template load<TAIL>(src + it.d0, it.n0);
        if (it.n1 > 0)
            it.x1.template load<TAIL>(src + it.d1, it.n1);
        return true;
    };
    const auto turn = [&](Item &it) {
        float y0[V], y1[V];
        if constexpr (NEIGHBOURS) {
#pragma unroll
            for (int j = 0; j < V; j += 2) {
                const float2 u = it.cs[j / 2];
                const float2 w = it.cs[(TAIL ? V : p.pairs) / 2 + j / 2];
                y0[j] = it.x0.get(j) * u.x - it.x0.get(j + 1) * u.y;
                y0[j + 1] = it.x0.get(j + 1) * u.x + it.x0.get(j) * u.y;
                y1[j] = it.x1.get(j) * w.x - it.x1.get(j + 1) * w.y;
                y1[j + 1] = it.x1.get(j + 1) * w.x + it.x1.get(j) * w.y;
            }
        } else {
#pragma unroll
            for (int j = 0; j < V; ++j) {
                const float2 u = it.cs[j];
                y0[j] = it.x0.get(j) * u.x - it.x1.get(j) * u.y;
                y1[j] = it.x1.get(j) * u.x + it.x0.get(j) * u.y;
            }
        }
        it.x0.set(y0);
        it.x1.set(y1);
    };
    const unsigned items = n * p.items.d;
    for (unsigned first = 0; first < items; first += kThreads) {
        const unsigned i = first + threadIdx.x;
        Item it;
        const bool live = i < items && fetch(i, it);
        if (first == 0) {
            // The angles while the first rows are on their way.
            for (unsigned j = threadIdx.x; j < unsigned(n * p.pairs); j += kThreads) {
                const unsigned t = p.pairs_by.quotient(j), pair = j - t * p.pairs;
                const Place at = place(t);
                const int a = p.axis ? min(int(p.axis[pair]), p.axes - 1) : 0;
                // In turns, in 64 bits: a far position's angle keeps its place within the
                // turn to 2^-53 of itself.
                const double turns =
                    double(p.pos[at.b * p.pos_batch + int64_t(at.s) * p.axes + a]) *
                    p.freqs[pair] * 0.15915494309189535;
                // bf16 outputs lose nothing to cosines in f32 (2 ulp; 64 bits cost 2 to 6 %
                // there, nothing in f32).
                const double part = turns - rint(turns);
                float sn, cs;
                if constexpr (sizeof(T) == 4) {
                    double s64, c64;
                    sincospi(2.0 * part, &s64, &c64);
                    sn = float(s64);
                    cs = float(c64);
                } else {
                    sincospif(2.0f * float(part), &sn, &cs);
                }
                table[j] = float2{cs, p.inverse ? -sn : sn};
            }
            __syncthreads();
        }
        if (!live)
            continue;
        if (it.turn)
            turn(it);
        it.x0.template store<TAIL>(it.dst + it.d0, it.n0);
        if (it.n1 > 0)
            it.x1.template store<TAIL>(it.dst + it.d1, it.n1);
    }
}

template <typename T, int V, bool TAIL>
bool run_rope(const RopeAxes &a, RopeArgs &p, bool copies, hipStream_t st)
{
    const int heads = a.H_q + a.H_k;
    p.turned = (a.pairs + V - 1) / V;
    const int rest = copies ? (a.D - 2 * a.pairs + 2 * V - 1) / (2 * V) : 0;
    const int chunks = p.turned + rest;
    // At most 1024 chunks of a head and 2^12 heads: every quotient is exact.
    p.chunks = Divisor(unsigned(chunks));
    p.items = Divisor(unsigned(chunks * heads));
    // A chunk a thread, or two that share their angles' table where the GPU is full anyway
    // (30003 tokens of 12 + 2 bf16 heads of 64 18.5 us from the last-level cache, where the
    // products before leave them, with one each 19.5, though from cold memory 25.7 and 24.8; 8
    // tokens of 16 + 4 heads of 128 3.7 and 2.9), and no more angles than the table holds.
    const int each = p.tokens * chunks * heads > 2048 * kThreads ? 2 : 1;
    p.per_block = std::max(1, std::min(each * kThreads / (chunks * heads), kTable / a.pairs));
    p.pairs_by = Divisor(unsigned(a.pairs));
    p.sequence = Divisor(unsigned(std::min(a.S, 2 * kThreads)));
    const int64_t blocks = (p.tokens + p.per_block - 1) / p.per_block;
    if (blocks > UINT32_MAX / kThreads)
        return fail("rope_axes_dev: too many tokens for one launch");
    const dim3 grid(static_cast<unsigned>(blocks));
    if (a.interleaved)
        hipLaunchKernelGGL((rope_axes_kernel<T, V, true, TAIL>), grid, dim3(kThreads), 0, st, p);
    else
        hipLaunchKernelGGL((rope_axes_kernel<T, V, false, TAIL>), grid, dim3(kThreads), 0, st, p);
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
    // A row that is not turned in place has a rest to copy.
    const bool copies = (a.H_q > 0 && a.q != a.q_out) || (a.H_k > 0 && a.k != a.k_out);
    // 16 bytes a vector, wherever rows begin.  Heads that these do not divide end in a shorter
    // chunk, element by element: bf16 then moves 8 bytes (12 heads of 78, 10001 tokens from the
    // last-level cache: 18.5 us, by 16 bytes 21.9, by 4 21.3, by single elements 24.3; from cold
    // memory 25.1).
    const int split = a.pairs | a.D;
    if (a.type == kMx4F32)
        return split % 4 == 0 ? run_rope<float, 4, false>(a, p, copies, st)
                              : run_rope<float, 4, true>(a, p, copies, st);
    if (split % 8 == 0)
        return run_rope<uint16_t, 8, false>(a, p, copies, st);
    return split % 4 == 0 ? run_rope<uint16_t, 4, false>(a, p, copies, st)
                          : run_rope<uint16_t, 4, true>(a, p, copies, st);
}

}  // namespace anima_hip
