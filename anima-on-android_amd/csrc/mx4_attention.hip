// Attention over a 4-bit K/V cache (mx4.h rows): O = softmax(scale Q K^T) V
// with K and V decoded to bf16 in registers, where they are exact, and f32
// scores, softmax statistics and sums.
//
// A K/V head serves H / H_kv query heads; its query rows are numbered
// r = s * (H / H_kv) + (head within the group), so that neighbouring rows see
// nearly the same keys under a causal mask.  S^T = K Q^T and O^T = V^T P^T are
// computed, so that a query row is one column of every accumulator.  bf16
// queries enter as they are and P as one bf16 term, as in the other bf16 attention
// kernels: off by at most half a bf16 step a key, which is the output's own
// rounding, where three terms would be three times the second product's MFMAs
// (cross-attention 4096 x 512 x 16 heads of 128, B = 2: 58 us, and 123 with f32
// queries).  The token kernel sums the probabilities before that rounding, the
// tile kernel after it.  f32 queries and their P enter as three terms each
// (mx4::terms2), so products are exact to f32.
//
//   * token kernel: 16 or 32 query rows per wave on v_mfma_f32_16x16x32_bf16, the
//     waves of a workgroup and the workgroups of a split sharing the keys.  32 rows
//     read and decode a key once where 16 do so twice: 16 sequences of up to 8192
//     keys, 8 queries, 32 heads on 8 of 128, bf16, 44.8 -> 35.5 us; in f32 at D = 128
//     they take more registers than there are (56 -> 87).
//     Bound by the one pass over the cache (17/16 byte per key and dimension
//     for K and V together: 91 MB in 22 us, 4.2 TB/s, for a query each of 16
//     sequences of up to 16384 keys), by latency where the cache is short (200
//     keys 8 us), and by its VALU work where the rows are many.  Codes go
//     from memory to registers to the MFMA and nothing is staged in LDS: a
//     lane's 16 bytes of a K row are one scale group (the MFMA's k index runs
//     over d in the order the lanes hold it), and V^T fragments are pairs of
//     V rows transposed by two byte permutes per two codes.
//   * tile kernel: many query rows.  Tiles of 64 keys are decoded once per
//     workgroup of 128 query rows into LDS, K as rows and V transposed, while
//     the codes of the tile after next are on their way; 32 query rows per wave
//     on v_mfma_f32_32x32x16_bf16, two workgroups on a CU.  Bound by the
//     softmax's VALU work and the MFMAs, which overlap only between the two
//     waves of a SIMD: bf16 303 us (0.91 PFLOP/s) at 4096 x 4096 x 16 heads x 2,
//     50 us at 4096 x 512 (24 us for its MFMAs alone, 141 us by the first
//     token kernel).  Workgroups of 256 rows over 128 keys, one on a CU, take
//     2 to 6 % less at whole multiples of 256 rows and more elsewhere; the
//     scores of the next tile computed between the exponentials of this one take
//     18 % more, the registers for both tiles' scores being short.
//
// A masked key never reaches a row: its score is left out of the maximum and
// the sum, and the decoded V of keys past the cache's length is finite.  Inside
// the length a V group may be NaN (scale byte 255) while some rows may not see
// its key: such groups are decoded as zero and their NaN is added to the rows
// that do see them.  The tile kernel looks for them in all its keys' scale bytes
// once it has met one: 250 queries, 16 heads on 1, 9000 keys, 53 us, and 314 with one
// NaN group.
#include "mx4.h"
#include "mx4_plan.h"

#include <algorithm>
#include <cmath>

// No fused score: exp2(s - max) is taken of the rounded score the maximum was
// taken of, so the largest probability is 1.
#pragma clang fp contract(off)

namespace anima_hip {
namespace {

using namespace flash_tile;
using mx4::decode2_at;
using mx4::decode8;
using mx4::mfma16;
using mx4::scale_of;
using mx4::terms2;
using mx4::u32x2;
using namespace mx4_plan;

template <typename T>
constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;

__device__ __forceinline__ void store_o(float *o, float v) { *o = v; }
__device__ __forceinline__ void store_o(uint16_t *o, float v)
{
    const __bf16 b = static_cast<__bf16>(v);
    *o = __builtin_bit_cast(uint16_t, b);
}

// Max over the four lanes n, n + 16, n + 32, n + 48 of a query.
__device__ __forceinline__ float quad_max(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false,
                                                    false);
    return row_pair_max(fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1])));
}

// bf16 queries: a row whose scaled maximum m2 has no fraction left.  Its scores
// take their distance from the maximum first.
constexpr float kFarLog2 = 0x1p24f;
template <int NT>
__device__ __forceinline__ bool far_row(float m2)
{
    return NT == 1 && fabsf(m2) > kFarLog2;
}

// What scores are taken against.  A row whose scores are all -inf so far (products past
// the range of f32) has no distance from its maximum, which would be NaN: against
// zero each of them weighs nothing, and a NaN score stays one.
__device__ __forceinline__ float max_or_zero(float mx) { return mx == -INFINITY ? 0.0f : mx; }

// The argument of a probability's exponential.  f32 queries and far rows (whose scores
// are distances by then, with m2 = 0): (score - mx) * scale2.  Other rows of bf16 queries: one
// fused operation, which takes the scaled maximum as it was rounded; base_shift is what that
// adds to all arguments against the same maximum.
template <int NT>
__device__ __forceinline__ float exponent(float score, float mx, float scale2, float m2)
{
    return NT == 1 ? __builtin_fmaf(score, scale2, -m2) : (score - mx) * scale2;
}
template <int NT>
__device__ __forceinline__ float base_shift(float mx, float scale2)
{
    const float m2 = mx * scale2;
    return NT == 3 || mx == -INFINITY || far_row<NT>(m2) ? 0.0f
                                                          : __builtin_fmaf(mx, scale2, -m2);
}

// What takes probabilities and their sums from the maximum `from` to `to`, both raw scores:
// waves, splits and the steps of one wave meet at their distance, which stays exact where
// their scaled values have lost it, and at the shifts their exponents hold (up to 0.5).
// Halves, whose distance is always a number: the scale may be small, or 0.
template <int NT>
__device__ __forceinline__ float rebase(float from, float to, float scale2)
{
    return __builtin_amdgcn_exp2f(2.0f * ((0.5f * from - 0.5f * to) * scale2) +
                                  (base_shift<NT>(to, scale2) - base_shift<NT>(from, scale2)));
}

// A partial result times its weight.  A NaN value reaches the row however little its
// key weighs beside the others, wherever it lies; a sum that passed the range of f32 among
// keys that weigh nothing does not.
__device__ __forceinline__ float weighed(float w, float x)
{
    return w != 0.0f || x != x ? w * x : 0.0f;
}

struct AttnArgs {
    Kv4Attention p;
    float scale2;   // softmax scale * log2(e) / q_factor, not negative
    float q_factor;  // on the queries: the scale's sign, and for f32 part of a tiny scale
    int group;      // H / H_kv
    int rows;       // S_q * group
    int tiles;      // query tiles of a K/V head
    int splits;
    float *part;    // [splits][B * S_q * H][D] O of each split, normalised
    float2 *ml;     // [splits][B * S_q * H] (max of the raw scores, sum); sum 0: no weight
};

// The sequence a workgroup works on.
struct Seq {
    int len, nq;      // cached keys, query tokens
    int64_t kv_row;   // first cache row of the K/V head
    __device__ __forceinline__ Seq(const Kv4Attention &p, int b, int hk)
    {
        const int bk = p.Bk == 1 ? 0 : b;
        len = min(max(p.lens[bk], 0), p.S_max);
        nq = p.counts ? min(max(p.counts[b], 0), p.S_q) : p.S_q;
        kv_row = (int64_t(bk) * p.H_kv + hk) * p.S_max;
    }
    // Keys that query token s sees: 0 .. limit - 1.
    __device__ __forceinline__ int limit(const Kv4Attention &p, int s) const
    {
        return p.causal ? min(max(len - nq + s + 1, 0), len) : len;
    }
};

// A query row's eight values from d times the factor (bf16: 1 or -1) as bf16 terms.
__device__ __forceinline__ void q_terms(const uint16_t *q, bool wide, float factor, bf16x8 (&t)[1])
{
    u32x4 u;
    if (wide)
        u = *reinterpret_cast<const u32x4 *>(q);
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            u[i] = unsigned(q[2 * i]) | unsigned(q[2 * i + 1]) << 16;
    }
    t[0] = __builtin_bit_cast(bf16x8, factor < 0.0f ? u ^ 0x80008000u : u);
}

template <bool INF = true>
__device__ __forceinline__ void terms8(const float (&x)[8], bf16x8 (&t)[3])
{
    u32x4 u[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned w[3];
        terms2<3, INF>(x[2 * i], x[2 * i + 1], w);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            u[j][i] = w[j];
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
        t[j] = __builtin_bit_cast(bf16x8, u[j]);
}

__device__ __forceinline__ void q_terms(const float *q, bool, float factor, bf16x8 (&t)[3])
{
    float x[8];
#pragma unroll
    for (int i = 0; i < 8; ++i)
        x[i] = q[i] * factor;
    terms8(x, t);
}

// Eight probabilities as the P operand: one rounded term or three exact ones.
__device__ __forceinline__ void p_terms(const float (&p)[8], bf16x8 (&t)[1])
{
    u32x4 u;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        u[i] = __builtin_bit_cast(
            unsigned, __builtin_convertvector(f32x2{p[2 * i], p[2 * i + 1]}, bf16x2));
    t[0] = __builtin_bit_cast(bf16x8, u);
}
__device__ __forceinline__ void p_terms(const float (&p)[8], bf16x8 (&t)[3])
{
    terms8<false>(p, t);  // at most 2^8
}

// ----------------------------------------------------------- token kernel

// A wave's loads for 32 keys.  Lane (m, g): K rows t0 + m and t0 + 16 + m,
// dimensions g * D/4 .. ; V rows of the eight keys 4g + 0..3 and 16 + 4g +
// 0..3, dimensions m * D/16 .. .  Addresses are a base of the wave plus an
// offset of the lane that stays the same from step to step.
template <int D>
struct TokLoads {
    static constexpr int GROUPS = D / 32;
    static constexpr int ROW = D / 2;  // bytes of a row's codes
    unsigned kc[2][D / 32];
    unsigned ks[2];
    unsigned vc[8];
    unsigned vs[8];

    __device__ __forceinline__ void load_k(const uint8_t *codes, const uint8_t *scales, int h,
                                           unsigned key, unsigned g)
    {
        const uint8_t *src = codes + (key * ROW + g * (D / 8));
        if constexpr (D == 128) {
            const u32x4 w = *reinterpret_cast<const u32x4 *>(src);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                kc[h][i] = w[i];
        } else {
            const u32x2 w = *reinterpret_cast<const u32x2 *>(src);
            kc[h][0] = w[0];
            kc[h][1] = w[1];
        }
        ks[h] = scales[key * GROUPS + g * GROUPS / 4];
    }
    __device__ __forceinline__ void load_v(const uint8_t *codes, const uint8_t *scales, int j,
                                           unsigned key, unsigned m)
    {
        const uint8_t *src = codes + (key * ROW + m * (D / 32));
        if constexpr (D == 128)
            vc[j] = *reinterpret_cast<const unsigned *>(src);
        else
            vc[j] = *reinterpret_cast<const uint16_t *>(src);
        vs[j] = scales[key * GROUPS + m * GROUPS / 16];
    }
    // Keys row .. row + 31 of the cache; past row + over, that key again.
    template <bool TAIL>
    __device__ __forceinline__ void load(const Kv4Cache &c, int64_t row, unsigned over, unsigned m,
                                         unsigned g)
    {
        const uint8_t *kc0 = c.k + row * ROW, *ks0 = c.k_scales + row * GROUPS;
        const uint8_t *vc0 = c.v + row * ROW, *vs0 = c.v_scales + row * GROUPS;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const unsigned key = 16 * h + m;
            load_k(kc0, ks0, h, TAIL ? min(key, over) : key, g);
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const unsigned key = 16 * (j >> 2) + 4 * g + (j & 3);
            load_v(vc0, vs0, j, TAIL ? min(key, over) : key, m);
        }
    }
};

template <typename T, int D, int RB>
__global__ __launch_bounds__(kTokWaves * 64, 2) void kv4_token_kernel(AttnArgs a)
{
    constexpr int NT = kTerms<T>;
    constexpr int STEPS = D / 32;  // MFMA steps of a score; V^T blocks of 16 are D / 16
    constexpr int VB = D / 16;
    constexpr int OPITCH = D + 4, ROWS = RB * kTokRows;
    __shared__ __attribute__((aligned(16))) float so[kTokWaves][ROWS][OPITCH];
    __shared__ float sm[kTokWaves][ROWS], sl[kTokWaves][ROWS];

    const Kv4Attention &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    // Neighbouring workgroups go to different XCDs, and the shares of a long
    // sequence with them.
    const int blk = blockIdx.x;
    const int split = blk % a.splits;
    const int bh = (blk / a.splits) % (p.B * p.H_kv);
    const int tile = (blk / a.splits) / (p.B * p.H_kv);
    const int b = bh / p.H_kv, hk = bh - b * p.H_kv;

    // This lane's query rows (column n of the accumulators).  Rows past the last
    // read that one and are not written; a column's values stay its own.
    const Seq seq(p, b, hk);
    // Scores are kept unscaled; the sign of the scale is in the queries.
    const float scale2 = a.scale2;
    bf16x8 qf[RB][STEPS][NT];
    int limit[RB], most = 0, least = INT32_MAX;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = tile * ROWS + kTokRows * rb + n;
        const int rc = min(row, a.rows - 1);
        const int s = rc / a.group, hq = hk * a.group + (rc - s * a.group);
        const T *q = static_cast<const T *>(p.q);
        const T *qr = q + b * p.qs.b + hq * p.qs.h + s * p.qs.s;
        const bool wide = ((reinterpret_cast<uintptr_t>(q) & 15) |
                           ((p.qs.b | p.qs.h | p.qs.s) & 7)) == 0;
#pragma unroll
        for (int st = 0; st < STEPS; ++st)
            q_terms(qr + g * (D / 4) + 8 * st, wide, a.q_factor, qf[rb][st]);
        const bool live = row < a.rows && s < seq.nq;
        limit[rb] = live ? seq.limit(p, s) : 0;
        most = max(most, limit[rb]);
        least = min(least, live ? limit[rb] : INT32_MAX);
    }
    // Keys any row of the tile sees, and keys all of its live rows see.
#pragma unroll
    for (int o = 8; o; o >>= 1) {
        most = max(most, __shfl_xor(most, o));
        least = min(least, __shfl_xor(least, o));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);

    // This workgroup's share of the keys, in steps of 32; its waves take turns.
    const int steps = (most + kTokKeys - 1) / kTokKeys;
    const int per = (steps + a.splits - 1) / a.splits;
    const int first = split * per, end = min(first + per, steps);

    f32x4 o[RB][VB];
    float mx[RB], sum[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int i = 0; i < VB; ++i)
            o[rb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        mx[rb] = -INFINITY;
        sum[rb] = 0.0f;
    }

    auto step = [&](const TokLoads<D> &ld, int t0, auto masked) {
        constexpr bool MASK = decltype(masked)::value;
        // Scores: key 16 h + 4 g + r of query n in sc[rb][4 h + r].
        float sc[RB][8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 acc[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
                acc[rb] = f32x4{0.f, 0.f, 0.f, 0.f};
            const float ksc = scale_of(ld.ks[h]);
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const bf16x8 kf = decode8(ld.kc[h][st], ksc);
#pragma unroll
                for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        acc[rb] = mfma16(kf, qf[rb][st][j], acc[rb]);
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    sc[rb][4 * h + r] = acc[rb][r];
        }
        bf16x8 pf[RB][NT];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int room = limit[rb] - t0 - 4 * g;  // keys 16 h + r below it are seen
            float mt = -INFINITY;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!MASK || 16 * (i >> 2) + (i & 3) < room)
                    mt = fmaxf(mt, sc[rb][i]);
            mt = quad_max(mt);
            // The maximum moves when a row has none yet or is 2^8 behind: until
            // then probabilities stay below 2^8 and nothing is rescaled.
            const bool move =
                mx[rb] == -INFINITY ? mt > mx[rb] : (mt - mx[rb]) * scale2 > kRescaleLog2;
            if (__builtin_amdgcn_ballot_w64(move) != 0) {
                const float mn = move ? mt : mx[rb];
                const float alpha = mx[rb] == mn || mx[rb] == -INFINITY
                                        ? 1.0f
                                        : rebase<NT>(mx[rb], mn, scale2);
                mx[rb] = mn;
                sum[rb] *= alpha;
#pragma unroll
                for (int i = 0; i < VB; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        o[rb][i][r] *= alpha;
            }
            const float mref = max_or_zero(mx[rb]);
            float m2 = mref * scale2;
            const bool far = far_row<NT>(m2);
            if (NT == 1 && __builtin_amdgcn_ballot_w64(far) != 0) {
                const float back = far ? mref : 0.0f;  // the wave's other rows stay as they are
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    float x = sc[rb][i] - back;
                    asm volatile("" : "+v"(x));  // stays behind the branch
                    sc[rb][i] = x;
                }
                m2 = far ? 0.0f : m2;
            }
            float pr[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                pr[i] = __builtin_amdgcn_exp2f(exponent<NT>(sc[rb][i], mref, scale2, m2));
                if (MASK && 16 * (i >> 2) + (i & 3) >= room)
                    pr[i] = 0.0f;
                sum[rb] += pr[i];
            }
            p_terms(pr, pf[rb]);
        }
        float vsc[8];
        unsigned nan = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            unsigned byte = ld.vs[j];
            if (MASK) {
                nan |= byte == unsigned(mx4::kNanScale) ? 1u << j : 0u;
                byte = byte == unsigned(mx4::kNanScale) ? 0u : byte;
            }
            vsc[j] = scale_of(byte);
        }
        // V^T blocks 2c and 2c + 1: dimensions m * VB + 2c and + 2c + 1 of keys j.
#pragma unroll
        for (int c = 0; c < VB / 2; ++c) {
            u32x4 even, odd;
#pragma unroll
            for (int jj = 0; jj < 4; ++jj) {
                const unsigned x0 = decode2_at(ld.vc[2 * jj], vsc[2 * jj], c);
                const unsigned x1 = decode2_at(ld.vc[2 * jj + 1], vsc[2 * jj + 1], c);
                even[jj] = __builtin_amdgcn_perm(x1, x0, 0x05040100);
                odd[jj] = __builtin_amdgcn_perm(x1, x0, 0x07060302);
            }
#pragma unroll
            for (int rb = 0; rb < RB; ++rb)
#pragma unroll
                for (int j = 0; j < NT; ++j) {
                    o[rb][2 * c] =
                        mfma16(__builtin_bit_cast(bf16x8, even), pf[rb][j], o[rb][2 * c]);
                    o[rb][2 * c + 1] =
                        mfma16(__builtin_bit_cast(bf16x8, odd), pf[rb][j], o[rb][2 * c + 1]);
                }
        }
        if (MASK && __builtin_amdgcn_ballot_w64(nan != 0) != 0) {
            // NaN groups of V: to the rows that see their keys.  Lane (m, g')
            // holds the bytes of dimensions m * VB ..; the accumulators of
            // lane (n, g) hold m = 4 g + r.
#pragma unroll
            for (int gg = 0; gg < 4; ++gg)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const unsigned bits = unsigned(__shfl(int(nan), 16 * gg + 4 * g + r));
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) {
                        bool hit = false;
#pragma unroll
                        for (int j = 0; j < 8; ++j)
                            hit = hit || ((bits >> j & 1u) &&
                                          t0 + 16 * (j >> 2) + 4 * gg + (j & 3) < limit[rb]);
                        if (hit)
#pragma unroll
                            for (int i = 0; i < VB; ++i)
                                o[rb][i][r] = NAN;
                    }
                }
        }
    };

    auto load = [&](TokLoads<D> &ld, int i) {
        const int t0 = i * kTokKeys;
        const int64_t at = seq.kv_row + t0;
        if (t0 + kTokKeys <= seq.len)
            ld.template load<false>(p.cache, at, 0, n, g);
        else
            ld.template load<true>(p.cache, at, unsigned(seq.len - 1 - t0), n, g);
    };
    // The next step's codes are on their way while this one's are used.  Steps
    // that every row sees whole come first.
    TokLoads<D> cur, next;
    int i = first + wave;
    if (i < end)
        load(cur, i);
    for (; i < end && (i + 1) * kTokKeys <= least; i += kTokWaves) {
        if (i + kTokWaves < end)
            load(next, i + kTokWaves);
        step(cur, i * kTokKeys, std::false_type{});
        cur = next;
    }
    for (; i < end; i += kTokWaves) {
        if (i + kTokWaves < end)
            load(next, i + kTokWaves);
        step(cur, i * kTokKeys, std::true_type{});
        cur = next;
    }

    // Join the waves.  Lane (n, g) holds O^T rows d = (4 g + r) * VB + i of query n.
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int nr = kTokRows * rb + n;
        sum[rb] += __shfl_xor(sum[rb], 16);
        sum[rb] += __shfl_xor(sum[rb], 32);
#pragma unroll
        for (int r = 0; r < 4; ++r)
#pragma unroll
            for (int i = 0; i < VB; ++i)
                so[wave][nr][(4 * g + r) * VB + i] = o[rb][i][r];
        if (g == 0) {
            sm[wave][nr] = mx[rb];
            sl[wave][nr] = sum[rb];
        }
    }
    __syncthreads();
    constexpr int LANES = kTokWaves * 64 / ROWS;  // threads of a row
    const int jr = tid / LANES, jc = tid % LANES;
    const int jrow = tile * ROWS + jr;
    const int js = jrow / a.group, jh = hk * a.group + (jrow - js * a.group);
    if (jrow >= a.rows || js >= seq.nq)
        return;
    float jm = -INFINITY, jl = 0.0f, w[kTokWaves];
#pragma unroll
    for (int i = 0; i < kTokWaves; ++i)
        jm = fmaxf(jm, sm[i][jr]);
#pragma unroll
    for (int i = 0; i < kTokWaves; ++i) {
        w[i] = sl[i][jr] == 0.0f  ? 0.0f
               : sm[i][jr] == jm ? 1.0f
                                 : rebase<NT>(sm[i][jr], jm, scale2);
        jl += w[i] * sl[i][jr];
    }
    const float inv = jl == 0.0f ? 0.0f : 1.0f / jl;
    const int64_t orow = (int64_t(b) * p.S_q + js) * p.H + jh;
    T *out = static_cast<T *>(p.o) + b * p.os.b + jh * p.os.h + js * p.os.s;
    const int64_t plane = int64_t(p.B) * p.S_q * p.H;
    for (int d = jc; d < D; d += LANES) {
        float v = 0.0f;
#pragma unroll
        for (int i = 0; i < kTokWaves; ++i)
            v += weighed(w[i], so[i][jr][d]);
        v *= inv;
        if (a.splits > 1)
            a.part[(split * plane + orow) * D + d] = v;
        else
            store_o(out + d, v);
    }
    if (a.splits > 1 && jc == 0)
        a.ml[split * plane + orow] = float2{jm, jl};
}

// ------------------------------------------------------------ tile kernel

// 16-byte pieces of a staged K row (D / 8 of them) and V^T row (8), placed so
// that the 16 rows a ds_read_b128 quarter touches lie in distinct banks.
template <int D>
__device__ __forceinline__ int k_piece(int row, int piece)
{
    return D == 128 ? piece ^ (row & 15) : piece ^ ((row & 7) ^ ((row >> 3) & 1));
}
__device__ __forceinline__ int v_piece(int row, int piece)
{
    return piece ^ ((row & 7) ^ ((row >> 3) & 1));
}

template <typename T, int D>
__global__ __launch_bounds__(kTileWaves * 64, 2) void kv4_tile_kernel(AttnArgs a)
{
    constexpr int NT = kTerms<T>;
    constexpr int GROUPS = D / 32;
    constexpr int DB = D / 32;           // V^T blocks of 32 dimensions
    constexpr int KSTEPS = D / 16;       // MFMA steps of a score
    constexpr int KV_EL = kTileKeys * D;  // elements of a staged K or V^T tile
    constexpr int VD = D / 16;           // dimensions of V a thread decodes, of 4 keys
    __shared__ __attribute__((aligned(16))) u16 smem[4 * KV_EL];
    __shared__ int any_nan;  // of the workgroup's V

    const Kv4Attention &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int blk = xcd_major_block();
    const int split = blk % a.splits;
    // Under a causal mask the last query tiles are the longest: they go first.
    const int tile = a.tiles - 1 - (blk / a.splits) % a.tiles;
    const int bh = (blk / a.splits) / a.tiles;
    const int b = bh / p.H_kv, hk = bh - b * p.H_kv;
    const Seq seq(p, b, hk);

    // This lane's query row: column col of the accumulators.  Rows past the
    // last read that one and are not written.
    const int row = tile * kTileRows + wave * 32 + col;
    const int rc = min(row, a.rows - 1);
    const int s = rc / a.group, hq = hk * a.group + (rc - s * a.group);
    const bool live = row < a.rows && s < seq.nq;
    const int limit = live ? seq.limit(p, s) : 0;
    int most = limit, least = live ? limit : INT32_MAX;
#pragma unroll
    for (int o = 16; o; o >>= 1) {
        most = max(most, __shfl_xor(most, o));
        least = min(least, __shfl_xor(least, o));
    }
    most = __builtin_amdgcn_readfirstlane(most);
    least = __builtin_amdgcn_readfirstlane(least);
    // Keys that any row of the workgroup sees: those of its last live row.
    const int s_last = min((min((tile + 1) * kTileRows, a.rows) - 1) / a.group, seq.nq - 1);
    const int wg_most = s_last >= (tile * kTileRows) / a.group ? seq.limit(p, s_last) : 0;
    const int steps = (wg_most + kTileKeys - 1) / kTileKeys;
    const int per = (steps + a.splits - 1) / a.splits;
    const int first = min(split * per, steps), end = min(first + per, steps);

    // Scores are kept unscaled; the sign of the scale is in the queries.
    const float scale2 = a.scale2;
    bf16x8 qf[KSTEPS][NT];
    {
        const T *q = static_cast<const T *>(p.q);
        const T *qr = q + b * p.qs.b + hq * p.qs.h + s * p.qs.s;
        const bool wide = ((reinterpret_cast<uintptr_t>(q) & 15) |
                           ((p.qs.b | p.qs.h | p.qs.s) & 7)) == 0;
#pragma unroll
        for (int ks = 0; ks < KSTEPS; ++ks)
            q_terms(qr + 16 * ks + 8 * half, wide, a.q_factor, qf[ks]);
    }

    // What this thread decodes of a tile: D / 4 codes of one key's K, and V of
    // the four keys 4 va .. 4 va + 3 in VD dimensions.
    const int kt = tid >> 2, kpart = tid & 3;
    const int va = tid & 15, vd = tid >> 4;
    unsigned kc[D / 32], kscale, vc[4], vscale[4];
    auto load = [&](int j) {
        // Keys past the cache's length read its last one again.
        const unsigned over = unsigned(min(seq.len - 1 - j * kTileKeys, kTileKeys - 1));
        const int64_t row = seq.kv_row + int64_t(j) * kTileKeys;
        const uint8_t *kc0 = p.cache.k + row * (D / 2), *ks0 = p.cache.k_scales + row * GROUPS;
        const uint8_t *vc0 = p.cache.v + row * (D / 2), *vs0 = p.cache.v_scales + row * GROUPS;
        {
            const unsigned key = min(unsigned(kt), over);
            const uint8_t *src = kc0 + (key * (D / 2) + kpart * (D / 8));
            if constexpr (D == 128) {
                const u32x4 w = *reinterpret_cast<const u32x4 *>(src);
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    kc[i] = w[i];
            } else {
                const u32x2 w = *reinterpret_cast<const u32x2 *>(src);
                kc[0] = w[0];
                kc[1] = w[1];
            }
            kscale = ks0[key * GROUPS + kpart * GROUPS / 4];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const unsigned key = min(unsigned(4 * va + i), over);
            const uint8_t *src = vc0 + (key * (D / 2) + vd * (D / 32));
            if constexpr (D == 128)
                vc[i] = *reinterpret_cast<const unsigned *>(src);
            else
                vc[i] = *reinterpret_cast<const uint16_t *>(src);
            vscale[i] = vs0[key * GROUPS + vd * GROUPS / 16];
        }
    };
    // Quad va of keys within its row of 64: groups of 16 keys hold their quads
    // in the order 0, 2, 1, 3, so that 16 bytes are the eight keys a lane half
    // holds in its accumulator registers.
    const int vq = va & 3;
    const int vpiece = 2 * (va >> 2) + (vq & 1), vsub = vq >> 1;
    auto store = [&](int stage) {
        unsigned ko = stage * KV_EL + kt * D + k_piece<D>(kt, kpart * (D / 32)) * 8;
        unsigned vo = (2 + stage) * KV_EL + vd * VD * kTileKeys + v_piece(vd * VD, vpiece) * 8 +
                      4 * vsub;
        asm volatile("" : "+v"(ko), "+v"(vo));
        const float ks = scale_of(kscale);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
            *reinterpret_cast<bf16x8 *>(smem + (ko ^ 8 * i)) = decode8(kc[i], ks);
        bool nan = false;
        float vs[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const bool bad = vscale[i] == unsigned(mx4::kNanScale);
            nan = nan || bad;
            vs[i] = scale_of(bad ? 0u : vscale[i]);
        }
#pragma unroll
        for (int c = 0; c < VD / 2; ++c) {
            u32x2 even, odd;
#pragma unroll
            for (int jj = 0; jj < 2; ++jj) {
                const unsigned x0 = decode2_at(vc[2 * jj], vs[2 * jj], c);
                const unsigned x1 = decode2_at(vc[2 * jj + 1], vs[2 * jj + 1], c);
                even[jj] = __builtin_amdgcn_perm(x1, x0, 0x05040100);
                odd[jj] = __builtin_amdgcn_perm(x1, x0, 0x07060302);
            }
            // Rows vd * VD + 2 c and + 1: the swizzle's low bits are the row's.
            *reinterpret_cast<u32x2 *>(smem + 2 * c * kTileKeys + (vo ^ 8 * (2 * c))) = even;
            *reinterpret_cast<u32x2 *>(smem + (2 * c + 1) * kTileKeys + (vo ^ 8 * (2 * c + 1))) =
                odd;
        }
        if (nan)
            any_nan = 1;
    };

    f32x16 o[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r)
            o[i][r] = 0.0f;
    float mx = -INFINITY, sum = 0.0f;

    // Offsets of this lane's K rows and V^T rows, with its half's first piece,
    // in stage 0; other pieces differ in bits that a row's start leaves clear.
    // Recomputed per tile: kept in registers for every piece they would spill.
    const unsigned ko0 = col * D + k_piece<D>(col, half) * 8;
    const unsigned vo0 = 2 * KV_EL + col * kTileKeys + v_piece(col, half) * 8;
    f32x16 sc[2];  // key t0 + 32 kb + acc_row(r, half) in sc[kb][r]
    auto scores = [&](int stage) {
        unsigned ko = ko0 + stage * KV_EL;
        asm volatile("" : "+v"(ko));
#pragma unroll
        for (int kb = 0; kb < 2; ++kb) {
#pragma unroll
            for (int r = 0; r < 16; ++r)
                sc[kb][r] = 0.0f;
            asm volatile("" ::: "memory");
#pragma unroll
            for (int ks = 0; ks < KSTEPS; ++ks) {
                const bf16x8 kf =
                    *reinterpret_cast<const bf16x8 *>(smem + 32 * kb * D + (ko ^ 16 * ks));
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    sc[kb] = mfma_bf16(kf, qf[ks][t], sc[kb]);
            }
        }
    };
    auto softmax_pv = [&](int j, int stage) {
        const int t0 = j * kTileKeys;
        const bool masked = t0 + kTileKeys > least;  // uniform over the wave
        const int room = limit - t0 - 4 * half;
        unsigned vo = vo0 + stage * KV_EL;
        asm volatile("" : "+v"(vo));
        if (masked)
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float x = 32 * kb + 8 * (r >> 2) + (r & 3) < room ? sc[kb][r] : -INFINITY;
                    asm volatile("" : "+v"(x));  // stays behind the branch
                    sc[kb][r] = x;
                }
        float mt = -INFINITY;
#pragma unroll
        for (int kb = 0; kb < 2; ++kb)
#pragma unroll
            for (int r = 0; r < 16; ++r)
                mt = fmaxf(mt, sc[kb][r]);
        mt = row_pair_max(mt);
        // The maximum moves when a row has none yet or is 2^8 behind: until
        // then probabilities stay below 2^8 and nothing is rescaled.
        const bool move = mx == -INFINITY ? mt > mx : (mt - mx) * scale2 > kRescaleLog2;
        if (__builtin_amdgcn_ballot_w64(move) != 0) {
            const float mn = move ? mt : mx;
            const float alpha =
                mx == mn || mx == -INFINITY ? 1.0f : rebase<NT>(mx, mn, scale2);
            mx = mn;
            sum *= alpha;
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    o[i][r] *= alpha;
        }
        const float mref = max_or_zero(mx);
        float m2 = mref * scale2;
        const bool far = far_row<NT>(m2);
        if (NT == 1 && __builtin_amdgcn_ballot_w64(far) != 0) {
            const float back = far ? mref : 0.0f;  // the wave's other rows stay as they are
#pragma unroll
            for (int kb = 0; kb < 2; ++kb)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    float x = sc[kb][r] - back;
                    asm volatile("" : "+v"(x));
                    sc[kb][r] = x;
                }
            m2 = far ? 0.0f : m2;
        }
        // Sixteen keys at a time: the MFMAs of one group run under the
        // exponentials of the next.
#pragma unroll
        for (int kg = 0; kg < 4; ++kg) {
            asm volatile("" ::: "memory");
            bf16x8 vf[DB];
#pragma unroll
            for (int i = 0; i < DB; ++i)
                vf[i] = *reinterpret_cast<const bf16x8 *>(smem + 32 * i * kTileKeys +
                                                          (vo ^ 16 * kg));
            float pr[8];
#pragma unroll
            for (int r = 0; r < 8; ++r)
                pr[r] = __builtin_amdgcn_exp2f(
                    exponent<NT>(sc[kg >> 1][8 * (kg & 1) + r], mref, scale2, m2));
            // Not left to exp2(-inf): the scale may be 0.
            if (masked)
#pragma unroll
                for (int r = 0; r < 8; ++r) {
                    float x = 16 * kg + 8 * (r >> 2) + (r & 3) < room ? pr[r] : 0.0f;
                    asm volatile("" : "+v"(x));
                    pr[r] = x;
                }
            bf16x8 pf[NT];
            p_terms(pr, pf);
            if constexpr (NT == 1)
                sum = row_sum8(pf[0], sum);
            else
#pragma unroll
                for (int r = 0; r < 8; ++r)
                    sum += pr[r];
#pragma unroll
            for (int i = 0; i < DB; ++i)
#pragma unroll
                for (int t = 0; t < NT; ++t)
                    o[i] = mfma_bf16(vf[i], pf[t], o[i]);
        }
    };

    if (tid == 0)
        any_nan = 0;
    __syncthreads();
    if (first < end) {
        load(first);
        store(0);
        if (first + 1 < end)
            load(first + 1);
    }
    __syncthreads();
    for (int j = first; j < end; ++j) {
        const int stage = (j - first) & 1;
        // The next tile is decoded under the scores' MFMAs.
        const bool seen = j * kTileKeys < most;
        if (seen)
            scores(stage);
        if (j + 1 < end) {
            store(stage ^ 1);
            if (j + 2 < end)
                load(j + 2);
        }
        if (seen) {
            __builtin_amdgcn_s_setprio(1);
            softmax_pv(j, stage);
            __builtin_amdgcn_s_setprio(0);
        }
        __syncthreads();
    }

    // NaN groups of V, decoded as zero: to the rows that see their keys.
    if (any_nan)
        for (int t = first * kTileKeys; t < min(end * kTileKeys, seq.len); ++t)
#pragma unroll
            for (int i = 0; i < DB; ++i)
                if (p.cache.v_scales[(seq.kv_row + t) * GROUPS + i] == mx4::kNanScale && t < limit)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        o[i][r] = NAN;

    // Row sums over the two halves; then O^T through the stages' LDS (every
    // wave has left them), so that rows go out whole: f32 rows of D / 4 pieces
    // of 16 bytes, placed by their row's low bits against bank conflicts.
    sum += __shfl_xor(sum, 32);
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    float *so = reinterpret_cast<float *>(smem) + wave * 32 * D;
    constexpr int PIECES = D / 4;
#pragma unroll
    for (int i = 0; i < DB; ++i)
#pragma unroll
        for (int r = 0; r < 16; r += 4)
            *reinterpret_cast<f32x4 *>(so + col * D +
                                       ((8 * i + acc_row(r, half) / 4) ^ (col & 15)) * 4) =
                f32x4{o[i][r] * inv, o[i][r + 1] * inv, o[i][r + 2] * inv, o[i][r + 3] * inv};
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    const bool parts = a.splits > 1;
    const int64_t plane = int64_t(p.B) * p.S_q * p.H;
    const int64_t prow = split * plane + (int64_t(b) * p.S_q + s) * p.H + hq;
    if (parts && live && half == 0)
        a.ml[prow] = float2{mx, sum};
    // Where this lane's row starts (elements), for the lanes that write it.
    const int64_t at = !live   ? -1
                       : parts ? prow * D
                               : b * p.os.b + hq * p.os.h + s * p.os.s;
    const bool wide_o = ((reinterpret_cast<uintptr_t>(p.o) & 15) |
                         ((p.os.b | p.os.h | p.os.s) & 7)) == 0;
    if (parts || NT == 3) {
        float *dst = parts ? a.part : static_cast<float *>(p.o);
#pragma unroll
        for (int i = 0; i < PIECES / 2; ++i) {
            const int f = i * 64 + lane, r = f / PIECES, piece = f % PIECES;
            const int64_t off = __shfl(at, r);
            const f32x4 v = *reinterpret_cast<const f32x4 *>(so + r * D + (piece ^ (r & 15)) * 4);
            if (off < 0)
                continue;
            if (parts || wide_o)
                *reinterpret_cast<f32x4 *>(dst + off + 4 * piece) = v;
            else
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    dst[off + 4 * piece + e] = v[e];
        }
    } else {
        u16 *dst = static_cast<u16 *>(p.o);
#pragma unroll
        for (int i = 0; i < PIECES / 4; ++i) {
            const int f = i * 64 + lane, r = f / (PIECES / 2), piece = f % (PIECES / 2) * 2;
            const int64_t off = __shfl(at, r);
            const float *src = so + r * D;
            const f32x4 v0 = *reinterpret_cast<const f32x4 *>(src + (piece ^ (r & 15)) * 4);
            const f32x4 v1 = *reinterpret_cast<const f32x4 *>(src + ((piece + 1) ^ (r & 15)) * 4);
            if (off < 0)
                continue;
            const float v[8] = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
            if (wide_o) {
                bf16x8 t[1];
                p_terms(v, t);
                *reinterpret_cast<bf16x8 *>(dst + off + 4 * piece) = t[0];
            } else
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    store_o(dst + off + 4 * piece + e, v[e]);
        }
    }
}

// O = sum_s w_s P_s / sum_s w_s, w_s = l_s rebase(m_s, max m), over the splits (at most
// 64); one of which no key was seen has l_s = 0.  PER waves per row: in each, lane s
// weighs split s; wave w adds the splits w, w + PER, .., at most 16, its loads all in
// flight, D / 64 dimensions per lane, and the waves' sums are added in their order.
template <typename T, int D, int PER>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttnArgs a)
{
    constexpr int E = D / 64;
    const Kv4Attention &p = a.p;
    const int64_t plane = int64_t(p.B) * p.S_q * p.H;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const unsigned row = blockIdx.x * unsigned(4 / PER) + unsigned(PER == 4 ? 0 : wave);
    const int first = PER == 4 ? wave : 0;
    if (row >= unsigned(plane))
        return;  // whole wave; with PER == 4 no workgroup
    const unsigned bs = row / unsigned(p.H), b = bs / unsigned(p.S_q);
    const int h = int(row - bs * unsigned(p.H)), s = int(bs - b * unsigned(p.S_q));
    if (p.counts && s >= p.counts[b])
        return;  // likewise
    const float *src = a.part + int64_t(row) * D + lane * E;
    float x[kAttnMaxSplits / 4][E], v[E] = {};
#pragma unroll
    for (int k = 0; k < kAttnMaxSplits / 4; ++k)
        if (first + PER * k < a.splits)
#pragma unroll
            for (int e = 0; e < E; ++e)
                x[k][e] = src[(first + PER * k) * plane * D + e];
    const float2 ml = lane < a.splits ? a.ml[lane * plane + row] : float2{-INFINITY, 0.0f};
    float m = ml.y == 0.0f ? -INFINITY : ml.x;
#pragma unroll
    for (int o = 32; o; o >>= 1)
        m = fmaxf(m, __shfl_xor(m, o));
    // A split of which no key was seen weighs nothing, whatever its maximum.
    const float w =
        ml.y == 0.0f
            ? 0.0f
            : (ml.x == m ? 1.0f : rebase<kTerms<T>>(ml.x, m, a.scale2)) * ml.y;
    float l = w;
#pragma unroll
    for (int o = 32; o; o >>= 1)
        l += __shfl_xor(l, o);
#pragma unroll
    for (int k = 0; k < kAttnMaxSplits / 4; ++k)
        if (first + PER * k < a.splits) {
            const float wk = __shfl(w, first + PER * k);
#pragma unroll
            for (int e = 0; e < E; ++e)
                v[e] += weighed(wk, x[k][e]);
        }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    T *out = static_cast<T *>(p.o) + b * p.os.b + h * p.os.h + s * p.os.s;
    if constexpr (PER == 1) {
#pragma unroll
        for (int e = 0; e < E; ++e)
            store_o(out + lane * E + e, v[e] * inv);
    } else {
        __shared__ float part[4][D];
#pragma unroll
        for (int e = 0; e < E; ++e)
            part[wave][lane * E + e] = v[e];
        __syncthreads();
        const int d = threadIdx.x;
        if (d < D)
            store_o(out + d, (part[0][d] + part[1][d] + part[2][d] + part[3][d]) * inv);
    }
}

int64_t part_bytes(int B, int S_q, int H, int D, int splits)
{
    return int64_t(B) * S_q * H * splits * (int64_t(D) * 4 + 8);
}

template <typename T, int D>
bool run_attention_kv4(AttnArgs &a, const AttnPlan &pl, hipStream_t st)
{
    const int64_t blocks = int64_t(a.p.B) * a.p.H_kv * a.tiles * a.splits;
    const int64_t rows = int64_t(a.p.B) * a.p.S_q * a.p.H;
    if (!launch_fits(blocks, 256) || !launch_fits(a.splits > 1 ? rows : 0, 256))
        return fail("kv4_attention_dev: too many query rows for one launch");
    const dim3 grid{unsigned(blocks)};
    if (pl.tile)
        hipLaunchKernelGGL((kv4_tile_kernel<T, D>), grid, dim3(kTileWaves * 64), 0, st, a);
    else if (pl.row_blocks == 1)
        hipLaunchKernelGGL((kv4_token_kernel<T, D, 1>), grid, dim3(kTokWaves * 64), 0, st, a);
    else if constexpr (two_row_blocks(kTerms<T> == 3, D))
        hipLaunchKernelGGL((kv4_token_kernel<T, D, 2>), grid, dim3(kTokWaves * 64), 0, st, a);
    if (!hip_ok(hipGetLastError(), "kv4 attention launch"))
        return false;
    if (a.splits == 1)
        return true;
    // A workgroup per row where rows are few: 16 rows of 16 splits 10.9 us in all
    // against 11.4, 32000 rows of 2 splits 76 against 45.
    if (a.splits > kAttnMaxSplits / 4 || rows <= 1024)
        hipLaunchKernelGGL((kv4_join_kernel<T, D, 4>), dim3(unsigned(rows)), dim3(256), 0, st, a);
    else
        hipLaunchKernelGGL((kv4_join_kernel<T, D, 1>), dim3(unsigned((rows + 3) / 4)), dim3(256),
                           0, st, a);
    return hip_ok(hipGetLastError(), "kv4_join_kernel launch");
}

}  // namespace

size_t kv4_attention_scratch_bytes(int B, int S_q, int H, int H_kv, int D, int S_max, Mx4Type type)
{
    if (B <= 0 || S_q <= 0 || H <= 0 || H_kv <= 0 || D <= 0 || S_max <= 0 || H % H_kv)
        return 0;
    // With a causal mask or without.
    const int splits = std::max(attn_plan(B, S_q, H, H_kv, D, S_max, type == kMx4F32, true).splits,
                                attn_plan(B, S_q, H, H_kv, D, S_max, type == kMx4F32, false).splits);
    return splits > 1 ? size_t(part_bytes(B, S_q, H, D, splits)) : 0;
}

bool launch_kv4_attention(const Kv4Attention &p, void *scratch, size_t scratch_bytes,
                          hipStream_t st)
{
    if (p.B <= 0 || p.S_q <= 0 || p.H <= 0)
        return true;
    const AttnPlan pl = attn_plan(p.B, p.S_q, p.H, p.H_kv, p.D, p.S_max, p.type == kMx4F32,
                                  p.causal);
    AttnArgs a{};
    a.p = p;
    a.scale2 = std::fabs(p.scale * kLog2e);
    a.q_factor = p.scale < 0.0f ? -1.0f : 1.0f;
    // f32 queries' exponents take the distance of two scores.  One past f32's range is a
    // weight of 0 under scales from 2^9 / 2^128 on, but not under smaller ones or 0: part of
    // those goes into the queries, whose bits lost by it count for less than 2^-50.
    if (p.type == kMx4F32 && a.scale2 < 0x1p-119f) {
        a.scale2 *= 0x1p64f;
        a.q_factor *= 0x1p-64f;
    }
    a.group = p.H / p.H_kv;
    a.rows = p.S_q * a.group;
    a.tiles = pl.tiles;
    a.splits = pl.splits;
    const size_t need = kv4_attention_scratch_bytes(p.B, p.S_q, p.H, p.H_kv, p.D, p.S_max, p.type);
    if (need > 0) {
        if (!scratch || scratch_bytes < need)
            return fail(
                "kv4_attention_dev: scratch smaller than anima_hip_kv4_attention_scratch_bytes");
        if (!aligned(scratch, 16))
            return fail("kv4_attention_dev: scratch must be 16-byte aligned");
    }
    if (pl.splits > 1) {
        a.part = static_cast<float *>(scratch);
        a.ml = reinterpret_cast<float2 *>(a.part + int64_t(p.B) * p.S_q * p.H * pl.splits * p.D);
    }
    if (p.type == kMx4F32)
        return p.D == 128 ? run_attention_kv4<float, 128>(a, pl, st)
                          : run_attention_kv4<float, 64>(a, pl, st);
    return p.D == 128 ? run_attention_kv4<uint16_t, 128>(a, pl, st)
                      : run_attention_kv4<uint16_t, 64>(a, pl, st);
}

}  // namespace anima_hip
