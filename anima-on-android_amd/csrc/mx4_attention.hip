// Attention over a 4-bit K/V cache (mx4.h rows): O = softmax(scale Q K^T) V
// with K and V decoded to bf16 in registers, where they are exact, and f32
// scores, softmax statistics and sums.
//
// A K/V head serves H / H_kv query heads; its query rows are numbered
// r = s * (H / H_kv) + (head within the group), so that neighbouring rows see
// nearly the same keys under a causal mask.  S^T = K Q^T and O^T = V^T P^T are
// computed, so that a query row is one column of every accumulator.  bf16
// queries enter as they are and P as one bf16 term; f32 queries and their P
// enter as three terms each (mx4::terms2), so products are exact to f32.
//
// 16 query rows per wave on v_mfma_f32_16x16x32_bf16, the waves of a workgroup
// and the workgroups of a split sharing the keys.  Bound by the one pass over
// the cache (17/16 byte per key and dimension for K and V together), or by
// latency where the cache is short.  Codes go from memory to registers to the
// MFMA and nothing is staged in LDS: a lane's 16 bytes of a K row are one
// scale group (the MFMA's k index runs over d in the order the lanes hold it),
// and V^T fragments are pairs of V rows transposed by two byte permutes per
// two codes.
//
// A masked key never reaches a row: its score is left out of the maximum and
// the sum, and the decoded V of keys past the cache's length is finite.  Inside
// the length a V group may be NaN (scale byte 255) while some rows may not see
// its key: such groups are decoded as zero and their NaN is added to the rows
// that do see them.
#include "mx4.h"

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

template <typename T>
constexpr int kTerms = sizeof(T) == 4 ? 3 : 1;

__device__ __forceinline__ void store_o(float *o, float v) { *o = v; }
__device__ __forceinline__ void store_o(uint16_t *o, float v)
{
    const __bf16 b = static_cast<__bf16>(v);
    *o = __builtin_bit_cast(uint16_t, b);
}

struct AttnArgs {
    Kv4Attention p;
    float scale2;   // softmax scale * log2(e)
    int group;      // H / H_kv
    int rows;       // S_q * group
    int tiles;      // query tiles of a K/V head
    int splits;
    float *part;    // [splits][B * S_q * H][D] O of each split, normalised
    float2 *ml;     // [splits][B * S_q * H] (max in log2 units, sum); sum 0: no key seen
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

// A query row's eight values from d as bf16 terms.
__device__ __forceinline__ void q_terms(const uint16_t *q, bool wide, bf16x8 (&t)[1])
{
    u32x4 u;
    if (wide)
        u = *reinterpret_cast<const u32x4 *>(q);
    else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
            u[i] = unsigned(q[2 * i]) | unsigned(q[2 * i + 1]) << 16;
    }
    t[0] = __builtin_bit_cast(bf16x8, u);
}

__device__ __forceinline__ void q_terms(const float *q, bool, bf16x8 (&t)[3])
{
    u32x4 u[3];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        unsigned w[3];
        terms2<3>(q[2 * i], q[2 * i + 1], w);
#pragma unroll
        for (int j = 0; j < 3; ++j)
            u[j][i] = w[j];
    }
#pragma unroll
    for (int j = 0; j < 3; ++j)
        t[j] = __builtin_bit_cast(bf16x8, u[j]);
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
    q_terms(p, true, t);
}

// ----------------------------------------------------------- token kernel

constexpr int kTokRows = 16;   // query rows of a workgroup
constexpr int kTokKeys = 32;   // keys a wave takes at a time
constexpr int kTokWaves = 4;

// A wave's loads for 32 keys.  Lane (m, g): K rows t0 + m and t0 + 16 + m,
// dimensions g * D/4 .. ; V rows of the eight keys 4g + 0..3 and 16 + 4g +
// 0..3, dimensions m * D/16 .. .
template <int D>
struct TokLoads {
    static constexpr int GROUPS = D / 32;
    static constexpr int KW = D / 32;  // words of K codes per key and lane: D/4 codes
    unsigned kc[2][KW];
    unsigned ks[2];
    unsigned vc[8];
    unsigned vs[8];

    template <bool TAIL>
    __device__ __forceinline__ void load(const Kv4Cache &c, int64_t row0, int t0, int last, int m,
                                         int g)
    {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int t = TAIL ? min(t0 + 16 * h + m, last) : t0 + 16 * h + m;
            const int64_t row = row0 + t;
            const uint8_t *src = c.k + row * (D / 2) + g * (D / 8);
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
            ks[h] = c.k_scales[row * GROUPS + g * GROUPS / 4];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const int key = 16 * (j >> 2) + 4 * g + (j & 3);
            const int t = TAIL ? min(t0 + key, last) : t0 + key;
            const int64_t row = row0 + t;
            const uint8_t *src = c.v + row * (D / 2) + m * (D / 32);
            if constexpr (D == 128)
                vc[j] = *reinterpret_cast<const unsigned *>(src);
            else
                vc[j] = *reinterpret_cast<const uint16_t *>(src);
            vs[j] = c.v_scales[row * GROUPS + m * GROUPS / 16];
        }
    }
};

template <typename T, int D>
__global__ __launch_bounds__(kTokWaves * 64) void kv4_token_kernel(AttnArgs a)
{
    constexpr int NT = kTerms<T>;
    constexpr int STEPS = D / 32;  // MFMA steps of a score; V^T blocks of 16 are D / 16
    constexpr int VB = D / 16;
    constexpr int OPITCH = D + 4;
    __shared__ __attribute__((aligned(16))) float so[kTokWaves][kTokRows][OPITCH];
    __shared__ float sm[kTokWaves][kTokRows], sl[kTokWaves][kTokRows];

    const Kv4Attention &p = a.p;
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15, g = lane >> 4;
    const int blk = xcd_major_block();
    const int split = blk % a.splits;
    const int tile = (blk / a.splits) % a.tiles;
    const int bh = (blk / a.splits) / a.tiles;
    const int b = bh / p.H_kv, hk = bh - b * p.H_kv;
    const Seq seq(p, b, hk);

    // This lane's query row (column n of the accumulators).
    const int row = tile * kTokRows + n;
    const int s = row / a.group, hq = hk * a.group + (row - s * a.group);
    const bool live = row < a.rows && s < seq.nq;
    const int limit = live ? seq.limit(p, s) : 0;
    // Keys any row of the tile sees, and keys all of its live rows see.
    int most = limit, least = live ? limit : INT32_MAX;
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

    bf16x8 qf[STEPS][NT];
    {
        const T *q = static_cast<const T *>(p.q);
        const bool ok = live && limit > 0;
        const T *qr = ok ? q + b * p.qs.b + hq * p.qs.h + s * p.qs.s : nullptr;
        const bool wide = ((reinterpret_cast<uintptr_t>(q) & 15) |
                           ((p.qs.b | p.qs.h | p.qs.s) & 7)) == 0;
#pragma unroll
        for (int st = 0; st < STEPS; ++st) {
            if (ok)
                q_terms(qr + g * (D / 4) + 8 * st, wide, qf[st]);
            else
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    qf[st][j] = __builtin_bit_cast(bf16x8, u32x4{0, 0, 0, 0});
        }
    }

    f32x4 o[VB];
#pragma unroll
    for (int i = 0; i < VB; ++i)
        o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float mx = -INFINITY, sum = 0.0f;

    auto step = [&](const TokLoads<D> &ld, int t0, auto masked) {
        constexpr bool MASK = decltype(masked)::value;
        // Scores: key 16 h + 4 g + r of query n in sc[4 h + r].
        float sc[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            f32x4 acc = {0.f, 0.f, 0.f, 0.f};
            const float ksc = scale_of(ld.ks[h]);
#pragma unroll
            for (int st = 0; st < STEPS; ++st) {
                const bf16x8 kf = decode8(ld.kc[h][st], ksc);
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc = mfma16(kf, qf[st][j], acc);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r)
                sc[4 * h + r] = acc[r] * a.scale2;
        }
        float mt = -INFINITY;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (!MASK || t0 + 16 * (i >> 2) + 4 * g + (i & 3) < limit)
                mt = fmaxf(mt, sc[i]);
        }
        mt = fmaxf(mt, __shfl_xor(mt, 16));
        mt = fmaxf(mt, __shfl_xor(mt, 32));
        const float mn = fmaxf(mx, mt);
        // No key seen yet (or all scores -inf): nothing to rescale.
        const float alpha = mx == mn ? 1.0f : __builtin_amdgcn_exp2f(mx - mn);
        mx = mn;
        float pr[8], ps = 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const bool seen = !MASK || t0 + 16 * (i >> 2) + 4 * g + (i & 3) < limit;
            pr[i] = seen ? __builtin_amdgcn_exp2f(sc[i] - mn) : 0.0f;
            ps += pr[i];
        }
        sum = sum * alpha + ps;
        bf16x8 pf[NT];
        p_terms(pr, pf);
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
#pragma unroll
        for (int i = 0; i < VB; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                o[i][r] *= alpha;
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
            for (int j = 0; j < NT; ++j) {
                o[2 * c] = mfma16(__builtin_bit_cast(bf16x8, even), pf[j], o[2 * c]);
                o[2 * c + 1] = mfma16(__builtin_bit_cast(bf16x8, odd), pf[j], o[2 * c + 1]);
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
                    bool hit = false;
#pragma unroll
                    for (int j = 0; j < 8; ++j)
                        hit = hit || ((bits >> j & 1u) &&
                                      t0 + 16 * (j >> 2) + 4 * gg + (j & 3) < limit);
                    if (hit)
#pragma unroll
                        for (int i = 0; i < VB; ++i)
                            o[i][r] = NAN;
                }
        }
    };

    const int last = max(seq.len - 1, 0);
    for (int i = first + wave; i < end; i += kTokWaves) {
        const int t0 = i * kTokKeys;
        TokLoads<D> ld;
        if (t0 + kTokKeys <= least) {
            ld.template load<false>(p.cache, seq.kv_row, t0, last, n, g);
            step(ld, t0, std::false_type{});
        } else {
            ld.template load<true>(p.cache, seq.kv_row, t0, last, n, g);
            step(ld, t0, std::true_type{});
        }
    }

    // Join the waves.  Lane (n, g) holds O^T rows d = (4 g + r) * VB + i of query n.
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int i = 0; i < VB; ++i)
            so[wave][n][(4 * g + r) * VB + i] = o[i][r];
    if (g == 0) {
        sm[wave][n] = mx;
        sl[wave][n] = sum;
    }
    __syncthreads();
    constexpr int LANES = kTokWaves * 64 / kTokRows;  // threads of a row
    const int jr = tid / LANES, jc = tid % LANES;
    const int jrow = tile * kTokRows + jr;
    const int js = jrow / a.group, jh = hk * a.group + (jrow - js * a.group);
    if (jrow >= a.rows || js >= seq.nq)
        return;
    float jm = -INFINITY, jl = 0.0f, w[kTokWaves];
#pragma unroll
    for (int i = 0; i < kTokWaves; ++i)
        jm = fmaxf(jm, sm[i][jr]);
#pragma unroll
    for (int i = 0; i < kTokWaves; ++i) {
        w[i] = sl[i][jr] == 0.0f ? 0.0f : sm[i][jr] == jm ? 1.0f : __builtin_amdgcn_exp2f(sm[i][jr] - jm);
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
            if (w[i] != 0.0f)
                v += w[i] * so[i][jr][d];
        v *= inv;
        if (a.splits > 1)
            a.part[(split * plane + orow) * D + d] = v;
        else
            store_o(out + d, v);
    }
    if (a.splits > 1 && jc == 0)
        a.ml[split * plane + orow] = float2{jm, jl};
}

// O = sum_s w_s P_s / sum_s w_s, w_s = l_s 2^(m_s - max m), over the splits
// that saw a key.
template <typename T>
__global__ __launch_bounds__(256) void kv4_join_kernel(AttnArgs a)
{
    const Kv4Attention &p = a.p;
    const int64_t plane = int64_t(p.B) * p.S_q * p.H;
    const int64_t i = int64_t(blockIdx.x) * 256 + threadIdx.x;
    const int64_t row = i / p.D;
    if (row >= plane)
        return;
    const int d = int(i - row * p.D);
    const int h = int(row % p.H);
    const int64_t bs = row / p.H;
    const int b = int(bs / p.S_q), s = int(bs % p.S_q);
    if (p.counts && s >= p.counts[b])
        return;
    float m = -INFINITY;
    for (int k = 0; k < a.splits; ++k)
        m = fmaxf(m, a.ml[k * plane + row].x);
    float l = 0.0f, v = 0.0f;
    for (int k = 0; k < a.splits; ++k) {
        const float2 ml = a.ml[k * plane + row];
        if (ml.y == 0.0f)
            continue;
        const float w = (ml.x == m ? 1.0f : __builtin_amdgcn_exp2f(ml.x - m)) * ml.y;
        l += w;
        v += w * a.part[(k * plane + row) * p.D + d];
    }
    store_o(static_cast<T *>(p.o) + b * p.os.b + h * p.os.h + s * p.os.s + d,
            l == 0.0f ? 0.0f : v / l);
}

struct Plan {
    int tiles, splits;
};

Plan plan_of(int B, int S_q, int H, int H_kv, int S_max)
{
    const int64_t rows = int64_t(S_q) * (H / H_kv);
    Plan pl;
    pl.tiles = int((rows + kTokRows - 1) / kTokRows);
    const int64_t groups = std::max<int64_t>(1, int64_t(B) * H_kv * pl.tiles);
    // A workgroup's waves take 32 keys each at a time; splits until the grid
    // has about four workgroups per CU or a share is one round.
    const int64_t rounds = (int64_t(S_max) + kTokKeys * kTokWaves - 1) / (kTokKeys * kTokWaves);
    pl.splits = int(std::max<int64_t>(1, std::min<int64_t>({1024 / groups, rounds, 64})));
    return pl;
}

int64_t part_bytes(int B, int S_q, int H, int D, int splits)
{
    return int64_t(B) * S_q * H * splits * (int64_t(D) * 4 + 8);
}

template <typename T, int D>
bool run_attention_kv4(AttnArgs &a, hipStream_t st)
{
    const int64_t blocks = int64_t(a.p.B) * a.p.H_kv * a.tiles * a.splits;
    const int64_t elems = int64_t(a.p.B) * a.p.S_q * a.p.H * D;
    if (blocks > INT32_MAX || (elems + 255) / 256 > INT32_MAX)
        return fail("kv4_attention_dev: too many query rows");
    hipLaunchKernelGGL((kv4_token_kernel<T, D>), dim3(unsigned(blocks)), dim3(kTokWaves * 64), 0,
                       st, a);
    if (!hip_ok(hipGetLastError(), "kv4_token_kernel launch"))
        return false;
    if (a.splits == 1)
        return true;
    hipLaunchKernelGGL(kv4_join_kernel<T>, dim3(unsigned((elems + 255) / 256)), dim3(256), 0, st,
                       a);
    return hip_ok(hipGetLastError(), "kv4_join_kernel launch");
}

}  // namespace

size_t kv4_attention_scratch_bytes(int B, int S_q, int H, int H_kv, int D, int S_max, Mx4Type)
{
    if (B <= 0 || S_q <= 0 || H <= 0 || H_kv <= 0 || D <= 0 || S_max <= 0 || H % H_kv)
        return 0;
    const Plan pl = plan_of(B, S_q, H, H_kv, S_max);
    return pl.splits > 1 ? size_t(part_bytes(B, S_q, H, D, pl.splits)) : 0;
}

bool launch_kv4_attention(const Kv4Attention &p, void *scratch, size_t scratch_bytes,
                          hipStream_t st)
{
    if (p.B <= 0 || p.S_q <= 0 || p.H <= 0)
        return true;
    const Plan pl = plan_of(p.B, p.S_q, p.H, p.H_kv, p.S_max);
    AttnArgs a{};
    a.p = p;
    a.scale2 = p.scale * kLog2e;
    a.group = p.H / p.H_kv;
    a.rows = p.S_q * a.group;
    a.tiles = pl.tiles;
    a.splits = pl.splits;
    if (pl.splits > 1) {
        if (!scratch ||
            scratch_bytes < kv4_attention_scratch_bytes(p.B, p.S_q, p.H, p.H_kv, p.D, p.S_max,
                                                        p.type))
            return fail(
                "kv4_attention_dev: scratch smaller than anima_hip_kv4_attention_scratch_bytes");
        if (!aligned(scratch, 16))
            return fail("kv4_attention_dev: scratch must be 16-byte aligned");
        a.part = static_cast<float *>(scratch);
        a.ml = reinterpret_cast<float2 *>(a.part + int64_t(p.B) * p.S_q * p.H * pl.splits * p.D);
    }
    if (p.type == kMx4F32)
        return p.D == 128 ? run_attention_kv4<float, 128>(a, st)
                          : run_attention_kv4<float, 64>(a, st);
    return p.D == 128 ? run_attention_kv4<uint16_t, 128>(a, st)
                      : run_attention_kv4<uint16_t, 64>(a, st);
}

}  // namespace anima_hip
