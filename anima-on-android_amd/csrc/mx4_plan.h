// Launch plans of the 4-bit operators: which kernel, tile and split a call of
// given sizes takes, by predicted time.  Host code without HIP.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <iterator>

namespace anima_hip {
namespace mx4_plan {

// The runtime counts the threads of a launch in 32 bits.
inline bool launch_fits(int64_t blocks, int threads) { return blocks <= UINT32_MAX / threads; }

// ------------------------------------------------- linear (mx4_linear.hip)

constexpr int kFewRows = 16;  // most rows of A of the few-rows kernel
constexpr int kTileK = 64;    // K elements per chunk of the plain tiles: 128-byte rows of bf16
constexpr int kLinMaxSplits = 16;
constexpr int kStagedMaxK = 1 << 22;  // row offsets within a staged tile are 32-bit bytes

struct TileShape {
    int bm, bn;
    // Microseconds of a workgroup per chunk of K (256 bytes of a row of A) where half
    // the CUs have one, and where all have (large tiles: at a lower clock; small
    // ones: several workgroups on a CU, per workgroup).
    double half_us, full_us;
    bool pairs = false;  // two chunks at once where K has an even number of them
};
// Fitted, with the constants of the model below, to the times of 900 products, M from
// 17 to 8192, N from 256 to 16384, K from 256 to 11008; on 400 others the choice is
// 0.6 % behind the fastest shape and split on average, 9 % in the worst twentieth.
constexpr TileShape kBf16Shapes[] = {{192, 256, 2.04, 2.31},      {128, 256, 1.4, 1.7},
                                     {128, 128, 1.03, 1.25},      {64, 128, 0.69, 0.77, true},
                                     {64, 64, 0.42, 0.52, true},  {32, 64, 0.33, 0.34, true}};
constexpr TileShape kF32Shapes[] = {{256, 256, 4.32, 5.12}, {128, 256, 2.61, 2.76},
                                    {64, 128, 0.92, 0.98, true}, {32, 64, 0.39, 0.32, true}};
constexpr TileShape kTileShapes[] = {{32, 128, 0, 0}, {64, 128, 0, 0}, {128, 128, 0, 0}};
enum LinKernel { kFew, kTiles, kStaged };
struct LinPlan {
    LinKernel kernel = kFew;
    bool pad = false;  // staged, on copies of the operands with K padded to 128
    bool pairs = false;  // staged, two chunks at once
    int shape = 0;
    int tiles_m = 0, tiles_n = 0, splits = 1, per_split = 0, chunks = 0;
};

// The tile grid of a shape with K shared out over up to `splits` workgroups.
inline void set_grid(LinPlan &pl, const TileShape &t, int M, int N, int splits)
{
    pl.tiles_m = (M + t.bm - 1) / t.bm;
    pl.tiles_n = (N + t.bn - 1) / t.bn;
    pl.per_split = (pl.chunks + splits - 1) / splits;
    pl.pairs = t.pairs && pl.chunks % 2 == 0;
    if (pl.pairs)
        pl.per_split += pl.per_split & 1;
    pl.splits = pl.per_split ? (pl.chunks + pl.per_split - 1) / pl.per_split : 1;
}

// Predicted time of a staged grid: 4 us of latency and epilogue, the chunks of the
// fullest CU, and the sum of the planes.
inline double staged_us(const LinPlan &pl, const TileShape &t, int M, int N)
{
    const double wgs = double(pl.tiles_m) * pl.tiles_n * pl.splits;
    const double rounds = std::ceil(wgs / 256);
    const double load = std::min(1.0, std::max(0.0, wgs / 128 - 1));
    const double alone = t.half_us + (t.full_us > t.half_us ? (t.full_us - t.half_us) * load : 0);
    double us = 4.2 + pl.per_split * (rounds > 1 ? std::max(alone, rounds * t.full_us) : alone);
    if (pl.splits > 1)
        us += 1.9 + double(pl.splits) * M * N * 4 / 2e6;
    return us;
}

inline int lin_padded(int K) { return (K + 127) & ~127; }

// The staged shape and split of least predicted time, K a multiple of 128.
inline LinPlan staged_plan(int M, int N, int K, bool f32)
{
    const TileShape *shapes = f32 ? kF32Shapes : kBf16Shapes;
    const int n = f32 ? int(std::size(kF32Shapes)) : int(std::size(kBf16Shapes));
    LinPlan pl, best;
    pl.kernel = kStaged;
    pl.chunks = K / (f32 ? 64 : 128);
    double best_us = 1e300;
    for (pl.shape = 0; pl.shape < n; ++pl.shape)
        for (int splits = 1; splits <= 8; splits *= 2) {
            if (splits > 1 && (splits > pl.chunks || double(M) * N * splits > 1.6e7))
                break;
            set_grid(pl, shapes[pl.shape], M, N, splits);
            const double us = staged_us(pl, shapes[pl.shape], M, N);
            if (us < best_us) {
                best_us = us;
                best = pl;
            }
        }
    return best;
}

// `staged`: the rows of A suit the staged kernel (16-byte aligned, offsets in 32 bits).
inline LinPlan lin_plan(int M, int N, int K, bool f32, bool staged)
{
    LinPlan pl;
    // Few rows, unless their terms take long to stage in every workgroup.  Time by the
    // few-rows kernel over that by staged tiles, by the staged terms of a workgroup
    // (rows x terms x K): bf16 0.7 at 22000, 0.95 at 88000, 1.3 at 131000; f32 at 3 to 8
    // rows 0.6 to 0.8 at 49000, 0.9 at 132000, 1.1 at 197000, at 12 rows 0.8 at 51000,
    // 1.0 at 74000, 1.2 at 147000, at 16 rows 0.7 at 25000, 1.1 at 49000, 2 at 264000.
    // The limits are for K a multiple of 128: other K stay here at any size (f32, 16 rows,
    // N 2048: 39.8 us at K = 8200, where 8192 takes 13.5 by staged tiles).
    const int64_t limit = !f32 ? 90000 : M <= 8 ? 150000 : M <= 12 ? 100000 : 40000;
    if (M <= kFewRows && (!staged || K % 128 || int64_t(M) * (f32 ? 3 : 1) * K <= limit))
        return pl;
    if (K > 0 && K % 128 == 0 && K <= kStagedMaxK && staged)
        return staged_plan(M, N, K, f32);
    // Other K: copies padded to a multiple of 128 where the product is worth their
    // launch (333 x 2000 x 1500 bf16: 29.8 us on plain tiles, 15.4 with the copies;
    // 30 x 5000 x 700: 12.1 and 10.3).
    if (K % 128 && K <= kStagedMaxK && double(M) * N * K > 6e7) {
        pl = staged_plan(M, N, lin_padded(K), f32);
        pl.pad = true;
        return pl;
    }
    pl.kernel = kTiles;
    pl.shape = M <= 32 ? 0 : M <= 64 ? 1 : 2;
    pl.chunks = (K + kTileK - 1) / kTileK;
    const TileShape &t = kTileShapes[pl.shape];
    set_grid(pl, t, M, N, 1);
    const int64_t tiles = int64_t(pl.tiles_m) * pl.tiles_n;
    const int64_t splits = std::min<int64_t>({256 / tiles, pl.chunks / 4, kLinMaxSplits});
    if (splits > 1)
        set_grid(pl, t, M, N, int(splits));
    return pl;
}

// Scratch: the padded copies of A, the codes and the scales, then the planes of a
// split, each part 256-byte aligned.
struct LinScratch {
    int64_t a = 0, codes = 0, scales = 0, planes = 0, bytes = 0;
};
inline LinScratch lin_scratch(const LinPlan &pl, int M, int N, int K, bool f32)
{
    const auto round = [](int64_t n) { return (n + 255) & ~int64_t(255); };
    LinScratch s;
    if (pl.pad) {
        const int64_t kp = lin_padded(K);
        s.codes = s.a + round(M * kp * (f32 ? 4 : 2));
        s.scales = s.codes + round(N * kp / 2);
        s.planes = s.scales + round(N * kp / 32);
    }
    s.bytes = s.planes + (pl.splits > 1 ? int64_t(pl.splits) * M * N * 4 : 0);
    return s;
}

// -------------------------------------------- attention (mx4_attention.hip)

constexpr int kTokRows = 16;   // query rows of a block; a workgroup has one or two
constexpr int kTokKeys = 32;   // keys a wave takes at a time
constexpr int kTokWaves = 4;
constexpr int kTileWaves = 4;
constexpr int kTileRows = 32 * kTileWaves;  // query rows of a workgroup
constexpr int kTileKeys = 64;
constexpr int kAttnMaxSplits = 64;

// Two blocks of rows fit the token kernel's registers.
constexpr bool two_row_blocks(bool f32, int D) { return !f32 || D == 64; }

struct AttnPlan {
    bool tile = false;  // the tile kernel
    int row_blocks = 1;  // of the token kernel
    int tiles = 0, splits = 1;
};

// Microseconds of a workgroup per 128 keys (token kernel, 16 and 32 query rows) and per 64
// keys (tile kernel, 128 rows), alone on a CU and as its share of a CU that has two;
// bf16 and f32 queries, D of 64 and 128.  These and the constants of the model are
// fitted to the times of 1900 calls, 1 to 64 sequences of unequal lengths of 100
// to 30000 keys, 1 to 1000 queries, 1 to 32 K/V heads.
struct Rate {
    double alone[3], full[3];
};
constexpr Rate kRates[2][2] = {{{{0.64, 1.79, 1.51}, {0.52, 0.82, 0.98}},
                                {{0.92, 1.43, 1.72}, {0.58, 0.98, 0.98}}},
                               {{{0.8, 2.14, 1.79}, {0.67, 1.13, 1.81}},
                                {{1.03, 0, 6.63}, {0.96, 0, 3.73}}}};

// The kernel and the split that the model expects to take least: latency, the keys
// of the longest share or of a full CU (half a workgroup's more on the fullest, and
// part of the last round's empty places), and with splits the partial results
// written and joined.  On those calls it is 0.8 % behind the fastest of all kernels
// and splits on average, 11 % in the worst twentieth.  The token kernel, which meets
// at no barrier, is ahead to some hundred query rows of a K/V head and in f32
// further: 2048 rows of 512 keys, 4 K/V heads, take 10.8 us by it and 18.7 by the
// tile kernel (bf16); 4096 x 512 keys, 32 heads, 50 us by the tile kernel against 141
// by the first token kernel.
// The lengths are the device's, so the plan is for a full cache.  One that holds little of
// its capacity is shared out too far: 16 heads on 4 of 128, bf16, 512 tokens in caches of
// 512, 4096 and 32768, by one query 9.3, 10.3 and 10.9 us, by 64 10.0, 12.2 and 20.4, by
// 512 11.7, 24.2 and 32.7.
inline AttnPlan attn_plan(int B, int S_q, int H, int H_kv, int D, int S_max, bool f32,
                          bool causal)
{
    const Rate &rate = kRates[f32][D == 128];
    const int64_t rows = int64_t(S_q) * (H / H_kv);
    // Under a causal mask the query tiles see S_max - S_q .. S_max keys.
    const double part = causal && S_q > 1 && S_max > 0
                            ? 1.0 - 0.5 * std::min(S_q, S_max) / S_max : 1.0;
    AttnPlan best;
    double best_us = 1e300;
    for (int kind = 0; kind < 3; ++kind) {
        AttnPlan pl;
        pl.tile = kind == 2;
        pl.row_blocks = kind == 1 ? 2 : 1;
        if (kind == 1 && (rows <= kTokRows || !two_row_blocks(f32, D)))
            continue;
        const int per_tile = pl.tile ? kTileRows : pl.row_blocks * kTokRows;
        pl.tiles = int((rows + per_tile - 1) / per_tile);
        const double groups = double(B) * H_kv * pl.tiles;
        const int keys = pl.tile ? kTileKeys : kTokKeys * kTokWaves;
        const int64_t rounds = (int64_t(S_max) + keys - 1) / keys;
        for (pl.splits = 1; pl.splits <= kAttnMaxSplits; pl.splits *= 2) {
            const double bytes = double(B) * S_q * H * pl.splits * D * 4;
            if (pl.splits > 1 && (pl.splits > rounds || bytes > 512e6))
                break;
            const double share = std::ceil(double(rounds) / pl.splits);
            const double load = groups * pl.splits / 256;  // workgroups per CU
            // The longest share, or the work of a full CU.
            const double rest = load > 1 ? 0.3 * (std::ceil(load) - load) : 0.0;
            const double work = part * (load + rest) + 0.5 * std::min(load, 1.0);
            double us = 6.6 + std::max(share * rate.alone[kind], share * work * rate.full[kind]) +
                        5.4 * std::max(0.0, load / 2 - 1);
            if (pl.splits > 1)
                us += 3.2 + bytes / 1.8e6;
            if (us < best_us) {
                best_us = us;
                best = pl;
            }
        }
    }
    return best;
}

}  // namespace mx4_plan
}  // namespace anima_hip
