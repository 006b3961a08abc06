// Launch plans of the 8-bit linear layer: which kernel, tile and split a call of
// given sizes takes, by predicted time.  Host code without HIP.
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <iterator>

namespace anima_hip {
namespace fp8_plan {

// The runtime counts the threads of a launch in 32 bits.
inline bool launch_fits(int64_t blocks, int threads) { return blocks <= UINT32_MAX / threads; }

constexpr int kMaxSplits = 16;
constexpr int kStagedMaxGroups = 1 << 15;  // row offsets within a staged tile are 32-bit bytes

struct TileShape {
    int bm, bn;
    int groups;  // of K at once
    int room;    // workgroups that a CU holds
    // Time in us of one group of K while at most half of the CUs work and when all do (a
    // CU's two workgroups together where there is room for two), and of a tile's start and
    // end.  Fitted to whole calls to rank the shapes, not times that a part of the kernel
    // takes: nothing here counts bytes, and the 32 x 64 tiles of two groups come out faster
    // when all CUs work.  Where memory bounds a call it is predicted too fast
    // (bf16 1 x 16384 x 8192 12.0 us, measured 31.9).
    double us_alone, us_full, us_tile;
};
constexpr TileShape kBf16Shapes[] = {
    {256, 256, 1, 1, 1.221, 1.488, 6.736},
    {192, 256, 1, 1, 0.981, 1.195, 3.728},
    {128, 256, 1, 1, 0.773, 0.883, 4.003},
    {128, 128, 1, 2, 0.636, 0.998, 2.375},
    {128, 64, 1, 2, 0.331, 0.629, 1.957},
    {64, 128, 1, 2, 0.346, 0.690, 2.080},
    {64, 64, 1, 2, 0.215, 0.420, 1.550},
    {64, 64, 2, 1, 0.167, 0.227, 1.912},
    {32, 64, 1, 2, 0.220, 0.305, 1.456},
    {32, 64, 2, 1, 0.172, 0.129, 1.540}};
constexpr TileShape kF32Shapes[] = {
    {256, 256, 1, 1, 2.340, 2.809, 8.118},
    {192, 256, 1, 1, 1.842, 2.277, 3.297},
    {128, 256, 1, 1, 1.200, 1.568, 3.065},
    {128, 128, 1, 2, 0.779, 1.667, 2.312},
    {64, 128, 1, 2, 0.535, 1.080, 1.756},
    {64, 128, 2, 1, 0.417, 0.562, 2.357},
    {64, 64, 1, 2, 0.425, 0.700, 1.125},
    {64, 64, 2, 1, 0.284, 0.369, 1.638},
    {32, 64, 1, 2, 0.290, 0.399, 1.126},
    {32, 64, 2, 1, 0.197, 0.163, 1.358}};

// What belongs to a call rather than to a shape: us of a launch; us and bytes a us of the
// planes' sum; then the few-rows kernel's us of a launch, of a wave's group, and of a
// thousand groups of 16 weight rows, without and for 16 rows of A.
struct CallCost {
    double launch, sum_launch, sum_rate, few_launch, few_turn, few_weights, few_rows;
};
constexpr CallCost kBf16Cost = {2.195, 1.921, 1.886e6, 2.357, 0.809, 0.453, 0.265};
constexpr CallCost kF32Cost = {2.741, 1.753, 1.907e6, 2.300, 0.819, 0.466, 0.294};

struct LinPlan {
    bool staged = false;
    int waves = 1;  // few rows: of a workgroup
    // Staged: the shape and the split of K.
    int shape = 0, tiles_m = 0, tiles_n = 0, splits = 1, per_split = 0;  // per_split in groups
};

// The tile grid of a shape with K, a multiple of what it takes at once, shared out over up
// to `splits` workgroups.
inline void set_grid(LinPlan &pl, const TileShape &t, int M, int N, int groups, int splits)
{
    pl.staged = true;
    pl.tiles_m = (M + t.bm - 1) / t.bm;
    pl.tiles_n = (N + t.bn - 1) / t.bn;
    pl.per_split = (groups + splits - 1) / splits;
    pl.per_split += pl.per_split % t.groups;
    pl.splits = (groups + pl.per_split - 1) / pl.per_split;
}

inline int64_t strips(int M, int N) { return int64_t((N + 15) / 16) * ((M + 15) / 16); }

inline LinPlan few_plan(int M, int N, int groups)
{
    LinPlan pl;
    // Two waves for every SIMD of the GPU, but none without work.
    while (pl.waves < 8 && 2 * pl.waves <= groups && strips(M, N) * pl.waves < 2048)
        pl.waves *= 2;
    return pl;
}

inline double few_us(const LinPlan &pl, int M, int N, int groups, const CallCost &c)
{
    const int turns = (groups + pl.waves - 1) / pl.waves;
    // Latency, or the loads' rate.
    const double per_group = c.few_weights + c.few_rows * std::min(M, 16) / 16;
    return c.few_launch + std::max(turns * c.few_turn, strips(M, N) * groups * per_group / 1000);
}

inline double staged_us(const LinPlan &pl, const TileShape &t, int M, int N, const CallCost &c)
{
    const int64_t items = int64_t(pl.tiles_m) * pl.tiles_n * pl.splits;  // over 256 CUs
    double us = c.launch;
    if (t.room == 1) {
        const double slower = std::max(0.0, std::min(1.0, items / 128.0 - 1));
        const double group = t.us_alone + (t.us_full - t.us_alone) * slower;
        us += double((items + 255) / 256) * (pl.per_split * group + t.us_tile);
    } else {
        const int64_t pairs = items / 512, rest = items % 512;
        us += double(pairs) * (pl.per_split * t.us_full + t.us_tile);
        if (rest > 0)
            us += pl.per_split * (rest <= 256 ? t.us_alone : t.us_full) + t.us_tile;
    }
    if (pl.splits > 1)
        us += c.sum_launch + double(pl.splits) * M * N * 4 / c.sum_rate;
    return us;
}

// The plan whose predicted time is least.  The constants are fitted to 560 measured sizes
// of 1 to 8192 rows; on them the measured time of the choice is 2 % behind that of the best
// of the plans on average and 8 % in one of twenty, on 92 fresh ones 2 to 4 % on average.
// That is about the choice alone: the predicted times are further off (TileShape), also
// between sizes (bf16 256 x 2048 x 2048 predicted 5.8 us, 64 rows 6.5; measured 7.1 and 6.2).
inline LinPlan lin_plan(int M, int N, int groups, bool f32)
{
    LinPlan best = few_plan(M, N, groups);
    if (groups == 0 || groups > kStagedMaxGroups)
        return best;
    const CallCost &cost = f32 ? kF32Cost : kBf16Cost;
    double best_us = launch_fits(strips(M, N), best.waves * 64)
                         ? few_us(best, M, N, groups, cost) : HUGE_VAL;
    for (int shape = int(std::size(kBf16Shapes)) - 1; shape >= 0; --shape) {
        const TileShape &t = f32 ? kF32Shapes[shape] : kBf16Shapes[shape];
        if (groups % t.groups)
            continue;
        for (const int splits : {1, 2, 3, 4, 6, 8, 12, kMaxSplits}) {
            // One round of tiles at least, or the sum's launch: most shapes are too slow already.
            const double least = cost.launch + t.us_tile +
                                 (splits == 1 ? groups * std::min(t.us_alone, t.us_full)
                                              : cost.sum_launch);
            if (least >= best_us)
                continue;
            LinPlan pl;
            pl.shape = shape;
            set_grid(pl, t, M, N, groups, splits);
            const int64_t items = int64_t(pl.tiles_m) * pl.tiles_n * pl.splits;
            // K is shared out to fill the GPU, not beyond.
            if (pl.splits > 1 && items > 1024)
                break;
            if (!launch_fits(items, 512))
                continue;
            const double us = staged_us(pl, t, M, N, cost);
            if (us < best_us) {
                best = pl;
                best_us = us;
            }
        }
    }
    return best;
}

// Scratch: the planes of a split.
inline int64_t lin_scratch(const LinPlan &pl, int M, int N)
{
    return pl.staged && pl.splits > 1 ? int64_t(pl.splits) * M * N * 4 : 0;
}

}  // namespace fp8_plan
}  // namespace anima_hip
