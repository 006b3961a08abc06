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
    bool pairs;  // two groups of K at once where K has an even number of them
};
constexpr TileShape kBf16Shapes[] = {{256, 256, false}, {192, 256, false}, {128, 256, false},
                                     {128, 128, false}, {64, 128, true},   {64, 64, true},
                                     {32, 64, true}};
constexpr TileShape kF32Shapes[] = {{256, 256, false}, {128, 256, false}, {128, 128, false},
                                    {64, 128, true},   {64, 64, true},    {32, 64, true}};

struct LinPlan {
    bool staged = false;
    // Few rows: 16-row blocks of A a workgroup takes, and its waves.
    int blocks = 1, waves = 4;
    // Staged: the shape, whether it takes two groups at once, and the split of K.
    int shape = 0;
    bool pairs = false;
    int tiles_m = 0, tiles_n = 0, splits = 1, per_split = 0;  // per_split in groups
};

inline void set_grid(LinPlan &pl, const TileShape &t, int M, int N, int groups, int splits)
{
    pl.staged = true;
    pl.tiles_m = (M + t.bm - 1) / t.bm;
    pl.tiles_n = (N + t.bn - 1) / t.bn;
    pl.per_split = (groups + splits - 1) / splits;
    pl.pairs = t.pairs && groups % 2 == 0;
    if (pl.pairs)
        pl.per_split += pl.per_split & 1;
    pl.splits = pl.per_split ? (groups + pl.per_split - 1) / pl.per_split : 1;
}

inline LinPlan few_plan(int M, int N, int groups)
{
    LinPlan pl;
    pl.blocks = M <= 16 ? 1 : M <= 32 ? 2 : 4;
    const int64_t strips = int64_t((N + 15) / 16) * ((M + 16 * pl.blocks - 1) / (16 * pl.blocks));
    // Waves for every SIMD of the GPU to have some, but none without work.
    pl.waves = 1;
    while (pl.waves < 16 && pl.waves < groups && strips * pl.waves < 4096)
        pl.waves *= 2;
    return pl;
}

inline LinPlan lin_plan(int M, int N, int groups, bool f32)
{
    if (M <= 64 || groups == 0 || groups > kStagedMaxGroups)
        return few_plan(M, N, groups);
    LinPlan pl;
    pl.shape = M <= 512 ? (f32 ? 4 : 5) : (f32 ? 0 : 1);
    set_grid(pl, f32 ? kF32Shapes[pl.shape] : kBf16Shapes[pl.shape], M, N, groups, 1);
    return pl;
}

// Scratch: the planes of a split.
inline int64_t lin_scratch(const LinPlan &pl, int M, int N)
{
    return pl.staged && pl.splits > 1 ? int64_t(pl.splits) * M * N * 4 : 0;
}

}  // namespace fp8_plan
}  // namespace anima_hip
