// The plans csrc/fp8_plan.h makes: for every line "M N groups f32" one line "few <waves>" or
// "tile <shape> <splits>", then the scratch bytes.  Every plan is checked: its tiles and parts
// of K cover the product, none is empty, and its launches fit.
#include "fp8_plan.h"

#include <iostream>

using namespace anima_hip::fp8_plan;

int main()
{
    int M, N, groups, f32;
    while (std::cin >> M >> N >> groups >> f32) {
        const LinPlan p = lin_plan(M, N, groups, f32 != 0);
        const int64_t bytes = lin_scratch(p, M, N);
        if (!p.staged) {
            if (bytes != 0 || (p.waves > 1 && p.waves > groups) || p.waves > 8)
                return 1;
            std::cout << "few " << p.waves << " 0\n";
            continue;
        }
        const TileShape &t = f32 ? kF32Shapes[p.shape] : kBf16Shapes[p.shape];
        const int64_t items = int64_t(p.tiles_m) * p.tiles_n * p.splits;
        if (int64_t(p.tiles_m) * t.bm < M || int64_t(p.tiles_m - 1) * t.bm >= M ||
            int64_t(p.tiles_n) * t.bn < N || int64_t(p.tiles_n - 1) * t.bn >= N)
            return 2;
        if (int64_t(p.splits) * p.per_split < groups ||
            int64_t(p.splits - 1) * p.per_split >= groups || p.splits > kMaxSplits)
            return 3;
        if (groups % t.groups || p.per_split % t.groups)
            return 4;
        if (!launch_fits(items, 512))
            return 5;
        if (bytes != (p.splits > 1 ? int64_t(p.splits) * M * N * 4 : 0) ||
            (p.splits > 1 && !launch_fits((int64_t(M) * N + 255) / 256, 256)))
            return 6;
        std::cout << "tile " << p.shape << " " << p.splits << " " << bytes << "\n";
    }
    return 0;
}
