// The plans csrc/mx4_plan.h makes: for every line "linear M N K f32 staged" one line
// "few", "tiles <shape> <splits>", "staged <shape> <splits>" or "pad <shape> <splits>" (staged
// on padded copies), and for "attend B S_q H
// H_kv D S_max f32 causal" one line "token <splits>" or "tile <splits>".
#include "mx4_plan.h"

#include <iostream>
#include <string>

using namespace anima_hip::mx4_plan;

int main()
{
    std::string what;
    while (std::cin >> what) {
        if (what == "linear") {
            int M, N, K, f32, staged;
            std::cin >> M >> N >> K >> f32 >> staged;
            const LinPlan p = lin_plan(M, N, K, f32 != 0, staged != 0);
            if (p.kernel == kFew)
                std::cout << "few\n";
            else
                std::cout << (p.kernel == kTiles ? "tiles " : p.pad ? "pad " : "staged ") << p.shape << " "
                          << p.splits << "\n";
        } else {
            int B, S_q, H, H_kv, D, S_max, f32, causal;
            std::cin >> B >> S_q >> H >> H_kv >> D >> S_max >> f32 >> causal;
            const AttnPlan p = attn_plan(B, S_q, H, H_kv, D, S_max, f32 != 0, causal != 0);
            std::cout << (p.tile ? "tile " : "token ") << p.splits << "\n";
        }
    }
    return 0;
}
