// CPU check of the rotary frequency table (flash_deepseek_b200/csrc/moe_kv_host.h)
// away from its default configuration: reads lines of "dim theta scale orig_ctx
// beta_fast beta_slow", prints the turns per position of every pair, a line each.
#include <cstdio>

#include "../flash_deepseek_b200/csrc/moe_kv_host.h"

int main() {
    moe_rope_config r{};
    r.mscale = 1.0f;
    double turns[128];
    while (scanf("%d %f %f %f %f %f", &r.dim, &r.theta, &r.scale, &r.orig_ctx, &r.beta_fast, &r.beta_slow) == 6) {
        if (kv_bad_rope(&r)) return 1;
        kv_rope_turns(&r, turns);
        for (int i = 0; i < r.dim / 2; i++) printf("%.17g ", turns[i]);
        printf("\n");
    }
    return 0;
}
