// CPU check of the MLA attention's work division (moe_kv_plan.h) where
// sequence lengths near 2^31 meet page tables that span as many rows or more
// (repeated pages): no length, tile count or share may wrap.
#include <cstdio>
#include <vector>

#include "../flash_deepseek_b200/csrc/moe_kv_plan.h"

int main() {
    const int top = 0x7FFFFFFF;
    const int ctxs[] = {0, 1, 1 << 20, 1 << 30, top - 200, top - 64, top - 63, top - 1, top};
    const int64_t tables[] = {1, 1024, 1ll << 30, top - 64ll, top - 63ll, top - 1ll, top, 1ll << 31, (1ll << 31) + 1024, 1ll << 41};
    int cases = 0;
    for (int64_t table : tables)
        for (int ctx : ctxs)
            for (int n : {0, 1, 63, 64, 1 << 20}) {
                // a sane sequence on each side: their shares must not be touched
                auto at = [&](int b) {
                    return b == 1 ? mla_seq(5, 5 + n, ctx, 2 << 20, 128, table) : mla_seq(b ? 5 + n : 0, b ? 8 + n : 5, 100, 2 << 20, 128, 4096);
                };
                const MlaSeq s = at(1);
                const int64_t len = (int64_t)ctx + n;
                const bool ok = s.len >= 0 && s.tiles >= 0 && s.work() >= 0 && s.len <= table && s.len <= len &&
                                (n == 0 || (s.tiles >= 1 && (int64_t)s.tiles * MLA_N >= s.len && ((int64_t)s.tiles - 1) * MLA_N < s.len &&
                                            (int64_t)s.tiles * MLA_N <= top && (s.len == len || s.bad)));
                // a length that fits is not cut
                const bool whole = len > table || len > top - 64ll || n == 0 || (s.len == len && !s.bad);
                int64_t total = 0;
                for (int b = 0; b < 3; b++) total += at(b).work();
                bool shares = total >= 0;
                for (int p = 0; p < 74 && shares; p++) shares = mla_share(total, p, 74) <= mla_share(total, p + 1, 74);
                // the walk of the last pair ends in the last sequence
                MlaWalk w{};
                w.w = mla_share(total, 73, 74), w.w1 = total, w.n_seqs = 3;
                int64_t off = w.w;
                while (w.seq < 3 && off >= at(w.seq).work()) off -= at(w.seq++).work();
                w.off = off;
                MlaSeg g{};
                int64_t sum = 0;
                const int64_t share = w.w1 - w.w;
                bool in = true;
                for (int k = 0; k < 1000 && w.next(g, at); k++) sum += g.tile1 - g.tile0, in = in && g.tile0 >= 0 && g.tile1 <= w.s.tiles;
                const bool walk = in && (sum == share || sum > 0);
                if (!ok || !whole || !shares || !walk) {
                    printf("table %lld ctx %d n %d: len %d tiles %d bad %d (%d %d %d %d)\n", (long long)table, ctx, n, s.len, s.tiles, s.bad, ok,
                           whole, shares, walk);
                    return 1;
                }
                cases++;
            }
    printf("ok %d\n", cases);
    return 0;
}
