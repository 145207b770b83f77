// CPU check of the MLA attention's work division (moe_kv_plan.h): for random
// batches every (sequence, block, tile) is walked exactly once, pieces of a
// cut unit are where the join looks for them, shares differ by one tile at most.
#include <cstdio>
#include <cstdlib>
#include <map>
#include <random>
#include <set>
#include <tuple>
#include <vector>

#include "../flash_deepseek_b200/csrc/moe_kv_plan.h"

#define CHECK(x)                                                   \
    do {                                                           \
        if (!(x)) {                                                \
            printf("round %d: %s (line %d)\n", round, #x, __LINE__); \
            return 1;                                              \
        }                                                          \
    } while (0)

int main() {
    std::mt19937 rng(1);
    long cut = 0, whole = 0;
    for (int round = 0; round < 400; round++) {
        const int n_seqs = 1 + rng() % (round % 5 == 0 ? 200 : 6), heads = 1 + rng() % 130, pairs = 1 + rng() % 80;
        const int page_rows = 8 << rng() % 5, per = 1 + rng() % 60;
        std::vector<int> q{(int)(rng() % 3)}, ctx;
        for (int b = 0; b < n_seqs; b++) {
            q.push_back(q.back() + (rng() % 3 ? rng() % 9 : 0));
            ctx.push_back(rng() % 11 == 0 ? -3 : (int)(rng() % (rng() % 4 ? 300 : 3000)));
        }
        const int n_tokens = q.back() - (rng() % 13 == 0);
        auto at = [&](int b) { return mla_seq(q[b], q[b + 1], ctx[b], n_tokens, heads, (int64_t)per * page_rows); };
        int64_t total = 0;
        for (int b = 0; b < n_seqs; b++) {
            const MlaSeq s = at(b);
            CHECK(s.work() >= 0 && (s.n == 0 || s.bad || s.len == s.ctx + s.n));
            CHECK(s.n == 0 || (s.blocks > 0 && s.tiles > 0 && s.tiles <= (per * page_rows + 63) / 64));
            total += s.work();
        }
        std::map<std::tuple<int, int, int>, int> seen;
        std::map<std::pair<int, int>, std::vector<std::pair<int, int>>> pieces;   // unit -> (pair, slot)
        std::map<std::pair<int, int>, std::pair<int, int>> tails;                 // unit -> (first pair, last pair)
        for (int p = 0; p < pairs; p++) {
            const int64_t w0 = mla_share(total, p, pairs), w1 = mla_share(total, p + 1, pairs);
            CHECK(w0 <= w1 && w1 - w0 <= total / pairs + 1 && (p || w0 == 0) && (p + 1 < pairs || w1 == total));
            CHECK(w0 < w1 || w1 == total);
            if (w0 == w1) continue;
            MlaWalk w{};
            w.w = w0, w.w1 = w1, w.n_seqs = n_seqs;
            int64_t off = w0;
            while (off >= at(w.seq).work()) off -= at(w.seq++).work();
            w.off = off;
            MlaSeg g{};
            int64_t sum = 0;
            int rest = 0;
            while (w.next(g, at)) {
                CHECK(g.tile0 < g.tile1 && g.tile1 <= w.s.tiles && g.block < w.s.blocks);
                for (int t = g.tile0; t < g.tile1; t++) CHECK(++seen[std::make_tuple(g.seq, g.block, t)] == 1);
                sum += g.tile1 - g.tile0;
                rest = w.s.tiles - g.tile1;
                CHECK(g.whole == (g.tile0 == 0 && rest == 0));
                if (!g.whole) pieces[{g.seq, g.block}].push_back({p, g.tile0 == 0});
                (g.whole ? whole : cut)++;
            }
            CHECK(sum == w1 - w0 && w.w == w1);
            if (rest > 0 && g.tile0 == 0) tails[{g.seq, g.block}] = {p, mla_last_pair(total, p, pairs, w1, rest)};
        }
        CHECK((int64_t)seen.size() == total);
        CHECK(tails.size() == pieces.size());
        for (auto &u : pieces) {
            const auto t = tails.at(u.first);
            CHECK((int)u.second.size() == t.second - t.first + 1);
            for (size_t k = 0; k < u.second.size(); k++)
                CHECK(u.second[k].first == t.first + (int)k && u.second[k].second == (k == 0));
        }
    }
    printf("ok %ld cut %ld whole\n", cut, whole);
    return 0;
}
