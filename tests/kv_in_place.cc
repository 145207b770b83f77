// CPU check: the attention refuses an output that is one of its query's
// buffers (flash_deepseek_b200/csrc/moe_kv_host.h); one line per case.
#include <cstdio>

#include "../flash_deepseek_b200/csrc/moe_kv_host.h"

int main() {
    alignas(256) static char a[64], b[64], c[64];
    const moe_kv_batch batch{1, 2, nullptr, nullptr, nullptr, 1}, none{0, 2, nullptr, nullptr, nullptr, 0};
    auto say = [&](const char *name, const moe_kv_batch &k, const void *ql, const void *qr, void *out) {
        moe_mla_query q{};
        q.q_latent = ql, q.q_rope = qr, q.out = out;
        const char *bad = kv_bad_in_place(&k, &q);
        printf("%s: %s\n", name, bad ? bad : "ok");
    };
    say("apart", batch, a, b, c);
    say("query_twice", batch, a, a, c);
    say("latent", batch, a, b, a);
    say("rope", batch, a, b, b);
    say("nothing_to_do", none, a, a, a);
    return 0;
}
