// CPU check of the MLA attention entry points' refusals and of the rotary
// frequency table (flash_deepseek_b200/csrc/moe_kv_host.h): prints one line
// per case, name and "ok" or the reason.
#include <cstdio>
#include <limits>

#include "../flash_deepseek_b200/csrc/moe_kv_host.h"

static void say(const char *name, const char *bad) { printf("%s: %s\n", name, bad ? bad : "ok"); }

int main() {
    alignas(256) static char mem[1024];
    int *ip = reinterpret_cast<int *>(mem);
    const moe_kv_cache kv{mem, MOE_KV_BF16, 512, 64, 100};
    const moe_kv_batch b{2, 8, ip, ip, ip, 4};
    const moe_rope_config r{64, 0, 10000.0f, 40.0f, 4096.0f, 32.0f, 1.0f, 1.0f};
    const moe_mla_query q{mem, 128 * 512, 512, mem, 128 * 64, 64, 128, 0.1f, nullptr, 0, mem, 128 * 512, 512, nullptr};
    const float nan = std::numeric_limits<float>::quiet_NaN();

    say("cache", kv_bad_cache(&kv, &b));
    say("cache_null", kv_bad_cache(nullptr, &b));
    say("batch_null", kv_bad_cache(&kv, nullptr));
#define KV(name, field, value) { moe_kv_cache k = kv; k.field = value; say(name, kv_bad_cache(&k, &b)); }
#define BT(name, field, value) { moe_kv_batch k = b; k.field = value; say(name, kv_bad_cache(&kv, &k)); }
    KV("format", format, 2) KV("latent_odd", latent, 500) KV("latent_big", latent, 640) KV("latent_0", latent, 0)
    KV("page_48", page_size, 48) KV("page_4", page_size, 4) KV("page_2048", page_size, 2048) KV("page_neg", page_size, -64)
    KV("pages_0", n_pages, 0) KV("pages_many", n_pages, 1 << 26) KV("data_null", data, nullptr) KV("data_off", data, mem + 16)
    BT("seqs_neg", n_seqs, -1) BT("seqs_many", n_seqs, 4097) BT("tokens_neg", n_tokens, -1) BT("tokens_many", n_tokens, (1 << 30) + 1) BT("start_null", q_start, nullptr)
    BT("ctx_null", ctx_len, nullptr) BT("table_null", pages, nullptr) BT("table_0", pages_per_seq, 0)
    { moe_kv_batch k{0, 0, nullptr, nullptr, nullptr, 0}; say("no_seqs", kv_bad_cache(&kv, &k)); }

    auto rope = [&](const char *name, const moe_rope_config &c, const void *x, int xt, int64_t s0, int64_t s1, const void *y,
                    int yt, int64_t t0, int64_t t1, int T, int H, int D, int off) {
        say(name, kv_bad_rope_call(&c, x, xt, s0, s1, y, yt, t0, t1, ip, T, H, D, off));
    };
    char *y = mem + 512;
    rope("rope", r, mem, 0, 192, 64, y, 30, 192, 64, 2, 3, 64, 0);
    rope("rope_in_place", r, mem, 1, 192, 64, mem, 1, 192, 64, 2, 3, 64, 0);
    rope("rope_in_place_type", r, mem, 1, 192, 64, mem, 30, 192, 64, 2, 3, 64, 0);
    rope("rope_in_place_stride", r, mem, 1, 192, 64, mem, 1, 256, 64, 2, 3, 64, 0);
    rope("rope_type", r, mem, 12, 192, 64, y, 1, 192, 64, 2, 3, 64, 0);
    rope("rope_offset", r, mem, 1, 192, 64, y, 1, 192, 64, 2, 3, 64, 1);
    rope("rope_overlap", r, mem, 1, 192, 64, y, 1, 191, 64, 2, 3, 64, 0);
    rope("rope_head_major", r, mem, 1, 64, 128, y, 1, 64, 128, 2, 3, 64, 0);
    rope("rope_neg", r, mem, 1, -192, 64, y, 1, 192, 64, 2, 3, 64, 0);
    rope("rope_off_align", r, mem + 1, 1, 192, 64, y, 1, 192, 64, 2, 3, 64, 0);
    rope("rope_nothing", r, nullptr, 1, 192, 64, nullptr, 1, 192, 64, 0, 3, 64, 0);
    rope("rope_many", r, mem, 1, 192, 64, y, 1, 192, 64, (1 << 30) + 1, 3, 64, 0);
    rope("rope_null", r, nullptr, 1, 192, 64, y, 1, 192, 64, 1, 3, 64, 0);
    rope("rope_broadcast_in", r, mem, 1, 0, 0, y, 1, 192, 64, 2, 3, 64, 0);
#define RP(name, field, value) { moe_rope_config k = r; k.field = value; say(name, kv_bad_rope(&k)); }
    RP("dim_odd", dim, 63) RP("dim_0", dim, 0) RP("dim_258", dim, 258) RP("theta_1", theta, 1.0f) RP("theta_nan", theta, nan)
    RP("scale_low", scale, 0.5f) RP("orig_0", orig_ctx, 0.0f) RP("beta_neg", beta_fast, -1.0f) RP("mscale_nan", mscale, nan)
    { moe_rope_config k = r; k.scale = 1.0f; k.orig_ctx = 0.0f; say("no_scaling", kv_bad_rope(&k)); }

    say("write", kv_bad_write(&b, mem, 0, 576, nullptr, 1e-6f, &r, ip));
    say("write_bare", kv_bad_write(&b, mem, 0, 576, nullptr, 1e-6f, nullptr, nullptr));
    say("write_no_pos", kv_bad_write(&b, mem, 0, 576, nullptr, 1e-6f, &r, nullptr));
    say("write_type", kv_bad_write(&b, mem, 14, 576, nullptr, 1e-6f, &r, ip));
    say("write_eps", kv_bad_write(&b, mem, 0, 576, nullptr, nan, &r, ip));
    { moe_rope_config k = r; k.dim = 32; say("write_dim", kv_bad_write(&b, mem, 0, 576, nullptr, 0.0f, &k, ip)); }
    say("read", kv_bad_read(&kv, &b, mem, 30, 576));
    say("read_overlap", kv_bad_read(&kv, &b, mem, 30, 575));
    say("read_null", kv_bad_read(&kv, &b, nullptr, 30, 576));

    say("query", kv_bad_query(&kv, &b, &q, mem, 256, 256));
    say("query_ws", kv_bad_query(&kv, &b, &q, mem, 255, 256));
    say("query_ws_off", kv_bad_query(&kv, &b, &q, mem + 128, 256, 256));
    say("query_null", kv_bad_query(&kv, &b, nullptr, mem, 256, 256));
#define QY(name, field, value) { moe_mla_query k = q; k.field = value; say(name, kv_bad_query(&kv, &b, &k, mem, 256, 256)); }
    QY("heads_0", n_heads, 0) QY("heads_1025", n_heads, 1025) QY("scale_nan", scale, nan) QY("stride_7", q_rope_head_stride, 65)
    QY("stride_neg", out_token_stride, -512) QY("out_overlap", out_head_stride, 504) QY("out_off", out, mem + 8)
    QY("q_null", q_latent, nullptr) QY("lse_off", lse, reinterpret_cast<float *>(mem + 2))
    { moe_mla_query k = q; k.tree = reinterpret_cast<const uint32_t *>(mem); say("tree_words", kv_bad_query(&kv, &b, &k, mem, 256, 256)); }
    { moe_kv_batch k = b; k.n_tokens = 1 << 25; say("rows_many", kv_bad_query(&kv, &k, &q, mem, 256, 256)); }

    double turns[128];
    kv_rope_turns(&r, turns);
    for (int i = 0; i < 32; i++) printf("turn %d %.17g\n", i, turns[i]);
    return 0;
}
