// moe_kv_host.h -- argument checks of the MLA attention entry points and the
// rotary frequency table, in plain C++ (no CUDA), so that a CPU test reaches
// every refusal.  Each check returns nullptr or the reason of the refusal.
#pragma once
#include <math.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>

#include "../../include/moe_cuda.h"

inline bool kv_fmt_fp8(int fmt) { return fmt == MOE_KV_FP8_F16 || fmt == MOE_KV_FP8_BF16; }
inline bool kv_fmt_known(int fmt) { return fmt == MOE_KV_F16 || fmt == MOE_KV_BF16 || kv_fmt_fp8(fmt); }
inline bool kv_float_type(int t) { return t == MOE_TYPE_F32 || t == MOE_TYPE_F16 || t == MOE_TYPE_BF16; }
inline size_t kv_float_size(int t) { return t == MOE_TYPE_F32 ? 4 : 2; }
inline bool kv_off(const void *p, size_t a) { return ((uintptr_t)p % a) != 0; }

// 0 when the format or the number of latent values is not supported
inline size_t kv_host_row_bytes(int format, int latent) {
    if (!kv_fmt_known(format) || latent < 128 || latent > 512 || latent % 128) return 0;
    if (!kv_fmt_fp8(format)) return 2 * ((size_t)latent + MOE_KV_ROPE);
    return ((size_t)latent + 2 * MOE_KV_ROPE + latent / 32 + 15) / 16 * 16;
}

// [n0][n1] blocks of `len` values at strides s0, s1 that do not overlap
inline bool kv_disjoint(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t len) {
    if (n0 <= 1) return n1 <= 1 || s1 >= len;
    if (n1 <= 1) return s0 >= len;
    return (s1 >= len && s0 >= (n1 - 1) * s1 + len) || (s0 >= len && s1 >= (n0 - 1) * s0 + len);
}

inline const char *kv_bad_cache(const moe_kv_cache *kv, const moe_kv_batch *b) {
    if (!kv || !b) return "null cache or batch";
    if (!kv_host_row_bytes(kv->format, kv->latent)) return "cache format or number of latent values not supported";
    if (kv->page_size < 8 || kv->page_size > 1024 || (kv->page_size & (kv->page_size - 1)))
        return "page_size is not a power of two in 8..1024";
    if (kv->n_pages <= 0 || (int64_t)kv->n_pages * kv->page_size > 0x7FFFFFFFll) return "n_pages out of range";
    if (!kv->data || kv_off(kv->data, 128)) return "cache buffer null or not 128-byte aligned";
    if (b->n_seqs < 0 || b->n_seqs > 4096 || b->n_tokens < 0 || b->n_tokens > (1 << 30)) return "number of sequences or tokens out of range";
    if (b->n_seqs > 0 && (!b->q_start || !b->ctx_len || !b->pages || b->pages_per_seq <= 0 || kv_off(b->q_start, 4) ||
                          kv_off(b->ctx_len, 4) || kv_off(b->pages, 4)))
        return "sequence bounds or page table null or not aligned";
    return nullptr;
}

inline const char *kv_bad_rope(const moe_rope_config *r) {
    if (!r) return "null rope configuration";
    if (r->dim < 2 || r->dim > 256 || r->dim % 2) return "rope dim is not even in 2..256";
    if (!(r->theta > 1.0f) || !(r->scale >= 1.0f) || !std::isfinite(r->theta) || !std::isfinite(r->scale) ||
        !std::isfinite(r->mscale))
        return "rope theta must be above 1, scale at least 1, all finite";
    if (r->scale > 1.0f && !(r->orig_ctx > 0.0f && r->beta_fast > 0.0f && r->beta_slow > 0.0f &&
                             std::isfinite(r->orig_ctx) && std::isfinite(r->beta_fast) && std::isfinite(r->beta_slow)))
        return "rope scaling needs orig_ctx, beta_fast and beta_slow above 0";
    return nullptr;
}

// turns per position of each of the dim / 2 pairs, in 64 bits
inline void kv_rope_turns(const moe_rope_config *r, double *turns) {
    const double tau = 6.283185307179586476925, theta = r->theta, dim = r->dim;
    const int pairs = r->dim / 2;
    double lo = 0, hi = 1;
    if (r->scale > 1.0f) {
        lo = std::max(floor(dim * log(r->orig_ctx / (r->beta_fast * tau)) / (2 * log(theta))), 0.0);
        hi = std::min(ceil(dim * log(r->orig_ctx / (r->beta_slow * tau)) / (2 * log(theta))), (double)(pairs - 1));
        hi = std::max(hi, lo + 1);
    }
    for (int i = 0; i < pairs; i++) {
        const double f = pow(theta, -2.0 * i / dim);
        const double ramp = r->scale > 1.0f ? std::min(std::max((i - lo) / (hi - lo), 0.0), 1.0) : 0.0;
        turns[i] = (f / r->scale * ramp + f * (1 - ramp)) / tau;
    }
}

inline const char *kv_bad_rope_call(const moe_rope_config *rope, const void *x, int x_type, int64_t xt, int64_t xh,
                                    const void *y, int y_type, int64_t yt, int64_t yh, const int *pos, int T,
                                    int n_heads, int head_dim, int offset) {
    if (const char *bad = kv_bad_rope(rope)) return bad;
    if (!kv_float_type(x_type) || !kv_float_type(y_type)) return "type not supported";
    if (T < 0 || T > (1 << 30) || n_heads < 0 || n_heads > 65536 || head_dim <= 0 || head_dim > 65536 || offset < 0 ||
        offset > head_dim - rope->dim || (int64_t)n_heads * head_dim > 0x3FFFFFFF)
        return "tokens, heads or rotated values out of range";
    if (xt < 0 || xh < 0 || yt < 0 || yh < 0) return "negative stride";
    if (T == 0 || n_heads == 0) return nullptr;
    if (!x || !y || !pos || kv_off(x, kv_float_size(x_type)) || kv_off(y, kv_float_size(y_type)) || kv_off(pos, 4))
        return "buffer null or not aligned to its type";
    if (x == y && (x_type != y_type || xt != yt || xh != yh)) return "in place needs the same type and strides";
    if (!kv_disjoint(T, yt, n_heads, yh, head_dim)) return "output strides overlap";
    return nullptr;
}

inline const char *kv_bad_write(const moe_kv_batch *b, const void *x, int type, int64_t stride, const float *norm_w,
                                float eps, const moe_rope_config *rope, const int *pos) {
    if (rope) {
        if (const char *bad = kv_bad_rope(rope)) return bad;
        if (rope->dim != MOE_KV_ROPE) return "rope dim is not 64";
    }
    if (!kv_float_type(type)) return "type not supported";
    if (stride < 0 || !(eps >= 0.0f)) return "negative stride or eps";
    if (b->n_tokens == 0 || b->n_seqs == 0) return nullptr;
    if (!x || (rope && !pos) || kv_off(x, kv_float_size(type)) || kv_off(norm_w, 4) || kv_off(pos, 4))
        return "buffer null or not aligned to its type";
    return nullptr;
}

inline const char *kv_bad_read(const moe_kv_cache *kv, const moe_kv_batch *b, const void *y, int type, int64_t stride) {
    if (!kv_float_type(type)) return "type not supported";
    if (stride < 0 || !kv_disjoint(b->n_tokens, stride, 1, 0, kv->latent + MOE_KV_ROPE)) return "rows overlap";
    if (b->n_tokens == 0 || b->n_seqs == 0) return nullptr;
    if (!y || kv_off(y, kv_float_size(type))) return "buffer null or not aligned to its type";
    return nullptr;
}

inline const char *kv_bad_query(const moe_kv_cache *kv, const moe_kv_batch *b, const moe_mla_query *q, const void *ws,
                                size_t ws_bytes, size_t ws_need) {
    if (!q) return "null query";
    if (q->n_heads <= 0 || q->n_heads > 1024 || (int64_t)b->n_tokens * q->n_heads > 0x7FFFFFFFll)
        return "number of heads or tokens out of range";
    if (!std::isfinite(q->scale)) return "scale is not finite";
    const int64_t st[6] = {q->q_latent_token_stride, q->q_latent_head_stride, q->q_rope_token_stride,
                           q->q_rope_head_stride, q->out_token_stride, q->out_head_stride};
    for (int64_t v : st)
        if (v < 0 || v % 8) return "a stride is negative or not a multiple of 8";
    if (q->tree && q->tree_words <= 0) return "tree_words is not positive";
    if (!kv_disjoint(b->n_tokens, st[4], q->n_heads, st[5], kv->latent)) return "output strides overlap";
    if (b->n_tokens == 0 || b->n_seqs == 0) return nullptr;
    if (!q->q_latent || !q->q_rope || !q->out || kv_off(q->q_latent, 16) || kv_off(q->q_rope, 16) || kv_off(q->out, 16))
        return "query or output buffer null or not 16-byte aligned";
    if (kv_off(q->lse, 4) || kv_off(q->tree, 4)) return "lse or tree not aligned";
    if (!ws || kv_off(ws, 256) || ws_bytes < ws_need) return "workspace null, not 256-byte aligned or too small";
    return nullptr;
}

// The attention's output may not be one of its query's buffers: the CTAs that share a block of query rows, and the pairs
// that share a unit, read the query at their own times, while others store results.
inline const char *kv_bad_in_place(const moe_kv_batch *b, const moe_mla_query *q) {
    if (b->n_tokens == 0 || b->n_seqs == 0) return nullptr;
    if (q->out == q->q_latent || q->out == q->q_rope) return "output and query are the same buffer";
    return nullptr;
}
