// moe_kv.cu -- rotary positions, and the rows of the paged latent cache
// written and read back (formats in moe_kv.cuh).  All three are bound by the
// bytes they move; apply_rope_q / apply_rope_k (infer.m:628-656) and the
// cache append of mla_forward (infer.m:665-675, 760-790) are the reference's
// counterparts, one token at a time.
#include "moe_kv.cuh"

#define LAUNCH_COUNT(p) \
    do {                \
        if (p) (*(p))++; \
    } while (0)

namespace {

// ---------------------------------------------------------------------------
// Rotary positions.  y = x with the pairs of dims [offset, offset + dim) of
// every head rotated: (a, b) -> (a cos - b sin, a sin + b cos), the other
// dims copied.  One CTA takes (part of) the heads of one token, so the angles
// (one reduction in fp64 and one sincospi per pair) are formed once per CTA
// and read from shared memory by all heads.
// ---------------------------------------------------------------------------
constexpr int RP_THREADS = 256;
constexpr int RP_PAIRS = 128;

struct RopeArgs {
    const void *x;
    void *y;
    long long xt, xh, yt, yh;   // strides in elements: token, head
    const int *pos;
    int n_heads, head_dim, offset;
    int in_place;
    int units;                  // work units of one token
    int units_per_cta;
};

template <typename TI, typename TO, bool VEC>
__global__ void __launch_bounds__(RP_THREADS) k_rope(RopeArgs a, MoeRopeDev rope) {
    __shared__ float cs[RP_PAIRS], sn[RP_PAIRS];
    const int t = blockIdx.x, m = rope.pairs;
    const int p = __ldg(a.pos + t);
    if ((int)threadIdx.x < m) kv_cos_sin(p, rope.turns[threadIdx.x], rope.mscale, cs[threadIdx.x], sn[threadIdx.x]);
    __syncthreads();
    const TI *x = reinterpret_cast<const TI *>(a.x) + (long long)t * a.xt;
    TO *y = reinterpret_cast<TO *>(a.y) + (long long)t * a.yt;
    // a unit is W elements (an interleaved block, or a copied one), or W
    // elements of the first half together with their partners in the second
    constexpr int W = VEC ? 8 : 1;
    const int rot = rope.half_layout ? m / W : (VEC ? 2 * m / W : m);   // rotated units of a head
    const int per = rot + (a.in_place ? 0 : (a.head_dim - 2 * m) / W);
    const int u1 = min(a.units, (int)(blockIdx.y + 1) * a.units_per_cta);
#pragma unroll 4
    for (int u = blockIdx.y * a.units_per_cta + threadIdx.x; u < u1; u += RP_THREADS) {
        const int h = u / per, j = u - h * per;
        const TI *xh = x + (long long)h * a.xh;
        TO *yh = y + (long long)h * a.yh;
        if (j >= rot) {   // copied
            int e = (j - rot) * W;
            if (e >= a.offset) e += 2 * m;
            if (VEC) {
                float v[8];
                kv_load8<TI, true>(xh + e, v);
                kv_store8<TO, true>(yh + e, v);
            } else {
                yh[e] = KvType<TO>::from_f(KvType<TI>::to_f(xh[e]));
            }
        } else if (rope.half_layout) {
            const int i = j * W, e = a.offset + i;
            if (VEC) {
                float u0[8], u2[8], v0[8], v2[8];
                kv_load8<TI, true>(xh + e, u0);
                kv_load8<TI, true>(xh + e + m, u2);
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float c = cs[i + k], s = sn[i + k];
                    v0[k] = u0[k] * c - u2[k] * s;
                    v2[k] = u0[k] * s + u2[k] * c;
                }
                kv_store8<TO, true>(yh + e, v0);
                kv_store8<TO, true>(yh + e + m, v2);
            } else {
                const float c = cs[i], s = sn[i];
                const float p0 = KvType<TI>::to_f(xh[e]), p1 = KvType<TI>::to_f(xh[e + m]);
                yh[e] = KvType<TO>::from_f(p0 * c - p1 * s);
                yh[e + m] = KvType<TO>::from_f(p0 * s + p1 * c);
            }
        } else if (VEC) {
            const int e = a.offset + j * 8;
            float v[8], w[8];
            kv_load8<TI, true>(xh + e, v);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const float c = cs[j * 4 + k], s = sn[j * 4 + k];
                w[2 * k] = v[2 * k] * c - v[2 * k + 1] * s;
                w[2 * k + 1] = v[2 * k] * s + v[2 * k + 1] * c;
            }
            kv_store8<TO, true>(yh + e, w);
        } else {
            const int e = a.offset + 2 * j;
            const float c = cs[j], s = sn[j];
            const float p0 = KvType<TI>::to_f(xh[e]), p1 = KvType<TI>::to_f(xh[e + 1]);
            yh[e] = KvType<TO>::from_f(p0 * c - p1 * s);
            yh[e + 1] = KvType<TO>::from_f(p0 * s + p1 * c);
        }
    }
}

// ---------------------------------------------------------------------------
// Cache rows.  One warp per row: a lane holds 8 consecutive latent values of
// every 256 (so a group of 32 is 4 lanes, and loads and stores of a warp are
// contiguous) and one rotary pair.
// ---------------------------------------------------------------------------
constexpr int KV_WARPS = 4;
constexpr int KV_CHUNKS = 2;   // 256-value chunks of the widest latent part (512)

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename TI, typename TC, bool FP8, bool VEC>
__global__ void __launch_bounds__(KV_WARPS * 32) k_kv_write(MoeKvDev kv, MoeKvBatchDev b, const TI *__restrict__ x,
                                                            long long stride, const float *__restrict__ norm_w,
                                                            float eps, int rotate, MoeRopeDev rope,
                                                            const int *__restrict__ pos, int *error) {
    const int t = blockIdx.x * KV_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= b.n_tokens) return;
    const int L = kv.latent;
    const TI *row = x + (long long)t * stride;
    // the row itself first: these loads do not wait for the page lookup
    float v[KV_CHUNKS][8], w[KV_CHUNKS][8];
#pragma unroll
    for (int c = 0; c < KV_CHUNKS; c++) {
        const int e = c * 256 + lane * 8;
        if (e < L) {
            kv_load8<TI, VEC>(row + e, v[c]);
            if (norm_w) kv_load8<float, VEC>(norm_w + e, w[c]);
        }
    }
    const int ia = rotate && rope.half_layout ? lane : 2 * lane;
    const int ib = rotate && rope.half_layout ? lane + MOE_KV_ROPE / 2 : 2 * lane + 1;
    float ra = KvType<TI>::to_f(row[L + ia]), rb = KvType<TI>::to_f(row[L + ib]);
    float cs = 1.0f, sn = 0.0f;
    if (rotate) kv_cos_sin(__ldg(pos + t), rope.turns[lane], rope.mscale, cs, sn);
    const int seq = kv_seq_of(b, t);
    if (seq < 0) return;   // behind the last sequence: nothing is written
    const long long at = kv_flat_row(kv, b, seq, (long long)__ldg(b.ctx_len + seq) + (t - __ldg(b.q_start + seq)));
    if (at < 0) {
        if (lane == 0) kv_error(error, KV_ERR_BATCH);
        return;
    }
    if (norm_w) {
        float ss = 0.0f;
#pragma unroll
        for (int c = 0; c < KV_CHUNKS; c++)
            if (c * 256 + lane * 8 < L)
#pragma unroll
                for (int k = 0; k < 8; k++) ss = fmaf(v[c][k], v[c][k], ss);
        const float r = 1.0f / sqrtf(warp_sum(ss) / (float)L + eps);
#pragma unroll
        for (int c = 0; c < KV_CHUNKS; c++)
            if (c * 256 + lane * 8 < L)
#pragma unroll
                for (int k = 0; k < 8; k++) v[c][k] = v[c][k] * r * w[c][k];
    }
    if (rotate) {
        const float a = ra;
        ra = a * cs - rb * sn;
        rb = a * sn + rb * cs;
    }
    uint8_t *dst = kv.data + at * kv.row_bytes;
    TC *drope = reinterpret_cast<TC *>(dst + (FP8 ? L : 2 * L));
#pragma unroll
    for (int c = 0; c < KV_CHUNKS; c++) {
        const int e = c * 256 + lane * 8;
        if (!FP8) {
            if (e < L) kv_store8<TC, true>(reinterpret_cast<TC *>(dst) + e, v[c]);
            continue;
        }
        // the group's largest magnitude over its 4 lanes (every lane takes
        // part in the shuffles; L is a multiple of 128, so groups are whole)
        uint32_t big = 0;
        if (e < L)
#pragma unroll
            for (int k = 0; k < 8; k++) big = max(big, __float_as_uint(v[c][k]) & 0x7FFFFFFFu);
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 1));
        big = max(big, __shfl_xor_sync(0xffffffffu, big, 2));
        if (e >= L) continue;
        // the least k with amax <= 448 * 2^k, 448 = 1.75 * 2^8 (exact: exponent and mantissa compared as integers)
        int k = (int)(big >> 23) - 127 - 8 + ((big & 0x7FFFFFu) > 0x600000u);
        k = min(max(k, KV_K_MIN), KV_K_MAX);
        const bool bad = big >= 0x7F800000u;
        const float inv = __uint_as_float((uint32_t)(127 - k) << 23);
        uint32_t q[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float2 lo = make_float2(v[c][4 * i] * inv, v[c][4 * i + 1] * inv);
            const float2 hi = make_float2(v[c][4 * i + 2] * inv, v[c][4 * i + 3] * inv);
            q[i] = (uint32_t)__nv_cvt_float2_to_fp8x2(lo, __NV_SATFINITE, __NV_E4M3) |
                   (uint32_t)__nv_cvt_float2_to_fp8x2(hi, __NV_SATFINITE, __NV_E4M3) << 16;
        }
        *reinterpret_cast<uint2 *>(dst + e) = make_uint2(q[0], q[1]);
        if ((lane & 3) == 0) dst[L + 2 * MOE_KV_ROPE + e / KV_GROUP] = bad ? 255 : (uint8_t)(127 + k);
    }
    drope[ia] = KvType<TC>::from_f(ra);
    drope[ib] = KvType<TC>::from_f(rb);
}

template <typename TO, typename TC, bool FP8, bool VEC>
__global__ void __launch_bounds__(KV_WARPS * 32) k_kv_read(MoeKvDev kv, MoeKvBatchDev b, TO *__restrict__ y,
                                                           long long stride, int *error) {
    const int t = blockIdx.x * KV_WARPS + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (t >= b.n_tokens) return;
    const int seq = kv_seq_of(b, t);
    if (seq < 0) return;
    const int L = kv.latent;
    const long long at = kv_flat_row(kv, b, seq, (long long)__ldg(b.ctx_len + seq) + (t - __ldg(b.q_start + seq)));
    if (at < 0 && lane == 0) kv_error(error, KV_ERR_BATCH);   // the row reads as zeros
    const uint8_t *src = kv.data + (at < 0 ? 0 : at) * kv.row_bytes;
    TO *dst = y + (long long)t * stride;
    const TC *srope = reinterpret_cast<const TC *>(src + (FP8 ? L : 2 * L));
    float v[KV_CHUNKS][8];
#pragma unroll
    for (int c = 0; c < KV_CHUNKS; c++) {
        const int e = c * 256 + lane * 8;
#pragma unroll
        for (int k = 0; k < 8; k++) v[c][k] = 0.0f;
        if (e >= L || at < 0) continue;
        if (!FP8) {
            kv_load8<TC, true>(reinterpret_cast<const TC *>(src) + e, v[c]);
            continue;
        }
        const uint2 q = __ldg(reinterpret_cast<const uint2 *>(src + e));
        const int sb = __ldg(src + L + 2 * MOE_KV_ROPE + e / KV_GROUP);
        const float sc = sb == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)sb << 23);
        kv_e4m3x4(q.x, &v[c][0]);
        kv_e4m3x4(q.y, &v[c][4]);
#pragma unroll
        for (int k = 0; k < 8; k++) v[c][k] *= sc;
    }
    float ra = 0.0f, rb = 0.0f;
    if (at >= 0) {
        ra = KvType<TC>::to_f(srope[2 * lane]);
        rb = KvType<TC>::to_f(srope[2 * lane + 1]);
    }
#pragma unroll
    for (int c = 0; c < KV_CHUNKS; c++) {
        const int e = c * 256 + lane * 8;
        if (e < L) kv_store8<TO, VEC>(dst + e, v[c]);
    }
    dst[L + 2 * lane] = KvType<TO>::from_f(ra);
    dst[L + 2 * lane + 1] = KvType<TO>::from_f(rb);
}

bool aligned16(const void *p, long long bytes) { return ((uintptr_t)p & 15) == 0 && (bytes & 15) == 0; }

size_t type_size(int type) { return type == MOE_TYPE_F32 ? 4 : 2; }

template <typename F>
void by_type(int type, F &&f) {
    if (type == MOE_TYPE_F32) f(float());
    else if (type == MOE_TYPE_F16) f(__half());
    else f(__nv_bfloat16());
}

}  // namespace

void moe_launch_rope(const MoeRopeDev &rope, const void *x, int x_type, long long xt, long long xh, void *y,
                     int y_type, long long yt, long long yh, const int *pos, int n_tokens, int n_heads, int head_dim,
                     int offset, cudaStream_t s, uint64_t *launches) {
    if (n_tokens <= 0 || n_heads <= 0) return;
    RopeArgs a{x, y, xt, xh, yt, yh, pos, n_heads, head_dim, offset, 0, 0, 0};
    a.in_place = x == y;
    const size_t xs = type_size(x_type), ys = type_size(y_type);
    // Whole 8-element vectors when every block of 8 starts on 16 bytes and no
    // block holds both rotated and copied dims; else element by element.
    const bool vec = aligned16(x, xt * xs) && aligned16(y, yt * ys) && (xh * xs) % 16 == 0 && (yh * ys) % 16 == 0 &&
                     head_dim % 8 == 0 && offset % 8 == 0 && rope.pairs % (rope.half_layout ? 8 : 4) == 0;
    const int w = vec ? 8 : 1, m = rope.pairs;
    const int rot = rope.half_layout ? m / w : (vec ? 2 * m / w : m);
    a.units = n_heads * (rot + (a.in_place ? 0 : (head_dim - 2 * m) / w));
    // Up to 16 units per thread (the angles of a CTA are formed once for
    // them), fewer while that leaves SMs without a CTA.
    int k = 16;
    while (k > 1 && (long long)n_tokens * ((a.units + RP_THREADS * k - 1) / (RP_THREADS * k)) < 148 * 4) k >>= 1;
    a.units_per_cta = RP_THREADS * k;
    const dim3 grid(n_tokens, (a.units + a.units_per_cta - 1) / a.units_per_cta);
    by_type(x_type, [&](auto ti) {
        by_type(y_type, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            if (vec) k_rope<TI, TO, true><<<grid, RP_THREADS, 0, s>>>(a, rope);
            else k_rope<TI, TO, false><<<grid, RP_THREADS, 0, s>>>(a, rope);
        });
    });
    LAUNCH_COUNT(launches);
}

template <typename T, typename F>
static void by_format(int fmt, F &&f) {
    if (fmt == MOE_KV_F16) f(T(), __half(), std::false_type());
    else if (fmt == MOE_KV_BF16) f(T(), __nv_bfloat16(), std::false_type());
    else if (fmt == MOE_KV_FP8_F16) f(T(), __half(), std::true_type());
    else f(T(), __nv_bfloat16(), std::true_type());
}

void moe_launch_kv_write(const MoeKvDev &kv, const MoeKvBatchDev &b, const void *x, int type, long long stride,
                         const float *norm_w, float eps, const MoeRopeDev *rope, const int *pos, int *error,
                         cudaStream_t s, uint64_t *launches) {
    if (b.n_tokens <= 0 || b.n_seqs <= 0) return;
    const int grid = (b.n_tokens + KV_WARPS - 1) / KV_WARPS;
    const bool vec = aligned16(x, stride * type_size(type)) && ((uintptr_t)norm_w & 15) == 0;
    MoeRopeDev none{};
    const MoeRopeDev &r = rope ? *rope : none;
    const int rotate = rope ? 1 : 0;
    by_type(type, [&](auto ti) {
        by_format<decltype(ti)>(kv.format, [&](auto t, auto tc, auto fp8) {
            using TI = decltype(t);
            using TC = decltype(tc);
            constexpr bool F = decltype(fp8)::value;
            const TI *p = reinterpret_cast<const TI *>(x);
            if (vec) k_kv_write<TI, TC, F, true><<<grid, KV_WARPS * 32, 0, s>>>(kv, b, p, stride, norm_w, eps, rotate, r, pos, error);
            else k_kv_write<TI, TC, F, false><<<grid, KV_WARPS * 32, 0, s>>>(kv, b, p, stride, norm_w, eps, rotate, r, pos, error);
        });
    });
    LAUNCH_COUNT(launches);
}

void moe_launch_kv_read(const MoeKvDev &kv, const MoeKvBatchDev &b, void *y, int type, long long stride, int *error,
                        cudaStream_t s, uint64_t *launches) {
    if (b.n_tokens <= 0 || b.n_seqs <= 0) return;
    const int grid = (b.n_tokens + KV_WARPS - 1) / KV_WARPS;
    const bool vec = aligned16(y, stride * type_size(type));
    by_type(type, [&](auto to) {
        by_format<decltype(to)>(kv.format, [&](auto t, auto tc, auto fp8) {
            using TO = decltype(t);
            using TC = decltype(tc);
            constexpr bool F = decltype(fp8)::value;
            TO *p = reinterpret_cast<TO *>(y);
            if (vec) k_kv_read<TO, TC, F, true><<<grid, KV_WARPS * 32, 0, s>>>(kv, b, p, stride, error);
            else k_kv_read<TO, TC, F, false><<<grid, KV_WARPS * 32, 0, s>>>(kv, b, p, stride, error);
        });
    });
    LAUNCH_COUNT(launches);
}
