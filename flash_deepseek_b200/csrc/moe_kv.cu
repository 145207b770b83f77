// moe_kv.cu -- rotary positions, and the rows of the paged latent cache
// written and read back (formats in moe_kv.cuh).  All three are bound by the
// bytes they move; apply_rope_q / apply_rope_k (infer.m:628-656) and the
// cache append of mla_forward (infer.m:665-675, 760-790) are the reference's
// counterparts, one token at a time.
#include <type_traits>

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
// and read from shared memory by all heads.  4096 tokens x 128 heads x 192
// bf16: 85 us, 4.7 TB/s.
// ---------------------------------------------------------------------------
constexpr int RP_THREADS = 256;
constexpr int RP_PAIRS = 128;
// units of a thread in flight: 1 / 2 / 3 / 4 / 6 took 108 / 90 / 85 / 98 / 105 us for 4096 tokens x 128 heads x 192 bf16
constexpr int RP_UNITS = 3;

struct RopeArgs {
    const void *x;
    void *y;
    long long xt, xh, yt, yh;   // strides in elements: token, head
    const int *pos;
    int n_tokens, n_heads, head_dim, offset;
    int in_place;
    int units;                  // work units of one token
    int parts;                  // work items of one token
};

// A unit is 8 elements (4 interleaved pairs, or copied ones), or 8 of the first half together with their 8 partners
// in the second.  U units of a thread are loaded before the first is stored; CTAs walk over (token, part) items and
// form the next item's angles while this one's loads are under way.
template <typename TI, typename TO, int U, bool IN_PLACE>
__global__ void __launch_bounds__(RP_THREADS) k_rope(RopeArgs a, MoeRopeDev rope) {
    __shared__ float cs[2][RP_PAIRS], sn[2][RP_PAIRS];
    const int m = rope.pairs, items = a.n_tokens * a.parts, tid = threadIdx.x;
    const bool half = rope.half_layout != 0;
    const int rot = half ? m / 8 : m / 4, per = rot + (a.in_place ? 0 : (a.head_dim - 2 * m) / 8);
    const int first = blockIdx.x;
    auto angles = [&](int item, int buf) {
        if (tid < m && item < items)
            kv_cos_sin(__ldg(a.pos + item / a.parts), rope.turns[tid], rope.mscale, cs[buf][tid], sn[buf][tid]);
    };
    angles(first, 0);
    for (int item = first, buf = 0; item < items; item += gridDim.x, buf ^= 1) {
        __syncthreads();   // the item's angles are there, the other buffer is read
        const int t = item / a.parts, part = item - t * a.parts;
        const TI *x = reinterpret_cast<const TI *>(a.x) + (long long)t * a.xt;
        TO *y = reinterpret_cast<TO *>(a.y) + (long long)t * a.yt;
        const int lo = (int)((long long)a.units * part / a.parts), hi = (int)((long long)a.units * (part + 1) / a.parts);
        bool next = true;
        for (int u0 = lo + tid; u0 < hi || next; u0 += RP_THREADS * U) {
            KvRaw8<TI> f[U], g[U];
            int at[U], hd[U];
#pragma unroll
            for (int k = 0; k < U; k++) {
                const int u = u0 + k * RP_THREADS;
                if (u >= hi) continue;
                const int h = u / per, j = u - h * per;
                int e = j < rot ? a.offset + j * 8 : (j - rot) * 8;
                if (j >= rot && e >= a.offset) e += 2 * m;
                hd[k] = h;
                at[k] = j < rot ? e : ~e;   // copied: below zero
                kv_load_raw<TI, IN_PLACE>(x + h * a.xh + e, f[k]);
                if (half && j < rot) kv_load_raw<TI, IN_PLACE>(x + h * a.xh + e + m, g[k]);
            }
            if (next) angles(item + gridDim.x, buf ^ 1);
            next = false;
#pragma unroll
            for (int k = 0; k < U; k++) {
                if (u0 + k * RP_THREADS >= hi) continue;
                const bool turn = at[k] >= 0;
                const int e = turn ? at[k] : ~at[k], i = e - a.offset;
                TO *py = y + hd[k] * a.yh + e;
                float v[8];
                kv_unraw<TI>(f[k], v);
                if (turn && half) {
                    float w[8];
                    kv_unraw<TI>(g[k], w);
#pragma unroll
                    for (int j = 0; j < 8; j++) {
                        const float c = cs[buf][i + j], s = sn[buf][i + j], b = v[j];
                        v[j] = b * c - w[j] * s;
                        w[j] = b * s + w[j] * c;
                    }
                    kv_store8<TO, true>(py + m, w);
                } else if (turn) {
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        const float c = cs[buf][i / 2 + j], s = sn[buf][i / 2 + j], b = v[2 * j];
                        v[2 * j] = b * c - v[2 * j + 1] * s;
                        v[2 * j + 1] = b * s + v[2 * j + 1] * c;
                    }
                }
                kv_store8<TO, true>(py, v);
            }
        }
    }
}

// element by element, for rows that do not start on 16 bytes or blocks that hold rotated and copied values
template <typename TI, typename TO>
__global__ void __launch_bounds__(RP_THREADS) k_rope_any(RopeArgs a, MoeRopeDev rope) {
    __shared__ float cs[RP_PAIRS], sn[RP_PAIRS];
    const int m = rope.pairs, t = blockIdx.x / a.parts, part = blockIdx.x - t * a.parts;
    if ((int)threadIdx.x < m) kv_cos_sin(__ldg(a.pos + t), rope.turns[threadIdx.x], rope.mscale, cs[threadIdx.x], sn[threadIdx.x]);
    __syncthreads();
    const TI *x = reinterpret_cast<const TI *>(a.x) + (long long)t * a.xt;
    TO *y = reinterpret_cast<TO *>(a.y) + (long long)t * a.yt;
    const bool half = rope.half_layout != 0;
    const int per = m + (a.in_place ? 0 : a.head_dim - 2 * m);
    const int lo = (int)((long long)a.units * part / a.parts), hi = (int)((long long)a.units * (part + 1) / a.parts);
    for (int u = lo + threadIdx.x; u < hi; u += RP_THREADS) {
        const int h = u / per, j = u - h * per;
        const TI *px = x + h * a.xh;
        TO *py = y + h * a.yh;
        if (j < m) {
            const int e = a.offset + (half ? j : 2 * j), f = e + (half ? m : 1);
            const float p = KvType<TI>::to_f(px[e]), q = KvType<TI>::to_f(px[f]), c = cs[j], s = sn[j];
            py[e] = KvType<TO>::from_f(p * c - q * s);
            py[f] = KvType<TO>::from_f(p * s + q * c);
        } else {
            int e = j - m;
            if (e >= a.offset) e += 2 * m;
            py[e] = KvType<TO>::from_f(KvType<TI>::to_f(px[e]));
        }
    }
}

// ---------------------------------------------------------------------------
// Cache rows.  One warp per row: a lane holds 8 consecutive latent values of
// every 256 (so a group of 32 is 4 lanes, and loads and stores of a warp are
// contiguous) and one rotary pair.  32,762 fp32 rows into 8 bits: 25 us (3.9
// TB/s); 130,000 8-bit rows out as bf16: 39 to 42 us by box (6.0 to 5.7 TB/s).
// ---------------------------------------------------------------------------
constexpr int KV_WARPS = 4;
// rows of a reading warp in flight: 1 / 2 / 3 / 4 took 43.4 / 39.4 / 39.6 / 39.5 us for 130,000 8-bit rows on one box
constexpr int KV_RPW = 2;
constexpr int KV_CHUNKS = 2;   // 256-value chunks of the widest latent part (512)

__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// One row per warp: the row's own loads are issued before the page lookup, which waits for three dependent ones.  (Two
// rows per warp as in the read: 28.8 against 25.0 us for 32,762 fp32 rows into 8 bits; more registers, fewer warps.)
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

// the flat row of row t0 + lane of a warp's RPW rows: -2 in no sequence, -1 (reported) without a page
template <int RPW>
__device__ __forceinline__ long long kv_lookup(const MoeKvDev &kv, const MoeKvBatchDev &b, int t0, int lane, int *error) {
    const int t = t0 + lane;
    if (lane >= RPW || t >= b.n_tokens) return -2;
    const int seq = kv_seq_of(b, t);
    if (seq < 0) return -2;
    const long long at = kv_flat_row(kv, b, seq, (long long)__ldg(b.ctx_len + seq) + (t - __ldg(b.q_start + seq)));
    if (at < 0) kv_error(error, KV_ERR_BATCH);
    return at;
}

// A warp reads RPW rows, all of their loads in front of the first store; lane k looks up row k.
template <typename TO, typename TC, bool FP8, bool VEC, int RPW>
__global__ void __launch_bounds__(KV_WARPS * 32) k_kv_read(MoeKvDev kv, MoeKvBatchDev b, TO *__restrict__ y,
                                                           long long stride, int *error) {
    const int t0 = (blockIdx.x * KV_WARPS + (threadIdx.x >> 5)) * RPW, lane = threadIdx.x & 31;
    if (t0 >= b.n_tokens) return;
    const int L = kv.latent;
    const long long found = kv_lookup<RPW>(kv, b, t0, lane, error);   // -1: the row reads as zeros
    uint4 q[RPW][KV_CHUNKS];
    int sb[RPW][KV_CHUNKS];
    uint32_t rp[RPW];
#pragma unroll
    for (int k = 0; k < RPW; k++) {
        const long long at = __shfl_sync(0xffffffffu, found, k);
        const uint8_t *src = kv.data + (at < 0 ? 0 : at) * kv.row_bytes;
        rp[k] = at < 0 ? 0u : __ldg(reinterpret_cast<const uint32_t *>(src + (FP8 ? L : 2 * L)) + lane);
#pragma unroll
        for (int c = 0; c < KV_CHUNKS; c++) {
            const int e = c * 256 + lane * 8;
            const bool in = e < L && at >= 0;
            q[k][c] = make_uint4(0, 0, 0, 0);
            sb[k][c] = 127;
            if (in && !FP8) q[k][c] = __ldg(reinterpret_cast<const uint4 *>(src + 2 * e));
            if (in && FP8) {
                const uint2 h = __ldg(reinterpret_cast<const uint2 *>(src + e));
                q[k][c].x = h.x, q[k][c].y = h.y;
                sb[k][c] = __ldg(src + L + 2 * MOE_KV_ROPE + e / KV_GROUP);
            }
        }
    }
#pragma unroll
    for (int k = 0; k < RPW; k++) {
        if (__shfl_sync(0xffffffffu, found, k) == -2) continue;   // left as it is
        TO *dst = y + (long long)(t0 + k) * stride;
#pragma unroll
        for (int c = 0; c < KV_CHUNKS; c++) {
            const int e = c * 256 + lane * 8;
            if (e >= L) continue;
            float v[8];
            if (FP8) {
                const int x = sb[k][c];
                const float sc = x == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)x << 23);
                kv_e4m3x4(q[k][c].x, &v[0]);
                kv_e4m3x4(q[k][c].y, &v[4]);
#pragma unroll
                for (int j = 0; j < 8; j++) v[j] *= sc;
            } else {
                kv_unraw<TC>(reinterpret_cast<const KvRaw8<TC> &>(q[k][c]), v);
            }
            kv_store8<TO, VEC>(dst + e, v);
        }
        const TC *h = reinterpret_cast<const TC *>(&rp[k]);
        dst[L + 2 * lane] = KvType<TO>::from_f(KvType<TC>::to_f(h[0]));
        dst[L + 2 * lane + 1] = KvType<TO>::from_f(KvType<TC>::to_f(h[1]));
    }
}

// rows of a warp: KV_RPW once that leaves every SM 16 warps, else 1 (a short call is all latency)
int rows_per_warp(int rows, int sms) { return rows >= KV_RPW * 16 * sms ? KV_RPW : 1; }

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
                     int offset, int sms, cudaStream_t s, uint64_t *launches) {
    if (n_tokens <= 0 || n_heads <= 0) return;
    RopeArgs a{x, y, xt, xh, yt, yh, pos, n_tokens, n_heads, head_dim, offset, x == y, 0, 1};
    const size_t xs = type_size(x_type), ys = type_size(y_type);
    // Whole 8-element vectors when every block of 8 starts on 16 bytes and no
    // block holds both rotated and copied values; else element by element.
    const bool vec = aligned16(x, xt * xs) && aligned16(y, yt * ys) && (xh * xs) % 16 == 0 && (yh * ys) % 16 == 0 &&
                     head_dim % 8 == 0 && offset % 8 == 0 && rope.pairs % (rope.half_layout ? 8 : 4) == 0;
    const int w = vec ? 8 : 1, m = rope.pairs;
    const int rot = vec ? (rope.half_layout ? m / 8 : m / 4) : m;
    a.units = n_heads * (rot + (a.in_place ? 0 : (head_dim - 2 * m) / w));
    // A token is one work item, or parts of RP_THREADS units where tokens alone leave SMs without work (and at most
    // some 8 units per thread, so that the last items end together)
    const int most = (a.units + RP_THREADS - 1) / RP_THREADS;
    a.parts = (a.units + RP_THREADS * 8 - 1) / (RP_THREADS * 8);
    while (a.parts < most && (long long)n_tokens * a.parts < 8 * sms) a.parts++;
    const long long items = (long long)n_tokens * a.parts;
    by_type(x_type, [&](auto ti) {
        by_type(y_type, [&](auto to) {
            using TI = decltype(ti);
            using TO = decltype(to);
            const unsigned ctas = (unsigned)(items < 8 * sms ? items : 8 * sms);
            constexpr bool SAME = std::is_same<TI, TO>::value;   // in place: the same type (checked by the caller)
            if (vec && a.in_place) k_rope<TI, TO, RP_UNITS, SAME><<<ctas, RP_THREADS, 0, s>>>(a, rope);
            else if (vec) k_rope<TI, TO, RP_UNITS, false><<<ctas, RP_THREADS, 0, s>>>(a, rope);
            else k_rope_any<TI, TO><<<(unsigned)items, RP_THREADS, 0, s>>>(a, rope);
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
    const bool vec = aligned16(x, stride * type_size(type)) && ((uintptr_t)norm_w & 15) == 0;
    const int grid = (b.n_tokens + KV_WARPS - 1) / KV_WARPS;
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

void moe_launch_kv_read(const MoeKvDev &kv, const MoeKvBatchDev &b, void *y, int type, long long stride, int sms,
                        int *error, cudaStream_t s, uint64_t *launches) {
    if (b.n_tokens <= 0 || b.n_seqs <= 0) return;
    const bool vec = aligned16(y, stride * type_size(type));
    const int rpw = rows_per_warp(b.n_tokens, sms), grid = (b.n_tokens + KV_WARPS * rpw - 1) / (KV_WARPS * rpw);
    by_type(type, [&](auto to) {
        by_format<decltype(to)>(kv.format, [&](auto t, auto tc, auto fp8) {
            using TO = decltype(t);
            using TC = decltype(tc);
            constexpr bool F = decltype(fp8)::value;
            TO *p = reinterpret_cast<TO *>(y);
            auto kernel = rpw == 1 ? (vec ? k_kv_read<TO, TC, F, true, 1> : k_kv_read<TO, TC, F, false, 1>)
                                   : (vec ? k_kv_read<TO, TC, F, true, KV_RPW> : k_kv_read<TO, TC, F, false, KV_RPW>);
            kernel<<<grid, KV_WARPS * 32, 0, s>>>(kv, b, p, stride, error);
        });
    });
    LAUNCH_COUNT(launches);
}
