// moe_mla.cu -- absorbed MLA attention of drafted tokens over the paged
// latent cache (mla_forward, infer.m:665-903, whose decode step is the case of
// one token): scores of every row that a token sees, softmax, the weighted
// mean of the rows' latent parts, for all heads of a token over one cached row.
#include "moe_kv.cuh"

#define LAUNCH_COUNT(p) \
    do {                \
        if (p) (*(p))++; \
    } while (0)

namespace {

constexpr int MS_HEADS = 16, MS_ROWS = 16, MS_THREADS = 256;

// Whether the token numbered `i` of its sequence sees row `pos`.
__device__ __forceinline__ bool mla_sees(const MoeMlaQuery &q, int token, int i, long long pos, int ctx, int n) {
    if (pos < ctx) return true;
    const long long j = pos - ctx;
    if (j >= n) return false;
    if (!q.tree) return j <= i;
    return j < 32ll * q.tree_words && (__ldg(q.tree + (size_t)token * q.tree_words + (j >> 5)) >> (j & 31) & 1);
}

// One CTA per (token, 16 heads): 16 cache rows at a time decoded to fp32 in
// shared memory, one (head, row) score per thread, a running maximum and sum
// per head, the output in registers (2 latent values of all 16 heads a thread).
template <typename TC, bool FP8>
__global__ void __launch_bounds__(MS_THREADS) k_mla(MoeKvDev kv, MoeKvBatchDev b, MoeMlaQuery q, int *error) {
    extern __shared__ float sm[];
    const int L = kv.latent, W = L + MOE_KV_ROPE, tid = threadIdx.x;
    float *sq = sm, *sk = sq + MS_HEADS * W, *sp = sk + MS_ROWS * (W + 1), *sm_m = sp + MS_HEADS * MS_ROWS,
          *sm_c = sm_m + MS_HEADS, *sm_l = sm_c + MS_HEADS;
    __shared__ int seen[MS_ROWS];
    const int t = blockIdx.x, h0 = blockIdx.y * MS_HEADS;
    const int seq = kv_seq_of(b, t);
    if (seq < 0) return;
    const int i = t - b.q_start[seq], n = b.q_start[seq + 1] - b.q_start[seq], ctx = b.ctx_len[seq];
    const long long len = max((long long)ctx + n, 0ll);
    for (int e = tid; e < MS_HEADS * W; e += MS_THREADS) {
        const int h = e / W, d = e % W;
        float v = 0.0f;
        if (h0 + h < q.n_heads) {
            const TC *p = d < L ? (const TC *)q.latent + t * q.lt + (h0 + h) * q.lh + d
                                : (const TC *)q.rope + t * q.rt + (h0 + h) * q.rh + d - L;
            v = KvType<TC>::to_f(*p);
        }
        sq[e] = v;
    }
    if (tid < MS_HEADS) sm_m[tid] = -INFINITY, sm_l[tid] = 0.0f;
    float acc[MS_HEADS][2] = {};
    const int hh = tid / MS_ROWS, r = tid % MS_ROWS;
    for (long long r0 = 0; r0 < len; r0 += MS_ROWS) {
        __syncthreads();
        if (tid < MS_ROWS) {
            const long long pos = r0 + tid;
            const bool s = pos < len && mla_sees(q, t, i, pos, ctx, n);
            const long long at = s ? kv_flat_row(kv, b, seq, pos) : -1;
            if (s && at < 0) kv_error(error, KV_ERR_BATCH);
            seen[tid] = (int)at;
        }
        __syncthreads();
        for (int e = tid; e < MS_ROWS * W; e += MS_THREADS) {
            const int k = e / W, d = e % W;
            float v = 0.0f;
            if (seen[k] >= 0) {
                const uint8_t *row = kv.data + (size_t)seen[k] * kv.row_bytes;
                if (!FP8) v = KvType<TC>::to_f(((const TC *)row)[d]);
                else if (d >= L) v = KvType<TC>::to_f(((const TC *)(row + L))[d - L]);
                else {
                    float w4[4];
                    kv_e4m3x4(row[d], w4);
                    const int sb = row[L + 2 * MOE_KV_ROPE + d / KV_GROUP];
                    v = w4[0] * (sb == 255 ? __uint_as_float(0x7FC00000u) : __uint_as_float((uint32_t)sb << 23));
                }
            }
            sk[k * (W + 1) + d] = v;
        }
        __syncthreads();
        float s = 0.0f;
        for (int d = 0; d < W; d++) s = fmaf(sq[hh * W + d], sk[r * (W + 1) + d], s);
        s = seen[r] >= 0 ? s * q.scale : -INFINITY;
        float m = s;
        for (int o = MS_ROWS / 2; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        const float old = sm_m[hh], nm = fmaxf(old, m), ref = nm == -INFINITY ? 0.0f : nm;
        const float p = expf(s - ref), c = expf(old - ref);
        float l = p;
        for (int o = MS_ROWS / 2; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        sp[hh * MS_ROWS + r] = p;
        __syncwarp();
        if (r == 0) sm_m[hh] = nm, sm_c[hh] = c, sm_l[hh] = sm_l[hh] * c + l;
        __syncthreads();
#pragma unroll
        for (int h = 0; h < MS_HEADS; h++) {
            const float f = sm_c[h];
            acc[h][0] *= f;
            acc[h][1] *= f;
        }
        for (int k = 0; k < MS_ROWS; k++) {
            if (seen[k] < 0) continue;
            const float v0 = tid < L ? sk[k * (W + 1) + tid] : 0.0f;
            const float v1 = tid + MS_THREADS < L ? sk[k * (W + 1) + tid + MS_THREADS] : 0.0f;
#pragma unroll
            for (int h = 0; h < MS_HEADS; h++) {
                const float pk = sp[h * MS_ROWS + k];
                acc[h][0] = fmaf(pk, v0, acc[h][0]);
                acc[h][1] = fmaf(pk, v1, acc[h][1]);
            }
        }
    }
    __syncthreads();
#pragma unroll
    for (int h = 0; h < MS_HEADS; h++) {
        if (h0 + h >= q.n_heads) break;
        const float l = sm_l[h], f = l == 0.0f ? 0.0f : 1.0f / l;
        TC *o = (TC *)q.out + t * q.ot + (h0 + h) * q.oh;
        if (tid < L) o[tid] = KvType<TC>::from_f(acc[h][0] * f);
        if (tid + MS_THREADS < L) o[tid + MS_THREADS] = KvType<TC>::from_f(acc[h][1] * f);
        if (tid == 0 && q.lse) q.lse[(size_t)t * q.n_heads + h0 + h] = l == 0.0f ? -INFINITY : sm_m[h] + logf(l);
    }
}

}  // namespace

size_t moe_mla_ws_bytes(int latent, int sms) { return 256; }

int moe_launch_mla(const MoeKvDev &kv, const MoeKvBatchDev &b, const MoeMlaQuery &q, void *ws, int sms, int *error,
                   cudaStream_t s, uint64_t *launches) {
    const int W = kv.latent + MOE_KV_ROPE;
    const size_t smem = sizeof(float) * (MS_HEADS * W + MS_ROWS * (W + 1) + MS_HEADS * MS_ROWS + 3 * MS_HEADS);
    const dim3 grid(b.n_tokens, (q.n_heads + MS_HEADS - 1) / MS_HEADS);
    static size_t d0[MOE_MAX_DEVICES], d1[MOE_MAX_DEVICES], d2[MOE_MAX_DEVICES], d3[MOE_MAX_DEVICES];
    switch (kv.format) {
        case MOE_KV_F16: moe_smem_limit(k_mla<__half, false>, smem, d0); k_mla<__half, false><<<grid, MS_THREADS, smem, s>>>(kv, b, q, error); break;
        case MOE_KV_BF16: moe_smem_limit(k_mla<__nv_bfloat16, false>, smem, d1); k_mla<__nv_bfloat16, false><<<grid, MS_THREADS, smem, s>>>(kv, b, q, error); break;
        case MOE_KV_FP8_F16: moe_smem_limit(k_mla<__half, true>, smem, d2); k_mla<__half, true><<<grid, MS_THREADS, smem, s>>>(kv, b, q, error); break;
        default: moe_smem_limit(k_mla<__nv_bfloat16, true>, smem, d3); k_mla<__nv_bfloat16, true><<<grid, MS_THREADS, smem, s>>>(kv, b, q, error);
    }
    LAUNCH_COUNT(launches);
    return 0;
}
