// moe_mla.cu -- absorbed MLA attention of drafted tokens over the paged
// latent cache (mla_forward, infer.m:665-903, whose decode step is the case of
// one token), on the fifth-generation tensor cores.
//
// Mathematics.  For a query row q (one head of one token) and the cache rows
// r that its token sees: s_r = scale * q . k_r over latent + 64 values,
// out = sum_r e^(s_r - m) c_r / sum_r e^(s_r - m), c_r the latent part of k_r.
// One pass over the cache with a running reference m: all heads of a token
// share the rows, so 128 query rows (MLA_M) meet tiles of 64 cache rows.
//
// Why this split.  The output of 128 rows in fp32 (512 columns) would fill
// tensor memory, so two CTAs share a block of query rows, each with half of
// the latent columns of the output (256 columns) and the whole of the scores,
// which both compute: 832 / 1088 of the products of one row a CTA, but no
// exchange between the CTAs.  The query block does not fit shared memory
// beside the cache tiles either: its first chunks live in tensor memory (the
// A operand of the score product may come from there), the rest in shared
// memory.  Both CTAs of a pair walk over the same tiles at the same time, so
// the second read of a tile comes from L2.
//
// A CTA: one warp loads (TMA, one box per page piece; the 8-bit formats: 8
// warps that load codes, expand them to 16 bits exactly and write the
// swizzled tile), one issues the MMAs, four hold one query row per thread
// (softmax, output).  Order on the tensor pipe: scores of tile i + 1, then
// the output product of tile i, so the softmax of one tile runs under the
// products of its neighbours.  A tile's latent chunks of this CTA's half stay
// until its output product is done (ring B, 3 tiles); the other half and the
// rotary chunk are only scores' operands and leave chunk by chunk (ring A).
// Work division: moe_kv_plan.h; cut units are joined by k_mla_join.
#include "moe_common.cuh"
#include "moe_kv.cuh"
#include "moe_kv_plan.h"
#include "moe_umma.cuh"

#define LAUNCH_COUNT(p) \
    do {                \
        if (p) (*(p))++; \
    } while (0)

namespace {

constexpr int MLA_CHUNK = MLA_N * 128;      // bytes of a 64-row x 64-value chunk
constexpr int MLA_QCHUNK = MLA_M * 128;     // bytes of a 128-row x 64-value query chunk
constexpr int MLA_RA = 8;                   // chunks of ring A
constexpr int MLA_SB = 3;                   // tiles of ring B
constexpr int MLA_TM_S = 256, MLA_TM_P = 320, MLA_TM_Q = 352;   // tensor-memory columns (the output from 0)
constexpr float MLA_RAISE = 8.0f;           // log2: how far scores may pass the reference before it is raised

// Tensor memory left for query chunks of 32 columns (64 values) each: all of
// them for up to 384 latent values, 5 of 9 for 512.
__host__ __device__ constexpr int mla_q_tm(int latent) {
    const int all = latent / 64 + 1, fit = (512 - MLA_TM_Q + (256 - latent / 2)) / 32;
    return all < fit ? all : fit;
}

struct MlaCtl {   // control block behind the tiles
    uint64_t full_a[MLA_RA], empty_a[MLA_RA], full_b[MLA_SB], empty_b[MLA_SB];
    uint64_t s_full, s_empty, p_full, pv_done, q_ready, drain;
    uint64_t nonfinite[2];       // by tile parity: rows of a tile with an infinity or a NaN in this CTA's latent half
    uint8_t valid[MLA_SB][8];    // 8-row groups of a tile whose page exists
    int64_t w0, w1, off0;        // the pair's share: first and last tile, place of the first in its sequence
    int64_t scan[32];
    int64_t total;
    int seq0;
    uint32_t tmem;
    int dead;                    // a bounded wait gave up
};

// Pieces of cut units: [pair][slot][latent][128 rows] sums, [pair][slot][2][128] references and sums of weights
struct MlaWs {
    struct Tail {                // the unit that pair p begins and does not end
        int seq, block, last, on;
    } *tail;
    float *ml, *o;
};

__host__ __device__ MlaWs mla_ws(void *ws, int latent, int pairs) {
    MlaWs w;
    uint8_t *b = reinterpret_cast<uint8_t *>(ws);
    w.tail = reinterpret_cast<MlaWs::Tail *>(b);
    b += ((size_t)pairs * sizeof(MlaWs::Tail) + 255) / 256 * 256;
    w.ml = reinterpret_cast<float *>(b);
    b += (size_t)pairs * 2 * 2 * MLA_M * sizeof(float);
    w.o = reinterpret_cast<float *>(b);
    return w;
}

struct MlaSeqAt {
    MoeKvBatchDev b;
    int heads, page_shift;
    __device__ __forceinline__ MlaSeq operator()(int i) const {
        return mla_seq(__ldg(b.q_start + i), __ldg(b.q_start + i + 1), __ldg(b.ctx_len + i), b.n_tokens, heads,
                       (int64_t)b.pages_per_seq << page_shift);
    }
};

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// 4 e4m3 codes times a group's scale as 4 16-bit values.  The code's exponent
// and mantissa bits placed in the 16-bit format's fields are the value over
// 2^120 (bf16) or 2^8 (fp16), subnormals too; f holds 2^(120 + k) or 2^(8 + k).
template <bool BF16>
__device__ __forceinline__ uint2 expand4(uint32_t w, uint32_t f) {
    const uint32_t lo = __byte_perm(w, 0, 0x1404), hi = __byte_perm(w, 0, 0x3424);
    uint2 r;
    if (BF16) {
        r.x = (lo & 0x80008000u) | ((lo & 0x7F007F00u) >> 4);
        r.y = (hi & 0x80008000u) | ((hi & 0x7F007F00u) >> 4);
        asm("mul.bf16x2 %0, %0, %1;" : "+r"(r.x) : "r"(f));
        asm("mul.bf16x2 %0, %0, %1;" : "+r"(r.y) : "r"(f));
    } else {
        r.x = (lo & 0x80008000u) | ((lo & 0x7F007F00u) >> 1);
        r.y = (hi & 0x80008000u) | ((hi & 0x7F007F00u) >> 1);
        asm("mul.f16x2 %0, %0, %1;" : "+r"(r.x) : "r"(f));
        asm("mul.f16x2 %0, %0, %1;" : "+r"(r.y) : "r"(f));
    }
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t scale2(uint32_t sb) {
    const uint32_t h = sb == 255 ? 0x7FFFu : BF16 ? ((sb + 120) & 255) << 7 : ((sb - 104) & 31) << 10;
    return h | h << 16;
}

// 64 visibility bits of a row for tile rows pos0 .. pos0 + 63: below ctx all,
// from there on the token's tree bits (or a chain up to itself)
__device__ __forceinline__ uint64_t low_bits(int64_t n) { return n <= 0 ? 0 : n >= 64 ? ~0ull : (1ull << n) - 1; }
__device__ __forceinline__ uint32_t tree_word(const uint32_t *t, int64_t w, int words) {
    return w >= 0 && w < words ? __ldg(t + w) : 0u;
}
__device__ __forceinline__ uint64_t mla_visible(const MoeMlaQuery &q, const MlaSeq &s, int token, int64_t pos0) {
    const uint64_t old = low_bits(s.ctx - pos0), all = low_bits(s.len - pos0);
    if (!q.tree) return (old | low_bits((int64_t)s.ctx + token + 1 - pos0)) & all;
    const uint32_t *t = q.tree + (int64_t)(s.q0 + token) * q.tree_words;
    const int64_t j0 = pos0 - s.ctx;   // drafted row of bit 0 (may be negative, above -64 where it matters)
    uint64_t v;
    if (j0 <= -64) v = 0;
    else if (j0 < 0) v = (tree_word(t, 0, q.tree_words) | (uint64_t)tree_word(t, 1, q.tree_words) << 32) << -j0;
    else {
        const int64_t w = j0 >> 5;
        const int sh = (int)(j0 & 31);
        const uint64_t a = tree_word(t, w, q.tree_words) | (uint64_t)tree_word(t, w + 1, q.tree_words) << 32;
        v = a >> sh;
        if (sh) v |= (uint64_t)tree_word(t, w + 2, q.tree_words) << (64 - sh);
    }
    return (old | v) & all;
}

// ---------------------------------------------------------------------------
template <bool BF16, bool FP8>
struct MlaKernel {
    static constexpr int THREADS = FP8 ? 512 : 256;

    const MoeKvDev &kv;
    const MlaSeqAt &seq_at;
    const MoeMlaQuery &q;
    const CUtensorMap *tm;
    MlaWs ws;
    int *error;
    uint8_t *ring_b, *ring_a, *sq;
    MlaCtl *c;
    int half, pair, pairs, nv, nc, nq;   // latent chunks of a half, chunks of a row, query chunks in tensor memory
    int lane, warp;

    // the chunk (64 values of a row) at place p of the order: own half, other half, rotary
    __device__ __forceinline__ int chunk_at(int p) const {
        return p < nv ? half * nv + p : p < 2 * nv ? (1 - half) * nv + p - nv : 2 * nv;
    }
    __device__ __forceinline__ MlaWalk walk() const {
        MlaWalk w{};
        w.w = c->w0, w.w1 = c->w1, w.off = c->off0, w.seq = c->seq0, w.n_seqs = seq_at.b.n_seqs;
        return w;
    }
    __device__ __forceinline__ void give_up() {
        if (lane == 0) {
            c->dead = 1;
            kv_error(error, KV_ERR_TIMEOUT);
        }
    }
    __device__ __forceinline__ long long flat(int seq, const MlaSeq &s, int64_t pos) const {
        if (pos >= s.len) return -2;   // behind the sequence: no error
        return kv_flat_row(kv, seq_at.b, seq, pos);
    }

    // after a wait gave up: none of the copies issued so far may land after the CTA has ended
    __device__ void stop_tma(int ia, int ib) {
        give_up();
        tc_drain(c->full_a, ia, MLA_RA);
        tc_drain(c->full_b, ib, MLA_SB);
    }

    // ---- loads, 16-bit formats: lane j < 8 handles rows 8 j .. of a tile
    __device__ void produce_tma() {
        MlaWalk w = walk();
        MlaSeg g;
        int ia = 0, ib = 0;
        const int rows_box = min(1 << kv.page_shift, MLA_N);
        const int outside = kv.n_pages << kv.page_shift;   // a box there reads zeros
        while (w.next(g, seq_at)) {
            for (int t = g.tile0; t < g.tile1; t++, ib++) {
                const int st = ib % MLA_SB;
                int row = outside;
                bool ok = false;
                if (lane < 8) {
                    const long long f = flat(g.seq, w.s, (int64_t)t * MLA_N + lane * 8);
                    ok = f >= 0;
                    if (ok) row = (int)f;
                    if (f == -1) kv_error(error, KV_ERR_BATCH);
                }
                const bool box = lane < 8 && (lane * 8) % rows_box == 0;
                const int off = lane * 8 * 128;
                if (!tc_wait_warp(&c->empty_b[st], (ib / MLA_SB + 1) & 1)) return stop_tma(ia, ib);
                if (lane < 8) c->valid[st][lane] = ok;
                __syncwarp();
                if (lane == 0) tc_expect(&c->full_b[st], (uint32_t)nv * MLA_CHUNK);
                __syncwarp();
                if (box)
                    for (int p = 0; p < nv; p++)
                        tc_tma2(ring_b + (st * nv + p) * MLA_CHUNK + off, tm, chunk_at(p) * 64, row, &c->full_b[st]);
                for (int p = nv; p < nc; p++, ia++) {
                    const int sa = ia % MLA_RA;
                    if (!tc_wait_warp(&c->empty_a[sa], (ia / MLA_RA + 1) & 1)) return stop_tma(ia, ib + 1);
                    if (lane == 0) tc_expect(&c->full_a[sa], MLA_CHUNK);
                    __syncwarp();
                    if (box) tc_tma2(ring_a + sa * MLA_CHUNK + off, tm, chunk_at(p) * 64, row, &c->full_a[sa]);
                }
            }
        }
    }

    // ---- loads, 8-bit formats: 8 warps, 4 threads per row, 16 codes of every chunk each.  The next tile's
    // loads are issued as this tile's chunks are expanded, so a tile's bytes are always in flight.
    __device__ void produce_expand() {
        const int tid = threadIdx.x - 256, r = tid >> 2, qd = tid & 3, L = kv.latent;
        MlaWalk w = walk();
        MlaSeg g;
        int ia = 0, ib = 0;
        uint4 code[8], rope[2], sc;
        const uint4 zero = make_uint4(0, 0, 0, 0);
        // loads of tile t of the current segment
        const uint8_t *row;
        bool ok;
        auto locate = [&](int seq, const MlaSeq &s, int t) {
            const long long f = flat(seq, s, (int64_t)t * MLA_N + r);
            ok = f >= 0;
            if (f == -1) kv_error(error, KV_ERR_BATCH);
            row = ok ? kv.data + f * kv.row_bytes : nullptr;
        };
        auto load_sc = [&]() {
            sc = zero;
            if (!row) return;
            const uint32_t *p = reinterpret_cast<const uint32_t *>(row + L + 2 * MOE_KV_ROPE);
            sc.x = __ldg(p);
            if (L > 128) sc.y = __ldg(p + 1);
            if (L > 256) sc.z = __ldg(p + 2);
            if (L > 384) sc.w = __ldg(p + 3);
        };
        auto load_code = [&](int p) { return row ? __ldg(reinterpret_cast<const uint4 *>(row + chunk_at(p) * 64) + qd) : zero; };
        auto load_rope = [&](int k) { return row ? __ldg(reinterpret_cast<const uint4 *>(row + L) + 2 * qd + k) : zero; };
        if (!w.next(g, seq_at)) return;
        int t = g.tile0;
        locate(g.seq, w.s, t);
        load_sc();
#pragma unroll
        for (int p = 0; p < 8; p++)
            if (p < 2 * nv) code[p] = load_code(p);
        rope[0] = load_rope(0), rope[1] = load_rope(1);
        for (bool more = true; more; ib++) {
            const int st = ib % MLA_SB;
            const bool cur_ok = ok;
            const uint4 s4 = sc;
            // the next tile
            if (++t >= g.tile1) {
                more = w.next(g, seq_at);
                t = g.tile0;
            }
            if (more) {
                locate(g.seq, w.s, t);
                load_sc();
            } else {
                row = nullptr;
            }
            if (!tc_wait_warp(&c->empty_b[st], (ib / MLA_SB + 1) & 1)) return give_up();
            if (lane == 0) c->valid[st][warp - 8] = cur_ok;   // a warp holds the 8 rows of one group
            const uint32_t sw = (uint32_t)(r & 7);
            const uint32_t at = (uint32_t)(r >> 3) * 1024 + sw * 128;
#pragma unroll
            for (int p = 0; p < 9; p++) {
                if (p >= nc) break;
                uint8_t *dst;
                if (p < nv) dst = ring_b + (st * nv + p) * MLA_CHUNK;
                else {
                    const int sa = ia % MLA_RA;
                    if (!tc_wait_warp(&c->empty_a[sa], (ia / MLA_RA + 1) & 1)) return give_up();
                    dst = ring_a + sa * MLA_CHUNK;
                }
                uint4 lo, hi;
                if (p < 2 * nv) {
                    const uint4 v = code[p < 8 ? p : 7];
                    const int grp = 2 * chunk_at(p) + (qd >> 1);
                    const uint32_t word = grp < 4 ? s4.x : grp < 8 ? s4.y : grp < 12 ? s4.z : s4.w;
                    const uint32_t f = scale2<BF16>(word >> (8 * (grp & 3)) & 255);
                    const uint2 a = expand4<BF16>(v.x, f), b = expand4<BF16>(v.y, f);
                    const uint2 d = expand4<BF16>(v.z, f), e = expand4<BF16>(v.w, f);
                    lo = make_uint4(a.x, a.y, b.x, b.y);
                    hi = make_uint4(d.x, d.y, e.x, e.y);
                    if (p < 8) code[p] = load_code(p);
                } else {
                    lo = rope[0], hi = rope[1];
                    rope[0] = load_rope(0), rope[1] = load_rope(1);
                }
                if (!cur_ok) lo = zero, hi = zero;
                *reinterpret_cast<uint4 *>(dst + at + ((2 * qd) ^ sw) * 16) = lo;
                *reinterpret_cast<uint4 *>(dst + at + ((2 * qd + 1) ^ sw) * 16) = hi;
                fence_async_smem();
                __syncwarp();
                if (p >= nv) {
                    if (lane == 0) tc_arrive(&c->full_a[ia % MLA_RA]);
                    ia++;
                } else if (p == nv - 1) {
                    if (lane == 0) tc_arrive(&c->full_b[st]);
                }
            }
        }
    }

    // ---- MMA issue: one warp, every lane runs the loop, an elected lane issues
    __device__ void issue() {
        const uint32_t tmem = c->tmem;
        const uint32_t id_s = umma_idesc_16(MLA_M, MLA_N, BF16, 0), id_o = umma_idesc_16(MLA_M, kv.latent / 2, BF16, 1);
        MlaWalk w = walk();
        MlaSeg g;
        int ia = 0, it = 0, seg = 0;   // ring A chunks, tiles, segments so far
        auto output = [&](int i, bool first) -> bool {
            const int st = i % MLA_SB;
            if (!tc_wait_warp(&c->p_full, i & 1)) return false;
            tmem_fence_after();
            const uint64_t d = umma_desc_sw128_mn(umma_smem_u32(ring_b + st * nv * MLA_CHUNK), MLA_CHUNK);
#pragma unroll
            for (int k = 0; k < MLA_N / 16; k++)   // 16 cache rows: 2048 bytes of the tile, 8 columns of P
                umma_f16_ta_warp(tmem, tmem + MLA_TM_P + k * 8, d + k * (2048 >> 4), id_o, !(first && k == 0));
            umma_commit_warp(&c->empty_b[st]);
            umma_commit_warp(&c->pv_done);
            return true;
        };
        bool ok = true;
        while (ok && w.next(g, seq_at)) {
            ok = tc_wait_warp(&c->q_ready, seg & 1);
            seg++;
            if (!ok) break;
            for (int t = g.tile0; ok && t < g.tile1; t++, it++) {
                const int st = it % MLA_SB;
                ok = (it == 0 || tc_wait_warp(&c->s_empty, (it - 1) & 1)) && tc_wait_warp(&c->full_b[st], (it / MLA_SB) & 1);
                if (!ok) break;
                tmem_fence_after();
                for (int p = 0; p < nc; p++) {
                    const uint8_t *src;
                    if (p < nv) src = ring_b + (st * nv + p) * MLA_CHUNK;
                    else {
                        const int sa = ia % MLA_RA;
                        ok = tc_wait_warp(&c->full_a[sa], (ia / MLA_RA) & 1);
                        if (!ok) break;
                        src = ring_a + sa * MLA_CHUNK;
                    }
                    const uint64_t b = umma_desc_sw128(umma_smem_u32(src));
                    if (p < nq) {
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            umma_f16_ta_warp(tmem + MLA_TM_S, tmem + q_col(p) + k * 8, b + k * 2, id_s, p > 0 || k > 0);
                    } else {
                        const uint64_t a = umma_desc_sw128(umma_smem_u32(sq + (p - nq) * MLA_QCHUNK));
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            umma_f16_warp(tmem + MLA_TM_S, a + k * 2, b + k * 2, id_s, p > 0 || k > 0);
                    }
                    if (p >= nv) umma_commit_warp(&c->empty_a[ia++ % MLA_RA]);
                }
                if (!ok) break;
                umma_commit_warp(&c->s_full);
                if (t > g.tile0) ok = output(it - 1, t - 1 == g.tile0);
            }
            if (ok) ok = output(it - 1, g.tile1 - 1 == g.tile0);
        }
        if (!ok) give_up();
        // nothing of this warp's is in flight when the CTA ends
        umma_commit_warp(&c->drain);
        tc_wait_warp(&c->drain, 0);
    }
    // tensor-memory column of the query chunk at place p
    __device__ __forceinline__ uint32_t q_col(int p) const {
        // below 512 latent values the output takes fewer columns: the first chunks go behind it
        const int spare = (256 - kv.latent / 2) / 32;
        return p < spare ? kv.latent / 2 + p * 32 : MLA_TM_Q + (p - spare) * 32;
    }

    // ---- softmax and output: 4 warps, one query row per thread
    __device__ void rows() {
        const uint32_t tmem = c->tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const int r = (warp & 3) * 32 + lane, L = kv.latent, half_cols = L / 2;
        const float c2 = q.scale * 1.4426950408889634f;
        MlaWalk w = walk();
        MlaSeg g;
        int it = 0;
        bool ok = true;
        while (ok && w.next(g, seq_at)) {
            const MlaSeq s = w.s;
            const int64_t row = (int64_t)g.block * MLA_M + r;
            const bool live = row < (int64_t)s.n * q.n_heads;
            const int token = live ? (int)(row / q.n_heads) : 0, head = live ? (int)(row - (int64_t)token * q.n_heads) : 0;
            load_query(r, live, (int64_t)s.q0 + token, head);
            float ref = -INFINITY, l = 0.0f;
            for (int t = g.tile0; t < g.tile1; t++, it++) {
                const int st = it % MLA_SB;
                const int64_t pos0 = (int64_t)t * MLA_N;
                ok = tc_wait_warp(&c->s_full, it & 1);
                if (!ok) break;
                tmem_fence_after();
                float v[64];
                tmem_ld32(tmem + MLA_TM_S, *reinterpret_cast<float(*)[32]>(v));
                tmem_ld32(tmem + MLA_TM_S + 32, *reinterpret_cast<float(*)[32]>(v + 32));
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) tc_arrive(&c->s_empty);
                // a tile that reaches the drafted rows, or lacks a page: hide what the row does not see
                ok = tc_wait_warp(&c->full_b[st], (it / MLA_SB) & 1);   // long complete: orders the valid bytes
                if (!ok) break;
#pragma unroll
                for (int k = 0; k < 64; k++) v[k] *= c2;
                const uint64_t pages = *reinterpret_cast<const volatile uint64_t *>(c->valid[st]);
                if (pos0 + MLA_N > s.ctx || pages != 0x0101010101010101ull) {
                    uint64_t see = mla_visible(q, s, token, pos0) & pages * 255;
                    const uint64_t nf = clean(st, it & 1);
#pragma unroll
                    for (int k = 0; k < 64; k++) {
                        if (nf >> k & 1) v[k] = __uint_as_float(0x7FC00000u);
                        if (!(see >> k & 1)) v[k] = -INFINITY;
                    }
                }
                float mx[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
                for (int k = 4; k < 64; k++) mx[k & 3] = fmaxf(mx[k & 3], v[k]);
                const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3]));
                if (it > 0) {   // the previous output product is done: P may be written, the output rescaled
                    ok = tc_wait_warp(&c->pv_done, (it - 1) & 1);
                    if (!ok) break;
                    tmem_fence_after();
                }
                if (t == g.tile0) ref = top;
                else if (__any_sync(0xffffffffu, top > ref + MLA_RAISE)) {
                    // raise the reference: weights stay below 2^8 of it, so fp16 and bf16 hold them
                    const float m = fmaxf(ref, top), f = m == -INFINITY ? 1.0f : ex2(ref - m);
                    l *= f;
                    ref = m;
                    for (int col = 0; col < half_cols; col += 32) {
                        float o[32];
                        uint32_t u[32];
                        tmem_ld32(tmem + col, o);
#pragma unroll
                        for (int k = 0; k < 32; k++) u[k] = __float_as_uint(o[k] * f);
                        tmem_st32(tmem + col, u);
                    }
                    tmem_wait_st();
                }
                const float m0 = ref == -INFINITY ? 0.0f : ref;
                float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                uint32_t pk[32];
#pragma unroll
                for (int k = 0; k < 64; k += 2) {
                    const float a = ex2(v[k] - m0), b = ex2(v[k + 1] - m0);
                    sum[k & 2] += a;
                    sum[(k & 2) + 1] += b;
                    pk[k / 2] = pack2<BF16>(a, b);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                tmem_st32(tmem + MLA_TM_P, pk);
                tmem_wait_st();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) tc_arrive(&c->p_full);
            }
            if (!ok) break;
            ok = tc_wait_warp(&c->pv_done, (it - 1) & 1);
            if (!ok) break;
            tmem_fence_after();
            if (g.whole) store_out(tmem, live, (int64_t)s.q0 + token, head, ref, l);
            else store_piece(tmem, g, w, live, r, ref, l);
        }
        if (!ok) give_up();
    }

    // The query row into tensor memory and shared memory (zeros behind the block's last row)
    __device__ __forceinline__ void load_query(int r, bool live, int64_t token, int head) {
        const uint4 *ql = reinterpret_cast<const uint4 *>(reinterpret_cast<const __half *>(q.latent) + token * q.lt + head * q.lh);
        const uint4 *qr = reinterpret_cast<const uint4 *>(reinterpret_cast<const __half *>(q.rope) + token * q.rt + head * q.rh);
        const uint32_t tmem = c->tmem + ((uint32_t)((warp & 3) * 32) << 16);
        for (int p = 0; p < nc; p++) {
            const int g = chunk_at(p);
            const uint4 *src = g < 2 * nv ? ql + g * 8 : qr;
            uint32_t u[32];
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint4 x = live ? __ldg(src + k) : make_uint4(0, 0, 0, 0);
                u[4 * k] = x.x, u[4 * k + 1] = x.y, u[4 * k + 2] = x.z, u[4 * k + 3] = x.w;
            }
            if (p < nq) {
                tmem_st32(tmem + q_col(p), u);
            } else {
                uint8_t *dst = sq + (p - nq) * MLA_QCHUNK + (r >> 3) * 1024 + (r & 7) * 128;
#pragma unroll
                for (int k = 0; k < 8; k++)
                    *reinterpret_cast<uint4 *>(dst + (k ^ (r & 7)) * 16) = make_uint4(u[4 * k], u[4 * k + 1], u[4 * k + 2], u[4 * k + 3]);
            }
        }
        tmem_wait_st();
        fence_async_smem();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&c->q_ready);
    }

    // Rows of the tile with an infinity or a NaN among this CTA's output columns become zeros there (a weight of
    // zero times a NaN is a NaN), and are named to the caller.  Two threads per row.
    __device__ __forceinline__ uint64_t clean(int st, int par) {
        const int tid = (warp & 3) * 32 + lane, r = tid >> 1, h = tid & 1;
        if (tid == 0) c->nonfinite[par] = 0;
        __syncwarp();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const uint32_t top = BF16 ? 0x7F80u : 0x7C00u;
        bool bad = false;
        for (int p = 0; p < nv; p++) {
            const uint4 *src = reinterpret_cast<const uint4 *>(ring_b + (st * nv + p) * MLA_CHUNK + r * 128 + h * 64);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint4 x = src[k];
                const uint32_t u[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 0; j < 4; j++) bad |= (u[j] & top) == top || (u[j] >> 16 & top) == top;
            }
        }
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 1) != 0;
        if (bad) {
            if (h == 0) atomicOr(reinterpret_cast<unsigned long long *>(&c->nonfinite[par]), 1ull << r);
            for (int p = 0; p < nv; p++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    reinterpret_cast<uint4 *>(ring_b + (st * nv + p) * MLA_CHUNK + r * 128 + h * 64)[k] = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        __syncwarp();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        return *reinterpret_cast<volatile uint64_t *>(&c->nonfinite[par]);
    }

    __device__ __forceinline__ void store_out(uint32_t tmem, bool live, int64_t token, int head, float ref, float l) {
        const int half_cols = kv.latent / 2;
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        __half *out = reinterpret_cast<__half *>(q.out) + token * q.ot + head * q.oh + half * half_cols;
        for (int col = 0; col < half_cols; col += 32) {
            float o[32];
            tmem_ld32(tmem + col, o);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint4 x;
                x.x = pack2<BF16>(o[8 * k] * f, o[8 * k + 1] * f);
                x.y = pack2<BF16>(o[8 * k + 2] * f, o[8 * k + 3] * f);
                x.z = pack2<BF16>(o[8 * k + 4] * f, o[8 * k + 5] * f);
                x.w = pack2<BF16>(o[8 * k + 6] * f, o[8 * k + 7] * f);
                if (live) reinterpret_cast<uint4 *>(out + col)[k] = x;
            }
            __syncwarp();
        }
        if (live && half == 0 && q.lse)
            q.lse[token * q.n_heads + head] = l == 0.0f ? -INFINITY : ref * 0.69314718055994531f + logf(l);
    }

    __device__ __forceinline__ void store_piece(uint32_t tmem, const MlaSeg &g, const MlaWalk &w, bool live, int r, float ref, float l) {
        const int L = kv.latent, half_cols = L / 2;
        const int slot = 2 * pair + (g.tile0 == 0);
        float *o = ws.o + ((size_t)slot * L + half * half_cols) * MLA_M + r;
        for (int col = 0; col < half_cols; col += 32) {
            float v[32];
            tmem_ld32(tmem + col, v);
#pragma unroll
            for (int k = 0; k < 32; k++)
                if (live) o[(size_t)(col + k) * MLA_M] = v[k];
            __syncwarp();
        }
        if (half == 0 && live) {
            ws.ml[(size_t)slot * 2 * MLA_M + r] = ref;
            ws.ml[(size_t)slot * 2 * MLA_M + MLA_M + r] = l;
        }
    }
};

template <bool BF16, bool FP8>
__global__ void __launch_bounds__(FP8 ? 512 : 256, 1)
    k_mla(MoeKvDev kv, MlaSeqAt seq_at, MoeMlaQuery q, const __grid_constant__ CUtensorMap tm, void *ws, int *error) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    const int L = kv.latent, nv = L / 128, nc = 2 * nv + 1, nq = mla_q_tm(L);
    const int pairs = gridDim.x / 2;
    uint8_t *ring_b = base, *ring_a = ring_b + MLA_SB * nv * MLA_CHUNK, *sq = ring_a + MLA_RA * MLA_CHUNK;
    MlaCtl *c = reinterpret_cast<MlaCtl *>(sq + (nc - nq) * MLA_QCHUNK);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int PROD = FP8 ? 8 : 1;
    if (tid == 0) {
        for (int i = 0; i < MLA_RA; i++) tc_mbar_init(&c->full_a[i], PROD), tc_mbar_init(&c->empty_a[i], 1);
        for (int i = 0; i < MLA_SB; i++) tc_mbar_init(&c->full_b[i], PROD), tc_mbar_init(&c->empty_b[i], 1);
        tc_mbar_init(&c->s_full, 1), tc_mbar_init(&c->s_empty, 4), tc_mbar_init(&c->p_full, 4);
        tc_mbar_init(&c->pv_done, 1), tc_mbar_init(&c->q_ready, 4), tc_mbar_init(&c->drain, 1);
        c->dead = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 2) tmem_alloc(&c->tmem, 512);
    moe_pdl_wait();
    // the pair's share of all tiles: every thread sums a stretch of sequences, a scan over threads, then the
    // thread whose stretch holds the share's first tile finds its sequence
    const int pair = blockIdx.x >> 1, n = seq_at.b.n_seqs;
    const int per = (n + blockDim.x - 1) / blockDim.x, b0 = min(n, tid * per), b1 = min(n, b0 + per);
    int64_t mine = 0;
    for (int b = b0; b < b1; b++) {
        const MlaSeq s = seq_at(b);
        mine += s.work();
        if (s.bad && blockIdx.x == 0) kv_error(error, KV_ERR_BATCH);
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += y;
    }
    if (lane == 31) c->scan[warp] = incl;
    __syncthreads();
    int64_t before = incl - mine, total = 0;
    for (int k = 0; k < (int)(blockDim.x >> 5); k++) {
        if (k < warp) before += c->scan[k];
        total += c->scan[k];
    }
    const int64_t w0 = mla_share(total, pair, pairs), w1 = mla_share(total, pair + 1, pairs);
    if (tid == 0) c->w0 = w0, c->w1 = w1, c->total = total;
    if (w0 < w1 && w0 >= before && w0 < before + mine) {
        int64_t off = w0 - before;
        int b = b0;
        for (;; b++) {
            const int64_t k = seq_at(b).work();
            if (off < k) break;
            off -= k;
        }
        c->off0 = off, c->seq0 = b;
    }
    tmem_fence_before();
    __syncthreads();
    tmem_fence_after();
    MlaKernel<BF16, FP8> k{kv, seq_at, q, &tm, mla_ws(ws, L, pairs), error, ring_b, ring_a, sq, c,
                           (int)(blockIdx.x & 1), pair, pairs, nv, nc, nq, lane, warp};
    if (k.half == 0 && warp == 3 && lane == 0) {
        // the unit that this pair begins and another one ends (k_mla_join); every call writes the entry
        MlaWalk w = k.walk();
        MlaSeg g{};
        MlaWs::Tail tail{0, 0, 0, 0};
        int rest = 0;
        while (w.next(g, seq_at)) rest = w.s.tiles - g.tile1;
        if (w0 < w1 && rest > 0 && g.tile0 == 0)
            tail = MlaWs::Tail{g.seq, g.block, mla_last_pair(total, pair, pairs, w1, rest), 1};
        k.ws.tail[pair] = tail;
    }
    if (w0 < w1) {
        if (FP8 && warp >= 8) k.produce_expand();
        else if (!FP8 && warp == 0) k.produce_tma();
        else if (warp == 1) k.issue();
        else if (warp >= 4 && warp < 8) k.rows();
    }
    __syncwarp();
    tmem_fence_before();
    __syncthreads();
    if (warp == 2) tmem_free(c->tmem, 512);
}

// ---------------------------------------------------------------------------
// Joins the pieces of the unit that pair blockIdx.x began and did not end: per
// row the pieces' sums, each times 2^(its reference - the largest), in the
// order of the pairs (the same bits every time).  One thread per (row, 8
// columns, quarter of the pieces); the quarters meet in shared memory.
// ---------------------------------------------------------------------------
constexpr int MJ_COLS = 8, MJ_PARTS = 4;

template <bool BF16>
__global__ void __launch_bounds__(MLA_M *MJ_PARTS) k_mla_join(MoeKvDev kv, MlaSeqAt seq_at, MoeMlaQuery q, void *wsp, int pairs) {
    __shared__ float acc[MJ_PARTS][MJ_COLS + 1][MLA_M];
    moe_pdl_wait();
    const MlaWs ws = mla_ws(wsp, kv.latent, pairs);
    const int p = blockIdx.x, r = threadIdx.x % MLA_M, part = threadIdx.x / MLA_M;
    const MlaWs::Tail t = ws.tail[p];
    if (!t.on) return;
    const MlaSeq s = seq_at(t.seq);
    const int64_t row = (int64_t)t.block * MLA_M + r;
    const bool live = row < (int64_t)s.n * q.n_heads;
    const int L = kv.latent, col = blockIdx.y * MJ_COLS, pieces = t.last - p + 1;
    // piece 0 is this pair's second slot, piece k > 0 pair p + k's first
    auto slot = [&](int k) { return k == 0 ? 2 * p + 1 : 2 * (p + k); };
    float m = -INFINITY;
    if (live)
#pragma unroll 8
        for (int k = 0; k < pieces; k++) m = fmaxf(m, ws.ml[(size_t)slot(k) * 2 * MLA_M + r]);
    const float m0 = m == -INFINITY ? 0.0f : m;
    float l = 0.0f, o[MJ_COLS] = {};
    const int k0 = pieces * part / MJ_PARTS, k1 = pieces * (part + 1) / MJ_PARTS;
    if (live)
#pragma unroll 4
        for (int k = k0; k < k1; k++) {
            const float *ml = ws.ml + (size_t)slot(k) * 2 * MLA_M + r;
            const float f = ex2(ml[0] - m0);
            const float *src = ws.o + ((size_t)slot(k) * L + col) * MLA_M + r;
            l = fmaf(f, ml[MLA_M], l);
#pragma unroll
            for (int j = 0; j < MJ_COLS; j++) o[j] = fmaf(f, src[j * MLA_M], o[j]);
        }
#pragma unroll
    for (int j = 0; j < MJ_COLS; j++) acc[part][j][r] = o[j];
    acc[part][MJ_COLS][r] = l;
    __syncthreads();
    if (part || !live) return;
#pragma unroll
    for (int k = 1; k < MJ_PARTS; k++) {
        l += acc[k][MJ_COLS][r];
#pragma unroll
        for (int j = 0; j < MJ_COLS; j++) o[j] += acc[k][j][r];
    }
    const float f = l == 0.0f ? 0.0f : 1.0f / l;
    const int64_t token = s.q0 + row / q.n_heads, head = row % q.n_heads;
    uint4 x;
    x.x = pack2<BF16>(o[0] * f, o[1] * f);
    x.y = pack2<BF16>(o[2] * f, o[3] * f);
    x.z = pack2<BF16>(o[4] * f, o[5] * f);
    x.w = pack2<BF16>(o[6] * f, o[7] * f);
    *reinterpret_cast<uint4 *>(reinterpret_cast<__half *>(q.out) + token * q.ot + head * q.oh + col) = x;
    if (col == 0 && q.lse) q.lse[token * q.n_heads + head] = l == 0.0f ? -INFINITY : m * 0.69314718055994531f + logf(l);
}

size_t mla_smem(int latent) {
    const int nv = latent / 128, nc = 2 * nv + 1;
    return 1024 + (size_t)(MLA_SB * nv + MLA_RA) * MLA_CHUNK + (size_t)(nc - mla_q_tm(latent)) * MLA_QCHUNK + sizeof(MlaCtl);
}

template <bool BF16, bool FP8>
void launch(const MoeKvDev &kv, const MlaSeqAt &at, const MoeMlaQuery &q, const CUtensorMap &tm, void *ws, int pairs,
            int *error, cudaStream_t s) {
    static size_t done[MOE_MAX_DEVICES];
    const size_t smem = mla_smem(kv.latent);
    moe_smem_limit(k_mla<BF16, FP8>, smem, done);
    moe_launch_pdl(k_mla<BF16, FP8>, dim3(2 * pairs), dim3(FP8 ? 512 : 256), smem, s, kv, at, q, tm, ws, error);
    moe_launch_pdl(k_mla_join<BF16>, dim3(pairs, kv.latent / MJ_COLS), dim3(MLA_M * MJ_PARTS), 0, s, kv, at, q, ws, pairs);
}

}  // namespace

size_t moe_mla_ws_bytes(int latent, int sms) {
    const int pairs = sms / 2;
    return ((size_t)pairs * sizeof(MlaWs::Tail) + 255) / 256 * 256 + (size_t)pairs * 2 * (2 + latent) * MLA_M * sizeof(float);
}

int moe_launch_mla(const MoeKvDev &kv, const MoeKvBatchDev &b, const MoeMlaQuery &q, void *ws, int sms, int *error,
                   cudaStream_t s, uint64_t *launches) {
    const MlaSeqAt at{b, q.n_heads, kv.page_shift};
    const bool fp8 = kv.format == MOE_KV_FP8_F16 || kv.format == MOE_KV_FP8_BF16;
    CUtensorMap tm{};
    if (!fp8 && moe_make_map_f16_sw128(&tm, kv.data, kv.latent + MOE_KV_ROPE, (uint64_t)kv.n_pages << kv.page_shift, 64,
                                       kv.page_shift >= 6 ? MLA_N : 1u << kv.page_shift))
        return -1;
    switch (kv.format) {
        case MOE_KV_F16: launch<false, false>(kv, at, q, tm, ws, sms / 2, error, s); break;
        case MOE_KV_BF16: launch<true, false>(kv, at, q, tm, ws, sms / 2, error, s); break;
        case MOE_KV_FP8_F16: launch<false, true>(kv, at, q, tm, ws, sms / 2, error, s); break;
        default: launch<true, true>(kv, at, q, tm, ws, sms / 2, error, s);
    }
    LAUNCH_COUNT(launches);
    LAUNCH_COUNT(launches);
    return 0;
}
