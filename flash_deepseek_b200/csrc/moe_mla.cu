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
// products of its neighbours.  (Scores of tile i + 2 wait until that product
// is done: they take the place of its weights.)  A tile's latent chunks of this
// CTA's half stay until its output product is done (ring B, 3 tiles); the other
// half and the rotary chunk are only scores' operands and leave chunk by chunk
// (ring A).
// Work division: moe_kv_plan.h; cut units are joined by k_mla_join.
//
// Measured.  A tile's products take 1,984 cycles (128 x 64 scores: 32 cycles per
// 16 values with the query in tensor memory, 48 from shared memory, whose reads
// bound it; 128 x 256 output: 128 cycles per 16 rows); a tile takes some 2,900
// (1.7 us) in 16 bits and 3,200 (1.9 us) in 8 bits, where the pair runs in
// lockstep, and a launch 14 to 17 us beside its tiles.  With the join (10 to 23
// us, partly under it): 32 sequences of 8192 bf16 rows, one token of 128 heads:
// 113 to 134 us by box (2.4 to 2.1 TB/s, 0.57 to 0.48 PFLOP/s); 8 trees of 13
// tokens over 16,384 8-bit rows: 0.65 to 0.70 ms (0.66 to 0.61 PFLOP/s).
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
constexpr int MLA_RA = 6;                   // chunks of ring A
constexpr int MLA_SB = 3;                   // tiles of ring B
// Tensor-memory columns: the output from 0 (at most 256), two score tiles of 64 (the weights of a tile, 32 columns of
// 16-bit pairs, take the place of its second half), the query's chunks.
constexpr int MLA_TM_S = 256, MLA_TM_P = 32, MLA_TM_Q = 384;
constexpr int MLA_XW = 8;                   // warps that expand the 8-bit formats (4: 667 us where 8 take 626)
constexpr float MLA_RAISE = 8.0f;           // log2: how far scores may pass the reference before it is raised
// log2 of the weight of a score at the reference.  fp16 weights are normal from 2^-14 and zero below 2^-25, so they are
// put as high as 2^(lift + MLA_RAISE) = 2^15 allows: full precision down to 2^-21 of the reference's weight, and an error
// of at most 2^-32 of it below.  (Lifted by 0, rows 17 nats below the reference weighed twice too much or nothing: 10^5
// of them behind one strong row are a part of the result that shows.)  bf16 has fp32's exponents and needs none.  Nor do
// scores from 2^20 on, whose own rounding is 2^-4 and more: there the room up to fp16's 2^16 is for that.
template <bool BF16>
__device__ __forceinline__ float mla_lift(float score) { return !BF16 && fabsf(score) < 1048576.0f ? 7.0f : 0.0f; }

// Log of the sum of exponentials, from the reference and the sum of weights relative to it: added in log2, where a lift
// cancels exactly
__device__ __forceinline__ float mla_lse(float ref, float l) {
    return l == 0.0f ? -INFINITY : (ref + log2f(l)) * 0.69314718055994531f;
}

// Tensor memory left for query chunks of 32 columns (64 values) each: all of
// them for up to 256 latent values, 6 of 7 for 384, 4 of 9 for 512.
__host__ __device__ constexpr int mla_q_tm(int latent) {
    const int all = latent / 64 + 1, fit = (512 - MLA_TM_Q + (256 - latent / 2)) / 32;
    return all < fit ? all : fit;
}

// Query chunks in shared memory: the others, or room for those on their way into tensor memory
__host__ __device__ constexpr int mla_q_sm(int latent) {
    const int tm = mla_q_tm(latent), rest = latent / 64 + 1 - tm;
    return rest > tm ? rest : tm;
}

struct MlaCtl {   // control block behind the tiles
    uint64_t full_a[MLA_RA], empty_a[MLA_RA], full_b[MLA_SB], empty_b[MLA_SB];   // chunks of ring A, tiles of ring B
    uint64_t full_r[2], empty_r[2];   // 8-bit formats: rotary chunks by tile parity
    uint64_t s_full[2], p_full[2], pv_done[2], q_ready, drain;   // by tile parity
    uint64_t clean;              // the softmax warps meet (clean)
    uint64_t nonfinite[2];       // by tile parity: rows of a tile with an infinity or a NaN in this CTA's latent half
    struct Rows {                // each softmax warp's walk over the segments (in registers it would cost them 30)
        MlaWalk w;
        MlaSeg g;
        int more, met;           // met: phases of `clean` so far
    } rows[4];
    uint8_t valid[4][8];         // by tile: 8-row groups whose page exists
    int64_t w0, w1, off0;        // the pair's share: first and last tile, place of the first in its sequence
    int64_t scan[32];
    int seq0;
    uint32_t tmem;
    int used;                    // 8-bit formats: tiles whose copies the other CTA's scores are done with
};

// Pieces of cut units: [pair][slot][latent][128 rows] sums, [pair][slot][half][2][128] references and sums of weights.
// Each half of the columns has its CTA's own: the two CTAs sum a score's chunks in different orders, so their scores
// differ in the last bits, and one may raise its reference where the other does not (by up to MLA_RAISE apart then).
constexpr int MLA_STATS = 2 * 2 * MLA_M;   // floats of a slot
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
    b += (size_t)pairs * 2 * MLA_STATS * sizeof(float);
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

// The warp waits for a phase (tc_wait_warp); the polling is out of line: the
// loops of this kernel's roles share one instruction cache of some 32 KB, and
// with everything unrolled and inlined the wait for instructions cost more than
// any other stall (8-bit rows: 0.80 against 0.64 ms).
__device__ __noinline__ bool poll(uint64_t *b, uint32_t parity) { return tc_wait_warp(b, parity); }
__device__ __forceinline__ bool wait_phase(uint64_t *b, uint32_t parity) {
    return __all_sync(0xffffffffu, tc_test(b, parity)) || poll(b, parity);
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if (BF16) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t *>(&v);
    }
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&v);
}

// a number handed from one thread of the CTA to others, with what the writer saw and wrote before it
__device__ __forceinline__ void store_release(int *p, int v) {
    asm volatile("st.release.cta.shared::cta.s32 [%0], %1;\n" ::"r"(umma_smem_u32(p)), "r"(v) : "memory");
}
__device__ __forceinline__ int load_acquire(const int *p) {
    int v;
    asm volatile("ld.acquire.cta.shared::cta.s32 %0, [%1];\n" : "=r"(v) : "r"(umma_smem_u32(p)) : "memory");
    return v;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// two fp32 values in one 64-bit register, one instruction for both
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}
__device__ __forceinline__ void unpair2(uint64_t r, float &a, float &b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(r)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// 4 e4m3 codes times a group's scale as 4 16-bit values.  The code's exponent
// and mantissa bits placed in the 16-bit format's fields are the value over
// 2^120 (bf16) or 2^8 (fp16), subnormals too; f holds 2^(120 + k) or 2^(8 + k).
// Each half word holds a code: shifted up by a product, then the sign (bit 11 or
// 14) moved to bit 15 by adding 15 times or once itself; products and sums run
// on another pipe than the byte permutes and masks, which bound this.
template <bool BF16>
__device__ __forceinline__ uint2 expand4(uint32_t w, uint32_t f) {
    constexpr uint32_t up = BF16 ? 16 : 128, sign = BF16 ? 0x08000800u : 0x40004000u, times = BF16 ? 15 : 1;
    const uint32_t lo = __byte_perm(w, 0, 0x4140) * up, hi = __byte_perm(w, 0, 0x4342) * up;
    uint2 r = make_uint2((lo & sign) * times + lo, (hi & sign) * times + hi);
    if (BF16) {
        asm("mul.bf16x2 %0, %0, %1;" : "+r"(r.x) : "r"(f));
        asm("mul.bf16x2 %0, %0, %1;" : "+r"(r.y) : "r"(f));
    } else {
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
template <bool BF16, bool FP8, int NV>   // NV: latent chunks (of 64 values) of a CTA's half
struct MlaKernel {
    static constexpr int NC = 2 * NV + 1, NQ = mla_q_tm(128 * NV);   // chunks of a row; of the query in tensor memory

    const MoeKvDev &kv;
    const MlaSeqAt &seq_at;
    const MoeMlaQuery &q;
    const CUtensorMap *tm;
    MlaWs ws;
    int *error;
    uint8_t *ring_b, *ring_a, *ring_r, *sq;
    MlaCtl *c;
    int half, pair;
    int lane, warp;

    // the chunk (64 values of a row) at place p of the order: own half, other half, rotary
    __device__ __forceinline__ int chunk_at(int p) const {
        return p < NV ? half * NV + p : p < 2 * NV ? (1 - half) * NV + p - NV : 2 * NV;
    }
    __device__ __forceinline__ MlaWalk walk() const {
        MlaWalk w{};
        w.w = c->w0, w.w1 = c->w1, w.off = c->off0, w.seq = c->seq0, w.n_seqs = seq_at.b.n_seqs;
        return w;
    }
    __device__ __forceinline__ void give_up() {
        if (lane == 0) kv_error(error, KV_ERR_TIMEOUT);
    }
    __device__ __forceinline__ long long flat(int seq, const MlaSeq &s, int64_t pos) const {
        if (pos >= s.len) return -2;   // behind the sequence: no error
        return kv_flat_row(kv, seq_at.b, seq, pos);
    }

    // after a wait gave up: none of the copies issued so far may land after the CTA has ended
    __device__ void stop_tma(int ia, int ib, int ir) {
        give_up();
        if (FP8) return tc_drain(c->full_r, ir, 2);
        tc_drain(c->full_a, ia, MLA_RA);
        tc_drain(c->full_b, ib, MLA_SB);
    }

    // ---- TMA: lane j < 8 handles rows 8 j .. of a tile.  16-bit formats: all chunks; 8-bit formats: the rotary one.
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
                if (FP8) {
                    // valid[] of tile ib - 4 is read: its output product was issued before the scores of tile ib - 2
                    const int sr = ib & 1;
                    if (!wait_phase(&c->empty_r[sr], (ib / 2 + 1) & 1)) return stop_tma(0, 0, ib);
                    if (lane < 8) c->valid[ib & 3][lane] = ok;
                    __syncwarp();
                    if (lane == 0) tc_expect(&c->full_r[sr], MLA_CHUNK);
                    __syncwarp();
                    if (box) tc_tma2(ring_r + sr * MLA_CHUNK + off, tm, 64 * NV, row, &c->full_r[sr]);   // 16-bit units
                    continue;
                }
                if (!wait_phase(&c->empty_b[st], (ib / MLA_SB + 1) & 1)) return stop_tma(ia, ib, 0);
                if (lane < 8) c->valid[ib & 3][lane] = ok;
                __syncwarp();
                if (lane == 0) tc_expect(&c->full_b[st], (uint32_t)NV * MLA_CHUNK);
                __syncwarp();
                if (box)
#pragma unroll 1
                    for (int p = 0; p < NV; p++)
                        tc_tma2(ring_b + (st * NV + p) * MLA_CHUNK + off, tm, chunk_at(p) * 64, row, &c->full_b[st]);
#pragma unroll 1
                for (int p = NV; p < NC; p++, ia++) {
                    const int sa = ia % MLA_RA;
                    if (!wait_phase(&c->empty_a[sa], (ia / MLA_RA + 1) & 1)) return stop_tma(ia, ib + 1, 0);
                    if (lane == 0) tc_expect(&c->full_a[sa], MLA_CHUNK);
                    __syncwarp();
                    if (box) tc_tma2(ring_a + sa * MLA_CHUNK + off, tm, chunk_at(p) * 64, row, &c->full_a[sa]);
                }
            }
        }
    }

    // ---- 8-bit formats: 8 warps expand the chunks of this CTA's half into ring B, 4 threads per row, 16 codes of a chunk
    // each; from there they are copied into ring A of the other CTA, whose scores need them too.  So each CTA reads and
    // expands half of a row.  Codes are loaded a tile ahead, page numbers two.
    struct Cursor {   // a place in the pair's tiles
        MlaWalk w;
        MlaSeg g;
        int t;
        bool more;
    };
    __device__ __forceinline__ void step(Cursor &u) {
        if (u.more && ++u.t >= u.g.tile1) {
            u.more = u.w.next(u.g, seq_at);
            u.t = u.g.tile0;
        }
    }
    // the page of this thread's row of the cursor's tile (-1: none, -2: behind the sequence)
    __device__ __forceinline__ int page_of(const Cursor &u, int r, int &in_page) {
        const int64_t pos = (int64_t)u.t * MLA_N + r;
        in_page = (int)(pos & ((1 << kv.page_shift) - 1));
        if (!u.more || pos >= u.w.s.len) return -2;
        const int64_t pi = pos >> kv.page_shift;
        return pi < seq_at.b.pages_per_seq ? __ldg(seq_at.b.pages + (size_t)u.g.seq * seq_at.b.pages_per_seq + pi) : -1;
    }
    __device__ __forceinline__ const uint8_t *row_of(int page, int in_page) {
        // (a page out of range: the TMA warp reports it and hides the row)
        return page < 0 || page >= kv.n_pages ? nullptr : kv.data + (((int64_t)page << kv.page_shift) + in_page) * kv.row_bytes;
    }
    __device__ void produce_expand() {
        constexpr int L = 128 * NV;
        static_assert(MLA_XW * 32 == MLA_N * 4, "4 threads for each row of a tile");
        const int tid = threadIdx.x - 256, r = tid >> 2, qd = tid & 3;
        const int n = (int)(c->w1 - c->w0);
        const uint32_t sw = (uint32_t)(r & 7), at = (uint32_t)(r >> 3) * 1024 + sw * 128;
        const uint32_t lo_at = at + ((2 * qd) ^ sw) * 16, hi_at = at + ((2 * qd + 1) ^ sw) * 16;
        const int code_at = half * NV * 64 + qd * 16, scale_at = L + 2 * MOE_KV_ROPE + half * NV * 2 + (qd >> 1);
        uint4 code[NV];
        uint32_t sb[NV];
        auto load = [&](const uint8_t *row, int p, uint4 &v, uint32_t &b) {
            v = row ? __ldg(reinterpret_cast<const uint4 *>(row + code_at + p * 64)) : make_uint4(0, 0, 0, 0);
            b = row ? __ldg(row + scale_at + p * 2) : 127u;
        };
        Cursor u{walk(), MlaSeg{}, 0, true};
        u.more = u.w.next(u.g, seq_at);
        u.t = u.g.tile0;
        int in_page, page = page_of(u, r, in_page);
        const uint8_t *row = row_of(page, in_page);
#pragma unroll
        for (int p = 0; p < NV; p++) load(row, p, code[p], sb[p]);
        step(u);
        page = page_of(u, r, in_page);
#pragma unroll 1
        for (int i = 0; i < n; i++) {
            const int st = i % MLA_SB;
            row = row_of(page, in_page);         // of tile i + 1
            step(u);
            page = page_of(u, r, in_page);       // of tile i + 2
            if (!wait_phase(&c->empty_b[st], (i / MLA_SB + 1) & 1)) return give_up();
#pragma unroll
            for (int p = 0; p < NV; p++) {
                const uint32_t f = scale2<BF16>(sb[p]);
                const uint4 v = code[p];
                load(row, p, code[p], sb[p]);
                const uint2 a = expand4<BF16>(v.x, f), b = expand4<BF16>(v.y, f);
                const uint2 d = expand4<BF16>(v.z, f), e = expand4<BF16>(v.w, f);
                uint8_t *dst = ring_b + (st * NV + p) * MLA_CHUNK;
                *reinterpret_cast<uint4 *>(dst + lo_at) = make_uint4(a.x, a.y, b.x, b.y);
                *reinterpret_cast<uint4 *>(dst + hi_at) = make_uint4(d.x, d.y, e.x, e.y);
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) tc_arrive(&c->full_b[st]);
        }
    }
    // One warp copies each expanded chunk to the other CTA once its scores of the tile before are done with the slot
    // (bulk copies: 16-byte remote stores from the expanding threads took 4500 cycles a tile, against 2700 for the rest).
    // A stage of ring B is free when its output product is done and the other CTA has used what was copied from it.
    __device__ void forward() {
        const int n = (int)(c->w1 - c->w0);
        const uint32_t other = half ^ 1, ra = cluster_map(ring_a, other), fa = cluster_map(c->full_a, other);
        for (int i = 0; i <= n; i++) {
            const int st = i % MLA_SB;
            if (i < n && !wait_phase(&c->full_b[st], (i / MLA_SB) & 1)) return stop_forward();
#pragma unroll 1
            for (int p = 0; p < NV; p++) {   // the slot: its tile i - 1 is used
                if (!wait_phase(&c->empty_a[p], (i + 1) & 1)) return stop_forward();
                if (lane == 0 && i < n)
                    cluster_copy_async(ra + p * MLA_CHUNK, ring_b + (st * NV + p) * MLA_CHUNK, MLA_CHUNK, fa + p * 8);
            }
            if (lane == 0 && i > 0) {
                store_release(&c->used, i);
                tc_arrive(&c->empty_b[(i - 1) % MLA_SB]);
            }
            __syncwarp();
        }
    }
    // after a wait gave up: the copies into the other CTA that are under way land long before it can end
    __device__ void stop_forward() {
        give_up();
        __nanosleep(100000);
    }

    // ---- MMA issue: one warp, every lane runs the loop, an elected lane issues.  Operands are broadcast from lane 0
    // and every branch goes by a vote: where the compiler cannot prove operands and control flow uniform, an MMA takes
    // 90 cycles to issue, against 32 (scores) to run.
    // Barriers are tested ahead, before the MMAs in front of their use: a test of a completed phase takes 100 cycles
    // from issue to branch, which the tensor pipe would stand idle.
    __device__ __forceinline__ bool then_wait(uint32_t seen, uint64_t *b, uint32_t parity) {
        return __all_sync(0xffffffffu, seen) || poll(b, parity);
    }
    struct Issue {
        uint32_t tmem, rb, ra, rr, sq;     // base addresses
        int st, sa, phase_b, phase_a;      // next tile's stage and next chunk's slot, their parities
        uint32_t seen_b;                   // the test of the next tile's ring B stage
    };
    // the weights of tile i times its latent chunks; nb: the stage's parity of the tile behind
    __device__ bool output(Issue &x, int i, int st, uint32_t seen, uint32_t more) {
        constexpr uint32_t id = umma_idesc_16(MLA_M, 64 * NV, BF16, 1);
        if (!then_wait(seen, &c->p_full[i & 1], (i >> 1) & 1)) return false;
        x.seen_b = tc_test(&c->full_b[x.st], x.phase_b);
        tmem_fence_after();
        const uint32_t ts = x.tmem + MLA_TM_S + (i & 1) * 64 + MLA_TM_P;
        const uint64_t d = umma_desc_sw128_mn(x.rb + st * NV * MLA_CHUNK, MLA_CHUNK);
        // four steps of 16 cache rows: 2048 bytes of the tile, 8 columns of weights each
        static_assert(MLA_N == 64, "four steps");
        umma_f16_ta_warp4<(2048 >> 4)>(x.tmem, ts, d, id, more);
        umma_commit_warp(&c->empty_b[st]);
        umma_commit_warp(&c->pv_done[i & 1]);
        return true;
    }
    // the scores of tile `it`; `seen`: the test of the weights of the tile before, made before the last chunk
    __device__ bool scores(Issue &x, int it, uint32_t &seen) {
        constexpr uint32_t id = umma_idesc_16(MLA_M, MLA_N, BF16, 0);
        if (!then_wait(x.seen_b, &c->full_b[x.st], x.phase_b)) return false;
        x.seen_b = 0;   // of this tile only: the first tile of a segment has no output() behind it that tests the next
        // The score tile it & 1 is free once the product that reads its weights (tile it - 2) is done.  The issue order
        // does not say so: products of another accumulator and shape are not ordered with it.  (The barrier is at most
        // one phase behind: the product of tile it itself is issued later.)
        if (!wait_phase(&c->pv_done[it & 1], ((it >> 1) + 1) & 1)) return false;
        tmem_fence_after();
        const uint32_t ts = x.tmem + MLA_TM_S + (it & 1) * 64;
        uint32_t seen_a = 0;
        auto chunk_tm = [&](uint32_t q_at, uint32_t k_at, uint32_t first) {   // the query's chunk in tensor memory
            umma_f16_ta_warp4<2>(ts, q_at, umma_desc_sw128(k_at), id, first);
        };
        auto chunk_sm = [&](uint32_t q_at, uint32_t k_at) {                   // in shared memory
            umma_f16_warp4(ts, umma_desc_sw128(q_at), umma_desc_sw128(k_at), id);
        };
        static_assert(NQ >= NV, "the own half's query chunks are in tensor memory");
        const uint32_t rb = x.rb + x.st * NV * MLA_CHUNK;
#pragma unroll
        for (int p = 0; p < NV; p++) {
            if (p == NV - 1) seen_a = FP8 ? tc_test(&c->full_a[0], it & 1) : tc_test(&c->full_a[x.sa], x.phase_a);
            chunk_tm(x.tmem + q_col(p), rb + p * MLA_CHUNK, p > 0);
        }
        if (FP8) {
            // ring A: one slot per chunk, filled by the other CTA; armed for the next tile as soon as this one is in
#pragma unroll
            for (int p = NV; p < 2 * NV; p++) {
                const int sa = p - NV;
                if (!then_wait(seen_a, &c->full_a[sa], it & 1)) return false;
                if (lane == 0) tc_expect(&c->full_a[sa], MLA_CHUNK);
                seen_a = sa + 1 < NV ? tc_test(&c->full_a[sa + 1], it & 1) : tc_test(&c->full_r[it & 1], (it >> 1) & 1);
                if (p < NQ) chunk_tm(x.tmem + q_col(p), x.ra + sa * MLA_CHUNK, 1u);
                else chunk_sm(x.sq + (uint32_t)(p - NQ) * MLA_QCHUNK, x.ra + sa * MLA_CHUNK);
                umma_commit_to_warp(&c->empty_a[sa], (uint16_t)(1u << (half ^ 1)));
            }
            if (!then_wait(seen_a, &c->full_r[it & 1], (it >> 1) & 1)) return false;
            seen = tc_test(&c->p_full[(it + 1) & 1], (uint32_t)(it - 1) >> 1 & 1);
            if (2 * NV < NQ) chunk_tm(x.tmem + q_col(2 * NV), x.rr + (it & 1) * MLA_CHUNK, 1u);
            else chunk_sm(x.sq + (uint32_t)(2 * NV - NQ) * MLA_QCHUNK, x.rr + (it & 1) * MLA_CHUNK);
            umma_commit_warp(&c->empty_r[it & 1]);
        } else {
#pragma unroll
            for (int p = NV; p < NC; p++) {
                const int sa = x.sa;
                if (!then_wait(seen_a, &c->full_a[sa], x.phase_a)) return false;
                if (++x.sa == MLA_RA) x.sa = 0, x.phase_a ^= 1;
                if (p < NC - 1) seen_a = tc_test(&c->full_a[x.sa], x.phase_a);
                else seen = tc_test(&c->p_full[(it + 1) & 1], (uint32_t)(it - 1) >> 1 & 1);
                if (p < NQ) chunk_tm(x.tmem + q_col(p), x.ra + sa * MLA_CHUNK, 1u);
                else chunk_sm(x.sq + (uint32_t)(p - NQ) * MLA_QCHUNK, x.ra + sa * MLA_CHUNK);
                umma_commit_warp(&c->empty_a[sa]);
            }
        }
        umma_commit_warp(&c->s_full[it & 1]);
        if (++x.st == MLA_SB) x.st = 0, x.phase_b ^= 1;
        return true;
    }
    __device__ void issue() {
        Issue x{uni(c->tmem), uni(umma_smem_u32(ring_b)), uni(umma_smem_u32(ring_a)), uni(umma_smem_u32(ring_r)), uni(umma_smem_u32(sq)), 0, 0, 0, 0, 0};
        MlaWalk w = walk();
        MlaSeg g;
        int it = 0, seg = 0, prev = 0;   // tiles, segments so far; the stage of the tile before
        uint32_t seen = 0;
        bool ok = true;
        while (__all_sync(0xffffffffu, ok && w.next(g, seq_at))) {
            const int n = uni(g.tile1 - g.tile0);
            ok = wait_phase(&c->q_ready, seg & 1);
            seg++;
            for (int t = 0; __all_sync(0xffffffffu, ok && t < n); t++, it++) {
                const int st = x.st;
                ok = scores(x, it, seen);
                if (__all_sync(0xffffffffu, ok && t > 0)) ok = output(x, it - 1, prev, seen, t > 1);
                prev = st;
            }
            if (__all_sync(0xffffffffu, ok)) ok = output(x, it - 1, prev, 0, n > 1);
        }
        if (!ok) give_up();
        // nothing of this warp's is in flight when the CTA ends, nor an arrival of the other CTA's on a barrier here
        if (FP8) umma_commit_to_warp(&c->drain, 3);
        else umma_commit_warp(&c->drain);
        wait_phase(&c->drain, 0);
    }
    static __device__ __forceinline__ uint32_t uni(uint32_t x) { return __shfl_sync(0xffffffffu, x, 0); }
    // tensor-memory column of the query chunk at place p
    static __device__ __forceinline__ uint32_t q_col(int p) {
        // below 512 latent values the output takes fewer columns: the first chunks go behind it
        constexpr int spare = (256 - 64 * NV) / 32;
        return p < spare ? 64 * NV + p * 32 : MLA_TM_Q + (p - spare) * 32;
    }

    // The output product of tile i is done.  Each parity has a barrier: this warp has seen the scores of tile i or i + 1,
    // so the product of tile i - 2 is done and the barrier at most one phase behind (a wait by parity that is two phases
    // behind would never end).
    __device__ __forceinline__ bool output_done(int i) { return wait_phase(&c->pv_done[i & 1], (i >> 1) & 1); }

    // ---- softmax and output: 4 warps, one query row per thread
    __device__ void rows() {
        const uint32_t tmem = c->tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const int r = (warp & 3) * 32 + lane, L = 128 * NV, half_cols = 64 * NV;
        // scores in units of log2: a negative scale flips the query's signs, a scale of zero makes the query zero, so
        // that the factor is positive and the largest product gives the largest score
        const float c2 = q.scale == 0.0f ? 1.0f : fabsf(q.scale) * 1.4426950408889634f;
        MlaCtl::Rows &u = c->rows[warp & 3];
        const MlaSeg &g = u.g;
        const MlaSeq &s = u.w.s;
        if (lane == 0) u.w = walk(), u.met = 0;
        int it = 0;
        bool ok = true;
        for (;;) {
            if (lane == 0) u.more = ok && u.w.next(u.g, seq_at);
            __syncwarp();
            if (!u.more) break;
            const uint32_t row = (uint32_t)g.block * MLA_M + r;
            const bool live = row < (uint32_t)s.n * q.n_heads;
            const int token = live ? row / (uint32_t)q.n_heads : 0;
            const int tile0 = g.tile0, tile1 = g.tile1, ctx = s.ctx;
            load_query(r, s, (uint32_t)g.block * MLA_M);
            float ref = -INFINITY, l = 0.0f;   // ref: the score whose weight is 1
            for (int t = tile0; t < tile1; t++, it++) {
                const int64_t pos0 = (int64_t)t * MLA_N;
                ok = wait_phase(&c->s_full[it & 1], (it >> 1) & 1);
                if (!ok) break;
                tmem_fence_after();
                // a tile that reaches the drafted rows, or lacks a page: hide what the row does not see
                const uint64_t pages = *reinterpret_cast<const volatile uint64_t *>(c->valid[it & 3]);
                uint64_t see = ~0ull, nf = 0;
                const bool part = pos0 + MLA_N > ctx || pages != 0x0101010101010101ull;
                if (part) {
                    see = mla_visible(q, s, token, pos0) & pages * 255;
                    ok = (!FP8 || copies_used(it)) && clean(it % MLA_SB, it & 1, u, nf);
                    if (!ok) break;
                }
                // the scores are read twice (largest, weights), half a tile at a time, in loops that stay rolled
                const uint32_t ts = tmem + MLA_TM_S + (it & 1) * 64;
                float v[32], top = -INFINITY;
#pragma unroll 1
                for (int h = 0; h < 2; h++) {
                    tmem_ld32(ts + 32 * h, v);
                    if (part) hide(v, (uint32_t)(see >> 32 * h), (uint32_t)(nf >> 32 * h));
                    float m0 = fmaxf(fmaxf(top, v[0]), v[1]), m1 = fmaxf(fmaxf(v[2], v[3]), v[4]);
#pragma unroll
                    for (int k = 5; k < 29; k += 4) {
                        m0 = fmaxf(fmaxf(m0, v[k]), v[k + 1]);
                        m1 = fmaxf(fmaxf(m1, v[k + 2]), v[k + 3]);
                    }
                    m0 = fmaxf(fmaxf(m0, v[29]), v[30]);
                    top = fmaxf(fmaxf(m0, m1), v[31]);
                }
                top *= c2;
                if (t == tile0) ref = top - mla_lift<BF16>(top);
                else if (__any_sync(0xffffffffu, top > ref + (mla_lift<BF16>(ref) + MLA_RAISE))) {
                    // raise the reference: weights stay below 2^8 of its own, so fp16 and bf16 hold them
                    const float m = fmaxf(ref, top - mla_lift<BF16>(top)), f = m == -INFINITY ? 1.0f : ex2(ref - m);
                    l *= f;
                    ref = m;
                    ok = output_done(it - 1);   // the output holds all tiles before this one
                    if (!ok) break;
                    tmem_fence_after();
#pragma unroll 1
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
                const float m0 = ref == -INFINITY ? 0.0f : -ref;
                const uint64_t cc = pair2(c2, c2), mm = pair2(m0, m0);
                uint64_t sum[2] = {0, 0};
#pragma unroll 1
                for (int h = 1; h >= 0; h--) {
                    tmem_ld32(ts + 32 * h, v);
                    if (part) hide(v, (uint32_t)(see >> 32 * h), (uint32_t)(nf >> 32 * h));
                    uint32_t pk[16];
#pragma unroll
                    for (int k = 0; k < 32; k += 2) {
                        float a, b;
                        unpair2(fma2(pair2(v[k], v[k + 1]), cc, mm), a, b);
                        a = ex2(a), b = ex2(b);
                        sum[k >> 1 & 1] = add2(sum[k >> 1 & 1], pair2(a, b));
                        pk[k / 2] = pack2<BF16>(a, b);
                    }
                    tmem_st16(ts + MLA_TM_P + 16 * h, pk);   // over the second half's scores, which no one reads again
                }
                float sa, sb;
                unpair2(add2(sum[0], sum[1]), sa, sb);
                l += sa + sb;
                tmem_wait_st();
                tmem_fence_before();
                __syncwarp();
                if (lane == 0) tc_arrive(&c->p_full[it & 1]);
            }
            if (!ok) break;
            ok = output_done(it - 1);
            if (!ok) break;
            tmem_fence_after();
            if (g.whole) store_out(tmem, live, (int64_t)s.q0 + token, row - (uint32_t)token * q.n_heads, ref, l);
            else store_piece(tmem, tile0 == 0, live, r, ref, l);
            __syncwarp();
        }
        if (!ok) give_up();
    }

    // Scores of rows that are not seen become -infinity, of seen ones that hold an infinity or a NaN a NaN
    static __device__ __forceinline__ void hide(float (&v)[32], uint32_t see, uint32_t nf) {
#pragma unroll
        for (int k = 0; k < 32; k++) {
            if (nf >> k & 1) v[k] = __uint_as_float(0x7FC00000u);
            if (!(see >> k & 1)) v[k] = -INFINITY;
        }
    }

    // The block's query rows into tensor memory and shared memory (zeros behind the last row).  A warp loads its own 32
    // rows, 8 lanes per 128-byte line (a lane per row touches 32 lines with every load: 11,000 cycles a block).  The
    // chunks for tensor memory pass through the shared ones' place, from lanes across a row to a lane per row.
    __device__ __forceinline__ void load_query(int r, const MlaSeq s, uint32_t row0) {
        const uint32_t tmem = c->tmem + ((uint32_t)((warp & 3) * 32) << 16);
        uint8_t *mine = sq + (r >> 5) * 4096;   // this warp's rows of a chunk
        query_lines<0, NQ>(mine, s, row0 + (r & ~31));
        __syncwarp();
#pragma unroll 1
        for (int p = 0; p < NQ; p++) {
            uint32_t v[32];
            const uint8_t *src = mine + p * MLA_QCHUNK + (lane >> 3) * 1024 + (lane & 7) * 128;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const uint4 y = *reinterpret_cast<const uint4 *>(src + (k ^ (lane & 7)) * 16);
                v[4 * k] = y.x, v[4 * k + 1] = y.y, v[4 * k + 2] = y.z, v[4 * k + 3] = y.w;
            }
            tmem_st32(tmem + q_col(p), v);
        }
        __syncwarp();
        if constexpr (NQ < NC) query_lines<NQ, NC>(mine, s, row0 + (r & ~31));
        tmem_wait_st();
        fence_async_smem();
        tmem_fence_before();
        __syncwarp();
        if (lane == 0) tc_arrive(&c->q_ready);
    }
    // chunks P0 .. P1 - 1 of 32 rows, swizzled, into consecutive chunks: lane = 16 bytes (lane % 8) of rows lane / 8 + 4 i
    template <int P0, int P1>
    __device__ __forceinline__ void query_lines(uint8_t *dst, const MlaSeq &s, uint32_t row0) {
        const uint32_t rows = (uint32_t)s.n * q.n_heads;   // below 2^31, as n_tokens * n_heads is
        const uint32_t flip = q.scale < 0.0f ? 0x80008000u : 0u;
        const int u = lane & 7;
        const uint32_t my_token = (row0 + lane) / (uint32_t)q.n_heads, my_head = row0 + lane - my_token * q.n_heads;
#pragma unroll(FP8 ? 4 : 8)
        for (int i = 0; i < 8; i++) {   // all of them in flight where the registers allow
            const int k = (lane >> 3) + 4 * i;
            const bool live = row0 + k < rows && q.scale != 0.0f;
            uint32_t token = __shfl_sync(0xffffffffu, my_token, k), head = __shfl_sync(0xffffffffu, my_head, k);
            if (!live) token = head = 0;
            const __half *ql = reinterpret_cast<const __half *>(q.latent) + (int64_t)(s.q0 + token) * q.lt + head * q.lh + u * 8;
            const __half *qr = reinterpret_cast<const __half *>(q.rope) + (int64_t)(s.q0 + token) * q.rt + head * q.rh + u * 8;
            uint4 x[P1 - P0];
#pragma unroll
            for (int p = P0; p < P1; p++) {
                const uint4 *src = reinterpret_cast<const uint4 *>(p == 2 * NV ? qr : ql + chunk_at(p) * 64);
                x[p - P0] = live ? __ldg(src) : make_uint4(0, 0, 0, 0);
            }
            uint8_t *at = dst + (k >> 3) * 1024 + (k & 7) * 128 + (u ^ (k & 7)) * 16;
#pragma unroll
            for (int p = P0; p < P1; p++)
                *reinterpret_cast<uint4 *>(at + (p - P0) * MLA_QCHUNK) =
                    make_uint4(x[p - P0].x ^ flip, x[p - P0].y ^ flip, x[p - P0].z ^ flip, x[p - P0].w ^ flip);
        }
    }

    // Before rows of a tile are changed here (clean), the other CTA has to be done with what is copied from them.
    __device__ __forceinline__ bool copies_used(int it) {
        const long long t0 = clock64();
        bool ok = true;
        while (ok && load_acquire(&c->used) <= it) ok = clock64() - t0 <= TC_WAIT_CYCLES;
        return __all_sync(0xffffffffu, ok);
    }
    // The four softmax warps meet.  By an mbarrier, whose wait is bounded: a warp whose own wait gave up does not come,
    // and the others must not stand at a block barrier for good.
    __device__ __forceinline__ bool meet(MlaCtl::Rows &u) {
        const uint32_t phase = u.met & 1;
        __syncwarp();
        if (lane == 0) u.met++, tc_arrive(&c->clean);
        return wait_phase(&c->clean, phase);
    }
    // Rows of the tile with an infinity or a NaN among this CTA's output columns become zeros there (a weight of
    // zero times a NaN is a NaN), and are named to the caller.  Two threads per row.
    __device__ __forceinline__ bool clean(int st, int par, MlaCtl::Rows &u, uint64_t &nf) {
        const int tid = (warp & 3) * 32 + lane, r = tid >> 1, h = tid & 1;
        if (tid == 0) c->nonfinite[par] = 0;
        if (!meet(u)) return false;
        const uint32_t top = BF16 ? 0x7F80u : 0x7C00u;
        bool bad = false;
        for (int p = 0; p < NV; p++) {
            const uint4 *src = reinterpret_cast<const uint4 *>(ring_b + (st * NV + p) * MLA_CHUNK + r * 128 + h * 64);
#pragma unroll
            for (int k = 0; k < 4; k++) {
                const uint4 x = src[k];
                const uint32_t v[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int j = 0; j < 4; j++) bad |= (v[j] & top) == top || (v[j] >> 16 & top) == top;
            }
        }
        bad |= __shfl_xor_sync(0xffffffffu, (int)bad, 1) != 0;
        if (bad) {
            if (h == 0) atomicOr(reinterpret_cast<unsigned long long *>(&c->nonfinite[par]), 1ull << r);
            for (int p = 0; p < NV; p++)
#pragma unroll
                for (int k = 0; k < 4; k++)
                    reinterpret_cast<uint4 *>(ring_b + (st * NV + p) * MLA_CHUNK + r * 128 + h * 64)[k] = make_uint4(0, 0, 0, 0);
        }
        fence_async_smem();
        if (!meet(u)) return false;
        nf = *reinterpret_cast<volatile uint64_t *>(&c->nonfinite[par]);
        return true;
    }

    __device__ __forceinline__ void store_out(uint32_t tmem, bool live, int64_t token, int head, float ref, float l) {
        constexpr int half_cols = 64 * NV;
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        __half *out = reinterpret_cast<__half *>(q.out) + token * q.ot + head * q.oh + half * half_cols;
#pragma unroll 1
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
            q.lse[token * q.n_heads + head] = mla_lse(ref, l);
    }

    __device__ __forceinline__ void store_piece(uint32_t tmem, bool begins, bool live, int r, float ref, float l) {
        const int L = 128 * NV, half_cols = 64 * NV;
        const int slot = 2 * pair + begins;
        float *o = ws.o + ((size_t)slot * L + half * half_cols) * MLA_M + r;
#pragma unroll 1
        for (int col = 0; col < half_cols; col += 32) {
            float v[32];
            tmem_ld32(tmem + col, v);
#pragma unroll
            for (int k = 0; k < 32; k++)
                if (live) o[(size_t)(col + k) * MLA_M] = v[k];
            __syncwarp();
        }
        if (live) {
            float *ml = ws.ml + (size_t)slot * MLA_STATS + half * 2 * MLA_M + r;
            ml[0] = ref;
            ml[MLA_M] = l;
        }
    }
};

template <bool BF16, bool FP8, int NV>
__global__ void __launch_bounds__(FP8 ? 256 + 32 * MLA_XW : 256, 1)
    k_mla(MoeKvDev kv, MlaSeqAt seq_at, MoeMlaQuery q, const __grid_constant__ CUtensorMap tm, void *ws, int *error) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t *base = reinterpret_cast<uint8_t *>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
    using K = MlaKernel<BF16, FP8, NV>;
    const int pairs = gridDim.x / 2;
    uint8_t *ring_b = base, *ring_a = ring_b + MLA_SB * NV * MLA_CHUNK;
    uint8_t *ring_r = ring_a + NV * MLA_CHUNK, *sq = FP8 ? ring_r + 2 * MLA_CHUNK : ring_a + MLA_RA * MLA_CHUNK;
    MlaCtl *c = reinterpret_cast<MlaCtl *>(sq + mla_q_sm(128 * NV) * MLA_QCHUNK);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    constexpr int PROD = FP8 ? MLA_XW : 1;   // arrivals that fill a tile of ring B: the expanding warps, or the TMA's one
    if (tid == 0) {
        for (int i = 0; i < MLA_RA; i++) tc_mbar_init(&c->full_a[i], 1), tc_mbar_init(&c->empty_a[i], 1);
        for (int i = 0; i < 2; i++) tc_mbar_init(&c->full_r[i], 1), tc_mbar_init(&c->empty_r[i], 1);
        for (int i = 0; i < MLA_SB; i++) tc_mbar_init(&c->full_b[i], PROD), tc_mbar_init(&c->empty_b[i], FP8 ? 2 : 1);
        tc_mbar_init(&c->s_full[0], 1), tc_mbar_init(&c->s_full[1], 1);
        tc_mbar_init(&c->p_full[0], 4), tc_mbar_init(&c->p_full[1], 4);
        tc_mbar_init(&c->pv_done[0], 1), tc_mbar_init(&c->pv_done[1], 1);
        tc_mbar_init(&c->q_ready, 4), tc_mbar_init(&c->clean, 4), tc_mbar_init(&c->drain, FP8 ? 2 : 1);
        c->used = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        if (FP8)
            for (int i = 0; i < NV; i++) tc_expect(&c->full_a[i], MLA_CHUNK);   // the other CTA's first chunks
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
    if (tid == 0) c->w0 = w0, c->w1 = w1;
    if (w0 < w1 && w0 >= before && w0 < before + mine) {
        int64_t off = w0 - before;
        int b = b0;
        for (; b < b1 - 1; b++) {   // w0 lies in this stretch, so in its last sequence if in none before
            const int64_t k = seq_at(b).work();
            if (off < k) break;
            off -= k;
        }
        c->off0 = off, c->seq0 = b;
    }
    tmem_fence_before();
    if (FP8) cluster_sync_all();   // the other CTA's barriers are ready
    __syncthreads();
    tmem_fence_after();
    K k{kv, seq_at, q, &tm, mla_ws(ws, 128 * NV, pairs), error, ring_b, ring_a, ring_r, sq, c, (int)(blockIdx.x & 1), pair, lane, warp};
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
    moe_pdl_trigger();   // the join may take the SMs as they come free
    if (w0 < w1) {
        if (FP8 && warp >= 8) k.produce_expand();
        else if (warp == 0) k.produce_tma();
        else if (warp == 1) k.issue();
        else if (FP8 && warp == 2) k.forward();
        else if (warp >= 4 && warp < 8) k.rows();
    }
    __syncwarp();
    tmem_fence_before();
    if (FP8) cluster_sync_all();   // nothing of the other CTA's reaches this one any more
    __syncthreads();
    if (warp == 2) tmem_free(c->tmem, 512);
}

// ---------------------------------------------------------------------------
// Joins the pieces of cut units: per row the pieces' sums, each times
// 2^(its reference - the largest), in the order of the pairs (the same bits
// every time).  Every CTA reads the pairs' entries, so that the columns of the
// units that were cut (one for a single long sequence, up to one per pair)
// spread over the whole grid: 4 to 64 columns of a unit per CTA, each thread
// one row and a quarter of them.
// ---------------------------------------------------------------------------
constexpr int MLA_PAIRS = 256;   // CTA pairs at most
static_assert(MLA_PAIRS <= 4 * MLA_M, "a thread of the join per pair");
constexpr int MJ_THREADS = 4 * MLA_M;

// Columns col .. col + W - 1 of a thread's row over all pieces, U pieces' loads in flight: as many as the compiler fits
// into 64 registers for all three W without spilling.  1 x 25 joins 74 pieces of 80 rows in 19.9 us; 1 x 32 spills and
// takes 25.1; 1 x 16 takes 18.9 but makes it spill elsewhere (units of 2 or 3 pieces: 13.0 instead of 12.5).  4 x 4 for
// up to 4 pieces: half of 4 x 8's loads would be idle (32 sequences of 8192 rows: 113.1 against 114.5 us a call).
template <int W, int U, typename S>
__device__ __forceinline__ void join_columns(const float *o, const float *sw, int r, int pieces, size_t stride, S &&slot, float (&sum)[W]) {
    for (int k0 = 0; k0 < pieces; k0 += U) {
        float v[U][W], g[U];
#pragma unroll
        for (int k = 0; k < U; k++) {
            const bool in = k0 + k < pieces;
            const float *src = o + slot(in ? k0 + k : 0) * stride;
            g[k] = in ? sw[(k0 + k) * MLA_M + r] : 0.0f;
#pragma unroll
            for (int j = 0; j < W; j++) v[k][j] = in ? src[j * MLA_M] : 0.0f;
        }
#pragma unroll
        for (int k = 0; k < U; k++)
#pragma unroll
            for (int j = 0; j < W; j++) sum[j] = fmaf(g[k], v[k][j], sum[j]);
    }
}

template <bool BF16>
__global__ void __launch_bounds__(MJ_THREADS, 2) k_mla_join(MoeKvDev kv, MlaSeqAt seq_at, MoeMlaQuery q, void *wsp, int pairs) {
    extern __shared__ float sw[];   // [pieces][128] references, then factors
    __shared__ float sl[4][MLA_M];
    __shared__ int on[MLA_PAIRS], units[MLA_PAIRS], n_units;
    moe_pdl_wait();
    const MlaWs ws = mla_ws(wsp, kv.latent, pairs);
    const int r = threadIdx.x % MLA_M, part = threadIdx.x / MLA_M, L = kv.latent;
    const int me = threadIdx.x;
    if (me < pairs) on[me] = ws.tail[me].on;
    __syncthreads();
    if (me < pairs) {   // the pairs that begin a cut unit, in order
        int rank = 0;
        for (int j = 0; j < me; j++) rank += on[j];
        if (on[me]) units[rank] = me;
        if (me == pairs - 1) n_units = rank + on[me];
    }
    __syncthreads();
    const int n = n_units;
    int cols = 4;   // of an item: as few as give each CTA one
    while (cols < 64 && n * (L / cols) > (int)gridDim.x) cols <<= 1;
    const int per = L / cols, items = n * per;
    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int p = units[item / per], col0 = (item % per) * cols;
        const float *ml = ws.ml + (2 * col0 < L ? 0 : 2 * MLA_M) + r;   // (an item's columns lie in one half)
        const MlaWs::Tail t = ws.tail[p];
        const MlaSeq s = seq_at(t.seq);
        const uint32_t row = (uint32_t)t.block * MLA_M + r;
        const bool live = row < (uint32_t)s.n * q.n_heads;
        const int pieces = t.last - p + 1;
        // piece 0 is this pair's second slot, piece k > 0 pair p + k's first
        auto slot = [&](int k) { return (size_t)(k == 0 ? 2 * p + 1 : 2 * (p + k)); };
        __syncthreads();
#pragma unroll 8
        for (int k = part; k < pieces; k += 4) sw[k * MLA_M + r] = live ? ml[slot(k) * MLA_STATS] : -INFINITY;
        __syncthreads();
        float m = -INFINITY;
#pragma unroll 8
        for (int k = 0; k < pieces; k++) m = fmaxf(m, sw[k * MLA_M + r]);
        const float m0 = m == -INFINITY ? 0.0f : m;
        float l = 0.0f;
        __syncthreads();
#pragma unroll 8
        for (int k = part; k < pieces; k += 4) {
            const float f = ex2(sw[k * MLA_M + r] - m0);
            sw[k * MLA_M + r] = f;
            if (live) l = fmaf(f, ml[slot(k) * MLA_STATS + MLA_M], l);
        }
        sl[part][r] = l;
        __syncthreads();
        l = (sl[0][r] + sl[1][r]) + (sl[2][r] + sl[3][r]);
        const float f = l == 0.0f ? 0.0f : 1.0f / l;
        const int64_t token = s.q0 + row / (uint32_t)q.n_heads, head = row % (uint32_t)q.n_heads;
        if (live) {
            const int mine = cols / 4;   // 1, 2, 4, 8 or 16
            __half *out = reinterpret_cast<__half *>(q.out) + token * q.ot + head * q.oh;
            const size_t stride = (size_t)L * MLA_M;
            for (int c0 = 0; c0 < mine; c0 += 4) {
                const int col = col0 + part * mine + c0;
                const float *o = ws.o + (size_t)col * MLA_M + r;
                if (mine >= 4) {
                    float a[4] = {};
                    if (pieces <= 4) join_columns<4, 4>(o, sw, r, pieces, stride, slot, a);
                    else join_columns<4, 8>(o, sw, r, pieces, stride, slot, a);
                    *reinterpret_cast<uint2 *>(out + col) = make_uint2(pack2<BF16>(a[0] * f, a[1] * f), pack2<BF16>(a[2] * f, a[3] * f));
                } else if (mine == 2) {
                    float a[2] = {};
                    join_columns<2, 16>(o, sw, r, pieces, stride, slot, a);
                    *reinterpret_cast<uint32_t *>(out + col) = pack2<BF16>(a[0] * f, a[1] * f);
                } else {
                    float a[1] = {};
                    join_columns<1, 25>(o, sw, r, pieces, stride, slot, a);
                    *reinterpret_cast<uint16_t *>(out + col) = (uint16_t)pack2<BF16>(a[0] * f, 0.0f);
                }
            }
            if (col0 == 0 && part == 0 && q.lse)
                q.lse[token * q.n_heads + head] = mla_lse(m, l);
        }
    }
}

size_t mla_smem(int latent, bool fp8) {
    const int nv = latent / 128;
    return 1024 + (size_t)(MLA_SB * nv + (fp8 ? nv + 2 : MLA_RA)) * MLA_CHUNK + (size_t)mla_q_sm(latent) * MLA_QCHUNK + sizeof(MlaCtl);
}

template <bool BF16, bool FP8, int NV>
void launch(const MoeKvDev &kv, const MlaSeqAt &at, const MoeMlaQuery &q, const CUtensorMap &tm, void *ws, int pairs,
            int *error, cudaStream_t s) {
    static size_t done[MOE_MAX_DEVICES];
    const size_t smem = mla_smem(kv.latent, FP8);
    moe_smem_limit(k_mla<BF16, FP8, NV>, smem, done);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * pairs);
    cfg.blockDim = dim3(FP8 ? 256 + 32 * MLA_XW : 256);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim = {FP8 ? 2u : 1u, 1, 1};
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    cudaLaunchKernelEx(&cfg, k_mla<BF16, FP8, NV>, kv, at, q, tm, ws, error);
    moe_launch_pdl(k_mla_join<BF16>, dim3(4 * pairs), dim3(MJ_THREADS), sizeof(float) * pairs * MLA_M, s, kv, at, q, ws, pairs);
}

template <bool BF16, bool FP8, typename... A>
void by_latent(const MoeKvDev &kv, A &&...a) {
    switch (kv.latent) {
        case 128: launch<BF16, FP8, 1>(kv, a...); break;
        case 256: launch<BF16, FP8, 2>(kv, a...); break;
        case 384: launch<BF16, FP8, 3>(kv, a...); break;
        default: launch<BF16, FP8, 4>(kv, a...);
    }
}

int mla_pairs(int sms) { return sms / 2 < 1 ? 1 : sms / 2 > MLA_PAIRS ? MLA_PAIRS : sms / 2; }

}  // namespace

size_t moe_mla_ws_bytes(int latent, int sms) {
    const int pairs = mla_pairs(sms);
    return ((size_t)pairs * sizeof(MlaWs::Tail) + 255) / 256 * 256 + (size_t)pairs * 2 * (MLA_STATS + latent * MLA_M) * sizeof(float);
}

int moe_launch_mla(const MoeKvDev &kv, const MoeKvBatchDev &b, const MoeMlaQuery &q, void *ws, int sms, int *error,
                   cudaStream_t s, uint64_t *launches) {
    const MlaSeqAt at{b, q.n_heads, kv.page_shift};
    CUtensorMap tm{};
    // rows as 16-bit units (8-bit formats: the TMA only loads the rotary values, which start at unit latent / 2)
    if (moe_make_map_f16_sw128(&tm, kv.data, kv.row_bytes / 2, (uint64_t)kv.n_pages << kv.page_shift, 64,
                               kv.page_shift >= 6 ? MLA_N : 1u << kv.page_shift))
        return -1;
    switch (kv.format) {
        case MOE_KV_F16: by_latent<false, false>(kv, at, q, tm, ws, mla_pairs(sms), error, s); break;
        case MOE_KV_BF16: by_latent<true, false>(kv, at, q, tm, ws, mla_pairs(sms), error, s); break;
        case MOE_KV_FP8_F16: by_latent<false, true>(kv, at, q, tm, ws, mla_pairs(sms), error, s); break;
        default: by_latent<true, true>(kv, at, q, tm, ws, mla_pairs(sms), error, s);
    }
    LAUNCH_COUNT(launches);
    LAUNCH_COUNT(launches);
    return 0;
}
