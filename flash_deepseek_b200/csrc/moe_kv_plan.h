// moe_kv_plan.h -- how the MLA attention kernel divides its work, for the
// device and for a CPU test.
//
// The query rows of a sequence (n tokens x heads, token-major) are cut into
// blocks of MLA_M rows; a block against the sequence's cache rows, in tiles of
// MLA_N, is a unit.  All units' tiles, one after the other, are divided evenly
// among the CTA pairs, so a pair walks over segments: whole units, the end of
// one that an earlier pair began, the start of one that a later pair ends.
// Units that are cut are joined afterwards from the pieces' sums.
#pragma once
#include <stdint.h>

#define MLA_M 128   // query rows of a block (rows of the tensor core's tile)
#define MLA_N 64    // cache rows of a tile

#ifdef __CUDACC__
#define KV_HD __host__ __device__ __forceinline__
#else
#define KV_HD inline
#endif

struct MlaSeq {
    int q0, n;        // first row of the call, rows of the call
    int ctx, len;     // rows in front of them, rows in all (as far as the page table reaches)
    int blocks, tiles;
    int bad;          // bounds out of range: the sequence is skipped; or the page table is too short
    KV_HD int64_t work() const { return (int64_t)blocks * tiles; }
};

// (A table may span more rows than an int holds, pages repeated; no sequence gets past 2^31 - 65.)
KV_HD MlaSeq mla_seq(int q0, int q1, int ctx, int n_tokens, int heads, int64_t table_rows) {
    constexpr int64_t most = 0x7FFFFFFF - MLA_N;   // s.len and its last tile's end are ints
    MlaSeq s{};
    if (table_rows > most) table_rows = most;
    if (q0 < 0 || q1 < q0 || q1 > n_tokens || ctx < 0) {
        s.bad = 1;
        return s;
    }
    s.q0 = q0;
    s.n = q1 - q0;
    if (s.n == 0) return s;
    s.ctx = ctx;
    const int64_t len = (int64_t)ctx + s.n;
    s.bad = len > table_rows;
    s.len = (int)(s.bad ? table_rows : len);
    s.blocks = (int)(((int64_t)s.n * heads + MLA_M - 1) / MLA_M);
    s.tiles = (s.len + MLA_N - 1) / MLA_N;   // at least 1: a page table has a row
    return s;
}

// First tile of pair p's share (pair p + 1's is its end): as even as tiles go,
// and pairs without any only behind the last one that has some.
KV_HD int64_t mla_share(int64_t total, int p, int pairs) {
    const int64_t each = total / pairs, more = total % pairs;
    return each * p + (p < more ? p : more);
}

struct MlaSeg {
    int seq, block, tile0, tile1;
    int whole;        // the unit begins and ends here
};

// The walk over a pair's segments.  `seq_at(b)` gives sequence b.
struct MlaWalk {
    int64_t w, w1, off;   // next tile, end of the share, the next tile's place in its sequence
    int seq, n_seqs;
    MlaSeq s;             // of the last segment

    template <typename F>
    KV_HD bool next(MlaSeg &g, F &&seq_at) {
        if (w >= w1) return false;
        s = seq_at(seq);
        while (off >= s.work()) {   // past its end, or nothing to do in it
            if (++seq >= n_seqs) return false;
            off = 0;
            s = seq_at(seq);
        }
        g.seq = seq;
        g.block = (int)(off / s.tiles);
        g.tile0 = (int)(off - (int64_t)g.block * s.tiles);
        const int64_t left = w1 - w;
        g.tile1 = left < s.tiles - g.tile0 ? g.tile0 + (int)left : s.tiles;
        g.whole = g.tile0 == 0 && g.tile1 == s.tiles;
        w += g.tile1 - g.tile0;
        off += g.tile1 - g.tile0;
        return true;
    }
};

// The last pair that holds a piece of a unit of which `rest` > 0 tiles follow
// behind pair p's share, which ends at tile w.
KV_HD int mla_last_pair(int64_t total, int p, int pairs, int64_t w, int64_t rest) {
    int last = p + 1;
    while (mla_share(total, last + 1, pairs) < w + rest) last++;
    return last;
}
