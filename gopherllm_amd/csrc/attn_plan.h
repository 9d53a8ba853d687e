// attn_plan.h -- how attention over cache ranges is split over workgroups and
// what its workspace holds.  Host arithmetic only, so it is tested without a device.
#pragma once

#include <stddef.h>

#include <algorithm>

namespace gllm {

constexpr int kSeqWaves = 4;                  // waves of a workgroup
constexpr int kSeqQuantum = 128;              // positions: one step of every shape of workgroup, or more
constexpr int kSeqTarget = 512;               // workgroups: two for each of the 256 CUs
constexpr int kSeqMaxSplits = 64;             // partial results of a query row from one range
constexpr int kSeqMaxRows = 1 << 22;          // n * n_heads: a workgroup each has to fit a launch

// Query rows of a kv head: n tokens x r heads.
struct SeqPlan {
    int r;                    // query heads of a kv head
    int nq, rw, row_blocks;   // of the shared range: blocks of 16 nq rw rows, over rw waves
    int chunk, chunks;        // positions of a workgroup, workgroups per row block
    int own_blocks, splits;   // of each token's own range (16 rows a block)
    int slots;                // partial results of a query row
    size_t rows;              // n * n_heads
    size_t parts;             // partial results that the workspace has room for
};

inline int ceil_div(int a, int b) { return (int)(((long long)a + b - 1) / b); }

inline bool seq_much(long long per_kv, int n_kv, int hd, int len) { return per_kv * (double)len * n_kv * hd > 4.0e9; }

// Room for rows x slots partial results that never falls as n, len or most grow,
// so a workspace for the most of each serves every smaller call (the slots
// themselves fall where a chunk grows by a step: 64 over 8192 positions, 33 over
// 8193).  A row has at most 64 and one for each 128 positions of either range, and
//   shared  n_kv * row_blocks * chunks <= kSeqTarget, or one chunk, with row_blocks
//           of at most 16 nq rw of a kv head's rows (nq as for the largest head)
//   own     n * n_kv * own_blocks * splits <= kSeqTarget, or one split
inline size_t seq_parts(int n, int n_heads, int n_kv, int len, int most) {
    const size_t rows = (size_t)n * n_heads;
    const int r = n_heads / n_kv;
    const long long per_kv = (long long)n * r;
    const auto cap = [&](int positions) { return rows * std::min(kSeqMaxSplits, ceil_div(positions, kSeqQuantum)); };
    size_t parts = 0;
    if (len > 0) {
        const size_t block = per_kv <= 16 ? 16 : per_kv > 64 && seq_much(per_kv, n_kv, 128, len) ? 32 * kSeqWaves : 16 * kSeqWaves;
        parts += std::min(cap(len), std::max(rows, kSeqTarget * block));
    }
    if (most > 0) {
        const size_t own_blocks = ceil_div(r, 16);
        parts += std::min(cap(most), std::max(rows, ((size_t)kSeqTarget * r + own_blocks - 1) / own_blocks));
    }
    return parts;
}

// n tokens, heads / kv heads of hd, `len` shared positions, own ranges planned for
// `most` positions (0: none).
inline SeqPlan seq_plan(int n, int n_heads, int n_kv, int hd, int len, int most) {
    SeqPlan p{};
    p.r = n_heads / n_kv;
    p.rows = (size_t)n * n_heads;
    const long long per_kv = (long long)n * p.r;
    // Up to 16 rows: the waves split positions.  More: they share the positions,
    // 16 rows each, or 32 where that leaves no more padding and there is work
    // enough that reading the tiles half as often counts.  With 16 and 32 rows, 8
    // kv heads of 128, rows x positions: 256 x 32768 79 and 74 us, 1024 x 4000 59
    // and 54, 256 x 16000 45.1 and 45.5, 256 x 8000 29 and 33, 128 x 8000 22 and
    // 28; 8 of 80: 640 x 10000 56 and 54, 640 x 4000 33 and 35; 2 of 64: 1024 x
    // 32768 55 and 52, 1024 x 8000 24 and 28; one of 128: 2048 x 64000 147 and 131,
    // 2048 x 16000 46.3 and 46.9, 2048 x 4000 26 and 28; 4 of 32: 2048 x 16000 72
    // and 59, 2048 x 4000 28.9 and 28.4.
    p.rw = per_kv <= 16 ? 1 : kSeqWaves;
    const bool fits = (per_kv + 63) / 64 * 64 == (per_kv + 127) / 128 * 128;
    p.nq = fits && seq_much(per_kv, n_kv, hd, len) ? 2 : 1;
    p.row_blocks = (int)((per_kv + 16 * p.nq * p.rw - 1) / (16 * p.nq * p.rw));
    if (len > 0) {
        const long long per_chunk = (long long)n_kv * p.row_blocks;
        const auto chunks = [&](int target) { return (int)std::max(1LL, std::min((long long)kSeqMaxSplits, target / per_chunk)); };
        // Many rows of a shared range keep the matrix cores busy and the own
        // ranges memory: where these are planned as long, half the shared workgroups
        // leave room for both on a CU that holds two of them, as it does for heads
        // past 96 (64 requests of 32 / 8 heads of 128 over 32768 rows and 513 of
        // their own: 98 us with 512, 92 with 256; while those are one row, 81 and
        // 84).  For smaller heads three or four fit (64 of 80: 87 and 112 us; of 64:
        // 51 and 61), and there only chunks of a few steps do better halved (64 of
        // 96 over 2000 rows: 22 and 18).
        int want = chunks(kSeqTarget);
        if (p.rw > 1 && (long long)n * most >= len && (hd > 96 || ceil_div(len, want) <= kSeqQuantum)) want = chunks(kSeqTarget / 2);
        p.chunk = ceil_div(ceil_div(len, want), kSeqQuantum) * kSeqQuantum;
        p.chunks = ceil_div(len, p.chunk);
    }
    if (most > 0) {
        p.own_blocks = ceil_div(p.r, 16);
        const long long per_split = (long long)n * n_kv * p.own_blocks;
        // as many as the shared range's workgroups leave, and kSeqTarget / 4 at least
        // (8 requests over 4001 rows and up to 640 of their own: 16.3 us with 320
        // workgroups for these, 14.9 with the 256 that are left).  More tokens x kv
        // heads than that wait for shared ones to end: 33 requests of 8 kv heads
        // are 264 beside 480, 64 are 512 beside 256.
        const int left = std::max(kSeqTarget - n_kv * p.row_blocks * p.chunks, kSeqTarget / 4);
        const int want = (int)std::max(1LL, std::min((long long)kSeqMaxSplits, left / per_split));
        p.splits = std::min(want, ceil_div(most, kSeqQuantum));
    }
    p.slots = p.chunks + p.splits;
    p.parts = seq_parts(n, n_heads, n_kv, len, most);
    return p;
}

// Floats of the partial results: base and sum of each, and its output.
inline size_t seq_floats(const SeqPlan& p, int hd) { return p.parts * (2 + (size_t)hd) + 64; }

// What attention with weights works in, in floats: one token's query rows (up to
// 16 a kv head) keep their scores, more keep their operands (f16 pairs, in the matrix cores' order),
// scales and final base and 1 / sum; then the partial results.
struct MassSpace {
    bool kept;
    int sstride;  // of a row's scores
    int tiles;    // of 16 query rows of a kv head
    size_t scale, ml, parts;
};
inline MassSpace mass_space(const SeqPlan& p, int hd, int n_kv, int len) {
    MassSpace m{};
    m.kept = p.rw == 1 && p.rows == (size_t)n_kv * p.r;
    if (m.kept) {
        m.sstride = (int)(((size_t)len + 3) / 4 * 4);
        m.parts = p.rows * (size_t)m.sstride;
    } else {
        m.tiles = p.row_blocks * p.rw * p.nq;
        const size_t all = (size_t)m.tiles * n_kv;
        m.scale = all * 2 * ceil_div(hd, 32) * 64 * 4;  // 16 bytes a lane for each 32 dims of both parts
        m.ml = m.scale + all * 16;
        m.parts = m.ml + (p.rows * 2 + 3) / 4 * 4;
    }
    return m;
}

// Floats of it with the partial results: like seq_parts, as many as any call of
// fewer tokens over fewer positions needs, one token's kept scores among them.
inline size_t mass_floats(const SeqPlan& p, int hd, int n_kv, int len) {
    const int n_heads = p.r * n_kv, n = (int)(p.rows / n_heads);
    const size_t one = p.r <= 16 ? n_heads * (((size_t)len + 3) / 4 * 4) : 0;
    return std::max(mass_space(p, hd, n_kv, len).parts, one) + seq_parts(n, n_heads, n_kv, len, n - 1) * (2 + (size_t)hd) + 64;
}

// Rows a .. b - 1 of a cache of max_len rows that the range start, len names.
struct RowSpan {
    int a, b;
};
#ifdef __HIPCC__
__host__ __device__
#endif
inline RowSpan clip_rows(int start, int len, int max_len) {
    const long long lo = start < 0 ? 0 : start;
    long long hi = (long long)start + (len < 0 ? 0 : len);
    if (hi > max_len) hi = max_len;
    RowSpan s;
    s.a = lo > max_len ? max_len : (int)lo;
    s.b = hi < s.a ? s.a : (int)hi;
    return s;
}

}  // namespace gllm
