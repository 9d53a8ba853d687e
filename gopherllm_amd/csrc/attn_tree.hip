// attn_tree.hip -- attention of drafted tokens: each of n requests has a context
// in the cache and, in the rows behind it, a tree of up to 256 drafted tokens.  A
// token sees the context, its ancestors and itself.  No counterpart in the
// reference, which decodes one token at a time (attendHeadGroup model.go:1516).
//
// The mathematics and the layout are attn_seq.h's.  The context and the drafted
// rows are one range, split over workgroups; only its last steps look at the tree.
// A second launch joins the parts, unless one workgroup has them all.
#include <algorithm>
#include <type_traits>

#include "attn_seq.h"

namespace gllm {

constexpr int kTreeTokens = 256, kTreeWords = kTreeTokens / 32;

struct TreeArgs {
    const float* q;  // [n][m][n_heads][hd]
    float* out;
    const uint16_t *K, *V;  // row 0 of the layer
    int kd_k, kd_v;         // row strides
    int n, m, n_heads, n_kv, r, hd, max_len;
    int row_blocks, target, splits;  // blocks of all m tokens; units to make; partial results that a row has room for
    const int32_t *starts, *lens, *parents, *counts;  // counts: or null, m each
    float scale;  // scale * log2(e)
    float per_r, per_target, per_split;  // 1 / r; a little above 1 / target and 1 / splits
    float *pm, *pl, *po;  // [request][token][head][split] base, sum, [hd] output
    int32_t* used;        // [request] splits
};

// The token of query row rr of a kv head, rr / r: rr + 1/2 is at least 1 / 2r away
// from a multiple of r, more than the product's rounding for the 2^20 rows taken.
__device__ __forceinline__ int tree_token(const TreeArgs& t, int rr) { return (int)(((float)rr + 0.5f) * t.per_r); }

// The rows lo .. hi - 1 that a request's tokens see, drafted ones from d0 on.
struct TreeSpan {
    int count, lo, hi, d0;
};
struct TreeInts {
    int count, start, len;
};
__device__ __forceinline__ TreeInts tree_ints(const TreeArgs& t, int i) {  // all three on their way at once
    return {*(t.counts ? t.counts + i : t.lens + i), t.starts[i], t.lens[i]};
}
__device__ __forceinline__ TreeSpan tree_span(const TreeArgs& t, const TreeInts& x) {
    TreeSpan s;
    s.count = t.counts ? min(max(x.count, 0), t.m) : t.m;
    const long long start = x.start, behind = start + max(x.len, 0);
    s.d0 = (int)max(min(behind, (long long)t.max_len), (long long)-kTreeTokens);
    s.lo = (int)min(max(start, 0LL), (long long)t.max_len);
    s.hi = max(s.lo, (int)max(min(behind + s.count, (long long)t.max_len), 0LL));
    return s;
}

// Rows of a unit: so many that the requests' ranges make no more than `target` units
// and a rest each, and none more than `splits`.  The quotients may come out one too
// large, never too small.
template <int QUANTUM>
__device__ __forceinline__ int tree_chunk(const TreeArgs& t, float total, int longest) {
    const int c = max((int)fminf(total * t.per_target, (float)kSeqMaxLen), (int)((float)longest * t.per_split)) + 1;
    return (max(c, kSeqQuantum) + QUANTUM - 1) / QUANTUM * QUANTUM;
}
__device__ __forceinline__ int tree_used(const TreeSpan& s, int chunk) {
    return max(1, (int)(((unsigned)(s.hi - s.lo) + (unsigned)chunk - 1) / (unsigned)chunk));
}

// Of several requests, the one that unit u belongs to, the unit's number in it, and
// the rows of a unit: a request a lane, 64 at a time.  Ranges are split by what the
// requests have, so that long ones take more workgroups than short ones (16 requests
// of up to 2500 rows, split alike: 40 us, so: 24).
template <int BLOCK, int QUANTUM>
__device__ __forceinline__ bool tree_find(const TreeArgs& t, int u, int& i, int& rest, int& chunk, TreeSpan& span) {
    const auto blocks = [&](const TreeSpan& s) { return (int)((unsigned)(s.count * t.r + BLOCK - 1) / BLOCK); };
    const int lane = threadIdx.x & 63;
    TreeSpan s{};
    const auto load = [&](int i0) {
        s = TreeSpan{};
        if (i0 + lane < t.n) s = tree_span(t, tree_ints(t, i0 + lane));
    };
    float total = 0.0f;  // off by up to n 2^-30 of itself, which per_target has in it
    int longest = 0;
    for (int i0 = 0; i0 < t.n; i0 += 64) {
        load(i0);
        if (s.count) {
            total += (float)(s.hi - s.lo) * (float)blocks(s);
            longest = max(longest, s.hi - s.lo);
        }
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) total += __shfl_xor(total, off);
    chunk = tree_chunk<QUANTUM>(t, total, (int)wave_max_u32((uint32_t)longest));
    int before = 0;
    for (int i0 = 0; i0 < t.n; i0 += 64) {
        if (t.n > 64) load(i0);  // the last 64 are in registers
        const int units = s.count ? tree_used(s, chunk) * blocks(s) : 0;
        int upto = units;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int x = __shfl_up(upto, off);
            if (lane >= off) upto += x;
        }
        const uint64_t past = __ballot(before + upto > u);
        if (past) {
            const int at = __ffsll((unsigned long long)past) - 1;
            i = i0 + at;
            rest = u - before - __builtin_amdgcn_readlane(upto - units, at);
            span.count = __builtin_amdgcn_readlane(s.count, at);
            span.lo = __builtin_amdgcn_readlane(s.lo, at);
            span.hi = __builtin_amdgcn_readlane(s.hi, at);
            span.d0 = __builtin_amdgcn_readlane(s.d0, at);
            return true;
        }
        before += __builtin_amdgcn_readlane(upto, 63);
    }
    return false;
}

// What each token sees of the drafted ones: bit j of seen[..][t] is token j, with
// a word of zeros behind the last.  A token goes up from parent to parent, over a
// run of tokens that follow each other a word at a time (run: bit t is whether t's
// parent is t - 1).  A parent that is not an earlier token is none.  Every thread
// of the workgroup calls this, with its token's parent.
struct TreeSeen {
    uint32_t seen[kTreeWords + 1][kTreeTokens];
    int up[kTreeTokens];
    uint32_t run[kTreeWords];
};
__device__ __forceinline__ void tree_seen(int parent, int count, TreeSeen& s) {
    const int t = threadIdx.x, words = (count + 31) / 32;
    const int p = t < count && parent < t ? parent : -1;
    const uint64_t runs = __ballot(t > 0 && p == t - 1);
    if (t < kTreeTokens) {
        s.up[t] = p;
        if ((t & 31) == 0) s.run[t >> 5] = (uint32_t)(runs >> (t & 32));
#pragma unroll
        for (int w = 0; w <= kTreeWords; w++)
            if (w <= words) s.seen[w][t] = 0;
    }
    __syncthreads();
    if (t < count) {
        int cur = t, word = t >> 5;
        uint32_t bits = 0;
        while (cur >= 0) {  // falls in every round
            if (cur >> 5 != word) {
                s.seen[word][t] = bits;
                bits = 0;
                word = cur >> 5;
            }
            const uint32_t upto = (2u << (cur & 31)) - 1, ends = ~s.run[word] & upto;
            const int first = ends ? 31 - __clz((int)ends) : 0;  // of the run in this word
            bits |= upto & ~((1u << first) - 1);
            cur = ends ? s.up[32 * word + first] : 32 * word - 1;
        }
        s.seen[word][t] = bits;
    }
    __syncthreads();
}

// Bit i: whether token tok sees row pb + i, below p1.
__device__ __forceinline__ uint32_t tree_bits(const TreeSeen& s, int tok, int d0, int pb, int p1) {
    const int j = pb - d0;  // the drafted token of row pb
    uint32_t b;
    if (j < 0) {  // above -kStep
        b = ((1u << -j) - 1) | s.seen[0][tok] << -j;
    } else {
        const uint64_t two = (uint64_t)s.seen[(j >> 5) + 1][tok] << 32 | s.seen[j >> 5][tok];
        b = (uint32_t)(two >> (j & 31));
    }
    return p1 - pb < 32 ? b & ((1u << (p1 - pb)) - 1) : b;
}

// A step of 32 positions: scores from the K tile at kt (LDS), weights, and the
// weighted rows of the V tile at vt added to the sums.  TREE: position i of the
// step counts where bits[nq] has it.
template <int HD, int NQ, bool TREE>
__device__ __forceinline__ void tree_step(SeqRows<HD, NQ>& q, const char* kt, const char* vt, const uint32_t (&bits)[NQ], float minus1) {
    constexpr int KK = HD / 32, DT = HD / 16;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const float ninf = -__int_as_float(0x7f800000);
    h8 k[2][KK];
#pragma unroll
    for (int kk = 0; kk < KK; kk++)
#pragma unroll
        for (int t = 0; t < 2; t++) k[t][kk] = *(const h8*)(kt + (16 * t + col) * HD * 2 + 16 * ((4 * kk + grp) ^ k_swizzle<HD>(col)));
    // V operand k = 8 grp + 4 t + j is position 16 t + 4 grp + j
    const int vr = 4 * grp + (col >> 2);
    const char* vp = vt + vr * HD * 2 + 8 * (col & 1);
    const auto rows = [&](int dt) {
        s4 x[2];
#pragma unroll
        for (int t = 0; t < 2; t++)  // rows 16 apart share their swizzle
            x[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(
                vp + 16 * t * HD * 2 + 16 * ((2 * dt + ((col & 3) >> 1)) ^ v_swizzle<HD>(vr))));
        h8 f;
        const h4 y0 = __builtin_bit_cast(h4, x[0]), y1 = __builtin_bit_cast(h4, x[1]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            f[j] = y0[j];
            f[4 + j] = y1[j];
        }
        return f;
    };
    __builtin_amdgcn_sched_barrier(0);  // all of K is on its way before the first product
    f4 s[NQ][2];
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int t = 0; t < 2; t++) s[nq][t] = f4{0, 0, 0, 0};
#pragma unroll
    for (int kk = 0; kk < KK; kk++) {
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) s[nq][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][kk], q.lo[nq][kk], s[nq][t], 0, 0, 0);
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) s[nq][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][kk], q.hi[nq][kk], s[nq][t], 0, 0, 0);
    }
    float cc[NQ], mx[NQ];
    bool over = false;
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        cc[nq] = TREE ? 1.0f : q.c[nq];
        mx[nq] = ninf;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                if constexpr (TREE) s[nq][t][j] = bits[nq] >> (16 * t + 4 * grp + j) & 1 ? s[nq][t][j] * q.c[nq] : ninf;
                mx[nq] = fmaxf(mx[nq], s[nq][t][j]);
            }
        over |= mx[nq] * cc[nq] - q.base[nq] > kSeqRoom;
    }
    // a query whose scores pass what its base allows gets a new one
    if (__any(over)) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            float top = fmaxf(mx[nq], __shfl_xor(mx[nq], 16));
            top = fmaxf(top, __shfl_xor(top, 32)) * cc[nq];
            const float nb = top - q.base[nq] > kSeqRoom ? top - kSeqLift : q.base[nq];
            const float f = __builtin_amdgcn_exp2f(q.base[nq] - nb);
            q.l[nq] *= f;
#pragma unroll
            for (int dt = 0; dt < DT; dt++) q.o[nq][dt] *= f;
            q.base[nq] = nb;
        }
    }
    h8 wh[NQ], wl[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; nq++)
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                // the two parts of a weight, to nearest (what cannot be held must not
                // all be on one side)
                const float w0 = __builtin_amdgcn_exp2f(fmaf(s[nq][t][j], cc[nq], -q.base[nq]));
                const float w1 = __builtin_amdgcn_exp2f(fmaf(s[nq][t][j + 1], cc[nq], -q.base[nq]));
                q.l[nq] += w0 + w1;
                const h2 hi = __builtin_convertvector((f2{w0, w1}), h2);
                const h2 lo = __builtin_convertvector((f2{fmaf((float)hi[0], minus1, w0), fmaf((float)hi[1], minus1, w1)}), h2);
                wh[nq][4 * t + j] = hi[0];
                wh[nq][4 * t + j + 1] = hi[1];
                wl[nq][4 * t + j] = lo[0];
                wl[nq][4 * t + j + 1] = lo[1];
            }
    u4 cut = {0, 0, 0, 0};
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
        h8 x = rows(dt);
        if constexpr (TREE) {
            // Infinities and NaN of drafted tokens must not meet the weight of 0 that
            // others have for them: they are taken as the largest finite values, and
            // who sees their row gets NaN.
            const h8 y = __builtin_elementwise_min(__builtin_elementwise_max(x, (h8)(_Float16)-65504.0f), (h8)(_Float16)65504.0f);
            cut |= __builtin_bit_cast(u4, x) ^ __builtin_bit_cast(u4, y);
            x = y;
        }
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) q.o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, wl[nq], q.o[nq][dt], 0, 0, 0);
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) q.o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, wh[nq], q.o[nq][dt], 0, 0, 0);
    }
    if constexpr (TREE) {
#pragma unroll
        for (int i = 0; i < 4; i++) {  // over the 16 lanes that have the same positions
            cut[i] |= dpp_u<kQuadXor1>(cut[i]);
            cut[i] |= dpp_u<kQuadXor2>(cut[i]);
            cut[i] |= dpp_u<kRowHalfMirror>(cut[i]);
            cut[i] |= dpp_u<kRowMirror>(cut[i]);
        }
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t hit = j & 1 ? cut[2 * t + (j >> 1)] >> 16 : cut[2 * t + (j >> 1)] & 0xFFFFu;
#pragma unroll
                for (int nq = 0; nq < NQ; nq++)
                    if (hit && bits[nq] >> (16 * t + 4 * grp + j) & 1) q.l[nq] = __int_as_float(0x7fc00000);
            }
    }
}

// LDS of a workgroup of RW x PW waves: a ring of ST stages for each of the PW parts
// of the positions, then the parts' sums.
template <int HD, int NQ, int RW, int PW, int ST>
struct TreeLds {
    static constexpr int STAGE = 2 * kStep * HD * 2;  // bytes of K and V of a step
    static constexpr int RING = PW * ST * STAGE;
    static constexpr int SUMS = PW > 1 ? RW * PW * NQ * (HD / 16) * 64 * 16 : 0;
    static constexpr int BYTES = RING > SUMS ? RING : SUMS;
};

// RW waves take 16 NQ query rows each over the same positions and share K and V
// tiles that direct copies bring into a ring of ST stages; PW such groups of waves
// take a part of the workgroup's positions each and join their sums in LDS.
//
// Long contexts of many rows are bound by the matrix cores and what waits between
// their products: 64 tokens of 32 / 8 heads of 128 over 32768 rows (134 MB, 69 GFLOP
// with both parts) take 69 us, 1.0 PFLOP/s where a large library product reaches 1.15;
// the cores are busy 52 % of the waves' time, LDS 15 %, without a bank conflict.
// Two stages are enough, as the steps of a CU's waves do not run in time with each
// other: rings of three and four measured the same.  With 16 rows a wave they would also
// leave a CU fewer waves; with 32 the joined sums fill LDS (128 KB for heads of 128, as
// much as a ring of four) and a CU has one workgroup either way.  Short
// contexts are bound by latency: 33 tokens over 4001 rows take 16 to 18 us, seven steps of
// about 1 us and the rest the start (lengths, queries, first tiles) and the end (sums
// joined in LDS, partial results written).  One step's latency is K's reads, 8 products in a row, exponentials, V's reads and
// products; starting the next step's reads under them took registers and no time off.
template <int HD, int NQ, int RW, int PW, int ST>
__global__ __launch_bounds__(64 * RW * PW, 2) void tree_attend_kernel(TreeArgs t) {
    constexpr int DT = HD / 16, CH = HD / 8, TILE = kStep * HD * 2, STAGE = TreeLds<HD, NQ, RW, PW, ST>::STAGE;
    constexpr int COPIES = 2 * kStep * CH / 64, U = COPIES / RW;  // copies of a stage, 64 chunks each, and of a wave
    static_assert(COPIES % RW == 0, "as many copies for each wave");
    static_assert(64 * RW * PW >= kTreeTokens, "a token a thread");
    __shared__ __align__(16) char lds[TreeLds<HD, NQ, RW, PW, ST>::BYTES];
    __shared__ TreeSeen seen;
    __shared__ float sm[PW][RW][NQ][16], sl[PW][RW][NQ][16];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4, pw = wave / RW, rw = wave % RW;
    const int g = blockIdx.x % t.n_kv;
    // the unit: rows a0 .. a1 - 1 of request i for the query rows of its block rb
    int i = 0, rb, slot, chunk = 0;
    TreeSpan span{};
    TreeInts ints{};
    // one request, or a workgroup for each range: its place is known before the lengths are
    const bool fixed = t.n == 1 || t.splits == 1;
    if (fixed) {
        const unsigned u = blockIdx.x / t.n_kv, q = u / (unsigned)t.row_blocks;
        rb = (int)(u - q * t.row_blocks);
        i = t.n == 1 ? 0 : (int)q;
        slot = t.n == 1 ? (int)q : 0;
        ints = tree_ints(t, i);
    } else {
        int rest = 0;
        if (!tree_find<16 * NQ * RW, kStep * PW>(t, blockIdx.x / t.n_kv, i, rest, chunk, span)) return;
        i = __builtin_amdgcn_readfirstlane(i);
        rest = __builtin_amdgcn_readfirstlane(rest);
        const unsigned rbs = __builtin_amdgcn_readfirstlane((unsigned)(span.count * t.r + 16 * NQ * RW - 1) / (16 * NQ * RW));
        slot = rbs == 1 ? rest : (int)((unsigned)rest / rbs);
        rb = rest - slot * (int)rbs;
    }
    const size_t first = (size_t)i * t.m * t.n_heads;  // the request's first query row
    const int row0 = (rb * RW + rw) * 16 * NQ;
    SeqQueries<HD, NQ> x;
    seq_load_queries<HD, NQ>(t.q + first * t.hd, t.n_heads, t.m * t.r, t.r, t.hd, g, row0, [&](int rr) { return tree_token(t, rr); }, x);
    int parent = (int)threadIdx.x < t.m ? t.parents[(size_t)i * t.m + threadIdx.x] : -1;
    if (fixed) {
        span = tree_span(t, ints);
        chunk = tree_chunk<kStep * PW>(t, (float)(span.hi - span.lo) * (float)t.row_blocks, span.hi - span.lo);
    }
    // one value for the wave, which the compiler cannot see
    const int count = __builtin_amdgcn_readfirstlane(span.count), lo = __builtin_amdgcn_readfirstlane(span.lo);
    const int hi = __builtin_amdgcn_readfirstlane(span.hi), d0 = __builtin_amdgcn_readfirstlane(span.d0);
    chunk = __builtin_amdgcn_readfirstlane(chunk);
    const int used = __builtin_amdgcn_readfirstlane(tree_used(TreeSpan{count, lo, hi, d0}, chunk)), rows = count * t.r;
    if (slot >= used || rb * RW * 16 * NQ >= rows) return;
    const int a0 = min(hi, lo + slot * chunk), a1 = a0 + min(hi - a0, chunk);
    const bool tree = a1 > d0 && a1 > a0;
    const int steps = ((a1 - a0 + PW - 1) / PW + kStep - 1) / kStep;  // of the longest part
    const int p0 = min(a1, a0 + pw * steps * kStep), p1 = min(a1, p0 + steps * kStep);

    int off[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int c = RW * u + rw;  // of the stage
        const bool v = c >= COPIES / 2;
        const int e = 64 * (v ? c - COPIES / 2 : c) + lane, rr = e / CH, d = 8 * (e % CH ^ (v ? v_swizzle<HD>(rr) : k_swizzle<HD>(rr)));
        off[u] = d < t.hd ? (rr * (v ? t.kd_v : t.kd_k) + d) * 2 : kPastEnd;
    }
    char* ring = lds + pw * ST * STAGE;
    const uint32_t ring_at = lds_addr(ring);
    const auto copy = [&](int step) {  // past the last step the buffers are empty, and nothing is read
        const int pb = min(p0 + step * kStep, p1);
        const u4 k = SeqBuffer(t.K, t.kd_k, t.hd, g, pb, p1).words(), v = SeqBuffer(t.V, t.kd_v, t.hd, g, pb, p1).words();
        const uint32_t to = ring_at + (step % ST) * STAGE;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int c = RW * u + rw;
            lds_buffer16(c >= COPIES / 2 ? v : k, off[u], to + 1024 * c);
        }
    };
#pragma unroll
    for (int i = 0; i < ST - 1; i++) copy(i);
    SeqRows<HD, NQ> q;
    seq_split_queries<HD, NQ>(t.scale, x, q);
    if (tree) tree_seen(parent, count, seen);
    float minus1 = -1.0f;  // a register, so that w - hi is one mixed-precision fma of hi as it lies
    asm volatile("" : "+v"(minus1));
    const bool busy = row0 < rows;  // a wave without rows only copies
    const auto step = [&](int it, auto kind) {
        // this wave's copies of the stage are in (ST - 2 later stages may be out),
        // and its reads of the stage before, whose place the next copies take
        wait_vmem_le<(ST - 2) * U>();
        wait_lgkm0();
        lds_barrier();
        copy(it + ST - 1);
        const int pb = p0 + it * kStep;
        if (!busy || pb >= p1) return;
        const char* kt = ring + (it % ST) * STAGE;
        uint32_t bits[NQ];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) bits[nq] = kind ? tree_bits(seen, min(tree_token(t, row0 + 16 * nq + col), count - 1), d0, pb, p1) : 0;
        tree_step<HD, NQ, decltype(kind)::value>(q, kt, kt + TILE, bits, minus1);
    };
    // loops of their own: with both steps in one, wide heads spill 43 registers
    int it = 0;
    for (; it < steps && p0 + (it + 1) * kStep <= d0; it++) step(it, std::false_type{});
    for (; it < steps; it++) step(it, std::true_type{});
    wait_vmem_le<0>();  // no copy outlives the workgroup

    float l[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        l[nq] = q.l[nq];
        l[nq] += __shfl_xor(l[nq], 16);
        l[nq] += __shfl_xor(l[nq], 32);
    }
    if (t.splits > 1 && slot == 0 && rb == 0 && g == 0 && threadIdx.x == 0) t.used[i] = used;
    const auto row_of = [&](int nq) {  // or past the end
        const int rr = row0 + 16 * nq + col;
        const int token = tree_token(t, rr);
        return rr < rows ? first + (size_t)token * t.n_heads + g * t.r + (rr - token * t.r) : ~(size_t)0;
    };
    const auto store = [&](size_t row, int dt, f4 o, float inv) {
        const int d = 16 * dt + 4 * grp;
        if (row == ~(size_t)0 || d >= t.hd) return;
        if (used == 1) *(f4*)(t.out + row * t.hd + d) = o * inv;
        else *(f4*)(t.po + (row * t.splits + slot) * t.hd + d) = o;
    };
    const auto store_sums = [&](size_t row, float M, float L) {
        if (row == ~(size_t)0 || grp || used == 1) return;
        t.pm[row * t.splits + slot] = M;
        t.pl[row * t.splits + slot] = L;
    };
    if constexpr (PW == 1) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            const size_t row = row_of(nq);
            const float inv = l[nq] == 0.0f ? 0.0f : 1.0f / l[nq];
            store_sums(row, q.base[nq], l[nq]);
#pragma unroll
            for (int dt = 0; dt < DT; dt++) store(row, dt, q.o[nq][dt], inv);
        }
    } else {
        __syncthreads();  // the rings have been read
        f4* sums = (f4*)lds;  // [part][wave][16 rows][16 dims][lane]
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            if (grp == 0) {
                sm[pw][rw][nq][col] = q.base[nq];
                sl[pw][rw][nq][col] = l[nq];
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) sums[(((pw * RW + rw) * NQ + nq) * DT + dt) * 64 + lane] = q.o[nq][dt];
        }
        __syncthreads();
        constexpr int D = (DT + PW - 1) / PW;  // 16 dims each that a part's waves join
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            const size_t row = row_of(nq);
            float M = kNoBase, L = 0.0f, f[PW];
#pragma unroll
            for (int p = 0; p < PW; p++) M = fmaxf(M, sm[p][rw][nq][col]);
#pragma unroll
            for (int p = 0; p < PW; p++) {
                f[p] = __builtin_amdgcn_exp2f(sm[p][rw][nq][col] - M);
                L = fmaf(sl[p][rw][nq][col], f[p], L);
            }
            const float inv = L == 0.0f ? 0.0f : 1.0f / L;
            if (pw == 0) store_sums(row, M, L);
#pragma unroll
            for (int i = 0; i < D; i++) {
                const int dt = pw * D + i;
                if (dt >= DT) break;
                f4 o = {0, 0, 0, 0};
#pragma unroll
                for (int p = 0; p < PW; p++) o += f[p] * sums[(((p * RW + rw) * NQ + nq) * DT + dt) * 64 + lane];
                store(row, dt, o, inv);
            }
        }
    }
}

// out[row] = sum_s 2^(base_s - M) o_s / sum_s 2^(base_s - M) l_s, zero for a row
// that saw nothing; nothing for tokens past their request's count and for requests
// whose rows one workgroup had.  32 threads take a part, 4 dims each; the first 16
// parts are on their way before it is known how many there are.  Bound by latency:
// 4.0 us for 1056 rows of 10 parts (5.6 MB), 5.8 for 8320 rows of up to 8, 5.0 for 2048
// of 16 (17 MB, from the last-level cache).
__global__ __launch_bounds__(128) void tree_merge_kernel(TreeArgs t) {
    constexpr int E = 4;
    __shared__ __align__(16) float red[4][128];
    __shared__ float f[kSeqMaxSplits];
    __shared__ float s_inv;
    const unsigned row = blockIdx.x, token = row / (unsigned)t.n_heads, i = token / (unsigned)t.m;
    const int tid = threadIdx.x, sub = tid >> 5, d = 4 * (tid & 31);
    const int count = t.counts ? t.counts[i] : t.m, used = t.used[i];  // left as it was where there is no token
    const size_t at = (size_t)row * t.splits;
    const float* p = t.po + at * t.hd + d;
    f4 x[E];
#pragma unroll
    for (int e = 0; e < E; e++)
        if (d < t.hd && sub + 4 * e < t.splits) x[e] = *(const f4*)(p + (size_t)(sub + 4 * e) * t.hd);
    float m = 0.0f, l = 0.0f;
    if (tid < t.splits) {
        m = t.pm[at + tid];
        l = t.pl[at + tid];
    }
    if ((int)(token - i * t.m) >= count || used == 1) return;
    if (tid < 64) {
        m = tid < used ? m : kNoBase;
        l = tid < used ? l : 0.0f;
        const float M = wave_max(m), w = __builtin_amdgcn_exp2f(m - M);
        float L = l * w;
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) L += __shfl_xor(L, off);
        f[tid] = w;
        if (tid == 0) s_inv = L == 0.0f ? 0.0f : 1.0f / L;
    }
    __syncthreads();
    f4 o = {0, 0, 0, 0};
    if (d < t.hd) {
#pragma unroll
        for (int e = 0; e < E; e++)
            if (sub + 4 * e < used) o += f[sub + 4 * e] * x[e];
#pragma unroll 4
        for (int s = sub + 4 * E; s < used; s += 4) o += f[s] * *(const f4*)(p + (size_t)s * t.hd);
    }
    *(f4*)&red[sub][d] = o;
    __syncthreads();
    if (tid < t.hd) t.out[(size_t)row * t.hd + tid] = s_inv == 0.0f ? 0.0f : ((red[0][tid] + red[1][tid]) + (red[2][tid] + red[3][tid])) * s_inv;
}

template <int NQ, int RW, int PW, int ST>
static void tree_launch(const TreeArgs& a, unsigned blocks, hipStream_t s) {
    const dim3 grid(blocks), block(64 * RW * PW);
    if (a.hd <= 32) hipLaunchKernelGGL((tree_attend_kernel<32, NQ, RW, PW, ST>), grid, block, 0, s, a);
    else if (a.hd <= 64) hipLaunchKernelGGL((tree_attend_kernel<64, NQ, RW, PW, ST>), grid, block, 0, s, a);
    else if (a.hd <= 96) hipLaunchKernelGGL((tree_attend_kernel<96, NQ, RW, PW, ST>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((tree_attend_kernel<128, NQ, RW, PW, ST>), grid, block, 0, s, a);
}

}  // namespace gllm

using namespace gllm;

extern "C" {

size_t gllm_hip_attend_tree_bytes(int n, int m, int n_heads, int n_kv_heads, int hd, int most) {
    if (most < 0 || !seq_sizes(n, n_heads, n_kv_heads, hd, 0) || m < 1 || m > kTreeTokens || (long long)n * m * n_heads > kSeqMaxRows ||
        (long long)m * (n_heads / n_kv_heads) > 1 << 20)
        return 0;
    return 4 * tree_floats(tree_plan(n, m, n_heads, n_kv_heads, hd, most), n, hd);
}

int gllm_hip_attend_tree_dev(gllm_hip_kv* kv, int l, const float* d_q, int n, int m, int n_heads, int n_kv_heads, int hd,
                             const int32_t* d_starts, const int32_t* d_lens, int most, const int32_t* d_parents,
                             const int32_t* d_counts, float scale, float* d_out, void* d_work, size_t work_bytes,
                             void* stream) {
    const char* what = "gllm_hip_attend_tree_dev";
    if (m < 1 || m > kTreeTokens) return fail(GLLM_EINVAL, "%s: %d drafted tokens, 1 to %d are taken", what, m, kTreeTokens);
    if (n > kSeqMaxRows) return fail(GLLM_EINVAL, "%s: %d requests are too many", what, n);
    GLLM_TRY(seq_check(what, kv, l, d_q, n * m, n_heads, n_kv_heads, hd, d_out));
    if (most < 0) return fail(GLLM_EINVAL, "%s: contexts of up to %d rows", what, most);
    if (!d_starts || !d_lens || !d_parents) return fail(GLLM_EINVAL, "%s: null pointer", what);
    if ((long long)m * (n_heads / n_kv_heads) > 1 << 20) return fail(GLLM_EINVAL, "%s: %d tokens of %d heads to a kv head are too many", what, m, n_heads / n_kv_heads);
    hipStream_t s = (hipStream_t)stream;
    const TreePlan p = tree_plan(n, m, n_heads, n_kv_heads, hd, most);
    const size_t need = tree_floats(p, n, hd) * 4;
    if (d_work) {
        const auto meets = [&](const void* x, size_t bytes) { return x && bytes_meet(d_work, need, x, bytes); };
        if (meets(d_q, p.rows * hd * 4) || meets(d_out, p.rows * hd * 4) || meets(d_starts, (size_t)n * 4) || meets(d_lens, (size_t)n * 4) ||
            meets(d_counts, (size_t)n * 4) || meets(d_parents, (size_t)n * m * 4))
            return fail(GLLM_EINVAL, "%s: the workspace overlaps the tensors", what);
    }
    float* w;
    GLLM_TRY(seq_work(what, kv, need / 4, d_work, work_bytes, s, &w));
    const size_t parts = p.rows * p.splits;
    TreeArgs a{d_q, d_out, kv->k[l], kv->v[l], kv->kv_dim_k, kv->kv_dim_v, n, m, n_heads, n_kv_heads, p.r, hd, kv->max_len,
               p.row_blocks, p.target, p.splits, d_starts, d_lens, d_parents, d_counts, scale * 1.44269504088896340736f,
               1.0f / p.r, (1.0001f + n * 0x1p-29f) / p.target, 1.0001f / p.splits, w + parts * hd, w + parts * (hd + 1), w, (int32_t*)(w + parts * (hd + 2))};
    const unsigned blocks = (unsigned)(n_kv_heads * p.units);
    if (p.rw == 1) tree_launch<1, 1, 4, 2>(a, blocks, s);
    else if (p.rw == 2) tree_launch<1, 2, 4, 2>(a, blocks, s);
    else if (p.nq == 2) tree_launch<2, 4, 2, 2>(a, blocks, s);
    else if (p.pw == 2) tree_launch<1, 4, 2, 2>(a, blocks, s);
    else tree_launch<1, 4, 1, 2>(a, blocks, s);
    GLLM_HIP(hipGetLastError());
    if (p.splits > 1) {
        hipLaunchKernelGGL(tree_merge_kernel, dim3((unsigned)p.rows), dim3(128), 0, s, a);
        GLLM_HIP(hipGetLastError());
    }
    return GLLM_OK;
}

}  // extern "C"
