// attn_shared.hip -- decode attention over ranges of cache rows on the f16
// matrix cores: a batch of requests that share a prefix and have rows of
// their own, and the last tokens of one sequence with the weight that every
// row received.  The reference attends one sequence at a time (attendHeadGroup
// model.go:1516); these serve callers that batch or bound it.
//
//   t_p   = (q . k_p) * scale * log2(e)
//   w_p   = 2^(t_p - base)            base: 8 to 15 below the running maximum of t
//   out   = sum w_p v_p / sum w_p     over the shared rows, then the own rows
//
// K and V are f16 and q and w are float32.  Each of q and w is the sum of two
// f16 values (its rounding and the rounding of the rest, both to nearest: off by
// at most 2^-23 of its power of two), so two
// f16 matrix products, whose products are exact in the float32 accumulator,
// stand for one float32 product at an eighth of its matrix-core time.  q is
// first scaled by a power of two to a maximum in [2^14, 2^15), and base lifts
// the weights, so that the second part stays normal where it counts: below,
// f16's step of 2^-24 leaves a weight off by up to 2^-33 of the row's largest.
//
// A workgroup's four waves split the positions of a chunk, or its query rows
// where there are many.  Per 32 positions a wave forms the transposed scores
// S^T = K Q^T and the transposed output O^T += V^T W^T: the accumulator layout
// of S^T (query = lane & 15, position = 4 * (lane / 16) + register) is, for two
// tiles of 16 positions, the operand layout of W^T, so the weights never leave
// the lane.  V^T is read from an LDS tile with the transposing loads.
#include <algorithm>

#include "attn_plan.h"
#include "gllm_common.h"
#include "kv_cache.h"

namespace gllm {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef float f2 __attribute__((ext_vector_type(2)));
typedef _Float16 h2 __attribute__((ext_vector_type(2)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct SeqArgs {
    const float* q;       // [n][n_heads][hd]
    const uint16_t* K;    // row 0 of the layer
    const uint16_t* V;
    int kd_k, kd_v;       // row strides
    int n, n_heads, n_kv, r, hd, max_len;
    int start, len;       // shared rows
    int row_blocks, chunk;
    const int32_t* starts;  // own rows, or null: token i has the i rows from own_row on
    const int32_t* lens;
    int own_row;
    int own_blocks, splits;
    int shared_wgs;       // workgroups of the shared range
    int slot0, slots;     // first partial of the own ranges, partials per row
    float scale;          // scale * log2(e)
    float* pm;            // [row][slot] base
    float* pl;            //             sum
    float* po;            //             [hd] output
    float* scores;        // one token: [row][sstride], or null
    int sstride;
    u4* q_parts;          // more: the queries' operands [kv head][tile of 16 rows][lo, hi][32 dims][lane], or null
    float* q_scale;       // [kv head][tile][16]: score of a dot of theirs, in powers of two
    int tiles;            // of a kv head
};

// A new base puts the largest weight so far at 2^8; it stays until a weight
// would pass 2^15, so that most steps leave the sums as they are (f16 ends at
// 2^16).  At the other end a weight's second part is rounded to f16's steps of
// 2^-24, 2^-33 of the largest weight, to nearest: cut towards zero, which takes as
// long, the losses of many small weights add up (rows 2^18 below the heaviest
// ones came out 2.7e-5 low, now 1e-6 either way).
constexpr float kSeqLift = 8.0f, kSeqRoom = 15.0f;
constexpr float kNoBase = -3.0e38f;  // of a query without positions so far: every factor of its zero sums is finite
constexpr int kBufferWord3 = 0x00020000;  // raw buffer of 32-bit data; reads past its end give 0

// 16-byte chunk c of row r of an LDS tile lies at chunk c ^ f(r) of that row, so
// that the eight rows of a phase of 16-byte reads (K) and the four rows of 32
// bytes of a phase of transposing reads (V) meet different banks.
template <int HD>
__device__ __forceinline__ int k_swizzle(int r) {
    return HD % 64 == 0 ? r & 7 : (r >> 1) & 3;
}
template <int HD>
__device__ __forceinline__ int v_swizzle(int r) {
    return HD % 64 == 0 ? 2 * (r & 3) : 2 * ((r >> 1) & 1);
}

constexpr int kStep = 32;    // positions of a step
constexpr int kStages = 4;   // tiles of the ring that row waves share, three of them on their way

template <int HD, int RW>
struct SeqLds {
    static constexpr int TILE = kStep * HD * 2;  // bytes of K or V of a step
    static constexpr int MERGE = kSeqWaves * 16 * (HD + 4) * 4;
    static constexpr int OWN = kSeqWaves * TILE > MERGE ? kSeqWaves * TILE : MERGE;
    static constexpr int RING = RW > 1 ? kStages * 2 * TILE : 0;
    static constexpr int BYTES = RING > OWN ? RING : OWN;
};

// NQ tiles of 16 query rows, one row a lane (col = lane & 15), dims 32 kk + 8 grp.
template <int HD, int NQ>
struct SeqRows {
    h8 hi[NQ][HD / 32], lo[NQ][HD / 32];
    float c[NQ];
    // and the sums so far: out^T tiles of 16 dims, base and sum of weights of this lane's positions
    f4 o[NQ][HD / 16];
    float base[NQ], l[NQ];
};

template <int HD, int NQ, bool OWN>
__device__ __forceinline__ void seq_queries(const SeqArgs& a, int g, int tok, int row0, SeqRows<HD, NQ>& q) {
    constexpr int KK = HD / 32;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const int rows = OWN ? a.r : a.n * a.r;
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        const int rr = row0 + 16 * nq + col;
        const bool on = rr < rows;
        const int i = OWN ? tok : rr / a.r, hh = OWN ? rr : rr - i * a.r;
        const size_t row = on ? (size_t)i * a.n_heads + g * a.r + hh : 0;
        f4 x[KK][2];
        float mx = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            const int d = 32 * kk + 8 * grp;
            x[kk][0] = x[kk][1] = f4{0, 0, 0, 0};
            if (on && d < a.hd) {
                const float* p = a.q + row * a.hd + d;
                x[kk][0] = *(const f4*)p;
                x[kk][1] = *(const f4*)(p + 4);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) mx = fmaxf(mx, fmaxf(fabsf(x[kk][0][j]), fabsf(x[kk][1][j])));
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        // 2^k mx in [2^14, 2^15); rows of zeros, infinities and NaN as they are
        int e = 15;
        if (mx > 0.0f && mx < __int_as_float(0x7f800000)) (void)frexpf(mx, &e);
        const int k = 15 - e;
        q.c[nq] = ldexpf(fabsf(a.scale), -k);  // the sign goes into q, so a larger dot is a larger score
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = ldexpf(a.scale < 0.0f ? -x[kk][j >> 2][j & 3] : x[kk][j >> 2][j & 3], k);
                const _Float16 hi = (_Float16)v;
                q.hi[nq][kk][j] = hi;
                q.lo[nq][kk][j] = (_Float16)(v - (float)hi);
            }
        q.base[nq] = kNoBase;
        q.l[nq] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < HD / 16; dt++) q.o[nq][dt] = f4{0, 0, 0, 0};
    }
}

// The operands of the query rows from row0 on, for seq_mass_kernel
template <int HD, int NQ>
__device__ __forceinline__ void seq_keep_queries(const SeqArgs& a, int g, int row0, const SeqRows<HD, NQ>& q) {
    constexpr int KK = HD / 32;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        const size_t tile = (size_t)g * a.tiles + row0 / 16 + nq;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            a.q_parts[(tile * 2 * KK + kk) * 64 + lane] = __builtin_bit_cast(u4, q.lo[nq][kk]);
            a.q_parts[(tile * 2 * KK + KK + kk) * 64 + lane] = __builtin_bit_cast(u4, q.hi[nq][kk]);
        }
        if (lane < 16) a.q_scale[tile * 16 + lane] = q.c[nq];
    }
}

// s[nq][t] += K rows (16 positions of tile t) times the query rows
template <int HD, int NQ>
__device__ __forceinline__ void seq_dot(const h8 (&k)[HD / 32], const SeqRows<HD, NQ>& q, f4 (&s)[NQ][2], int t) {
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) s[nq][t] = f4{0, 0, 0, 0};
#pragma unroll
    for (int kk = 0; kk < HD / 32; kk++) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) s[nq][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[kk], q.lo[nq][kk], s[nq][t], 0, 0, 0);
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) s[nq][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[kk], q.hi[nq][kk], s[nq][t], 0, 0, 0);
    }
}

// The step at position pb of a range that ends at p1: scores s to weights, and
// the weighted rows of the V tile at vt (LDS) added to the sums.
template <int HD, int NQ>
__device__ __forceinline__ void seq_step(const SeqArgs& a, int g, int row0, int pb, int p1, bool scored, f4 (&s)[NQ][2],
                                         SeqRows<HD, NQ>& q, const char* vt, float minus1) {
    constexpr int DT = HD / 16;
    const int lane = threadIdx.x & 63, col = lane & 15, grp = lane >> 4;
    const float ninf = -__int_as_float(0x7f800000);
    // in the range's last step, scaled scores with -Inf past its end
    float cc[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) cc[nq] = q.c[nq];
    if (pb + kStep > p1) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            cc[nq] = 1.0f;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) s[nq][t][j] = pb + 16 * t + 4 * grp + j < p1 ? s[nq][t][j] * q.c[nq] : ninf;
        }
    }
    if (scored) {
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            const int rr = row0 + 16 * nq + col;
            if (rr < a.n * a.r) {
                const int i = rr / a.r;
                float* to = a.scores + ((size_t)i * a.n_heads + g * a.r + (rr - i * a.r)) * a.sstride - a.start;
#pragma unroll
                for (int t = 0; t < 2; t++)
                    if (pb + 16 * t + 4 * grp < p1) *(f4*)(to + pb + 16 * t + 4 * grp) = s[nq][t] * cc[nq];
            }
        }
    }
    // a query whose scores pass what its base allows gets a new one
    float mx[NQ];
    bool over = false;
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        mx[nq] = ninf;
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) mx[nq] = fmaxf(mx[nq], s[nq][t][j]);
        over |= mx[nq] * cc[nq] - q.base[nq] > kSeqRoom;
    }
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
    // V operand k = 8 grp + 4 t + j is position 16 t + 4 grp + j
    const int vr = 4 * grp + (col >> 2);
    const char* vp = vt + vr * HD * 2 + 8 * (col & 1);
#pragma unroll
    for (int dt = 0; dt < DT; dt++) {
        s4 x[2];
#pragma unroll
        for (int t = 0; t < 2; t++)  // rows 16 apart share their swizzle
            x[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)(
                vp + 16 * t * HD * 2 + 16 * ((2 * dt + ((col & 3) >> 1)) ^ v_swizzle<HD>(vr))));
        h8 vf;
        const h4 y0 = __builtin_bit_cast(h4, x[0]), y1 = __builtin_bit_cast(h4, x[1]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            vf[j] = y0[j];
            vf[4 + j] = y1[j];
        }
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) q.o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wl[nq], q.o[nq][dt], 0, 0, 0);
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) q.o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wh[nq], q.o[nq][dt], 0, 0, 0);
    }
}

// Rows pb .. min(pb + kStep, p1) - 1 of a kv head as a buffer: what is past its
// end reads as zero without a branch (V has to: the weight there is 0, and
// 0 * Inf is not).  A lane gives dims past hd an offset past any buffer.
struct SeqBuffer {
    const uint16_t* at;
    int bytes;
    __device__ __forceinline__ SeqBuffer(const uint16_t* base, int kd, int hd, int g, int pb, int p1) {
        const int n = min(p1 - pb, kStep);
        at = base + (size_t)pb * kd + g * hd;
        bytes = n > 0 ? ((n - 1) * kd + hd) * 2 : 0;
    }
    __device__ __forceinline__ u4 words() const {
        const uint64_t p = (uint64_t)at;
        return u4{(uint32_t)p, (uint32_t)(p >> 32) & 0xFFFFu, (uint32_t)bytes, (uint32_t)kBufferWord3};
    }
    __device__ __forceinline__ u4 load(int off) const {
        return __builtin_amdgcn_raw_buffer_load_b128(__builtin_amdgcn_make_buffer_rsrc((void*)at, 0, bytes, kBufferWord3), off, 0, 0);
    }
};
constexpr int kPastEnd = (int)0x80000000;

__device__ __forceinline__ size_t seq_part(const SeqArgs& a, bool own, int g, int tok, int rr, int slot) {
    const int i = own ? tok : rr / a.r, hh = own ? rr : rr - i * a.r;
    return ((size_t)i * a.n_heads + g * a.r + hh) * a.slots + slot + (own ? a.slot0 : 0);
}

// Up to 16 query rows: the four waves take different positions, each with K
// straight from memory into operand order and V through its own LDS tile, and
// join their sums in LDS.  Bound by memory: one request over 32768 rows of 8
// kv heads of 128 (134 MB) takes 26 us with the joining launch, 5.1 TB/s.
// HD: head size rounded up to 32 (hd <= HD, hd % 8 == 0); OWN: each token's own
// rows, not the shared ones.
template <int HD, bool OWN>
__device__ __forceinline__ void seq_few(const SeqArgs& a, int b, char* lds, float (*sm)[16], float (*sl)[16]) {
    constexpr int KK = HD / 32, DT = HD / 16, CH = HD / 8, LD = kStep * CH / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int g = b % a.n_kv;
    b /= a.n_kv;
    int rb, slot, tok = 0, a0, a1;  // rows a0 .. a1 - 1 of the cache
    if (OWN) {
        rb = b % a.own_blocks;
        b /= a.own_blocks;
        tok = b % a.n;
        slot = b / a.n;
        const RowSpan s = a.starts ? clip_rows(a.starts[tok], a.lens[tok], a.max_len) : RowSpan{a.own_row, a.own_row + tok};
        const int chunk = (((s.b - s.a) + a.splits - 1) / a.splits + kSeqQuantum - 1) / kSeqQuantum * kSeqQuantum;
        a0 = min(s.b, s.a + slot * chunk);
        a1 = min(s.b, a0 + chunk);
    } else {
        rb = b % a.row_blocks;
        slot = b / a.row_blocks;
        a0 = a.start + slot * a.chunk;
        a1 = min(a.start + a.len, a0 + a.chunk);
    }
    const int part = ((a1 - a0 + kSeqWaves * kStep - 1) / (kSeqWaves * kStep)) * kStep;  // positions of a wave
    const int p0 = min(a1, a0 + wave * part), p1 = min(a1, p0 + part);
    const int rows = OWN ? a.r : a.n * a.r, row0 = rb * 16;

    u4 kr[2][KK], vr[LD];
    const auto load_k = [&](int pb) {
        const SeqBuffer r(a.K, a.kd_k, a.hd, g, pb, p1);
#pragma unroll
        for (int t = 0; t < 2; t++)
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                const int d = 32 * kk + 8 * grp;
                kr[t][kk] = r.load(d < a.hd ? ((16 * t + col) * a.kd_k + d) * 2 : kPastEnd);
            }
    };
    const auto load_v = [&](int pb) {
        const SeqBuffer r(a.V, a.kd_v, a.hd, g, pb, p1);
#pragma unroll
        for (int u = 0; u < LD; u++) {
            const int e = 64 * u + lane, d = 8 * (e % CH);
            vr[u] = r.load(d < a.hd ? (e / CH * a.kd_v + d) * 2 : kPastEnd);
        }
    };
    if (p0 < p1) {  // on their way while the query rows are read and split
        load_v(p0);
        load_k(p0);
    }
    SeqRows<HD, 1> q;
    seq_queries<HD, 1, OWN>(a, g, tok, row0, q);
    if (!OWN && a.q_parts && slot == 0 && wave == 0) seq_keep_queries<HD, 1>(a, g, row0, q);
    float minus1 = -1.0f;  // a register, so that w - hi is one mixed-precision fma of hi as it lies
    asm volatile("" : "+v"(minus1));
    char* vt = lds + wave * SeqLds<HD, 1>::TILE;
    for (int pb = p0; pb < p1; pb += kStep) {
        const bool more = pb + kStep < p1;
#pragma unroll
        for (int u = 0; u < LD; u++) {
            const int e = 64 * u + lane, rr = e / CH;
            *(u4*)(vt + rr * HD * 2 + 16 * (e % CH ^ v_swizzle<HD>(rr))) = vr[u];
        }
        if (more) load_v(pb + kStep);
        f4 s[1][2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            h8 k[KK];
#pragma unroll
            for (int kk = 0; kk < KK; kk++) k[kk] = __builtin_bit_cast(h8, kr[t][kk]);
            seq_dot<HD, 1>(k, q, s, t);
        }
        if (more) load_k(pb + kStep);
        seq_step<HD, 1>(a, g, row0, pb, p1, !OWN && a.scores, s, q, vt, minus1);
        asm volatile("" ::: "memory");
    }

    float ls = q.l[0];
    ls += __shfl_xor(ls, 16);
    ls += __shfl_xor(ls, 32);
    float* so = (float*)lds;  // [wave][16][HD + 4]
    __syncthreads();
    if (grp == 0) {
        sm[wave][col] = q.base[0];
        sl[wave][col] = ls;
    }
#pragma unroll
    for (int dt = 0; dt < DT; dt++) *(f4*)(so + (wave * 16 + col) * (HD + 4) + 16 * dt + 4 * grp) = q.o[0][dt];
    __syncthreads();
    // 16 threads a row, dims 4 (t % 16) + 64 v
    const int row = threadIdx.x >> 4, rr = row0 + row;
    if (rr >= rows) return;
    float M = kNoBase, L = 0.0f, f[kSeqWaves];
#pragma unroll
    for (int w = 0; w < kSeqWaves; w++) M = fmaxf(M, sm[w][row]);
#pragma unroll
    for (int w = 0; w < kSeqWaves; w++) {
        f[w] = __builtin_amdgcn_exp2f(sm[w][row] - M);
        L = fmaf(sl[w][row], f[w], L);
    }
    const size_t at = seq_part(a, OWN, g, tok, rr, slot);
    if ((threadIdx.x & 15) == 0) {
        a.pm[at] = M;
        a.pl[at] = L;
    }
    for (int d = 4 * (threadIdx.x & 15); d < a.hd; d += 64) {
        f4 x = {0, 0, 0, 0};
#pragma unroll
        for (int w = 0; w < kSeqWaves; w++) x += f[w] * *(const f4*)(so + (w * 16 + row) * (HD + 4) + d);
        *(f4*)(a.po + at * a.hd + d) = x;
    }
}

// Many query rows: the four waves take 16 NQ rows each over the same positions
// and share the K and V tiles, which direct copies bring into a ring of stages
// three steps ahead (with registers, one step ahead, 64 requests over 32768 rows
// took 85 us).  Bound by the matrix cores: 256 rows of each of 8 kv heads over
// 32768 positions take 73 us, 54 of them in this loop: 69 GFLOP at 1270
// TFLOP/s, the rate of a large library product here; the rest is the launch,
// the queries, the first tiles (10 us) and the partial results (8).
template <int HD, int NQ>
__device__ __forceinline__ void seq_many(const SeqArgs& a, int b, char* lds) {
    constexpr int KK = HD / 32, DT = HD / 16, CH = HD / 8, TILE = SeqLds<HD, 4>::TILE;
    constexpr int U = 2 * kStep * CH / 256;  // copies of a wave for a stage: 64 chunks each, K first, then V
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int g = b % a.n_kv;
    b /= a.n_kv;
    const int rb = b % a.row_blocks, slot = b / a.row_blocks;
    const int p0 = a.start + slot * a.chunk, p1 = min(a.start + a.len, p0 + a.chunk);
    const int rows = a.n * a.r, row0 = (rb * kSeqWaves + wave) * 16 * NQ;

    int off[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const int w = kSeqWaves * u + wave, per = kStep * CH / 64;  // copy w of the stage
        const bool v = w >= per;
        const int e = 64 * (v ? w - per : w) + lane, r = e / CH, d = 8 * (e % CH ^ (v ? v_swizzle<HD>(r) : k_swizzle<HD>(r)));
        off[u] = d < a.hd ? (r * (v ? a.kd_v : a.kd_k) + d) * 2 : kPastEnd;
    }
    const uint32_t ring = lds_addr(lds);
    const auto copy = [&](int step) {  // past the last step the buffers are empty, and nothing is read
        const int pb = min(p0 + step * kStep, p1);
        const u4 k = SeqBuffer(a.K, a.kd_k, a.hd, g, pb, p1).words(), v = SeqBuffer(a.V, a.kd_v, a.hd, g, pb, p1).words();
        const uint32_t to = ring + (step % kStages) * 2 * TILE;
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int w = kSeqWaves * u + wave;
            lds_buffer16(w >= kStep * CH / 64 ? v : k, off[u], to + 1024 * w);
        }
    };
    copy(0);  // the queries' loads wait for it, not for the stages after
    SeqRows<HD, NQ> q;
    seq_queries<HD, NQ, false>(a, g, 0, row0, q);
#pragma unroll
    for (int i = 1; i < kStages - 1; i++) copy(i);
    if (a.q_parts && slot == 0) seq_keep_queries<HD, NQ>(a, g, row0, q);
    float minus1 = -1.0f;  // a register, so that w - hi is one mixed-precision fma of hi as it lies
    asm volatile("" : "+v"(minus1));
    const int steps = (p1 - p0 + kStep - 1) / kStep;
    for (int it = 0; it < steps; it++) {
        // this wave's copies of the stage are in (two later stages may be out),
        // and its reads of the stage before, whose place the next copies take
        wait_vmem_le<2 * U>();
        wait_lgkm0();
        lds_barrier();
        copy(it + kStages - 1);
        const char* kt = lds + (it % kStages) * 2 * TILE;
        f4 s[NQ][2];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            h8 k[KK];
#pragma unroll
            for (int kk = 0; kk < KK; kk++)
                k[kk] = *(const h8*)(kt + (16 * t + col) * HD * 2 + 16 * ((4 * kk + grp) ^ k_swizzle<HD>(col)));
            seq_dot<HD, NQ>(k, q, s, t);
        }
        const int pb = p0 + it * kStep;
        seq_step<HD, NQ>(a, g, row0, pb, p1, false, s, q, kt + TILE, minus1);
    }
    wait_vmem_le<0>();  // no copy outlives the workgroup
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        float ls = q.l[nq];
        ls += __shfl_xor(ls, 16);
        ls += __shfl_xor(ls, 32);
        const int rr = row0 + 16 * nq + col;
        if (rr < rows) {
            const size_t at = seq_part(a, false, g, 0, rr, slot);
            if (grp == 0) {
                a.pm[at] = q.base[nq];
                a.pl[at] = ls;
            }
#pragma unroll
            for (int dt = 0; dt < DT; dt++)
                if (16 * dt + 4 * grp < a.hd) *(f4*)(a.po + at * a.hd + 16 * dt + 4 * grp) = q.o[nq][dt];
        }
    }
}

// Shared and own ranges in one launch, the shared ones first.
template <int HD, int NQ, int RW>
__global__ __launch_bounds__(256, 2) void seq_attend_kernel(SeqArgs a) {
    __shared__ __align__(16) char lds[SeqLds<HD, RW>::BYTES];
    __shared__ float sm[kSeqWaves][16], sl[kSeqWaves][16];
    const int b = blockIdx.x;
    if (b >= a.shared_wgs) seq_few<HD, true>(a, b - a.shared_wgs, lds, sm, sl);
    else if constexpr (RW == 1) seq_few<HD, false>(a, b, lds, sm, sl);
    else seq_many<HD, NQ>(a, b, lds);
}

// The factor of each of a row's slots (two a lane), and the row's base and sum.
struct SlotFactors {
    float f0, f1, M, L;
};
__device__ __forceinline__ SlotFactors slot_factors(const float* pm, const float* pl, size_t at, int slots, int lane) {
    static_assert(2 * kSeqMaxSplits == 128, "two slots a lane");
    const float m0 = lane < slots ? pm[at + lane] : kNoBase, m1 = lane + 64 < slots ? pm[at + lane + 64] : kNoBase;
    const float l0 = lane < slots ? pl[at + lane] : 0.0f, l1 = lane + 64 < slots ? pl[at + lane + 64] : 0.0f;
    SlotFactors r;
    r.M = wave_max(fmaxf(m0, m1));
    r.f0 = __builtin_amdgcn_exp2f(m0 - r.M);
    r.f1 = __builtin_amdgcn_exp2f(m1 - r.M);
    r.L = fmaf(l0, r.f0, l1 * r.f1);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) r.L += __shfl_xor(r.L, off);
    return r;
}

struct MergeArgs {
    const float *pm, *pl, *po;
    float* out;
    float2* ml;           // base and 1 / sum of each row, or null
    int slots, hd;
    const float* scores;  // one token: [row][sstride], or null
    float* mass;          // [kv head][mass_stride], from the first attended row on
    int sstride, n, n_heads, n_kv, r, len, mass_stride, mass_wgs;
};

constexpr int kFewRows = 16;         // query rows of a kv head up to which scores are kept
constexpr int kMassPositions = 512;  // of a workgroup

// Workgroups below mass_wgs add the weights of 512 positions to mass, from the
// kept scores of one token's up to 16 query rows a kv head; the others make a row's output:
// out[row] = sum_s 2^(base_s - M) o_s / sum_s 2^(base_s - M) l_s, zero for a row
// without positions; 32 threads take a slot, 4 dims each, eight slots at a time.
__global__ __launch_bounds__(256) void seq_merge_kernel(MergeArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    if ((int)blockIdx.x >= a.mass_wgs) {
        __shared__ __align__(16) float red[8][128];
        __shared__ float f[2 * kSeqMaxSplits];
        const size_t row = blockIdx.x - a.mass_wgs, at = row * a.slots;
        const SlotFactors s = slot_factors(a.pm, a.pl, at, a.slots, lane);
        const float inv = s.L == 0.0f ? 0.0f : 1.0f / s.L;
        if (wave == 0) {
            f[lane] = s.f0;
            f[lane + 64] = s.f1;
            if (a.ml && lane == 0) a.ml[row] = make_float2(s.L == 0.0f ? 0.0f : s.M, inv);
        }
        __syncthreads();
        const int sub = tid >> 5, d = 4 * (tid & 31);
        f4 o = {0, 0, 0, 0};
        if (d < a.hd) {
            const float* p = a.po + at * a.hd + d;
#pragma unroll 4
            for (int t = sub; t < a.slots; t += 8) o += f[t] * *(const f4*)(p + (size_t)t * a.hd);
        }
        *(f4*)&red[sub][d] = o;
        __syncthreads();
        if (tid < a.hd) {
            float x = 0.0f;
#pragma unroll
            for (int t = 0; t < 8; t++) x += red[t][tid];
            a.out[row * a.hd + tid] = s.L == 0.0f ? 0.0f : x * inv;
        }
        return;
    }
    __shared__ float2 ml[kFewRows];
    const int g = blockIdx.x % a.n_kv, t = (blockIdx.x / a.n_kv) * kMassPositions + 2 * tid;
    const int rows = a.n * a.r;
    const auto row_of = [&](int q) { return (size_t)(q / a.r) * a.n_heads + g * a.r + q % a.r; };
    for (int q = wave; q < rows; q += 4) {
        const SlotFactors s = slot_factors(a.pm, a.pl, row_of(q) * a.slots, a.slots, lane);
        if (lane == 0) ml[q] = make_float2(s.L == 0.0f ? 0.0f : s.M, s.L == 0.0f ? 0.0f : 1.0f / s.L);
    }
    __syncthreads();
    float s0 = 0.0f, s1 = 0.0f;
    if (t < a.len) {
#pragma unroll 8
        for (int q = 0; q < rows; q++) {
            const float2 x = *(const float2*)(a.scores + row_of(q) * a.sstride + t), b = ml[q];
            s0 = fmaf(__builtin_amdgcn_exp2f(x.x - b.x), b.y, s0);
            s1 = fmaf(__builtin_amdgcn_exp2f(x.y - b.x), b.y, s1);
        }
    }
    float* to = a.mass + (size_t)g * a.mass_stride + t;
    if (t < a.len) to[0] += s0;
    if (t + 1 < a.len) to[1] += s1;
}

struct MassArgs {
    const uint16_t* K;
    const u4* q_parts;
    const float* q_scale;
    const float2* ml;
    float* mass;  // from the first attended row on
    int kd_k, hd, n, n_heads, n_kv, r, tiles, start, len, mass_stride;
};

// The weights of several tokens, from their scores made again: a wave holds 64
// positions' keys in registers and takes the rows' operands, 16 rows at a time,
// as the attention left them.  For 32 tokens over 16001 rows of 8 heads of 128
// this takes 17.5 us; writing their scores (65 MB) took the attention 16 us
// more, and reading them 35.
template <int HD>
__global__ __launch_bounds__(256, 2) void seq_mass_kernel(MassArgs a) {
    constexpr int KK = HD / 32, PT = 4;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int g = blockIdx.x % a.n_kv, p0 = (blockIdx.x / a.n_kv) * 256 + wave * 64;
    if (p0 >= a.len) return;
    h8 k[PT][KK];
#pragma unroll
    for (int t = 0; t < PT; t += 2) {
        const SeqBuffer b(a.K, a.kd_k, a.hd, g, a.start + min(p0 + 16 * t, a.len), a.start + a.len);
#pragma unroll
        for (int u = 0; u < 2; u++)
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                const int d = 32 * kk + 8 * grp;
                k[t + u][kk] = __builtin_bit_cast(h8, b.load(d < a.hd ? ((16 * u + col) * a.kd_k + d) * 2 : kPastEnd));
            }
    }
    f4 sum[PT];
#pragma unroll
    for (int t = 0; t < PT; t++) sum[t] = f4{0, 0, 0, 0};
    const u4* parts = a.q_parts + (size_t)g * a.tiles * 2 * KK * 64 + lane;
    const int rows = a.n * a.r, tiles = (rows + 15) / 16;
    // a tile's operands, and its rows' scale, base and 1 / sum, are read one tile ahead
    u4 next[2 * KK];
    float2 next_b;
    float next_c;
    int next_i;
    const auto load = [&](int tile) {
#pragma unroll
        for (int j = 0; j < 2 * KK; j++) next[j] = parts[(tile * 2 * KK + j) * 64];
        const int rr = min(16 * tile + col, rows - 1);
        next_i = rr / a.r;
        next_b = a.ml[(size_t)next_i * a.n_heads + g * a.r + (rr - next_i * a.r)];
        next_c = a.q_scale[((size_t)g * a.tiles + tile) * 16 + col];
    };
    load(0);
    for (int tile = 0; tile < tiles; tile++) {
        h8 q[2 * KK];
#pragma unroll
        for (int i = 0; i < 2 * KK; i++) q[i] = __builtin_bit_cast(h8, next[i]);
        const float2 b = next_b;
        const float c = next_c, inv = b.y;
        // positions from lim on are masked, all of them for a row that only fills the
        // tile: its dots are 0 and its base another row's, so its weight can be Inf
        const int lim = 16 * tile + col < rows ? a.len - (a.n - 1 - next_i) : 0;
        if (tile + 1 < tiles) load(tile + 1);
        f4 s[PT];
#pragma unroll
        for (int t = 0; t < PT; t++) s[t] = f4{0, 0, 0, 0};
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
#pragma unroll
            for (int t = 0; t < PT; t++) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][kk], q[kk], s[t], 0, 0, 0);
#pragma unroll
            for (int t = 0; t < PT; t++) s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[t][kk], q[KK + kk], s[t], 0, 0, 0);
        }
#pragma unroll
        for (int t = 0; t < PT; t++)
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const float w = __builtin_amdgcn_exp2f(fmaf(s[t][j], c, -b.x)) * inv;
                sum[t][j] += p0 + 16 * t + 4 * grp + j < lim ? w : 0.0f;
            }
    }
    // over the 16 rows of the tiles; lane col keeps position 16 (col / 4) + 4 grp + col % 4
    float mine = 0.0f;
#pragma unroll
    for (int t = 0; t < PT; t++)
#pragma unroll
        for (int j = 0; j < 4; j++) {
            float x = sum[t][j];
            x += dpp_f<kQuadXor1>(x);
            x += dpp_f<kQuadXor2>(x);
            x += dpp_f<kRowHalfMirror>(x);
            x += dpp_f<kRowMirror>(x);
            mine = col == 4 * t + j ? x : mine;
        }
    const int p = p0 + 16 * (col >> 2) + 4 * grp + (col & 3);
    if (p < a.len) a.mass[(size_t)g * a.mass_stride + p] += mine;
}

template <int NQ, int RW>
static void seq_launch_hd(const SeqArgs& a, int blocks, hipStream_t s) {
    if (a.hd <= 32) hipLaunchKernelGGL((seq_attend_kernel<32, NQ, RW>), dim3(blocks), dim3(256), 0, s, a);
    else if (a.hd <= 64) hipLaunchKernelGGL((seq_attend_kernel<64, NQ, RW>), dim3(blocks), dim3(256), 0, s, a);
    else if (a.hd <= 96) hipLaunchKernelGGL((seq_attend_kernel<96, NQ, RW>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((seq_attend_kernel<128, NQ, RW>), dim3(blocks), dim3(256), 0, s, a);
}

constexpr int kSeqMaxLen = 1 << 30;  // rows of a cache

// Sizes that seq_check takes, for the workspaces
static bool seq_sizes(int n, int n_heads, int n_kv, int hd, int len) {
    return n >= 1 && n_kv >= 1 && n_heads >= 1 && n_heads % n_kv == 0 && hd >= 8 && hd % 8 == 0 && hd <= 128 && len >= 0 &&
           len <= kSeqMaxLen && (long long)n * n_heads <= kSeqMaxRows;
}

static int seq_check(const char* what, const gllm_hip_kv* kv, int l, const float* d_q, int n, int n_heads, int n_kv,
                     int hd, const float* d_out) {
    if (n < 1) return fail(GLLM_EINVAL, "%s: %d tokens", what, n);
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv) return fail(GLLM_EINVAL, "%s: %d heads over %d kv heads", what, n_heads, n_kv);
    if (hd < 8 || hd % 8 || hd > 128) return fail(GLLM_EINVAL, "%s: head size %d is not a multiple of 8 up to 128", what, hd);
    if ((long long)n * n_heads > kSeqMaxRows) return fail(GLLM_EINVAL, "%s: %d tokens of %d heads are too many", what, n, n_heads);
    if (!kv || !d_q || !d_out) return fail(GLLM_EINVAL, "%s: null pointer", what);
    if (l < 0 || l >= kv->layers) return fail(GLLM_EINVAL, "%s: layer %d out of range", what, l);
    if ((long long)n_kv * hd > kv->kv_dim_k || (long long)n_kv * hd > kv->kv_dim_v)
        return fail(GLLM_EINVAL, "%s: %d kv heads of %d do not fit the cache", what, n_kv, hd);
    if (kv->max_len > kSeqMaxLen || kv->kv_dim_k > 1 << 24 || kv->kv_dim_v > 1 << 24)
        return fail(GLLM_EUNSUP, "%s: a cache of %d rows of %d and %d values", what, kv->max_len, kv->kv_dim_k, kv->kv_dim_v);
    if (kv->kv_dim_k % 8 || kv->kv_dim_v % 8)
        return fail(GLLM_EUNSUP, "%s: cache rows of %d and %d values are not 16-byte aligned", what, kv->kv_dim_k, kv->kv_dim_v);
    if (((uintptr_t)d_q | (uintptr_t)d_out) & 15) return fail(GLLM_EINVAL, "%s: q and out must be 16-byte aligned", what);
    return GLLM_OK;
}

// Device and workspace: the caller's, or the calling thread's scratch for the stream.
static int seq_work(const char* what, const gllm_hip_kv* kv, size_t floats, void* d_work, size_t work_bytes, hipStream_t s, float** out) {
    int dev = -1;
    GLLM_HIP(hipGetDevice(&dev));
    if (dev != kv->device) return fail(GLLM_EINVAL, "%s: the cache is on device %d, the current one is %d", what, kv->device, dev);
    if (d_work) {
        if (((uintptr_t)d_work & 15) || work_bytes < floats * 4)
            return fail(GLLM_EINVAL, "%s: the workspace needs %zu bytes, 16-byte aligned", what, floats * 4);
        *out = (float*)d_work;
        return GLLM_OK;
    }
    *out = (float*)thread_scratch(10, floats * 4, s);
    return *out ? GLLM_OK : scratch_error();
}

static SeqArgs seq_args(const gllm_hip_kv* kv, int l, const float* d_q, int n, int n_heads, int n_kv, int hd,
                        float scale, const SeqPlan& p, float* parts) {
    SeqArgs a{};
    a.q = d_q;
    a.K = kv->k[l];
    a.V = kv->v[l];
    a.kd_k = kv->kv_dim_k;
    a.kd_v = kv->kv_dim_v;
    a.n = n;
    a.n_heads = n_heads;
    a.n_kv = n_kv;
    a.r = p.r;
    a.hd = hd;
    a.max_len = kv->max_len;
    a.row_blocks = p.row_blocks;
    a.chunk = p.chunk;
    a.own_blocks = p.own_blocks;
    a.splits = p.splits;
    a.slots = p.slots;
    a.scale = scale * 1.44269504088896340736f;
    a.po = parts;
    a.pm = parts + p.rows * p.slots * (size_t)hd;
    a.pl = a.pm + p.rows * p.slots;
    return a;
}

static MergeArgs merge_args(const SeqArgs& a, const SeqPlan& p, float* d_out) {
    MergeArgs m{};
    m.pm = a.pm;
    m.pl = a.pl;
    m.po = a.po;
    m.out = d_out;
    m.slots = p.slots;
    m.hd = a.hd;
    m.n = a.n;
    m.n_heads = a.n_heads;
    m.n_kv = a.n_kv;
    m.r = a.r;
    m.len = a.len;
    return m;
}

static int seq_launch(SeqArgs a, const SeqPlan& p, hipStream_t s) {
    a.shared_wgs = a.n_kv * p.row_blocks * p.chunks;
    a.slot0 = p.chunks;
    const long long blocks = a.shared_wgs + (long long)a.n_kv * p.own_blocks * a.n * p.splits;
    if (blocks == 0) return GLLM_OK;
    if (p.rw == 1) seq_launch_hd<1, 1>(a, (int)blocks, s);
    else if (p.nq == 1) seq_launch_hd<1, 4>(a, (int)blocks, s);
    else seq_launch_hd<2, 4>(a, (int)blocks, s);
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

}  // namespace gllm

using namespace gllm;

extern "C" {

size_t gllm_hip_attend_shared_bytes(int n, int n_heads, int n_kv_heads, int hd, int len, int most) {
    if (!seq_sizes(n, n_heads, n_kv_heads, hd, len) || most < 0) return 0;
    return 4 * seq_floats(seq_plan(n, n_heads, n_kv_heads, hd, len, most), hd);
}

int gllm_hip_attend_shared_dev(gllm_hip_kv* kv, int l, const float* d_q, int n, int n_heads, int n_kv_heads, int hd,
                               int start, int len, const int32_t* d_starts, const int32_t* d_lens, int most, float scale,
                               float* d_out, void* d_work, size_t work_bytes, void* stream) {
    const char* what = "gllm_hip_attend_shared_dev";
    GLLM_TRY(seq_check(what, kv, l, d_q, n, n_heads, n_kv_heads, hd, d_out));
    if (start < 0 || len < 0 || (long long)start + len > kv->max_len)
        return fail(GLLM_EINVAL, "%s: shared rows %d + %d outside 0..%d", what, start, len, kv->max_len - 1);
    if (most < 0 || (most > 0) != (d_starts != nullptr) || (most > 0) != (d_lens != nullptr))
        return fail(GLLM_EINVAL, "%s: own rows need starts, lens and most > 0 together", what);
    hipStream_t s = (hipStream_t)stream;
    const SeqPlan p = seq_plan(n, n_heads, n_kv_heads, hd, len, most);
    float* w;
    GLLM_TRY(seq_work(what, kv, seq_floats(p, hd), d_work, work_bytes, s, &w));
    SeqArgs a = seq_args(kv, l, d_q, n, n_heads, n_kv_heads, hd, scale, p, w);
    a.start = start;
    a.len = len;
    a.starts = d_starts;
    a.lens = d_lens;
    GLLM_TRY(seq_launch(a, p, s));
    hipLaunchKernelGGL(seq_merge_kernel, dim3((unsigned)p.rows), dim3(256), 0, s, merge_args(a, p, d_out));
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

size_t gllm_hip_attend_mass_bytes(int n, int n_heads, int n_kv_heads, int hd, int len) {
    if (!seq_sizes(n, n_heads, n_kv_heads, hd, len) || n > len) return 0;
    return 4 * mass_floats(seq_plan(n, n_heads, n_kv_heads, hd, len - (n - 1), n - 1), hd, n_kv_heads, len);
}

int gllm_hip_attend_mass_dev(gllm_hip_kv* kv, int l, const float* d_q, int n, int n_heads, int n_kv_heads, int hd,
                             int start, int end, float scale, float* d_mass, int mass_stride, float* d_out,
                             void* d_work, size_t work_bytes, void* stream) {
    const char* what = "gllm_hip_attend_mass_dev";
    GLLM_TRY(seq_check(what, kv, l, d_q, n, n_heads, n_kv_heads, hd, d_out));
    if (start < 0 || end >= kv->max_len || (long long)end - start + 1 < n)
        return fail(GLLM_EINVAL, "%s: %d tokens over positions %d..%d of 0..%d", what, n, start, end, kv->max_len - 1);
    if (!d_mass || mass_stride <= end) return fail(GLLM_EINVAL, "%s: mass rows of %d values do not hold position %d", what, mass_stride, end);
    hipStream_t s = (hipStream_t)stream;
    const int len = end - start + 1;
    // what every token attends is the shared range; token i has i rows more
    const SeqPlan p = seq_plan(n, n_heads, n_kv_heads, hd, len - (n - 1), n - 1);
    float* w;
    GLLM_TRY(seq_work(what, kv, mass_floats(p, hd, n_kv_heads, len), d_work, work_bytes, s, &w));
    const MassSpace m = mass_space(p, hd, n_kv_heads, len);
    SeqArgs a = seq_args(kv, l, d_q, n, n_heads, n_kv_heads, hd, scale, p, w + m.parts);
    a.start = start;
    a.len = len - (n - 1);
    a.own_row = start + a.len;
    if (m.kept) {
        a.scores = w;
        a.sstride = m.sstride;
    } else {
        a.q_parts = (u4*)w;
        a.q_scale = w + m.scale;
        a.tiles = m.tiles;
    }
    GLLM_TRY(seq_launch(a, p, s));
    MergeArgs g = merge_args(a, p, d_out);
    g.len = len;
    g.mass = d_mass + start;
    g.mass_stride = mass_stride;
    if (m.kept) {
        g.scores = w;
        g.sstride = m.sstride;
        g.mass_wgs = n_kv_heads * ((len + kMassPositions - 1) / kMassPositions);
    } else {
        g.ml = (float2*)(w + m.ml);
    }
    hipLaunchKernelGGL(seq_merge_kernel, dim3((unsigned)(g.mass_wgs + p.rows)), dim3(256), 0, s, g);
    GLLM_HIP(hipGetLastError());
    if (!m.kept) {
        const MassArgs b{a.K, a.q_parts, a.q_scale, g.ml, g.mass, a.kd_k, hd, n, n_heads, n_kv_heads, p.r, m.tiles, start, len, mass_stride};
        const dim3 grid((unsigned)(n_kv_heads * ((len + 255) / 256)));
        if (hd <= 32) hipLaunchKernelGGL(seq_mass_kernel<32>, grid, dim3(256), 0, s, b);
        else if (hd <= 64) hipLaunchKernelGGL(seq_mass_kernel<64>, grid, dim3(256), 0, s, b);
        else if (hd <= 96) hipLaunchKernelGGL(seq_mass_kernel<96>, grid, dim3(256), 0, s, b);
        else hipLaunchKernelGGL(seq_mass_kernel<128>, grid, dim3(256), 0, s, b);
        GLLM_HIP(hipGetLastError());
    }
    return GLLM_OK;
}

}  // extern "C"
