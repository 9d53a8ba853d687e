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
// f16 values (its rounding and the rounding of the rest, 22 bits), so two
// f16 matrix products, whose products are exact in the float32 accumulator,
// stand for one float32 product at an eighth of its matrix-core time.  q is
// first scaled by a power of two to a maximum in [2^14, 2^15), and base lifts
// the weights, so that the second part stays normal where it counts.
//
// A workgroup's four waves split the positions of a chunk, or its query rows
// where there are many.  Per 32 positions a wave forms the transposed scores S^T = K Q^T and the transposed output
// O^T += V^T W^T: the accumulator layout of S^T (query = lane & 15, position
// = 4 * (lane / 16) + register) is, for two tiles of 16 positions, the
// operand layout of W^T, so the weights never leave the lane.  V^T is read
// from an LDS tile with the transposing loads.
#include <algorithm>

#include "attn_plan.h"
#include "gllm_common.h"
#include "kv_cache.h"

namespace gllm {

typedef _Float16 h8 __attribute__((ext_vector_type(8)));
typedef _Float16 h4 __attribute__((ext_vector_type(4)));
typedef short s4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef uint32_t u4 __attribute__((ext_vector_type(4)));

struct SeqArgs {
    const float* q;       // [n][n_heads][hd]
    const uint16_t* K;    // row 0 of the layer
    const uint16_t* V;
    int kd_k, kd_v;       // row strides
    int n, n_heads, n_kv, r, hd, max_len;
    int start, len;       // shared rows
    int causal;           // token i ends n - 1 - i rows earlier
    int row_blocks, chunk;
    const int32_t* starts;  // own rows
    const int32_t* lens;
    int own_blocks, splits;
    int shared_wgs;       // workgroups of the shared range
    int slot0, slots;     // first partial of the own ranges, partials per row
    float scale;          // scale * log2(e)
    float* pm;            // [row][slot] base
    float* pl;            //             sum
    float* po;            //             [hd] output
    float* scores;        // [row][sstride] or null
    int sstride;
};

// A new base puts the largest weight so far at 2^8; it stays until a weight
// would pass 2^15, so that most steps leave the sums as they are (f16 ends at
// 2^16; at the other end a weight's second part ends 2^-32 below the largest).
constexpr float kSeqLift = 8.0f, kSeqRoom = 15.0f;
constexpr float kNoBase = -3.0e38f;  // of a query without positions so far: every factor of its zero sums is finite
constexpr int kBufferWord3 = 0x00020000;  // raw buffer of 32-bit data; reads past its end give 0

// Bytes between rows of an LDS tile.  K rows are read 16 bytes a lane, eight
// rows at a time: 16 bytes of padding spread them over the banks.  V rows are
// read 32 bytes a row, four rows at a time, by the transposing loads: rows of
// 256 and 128 bytes need 32 bytes of padding, 192 and 64 spread by themselves.
template <int HD>
struct Lds {
    static constexpr int k_row = HD * 2 + 16;
    static constexpr int v_row = HD * 2 + (HD % 64 == 0 ? 32 : 0);
};

template <int HD, int NQ, int RW>
struct SeqShape {
    static constexpr int PW = kSeqWaves / RW;                // position groups
    static constexpr int STEP = RW == 4 && HD % 64 ? 64 : 32;           // positions of a step
    static constexpr int TILE = STEP * ((RW > 1 ? Lds<HD>::k_row : 0) + Lds<HD>::v_row);
    static constexpr int BUFS = RW > 1 ? 2 : 1;
    static constexpr int MERGE = PW > 1 ? kSeqWaves * 16 * (HD + 4) * 4 : 0;
    static constexpr int BYTES = PW * BUFS * TILE > MERGE ? PW * BUFS * TILE : MERGE;
};

__device__ __forceinline__ h8 join(s4 a, s4 b) {
    h8 r;
    const h4 x = __builtin_bit_cast(h4, a), y = __builtin_bit_cast(h4, b);
#pragma unroll
    for (int j = 0; j < 4; j++) {
        r[j] = x[j];
        r[4 + j] = y[j];
    }
    return r;
}

// HD: head size rounded up to 32 (hd <= HD, hd % 8 == 0); NQ: tiles of 16
// query rows of a wave; RW: waves that take different query rows over the same
// positions, sharing the K and V tiles; the kSeqWaves / RW groups of such waves
// take different positions.  OWN: each token's own rows, not the shared ones.
template <int HD, int NQ, int RW, bool OWN>
__device__ __forceinline__ void seq_run(const SeqArgs& a, int b, char* lds, float (*sm)[16], float (*sl)[16]) {
    using S = SeqShape<HD, NQ, RW>;
    constexpr int KK = HD / 32, DT = HD / 16, CH = HD / 8, PW = S::PW, STEP = S::STEP, ST = STEP / 16;
    constexpr int GT = RW * 64;                    // threads of a position group
    constexpr int LD = STEP * CH / GT;             // 16-byte loads of a thread for a tile
    static_assert(STEP * CH % GT == 0, "a tile is a whole number of loads");
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, grp = lane >> 4;
    const int pg = wave / RW, rw = wave % RW;
    const float ninf = -__int_as_float(0x7f800000);

    const int g = b % a.n_kv;
    b /= a.n_kv;
    int rb, slot, tok = 0, a0, a1;  // rows a0 .. a1 - 1 of the cache
    if (OWN) {
        rb = b % a.own_blocks;
        b /= a.own_blocks;
        tok = b % a.n;
        slot = b / a.n;
        const RowSpan s = clip_rows(a.starts[tok], a.lens[tok], a.max_len);
        const int chunk = (((s.b - s.a) + a.splits - 1) / a.splits + kSeqQuantum - 1) / kSeqQuantum * kSeqQuantum;
        a0 = min(s.b, s.a + slot * chunk);
        a1 = min(s.b, a0 + chunk);
    } else {
        rb = b % a.row_blocks;
        slot = b / a.row_blocks;
        a0 = a.start + slot * a.chunk;
        a1 = min(a.start + a.len, a0 + a.chunk);
    }
    const int part = ((a1 - a0 + PW * STEP - 1) / (PW * STEP)) * STEP;  // positions of a group
    const int p0 = min(a1, a0 + pg * part), p1 = min(a1, p0 + part);

    // A tile's K and V as loads.  V, and K where waves share it, go to LDS: 16-byte
    // chunk e = GT u + thread of the group; K of a wave's own goes straight into
    // operand order, u = t * KK + kk: position 16 t + col, dims 32 kk + 8 grp.
    // The buffer ends with the range's last row, so what is past it reads as
    // zero without a branch (V has to: the weight there is 0, and 0 * Inf is not);
    // dims past hd get an offset past any buffer.
    const int gt = rw * 64 + lane;
    u4 kr[LD], vr[LD];
    const auto rsrc = [&](const uint16_t* base, int kd, int pb) {
        const int n = min(p1 - pb, STEP);
        return __builtin_amdgcn_make_buffer_rsrc((void*)(base + (size_t)pb * kd + g * a.hd), 0,
                                                 n > 0 ? ((n - 1) * kd + a.hd) * 2 : 0, kBufferWord3);
    };
    const auto chunk_off = [&](int u, int kd) {
        const int e = GT * u + gt, d = 8 * (e % CH);
        return d < a.hd ? (e / CH * kd + d) * 2 : (int)0x80000000;
    };
    const auto load_k = [&](int pb) {
        const auto r = rsrc(a.K, a.kd_k, pb);
#pragma unroll
        for (int u = 0; u < LD; u++) {
            const int t = u / KK, d = 32 * (u % KK) + 8 * grp;
            const int off = RW > 1 ? chunk_off(u, a.kd_k) : d < a.hd ? ((16 * t + col) * a.kd_k + d) * 2 : (int)0x80000000;
            kr[u] = __builtin_amdgcn_raw_buffer_load_b128(r, off, 0, 0);
        }
    };
    const auto load_v = [&](int pb) {
        const auto r = rsrc(a.V, a.kd_v, pb);
#pragma unroll
        for (int u = 0; u < LD; u++) vr[u] = __builtin_amdgcn_raw_buffer_load_b128(r, chunk_off(u, a.kd_v), 0, 0);
    };
    const int steps = part / STEP;  // the same for every wave of the workgroup
    if (steps > 0) {  // on their way while the query rows are read and split
        load_v(p0);
        load_k(p0);
    }

    // query rows: rb * 16 * NQ * RW + 16 * (rw * NQ + nq) + col of this kv head
    const int rows = OWN ? a.r : a.n * a.r;
    const int row0 = (rb * RW + rw) * 16 * NQ;
    h8 qh[NQ][KK], ql[NQ][KK];
    float c[NQ];
    int lim[NQ];  // rows from it on are masked
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        const int rr = row0 + 16 * nq + col;
        const bool on = rr < rows;
        const int i = OWN ? tok : rr / a.r, hh = OWN ? rr : rr - i * a.r;
        const size_t row = on ? (size_t)i * a.n_heads + g * a.r + hh : 0;
        lim[nq] = a.causal ? min(p1, a.start + a.len - (a.n - 1 - (on ? i : 0))) : p1;
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
        c[nq] = ldexpf(fabsf(a.scale), -k);  // the sign goes into q, so a larger dot is a larger score
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = ldexpf(a.scale < 0.0f ? -x[kk][j >> 2][j & 3] : x[kk][j >> 2][j & 3], k);
                const _Float16 hi = (_Float16)v;
                qh[nq][kk][j] = hi;
                ql[nq][kk][j] = (_Float16)(v - (float)hi);
            }
    }
    int lim_all = a1;  // rows that no row of this wave masks
    if (!OWN && a.causal) lim_all = a.start + a.len - (a.n - 1 - min(row0 / a.r, a.n - 1));

    f4 o[NQ][DT];
    float base[NQ], l[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        base[nq] = kNoBase;
        l[nq] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[nq][dt] = f4{0, 0, 0, 0};
    }

    char* tile = lds + pg * S::BUFS * S::TILE;
    const auto store_tile = [&](char* to) {
#pragma unroll
        for (int u = 0; u < LD; u++) {
            const int e = GT * u + gt, rr = e / CH, ch = e % CH;
            if (RW > 1) *(u4*)(to + rr * Lds<HD>::k_row + 16 * ch) = kr[u];
            *(u4*)(to + (RW > 1 ? STEP * Lds<HD>::k_row : 0) + rr * Lds<HD>::v_row + 16 * ch) = vr[u];
        }
    };

    float minus1 = -1.0f;  // a register, so that w - hi is one mixed-precision fma of hi as it lies
    asm volatile("" : "+v"(minus1));
    if (RW > 1 && steps > 0) {
        store_tile(tile);
        __syncthreads();
    }
    for (int it = 0; it < steps; it++) {
        const int pb = p0 + it * STEP;
        const bool more = it + 1 < steps;
        char* cur = tile + (RW > 1 ? (it & 1) * S::TILE : 0);
        h8 kf[ST][KK];
        if (RW == 1) {
            if (pb >= p1) break;  // no barrier in this loop
            store_tile(cur);
            if (more) load_v(pb + STEP);
#pragma unroll
            for (int t = 0; t < ST; t++)
#pragma unroll
                for (int kk = 0; kk < KK; kk++) kf[t][kk] = __builtin_bit_cast(h8, kr[(t * KK + kk) % LD]);
        } else {
            if (more) {
                load_k(pb + STEP);
                load_v(pb + STEP);
            }
        }
        f4 s[NQ][ST];
#pragma unroll
        for (int t = 0; t < ST; t++) {
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) s[nq][t] = f4{0, 0, 0, 0};
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                const h8 k = RW == 1 ? kf[t][kk]
                                     : *(const h8*)(cur + (16 * t + col) * Lds<HD>::k_row + 64 * kk + 16 * grp);
#pragma unroll
                for (int nq = 0; nq < NQ; nq++) s[nq][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, ql[nq][kk], s[nq][t], 0, 0, 0);
#pragma unroll
                for (int nq = 0; nq < NQ; nq++) s[nq][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, qh[nq][kk], s[nq][t], 0, 0, 0);
            }
        }
        if (RW == 1 && more) load_k(pb + STEP);
        // where the tile holds masked positions, scaled scores with -Inf in their places
        float cc[NQ];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) cc[nq] = c[nq];
        if (pb + STEP > min(p1, lim_all)) {
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
                cc[nq] = 1.0f;
#pragma unroll
                for (int t = 0; t < ST; t++)
#pragma unroll
                    for (int j = 0; j < 4; j++) s[nq][t][j] = pb + 16 * t + 4 * grp + j < lim[nq] ? s[nq][t][j] * c[nq] : ninf;
            }
        }
        if (!OWN && a.scores) {
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
                const int rr = row0 + 16 * nq + col;
                if (rr < rows) {
                    const int i = rr / a.r;
                    float* to = a.scores + ((size_t)i * a.n_heads + g * a.r + (rr - i * a.r)) * a.sstride - a.start;
#pragma unroll
                    for (int t = 0; t < ST; t++)
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
            for (int t = 0; t < ST; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) mx[nq] = fmaxf(mx[nq], s[nq][t][j]);
            over |= mx[nq] * cc[nq] - base[nq] > kSeqRoom;
        }
        if (__any(over)) {
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
                float top = fmaxf(mx[nq], __shfl_xor(mx[nq], 16));
                top = fmaxf(top, __shfl_xor(top, 32)) * cc[nq];
                const float nb = top - base[nq] > kSeqRoom ? top - kSeqLift : base[nq];
                const float f = __builtin_amdgcn_exp2f(base[nq] - nb);
                l[nq] *= f;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[nq][dt] *= f;
                base[nq] = nb;
            }
        }
        // V operand k = 8 grp + 4 t + j of step u is position 32 u + 16 t + 4 grp + j
        const char* vt = cur + (RW > 1 ? STEP * Lds<HD>::k_row : 0) + (4 * grp + (col >> 2)) * Lds<HD>::v_row + 8 * (col & 3);
#pragma unroll
        for (int u = 0; u < ST / 2; u++) {
            h8 wh[NQ], wl[NQ];
#pragma unroll
            for (int nq = 0; nq < NQ; nq++)
#pragma unroll
                for (int t = 0; t < 2; t++)
#pragma unroll
                    for (int j = 0; j < 4; j += 2) {
                        // the two parts of a weight, both cut short: 21 bits
                        const f4 x = s[nq][2 * u + t];
                        const float w0 = __builtin_amdgcn_exp2f(fmaf(x[j], cc[nq], -base[nq]));
                        const float w1 = __builtin_amdgcn_exp2f(fmaf(x[j + 1], cc[nq], -base[nq]));
                        l[nq] += w0 + w1;
                        const auto hi = __builtin_amdgcn_cvt_pkrtz(w0, w1);
                        const auto lo = __builtin_amdgcn_cvt_pkrtz(fmaf((float)hi[0], minus1, w0), fmaf((float)hi[1], minus1, w1));
                        wh[nq][4 * t + j] = (_Float16)hi[0];
                        wh[nq][4 * t + j + 1] = (_Float16)hi[1];
                        wl[nq][4 * t + j] = (_Float16)lo[0];
                        wl[nq][4 * t + j + 1] = (_Float16)lo[1];
                    }
#pragma unroll
            for (int dt = 0; dt < DT; dt++) {
                s4 x[2];
#pragma unroll
                for (int t = 0; t < 2; t++)
                    x[t] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                        (__attribute__((address_space(3))) s4*)(vt + (32 * u + 16 * t) * Lds<HD>::v_row + 32 * dt));
                const h8 vf = join(x[0], x[1]);
#pragma unroll
                for (int nq = 0; nq < NQ; nq++) o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wl[nq], o[nq][dt], 0, 0, 0);
#pragma unroll
                for (int nq = 0; nq < NQ; nq++) o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wh[nq], o[nq][dt], 0, 0, 0);
            }
        }
        asm volatile("" ::: "memory");
        if (RW > 1) {
            if (more) store_tile(tile + ((it + 1) & 1) * S::TILE);
            __syncthreads();
        }
    }

    // results: straight to the partials, or the position groups' joined in LDS,
    // one tile of query rows of every row wave at a time
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        float ls = l[nq];
        ls += __shfl_xor(ls, 16);
        ls += __shfl_xor(ls, 32);
        if (PW == 1) {
            const int rr = row0 + 16 * nq + col;
            if (rr < rows) {
                const int i = OWN ? tok : rr / a.r, hh = OWN ? rr : rr - i * a.r;
                const size_t at = ((size_t)i * a.n_heads + g * a.r + hh) * a.slots + slot + (OWN ? a.slot0 : 0);
                if (grp == 0) {
                    a.pm[at] = base[nq];
                    a.pl[at] = ls;
                }
#pragma unroll
                for (int dt = 0; dt < DT; dt++)
                    if (16 * dt + 4 * grp < a.hd) *(f4*)(a.po + at * a.hd + 16 * dt + 4 * grp) = o[nq][dt];
            }
            continue;
        }
        float* so = (float*)lds;  // [wave][16][HD + 4]
        __syncthreads();
        if (grp == 0) {
            sm[wave][col] = base[nq];
            sl[wave][col] = ls;
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) *(f4*)(so + (wave * 16 + col) * (HD + 4) + 16 * dt + 4 * grp) = o[nq][dt];
        __syncthreads();
        // 16 threads a row: RW * 16 rows, dims 4 (t % 16) + 64 v
#pragma unroll
        for (int q = 0; q < RW; q++) {
            const int row = threadIdx.x >> 4, rr = (rb * RW + q) * 16 * NQ + 16 * nq + row;
            float M = kNoBase, L = 0.0f, f[PW];
#pragma unroll
            for (int w = 0; w < PW; w++) M = fmaxf(M, sm[w * RW + q][row]);
#pragma unroll
            for (int w = 0; w < PW; w++) {
                f[w] = __builtin_amdgcn_exp2f(sm[w * RW + q][row] - M);
                L = fmaf(sl[w * RW + q][row], f[w], L);
            }
            if (rr < rows) {
                const int i = OWN ? tok : rr / a.r, hh = OWN ? rr : rr - i * a.r;
                const size_t at = ((size_t)i * a.n_heads + g * a.r + hh) * a.slots + slot + (OWN ? a.slot0 : 0);
                if ((threadIdx.x & 15) == 0) {
                    a.pm[at] = M;
                    a.pl[at] = L;
                }
                for (int d = 4 * (threadIdx.x & 15); d < a.hd; d += 64) {
                    f4 x = {0, 0, 0, 0};
#pragma unroll
                    for (int w = 0; w < PW; w++) x += f[w] * *(const f4*)(so + ((w * RW + q) * 16 + row) * (HD + 4) + d);
                    *(f4*)(a.po + at * a.hd + d) = x;
                }
            }
        }
    }
}

// Shared and own ranges in one launch: own_wgs workgroups of own ranges among
// the shared ones.
template <int HD, int NQ, int RW>
__global__ __launch_bounds__(256, 2) void seq_attend_kernel(SeqArgs a) {
    constexpr int A = SeqShape<HD, NQ, RW>::BYTES, B = SeqShape<HD, 1, 1>::BYTES;
    __shared__ __align__(16) char lds[A > B ? A : B];
    __shared__ float sm[kSeqWaves][16], sl[kSeqWaves][16];
    const int b = blockIdx.x;
    if (b < a.shared_wgs) seq_run<HD, NQ, RW, false>(a, b, lds, sm, sl);
    else seq_run<HD, 1, 1, true>(a, b - a.shared_wgs, lds, sm, sl);
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
    int rows, slots, hd;
    const float* scores;  // [row][sstride], or null: no mass
    float* mass;          // [kv head][mass_stride], from the first attended row on
    int sstride, n, n_heads, n_kv, r, len, mass_stride, mass_wgs;
};

constexpr int kMassRows = 64;  // query rows whose base and 1 / sum a workgroup holds at a time

// Workgroups below mass_wgs add the weights of 512 positions to mass, the
// others make a row's output:
// out[row] = sum_s 2^(base_s - M) o_s / sum_s 2^(base_s - M) l_s, zero for a row
// without positions; 32 threads take a slot, 4 dims each, eight slots at a time.
__global__ __launch_bounds__(256) void seq_merge_kernel(MergeArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    __shared__ __align__(16) float red[8][128];
    if ((int)blockIdx.x >= a.mass_wgs) {
        const size_t row = blockIdx.x - a.mass_wgs, at = row * a.slots;
        const SlotFactors s = slot_factors(a.pm, a.pl, at, a.slots, lane);
        const float inv = s.L == 0.0f ? 0.0f : 1.0f / s.L;
        __shared__ float f[2 * kSeqMaxSplits];
        if (wave == 0) {
            f[lane] = s.f0;
            f[lane + 64] = s.f1;
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
    __shared__ float2 ml[kMassRows];  // base, 1 / sum
    const int g = blockIdx.x % a.n_kv, t = (blockIdx.x / a.n_kv) * 512 + 2 * tid;
    const int rows = a.n * a.r;
    float s0 = 0.0f, s1 = 0.0f;
    for (int r0 = 0; r0 < rows; r0 += kMassRows) {
        const int m = min(kMassRows, rows - r0);
        __syncthreads();
        for (int q = wave; q < m; q += 4) {
            const int i = (r0 + q) / a.r;
            const size_t row = (size_t)i * a.n_heads + g * a.r + (r0 + q - i * a.r);
            const SlotFactors s = slot_factors(a.pm, a.pl, row * a.slots, a.slots, lane);
            if (lane == 0) ml[q] = make_float2(s.L == 0.0f ? 0.0f : s.M, s.L == 0.0f ? 0.0f : 1.0f / s.L);
        }
        __syncthreads();
        if (t < a.len) {
#pragma unroll 8
            for (int q = 0; q < m; q++) {
                const int i = (r0 + q) / a.r;
                const size_t row = (size_t)i * a.n_heads + g * a.r + (r0 + q - i * a.r);
                const float2 x = *(const float2*)(a.scores + row * a.sstride + t), b = ml[q];
                s0 = fmaf(__builtin_amdgcn_exp2f(x.x - b.x), b.y, s0);
                s1 = fmaf(__builtin_amdgcn_exp2f(x.y - b.x), b.y, s1);
            }
        }
    }
    float* to = a.mass + (size_t)g * a.mass_stride + t;
    if (t < a.len) to[0] += s0;
    if (t + 1 < a.len) to[1] += s1;
}

template <int NQ, int RW>
static void seq_launch_hd(const SeqArgs& a, int blocks, hipStream_t s) {
    if (a.hd <= 32) hipLaunchKernelGGL((seq_attend_kernel<32, NQ, RW>), dim3(blocks), dim3(256), 0, s, a);
    else if (a.hd <= 64) hipLaunchKernelGGL((seq_attend_kernel<64, NQ, RW>), dim3(blocks), dim3(256), 0, s, a);
    else if (a.hd <= 96) hipLaunchKernelGGL((seq_attend_kernel<96, NQ, RW>), dim3(blocks), dim3(256), 0, s, a);
    else hipLaunchKernelGGL((seq_attend_kernel<128, NQ, RW>), dim3(blocks), dim3(256), 0, s, a);
}

static int seq_check(const char* what, const gllm_hip_kv* kv, int l, const float* d_q, int n, int n_heads, int n_kv,
                     int hd, const float* d_out) {
    if (n < 1) return fail(GLLM_EINVAL, "%s: %d tokens", what, n);
    if (n_kv < 1 || n_heads < 1 || n_heads % n_kv) return fail(GLLM_EINVAL, "%s: %d heads over %d kv heads", what, n_heads, n_kv);
    if (hd < 8 || hd % 8 || hd > 128) return fail(GLLM_EINVAL, "%s: head size %d is not a multiple of 8 up to 128", what, hd);
    if ((long long)n * n_heads > (1 << 24)) return fail(GLLM_EINVAL, "%s: %d tokens of %d heads are too many", what, n, n_heads);
    if (!kv || !d_q || !d_out) return fail(GLLM_EINVAL, "%s: null pointer", what);
    if (l < 0 || l >= kv->layers) return fail(GLLM_EINVAL, "%s: layer %d out of range", what, l);
    if ((long long)n_kv * hd > kv->kv_dim_k || (long long)n_kv * hd > kv->kv_dim_v)
        return fail(GLLM_EINVAL, "%s: %d kv heads of %d do not fit the cache", what, n_kv, hd);
    if (kv->max_len > 1 << 30) return fail(GLLM_EUNSUP, "%s: a cache of %d rows", what, kv->max_len);
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
    m.rows = (int)p.rows;
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
    else if (p.nq == 1) seq_launch_hd<1, 2>(a, (int)blocks, s);
    else if (p.rw == 2) seq_launch_hd<2, 2>(a, (int)blocks, s);
    else seq_launch_hd<2, 4>(a, (int)blocks, s);
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

}  // namespace gllm

using namespace gllm;

extern "C" {

size_t gllm_hip_attend_shared_bytes(int n, int n_heads, int n_kv_heads, int hd, int len, int most) {
    if (n < 1 || n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads || hd < 1 || len < 0 || most < 0 ||
        (long long)n * n_heads > (1 << 24))
        return 0;
    return 4 * seq_floats(seq_plan(n, n_heads, n_kv_heads, len, most), hd, 0);
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
    const SeqPlan p = seq_plan(n, n_heads, n_kv_heads, len, most);
    float* w;
    GLLM_TRY(seq_work(what, kv, seq_floats(p, hd, 0), d_work, work_bytes, s, &w));
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
    if (n < 1 || n_kv_heads < 1 || n_heads < 1 || n_heads % n_kv_heads || hd < 1 || len < 1 ||
        (long long)n * n_heads > (1 << 24))
        return 0;
    return 4 * seq_floats(seq_plan(n, n_heads, n_kv_heads, len, 0), hd, ((size_t)len + 3) / 4 * 4);
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
    const int sstride = (int)(((size_t)len + 3) / 4 * 4);
    const SeqPlan p = seq_plan(n, n_heads, n_kv_heads, len, 0);
    float* w;
    GLLM_TRY(seq_work(what, kv, seq_floats(p, hd, sstride), d_work, work_bytes, s, &w));
    SeqArgs a = seq_args(kv, l, d_q, n, n_heads, n_kv_heads, hd, scale, p, w + p.rows * (size_t)sstride);
    a.start = start;
    a.len = len;
    a.causal = 1;
    a.scores = w;
    a.sstride = sstride;
    GLLM_TRY(seq_launch(a, p, s));
    MergeArgs m = merge_args(a, p, d_out);
    m.scores = w;
    m.sstride = sstride;
    m.mass = d_mass + start;
    m.mass_stride = mass_stride;
    m.mass_wgs = n_kv_heads * ((len + 511) / 512);
    hipLaunchKernelGGL(seq_merge_kernel, dim3((unsigned)(m.mass_wgs + p.rows)), dim3(256), 0, s, m);
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

}  // extern "C"
