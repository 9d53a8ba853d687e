// attn_shared.hip -- decode attention over ranges of cache rows on the f16
// matrix cores: a batch of requests that share a prefix and have rows of
// their own, and the last tokens of one sequence with the weight that every
// row received.  The reference attends one sequence at a time (attendHeadGroup
// model.go:1516); these serve callers that batch or bound it.
//
//   t_p   = (q . k_p) * scale * log2(e)
//   w_p   = 2^(t_p - base)            base = (running maximum of t) - 15
//   out   = sum w_p v_p / sum w_p     over the shared rows, then the own rows
//
// K and V are f16 and q and w are float32.  Each of q and w is the sum of two
// f16 values (its rounding and the rounding of the rest, 22 bits), so two
// f16 matrix products, whose products are exact in the float32 accumulator,
// stand for one float32 product at an eighth of its matrix-core time.  q is
// first scaled by a power of two to a maximum in [2^14, 2^15), and the
// weights by 2^15 (the 15 in base), so that the second part stays normal.
//
// A workgroup's four waves split the positions of a chunk.  Per 32 positions
// a wave forms the transposed scores S^T = K Q^T and the transposed output
// O^T += V^T W^T: the accumulator layout of S^T (query = lane & 15, position
// = 4 * (lane / 16) + register) is, for two tiles of 16 positions, the
// operand layout of W^T, so the weights never leave the lane.  V^T is read
// from a wave's own LDS tile with the transposing loads.
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
    int slot0, slots;     // first partial of this launch, partials per row
    float scale;          // scale * log2(e)
    float* pm;            // [row][slot] base
    float* pl;            //             sum
    float* po;            //             [hd] output
    float* scores;        // [row][sstride] or null
    int sstride;
};

constexpr float kSeqLift = 15.0f;

// XOR on the 16-byte chunk index of V row r, so that the four rows that a
// 16-lane group of a transposing load reads lie in different banks.
template <int HD>
__device__ __forceinline__ int v_swizzle(int r) {
    if (HD == 128) return 2 * (r & 3);
    if (HD == 64) return 2 * ((r >> 1) & 1);
    return 0;  // 192- and 64-byte rows spread by themselves
}

// HD: head size rounded up to 32 (hd <= HD, hd % 8 == 0); NQ: tiles of 16
// query rows; OWN: each token's own rows instead of the shared ones.
template <int HD, int NQ, bool OWN>
__global__ __launch_bounds__(256) void seq_attend_kernel(SeqArgs a) {
    constexpr int KK = HD / 32, DT = HD / 16, CH = HD / 8;
    constexpr int VB = kSeqTile * HD;  // halves of a V tile
    __shared__ __align__(16) _Float16 vs[kSeqWaves][VB];
    __shared__ __align__(16) float so[kSeqWaves][16][HD];
    __shared__ float sm[kSeqWaves][16], sl[kSeqWaves][16];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int col = lane & 15, grp = lane >> 4;
    const float ninf = -__int_as_float(0x7f800000);

    int g, rb, slot, tok = 0, a0, a1;  // rows a0 .. a1 - 1 of the cache
    int b = blockIdx.x;
    g = b % a.n_kv;
    b /= a.n_kv;
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
    const int part = ((a1 - a0 + kSeqQuantum - 1) / kSeqQuantum) * kSeqTile;  // positions of a wave
    const int p0 = min(a1, a0 + wave * part), p1 = min(a1, p0 + part);

    // query rows: row = rb * 16 * NQ + 16 * nq + col of this kv head
    const int rows = OWN ? a.r : a.n * a.r;
    h8 qh[NQ][KK], ql[NQ][KK];
    float c[NQ];
    int lim[NQ];  // rows past it are masked
    size_t part_row[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        const int rr = rb * 16 * NQ + 16 * nq + col;
        const bool on = rr < rows;
        const int i = OWN ? tok : rr / a.r, hh = OWN ? rr : rr - i * a.r;
        const size_t row = on ? (size_t)i * a.n_heads + g * a.r + hh : 0;
        part_row[nq] = row;
        lim[nq] = a.causal ? a.start + a.len - (a.n - 1 - (on ? i : 0)) : a1;
        float x[KK][8];
        float mx = 0.0f;
#pragma unroll
        for (int kk = 0; kk < KK; kk++) {
            const int d = 32 * kk + 8 * grp;
            f4 u = {0, 0, 0, 0}, v = {0, 0, 0, 0};
            if (on && d < a.hd) {
                const float* p = a.q + row * a.hd + d;
                u = *(const f4*)p;
                v = *(const f4*)(p + 4);
            }
#pragma unroll
            for (int j = 0; j < 4; j++) {
                x[kk][j] = u[j];
                x[kk][4 + j] = v[j];
                mx = fmaxf(mx, fmaxf(fabsf(u[j]), fabsf(v[j])));
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        // 2^k mx in [2^14, 2^15); rows of zeros, infinities and NaN as they are
        int e = 15;
        if (mx > 0.0f && mx < __int_as_float(0x7f800000)) (void)frexpf(mx, &e);
        const int k = 15 - e;
        c[nq] = ldexpf(a.scale, -k);
#pragma unroll
        for (int kk = 0; kk < KK; kk++)
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const float v = ldexpf(x[kk][j], k);
                const _Float16 hi = (_Float16)v;
                qh[nq][kk][j] = hi;
                ql[nq][kk][j] = (_Float16)(v - (float)hi);
            }
    }

    f4 o[NQ][DT];
    float base[NQ], l[NQ];
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        base[nq] = ninf;
        l[nq] = 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; dt++) o[nq][dt] = f4{0, 0, 0, 0};
    }
    _Float16* vt = vs[wave];
    for (int pb = p0; pb < p1; pb += kSeqTile) {
        // K operands: position 16 t + col, 8 dims at 32 kk + 8 grp
        h8 kf[2][KK];
#pragma unroll
        for (int t = 0; t < 2; t++) {
            const int pos = pb + 16 * t + col;
            const uint16_t* p = a.K + (size_t)min(pos, p1 - 1) * a.kd_k + g * a.hd;
#pragma unroll
            for (int kk = 0; kk < KK; kk++) {
                const int d = 32 * kk + 8 * grp;
                u4 v = {0, 0, 0, 0};
                if (d < a.hd && pos < p1) v = *(const u4*)(p + d);
                kf[t][kk] = __builtin_bit_cast(h8, v);
            }
        }
        // V tile: rows past the range are zero, as their weights are (0 * Inf is not)
#pragma unroll
        for (int i = 0; i < kSeqTile * CH / 64; i++) {
            const int e = 64 * i + lane, rr = e / CH, ch = e % CH;
            const int pos = pb + rr;
            u4 v = {0, 0, 0, 0};
            if (8 * ch < a.hd && pos < p1) v = *(const u4*)(a.V + (size_t)pos * a.kd_v + g * a.hd + 8 * ch);
            *(u4*)(vt + rr * HD + 8 * (ch ^ v_swizzle<HD>(rr))) = v;
        }
        asm volatile("" ::: "memory");
        h8 wh[NQ], wl[NQ];
#pragma unroll
        for (int nq = 0; nq < NQ; nq++) {
            f4 s[2];
#pragma unroll
            for (int t = 0; t < 2; t++) {
                s[t] = f4{0, 0, 0, 0};
#pragma unroll
                for (int kk = 0; kk < KK; kk++) {
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][kk], ql[nq][kk], s[t], 0, 0, 0);
                    s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf[t][kk], qh[nq][kk], s[t], 0, 0, 0);
                }
            }
            float mx = ninf;
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int pos = pb + 16 * t + 4 * grp + j;
                    s[t][j] = pos < min(lim[nq], p1) ? s[t][j] * c[nq] : ninf;
                    mx = fmaxf(mx, s[t][j]);
                }
            if (a.scores) {
                const int rr = rb * 16 * NQ + 16 * nq + col;
#pragma unroll
                for (int t = 0; t < 2; t++) {
                    const int pos = pb + 16 * t + 4 * grp;
                    if (rr < rows && pos < p1)
                        *(f4*)(a.scores + part_row[nq] * a.sstride + (pos - a.start)) = s[t];
                }
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16));
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float nb = fmaxf(base[nq], mx - kSeqLift);
            if (__any(nb > base[nq])) {
                const float f = base[nq] == ninf ? 0.0f : __builtin_amdgcn_exp2f(base[nq] - nb);
                l[nq] *= f;
#pragma unroll
                for (int dt = 0; dt < DT; dt++) o[nq][dt] *= f;
                base[nq] = nb;
            }
            const float bs = nb == ninf ? 0.0f : nb;  // nothing so far: every weight is 0
#pragma unroll
            for (int t = 0; t < 2; t++)
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float w = __builtin_amdgcn_exp2f(s[t][j] - bs);
                    l[nq] += w;
                    const _Float16 hi = (_Float16)w;
                    wh[nq][4 * t + j] = hi;
                    wl[nq][4 * t + j] = (_Float16)(w - (float)hi);
                }
        }
        // operand k = 8 grp + 4 t + j is position 16 t + 4 grp + j
#pragma unroll
        for (int dt = 0; dt < DT; dt++) {
            h8 vf;
#pragma unroll
            for (int t = 0; t < 2; t++) {
                const int rr = 16 * t + 4 * grp + (col >> 2), d = 16 * dt + 4 * (col & 3);
                s4 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (__attribute__((address_space(3))) s4*)(vt + rr * HD + 8 * ((d >> 3) ^ v_swizzle<HD>(rr)) + (d & 7)));
                const h4 y = __builtin_bit_cast(h4, x);
#pragma unroll
                for (int j = 0; j < 4; j++) vf[4 * t + j] = y[j];
            }
#pragma unroll
            for (int nq = 0; nq < NQ; nq++) {
                o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wl[nq], o[nq][dt], 0, 0, 0);
                o[nq][dt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vf, wh[nq], o[nq][dt], 0, 0, 0);
            }
        }
        asm volatile("" ::: "memory");
    }
    // the waves' results: one tile of query rows at a time through LDS
#pragma unroll
    for (int nq = 0; nq < NQ; nq++) {
        float ls = l[nq];
        ls += __shfl_xor(ls, 16);
        ls += __shfl_xor(ls, 32);
        __syncthreads();
        if (grp == 0) {
            sm[wave][col] = base[nq];
            sl[wave][col] = ls;
        }
#pragma unroll
        for (int dt = 0; dt < DT; dt++) *(f4*)&so[wave][col][16 * dt + 4 * grp] = o[nq][dt];
        __syncthreads();
        // thread t: row t / 16, dims (t % 16) * 4 + 64 u
        const int row = threadIdx.x >> 4, rr = rb * 16 * NQ + 16 * nq + row;
        float M = ninf, L = 0.0f, f[kSeqWaves];
#pragma unroll
        for (int w = 0; w < kSeqWaves; w++) M = fmaxf(M, sm[w][row]);
#pragma unroll
        for (int w = 0; w < kSeqWaves; w++) {
            f[w] = sm[w][row] == ninf ? 0.0f : __builtin_amdgcn_exp2f(sm[w][row] - M);
            L = fmaf(sl[w][row], f[w], L);
        }
        if (rr < rows) {
            const int i = OWN ? tok : rr / a.r, hh = OWN ? rr : rr - i * a.r;
            const size_t at = ((size_t)i * a.n_heads + g * a.r + hh) * a.slots + a.slot0 + slot;
            if ((threadIdx.x & 15) == 0) {
                a.pm[at] = M;
                a.pl[at] = L;
            }
            for (int d = 4 * (threadIdx.x & 15); d < a.hd; d += 64) {
                f4 x = {0, 0, 0, 0};
#pragma unroll
                for (int w = 0; w < kSeqWaves; w++) x += f[w] * *(const f4*)&so[w][row][d];
                *(f4*)(a.po + at * a.hd + d) = x;
            }
        }
    }
}

// out[row] = sum_s 2^(base_s - M) o_s / sum_s 2^(base_s - M) l_s; a row
// without positions is zero.  ml, if set: M and 1 / sum of each row.
__global__ __launch_bounds__(128) void seq_merge_kernel(const float* __restrict__ pm, const float* __restrict__ pl,
                                                        const float* __restrict__ po, int slots, int hd,
                                                        float* __restrict__ out, float* __restrict__ ml) {
    const size_t row = blockIdx.x;
    const int d = threadIdx.x;
    const float ninf = -__int_as_float(0x7f800000);
    pm += row * slots;
    pl += row * slots;
    float M = ninf;
    for (int s = 0; s < slots; s++) M = fmaxf(M, pm[s]);
    float L = 0.0f, o = 0.0f;
    for (int s = 0; s < slots; s++) {
        const float f = pm[s] == ninf ? 0.0f : __builtin_amdgcn_exp2f(pm[s] - M);
        L = fmaf(pl[s], f, L);
        if (d < hd) o = fmaf(po[(row * slots + s) * hd + d], f, o);
    }
    const float inv = L == 0.0f ? 0.0f : 1.0f / L;
    if (d < hd) out[row * hd + d] = L == 0.0f ? 0.0f : o * inv;
    if (ml && d == 0) {
        ml[2 * row] = M;
        ml[2 * row + 1] = inv;
    }
}

// mass[g][start + t] += the weights of position t over the rows of kv head g
__global__ __launch_bounds__(256) void seq_mass_kernel(const float* __restrict__ scores, int sstride,
                                                       const float* __restrict__ ml, int n, int n_heads, int r,
                                                       int len, float* __restrict__ mass, int mass_stride) {
    const int g = blockIdx.y, t = blockIdx.x * 256 + threadIdx.x;
    if (t >= len) return;
    float sum = 0.0f;
    for (int i = 0; i < n; i++)
        for (int h = 0; h < r; h++) {
            const size_t row = (size_t)i * n_heads + g * r + h;
            const float inv = ml[2 * row + 1];
            if (inv != 0.0f) sum += __builtin_amdgcn_exp2f(scores[row * sstride + t] - ml[2 * row]) * inv;
        }
    mass[(size_t)g * mass_stride + t] += sum;
}

template <int HD, int NQ, bool OWN>
static void seq_launch(const SeqArgs& a, int blocks, hipStream_t s) {
    hipLaunchKernelGGL((seq_attend_kernel<HD, NQ, OWN>), dim3(blocks), dim3(256), 0, s, a);
}

template <int NQ, bool OWN>
static void seq_launch_hd(const SeqArgs& a, int blocks, hipStream_t s) {
    if (a.hd <= 32) seq_launch<32, NQ, OWN>(a, blocks, s);
    else if (a.hd <= 64) seq_launch<64, NQ, OWN>(a, blocks, s);
    else if (a.hd <= 96) seq_launch<96, NQ, OWN>(a, blocks, s);
    else seq_launch<128, NQ, OWN>(a, blocks, s);
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

static void seq_shared(const SeqArgs& a, const SeqPlan& p, hipStream_t s) {
    const int blocks = a.n_kv * p.row_blocks * p.chunks;
    if (p.nq == 1) seq_launch_hd<1, false>(a, blocks, s);
    else if (p.nq == 2) seq_launch_hd<2, false>(a, blocks, s);
    else seq_launch_hd<4, false>(a, blocks, s);
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
    if (p.chunks) {
        seq_shared(a, p, s);
        GLLM_HIP(hipGetLastError());
    }
    if (p.splits) {
        a.slot0 = p.chunks;
        seq_launch_hd<1, true>(a, n_kv_heads * p.own_blocks * n * p.splits, s);
        GLLM_HIP(hipGetLastError());
    }
    hipLaunchKernelGGL(seq_merge_kernel, dim3((unsigned)p.rows), dim3(128), 0, s, a.pm, a.pl, a.po, p.slots, hd, d_out,
                       (float*)nullptr);
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
    float* ml = w + p.rows * (size_t)sstride;
    SeqArgs a = seq_args(kv, l, d_q, n, n_heads, n_kv_heads, hd, scale, p, ml + (p.rows * 2 + 3) / 4 * 4);
    a.start = start;
    a.len = len;
    a.causal = 1;
    a.scores = w;
    a.sstride = sstride;
    seq_shared(a, p, s);
    GLLM_HIP(hipGetLastError());
    hipLaunchKernelGGL(seq_merge_kernel, dim3((unsigned)p.rows), dim3(128), 0, s, a.pm, a.pl, a.po, p.slots, hd, d_out, ml);
    GLLM_HIP(hipGetLastError());
    hipLaunchKernelGGL(seq_mass_kernel, dim3((len + 255) / 256, n_kv_heads), dim3(256), 0, s, w, sstride, ml, n, n_heads,
                       p.r, len, d_mass + start, mass_stride);
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

}  // extern "C"
