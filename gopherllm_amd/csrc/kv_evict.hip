// kv_evict.hip -- which rows of a cache stay, by the attention weight they
// have received (gllm_hip_attend_mass_dev): a prompt's rows copied down to a
// budget, and a new token's row in place of the one of least weight.  No
// counterpart in the reference, whose cache ends at max_len.
//
// Per (layer, kv head), since each head attends on its own.  Order of rows:
// protected ones first (the first `sinks` positions and the newest `recent`),
// all alike, then by weight, NaN below every number.
#include <algorithm>

#include "gllm_common.h"
#include "kv_cache.h"

namespace gllm {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

// Order-preserving image of a weight in 32 bits, below 0xFFFFFFFF; -0 is 0
// and NaN is 0, below every number's.
__device__ __forceinline__ uint32_t mass_key(float m) {
    if (m != m) return 0;
    const uint32_t u = __float_as_uint(m + 0.0f);
    return (u >> 31) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ bool kept_always(int pos, int sinks, long long from) { return pos < sinks || pos >= from; }

struct KeepArgs {
    const float* mass;   // [layer][kv head][stride]
    const int32_t* pos;  // same, or null: a row is its position
    float* mass_out;     // [layer][kv head][out_stride]
    int32_t* pos_out;
    int32_t* list;       // [layer][kv head][budget] kept rows
    int n_kv, stride, out_stride, start, dst_start, len, budget, sinks;
    long long from;      // now - recent
};

constexpr int kKeepThreads = 1024, kKeepWaves = kKeepThreads / 64;

// Sum over the threads after this one, and over all: for counts below 2^31.
__device__ __forceinline__ int sum_after(int v, int* wave_sums) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int s = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int x = __shfl_down(s, off);
        if (lane + off < 64) s += x;
    }
    __syncthreads();  // the sums of an earlier call have been read
    if (lane == 0) wave_sums[wave] = s;
    __syncthreads();
    int after = s - v;
#pragma unroll
    for (int w = 0; w < kKeepWaves; w++) after += w > wave ? wave_sums[w] : 0;
    return after;
}

// One workgroup per (layer, kv head).  The budget-th largest key by three
// histograms in LDS of its 12, 10 and 10 leading bits: 12, because weights
// share their sign and most of their exponent, and an LDS counter that many
// lanes want serves them one by one (16384 rows of 24 layers x 8 heads take 21
// us; digits of 8 bits took 100, counting by ballots, two bits a pass, 52).
// Then the kept rows in row order, from the counts of every run of 64 rows.
//
// KPT: rows of a thread in a tile (row = 1024 (tile KPT + i) + thread); the
// keys of a single tile stay in registers, those of more are read per pass.
template <int KPT>
__global__ __launch_bounds__(kKeepThreads) void keep_select_kernel(KeepArgs a) {
    constexpr int kTile = KPT * kKeepThreads, kRuns = KPT * kKeepWaves, kBins = 4096;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t lg = blockIdx.x;
    const float* mass = a.mass + lg * a.stride + a.start;
    const int32_t* pos = a.pos ? a.pos + lg * a.stride + a.start : nullptr;
    __shared__ __align__(16) int hist[kBins];
    __shared__ int wave_sums[kKeepWaves], wave_at[kKeepWaves];
    __shared__ uint32_t s_thr;
    __shared__ int s_left;
    uint32_t key[KPT];
    const auto load = [&](int t0) {
        float m[KPT];  // all on their way before the first is looked at
        int p[KPT];
#pragma unroll
        for (int i = 0; i < KPT; i++) {
            const int t = min(t0 + kKeepThreads * i + tid, a.len - 1);
            m[i] = mass[t];
            p[i] = a.start + t;
        }
        if (pos) {
#pragma unroll
            for (int i = 0; i < KPT; i++) p[i] = pos[min(t0 + kKeepThreads * i + tid, a.len - 1)];
        }
#pragma unroll
        for (int i = 0; i < KPT; i++) key[i] = kept_always(p[i], a.sinks, a.from) ? 0xFFFFFFFFu : mass_key(m[i]);
    };
    const bool one = a.len <= kTile;
    if (one) load(0);
    uint32_t thr = 0;
    int left = a.budget;  // rows still wanted among the keys with these leading bits
#pragma unroll
    for (int pass = 0; pass < 3; pass++) {
        const int shift = pass == 0 ? 20 : pass == 1 ? 10 : 0, bins = pass == 0 ? kBins : 1024;
        for (int i = tid; i < bins; i += kKeepThreads) hist[i] = 0;
        __syncthreads();
        for (int t0 = 0; t0 < a.len; t0 += kTile) {
            if (!one) load(t0);
#pragma unroll
            for (int i = 0; i < KPT; i++) {
                const bool in = pass == 0 || ((key[i] ^ thr) >> (pass == 1 ? 20 : 10)) == 0;
                if (in && t0 + kKeepThreads * i + tid < a.len) atomicAdd(&hist[(key[i] >> shift) & (bins - 1)], 1);
            }
        }
        __syncthreads();
        // thread t holds the bins 4 t .. 4 t + 3, or t; after: keys in the bins above
        const int per = bins / kKeepThreads;
        int c[4] = {0, 0, 0, 0}, mine = 0;
#pragma unroll
        for (int j = 0; j < 4; j++)
            if (j < per) mine += c[j] = hist[per * tid + j];
        int after = sum_after(mine, wave_sums);
        if (after < left && after + mine >= left) {
#pragma unroll
            for (int j = 3; j >= 0; j--) {
                if (j < per && after < left && after + c[j] >= left) {
                    s_thr = thr | (uint32_t)(per * tid + j) << shift;
                    s_left = left - after;
                    break;
                }
                after += c[j];
            }
        }
        __syncthreads();
        thr = s_thr;
        left = s_left;
    }
    // kept: keys above the threshold, and the first `left` rows at it
    int* above = hist;  // of each run, then before each run
    int* at_it = hist + kRuns;
    static_assert(2 * kRuns <= kBins, "the runs' counts reuse the histogram");
    int done = 0, at_done = 0;  // rows kept, and keys at the threshold, before this tile
    for (int t0 = 0; t0 < a.len; t0 += kTile) {
        if (!one) load(t0);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KPT; i++) {
            const bool in = t0 + kKeepThreads * i + tid < a.len;
            const int up = __popcll(__ballot(in && key[i] > thr)), eq = __popcll(__ballot(in && key[i] == thr));
            if (lane == 0) {
                above[i * kKeepWaves + wave] = up;
                at_it[i * kKeepWaves + wave] = eq;
            }
        }
        __syncthreads();
        const int u = tid < kRuns ? above[tid] : 0, e = tid < kRuns ? at_it[tid] : 0;
        int su = u, se = e;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int x = __shfl_up(su, off), y = __shfl_up(se, off);
            if (lane >= off) {
                su += x;
                se += y;
            }
        }
        if (lane == 63) {
            wave_sums[wave] = su;
            wave_at[wave] = se;
        }
        __syncthreads();
        int bu = 0, be = 0, up_all = 0, at_all = 0;
        for (int w = 0; w < kKeepWaves; w++) {
            bu += w < wave ? wave_sums[w] : 0;
            be += w < wave ? wave_at[w] : 0;
            up_all += wave_sums[w];
            at_all += wave_at[w];
        }
        if (tid < kRuns) {
            above[tid] = bu + su - u;
            at_it[tid] = be + se - e;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < KPT; i++) {
            const int t = t0 + kKeepThreads * i + tid;
            const bool gt = t < a.len && key[i] > thr, eq = t < a.len && key[i] == thr;
            const uint64_t below = (1ull << lane) - 1;
            const int up = above[i * kKeepWaves + wave] + __popcll(__ballot(gt) & below);
            const int before = at_done + at_it[i * kKeepWaves + wave] + __popcll(__ballot(eq) & below);
            if (gt || (eq && before < left)) {
                const int at = done + up + min(before, left) - min(at_done, left);
                // always below the budget, unless another stream changes the weights meanwhile
                if (at < a.budget) a.list[lg * a.budget + at] = a.start + t;  // the copy brings its mass and position
            }
        }
        done += up_all + min(at_done + at_all, left) - min(at_done, left);
        at_done += at_all;
    }
}

constexpr int kKeepLayers = 32;  // layers of a copy launch: their pointers are its arguments
struct KeepPtrs {
    const uint16_t *k[kKeepLayers], *v[kKeepLayers];
    uint16_t *dk[kKeepLayers], *dv[kKeepLayers];
};

// dst row dst_start + j of head g = src row list[j], with its mass and
// position; 16 bytes a thread.  Bound by memory: 2048 rows of 24 layers x 8
// heads of 128 (403 MB) take 82 us, 4.9 TB/s.
__global__ __launch_bounds__(256) void keep_copy_kernel(KeepPtrs p, KeepArgs a, int layer0, int hd, int sk, int sv, int dk,
                                                        int dv) {
    const int l = blockIdx.y, ch = hd / 8;
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;  // (row, head, chunk)
    if (e >= (long long)a.budget * a.n_kv * ch) return;
    const int c = (int)(e % ch), g = (int)(e / ch % a.n_kv), j = (int)(e / ch / a.n_kv);
    const size_t lg = (size_t)(layer0 + l) * a.n_kv + g;
    // in the range whatever the list holds after such a race
    const size_t row = min(max(a.list[lg * a.budget + j], a.start), a.start + a.len - 1), to = (size_t)a.dst_start + j;
    const int col = g * hd + 8 * c;
    const u4 kk = *(const u4*)(p.k[l] + row * sk + col), vv = *(const u4*)(p.v[l] + row * sv + col);
    *(u4*)(p.dk[l] + to * dk + col) = kk;
    *(u4*)(p.dv[l] + to * dv + col) = vv;
    if (c == 0) {
        a.mass_out[lg * a.out_stride + to] = a.mass[lg * a.stride + row];
        a.pos_out[lg * a.out_stride + to] = a.pos ? a.pos[lg * a.stride + row] : (int)row;
    }
}

struct EvictArgs {
    const float *k, *v;
    float* mass;   // [kv head][stride]
    int32_t* pos;
    const int32_t* now;
    int32_t* rows_out;
    uint16_t *K, *V;
    int stride, start, len, sinks, recent, hd, kd_k, kd_v;
};

// One workgroup per kv head: the least (key, row), then the store.  A launch's
// length up to a few thousand rows (3.6 us for 1024), then one CU's reads.
__global__ __launch_bounds__(kKeepThreads) void evict_store_kernel(EvictArgs a) {
    const int g = blockIdx.x, tid = threadIdx.x;
    float* mass = a.mass + (size_t)g * a.stride + a.start;
    int32_t* pos = a.pos + (size_t)g * a.stride + a.start;
    const int now = *a.now;
    const long long from = (long long)now - a.recent;
    uint64_t best = ~0ull;
    constexpr int kBatch = 8;  // rows of a thread on their way at a time (32768 rows: 10 us one by one, 6 so)
    for (int t0 = 0; t0 < a.len; t0 += kBatch * kKeepThreads) {
        float m[kBatch];
        int p[kBatch];
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            const int t = min(t0 + kKeepThreads * i + tid, a.len - 1);  // again the last row: the same candidate
            m[i] = mass[t];
            p[i] = pos[t];
        }
#pragma unroll
        for (int i = 0; i < kBatch; i++) {
            const int t = min(t0 + kKeepThreads * i + tid, a.len - 1);
            const uint32_t k = kept_always(p[i], a.sinks, from) ? 0xFFFFFFFFu : mass_key(m[i]);
            best = min(best, (uint64_t)k << 32 | (uint32_t)t);
        }
    }
    __shared__ uint64_t wb[kKeepWaves];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) best = min(best, (uint64_t)__shfl_xor((unsigned long long)best, off));
    if ((tid & 63) == 0) wb[tid >> 6] = best;
    __syncthreads();
    best = wb[0];
    for (int w = 1; w < kKeepWaves; w++) best = min(best, wb[w]);
    const int t = (int)(uint32_t)best;
    const size_t row = (size_t)a.start + t;
    if (tid < a.hd) {
        a.K[row * a.kd_k + g * a.hd + tid] = f32_to_f16_bits(a.k[g * a.hd + tid]);
        a.V[row * a.kd_v + g * a.hd + tid] = f32_to_f16_bits(a.v[g * a.hd + tid]);
    }
    if (tid == 0) {
        mass[t] = 0.0f;
        pos[t] = now;
        if (a.rows_out) a.rows_out[g] = (int)row;
    }
}

static int current_is(const char* what, const gllm_hip_kv* kv) {
    int dev = -1;
    GLLM_HIP(hipGetDevice(&dev));
    if (dev != kv->device) return fail(GLLM_EINVAL, "%s: the cache is on device %d, the current one is %d", what, kv->device, dev);
    return GLLM_OK;
}

}  // namespace gllm

using namespace gllm;

extern "C" {

size_t gllm_hip_kv_keep_bytes(int layers, int n_kv_heads, int budget) {
    if (layers < 1 || n_kv_heads < 1 || budget < 1) return 0;
    return (size_t)layers * n_kv_heads * budget * 4;
}

int gllm_hip_kv_keep_dev(const gllm_hip_kv* src, gllm_hip_kv* dst, int n_kv_heads, int hd, int start, int len,
                         int dst_start, int budget, int sinks, int recent, int now, const float* d_mass,
                         const int32_t* d_pos, int stride, float* d_mass_out, int32_t* d_pos_out, int out_stride,
                         void* d_work, size_t work_bytes, void* stream) {
    const char* what = "gllm_hip_kv_keep_dev";
    if (n_kv_heads < 1 || hd < 8 || hd % 8) return fail(GLLM_EINVAL, "%s: %d kv heads of %d", what, n_kv_heads, hd);
    if (len < 1 || budget < 1 || budget > len) return fail(GLLM_EINVAL, "%s: budget %d of %d rows", what, budget, len);
    if (sinks < 0 || recent < 0 || now < 0) return fail(GLLM_EINVAL, "%s: sinks %d, recent %d, now %d", what, sinks, recent, now);
    if (!src || !dst || !d_mass || !d_mass_out || !d_pos_out) return fail(GLLM_EINVAL, "%s: null pointer", what);
    if (src == dst) return fail(GLLM_EINVAL, "%s: the rows go to another cache", what);
    if (src->layers != dst->layers) return fail(GLLM_EINVAL, "%s: caches of %d and %d layers", what, src->layers, dst->layers);
    const long long dim = (long long)n_kv_heads * hd;
    if (dim > src->kv_dim_k || dim > src->kv_dim_v || dim > dst->kv_dim_k || dim > dst->kv_dim_v)
        return fail(GLLM_EINVAL, "%s: %d kv heads of %d do not fit the caches", what, n_kv_heads, hd);
    if ((src->kv_dim_k | src->kv_dim_v | dst->kv_dim_k | dst->kv_dim_v) % 8)
        return fail(GLLM_EUNSUP, "%s: cache rows are not 16-byte aligned", what);
    if (start < 0 || (long long)start + len > src->max_len || dst_start < 0 || (long long)dst_start + budget > dst->max_len)
        return fail(GLLM_EINVAL, "%s: rows %d + %d of %d, to %d + %d of %d", what, start, len, src->max_len, dst_start, budget, dst->max_len);
    if (src->max_len > 1 << 30 || dst->max_len > 1 << 30 || budget * dim / 8 >= 1LL << 31)
        return fail(GLLM_EUNSUP, "%s: %d rows of %lld values from %d", what, budget, dim, src->max_len);
    if (stride < start + len || out_stride < dst_start + budget)
        return fail(GLLM_EINVAL, "%s: mass rows of %d and %d values do not hold the rows", what, stride, out_stride);
    const size_t heads = (size_t)src->layers * n_kv_heads;
    const auto apart = [&](const void* in, const void* out) {
        const uintptr_t i = (uintptr_t)in, o = (uintptr_t)out;
        return !in || i + heads * stride * 4 <= o || o + heads * out_stride * 4 <= i;
    };
    if (!apart(d_mass, d_mass_out) || !apart(d_mass, d_pos_out) || !apart(d_pos, d_mass_out) || !apart(d_pos, d_pos_out))
        return fail(GLLM_EINVAL, "%s: outputs overlap the inputs", what);
    const size_t bytes = gllm_hip_kv_keep_bytes(src->layers, n_kv_heads, budget);
    if (d_work && (((uintptr_t)d_work & 15) || work_bytes < bytes))
        return fail(GLLM_EINVAL, "%s: the workspace needs %zu bytes, 16-byte aligned", what, bytes);
    const auto off_work = [&](const void* p, int row) {
        const uintptr_t w = (uintptr_t)d_work, t = (uintptr_t)p;
        return !p || !d_work || w + bytes <= t || t + heads * row * 4 <= w;
    };
    if (!off_work(d_mass, stride) || !off_work(d_pos, stride) || !off_work(d_mass_out, out_stride) || !off_work(d_pos_out, out_stride))
        return fail(GLLM_EINVAL, "%s: the workspace overlaps the tensors", what);
    GLLM_TRY(current_is(what, src));
    GLLM_TRY(current_is(what, dst));
    hipStream_t s = (hipStream_t)stream;
    int32_t* list = d_work ? (int32_t*)d_work : (int32_t*)thread_scratch(11, bytes, s);
    if (!list) return scratch_error();
    KeepArgs a{d_mass, d_pos, d_mass_out, d_pos_out, list, n_kv_heads, stride, out_stride, start, dst_start, len, budget, sinks,
               (long long)now - recent};
    const dim3 grid((unsigned)(src->layers * n_kv_heads)), block(kKeepThreads);
    // one tile of keys in registers where it holds them all: 2000 rows take 8.3 us
    // with 4 rows a thread and 13.1 with 16, which 16384 rows need
    if (len <= 4 * kKeepThreads) hipLaunchKernelGGL(keep_select_kernel<4>, grid, block, 0, s, a);
    else hipLaunchKernelGGL(keep_select_kernel<16>, grid, block, 0, s, a);
    GLLM_HIP(hipGetLastError());
    const long long items = (long long)budget * n_kv_heads * (hd / 8);
    for (int l0 = 0; l0 < src->layers; l0 += kKeepLayers) {
        const int n = std::min(kKeepLayers, src->layers - l0);
        KeepPtrs p{};
        for (int i = 0; i < n; i++) {
            p.k[i] = src->k[l0 + i];
            p.v[i] = src->v[l0 + i];
            p.dk[i] = dst->k[l0 + i];
            p.dv[i] = dst->v[l0 + i];
        }
        hipLaunchKernelGGL(keep_copy_kernel, dim3((unsigned)((items + 255) / 256), (unsigned)n), dim3(256), 0, s, p, a, l0, hd,
                           src->kv_dim_k, src->kv_dim_v, dst->kv_dim_k, dst->kv_dim_v);
        GLLM_HIP(hipGetLastError());
    }
    return GLLM_OK;
}

int gllm_hip_kv_evict_store_dev(gllm_hip_kv* kv, int l, int n_kv_heads, int hd, const float* d_k, const float* d_v,
                                int start, int len, int sinks, int recent, float* d_mass, int32_t* d_pos, int stride,
                                const int32_t* d_now, int32_t* d_rows_out, void* stream) {
    const char* what = "gllm_hip_kv_evict_store_dev";
    if (n_kv_heads < 1 || hd < 1 || hd > kKeepThreads) return fail(GLLM_EINVAL, "%s: %d kv heads of %d", what, n_kv_heads, hd);
    if (len < 1) return fail(GLLM_EINVAL, "%s: no row to give up", what);
    if (sinks < 0 || recent < 0) return fail(GLLM_EINVAL, "%s: sinks %d, recent %d", what, sinks, recent);
    if (!kv || !d_k || !d_v || !d_mass || !d_pos || !d_now) return fail(GLLM_EINVAL, "%s: null pointer", what);
    if (l < 0 || l >= kv->layers) return fail(GLLM_EINVAL, "%s: layer %d out of range", what, l);
    if ((long long)n_kv_heads * hd > kv->kv_dim_k || (long long)n_kv_heads * hd > kv->kv_dim_v)
        return fail(GLLM_EINVAL, "%s: %d kv heads of %d do not fit the cache", what, n_kv_heads, hd);
    if (start < 0 || (long long)start + len > kv->max_len || stride < start + len)
        return fail(GLLM_EINVAL, "%s: rows %d + %d of %d, mass rows of %d", what, start, len, kv->max_len, stride);
    if (kv->max_len > 1 << 30) return fail(GLLM_EUNSUP, "%s: a cache of %d rows", what, kv->max_len);
    GLLM_TRY(current_is(what, kv));
    EvictArgs a{d_k, d_v, d_mass, d_pos, d_now, d_rows_out, kv->k[l], kv->v[l], stride, start, len, sinks, recent, hd,
                kv->kv_dim_k, kv->kv_dim_v};
    hipLaunchKernelGGL(evict_store_kernel, dim3((unsigned)n_kv_heads), dim3(kKeepThreads), 0, (hipStream_t)stream, a);
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

}  // extern "C"
