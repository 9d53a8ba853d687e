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

constexpr int kKeepThreads = 1024;

// One workgroup per (layer, kv head): the budget-th largest key by four
// passes of a byte each, then the kept rows in row order.
__global__ __launch_bounds__(kKeepThreads) void keep_select_kernel(KeepArgs a) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const size_t lg = blockIdx.x;
    const float* mass = a.mass + lg * a.stride + a.start;
    const int32_t* pos = a.pos ? a.pos + lg * a.stride + a.start : nullptr;
    __shared__ int hist[256];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    __shared__ int w_gt[kKeepThreads / 64], w_eq[kKeepThreads / 64];
    const auto key = [&](int t) {
        const int p = pos ? pos[t] : a.start + t;
        return kept_always(p, a.sinks, a.from) ? 0xFFFFFFFFu : mass_key(mass[t]);
    };
    uint32_t prefix = 0;
    int need = a.budget;  // rows still wanted among those with this prefix
    for (int shift = 24; shift >= 0; shift -= 8) {
        if (tid < 256) hist[tid] = 0;
        __syncthreads();
        const uint32_t mask = shift == 24 ? 0u : 0xFFFFFFFFu << (shift + 8);
        for (int t = tid; t < a.len; t += kKeepThreads) {
            const uint32_t k = key(t);
            if ((k & mask) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
        }
        __syncthreads();
        if (tid == 0) {
            int b = 255, left = need;
            while (b > 0 && hist[b] < left) left -= hist[b--];
            s_prefix = prefix | ((uint32_t)b << shift);
            s_need = left;
        }
        __syncthreads();
        prefix = s_prefix;
        need = s_need;
    }
    // rows above the threshold, and the first `need` rows at it
    int done = 0, eq_done = 0;
    for (int t0 = 0; t0 < a.len; t0 += kKeepThreads) {
        const int t = t0 + tid;
        const uint32_t k = t < a.len ? key(t) : 0;
        const bool eq = t < a.len && k == prefix, gt = t < a.len && k > prefix;
        const uint64_t be = __ballot(eq), bg = __ballot(gt);
        if (lane == 0) {
            w_eq[wave] = __popcll(be);
            w_gt[wave] = __popcll(bg);
        }
        __syncthreads();
        int eq_before = eq_done, gt_before = 0, eq_all = eq_done, gt_all = 0;
        for (int w = 0; w < kKeepThreads / 64; w++) {
            if (w < wave) {
                eq_before += w_eq[w];
                gt_before += w_gt[w];
            }
            eq_all += w_eq[w];
            gt_all += w_gt[w];
        }
        const uint64_t below = (1ull << lane) - 1;
        eq_before += __popcll(be & below);
        gt_before += __popcll(bg & below);
        if (gt || (eq && eq_before < need)) {
            const int at = done + gt_before + min(eq_before, need) - min(eq_done, need);
            a.list[lg * a.budget + at] = a.start + t;
            a.mass_out[lg * a.out_stride + a.dst_start + at] = mass[t];
            a.pos_out[lg * a.out_stride + a.dst_start + at] = pos ? pos[t] : a.start + t;
        }
        done += gt_all + min(eq_all, need) - min(eq_done, need);
        eq_done = eq_all;
        __syncthreads();
    }
}

constexpr int kKeepLayers = 32;  // layers of a copy launch: their pointers are its arguments
struct KeepPtrs {
    const uint16_t *k[kKeepLayers], *v[kKeepLayers];
    uint16_t *dk[kKeepLayers], *dv[kKeepLayers];
};

// dst row dst_start + j of head g = src row list[j]; 16 bytes a thread.
__global__ __launch_bounds__(256) void keep_copy_kernel(KeepPtrs p, const int32_t* __restrict__ list, int layer0, int n_kv,
                                                        int hd, int budget, int dst_start, int sk, int sv, int dk, int dv) {
    const int l = blockIdx.y, ch = hd / 8;
    const long long e = (long long)blockIdx.x * 256 + threadIdx.x;  // (row, head, chunk)
    if (e >= (long long)budget * n_kv * ch) return;
    const int c = (int)(e % ch), g = (int)(e / ch % n_kv), j = (int)(e / ch / n_kv);
    const size_t row = list[((size_t)(layer0 + l) * n_kv + g) * budget + j], to = (size_t)dst_start + j;
    const int col = g * hd + 8 * c;
    const u4 kk = *(const u4*)(p.k[l] + row * sk + col), vv = *(const u4*)(p.v[l] + row * sv + col);
    *(u4*)(p.dk[l] + to * dk + col) = kk;
    *(u4*)(p.dv[l] + to * dv + col) = vv;
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

// One workgroup per kv head: the least (key, row), then the store.
__global__ __launch_bounds__(kKeepThreads) void evict_store_kernel(EvictArgs a) {
    const int g = blockIdx.x, tid = threadIdx.x;
    float* mass = a.mass + (size_t)g * a.stride + a.start;
    int32_t* pos = a.pos + (size_t)g * a.stride + a.start;
    const int now = *a.now;
    const long long from = (long long)now - a.recent;
    uint64_t best = ~0ull;
    for (int t = tid; t < a.len; t += kKeepThreads) {
        const uint32_t k = kept_always(pos[t], a.sinks, from) ? 0xFFFFFFFFu : mass_key(mass[t]);
        best = min(best, (uint64_t)k << 32 | (uint32_t)t);
    }
    __shared__ uint64_t wb[kKeepThreads / 64];
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) best = min(best, (uint64_t)__shfl_xor((unsigned long long)best, off));
    if ((tid & 63) == 0) wb[tid >> 6] = best;
    __syncthreads();
    best = wb[0];
    for (int w = 1; w < kKeepThreads / 64; w++) best = min(best, wb[w]);
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
    if (stride < start + len || out_stride < dst_start + budget)
        return fail(GLLM_EINVAL, "%s: mass rows of %d and %d values do not hold the rows", what, stride, out_stride);
    const size_t heads = (size_t)src->layers * n_kv_heads;
    const auto apart = [&](const void* in, const void* out) {
        const uintptr_t i = (uintptr_t)in, o = (uintptr_t)out;
        return !in || i + heads * stride * 4 <= o || o + heads * out_stride * 4 <= i;
    };
    if (!apart(d_mass, d_mass_out) || !apart(d_mass, d_pos_out) || !apart(d_pos, d_mass_out) || !apart(d_pos, d_pos_out))
        return fail(GLLM_EINVAL, "%s: outputs overlap the inputs", what);
    GLLM_TRY(current_is(what, src));
    GLLM_TRY(current_is(what, dst));
    hipStream_t s = (hipStream_t)stream;
    const size_t bytes = gllm_hip_kv_keep_bytes(src->layers, n_kv_heads, budget);
    if (d_work && (((uintptr_t)d_work & 15) || work_bytes < bytes))
        return fail(GLLM_EINVAL, "%s: the workspace needs %zu bytes, 16-byte aligned", what, bytes);
    int32_t* list = d_work ? (int32_t*)d_work : (int32_t*)thread_scratch(11, bytes, s);
    if (!list) return scratch_error();
    KeepArgs a{d_mass, d_pos, d_mass_out, d_pos_out, list, n_kv_heads, stride, out_stride, start, dst_start, len, budget, sinks,
               (long long)now - recent};
    hipLaunchKernelGGL(keep_select_kernel, dim3((unsigned)(src->layers * n_kv_heads)), dim3(kKeepThreads), 0, s, a);
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
        hipLaunchKernelGGL(keep_copy_kernel, dim3((unsigned)((items + 255) / 256), (unsigned)n), dim3(256), 0, s, p, list, l0,
                           n_kv_heads, hd, budget, dst_start, src->kv_dim_k, src->kv_dim_v, dst->kv_dim_k, dst->kv_dim_v);
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
    GLLM_TRY(current_is(what, kv));
    EvictArgs a{d_k, d_v, d_mass, d_pos, d_now, d_rows_out, kv->k[l], kv->v[l], stride, start, len, sinks, recent, hd,
                kv->kv_dim_k, kv->kv_dim_v};
    hipLaunchKernelGGL(evict_store_kernel, dim3((unsigned)n_kv_heads), dim3(kKeepThreads), 0, (hipStream_t)stream, a);
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

}  // extern "C"
