// rope.hip -- rotary positions for callers of the cache: any layout, part of
// the head, scaled frequencies (applyPreparedRope model.go:3051-3093,
// ropeInterleaved :3084), alone and with the store of the rotated keys and
// the values (storeKV model.go:1466).
//
//   angle = pos * inv_i   y0 = x0 c - x1 s   y1 = x0 s + x1 c
//
// The angle, its reduction and its sine and cosine are 64-bit (a float32
// product is 2^-8 rad off at a million), c and s are rounded to float32 once
// and shared by all heads of a token.
#include <math.h>

#include <algorithm>
#include <vector>

#include "gllm_common.h"
#include "kv_cache.h"
#include "rope_freq.h"

struct gllm_hip_rope {
    int head_dim, rot_dim, layout;
    double amp;
    double* d_inv;
    int device;
};

namespace gllm {

// Sine and cosine of a by reduction to [-pi/4, pi/4]: a - n pi/2 with pi/2 in
// two parts, each step one fma, then the Taylor series through r^13 and r^12
// (the first terms left out are below 2e-14 and 4e-13, a float32 rounding is
// 6e-8).  Exact to float32 for |a| < 2^31: n needs 31 bits and the products'
// rounding is absorbed by the fma.
__device__ __forceinline__ void sincos64(double a, double* s, double* c) {
    const double n = rint(a * 0.63661977236758134308);
    double r = fma(-n, 1.57079632679489655800, a);
    r = fma(-n, 6.12323399573676603587e-17, r);
    const double z = r * r;
    double ps = fma(z, 1.0 / 6227020800.0, -1.0 / 39916800.0);
    ps = fma(z, ps, 1.0 / 362880.0);
    ps = fma(z, ps, -1.0 / 5040.0);
    ps = fma(z, ps, 1.0 / 120.0);
    ps = fma(z, ps, -1.0 / 6.0);
    const double sn = fma(r * z, ps, r);
    double pc = fma(z, 1.0 / 479001600.0, -1.0 / 3628800.0);
    pc = fma(z, pc, 1.0 / 40320.0);
    pc = fma(z, pc, -1.0 / 720.0);
    pc = fma(z, pc, 1.0 / 24.0);
    pc = fma(z, pc, -0.5);
    const double cs = fma(z, pc, 1.0);
    const int q = (int)(long long)n & 3;
    const double u = (q & 1) ? cs : sn, v = (q & 1) ? sn : cs;
    *s = (q & 2) ? -u : u;
    *c = (q == 1 || q == 2) ? -v : v;
}

struct RopeArgs {
    const double* inv;
    double amp;
    int hd, rot, half_layout;
    const int32_t* pos;
    const float *q, *k, *v;
    float* q_out;
    int q_stride, k_stride, v_stride, out_stride, heads, n_kv;
    const int32_t* rows;  // cache rows, null: q alone
    uint16_t *K, *V;
    int kd_k, kd_v, max_len;
};

// One workgroup per token.
__global__ __launch_bounds__(256) void rope_kernel(RopeArgs a) {
    __shared__ float2 cs[512];
    const size_t t = blockIdx.x;
    const int half = a.rot / 2;
    for (int i = threadIdx.x; i < half; i += 256) {
        double s, c;
        sincos64((double)a.pos[t] * a.inv[i], &s, &c);
        cs[i] = make_float2((float)(c * a.amp), (float)(s * a.amp));
    }
    __syncthreads();
    const int row = a.rows ? a.rows[t] : -1;
    const bool store = row >= 0 && row < a.max_len;
    const int unit = half + a.hd - a.rot;  // pairs, then values that stay
    const int n_q = a.q ? a.heads * unit : 0, n_k = store ? a.n_kv * unit : 0;
    for (int e = threadIdx.x; e < n_q + n_k; e += 256) {
        const bool is_q = e < n_q;
        const int f = is_q ? e : e - n_q, h = f / unit, i = f - h * unit;
        const float* x = (is_q ? a.q + t * a.q_stride : a.k + t * a.k_stride) + h * a.hd;
        int i0, i1;
        float y0, y1;
        if (i < half) {
            i0 = a.half_layout ? i : 2 * i;
            i1 = a.half_layout ? i + half : 2 * i + 1;
            const float x0 = x[i0], x1 = x[i1];
            const float2 w = cs[i];
            y0 = fmaf(x0, w.x, -(x1 * w.y));
            y1 = fmaf(x0, w.y, x1 * w.x);
        } else {
            i0 = i1 = i + half;
            y0 = y1 = x[i0];
        }
        if (is_q) {
            float* o = a.q_out + t * a.out_stride + h * a.hd;
            o[i0] = y0;
            o[i1] = y1;
        } else {
            uint16_t* o = a.K + (size_t)row * a.kd_k + h * a.hd;
            o[i0] = f32_to_f16_bits(y0);
            o[i1] = f32_to_f16_bits(y1);
        }
    }
    if (store)
        for (int e = threadIdx.x; e < a.n_kv * a.hd; e += 256)
            a.V[(size_t)row * a.kd_v + e] = f32_to_f16_bits(a.v[t * a.v_stride + e]);
}

static int rope_launch(const RopeArgs& a, int n, hipStream_t s) {
    if (n == 0) return GLLM_OK;
    hipLaunchKernelGGL(rope_kernel, dim3((unsigned)n), dim3(256), 0, s, a);
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

static int rope_check(const char* what, const gllm_hip_rope* r, int n, const int32_t* d_pos) {
    if (!r) return fail(GLLM_EINVAL, "%s: null rope", what);
    if (n < 0 || (n > 0 && !d_pos)) return fail(GLLM_EINVAL, "%s: %d tokens without positions", what, n);
    int dev = -1;
    GLLM_HIP(hipGetDevice(&dev));
    if (dev != r->device) return fail(GLLM_EINVAL, "%s: the rope is on device %d, the current one is %d", what, r->device, dev);
    return GLLM_OK;
}

static RopeArgs rope_args(const gllm_hip_rope* r, const int32_t* d_pos) {
    RopeArgs a{};
    a.inv = r->d_inv;
    a.amp = r->amp;
    a.hd = r->head_dim;
    a.rot = r->rot_dim;
    a.half_layout = r->layout == GLLM_ROPE_HALF;
    a.pos = d_pos;
    return a;
}

}  // namespace gllm

using namespace gllm;

extern "C" {

int gllm_hip_rope_frequencies(const gllm_hip_rope_config* cfg, double* inv, double* amp) {
    if (!cfg || !inv || !amp) return fail(GLLM_EINVAL, "gllm_hip_rope_frequencies: null pointer");
    if (const char* why = rope_config_error(*cfg)) return fail(GLLM_EINVAL, "gllm_hip_rope_frequencies: %s", why);
    rope_frequencies(*cfg, inv, amp);
    return GLLM_OK;
}

gllm_hip_rope* gllm_hip_rope_new(const gllm_hip_rope_config* cfg) {
    if (!cfg) {
        fail(GLLM_EINVAL, "gllm_hip_rope_new: null configuration");
        return nullptr;
    }
    if (const char* why = rope_config_error(*cfg)) {
        fail(GLLM_EINVAL, "gllm_hip_rope_new: %s", why);
        return nullptr;
    }
    double inv[512];
    gllm_hip_rope r{cfg->head_dim, cfg->rot_dim, cfg->layout, 0.0, nullptr, 0};
    rope_frequencies(*cfg, inv, &r.amp);
    const size_t bytes = (size_t)(cfg->rot_dim / 2) * sizeof(double);
    if (check(hipGetDevice(&r.device), "gllm_hip_rope_new") != GLLM_OK) return nullptr;
    if (hipMalloc(&r.d_inv, bytes) != hipSuccess) {
        (void)hipGetLastError();
        fail(GLLM_ENOMEM, "gllm_hip_rope_new: out of device memory");
        return nullptr;
    }
    if (check(hipMemcpy(r.d_inv, inv, bytes, hipMemcpyHostToDevice), "gllm_hip_rope_new") != GLLM_OK) {
        (void)hipFree(r.d_inv);
        return nullptr;
    }
    return new gllm_hip_rope(r);
}

void gllm_hip_rope_release(gllm_hip_rope* r) {
    if (!r) return;
    (void)hipFree(r->d_inv);
    delete r;
}

int gllm_hip_rope_dev(const gllm_hip_rope* r, const float* d_x, int x_stride, int n, int heads, const int32_t* d_pos,
                      float* d_out, int out_stride, void* stream) {
    const char* what = "gllm_hip_rope_dev";
    GLLM_TRY(rope_check(what, r, n, d_pos));
    const long long dim = (long long)heads * r->head_dim;
    if (heads < 1 || x_stride < dim || out_stride < dim)
        return fail(GLLM_EINVAL, "%s: %d heads of %d do not fit rows of %d and %d", what, heads, r->head_dim, x_stride, out_stride);
    if (n > 0 && (!d_x || !d_out)) return fail(GLLM_EINVAL, "%s: null pointer", what);
    if (d_x == d_out && x_stride != out_stride) return fail(GLLM_EINVAL, "%s: in place needs one row stride", what);
    RopeArgs a = rope_args(r, d_pos);
    a.q = d_x;
    a.q_stride = x_stride;
    a.heads = heads;
    a.q_out = d_out;
    a.out_stride = out_stride;
    return rope_launch(a, n, (hipStream_t)stream);
}

int gllm_hip_kv_store_rope_dev(gllm_hip_kv* kv, int l, const gllm_hip_rope* r, const float* d_q, int q_stride,
                               int n_heads, const float* d_k, int k_stride, const float* d_v, int v_stride,
                               int n_kv_heads, int n, const int32_t* d_pos, const int32_t* d_rows, float* d_q_out,
                               int out_stride, void* stream) {
    const char* what = "gllm_hip_kv_store_rope_dev";
    GLLM_TRY(rope_check(what, r, n, d_pos));
    if (!kv) return fail(GLLM_EINVAL, "%s: null cache", what);
    if (l < 0 || l >= kv->layers) return fail(GLLM_EINVAL, "%s: layer %d out of range", what, l);
    if (kv->device != r->device) return fail(GLLM_EINVAL, "%s: the cache is on device %d, the rope on %d", what, kv->device, r->device);
    const long long kd = (long long)n_kv_heads * r->head_dim, qd = (long long)n_heads * r->head_dim;
    if (n_kv_heads < 1 || kd > kv->kv_dim_k || kd > kv->kv_dim_v || k_stride < kd || v_stride < kd)
        return fail(GLLM_EINVAL, "%s: %d kv heads of %d do not fit the cache or the rows of k and v", what, n_kv_heads, r->head_dim);
    if (d_q && (n_heads < 1 || q_stride < qd || out_stride < qd))
        return fail(GLLM_EINVAL, "%s: %d heads of %d do not fit rows of %d and %d", what, n_heads, r->head_dim, q_stride, out_stride);
    if (n > 0 && (!d_k || !d_v || !d_rows || (d_q && !d_q_out))) return fail(GLLM_EINVAL, "%s: null pointer", what);
    if (d_q && d_q == d_q_out && q_stride != out_stride) return fail(GLLM_EINVAL, "%s: in place needs one row stride", what);
    RopeArgs a = rope_args(r, d_pos);
    a.q = d_q;
    a.q_stride = q_stride;
    a.heads = n_heads;
    a.q_out = d_q_out;
    a.out_stride = out_stride;
    a.k = d_k;
    a.k_stride = k_stride;
    a.v = d_v;
    a.v_stride = v_stride;
    a.n_kv = n_kv_heads;
    a.rows = d_rows;
    a.K = kv->k[l];
    a.V = kv->v[l];
    a.kd_k = kv->kv_dim_k;
    a.kd_v = kv->kv_dim_v;
    a.max_len = kv->max_len;
    return rope_launch(a, n, (hipStream_t)stream);
}

}  // extern "C"
