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
#include <new>

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
// 6e-8).  |a| < 2^41 (an int32 position times an inverse frequency below 2^10):
// n pi/2 loses nothing that a itself, rounded once to 64 bits, still has.
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
    uint64_t unit_magic;  // ceil(2^32 / units of a head)
};

// cos and sin of a token's angles, times the amplitude, into cs
__device__ __forceinline__ void rope_angles(const RopeArgs& a, int t, float2* cs) {
    for (int i = threadIdx.x; i < a.rot / 2; i += 256) {
        double s, c;
        sincos64((double)a.pos[t] * a.inv[i], &s, &c);
        cs[i] = make_float2((float)(c * a.amp), (float)(s * a.amp));
    }
}

__device__ __forceinline__ float2 turn(float x0, float x1, float2 w) {
    return make_float2(fmaf(x0, w.x, -(x1 * w.y)), fmaf(x0, w.y, x1 * w.x));
}

// The row that unit e of a token is in
__device__ __forceinline__ const float* rope_source(const RopeArgs& a, size_t t, int e, int n_q, int n_k) {
    const bool is_q = e < n_q, is_k = e < n_q + n_k;
    const size_t stride = is_q ? a.q_stride : is_k ? a.k_stride : a.v_stride;
    const uintptr_t base = is_q ? (uintptr_t)a.q : is_k ? (uintptr_t)a.k : (uintptr_t)a.v;
    return (const float*)base + t * stride;
}

// A token's queries, keys and values in units of four values (HALF: of two
// such quads half a rotation apart), one a thread; blockIdx.y takes the
// units from its number times 256 on, in steps of the grid, and its first
// unit is on its way while the angles are made.  Bound by memory: 4001 tokens
// of 32 / 8 heads of 128 (180 MB) take 38 us, 4.7 TB/s (a pair a thread took 54).
template <bool HALF>
__global__ __launch_bounds__(256) void rope_quads_kernel(RopeArgs a) {
    __shared__ __align__(16) float2 cs[512];
    const size_t t = blockIdx.x;
    const int half = a.rot / 2;
    const int row = a.rows ? a.rows[t] : -1;
    const bool store = row >= 0 && row < a.max_len;
    const int unit = (HALF ? a.hd - half : a.hd) / 4;  // of a head
    const int n_q = a.q ? a.heads * unit : 0, n_k = store ? a.n_kv * unit : 0, n_v = store ? a.n_kv * a.hd / 4 : 0;
    const int all = n_q + n_k + n_v, step = 256 * gridDim.y;
    const float4 none = make_float4(0, 0, 0, 0);
    // unit e: its head's unit u (past the head's turning values for v), and its place in the row of heads
    const auto place = [&](int e, int& u) {
        if (e >= n_q + n_k) {
            u = a.hd;
            return 4 * (e - n_q - n_k);
        }
        const int f = e < n_q ? e : e - n_q, h = (int)(((uint64_t)f * a.unit_magic) >> 32);  // f / unit
        u = f - h * unit;
        return h * a.hd + 4 * u + (HALF && 4 * u >= half ? half : 0);
    };
    const auto finish = [&](int e, int u, int at, float4 x, float4 y) {
        const bool two = HALF && 4 * u < half;
        if (two) {
            const float4 w0 = *(const float4*)&cs[4 * u], w1 = *(const float4*)&cs[4 * u + 2];
            const float2 p0 = turn(x.x, y.x, make_float2(w0.x, w0.y)), p1 = turn(x.y, y.y, make_float2(w0.z, w0.w));
            const float2 p2 = turn(x.z, y.z, make_float2(w1.x, w1.y)), p3 = turn(x.w, y.w, make_float2(w1.z, w1.w));
            x = make_float4(p0.x, p1.x, p2.x, p3.x);
            y = make_float4(p0.y, p1.y, p2.y, p3.y);
        } else if (!HALF && 4 * u < a.rot) {
            const float4 w = *(const float4*)&cs[2 * u];
            const float2 p0 = turn(x.x, x.y, make_float2(w.x, w.y)), p1 = turn(x.z, x.w, make_float2(w.z, w.w));
            x = make_float4(p0.x, p0.y, p1.x, p1.y);
        }
        if (e < n_q) {
            float* o = a.q_out + t * a.out_stride + at;
            *(float4*)o = x;
            if (two) *(float4*)(o + half) = y;
        } else {
            const auto pack = [](float4 f) {
                return make_uint2(f32_to_f16_bits(f.x) | (uint32_t)f32_to_f16_bits(f.y) << 16,
                                  f32_to_f16_bits(f.z) | (uint32_t)f32_to_f16_bits(f.w) << 16);
            };
            uint16_t* o = (e < n_q + n_k ? a.K + (size_t)row * a.kd_k : a.V + (size_t)row * a.kd_v) + at;
            *(uint2*)o = pack(x);
            if (two) *(uint2*)(o + half) = pack(y);
        }
    };
    int e = blockIdx.y * 256 + threadIdx.x, u = 0, at = 0;
    float4 x = none, y = none;
    if (e < all) {
        at = place(e, u);
        const float* src = rope_source(a, t, e, n_q, n_k) + at;
        x = *(const float4*)src;
        if (HALF && 4 * u < half) y = *(const float4*)(src + half);
    }
    rope_angles(a, t, cs);
    __syncthreads();
    if (e < all) finish(e, u, at, x, y);
    for (e += step; e < all; e += step) {
        at = place(e, u);
        const float* src = rope_source(a, t, e, n_q, n_k) + at;
        x = *(const float4*)src;
        y = none;
        if (HALF && 4 * u < half) y = *(const float4*)(src + half);
        finish(e, u, at, x, y);
    }
}

// The same for any sizes and alignments, a pair or a value that stays at a
// time.  One workgroup per token.
__global__ __launch_bounds__(256) void rope_pairs_kernel(RopeArgs a) {
    __shared__ float2 cs[512];
    const size_t t = blockIdx.x;
    const int half = a.rot / 2;
    rope_angles(a, t, cs);
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
        float2 y;
        if (i < half) {
            i0 = a.half_layout ? i : 2 * i;
            i1 = a.half_layout ? i + half : 2 * i + 1;
            y = turn(x[i0], x[i1], cs[i]);
        } else {
            i0 = i1 = i + half;
            y.x = y.y = x[i0];
        }
        if (is_q) {
            float* o = a.q_out + t * a.out_stride + h * a.hd;
            o[i0] = y.x;
            o[i1] = y.y;
        } else {
            uint16_t* o = a.K + (size_t)row * a.kd_k + h * a.hd;
            o[i0] = f32_to_f16_bits(y.x);
            o[i1] = f32_to_f16_bits(y.y);
        }
    }
    if (store)
        for (int e = threadIdx.x; e < a.n_kv * a.hd; e += 256)
            a.V[(size_t)row * a.kd_v + e] = f32_to_f16_bits(a.v[t * a.v_stride + e]);
}

static int rope_launch(RopeArgs a, int n, hipStream_t s) {
    if (n == 0) return GLLM_OK;
    // quads: 16-byte loads and 8-byte f16 stores, and no quad that turns in part
    const uintptr_t ptrs = (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.k | (uintptr_t)a.v;
    const int strides = (a.q ? a.q_stride | a.out_stride : 0) | (a.rows ? a.k_stride | a.v_stride | a.kd_k | a.kd_v : 0);
    if (ptrs % 16 == 0 && strides % 4 == 0 && a.hd % 4 == 0 && a.rot % (a.half_layout ? 8 : 4) == 0) {
        const int unit = (a.half_layout ? a.hd - a.rot / 2 : a.hd) / 4;
        const long long all = (a.q ? (long long)a.heads * unit : 0) + (a.rows ? (long long)a.n_kv * (unit + a.hd / 4) : 0);
        if (all < 65536) {  // where the multiplication divides exactly
            a.unit_magic = (0x100000000ull + unit - 1) / unit;
            // a few tokens: their units over several workgroups (one token of 32 / 8
            // heads of 128 takes 3.2 us over 6, 5.1 in one)
            const int parts = std::max(1, std::min((int)((all + 255) / 256), 512 / n));
            if (a.half_layout) hipLaunchKernelGGL(rope_quads_kernel<true>, dim3((unsigned)n, parts), dim3(256), 0, s, a);
            else hipLaunchKernelGGL(rope_quads_kernel<false>, dim3((unsigned)n, parts), dim3(256), 0, s, a);
            GLLM_HIP(hipGetLastError());
            return GLLM_OK;
        }
    }
    hipLaunchKernelGGL(rope_pairs_kernel, dim3((unsigned)n), dim3(256), 0, s, a);
    GLLM_HIP(hipGetLastError());
    return GLLM_OK;
}

static int rope_check(const char* what, const gllm_hip_rope* r, int n, const int32_t* d_pos) {
    if (!r) return fail(GLLM_EINVAL, "%s: null rope", what);
    if (n < 0 || (n > 0 && !d_pos)) return fail(GLLM_EINVAL, "%s: %d tokens without positions", what, n);
    if (n >= 1 << 24) return fail(GLLM_EINVAL, "%s: %d tokens are more than a launch holds", what, n);
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
    gllm_hip_rope* out = new (std::nothrow) gllm_hip_rope(r);
    if (!out) {
        (void)hipFree(r.d_inv);
        fail(GLLM_ENOMEM, "gllm_hip_rope_new: out of memory");
    }
    return out;
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
