// kv_copy.hip -- rows of the F16 KV cache copied in every layer: the accepted
// tokens of a draft moved together behind their context, and ranges of rows
// forked, moved down over free ones, exchanged, or brought to another cache.  The
// reference copies whole prefixes on the host (runtime.go:1334).
#include <algorithm>
#include <new>

#include "copy_plan.h"
#include "gllm_common.h"
#include "kv_cache.h"

namespace gllm {

typedef uint32_t u4 __attribute__((ext_vector_type(4)));

constexpr int kCopyLayers = 32;  // layers of a launch: their pointers are its arguments
struct CopyPtrs {
    const uint16_t *k[kCopyLayers], *v[kCopyLayers];
    uint16_t *dk[kCopyLayers], *dv[kCopyLayers];
};

// A thread owns 16 bytes of a row, in one layer, for all rows of a request, so a
// path that goes up (path[k] >= k) needs no other thread's reads to be done: one
// launch, no barrier, no room beside the cache.  Bound by memory (64 requests of up to
// 9 rows of 8 heads of 128 in 24 layers, 64 MB read and written: 11 us) and by a launch
// and three dependent reads (one request: 4 us).
struct PathArgs {
    const int32_t *starts, *lens, *path, *accepted;
    int m, ck, cv, max_len;  // 16-byte pieces of a row of keys, of values
};

__global__ __launch_bounds__(256) void keep_path_kernel(CopyPtrs p, PathArgs a) {
    constexpr int U = 8;
    int c = blockIdx.x * 256 + threadIdx.x;
    const int i = blockIdx.y, l = blockIdx.z;
    if (c >= a.ck + a.cv) return;
    const bool v = c >= a.ck;
    if (v) c -= a.ck;
    const int per = v ? a.cv : a.ck;
    u4* rows = (u4*)(v ? p.dv[l] : p.dk[l]) + c;
    const int taken = min(max(a.accepted[i], 0), a.m);
    const long long base = (long long)a.starts[i] + max(a.lens[i], 0);
    const int32_t* path = a.path + (size_t)i * a.m;
    for (int k0 = 0; k0 < taken; k0 += U) {
        u4 x[U];
        long long from[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int k = k0 + u, j = k < taken ? path[k] : 0;
            from[u] = base + j;
            // what is in place already, or outside the tree or the cache, or would go there, stays
            if (k >= taken || j <= k || j >= a.m || base + k < 0 || from[u] >= a.max_len) from[u] = -1;
            if (from[u] >= 0) x[u] = rows[from[u] * per];
        }
#pragma unroll
        for (int u = 0; u < U; u++)
            if (from[u] >= 0) rows[(base + k0 + u) * per] = x[u];
    }
}

// Ranges of a launch.  Those that read the same rows are one group: the rows are
// read once.
constexpr int kCopyRanges = 96;
struct CopyArgs {
    int groups, ck, cv, sk, sv, dk, dv;  // pieces of a row; of a row's stride at the source, at the destination
    int tile[kCopyRanges + 1];           // the groups' first tiles
    int src[kCopyRanges], rows[kCopyRanges], to[kCopyRanges + 1];  // first destination of each
    int dst[kCopyRanges];
};

constexpr int kCopyTile = 32;  // rows of a workgroup

// Moves of which none writes what another reads.  COLS: threads across a row, so
// that 256 / COLS rows go at a time.  Rows that several moves read are read once.
// Bound by memory: 1.57 GB read and written (2000 rows of 8 heads of 128 in 24 layers, to
// 7 places) take 326 us, 4.8 TB/s, a large copy's rate; a few rows take 3.6 us, a launch.
template <int COLS>
__global__ __launch_bounds__(256) void copy_apart_kernel(CopyPtrs p, CopyArgs a) {
    constexpr int R = 256 / COLS, U = kCopyTile / R < 8 ? kCopyTile / R : 8;
    const int tile = blockIdx.x, l = blockIdx.z;
    int c = blockIdx.y * COLS + threadIdx.x % COLS;
    if (c >= a.ck + a.cv) return;
    int g = 0;
    for (int step = 64; step >= 1; step >>= 1)
        if (g + step < a.groups && a.tile[g + step] <= tile) g += step;
    const bool v = c >= a.ck;
    if (v) c -= a.ck;
    const int ss = v ? a.sv : a.sk, ds = v ? a.dv : a.dk;
    const int r0 = (tile - a.tile[g]) * kCopyTile, end = min(r0 + kCopyTile, a.rows[g]);
    const u4* from = (const u4*)(v ? p.v[l] : p.k[l]) + (size_t)a.src[g] * ss + c;
    u4* to = (u4*)(v ? p.dv[l] : p.dk[l]) + c;
    for (int r = r0 + (int)threadIdx.x / COLS; r < end; r += R * U) {
        u4 x[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (r + R * u < end) x[u] = from[(size_t)(r + R * u) * ss];
        for (int d = a.to[g]; d < a.to[g + 1]; d++) {
            u4* at = to + (size_t)(a.dst[d] + r) * ds;
#pragma unroll
            for (int u = 0; u < U; u++)
                if (r + R * u < end) at[(size_t)(R * u) * ds] = x[u];
        }
    }
}

// Moves in order, each of which may write what it or an earlier one reads.  A
// workgroup has COLS 16-byte pieces of a row, in one layer, to itself, and all rows:
// 4096 / COLS at a time, all read before the first is written (8 requests of 1000 to
// 2000 rows of 8 heads of 128 in 24 layers: 540 us for 2.6 GB read and written, 4.8
// TB/s, a large copy's rate).
struct OrderArgs {
    int moves, rows, ck, cv, step;  // step: the largest power of two below moves
    int begin[kCopyRanges + 1];     // the moves' first rows, of all rows in order
    int src[kCopyRanges], dst[kCopyRanges];
};

constexpr int kOrderVec = 16;
constexpr int kOrderWorkgroups = 96;  // fewer are slower than reading the rows twice
constexpr int order_rows(int cols) { return 256 / cols * kOrderVec; }  // that one step takes

template <int COLS>
__global__ __launch_bounds__(256) void copy_ordered_kernel(CopyPtrs p, OrderArgs a) {
    constexpr int R = 256 / COLS, U = kOrderVec;
    __shared__ int begin[kCopyRanges + 1], src[kCopyRanges], dst[kCopyRanges];
    for (int i = threadIdx.x; i < a.moves; i += 256) {
        begin[i] = a.begin[i];
        src[i] = a.src[i];
        dst[i] = a.dst[i];
    }
    if (threadIdx.x == 0) begin[a.moves] = a.rows;
    __syncthreads();
    const int l = blockIdx.y, kb = (a.ck + COLS - 1) / COLS;
    const bool v = (int)blockIdx.x >= kb;
    const int per = v ? a.cv : a.ck, c = ((int)blockIdx.x - (v ? kb : 0)) * COLS + threadIdx.x % COLS;
    u4* rows = (u4*)(v ? p.dv[l] : p.dk[l]) + c;
    const bool on = c < per;
    for (int r0 = 0; r0 < a.rows; r0 += R * U) {
        u4 x[U];
        int to[U];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int r = r0 + R * u + (int)threadIdx.x / COLS;
            to[u] = -1;
            if (on && r < a.rows) {
                int g = 0;
                for (int step = a.step; step >= 1; step >>= 1)
                    if (g + step < a.moves && begin[g + step] <= r) g += step;
                // up from the first row, or, where the rows go up, down from the last
                const int at = dst[g] < src[g] ? r - begin[g] : begin[g + 1] - 1 - r;
                to[u] = dst[g] + at;
                x[u] = rows[(size_t)(src[g] + at) * per];
            }
        }
        __syncthreads();
#pragma unroll
        for (int u = 0; u < U; u++)
            if (to[u] >= 0) rows[(size_t)to[u] * per] = x[u];
        // the next rows' reads may pass these writes: no later move reads what they write
    }
}

static int copy_current(const char* what, const gllm_hip_kv* kv) {
    int dev = -1;
    GLLM_HIP(hipGetDevice(&dev));
    if (dev != kv->device) return fail(GLLM_EINVAL, "%s: the cache is on device %d, the current one is %d", what, kv->device, dev);
    if (kv->max_len > 1 << 30 || kv->kv_dim_k > 1 << 24 || kv->kv_dim_v > 1 << 24 || (kv->kv_dim_k | kv->kv_dim_v) % 8)
        return fail(GLLM_EUNSUP, "%s: a cache of %d rows of %d and %d values", what, kv->max_len, kv->kv_dim_k, kv->kv_dim_v);
    return GLLM_OK;
}

// The moves, apart from each other, from rows at `from` to rows at `to`.
static int launch_apart(const std::vector<RowMove>& all, const CopyPtrs& p, int layers, int ck, int cv, hipStream_t s) {
    std::vector<RowMove> moves = all;
    std::sort(moves.begin(), moves.end(), [](const RowMove& a, const RowMove& b) {
        return a.src != b.src ? a.src < b.src : a.rows != b.rows ? a.rows < b.rows : a.dst < b.dst;
    });
    for (size_t i = 0; i < moves.size();) {
        CopyArgs a{};
        a.ck = a.sk = a.dk = ck;
        a.cv = a.sv = a.dv = cv;
        int n = 0;
        for (; i < moves.size() && n < kCopyRanges; i++, n++) {
            const RowMove& m = moves[i];
            if (n == 0 || m.src != a.src[a.groups - 1] || m.rows != a.rows[a.groups - 1]) {
                a.src[a.groups] = m.src;
                a.rows[a.groups] = m.rows;
                a.to[a.groups] = n;
                a.tile[a.groups + 1] = a.tile[a.groups] + (m.rows + kCopyTile - 1) / kCopyTile;
                a.groups++;
            }
            a.dst[n] = m.dst;
            a.to[a.groups] = n + 1;
        }
        const int cols = ck + cv;
        const unsigned tiles = (unsigned)a.tile[a.groups];
        const auto grid = [&](int c) { return dim3(tiles, (unsigned)((cols + c - 1) / c), (unsigned)layers); };
        if (cols <= 32) hipLaunchKernelGGL(copy_apart_kernel<32>, grid(32), dim3(256), 0, s, p, a);
        else if (cols <= 64) hipLaunchKernelGGL(copy_apart_kernel<64>, grid(64), dim3(256), 0, s, p, a);
        else if (cols <= 128) hipLaunchKernelGGL(copy_apart_kernel<128>, grid(128), dim3(256), 0, s, p, a);
        else hipLaunchKernelGGL(copy_apart_kernel<256>, grid(256), dim3(256), 0, s, p, a);
        GLLM_HIP(hipGetLastError());
    }
    return GLLM_OK;
}

static int order_slices(int cols, int ck, int cv) { return (ck + cols - 1) / cols + (cv + cols - 1) / cols; }
// Whole lines where that makes workgroups enough for launches of `layers` layers
static int order_cols(int layers, int ck, int cv) {
    return (long long)layers * order_slices(8, ck, cv) >= 2 * kOrderWorkgroups ? 8 : 4;
}

static int launch_ordered(const std::vector<RowMove>& moves, const CopyPtrs& p, int layers, int ck, int cv, int cols, hipStream_t s) {
    for (size_t i = 0; i < moves.size();) {
        OrderArgs a{};
        a.ck = ck;
        a.cv = cv;
        for (; i < moves.size() && a.moves < kCopyRanges; i++, a.moves++) {
            a.begin[a.moves] = a.rows;
            a.src[a.moves] = moves[i].src;
            a.dst[a.moves] = moves[i].dst;
            a.rows += moves[i].rows;
        }
        for (a.step = 1; 2 * a.step < a.moves;) a.step *= 2;
        const dim3 grid((unsigned)order_slices(cols, ck, cv), (unsigned)layers);
        if (cols == 8) hipLaunchKernelGGL(copy_ordered_kernel<8>, grid, dim3(256), 0, s, p, a);
        else hipLaunchKernelGGL(copy_ordered_kernel<4>, grid, dim3(256), 0, s, p, a);
        GLLM_HIP(hipGetLastError());
    }
    return GLLM_OK;
}

// Layers of a launch, about the same for each: as many as its arguments have room for
// and, where rows are set aside, a workspace of about 256 MB, one at least.
static int launch_layers(int layers, size_t staged_bytes) {
    size_t most = std::min(layers, kCopyLayers);
    if (staged_bytes) most = std::max<size_t>(1, std::min(most, ((size_t)256 << 20) / staged_bytes));
    const int launches = (layers + (int)most - 1) / (int)most;
    return (layers + launches - 1) / launches;
}

struct CopyWay {
    CopyPlan plan;
    size_t rows, layer;  // set aside, and their bytes in a layer
    int step, cols;      // layers of a launch; pieces of a row that a workgroup has in order
};

static int copy_check(const char* what, const gllm_hip_kv* src, const gllm_hip_kv* dst, const int32_t* moves, int n, CopyWay* way, size_t* bytes) {
    if (n < 0 || n > kCopyMost) return fail(GLLM_EINVAL, "%s: %d moves, up to %d are taken", what, n, kCopyMost);
    if (!src || !dst || (n > 0 && !moves)) return fail(GLLM_EINVAL, "%s: null pointer", what);
    if (src->layers != dst->layers || src->kv_dim_k != dst->kv_dim_k || src->kv_dim_v != dst->kv_dim_v)
        return fail(GLLM_EINVAL, "%s: caches of %d and %d layers of %d / %d and %d / %d values", what, src->layers, dst->layers,
                    src->kv_dim_k, src->kv_dim_v, dst->kv_dim_k, dst->kv_dim_v);
    size_t rows = 0;
    for (int i = 0; i < n; i++) {
        const int32_t* m = moves + 3 * i;
        if (m[2] < 0 || m[0] < 0 || m[1] < 0 || (long long)m[0] + m[2] > src->max_len || (long long)m[1] + m[2] > dst->max_len)
            return fail(GLLM_EINVAL, "%s: move %d of %d rows from %d of %d to %d of %d", what, i, m[2], m[0], src->max_len, m[1], dst->max_len);
        rows += (size_t)m[2];
    }
    if (rows > (size_t)1 << 28) return fail(GLLM_EUNSUP, "%s: %zu rows", what, rows);
    CopyPlan& p = way->plan;
    const int ck = src->kv_dim_k / 8, cv = src->kv_dim_v / 8;
    const auto lay_out = [&] {
        way->rows = 0;
        for (const RowMove& m : p.staged) way->rows += m.rows;
        way->layer = way->rows * ((size_t)src->kv_dim_k + src->kv_dim_v) * 2;
        way->step = launch_layers(src->layers, way->layer);
        way->cols = order_cols(way->step, ck, cv);
    };
    try {
        p = copy_plan(moves, n, src == dst);
        if (!p.ok) return fail(GLLM_EINVAL, "%s: two moves write the same rows", what);
        const int once = order_cols(launch_layers(src->layers, 0), ck, cv);
        if (!p.apart && rows <= (size_t)order_rows(once) && p.moves.size() + p.staged.size() <= kCopyRanges) {
            // all rows are read before one is written
            p.moves.insert(p.moves.end(), p.staged.begin(), p.staged.end());
            p.staged.clear();
        }
        lay_out();
        if (!p.apart && rows > (size_t)4 * order_rows(4) && (long long)way->step * order_slices(8, ck, cv) < kOrderWorkgroups) {
            // many rows twice, by all of the device, rather than in order by a few of its
            // CUs: 12000 rows of 8 heads of 128 take 50 us in order and 30 staged in one
            // layer, 99 and 77 in two, 137 and 160 in four; 700 rows 8 and 12.  What counts
            // is the layers of a launch: two places of 65536 such rows exchanged in 24
            // layers, one a launch, 22.6 and 9.9 ms; 12000 rows of one head of 128 moved
            // down by 5 in 33, 17 a launch, 0.18 and 0.11
            p.staged.insert(p.staged.end(), p.moves.begin(), p.moves.end());
            p.moves.clear();
            lay_out();
        }
    } catch (const std::bad_alloc&) {
        return fail(GLLM_ENOMEM, "%s: no host memory for %d moves", what, n);
    }
    *bytes = way->layer * way->step;
    return GLLM_OK;
}

}  // namespace gllm

using namespace gllm;

extern "C" {

int gllm_hip_kv_keep_path_dev(gllm_hip_kv* kv, int n, int m, const int32_t* d_starts, const int32_t* d_lens, const int32_t* d_path,
                              const int32_t* d_accepted, void* stream) {
    const char* what = "gllm_hip_kv_keep_path_dev";
    if (n < 1 || n > 65535 || m < 1) return fail(GLLM_EINVAL, "%s: %d requests of %d tokens", what, n, m);
    if (!kv || !d_starts || !d_lens || !d_path || !d_accepted) return fail(GLLM_EINVAL, "%s: null pointer", what);
    GLLM_TRY(copy_current(what, kv));
    const PathArgs a{d_starts, d_lens, d_path, d_accepted, m, kv->kv_dim_k / 8, kv->kv_dim_v / 8, kv->max_len};
    for (int l0 = 0; l0 < kv->layers; l0 += kCopyLayers) {
        const int layers = std::min(kCopyLayers, kv->layers - l0);
        CopyPtrs p{};
        for (int i = 0; i < layers; i++) {
            p.dk[i] = kv->k[l0 + i];
            p.dv[i] = kv->v[l0 + i];
        }
        hipLaunchKernelGGL(keep_path_kernel, dim3((unsigned)((a.ck + a.cv + 255) / 256), (unsigned)n, (unsigned)layers), dim3(256), 0,
                           (hipStream_t)stream, p, a);
        GLLM_HIP(hipGetLastError());
    }
    return GLLM_OK;
}

size_t gllm_hip_kv_copy_rows_bytes(const gllm_hip_kv* src, const gllm_hip_kv* dst, const int32_t* moves, int n) {
    CopyWay way;
    size_t bytes = 0;
    return copy_check("gllm_hip_kv_copy_rows_bytes", src, dst, moves, n, &way, &bytes) == GLLM_OK ? bytes : 0;
}

int gllm_hip_kv_copy_rows_dev(const gllm_hip_kv* src, gllm_hip_kv* dst, const int32_t* moves, int n, void* d_work, size_t work_bytes,
                              void* stream) {
    const char* what = "gllm_hip_kv_copy_rows_dev";
    CopyWay way;
    size_t bytes = 0;
    GLLM_TRY(copy_check(what, src, dst, moves, n, &way, &bytes));
    const CopyPlan& plan = way.plan;
    GLLM_TRY(copy_current(what, src));
    GLLM_TRY(copy_current(what, dst));
    if (d_work && (((uintptr_t)d_work & 15) || work_bytes < bytes))
        return fail(GLLM_EINVAL, "%s: the workspace needs %zu bytes, 16-byte aligned", what, bytes);
    if (d_work && bytes)
        for (int l = 0; l < src->layers; l++)
            for (const gllm_hip_kv* c : {src, (const gllm_hip_kv*)dst})
                if (bytes_meet(d_work, bytes, c->k[l], (size_t)c->max_len * c->kv_dim_k * 2) ||
                    bytes_meet(d_work, bytes, c->v[l], (size_t)c->max_len * c->kv_dim_v * 2))
                    return fail(GLLM_EINVAL, "%s: the workspace overlaps a cache", what);
    if (plan.moves.empty() && plan.staged.empty()) return GLLM_OK;
    hipStream_t s = (hipStream_t)stream;
    char* work = nullptr;
    if (bytes) {
        work = (char*)(d_work ? d_work : thread_scratch(13, bytes, s));
        if (!work) return scratch_error();
    }
    const int ck = src->kv_dim_k / 8, cv = src->kv_dim_v / 8;
    try {
        size_t rows = 0;
        std::vector<RowMove> out, in;  // to the workspace, and from it
        for (const RowMove& m : plan.staged) {
            out.push_back({m.src, (int)rows, m.rows});
            in.push_back({(int)rows, m.dst, m.rows});
            rows += m.rows;
        }
        for (int l0 = 0; l0 < src->layers; l0 += way.step) {
            const int layers = std::min(way.step, src->layers - l0);
            CopyPtrs p{}, there{}, back{};
            for (int i = 0; i < layers; i++) {
                p.k[i] = there.k[i] = src->k[l0 + i];
                p.v[i] = there.v[i] = src->v[l0 + i];
                p.dk[i] = back.dk[i] = dst->k[l0 + i];
                p.dv[i] = back.dv[i] = dst->v[l0 + i];
                uint16_t* at = (uint16_t*)(work + way.layer * i);
                back.k[i] = there.dk[i] = at;
                back.v[i] = there.dv[i] = at + rows * ck * 8;
            }
            if (plan.apart) {
                GLLM_TRY(launch_apart(plan.moves, p, layers, ck, cv, s));
                continue;
            }
            GLLM_TRY(launch_apart(out, there, layers, ck, cv, s));
            GLLM_TRY(launch_ordered(plan.moves, p, layers, ck, cv, way.cols, s));
            GLLM_TRY(launch_apart(in, back, layers, ck, cv, s));
        }
    } catch (const std::bad_alloc&) {
        return fail(GLLM_ENOMEM, "%s: no host memory for %d moves", what, n);
    }
    return GLLM_OK;
}

}  // extern "C"
