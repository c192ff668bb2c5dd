// Global gradient norm over a list of tensors, clipping, and the clipped AdamW update:
//     norm = sqrt(sum over all tensors of g^2);   f = min(1, max_norm / (norm + 1e-6));
//     clip:   g <- f g
//     AdamW (no bias correction, eps added to sqrt(v), weight decay on the parameter: gzsl_adamw_nobias_step's formula):
//             m <- b1 m + (1 - b1) f g;  v <- b2 v + (1 - b2) (f g)^2;  p <- p - lr (m / (sqrt(v) + eps) + wd p)
// Two launches: every workgroup of the first adds the squares of its share in 64 bits (no overflow, no order worth speaking
// of) and stores one partial sum; every workgroup of the second adds ALL partial sums in the same order, so the factor is
// the same everywhere, needs no atomics, and two runs agree bit for bit.  The tensors' addresses travel as kernel arguments:
// nothing is copied to the device and a captured graph keeps them.
// Memory-bound.  A share is 4096 elements (16 KB of fp32): four 16-byte loads a thread, all in flight at once; the second launch
// has its first loads under way while it adds the partial sums.  Equal workgroups of both launches take equal shares, so what
// the first read the second finds in the same XCD's L2 up to 32 MB of gradients.  5.3 M fp32 gradients: 14 us with both launches (43 MB
// at the rate of a copy: 8); AdamW of 10.7 M parameters 71 us (300 MB: 59, and 8 for the norm's own read).
#include "common.h"
#include "../../include/gzsl_hip.h"

typedef __bf16 bf16;

#define CL_TENSORS 64    // tensors of a launch
#define CL_SHARE 4096    // elements of a workgroup's share, at least
#define CL_BLOCKS 2048   // shares of a call, about
#define CL_U 4           // 16-byte loads of a thread in flight
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf8 __attribute__((ext_vector_type(8)));

struct ClBatch {
    void *g[CL_TENSORS];
    long long n[CL_TENSORS];
    int first[CL_TENSORS + 1];  // first workgroup of a tensor, in this launch
    unsigned long long half;    // bit i: tensor i is bf16
    long long share;
    int count, base, total;     // tensors; index of this launch's first partial sum; partial sums of the call
};
struct ClState {
    float *p[CL_TENSORS], *m[CL_TENSORS], *v[CL_TENSORS];
};

__device__ __forceinline__ int cl_find(const ClBatch& t, int blk) {
    int lo = 0, hi = t.count;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (t.first[mid] <= blk) lo = mid;
        else hi = mid;
    }
    return lo;
}
__device__ __forceinline__ double cl_block_sum(double v, double* sh) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o);
    if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
    __syncthreads();
    return sh[0] + sh[1] + sh[2] + sh[3];
}

struct ClPiece {
    int i;
    long long lo, n;  // first element in the tensor, elements
};
__device__ __forceinline__ ClPiece cl_piece(const ClBatch& t) {
    ClPiece c;
    c.i = cl_find(t, blockIdx.x);
    c.lo = (long long)(blockIdx.x - t.first[c.i]) * t.share;
    c.n = min(t.share, t.n[c.i] - c.lo);
    return c;
}
__device__ __forceinline__ bool cl_aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename V>
__device__ __forceinline__ double cl_squares(const V& v, double s) {
    constexpr int n = sizeof(V) / sizeof(v[0]);
#pragma unroll
    for (int j = 0; j < n; ++j) s = fma((double)(float)v[j], (double)(float)v[j], s);
    return s;
}
// Sum of squares of n elements; V: 16-byte vectors of the type E.
template <typename E, typename V>
__device__ __forceinline__ double cl_sum_of(const E* g, long long n) {
    constexpr int W = 16 / sizeof(E);
    double s = 0.0;
    long long done = 0;
    if (cl_aligned(g)) {
        const long long nv = n / W;
        const V* p = reinterpret_cast<const V*>(g);
        for (long long k = threadIdx.x; k < nv; k += 256 * CL_U) {
            V v[CL_U];
#pragma unroll
            for (int u = 0; u < CL_U; ++u) v[u] = k + 256 * u < nv ? p[k + 256 * u] : V(0);
#pragma unroll
            for (int u = 0; u < CL_U; ++u) s = cl_squares(v[u], s);
        }
        done = nv * W;
    }
    for (long long k = done + threadIdx.x; k < n; k += 256) s = fma((double)(float)g[k], (double)(float)g[k], s);
    return s;
}
__global__ __launch_bounds__(256) void cl_sum_kernel(ClBatch t, double* partial) {
    __shared__ double sh[4];
    const ClPiece c = cl_piece(t);
    double s = (t.half >> c.i & 1) ? cl_sum_of<bf16, bf8>((const bf16*)t.g[c.i] + c.lo, c.n) : cl_sum_of<float, f4>((const float*)t.g[c.i] + c.lo, c.n);
    s = cl_block_sum(s, sh);
    if (threadIdx.x == 0) partial[t.base + blockIdx.x] = s;
}
__device__ __forceinline__ float cl_factor(const double* partial, int total, float max_norm, float* norm, bool write, double* sh) {
    double s = 0.0;
#pragma unroll 8
    for (int k = threadIdx.x; k < total; k += 256) s += partial[k];
    s = sqrt(cl_block_sum(s, sh));
    if (write && threadIdx.x == 0) *norm = (float)s;
    const double f = (double)max_norm / (s + 1e-6);
    return f < 1.0 ? (float)f : (f != f ? (float)f : 1.f);  // a norm that is no number makes every gradient one
}
template <typename E, typename V>
__device__ __forceinline__ void cl_scale_piece(E* g, long long n, const ClBatch& t, const double* partial, float max_norm, float* norm, double* sh) {
    constexpr int W = 16 / sizeof(E);
    const bool vec = cl_aligned(g);
    const long long nv = vec ? n / W : 0;
    V* p = reinterpret_cast<V*>(g);
    V v[CL_U];
    auto load = [&](long long k) {
#pragma unroll
        for (int u = 0; u < CL_U; ++u) v[u] = k + 256 * u < nv ? p[k + 256 * u] : V(0);
    };
    load(threadIdx.x);
    const float f = cl_factor(partial, t.total, max_norm, norm, t.base + blockIdx.x == 0, sh);
    for (long long k = threadIdx.x; k < nv;) {
#pragma unroll
        for (int u = 0; u < CL_U; ++u) {
            if (k + 256 * u >= nv) break;
#pragma unroll
            for (int j = 0; j < W; ++j) v[u][j] = (E)((float)v[u][j] * f);
            p[k + 256 * u] = v[u];
        }
        k += 256 * CL_U;
        load(k);
    }
    for (long long k = nv * W + threadIdx.x; k < n; k += 256) g[k] = (E)((float)g[k] * f);
}
__global__ __launch_bounds__(256) void cl_scale_kernel(ClBatch t, const double* partial, float max_norm, float* norm) {
    __shared__ double sh[4];
    const ClPiece c = cl_piece(t);
    if (t.half >> c.i & 1) cl_scale_piece<bf16, bf8>((bf16*)t.g[c.i] + c.lo, c.n, t, partial, max_norm, norm, sh);
    else cl_scale_piece<float, f4>((float*)t.g[c.i] + c.lo, c.n, t, partial, max_norm, norm, sh);
}
struct ClHyper {
    float lr, b1, c1, b2, c2, eps, wd;  // c = 1 - b, taken in 64 bits
};
__device__ __forceinline__ void cl_update(float& p, float g, float& m, float& v, float f, const ClHyper& h) {
    g *= f;
    m = h.b1 * m + h.c1 * g;
    v = h.b2 * v + h.c2 * g * g;
    float upd = m / (sqrtf(v) + h.eps);
    if (h.wd > 0.f) upd += h.wd * p;
    p -= h.lr * upd;
}
__global__ __launch_bounds__(256) void cl_adamw_kernel(ClBatch t, ClState st, const double* partial, float max_norm, float* norm, ClHyper h) {
    __shared__ double sh[4];
    constexpr int U = 2;
    const ClPiece c = cl_piece(t);
    const float* g = (const float*)t.g[c.i] + c.lo;
    float *p = st.p[c.i] + c.lo, *m = st.m[c.i] + c.lo, *v = st.v[c.i] + c.lo;
    const long long nv = cl_aligned(g) && cl_aligned(p) && cl_aligned(m) && cl_aligned(v) ? c.n / 4 : 0;
    f4 x[4][U];
    auto load = [&](long long k) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (k + 256 * u < nv) {
                x[0][u] = reinterpret_cast<const f4*>(g)[k + 256 * u], x[1][u] = reinterpret_cast<f4*>(p)[k + 256 * u];
                x[2][u] = reinterpret_cast<f4*>(m)[k + 256 * u], x[3][u] = reinterpret_cast<f4*>(v)[k + 256 * u];
            }
    };
    load(threadIdx.x);
    const float f = cl_factor(partial, t.total, max_norm, norm, t.base + blockIdx.x == 0, sh);
    for (long long k = threadIdx.x; k < nv;) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k + 256 * u >= nv) break;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float pp = x[1][u][j], mm = x[2][u][j], vv = x[3][u][j];
                cl_update(pp, x[0][u][j], mm, vv, f, h);
                x[1][u][j] = pp, x[2][u][j] = mm, x[3][u][j] = vv;
            }
            reinterpret_cast<f4*>(p)[k + 256 * u] = x[1][u];
            reinterpret_cast<f4*>(m)[k + 256 * u] = x[2][u];
            reinterpret_cast<f4*>(v)[k + 256 * u] = x[3][u];
        }
        k += 256 * U;
        load(k);
    }
    for (long long k = 4 * nv + threadIdx.x; k < c.n; k += 256) cl_update(p[k], g[k], m[k], v[k], f, h);
}

// shares of a call: CL_SHARE elements, more where that would make over CL_BLOCKS of them (rounded to 16 bytes of bf16)
static long long cl_share(const long long* sizes, int n, long long& blocks) {
    long long all = 0;
    for (int i = 0; i < n; ++i) all += sizes[i];
    long long share = (all + CL_BLOCKS - 1) / CL_BLOCKS;
    share = share < CL_SHARE ? CL_SHARE : (share + 1023) / 1024 * 1024;
    blocks = 0;
    for (int i = 0; i < n; ++i) blocks += (sizes[i] + share - 1) / share;
    return share;
}
static int cl_check(const long long* sizes, int n, float max_norm) {
    if (n < 0 || (n > 0 && !sizes) || !(max_norm > 0.f)) return GZSL_EINVAL;
    for (int i = 0; i < n; ++i)
        if (sizes[i] < 0) return GZSL_EINVAL;
    return 0;
}
static int cl_run(void* const* g, const long long* sizes, const int* dtypes, int n, float max_norm, float* norm, float* const* p, float* const* m,
                  float* const* v, const ClHyper* hyper, void* work, long long work_bytes, hipStream_t st) {
    long long blocks;
    const long long share = cl_share(sizes, n, blocks);
    if (blocks > 0x3FFFFFFF) return GZSL_ETOOBIG;
    if (!norm || (blocks > 0 && (!work || work_bytes < 8 * blocks || ((uintptr_t)work & 7)))) return GZSL_EINVAL;
    for (int i = 0; i < n; ++i)
        if (sizes[i] > 0 && (!g[i] || (hyper && (!p[i] || !m[i] || !v[i])))) return GZSL_EINVAL;
    double* partial = (double*)work;
    for (int pass = 0; pass < 2; ++pass) {
        int base = 0;
        ClBatch t;
        ClState s;
        t.share = share, t.total = (int)blocks, t.count = 0, t.half = 0, t.first[0] = 0;
        auto flush = [&]() {
            // (with nothing at all to update one workgroup still writes the norm, 0)
            if (t.count == 0 && !(blocks == 0 && pass == 1)) return;
            t.base = base;
            const int grid = t.count ? t.first[t.count] : 1;
            if (t.count == 0) t.n[0] = 0, t.g[0] = nullptr, s.p[0] = s.m[0] = s.v[0] = nullptr, t.count = 1, t.first[1] = 1;
            if (pass == 0) hipLaunchKernelGGL(cl_sum_kernel, dim3(grid), dim3(256), 0, st, t, partial);
            else if (hyper)
                hipLaunchKernelGGL(cl_adamw_kernel, dim3(grid), dim3(256), 0, st, t, s, partial, max_norm, norm, *hyper);
            else hipLaunchKernelGGL(cl_scale_kernel, dim3(grid), dim3(256), 0, st, t, partial, max_norm, norm);
            base += grid;
            t.count = 0, t.half = 0;
        };
        for (int i = 0; i < n; ++i) {
            if (sizes[i] == 0) continue;
            const int k = t.count++;
            t.g[k] = g[i], t.n[k] = sizes[i];
            t.first[k + 1] = t.first[k] + (int)((sizes[i] + share - 1) / share);
            if (dtypes && dtypes[i] == GZSL_BF16) t.half |= 1ULL << k;
            if (hyper) s.p[k] = p[i], s.m[k] = m[i], s.v[k] = v[i];
            if (t.count == CL_TENSORS) flush();
        }
        flush();
        GZSL_CHECK_LAUNCH();
    }
    return 0;
}

extern "C" long long gzsl_clip_work_bytes(const long long* sizes, int n) {
    if (cl_check(sizes, n, 1.f)) return -1;
    long long blocks;
    cl_share(sizes, n, blocks);
    return 8 * blocks;
}

extern "C" int gzsl_clip_grad_norm(void* const* grads, const long long* sizes, const int* dtypes, int n, float max_norm, float* norm, void* work,
                                   long long work_bytes, void* stream) {
    if (int e = cl_check(sizes, n, max_norm)) return e;
    if (n > 0 && (!grads || !dtypes)) return GZSL_EINVAL;
    for (int i = 0; i < n; ++i)
        if (dtypes[i] != GZSL_F32 && dtypes[i] != GZSL_BF16) return GZSL_EINVAL;
    return cl_run(grads, sizes, dtypes, n, max_norm, norm, nullptr, nullptr, nullptr, nullptr, work, work_bytes, (hipStream_t)stream);
}

extern "C" int gzsl_adamw_clip_step(float* const* p, const float* const* g, float* const* m, float* const* v, const long long* sizes, int n,
                                    float max_norm, double lr, double beta1, double beta2, double eps, double wd, float* norm, void* work,
                                    long long work_bytes, void* stream) {
    if (int e = cl_check(sizes, n, max_norm)) return e;
    if (n > 0 && (!p || !g || !m || !v)) return GZSL_EINVAL;
    const ClHyper hyper = {(float)lr, (float)beta1, (float)(1.0 - beta1), (float)beta2, (float)(1.0 - beta2), (float)eps, (float)wd};
    return cl_run((void* const*)g, sizes, nullptr, n, max_norm, norm, p, m, v, &hyper, work, work_bytes, (hipStream_t)stream);
}
