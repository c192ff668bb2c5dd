// Global gradient norm over a list of tensors, clipping, and the clipped AdamW update:
//     norm = sqrt(sum over all tensors of g^2);   f = min(1, max_norm / (norm + 1e-6));
//     clip:   g <- f g
//     AdamW (no bias correction, eps added to sqrt(v), weight decay on the parameter: gzsl_adamw_nobias_step's formula):
//             m <- b1 m + (1 - b1) f g;  v <- b2 v + (1 - b2) (f g)^2;  p <- p - lr (m / (sqrt(v) + eps) + wd p)
// Two launches: every workgroup of the first adds the squares of its share in 64 bits (no overflow, no order worth speaking
// of) and stores one partial sum; every workgroup of the second adds ALL partial sums in the same order, so the factor is
// the same everywhere, needs no atomics, and two runs agree bit for bit.  The tensors' addresses travel as kernel arguments:
// nothing is copied to the device and a captured graph keeps them.
#include "common.h"
#include "../../include/gzsl_hip.h"

typedef __bf16 bf16;

#define CL_TENSORS 64    // tensors of a launch
#define CL_SHARE 16384   // elements of a workgroup's share, at least
#define CL_BLOCKS 2048   // shares of a call, about

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

__global__ __launch_bounds__(256) void cl_sum_kernel(ClBatch t, double* partial) {
    __shared__ double sh[4];
    const int i = cl_find(t, blockIdx.x);
    const long long lo = (long long)(blockIdx.x - t.first[i]) * t.share, hi = lo + t.share < t.n[i] ? lo + t.share : t.n[i];
    double s = 0.0;
    if (t.half >> i & 1) {
        const bf16* g = (const bf16*)t.g[i];
        for (long long k = lo + threadIdx.x; k < hi; k += 256) s += (double)(float)g[k] * (double)(float)g[k];
    } else {
        const float* g = (const float*)t.g[i];
        for (long long k = lo + threadIdx.x; k < hi; k += 256) s += (double)g[k] * (double)g[k];
    }
    s = cl_block_sum(s, sh);
    if (threadIdx.x == 0) partial[t.base + blockIdx.x] = s;
}
__device__ __forceinline__ float cl_factor(const double* partial, int total, float max_norm, float* norm, bool write, double* sh) {
    double s = 0.0;
    for (int k = threadIdx.x; k < total; k += 256) s += partial[k];
    s = sqrt(cl_block_sum(s, sh));
    if (write && threadIdx.x == 0) *norm = (float)s;
    const double f = (double)max_norm / (s + 1e-6);
    return f < 1.0 ? (float)f : (f != f ? (float)f : 1.f);  // a norm that is no number makes every gradient one
}
__global__ __launch_bounds__(256) void cl_scale_kernel(ClBatch t, const double* partial, float max_norm, float* norm) {
    __shared__ double sh[4];
    const float f = cl_factor(partial, t.total, max_norm, norm, blockIdx.x == 0, sh);
    const int i = cl_find(t, blockIdx.x);
    const long long lo = (long long)(blockIdx.x - t.first[i]) * t.share, hi = lo + t.share < t.n[i] ? lo + t.share : t.n[i];
    if (t.half >> i & 1) {
        bf16* g = (bf16*)t.g[i];
        for (long long k = lo + threadIdx.x; k < hi; k += 256) g[k] = (bf16)((float)g[k] * f);
    } else {
        float* g = (float*)t.g[i];
        for (long long k = lo + threadIdx.x; k < hi; k += 256) g[k] *= f;
    }
}
__global__ __launch_bounds__(256) void cl_adamw_kernel(ClBatch t, ClState st, const double* partial, float max_norm, float* norm, float lr, float b1, float b2,
                                                       float eps, float wd) {
    __shared__ double sh[4];
    const float f = cl_factor(partial, t.total, max_norm, norm, blockIdx.x == 0, sh);
    const int i = cl_find(t, blockIdx.x);
    const long long lo = (long long)(blockIdx.x - t.first[i]) * t.share, hi = lo + t.share < t.n[i] ? lo + t.share : t.n[i];
    const float* g = (const float*)t.g[i];
    float *p = st.p[i], *m = st.m[i], *v = st.v[i];
    for (long long k = lo + threadIdx.x; k < hi; k += 256) {
        const float gg = g[k] * f, mm = b1 * m[k] + (1.f - b1) * gg, vv = b2 * v[k] + (1.f - b2) * gg * gg;
        m[k] = mm;
        v[k] = vv;
        float upd = mm / (sqrtf(vv) + eps);
        if (wd > 0.f) upd += wd * p[k];
        p[k] -= lr * upd;
    }
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
                  float* const* v, const float* hyper, void* work, long long work_bytes, hipStream_t st) {
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
                hipLaunchKernelGGL(cl_adamw_kernel, dim3(grid), dim3(256), 0, st, t, s, partial, max_norm, norm, hyper[0], hyper[1], hyper[2], hyper[3], hyper[4]);
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
                                    float max_norm, float lr, float beta1, float beta2, float eps, float wd, float* norm, void* work,
                                    long long work_bytes, void* stream) {
    if (int e = cl_check(sizes, n, max_norm)) return e;
    if (n > 0 && (!p || !g || !m || !v)) return GZSL_EINVAL;
    const float hyper[5] = {lr, beta1, beta2, eps, wd};
    return cl_run((void* const*)g, sizes, nullptr, n, max_norm, norm, p, m, v, hyper, work, work_bytes, (hipStream_t)stream);
}
