// Gated linear recurrence over packed notes, forward and backward, and its single-token step:
//     z = sigmoid(g);   h_t = (1 - z_t) h_{t-1} + z_t c_t          (t runs through a note's rows, or back through them)
//     backward:  lam_t = dh_t + (1 - z_{t+1}) lam_{t+1};   dc = lam z;   dg = lam (c - h_{t-1}) z (1 - z);   dh_0 = (1 - z_1) lam_1
// The states are fp32 throughout; tensors of 16 bits are widened when read and rounded once when written.
#include "packed.h"
#include "../../include/gzsl_hip.h"

struct GsArgs {
    const void *g, *c;
    const int64_t* spans;
    const float* h0;
    long long rows, ldg, ldc;
    int B, max_len, H, reverse;
    void* h;
    float* last;
    const void *ch, *dh;
    const float* dlast;
    void *dg, *dc;
    float* dh0;
};

// z = sigmoid(g) and a = 1 - z = sigmoid(-g), both to full relative accuracy (e^-|g| never overflows)
__device__ __forceinline__ void gs_gate(float g, float& z, float& a) {
    const float e = expf(-fabsf(g)), big = 1.f / (1.f + e), small = e * big;
    z = g >= 0.f ? big : small;
    a = g >= 0.f ? small : big;
    if (g != g) z = a = g;
}

// one thread per (note, channel)
template <typename T>
__global__ __launch_bounds__(64) void gs_fwd_kernel(GsArgs a) {
    const int ch = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (ch >= a.H) return;
    const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len);
    const T *g = (const T*)a.g + ch, *c = (const T*)a.c + ch;
    T* out = (T*)a.h + ch;
    float h = a.h0 ? a.h0[(long long)b * a.H + ch] : 0.f;
    for (int t = 0; t < sp.len; ++t) {
        const long long row = sp.start + (a.reverse ? sp.len - 1 - t : t);
        float z, k;
        gs_gate((float)g[row * a.ldg], z, k);
        h = fmaf(k, h, z * (float)c[row * a.ldc]);
        out[row * a.H] = (T)h;
    }
    a.last[(long long)b * a.H + ch] = h;
}

template <typename T>
__global__ __launch_bounds__(64) void gs_bwd_kernel(GsArgs a) {
    const int ch = blockIdx.x * 64 + threadIdx.x, b = blockIdx.y;
    if (ch >= a.H) return;
    const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len);
    const T *g = (const T*)a.g + ch, *c = (const T*)a.c + ch, *h = (const T*)a.ch + ch, *dh = (const T*)a.dh + ch;
    T *dg = (T*)a.dg + ch, *dc = (T*)a.dc + ch;
    const long long at = (long long)b * a.H + ch;
    const float h0 = a.h0 ? a.h0[at] : 0.f;
    float carry = a.dlast ? a.dlast[at] : 0.f;
    for (int t = sp.len - 1; t >= 0; --t) {
        const long long row = sp.start + (a.reverse ? sp.len - 1 - t : t), prev = a.reverse ? row + 1 : row - 1;
        float z, k;
        gs_gate((float)g[row * a.ldg], z, k);
        const float lam = carry + (a.dh ? (float)dh[row * a.H] : 0.f), before = t > 0 ? (float)h[prev * a.H] : h0;
        dc[row * a.H] = (T)(lam * z);
        dg[row * a.H] = (T)(lam * ((float)c[row * a.ldc] - before) * (z * k));
        carry = lam * k;
    }
    if (a.dh0) a.dh0[at] = carry;
}

template <typename T>
__global__ __launch_bounds__(256) void gs_step_kernel(const T* g, const T* c, float* state, const uint8_t* active, int H, long long ldg, long long ldc, long long n) {
    const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const long long b = i / H;
    const int ch = (int)(i - b * H);
    if (active && !active[b]) return;
    float z, k;
    gs_gate((float)g[b * ldg + ch], z, k);
    state[i] = fmaf(k, state[i], z * (float)c[b * ldc + ch]);
}

static int gs_check(const GzslGatedScan* d) {
    if (!d || d->B < 0 || d->rows < 0 || d->max_len < 0 || d->H < 1 || d->ldg < d->H || d->ldc < d->H) return GZSL_EINVAL;
    if (d->dtype != GZSL_F32 && d->dtype != GZSL_BF16) return GZSL_EINVAL;
    if (d->B > 65534) return GZSL_ETOOBIG;
    if (d->B > 0 && !d->spans) return GZSL_EINVAL;
    if (d->rows > 0 && (!d->gates || !d->cands)) return GZSL_EINVAL;
    return 0;
}
static GsArgs gs_args(const GzslGatedScan& d) {
    GsArgs a{};
    a.g = d.gates, a.c = d.cands, a.spans = d.spans, a.h0 = d.h0, a.rows = d.rows, a.ldg = d.ldg, a.ldc = d.ldc;
    a.B = d.B, a.max_len = d.max_len, a.H = d.H, a.reverse = d.reverse;
    return a;
}

template <typename T>
static int gs_fwd(const GsArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(gs_fwd_kernel<T>, dim3(cdiv(a.H, 64), a.B), dim3(64), 0, st, a);
    hipLaunchKernelGGL(zero_gaps_kernel<T>, dim3(16, a.B + 1), dim3(256), 0, st, a.spans, a.rows, a.B, a.max_len, (T*)a.h, a.H, (T*)nullptr, 0);
    GZSL_CHECK_LAUNCH();
    return 0;
}
template <typename T>
static int gs_bwd(const GsArgs& a, hipStream_t st) {
    hipLaunchKernelGGL(gs_bwd_kernel<T>, dim3(cdiv(a.H, 64), a.B), dim3(64), 0, st, a);
    hipLaunchKernelGGL(zero_gaps_kernel<T>, dim3(16, a.B + 1), dim3(256), 0, st, a.spans, a.rows, a.B, a.max_len, (T*)a.dg, a.H, (T*)a.dc, a.H);
    GZSL_CHECK_LAUNCH();
    return 0;
}

extern "C" long long gzsl_gated_scan_work_bytes(const GzslGatedScan* d, int backward) {
    (void)backward;
    return gs_check(d) ? -1 : 0;
}

extern "C" int gzsl_gated_scan_fwd(const GzslGatedScan* d, void* h, float* h_last, void* work, long long work_bytes, void* stream) {
    (void)work, (void)work_bytes;
    if (int e = gs_check(d)) return e;
    if (d->B == 0) return d->rows == 0 ? 0 : GZSL_EINVAL;
    if (!h_last || (d->rows > 0 && !h)) return GZSL_EINVAL;
    GsArgs a = gs_args(*d);
    a.h = h, a.last = h_last;
    return d->dtype == GZSL_F32 ? gs_fwd<float>(a, (hipStream_t)stream) : gs_fwd<bf16>(a, (hipStream_t)stream);
}

extern "C" int gzsl_gated_scan_bwd(const GzslGatedScan* d, const void* h, const void* dh, const float* dlast, void* dgates, void* dcands, float* dh0,
                                   void* work, long long work_bytes, void* stream) {
    (void)work, (void)work_bytes;
    if (int e = gs_check(d)) return e;
    if (d->B == 0) return d->rows == 0 ? 0 : GZSL_EINVAL;
    if (d->rows > 0 && (!h || !dgates || !dcands)) return GZSL_EINVAL;
    GsArgs a = gs_args(*d);
    a.ch = h, a.dh = dh, a.dlast = dlast, a.dg = dgates, a.dc = dcands, a.dh0 = dh0;
    return d->dtype == GZSL_F32 ? gs_bwd<float>(a, (hipStream_t)stream) : gs_bwd<bf16>(a, (hipStream_t)stream);
}

extern "C" int gzsl_gated_scan_step(const void* gates, const void* cands, float* state, const uint8_t* active, int B, int H, long long ldg,
                                    long long ldc, int dtype, void* stream) {
    if (B < 0 || H < 1 || ldg < H || ldc < H || (dtype != GZSL_F32 && dtype != GZSL_BF16)) return GZSL_EINVAL;
    if (B == 0) return 0;
    if (!gates || !cands || !state) return GZSL_EINVAL;
    const long long n = (long long)B * H;
    if (n > 0x7FFFFFFFLL * 128) return GZSL_ETOOBIG;
    const dim3 grid((unsigned)((n + 255) / 256));
    if (dtype == GZSL_F32)
        hipLaunchKernelGGL(gs_step_kernel<float>, grid, dim3(256), 0, (hipStream_t)stream, (const float*)gates, (const float*)cands, state, active, H, ldg, ldc, n);
    else
        hipLaunchKernelGGL(gs_step_kernel<bf16>, grid, dim3(256), 0, (hipStream_t)stream, (const bf16*)gates, (const bf16*)cands, state, active, H, ldg, ldc, n);
    GZSL_CHECK_LAUNCH();
    return 0;
}
