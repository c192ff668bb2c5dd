// Kernels and entry points of the packed label attention; the mathematics, fragments and tile images are in packed_attn.h.
#include "packed_attn.h"

// ------------------------------------------------------------------------------------------------------------- pre-pass
// One 16-byte chunk of an image row from a row of W elements (nullptr: zeros).
template <typename T>
__device__ __forceinline__ u32x4 pa_chunk(const T* row, int e0, int W) {
    constexpr int KF = 16 / sizeof(T);
    if (row == nullptr || e0 >= W) return u32x4{0, 0, 0, 0};
    const T* p = row + e0;
    if (e0 + KF <= W) {
        if (((uintptr_t)p & 15) == 0) return *reinterpret_cast<const u32x4*>(p);
        if (((uintptr_t)p & 7) == 0) {
            const u32x2 lo = reinterpret_cast<const u32x2*>(p)[0], hi = reinterpret_cast<const u32x2*>(p)[1];
            return u32x4{lo[0], lo[1], hi[0], hi[1]};
        }
    }
    T v[KF];
#pragma unroll
    for (int j = 0; j < KF; ++j) v[j] = e0 + j < W ? p[j] : (T)0.f;
    return __builtin_bit_cast(u32x4, v);
}
template <typename T>
__device__ __forceinline__ void pa_image(char* img, int pitch, const T* src, long long ld, int row0, int nrows, int W, int tid, int nt) {
    const int per = pitch / 16;
    for (int c = tid; c < PA_ROWS * per; c += nt) {
        const int r = c / per, k = c - r * per;
        const u32x4 v = pa_chunk<T>(row0 + r < nrows ? src + (long long)(row0 + r) * ld : nullptr, k * (16 / (int)sizeof(T)), W);
        *reinterpret_cast<u32x4*>(img + r * pitch + 16 * k) = v;
    }
}
// Blocks [0, B nT): key and value images of a token tile; then nQ blocks of query images.
template <typename T, class G>
__global__ __launch_bounds__(256) void pa_pack_kernel(PaArgs a) {
    const int id = blockIdx.x, nTok = a.B * a.nT;
    if (id < nTok) {
        const int b = id / a.nT, t = id % a.nT;
        const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len);
        if (t * PA_ROWS >= sp.len) return;
        char* img = a.KV + (long long)id * G::KV;
        pa_image<T>(img, G::PE, (const T*)a.keys + sp.start * a.ldk, a.ldk, t * PA_ROWS, sp.len, a.E, threadIdx.x, 256);
        pa_image<T>(img + G::EB, G::PF, (const T*)a.values + sp.start * a.ldv, a.ldv, t * PA_ROWS, sp.len, a.F, threadIdx.x, 256);
    } else {
        const int q = id - nTok;
        pa_image<T>(a.Q + (long long)q * G::EB, G::PE, (const T*)a.queries, a.ldq, q * PA_ROWS, a.L, a.E, threadIdx.x, 256);
    }
}
// Backward: dO images of (note, label tile) with lse (in units of log 2; +inf past the last label, so that P = 0 there) and
// delta[l] = <dO_l, O_l> behind the rows; eight threads a row for the sum.
template <typename T, class G>
__global__ __launch_bounds__(256) void pa_pack_do_kernel(PaArgs a) {
    const int q = blockIdx.x, b = blockIdx.y, tid = threadIdx.x;
    char* img = a.DO + ((long long)b * a.nQ + q) * G::OB;
    const T* dO = (const T*)a.dO + (long long)b * a.L * a.F;
    pa_image<T>(img, G::PF, dO, a.F, q * PA_ROWS, a.L, a.F, tid, 256);
    const int r = tid >> 3, l = q * PA_ROWS + r;
    float s = 0.f;
    if (l < a.L) {
        const T *x = dO + (long long)l * a.F, *y = (const T*)a.cO + ((long long)b * a.L + l) * a.F;
        for (int f = tid & 7; f < a.F; f += 8) s = fmaf((float)x[f], (float)y[f], s);
    }
    s += __shfl_xor(s, 1);
    s += __shfl_xor(s, 2);
    s += __shfl_xor(s, 4);
    if ((tid & 7) == 0) {
        float* aux = reinterpret_cast<float*>(img + G::FB);
        aux[r] = l < a.L ? a.cLSE[(long long)b * a.L + l] * PA_LOG2E : INFINITY;
        aux[32 + r] = s;
    }
}
// -------------------------------------------------------------------------------------------------------------- forward
// Workgroup = WAVES waves x NL x 16 labels of one note (and one share of its tokens); labels on the lane axis.
template <typename T, class G, int WAVES, int NL, bool DROP>
__global__ __launch_bounds__(WAVES * 64, 2) void pa_fwd_kernel(PaArgs a) {
    typedef typename PaTy<T>::frag frag;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int nLT = (a.L + 16 * NL * WAVES - 1) / (16 * NL * WAVES);
    const int lt = blockIdx.x % nLT, b = blockIdx.x / nLT % a.B, split = blockIdx.x / (nLT * a.B);
    const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len);
    const int tiles = (sp.len + PA_ROWS - 1) / PA_ROWS, per = (tiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(tiles, t0 + per);
    const int l0 = (lt * WAVES + wave) * 16 * NL;
    const PaCap cap = pa_cap(a.cap);

    frag qf[NL][G::SE];
    uint32_t key[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int l = min(l0 + 16 * i + n, a.nQ * PA_ROWS - 1);
        const char* row = a.Q + (long long)(l / PA_ROWS) * G::EB + (l % PA_ROWS) * G::PE + 16 * g;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) qf[i][s] = *reinterpret_cast<const frag*>(row + 64 * s);
        key[i] = gz_row_key(a.seed, GZSL_STREAM_ATTN, (uint32_t)b * a.L_total + a.l_offset + (uint32_t)(l0 + 16 * i + n));
    }
    f32x4 acc[NL][G::NF];
    float m[NL], sum[NL];
    // Capped scores lie in [-cap, cap]: up to 30 the bound itself can stand for the running maximum (e^-60 is a normal
    // number), so nothing is ever rescaled.  Otherwise a tile whose maximum exceeds m by more than 2^12 moves it.
    const float m0 = a.cap > 0.f && a.cap <= 30.f ? cap.c2 : -INFINITY;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        m[i] = m0, sum[i] = 0.f;
#pragma unroll
        for (int j = 0; j < G::NF; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const char* kv = a.KV + (long long)b * a.nT * G::KV;
    if (t0 < t1) pa_dma<WAVES>(kv + (long long)t0 * G::KV, sm, G::KV, wave, lane);
    pa_arrive();
    for (int t = t0; t < t1; ++t) {
        const char* K = sm + ((t - t0) & 1) * G::KV;
        const char* V = K + G::EB;
        if (t + 1 < t1) pa_dma<WAVES>(kv + (long long)(t + 1) * G::KV, sm + ((t - t0 + 1) & 1) * G::KV, G::KV, wave, lane);
        f32x4 s[2][NL];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < NL; ++i) s[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int k = 0; k < G::SE; ++k)
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const frag kf = pa_row<T>(K, G::PE, 16 * u, k, n, g);
#pragma unroll
                for (int i = 0; i < NL; ++i) s[u][i] = pa_mma(kf, qf[i][k], s[u][i]);
            }
        frag pf[NL][G::KS];
        const int left = sp.len - t * PA_ROWS;  // tokens of this tile
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            float y[2][4], p[2][4], mt = -INFINITY;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float th;
                    y[u][r] = a.cap > 0.f ? pa_score2<T>(s[u][i][r], cap, th) : s[u][i][r] * PA_LOG2E;
                    if (left < PA_ROWS && 16 * u + 4 * g + r >= left) y[u][r] = -INFINITY;
                    mt = fmaxf(mt, y[u][r]);
                }
            if (__any(mt > m[i] + 12.f)) {  // m is the same in the four lanes of a column
                mt = fmaxf(mt, __shfl_xor(mt, 16));
                mt = fmaxf(mt, __shfl_xor(mt, 32));
                const float mn = fmaxf(m[i], mt), alpha = mn == m[i] ? 1.f : __builtin_amdgcn_exp2f(m[i] - mn);
#pragma unroll
                for (int j = 0; j < G::NF; ++j) acc[i][j] *= alpha;
                sum[i] *= alpha;
                m[i] = mn;
            }
            const float mi = m[i] == -INFINITY ? 0.f : m[i];  // (no finite score yet: every weight is e^-inf = 0)
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[u][r] = __builtin_amdgcn_exp2f(y[u][r] - mi);
                    sum[i] += p[u][r];
                    if (DROP) p[u][r] = gz_u32(key[i], (uint32_t)(t * PA_ROWS + 16 * u + 4 * g + r)) >= a.thresh ? p[u][r] * a.scale : 0.f;
                }
#pragma unroll
            for (int k = 0; k < G::KS; ++k) pa_pack(p, k, pf[i][k]);
        }
#pragma unroll
        for (int k = 0; k < G::KS; ++k)
#pragma unroll
            for (int j = 0; j < G::NF; ++j) {
                const frag vf = pa_col<T>(V, G::PF, k * G::KK, 16 * j, n, g);
#pragma unroll
                for (int i = 0; i < NL; ++i) acc[i][j] = pa_mma(vf, pf[i][k], acc[i][j]);
            }
        pa_arrive();
    }
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int l = l0 + 16 * i + n;
        sum[i] += __shfl_xor(sum[i], 16);
        sum[i] += __shfl_xor(sum[i], 32);
        if (l >= a.L) continue;
        const long long row = (long long)b * a.L + l;
        if (a.nsplit > 1) {
            const long long pr = (long long)split * a.B * a.L + row;
            if (g == 0) a.ml[2 * pr] = m[i], a.ml[2 * pr + 1] = sum[i];
#pragma unroll
            for (int j = 0; j < G::NF; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * j + 4 * g + r < a.F) a.part[pr * a.F + 16 * j + 4 * g + r] = acc[i][j][r];
        } else {
            const float inv = sp.len > 0 ? 1.f / sum[i] : 0.f;
            if (g == 0) a.LSE[row] = sp.len > 0 ? (m[i] + __builtin_amdgcn_logf(sum[i])) * PA_LN2 : -INFINITY;
            T* out = (T*)a.O + row * a.F;
#pragma unroll
            for (int j = 0; j < G::NF; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * j + 4 * g + r < a.F) out[16 * j + 4 * g + r] = (T)(acc[i][j][r] * inv);
        }
    }
}
// Joins the token splits of a (note, label): one wave a row, splits in order.
template <typename T>
__global__ __launch_bounds__(256) void pa_join_kernel(PaArgs a) {
    const long long row = (long long)blockIdx.x * 4 + (threadIdx.x >> 6), all = (long long)a.B * a.L;
    const int lane = threadIdx.x & 63;
    if (row >= all) return;
    float M = -INFINITY, sum = 0.f;
    for (int s = 0; s < a.nsplit; ++s) {
        const float* ml = a.ml + 2 * (s * all + row);
        if (ml[1] != 0.f) M = fmaxf(M, ml[0]);  // (a share without tokens has sum 0)
    }
    float o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < a.nsplit; ++s) {
        const float* ml = a.ml + 2 * (s * all + row);
        if (ml[1] == 0.f) continue;
        const float w = __builtin_amdgcn_exp2f(ml[0] - M);
        sum = fmaf(w, ml[1], sum);
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (lane + 64 * k < a.F) o[k] = fmaf(w, a.part[(s * all + row) * a.F + lane + 64 * k], o[k]);
    }
    const float inv = sum != 0.f ? 1.f / sum : 0.f;
    if (lane == 0) a.LSE[row] = sum != 0.f ? (M + __builtin_amdgcn_logf(sum)) * PA_LN2 : -INFINITY;
#pragma unroll
    for (int k = 0; k < 4; ++k)
        if (lane + 64 * k < a.F) ((T*)a.O)[row * a.F + lane + 64 * k] = (T)(o[k] * inv);
}

// ------------------------------------------------------------------------------------------------------------- backward
// P and dS of one 32 (rows) x 16 (columns) pair of score tiles.  lse2 / delta are indexed by the label, which is the row
// (dK / dV sweep) or the column (dQ sweep).
template <typename T>
__device__ __forceinline__ void pa_grad(float s, float dp, float lse2, float delta, bool on, float keep, const PaCap& c, float& p, float& ds) {
    float th = 0.f;
    const float y = c.cap > 0.f ? pa_score2<T>(s, c, th) : s * PA_LOG2E;
    const float w = on ? __builtin_amdgcn_exp2f(y - lse2) : 0.f;
    p = w * keep;
    ds = w * (dp * keep - delta);
    if (c.cap > 0.f) ds *= fmaf(-th, th, 1.f);
    if (!on) ds = 0.f;
}

// dK / dV: workgroup = WAVES x 16 tokens of one note (token on the lane axis), sweeping its share of the labels.
template <typename T, class G, int WAVES, bool DROP>
__global__ __launch_bounds__(WAVES * 64, 2) void pa_bwd_kv_kernel(PaArgs a) {
    typedef typename PaTy<T>::frag frag;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    constexpr int BUF = G::EB + G::OB;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int nTT = (a.max_len + 16 * WAVES - 1) / (16 * WAVES);
    const int tt = blockIdx.x % nTT, b = blockIdx.x / nTT % a.B, split = blockIdx.x / (nTT * a.B);
    const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len);
    if (tt * 16 * WAVES >= sp.len) return;
    const int per = (a.nQ + a.nsplit - 1) / a.nsplit, q0 = split * per, q1 = min(a.nQ, q0 + per);
    const int tok = (tt * WAVES + wave) * 16 + n;
    const PaCap cap = pa_cap(a.cap);
    frag kf[G::SE], vf[G::SF];
    {
        const int t = min(tok, (sp.len - 1) / PA_ROWS * PA_ROWS + PA_ROWS - 1);  // inside the note's last tile image
        const char* img = a.KV + ((long long)b * a.nT + t / PA_ROWS) * G::KV + 16 * g;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) kf[s] = *reinterpret_cast<const frag*>(img + (t % PA_ROWS) * G::PE + 64 * s);
#pragma unroll
        for (int s = 0; s < G::SF; ++s) vf[s] = *reinterpret_cast<const frag*>(img + G::EB + (t % PA_ROWS) * G::PF + 64 * s);
    }
    f32x4 dv[G::NF], dk[G::NE];
#pragma unroll
    for (int j = 0; j < G::NF; ++j) dv[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < G::NE; ++j) dk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char* dO = a.DO + (long long)b * a.nQ * G::OB;
    auto fetch = [&](int q, char* buf) {
        pa_dma<WAVES>(a.Q + (long long)q * G::EB, buf, G::EB, wave, lane);
        pa_dma<WAVES>(dO + (long long)q * G::OB, buf + G::EB, G::OB, wave, lane);
    };
    if (q0 < q1) fetch(q0, sm);
    pa_arrive();
    for (int q = q0; q < q1; ++q) {
        const char* Q = sm + ((q - q0) & 1) * BUF;
        const char* D = Q + G::EB;
        const float* aux = reinterpret_cast<const float*>(D + G::FB);
        if (q + 1 < q1) fetch(q + 1, sm + ((q - q0 + 1) & 1) * BUF);
        float p[2][4], ds[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f}, dp = s;
#pragma unroll
            for (int k = 0; k < G::SE; ++k) s = pa_mma(pa_row<T>(Q, G::PE, 16 * u, k, n, g), kf[k], s);
#pragma unroll
            for (int k = 0; k < G::SF; ++k) dp = pa_mma(pa_row<T>(D, G::PF, 16 * u, k, n, g), vf[k], dp);
            const f32x4 lse = *reinterpret_cast<const f32x4*>(aux + 16 * u + 4 * g), delta = *reinterpret_cast<const f32x4*>(aux + 32 + 16 * u + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float keep = 1.f;
                if (DROP) {
                    const uint32_t l = (uint32_t)(q * PA_ROWS + 16 * u + 4 * g + r);
                    const uint32_t key = gz_row_key(a.seed, GZSL_STREAM_ATTN, (uint32_t)b * a.L_total + a.l_offset + l);
                    keep = gz_u32(key, (uint32_t)tok) >= a.thresh ? a.scale : 0.f;
                }
                pa_grad<T>(s[r], dp[r], lse[r], delta[r], true, keep, cap, p[u][r], ds[u][r]);
            }
        }
#pragma unroll
        for (int k = 0; k < G::KS; ++k) {
            frag pf, sf;
            pa_pack(p, k, pf);
            pa_pack(ds, k, sf);
#pragma unroll
            for (int j = 0; j < G::NF; ++j) dv[j] = pa_mma(pa_col<T>(D, G::PF, k * G::KK, 16 * j, n, g), pf, dv[j]);
#pragma unroll
            for (int j = 0; j < G::NE; ++j) dk[j] = pa_mma(pa_col<T>(Q, G::PE, k * G::KK, 16 * j, n, g), sf, dk[j]);
        }
        pa_arrive();
    }
    if (tok >= sp.len) return;
    const long long row = sp.start + tok;
    if (a.nsplit > 1) {
        float* out = a.dkv + ((long long)split * a.rows + row) * (a.E + a.F);
#pragma unroll
        for (int j = 0; j < G::NE; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * j + 4 * g + r < a.E) out[16 * j + 4 * g + r] = dk[j][r];
#pragma unroll
        for (int j = 0; j < G::NF; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * j + 4 * g + r < a.F) out[a.E + 16 * j + 4 * g + r] = dv[j][r];
        return;
    }
    T *ok = (T*)a.dK + row * a.E, *ov = (T*)a.dV + row * a.F;
#pragma unroll
    for (int j = 0; j < G::NE; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (16 * j + 4 * g + r < a.E) ok[16 * j + 4 * g + r] = (T)dk[j][r];
#pragma unroll
    for (int j = 0; j < G::NF; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (16 * j + 4 * g + r < a.F) ov[16 * j + 4 * g + r] = (T)dv[j][r];
}
// dK / dV from the label splits, in order.  Rows of no note are skipped (zeroed by zero_gaps_kernel).
template <typename T>
__global__ __launch_bounds__(256) void pa_kv_join_kernel(PaArgs a) {
    const int b = blockIdx.y, W = a.E + a.F;
    const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len);
    const long long all = (long long)sp.len * W, slab = a.rows * W;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long long)gridDim.x * 256) {
        const long long row = sp.start + i / W;
        const int c = (int)(i % W);
        float s = 0.f;
        for (int k = 0; k < a.nsplit; ++k) s += a.dkv[k * slab + row * W + c];
        if (c < a.E) ((T*)a.dK)[row * a.E + c] = (T)s;
        else ((T*)a.dV)[row * a.F + c - a.E] = (T)s;
    }
}

// dQ: workgroup = WAVES x NL x 16 labels (label on the lane axis) over its share of one note's tokens; a slab per share.
template <typename T, class G, int WAVES, int NL, bool DROP>
__global__ __launch_bounds__(WAVES * 64, 2) void pa_bwd_q_kernel(PaArgs a) {
    typedef typename PaTy<T>::frag frag;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int nLT = (a.L + 16 * NL * WAVES - 1) / (16 * NL * WAVES);
    const int lt = blockIdx.x % nLT, b = blockIdx.x / nLT % a.B, split = blockIdx.x / (nLT * a.B);
    const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len);
    const int tiles = (sp.len + PA_ROWS - 1) / PA_ROWS, per = (tiles + a.nsplit - 1) / a.nsplit;
    const int t0 = split * per, t1 = min(tiles, t0 + per);
    const int l0 = (lt * WAVES + wave) * 16 * NL;
    const PaCap cap = pa_cap(a.cap);
    frag qf[NL][G::SE], df[NL][G::SF];
    float lse[NL], delta[NL];
    uint32_t key[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int l = min(l0 + 16 * i + n, a.nQ * PA_ROWS - 1);
        const char* qr = a.Q + (long long)(l / PA_ROWS) * G::EB + (l % PA_ROWS) * G::PE + 16 * g;
        const char* dimg = a.DO + ((long long)b * a.nQ + l / PA_ROWS) * G::OB;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) qf[i][s] = *reinterpret_cast<const frag*>(qr + 64 * s);
#pragma unroll
        for (int s = 0; s < G::SF; ++s) df[i][s] = *reinterpret_cast<const frag*>(dimg + (l % PA_ROWS) * G::PF + 16 * g + 64 * s);
        const float* aux = reinterpret_cast<const float*>(dimg + G::FB);
        lse[i] = aux[l % PA_ROWS], delta[i] = aux[32 + l % PA_ROWS];
        key[i] = gz_row_key(a.seed, GZSL_STREAM_ATTN, (uint32_t)b * a.L_total + a.l_offset + (uint32_t)(l0 + 16 * i + n));
    }
    f32x4 dq[NL][G::NE];
#pragma unroll
    for (int i = 0; i < NL; ++i)
#pragma unroll
        for (int j = 0; j < G::NE; ++j) dq[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char* kv = a.KV + (long long)b * a.nT * G::KV;
    if (t0 < t1) pa_dma<WAVES>(kv + (long long)t0 * G::KV, sm, G::KV, wave, lane);
    pa_arrive();
    for (int t = t0; t < t1; ++t) {
        const char* K = sm + ((t - t0) & 1) * G::KV;
        const char* V = K + G::EB;
        if (t + 1 < t1) pa_dma<WAVES>(kv + (long long)(t + 1) * G::KV, sm + ((t - t0 + 1) & 1) * G::KV, G::KV, wave, lane);
        f32x4 s[2][NL], dp[2][NL];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int i = 0; i < NL; ++i) s[u][i] = dp[u][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int k = 0; k < G::SE; ++k) {
                const frag f = pa_row<T>(K, G::PE, 16 * u, k, n, g);
#pragma unroll
                for (int i = 0; i < NL; ++i) s[u][i] = pa_mma(f, qf[i][k], s[u][i]);
            }
#pragma unroll
            for (int k = 0; k < G::SF; ++k) {
                const frag f = pa_row<T>(V, G::PF, 16 * u, k, n, g);
#pragma unroll
                for (int i = 0; i < NL; ++i) dp[u][i] = pa_mma(f, df[i][k], dp[u][i]);
            }
        }
        const int left = sp.len - t * PA_ROWS;
        frag sf[NL][G::KS];
#pragma unroll
        for (int i = 0; i < NL; ++i) {
            float p, ds[2][4];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int row = 16 * u + 4 * g + r;
                    float keep = 1.f;
                    if (DROP) keep = gz_u32(key[i], (uint32_t)(t * PA_ROWS + row)) >= a.thresh ? a.scale : 0.f;
                    pa_grad<T>(s[u][i][r], dp[u][i][r], lse[i], delta[i], row < left, keep, cap, p, ds[u][r]);
                }
#pragma unroll
            for (int k = 0; k < G::KS; ++k) pa_pack(ds, k, sf[i][k]);
        }
#pragma unroll
        for (int k = 0; k < G::KS; ++k)
#pragma unroll
            for (int j = 0; j < G::NE; ++j) {
                const frag f = pa_col<T>(K, G::PE, k * G::KK, 16 * j, n, g);
#pragma unroll
                for (int i = 0; i < NL; ++i) dq[i][j] = pa_mma(f, sf[i][k], dq[i][j]);
            }
        pa_arrive();
    }
    float* slab = a.dq + ((long long)split * a.B + b) * a.L * a.E;
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int l = l0 + 16 * i + n;
        if (l >= a.L) continue;
#pragma unroll
        for (int j = 0; j < G::NE; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * j + 4 * g + r < a.E) slab[(long long)l * a.E + 16 * j + 4 * g + r] = dq[i][j][r];
    }
}
// dQ = sum of the slabs, in order.
template <typename T>
__global__ __launch_bounds__(256) void pa_q_join_kernel(const float* slab, T* out, long long n, int nslab) {
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = 0.f;
        for (int k = 0; k < nslab; ++k) s += slab[k * n + i];
        out[i] = (T)s;
    }
}

// ---------------------------------------------------------------------------------------------------------------- launch
static inline long long up256(long long n) { return (n + 255) / 256 * 256; }

struct PaPlan {
    int nT, nQ, wide;              // wide: E > 112
    int fs, qs, ks;                // forward token splits, dQ token splits, dK / dV label splits
    long long kv, q, dO, part, ml, dq, dkv, bytes;
};
#define PA_LABELS 128  // labels (forward, dQ) or tokens (dK / dV) of a workgroup, both types

template <class G>
static void pa_sizes(PaPlan& p, const GzslPackedAttn& d, int backward) {
    p.kv = up256((long long)d.B * p.nT * G::KV);
    p.q = up256((long long)p.nQ * G::EB);
    p.dO = backward ? up256((long long)d.B * p.nQ * G::OB) : 0;
}
// Shares of an axis: enough workgroups for two rounds of 256 compute units, eight tiles a share at least.
static int pa_splits(long long wgs, int tiles, int least) {
    long long s = wgs > 0 ? 512 / wgs : 1;
    if (s > tiles / least) s = tiles / least;
    return (int)(s < 1 ? 1 : (s > 256 ? 256 : s));
}
static int pa_plan(const GzslPackedAttn* d, int backward, PaPlan& p) {
    if (!d || d->B < 0 || d->rows < 0 || d->max_len < 0 || d->L < 0 || d->E < 1 || d->F < 1 || d->E > 208 || d->F > 208) return GZSL_EINVAL;
    if (d->dtype != GZSL_F32 && d->dtype != GZSL_BF16) return GZSL_EINVAL;
    if (!(d->cap >= 0.f) || d->cap > 1e30f) return GZSL_EINVAL;
    if (d->ldk < d->E || d->ldv < d->F || d->ldq < d->E) return GZSL_EINVAL;
    p = PaPlan{};
    p.nT = (int)(((long long)d->max_len + PA_ROWS - 1) / PA_ROWS), p.nQ = (int)(((long long)d->L + PA_ROWS - 1) / PA_ROWS);
    p.wide = d->E > 112;
    const long long nLT = cdiv(d->L, PA_LABELS), nTT = cdiv(d->max_len, PA_LABELS);
    if ((long long)d->B * (p.nT + 1) + p.nQ > 0x3FFFFFFF || (long long)d->B * (nLT + nTT + 1) > 0x3FFFFFFF || d->B > 65534 || p.nQ > 0x3FFFFFFF) return GZSL_ETOOBIG;
    p.fs = pa_splits(d->B * nLT, p.nT, 8);
    p.qs = pa_splits(d->B * nLT, p.nT, 8);
    p.ks = pa_splits(d->B * nTT, p.nQ, 4);
    if (d->dtype == GZSL_F32) p.wide ? pa_sizes<PaGeo<float, 13, 13>>(p, *d, backward) : pa_sizes<PaGeo<float, 7, 13>>(p, *d, backward);
    else p.wide ? pa_sizes<PaGeo<bf16, 13, 13>>(p, *d, backward) : pa_sizes<PaGeo<bf16, 7, 13>>(p, *d, backward);
    if (!backward && p.fs > 1) {
        p.part = up256(4LL * p.fs * d->B * d->L * d->F);
        p.ml = up256(8LL * p.fs * d->B * d->L);
    }
    if (backward) {
        p.dq = up256(4LL * p.qs * d->B * d->L * d->E);
        if (p.ks > 1) p.dkv = up256(4LL * p.ks * d->rows * (d->E + d->F));
    }
    p.bytes = p.kv + p.q + p.dO + p.part + p.ml + p.dq + p.dkv;
    return 0;
}
static void pa_fill(PaArgs& a, const GzslPackedAttn& d, const PaPlan& p, void* work) {
    a.keys = d.keys, a.values = d.values, a.queries = d.queries, a.spans = d.spans;
    a.rows = d.rows, a.ldk = d.ldk, a.ldv = d.ldv, a.ldq = d.ldq;
    a.B = d.B, a.max_len = d.max_len, a.L = d.L, a.E = d.E, a.F = d.F, a.nT = p.nT, a.nQ = p.nQ;
    a.cap = d.cap, a.l_offset = (uint32_t)d.l_offset, a.L_total = (uint32_t)d.L_total, a.seed = d.seed, a.thresh = d.drop_thresh, a.scale = d.drop_scale;
    char* w = (char*)work;
    a.KV = w, w += p.kv;
    a.Q = w, w += p.q;
    a.DO = w, w += p.dO;
    a.part = (float*)w, w += p.part;
    a.ml = (float*)w, w += p.ml;
    a.dq = (float*)w, w += p.dq;
    a.dkv = (float*)w;
}
template <typename T>
struct PaCfg;
template <>
struct PaCfg<float> {
    static constexpr int WAVES = 8, NL = 1;
};
template <>
struct PaCfg<bf16> {
    static constexpr int WAVES = 4, NL = 2;
};

template <typename T, class G, bool DROP>
static int pa_fwd(PaArgs& a, const PaPlan& p, hipStream_t st) {
    constexpr int W = PaCfg<T>::WAVES, NL = PaCfg<T>::NL;
    static_assert(W * NL * 16 == PA_LABELS, "labels of a workgroup");
    auto k = pa_fwd_kernel<T, G, W, NL, DROP>;
    const int lds = 2 * G::KV;
    a.nsplit = p.fs;
    hipLaunchKernelGGL((pa_pack_kernel<T, G>), dim3(a.B * a.nT + a.nQ), dim3(256), 0, st, a);
    hipLaunchKernelGGL(k, dim3(cdiv(a.L, PA_LABELS) * a.B * p.fs), dim3(W * 64), lds, st, a);
    if (p.fs > 1) hipLaunchKernelGGL(pa_join_kernel<T>, dim3(cdiv((long)a.B * a.L, 4)), dim3(256), 0, st, a);
    GZSL_CHECK_LAUNCH();
    return 0;
}
template <typename T, class G, bool DROP>
static int pa_bwd(PaArgs& a, const PaPlan& p, hipStream_t st) {
    constexpr int W = PaCfg<T>::WAVES, NL = PaCfg<T>::NL, WK = PA_LABELS / 16;
    auto kk = pa_bwd_kv_kernel<T, G, WK, DROP>;
    auto kq = pa_bwd_q_kernel<T, G, W, NL, DROP>;
    const int lk = 2 * (G::EB + G::OB), lq = 2 * G::KV;
    hipLaunchKernelGGL((pa_pack_kernel<T, G>), dim3(a.B * a.nT + a.nQ), dim3(256), 0, st, a);
    hipLaunchKernelGGL((pa_pack_do_kernel<T, G>), dim3(a.nQ, a.B), dim3(256), 0, st, a);
    if (a.nT > 0) {
        a.nsplit = p.ks;
        hipLaunchKernelGGL(kk, dim3(cdiv(a.max_len, PA_LABELS) * a.B * p.ks), dim3(WK * 64), lk, st, a);
        if (p.ks > 1) hipLaunchKernelGGL(pa_kv_join_kernel<T>, dim3(cdiv((long)a.max_len * (a.E + a.F), 1024), a.B), dim3(256), 0, st, a);
    }
    hipLaunchKernelGGL(zero_gaps_kernel<T>, dim3(16, a.B + 1), dim3(256), 0, st, a.spans, a.rows, a.B, a.max_len, (T*)a.dK, a.E, (T*)a.dV, a.F);
    a.nsplit = p.qs;
    hipLaunchKernelGGL(kq, dim3(cdiv(a.L, PA_LABELS) * a.B * p.qs), dim3(W * 64), lq, st, a);
    const long long n = (long long)a.L * a.E;
    hipLaunchKernelGGL(pa_q_join_kernel<T>, dim3((unsigned)(n < 256 * 4096 ? cdiv((long)n, 256) : 4096)), dim3(256), 0, st, a.dq, (T*)a.dQ, n, p.qs * a.B);
    GZSL_CHECK_LAUNCH();
    return 0;
}
template <typename T, class G>
static int pa_go(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    if (backward) return a.thresh ? pa_bwd<T, G, true>(a, p, st) : pa_bwd<T, G, false>(a, p, st);
    return a.thresh ? pa_fwd<T, G, true>(a, p, st) : pa_fwd<T, G, false>(a, p, st);
}
static int pa_run(const GzslPackedAttn& d, PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    if (d.dtype == GZSL_F32) return p.wide ? pa_go<float, PaGeo<float, 13, 13>>(a, p, backward, st) : pa_go<float, PaGeo<float, 7, 13>>(a, p, backward, st);
    return p.wide ? pa_go<bf16, PaGeo<bf16, 13, 13>>(a, p, backward, st) : pa_go<bf16, PaGeo<bf16, 7, 13>>(a, p, backward, st);
}

extern "C" long long gzsl_packed_attn_work_bytes(const GzslPackedAttn* d, int backward) {
    PaPlan p;
    return pa_plan(d, backward, p) ? -1 : p.bytes;
}

extern "C" int gzsl_packed_attn_fwd(const GzslPackedAttn* d, void* O, float* LSE, void* work, long long work_bytes, void* stream) {
    PaPlan p;
    if (int e = pa_plan(d, 0, p)) return e;
    if (d->B == 0 || d->L == 0) return 0;
    if (!O || !LSE || !d->spans || !d->queries || (d->rows > 0 && (!d->keys || !d->values)) || work_bytes < p.bytes || !work || ((uintptr_t)work & 15)) return GZSL_EINVAL;
    PaArgs a{};
    pa_fill(a, *d, p, work);
    a.O = O, a.LSE = LSE;
    return pa_run(*d, a, p, false, (hipStream_t)stream);
}

extern "C" int gzsl_packed_attn_bwd(const GzslPackedAttn* d, const void* O, const float* LSE, const void* dO, void* dkeys, void* dvalues, void* dqueries,
                                    void* work, long long work_bytes, void* stream) {
    PaPlan p;
    if (int e = pa_plan(d, 1, p)) return e;
    if (d->L == 0 && d->rows == 0) return 0;
    if (d->B == 0 || d->L == 0) return GZSL_EINVAL;  // nothing was attended: the gradients are the caller's zeros
    if (!O || !LSE || !dO || !dqueries || !d->spans || !d->queries || (d->rows > 0 && (!d->keys || !d->values || !dkeys || !dvalues)) || work_bytes < p.bytes || !work ||
        ((uintptr_t)work & 15))
        return GZSL_EINVAL;
    PaArgs a{};
    pa_fill(a, *d, p, work);
    a.cO = O, a.cLSE = LSE, a.dO = dO, a.dK = dkeys, a.dV = dvalues, a.dQ = dqueries;
    return pa_run(*d, a, p, true, (hipStream_t)stream);
}
