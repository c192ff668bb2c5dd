// Kernels of the packed label attention, instantiated for fp32 in packed_attn_f32.hip and for bf16 in packed_attn_bf16.hip; the
// mathematics, the fragments, the tile images and the cut of the work are in packed_attn.h.
#pragma once
#include <type_traits>
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
template <typename T, int ROWS>
__device__ __forceinline__ void pa_image(char* img, int pitch, const T* src, long long ld, int row0, int nrows, int W, int tid, int nt) {
    const int per = pitch / 16;
    for (int c = tid; c < ROWS * per; c += nt) {
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
        if (t * G::ROWS >= sp.len) return;
        char* img = a.KV + (long long)id * G::KV;
        pa_image<T, G::ROWS>(img, G::PE, (const T*)a.keys + sp.start * a.ldk, a.ldk, t * G::ROWS, sp.len, a.E, threadIdx.x, 256);
        pa_image<T, G::ROWS>(img + G::EB, G::PF, (const T*)a.values + sp.start * a.ldv, a.ldv, t * G::ROWS, sp.len, a.F, threadIdx.x, 256);
    } else {
        const int q = id - nTok;
        pa_image<T, G::ROWS>(a.Q + (long long)q * G::QB, G::PE, (const T*)a.queries, a.ldq, q * G::ROWS, a.L, a.E, threadIdx.x, 256);
    }
}
// Backward: dO images of (note, label tile); behind the rows, for each label, off and scale of its weights
// P = exp2(y - off) * scale (from the forward's own maximum and sum; from LSE where the caller has only that; scale 0 past the
// last label) and delta = <dO_l, O_l> (with what the rounding of O dropped, where it is known).  `TPR` threads a row.
template <typename T, class G>
__global__ __launch_bounds__(256) void pa_pack_do_kernel(PaArgs a) {
    constexpr int TPR = 256 / G::ROWS;
    const int q = blockIdx.x % a.nQ, b = blockIdx.x / a.nQ, tid = threadIdx.x;
    char* img = a.DO + ((long long)b * a.nQ + q) * G::OB;
    const T* dO = (const T*)a.dO + (long long)b * a.L * a.F;
    pa_image<T, G::ROWS>(img, G::PF, dO, a.F, q * G::ROWS, a.L, a.F, tid, 256);
    const int r = tid / TPR, l = q * G::ROWS + r;
    const long long row = (long long)b * a.L + l;
    float s = 0.f;
    if (l < a.L) {
        const T *x = dO + (long long)l * a.F, *y = (const T*)a.cO + row * a.F;
        const bf16* low = sizeof(T) == 2 && a.crest ? reinterpret_cast<const bf16*>(a.crest + 2LL * a.B * a.L) + row * a.F : nullptr;
        for (int f = tid % TPR; f < a.F; f += TPR) s = fmaf((float)x[f], (float)y[f] + (low ? (float)low[f] : 0.f), s);
    }
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) s += __shfl_xor(s, o);
    if (tid % TPR == 0) {
        float* aux = reinterpret_cast<float*>(img + G::FB);
        float off = 0.f, scale = 0.f;
        if (l < a.L) {
            if (a.crest) off = a.crest[2 * row], scale = a.crest[2 * row + 1];
            else off = a.cLSE[row] * PA_LOG2E, scale = 1.f;
        }
        aux[r] = off;
        aux[G::ROWS + r] = scale;
        aux[2 * G::ROWS + r] = s;
    }
}

// Four consecutive values of an output row, and what rounding them dropped.
template <typename T>
__device__ __forceinline__ void pa_out(const f32x4& v, T* row, bf16* low, int c, int W) {
    if (c >= W) return;
    T* p = row + c;
    if (c + 4 <= W && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0) {
        typedef T vec __attribute__((ext_vector_type(4)));
        vec x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = (T)v[r];
        *reinterpret_cast<vec*>(p) = x;
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (c + r < W) p[r] = (T)v[r];
    }
    if (sizeof(T) == 2 && low) {
        bf16* q = low + c;
        bf16x4 x;
#pragma unroll
        for (int r = 0; r < 4; ++r) x[r] = (bf16)(v[r] - (float)(T)v[r]);
        if (c + 4 <= W && ((uintptr_t)q & 7) == 0) {
            *reinterpret_cast<bf16x4*>(q) = x;
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (c + r < W) q[r] = x[r];
        }
    }
}

// -------------------------------------------------------------------------------------------------------------- forward
// Workgroup = WAVES x 16 labels of one note (or of one chunk of it); labels on the lane axis.
template <typename T, class G, int WAVES, bool CAP, bool DROP>
__global__ __launch_bounds__(WAVES * 64, (sizeof(T) == 2 && G::NE == 7) ? 4 : (sizeof(T) == 2 ? 3 : 2)) void pa_fwd_kernel(PaArgs a) {
    typedef typename PaTy<T>::frag frag;
    constexpr int U = G::U;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int lt = blockIdx.x % a.nLT;
    const PaUnit un = pa_unit<G::ROWS>(a, blockIdx.x / a.nLT);
    if (un.ci >= un.all) return;
    const int b = un.b, len = un.sp.len;
    const int t0 = un.c * (un.chunk / G::ROWS), t1 = (int)min((long long)(len + G::ROWS - 1) / G::ROWS, (long long)t0 + un.chunk / G::ROWS);
    const int l0 = (lt * WAVES + wave) * 16;
    const PaCap cap = pa_cap(a.cap);

    frag qf[G::SE];
    {
        const int l = min(l0 + n, a.nQ * G::ROWS - 1);
        const char* row = a.Q + (long long)(l / G::ROWS) * G::QB + (l % G::ROWS) * G::PE + 16 * g;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) qf[s] = *reinterpret_cast<const frag*>(row + 64 * s);
    }
    const uint32_t key = gz_row_key(a.seed, GZSL_STREAM_ATTN, (uint32_t)b * a.L_total + a.l_offset + (uint32_t)(l0 + n));
    f32x4 acc[G::NF];
#pragma unroll
    for (int j = 0; j < G::NF; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    // Scores capped at 30 lie within 2^+-44: their exponentials and sums are plain fp32 numbers without a maximum taken off, and
    // nothing is ever rescaled.  Otherwise a tile whose maximum exceeds the running one by more than 2^12 moves it.
    const bool fixed = CAP && a.cap <= 30.f;
    float m = fixed ? 0.f : -INFINITY, sum = 0.f;
    const char* kv = a.KV + (long long)b * a.nT * G::KV;
    if (t0 < t1) pa_dma<WAVES>(kv + (long long)t0 * G::KV, sm, G::KV, wave, lane);
    pa_arrive();
    auto step = [&](int t, auto last) {  // last: the tile may end behind the note
        const char* K = sm + ((t - t0) & 1) * G::KV;
        const char* V = K + G::EB;
        if (t + 1 < t1) pa_dma<WAVES>(kv + (long long)(t + 1) * G::KV, sm + ((t - t0 + 1) & 1) * G::KV, G::KV, wave, lane);
        f32x4 s[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < G::SE; ++k) s[u] = pa_mma(pa_row<T>(K, G::PE, 16 * u, k, n, g), qf[k], s[u]);
        }
        float y[U][4], th[U][4];
        pa_scores<T, CAP, U, false>(s, cap, y, th);
        if constexpr (decltype(last)::value) {
            const int left = len - t * G::ROWS;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * u + 4 * g + r >= left) y[u][r] = -INFINITY;
        }
        if (!fixed) {
            float mt = -INFINITY;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) mt = fmaxf(mt, y[u][r]);
            if (__any(mt > m + 12.f)) {  // m is the same in the four lanes of a column
                mt = fmaxf(mt, __shfl_xor(mt, 16));
                mt = fmaxf(mt, __shfl_xor(mt, 32));
                const float mn = fmaxf(m, mt), alpha = mn == m ? 1.f : __builtin_amdgcn_exp2f(m - mn);
#pragma unroll
                for (int j = 0; j < G::NF; ++j) acc[j] *= alpha;
                sum *= alpha;
                m = mn;
            }
            const float mi = m == -INFINITY ? 0.f : m;  // (no finite score yet: every weight is 2^-inf = 0)
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) y[u][r] -= mi;
        }
        frag pf;
        {
            float p[U][4];
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[u][r] = __builtin_amdgcn_exp2f(y[u][r]);
                    sum += p[u][r];
                    if (DROP) p[u][r] = gz_u32(key, (uint32_t)(t * G::ROWS + 16 * u + 4 * g + r)) >= a.thresh ? p[u][r] * a.scale : 0.f;
                }
            pa_pack(p, pf);
        }
#pragma unroll
        for (int j = 0; j < G::NF; ++j) acc[j] = pa_mma(pa_col<T>(V, G::PF, 0, 16 * j, n, g), pf, acc[j]);
        pa_arrive();
    };
    for (int t = t0; t < t1 - 1; ++t) step(t, std::false_type{});
    if (t0 < t1) step(t1 - 1, std::true_type{});
    const int l = l0 + n;
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (l >= a.L) return;
    const long long row = (long long)b * a.L + l;
    if (un.nch > 1) {
        const long long pr = (long long)un.ci * a.L + l;
        if (g == 0) a.ml[2 * pr] = m, a.ml[2 * pr + 1] = sum;
#pragma unroll
        for (int j = 0; j < G::NF; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * j + 4 * g + r < a.F) a.part[pr * a.F + 16 * j + 4 * g + r] = acc[j][r];
        return;
    }
    const float inv = len > 0 ? 1.f / sum : 0.f;
    if (g == 0) {
        a.LSE[row] = len > 0 ? (m + __builtin_amdgcn_logf(sum)) * PA_LN2 : -INFINITY;
        if (a.rest) a.rest[2 * row] = m, a.rest[2 * row + 1] = inv;
    }
    T* out = (T*)a.O + row * a.F;
    bf16* low = sizeof(T) == 2 && a.rest ? reinterpret_cast<bf16*>(a.rest + 2LL * a.B * a.L) + row * a.F : nullptr;
#pragma unroll
    for (int j = 0; j < G::NF; ++j) pa_out<T>(acc[j] * inv, out, low, 16 * j + 4 * g, a.F);
}
// Joins the chunks of a (note, label), in order.  G waves share a row's chunks (few rows over many chunks) and meet in LDS; a row
// is 64 lanes over the widths.
template <typename T, int ROWS, int G>
__global__ __launch_bounds__(256) void pa_join_kernel(PaArgs a) {
    __shared__ float so[4][256], ss[4], sM[4];
    constexpr int R = 4 / G;  // rows of a workgroup
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, part = w % G, nb = (a.L + R - 1) / R;
    const int l = blockIdx.x % nb * R + w / G;
    const PaUnit un = pa_unit<ROWS>(a, 0, blockIdx.x / nb);
    if (un.nch == 1) return;
    const bool on = l < a.L;
    const int per = (un.nch + G - 1) / G, c0 = on ? part * per : 0, c1 = on ? min(un.nch, c0 + per) : 0;
    float M = -INFINITY;
    for (int c = c0 + lane; c < c1; c += 64) {
        const float* ml = a.ml + 2 * ((long long)(un.ci + c) * a.L + l);
        if (ml[1] != 0.f) M = fmaxf(M, ml[0]);  // (no finite score in this chunk: sum 0)
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    if (G > 1) {
        if (lane == 0) sM[w] = M;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < G; ++k) M = fmaxf(M, sM[w - part + k]);
    }
    float sum = 0.f, o4[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int c = c0; c < c1; ++c) {
        const long long pr = (long long)(un.ci + c) * a.L + l;
        const float s = a.ml[2 * pr + 1], f = s != 0.f ? __builtin_amdgcn_exp2f(a.ml[2 * pr] - M) : 0.f;
        sum = fmaf(f, s, sum);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const float x = lane + 64 * k < a.F ? a.part[pr * a.F + lane + 64 * k] : 0.f;
            o4[k] = f != 0.f ? fmaf(f, x, o4[k]) : o4[k];
        }
    }
    if (G > 1) {
#pragma unroll
        for (int k = 0; k < 4; ++k) so[w][lane + 64 * k] = o4[k];
        if (lane == 0) ss[w] = sum;
        __syncthreads();
        if (part > 0) return;
        for (int q = 1; q < G; ++q) {
            sum += ss[w + q];
#pragma unroll
            for (int k = 0; k < 4; ++k) o4[k] += so[w + q][lane + 64 * k];
        }
    }
    if (!on) return;
    const long long row = (long long)un.b * a.L + l;
    const float inv = 1.f / sum;
    if (lane == 0) {
        a.LSE[row] = (M + __builtin_amdgcn_logf(sum)) * PA_LN2;
        if (a.rest) a.rest[2 * row] = M, a.rest[2 * row + 1] = inv;
    }
    bf16* low = sizeof(T) == 2 && a.rest ? reinterpret_cast<bf16*>(a.rest + 2LL * a.B * a.L) + row * a.F : nullptr;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        const int f = lane + 64 * k;
        if (f >= a.F) continue;
        const float o = o4[k] * inv;
        const T r = (T)o;
        ((T*)a.O)[row * a.F + f] = r;
        if (low) low[f] = (bf16)(o - (float)r);
    }
}

// ------------------------------------------------------------------------------------------------------------- backward
// P and dS of a tile: weights w = exp2(y - off) * scale, dropout factor keep.
template <bool CAP>
__device__ __forceinline__ void pa_grad(float y, float th, float dp, float off, float scale, float delta, float keep, float& p, float& ds) {
    const float w = __builtin_amdgcn_exp2f(y - off) * scale;
    p = w * keep;
    ds = w * fmaf(dp, keep, -delta);
    if (CAP) ds *= fmaf(-th, th, 1.f);
}

// dK / dV: workgroup = 64 tokens of one note (16 a wave, tokens on the lane axis), sweeping its share of the labels.
template <typename T, class G, bool CAP, bool DROP>
__global__ __launch_bounds__(256, 2) void pa_bwd_kv_kernel(PaArgs a) {
    typedef typename PaTy<T>::frag frag;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    constexpr int BUF = G::QB + G::OB, WAVES = PA_TILE / 16, U = G::U;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const PaTileUnit un = pa_tile_unit(a, blockIdx.x);
    if (un.b < 0) return;
    const int b = un.b, len = un.sp.len;
    const int per = (a.nQ + un.shares - 1) / un.shares, q0 = un.share * per, q1 = min(a.nQ, q0 + per);
    const int tok = (un.tile * WAVES + wave) * 16 + n;
    const PaCap cap = pa_cap(a.cap);
    frag kf[G::SE], vf[G::SF];
    {
        const int t = min(tok, (len - 1) / G::ROWS * G::ROWS + G::ROWS - 1);  // inside the note's last tile image
        const char* img = a.KV + ((long long)b * a.nT + t / G::ROWS) * G::KV + 16 * g;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) kf[s] = *reinterpret_cast<const frag*>(img + (t % G::ROWS) * G::PE + 64 * s);
#pragma unroll
        for (int s = 0; s < G::SF; ++s) vf[s] = *reinterpret_cast<const frag*>(img + G::EB + (t % G::ROWS) * G::PF + 64 * s);
    }
    f32x4 dv[G::NF], dk[G::NE];
#pragma unroll
    for (int j = 0; j < G::NF; ++j) dv[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < G::NE; ++j) dk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char* dO = a.DO + (long long)b * a.nQ * G::OB;
    auto fetch = [&](int q, char* buf) {
        pa_dma<WAVES>(a.Q + (long long)q * G::QB, buf, G::QB, wave, lane);
        pa_dma<WAVES>(dO + (long long)q * G::OB, buf + G::QB, G::OB, wave, lane);
    };
    if (q0 < q1) fetch(q0, sm);
    pa_arrive();
    for (int q = q0; q < q1; ++q) {
        const char* Q = sm + ((q - q0) & 1) * BUF;
        const char* D = Q + G::QB;
        const float* aux = reinterpret_cast<const float*>(D + G::FB);
        if (q + 1 < q1) fetch(q + 1, sm + ((q - q0 + 1) & 1) * BUF);
        float p[U][4], ds[U][4], y[U][4], th[U][4];
        f32x4 s[U], dp[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = dp[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < G::SF; ++k) {
                if (k < G::SE) s[u] = pa_mma(pa_row<T>(Q, G::PE, 16 * u, k, n, g), kf[k], s[u]);
                dp[u] = pa_mma(pa_row<T>(D, G::PF, 16 * u, k, n, g), vf[k], dp[u]);
            }
        }
        pa_scores<T, CAP, U, true>(s, cap, y, th);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const f32x4 off = *reinterpret_cast<const f32x4*>(aux + 16 * u + 4 * g), scale = *reinterpret_cast<const f32x4*>(aux + G::ROWS + 16 * u + 4 * g),
                        delta = *reinterpret_cast<const f32x4*>(aux + 2 * G::ROWS + 16 * u + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float keep = 1.f;
                if (DROP) {
                    const uint32_t l = (uint32_t)(q * G::ROWS + 16 * u + 4 * g + r);
                    const uint32_t key = gz_row_key(a.seed, GZSL_STREAM_ATTN, (uint32_t)b * a.L_total + a.l_offset + l);
                    keep = gz_u32(key, (uint32_t)tok) >= a.thresh ? a.scale : 0.f;
                }
                pa_grad<CAP>(y[u][r], th[u][r], dp[u][r], off[r], scale[r], delta[r], keep, p[u][r], ds[u][r]);
            }
        }
        frag pf, sf;
        pa_pack(p, pf);
        pa_pack(ds, sf);
#pragma unroll
        for (int j = 0; j < G::NF; ++j) dv[j] = pa_mma(pa_col<T>(D, G::PF, 0, 16 * j, n, g), pf, dv[j]);
        if constexpr (sizeof(T) == 2) {
            frag sl;
            pa_pack_low(ds, sl);
#pragma unroll
            for (int j = 0; j < G::NE; ++j) {
                const frag f = pa_col<T>(Q, G::PE, 0, 16 * j, n, g);
                dk[j] = pa_mma(f, sf, pa_mma(f, sl, dk[j]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < G::NE; ++j) dk[j] = pa_mma(pa_col<T>(Q, G::PE, 0, 16 * j, n, g), sf, dk[j]);
        }
        pa_arrive();
    }
    if (tok >= len) return;
    const long long row = un.sp.start + tok;
    if (un.shares > 1) {
        float* out = a.dkv + ((long long)un.unit * PA_TILE + wave * 16 + n) * (a.E + a.F);
#pragma unroll
        for (int j = 0; j < G::NE; ++j) pa_out<float>(dk[j], out, nullptr, 16 * j + 4 * g, a.E);
#pragma unroll
        for (int j = 0; j < G::NF; ++j) pa_out<float>(dv[j], out + a.E, nullptr, 16 * j + 4 * g, a.F);
        return;
    }
#pragma unroll
    for (int j = 0; j < G::NE; ++j) pa_out<T>(dk[j], (T*)a.dK + row * a.E, nullptr, 16 * j + 4 * g, a.E);
#pragma unroll
    for (int j = 0; j < G::NF; ++j) pa_out<T>(dv[j], (T*)a.dV + row * a.F, nullptr, 16 * j + 4 * g, a.F);
}
// dK / dV from the label shares, in order, and zeros in the rows of no note: 16 rows a workgroup, counted from a note's first
// (blockIdx.y = B: the rows in front of the first note), a wave to a row.
#define PA_JOIN_ROWS 16
template <typename T>
__global__ __launch_bounds__(256) void pa_kv_finish_kernel(PaArgs a) {
    const int b = blockIdx.y, W = a.E + a.F, lane = threadIdx.x & 63, w = threadIdx.x >> 6, last = gridDim.x - 1;
    long long start = 0, len = 0, end;  // rows [start + len, end) belong to no note
    PaTileUnit un;
    un.shares = 1;
    if (b == a.B) {
        end = note_span(a.spans, 0, a.rows, a.max_len).start;
    } else {
        un = pa_tile_unit(a, 0, b);
        start = un.sp.start, len = un.sp.len;
        end = b + 1 < a.B ? note_span(a.spans, b + 1, a.rows, a.max_len).start : a.rows;
    }
    // (the last workgroup of a note takes all that is left behind it)
    const long long stop = (int)blockIdx.x == last ? max(end - start, len) : (long long)(blockIdx.x + 1) * PA_JOIN_ROWS;
    for (long long r = (long long)blockIdx.x * PA_JOIN_ROWS + w; r < stop; r += 4) {
        const long long row = start + r;
        if (r < len) {
            if (un.shares == 1) continue;
            const float* slab = a.dkv + ((un.tile + r / PA_TILE) * un.shares * PA_TILE + r % PA_TILE) * W;
            if (((a.E | a.F) & 3) == 0) {
                for (int c = 4 * lane; c < W; c += 256) {
                    f32x4 s = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
                    for (int k = 0; k < un.shares; ++k) s += *reinterpret_cast<const f32x4*>(slab + (long long)k * PA_TILE * W + c);
                    if (c < a.E) pa_out<T>(s, (T*)a.dK + row * a.E, nullptr, c, a.E);
                    else pa_out<T>(s, (T*)a.dV + row * a.F, nullptr, c - a.E, a.F);
                }
                continue;
            }
            for (int c = lane; c < W; c += 64) {
                float s = 0.f;
#pragma unroll 4
                for (int k = 0; k < un.shares; ++k) s += slab[(long long)k * PA_TILE * W + c];
                if (c < a.E) ((T*)a.dK)[row * a.E + c] = (T)s;
                else ((T*)a.dV)[row * a.F + c - a.E] = (T)s;
            }
        } else if (row < end) {
            for (int c = lane; c < a.E; c += 64) ((T*)a.dK)[row * a.E + c] = (T)0.f;
            for (int c = lane; c < a.F; c += 64) ((T*)a.dV)[row * a.F + c] = (T)0.f;
        }
    }
}

// dQ: workgroup = WAVES x 16 labels (label on the lane axis) over one note or one chunk of it; a slab per chunk.
template <typename T, class G, int WAVES, bool CAP, bool DROP>
__global__ __launch_bounds__(WAVES * 64, 2) void pa_bwd_q_kernel(PaArgs a) {
    typedef typename PaTy<T>::frag frag;
    constexpr int U = G::U;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 15, g = lane >> 4;
    const int lt = blockIdx.x % a.nLT;
    const PaUnit un = pa_unit<G::ROWS>(a, blockIdx.x / a.nLT);
    if (un.ci >= un.all) return;
    const int b = un.b, len = un.sp.len;
    const int t0 = un.c * (un.chunk / G::ROWS), t1 = (int)min((long long)(len + G::ROWS - 1) / G::ROWS, (long long)t0 + un.chunk / G::ROWS);
    const int l0 = (lt * WAVES + wave) * 16;
    const PaCap cap = pa_cap(a.cap);
    frag qf[G::SE], df[G::SF];
    float off, scale, delta;
    {
        const int l = min(l0 + n, a.nQ * G::ROWS - 1);
        const char* qr = a.Q + (long long)(l / G::ROWS) * G::QB + (l % G::ROWS) * G::PE + 16 * g;
        const char* dimg = a.DO + ((long long)b * a.nQ + l / G::ROWS) * G::OB;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) qf[s] = *reinterpret_cast<const frag*>(qr + 64 * s);
#pragma unroll
        for (int s = 0; s < G::SF; ++s) df[s] = *reinterpret_cast<const frag*>(dimg + (l % G::ROWS) * G::PF + 16 * g + 64 * s);
        const float* aux = reinterpret_cast<const float*>(dimg + G::FB);
        off = aux[l % G::ROWS], scale = aux[G::ROWS + l % G::ROWS], delta = aux[2 * G::ROWS + l % G::ROWS];
    }
    const uint32_t key = gz_row_key(a.seed, GZSL_STREAM_ATTN, (uint32_t)b * a.L_total + a.l_offset + (uint32_t)(l0 + n));
    f32x4 dq[G::NE];
#pragma unroll
    for (int j = 0; j < G::NE; ++j) dq[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const char* kv = a.KV + (long long)b * a.nT * G::KV;
    if (t0 < t1) pa_dma<WAVES>(kv + (long long)t0 * G::KV, sm, G::KV, wave, lane);
    pa_arrive();
    auto step = [&](int t, auto last) {  // last: the tile may end behind the note
        const char* K = sm + ((t - t0) & 1) * G::KV;
        const char* V = K + G::EB;
        if (t + 1 < t1) pa_dma<WAVES>(kv + (long long)(t + 1) * G::KV, sm + ((t - t0 + 1) & 1) * G::KV, G::KV, wave, lane);
        float ds[U][4], y[U][4], th[U][4];
        f32x4 s[U], dp[U];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s[u] = dp[u] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < G::SF; ++k) {
                if (k < G::SE) s[u] = pa_mma(pa_row<T>(K, G::PE, 16 * u, k, n, g), qf[k], s[u]);
                dp[u] = pa_mma(pa_row<T>(V, G::PF, 16 * u, k, n, g), df[k], dp[u]);
            }
        }
        pa_scores<T, CAP, U, true>(s, cap, y, th);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float keep = 1.f, p;
                if (DROP) keep = gz_u32(key, (uint32_t)(t * G::ROWS + 16 * u + 4 * g + r)) >= a.thresh ? a.scale : 0.f;
                pa_grad<CAP>(y[u][r], th[u][r], dp[u][r], off, scale, delta, keep, p, ds[u][r]);
            }
        if constexpr (decltype(last)::value) {  // (a key of zeros has the score 0, which may be far above the note's own)
            const int left = len - t * G::ROWS;
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (16 * u + 4 * g + r >= left) ds[u][r] = 0.f;
        }
        frag sf;
        pa_pack(ds, sf);
        if constexpr (sizeof(T) == 2) {
            frag sl;
            pa_pack_low(ds, sl);
#pragma unroll
            for (int j = 0; j < G::NE; ++j) {
                const frag f = pa_col<T>(K, G::PE, 0, 16 * j, n, g);
                dq[j] = pa_mma(f, sf, pa_mma(f, sl, dq[j]));
            }
        } else {
#pragma unroll
            for (int j = 0; j < G::NE; ++j) dq[j] = pa_mma(pa_col<T>(K, G::PE, 0, 16 * j, n, g), sf, dq[j]);
        }
        pa_arrive();
    };
    for (int t = t0; t < t1 - 1; ++t) step(t, std::false_type{});
    if (t0 < t1) step(t1 - 1, std::true_type{});
    const int l = l0 + n;
    if (l >= a.L) return;
    float* out = a.dq + ((long long)un.ci * a.L + l) * a.E;
#pragma unroll
    for (int j = 0; j < G::NE; ++j) pa_out<float>(dq[j], out, nullptr, 16 * j + 4 * g, a.E);
}
// dQ = sum of the slabs, in order.
template <typename T, int ROWS>
__global__ __launch_bounds__(256) void pa_q_join_kernel(PaArgs a) {
    const int all = pa_unit<ROWS>(a, 0).all;
    const long long n = (long long)a.L * a.E;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
        float s = 0.f;
#pragma unroll 4
        for (int k = 0; k < all; ++k) s += a.dq[k * n + i];
        ((T*)a.dQ)[i] = (T)s;
    }
}

// --------------------------------------------------------------------------------------------------------------- launch
template <typename T, class G, int W, bool CAP, bool DROP>
static int pa_fwd(PaArgs& a, hipStream_t st) {
    hipLaunchKernelGGL((pa_pack_kernel<T, G>), dim3(a.B * a.nT + a.nQ), dim3(256), 0, st, a);
    hipLaunchKernelGGL((pa_fwd_kernel<T, G, W, CAP, DROP>), dim3(a.nLT * (a.B + a.extra)), dim3(W * 64), 2 * G::KV, st, a);
    if (a.extra > 0) {
        if ((long long)a.B * a.L <= 1024) hipLaunchKernelGGL((pa_join_kernel<T, G::ROWS, 4>), dim3(a.B * a.L), dim3(256), 0, st, a);
        else hipLaunchKernelGGL((pa_join_kernel<T, G::ROWS, 1>), dim3(a.B * cdiv(a.L, 4)), dim3(256), 0, st, a);
    }
    GZSL_CHECK_LAUNCH();
    return 0;
}
template <typename T, class G, int W, bool CAP, bool DROP>
static int pa_bwd(PaArgs& a, const PaPlan& p, hipStream_t st) {
    hipLaunchKernelGGL((pa_pack_kernel<T, G>), dim3(a.B * a.nT + a.nQ), dim3(256), 0, st, a);
    hipLaunchKernelGGL((pa_pack_do_kernel<T, G>), dim3(a.nQ * a.B), dim3(256), 0, st, a);
    if (p.units > 0) hipLaunchKernelGGL((pa_bwd_kv_kernel<T, G, CAP, DROP>), dim3((unsigned)p.units), dim3(256), 2 * (G::QB + G::OB), st, a);
    hipLaunchKernelGGL(pa_kv_finish_kernel<T>, dim3(a.max_len > 0 ? cdiv(a.max_len, PA_JOIN_ROWS) : 1, a.B + 1), dim3(256), 0, st, a);
    hipLaunchKernelGGL((pa_bwd_q_kernel<T, G, W, CAP, DROP>), dim3(a.nLT * (a.B + a.extra)), dim3(W * 64), 2 * G::KV, st, a);
    const long long n = (long long)a.L * a.E;
    hipLaunchKernelGGL((pa_q_join_kernel<T, G::ROWS>), dim3((unsigned)(n < 256 * 4096 ? cdiv((long)n, 256) : 4096)), dim3(256), 0, st, a);
    GZSL_CHECK_LAUNCH();
    return 0;
}
template <typename T, class G, int W, bool CAP>
static int pa_go2(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    if (backward) return a.thresh ? pa_bwd<T, G, W, CAP, true>(a, p, st) : pa_bwd<T, G, W, CAP, false>(a, p, st);
    return a.thresh ? pa_fwd<T, G, W, CAP, true>(a, st) : pa_fwd<T, G, W, CAP, false>(a, st);
}
template <typename T, int W>
static int pa_go(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    typedef PaGeo<T, 7, 13> A;
    typedef PaGeo<T, 13, 13> B;
    if (a.cap > 0.f) return p.wide ? pa_go2<T, B, W, true>(a, p, backward, st) : pa_go2<T, A, W, true>(a, p, backward, st);
    return p.wide ? pa_go2<T, B, W, false>(a, p, backward, st) : pa_go2<T, A, W, false>(a, p, backward, st);
}
