// Kernels of the packed label attention, instantiated by kind of product in packed_attn_{bf16,x3,f32}.hip; the mathematics, the
// fragments, the tile images and the cut of the work are in packed_attn.h.
#pragma once
#include <type_traits>
#include "packed_attn.h"

// The KF elements x of one lane -> its 16 bytes of a fragment (of each plane).
template <class K, class G>
__device__ __forceinline__ typename K::frag pa_cut(const typename K::T (&x)[G::KF]) {
    if constexpr (K::PL == 1) {
        return __builtin_bit_cast(typename K::frag, x);
    } else {
        PaPieces f;
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            bf16 h, m, l;
            pa_split(x[j], h, m, l);
            f.p[0][j] = h, f.p[1][j] = m, f.p[2][j] = l;
            top = fmaxf(top, fabsf(x[j]));
        }
        if (__any(top >= PA_ROUNDS_OVER))
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                bf16 h, m, l;
                pa_split_any(x[j], h, m, l);
                f.p[0][j] = h, f.p[1][j] = m, f.p[2][j] = l;
            }
        return f;
    }
}
template <class K, int COUNT>
__device__ __forceinline__ void pa_put(char* img, int i, const typename K::frag& f, int lane) {
    if constexpr (K::PL == 1) {
        *reinterpret_cast<typename K::frag*>(img + i * 1024 + lane * 16) = f;
    } else {
#pragma unroll
        for (int p = 0; p < 3; ++p) *reinterpret_cast<bf16x8*>(img + (p * COUNT + i) * 1024 + lane * 16) = f.p[p];
    }
}
// ------------------------------------------------------------------------------------------------------------- pre-pass
// A tile's rows into LDS, zeros past nrows (at least 1; REPEAT: its last row again) and past W (row stride P elements).  Addresses are clamped, not branched around,
// and loaded in batches: a batch is on its way together.
template <typename T, int ROWS, bool REPEAT = false, int P>
__device__ __forceinline__ void pa_stage(T (*sh)[P], const T* src, long long ld, int row0, int nrows, int W, int tid) {
    if (((uintptr_t)src & 15) == 0 && ld % (16 / sizeof(T)) == 0 && W % (16 / sizeof(T)) == 0) {
        constexpr int V = 16 / sizeof(T), C = P / V, N = (ROWS * C + 255) / 256;
        typedef T vec __attribute__((ext_vector_type(V)));
        vec v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + 256 * i;
            v[i] = *reinterpret_cast<const vec*>(src + (long long)min(row0 + c / C, nrows - 1) * ld + min(c % C * V, W - V));
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int c = tid + 256 * i, r = c / C, e = c % C * V;
            if (!((REPEAT || row0 + r < nrows) && e < W))
#pragma unroll
                for (int k = 0; k < V; ++k) v[i][k] = (T)0.f;
            if (c < ROWS * C) *reinterpret_cast<vec*>(&sh[r][e]) = v[i];
        }
    } else {
        constexpr int N = (ROWS * P + 255) / 256, D = 8;
#pragma unroll 1
        for (int i0 = 0; i0 < N; i0 += D) {
            T v[D];
#pragma unroll
            for (int i = 0; i < D; ++i) {
                const int c = tid + 256 * (i0 + i);
                v[i] = src[(long long)min(row0 + c / P, nrows - 1) * ld + min(c % P, W - 1)];
            }
#pragma unroll
            for (int i = 0; i < D; ++i) {
                const int c = tid + 256 * (i0 + i), r = c / P, e = c % P;
                if (c < ROWS * P) sh[r][e] = (REPEAT || row0 + r < nrows) && e < W ? v[i] : (T)0.f;
            }
        }
    }
}
// Row (ROW) or column fragments of the staged tile: N of them (a plane), written 1 KB a wave.
template <class K, class G, int N, int STEPS, bool ROW, int P>
__device__ __forceinline__ void pa_emit(typename K::T (*sh)[P], char* img, int tid) {
    typedef typename K::T T;
    const int lane = tid & 63, n = lane & 15, g = lane >> 4;
#pragma unroll
    for (int q0 = 0; q0 < N; q0 += 4) {
        const int i = q0 + (tid >> 6);
        if (i >= N) break;
        T x[G::KF];
        if (ROW) {
            constexpr int V = 16 / (int)sizeof(T);
            typedef T vec __attribute__((ext_vector_type(V)));
            const T* row = &sh[16 * (i / STEPS) + n][i % STEPS * G::KK + g * G::KF];
#pragma unroll
            for (int j = 0; j < G::KF; j += V) {
                const vec v = *reinterpret_cast<const vec*>(row + j);
#pragma unroll
                for (int k = 0; k < V; ++k) x[j + k] = v[k];
            }
        } else {
#pragma unroll
            for (int j = 0; j < G::KF; ++j) x[j] = sh[16 * (j >> 2) + 4 * g + (j & 3)][16 * i + n];
        }
        pa_put<K, N>(img, i, pa_cut<K, G>(x), lane);
    }
}
// Blocks [0, slots): a token tile (keys, values); then nQ blocks of queries.  Memory-bound: reads each operand once, writes its image
// (17404 tokens of 200 + 200 bf16: 8 us).
template <class K, class G, bool BWD>
__global__ __launch_bounds__(256) void pa_pack_kernel(PaArgs a) {
    typedef typename K::T T;
    constexpr int PE = G::SE * G::KK, PF = G::SF * G::KK;
    __shared__ __attribute__((aligned(16))) T se[G::ROWS][PE + 16 / sizeof(T)], sf[G::ROWS][PF + 16 / sizeof(T)];
    const int id = blockIdx.x, tid = threadIdx.x;
    if (id < a.slots) {
        const PaTile un = pa_slot<G::ROWS>(a, id);
        if (un.b < 0) return;
        const int t = un.tile;
        const NoteSpan sp = un.sp;
        pa_stage<T, G::ROWS>(se, (const T*)a.keys + sp.start * a.ldk, a.ldk, t * G::ROWS, sp.len, a.E, tid);
        pa_stage<T, G::ROWS>(sf, (const T*)a.values + sp.start * a.ldv, a.ldv, t * G::ROWS, sp.len, a.F, tid);
        __syncthreads();
        char* img = a.TK + (long long)id * (BWD ? G::TOK : G::FWD) * 1024;
        pa_emit<K, G, G::RE, G::SE, true>(se, img, tid);
        img += G::PL * G::RE * 1024;
        if (!BWD) {
            pa_emit<K, G, G::NF, 1, false>(sf, img, tid);
        } else {
            pa_emit<K, G, G::RF, G::SF, true>(sf, img, tid);
            if (!G::TRT) pa_emit<K, G, G::NE, 1, false>(se, img + G::PL * G::RF * 1024, tid);
        }
    } else {
        const int q = id - a.slots;
        // (past the last label that label again, with weights scaled by 0: of zeros an infinite key would make a score that is no number)
        pa_stage<T, G::ROWS, true>(se, (const T*)a.queries, a.ldq, q * G::ROWS, a.L, a.E, tid);
        __syncthreads();
        char* img = a.Q + (long long)q * (BWD ? G::QRY : G::PL * G::RE) * 1024;
        pa_emit<K, G, G::RE, G::SE, true>(se, img, tid);
        if (BWD && !G::TRL) pa_emit<K, G, G::NE, 1, false>(se, img + G::RE * 1024, tid);
    }
}
// Backward: dO images of (note, label tile); behind the fragments, for each label, off and scale of its weights
// P = e^(y - off) * scale (from the forward's own maximum and sum; from LSE where the caller has only that; past the last label its
// off again and scale 0) and delta = <dO_l, O_l> (with what the rounding of O dropped, where it is known).  TPR threads a row.  Memory-bound
// (16 x 1999 rows of 200 bf16: 67 MB in 14 us).
template <class K, class G>
__global__ __launch_bounds__(256) void pa_pack_do_kernel(PaArgs a) {
    typedef typename K::T T;
    constexpr int TPR = 256 / G::ROWS, PF = G::SF * G::KK;
    __shared__ __attribute__((aligned(16))) T sf[G::ROWS][PF + 16 / sizeof(T)];
    const int q = blockIdx.x % a.nQ, b = blockIdx.x / a.nQ, tid = threadIdx.x;
    char* img = a.DO + ((long long)b * a.nQ + q) * G::OUT * 1024;
    pa_stage<T, G::ROWS>(sf, (const T*)a.dO + (long long)b * a.L * a.F, a.F, q * G::ROWS, a.L, a.F, tid);
    __syncthreads();
    const int r = tid / TPR, l = q * G::ROWS + r;
    const long long row = (long long)b * a.L + l;
    float s = 0.f;
    if (l < a.L) {
        const T* y = (const T*)a.cO + row * a.F;
        const bf16* low = sizeof(T) == 2 && a.crest ? reinterpret_cast<const bf16*>(a.crest + 2LL * a.B * a.L) + row * a.F : nullptr;
        constexpr int V = 16 / (int)sizeof(T), N = (208 / V + TPR - 1) / TPR;  // (F <= 208)
        typedef T vec __attribute__((ext_vector_type(V)));
        if (a.F % V == 0 && (((uintptr_t)y | (uintptr_t)low) & 15) == 0) {
            vec v[N], w[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int f = min((tid % TPR + i * TPR) * V, a.F - V);
                v[i] = *reinterpret_cast<const vec*>(y + f);
                if (sizeof(T) == 2) w[i] = low ? *reinterpret_cast<const vec*>(low + f) : v[i];
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const int f = (tid % TPR + i * TPR) * V;
                if (f < a.F)
#pragma unroll
                    for (int k = 0; k < V; ++k) s = fmaf((float)sf[r][f + k], (float)v[i][k] + (low ? (float)w[i][k] : 0.f), s);
            }
        } else {
#pragma unroll 4
            for (int f = tid % TPR; f < a.F; f += TPR) s = fmaf((float)sf[r][f], (float)y[f] + (low ? (float)low[f] : 0.f), s);
        }
    }
#pragma unroll
    for (int o = 1; o < TPR; o <<= 1) s += __shfl_xor(s, o);
    if (tid % TPR == 0) {
        float* aux = reinterpret_cast<float*>(img + (G::OUT - 1) * 1024);
        float off = 0.f, scale = 0.f;
        const long long at = min(row, (long long)b * a.L + a.L - 1);
        if (a.crest) off = a.crest[2 * at], scale = a.crest[2 * at + 1];
        else if (a.cLSE[at] != -INFINITY) off = a.cLSE[at] * (a.cap > 0.f ? PA_LOG2E : 1.f), scale = 1.f;
        if (l >= a.L) scale = 0.f;
        aux[r] = off;
        aux[G::ROWS + r] = scale;
        aux[2 * G::ROWS + r] = s;
    }
    pa_emit<K, G, G::RF, G::SF, true>(sf, img, tid);
    if (!G::TRL) pa_emit<K, G, G::NF, 1, false>(sf, img + G::PL * G::RF * 1024, tid);
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
// One wave's 16 labels (on the lane axis) against one token tile.
template <class K, class G>
struct PaFwdState {
    typename K::frag qf[G::SE];
    f32x4 acc[G::NF];
    float m, sum;
    uint32_t key;
    bool fixed;
};
template <class K, class G>
__device__ __forceinline__ void pa_fwd_begin(PaFwdState<K, G>& w, const PaArgs& a, bool cap, int b, int l) {
#pragma unroll
    for (int j = 0; j < G::NF; ++j) w.acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    w.key = gz_row_key(a.seed, GZSL_STREAM_ATTN, (uint32_t)b * a.L_total + a.l_offset + (uint32_t)l);
    // Scores capped at 30 lie within 2^+-44: their exponentials and sums are plain fp32 numbers without a maximum taken off, and
    // nothing is ever rescaled.  Otherwise a tile whose maximum exceeds the running one by more than 2^12 moves it.
    w.fixed = cap && a.cap <= 30.f;
    w.m = w.fixed ? 0.f : -INFINITY, w.sum = 0.f;
}
// KR: row fragments of the keys, VC: column fragments of the values; t0: the tile's first token, LAST: it may end behind the note (left
// tokens are the note's).
template <class K, class G, int CAP, bool DROP, bool LAST>
__device__ __forceinline__ void pa_fwd_tile(PaFwdState<K, G>& w, const PaArgs& a, const PaCap& cap, const char* KR, const char* VC, int t0, int left,
                                            int lane) {
    typedef typename K::frag frag;
    constexpr bool TWO = sizeof(typename K::T) == 2;  // the weights go in two bf16 pieces
    constexpr int U = G::U, D = G::PL == 3 || (TWO && CAP == PA_SERIES) ? 2 : (TWO && DROP ? 3 : 4);  // (where four ahead would spill)
    const int g = lane >> 4;
    f32x4 s[U];
#pragma unroll
    for (int u = 0; u < U; ++u) s[u] = f32x4{0.f, 0.f, 0.f, 0.f};
    frag ring[D];
    auto ldk = [&](int i) { return pa_frag<K, G::RE>(KR, i % U * G::SE + i / U, lane); };
    auto ldv = [&](int j) { return pa_frag<K, G::NF>(VC, j, lane); };
    pa_fill_ring<G::RE>(ring, ldk);
    pa_run_ring<G::RE>(ring, ldk, [&](int i, const frag& f) { s[i % U] = pa_mma(f, w.qf[i / U], s[i % U]); });
    pa_fill_ring<G::NF>(ring, ldv);  // under way during the softmax
    float y[U][4], th[U][4];
    pa_scores<CAP, U, false>(s, cap, y, th);
    if (LAST) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (16 * u + 4 * g + r >= left) y[u][r] = -INFINITY;
    }
    if (!w.fixed) {
        float mt = -INFINITY;
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) mt = fmaxf(mt, y[u][r]);
        if (__any(mt > w.m + (CAP ? 12.f : 12.f * PA_LN2))) {  // m is the same in the four lanes of a column
            mt = fmaxf(mt, __shfl_xor(mt, 16));
            mt = fmaxf(mt, __shfl_xor(mt, 32));
            const float mn = fmaxf(w.m, mt), alpha = mn == w.m ? 1.f : pa_exp<CAP>(w.m - mn);
#pragma unroll
            for (int j = 0; j < G::NF; ++j) w.acc[j] *= alpha;
            w.sum *= alpha;
            w.m = mn;
        }
        const float mi = w.m == -INFINITY ? 0.f : w.m;  // (no finite score yet: every weight is 2^-inf = 0)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[u][r] -= mi;
    }
    frag pf;
    bf16x8 pl;
    {
        float p[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[u][r] = pa_exp<CAP>(y[u][r]);
                w.sum += p[u][r];
                if (DROP) p[u][r] = gz_u32(w.key, (uint32_t)(t0 + 16 * u + 4 * g + r)) >= a.thresh ? p[u][r] * a.scale : 0.f;
            }
        if constexpr (TWO) pa_pack_two(p, pf, pl);
        else pa_pack(p, pf);
    }
    pa_run_ring<G::NF>(ring, ldv, [&](int j, const frag& f) {
        if constexpr (TWO) w.acc[j] = pa_mma(f, pl, w.acc[j]);
        w.acc[j] = pa_mma(f, pf, w.acc[j]);
    });
}
// Output rows, or a chunk's part of them.  A row without a finite score (sum 0) is one of no tokens.
__device__ __forceinline__ float pa_lse(const PaArgs& a, float m, float sum) {
    return sum == 0.f ? -INFINITY : fmaf(__builtin_amdgcn_logf(sum), PA_LN2, a.cap > 0.f ? m * PA_LN2 : m);
}
template <class K, class G>
__device__ __forceinline__ void pa_fwd_end(PaFwdState<K, G>& w, const PaArgs& a, const PaUnit& un, int l, int lane) {
    typedef typename K::T T;
    const int g = lane >> 4;
    float sum = w.sum;
    sum += __shfl_xor(sum, 16);
    sum += __shfl_xor(sum, 32);
    if (l >= a.L) return;
    const long long row = (long long)un.b * a.L + l;
    if (un.nch > 1) {
        const long long pr = (long long)un.ci * a.L + l;
        if (g == 0) a.ml[2 * pr] = w.m, a.ml[2 * pr + 1] = sum;
#pragma unroll
        for (int j = 0; j < G::NF; ++j) pa_out<float>(w.acc[j], a.part + pr * a.F, nullptr, 16 * j + 4 * g, a.F);
        return;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (g == 0) {
        a.LSE[row] = pa_lse(a, w.m, sum);
        if (a.rest) a.rest[2 * row] = sum == 0.f ? 0.f : w.m, a.rest[2 * row + 1] = inv;
    }
    T* out = (T*)a.O + row * a.F;
    bf16* low = sizeof(T) == 2 && a.rest ? reinterpret_cast<bf16*>(a.rest + 2LL * a.B * a.L) + row * a.F : nullptr;
#pragma unroll
    for (int j = 0; j < G::NF; ++j) pa_out<T>(w.acc[j] * inv, out, low, 16 * j + 4 * g, a.F);
}

// Workgroup = WAVES x 16 labels of one note (or of one chunk of it), token tiles from the pre-pass's images.  An image is read by all
// label workgroups of a note and comes from L2; a wave's 16 queries and its output tile stay in registers.  Bound by the matrix pipe
// (bf16 62 % busy, PaX3 70 %) and the softmax's vector instructions, which overlap with other waves' matrix instructions only in part:
// 19309 tokens x 9000 labels (100, 200; capped) bf16 175 us, 1090 TFLOP/s of the padded products, the second pieces' among them (1255 is what a large library product
// reaches, whose clock is as low); without the softmax 97.  Tried at that size and no faster: 32 labels a wave (half the LDS
// reads), three tiles on their way instead of two, priorities by phase or by workgroup.  PaX3: 7339 x 9000 220 us.
template <class K, class G, int WAVES, int OCC, int CAP, bool DROP>
__global__ __launch_bounds__(WAVES * 64, OCC) void pa_fwd_kernel(PaArgs a) {
    extern __shared__ __attribute__((aligned(16))) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = pa_scalar(tid >> 6), n = lane & 15;
    const int lt = blockIdx.x % a.nLT;
    const PaUnit un = pa_unit<G::ROWS>(a, blockIdx.x / a.nLT);
    if (un.ci >= un.all) return;
    const int b = un.b, len = un.sp.len;
    const int t0 = un.c * (un.chunk / G::ROWS), t1 = (int)min((long long)(len + G::ROWS - 1) / G::ROWS, (long long)t0 + un.chunk / G::ROWS);
    const int l0 = (lt * WAVES + wave) * 16;
    const bool idle = l0 >= a.L;  // (wave-uniform: copies and barriers only)
    const PaCap cap = pa_cap(a.cap);
    PaFwdState<K, G> w;
    pa_fwd_begin(w, a, CAP != PA_NONE, b, l0 + n);
    {
        const int c = min(l0, a.nQ * G::ROWS - 16);
        const char* img = a.Q + (long long)(c / G::ROWS) * G::PL * G::RE * 1024;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) w.qf[s] = pa_frag<K, G::RE>(img, (c % G::ROWS / 16) * G::SE + s, lane);
    }
    const PaImages tk = pa_images<G::ROWS>(a, b, un.sp.start, G::FWD);
    if (t0 < t1) pa_dma<WAVES, G::FWD>(tk(t0), sm, wave, lane);
    pa_arrive();
    auto step = [&](int t, auto last) {
        const char* KR = sm + ((t - t0) & 1) * G::FWD * 1024;
        if (t + 1 < t1) pa_dma<WAVES, G::FWD>(tk(t + 1), sm + ((t - t0 + 1) & 1) * G::FWD * 1024, wave, lane);
        if (!idle) pa_fwd_tile<K, G, CAP, DROP, decltype(last)::value>(w, a, cap, KR, KR + G::PL * G::RE * 1024, t * G::ROWS, len - t * G::ROWS, lane);
        pa_arrive();
    };
    for (int t = t0; t < t1 - 1; ++t) step(t, std::false_type{});
    if (t0 < t1) step(t1 - 1, std::true_type{});
    pa_fwd_end(w, a, un, l0 + n, lane);
}

// KF consecutive elements of a row from e0 (clamped address, no branch around a load).  wide: 16-byte loads are allowed.
template <class G, typename T>
__device__ __forceinline__ void pa_row_load(const T* row, int e0, int W, bool wide, T (&x)[G::KF]) {
    constexpr int V = 16 / (int)sizeof(T);
    typedef T vec __attribute__((ext_vector_type(V)));
    if (wide) {
#pragma unroll
        for (int j = 0; j < G::KF; j += V) {
            const vec v = *reinterpret_cast<const vec*>(row + min(e0 + j, W - V));
#pragma unroll
            for (int k = 0; k < V; ++k) x[j + k] = v[k];
        }
    } else {
#pragma unroll
        for (int j = 0; j < G::KF; ++j) x[j] = row[min(e0 + j, W - 1)];
    }
}

// The same for at most WAVES x 16 labels (one label workgroup a note or chunk): every token tile is then read by one workgroup
// alone, which cuts its fragments itself: each wave loads the elements of its share of the next tile's fragments while it works on the
// current one.  No images and one launch less: 2 notes of 59 tokens in all x 70 labels 16 -> 13 us, 40003 tokens x 50 labels 58 -> 40.
// With more labels every label workgroup would cut the fragments again.  What bounds it is latency: five tiles a workgroup at 256
// workgroups (24 us for 48 MB); a second tile on its way changed nothing.
template <class K, class G, int WAVES, int CAP, bool DROP>
__global__ __launch_bounds__(WAVES * 64, 2) void pa_fwd_direct_kernel(PaArgs a) {
    typedef typename K::T T;
    constexpr int V = 16 / (int)sizeof(T), NR = (G::RE + WAVES - 1) / WAVES, NC = (G::NF + WAVES - 1) / WAVES;  // fragments of a wave
    extern __shared__ __attribute__((aligned(16))) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = pa_scalar(tid >> 6), n = lane & 15, g = lane >> 4;
    const PaUnit un = pa_unit<G::ROWS>(a, blockIdx.x);
    if (un.ci >= un.all) return;
    const int b = un.b, len = un.sp.len;
    const int t0 = un.c * (un.chunk / G::ROWS), t1 = (int)min((long long)(len + G::ROWS - 1) / G::ROWS, (long long)t0 + un.chunk / G::ROWS);
    const int l0 = wave * 16;
    const bool idle = l0 >= a.L;
    const PaCap cap = pa_cap(a.cap);
    const T *kp = (const T*)a.keys + un.sp.start * a.ldk, *vp = (const T*)a.values + un.sp.start * a.ldv;
    const bool kwide = a.E % V == 0 && a.ldk % V == 0 && ((uintptr_t)kp & 15) == 0;
    T xk[NR][G::KF], xv[NC][G::KF];
    auto load = [&](int t) {
#pragma unroll
        for (int q = 0; q < NR; ++q) {
            const int i = min(wave + q * WAVES, G::RE - 1), row = min(t * G::ROWS + 16 * (i / G::SE) + n, len - 1);
            pa_row_load<G>(kp + row * a.ldk, i % G::SE * G::KK + g * G::KF, a.E, kwide, xk[q]);
        }
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            const int c = min(16 * min(wave + q * WAVES, G::NF - 1) + n, a.F - 1);
#pragma unroll
            for (int j = 0; j < G::KF; ++j) xv[q][j] = vp[min(t * G::ROWS + 16 * (j >> 2) + 4 * g + (j & 3), len - 1) * a.ldv + c];
        }
    };
    // zeros past the note's end and past E / F
    auto store = [&](int t, char* buf) {
#pragma unroll
        for (int q = 0; q < NR; ++q) {
            const int i = wave + q * WAVES, e0 = i % G::SE * G::KK + g * G::KF;
            if (i >= G::RE) break;
            const bool in = t * G::ROWS + 16 * (i / G::SE) + n < len;
#pragma unroll
            for (int j = 0; j < G::KF; ++j) xk[q][j] = in && e0 + j < a.E ? xk[q][j] : (T)0.f;
            pa_put<K, G::RE>(buf, i, pa_cut<K, G>(xk[q]), lane);
        }
#pragma unroll
        for (int q = 0; q < NC; ++q) {
            const int i = wave + q * WAVES;
            if (i >= G::NF) break;
#pragma unroll
            for (int j = 0; j < G::KF; ++j) xv[q][j] = t * G::ROWS + 16 * (j >> 2) + 4 * g + (j & 3) < len && 16 * i + n < a.F ? xv[q][j] : (T)0.f;
            pa_put<K, G::NF>(buf + G::PL * G::RE * 1024, i, pa_cut<K, G>(xv[q]), lane);
        }
    };
    if (t0 < t1) load(t0);
    PaFwdState<K, G> w;
    pa_fwd_begin(w, a, CAP != PA_NONE, b, l0 + n);
    {
        const T* row = (const T*)a.queries + (long long)min(l0 + n, a.L - 1) * a.ldq;
        const bool qwide = a.E % V == 0 && a.ldq % V == 0 && ((uintptr_t)a.queries & 15) == 0;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) {
            const int e0 = s * G::KK + g * G::KF;
            T x[G::KF];
            pa_row_load<G>(row, e0, a.E, qwide, x);
#pragma unroll
            for (int j = 0; j < G::KF; ++j) x[j] = l0 + n < a.L && e0 + j < a.E ? x[j] : (T)0.f;
            w.qf[s] = pa_cut<K, G>(x);
        }
    }
    if (t0 < t1) store(t0, sm);
    if (t0 + 1 < t1) load(t0 + 1);
    __syncthreads();
    for (int t = t0; t < t1; ++t) {  // (the masked form for every tile: one copy of the code, whose first run is part of a short call)
        const char* KR = sm + ((t - t0) & 1) * G::FWD * 1024;
        if (!idle) pa_fwd_tile<K, G, CAP, DROP, true>(w, a, cap, KR, KR + G::PL * G::RE * 1024, t * G::ROWS, len - t * G::ROWS, lane);
        if (t + 1 < t1) store(t + 1, sm + ((t - t0 + 1) & 1) * G::FWD * 1024);
        if (t + 2 < t1) load(t + 2);
        __syncthreads();
    }
    pa_fwd_end(w, a, un, l0 + n, lane);
}
// Joins the chunks of a (note, label), in order: a workgroup of 4 rows of one wave each, or (G > 1, few rows over many chunks) of one
// row whose chunks G waves share and join in LDS.  A lane weighs one chunk; a row's F values lie over the lanes.  Latency-bound (50 rows
// of 250 chunks: 9.6 us, 12.7 with the parts loaded behind the weights).
template <typename T, int ROWS, int G>
__global__ __launch_bounds__(G == 1 ? 256 : 64 * G) void pa_join_kernel(PaArgs a) {
    __shared__ float so[G == 1 ? 4 : G][256], ss[G == 1 ? 4 : G], sM[G];
    constexpr int R = G == 1 ? 4 : 1;
    const int lane = threadIdx.x & 63, w = pa_scalar((int)threadIdx.x >> 6), part = w % G, nb = (a.L + R - 1) / R;
    const int l = blockIdx.x % nb * R + w / G;
    const PaUnit un = pa_unit<ROWS>(a, 0, blockIdx.x / nb);
    if (un.nch == 1) return;
    const bool on = l < a.L, vec = a.F % 4 == 0;
    const int per = (un.nch + G - 1) / G, c0 = on ? part * per : 0, c1 = on ? min(un.nch, c0 + per) : 0;
    const float* ml = a.ml + 2 * ((long long)un.ci * a.L + l);
    const float* pr = a.part + ((long long)un.ci * a.L + l) * a.F;
    constexpr int D = 4;  // parts of a row on their way, the first of them while the weights are worked out
    f32x4 v[D];           // values 4 lane .. + 3 (vec), else lane + 64 k
    auto load = [&](int c) {
#pragma unroll
        for (int i = 0; i < D; ++i) {
            const float* x = pr + (long long)min(c + i, c1 - 1) * a.L * a.F;
            if (vec) {
                v[i] = *reinterpret_cast<const f32x4*>(x + min(4 * lane, a.F - 4));
            } else {
#pragma unroll
                for (int k = 0; k < 4; ++k) v[i][k] = x[min(lane + 64 * k, a.F - 1)];
            }
        }
    };
    if (c0 < c1) load(c0);
    float M = -INFINITY;
    for (int c = c0 + lane; c < c1; c += 64)
        if (ml[2LL * c * a.L + 1] != 0.f) M = fmaxf(M, ml[2LL * c * a.L]);  // (no finite score in this chunk: sum 0)
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o));
    if (G > 1) {
        if (lane == 0) sM[part] = M;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < G; ++k) M = fmaxf(M, sM[k]);
    }
    float sum = 0.f, f = 0.f;
    f32x4 o4 = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int b0 = c0; b0 < c1; b0 += D) {
        if ((b0 - c0) % 64 == 0) {
            const int c = min(b0 + lane, c1 - 1);
            const float s = b0 + lane < c1 ? ml[2LL * c * a.L + 1] : 0.f;
            f = s != 0.f ? __builtin_amdgcn_exp2f((ml[2LL * c * a.L] - M) * (a.cap > 0.f ? 1.f : PA_LOG2E)) : 0.f;
            sum = fmaf(f, s, sum);
        }
#pragma unroll
        for (int i = 0; i < D; ++i) {
            const float fi = __shfl(f, (b0 - c0) % 64 + i);
            if (b0 + i < c1)  // (a part that is no number stays one behind a weight of 0)
#pragma unroll
                for (int k = 0; k < 4; ++k) o4[k] = fmaf(fi, v[i][k], o4[k]);
        }
        if (b0 + D < c1) load(b0 + D);
    }
    sum = wave_sum(sum);
#pragma unroll
    for (int k = 0; k < 4; ++k) so[w][vec ? 4 * lane + k : lane + 64 * k] = o4[k];
    if (lane == 0) ss[w] = sum;
    __syncthreads();
    // one thread a value from here on
    const long long row = (long long)un.b * a.L + l;
    bf16* low = sizeof(T) == 2 && a.rest ? reinterpret_cast<bf16*>(a.rest + 2LL * a.B * a.L) + row * a.F : nullptr;
    const int f0 = G == 1 ? lane : threadIdx.x, step = G == 1 ? 64 : 64 * G, w0 = G == 1 ? w : 0;
    if (!on) return;
    sum = 0.f;
#pragma unroll
    for (int q = 0; q < G; ++q) sum += ss[w0 + q];
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    if (f0 == 0) {
        a.LSE[row] = pa_lse(a, M, sum);
        if (a.rest) a.rest[2 * row] = sum == 0.f ? 0.f : M, a.rest[2 * row + 1] = inv;
    }
    for (int f = f0; f < a.F; f += step) {
        float o = 0.f;
#pragma unroll
        for (int q = 0; q < G; ++q) o += so[w0 + q][f];
        o *= inv;
        const T r = (T)o;
        ((T*)a.O)[row * a.F + f] = r;
        if (low) low[f] = (bf16)(o - (float)r);
    }
}

// ------------------------------------------------------------------------------------------------------------- backward
// P and dS of a tile: weights w = e^(y - off) * scale, dropout factor keep.
template <int CAP, bool TH>
__device__ __forceinline__ void pa_grad(float y, float th, float dp, float off, float scale, float delta, float keep, float& p, float& ds) {
    const float w = pa_exp<CAP>(y - off) * scale;
    p = w * keep;
    ds = w * fmaf(dp, keep, -delta);
    if (TH) ds *= fmaf(-th, th, 1.f);
}

// dK / dV: workgroup = one run of steps, 128 tokens of one note (16 a wave, tokens on the lane axis) by a label tile each.  One
// workgroup a compute unit by its LDS and registers, so two waves a SIMD: what they wait for one another, for fragments and at the
// barrier of a step is what is left (PaBF, E, F = 200: matrix pipe 51 % busy, LDS 39 %; PaX3 62 to 64 and 42 to 52 %).  17404 tokens x 1999
// labels of 200 bf16 98 us, 7339 x 9000 of 100 and 200 fp32 305 + 233.
// PaX3 takes dV and dK in two launches (PART 1 and 2): the pieces of K and V and both accumulators are more than the 256 registers of a
// wave at two waves a SIMD, and the scores a second time are a fifth of the products.
template <class K, class G, int PART, int CAP, bool DROP>
__global__ __launch_bounds__(PA_TILE * 4, 2) void pa_bwd_kv_kernel(PaArgs a) {
    typedef typename K::T T;
    typedef typename K::frag frag;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    constexpr int BUF = (G::QRY + G::OUT) * 1024, WAVES = PA_TILE / 16, U = G::U;
    constexpr int D = G::PL == 3 || (G::NE > 7 && (CAP || G::SZ == 4)) ? 2 : 4;  // (where four fragments ahead would spill)
    constexpr bool DV = PART & 1, DK = PART & 2;
    const int tid = threadIdx.x, lane = tid & 63, wave = pa_scalar(tid >> 6), n = lane & 15, g = lane >> 4;
    long long before;
    const PaRuns runs(pa_all_tiles(a, 0, before), a.nQ);
    const int end = min(runs.steps, ((int)blockIdx.x + 1) * runs.per);
    const PaCap cap = pa_cap(a.cap);
    for (int at = (int)blockIdx.x * runs.per; at < end;) {
        const int tile = at / a.nQ, q0 = at % a.nQ, q1 = min(a.nQ, q0 + end - at);
        at += q1 - q0;
        const PaTile un = pa_tile(a, tile);
        const int b = un.b, len = un.sp.len;
        const int tok0 = (un.tile * WAVES + wave) * 16, tok = tok0 + n;
        const bool idle = tok0 >= len;  // (wave-uniform: copies and barriers only)
        frag kf[G::SE], vf[DK ? G::SF : 1];
        {
            const int c = min(tok0, (len - 1) / 16 * 16);
            const char* img = pa_images<G::ROWS>(a, b, un.sp.start, G::TOK)(pa_scalar(c / G::ROWS));
#pragma unroll
            for (int s = 0; s < G::SE; ++s) kf[s] = pa_frag<K, G::RE>(img, (c % G::ROWS / 16) * G::SE + s, lane);
            if (DK)
#pragma unroll
                for (int s = 0; s < G::SF; ++s) vf[s] = pa_frag<K, G::RF>(img + G::PL * G::RE * 1024, (c % G::ROWS / 16) * G::SF + s, lane);
        }
        f32x4 dv[DV ? G::NF : 1], dk[DK ? G::NE : 1];
#pragma unroll
        for (int j = 0; j < (DV ? G::NF : 1); ++j) dv[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < (DK ? G::NE : 1); ++j) dk[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        const char* dO = a.DO + (long long)b * a.nQ * G::OUT * 1024;
        auto fetch = [&](int q, char* buf) {
            pa_dma<WAVES, G::QRY>(a.Q + (long long)q * G::QRY * 1024, buf, wave, lane);
            pa_dma<WAVES, G::OUT>(dO + (long long)q * G::OUT * 1024, buf + G::QRY * 1024, wave, lane);
        };
        fetch(q0, sm);
        pa_arrive();
        for (int q = q0; q < q1; ++q) {
            const char* QR = sm + ((q - q0) & 1) * BUF;
            const char* DR = QR + G::QRY * 1024;
            const float* aux = reinterpret_cast<const float*>(DR + (G::OUT - 1) * 1024);
            if (q + 1 < q1) fetch(q + 1, sm + ((q - q0 + 1) & 1) * BUF);
            if (!idle) {
                f32x4 s[U], dp[U];
#pragma unroll
                for (int u = 0; u < U; ++u) s[u] = dp[u] = f32x4{0.f, 0.f, 0.f, 0.f};
                frag ring[D];
                // rows of the queries, then rows of dO
                constexpr int NS = G::RE + (DK ? G::RF : 0);
                auto ldr = [&](int i) {
                    return i < G::RE ? pa_frag<K, G::RE>(QR, i % U * G::SE + i / U, lane) : pa_frag<K, G::RF>(DR, (i - G::RE) % U * G::SF + (i - G::RE) / U, lane);
                };
                pa_fill_ring<NS>(ring, ldr);
                pa_run_ring<NS>(ring, ldr, [&](int i, const frag& f) {
                    if (i < G::RE) s[i % U] = pa_mma(f, kf[i / U], s[i % U]);
                    else dp[(i - G::RE) % U] = pa_mma(f, vf[DK ? (i - G::RE) / U : 0], dp[(i - G::RE) % U]);
                });
                auto ldv = [&](int j) {
                    if constexpr (G::TRL) return pa_col_tr<K, G::SF>(DR, j, n, g);
                    else return pa_frag<K, G::NF>(DR + G::RF * 1024, j, lane);
                };
                auto ldk = [&](int j) {
                    if constexpr (G::TRL) return pa_col_tr<K, G::SE>(QR, j, n, g);
                    else return pa_frag<K, G::NE>(QR + G::RE * 1024, j, lane);
                };
                constexpr int NC = (DV ? G::NF : 0) + (DK ? G::NE : 0);
                auto ldc = [&](int j) { return DV && j < G::NF ? ldv(j) : ldk(j - (DV ? G::NF : 0)); };
                pa_fill_ring<NC>(ring, ldc);
                float p[U][4], ds[U][4], y[U][4], th[U][4];
                pa_scores<CAP, U, DK>(s, cap, y, th);
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
                        pa_grad<CAP, CAP != PA_NONE && DK>(y[u][r], th[u][r], dp[u][r], off[r], scale[r], delta[r], keep, p[u][r], ds[u][r]);
                    }
                }
                frag pf, sf;
                bf16x8 pl, sl;  // (bf16: what rounding dropped)
                if (DV) pa_pack(p, pf);
                if (DK) pa_pack(ds, sf);
                if constexpr (DK && sizeof(T) == 2) pa_pack_low(ds, sl);
                if constexpr (DV && sizeof(T) == 2) pa_pack_low(p, pl);
                pa_run_ring<NC>(ring, ldc, [&](int j, const frag& f) {
                    if (DV && j < G::NF) {
                        if constexpr (sizeof(T) == 2) dv[DV ? j : 0] = pa_mma(f, pl, dv[DV ? j : 0]);
                        dv[DV ? j : 0] = pa_mma(f, pf, dv[DV ? j : 0]);
                    } else {
                        const int e = DK ? j - (DV ? G::NF : 0) : 0;
                        if constexpr (sizeof(T) == 2) dk[e] = pa_mma(f, sl, dk[e]);
                        dk[e] = pa_mma(f, sf, dk[e]);
                    }
                });
            }
            pa_arrive();
        }
        if (tok < len) {
            const long long row = un.sp.start + tok;
            const bool slab = q1 - q0 < a.nQ;
            int E = a.E, F = a.F;
            asm volatile("" : "+s"(E), "+s"(F));  // (or the masks of all columns below are worked out in front of the loop, and spilled)
            float* part = a.dkv + ((2LL * blockIdx.x + (q0 == 0)) * PA_TILE + wave * 16 + n) * (E + F);
            if (DK)
#pragma unroll
                for (int j = 0; j < G::NE; ++j) {
                    if (slab) pa_out<float>(dk[j], part, nullptr, 16 * j + 4 * g, E);
                    else pa_out<T>(dk[j], (T*)a.dK + row * E, nullptr, 16 * j + 4 * g, E);
                }
            if (DV)
#pragma unroll
                for (int j = 0; j < G::NF; ++j) {
                    if (slab) pa_out<float>(dv[j], part + E, nullptr, 16 * j + 4 * g, F);
                    else pa_out<T>(dv[j], (T*)a.dV + row * F, nullptr, 16 * j + 4 * g, F);
                }
        }
    }
}
// dK / dV of the tiles that runs share, in order, and zeros in the rows of no note: 1, 4 or 16 rows a workgroup, counted from a note's first
// (blockIdx.y = B: the rows in front of the first note), a wave to a row.
template <typename T>
__global__ __launch_bounds__(256) void pa_kv_finish_kernel(PaArgs a) {
    const int b = blockIdx.y, W = a.E + a.F, lane = threadIdx.x & 63, w = pa_scalar((int)threadIdx.x >> 6);
    const NoteSpan sp = b < a.B ? note_span(a.spans, b, a.rows, a.max_len) : NoteSpan{0, 0};
    const long long end = note_gap(a.spans, a.B, a.rows, a.max_len, b < a.B ? sp.start + sp.len : -1);  // of the gap behind this note
    long long first;
    const PaRuns runs(pa_all_tiles(a, b, first), a.nQ);
    if (a.join_rows == 1) {  // few tiles of many runs each: the four waves share one row's parts and join in LDS
        __shared__ float sh[4][7 * 64];
        for (long long r = blockIdx.x; r < max((long long)sp.len, end - sp.start); r += gridDim.x) {
            const long long row = sp.start + r;
            float s[7] = {};  // E + F <= 416
            if (r < sp.len) {
                if (runs.steps == 0) continue;
                const int at = (int)(first + r / PA_TILE) * a.nQ, u0 = at / runs.per, n = (at + a.nQ - 1) / runs.per - u0, per = n / 4 + 1;
                if (n == 0) continue;
                const float* slab = a.dkv + (2LL * u0 * PA_TILE + r % PA_TILE) * W;
#pragma unroll 4
                for (int k = w * per; k < min(n + 1, (w + 1) * per); ++k)
#pragma unroll
                    for (int j = 0; j < 7; ++j) s[j] += slab[(k > 0 ? 2LL * k : 1LL) * PA_TILE * W + min(lane + 64 * j, W - 1)];
            } else if (row >= end) {
                continue;
            }
#pragma unroll
            for (int j = 0; j < 7; ++j) sh[w][lane + 64 * j] = s[j];
            __syncthreads();
            for (int c = threadIdx.x; c < W; c += 256) {
                const T o = (T)(((sh[0][c] + sh[1][c]) + sh[2][c]) + sh[3][c]);
                if (c < a.E) ((T*)a.dK)[row * a.E + c] = o;
                else ((T*)a.dV)[row * a.F + c - a.E] = o;
            }
            __syncthreads();
        }
        return;
    }
    for (long long r0 = (long long)blockIdx.x * a.join_rows; r0 < max((long long)sp.len, end - sp.start); r0 += (long long)gridDim.x * a.join_rows) {
        int u0 = 0, u1 = 0;  // the runs of this tile
        if (r0 < sp.len && runs.steps > 0) {
            const int at = (int)(first + r0 / PA_TILE) * a.nQ;
            u0 = at / runs.per, u1 = (at + a.nQ - 1) / runs.per;
        }
        for (long long r = r0 + w; r < r0 + a.join_rows; r += 4) {
            const long long row = sp.start + r;
            if (r < sp.len) {
                if (u0 == u1) continue;
                // parts: the first run's second slab, then the first slabs of those behind it
                const float* slab = a.dkv + (2LL * u0 * PA_TILE + r % PA_TILE) * W;
                const int n = u1 - u0;
                if (((a.E | a.F) & 3) == 0) {
                    f32x4 s[2];  // E + F <= 416: all of the row on its way at once
#pragma unroll
                    for (int j = 0; j < 2; ++j) s[j] = *reinterpret_cast<const f32x4*>(slab + (long long)PA_TILE * W + min(4 * lane + 256 * j, W - 4));
#pragma unroll 4
                    for (int k = 1; k <= n; ++k)
#pragma unroll
                        for (int j = 0; j < 2; ++j) s[j] += *reinterpret_cast<const f32x4*>(slab + 2LL * k * PA_TILE * W + min(4 * lane + 256 * j, W - 4));
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        const int c = 4 * lane + 256 * j;
                        if (c < a.E) pa_out<T>(s[j], (T*)a.dK + row * a.E, nullptr, c, a.E);
                        else if (c < W) pa_out<T>(s[j], (T*)a.dV + row * a.F, nullptr, c - a.E, a.F);
                    }
                    continue;
                }
                float s[7];
#pragma unroll
                for (int j = 0; j < 7; ++j) s[j] = slab[(long long)PA_TILE * W + min(lane + 64 * j, W - 1)];
#pragma unroll 4
                for (int k = 1; k <= n; ++k)
#pragma unroll
                    for (int j = 0; j < 7; ++j) s[j] += slab[2LL * k * PA_TILE * W + min(lane + 64 * j, W - 1)];
#pragma unroll
                for (int j = 0; j < 7; ++j) {
                    const int c = lane + 64 * j;
                    if (c < a.E) ((T*)a.dK)[row * a.E + c] = (T)s[j];
                    else if (c < W) ((T*)a.dV)[row * a.F + c - a.E] = (T)s[j];
                }
            } else if (row < end) {
                for (int c = lane; c < a.E; c += 64) ((T*)a.dK)[row * a.E + c] = (T)0.f;
                for (int c = lane; c < a.F; c += 64) ((T*)a.dV)[row * a.F + c] = (T)0.f;
            }
        }
    }
}

// dQ: workgroup = WAVES x 16 labels (label on the lane axis) over one note or one chunk of it; a slab per chunk.  H = 2: twice the
// waves, which take turns at the token tiles and add up in LDS (few labels: half the way through the longest note).  Bound as dK / dV is
// (17404 tokens x 1999 labels of 200 bf16 70 us, 7339 x 9000 of 100 and 200 fp32 325).
template <class K, class G, int WAVES, int H, int CAP, bool DROP>
__global__ __launch_bounds__(WAVES * H * 64, 2) void pa_bwd_q_kernel(PaArgs a) {
    typedef typename K::T T;
    typedef typename K::frag frag;
    constexpr int U = G::U, D = G::PL == 3 ? 2 : 4;
    extern __shared__ __attribute__((aligned(16))) char sm[];
    const int tid = threadIdx.x, lane = tid & 63, wave = pa_scalar(tid >> 6) % WAVES, h = pa_scalar(tid >> 6) / WAVES, n = lane & 15, g = lane >> 4;
    const int lt = blockIdx.x % a.nLT;
    const PaUnit un = pa_unit<G::ROWS>(a, blockIdx.x / a.nLT);
    if (un.ci >= un.all) return;
    const int b = un.b, len = un.sp.len;
    const int t0 = un.c * (un.chunk / G::ROWS), t1 = (int)min((long long)(len + G::ROWS - 1) / G::ROWS, (long long)t0 + un.chunk / G::ROWS);
    const int l0 = (lt * WAVES + wave) * 16;
    const bool idle = l0 >= a.L;
    const PaCap cap = pa_cap(a.cap);
    frag qf[G::SE], df[G::SF];
    float off, scale, delta;
    {
        const int c = min(l0, a.nQ * G::ROWS - 16), u = c % G::ROWS / 16;
        const char* qi = a.Q + (long long)(c / G::ROWS) * G::QRY * 1024;
        const char* di = a.DO + ((long long)b * a.nQ + c / G::ROWS) * G::OUT * 1024;
#pragma unroll
        for (int s = 0; s < G::SE; ++s) qf[s] = pa_frag<K, G::RE>(qi, u * G::SE + s, lane);
#pragma unroll
        for (int s = 0; s < G::SF; ++s) df[s] = pa_frag<K, G::RF>(di, u * G::SF + s, lane);
        const float* aux = reinterpret_cast<const float*>(di + (G::OUT - 1) * 1024) + 16 * u + n;
        off = aux[0], scale = aux[G::ROWS], delta = aux[2 * G::ROWS];
    }
    const uint32_t key = gz_row_key(a.seed, GZSL_STREAM_ATTN, (uint32_t)b * a.L_total + a.l_offset + (uint32_t)(l0 + n));
    f32x4 dq[G::NE];
#pragma unroll
    for (int j = 0; j < G::NE; ++j) dq[j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const PaImages tk = pa_images<G::ROWS>(a, b, un.sp.start, G::TOK);
    auto fetch = [&](int t, int k) {
        if (t < t1) pa_dma<WAVES, G::TOK>(tk(t), sm + (2 * h + (k & 1)) * G::TOK * 1024, wave, lane);
    };
    fetch(t0 + h, 0);
    pa_arrive();
    const int steps = (t1 - t0 + H - 1) / H;
    auto step = [&](int k, auto last) {  // last: the tile may end behind the note, or there is none for this half
        const char* KR = sm + (2 * h + (k & 1)) * G::TOK * 1024;
        const char* VR = KR + G::PL * G::RE * 1024;
        const int t = t0 + k * H + h;
        fetch(t + H, k + 1);
        if (!idle && (!decltype(last)::value || t < t1)) {
            f32x4 s[U], dp[U];
#pragma unroll
            for (int u = 0; u < U; ++u) s[u] = dp[u] = f32x4{0.f, 0.f, 0.f, 0.f};
            frag ring[D];
            constexpr int NS = G::RE + G::RF;
            auto ldr = [&](int i) {
                return i < G::RE ? pa_frag<K, G::RE>(KR, i % U * G::SE + i / U, lane) : pa_frag<K, G::RF>(VR, (i - G::RE) % U * G::SF + (i - G::RE) / U, lane);
            };
            pa_fill_ring<NS>(ring, ldr);
            pa_run_ring<NS>(ring, ldr, [&](int i, const frag& f) {
                if (i < G::RE) s[i % U] = pa_mma(f, qf[i / U], s[i % U]);
                else dp[(i - G::RE) % U] = pa_mma(f, df[(i - G::RE) / U], dp[(i - G::RE) % U]);
            });
            auto ldc = [&](int j) {
                if constexpr (G::TRT) return pa_col_tr<K, G::SE>(KR, j, n, g);
                else return pa_frag<K, G::NE>(VR + G::RF * 1024, j, lane);
            };
            pa_fill_ring<G::NE>(ring, ldc);
            float ds[U][4], y[U][4], th[U][4];
            pa_scores<CAP, U, true>(s, cap, y, th);
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float keep = 1.f, p;
                    if (DROP) keep = gz_u32(key, (uint32_t)(t * G::ROWS + 16 * u + 4 * g + r)) >= a.thresh ? a.scale : 0.f;
                    pa_grad<CAP, CAP != PA_NONE>(y[u][r], th[u][r], dp[u][r], off, scale, delta, keep, p, ds[u][r]);
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
            bf16x8 sl;
            pa_pack(ds, sf);
            if constexpr (sizeof(T) == 2) pa_pack_low(ds, sl);
            pa_run_ring<G::NE>(ring, ldc, [&](int j, const frag& f) {
                if constexpr (sizeof(T) == 2) dq[j] = pa_mma(f, sl, dq[j]);
                dq[j] = pa_mma(f, sf, dq[j]);
            });
        }
        pa_arrive();
    };
    for (int k = 0; k < steps - 1; ++k) step(k, std::false_type{});
    if (steps > 0) step(steps - 1, std::true_type{});
    if constexpr (H == 2) {
        f32x4* sum = reinterpret_cast<f32x4*>(sm) + wave * G::NE * 64 + lane;
        static_assert(WAVES * G::NE <= 4 * G::TOK, "fits the buffers");
        if (h == 1)
#pragma unroll
            for (int j = 0; j < G::NE; ++j) sum[64 * j] = dq[j];
        __syncthreads();
        if (h == 1) return;
#pragma unroll
        for (int j = 0; j < G::NE; ++j) dq[j] += sum[64 * j];
    }
    const int l = l0 + n;
    if (l >= a.L) return;
    float* out = a.dq + ((long long)un.ci * a.L + l) * a.E;
#pragma unroll
    for (int j = 0; j < G::NE; ++j) pa_out<float>(dq[j], out, nullptr, 16 * j + 4 * g, a.E);
}
// dQ = sum of the slabs, in a fixed order: a thread an element, or (G > 1, many slabs of few elements: 56 labels of 31, 258 slabs, 22 us
// with one thread, 6 so) G waves share the slabs of 64 elements and join in LDS.
template <typename T, int ROWS, int G>
__global__ __launch_bounds__(G == 1 ? 256 : 64 * G) void pa_q_join_kernel(PaArgs a) {
    __shared__ float sh[G][64];
    const int all = pa_unit<ROWS>(a, 0).all;
    const long long n = (long long)a.L * a.E;
    if constexpr (G == 1) {
        for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
            float s = 0.f;
#pragma unroll 4
            for (int k = 0; k < all; ++k) s += a.dq[k * n + i];
            ((T*)a.dQ)[i] = (T)s;
        }
    } else {
        const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, per = (all + G - 1) / G;
        const long long i = (long long)blockIdx.x * 64 + lane;
        float s = 0.f;
        if (i < n)
#pragma unroll 8
            for (int k = w * per; k < min(all, (w + 1) * per); ++k) s += a.dq[k * n + i];
        sh[w][lane] = s;
        __syncthreads();
        if (w > 0 || i >= n) return;
#pragma unroll
        for (int k = 1; k < G; ++k) s += sh[k][lane];
        ((T*)a.dQ)[i] = (T)s;
    }
}

// --------------------------------------------------------------------------------------------------------------- launch
template <class K, class G, int W, int OCC, int CAP, bool DROP>
static int pa_fwd(PaArgs& a, hipStream_t st) {
    typedef typename K::T T;
    if constexpr (W == 8) if (a.nLT == 1) {
        hipLaunchKernelGGL((pa_fwd_direct_kernel<K, G, W, CAP, DROP>), dim3(a.B + a.extra), dim3(W * 64), 2 * G::FWD * 1024, st, a);
    }
    if (W != 8 || a.nLT > 1) {
        hipLaunchKernelGGL((pa_pack_kernel<K, G, false>), dim3(a.slots + a.nQ), dim3(256), 0, st, a);
        hipLaunchKernelGGL((pa_fwd_kernel<K, G, W, OCC, CAP, DROP>), dim3(a.nLT * (a.B + a.extra)), dim3(W * 64), 2 * G::FWD * 1024, st, a);
    }
    if (a.extra > 0) {
        if ((long long)a.B * a.L <= 1024) hipLaunchKernelGGL((pa_join_kernel<T, G::ROWS, 16>), dim3(a.B * a.L), dim3(1024), 0, st, a);
        else hipLaunchKernelGGL((pa_join_kernel<T, G::ROWS, 1>), dim3(a.B * cdiv(a.L, 4)), dim3(256), 0, st, a);
    }
    GZSL_CHECK_LAUNCH();
    return 0;
}
template <class K, class G, int W, int H, int CAP, bool DROP>
static int pa_bwd(PaArgs& a, const PaPlan& p, hipStream_t st) {
    typedef typename K::T T;
    constexpr int lds = 2 * (G::QRY + G::OUT) * 1024;
    static_assert(lds <= 160 * 1024 && 2 * H * G::TOK <= 160 && 2 * G::FWD <= 160, "two buffers in LDS");
    hipLaunchKernelGGL((pa_pack_kernel<K, G, true>), dim3(a.slots + a.nQ), dim3(256), 0, st, a);
    hipLaunchKernelGGL((pa_pack_do_kernel<K, G>), dim3(a.nQ * a.B), dim3(256), 0, st, a);
    if (p.units > 0) {
        if constexpr (G::PL == 3) {
            hipLaunchKernelGGL((pa_bwd_kv_kernel<K, G, 1, CAP, DROP>), dim3(p.units), dim3(PA_TILE * 4), lds, st, a);
            hipLaunchKernelGGL((pa_bwd_kv_kernel<K, G, 2, CAP, DROP>), dim3(p.units), dim3(PA_TILE * 4), lds, st, a);
        } else {
            hipLaunchKernelGGL((pa_bwd_kv_kernel<K, G, 3, CAP, DROP>), dim3(p.units), dim3(PA_TILE * 4), lds, st, a);
        }
    }
    // (a workgroup's rows repeat every gridDim.x: of many notes and one long one most workgroups would find none)
    const int gx = cdiv(a.max_len, a.join_rows), most = 65536 / (a.B + 1) + 1;
    hipLaunchKernelGGL(pa_kv_finish_kernel<T>, dim3(gx < 1 ? 1 : (gx < most ? gx : most), a.B + 1), dim3(256), 0, st, a);
    hipLaunchKernelGGL((pa_bwd_q_kernel<K, G, W, H, CAP, DROP>), dim3(a.nLT * (a.B + a.extra)), dim3(W * H * 64), 2 * H * G::TOK * 1024, st, a);
    const long long n = (long long)a.L * a.E;
    if (n <= 64 * 512 && a.B + a.extra > 32) hipLaunchKernelGGL((pa_q_join_kernel<T, G::ROWS, 16>), dim3((unsigned)cdiv((long)n, 64)), dim3(1024), 0, st, a);
    else hipLaunchKernelGGL((pa_q_join_kernel<T, G::ROWS, 1>), dim3((unsigned)(n < 256 * 4096 ? cdiv((long)n, 256) : 4096)), dim3(256), 0, st, a);
    GZSL_CHECK_LAUNCH();
    return 0;
}
// f(how scores are capped, whether weights are dropped)
template <class K, class F>
static int pa_form(const PaArgs& a, F&& f) {
    auto drop = [&](auto cap) { return a.thresh ? f(cap, std::true_type{}) : f(cap, std::false_type{}); };
    if (a.cap == 0.f) return drop(std::integral_constant<int, PA_NONE>{});
    if constexpr (sizeof(typename K::T) == 2)
        if (a.cap <= PA_CLOSED) return drop(std::integral_constant<int, PA_FORM>{});
    return drop(std::integral_constant<int, PA_SERIES>{});
}
// W waves, OCC waves a SIMD asked of the compiler
template <class K, class G, int W, int OCC>
static int pa_go_fwd(PaArgs& a, hipStream_t st) {
    return pa_form<K>(a, [&](auto cap, auto drop) { return pa_fwd<K, G, W, OCC, decltype(cap)::value, decltype(drop)::value>(a, st); });
}
template <class K, class G, int W, int H>
static int pa_go_bwd(PaArgs& a, const PaPlan& p, hipStream_t st) {
    return pa_form<K>(a, [&](auto cap, auto drop) { return pa_bwd<K, G, W, H, decltype(cap)::value, decltype(drop)::value>(a, p, st); });
}
