// Label-wise attention over packed notes, forward and backward, for fp32 and bf16 tensors (gfx950).
//
//     x[l,t] = <q_l, k_t>;   y = cap tanh(x / cap)  (cap = 0: y = x);   P[l,t] = softmax of y[l,.] over the note's own tokens
//     O[b,l] = sum_t drop(P[l,t]) v_t;   lse[b,l] = log sum_t exp y[l,t]           (a note of no tokens: O = 0, lse = -inf)
//     backward, with delta = <dO, O>:  dV_t += drop(P) dO_l;   dS = P (drop(<dO_l, v_t>) - delta) (1 - (y / cap)^2);
//                                      dK_t = sum_l dS q_l;    dQ_l = sum_{b,t} dS k_t
//
// One set of kernels, three kinds of product:
//   PaBF   bf16 tensors: v_mfma_f32_16x16x32_bf16.
//   PaX3   fp32 tensors, E <= 112: every operand is split exactly into three bf16 pieces (8 significant bits each) and a product is
//          the six cross terms of weight >= 2^-16 of them (what is dropped is below 2^-24 of the product), each the same MFMA:
//          6 x 16 cycles per 32 k against 8 x 32 of the fp32 MFMA.
//   PaF32  fp32 tensors, E > 112 (three pieces of both tiles no longer fit LDS twice): v_mfma_f32_16x16x4_f32, exact.
// Sums are fp32 in all of them.  P and dS of bf16 tensors enter their products in two bf16 pieces (16 bits, one more product each).  With
// P in one, a score row whose pooled values cancel was off by many times its own rounding (values of both signs, 517 tokens: 3.3e-4 for
// 0.8e-4), and O 1.0 to 1.3 times as far off as a rounded exact result where they do not; dS sums to zero over a row, so its products cancel
// always, and delta = <dO, O> has to be that of the same P: dK and dQ were up to 2.4 times as far off, dV 1.4 times.  So all are within a
// hundredth of rounded exact results (forward of 19309 tokens x 9000 labels 139 -> 172 us, of 17404 x 1999 labels of 200 50 -> 60, dK / dV
// there 88 -> 98).
//
// Everything is moved as FRAGMENTS: 1 KB, 16 bytes a lane, exactly one operand of one matrix instruction (eight bf16 of a lane;
// four fp32, which feed four instructions).  With n = lane & 15, g = lane >> 4:
//   row fragment (u, s) of a tile [row][k]:  row 16 u + n, 16 bytes of k from 64 s + 16 g (bytes)
//   column fragment (j) of the same tile:    column 16 j + n, its rows 4 g + i (bf16: and 16 + 4 g + i): exactly the order in which
//                                            the accumulator registers of the tile's 16 x 16 score tiles hold their rows, so P and
//                                            dS go from accumulator to operand without touching LDS.
// A pre-pass writes the operands as tile images made of such fragments (a tile: the rows of one k step of the second product, 32,
// or 16 of PaF32), zero-filled past the note's end, past the last label and past E / F.  The sweeps copy images by LDS-DMA and read
// them 16 bytes a lane at one address plus constants, free of bank conflicts without padding; odd widths, row pitches, alignment
// and whatever lies between the notes (NaN included) end in the pre-pass.  The backward
// takes the column fragments of bf16 pieces out of the row fragments with ds_read_b64_tr_b16, PaX3 all of them for lack of LDS, PaBF
// those of the keys (dQ 87 -> 78 us at 17404 tokens x 1999 labels of 200; of the labels' tiles it was no gain).  A tenth to a third of
// their LDS cycles are bank conflicts; lanes exchanged in the images to avoid them cost the 16-byte reads more (dK / dV 88 -> 111 us).
#pragma once
#include "packed.h"
#include "rng.h"
#include "../../include/gzsl_hip.h"

#define PA_LOG2E 1.4426950408889634f
#define PA_LN2 0.6931471805599453f
#define PA_TILE 128  // tokens of a workgroup in the dK / dV sweep

struct PaF32 {
    typedef float T;
    typedef float M;  // element of a fragment
    typedef f32x4 frag;
    static constexpr int PL = 1;
};
struct PaBF {
    typedef bf16 T;
    typedef bf16 M;
    typedef bf16x8 frag;
    static constexpr int PL = 1;
};
struct PaPieces {
    bf16x8 p[3];
};
struct PaX3 {
    typedef float T;
    typedef bf16 M;
    typedef PaPieces frag;
    static constexpr int PL = 3;
};

// NE / NF: 16-wide tiles of the key / value width (E <= 16 NE, F <= 16 NF).  Sizes in KB = fragments.
template <class K, int NE_, int NF_>
struct PaGeo {
    static constexpr int NE = NE_, NF = NF_, PL = K::PL, SZ = sizeof(typename K::M), KF = 16 / SZ, KK = 4 * KF, ROWS = KK, U = ROWS / 16;
    static constexpr int SE = (NE * 16 + KK - 1) / KK, SF = (NF * 16 + KK - 1) / KK;  // k steps over e / f
    static constexpr int RE = U * SE, RF = U * SF;                                    // row fragments of a tile (one plane)
    static constexpr bool TRT = SZ == 2, TRL = PL == 3;                               // backward, columns of token and label tiles: by transposed reads
    static constexpr int FWD = PL * (RE + NF);                                        // token tile, forward: keys by rows, values by columns
    static constexpr int TOK = PL * (RE + RF) + (TRT ? 0 : NE);                        // token tile, backward: keys, values by rows, keys by columns
    static constexpr int QRY = PL * RE + (TRL ? 0 : NE);                               // label tile: queries by rows (and columns)
    static constexpr int OUT = PL * RF + (TRL ? 0 : NF) + 1;                           // label tile: dO by rows (and columns), then off, scale, delta
};

__device__ __forceinline__ f32x4 pa_mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = mfma16(a[j], b[j], c);
    return c;
}
__device__ __forceinline__ f32x4 pa_mma(bf16x8 a, bf16x8 b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x4 pa_mma(const PaPieces& a, const PaPieces& b, f32x4 c) {  // smallest terms first
    c = pa_mma(a.p[2], b.p[0], c);
    c = pa_mma(a.p[0], b.p[2], c);
    c = pa_mma(a.p[1], b.p[1], c);
    c = pa_mma(a.p[1], b.p[0], c);
    c = pa_mma(a.p[0], b.p[1], c);
    return pa_mma(a.p[0], b.p[0], c);
}

// Fragment i of `count` (a plane) at `img`; planes follow one another.
template <class K, int COUNT>
__device__ __forceinline__ typename K::frag pa_frag(const char* img, int i, int lane) {
    if constexpr (K::PL == 1) {
        return *reinterpret_cast<const typename K::frag*>(img + i * 1024 + lane * 16);
    } else {
        PaPieces f;
#pragma unroll
        for (int p = 0; p < 3; ++p) f.p[p] = *reinterpret_cast<const bf16x8*>(img + (p * COUNT + i) * 1024 + lane * 16);
        return f;
    }
}
// Column fragment j out of the row fragments (SK k steps, U = 2) of a tile.  Row r, columns 16 j + 4 q .. + 3 lie in k step j / 2, lane
// (16 (2 (j & 1) + q / 2) + r), bytes 8 (q & 1); the transposed read gives lane n of a 16-lane group column n of its 4 x 16 block.
template <class K, int SK>
__device__ __forceinline__ typename K::frag pa_col_tr(const char* img, int j, int n, int g) {
    const int r = 4 * g + (n >> 2), q = n & 3;
    const char* at = img + (j >> 1) * 1024 + ((2 * (j & 1) + (q >> 1)) * 16 + r) * 16 + 8 * (q & 1);
    bf16x8 f[K::PL];
#pragma unroll
    for (int p = 0; p < K::PL; ++p) {
        const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GZ_LDS s16x4*)(at + p * 2 * SK * 1024));
        const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GZ_LDS s16x4*)(at + (p * 2 + 1) * SK * 1024));
        f[p] = __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
    }
    return __builtin_bit_cast(typename K::frag, f);
}
// accumulator registers of the tile's score tiles -> operand fragment
__device__ __forceinline__ void pa_pack(const float (&p)[1][4], f32x4& out) { out = f32x4{p[0][0], p[0][1], p[0][2], p[0][3]}; }
__device__ __forceinline__ void pa_pack(const float (&p)[2][4], bf16x8& out) {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = (bf16)p[j >> 2][j & 3];
}
__device__ __forceinline__ void pa_split(float x, bf16& h, bf16& m, bf16& l) {  // x = h + m + l
    h = (bf16)x;
    const float r = x - (float)h;
    m = (bf16)r;
    l = (bf16)(r - (float)m);
}
// An input of any value.  An infinity as (+-1, 0, +-inf): it meets the other operand's first piece alone, whose sign is the number's, and
// not the lower ones, which may be zero or of the other sign; two infinities meet twice, with one sign.  What would round to an
// infinity is cut instead.
#define PA_ROUNDS_OVER 0x1.ffp127f  // the least number that rounds to an infinite bf16
__device__ __forceinline__ void pa_split_any(float x, bf16& h, bf16& m, bf16& l) {
    if (fabsf(x) == INFINITY) {
        h = (bf16)copysignf(1.f, x), m = (bf16)0.f, l = (bf16)x;
    } else if (fabsf(x) >= PA_ROUNDS_OVER) {
        const float c = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u), r = x - c;
        h = (bf16)c, m = (bf16)r, l = (bf16)(r - (float)m);
    } else {
        pa_split(x, h, m, l);
    }
}
__device__ __forceinline__ void pa_pack(const float (&p)[2][4], PaPieces& out) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        bf16 h, m, l;
        pa_split(p[j >> 2][j & 3], h, m, l);
        out.p[0][j] = h, out.p[1][j] = m, out.p[2][j] = l;
    }
}
// Weights p >= 0 in two pieces that are positive where p is, so that an infinite value stays one: the first cut, not rounded, the
// second with 2^-23 p on top (it stays within 2^-16 p).
__device__ __forceinline__ void pa_pack_two(const float (&p)[2][4], bf16x8& hi, bf16x8& lo) {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const float x = p[j >> 2][j & 3], c = __uint_as_float(__float_as_uint(x) & 0xFFFF0000u);
        hi[j] = (bf16)c, lo[j] = (bf16)fmaf(x, 1.f + 0x1p-23f, -c);
    }
}
// what rounding to bf16 dropped
__device__ __forceinline__ void pa_pack_low(const float (&p)[2][4], bf16x8& out) {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = (bf16)(p[j >> 2][j & 3] - (float)(bf16)p[j >> 2][j & 3]);
}

// N fragments through a ring of D: a fragment's read is issued D products ahead of its use and kept there (left alone, the
// compiler reads each one right before its product and waits for it).  ld(i) reads, use(i, f) multiplies.
template <int N, int D, class F, class LD, class USE>
__device__ __forceinline__ void pa_run_ring(F (&ring)[D], LD&& ld, USE&& use) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
        use(i, ring[i % D]);
        if (i + D < N) ring[i % D] = ld(i + D);
        __builtin_amdgcn_sched_barrier(0);
    }
}
template <int N, int D, class F, class LD>
__device__ __forceinline__ void pa_fill_ring(F (&ring)[D], LD&& ld) {
#pragma unroll
    for (int i = 0; i < D && i < N; ++i) ring[i] = ld(i);
    __builtin_amdgcn_sched_barrier(0);
}

enum { PA_NONE = 0, PA_FORM = 1, PA_SERIES = 2 };  // how scores are capped: pa_scores
// 2^ of a difference of scores: in units of log 2, or (no cap) of 1
template <int CAP>
__device__ __forceinline__ float pa_exp(float d) {
    return __builtin_amdgcn_exp2f(CAP ? d : d * PA_LOG2E);
}
struct PaCap {
    float inv, k1, c2, kt;  // 1 / cap, 2 log2(e) / cap, cap log2(e), 1 / (cap log2(e))
};
__device__ __forceinline__ PaCap pa_cap(float cap) {
    const float inv = cap > 0.f ? 1.f / cap : 0.f;
    return {inv, 2.f * PA_LOG2E * inv, cap * PA_LOG2E, PA_LN2 * inv};
}
__device__ __forceinline__ float pa_far(float x, const PaCap& c) {  // cap log2(e) tanh(x / cap) = cap log2(e) (1 - 2 / (1 + e^{2 x / cap}))
    return fmaf(__builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * c.k1)), -2.f * c.c2, c.c2);
}
#define PA_NEAR 0.35f
// How scores are capped (the kernels' CAP):
//   1  the closed form: exact limits at +-inf, absolute error of a few 2^-24 cap log2(e).  bf16 tensors with a cap of at most PA_CLOSED,
//      whose weights it leaves as good as their two pieces do.
//   2  the odd series below |x / cap| = 0.35 (the next term is below 2^-26 of the value) and the closed form only where a wave's tile
//      holds a larger one: an error relative to the score, whatever the cap.  fp32 tensors, whose products of the gradient still have
//      that accuracy, and larger caps, at which the closed form's error grows past the scores (at 1e6 weights were off by a fifth).
//      For small caps of bf16 it is the longer way: 180 us against 176 for 19309 tokens x 9000 labels.
#define PA_CLOSED 64.f
// Scores x of a tile -> y = cap tanh(x / cap) in units of log 2, and th = tanh(x / cap) for the gradient.  Without a cap y is x itself, and
// maxima stay in its units: in those of log 2 a row of the type's lowest values would run over.
template <int CAP, int U, bool TH>
__device__ __forceinline__ void pa_scores(const f32x4 (&x)[U], const PaCap& c, float (&y)[U][4], float (&th)[U][4]) {
    float most = 0.f;
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            if (CAP == PA_NONE) {
                y[u][r] = x[u][r];
            } else if (CAP == PA_FORM) {
                y[u][r] = pa_far(x[u][r], c);
            } else {
                const float v = x[u][r] * c.inv, w = v * v;
                most = fmaxf(most, fabsf(v));  // (a NaN passes it by and stays one in the series)
                float t = fmaf(w, -1382.f / 155925.f * PA_LOG2E, 62.f / 2835.f * PA_LOG2E);
                t = fmaf(w, fmaf(w, fmaf(w, fmaf(w, t, -17.f / 315.f * PA_LOG2E), 2.f / 15.f * PA_LOG2E), -1.f / 3.f * PA_LOG2E), PA_LOG2E);
                y[u][r] = x[u][r] * t;
            }
        }
    if (CAP == PA_SERIES && __any(most >= PA_NEAR)) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (fabsf(x[u][r] * c.inv) >= PA_NEAR) y[u][r] = pa_far(x[u][r], c);
    }
    if (CAP && TH)
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) th[u][r] = y[u][r] * c.kt;
}

// Copies KB KB of a tile image into LDS: 1 KB per wave instruction, spread over the workgroup's waves.  `src` and `wave` are scalars.
// The caller waits with pa_arrive() before anyone reads.  (Buffer loads: after the global form the compiler takes every LDS read for
// one that may return out of order and waits for all of them each time.)
template <int WAVES, int KB>
__device__ __forceinline__ void pa_dma(const char* src, char* dst, int wave, int lane) {
    const __amdgpu_buffer_rsrc_t from = __builtin_amdgcn_make_buffer_rsrc(const_cast<char*>(src), 0, KB * 1024, 0x00020000);
#pragma unroll
    for (int i = 0; i < (KB + WAVES - 1) / WAVES; ++i) {
        const int o = (wave + i * WAVES) * 1024;
        if (KB % WAVES == 0 || i < KB / WAVES || o < KB * 1024)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (GZ_LDS void*)(dst + o), 16, 16 * lane, o, 0, 0);
    }
}
__device__ __forceinline__ int pa_scalar(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ long long pa_scalar(long long x) {
    return (long long)(uint32_t)pa_scalar((int)x) | (long long)pa_scalar((int)(x >> 32)) << 32;
}
// this wave's copies have landed, all but the newest LEFT of them, and every wave is past its reads of the other buffers
template <int LEFT = 0>
__device__ __forceinline__ void pa_arrive() {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"(LEFT) : "memory");
    __syncthreads();
}

struct PaArgs {
    const void *keys, *values, *queries;
    const int64_t* spans;
    long long rows, ldk, ldv, ldq;
    int B, max_len, L, E, F, nT, nQ;  // nT: token tiles of the longest note (0: images by rows, see pa_images), nQ: label tiles
    int slots;                        // token tiles that have an image
    float cap;
    uint32_t l_offset, L_total, seed, thresh;
    float scale;
    int join_rows;                    // rows of a workgroup of pa_kv_finish_kernel
    int nLT, extra, least;            // label workgroups of a note; token chunks beyond one a note (0: notes are not cut), their tokens at least
    // workspace
    char *TK, *Q, *DO;  // images: token tiles [slots], queries [nQ], dO [B][nQ]
    float *part, *ml;  // forward, notes cut: unnormalised O [chunk][L][F] and (max, sum) [chunk][L][2]
    float *dq, *dkv;   // backward: [chunk][L][E]; [slab][PA_TILE][E + F]
    // results and the backward's inputs
    void* O;
    float *LSE, *rest;  // rest: (max in the scores' units, 1 / sum) [B][L][2], then for bf16 what the rounding of O dropped, [B][L][F]
    const void *cO, *dO;
    const float *cLSE, *crest;
    void *dK, *dV, *dQ;
};

// ---- where a token tile's image lies.  [B][nT] where that is at most PA_WASTE times what disjoint notes can fill.  Otherwise, of notes of
// very different lengths (512 notes of 200000 rows, one of 65536: 67 GB), by rows: a note's first tile at [b], its tile t behind B at
// start / ROWS + t - 1.  Of disjoint notes no two meet there, in whatever order the table has them: the row in front of a tile t > 0 is
// its own note's, and so is every row of ROWS in front, so no other tile t > 0 begins in the same ROWS rows.
#define PA_WASTE 4
struct PaImages {
    const char *first, *rest;
    long long bytes;
    __device__ __forceinline__ const char* operator()(int t) const { return (t ? rest : first) + t * bytes; }
};
template <int ROWS>
__device__ __forceinline__ PaImages pa_images(const PaArgs& a, int b, long long start, int kb) {
    PaImages m;
    m.bytes = 1024LL * kb;
    m.rest = a.TK + (a.nT ? (long long)b * a.nT : a.B + start / ROWS - 1) * m.bytes;
    m.first = a.nT ? m.rest : a.TK + b * m.bytes;
    return m;
}

// ---- how the work is cut.  The host knows max_len, not the lengths: every wave works the cut out from the span table, so the
// kernels agree on it without a table in memory.  Per 64 notes: one load and a few lane exchanges.
struct PaUnit {
    int b, c, nch;        // note, its chunk, the note's chunks
    int chunk, ci, all;   // tokens of a chunk, number of this chunk among all, chunks in all
    NoteSpan sp;
};
// Chunks of ROWS-aligned `chunk` tokens, about a.extra of them beyond one a note.  Up to 64 notes are taken longest first, so
// that the last workgroups of the grid are the short ones; more notes are taken in their order.
template <int ROWS>
__device__ __forceinline__ PaUnit pa_unit(const PaArgs& a, int ci, int want_b = -1) {
    const int lane = threadIdx.x & 63;
    PaUnit u;
    u.ci = ci;
    u.b = -1;
    int chunk = 0x7FFFFFC0;
    auto span = [&](int b) { return b < a.B ? note_span(a.spans, b, a.rows, a.max_len) : NoteSpan{0, 0}; };
    NoteSpan sp = span(lane);
    if (a.extra > 0) {
        long long n = sp.len;
        for (int b0 = 64; b0 < a.B; b0 += 64) n += span(b0 + lane).len;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
        long long per = (n + a.extra - 1) / a.extra;
        if (per < a.least) per = a.least;
        chunk = (int)min(per / ROWS * ROWS + ROWS, (long long)0x7FFFFFC0);
    }
    chunk = pa_scalar(chunk);
    u.chunk = chunk;
    int base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        if (b0) sp = span(b0 + lane);
        int note = b0 + lane, len = sp.len;
        if (a.B <= 64) {  // order by length, longest first (ties: lower note first)
            int rank = 0;
            for (int j = 0; j < a.B; ++j) {
                const int other = __builtin_amdgcn_readlane(len, j);
                rank += other > len || (other == len && j < lane);
            }
            if (lane >= a.B) rank = lane;
            note = __builtin_amdgcn_ds_permute(rank << 2, note);
            len = __builtin_amdgcn_ds_permute(rank << 2, len);
        }
        const int nch = note < a.B ? max(1, (int)(((uint32_t)len + (uint32_t)chunk - 1) / (uint32_t)chunk)) : 0;
        int incl = nch;  // chunks up to and with this lane
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned long long hit = want_b >= 0 ? __ballot(note == want_b) : __ballot(base + incl > ci);
        if (u.b < 0 && hit) {
            const int src = __ffsll((long long)hit) - 1;
            u.b = pa_scalar(__shfl(note, src));
            u.nch = pa_scalar(__shfl(nch, src));
            const int first = base + pa_scalar(__shfl(incl, src)) - u.nch;
            u.c = ci - first;
            if (want_b >= 0) u.c = 0, u.ci = first;
            u.sp = {pa_scalar(__shfl(sp.start, u.b - b0)), pa_scalar(__shfl(len, src))};
        }
        base += pa_scalar(__shfl(incl, 63));
    }
    u.all = base;
    return u;
}
// dK / dV: the steps of the sweep, token tile by token tile (PA_TILE tokens x the label tiles), in PA_UNITS equal runs, one for each
// compute unit (less where a run would be under PA_RUN steps): every compute unit works for the same time, and only the tiles at a run's
// two ends are shared and go through slabs (2 u for one that the run begins inside of, 2 u + 1 for the one that it ends in).  With
// equal parts of a tile instead, as many as a cost rule found best, 17404 tokens x 1999 labels of 200 bf16 (weights in one piece) took
// 99 us, so 88; x 9000 labels, with their slabs' join, 415 and 380.
#define PA_UNITS 256
#define PA_RUN 2  // steps of a run, at least (of 4: 60 us against 35 of its two launches for 1000 tokens x 428 labels, fp32)
struct PaTile {
    int b, tile;  // note, token tile in it
    NoteSpan sp;
};
__device__ __forceinline__ int pa_tiles(int len) { return (int)(((uint32_t)len + PA_TILE - 1) / PA_TILE); }
// Token tiles of all notes, and of those in front of note b.
__device__ __forceinline__ long long pa_all_tiles(const PaArgs& a, int b, long long& before) {
    const int lane = threadIdx.x & 63;
    long long n = 0, m = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int t = b0 + lane < a.B ? pa_tiles(note_span(a.spans, b0 + lane, a.rows, a.max_len).len) : 0;
        n += t;
        m += b0 + lane < b ? t : 0;
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o), m += __shfl_xor(m, o);
    before = pa_scalar(m);
    return pa_scalar(n);
}
// Token tile i of all.
__device__ __forceinline__ PaTile pa_tile(const PaArgs& a, int i) {
    const int lane = threadIdx.x & 63;
    PaTile u;
    u.b = -1;
    int base = 0;
    for (int b0 = 0; b0 < a.B && u.b < 0; b0 += 64) {
        const NoteSpan sp = b0 + lane < a.B ? note_span(a.spans, b0 + lane, a.rows, a.max_len) : NoteSpan{0, 0};
        const int nt = pa_tiles(sp.len);
        int incl = nt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned long long hit = __ballot(base + incl > i);
        if (hit) {
            const int src = __ffsll((long long)hit) - 1;
            u.b = b0 + src;
            u.tile = i - base - pa_scalar(__shfl(incl, src) - __shfl(nt, src));
            u.sp = {pa_scalar(__shfl(sp.start, src)), pa_scalar(__shfl(sp.len, src))};
        }
        base += pa_scalar(__shfl(incl, 63));
    }
    return u;
}
// The token tile whose image is at `slot` (b = -1: none).
template <int ROWS>
__device__ __forceinline__ PaTile pa_slot(const PaArgs& a, int slot) {
    PaTile u;
    u.b = -1;
    if (a.nT || slot < a.B) {
        u.b = a.nT ? slot / a.nT : slot, u.tile = a.nT ? slot % a.nT : 0;
        u.sp = note_span(a.spans, u.b, a.rows, a.max_len);
        if ((long long)u.tile * ROWS >= u.sp.len) u.b = -1;
        return u;
    }
    const int lane = threadIdx.x & 63;
    const long long cell = slot - a.B + 1;
    for (int b0 = 0; b0 < a.B && u.b < 0; b0 += 64) {
        const NoteSpan sp = b0 + lane < a.B ? note_span(a.spans, b0 + lane, a.rows, a.max_len) : NoteSpan{0, 0};
        const long long t = cell - sp.start / ROWS;
        const unsigned long long hit = __ballot(t > 0 && t * ROWS < sp.len);
        if (hit) {
            const int src = __ffsll((long long)hit) - 1;
            u.b = b0 + src;
            u.sp = {pa_scalar(__shfl(sp.start, src)), pa_scalar(__shfl(sp.len, src))};
            u.tile = (int)(cell - u.sp.start / ROWS);
        }
    }
    return u;
}
struct PaRuns {
    int steps, per, units;  // in all, of a run (the last may be shorter), runs
    __device__ __forceinline__ PaRuns(long long tiles, int nQ) {
        // The host has seen that the steps of disjoint notes fit; of a table that is not, nothing is done where they do not.
        steps = tiles <= 0x7FFFFF00 / nQ ? (int)tiles * nQ : 0;
        per = max(PA_RUN, (steps - 1) / PA_UNITS + 1);
        units = (steps + per - 1) / per;
    }
};

struct PaPlan {
    long long slots;
    int max_len, nT, nQ, kind, waves, extra, least, units, nLT;  // kind: 0 PaBF, 1 PaBF wide, 2 PaX3, 3 PaF32 (wide: E > 112)
    long long kv, q, dO, part, ml, dq, dkv, bytes;
};
// packed_attn_bf16.hip, packed_attn_x3.hip, packed_attn_f32.hip
int pa_run_bf16(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st);
int pa_run_x3(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st);
int pa_run_f32(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st);
