// Label-wise attention over packed notes, forward and backward, for fp32 and bf16 tensors (gfx950).
//
//     x[l,t] = <q_l, k_t>;   y = cap tanh(x / cap)  (cap = 0: y = x);   P[l,t] = softmax of y[l,.] over the note's own tokens
//     O[b,l] = sum_t drop(P[l,t]) v_t;   lse[b,l] = log sum_t exp y[l,t]           (a note of no tokens: O = 0, lse = -inf)
//     backward, with delta = <dO, O>:  dV_t += drop(P) dO_l;   dS = P (drop(<dO_l, v_t>) - delta) (1 - (y / cap)^2);
//                                      dK_t = sum_l dS q_l;    dQ_l = sum_{b,t} dS k_t
//
// One set of kernels serves both types.  A "fragment" is 16 bytes per lane: eight bf16 (one v_mfma_f32_16x16x32_bf16) or
// four fp32 (four v_mfma_f32_16x16x4_f32, exact), so a k step of 64 bytes and every LDS offset are the same for both.
//   row fragment of an image [row][k]:   lane (n = lane & 15, g = lane >> 4) holds row n, bytes 64 s + 16 g .. + 15
//   column fragment of the same image (k down the rows): bf16 by ds_read_b64_tr_b16 (k order 16 h + 4 g + j), fp32 by four
//   ds_read_b32 (k = 4 g + j): exactly the order in which the accumulator registers of two (one) 16 x 16 score tiles hold
//   their rows, so P and dS go from accumulator to operand without touching LDS.
// Sums are fp32.  P is rounded to the tensors' type for its products (bf16: half a step of 2^-8, as the inputs' own rounding;
// nothing for fp32); the softmax sum uses P before that rounding.  dS sums to zero over a row, so its products cancel: as one
// bf16 piece it made dK and dQ 1.6 times as far off as rounded results are, so it goes in two (16 bits, one more product).
//
// A pre-pass writes the operands as TILE IMAGES of 32 rows that are byte for byte the LDS layout (row pitch 64 s + 32 bytes:
// conflict-free for both ways of reading), zero-filled past the note's end, past the last label and past E / F.  The sweeps
// then copy whole tiles by LDS-DMA, and odd widths, row pitches, alignment and whatever lies between the notes
// (NaN included) end in the pre-pass.
#pragma once
#include "packed.h"
#include "rng.h"
#include "../../include/gzsl_hip.h"

#define PA_LOG2E 1.4426950408889634f
#define PA_LN2 0.6931471805599453f
#define PA_TILE 64  // tokens of a workgroup in the dK / dV sweep

template <typename T>
struct PaTy;
template <>
struct PaTy<float> {
    typedef f32x4 frag;
};
template <>
struct PaTy<bf16> {
    typedef bf16x8 frag;
};

// NE / NF: 16-wide tiles of the key / value width (E <= 16 NE, F <= 16 NF).  A tile image holds one k step of the second
// product: 32 rows of bf16, 16 of fp32.
template <typename T, int NE_, int NF_>
struct PaGeo {
    static constexpr int NE = NE_, NF = NF_, SZ = sizeof(T), KF = 16 / SZ, ROWS = 4 * KF, U = ROWS / 16;
    static constexpr int SE = (NE * 16 * SZ + 63) / 64, SF = (NF * 16 * SZ + 63) / 64;  // 64-byte k steps over e / f
    static constexpr int PE = 64 * SE + 32, PF = 64 * SF + 32;                          // row pitches in bytes
    static constexpr int EB = ROWS * PE, FB = ROWS * PF;
    static constexpr int KV = EB + FB;                                  // token tile: keys, values
    static constexpr int QB = (EB + 1023) / 1024 * 1024;                // label tile: queries
    static constexpr int OB = (FB + 12 * ROWS + 1023) / 1024 * 1024;    // label tile: dO rows, then off[], scale[], delta[] of its labels
    static_assert(KV % 1024 == 0, "whole KB: the copies move 1 KB per wave instruction");
};

__device__ __forceinline__ f32x4 pa_mma(f32x4 a, f32x4 b, f32x4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = mfma16(a[j], b[j], c);
    return c;
}
__device__ __forceinline__ f32x4 pa_mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

template <typename T>
__device__ __forceinline__ typename PaTy<T>::frag pa_row(const char* img, int pitch, int row0, int s, int n, int g) {
    return *reinterpret_cast<const typename PaTy<T>::frag*>(img + (row0 + n) * pitch + 64 * s + 16 * g);
}
template <typename T>
__device__ __forceinline__ typename PaTy<T>::frag pa_col(const char* img, int pitch, int row0, int col0, int n, int g);
template <>
__device__ __forceinline__ f32x4 pa_col<float>(const char* img, int pitch, int row0, int col0, int n, int g) {
    f32x4 v;
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = *reinterpret_cast<const float*>(img + (row0 + 4 * g + j) * pitch + 4 * (col0 + n));
    return v;
}
template <>
__device__ __forceinline__ bf16x8 pa_col<bf16>(const char* img, int pitch, int row0, int col0, int n, int g) {
    const char* p = img + (row0 + 4 * g + (n >> 2)) * pitch + 2 * col0 + 8 * (n & 3);
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GZ_LDS s16x4*)p);
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((GZ_LDS s16x4*)(p + 16 * pitch));
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
}
// accumulator registers of the tile's 16-row score tiles -> operand fragment
__device__ __forceinline__ void pa_pack(const float (&p)[1][4], f32x4& out) {
    out = f32x4{p[0][0], p[0][1], p[0][2], p[0][3]};
}
__device__ __forceinline__ void pa_pack(const float (&p)[2][4], bf16x8& out) {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = (bf16)p[j >> 2][j & 3];
}
// what that rounding dropped
__device__ __forceinline__ void pa_pack_low(const float (&p)[2][4], bf16x8& out) {
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = (bf16)(p[j >> 2][j & 3] - (float)(bf16)p[j >> 2][j & 3]);
}

struct PaCap {
    float inv, k1, c2;  // 1 / cap, 2 log2(e) / cap, cap log2(e)
};
__device__ __forceinline__ PaCap pa_cap(float cap) {
    return {cap > 0.f ? 1.f / cap : 0.f, cap > 0.f ? 2.f * PA_LOG2E / cap : 0.f, cap * PA_LOG2E};
}
// tanh u = 1 - 2 / (1 + e^{2u}): exact limits at +-inf, absolute error of a few 2^-24.  fp32 tensors take the odd series below
// |u| = 0.35 (the next term is below 2^-26 of the value there), where the difference would lose relative accuracy that the
// products of the gradient still have.  `far` (the same in the whole wave): some lane needs the exponential.
__device__ __forceinline__ float pa_sech(float x, const PaCap& c) {  // 1 / (1 + e^{2 x / cap})
    return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(x * c.k1));
}
__device__ __forceinline__ float pa_series(float u) {
    const float w = u * u;
    return u * fmaf(w, fmaf(w, fmaf(w, fmaf(w, fmaf(w, -1382.f / 155925.f, 62.f / 2835.f), -17.f / 315.f), 2.f / 15.f), -1.f / 3.f), 1.f);
}
#define PA_NEAR 0.35f
// Scores x of a tile -> y in units of log 2 (and th = tanh(x / cap) for the gradient).
template <typename T, bool CAP, int U, bool TH>
__device__ __forceinline__ void pa_scores(const f32x4 (&x)[U], const PaCap& c, float (&y)[U][4], float (&th)[U][4]) {
    if (!CAP) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) y[u][r] = x[u][r] * PA_LOG2E;
    } else if (sizeof(T) == 2) {
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float q = pa_sech(x[u][r], c);
                y[u][r] = fmaf(q, -2.f * c.c2, c.c2);
                if (TH) th[u][r] = fmaf(q, -2.f, 1.f);
            }
    } else {
        bool near = true;
        float t[U][4];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const float v = x[u][r] * c.inv;
                near = near && fabsf(v) < PA_NEAR;  // (false for a NaN)
                t[u][r] = pa_series(v);
            }
        if (!__all(near)) {
#pragma unroll
            for (int u = 0; u < U; ++u)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!(fabsf(x[u][r] * c.inv) < PA_NEAR)) t[u][r] = fmaf(pa_sech(x[u][r], c), -2.f, 1.f);
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                y[u][r] = t[u][r] * c.c2;
                if (TH) th[u][r] = t[u][r];
            }
    }
}

// Copies `bytes` (whole KB) of a tile image into LDS: 1 KB per wave instruction, spread over the workgroup's waves.  The
// caller waits with pa_arrive() before anyone reads.
template <int WAVES>
__device__ __forceinline__ void pa_dma(const char* src, char* dst, int bytes, int wave, int lane) {
    for (int o = wave * 1024; o < bytes; o += WAVES * 1024)
        __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(src + o + 16 * lane), (GZ_LDS void*)(dst + o), 16, 0, 0);
}
// this wave's copies have landed and every wave is past its reads of the other buffer
__device__ __forceinline__ void pa_arrive() {
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
}

struct PaArgs {
    const void *keys, *values, *queries;
    const int64_t* spans;
    long long rows, ldk, ldv, ldq;
    int B, max_len, L, E, F, nT, nQ;  // nT: token tiles of the longest note, nQ: label tiles
    float cap;
    uint32_t l_offset, L_total, seed, thresh;
    float scale;
    int nLT, extra;                   // label workgroups of a note; token chunks beyond one a note (0: notes are not cut)
    int shares, slots;                // dK / dV: label shares of a token tile at most, slabs that the workspace has room for
    // workspace
    char *KV, *Q, *DO;
    float *part, *ml;  // forward, notes cut: unnormalised O [chunk][L][F] and (max, sum) [chunk][L][2]
    float *dq, *dkv;   // backward: [chunk][L][E]; [unit][PA_TILE][E + F]
    // results and the backward's inputs
    void* O;
    float *LSE, *rest;  // rest: (max in log 2, 1 / sum) [B][L][2], then for bf16 what the rounding of O dropped, [B][L][F]
    const void *cO, *dO;
    const float *cLSE, *crest;
    void *dK, *dV, *dQ;
};

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
    auto length = [&](int b) { return b < a.B ? note_span(a.spans, b, a.rows, a.max_len).len : 0; };
    int len = length(lane);
    if (a.extra > 0) {
        long long n = 0;
        for (int b0 = 0; b0 < a.B; b0 += 64) n += b0 ? length(b0 + lane) : len;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
        long long per = (n + a.extra - 1) / a.extra;
        if (per < 256) per = 256;  // a share that pays for its own start and its part in the join
        chunk = (int)min(per / ROWS * ROWS + ROWS, (long long)0x7FFFFFC0);
    }
    u.chunk = chunk;
    int base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        int note = b0 + lane;
        if (b0) len = length(note);
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
        const int nch = note < a.B ? max(1, (len + chunk - 1) / chunk) : 0;
        int incl = nch;  // chunks up to and with this lane
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned long long hit = want_b >= 0 ? __ballot(note == want_b) : __ballot(base + incl > ci);
        if (u.b < 0 && hit) {
            const int src = __ffsll((long long)hit) - 1;
            u.b = __shfl(note, src);
            u.nch = __shfl(nch, src);
            const int first = base + __shfl(incl, src) - u.nch;
            u.c = ci - first;
            if (want_b >= 0) u.c = 0, u.ci = first;
        }
        base += __shfl(incl, 63);
    }
    u.all = base;
    if (u.b >= 0) u.sp = note_span(a.spans, u.b, a.rows, a.max_len);
    return u;
}
// dK / dV: units of PA_TILE tokens x one of `shares` parts of the labels.  The parts are as many as fill the chip's 512 places
// (two workgroups a compute unit) best, a slab written and read again counted as 1 % a part.
struct PaTileUnit {
    int b, tile, share, shares, unit, tiles;
    NoteSpan sp;
};
__device__ __forceinline__ PaTileUnit pa_tile_unit(const PaArgs& a, int unit, int want_b = -1) {
    const int lane = threadIdx.x & 63;
    PaTileUnit u;
    u.b = -1;
    auto tiles_of = [&](int b) { return b < a.B ? (note_span(a.spans, b, a.rows, a.max_len).len + PA_TILE - 1) / PA_TILE : 0; };
    int n = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) n += tiles_of(b0 + lane);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
    u.tiles = n;
    u.shares = 1;
    float best = -1.f;
    for (int s = 1; s <= a.shares && (s == 1 || (long long)n * s <= a.slots); ++s) {
        const int all = n * s, rounds = (all + 511) / 512;
        const float fill = rounds > 0 ? (float)all / (512.f * rounds) - 0.01f * s : 0.f;
        if (fill > best) best = fill, u.shares = s;
    }
    u.unit = unit;
    const int t = unit / u.shares;
    u.share = unit % u.shares;
    int base = 0;
    for (int b0 = 0; b0 < a.B; b0 += 64) {
        const int nt = tiles_of(b0 + lane);
        int incl = nt;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int x = __shfl_up(incl, o);
            if (lane >= o) incl += x;
        }
        const unsigned long long hit = want_b >= 0 ? __ballot(b0 + lane == want_b) : __ballot(base + incl > t);
        if (u.b < 0 && hit) {
            const int src = __ffsll((long long)hit) - 1, first = base + __shfl(incl, src) - __shfl(nt, src);
            u.b = b0 + src;
            u.tile = want_b >= 0 ? first : t - first;  // want_b: the note's first tile among all
        }
        base += __shfl(incl, 63);
    }
    if (u.b >= 0) u.sp = note_span(a.spans, u.b, a.rows, a.max_len);
    return u;
}

struct PaPlan {
    int nT, nQ, wide, waves, extra, shares, slots, nLT;
    long long units;  // workgroups of the dK / dV sweep
    long long kv, q, dO, part, ml, dq, dkv, bytes;
};
// packed_attn_f32.hip / packed_attn_bf16.hip
int pa_run_f32(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st);
int pa_run_bf16(PaArgs& a, const PaPlan& p, bool backward, hipStream_t st);
