// Gated linear recurrence over packed notes, forward and backward, and its single-token step:
//     z = sigmoid(g);   h_t = (1 - z_t) h_{t-1} + z_t c_t          (t runs through a note's rows, or back through them)
//     backward:  lam_t = dh_t + (1 - z_{t+1}) lam_{t+1};   dc = lam z;   dg = lam (c - h_{t-1}) z (1 - z);   dh_0 = (1 - z_1) lam_1
// The states are fp32 throughout; tensors of 16 bits are widened when read and rounded once when written.  A forward that a backward
// follows also keeps what the rounding of h dropped (`rest`, 16 bits a value): c - h_{t-1} cancels where the state has settled near its
// candidate, and taken from the rounded h alone it left dg 2.7 times as far off as a rounded exact result for candidates of mean 3.
//
// Both directions are the recurrence x <- A x + B, whose steps join: (A1, B1) then (A2, B2) = (A2 A1, A2 B1 + B2).  The time axis is
// cut into chunks, one workgroup each (a thread owns V channels and S consecutive steps of a tile, all in registers):
//   1. gs_chunk_kernel reduces every chunk to its (A, B)         reads g and c (g and dh)
//   2. gs_join_kernel, where there are many chunks, joins the pairs to the state in front of each
//   3. gs_apply_kernel takes that state (or joins the pairs of the chunks before its own itself), then runs through its tiles:
//      each thread's steps to a pair, a scan of the pairs over the tile's threads in LDS, the steps again from the state in front.
// Memory-bound: 3 (6) tensors forward (backward), of which the first pass reads two once more (from the 256 MB last-level cache
// where they fit).  81600 x 256 bf16 forward: 21 + 8 + 28 us (4.0 and 4.5 TB/s in the first and the third; a copy reaches 5.1); 18388 x
// 200 fp32: 10 + 12 us, backward 9 + 21.  A workgroup takes whole rows: of narrower pieces, for more workgroups, the third took 44 for 39.
// The pairs meet in a fixed order, so results repeat bit for bit; tokens in front of a step never see it.
#include "packed.h"
#include "../../include/gzsl_hip.h"

#define GS_THREADS 256
#define GS_JTHREADS 512
#define GS_JGROUPS 4
#define GS_LOG2E 1.4426950408889634f

struct GsArgs {
    const void *g, *c;
    const int64_t* spans;
    const float* h0;
    long long rows, ldg, ldc;
    int B, max_len, H, reverse;
    void* h;
    float* last;
    bf16* rest;                              // [rows][H] or null: h - its rounding, written forward, read backward
    const void *ch, *dh;
    const float* dlast;
    void *dg, *dc;
    float* dh0;
    float* pair;                             // [B][nch][2][H]
    int joined;
    int* ascending;                          // of many notes: whether the table lists them in ascending order
    int ncg, nblk, TS, tiles, chunk, nch;    // channel groups of a workgroup, workgroups over the channels, threads over time, tiles of a chunk
};

// z = sigmoid(g) = 1 / (1 + w), a = 1 - z = w z with w = e^-g, both to a few roundings of their own size (the exponent |g| log2(e) is rounded
// once: |g| half steps): a difference 1 - z would be off by a half step of 1, which a far state multiplies.  w stops at 2^126, where its
// reciprocal is still a normal number; a gate that is no number stays one.
__device__ __forceinline__ void gs_gate(float g, float& z, float& a) {
    const float w = __builtin_amdgcn_exp2f(__builtin_elementwise_minimum(g * -GS_LOG2E, 126.f));
    z = __builtin_amdgcn_rcpf(1.f + w);
    a = w * z;
}

template <typename T, int V>
struct GsVec {
    typedef T type __attribute__((ext_vector_type(V)));
};
template <typename T>
struct GsVec<T, 1> {
    typedef T type;
};
template <typename T, int V>
__device__ __forceinline__ void gs_load(const T* p, float (&v)[V]) {
    typedef typename GsVec<T, V>::type vec;
    const vec x = *reinterpret_cast<const vec*>(p);
    if constexpr (V == 1) v[0] = (float)x;
    else
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = (float)x[i];
}
template <typename T, int V>
__device__ __forceinline__ void gs_store(T* p, const float (&v)[V]) {
    typedef typename GsVec<T, V>::type vec;
    vec x;
    if constexpr (V == 1) x = (T)v[0];
    else
#pragma unroll
        for (int i = 0; i < V; ++i) x[i] = (T)v[i];
    *reinterpret_cast<vec*>(p) = x;
}

// Inclusive scan of the threads' pairs along time (thread j of TS per channel group); returns the pair of the threads in front
// in (Ae, Be) and the whole tile's in (At, Bt).
template <int V>
__device__ __forceinline__ void gs_scan(float (&A)[V], float (&B)[V], float (&Ae)[V], float (&Be)[V], float (&At)[V], float (&Bt)[V], float* sh, int tid,
                                        int j, int TS, int ncg, int nt) {
    auto put = [&]() {
#pragma unroll
        for (int i = 0; i < V; ++i) sh[i * nt + tid] = A[i], sh[(V + i) * nt + tid] = B[i];
    };
    for (int d = 1; d < TS; d <<= 1) {
        put();
        __syncthreads();
        if (j >= d) {
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float pa = sh[i * nt + tid - d * ncg], pb = sh[(V + i) * nt + tid - d * ncg];
                B[i] = fmaf(A[i], pb, B[i]);
                A[i] *= pa;
            }
        }
        __syncthreads();
    }
    put();
    __syncthreads();
    const int lastt = tid - j * ncg + (TS - 1) * ncg;
#pragma unroll
    for (int i = 0; i < V; ++i) {
        Ae[i] = j > 0 ? sh[i * nt + tid - ncg] : 1.f;
        Be[i] = j > 0 ? sh[(V + i) * nt + tid - ncg] : 0.f;
        At[i] = sh[i * nt + lastt];
        Bt[i] = sh[(V + i) * nt + lastt];
    }
    __syncthreads();
}

// Where step i (in the order of the recurrence: forward from a note's first step, backward from its last) has its row.
template <bool BWD>
__device__ __forceinline__ long long gs_row(const NoteSpan& sp, int reverse, int i) {
    return (BWD != (reverse != 0)) ? sp.start + sp.len - 1 - i : sp.start + i;
}

struct GsPlace {
    int tid, nt, j, ch, b, k;
    bool on;
};
__device__ __forceinline__ GsPlace gs_place(const GsArgs& a, int V) {
    GsPlace p;
    p.tid = threadIdx.x, p.nt = blockDim.x;
    p.j = p.tid / a.ncg;
    p.k = blockIdx.x % a.nch;
    p.b = blockIdx.x / a.nch;
    p.ch = (blockIdx.y * a.ncg + p.tid % a.ncg) * V;
    p.on = p.ch < a.H;
    if (!p.on) p.ch = 0;
    return p;
}

// Waves a SIMD asked of the compiler where it would just miss them (81600 x 256 bf16 forward: 65 us at 5 and 2, 59 at 6 and 3).
constexpr int gs_waves(bool wide, bool bwd, bool chunk) { return wide && !bwd ? (chunk ? 6 : 3) : 1; }

template <typename T, int V, int S, bool BWD>
__global__ __launch_bounds__(GS_THREADS, gs_waves(V == 8, BWD, true)) void gs_chunk_kernel(GsArgs a) {
    extern __shared__ float sh[];
    const GsPlace p = gs_place(a, V);
    const NoteSpan sp = note_span(a.spans, p.b, a.rows, a.max_len);
    const long long first = (long long)p.k * a.chunk;
    if (first + a.chunk >= sp.len) return;  // nothing behind this chunk starts from it
    // this thread's share of the chunk: tiles * S consecutive steps, all inside the note
    const int n = a.tiles * S, i0 = (int)first + p.j * n;
    const T *x = (const T*)a.g + p.ch, *y = (BWD ? (const T*)a.dh : (const T*)a.c) + p.ch;
    const long long ldy = BWD ? a.H : a.ldc;
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
    for (int s0 = 0; s0 < n; s0 += S) {
        float g[S][V], u[S][V];
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const long long row = gs_row<BWD>(sp, a.reverse, i0 + s0 + s);
            gs_load<T, V>(x + row * a.ldg, g[s]);
            if (!BWD || a.dh) gs_load<T, V>(y + row * ldy, u[s]);
        }
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float z, k;
                gs_gate(g[s][v], z, k);
                if (BWD) B[v] = k * (B[v] + (a.dh ? u[s][v] : 0.f));
                else B[v] = fmaf(k, B[v], z * u[s][v]);
                A[v] *= k;
            }
    }
    float Ae[V], Be[V], At[V], Bt[V];
    gs_scan<V>(A, B, Ae, Be, At, Bt, sh, p.tid, p.j, a.TS, a.ncg, p.nt);
    if (p.on && p.j == 0) {
        float* out = a.pair + ((long long)p.b * a.nch + p.k) * 2 * a.H + p.ch;
#pragma unroll
        for (int v = 0; v < V; ++v) out[v] = At[v], out[a.H + v] = Bt[v];
    }
}

// The state in front of each chunk of a note, in place of its pair's A.  A workgroup takes GS_JGROUPS vectors of channels, its threads
// share out the chunks; latency-bound (512 chunks x 256 channels: 7 us; 256 or 1024 threads 9).
template <int V>
__global__ __launch_bounds__(GS_JTHREADS) void gs_join_kernel(GsArgs a, const float* init) {
    extern __shared__ float sh[];
    const int tid = threadIdx.x, cg = tid % GS_JGROUPS, j = tid / GS_JGROUPS, TS = GS_JTHREADS / GS_JGROUPS, b = blockIdx.x;
    int ch = (blockIdx.y * GS_JGROUPS + cg) * V;
    const bool on = ch < a.H;
    if (!on) ch = 0;
    const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len);
    const int n = (int)(((long long)sp.len + a.chunk - 1) / a.chunk);  // chunks of this note; the last one's pair is not there and not needed
    const int per = (n + TS - 1) / TS, q0 = min(n, j * per), q1 = min(n, q0 + per);
    float* pr = a.pair + (long long)b * a.nch * 2 * a.H + ch;
    float A[V], B[V];
#pragma unroll
    for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
#pragma unroll 8
    for (int q = q0; q < min(q1, n - 1); ++q) {
        float ka[V], kb[V];
        gs_load<float, V>(pr + (long long)q * 2 * a.H, ka);
        gs_load<float, V>(pr + (long long)q * 2 * a.H + a.H, kb);
#pragma unroll
        for (int v = 0; v < V; ++v) B[v] = fmaf(ka[v], B[v], kb[v]), A[v] *= ka[v];
    }
    float Ae[V], Be[V], At[V], Bt[V], x[V];
    gs_scan<V>(A, B, Ae, Be, At, Bt, sh, tid, j, TS, GS_JGROUPS, GS_JTHREADS);
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = fmaf(Ae[v], init ? init[(long long)b * a.H + ch + v] : 0.f, Be[v]);
    if (!on) return;
#pragma unroll 8
    for (int q = q0; q < q1; ++q) {
        float ka[V], kb[V];
        if (q < n - 1) {
            gs_load<float, V>(pr + (long long)q * 2 * a.H, ka);
            gs_load<float, V>(pr + (long long)q * 2 * a.H + a.H, kb);
        }
        gs_store<float, V>(pr + (long long)q * 2 * a.H, x);
        if (q < n - 1)
#pragma unroll
            for (int v = 0; v < V; ++v) x[v] = fmaf(ka[v], x[v], kb[v]);
    }
}

template <typename T, int V, int S, bool BWD>
__global__ __launch_bounds__(GS_THREADS, gs_waves(V == 8, BWD, false)) void gs_apply_kernel(GsArgs a) {
    extern __shared__ float sh[];
    const GsPlace p = gs_place(a, V);
    const NoteSpan sp = note_span(a.spans, p.b, a.rows, a.max_len);
    const long long first = (long long)p.k * a.chunk;
    {   // rows of no note: those behind this note, shared out like its own rows, and those in front of all notes, shared out over note 0's
        const bool known = a.ascending && *a.ascending;
        const long long end = sp.start + sp.len;
        const NoteSpan after = p.b + 1 < a.B ? note_span(a.spans, p.b + 1, a.rows, a.max_len) : NoteSpan{a.rows, 1};
        const bool look = !known && !(after.start == end && after.len > 0), front = p.b == 0 && sp.start > 0;
        __shared__ long long gap[2];
        if (look || front) {
            if (p.tid < 64) {  // (the last wave may be short of lanes)
                const long long g0 = look ? note_gap(a.spans, a.B, a.rows, a.max_len, end) : 0, g1 = note_gap(a.spans, a.B, a.rows, a.max_len, -1);
                if (p.tid == 0) gap[0] = g0, gap[1] = g1;
            }
            __syncthreads();
        }
        const long long next = look ? gap[0] : after.start;
        const long long lo = max(first, (long long)sp.len), hi = p.k == a.nch - 1 ? next - sp.start : min(first + a.chunk, next - sp.start);
        float zero[V];
#pragma unroll
        for (int v = 0; v < V; ++v) zero[v] = 0.f;
        auto clear = [&](long long r0, long long r1, int step) {
            for (long long r = r0 + p.j; r < r1; r += step) {
                if (!p.on) break;
                if (BWD) {
                    gs_store<T, V>((T*)a.dg + r * a.H + p.ch, zero);
                    gs_store<T, V>((T*)a.dc + r * a.H + p.ch, zero);
                } else {
                    gs_store<T, V>((T*)a.h + r * a.H + p.ch, zero);
                }
            }
        };
        clear(sp.start + lo, sp.start + hi, a.TS);
        if (front) clear((long long)p.k * a.TS, gap[1], a.nch * a.TS);
    }
    if (first >= sp.len && p.k > 0) return;
    const long long at = (long long)p.b * a.H + p.ch;
    const float* init = BWD ? a.dlast : a.h0;
    float x[V];  // the state in front of the current tile
#pragma unroll
    for (int v = 0; v < V; ++v) x[v] = init ? init[at + v] : 0.f;
    float Ae[V], Be[V], At[V], Bt[V];
    if (p.k > 0 && a.joined) {
        gs_load<float, V>(a.pair + ((long long)p.b * a.nch + p.k) * 2 * a.H + p.ch, x);
    } else if (p.k > 0) {
        // the pairs of the chunks in front, shared out over the threads along time
        const int per = (p.k + a.TS - 1) / a.TS, q0 = p.j * per, q1 = min(p.k, q0 + per);
        const float* pr = a.pair + (long long)p.b * a.nch * 2 * a.H + p.ch;
        float A[V], B[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
#pragma unroll 8
        for (int q = q0; q < q1; ++q) {
            float ka[V], kb[V];
            gs_load<float, V>(pr + (long long)q * 2 * a.H, ka);
            gs_load<float, V>(pr + (long long)q * 2 * a.H + a.H, kb);
#pragma unroll
            for (int v = 0; v < V; ++v) B[v] = fmaf(ka[v], B[v], kb[v]), A[v] *= ka[v];
        }
        gs_scan<V>(A, B, Ae, Be, At, Bt, sh, p.tid, p.j, a.TS, a.ncg, p.nt);
#pragma unroll
        for (int v = 0; v < V; ++v) x[v] = fmaf(At[v], x[v], Bt[v]);
    }
    const T *pg = (const T*)a.g + p.ch, *pc = (const T*)a.c + p.ch;
    for (int t = 0; t < a.tiles; ++t) {
        const long long base = first + (long long)t * a.TS * S;
        if (base >= sp.len) break;
        const int i0 = (int)base + p.j * S;
        float k[S][V], z[S][V], c[S][V], u[S][V];  // u: dh (backward)
#pragma unroll
        for (int s = 0; s < S; ++s) {
            const bool in = i0 + s < sp.len;
            const long long row = gs_row<BWD>(sp, a.reverse, in ? i0 + s : sp.len - 1);  // (past the end: read the last row, use nothing of it)
            gs_load<T, V>(pg + row * a.ldg, k[s]);
            gs_load<T, V>(pc + row * a.ldc, c[s]);
            if (BWD) {
                if (a.dh) gs_load<T, V>((const T*)a.dh + p.ch + row * a.H, u[s]);
                else
#pragma unroll
                    for (int v = 0; v < V; ++v) u[s][v] = 0.f;
                float before[V];
                const bool start = row == (a.reverse ? sp.start + sp.len - 1 : sp.start);  // the note's first step
                if (start) {
#pragma unroll
                    for (int v = 0; v < V; ++v) before[v] = a.h0 ? a.h0[at + v] : 0.f;
                } else {
                    const long long prev = (a.reverse ? row + 1 : row - 1) * a.H + p.ch;
                    gs_load<T, V>((const T*)a.ch + prev, before);
                    if (sizeof(T) == 2 && a.rest) {
                        float low[V];
                        gs_load<bf16, V>(a.rest + prev, low);
#pragma unroll
                        for (int v = 0; v < V; ++v) before[v] += low[v];
                    }
                }
#pragma unroll
                for (int v = 0; v < V; ++v) c[s][v] -= before[v];
            }
        }
        float A[V], B[V];
#pragma unroll
        for (int v = 0; v < V; ++v) A[v] = 1.f, B[v] = 0.f;
#pragma unroll
        for (int s = 0; s < S; ++s)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                gs_gate(k[s][v], z[s][v], k[s][v]);
                if (i0 + s >= sp.len) k[s][v] = 1.f, u[s][v] = c[s][v] = z[s][v] = 0.f;
                if (BWD) {
                    B[v] = k[s][v] * (B[v] + u[s][v]);
                } else {
                    z[s][v] *= c[s][v];
                    B[v] = fmaf(k[s][v], B[v], z[s][v]);
                }
                A[v] *= k[s][v];
            }
        // (a step past the end multiplies by 1 and adds nothing: in the backward that leaves k (B + u) = B)
        gs_scan<V>(A, B, Ae, Be, At, Bt, sh, p.tid, p.j, a.TS, a.ncg, p.nt);
        float y[V];
#pragma unroll
        for (int v = 0; v < V; ++v) {
            y[v] = fmaf(Ae[v], x[v], Be[v]);
            x[v] = fmaf(At[v], x[v], Bt[v]);
        }
#pragma unroll
        for (int s = 0; s < S; ++s) {
            if (i0 + s >= sp.len) break;
            const long long row = gs_row<BWD>(sp, a.reverse, i0 + s);
            float o[V], w[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                if (BWD) {
                    const float lam = y[v] + u[s][v];
                    o[v] = lam * z[s][v];
                    w[v] = lam * c[s][v] * (z[s][v] * k[s][v]);
                    y[v] = lam * k[s][v];
                } else {
                    y[v] = fmaf(k[s][v], y[v], z[s][v]);
                    o[v] = y[v];
                }
            }
            if (!p.on) continue;
            if (BWD) {
                gs_store<T, V>((T*)a.dc + row * a.H + p.ch, o);
                gs_store<T, V>((T*)a.dg + row * a.H + p.ch, w);
            } else {
                gs_store<T, V>((T*)a.h + row * a.H + p.ch, o);
                if (sizeof(T) == 2 && a.rest) {
#pragma unroll
                    for (int v = 0; v < V; ++v) w[v] = o[v] - (float)(T)o[v];
                    gs_store<bf16, V>(a.rest + row * a.H + p.ch, w);
                }
            }
        }
    }
    float* end = BWD ? a.dh0 : a.last;
    if (p.on && p.j == 0 && end && first + a.chunk >= sp.len)
#pragma unroll
        for (int v = 0; v < V; ++v) end[at + v] = x[v];
}

// Whether the notes stand in ascending order, disjoint: then a note's rows of no note end at the next one's start, and of many notes a
// workgroup need not go through the whole table for them.
__global__ __launch_bounds__(1024) void gs_order_kernel(GsArgs a) {
    bool ok = true;
    for (int b = threadIdx.x; b + 1 < a.B; b += 1024) {
        const NoteSpan sp = note_span(a.spans, b, a.rows, a.max_len), next = note_span(a.spans, b + 1, a.rows, a.max_len);
        ok = ok && sp.start + sp.len <= next.start;
    }
    ok = __syncthreads_and(ok);
    if (threadIdx.x == 0) *a.ascending = ok;
}

// Its launch is its time (64 x 200: 4.4 us with the call).
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
    if (d->B > 65534 || d->H > 65536 || d->max_len > 0x7FF00000) return GZSL_ETOOBIG;  // (positions of a last, partial tile stay below 2^31)
    if (d->B > 0 && !d->spans) return GZSL_EINVAL;
    if (d->rows > 0 && (!d->gates || !d->cands)) return GZSL_EINVAL;
    return 0;
}
static GsArgs gs_args(const GzslGatedScan& d) {
    GsArgs a{};
    a.g = d.gates, a.c = d.cands, a.spans = d.spans, a.h0 = d.h0, a.rows = d.rows, a.ldg = d.ldg, a.ldc = d.ldc;
    a.B = d.B, a.max_len = d.max_len < d.rows ? d.max_len : (int)d.rows, a.H = d.H, a.reverse = d.reverse;
    a.rest = d.dtype == GZSL_BF16 ? (bf16*)d.rest : nullptr;
    return a;
}

// Vectors of 16 bytes where the width and every address allow it, 8 bytes for bf16 of a width divisible by 4 only, else elements.
static int gs_width(const GzslGatedScan& d, uintptr_t addresses) {
    const int sz = d.dtype == GZSL_F32 ? 4 : 2;
    for (int V = 16 / sz; V >= 4; V >>= 1)
        if (d.H % V == 0 && d.ldg % V == 0 && d.ldc % V == 0 && addresses % (uintptr_t)(V * sz) == 0) return V;
    return 1;
}
// S V = 32 values of each operand in a thread's registers; up to GS_THREADS threads of at most 64 channel groups.
static int gs_steps(int V) { return V == 8 ? 4 : 8; }
static int gs_shape(GsArgs& a, int V) {
    const int groups = (a.H + V - 1) / V;
    a.ncg = groups < 64 ? groups : 64;
    a.nblk = (groups + a.ncg - 1) / a.ncg;
    a.TS = GS_THREADS / a.ncg;
    const long long tile = (long long)a.TS * gs_steps(V), all = (a.max_len + tile - 1) / tile, wgs = all * a.B * a.nblk;
    // a chunk is one tile until that makes over 1024 workgroups, four to a compute unit (81600 x 256 bf16: first pass and third 22 + 38 us
    // with half as many, 19 + 26 so, 18 + 28 with twice as many)
    long long m = wgs / 1024;
    if (m > all) m = all;
    if (m < 1) m = 1;
    a.tiles = (int)m, a.chunk = (int)(m * tile);
    a.nch = (int)(((long long)a.max_len + a.chunk - 1) / a.chunk);
    if (a.nch < 1) a.nch = 1;
    return (long long)a.nch * a.B > 0x7FFFFFFF ? GZSL_ETOOBIG : 0;
}

static long long gs_pair_bytes(const GsArgs& a) { return a.nch > 1 ? 8LL * a.B * a.nch * a.H : 0; }
// Up to 256 notes a workgroup finds its rows of no note in the table, four loads a wave; of more, a kernel looks at the order first.
static long long gs_work(const GsArgs& a) { return gs_pair_bytes(a) + (a.B > 256 ? 16 : 0); }

template <typename T, int V, bool BWD>
static int gs_go(GsArgs& a, void* work, long long work_bytes, hipStream_t st) {
    constexpr int S = V == 8 ? 4 : 8;
    if (int e = gs_shape(a, V)) return e;
    if (gs_work(a) > 0 && (!work || ((uintptr_t)work & 15) || work_bytes < gs_work(a))) return GZSL_EINVAL;
    a.pair = (float*)work;
    a.ascending = a.B > 256 ? (int*)((char*)work + gs_pair_bytes(a)) : nullptr;
    if (a.ascending) hipLaunchKernelGGL(gs_order_kernel, dim3(1), dim3(1024), 0, st, a);
    const dim3 grid(a.nch * a.B, a.nblk), block(a.ncg * a.TS);
    const size_t lds = sizeof(float) * 2 * V * block.x;
    if (a.nch > 1) hipLaunchKernelGGL((gs_chunk_kernel<T, V, S, BWD>), grid, block, lds, st, a);
    // Up to 64 chunks every workgroup joins the pairs in front of its own by itself (18388 x 200 fp32 in 40 chunks: a kernel for it would
    // take 6 us and save 1 to 3); of more, each would read more pairs than rows (512 chunks of 128 steps: 52 us against 26 + 7).
    a.joined = a.nch > 64;
    if (a.joined) {
        constexpr int JV = V >= 4 ? 4 : 1;
        const float* init = BWD ? a.dlast : a.h0;
        const dim3 jgrid(a.B, (a.H + JV * GS_JGROUPS - 1) / (JV * GS_JGROUPS));
        hipLaunchKernelGGL((gs_join_kernel<JV>), jgrid, dim3(GS_JTHREADS), sizeof(float) * 2 * JV * GS_JTHREADS, st, a, init);
    }
    hipLaunchKernelGGL((gs_apply_kernel<T, V, S, BWD>), grid, block, lds, st, a);
    GZSL_CHECK_LAUNCH();
    return 0;
}
template <bool BWD>
static int gs_run(const GzslGatedScan& d, GsArgs& a, int V, void* work, long long work_bytes, hipStream_t st) {
    if (d.dtype == GZSL_F32) return V == 4 ? gs_go<float, 4, BWD>(a, work, work_bytes, st) : gs_go<float, 1, BWD>(a, work, work_bytes, st);
    if (V == 8) return gs_go<bf16, 8, BWD>(a, work, work_bytes, st);
    return V == 4 ? gs_go<bf16, 4, BWD>(a, work, work_bytes, st) : gs_go<bf16, 1, BWD>(a, work, work_bytes, st);
}

extern "C" long long gzsl_gated_scan_work_bytes(const GzslGatedScan* d, int backward) {
    (void)backward;
    if (gs_check(d)) return -1;
    long long most = 0;  // over the vector widths, which the addresses decide
    for (int V = 1; V <= 8; V <<= 1) {
        GsArgs a = gs_args(*d);
        if (V == 2 || gs_shape(a, V)) continue;
        const long long n = gs_work(a);
        most = n > most ? n : most;
    }
    return most;
}

extern "C" long long gzsl_gated_scan_rest_bytes(const GzslGatedScan* d) {
    if (gs_check(d)) return -1;
    return d->dtype == GZSL_BF16 ? 2LL * d->rows * d->H : 0;
}

extern "C" int gzsl_gated_scan_fwd(const GzslGatedScan* d, void* h, float* h_last, void* work, long long work_bytes, void* stream) {
    if (int e = gs_check(d)) return e;
    if (d->B == 0) return d->rows == 0 ? 0 : GZSL_EINVAL;
    if (!h_last || (d->rows > 0 && !h)) return GZSL_EINVAL;
    GsArgs a = gs_args(*d);
    a.h = h, a.last = h_last;
    const int V = gs_width(*d, (uintptr_t)d->gates | (uintptr_t)d->cands | (uintptr_t)h | (uintptr_t)a.rest);
    return gs_run<false>(*d, a, V, work, work_bytes, (hipStream_t)stream);
}

extern "C" int gzsl_gated_scan_bwd(const GzslGatedScan* d, const void* h, const void* dh, const float* dlast, void* dgates, void* dcands, float* dh0,
                                   void* work, long long work_bytes, void* stream) {
    if (int e = gs_check(d)) return e;
    if (d->B == 0) return d->rows == 0 ? 0 : GZSL_EINVAL;
    if (d->rows > 0 && (!h || !dgates || !dcands)) return GZSL_EINVAL;
    GsArgs a = gs_args(*d);
    a.ch = h, a.dh = dh, a.dlast = dlast, a.dg = dgates, a.dc = dcands, a.dh0 = dh0;
    const int V = gs_width(*d, (uintptr_t)d->gates | (uintptr_t)d->cands | (uintptr_t)h | (uintptr_t)dh | (uintptr_t)dgates | (uintptr_t)dcands |
                                   (uintptr_t)a.rest);
    return gs_run<true>(*d, a, V, work, work_bytes, (hipStream_t)stream);
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
