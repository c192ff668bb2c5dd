// Host side of the packed label attention: argument checks, workspace plan, dispatch.
#include "packed_attn.h"

static inline long long up256(long long n) { return (n + 255) / 256 * 256; }

template <class G>
static void pa_sizes(PaPlan& p, const GzslPackedAttn& d, int backward) {
    p.nT = (int)(((long long)p.max_len + G::ROWS - 1) / G::ROWS), p.nQ = (int)(((long long)d.L + G::ROWS - 1) / G::ROWS);
    const long long most = d.rows / G::ROWS + d.B;  // tiles that disjoint notes can have
    p.slots = (long long)d.B * p.nT;
    if (p.slots > PA_WASTE * most) p.slots = most, p.nT = 0;
    p.kv = 1024LL * p.slots * (backward ? G::TOK : G::FWD);
    p.q = 1024LL * p.nQ * (backward ? G::QRY : G::PL * G::RE);
    p.dO = backward ? 1024LL * d.B * p.nQ * G::OUT : 0;
}
static int pa_plan(const GzslPackedAttn* d, int backward, PaPlan& p) {
    if (!d || d->B < 0 || d->rows < 0 || d->max_len < 0 || d->L < 0 || d->E < 1 || d->F < 1 || d->E > 208 || d->F > 208) return GZSL_EINVAL;
    if (d->dtype != GZSL_F32 && d->dtype != GZSL_BF16) return GZSL_EINVAL;
    if (d->cap != 0.f && !(d->cap >= 1e-30f && d->cap <= 1e30f)) return GZSL_EINVAL;
    if (d->ldk < d->E || d->ldv < d->F || d->ldq < d->E) return GZSL_EINVAL;
    if (d->B > 65534 || d->max_len > 0x7FFF0000 || d->L > 0x7FFF0000) return GZSL_ETOOBIG;
    p = PaPlan{};
    p.max_len = d->max_len < d->rows ? d->max_len : (int)d->rows;  // (no note is longer than the rows there are)
    p.kind = (d->dtype == GZSL_F32 ? 2 : 0) + (d->E > 112);
    if (p.kind == 0) pa_sizes<PaGeo<PaBF, 7, 13>>(p, *d, backward);
    else if (p.kind == 1) pa_sizes<PaGeo<PaBF, 13, 13>>(p, *d, backward);
    else if (p.kind == 2) pa_sizes<PaGeo<PaX3, 7, 13>>(p, *d, backward);
    else pa_sizes<PaGeo<PaF32, 13, 13>>(p, *d, backward);
    // 128 labels a workgroup (64: PaF32's forward, and bf16 where 128 leave fewer workgroups than the chip has places, two a compute
    // unit; dQ then has twice the waves share the tiles: 16 notes, 17404 tokens x 1999 labels of 200: 71 us against 87 without, x 9000
    // labels 326 against 286 of 128 a workgroup); notes are cut where the (note, label) workgroups alone would leave compute units
    // without one.
    const bool fits = !backward && d->L <= 128;  // one workgroup a note: it works from the rows themselves
    p.waves = !fits && ((p.kind == 3 && !backward) || (p.kind < 2 && (long long)d->B * cdiv(d->L, 128) < 512)) ? 4 : 8;
    p.nLT = cdiv(d->L, 16 * p.waves);
    const long long wgs = (long long)d->B * p.nLT;
    // tokens of a chunk that pay for its own start and its part in the join (fp32: 1500 tokens x 32 labels of 200, 28 + 6 us at 128, 25 + 7 at
    // 96, 20 + 6 at 64, but bf16 of 31, 21 + 8, 19 + 9, 19 + 9; dQ of 1000 tokens x 428 labels 38 us at 256, 25 at 128, 18 at 64; the
    // forward 27 us at 256, 18 at 128, 15 at 64, but 319 x 5380 25 us at 128 and 29 at 64)
    p.least = backward ? 64 : (fits ? 96 : 128);
    p.extra = wgs > 0 && wgs < 256 && p.max_len > p.least ? cdiv(p.waves == 4 && !backward ? 512 : 256, p.nLT) : 0;
    if (p.extra > (long long)d->B * (p.max_len / p.least + 1)) p.extra = d->B * (p.max_len / p.least + 1);
    const long long chunks = d->B + p.extra;
    if (fits) p.kv = p.q = 0;
    if (p.slots + p.nQ > 0x3FFFFFFF || chunks * p.nLT > 0x3FFFFFFF || (long long)d->B * p.nQ > 0x3FFFFFFF || (long long)d->B * d->L > 0x3FFFFFFF)
        return GZSL_ETOOBIG;
    if (!backward && p.extra > 0) {
        p.part = up256(4 * chunks * d->L * d->F);
        p.ml = up256(8 * chunks * d->L);
    }
    if (backward) {
        p.dq = up256(4 * chunks * d->L * d->E);
        long long tiles = (long long)d->B * cdiv(p.max_len, PA_TILE);  // at most
        if (tiles > d->rows / PA_TILE + d->B) tiles = d->rows / PA_TILE + d->B;
        const long long steps = tiles * p.nQ;  // at most: the runs are cut on the device
        if (steps > 0x7FFFFF00) return GZSL_ETOOBIG;
        // (of notes that overlap there may be more, as many as would fill B times max_len)
        const long long most = (long long)d->B * cdiv(p.max_len, PA_TILE);
        p.units = most >= PA_UNITS * PA_RUN || most * p.nQ >= PA_UNITS * PA_RUN ? PA_UNITS : (int)((most * p.nQ + PA_RUN - 1) / PA_RUN);
        p.dkv = up256(8LL * p.units * PA_TILE * (d->E + d->F));
    }
    p.bytes = p.kv + p.q + p.dO + p.part + p.ml + p.dq + p.dkv + 256;
    return 0;
}
static void pa_fill(PaArgs& a, const GzslPackedAttn& d, const PaPlan& p, void* work) {
    a.keys = d.keys, a.values = d.values, a.queries = d.queries, a.spans = d.spans;
    a.rows = d.rows, a.ldk = d.ldk, a.ldv = d.ldv, a.ldq = d.ldq;
    a.B = d.B, a.max_len = p.max_len, a.L = d.L, a.E = d.E, a.F = d.F, a.nT = p.nT, a.nQ = p.nQ, a.slots = (int)p.slots;
    a.cap = d.cap, a.l_offset = (uint32_t)d.l_offset, a.L_total = (uint32_t)d.L_total, a.seed = d.seed, a.thresh = d.drop_thresh, a.scale = d.drop_scale;
    a.nLT = p.nLT, a.extra = p.extra, a.least = p.least;
    // few rows: one a wave, for the time of one row's parts to come in (1000 tokens x 428 labels: 31 us with four a wave, 12 so); many: four,
    // to share out what a workgroup has to find out first (17404 x 1999: 21 us with one a wave, 19 so)
    // and few tiles of more than two runs each: one row for all four waves (500 tokens x 3917 labels, 51 runs a tile: 58 us with a row a
    // wave, 7 so; 6000 x 1999, 5 runs: 19 and 29)
    const long long at_most = (long long)p.max_len * d.B;
    a.join_rows = at_most <= 4096 && p.units > 2LL * d.B * cdiv(p.max_len, PA_TILE) ? 1 : (at_most <= 16384 ? 4 : 16);
    char* w = (char*)work;
    a.TK = w, w += p.kv;
    a.Q = w, w += p.q;
    a.DO = w, w += p.dO;
    a.part = (float*)w, w += p.part;
    a.ml = (float*)w, w += p.ml;
    a.dq = (float*)w, w += p.dq;
    a.dkv = (float*)w;
}
static int pa_run(const GzslPackedAttn& d, PaArgs& a, const PaPlan& p, bool backward, hipStream_t st) {
    if (p.kind == 3) return pa_run_f32(a, p, backward, st);
    return p.kind == 2 ? pa_run_x3(a, p, backward, st) : pa_run_bf16(a, p, backward, st);
}

extern "C" long long gzsl_packed_attn_work_bytes(const GzslPackedAttn* d, int backward) {
    PaPlan p;
    return pa_plan(d, backward, p) ? -1 : p.bytes;
}
extern "C" long long gzsl_packed_attn_rest_bytes(const GzslPackedAttn* d) {
    PaPlan p;
    if (pa_plan(d, 0, p)) return -1;
    return (long long)d->B * d->L * (8 + (d->dtype == GZSL_BF16 ? 2LL * d->F : 0));
}

extern "C" int gzsl_packed_attn_fwd(const GzslPackedAttn* d, void* O, float* LSE, void* rest, void* work, long long work_bytes, void* stream) {
    PaPlan p;
    if (int e = pa_plan(d, 0, p)) return e;
    if (d->B == 0 || d->L == 0) return 0;
    if (!O || !LSE || ((uintptr_t)rest & 15) || !d->spans || !d->queries || (d->rows > 0 && (!d->keys || !d->values)) || work_bytes < p.bytes || !work ||
        ((uintptr_t)work & 15))
        return GZSL_EINVAL;
    PaArgs a{};
    pa_fill(a, *d, p, work);
    a.O = O, a.LSE = LSE, a.rest = (float*)rest;
    return pa_run(*d, a, p, false, (hipStream_t)stream);
}

extern "C" int gzsl_packed_attn_bwd(const GzslPackedAttn* d, const void* O, const float* LSE, const void* rest, const void* dO, void* dkeys, void* dvalues,
                                    void* dqueries, void* work, long long work_bytes, void* stream) {
    PaPlan p;
    if (int e = pa_plan(d, 1, p)) return e;
    if (d->L == 0 && d->rows == 0) return 0;
    if (d->B == 0 || d->L == 0) return GZSL_EINVAL;  // nothing was attended: the gradients are the caller's zeros
    if (!O || !LSE || ((uintptr_t)rest & 15) || !dO || !dqueries || !d->spans || !d->queries ||
        (d->rows > 0 && (!d->keys || !d->values || !dkeys || !dvalues)) || work_bytes < p.bytes || !work || ((uintptr_t)work & 15))
        return GZSL_EINVAL;
    PaArgs a{};
    pa_fill(a, *d, p, work);
    a.cO = O, a.cLSE = LSE, a.crest = (const float*)rest, a.dO = dO, a.dK = dkeys, a.dV = dvalues, a.dQ = dqueries;
    return pa_run(*d, a, p, true, (hipStream_t)stream);
}
