// Shared pieces of the packed-note operators (packed_attn.hip, gated_scan.hip): notes of unequal length in one [rows, width]
// tensor, note b owning rows spans[b][0] .. spans[b][0] + spans[b][1] - 1, the notes in any order.
#pragma once
#include "common.h"

typedef __bf16 bf16;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
#define GZ_LDS __attribute__((address_space(3)))

struct NoteSpan {
    long long start;
    int len;
};
// Whatever the table holds, the result lies inside [0, rows) and is no longer than max_len: a wrong table gives wrong
// numbers, never an access out of range.
__device__ __forceinline__ NoteSpan note_span(const int64_t* spans, int b, long long rows, int max_len) {
    long long s = spans[2 * b], n = spans[2 * b + 1];
    s = s < 0 ? 0 : (s > rows ? rows : s);
    if (n > rows - s) n = rows - s;
    if (n > max_len) n = max_len;
    return {s, n < 0 ? 0 : (int)n};
}
// The first row from `end` on that a note owns which reaches past `end` (rows: none does): where the rows of no note behind a note that
// ends at `end` stop, in whatever order the table has the notes.  end = -1: the first row of any note.  Every wave works it out from the
// table by itself, a load and a few lane exchanges for 64 notes; all its lanes have to be there.
__device__ __forceinline__ long long note_gap(const int64_t* spans, int B, long long rows, int max_len, long long end) {
    long long g = rows;
    for (int b = threadIdx.x & 63; b < B; b += 64) {
        const NoteSpan sp = note_span(spans, b, rows, max_len);
        if (sp.start + sp.len > end) g = min(g, max(sp.start, end));
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) g = min(g, (long long)__shfl_xor(g, o));
    return g;
}
