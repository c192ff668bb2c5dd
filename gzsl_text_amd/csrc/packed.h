// Shared pieces of the packed-note operators (packed_attn.hip, gated_scan.hip): notes of unequal length in one [rows, width]
// tensor, note b owning rows spans[b][0] .. spans[b][0] + spans[b][1] - 1.
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
