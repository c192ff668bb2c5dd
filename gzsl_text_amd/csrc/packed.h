// Shared pieces of the packed-note operators (packed_attn.hip, gated_scan.hip): notes of unequal length in one [rows, width]
// tensor, note b owning rows spans[b][0] .. spans[b][0] + spans[b][1] - 1.
#pragma once
#include "common.h"

typedef __bf16 bf16;
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef unsigned u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
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

// Rows that belong to no note read as zero: those before the first note and those behind each note (spans ascend).
template <typename T>
static __global__ __launch_bounds__(256) void zero_gaps_kernel(const int64_t* spans, long long rows, int B, int max_len, T* x, int Wx, T* y, int Wy) {
    const int b = (int)blockIdx.y - 1;  // -1: in front of note 0
    long long r0 = 0, r1 = rows;
    if (b >= 0) {
        const NoteSpan sp = note_span(spans, b, rows, max_len);
        r0 = sp.start + sp.len;
    }
    if (b + 1 < B) r1 = note_span(spans, b + 1, rows, max_len).start;
    const long long step = (long long)gridDim.x * 256, first = (long long)blockIdx.x * 256 + threadIdx.x;
    for (long long i = r0 * Wx + first; i < r1 * Wx; i += step) x[i] = (T)0.f;
    if (y)
        for (long long i = r0 * Wy + first; i < r1 * Wy; i += step) y[i] = (T)0.f;
}
