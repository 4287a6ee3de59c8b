// Shared by the paged-cache kernels: element types, page arithmetic, and the tiling of a ragged batch of queries.
#pragma once
#include "common.h"

typedef __bf16 bf16;
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
// 16 bytes at any address that the element type allows (a head of 150 halfs starts at an odd multiple of 4 bytes): global memory
// takes a dword-x4 access at such an address as one instruction
typedef u32x4 u32x4_any __attribute__((aligned(2)));

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 without a divide: q = (mulhi(m, n) + n) >> s with s = ceil(log2 d) and
// m = floor(2^32 (2^s - d) / d) + 1 (Granlund and Montgomery 1994); the sum stays below 2^32 because n < 2^31.
struct JbDiv { unsigned d, m; int s; };
static inline JbDiv jb_make_div(unsigned d) {
    int s = 0;
    while (s < 31 && (1u << s) < d) ++s;
    return JbDiv{d, (unsigned)((((uint64_t)1 << 32) * (((uint64_t)1 << s) - d)) / d + 1), s};
}
// Whether no two of n1 x n2 x n3 rows of `len` elements, at these strides, share one -- of strides that nest: each at least what the smaller ones span
// (dimensions of one entry do not count).
static inline bool jb_apart(int64_t len, int64_t n1, int64_t s1, int64_t n2, int64_t s2, int64_t n3 = 1, int64_t s3 = 0) {
    int64_t n[3] = {n1, n2, n3}, s[3] = {s1, s2, s3}, span = len;
    for (int done = 0; done < 3; ++done) {
        int least = -1;
        for (int i = 0; i < 3; ++i)
            if (n[i] > 1 && (least < 0 || s[i] < s[least])) least = i;
        if (least < 0) break;
        if (s[least] < span) return false;
        span += (n[least] - 1) * s[least];
        n[least] = 1;
    }
    return true;
}
__device__ __forceinline__ unsigned jb_div(unsigned n, const JbDiv& v) { return (__umulhi(v.m, n) + n) >> v.s; }
