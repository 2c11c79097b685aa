// What the kernels of the paged key/value cache share: element types, division by a launch-time constant, and the batch.
#pragma once
#include "common.h"

typedef __bf16 bf16_t;
typedef bf16_t b2 __attribute__((ext_vector_type(2)));
typedef bf16_t b8 __attribute__((ext_vector_type(8)));
typedef float f8 __attribute__((ext_vector_type(8)));

enum { RDA_FP16 = 0, RDA_BF16 = 1, RDA_FP32 = 2 };  // the `type` arguments of include/rda.h

// Eight consecutive values as fp32, and back with one rounding (to nearest even).
__device__ __forceinline__ f8 load8(const half_t* p) { return __builtin_convertvector(*(const h8*)p, f8); }
__device__ __forceinline__ f8 load8(const bf16_t* p) {
    const u4v w = *(const u4v*)p;
    f8 x;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        x[2 * i] = __uint_as_float(w[i] << 16);
        x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
    return x;
}
__device__ __forceinline__ f8 load8(const float* p) { return __builtin_shufflevector(((const f4*)p)[0], ((const f4*)p)[1], 0, 1, 2, 3, 4, 5, 6, 7); }
__device__ __forceinline__ void store8(half_t* p, f8 x) { *(h8*)p = __builtin_convertvector(x, h8); }
__device__ __forceinline__ void store8(bf16_t* p, f8 x) { *(b8*)p = __builtin_convertvector(x, b8); }
__device__ __forceinline__ void store8(float* p, f8 x) {
    ((f4*)p)[0] = __builtin_shufflevector(x, x, 0, 1, 2, 3);
    ((f4*)p)[1] = __builtin_shufflevector(x, x, 4, 5, 6, 7);
}

// n / d for 0 <= n < 2^31 by a multiplication: with 2^s the least power of two >= d and m = floor(2^32 (2^s - d) / d) + 1,
// n / d = (hi32(n m) + n) >> s (the error of m / 2^32 + 1 as 2^s / d is below 2^-32, so the product's is below 2^-1 / d).
struct Div {
    u32 d, m, s;
};
static inline Div make_div(int d) {
    Div v = {(u32)d, 0, 0};
    while ((1ull << v.s) < (unsigned long long)d) v.s++;
    v.m = (u32)((((1ull << v.s) - d) << 32) / d) + 1;
    return v;
}
__device__ __forceinline__ int div_by(int n, const Div& v) { return (int)((__umulhi((u32)n, v.m) + (u32)n) >> v.s); }

// Values are read and written in vectors of eight: 16-byte aligned bases and strides.
static bool vector_rows(const void* p, const long* strides, int n, int type) {
    const long m = type == RDA_FP32 ? 4 : 8;
    for (int i = 0; i < n; i++)
        if (strides[i] % m) return false;
    return ((uintptr_t)p & 15) == 0;
}
