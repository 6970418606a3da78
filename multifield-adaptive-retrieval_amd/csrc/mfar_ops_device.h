// mfar_ops_device.h -- device helpers of the encoder / training operators (wave = 64 lanes, matrix tiles of 32 x 32).
//
// One fragment = 8 elements per lane.  Lane l of an A (or B) fragment holds row (column) l % 32 and the 8 places k = 8 * (l / 32) + j of a
// k range of 16; lane l of a result tile holds column l % 32 and the rows crow(i) = 8 * (i / 4) + 4 * (l / 32) + i % 4, i = 0..15.
// A product sums over k, so any order of k that A and B share is right: 16-bit types take one v_mfma_f32_32x32x16, fp32 eight
// v_mfma_f32_32x32x2 over the same fragments (element j of both halves makes one k pair).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32;
typedef unsigned long long u64;
typedef u32 u32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct Vec;
template <> struct Vec<float> { typedef f32x4 v4; typedef f32x8 v8; };
template <> struct Vec<_Float16> { typedef f16x4 v4; typedef f16x8 v8; };
template <> struct Vec<__bf16> { typedef bf16x4 v4; typedef bf16x8 v8; };
template <typename T> using V4 = typename Vec<T>::v4;
template <typename T> using V8 = typename Vec<T>::v8;

__device__ __forceinline__ int crow(int i, int half) { return 8 * (i >> 2) + 4 * half + (i & 3); }

__device__ __forceinline__ f32x16 mma(f16x8 a, f16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x8 a, f32x8 b, f32x16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

// c + the 8 elements, two at a time in the dot unit (fp16's smallest numbers count; each pair is added with an error under a step of fp32, so
// sums that run long take the result in by an ordinary addition)
__device__ __forceinline__ float add_up(f16x8 x, float c) {
    typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
    const f16x2 one = {(_Float16)1.0f, (_Float16)1.0f};
#pragma unroll
    for (int j = 0; j < 8; j += 2) c = __builtin_amdgcn_fdot2(f16x2{x[j], x[j + 1]}, one, c, false);
    return c;
}
__device__ __forceinline__ float add_up(bf16x8 x, float c) {
    typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
    const bf16x2 one = {(__bf16)1.0f, (__bf16)1.0f};
#pragma unroll
    for (int j = 0; j < 8; j += 2) c = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{x[j], x[j + 1]}, one, c, false);
    return c;
}

// the two halves' values of a column, in either half (v_permlane32_swap: no LDS round trip)
__device__ __forceinline__ void both_halves(float x, float& a, float& b) {
    typedef u32 u32x2 __attribute__((ext_vector_type(2)));
    const u32x2 y = __builtin_bit_cast(u32x2, __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false));
    a = __uint_as_float(y[0]), b = __uint_as_float(y[1]);
}
__device__ __forceinline__ float sum_halves(float x) {
    float a, b;
    both_halves(x, a, b);
    return a + b;
}
__device__ __forceinline__ float max_halves(float x) {
    float a, b;
    both_halves(x, a, b);
    return fmaxf(a, b);
}
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, below 2^-126 flushed to zero
#define LOG2E 1.44269504088896341f
#define LN2 0.693147180559945309f
