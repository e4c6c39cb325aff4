// What the kernels of the 8-bit key/value cache share.
//
// A block of the cache is the 64 rows (tokens) that one page holds of one key/value head, keys and values apart.  A value
// is code * s: the code in e4m3 (4 exponent bits, 3 mantissa bits, largest 448, steps of 2^-9 below 2^-6, one NaN, no
// infinity), s = 2^k one power of two a block, kept as a float.  With a power of two nothing but the code rounds: a block
// whose scale grows keeps its codes' mantissas (only codes that fall below 2^-6 round again), and the code times its scale
// is exact in bfloat16 and in float.
#pragma once
#include "common.cuh"
#include <cuda_fp8.h>
#include <cuda_fp16.h>
#include <math.h>

// One run's (layer's) part of the cache.  Keys: page p, head h, row t, channel d at k + p k_stride + (h 64 + t) hd + d;
// values: v + p v_stride + (h hd + d) 64 + t -- rows innermost, since the second product of attention contracts over them
// and an 8-bit operand has no transposed load.  scales[p scale_stride + plane n_kv + h] (plane 0 keys, 1 values).
// weights (or null): [p weight_stride + h 64 + t], the attention weight a row has gathered.  dropped (or null): by slot, how
// many rows of its sequence have been evicted: position p of the sequence is row p - dropped.  A view of the cache holds one, and the
// C entries copy it.
struct E4M3Pages {
    uint8_t* k;
    uint8_t* v;
    long long k_stride, v_stride;
    float* scales;
    long long scale_stride;
    float* weights;
    long long weight_stride;
    const int* block_table;
    int table_stride;
    const int* dropped;
    int n_kv, hd;
};

constexpr int kLeastExponent = -126;

// A kernel that only goes on with what the launch before it (of the same call) has left: it may begin while that one drains,
// whether the caller chains its kernels or not, and waits for it itself (chain_wait).
template <typename... Params, typename... Args>
static inline int launch_behind(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t stream, Args... args) {
    return launch_early(true, kernel, grid, block, smem, stream, args...);
}

// Lets `kernel` take up to `bytes` of shared memory on the current device, asked for once a device: the permission is the device's, and
// a size that differed by call could be lowered by another thread between here and the launch.  done: the kernel's own, one a device.
constexpr int kMaxDevices = 64;
static inline int allow_shared(const void* kernel, size_t bytes, bool (&done)[kMaxDevices]) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e != cudaSuccess) return (int)e;
    const bool counted = dev >= 0 && dev < kMaxDevices;
    if (counted && done[dev]) return 0;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    if (e != cudaSuccess) return (int)e;
    if (counted) done[dev] = true;
    return 0;
}

__device__ __forceinline__ bool finite_f32(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

__device__ __forceinline__ float min_or_nan(float a, float b) {
    float r;
    asm("min.NaN.f32 %0, %1, %2;\n" : "=f"(r) : "f"(a), "f"(b));
    return r;
}

// Where a score is computed once more, by other instructions than those that found its query's maximum `top` (both in powers of two),
// the two are apart by their sums' roundings.  From 2^20 on these are units: the winning row could come out at any probability
// between 0 and 1, and so what lies within this much of the maximum counts as the maximum.  Sums of 128 products agree to a few
// of the 64 steps of 2^-23 that this is; which of two rows that lie nearer is the larger, float scores cannot say.
constexpr float kLargeScore = 1048576.f;
__device__ __forceinline__ float score_slack(float top) { return fabsf(top) > kLargeScore ? fabsf(top) * 7.62939453125e-6f : 0.f; }

// The least power of two 2^k, k >= -126, with most <= 448 * 2^k, for finite most >= 0: 448 = 1.75 * 2^8, so k is the
// exponent less 8, one more where the mantissa exceeds 1.75.
__device__ __forceinline__ float e4m3_needed_scale(float most) {
    const uint32_t u = __float_as_uint(most);
    int k = (int)(u >> 23) - 127 - 8 + ((u & 0x7fffffu) > 0x600000u ? 1 : 0);
    k = max(k, kLeastExponent);
    return __uint_as_float((uint32_t)(k + 127) << 23);
}
// 1 / s for a power of two s between 2^-126 and 2^126 (also a power of two, exact).
__device__ __forceinline__ float pow2_inverse(float s) { return __uint_as_float(0x7f000000u - __float_as_uint(s)); }

// The nearest code, ties to even; what is not finite becomes the NaN code.
__device__ __forceinline__ uint8_t e4m3_code(float x) {
    return finite_f32(x) ? (uint8_t)__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3) : (uint8_t)0x7f;
}
__device__ __forceinline__ float e4m3_value(uint8_t c) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(c, __NV_E4M3);
    return __half2float(*reinterpret_cast<const __half*>(&h));
}
// Codes 0, 1 (the low half) and 2, 3 (the high half) of a word as pairs of halves, exact.
__device__ __forceinline__ uint32_t e4m3_pair_f16(uint32_t two_codes) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;\n" : "=r"(r) : "h"((unsigned short)two_codes));
    return r;
}
