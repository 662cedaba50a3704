// Element types, unaligned vectors and wave reductions of the training operators' kernels.
#pragma once

#include <hip/hip_runtime.h>

#include <cmath>

namespace ftrain::train {

using bf16 = __bf16;
using fp16 = _Float16;

constexpr int kWave = 64;
// Log2 of e, its inverse.
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

__device__ __forceinline__ float toFloat(float v) { return v; }
__device__ __forceinline__ float toFloat(bf16 v) {
    return __builtin_bit_cast(float, static_cast<unsigned>(__builtin_bit_cast(unsigned short, v)) << 16);
}
__device__ __forceinline__ float toFloat(fp16 v) { return static_cast<float>(v); }

// 16 bytes of T at any address a T may have: a global access of several dwords needs no alignment.
template <class T>
struct __attribute__((packed, aligned(alignof(T)))) Pack {
    static constexpr int kCount = 16 / sizeof(T);
    T v[kCount];
};

// Reductions over aligned groups of G lanes (a power of two); every lane gets the result.
template <int G>
__device__ __forceinline__ float groupMax(float v) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, kWave));
    return v;
}
template <int G, class V>
__device__ __forceinline__ V groupSum(V v) {
#pragma unroll
    for (int d = 1; d < G; d <<= 1) v += __shfl_xor(v, d, kWave);
    return v;
}

}  // namespace ftrain::train
