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

// exp(x) as 2^(x log2 e): the product's rounding is off by |x| 2^-24 of the result.
__device__ __forceinline__ float expFast(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }
// exp(x) to about an ulp: the rounding of x log2 e is carried along (2^(t + r) = 2^t (1 + r ln 2) for the
// tiny r).
__device__ __forceinline__ float expExact(float x) {
    constexpr float kLog2eLow = 1.9259629911266175e-8f;  // log2 e less kLog2e
    const float t = x * kLog2e;
    const float r = fmaf(x, kLog2eLow, fmaf(x, kLog2e, -t));
    const float p = __builtin_amdgcn_exp2f(t);
    // Where p is 0 or infinite (t may be) r is no number.
    return fabsf(t) < 126.f ? fmaf(p, r * kLn2, p) : p;
}

// Reductions over aligned groups of G lanes (a power of two); every lane gets the result.  Within 16
// lanes a step is the operation itself with a lane permutation (DPP: neighbours, pairs, then mirrored
// halves and rows, whose lanes agree by then); the last two exchange rows by permlane swaps.
template <int CTRL, class V>
__device__ __forceinline__ V permuted(V v) {
    static_assert(sizeof(V) == 4, "32-bit values");
    return __builtin_bit_cast(V, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}
// a and b with a's odd rows of 16 lanes (its upper 32 lanes) and b's even rows (lower lanes) exchanged.
// Assembly: of the builtin's two results this compiler returns the first twice.  The waits cover the
// hazards between a VALU write, the swap, and a DPP read of its results, which the compiler cannot see.
__device__ __forceinline__ void swap16(unsigned& a, unsigned& b) {
    asm volatile("s_nop 1\n\tv_permlane16_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}
__device__ __forceinline__ void swap32(unsigned& a, unsigned& b) {
    asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(a), "+v"(b));
}
template <int G, class V, class OP>
__device__ __forceinline__ V groupReduce(V v, OP&& op) {
    if constexpr (sizeof(V) == 4) {
        if constexpr (G > 1) v = op(v, permuted<0xB1>(v));    // quad_perm 1 0 3 2
        if constexpr (G > 2) v = op(v, permuted<0x4E>(v));    // quad_perm 2 3 0 1
        if constexpr (G > 4) v = op(v, permuted<0x141>(v));   // row_half_mirror
        if constexpr (G > 8) v = op(v, permuted<0x140>(v));   // row_mirror
        if constexpr (G > 16) {
            unsigned x = __builtin_bit_cast(unsigned, v), y = x;
            swap16(x, y);
            v = op(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y));
        }
        if constexpr (G > 32) {
            unsigned x = __builtin_bit_cast(unsigned, v), y = x;
            swap32(x, y);
            v = op(__builtin_bit_cast(V, x), __builtin_bit_cast(V, y));
        }
        return v;
    } else {
#pragma unroll
        for (int d = 1; d < G; d <<= 1) v = op(v, __shfl_xor(v, d, kWave));
        return v;
    }
}
template <int G>
__device__ __forceinline__ float groupMax(float v) {
    return groupReduce<G>(v, [](float a, float b) { return fmaxf(a, b); });
}
template <int G, class V>
__device__ __forceinline__ V groupSum(V v) {
    return groupReduce<G>(v, [](V a, V b) { return a + b; });
}
// The sum over the lanes that are the same in their groups of G, in each of them (DPP: rotations of 16 lanes).
template <int G>
__device__ __forceinline__ float acrossGroups(float v) {
    if constexpr (G <= 8) v += permuted<0x128>(v);
    if constexpr (G <= 4) v += permuted<0x124>(v);
    if constexpr (G <= 2) v += permuted<0x122>(v);
    if constexpr (G <= 1) v += permuted<0x121>(v);
    if constexpr (G <= 16) {
        unsigned x = __builtin_bit_cast(unsigned, v), y = x;
        swap16(x, y);
        v = __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
    }
    if constexpr (G <= 32) {
        unsigned x = __builtin_bit_cast(unsigned, v), y = x;
        swap32(x, y);
        v = __builtin_bit_cast(float, x) + __builtin_bit_cast(float, y);
    }
    return v;
}
// One wave's LDS accesses are done in order; this keeps the compiler from moving them across.
__device__ __forceinline__ void waveFence() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
}

}  // namespace ftrain::train
