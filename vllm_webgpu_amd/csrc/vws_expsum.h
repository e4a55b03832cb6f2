// vws_expsum.h -- sums of exponentials of a row's logits, exp((x - max) / T), shared by draft verification
// and the distillation loss, and the loads they are taken from.
//
// With c = log2(e) / T an element costs one fma and one exp2: exp2(x c - r), r = fl(n c) the running
// maximum n's product rounded.  r is off n c by up to half an ulp of r, so such a sum is off by a
// factor 2^d, which is divided out once the maximum is known (ExpSum::close).  That holds while d is
// small: beyond kExpFar a sum is taken anew, over differences from its maximum.  And r must not run far
// below zero while a thread has met only masked logits (a mask of -1e10 at T = 1 has d = 440, exp2(d) is
// infinite): it starts from exp_floor, below which nothing counts in a sum that kExpFar admits.
#pragma once

#include "vws_device.h"

namespace vws {

constexpr float kExpInf = __builtin_inff();
constexpr float kExpLog2e = 0x1.715476p+0f;

// The largest |max log2(e) / T| whose sum is taken by fma.  d <= 2^-11 there, and fl(x / T), which the
// sampler's arithmetic starts from, is within 2^-11 of x / T.
constexpr float kExpFar = 0x1p14f;

__device__ __forceinline__ float es_exp2(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float es_lane_xor(float v, int s) { return u2f(lane_xor(f2u(v), s)); }
__device__ __forceinline__ float es_wave_max(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = __builtin_fmaxf(v, es_lane_xor(v, o));
    return v;
}
__device__ __forceinline__ float es_wave_sum(float v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += es_lane_xor(v, o);
    return v;
}

// A maximum (finite) whose sum is to be taken over differences from it.
__device__ __forceinline__ bool exp_far(float m, float c) {
    return __builtin_fabsf(m) < kExpInf && !(__builtin_fabsf(m * c) <= kExpFar);
}
// The least reference of a thread's running sum: twice as far as kExpFar, so that what lies below it adds
// nothing (exp2 of less than -kExpFar) to a sum whose maximum is not far; finite for every c >= 0.
__device__ __forceinline__ float exp_floor(float c) { return __builtin_fmaxf(-2.0f * kExpFar / c, -0x1.fffffep127f); }

// (maximum m of some logits, sum of exp2((x - m) c)); the empty one is (-inf, 0).
struct ExpSum {
    float m = -kExpInf, s = 0.0f;
    __device__ __forceinline__ void merge(float om, float os, float c) {
        const float n = __builtin_fmaxf(m, om), ref = n == -kExpInf ? 0.0f : n;
        s = s * es_exp2((m - ref) * c) + os * es_exp2((om - ref) * c);
        m = n;
    }
    __device__ __forceinline__ void wave_merge(float c) {
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) merge(es_lane_xor(m, o), es_lane_xor(s, o), c);
    }
};

// A thread's running sum: of exp2(x c - ref), ref = fl(max(m, floor) c).
struct ExpRun {
    float m = -kExpInf, s = 0.0f, ref, floor;
    __device__ __forceinline__ explicit ExpRun(float c) : floor(exp_floor(c)) { ref = floor * c; }
    // Takes logits of maximum g in: returns the earlier ones' sum, relative to the new reference.
    __device__ __forceinline__ float raise(float g, float c) {
        const float was = ref;
        m = __builtin_fmaxf(m, g);
        ref = __builtin_fmaxf(m, floor) * c;
        return s * es_exp2(was - ref);
    }
    __device__ __forceinline__ ExpSum close(float c) const {
        ExpSum o;
        o.m = m;
        o.s = s * es_exp2(-__builtin_fmaf(__builtin_fmaxf(m, floor), c, -ref));
        return o;
    }
};

// 16 bytes at any element's address: rows of an odd vocabulary start unaligned.
template <typename T> struct RowVec { typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(2))); };
template <> struct RowVec<float> { typedef uint32_t U4 __attribute__((ext_vector_type(4), aligned(4))); };

// Vector vi of a row (a 32-bit offset, at most 2 MB, on its pointer).
template <typename T>
__device__ __forceinline__ void row_load(const T* row, int vi, uint32_t (&w)[4]) {
    const auto u = *reinterpret_cast<const typename RowVec<T>::U4*>(reinterpret_cast<const char*>(row) + 16u * (uint32_t)vi);
    w[0] = u[0]; w[1] = u[1]; w[2] = u[2]; w[3] = u[3];
}

}  // namespace vws
