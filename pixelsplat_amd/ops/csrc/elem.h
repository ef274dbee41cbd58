// Element types of the operators that take fp32, bf16 and fp16 tensors: 16-byte vectors of them, conversion to
// and from the fp32 all arithmetic is done in, and the activations with their slopes.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace ps {

typedef __bf16 bf16;
typedef _Float16 f16;

// V elements moved as one 4*V- or 2*V-byte access
template <typename T, int V>
struct alignas(sizeof(T) * V) Pack { T v[V]; };

template <typename T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <typename T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }   // round to nearest even

template <typename T> inline constexpr bool kNarrow = false;     // a type with fewer exponents than fp32 has
template <> inline constexpr bool kNarrow<f16> = true;

// parameters are stored in the tensors' type or in fp32
template <typename T>
__device__ __forceinline__ float load_param(const void* p, int is_f32, int64_t i) {
  return is_f32 ? reinterpret_cast<const float*>(p)[i] : to_f32(reinterpret_cast<const T*>(p)[i]);
}
template <typename T>
__device__ __forceinline__ void store_param(void* p, int is_f32, int64_t i, float v) {
  if (is_f32) reinterpret_cast<float*>(p)[i] = v;
  else reinterpret_cast<T*>(p)[i] = from_f32<T>(v);
}

// 0.5 (1 + erf(z / sqrt 2)) and exp(-z^2 / 2).  fp32 tensors use erff (an absolute error of 2^-24: far below zero, where the value
// itself is smaller than that, as in any form with 1 + erf).  16-bit tensors use, for the tail on z's far side,
// exp(-z^2 / 2) t P(t) with t = 1 / (1 + 0.4125 |z| / sqrt 2) and P of degree 5, which was fitted here to
// 0.5 erfc(x) exp(x^2), x = |z| / sqrt 2 = 0 .. 9.6, by minimising the larger of its absolute error (of erfc) over 2e-7 and its
// relative error over 2^-14.  In fp32 that is 2.5e-7 of 1 and, for z < 0, 2^-14.4 of the value itself: an eighth of half a step of fp16,
// down to where the value ends.  (A form that holds 1.5e-7 of 1 alone is 1.3 half steps of fp16 off at -4 and 8 of bf16 at
// -9.)  It shares the exponential with the slope, and it is a third of the instructions of erff.
template <bool EXACT>
__device__ __forceinline__ void normal_cdf(float z, float& cdf, float& bell) {
  bell = __expf(-0.5f * z * z);
  if (EXACT) {
    cdf = 0.5f * (1.f + erff(z * 0.70710678118654752f));
  } else {
    const float t = __builtin_amdgcn_rcpf(fmaf(0.4125f * 0.70710678118654752f, fabsf(z), 1.f));
    const float poly = t * fmaf(t, fmaf(t, fmaf(t, fmaf(t, fmaf(t, -0.086771145f, 0.2719236f), -0.07750261f), 0.17137343f),
                                       0.1036474f), 0.11732936f);
    const float tail = poly * bell;
    cdf = z < 0.f ? tail : 1.f - tail;
  }
}
__device__ __forceinline__ float sigmoid_f32(float z) { return 1.f / (1.f + __expf(-z)); }

// the PS_ACT_ values of pixelsplat_ops.h
enum Act { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3, ACT_SIGMOID = 4 };

template <int ACT, bool EXACT>
__device__ __forceinline__ float act_value(float z) {
  if constexpr (ACT == ACT_RELU) return z > 0.f || z != z ? z : 0.f;
  if constexpr (ACT == ACT_SILU) return z * sigmoid_f32(z);
  if constexpr (ACT == ACT_GELU) {
    float cdf, bell;
    normal_cdf<EXACT>(z, cdf, bell);
    return z * cdf;
  }
  if constexpr (ACT == ACT_SIGMOID) return sigmoid_f32(z);
  return z;
}
// act'(z); *value = act(z)
template <int ACT, bool EXACT>
__device__ __forceinline__ float act_slope(float z, float* value) {
  if constexpr (ACT == ACT_RELU) {
    *value = z > 0.f || z != z ? z : 0.f;
    return z > 0.f ? 1.f : 0.f;
  }
  if constexpr (ACT == ACT_SILU) {
    const float s = sigmoid_f32(z);
    *value = z * s;
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if constexpr (ACT == ACT_GELU) {
    float cdf, bell;
    normal_cdf<EXACT>(z, cdf, bell);
    *value = z * cdf;
    return fmaf(z * 0.39894228040143268f, bell, cdf);
  }
  if constexpr (ACT == ACT_SIGMOID) {
    const float e = __expf(-fabsf(z)), r = 1.f / (1.f + e);      // s (1 - s) would lose 1 - s where s is near 1
    *value = z < 0.f ? e * r : r;
    return e * r * r;
  }
  *value = z;
  return 1.f;
}

template <int A> struct ActTag { static constexpr int act = A; };
// f(ActTag<act>()): one branch around a kernel's loop, whose body then holds one activation's instructions.  (A branch
// an element left 16 - 28 KB of code in an epilogue, and the instruction cache's misses were most of a small call.)
template <typename F>
__device__ __forceinline__ void with_act(int act, F f) {
  switch (act) {
    case ACT_RELU: f(ActTag<ACT_RELU>()); break;
    case ACT_SILU: f(ActTag<ACT_SILU>()); break;
    case ACT_GELU: f(ActTag<ACT_GELU>()); break;
    case ACT_SIGMOID: f(ActTag<ACT_SIGMOID>()); break;
    default: f(ActTag<ACT_NONE>()); break;
  }
}

}  // namespace ps
