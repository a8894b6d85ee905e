// Activations and float conversions of the row-wise steps and of the products'
// epilogue. Device code.
#ifndef IREE_UK_AMD_ACTIVATION_H_
#define IREE_UK_AMD_ACTIVATION_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "iree_uk_amd.h"

namespace uk {

// x * sigmoid(t) = x / (1 + 2^(-t log2 e)). An exponent of 128 and more gives an
// infinity, and x over it zero, which is what the product tends to (from 2^126 on already:
// the reciprocal would be subnormal, and the hardware's is zero). The hardware's
// exponential and reciprocal are good to one unit in the last place each: the
// result to about three, and to |t| units where t is large and negative.
__device__ __forceinline__ float times_sigmoid(float x, float t) {
  return x * __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504f * t));
}

// The same closer, to 3.5 units and |t| / 40 of one: for f32 results, and for what an 8-bit form is
// made of, in which every unit more moves some elements across the middle between two steps. hi, the rounded exponent, is taken as it is:
// e^-t = 2^hi e^lo with lo = -t - hi ln 2, and e^lo = 1 + lo. (f8 2000 x 5001 with SILU: 9
// elements beside the 64-bit result's, 10 with correctly rounded steps; times_sigmoid has twice
// as many, and gate_pack takes 14.5 us with it, so 16.0, with a Newton step behind the
// reciprocal, too, 16.7.) Beyond 126 ln 2 the sigmoid is no normal f32 any more: below that it is
// zero, also times the lowest numbers, which masks are made of.
__device__ __forceinline__ float times_sigmoid_close(float x, float t) {
  constexpr float kLog2e = 1.44269502f, kLn2 = 0.693147182f, kMost = 87.3365448f;
  const bool none = t < -kMost;
  t = __builtin_amdgcn_fmed3f(t, -kMost, kMost);
  const float hi = -kLog2e * t;
  const float lo = __builtin_fmaf(-kLn2, hi, -t);
  const float e = __builtin_amdgcn_exp2f(hi);
  return x * (none ? 0.0f : __builtin_amdgcn_rcpf(__builtin_fmaf(e, lo, 1.0f + e)));
}

// x Phi(x) with Phi(x) = erfc(-x / sqrt 2) / 2. With s = |x| and tail = s erfc(s / sqrt 2) / 2
// it is s - tail for positive x and -tail for negative, so nothing cancels in the negative tail.
// erfc(s / sqrt 2) / 2 = e^(-s^2 / 2) p(t) with t = 1 / (1 + 0.4 s / sqrt 2), and p, without a
// constant term, was fitted for the smallest largest error of the tail: with the constants as they
// are rounded 7.5e-9 for all s and 1.2e-7 s near zero. With the roundings of f32 it is 3.2e-7 |x| off
// at most (measured from 1e-6 on, at |x| = 0.001), 3.4e-8 of the root mean square for normal x.
// (Of 10 million 8-bit roundings 3 are not those of exact values; with five terms, to 1.7e-7
// at their best, 5. erfcf is closer yet, at branches between lanes: gate 2048 x 28672
// 114 us where this takes 75.)
__device__ __forceinline__ float gelu(float x) {
  // (From 64 on the tail is zero, an infinite x, whose tail would be infinity times zero, among them.)
  const float s = __builtin_fminf(__builtin_fabsf(x), 64.0f);
  const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.282842726f, s, 1.0f));
  float p = __builtin_fmaf(-0.103000157f, t, 0.36618006f);
  p = __builtin_fmaf(p, t, -0.204105198f);
  p = __builtin_fmaf(p, t, 0.249023885f);
  p = __builtin_fmaf(p, t, 0.0750114322f);
  p = __builtin_fmaf(p, t, 0.116889864f);
  const float tail = s * (p * t * __builtin_amdgcn_exp2f(-0.72134752f * s * s));
  return (x < 0.0f ? 0.0f : x) - tail;   // (a NaN is not below zero, and stays)
}

// `act` is an IREE_UK_AMD_FLAG_ACTIVATION_* value, the same in all lanes. The comparison of
// RELU lets a NaN through.
template <bool CLOSE = false>
__device__ __forceinline__ float activate(float x, uint32_t act) {
  auto times_sigmoid = [](float v, float t) { return CLOSE ? times_sigmoid_close(v, t) : uk::times_sigmoid(v, t); };
  switch (act) {
    case IREE_UK_AMD_FLAG_ACTIVATION_RELU: return x < 0.0f ? 0.0f : x;
    case IREE_UK_AMD_FLAG_ACTIVATION_GELU: return gelu(x);
    // tanh(u) = 2 sigmoid(2 u) - 1, so x / 2 * (1 + tanh(u)) = x sigmoid(2 u).
    case IREE_UK_AMD_FLAG_ACTIVATION_GELU_TANH:
      return times_sigmoid(x, x * __builtin_fmaf(0.0713548163f, x * x, 1.59576912f));
    case IREE_UK_AMD_FLAG_ACTIVATION_SILU: return times_sigmoid(x, x);
    default: return x;
  }
}

// The activation of N elements, by one test of the activation for all of them.
template <bool CLOSE = false, int N>
__device__ __forceinline__ void activate_all(float (&z)[N], uint32_t act) {
  auto each = [&](auto act_c) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = activate<CLOSE>(z[i], decltype(act_c)::value);
  };
  if (act == IREE_UK_AMD_FLAG_ACTIVATION_NONE) return;
  if (act == IREE_UK_AMD_FLAG_ACTIVATION_SILU) each(std::integral_constant<uint32_t, IREE_UK_AMD_FLAG_ACTIVATION_SILU>{});
  else if (act == IREE_UK_AMD_FLAG_ACTIVATION_GELU_TANH)
    each(std::integral_constant<uint32_t, IREE_UK_AMD_FLAG_ACTIVATION_GELU_TANH>{});
  else if (act == IREE_UK_AMD_FLAG_ACTIVATION_GELU) each(std::integral_constant<uint32_t, IREE_UK_AMD_FLAG_ACTIVATION_GELU>{});
  else each(std::integral_constant<uint32_t, IREE_UK_AMD_FLAG_ACTIVATION_RELU>{});
}

// f32 to and from the 16-bit floats, rounded to nearest even, subnormals kept.
struct F32 {
  typedef float T;
  static __device__ __forceinline__ float to_f32(T v) { return v; }
  static __device__ __forceinline__ T from_f32(float v) { return v; }
};
struct F16 {
  typedef _Float16 T;
  static __device__ __forceinline__ float to_f32(T v) { return (float)v; }
  static __device__ __forceinline__ T from_f32(float v) { return (_Float16)v; }
};
struct BF16 {
  typedef __bf16 T;
  static __device__ __forceinline__ float to_f32(T v) { return (float)v; }
  static __device__ __forceinline__ T from_f32(float v) { return (__bf16)v; }
};

}  // namespace uk

#endif  // IREE_UK_AMD_ACTIVATION_H_
