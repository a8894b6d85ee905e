// What lies between the sums of a matrix-core product and the row-major matrix of
// iree_uk_amd_mmt4d_epilogue_unpack: scales, bias, activation, residual, and the one
// rounding to the matrix's type. Device code of the instances for Elem::k...Ep.
#ifndef IREE_UK_AMD_MMT4D_MFMA_EPILOGUE_H_
#define IREE_UK_AMD_MMT4D_MFMA_EPILOGUE_H_

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "uk_activation.h"

namespace uk_mfma {

struct Epilogue {
  uint32_t out_type, act;     // IREE_UK_AMD_FLAG_OUT_TYPE_*, IREE_UK_AMD_FLAG_ACTIVATION_*
  uint32_t out_bytes;         // of an element
  uint32_t swapped;           // mmt4d_mfma_thin.h: the kernel's rows are the caller's columns
  int64_t out_pitch;          // bytes between rows of the matrix
  const float* bias;          // of the caller's columns; null: none
  const char* residual;       // null: none
  int64_t residual_pitch;     // bytes
};

// N consecutive elements of a row of the out type, at any address of its elements.
template <typename F, int N>
struct RowPiece {
  typedef typename F::T V __attribute__((ext_vector_type(N)));
  typedef V Any __attribute__((aligned(sizeof(typename F::T))));
};

// f(F32{}), f(F16{}) or f(BF16{}), by the out type (the same in all lanes).
template <typename Body>
__device__ __forceinline__ void by_out_type(const Epilogue& ep, Body&& f) {
  if (ep.out_type == IREE_UK_AMD_FLAG_OUT_TYPE_BF16) f(uk::BF16{});
  else if (ep.out_type == IREE_UK_AMD_FLAG_OUT_TYPE_F16) f(uk::F16{});
  else f(uk::F32{});
}

// Elements (row, col) .. (row, col + N - 1) of the matrix, of which `left` exist (N and
// more: all): those of the residual (there is one) as f32, zeros where there are none.
template <typename F, int N>
__device__ __forceinline__ void load_residual(const Epilogue& ep, int row, int col, int left, float (&v)[N]) {
  const char* p = ep.residual + (int64_t)row * ep.residual_pitch + (int64_t)col * (int)sizeof(typename F::T);
  if (left >= N) {
    const auto x = *reinterpret_cast<const typename RowPiece<F, N>::Any*>(p);
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = F::to_f32(x[e]);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) v[e] = e < left ? F::to_f32(reinterpret_cast<const typename F::T*>(p)[e]) : 0.0f;
  }
}

// The same elements, rounded and stored.
template <typename F, int N>
__device__ __forceinline__ void store_row(const Epilogue& ep, char* out, int row, int col, int left, const float (&v)[N]) {
  char* p = out + (int64_t)row * ep.out_pitch + (int64_t)col * (int)sizeof(typename F::T);
  if (left >= N) {
    typename RowPiece<F, N>::V x;
#pragma unroll
    for (int e = 0; e < N; ++e) x[e] = F::from_f32(v[e]);
    *reinterpret_cast<typename RowPiece<F, N>::Any*>(p) = x;
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e)
      if (e < left) reinterpret_cast<typename F::T*>(p)[e] = F::from_f32(v[e]);
  }
}

// The activation of N elements, as close as the matrix's type shows: an f32 one shows the |t|
// units that a sigmoid may be off (3.7e-6 of the value near t = -80, so 3.7e-7), a 16-bit one,
// whose half steps are 4.9e-4 and more of it, does not.
template <int N>
__device__ __forceinline__ void activate_for(const Epilogue& ep, float (&z)[N]) {
  if (ep.out_type == IREE_UK_AMD_FLAG_OUT_TYPE_F32) uk::activate_all<true>(z, ep.act);
  else uk::activate_all(z, ep.act);
}

// residual + activation(z) of such elements, stored; z has its bias.
template <int N>
__device__ __forceinline__ void finish_row(const Epilogue& ep, char* out, int row, int col, int left, float (&z)[N]) {
  activate_for(ep, z);
  by_out_type(ep, [&](auto type) __attribute__((always_inline)) {
    using F = decltype(type);
    if (ep.residual) {
      float rv[N];
      load_residual<F>(ep, row, col, left, rv);
#pragma unroll
      for (int e = 0; e < N; ++e) z[e] += rv[e];
    }
    store_row<F>(ep, out, row, col, left, z);
  });
}

}  // namespace uk_mfma

#endif  // IREE_UK_AMD_MMT4D_MFMA_EPILOGUE_H_
