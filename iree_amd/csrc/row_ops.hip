// Row-wise steps into tiles: iree_uk_amd_rmsnorm_pack and iree_uk_amd_gate_pack.
//
// Norm: with h = in + residual, u = h * weight and r = 1 / sqrt(mean(h^2) + epsilon), the
// result is y = u * r. An 8-bit form divides y by max|y| / largest, in which r cancels:
// q = round(u * (largest / max|u|)), so one pass over a row gives both sums that its
// output needs (of h^2 and the maximum of |u|).
// Gate: u = activation(gate) * up and r = 1.
#include <hip/hip_runtime.h>

#include "uk_activation.h"
#include "uk_device_common.h"
#include "uk_hip_abi.h"
#include "uk_launch.h"

namespace {

constexpr int kThreads = 256;
constexpr float kLargestS8 = 127.0f, kLargestF8 = 448.0f;

struct RowArgs {
  const char* in;
  const char* second;   // residual or up; null: none
  char* sum;            // null: not asked for
  const char* weight;   // null: ones
  char* out;
  float* row_scale;
  int64_t in_stride, second_stride, sum_stride, out_stride;  // bytes
  int32_t rows, cols, padded_cols, M0, K0;
  uk::FastDiv by_m0, by_k0;
  float epsilon;
  uint32_t act;
};

// How the rows of a call end up in tiles.
enum class Form { kSame, kS8, kF8 };

// Bits of the largest |v|: as integers, NaN and infinity are above every number.
__device__ __forceinline__ uint32_t larger(uint32_t a, float v) {
  return max(a, __float_as_uint(v) & 0x7FFFFFFFu);
}

template <bool NORM, typename IN, Form FORM>
__global__ __launch_bounds__(kThreads) void row_op_kernel(RowArgs a) {
  using T = typename IN::T;
  const uint32_t row = blockIdx.x;
  const uint32_t pm = a.by_m0.div(row), m0 = row - pm * (uint32_t)a.M0;
  constexpr int OB = FORM == Form::kSame ? (int)sizeof(T) : 1;
  char* out = a.out + (int64_t)pm * a.out_stride + (int64_t)m0 * a.K0 * OB;
  auto at = [&](int c) {
    const int64_t kt = a.by_k0.div((uint32_t)c);
    return out + (kt * a.M0 * a.K0 + (c - kt * a.K0)) * OB;
  };
  auto put_zero = [&](int c) {
    if constexpr (FORM == Form::kSame) *reinterpret_cast<T*>(at(c)) = IN::from_f32(0.0f);
    else *at(c) = 0;
  };
  if ((int)row >= a.rows) {
    for (int c = threadIdx.x; c < a.padded_cols; c += kThreads) put_zero(c);
    return;
  }
  const T* in = reinterpret_cast<const T*>(a.in + (int64_t)row * a.in_stride);
  const T* second = reinterpret_cast<const T*>(a.second + (int64_t)row * a.second_stride);
  T* sum = reinterpret_cast<T*>(a.sum + (int64_t)row * a.sum_stride);
  const T* weight = reinterpret_cast<const T*>(a.weight);
  // h of column c (norm), then u.
  auto h_of = [&](int c) {
    float v = IN::to_f32(in[c]);
    if constexpr (NORM) {
      if (a.second) v += IN::to_f32(second[c]);
    }
    return v;
  };
  auto u_of = [&](int c, float h) {
    if constexpr (NORM) return a.weight ? h * IN::to_f32(weight[c]) : h;
    float v = uk::activate(h, a.act);
    return a.second ? v * IN::to_f32(second[c]) : v;
  };
  __shared__ float part_squares[kThreads];
  __shared__ uint32_t part_largest[kThreads];
  float squares = 0.0f;
  uint32_t largest = 0;
  for (int c = threadIdx.x; c < a.cols; c += kThreads) {
    const float h = h_of(c);
    if constexpr (NORM) squares += h * h;
    if constexpr (FORM != Form::kSame) largest = larger(largest, u_of(c, h));
  }
  part_squares[threadIdx.x] = squares;
  part_largest[threadIdx.x] = largest;
  __syncthreads();
  for (int half = kThreads / 2; half > 0; half /= 2) {
    if ((int)threadIdx.x < half) {
      part_squares[threadIdx.x] += part_squares[threadIdx.x + half];
      part_largest[threadIdx.x] = max(part_largest[threadIdx.x], part_largest[threadIdx.x + half]);
    }
    __syncthreads();
  }
  float r = 1.0f;
  if constexpr (NORM) {
    const float mean = a.cols ? part_squares[0] / (float)a.cols : 0.0f;
    // (an infinite sum is none that a norm can be taken of)
    r = mean < __builtin_inff() ? 1.0f / __builtin_sqrtf(mean + a.epsilon) : __builtin_nanf("");
    if (!a.cols) r = 1.0f;
  }
  float inverse = 0.0f;
  if constexpr (FORM != Form::kSame) {
    constexpr float kLargest = FORM == Form::kS8 ? kLargestS8 : kLargestF8;
    const float top = __uint_as_float(part_largest[0]), top_y = top * r;
    float scale;
    if (!(top_y < __builtin_inff())) scale = __builtin_nanf("");
    else if (top_y < 0x1p-100f || top < 0x1p-110f) scale = 0.0f;
    else { scale = top_y / kLargest; inverse = kLargest / top; }
    if (threadIdx.x == 0) a.row_scale[row] = scale;
  }
  for (int c = threadIdx.x; c < a.padded_cols; c += kThreads) {
    if (c >= a.cols) { put_zero(c); continue; }
    const float h = h_of(c), u = u_of(c, h);
    // (Where sum is one of the inputs, this thread alone has read what it now overwrites.)
    if constexpr (NORM) {
      if (a.sum) sum[c] = IN::from_f32(h);
    }
    if constexpr (FORM == Form::kSame) {
      *reinterpret_cast<T*>(at(c)) = IN::from_f32(u * r);
    } else {
      // (inverse 0: a row without an 8-bit form, zeros whatever it holds)
      float q = inverse != 0.0f ? u * inverse : 0.0f;
      constexpr float kLargest = FORM == Form::kS8 ? kLargestS8 : kLargestF8;
      q = __builtin_fminf(__builtin_fmaxf(q, -kLargest), kLargest);
      if constexpr (FORM == Form::kS8) *at(c) = (char)(int)__builtin_rintf(q);
      else *at(c) = (char)__builtin_amdgcn_cvt_pk_fp8_f32(q, q, 0, false);
    }
  }
}

}  // namespace

extern "C" int iree_uk_amd_hip_launch_row_op(const iree_uk_amd_row_op_t* p, void* stream_v,
                                             const char** kernel_name) {
  const uint32_t out = p->flags & IREE_UK_AMD_FLAG_OUT_TYPE_MASK;
  const Form form = out == IREE_UK_AMD_FLAG_OUT_TYPE_S8         ? Form::kS8
                    : out == IREE_UK_AMD_FLAG_OUT_TYPE_F8E4M3FN ? Form::kF8
                                                                : Form::kSame;
  const uint32_t in = p->flags & IREE_UK_AMD_FLAG_IN_TYPE_MASK;
  const int es = in == IREE_UK_AMD_FLAG_IN_TYPE_F32 ? 4 : 2, os = form == Form::kSame ? es : 1;
  RowArgs a{};
  a.in = (const char*)p->in;
  a.second = (const char*)p->second;
  a.sum = (char*)p->sum;
  a.weight = (const char*)p->weight;
  a.out = (char*)p->out;
  a.row_scale = p->row_scale;
  a.in_stride = p->in_stride0 * es;
  a.second_stride = p->second_stride0 * es;
  a.sum_stride = p->sum_stride0 * es;
  a.out_stride = p->out_stride0 * os;
  a.rows = (int32_t)p->rows;
  a.cols = (int32_t)p->cols;
  a.padded_cols = (int32_t)(p->K1 * p->K0);
  a.M0 = (int32_t)p->M0;
  a.K0 = (int32_t)p->K0;
  a.by_m0 = uk::FastDiv((uint32_t)p->M0);
  a.by_k0 = uk::FastDiv((uint32_t)p->K0);
  a.epsilon = p->epsilon;
  a.act = p->flags & IREE_UK_AMD_FLAG_ACTIVATION_MASK;
  const dim3 grid((uint32_t)(p->M1 * p->M0)), block(kThreads);
  hipStream_t stream = (hipStream_t)stream_v;
  *kernel_name = p->norm ? "rmsnorm_pack" : "gate_pack";
  auto go = [&](auto norm, auto in_type) {
    constexpr bool N = decltype(norm)::value;
    using IN = decltype(in_type);
    auto kernel = form == Form::kS8   ? row_op_kernel<N, IN, Form::kS8>
                  : form == Form::kF8 ? row_op_kernel<N, IN, Form::kF8>
                                      : row_op_kernel<N, IN, Form::kSame>;
    uk::launch(0, kernel, grid, block, 0, stream, a);
  };
  auto by_type = [&](auto norm) {
    if (in == IREE_UK_AMD_FLAG_IN_TYPE_F32) go(norm, uk::F32{});
    else if (in == IREE_UK_AMD_FLAG_IN_TYPE_F16) go(norm, uk::F16{});
    else go(norm, uk::BF16{});
  };
  if (p->norm) by_type(std::true_type{});
  else by_type(std::false_type{});
  return (int)hipGetLastError();
}
