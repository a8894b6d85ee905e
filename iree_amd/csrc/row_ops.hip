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
  int32_t rows, tiled_rows, cols, padded_cols, M0, K0;   // tiled_rows: M1 * M0
  int32_t log_waves, rows_a_block, piece;   // rows in registers: waves a row, rows a workgroup, columns next to each other
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

// 1 / sqrt(mean + epsilon); an infinite sum is none that a norm can be taken of, and a row
// without columns has nothing to divide.
__device__ __forceinline__ float reciprocal_norm(float squares, int cols, float epsilon) {
  if (cols == 0) return 1.0f;
  const float mean = squares / (float)cols;
  return mean < __builtin_inff() ? 1.0f / __builtin_sqrtf(mean + epsilon) : __builtin_nanf("");
}

// The scale of a row whose largest |u| is `top`, and the factor that takes u to its 8-bit
// form; 0 for a row that has none.
template <Form FORM>
__device__ __forceinline__ void eight_bit_scale(float top, float r, float& scale, float& factor) {
  constexpr float kLargest = FORM == Form::kS8 ? kLargestS8 : kLargestF8;
  const float top_y = top * r;
  factor = 0.0f;
  if (!(top_y < __builtin_inff())) scale = __builtin_nanf("");
  else if (top_y < 0x1p-100f || top < 0x1p-110f) scale = 0.0f;
  else {
    scale = top_y / kLargest;
    factor = kLargest / top;
  }
}

// ---- rows in registers ---------------------------------------------------------
//
// 2^a.log_waves waves a row, a lane holding C chunks of 8 columns, one 16-byte load of a
// 16-bit type, so that the loads of a wave cover neighbouring lines (chunks of two loads, whose
// lanes lie 32 bytes apart: norm 2048 x 8192 bf16 28.8 us, this 26.2; gate 2000 x 5001 17.8 and
// 16.0). A row is read once, its reductions go over the lanes and, through LDS, over the waves,
// and what is stored comes out of registers.
//
// Bound by memory, with every byte moved once (measured: norm 2048 x 8192 bf16 into f8 reads
// 67 MB and writes 49, gate 2048 x 28672 235 and 58): 26.2 us (4.5 TB/s) and 63.5 us (4.6 TB/s),
// where a copy of 1 GiB by torch moves 4.8 TB/s, by the best of the kernels tried 5.8. The
// vector ALU is busy for over half of the gate's time (the exponential and the reciprocal of
// SILU). Small calls are the launch and one round trip: norm 1 x 4096 4.6 us, pack of as many
// bytes 4.0.
constexpr int kChunk = 8;
constexpr int kMaxThreads = 1024;

template <typename T, int N>
struct Any {
  typedef T V __attribute__((ext_vector_type(N)));
  typedef V At __attribute__((aligned(sizeof(T))));   // at any address of its elements
};

// Columns c .. c + 7 of a row as they lie in memory. Loading and using them are two steps,
// and no lane branches in the first: what a kernel loads is then in flight together, one
// round trip to memory where `load, convert` for each of residual and weight made three.
template <typename IN>
struct Chunk {
  using T = typename IN::T;
  static constexpr int PIECES = (int)sizeof(T) / 2, N = kChunk / PIECES;   // of 16 bytes; columns of one
  uint32_t w[PIECES][4];

  // `row_bytes` > 0: of the row. A piece beyond its end is loaded from its last 16 bytes.
  __device__ __forceinline__ void load(const char* row, int c, uint32_t row_bytes) {
    typedef uint32_t v4u __attribute__((ext_vector_type(4)));
    typedef v4u v4u_any __attribute__((aligned(1)));
    const uint32_t off = (uint32_t)c * (uint32_t)sizeof(T);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      if (row_bytes >= 16) {   // (the same in all lanes)
        const v4u x = *reinterpret_cast<const v4u_any*>(row + uk::clipped_offset<16>(off + 16 * p, row_bytes));
#pragma unroll
        for (int i = 0; i < 4; ++i) w[p][i] = x[i];
      } else {
        uk::load_short_row<16>(w[p], row, off + 16 * p == 0 ? (int32_t)row_bytes : 0, 0);
      }
    }
  }
  // Those columns as f32, zeros beyond the row.
  __device__ __forceinline__ void values(int c, uint32_t row_bytes, float (&v)[kChunk]) {
    const uint32_t off = (uint32_t)c * (uint32_t)sizeof(T);
#pragma unroll
    for (int p = 0; p < PIECES; ++p) {
      if (row_bytes >= 16) uk::clip_piece<16>(w[p], uk::row_bytes_left(row_bytes, off + 16 * p), 0);
      const auto x = __builtin_bit_cast(typename Any<T, N>::V, w[p]);
#pragma unroll
      for (int e = 0; e < N; ++e) v[p * N + e] = IN::to_f32(x[e]);
    }
  }
};

// The elements of a chunk, of OB bytes, in words, to the tiles of a row: `at(column)` is where a column
// goes. Runs of `piece` columns lie next to each other (8, 4, or else single ones).
template <int OB, typename At>
__device__ __forceinline__ void store_chunk(const uint32_t (&w)[kChunk * OB / 4], int c, int padded_cols, int piece, At at) {
  typedef uint32_t v4u __attribute__((ext_vector_type(4)));
  typedef v4u v4u_any __attribute__((aligned(1)));
  typedef uint32_t v2u __attribute__((ext_vector_type(2)));
  typedef v2u v2u_any __attribute__((aligned(1)));
  typedef uint32_t u32_any __attribute__((aligned(1)));
  auto store_run = [&](auto columns) __attribute__((always_inline)) {
    constexpr int P = decltype(columns)::value, WORDS = P * OB / 4;
#pragma unroll
    for (int j = 0; j < kChunk; j += P) {
      if (c + j >= padded_cols) break;
      char* p = at(c + j);
      const int first = j * OB / 4;
      if constexpr (WORDS == 1) *reinterpret_cast<u32_any*>(p) = w[first];
      else if constexpr (WORDS == 2) *reinterpret_cast<v2u_any*>(p) = v2u{w[first], w[first + 1]};
      else
#pragma unroll
        for (int i = 0; i < WORDS; i += 4)
          *reinterpret_cast<v4u_any*>(p + 4 * i) = v4u{w[first + i], w[first + i + 1], w[first + i + 2], w[first + i + 3]};
    }
  };
  if (piece == 8) store_run(std::integral_constant<int, 8>{});
  else if (piece == 4) store_run(std::integral_constant<int, 4>{});
  else {
#pragma unroll
    for (int j = 0; j < kChunk; ++j) {
      if (c + j >= padded_cols) break;
      const uint32_t word = w[j * OB / 4];
      if constexpr (OB == 1) *at(c + j) = (char)(word >> 8 * (j % 4));
      else if constexpr (OB == 2) *reinterpret_cast<uint16_t*>(at(c + j)) = (uint16_t)(word >> 16 * (j % 2));
      else *reinterpret_cast<uint32_t*>(at(c + j)) = word;
    }
  }
}

template <bool NORM, typename IN, Form FORM, int C>
__global__ __launch_bounds__(kMaxThreads) void row_op_kernel(RowArgs a) {
  using T = typename IN::T;
  constexpr int OB = FORM == Form::kSame ? (int)sizeof(T) : 1;
  __shared__ float part_squares[kMaxThreads / 64];
  __shared__ uint32_t part_largest[kMaxThreads / 64];
  uk::fetch_arguments<sizeof(RowArgs)>();
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  // Consecutive workgroups go to the 8 XCDs in turn, each with an L2 of its own: every XCD
  // takes a contiguous share of the rows, so that the pieces which neighbouring rows put
  // into one line of a tile meet in one L2.
  const uint32_t per_xcd = gridDim.x >> 3;
  const uint32_t block = blockIdx.x < per_xcd * 8 ? (blockIdx.x & 7) * per_xcd + (blockIdx.x >> 3)
                                                          : blockIdx.x;
  const int log_waves = a.log_waves, waves = 1 << log_waves;
  const uint32_t row = block * (uint32_t)a.rows_a_block + (uint32_t)(wave >> log_waves);
  const bool exists = row < (uint32_t)a.rows, tiled = row < (uint32_t)a.tiled_rows;
  const int first = ((wave & (waves - 1)) * 64 + lane) * kChunk, step = waves * 64 * kChunk;
  const uint32_t pm = a.by_m0.div(row), m0 = row - pm * (uint32_t)a.M0;
  const char* in = a.in + (int64_t)row * a.in_stride;
  const char* second = a.second + (int64_t)row * a.second_stride;
  float u[C][kChunk];
  float squares[4] = {0.0f, 0.0f, 0.0f, 0.0f};
  uint32_t largest = 0;
  const uint32_t row_bytes = (uint32_t)a.cols * (uint32_t)sizeof(T);
  if (exists && a.cols > 0) {   // (the same in all lanes of a wave)
    // (Up to four chunks together: the registers of more.)
    constexpr int P = C <= 4 ? C : 4;
    Chunk<IN> x[P], y[P], z[NORM ? P : 1];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = first + i * step, k = i % P;
      if (k == 0) {
#pragma unroll
        for (int j = 0; j < P && i + j < C; ++j) {
          x[j].load(in, c + j * step, row_bytes);
          if (a.second) y[j].load(second, c + j * step, row_bytes);
          if (NORM && a.weight) z[j].load(a.weight, c + j * step, row_bytes);
        }
      }
      float v[kChunk];
      x[k].values(c, row_bytes, u[i]);
      if constexpr (NORM) {
        if (a.second) {
          y[k].values(c, row_bytes, v);
#pragma unroll
          for (int e = 0; e < kChunk; ++e) u[i][e] += v[e];
        }
#pragma unroll
        for (int e = 0; e < kChunk; ++e) squares[e % 4] += u[i][e] * u[i][e];
        if (a.sum && c < a.cols) {
          T* sum = reinterpret_cast<T*>(a.sum + (int64_t)row * a.sum_stride) + c;
          if (c + kChunk <= a.cols) {
            constexpr int N = 16 / sizeof(T);
#pragma unroll
            for (int j = 0; j < kChunk; j += N) {
              typename Any<T, N>::V h;
#pragma unroll
              for (int e = 0; e < N; ++e) h[e] = IN::from_f32(u[i][j + e]);
              *reinterpret_cast<typename Any<T, N>::At*>(sum + j) = h;
            }
          } else {
#pragma unroll
            for (int e = 0; e < kChunk; ++e)
              if (c + e < a.cols) sum[e] = IN::from_f32(u[i][e]);
          }
        }
        if (a.weight) {
          z[k].values(c, row_bytes, v);
#pragma unroll
          for (int e = 0; e < kChunk; ++e) u[i][e] *= v[e];
        }
      } else {
        uk::activate_all<true>(u[i], a.act);
        if (a.second) {
          y[k].values(c, row_bytes, v);
#pragma unroll
          for (int e = 0; e < kChunk; ++e) u[i][e] *= v[e];
        }
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int e = 0; e < kChunk; ++e) u[i][e] = 0.0f;
  }
  float total = (squares[0] + squares[1]) + (squares[2] + squares[3]);
  if constexpr (FORM != Form::kSame) {
#pragma unroll
    for (int i = 0; i < C; ++i)
#pragma unroll
      for (int e = 0; e < kChunk; ++e) largest = larger(largest, u[i][e]);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    if constexpr (NORM) total += __shfl_xor(total, d);
    if constexpr (FORM != Form::kSame) largest = max(largest, (uint32_t)__shfl_xor((int)largest, d));
  }
  if (waves > 1) {
    if (lane == 0) {
      part_squares[wave] = total;
      part_largest[wave] = largest;
    }
    __syncthreads();
    const int w0 = wave & ~(waves - 1);
    total = 0.0f;
    largest = 0;
    for (int w = 0; w < waves; ++w) {
      total += part_squares[w0 + w];
      largest = max(largest, part_largest[w0 + w]);
    }
  }
  if (!tiled) return;
  float r = 1.0f;
  if constexpr (NORM) r = reciprocal_norm(total, a.cols, a.epsilon);
  float factor = exists ? r : 0.0f;   // (a row beyond the matrix has no sum of squares, and r may be infinite)
  if constexpr (FORM != Form::kSame) {
    float scale;
    eight_bit_scale<FORM>(__uint_as_float(largest), r, scale, factor);
    if (exists && (threadIdx.x & (waves * 64 - 1)) == 0) a.row_scale[row] = scale;
    if (factor == 0.0f) {   // (a row without an 8-bit form)
#pragma unroll
      for (int i = 0; i < C; ++i)
#pragma unroll
        for (int e = 0; e < kChunk; ++e) u[i][e] = 0.0f;
    }
  }
  char* out = a.out + (int64_t)pm * a.out_stride + (int64_t)m0 * a.K0 * OB;
  auto at = [&](int c) {
    const uint32_t kt = a.by_k0.div((uint32_t)c);
    return out + ((int64_t)kt * a.M0 * a.K0 + (c - kt * a.K0)) * OB;
  };
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = first + i * step;
    if (c >= a.padded_cols) break;
    uint32_t w[kChunk * OB / 4];
#pragma unroll
    for (int e = 0; e < kChunk; ++e) u[i][e] *= factor;
    if constexpr (NORM && FORM == Form::kSame) {
      // A row that has no norm is NaN, and zero times that: not so the columns beyond it.
      if (!(factor < __builtin_inff())) {
#pragma unroll
        for (int e = 0; e < kChunk; ++e)
          if (c + e >= a.cols) u[i][e] = 0.0f;
      }
    }
    if constexpr (FORM == Form::kS8) {
      // Adding 1.5 * 2^23 rounds to an integer, whose low bits are the sum's.
#pragma unroll
      for (int e = 0; e < kChunk; e += 4) {
        uint32_t b[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) b[k] = __float_as_uint(u[i][e + k] + 12582912.0f);
        w[e / 4] = __builtin_amdgcn_perm(__builtin_amdgcn_perm(b[3], b[2], 0x0C0C0400u),
                                         __builtin_amdgcn_perm(b[1], b[0], 0x0C0C0400u), 0x05040100u);
      }
    } else if constexpr (FORM == Form::kF8) {
#pragma unroll
      for (int e = 0; e < kChunk; e += 4) {
        int v = __builtin_amdgcn_cvt_pk_fp8_f32(u[i][e], u[i][e + 1], 0, false);
        w[e / 4] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(u[i][e + 2], u[i][e + 3], v, true);
      }
    } else {
      constexpr int N = 4 / sizeof(T);
#pragma unroll
      for (int e = 0; e < kChunk; e += N) {
        typename Any<T, N>::V x;
#pragma unroll
        for (int k = 0; k < N; ++k) x[k] = IN::from_f32(u[i][e + k]);
        w[e / N] = __builtin_bit_cast(uint32_t, x);
      }
    }
    store_chunk<OB>(w, c, a.padded_cols, a.piece, at);
  }
}

// ---- rows longer than what a workgroup's registers hold ---------------------------
//
// One workgroup a row, which it reads twice: for the two sums, and for the output. (Columns are
// counted without a sign: up to 2^31 - 1 of them, and a step more.)
template <bool NORM, typename IN, Form FORM>
__global__ __launch_bounds__(kThreads) void row_op_long_kernel(RowArgs a) {
  using T = typename IN::T;
  const uint32_t row = blockIdx.x;
  const uint32_t pm = a.by_m0.div(row), m0 = row - pm * (uint32_t)a.M0;
  constexpr int OB = FORM == Form::kSame ? (int)sizeof(T) : 1;
  char* out = a.out + (int64_t)pm * a.out_stride + (int64_t)m0 * a.K0 * OB;
  auto at = [&](uint32_t c) {
    const int64_t kt = a.by_k0.div(c);
    return out + (kt * a.M0 * a.K0 + (c - kt * a.K0)) * OB;
  };
  auto put_zero = [&](uint32_t c) {
    if constexpr (FORM == Form::kSame) *reinterpret_cast<T*>(at(c)) = IN::from_f32(0.0f);
    else *at(c) = 0;
  };
  if ((int)row >= a.rows) {
    for (uint32_t c = threadIdx.x; c < (uint32_t)a.padded_cols; c += kThreads) put_zero(c);
    return;
  }
  const T* in = reinterpret_cast<const T*>(a.in + (int64_t)row * a.in_stride);
  const T* second = reinterpret_cast<const T*>(a.second + (int64_t)row * a.second_stride);
  T* sum = reinterpret_cast<T*>(a.sum + (int64_t)row * a.sum_stride);
  const T* weight = reinterpret_cast<const T*>(a.weight);
  // h of column c (norm), then u.
  auto h_of = [&](uint32_t c) {
    float v = IN::to_f32(in[c]);
    if constexpr (NORM) {
      if (a.second) v += IN::to_f32(second[c]);
    }
    return v;
  };
  auto u_of = [&](uint32_t c, float h) {
    if constexpr (NORM) return a.weight ? h * IN::to_f32(weight[c]) : h;
    float v = uk::activate<true>(h, a.act);
    return a.second ? v * IN::to_f32(second[c]) : v;
  };
  __shared__ float part_squares[kThreads];
  __shared__ uint32_t part_largest[kThreads];
  float squares = 0.0f;
  uint32_t largest = 0;
  for (uint32_t c = threadIdx.x; c < (uint32_t)a.cols; c += kThreads) {
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
  if constexpr (NORM) r = reciprocal_norm(part_squares[0], a.cols, a.epsilon);
  float inverse = 0.0f;
  if constexpr (FORM != Form::kSame) {
    float scale;
    eight_bit_scale<FORM>(__uint_as_float(part_largest[0]), r, scale, inverse);
    if (threadIdx.x == 0) a.row_scale[row] = scale;
  }
  for (uint32_t c = threadIdx.x; c < (uint32_t)a.padded_cols; c += kThreads) {
    if (c >= (uint32_t)a.cols) { put_zero(c); continue; }
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
  a.tiled_rows = (int32_t)(p->M1 * p->M0);
  if (p->M0 == 1) {   // (rows as they are: one tile as wide as a row)
    a.K0 = a.padded_cols;
    a.by_k0 = uk::FastDiv((uint32_t)a.padded_cols);
  }
  hipStream_t stream = (hipStream_t)stream_v;
  *kernel_name = p->norm ? "rmsnorm_pack" : "gate_pack";
  // Waves a row: as many as leave a lane with two chunks, up to eight; then more chunks a lane,
  // and sixteen waves where those are too many. us with four / eight / sixteen waves: norm 2048 x
  // 4096 bf16 13.7 / 13.6 / -, 2048 x 8192 32.3 / 29.2 / 27.6, gate 2048 x 14336 37.5 / 35.0 / 34.1, 2048 x
  // 28672 - / 68.4 / 76.3. f32, whose chunks are two loads: as many as leave it with one, up to
  // sixteen (norm 2048 x 4096 31.4 / 26.7 / 27.7, gate 2048 x 8192 59.0 / 60.1 / 49.8). Rows that leave
  // units idle take sixteen before they take a third chunk: gate 16 x 14336 8.6 / 7.3 / 7.0.
  const int64_t chunks = uk::ceil_div(a.padded_cols, kChunk), most = p->norm ? 4 : 8;
  const int64_t wanted = es == 4 ? 1 : 2;
  const int up_to = es == 4 || a.tiled_rows <= 256 ? 4 : 3;
  int log_waves = 0;
  while (log_waves < up_to && (wanted * 64 << log_waves) < chunks) ++log_waves;
  if (most * (64 << log_waves) < chunks) log_waves = 4;
  const int64_t each = uk::ceil_div(chunks, (int64_t)64 << log_waves);
  const bool in_registers = each <= most;
  a.log_waves = log_waves;
  const int row_threads = 64 << log_waves;
  const int threads = row_threads < 256 && a.tiled_rows > 1 ? 256 : row_threads;
  a.rows_a_block = threads / row_threads;
  a.piece = (int32_t)uk::pow2_divisor(a.K0, 8);
  auto go = [&](auto norm, auto in_type, auto form_c) {
    constexpr bool N = decltype(norm)::value;
    constexpr Form F = decltype(form_c)::value;
    using IN = decltype(in_type);
    // (An instance for every number of chunks: with powers of two alone gate 2048 x 11008 took
    // 29.6 us, so 26.2, 2048 x 28672 66.3 and 63.5, norm 2048 x 12288 38.5 and 37.0.)
    using Kernel = void (*)(RowArgs);
    static constexpr Kernel by_chunks[8] = {
        row_op_kernel<N, IN, F, 1>,         row_op_kernel<N, IN, F, 2>,         row_op_kernel<N, IN, F, 3>,
        row_op_kernel<N, IN, F, 4>,         row_op_kernel<N, IN, F, N ? 4 : 5>, row_op_kernel<N, IN, F, N ? 4 : 6>,
        row_op_kernel<N, IN, F, N ? 4 : 7>, row_op_kernel<N, IN, F, N ? 4 : 8>};
    const Kernel kernel = by_chunks[in_registers && each > 1 ? each - 1 : 0];
    // A grid has fewer than 2^32 threads: whole tiles of up to 2^21 rows a launch (a tile
    // has 4096 bytes at most, so 4096 rows).
    const int64_t most_panels = (1ll << 21) / p->M0;
    for (int64_t m = 0; m < p->M1; m += most_panels) {
      const int64_t first = m * p->M0, panels = p->M1 - m < most_panels ? p->M1 - m : most_panels;
      RowArgs b = a;
      b.in += first * a.in_stride;
      if (a.second) b.second += first * a.second_stride;
      if (a.sum) b.sum += first * a.sum_stride;
      b.out += m * a.out_stride;
      if (a.row_scale) b.row_scale += first;
      b.rows = (int32_t)(p->rows > first ? p->rows - first : 0);
      b.tiled_rows = (int32_t)(panels * p->M0);
      if (b.rows > b.tiled_rows) b.rows = b.tiled_rows;
      if (in_registers)
        uk::launch(0, kernel, dim3((uint32_t)uk::ceil_div(b.tiled_rows, a.rows_a_block)), dim3((uint32_t)threads), 0, stream, b);
      else
        uk::launch(0, row_op_long_kernel<N, IN, F>, dim3((uint32_t)b.tiled_rows), dim3(kThreads), 0, stream, b);
    }
  };
  auto by_form = [&](auto norm, auto in_type) {
    if (form == Form::kS8) go(norm, in_type, std::integral_constant<Form, Form::kS8>{});
    else if (form == Form::kF8) go(norm, in_type, std::integral_constant<Form, Form::kF8>{});
    else go(norm, in_type, std::integral_constant<Form, Form::kSame>{});
  };
  auto by_type = [&](auto norm) {
    if (in == IREE_UK_AMD_FLAG_IN_TYPE_F32) by_form(norm, uk::F32{});
    else if (in == IREE_UK_AMD_FLAG_IN_TYPE_F16) by_form(norm, uk::F16{});
    else by_form(norm, uk::BF16{});
  };
  if (p->norm) by_type(std::true_type{});
  else by_type(std::false_type{});
  return (int)hipGetLastError();
}
