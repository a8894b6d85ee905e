// mmt4d kernel selection: MFMA kernels where one covers (type, M0, N0, K0),
// otherwise the any-shape scalar kernel.
#include <hip/hip_runtime.h>

#include "mmt4d_mfma_epilogue.h"
#include "uk_device_common.h"
#include "uk_hip_abi.h"
#include "uk_launch.h"

extern "C" int iree_uk_amd_hip_launch_mmt4d_generic(
    const iree_uk_mmt4d_params_t* p, const iree_uk_amd_rowmajor_out_t* rowmajor,
    void* stream);
extern "C" int iree_uk_amd_hip_launch_mmt4d_mfma(
    const iree_uk_mmt4d_params_t* p, const iree_uk_amd_rowmajor_out_t* rowmajor,
    void* stream, int forced_variant, const char** kernel_name);
extern "C" int iree_uk_amd_hip_mmt4d_mfma_supported(int32_t M0, int32_t N0,
                                                    int32_t K0, uint32_t flags);
extern "C" int iree_uk_amd_hip_launch_mmt4d_s16_widened(
    const iree_uk_mmt4d_params_t* p, const iree_uk_amd_rowmajor_out_t* rowmajor,
    void* stream, const char** kernel_name);
extern "C" int iree_uk_amd_hip_launch_mmt4d_retiled(
    const iree_uk_mmt4d_params_t* p, const iree_uk_amd_rowmajor_out_t* rowmajor,
    void* stream, const char** kernel_name);
extern "C" int iree_uk_amd_hip_launch_mmt4d_dot2(
    const iree_uk_mmt4d_params_t* p, const iree_uk_amd_rowmajor_out_t* rowmajor,
    void* stream);

namespace uk_mfma {
void note_k_slices(int n);  // mmt4d_mfma.hip: records the slice count of the call
// mmt4d_mfma.hip: a device buffer kept per host thread and stream; 1: none to be had (a
// stream under capture, for one).
int acquire_product_workspace(size_t bytes, hipStream_t stream, char** base);
}

namespace {
// Calls on this thread that iree_uk_mmt4d_info advertises a matrix-core kernel
// for but that the scalar kernel served (see iree_uk_amd_mfma_decline_count).
thread_local uint64_t g_declined = 0;
}  // namespace

extern "C" IREE_UK_AMD_EXPORT uint64_t iree_uk_amd_mfma_decline_count(void) { return g_declined; }

extern "C" int iree_uk_amd_hip_mmt4d_has_mfma_kernel(int32_t M0, int32_t N0,
                                                     int32_t K0,
                                                     uint32_t flags) {
  return iree_uk_amd_hip_mmt4d_mfma_supported(M0, N0, K0, flags);
}

namespace {

// Epilogue of a product that is already in memory, in f32 and with its scales: eight
// columns of a row a thread. May run in place. Bound by memory.
struct ApartArgs {
  const char* z;   // rows x cols of f32
  int64_t z_pitch;
  char* out;
  int32_t rows, cols, pieces;   // pieces: of eight columns, in all rows
  uk::FastDiv by_pieces;        // of a row
  uk_mfma::Epilogue ep;
};

__global__ __launch_bounds__(256) void mmt4d_epilogue_kernel(ApartArgs a) {
  const uint32_t id = blockIdx.x * 256 + threadIdx.x;
  if (id >= (uint32_t)a.pieces) return;
  uint32_t row, piece;
  a.by_pieces.divmod(id, row, piece);
  const int col = (int)piece * 8, left = a.cols - col;
  float z[8];
  const char* src = a.z + (int64_t)row * a.z_pitch + (int64_t)col * 4;
  if (left >= 8) {
    const auto v = *reinterpret_cast<const uk_mfma::RowPiece<uk::F32, 8>::Any*>(src);
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = v[e];
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) z[e] = e < left ? reinterpret_cast<const float*>(src)[e] : 0.0f;
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) z[e] += a.ep.bias ? a.ep.bias[min(col + e, a.cols - 1)] : 0.0f;
  uk_mfma::finish_row(a.ep, a.out, (int)row, col, left, z);
}

// The most f32 results that wait in the library's buffer for their epilogue: as much as
// the memory-side cache (256 MB) holds beside the matrix they go to. Larger products run
// in several rows of tiles.
constexpr int64_t kApartBytes = 64ll << 20;

// Whether the matrix of the call and its residual have bytes in common.
bool overlaps(const char* a, int64_t a_bytes, const char* b, int64_t b_bytes) {
  return a < b + b_bytes && b < a + a_bytes;
}

// The scaled product of 8-bit floats in f32, in tile rows of any width: by the kernels that end
// in an epilogue (here one that adds nothing), which multiply as f16 what goes into an f32
// matrix; rows under 16 bytes are regrouped first. The other kernels for 8-bit floats lose bits
// that such a matrix shows: 1.5e-5 of the root mean square off, these 3e-8 (300 x 300 x 1000 in
// rows of 8 bytes). Returns a HIP status.
int launch_f8_into_f32(const iree_uk_mmt4d_params_t* p, const iree_uk_amd_rowmajor_out_t* rm, void* stream,
                       int kernel_mode, const char** kernel_name) {
  iree_uk_amd_rowmajor_out_t r = *rm;
  r.epilogue = 1;
  r.epilogue_flags = IREE_UK_AMD_FLAG_OUT_TYPE_F32 | IREE_UK_AMD_FLAG_ACTIVATION_NONE;
  r.bias = nullptr;
  r.residual = nullptr;
  int st = iree_uk_amd_hip_launch_mmt4d_mfma(p, &r, stream, 0, kernel_name);
  if (st < 0 && kernel_mode == IREE_UK_AMD_KERNEL_MODE_AUTO)
    st = iree_uk_amd_hip_launch_mmt4d_retiled(p, &r, stream, kernel_name);
  if (st >= 0) return st;
  *kernel_name = "mmt4d_generic";
  return iree_uk_amd_hip_launch_mmt4d_generic(p, &r, stream);
}

// Types and tiles that have no kernel with an epilogue of its own (mmt4d_mfma.hip): the
// product into f32 with its scales, on whatever kernel serves it (8-bit floats into f32: one
// that keeps their bits), and the epilogue as a second launch; in place where the matrix is f32
// and its residual another one, else from a buffer. Returns a HIP status, or -1 where there is
// no buffer to be had.
int launch_epilogue_apart(const iree_uk_mmt4d_params_t* p, const iree_uk_amd_rowmajor_out_t* rm, void* stream,
                          int kernel_mode, const char** kernel_name) {
  ApartArgs a{};
  a.ep.out_type = rm->epilogue_flags & IREE_UK_AMD_FLAG_OUT_TYPE_MASK;
  a.ep.act = rm->epilogue_flags & IREE_UK_AMD_FLAG_ACTIVATION_MASK;
  a.ep.out_bytes = a.ep.out_type == IREE_UK_AMD_FLAG_OUT_TYPE_F32 ? 4 : 2;
  a.ep.out_pitch = rm->stride0 * a.ep.out_bytes;
  a.ep.bias = rm->bias;
  a.ep.residual_pitch = rm->residual_stride0 * a.ep.out_bytes;
  const int64_t row_bytes = rm->size1 * a.ep.out_bytes;
  const bool in_place = a.ep.out_bytes == 4 &&
                        !(rm->residual && overlaps((const char*)p->out_buffer, (rm->size0 - 1) * a.ep.out_pitch + row_bytes,
                                                   (const char*)rm->residual,
                                                   (rm->size0 - 1) * a.ep.residual_pitch + row_bytes));
  const bool f8_into_f32 = (p->flags & IREE_UK_FLAG_MMT4D_TYPE_MASK) == IREE_UK_AMD_FLAG_MMT4D_TYPE_F8E4M3FNF8E4M3FNF32 &&
                           a.ep.out_bytes == 4;
  const int64_t pieces = uk::ceil_div(rm->size1, 8);
  // Rows of tiles a launch: what the buffer holds, and 32-bit numbers of pieces.
  const int64_t panel = (int64_t)p->M0 * (in_place ? pieces * 32 : rm->size1 * 4);
  const int64_t panels = panel >= kApartBytes ? 1 : kApartBytes / panel;
  if ((int64_t)p->M0 * pieces >= (1ll << 31)) return -1;
  char* buffer = nullptr;
  if (!in_place) {
    const int64_t rows = rm->size0 < panels * p->M0 ? rm->size0 : panels * p->M0;
    if (uk_mfma::acquire_product_workspace((size_t)(rows * rm->size1 * 4), (hipStream_t)stream, &buffer) != 0) return -1;
  }
  for (int64_t m = 0; m < p->M && m * p->M0 < rm->size0; m += panels) {
    const int64_t first = m * p->M0;
    iree_uk_mmt4d_params_t q = *p;
    q.M = p->M - m < panels ? p->M - m : panels;
    q.lhs_offset = p->lhs_offset + m * p->lhs_stride0;
    iree_uk_amd_rowmajor_out_t r = *rm;
    r.epilogue = 0;
    r.size0 = rm->size0 - first < q.M * p->M0 ? rm->size0 - first : q.M * p->M0;
    if (rm->row_scale) r.row_scale = rm->row_scale + first;
    a.out = (char*)p->out_buffer + first * a.ep.out_pitch;
    if (!in_place) {
      q.out_buffer = buffer;
      q.out_offset = 0;
      r.stride0 = rm->size1;
    } else {
      q.out_buffer = a.out;
      q.out_offset = 0;
    }
    const int st = f8_into_f32 ? launch_f8_into_f32(&q, &r, stream, kernel_mode, kernel_name)
                               : iree_uk_amd_hip_launch_mmt4d(&q, &r, stream, kernel_mode, kernel_name);
    if (st != 0) return st;
    a.z = (const char*)q.out_buffer;
    a.z_pitch = r.stride0 * 4;
    a.rows = (int32_t)r.size0;
    a.cols = (int32_t)rm->size1;
    a.pieces = (int32_t)(r.size0 * pieces);
    a.by_pieces = uk::FastDiv((uint32_t)pieces);
    a.ep.residual = rm->residual ? (const char*)rm->residual + first * a.ep.residual_pitch : nullptr;
    uk::launch(2, mmt4d_epilogue_kernel, dim3((uint32_t)uk::ceil_div(a.pieces, 256)), dim3(256), 0, (hipStream_t)stream, a);
    const int launched = (int)hipGetLastError();
    if (launched != 0) return launched;
  }
  return 0;
}

}  // namespace

extern "C" int iree_uk_amd_hip_launch_mmt4d(const iree_uk_mmt4d_params_t* p,
                                            const iree_uk_amd_rowmajor_out_t* rowmajor,
                                            void* stream, int kernel_mode,
                                            const char** kernel_name) {
  // Every call starts from "one K slice": the barrier-free matrix-core kernels and the
  // 128x128 blocks in slices report more (iree_uk_amd_last_k_slices).
  uk_mfma::note_k_slices(1);
  if (rowmajor && rowmajor->epilogue) {
    if (kernel_mode != IREE_UK_AMD_KERNEL_MODE_GENERIC && p->K != 0) {
      int st = iree_uk_amd_hip_launch_mmt4d_mfma(p, rowmajor, stream, 0, kernel_name);
      if (st < 0) st = launch_epilogue_apart(p, rowmajor, stream, kernel_mode, kernel_name);
      if (st >= 0) return st;
    }
    *kernel_name = "mmt4d_generic";
    return iree_uk_amd_hip_launch_mmt4d_generic(p, rowmajor, stream);
  }
  // s8 x s4 -> s32 and s16 x s16 -> s32 have an MFMA kernel for some shapes
  // only; the launcher says "not served" (negative) for the rest.
  const uint32_t type = p->flags & IREE_UK_FLAG_MMT4D_TYPE_MASK;
  const bool maybe = type == IREE_UK_FLAG_MMT4D_TYPE_S8S4S32 || type == IREE_UK_FLAG_MMT4D_TYPE_S16S16S32;
  if (kernel_mode != IREE_UK_AMD_KERNEL_MODE_GENERIC &&
      (maybe || iree_uk_amd_hip_mmt4d_mfma_supported(p->M0, p->N0, p->K0, p->flags))) {
    const int forced = kernel_mode >= IREE_UK_AMD_KERNEL_MODE_MFMA_VARIANT
                           ? kernel_mode - IREE_UK_AMD_KERNEL_MODE_MFMA_VARIANT
                           : 0;
    int st = iree_uk_amd_hip_launch_mmt4d_mfma(p, rowmajor, stream, forced, kernel_name);
    // A negative status means "not served after all" (a negative stride, an
    // operand spanning 2 GiB or more, a zero-fill): the scalar kernel, which
    // indexes with 64 bits, computes the same result. When the tile shape is
    // one the info query advertises, count the call so that the cliff shows.
    if (st >= 0) return st;
    if (!maybe && kernel_mode == IREE_UK_AMD_KERNEL_MODE_AUTO && p->K != 0) ++g_declined;
  }
  if (kernel_mode == IREE_UK_AMD_KERNEL_MODE_AUTO) {
    // Tile rows under 16 bytes in shapes the matrix-core kernels decline:
    // regrouped along K first (mmt4d_mfma.hip).
    const int st = iree_uk_amd_hip_launch_mmt4d_retiled(p, rowmajor, stream, kernel_name);
    if (st >= 0) return st;
  }
  if (kernel_mode == IREE_UK_AMD_KERNEL_MODE_AUTO) {
    // s16 x s8 and s16 x u4 with enough rows and columns: the matrix-core s16
    // kernel on a right-hand side widened to s16 (mmt4d_mfma_s16.hip).
    const int st = iree_uk_amd_hip_launch_mmt4d_s16_widened(p, rowmajor, stream, kernel_name);
    if (st >= 0) return st;
  }
  if (kernel_mode != IREE_UK_AMD_KERNEL_MODE_GENERIC) {
    // The 16-bit integer LHS types: vector dot products from LDS where the
    // tile shape allows (not a matrix-core kernel, so the info query does not
    // advertise it and callers pass the fallback flag as for the CPU library's
    // generic tiles).
    const int st = iree_uk_amd_hip_launch_mmt4d_dot2(p, rowmajor, stream);
    if (st >= 0) {
      *kernel_name = "mmt4d_dot2";
      return st;
    }
  }
  *kernel_name = "mmt4d_generic";
  return iree_uk_amd_hip_launch_mmt4d_generic(p, rowmajor, stream);
}
