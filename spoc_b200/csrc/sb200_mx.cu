// sb200_mx.cu — the C ABI of the microscaled operators and the root-mean-square norm (include/sb200.h): argument checks, the choice of a
// kernel's form, launches.
#include <cuda.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include <algorithm>
#include <atomic>

#include "../../include/sb200.h"
#include "gemm_mx.cuh"
#include "gemm_mx_plan.hpp"
#include "internal.hpp"
#include "microscale.cuh"
#include "rmsnorm.cuh"

using namespace sb200;

namespace {

constexpr int kMaxDevices = 16;
constexpr int64_t kMaxDim = 0x7fffffffLL - 128;

#define CU_TRY(call)                                           \
  do {                                                         \
    cudaError_t e__ = (call);                                  \
    if (e__ != cudaSuccess) return set_cuda_error(e__, #call); \
  } while (0)

inline cudaStream_t as_stream(uint64_t s) { return reinterpret_cast<cudaStream_t>(static_cast<uintptr_t>(s)); }
template <class T>
T* as_ptr(uint64_t p) {
  return reinterpret_cast<T*>(static_cast<uintptr_t>(p));
}
bool on_16(uint64_t p, int64_t ld) { return (p & 15) == 0 && (ld & 3) == 0; }

bool known_format(int format) { return format == SB200_MX_FP8 || format == SB200_MX_FP4; }
int64_t chunks_of(int64_t K) { return (K + MX_CHUNK - 1) / MX_CHUNK; }
uint64_t code_bytes(int format, int64_t rows, int64_t K) {
  return static_cast<uint64_t>(rows) * chunks_of(K) * (format == SB200_MX_FP4 ? 64 : 128);
}
uint64_t scale_bytes(int64_t rows, int64_t K) { return static_cast<uint64_t>((rows + 127) / 128) * chunks_of(K) * MX_TILE_BYTES; }

int check_shape(int64_t rows, int64_t K, const char* what) {
  if (rows < 0 || K < 0) return set_error(SB200_ERR_INVALID_VALUE, "%s: negative dimension (%lld x %lld)", what, (long long)rows, (long long)K);
  if (rows > kMaxDim || K > kMaxDim) return set_error(SB200_ERR_TOO_LARGE, "%s: dimension beyond 2^31 (%lld x %lld)", what, (long long)rows, (long long)K);
  // tiles of scales are counted in 32 bits
  if (static_cast<uint64_t>((rows + 127) / 128) * chunks_of(K) > 0x7fffffffull)
    return set_error(SB200_ERR_TOO_LARGE, "%s: %lld x %lld has more than 2^31 - 1 tiles of scales", what, (long long)rows, (long long)K);
  return SB200_OK;
}
int check_format(int format) {
  return known_format(format) ? SB200_OK : set_error(SB200_ERR_INVALID_VALUE, "unknown microscaled format %d", format);
}
// A microscaled operand that is there: both buffers, where TMA can read them.
int check_mx(uint64_t codes, uint64_t scales, const char* what) {
  if (!codes || !scales) return set_error(SB200_ERR_INVALID_VALUE, "%s: null codes or scales", what);
  if ((codes | scales) & 31) return set_error(SB200_ERR_ALIGNMENT, "%s: codes and scales start on 32 bytes", what);
  return SB200_OK;
}
// A float32 matrix that is there.
int check_matrix(uint64_t p, int64_t rows, int64_t cols, int64_t ld, const char* what) {
  if (!p) return set_error(SB200_ERR_INVALID_VALUE, "%s: null device pointer", what);
  if (p & 3) return set_error(SB200_ERR_ALIGNMENT, "%s: float32 matrices must be 4-byte aligned", what);
  if (ld < cols) return set_error(SB200_ERR_INVALID_VALUE, "%s: leading dimension %lld smaller than the row length %lld", what, (long long)ld, (long long)cols);
  if (ld > INT64_MAX / 8 / (rows > 0 ? rows : 1)) return set_error(SB200_ERR_TOO_LARGE, "%s: extent beyond 64 bits", what);
  return SB200_OK;
}
// A result may be an operand itself, row on row: with other row lengths a row would be written before another block has read it.
int check_in_place(uint64_t result, int64_t ldr, uint64_t operand, int64_t ldo, int64_t rows, const char* what) {
  if (!result || result != operand || ldr == ldo || rows < 2) return SB200_OK;
  return set_error(SB200_ERR_INVALID_VALUE, "%s: in place with another leading dimension (%lld, operand %lld)", what, (long long)ldr, (long long)ldo);
}
// What lies in a buffer of the library's ends there.
int mx_extent(int dev, int format, int64_t rows, int64_t K, uint64_t codes, uint64_t scales, const char* what) {
  if (int rc = operator_extent(dev, codes, code_bytes(format, rows, K), what)) return rc;
  return operator_extent(dev, scales, scale_bytes(rows, K), what);
}
int matrix_extent(int dev, uint64_t p, int64_t rows, int64_t cols, int64_t ld, const char* what) {
  return p && rows && cols ? operator_extent(dev, p, (static_cast<uint64_t>(rows - 1) * ld + cols) * 4, what) : SB200_OK;
}

// Quantising by rows, by columns and the way back share one division of L1 (half of it shared memory, of which columns need 70 KB for four blocks an SM):
// a kernel that wants another one waits until the SM is empty.  Left to the driver, four quantisations and two products of a layer's gradients
// (4096 x 4096 x 2048) take 118 us instead of 107, and 2047 x 1021 to 4 bits and back 8.4 instead of 6.2.
constexpr int kShared = 50;

// Blocks for `work` units, `per_block` each, at most `cap`.
unsigned grid_for(int64_t work, int64_t per_block, int64_t cap) {
  const int64_t blocks = (work + per_block - 1) / per_block;
  return static_cast<unsigned>(std::max<int64_t>(1, std::min(blocks, cap)));
}

// ------------------------------------------------------------------ norm
template <int FORMAT, bool VEC>
int launch_rmsnorm(int sm_count, cudaStream_t st, const RmsNorm& p) {
  const int64_t rows = FORMAT ? (p.rows + 127) / 128 * 128 : p.rows;
  constexpr int ACCESS = VEC ? ACCESS_VECTOR : FORMAT ? ACCESS_SINGLE : ACCESS_LANES;
  // The row in the registers of a warp or a block, and as many blocks an SM as leave a thread 48 registers (64 with eight float4).  Few rows, which
  // do not fill the chip, take wide blocks: 1 x 4096 to 8 bits 3.66 -> 2.93 us, 444 x 4096 9.3 -> 7.5, 444 x 1024 6.1 -> 3.0; 512 x 4096 is even,
  // 512 x 8192 goes 15.6 -> 17.8 and 8192 x 4096 70.8 -> 83.4.
#define SB200_NORM(THREADS, VECS, BLOCKS)                                                                                            \
  CU_TRY(launch_pdl(rmsnorm_kernel<FORMAT, THREADS, VECS, ACCESS, BLOCKS>, dim3(grid_for(rows, THREADS == 32 ? 4 : 1, 0x7fffffff)),  \
                    dim3(THREADS == 32 ? 128 : THREADS), 0, st, 1, p))
  const int cols = p.cols;
  const bool few = p.rows <= 3ll * sm_count;
  if (cols <= 128) SB200_NORM(32, 1, 12);
  else if (cols <= 256) SB200_NORM(32, 2, 12);
  else if (cols <= 512) SB200_NORM(32, 4, 10);
  else if (few && cols <= 1024) SB200_NORM(256, 1, 6);
  else if (cols <= 1024) SB200_NORM(32, 8, 8);
  else if (few && cols <= 2048) SB200_NORM(256, 2, 5);
  else if (cols <= 2048) SB200_NORM(128, 4, 10);
  else if (few && cols <= 4096) SB200_NORM(512, 2, 3);
  else if (cols <= 4096) SB200_NORM(256, 4, 5);
  else if (few && cols <= 8192) SB200_NORM(1024, 2, 1);
  else if (cols <= 8192) SB200_NORM(512, 4, 2);
  else if (cols <= 16384) SB200_NORM(512, 8, 2);
  else if (cols <= 32768) SB200_NORM(1024, 8, 1);
  else SB200_NORM(1024, 0, 1);
#undef SB200_NORM
  return operator_launched("rmsnorm_kernel");
}

int64_t dweight_parts(int64_t rows) { return std::min<int64_t>(rows, SB200_RMSNORM_MAX_PARTS); }

// As many blocks, or clusters, as are resident at once.
template <int TG, int G, int VECS, int STAGES, int ACCESS, bool WIDE = false>
int launch_backward_ring(const OperatorDevice& d, cudaStream_t st, RmsNormBackward p, unsigned* parts) {
  using Ring = BackwardRing<TG, G, VECS, STAGES, ACCESS>;
  auto kernel = rmsnorm_backward_ring_kernel<TG, G, VECS, STAGES, ACCESS, WIDE>;
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[d.index].load()) {
    CU_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Ring::kBytes));
    ready[d.index].store(true);
  }
  p.blocks = WIDE ? (p.cols + Ring::kCols - 1) / Ring::kCols : 1;
  p.slice = WIDE ? ((p.cols + p.blocks - 1) / p.blocks + 3) / 4 * 4 : p.cols;  // slices of rows on 16 bytes start there, too
  const int64_t units = std::max<int64_t>(1, WIDE ? cluster_capacity(p.blocks, d.sm_count) : d.sm_count);
  *parts = static_cast<unsigned>(std::min(units, dweight_parts(p.rows)));
  operator_waits(d.index);
  CU_TRY(launch_pdl(kernel, dim3(*parts * p.blocks), dim3(TG * G), Ring::kBytes, st, p.blocks, p));
  return operator_launched("rmsnorm_backward_ring_kernel");
}
template <int ACCESS>
int launch_backward(const OperatorDevice& d, cudaStream_t st, const RmsNormBackward& p, unsigned* parts) {
  const int cols = p.cols;
  // A block an SM with a ring of 196 KB.  Groups of the fewest warps that hold a row in four float4 a thread: with twice the threads and two float4
  // 4096 x 16384 took 178 us instead of 158 (and 255 without a cluster), 8192 x 8191 183 instead of 160.
  if (cols <= 128) return launch_backward_ring<32, 32, 1, 4, ACCESS>(d, st, p, parts);
  if (cols <= 256) return launch_backward_ring<32, 16, 2, 4, ACCESS>(d, st, p, parts);
  if (cols <= 512) return launch_backward_ring<32, 8, 4, 4, ACCESS>(d, st, p, parts);
  if (cols <= 1024) return launch_backward_ring<64, 4, 4, 4, ACCESS>(d, st, p, parts);
  if (cols <= 2048) return launch_backward_ring<128, 4, 4, 2, ACCESS>(d, st, p, parts);
  if (cols <= 4096) return launch_backward_ring<256, 2, 4, 2, ACCESS>(d, st, p, parts);
  if (cols <= 8192) return launch_backward_ring<512, 1, 4, 2, ACCESS>(d, st, p, parts);
  if (cols <= 8192 * RMS_MAX_CLUSTER) return launch_backward_ring<512, 1, 4, 2, ACCESS, true>(d, st, p, parts);
  *parts = static_cast<unsigned>(std::min<int64_t>(dweight_parts(p.rows), static_cast<int64_t>(d.sm_count) * 2));
  CU_TRY(launch_pdl(rmsnorm_backward_kernel<ACCESS>, dim3(*parts), dim3(1024), 0, st, 1, p));
  return operator_launched("rmsnorm_backward_kernel");
}
int launch_rmsnorm_backward(const OperatorDevice& d, cudaStream_t st, const RmsNormBackward& p, bool vec) {
  unsigned parts = 0;
  const int rc = vec ? launch_backward<ACCESS_VECTOR>(d, st, p, &parts) : launch_backward<ACCESS_LANES>(d, st, p, &parts);
  if (rc || !p.dweight) return rc;
  CU_TRY(launch_pdl(rmsnorm_dweight_kernel, dim3(grid_for(p.cols, 32, 1 << 20)), dim3(256), 0, st, 1, static_cast<const float*>(p.workspace),
                    static_cast<int>(parts), p.dweight, static_cast<long long>(p.cols)));
  return operator_launched("rmsnorm_dweight_kernel");
}

// --------------------------------------------------------------- product
template <bool FP4, int CTAS, int GROUPS, bool IN_CLUSTER = false>
int launch_mx(const OperatorDevice& d, cudaStream_t st, const CUtensorMap (&maps)[6], const MxGemm& p) {
  auto kernel = gemm_mx_kernel<FP4, CTAS, GROUPS, IN_CLUSTER>;
  constexpr int kMost = 1024 + MXG_CTRL_BYTES + MXG_RING_BYTES;
  // Blocks that wait for one another hold tensor memory while they do.  If two such blocks fitted an SM, the clusters of two launches on different
  // streams could each have allocated on one SM and wait for the other on the next, for good: each takes more than half of the shared memory.
  constexpr int kAlone = CTAS == 2 || IN_CLUSTER ? 114 * 1024 : 0;
  const int smem = std::max(kAlone, 1024 + MXG_CTRL_BYTES + std::max(p.stages * p.stage_bytes, IN_CLUSTER ? p.bt * 512 : 0));
  static std::atomic<bool> ready[kMaxDevices];
  if (!ready[d.index].load()) {
    CU_TRY(cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost));
    ready[d.index].store(true);
  }
  const int tiles = p.tiles_f * p.tiles_t, units = d.sm_count / CTAS;
  const int grid = p.splits > 1 ? tiles * p.splits : CTAS * std::min(tiles, units);
  operator_waits(d.index);
  CU_TRY(launch_pdl(kernel, dim3(static_cast<unsigned>(grid)), dim3(MXG_THREADS), smem, st, CTAS * p.splits, maps[0], maps[1], maps[2], maps[3], maps[4], maps[5], p));
  return operator_launched("gemm_mx_kernel");
}

int run_gemm_mx(const OperatorDevice& d, cudaStream_t st, int format_a, int format_b, int64_t K, uint64_t a_codes, uint64_t a_scales, uint64_t b_codes,
                uint64_t b_scales, MxGemm p) {
  const bool fp4 = format_a == SB200_MX_FP4 && format_b == SB200_MX_FP4;
  const MxPlan s = plan_gemm_mx(fp4, p.M, p.N, K, d.sm_count);
  if (s.tiles > INT_MAX / 16) return set_error(SB200_ERR_TOO_LARGE, "gemm_mx: %lld tiles", (long long)s.tiles);
  p.chunks = s.chunks;
  p.num_k_blocks = s.num_k_blocks;
  p.bt = s.bt;
  p.tiles_f = static_cast<int>((p.N + 128ll * s.ctas - 1) / (128 * s.ctas));
  p.tiles_t = static_cast<int>((p.M + static_cast<int64_t>(s.bt) - 1) / s.bt);
  p.splits = s.splits;
  p.split_k_blocks = s.split_k_blocks;
  p.stages = s.stages;
  p.stage_bytes = s.stage_bytes;
  p.slots = s.slots;
  p.tmem_cols = s.tmem_cols;
  p.acc1 = s.acc1;
  // spread: 4-bit codes that TMA spreads to a byte a value; a barrier counts the bytes that it reads
  const bool spread_w = !fp4 && format_b == SB200_MX_FP4, spread_x = !fp4 && format_a == SB200_MX_FP4;
  p.w_row_bytes = spread_w ? 64 : 128;
  p.x_row_bytes = spread_x ? 64 : 128;
  p.idesc = umma_idesc_mx(128u * s.ctas, static_cast<uint32_t>(s.bt), fp4 ? 1u : format_b == SB200_MX_FP4 ? 5u : 0u,
                          fp4 ? 1u : format_a == SB200_MX_FP4 ? 5u : 0u);
  p.status = d.status;
  CUtensorMap maps[6];
  auto codes_map = [&](CUtensorMap* map, uint64_t codes, int format, int64_t rows, bool spread, int box_rows) {
    const uint64_t row_bytes = static_cast<uint64_t>(p.chunks) * (format == SB200_MX_FP4 ? 64 : 128);
    return encode_tensor_map_2d(map, spread ? CU_TENSOR_MAP_DATA_TYPE_16U4_ALIGN16B : CU_TENSOR_MAP_DATA_TYPE_UINT8, as_ptr<void>(codes),
                                spread ? row_bytes * 2 : row_bytes, static_cast<uint64_t>(rows), row_bytes, 128, static_cast<uint32_t>(box_rows),
                                CU_TENSOR_MAP_SWIZZLE_128B);
  };
  auto scales_map = [&](CUtensorMap* map, uint64_t scales, int64_t rows) {
    return encode_tensor_map_2d(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, as_ptr<void>(scales), MX_TILE_BYTES / 4,
                                static_cast<uint64_t>((rows + 127) / 128) * p.chunks, MX_TILE_BYTES, MX_TILE_BYTES / 4,
                                fp4 ? 2 : 1, CU_TENSOR_MAP_SWIZZLE_NONE);
  };
  const int part_t = s.bt / s.ctas;
  const int w_tail = p.N % 128 ? p.N % 128 : 128, x_tail = p.M % part_t ? p.M % part_t : part_t;
  p.w_tail = w_tail;
  p.x_tail = x_tail;
  int rc;
  if ((rc = codes_map(&maps[0], b_codes, format_b, p.N, spread_w, 128)) || (rc = codes_map(&maps[1], a_codes, format_a, p.M, spread_x, part_t)) ||
      (w_tail < 128 && (rc = codes_map(&maps[2], b_codes, format_b, p.N, spread_w, w_tail))) ||
      (x_tail < part_t && (rc = codes_map(&maps[3], a_codes, format_a, p.M, spread_x, x_tail))) || (rc = scales_map(&maps[4], b_scales, p.N)) ||
      (rc = scales_map(&maps[5], a_scales, p.M)))
    return rc;
  if (w_tail == 128) maps[2] = maps[0];
  if (x_tail == part_t) maps[3] = maps[1];
  if (p.splits > 1) return fp4 ? launch_mx<true, 1, 1, true>(d, st, maps, p) : launch_mx<false, 1, 1, true>(d, st, maps, p);
  if (s.ctas == 1) return fp4 ? launch_mx<true, 1, 1>(d, st, maps, p) : launch_mx<false, 1, 1>(d, st, maps, p);
  if (s.groups == 1) return fp4 ? launch_mx<true, 2, 1>(d, st, maps, p) : launch_mx<false, 2, 1>(d, st, maps, p);
  return fp4 ? launch_mx<true, 2, 2>(d, st, maps, p) : launch_mx<false, 2, 2>(d, st, maps, p);
}

}  // namespace

extern "C" {

int sb200_mx_bytes(int format, int64_t rows, int64_t K, uint64_t* codes, uint64_t* scales) {
  if (int rc = check_format(format)) return rc;
  if (int rc = check_shape(rows, K, "mx_bytes")) return rc;
  if (!codes || !scales) return set_error(SB200_ERR_INVALID_VALUE, "mx_bytes: null result");
  *codes = code_bytes(format, rows, K);
  *scales = scale_bytes(rows, K);
  return SB200_OK;
}

int sb200_mx_quantize(int dev, uint64_t stream, int format, int64_t rows, int64_t K, uint64_t src, int64_t ld, int transposed, uint64_t codes,
                      uint64_t scales) {
  if (int rc = check_format(format)) return rc;
  if (int rc = check_shape(rows, K, "mx_quantize")) return rc;
  const int64_t src_rows = transposed ? K : rows, src_cols = transposed ? rows : K;
  const bool empty = rows == 0 || K == 0;
  if (!empty) {
    if (int rc = check_matrix(src, src_rows, src_cols, ld, "mx_quantize source")) return rc;
    if (int rc = check_mx(codes, scales, "mx_quantize result")) return rc;
  }
  OperatorDevice d;
  if (int rc = operator_device(dev, &d)) return rc;
  if (empty) return SB200_OK;
  if (int rc = matrix_extent(dev, src, src_rows, src_cols, ld, "mx_quantize source")) return rc;
  if (int rc = mx_extent(dev, format, rows, K, codes, scales, "mx_quantize result")) return rc;
  const MxQuantize q = {as_ptr<const float>(src), ld, rows, K, chunks_of(K), as_ptr<uint8_t>(codes), as_ptr<uint8_t>(scales)};
  const cudaStream_t st = as_stream(stream);
  const bool fp4 = format == SB200_MX_FP4;
  if (transposed) {
    const dim3 grid(grid_for((rows + 127) / 128 * (128 / MX_COLUMNS) * ((q.chunks + 1) / 2), 1, 0x7fffffff)), block(MX_COLUMNS_THREADS);
    CU_TRY(fp4 ? launch_pdl_sharing(kShared, mx_quantize_columns_kernel<true>, grid, block, 0, st, 1, q)
               : launch_pdl_sharing(kShared, mx_quantize_columns_kernel<false>, grid, block, 0, st, 1, q));
    return operator_launched("mx_quantize_columns_kernel");
  }
  const long long warps = (rows + 127) / 128 * 128 * ((q.chunks + MX_AHEAD - 1) / MX_AHEAD);
  const dim3 grid(grid_for(warps, MX_QUANTIZE_THREADS / 32, 0x7fffffff)), block(MX_QUANTIZE_THREADS);
  const bool vec = on_16(src, ld) && K % 4 == 0;
  CU_TRY(fp4 ? (vec ? launch_pdl_sharing(kShared, mx_quantize_rows_kernel<true, true>, grid, block, 0, st, 1, q, warps)
                    : launch_pdl_sharing(kShared, mx_quantize_rows_kernel<true, false>, grid, block, 0, st, 1, q, warps))
             : (vec ? launch_pdl_sharing(kShared, mx_quantize_rows_kernel<false, true>, grid, block, 0, st, 1, q, warps)
                    : launch_pdl_sharing(kShared, mx_quantize_rows_kernel<false, false>, grid, block, 0, st, 1, q, warps)));
  return operator_launched("mx_quantize_rows_kernel");
}

int sb200_mx_dequantize(int dev, uint64_t stream, int format, int64_t rows, int64_t K, uint64_t codes, uint64_t scales, uint64_t dst, int64_t ld) {
  if (int rc = check_format(format)) return rc;
  if (int rc = check_shape(rows, K, "mx_dequantize")) return rc;
  const bool empty = rows == 0 || K == 0;
  if (!empty) {
    if (int rc = check_mx(codes, scales, "mx_dequantize operand")) return rc;
    if (int rc = check_matrix(dst, rows, K, ld, "mx_dequantize result")) return rc;
  }
  OperatorDevice d;
  if (int rc = operator_device(dev, &d)) return rc;
  if (empty) return SB200_OK;
  if (int rc = mx_extent(dev, format, rows, K, codes, scales, "mx_dequantize operand")) return rc;
  if (int rc = matrix_extent(dev, dst, rows, K, ld, "mx_dequantize result")) return rc;
  const MxDequantize q = {as_ptr<const uint8_t>(codes), as_ptr<const uint8_t>(scales), as_ptr<float>(dst), ld, rows, K, chunks_of(K)};
  const cudaStream_t st = as_stream(stream);
  const bool fp4 = format == SB200_MX_FP4, vec = on_16(dst, ld) && K % 4 == 0;
  const long long warps = rows * ((q.chunks + MX_AHEAD - 1) / MX_AHEAD);
  const dim3 grid(grid_for(warps, MX_QUANTIZE_THREADS / 32, 0x7fffffff)), block(MX_QUANTIZE_THREADS);
  CU_TRY(fp4 ? (vec ? launch_pdl_sharing(kShared, mx_dequantize_kernel<true, true>, grid, block, 0, st, 1, q, warps)
                    : launch_pdl_sharing(kShared, mx_dequantize_kernel<true, false>, grid, block, 0, st, 1, q, warps))
             : (vec ? launch_pdl_sharing(kShared, mx_dequantize_kernel<false, true>, grid, block, 0, st, 1, q, warps)
                    : launch_pdl_sharing(kShared, mx_dequantize_kernel<false, false>, grid, block, 0, st, 1, q, warps)));
  return operator_launched("mx_dequantize_kernel");
}

int sb200_gemm_mx(int dev, uint64_t stream, int format_a, int format_b, int64_t M, int64_t N, int64_t K, uint64_t a_codes, uint64_t a_scales,
                  uint64_t b_codes, uint64_t b_scales, uint64_t D, int64_t ldd, float alpha, uint64_t C, int64_t ldc, float beta, uint64_t bias, int act) {
  if (int rc = check_format(format_a)) return rc;
  if (int rc = check_format(format_b)) return rc;
  if (int rc = check_shape(M, K, "gemm_mx")) return rc;
  if (int rc = check_shape(N, K, "gemm_mx")) return rc;
  if (act != SB200_ACT_NONE && act != SB200_ACT_RELU) return set_error(SB200_ERR_INVALID_VALUE, "unknown activation %d", act);
  const bool empty = M == 0 || N == 0;
  if (!empty) {
    if (K > 0) {
      if (int rc = check_mx(a_codes, a_scales, "gemm_mx operand A")) return rc;
      if (int rc = check_mx(b_codes, b_scales, "gemm_mx operand B")) return rc;
    }
    if (int rc = check_matrix(D, M, N, ldd, "gemm_mx result D")) return rc;
    if (C)
      if (int rc = check_matrix(C, M, N, ldc, "gemm_mx operand C")) return rc;
    if (int rc = check_in_place(D, ldd, C, ldc, M, "gemm_mx")) return rc;
    if (bias)
      if (int rc = check_matrix(bias, 1, N, N, "gemm_mx bias")) return rc;
  }
  OperatorDevice d;
  if (int rc = operator_device(dev, &d)) return rc;
  if (empty) return SB200_OK;
  if (K > 0) {
    if (int rc = mx_extent(dev, format_a, M, K, a_codes, a_scales, "gemm_mx operand A")) return rc;
    if (int rc = mx_extent(dev, format_b, N, K, b_codes, b_scales, "gemm_mx operand B")) return rc;
  }
  if (int rc = matrix_extent(dev, D, M, N, ldd, "gemm_mx result D")) return rc;
  if (int rc = matrix_extent(dev, C, M, N, ldc, "gemm_mx operand C")) return rc;
  if (int rc = matrix_extent(dev, bias, 1, N, N, "gemm_mx bias")) return rc;
  MxGemm p;
  memset(&p, 0, sizeof p);
  p.D = as_ptr<float>(D);
  p.C = as_ptr<const float>(C);
  p.bias = as_ptr<const float>(bias);
  p.ldd = ldd;
  p.ldc = ldc;
  p.M = static_cast<int>(M);
  p.N = static_cast<int>(N);
  p.alpha = alpha;
  p.beta = beta;
  p.act = act;
  if (K == 0) {
    CU_TRY(launch_pdl(gemm_mx_empty_kernel, dim3(grid_for(M * N, 256, static_cast<int64_t>(d.sm_count) * 16)), dim3(256), 0, as_stream(stream), 1, p));
    return operator_launched("gemm_mx_empty_kernel");
  }
  return run_gemm_mx(d, as_stream(stream), format_a, format_b, K, a_codes, a_scales, b_codes, b_scales, p);
}

int sb200_rmsnorm_f32(int dev, uint64_t stream, int64_t rows, int64_t cols, uint64_t x, int64_t ldx, uint64_t residual, int64_t ldr, uint64_t weight,
                      double eps, uint64_t sum, int64_t lds, uint64_t y, int64_t ldy, int format, uint64_t codes, uint64_t scales) {
  if (format != 0)
    if (int rc = check_format(format)) return rc;
  if (int rc = check_shape(rows, cols, "rmsnorm")) return rc;
  if (!(eps >= 0.0)) return set_error(SB200_ERR_INVALID_VALUE, "rmsnorm: eps must not be negative");
  if (!sum && !y && format == 0) return set_error(SB200_ERR_INVALID_VALUE, "rmsnorm: no result asked for");
  const bool empty = rows == 0 || cols == 0;
  if (!empty) {
    if (int rc = check_matrix(x, rows, cols, ldx, "rmsnorm x")) return rc;
    if (int rc = check_matrix(weight, 1, cols, cols, "rmsnorm weight")) return rc;
    if (residual)
      if (int rc = check_matrix(residual, rows, cols, ldr, "rmsnorm residual")) return rc;
    if (sum)
      if (int rc = check_matrix(sum, rows, cols, lds, "rmsnorm sum")) return rc;
    if (y)
      if (int rc = check_matrix(y, rows, cols, ldy, "rmsnorm y")) return rc;
    if (format)
      if (int rc = check_mx(codes, scales, "rmsnorm result")) return rc;
    if (sum && sum == y) return set_error(SB200_ERR_INVALID_VALUE, "rmsnorm: sum and y are the same matrix");
    const struct { uint64_t p; int64_t ld; } results[] = {{sum, lds}, {y, ldy}}, operands[] = {{x, ldx}, {residual, ldr}};
    for (const auto& r : results)
      for (const auto& o : operands)
        if (int rc = check_in_place(r.p, r.ld, o.p, o.ld, rows, "rmsnorm")) return rc;
  }
  OperatorDevice d;
  if (int rc = operator_device(dev, &d)) return rc;
  if (empty) return SB200_OK;
  if (int rc = matrix_extent(dev, x, rows, cols, ldx, "rmsnorm x")) return rc;
  if (int rc = matrix_extent(dev, weight, 1, cols, cols, "rmsnorm weight")) return rc;
  if (int rc = matrix_extent(dev, residual, rows, cols, ldr, "rmsnorm residual")) return rc;
  if (int rc = matrix_extent(dev, sum, rows, cols, lds, "rmsnorm sum")) return rc;
  if (int rc = matrix_extent(dev, y, rows, cols, ldy, "rmsnorm y")) return rc;
  if (format)
    if (int rc = mx_extent(dev, format, rows, cols, codes, scales, "rmsnorm result")) return rc;
  RmsNorm p;
  memset(&p, 0, sizeof p);
  p.x = as_ptr<const float>(x);
  p.residual = as_ptr<const float>(residual);
  p.weight = as_ptr<const float>(weight);
  p.h = as_ptr<float>(sum);
  p.y = as_ptr<float>(y);
  p.ldx = ldx;
  p.ldr = ldr;
  p.ldh = lds;
  p.ldy = ldy;
  p.rows = rows;
  p.cols = static_cast<int>(cols);
  p.chunks = static_cast<int>(chunks_of(cols));
  p.inv_cols = 1.0 / static_cast<double>(cols);
  p.eps = eps;
  if (format) {
    p.codes = as_ptr<uint8_t>(codes);
    p.scales = as_ptr<uint8_t>(scales);
  }
  // 128-bit accesses where every row of every matrix starts on 16 bytes and has whole vectors
  const bool vec = cols % 4 == 0 && on_16(x, ldx) && on_16(weight, 0) && (!residual || on_16(residual, ldr)) && (!sum || on_16(sum, lds)) && (!y || on_16(y, ldy));
  const cudaStream_t st = as_stream(stream);
  if (format == SB200_MX_FP8) return vec ? launch_rmsnorm<8, true>(d.sm_count, st, p) : launch_rmsnorm<8, false>(d.sm_count, st, p);
  if (format == SB200_MX_FP4) return vec ? launch_rmsnorm<4, true>(d.sm_count, st, p) : launch_rmsnorm<4, false>(d.sm_count, st, p);
  return vec ? launch_rmsnorm<0, true>(d.sm_count, st, p) : launch_rmsnorm<0, false>(d.sm_count, st, p);
}

int sb200_rmsnorm_workspace_bytes(int64_t rows, int64_t cols, uint64_t* bytes) {
  if (int rc = check_shape(rows, cols, "rmsnorm_workspace_bytes")) return rc;
  if (!bytes) return set_error(SB200_ERR_INVALID_VALUE, "rmsnorm_workspace_bytes: null result");
  *bytes = static_cast<uint64_t>(dweight_parts(rows)) * cols * 4;
  return SB200_OK;
}

int sb200_rmsnorm_backward_f32(int dev, uint64_t stream, int64_t rows, int64_t cols, uint64_t sum, int64_t lds, uint64_t weight, double eps,
                               uint64_t dy, int64_t lddy, uint64_t dsum, int64_t ldds, uint64_t dx, int64_t lddx, uint64_t dweight,
                               uint64_t workspace, uint64_t workspace_bytes) {
  if (int rc = check_shape(rows, cols, "rmsnorm_backward")) return rc;
  if (!(eps >= 0.0)) return set_error(SB200_ERR_INVALID_VALUE, "rmsnorm_backward: eps must not be negative");
  if (!dx && !dweight) return set_error(SB200_ERR_INVALID_VALUE, "rmsnorm_backward: no result asked for");
  const uint64_t need = static_cast<uint64_t>(dweight_parts(rows)) * cols * 4;
  if (cols > 0 && dweight)
    if (int rc = check_matrix(dweight, 1, cols, cols, "rmsnorm_backward dweight")) return rc;
  if (cols > 0 && rows > 0) {
    if (int rc = check_matrix(sum, rows, cols, lds, "rmsnorm_backward sum")) return rc;
    if (int rc = check_matrix(weight, 1, cols, cols, "rmsnorm_backward weight")) return rc;
    if (int rc = check_matrix(dy, rows, cols, lddy, "rmsnorm_backward dy")) return rc;
    if (dsum)
      if (int rc = check_matrix(dsum, rows, cols, ldds, "rmsnorm_backward dsum")) return rc;
    if (dx)
      if (int rc = check_matrix(dx, rows, cols, lddx, "rmsnorm_backward dx")) return rc;
    if (dweight && (!workspace || workspace_bytes < need))
      return set_error(SB200_ERR_INVALID_VALUE, "rmsnorm_backward: dweight needs a workspace of %llu bytes", static_cast<unsigned long long>(need));
    if (dweight && (workspace & 3)) return set_error(SB200_ERR_ALIGNMENT, "rmsnorm_backward: the workspace must be 4-byte aligned");
    if (int rc = check_in_place(dx, lddx, sum, lds, rows, "rmsnorm_backward dx")) return rc;
    if (int rc = check_in_place(dx, lddx, dy, lddy, rows, "rmsnorm_backward dx")) return rc;
    if (int rc = check_in_place(dx, lddx, dsum, ldds, rows, "rmsnorm_backward dx")) return rc;
  }
  OperatorDevice d;
  if (int rc = operator_device(dev, &d)) return rc;
  if (cols == 0) return SB200_OK;
  if (int rc = matrix_extent(dev, dweight, 1, cols, cols, "rmsnorm_backward dweight")) return rc;
  const cudaStream_t st = as_stream(stream);
  if (rows == 0) {  // an empty sum
    if (dweight) CU_TRY(cudaMemsetAsync(as_ptr<void>(dweight), 0, static_cast<size_t>(cols) * 4, st));
    return SB200_OK;
  }
  if (int rc = matrix_extent(dev, sum, rows, cols, lds, "rmsnorm_backward sum")) return rc;
  if (int rc = matrix_extent(dev, weight, 1, cols, cols, "rmsnorm_backward weight")) return rc;
  if (int rc = matrix_extent(dev, dy, rows, cols, lddy, "rmsnorm_backward dy")) return rc;
  if (int rc = matrix_extent(dev, dsum, rows, cols, ldds, "rmsnorm_backward dsum")) return rc;
  if (int rc = matrix_extent(dev, dx, rows, cols, lddx, "rmsnorm_backward dx")) return rc;
  if (dweight)
    if (int rc = operator_extent(dev, workspace, need, "rmsnorm_backward workspace")) return rc;
  RmsNormBackward p;
  memset(&p, 0, sizeof p);
  p.h = as_ptr<const float>(sum);
  p.weight = as_ptr<const float>(weight);
  p.dy = as_ptr<const float>(dy);
  p.dsum = as_ptr<const float>(dsum);
  p.dx = as_ptr<float>(dx);
  p.dweight = as_ptr<float>(dweight);
  p.workspace = as_ptr<float>(workspace);
  p.ldh = lds;
  p.lddy = lddy;
  p.ldds = ldds;
  p.lddx = lddx;
  p.rows = rows;
  p.cols = static_cast<int>(cols);
  p.least = eps < RMS_LEAST ? static_cast<float>(RMS_LEAST) : eps < 1e38 ? 0.0f : INFINITY;  // an eps past float32: no row's sums hold
  p.inv_cols = 1.0 / static_cast<double>(cols);
  p.eps = eps;
  const bool vec = cols % 4 == 0 && on_16(sum, lds) && on_16(weight, 0) && on_16(dy, lddy) && (!dsum || on_16(dsum, ldds)) && (!dx || on_16(dx, lddx));
  p.status = d.status;
  return launch_rmsnorm_backward(d, st, p, vec);
}

}  // extern "C"
