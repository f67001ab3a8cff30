// microscale.cuh — microscaled matrices: values of 8 or 4 bits with a power-of-two scale for every 32 of a row.
//
// A matrix of rows x K is two buffers (include/sb200.h gives the layout a caller sees):
//   codes   row by row, K padded with zeros to Kp, a multiple of 128; e4m3 bytes, or two e2m1 values a byte, the first in the low half
//   scales  one exponent byte (2^(byte - 127), 255: NaN) for 32 values, in tiles of 128 rows x 4 scales of 512 bytes: the scale of row r and
//           block b is byte (r % 32) * 16 + (r % 128) / 32 * 4 + b % 4 of tile (r / 128, b / 4).  A tile is what the tensor core wants in four
//           columns of tensor memory, so that the product copies tiles as they are; past the last row and K it holds zeros.
// A block's scale is 2^max(floor(log2 m) - e, -127), m its largest magnitude and e the exponent of the type's largest value (8, 2).  A value is
// multiplied by the inverse, which is exact, and rounded once, to the nearest, ties to even; what would round past the type's largest
// value is held there (m can be up to 512 in e4m3's units, whose largest value is 448, and 8 in e2m1's, whose is 6).  A block with a NaN or an
// infinity gets the scale NaN, which turns all it meets into NaN (SB200_ACT_RELU behind a product makes 0 of that, as in the other GEMMs).
#pragma once
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx_sm100.cuh"

namespace sb200 {

constexpr int MX_CHUNK = 128;        // values of a row whose scales lie side by side in a tile; K is padded to a multiple of it
constexpr int MX_TILE_BYTES = 512;   // 128 rows x 4 scales

template <bool FP4>
struct MxFormat {
  static constexpr int kLargestExponent = FP4 ? 2 : 8;
  static constexpr int kChunkBytes = FP4 ? 64 : 128;  // codes of MX_CHUNK values
};

// Where the four scales of row r and chunk c lie.
__device__ __forceinline__ long long mx_scale_offset(long long row, long long chunk, long long chunks) {
  return ((row >> 7) * chunks + chunk) * MX_TILE_BYTES + (row & 31) * 16 + ((row & 127) >> 5) * 4;
}

// The scale byte of a block whose largest magnitude has these bits, and the factor that its values are multiplied by.
template <bool FP4>
__device__ __forceinline__ uint32_t mx_scale_of(uint32_t largest_bits) {
  const int e = static_cast<int>(largest_bits >> 23);
  return e == 255 ? 255u : static_cast<uint32_t>(max(e - MxFormat<FP4>::kLargestExponent, 0));
}
__device__ __forceinline__ float mx_factor(uint32_t scale) {
  return __uint_as_float(scale == 255u ? 0u : (254u - scale) << 23);  // of a NaN block 0: finite values become zeros
}
__device__ __forceinline__ float mx_scale_value(uint32_t scale) {
  return __uint_as_float(scale == 255u ? 0x7fc00000u : scale == 0u ? 0x00400000u : scale << 23);
}

// Two products with one instruction, rounded as two are.
__device__ __forceinline__ float2 multiply2(float2 a, float2 b) {
  float2 v;
  asm("{\n.reg .b64 a, b;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %5};\nmul.rn.f32x2 a, a, b;\nmov.b64 {%0, %1}, a;\n}"
      : "=f"(v.x), "=f"(v.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return v;
}
// Four values, scaled, to four codes: 32 bits of e4m3, or 16 of e2m1.
template <bool FP4>
__device__ __forceinline__ uint32_t mx_codes4(float4 v, float factor) {
  const float2 f = make_float2(factor, factor), a = multiply2(make_float2(v.x, v.y), f), b = multiply2(make_float2(v.z, v.w), f);
  if constexpr (FP4)
    return static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(a, __NV_E2M1, cudaRoundNearest)) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp4x2(b, __NV_E2M1, cudaRoundNearest)) << 8;
  else
    return static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(a, __NV_SATFINITE, __NV_E4M3)) |
           static_cast<uint32_t>(__nv_cvt_float2_to_fp8x2(b, __NV_SATFINITE, __NV_E4M3)) << 16;
}
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t largest_bits4(const float4& v) {  // bits of magnitudes are ordered as they are; NaN above all
  return max(max(abs_bits(v.x), abs_bits(v.y)), max(abs_bits(v.z), abs_bits(v.w)));
}

// A warp's chunk of a row: lane l has values 4l .. 4l + 3, eight lanes a block.
__device__ __forceinline__ uint32_t largest_of_block(const float4& v) {
  uint32_t m = largest_bits4(v);
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
  m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
  return max(m, __shfl_xor_sync(0xffffffffu, m, 4));
}
// codes: of the chunk; scales: its four; c: the lane's four codes, scale: of their block.
template <bool FP4>
__device__ __forceinline__ void mx_store_codes(uint32_t c, uint32_t scale, uint8_t* codes, uint8_t* scales, int lane) {
  if constexpr (FP4)
    reinterpret_cast<uint16_t*>(codes)[lane] = static_cast<uint16_t>(c);
  else
    reinterpret_cast<uint32_t*>(codes)[lane] = c;
  if ((lane & 7) == 0) scales[lane >> 3] = static_cast<uint8_t>(scale);
}

template <bool FP4>
__device__ __forceinline__ void mx_store_chunk(const float4& v, uint32_t scale, uint8_t* codes, uint8_t* scales, int lane) {
  mx_store_codes<FP4>(mx_codes4<FP4>(v, mx_factor(scale)), scale, codes, scales, lane);
}

// Four values of a row; what is past `cols` counts for zero.  A thread has columns col .. col + 3, col a multiple of four: as a vector (ACCESS_VECTOR: the
// row starts on 16 bytes and `cols` is a multiple of four) or one by one (ACCESS_SINGLE); or, where it does not matter which thread has which
// columns, a warp has its 128 columns with 32 of them side by side in the lanes (ACCESS_LANES), which takes a quarter of the lines a load.
enum { ACCESS_SINGLE = 0, ACCESS_VECTOR = 1, ACCESS_LANES = 2 };
template <int ACCESS>
__device__ __forceinline__ float4 load4(const float* row, int col, int cols) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if constexpr (ACCESS == ACCESS_VECTOR) {
    if (col < cols) v = *reinterpret_cast<const float4*>(row + col);
    return v;
  }
  if constexpr (ACCESS == ACCESS_LANES) {
    const int c = (col & ~127) + ((col & 127) >> 2);
    if (c < cols) v.x = row[c];
    if (c + 32 < cols) v.y = row[c + 32];
    if (c + 64 < cols) v.z = row[c + 64];
    if (c + 96 < cols) v.w = row[c + 96];
    return v;
  }
  if (col < cols) v.x = row[col];
  if (col + 1 < cols) v.y = row[col + 1];
  if (col + 2 < cols) v.z = row[col + 2];
  if (col + 3 < cols) v.w = row[col + 3];
  return v;
}
template <int ACCESS>
__device__ __forceinline__ void store4(float* row, int col, int cols, const float4& v) {
  if constexpr (ACCESS == ACCESS_VECTOR) {
    if (col < cols) *reinterpret_cast<float4*>(row + col) = v;
    return;
  }
  if constexpr (ACCESS == ACCESS_LANES) {
    const int c = (col & ~127) + ((col & 127) >> 2);
    if (c < cols) row[c] = v.x;
    if (c + 32 < cols) row[c + 32] = v.y;
    if (c + 64 < cols) row[c + 64] = v.z;
    if (c + 96 < cols) row[c + 96] = v.w;
    return;
  }
  if (col < cols) row[col] = v.x;
  if (col + 1 < cols) row[col + 1] = v.y;
  if (col + 2 < cols) row[col + 2] = v.z;
  if (col + 3 < cols) row[col + 3] = v.w;
}

struct MxQuantize {
  const float* src;
  long long ld, rows, K, chunks;  // chunks: Kp / 128
  uint8_t *codes, *scales;
};
constexpr int MX_QUANTIZE_THREADS = 256;

// A warp's work in the kernels over rows: up to MX_AHEAD chunks side by side in one row, so that one division finds them (32 bits wide where the
// number of warps allows it: 64 bits take 100 instructions, as much as all else).
constexpr int MX_AHEAD = 4;
struct MxWarp {
  long long row;
  int chunk;
};
__device__ __forceinline__ MxWarp mx_warp(long long chunks, long long warps) {
  const long long at = static_cast<long long>(blockIdx.x) * (MX_QUANTIZE_THREADS / 32) + (threadIdx.x >> 5), groups = (chunks + MX_AHEAD - 1) / MX_AHEAD;
  MxWarp w;
  if (warps < (1ll << 31)) {
    const unsigned int row = static_cast<unsigned int>(at) / static_cast<unsigned int>(groups);
    w.row = row;
    w.chunk = static_cast<int>(static_cast<unsigned int>(at) - row * static_cast<unsigned int>(groups)) * MX_AHEAD;
  } else {
    w.row = at / groups;
    w.chunk = static_cast<int>(at - w.row * groups) * MX_AHEAD;
  }
  return w;
}

// A warp's chunk through 512 bytes of shared memory: from 32 columns side by side in the lanes (ACCESS_LANES) to four in a row a lane, and back.
__device__ __forceinline__ float4 turned(const float4& v, float4* chunk, int lane) {
  float* const flat = reinterpret_cast<float*>(chunk);
  __syncwarp();  // what was there before is read
  flat[lane] = v.x;
  flat[lane + 32] = v.y;
  flat[lane + 64] = v.z;
  flat[lane + 96] = v.w;
  __syncwarp();
  return chunk[lane];
}
__device__ __forceinline__ float4 turned_back(const float4& v, float4* chunk, int lane) {
  const float* const flat = reinterpret_cast<const float*>(chunk);
  __syncwarp();
  chunk[lane] = v;
  __syncwarp();
  return make_float4(flat[lane], flat[lane + 32], flat[lane + 64], flat[lane + 96]);
}

// Rows of a matrix.  Bound by HBM: 4 bytes read, 1 (1/2) and 1/32 written a value; 8192 x 8192 to 8 bits 49 us, 6.8 TB/s.  A warp takes MX_AHEAD chunks of a
// row, whose loads are all under way before the first is rounded.
template <bool FP4, bool VEC>
__global__ void __launch_bounds__(MX_QUANTIZE_THREADS) mx_quantize_rows_kernel(const MxQuantize q, long long warps) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, cols = static_cast<int>(q.K), chunks = static_cast<int>(q.chunks);
  const MxWarp w = mx_warp(q.chunks, warps);
  if (w.row >= (q.rows + 127) / 128 * 128) return;
  uint8_t* scales = q.scales + mx_scale_offset(w.row, w.chunk, q.chunks);
  if (w.row >= q.rows) {
    if (lane < MX_AHEAD && w.chunk + lane < chunks) *reinterpret_cast<uint32_t*>(scales + lane * MX_TILE_BYTES) = 0u;
    return;
  }
  const float* src = q.src + w.row * q.ld;
  uint8_t* codes = q.codes + (w.row * q.chunks + w.chunk) * MxFormat<FP4>::kChunkBytes;
  float4 v[MX_AHEAD];
#pragma unroll
  for (int u = 0; u < MX_AHEAD; ++u) v[u] = load4<VEC>(src, min(w.chunk + u, chunks) * MX_CHUNK + 4 * lane, cols);
#pragma unroll
  for (int u = 0; u < MX_AHEAD; ++u) {
    if (w.chunk + u >= chunks) break;
    mx_store_chunk<FP4>(v[u], mx_scale_of<FP4>(largest_of_block(v[u])), codes + u * MxFormat<FP4>::kChunkBytes, scales + u * MX_TILE_BYTES, lane);
  }
}

// Columns of a matrix stored K x rows: a block takes 64 of its columns (rows of the result) and 256 of its rows, a thread 32 values below one
// another, which is a block with one scale.  The codes go through shared memory, so that a row's 256 (128) bytes are written together.
// Bound by HBM as the kernel over rows is: 8192 x 8192 to 8 bits 51 us, 6.6 TB/s.
constexpr int MX_COLUMNS = 64;
constexpr int MX_COLUMNS_THREADS = 8 * MX_COLUMNS;
template <bool FP4>
__global__ void __launch_bounds__(MX_COLUMNS_THREADS) mx_quantize_columns_kernel(const MxQuantize q) {
  constexpr int BYTES = FP4 ? 16 : 32;            // codes of a block
  constexpr int PITCH = 8 * BYTES + 16;           // 16 more: rows start on different banks
  __shared__ __align__(16) uint8_t codes[MX_COLUMNS * PITCH];
  __shared__ __align__(8) uint8_t scales[MX_COLUMNS][8];
  grid_launch_dependents();
  grid_dependency_wait();
  const int column = threadIdx.x % MX_COLUMNS, block = threadIdx.x / MX_COLUMNS;
  const unsigned int row_tiles = static_cast<unsigned int>((q.rows + 127) / 128) * (128 / MX_COLUMNS), kt = blockIdx.x / row_tiles;
  const long long row0 = static_cast<long long>(blockIdx.x - kt * row_tiles) * MX_COLUMNS;
  const long long k0 = kt * 256ll + block * 32;
  float v[32];
  const float* src = q.src + k0 * q.ld + row0 + column;
  if (row0 + column < q.rows && k0 + 32 <= q.K) {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = src[i * q.ld];
  } else {
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = row0 + column < q.rows && k0 + i < q.K ? src[i * q.ld] : 0.0f;
  }
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 32; ++i) m = max(m, abs_bits(v[i]));
  const uint32_t scale = mx_scale_of<FP4>(m);
  const float factor = mx_factor(scale);
  uint32_t words[BYTES / 4];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = mx_codes4<FP4>(make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]), factor);
    if constexpr (FP4)
      words[i / 2] = i % 2 ? words[i / 2] | c << 16 : c;
    else
      words[i] = c;
  }
  uint8_t* to = codes + column * PITCH + block * BYTES;
#pragma unroll
  for (int i = 0; i < BYTES / 16; ++i)
    reinterpret_cast<uint4*>(to)[i] = make_uint4(words[4 * i], words[4 * i + 1], words[4 * i + 2], words[4 * i + 3]);
  scales[column][block] = static_cast<uint8_t>(scale);
  __syncthreads();
  constexpr int QUADS = 8 * BYTES / 16;  // 16-byte pieces of a row
  const int chunks = static_cast<int>(min(2ll, q.chunks - kt * 2ll)), pieces = chunks * (QUADS / 2);
#pragma unroll
  for (int i = threadIdx.x; i < MX_COLUMNS * QUADS; i += MX_COLUMNS_THREADS) {
    const int r = i / QUADS, piece = i % QUADS;
    if (row0 + r < q.rows && piece < pieces)
      *reinterpret_cast<uint4*>(q.codes + ((row0 + r) * q.chunks + kt * 2ll) * MxFormat<FP4>::kChunkBytes + piece * 16) =
          *reinterpret_cast<const uint4*>(codes + r * PITCH + piece * 16);
  }
  if (threadIdx.x < 2 * MX_COLUMNS) {
    const int r = threadIdx.x >> 1, half = threadIdx.x & 1;
    if (half < chunks) {
      const uint32_t four = *reinterpret_cast<const uint32_t*>(&scales[r][half * 4]);
      *reinterpret_cast<uint32_t*>(q.scales + mx_scale_offset(row0 + r, kt * 2ll + half, q.chunks)) = row0 + r < q.rows ? four : 0u;
    }
  }
}

// Back to float32: exact, for a code has at most four significant bits.  Rows that do not start on 16 bytes are stored with 32 columns side by side
// in the lanes: four single stores a lane write a quarter of each sector they touch (8192 x 4095 from 4 bits 39 us, 30 so).
struct MxDequantize {
  const uint8_t *codes, *scales;
  float* dst;
  long long ld, rows, K, chunks;
};
template <bool FP4, bool VEC>
__global__ void __launch_bounds__(MX_QUANTIZE_THREADS) mx_dequantize_kernel(const MxDequantize q, long long warps) {
  grid_launch_dependents();
  grid_dependency_wait();
  __shared__ float4 turn_of[VEC ? 1 : MX_QUANTIZE_THREADS];
  const int lane = threadIdx.x & 31, chunks = static_cast<int>(q.chunks);
  const MxWarp w = mx_warp(q.chunks, warps);
  if (w.row >= q.rows) return;
  const uint8_t* codes = q.codes + (w.row * q.chunks + w.chunk) * MxFormat<FP4>::kChunkBytes;
  const uint8_t* scales = q.scales + mx_scale_offset(w.row, w.chunk, q.chunks) + lane / 8;
  uint32_t c[MX_AHEAD], scale[MX_AHEAD];
#pragma unroll
  for (int u = 0; u < MX_AHEAD; ++u) {
    const int at = min(u, chunks - 1 - w.chunk);
    if constexpr (FP4)
      c[u] = reinterpret_cast<const uint16_t*>(codes + at * MxFormat<FP4>::kChunkBytes)[lane];
    else
      c[u] = reinterpret_cast<const uint32_t*>(codes + at * MxFormat<FP4>::kChunkBytes)[lane];
    scale[u] = scales[at * MX_TILE_BYTES];
  }
#pragma unroll
  for (int u = 0; u < MX_AHEAD; ++u) {
    if (w.chunk + u >= chunks) break;
    __half2_raw a, b;
    if constexpr (FP4) {
      a = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(c[u] & 255u), __NV_E2M1);
      b = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(c[u] >> 8), __NV_E2M1);
    } else {
      a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c[u] & 65535u), __NV_E4M3);
      b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c[u] >> 16), __NV_E4M3);
    }
    const float2 lo = __half22float2(__half2(a)), hi = __half22float2(__half2(b));
    const float f = mx_scale_value(scale[u]);
    float4 v = make_float4(lo.x * f, lo.y * f, hi.x * f, hi.y * f);
    if constexpr (!VEC) v = turned_back(v, turn_of + (threadIdx.x & ~31), lane);
    store4<VEC ? ACCESS_VECTOR : ACCESS_LANES>(q.dst + w.row * q.ld, (w.chunk + u) * MX_CHUNK + 4 * lane, static_cast<int>(q.K), v);
  }
}

}  // namespace sb200
