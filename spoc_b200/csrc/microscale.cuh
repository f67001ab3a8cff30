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
// infinity gets the scale NaN, which turns all it meets into NaN.
#pragma once
#include <cuda_fp4.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "ptx_sm100.cuh"

namespace sb200 {

constexpr int MX_BLOCK = 32;         // values that share a scale
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

// Four values, scaled, to four codes: 32 bits of e4m3, or 16 of e2m1.
template <bool FP4>
__device__ __forceinline__ uint32_t mx_codes4(float4 v, float factor) {
  const float2 a = make_float2(v.x * factor, v.y * factor), b = make_float2(v.z * factor, v.w * factor);
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
// codes: of the chunk; scales: its four.
template <bool FP4>
__device__ __forceinline__ void mx_store_chunk(float4 v, uint32_t scale, uint8_t* codes, uint8_t* scales, int lane) {
  const uint32_t c = mx_codes4<FP4>(v, mx_factor(scale));
  if constexpr (FP4)
    reinterpret_cast<uint16_t*>(codes)[lane] = static_cast<uint16_t>(c);
  else
    reinterpret_cast<uint32_t*>(codes)[lane] = c;
  if ((lane & 7) == 0) scales[lane >> 3] = static_cast<uint8_t>(scale);
}

// Four values of a row from column `col` on; what is past `cols` counts for zero.  VEC: the row starts on 16 bytes and `cols` is a multiple of
// four (the single elements beside the vectors cost the norm 30 registers a thread).
template <bool VEC>
__device__ __forceinline__ float4 load4(const float* row, int col, int cols) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (VEC) {
    if (col < cols) v = *reinterpret_cast<const float4*>(row + col);
    return v;
  }
  if (col < cols) v.x = row[col];
  if (col + 1 < cols) v.y = row[col + 1];
  if (col + 2 < cols) v.z = row[col + 2];
  if (col + 3 < cols) v.w = row[col + 3];
  return v;
}
template <bool VEC>
__device__ __forceinline__ void store4(float* row, int col, int cols, const float4& v) {
  if (VEC) {
    if (col < cols) *reinterpret_cast<float4*>(row + col) = v;
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

// Rows of a matrix: a warp a chunk, MX_AHEAD chunks in flight.  Bound by HBM: 4 bytes read, 1 (1/2) and 1/32 written a value.
template <bool FP4, bool VEC>
__global__ void __launch_bounds__(MX_QUANTIZE_THREADS) mx_quantize_rows_kernel(const MxQuantize q) {
  constexpr int AHEAD = 4;
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (MX_QUANTIZE_THREADS / 32);
  const long long first = static_cast<long long>(blockIdx.x) * (MX_QUANTIZE_THREADS / 32) + (threadIdx.x >> 5);
  const long long all = (q.rows + 127) / 128 * 128 * q.chunks;
  for (long long at = first * AHEAD; at < all; at += warps * AHEAD) {
    float4 v[AHEAD];
    long long row[AHEAD], chunk[AHEAD];
    row[0] = at / q.chunks;
    chunk[0] = at - row[0] * q.chunks;
#pragma unroll
    for (int u = 1; u < AHEAD; ++u) {
      const bool next = chunk[u - 1] + 1 == q.chunks;
      row[u] = row[u - 1] + (next ? 1 : 0);
      chunk[u] = next ? 0 : chunk[u - 1] + 1;
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
      v[u] = row[u] < q.rows ? load4<VEC>(q.src + row[u] * q.ld, static_cast<int>(chunk[u]) * MX_CHUNK + 4 * lane, static_cast<int>(q.K)) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      if (at + u >= all) break;
      uint8_t* scales = q.scales + mx_scale_offset(row[u], chunk[u], q.chunks);
      if (row[u] < q.rows)
        mx_store_chunk<FP4>(v[u], mx_scale_of<FP4>(largest_of_block(v[u])), q.codes + (row[u] * q.chunks + chunk[u]) * MxFormat<FP4>::kChunkBytes, scales, lane);
      else if (lane == 0)
        *reinterpret_cast<uint32_t*>(scales) = 0u;
    }
  }
}

// Columns of a matrix stored K x rows: a block takes 32 of its columns (rows of the result) and 256 of its rows, a thread 32 values below one
// another, which is a block with one scale.  The codes go through shared memory, so that a row's 256 (128) bytes are written together.
template <bool FP4>
__global__ void __launch_bounds__(256) mx_quantize_columns_kernel(const MxQuantize q) {
  constexpr int BYTES = FP4 ? 16 : 32;            // codes of a block
  constexpr int PITCH = 8 * BYTES + 16;           // 16 more: rows start on different banks
  __shared__ __align__(16) uint8_t codes[32 * PITCH];
  __shared__ uint8_t scales[32][8];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const long long row_tiles = (q.rows + 127) / 128 * 4, k_tiles = (q.chunks + 1) / 2;
  const long long tiles = row_tiles * k_tiles;
  for (long long tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    const long long kt = tile / row_tiles, row0 = (tile - kt * row_tiles) * 32;
    const long long k0 = kt * 256 + warp * 32;
    float v[32];
    const float* src = q.src + k0 * q.ld + row0 + lane;
    const bool in = row0 + lane < q.rows;
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] = in && k0 + i < q.K ? __ldg(src + i * q.ld) : 0.0f;
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
    uint8_t* to = codes + lane * PITCH + warp * BYTES;
#pragma unroll
    for (int i = 0; i < BYTES / 16; ++i)
      reinterpret_cast<uint4*>(to)[i] = make_uint4(words[4 * i], words[4 * i + 1], words[4 * i + 2], words[4 * i + 3]);
    scales[lane][warp] = static_cast<uint8_t>(scale);
    __syncthreads();
    constexpr int QUADS = 8 * BYTES / 16;  // 16-byte pieces of a row
    const int pieces = static_cast<int>(min(2ll, q.chunks - kt * 2)) * (QUADS / 2);
    for (int i = threadIdx.x; i < 32 * QUADS; i += 256) {
      const int r = i / QUADS, piece = i % QUADS;
      if (row0 + r < q.rows && piece < pieces)
        *reinterpret_cast<uint4*>(q.codes + ((row0 + r) * q.chunks + kt * 2) * MxFormat<FP4>::kChunkBytes + piece * 16) =
            *reinterpret_cast<const uint4*>(codes + r * PITCH + piece * 16);
    }
    if (threadIdx.x < 64) {
      const int r = threadIdx.x >> 1, half = threadIdx.x & 1;
      if (kt * 2 + half < q.chunks) {
        const uint32_t four = *reinterpret_cast<const uint32_t*>(&scales[r][half * 4]);
        *reinterpret_cast<uint32_t*>(q.scales + mx_scale_offset(row0 + r, kt * 2 + half, q.chunks)) = row0 + r < q.rows ? four : 0u;
      }
    }
    __syncthreads();
  }
}

// Back to float32: exact, for a code has at most four significant bits.
struct MxDequantize {
  const uint8_t *codes, *scales;
  float* dst;
  long long ld, rows, K, chunks;
};
template <bool FP4, bool VEC>
__global__ void __launch_bounds__(MX_QUANTIZE_THREADS) mx_dequantize_kernel(const MxDequantize q) {
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long warps = static_cast<long long>(gridDim.x) * (MX_QUANTIZE_THREADS / 32);
  for (long long at = static_cast<long long>(blockIdx.x) * (MX_QUANTIZE_THREADS / 32) + (threadIdx.x >> 5); at < q.rows * q.chunks; at += warps) {
    const long long row = at / q.chunks, chunk = at - row * q.chunks;
    const uint8_t* codes = q.codes + at * MxFormat<FP4>::kChunkBytes;
    const float scale = mx_scale_value(q.scales[mx_scale_offset(row, chunk, q.chunks) + lane / 8]);
    float2 lo, hi;
    if constexpr (FP4) {
      const uint32_t c = reinterpret_cast<const uint16_t*>(codes)[lane];
      const __half2_raw a = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(c & 255u), __NV_E2M1);
      const __half2_raw b = __nv_cvt_fp4x2_to_halfraw2(static_cast<__nv_fp4x2_storage_t>(c >> 8), __NV_E2M1);
      lo = __half22float2(__half2(a));
      hi = __half22float2(__half2(b));
    } else {
      const uint32_t c = reinterpret_cast<const uint32_t*>(codes)[lane];
      const __half2_raw a = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c & 65535u), __NV_E4M3);
      const __half2_raw b = __nv_cvt_fp8x2_to_halfraw2(static_cast<__nv_fp8x2_storage_t>(c >> 16), __NV_E4M3);
      lo = __half22float2(__half2(a));
      hi = __half22float2(__half2(b));
    }
    store4<VEC>(q.dst + row * q.ld, static_cast<int>(chunk) * MX_CHUNK + 4 * lane, static_cast<int>(q.K), make_float4(lo.x * scale, lo.y * scale, hi.x * scale, hi.y * scale));
  }
}

}  // namespace sb200
