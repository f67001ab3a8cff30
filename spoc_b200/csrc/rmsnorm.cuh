// rmsnorm.cuh — root-mean-square norm with the residual's addition, its result in float32 or microscaled, and its gradient.
//
//   h = x + residual (rounded to float32: it is stored, and the next layer adds to it),  y = h * weight / sqrt(mean(h^2) + eps)
//
// A code of 8 or 4 bits is the rounding of the exact y of the stored h, with the sum of squares and the root in 64 bits: next to a rounding border
// float32 falls on one side or the other depending on the order of the sum, one value in a million by a whole step, and so would all that is
// computed from it.  64 bits throughout are not needed for that: y in float32 is at most 2^-22 of it off (two products, and the scale, which is two of
// 2^-24 off).  Where a value of a warp's chunk has another code, or a block another scale, for 1 - RMS_DOUBT and 1 + RMS_DOUBT times it, or lies
// outside the range in which this holds, the warp does the chunk over in 64 bits (rmsnorm_chunk_exact), one chunk of 600.
//
// A block a row, or a warp up to 1024 columns, the row in registers (VECS float4 a thread; thread t has columns 4 (v * threads + t)), so that x
// and residual are read once.  Rows too long for that (32768 columns on) are read twice.  Bound by HBM: 8 bytes read, 5 written a value with
// 8-bit codes, and by the blocks in flight: 8192 x 8192 with a residual to 8 bits takes 143 us (135 at the copy bandwidth), with 126 registers a thread
// and one block an SM it took 337.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "microscale.cuh"

namespace sb200 {

constexpr float RMS_DOUBT = 4.76837158203125e-7f;  // 2^-21

struct RmsNorm {
  const float *x, *residual, *weight;  // residual may be null
  long long ldx, ldr, ldh, ldy;
  float *h, *y;                        // either may be null
  uint8_t *codes, *scales;             // null: no microscaled result
  long long rows;
  int cols, chunks;
  double inv_cols, eps;
};

// Sum over the block of a value a thread, the same in all threads and in every launch.
template <int THREADS, class T>
__device__ __forceinline__ T block_sum(T v, T* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (THREADS == 32) return v;
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  T s = shared[threadIdx.x & (THREADS / 32 - 1)];
#pragma unroll
  for (int o = THREADS / 64; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  return s;
}

// A double rounded toward zero to float32, with the last bit set where that lost something: rounding the result to any shorter type gives
// what rounding the double to it would.  Beyond float32's range: infinity.
__device__ __forceinline__ float round_to_odd(double y) {
  uint32_t b = __float_as_uint(__double2float_rz(y));
  const uint32_t hi = static_cast<uint32_t>(__double2hiint(y)) & 0x7fffffffu, lo = static_cast<uint32_t>(__double2loint(y));
  if (hi >= (1023u + 128u) << 20) return hi > 0x7ff00000u || (hi == 0x7ff00000u && lo) ? __uint_as_float(0x7fc00000u) : __uint_as_float((b & 0x80000000u) | 0x7f800000u);
  if ((lo & 0x1fffffffu) != 0 || (hi < (1023u - 126u) << 20 && static_cast<double>(__uint_as_float(b)) != y)) b |= 1u;
  return __uint_as_float(b);
}

template <bool FP4>
__device__ __noinline__ void rmsnorm_chunk_exact(float4 h, float4 w, double mean, uint8_t* codes, uint8_t* scales, int col, int cols) {
  const int lane = threadIdx.x & 31, left = cols - col;
  const double scale = 1.0 / sqrt(mean);
  float4 y = make_float4(round_to_odd(h.x * scale * w.x), round_to_odd(h.y * scale * w.y), round_to_odd(h.z * scale * w.z),
                         round_to_odd(h.w * scale * w.w));
  if (left < 4) {  // past K are zeros, where the mean is no number too
    if (left < 1) y.x = 0.f;
    if (left < 2) y.y = 0.f;
    if (left < 3) y.z = 0.f;
    y.w = 0.f;
  }
  mx_store_chunk<FP4>(y, mx_scale_of<FP4>(largest_of_block(y)), codes, scales, lane);
}

// 1 / sqrt(m) of a finite m: rsqrtf is two units in the last place off; a step of Newton's leaves the error of its own two roundings.
__device__ __forceinline__ float refined_root(float m) {
  const float s = rsqrtf(m);
  return fmaf(0.5f * s, fmaf(-m * s, s, 1.0f), s);
}
// 1 / sqrt(mean) is the result times *unit, which is 1, or a power of two that brings a mean far from 1 near to it.
__device__ __forceinline__ float inverse_root(double mean, float* unit) {
  const int half = (static_cast<int>(__double2hiint(mean) >> 20 & 0x7ff) - 1023) / 2;
  const float u = abs(half) < 45 ? 1.0f : __uint_as_float(static_cast<uint32_t>(min(max(127 - half, 1), 254)) << 23);
  float m = static_cast<float>(mean * u * u);
  // Only the eps of a row of zeros is so small: one of float32's smallest values in 2^31 makes a mean of 2^-329, and m 2^-75.
  if (m < 1.17549435e-38f && mean > 0.0) m = 1.17549435e-38f;
  const float s = refined_root(m);
  *unit = u;
  return m < INFINITY ? s : rsqrtf(m);  // of an infinite mean 0
}

// What a row's results need.
struct RmsRow {
  double mean;      // of the squares, plus eps
  float unit;       // 1, or a power of two that brings values of a mean far from 1 near to it
  float scale;      // 1 / (unit * sqrt(mean)), nearly
  float* y;         // the result's row, or null
  uint8_t *codes, *scales;  // of the warp's first chunk
};
template <int FORMAT>
__device__ __forceinline__ RmsRow rmsnorm_row(const RmsNorm& p, long long row, int first_chunk, double sum) {
  RmsRow r;
  r.mean = fma(sum, p.inv_cols, p.eps);
  r.scale = inverse_root(r.mean, &r.unit);
  r.y = p.y ? p.y + row * p.ldy : nullptr;
  r.codes = p.codes + (row * p.chunks + first_chunk) * (FORMAT == 4 ? 64 : 128);
  r.scales = p.scales + mx_scale_offset(row, first_chunk, p.chunks);
  return r;
}
// Four values of the normed row from column `col` on, `ahead` chunks behind the warp's first.  FORMAT: 0 float32 only, 4, 8.
template <int FORMAT, int ACCESS>
__device__ __forceinline__ void rmsnorm_emit(const RmsNorm& p, const RmsRow& row, int col, int ahead, const float4& h, int lane) {
  const float4 w = load4<ACCESS>(p.weight, col, p.cols);
  float4 y = h;
  if (row.unit != 1.0f) y = make_float4(h.x * row.unit, h.y * row.unit, h.z * row.unit, h.w * row.unit);
  const float2 s = make_float2(row.scale, row.scale);
  const float2 y01 = multiply2(multiply2(make_float2(y.x, y.y), s), make_float2(w.x, w.y)), y23 = multiply2(multiply2(make_float2(y.z, y.w), s), make_float2(w.z, w.w));
  y = make_float4(y01.x, y01.y, y23.x, y23.y);
  if (row.y) store4<ACCESS>(row.y, col, p.cols, y);
  if constexpr (FORMAT != 0) {
    constexpr bool FP4 = FORMAT == 4;
    if (col >> 7 >= p.chunks) return;  // the same in a whole warp
    uint8_t* codes = row.codes + static_cast<long long>(ahead) * MxFormat<FP4>::kChunkBytes;
    uint8_t* scales = row.scales + static_cast<long long>(ahead) * MX_TILE_BYTES;
    const uint32_t m = largest_of_block(y), block_scale = mx_scale_of<FP4>(m);
    const float f = mx_factor(block_scale), top = __uint_as_float(m);
    const uint32_t low = mx_codes4<FP4>(y, f * (1.0f - RMS_DOUBT)), high = mx_codes4<FP4>(y, f * (1.0f + RMS_DOUBT));
    // The estimate holds for weights below 2^40 and a largest value between 2^-60 and 2^100: products that fall below float32's range then lose
    // nothing that a code shows.  A block of zeros holds too, where h is zero.
    bool again = low != high || !(fmaxf(fmaxf(fabsf(w.x), fabsf(w.y)), fmaxf(fabsf(w.z), fabsf(w.w))) < 1.09951163e12f) || m - (67u << 23) >= 160u << 23 ||
                 ((__float_as_uint(top * (1.0f - RMS_DOUBT)) ^ __float_as_uint(top * (1.0f + RMS_DOUBT))) >> 23) != 0;
    if (__any_sync(0xffffffffu, again)) {
      if (m == 0 && low == high) again = (abs_bits(h.x) | abs_bits(h.y) | abs_bits(h.z) | abs_bits(h.w)) != 0;
      if (__any_sync(0xffffffffu, again)) {
        rmsnorm_chunk_exact<FP4>(h, w, row.mean, codes, scales, col, p.cols);
        return;
      }
    }
    mx_store_codes<FP4>(low, block_scale, codes, scales, lane);
  }
}
template <int ACCESS>
__device__ __forceinline__ float4 rmsnorm_input(const RmsNorm& p, long long row, int col) {
  float4 h = load4<ACCESS>(p.x + row * p.ldx, col, p.cols);
  if (p.residual) {
    const float4 r = load4<ACCESS>(p.residual + row * p.ldr, col, p.cols);
    h = make_float4(__fadd_rn(h.x, r.x), __fadd_rn(h.y, r.y), __fadd_rn(h.z, r.z), __fadd_rn(h.w, r.w));
  }
  return h;
}
__device__ __forceinline__ double squares(const float4& h) {
  return fma(static_cast<double>(h.x), static_cast<double>(h.x), static_cast<double>(h.y) * h.y) +
         fma(static_cast<double>(h.z), static_cast<double>(h.z), static_cast<double>(h.w) * h.w);
}
// THREADS: of a row; 32: a block has four rows.  VECS = 0: rows of any length, read twice (h may be x or residual itself: then the second
// reading takes h, which was stored).
template <int FORMAT, int THREADS, int VECS, int ACCESS, int BLOCKS>
__global__ void __launch_bounds__(THREADS == 32 ? 128 : THREADS, BLOCKS) rmsnorm_kernel(const RmsNorm p) {
  constexpr int ROWS = THREADS == 32 ? 4 : 1;
  constexpr int GLOBAL = VECS > 0 && ACCESS == ACCESS_SINGLE ? ACCESS_LANES : ACCESS;  // of x, residual and h
  __shared__ double shared[2][THREADS / 32];
  __shared__ float4 turn_of[GLOBAL == ACCESS ? 1 : THREADS == 32 ? 128 : THREADS];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, thread = THREADS == 32 ? lane : threadIdx.x, first = 4 * thread;
  const long long rows = FORMAT ? (p.rows + 127) / 128 * 128 : p.rows;
  int turn = 0;
  for (long long row = blockIdx.x * static_cast<long long>(ROWS) + (ROWS > 1 ? threadIdx.x >> 5 : 0); row < rows;
       row += gridDim.x * static_cast<long long>(ROWS), turn ^= 1) {
    if (FORMAT && row >= p.rows) {  // the scales' padding
      for (int c = thread; c < p.chunks; c += THREADS) *reinterpret_cast<uint32_t*>(p.scales + mx_scale_offset(row, c, p.chunks)) = 0u;
      continue;
    }
    if constexpr (VECS > 0) {
      float4 h[VECS];
#pragma unroll
      for (int v = 0; v < VECS; ++v) h[v] = rmsnorm_input<GLOBAL>(p, row, first + v * 4 * THREADS);
      double s = 0.0;
#pragma unroll
      for (int v = 0; v < VECS; ++v) s += squares(h[v]);
      if (p.h) {
        float* to = p.h + row * p.ldh;
#pragma unroll
        for (int v = 0; v < VECS; ++v) store4<GLOBAL>(to, first + v * 4 * THREADS, p.cols, h[v]);
      }
      if constexpr (GLOBAL != ACCESS) {
#pragma unroll
        for (int v = 0; v < VECS; ++v) h[v] = turned(h[v], turn_of + (threadIdx.x & ~31), lane);
      }
      const RmsRow r = rmsnorm_row<FORMAT>(p, row, first >> 7, block_sum<THREADS>(s, shared[turn]));
#pragma unroll
      for (int v = 0; v < VECS; ++v) rmsnorm_emit<FORMAT, ACCESS>(p, r, first + v * 4 * THREADS, v * (THREADS / 32), h[v], lane);
    } else {
      const long long padded = static_cast<long long>(p.chunks) * MX_CHUNK;
      double s = 0.0;
      for (long long c = first; c < padded; c += 4 * THREADS) {
        const int col = static_cast<int>(c);
        const float4 h = rmsnorm_input<ACCESS>(p, row, col);
        s += squares(h);
        if (p.h) store4<ACCESS>(p.h + row * p.ldh, col, p.cols, h);
      }
      const RmsRow r = rmsnorm_row<FORMAT>(p, row, first >> 7, block_sum<THREADS>(s, shared[turn]));
      for (long long c = first; c < padded; c += 4 * THREADS) {
        const int col = static_cast<int>(c);
        const float4 h = p.h ? load4<ACCESS>(p.h + row * p.ldh, col, p.cols) : rmsnorm_input<ACCESS>(p, row, col);
        rmsnorm_emit<FORMAT, ACCESS>(p, r, col, (col - first) >> 7, h, lane);
      }
    }
  }
}

// The gradient: with r = 1 / sqrt(mean(h^2) + eps), n = h r and g = dy * weight,
//   dx = dsum + r (g - n mean(g n)),   dweight = sum over the rows of dy n.
// A block (a cluster) takes rows blockIdx.x, + gridDim.x, ... and keeps its part of dweight; a second kernel adds the parts in the order of the
// blocks.  Bound by HBM: 12 bytes read and 4 written a value.
struct RmsNormBackward {
  const float *h, *weight, *dy, *dsum;  // dsum may be null
  long long ldh, lddy, ldds, lddx;
  float *dx, *dweight, *workspace;      // either of dx and dweight may be null
  int* status;
  long long rows;
  int cols;
  int blocks, slice;                    // of a row, where a cluster takes it
  float least;                          // sums of squares below it are too small for float32
  double inv_cols, eps;
};
// A row's two sums, of h^2 and of h g, are float32 where they hold: squares of values past 2^64 / sqrt(cols) are infinite, and r zero, and squares
// below 2^-126 lose bits, which nothing shows beside an eps of 2^-80 or a sum of that.  Other rows are summed again in 64 bits; doing so for every row
// took 8192 x 4095 from 87 to 106 us and 16384 x 256 from 14.5 to 15.6.
constexpr double RMS_LEAST = 8.271806125530277e-25;  // 2^-80
__device__ __forceinline__ bool sums_hold(const RmsNormBackward& p, const float2& s) {
  return s.x >= p.least && s.x < 8.507059e37f && fabsf(s.y) < 8.507059e37f;  // 2^126; false of NaN
}
__device__ __forceinline__ float2 sums_of_four(const float4& h, const float4& dy, const float4& w) {
  return make_float2(fmaf(h.x, h.x, h.y * h.y) + fmaf(h.z, h.z, h.w * h.w),
                     fmaf(h.x, dy.x * w.x, h.y * (dy.y * w.y)) + fmaf(h.z, dy.z * w.z, h.w * (dy.w * w.w)));
}
__device__ __forceinline__ void add_exactly(double2& s, float h, float dy, float w) {
  const double a = h;
  s.x = fma(a, a, s.x);
  s.y = fma(a, static_cast<double>(dy * w), s.y);
}
template <class T>
__device__ __forceinline__ void sum_over_warp(T& s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
    s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
  }
}
// The column of element j of a thread's four from `col` on, as load4 has them.
template <int ACCESS>
__device__ __forceinline__ int column_of(int col, int j) {
  return ACCESS == ACCESS_LANES ? (col & ~127) + ((col & 127) >> 2) + 32 * j : col + j;
}
// What a row's gradient needs of its sums: r, and the mean of g n.
__device__ __forceinline__ float2 backward_row(const RmsNormBackward& p, const double2& s) {
  float unit;
  const float r = inverse_root(fma(s.x, p.inv_cols, p.eps), &unit) * unit;
  return make_float2(r, static_cast<float>(s.y * p.inv_cols * r));
}
__device__ __forceinline__ float4 normed(const float4& h, float r) { return make_float4(h.x * r, h.y * r, h.z * r, h.w * r); }
// r (g - n mean(g n)) + dsum
__device__ __forceinline__ float4 backward_of(const float4& n, const float4& dy, const float4& w, const float4& dsum, const float2& row) {
  return make_float4(row.x * fmaf(-n.x, row.y, dy.x * w.x) + dsum.x, row.x * fmaf(-n.y, row.y, dy.y * w.y) + dsum.y,
                     row.x * fmaf(-n.z, row.y, dy.z * w.z) + dsum.z, row.x * fmaf(-n.w, row.y, dy.w * w.w) + dsum.w);
}
__device__ __forceinline__ float4 added(const float4& part, const float4& dy, const float4& n) {
  return make_float4(fmaf(dy.x, n.x, part.x), fmaf(dy.y, n.y, part.y), fmaf(dy.z, n.z, part.z), fmaf(dy.w, n.w, part.w));
}
// Rows of any length: h and dy are read twice, and the part of dweight is kept in the block's row of the workspace.  Four values are summed in
// float32, the fours, of which a thread may have half a million, in 64 bits.
template <int ACCESS>
__global__ void __launch_bounds__(1024) rmsnorm_backward_kernel(const RmsNormBackward p) {
  constexpr int THREADS = 1024, PART = ACCESS == ACCESS_VECTOR ? ACCESS_SINGLE : ACCESS;  // the workspace starts on 4 bytes
  __shared__ double2 shared[2][THREADS / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const int first = 4 * threadIdx.x;
  const long long padded = (p.cols + 127ll) / 128 * 128;
  float* const mine = p.workspace + static_cast<long long>(blockIdx.x) * p.cols;
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x) {
    const float *hr = p.h + row * p.ldh, *dyr = p.dy + row * p.lddy;
    auto over_block = [&](double2 s) {
      sum_over_warp(s);
      if ((threadIdx.x & 31) == 0) shared[turn][threadIdx.x >> 5] = s;
      __syncthreads();
      s = shared[turn][threadIdx.x & 31];
      sum_over_warp(s);
      turn ^= 1;
      return s;
    };
    double2 s = make_double2(0.0, 0.0);
    for (long long c = first; c < padded; c += 4 * THREADS) {
      const int col = static_cast<int>(c);
      const float2 t = sums_of_four(load4<ACCESS>(hr, col, p.cols), load4<ACCESS>(dyr, col, p.cols), load4<ACCESS>(p.weight, col, p.cols));
      s.x += t.x;
      s.y += t.y;
    }
    s = over_block(s);
    if (!sums_hold(p, make_float2(static_cast<float>(s.x), static_cast<float>(s.y)))) {
      s = make_double2(0.0, 0.0);
      for (long long c = threadIdx.x; c < p.cols; c += THREADS) add_exactly(s, hr[c], dyr[c], p.weight[c]);
      s = over_block(s);
    }
    const float2 of_row = backward_row(p, s);
    for (long long c = first; c < padded; c += 4 * THREADS) {
      const int col = static_cast<int>(c);
      const float4 n = normed(load4<ACCESS>(hr, col, p.cols), of_row.x), d = load4<ACCESS>(dyr, col, p.cols);
      if (p.dweight) {
        float4 part = make_float4(0.f, 0.f, 0.f, 0.f);
        if (row != blockIdx.x) part = load4<PART>(mine, col, p.cols);
        store4<PART>(mine, col, p.cols, added(part, d, n));
      }
      if (p.dx) {
        float4 ds = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p.dsum) ds = load4<ACCESS>(p.dsum + row * p.ldds, col, p.cols);
        store4<ACCESS>(p.dx + row * p.lddx, col, p.cols, backward_of(n, d, load4<ACCESS>(p.weight, col, p.cols), ds, of_row));
      }
    }
  }
}
// Rows that the registers of a block, or of a cluster, hold, read once: groups of TG threads go from row to row, each with a ring of STAGES rows of
// h, dy and dsum in shared memory that bulk copies fill ahead of it, so that the copies of one row run under the sums of another (8192 x 4096
// 131 us with a row's loads in front of its sums, 84 so, 83 at the copy bandwidth).  ACCESS_LANES: rows that do not all start on 16 bytes.
// Copies then begin and end at the multiples of 16 bytes around a row; the few bytes beside it are neither used nor beyond the 16 bytes of its first
// and last value.  WIDE: a cluster of p.blocks blocks a row, each with p.slice of its columns, which send one another their sums.
__device__ __forceinline__ uint32_t bulk_offset(const float* row) { return static_cast<uint32_t>(reinterpret_cast<uintptr_t>(row) >> 2 & 3); }
template <int TG, int G, int VECS, int STAGES, int ACCESS>
struct BackwardRing {
  static constexpr int kThreads = TG * G, kCols = TG * VECS * 4;
  static constexpr int kArrayBytes = kCols * 4 + (ACCESS == ACCESS_LANES ? 32 : 0), kStageBytes = 3 * kArrayBytes;
  static constexpr int kBytes = G * STAGES * kStageBytes + 128;  // the copies start on 128 bytes
  static_assert(G * kCols * 4 <= G * STAGES * kStageBytes, "the groups' parts of dweight fit the ring");
  static_assert(kArrayBytes % 16 == 0, "copies start on 16 bytes");
};
constexpr int RMS_MAX_CLUSTER = 8;
template <int TG, int G, int VECS, int STAGES, int ACCESS, bool WIDE>
__global__ void __launch_bounds__(TG * G, 1) rmsnorm_backward_ring_kernel(const RmsNormBackward p) {
  using Ring = BackwardRing<TG, G, VECS, STAGES, ACCESS>;
  static_assert(!WIDE || (G == 1 && TG >= 128), "a group of several warps");
  constexpr int PART = ACCESS == ACCESS_VECTOR ? ACCESS_SINGLE : ACCESS;  // the workspace starts on 4 bytes
  extern __shared__ uint8_t smem_raw[];
  __shared__ uint64_t full[G * STAGES];
  __shared__ float2 sums[2][G * TG / 32];
  __shared__ double2 exact_sums[G * TG / 32], exact_of_blocks[WIDE ? RMS_MAX_CLUSTER : 1];
  __shared__ float2 of_blocks[2][WIDE ? RMS_MAX_CLUSTER : 1];  // sums of the blocks of the cluster, rows in turn
  __shared__ uint64_t sent[3];                                 // and the barriers that count them; the last: exact sums
  __shared__ int abort_word;
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 127) & ~uintptr_t(127));
  const int group = threadIdx.x / TG, thread = threadIdx.x % TG, warp = threadIdx.x >> 5, lane = threadIdx.x & 31, first = 4 * thread;
  const int blocks = WIDE ? p.blocks : 1, rank = WIDE ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = WIDE ? static_cast<int>(blockIdx.x) / blocks : static_cast<int>(blockIdx.x);
  const int units = WIDE ? static_cast<int>(gridDim.x) / blocks : static_cast<int>(gridDim.x);
  const int col0 = WIDE ? rank * p.slice : 0, cols = WIDE ? min(p.slice, p.cols - col0) : p.cols;
  const float *const weight = p.weight + col0, *const h0 = p.h + col0, *const dy0 = p.dy + col0, *const dsum0 = p.dsum ? p.dsum + col0 : nullptr;
  uint8_t* mine = ring + group * STAGES * Ring::kStageBytes;
  if (threadIdx.x < G * STAGES) {
    mbar_init(smem_u32(&full[threadIdx.x]), 1);
    if (WIDE && threadIdx.x == 0)
      for (int k = 0; k < 3; ++k) mbar_init(smem_u32(&sent[k]), 1);
    mbar_fence_init();
  }
  if (threadIdx.x == 0) abort_word = 0;
  __syncthreads();
  if (WIDE) {  // the barriers are there before another block sends
    cluster_arrive_relaxed();
    cluster_wait();
  }
  grid_launch_dependents();
  grid_dependency_wait();
  const float inv_cols = 1.0f / static_cast<float>(p.cols), eps = static_cast<float>(p.eps);
  const long long step = static_cast<long long>(units) * G, row0 = unit + static_cast<long long>(units) * group;
  const uint32_t bytes = static_cast<uint32_t>(cols) * 4;
  auto fetch = [&](int stage, long long row) {  // one thread
    const uint32_t bar = smem_u32(&full[group * STAGES + stage]), to = smem_u32(mine) + stage * Ring::kStageBytes;
    auto size = [&](const float* from) { return ((ACCESS == ACCESS_VECTOR ? 0u : bulk_offset(from)) * 4 + bytes + 15) & ~15u; };
    auto copy = [&](int array, const float* from) {
      bulk_load(to + array * Ring::kArrayBytes, ACCESS == ACCESS_VECTOR ? from : from - bulk_offset(from), size(from), bar);
    };
    const float *h = h0 + row * p.ldh, *dy = dy0 + row * p.lddy, *ds = dsum0 + row * p.ldds;
    mbar_arrive_expect_tx(bar, size(h) + size(dy) + (p.dsum ? size(ds) : 0));
    copy(0, h);
    copy(1, dy);
    if (p.dsum) copy(2, ds);
  };
  if (thread == 0) {
#pragma unroll 1
    for (int s = 0; s < STAGES; ++s)
      if (row0 + s * step < p.rows) fetch(s, row0 + s * step);
  }
  float4 w[VECS], part[VECS];
#pragma unroll
  for (int v = 0; v < VECS; ++v) {
    w[v] = load4<ACCESS>(weight, first + v * 4 * TG, cols);
    part[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  }
  int stage = 0, turn = 0;
  uint32_t phase = 0, sent_phase = 0, exact_phase = 0;
  bool ok = true, ended = false;
  // The next copies come behind the row's stores: in front of them they hold those up (8192 x 8191 199 us, 160 so).  Rows of a cluster that do not
  // start on 16 bytes take them between their stores (4096 x 9999 139 -> 137, 1024 x 65535 189 -> 184; others lose: 6000 x 8196 141 -> 148).
  constexpr bool kFetchWithin = WIDE && ACCESS == ACCESS_LANES;
  for (long long row = row0; row < p.rows; row += step) {
    auto fetch_next = [&] {
      if (thread == 0 && row + STAGES * step < p.rows) fetch(stage, row + STAGES * step);
    };
    const uint8_t* from = mine + stage * Ring::kStageBytes;
    ok = mbar_wait_bounded(smem_u32(&full[group * STAGES + stage]), phase, &abort_word) && ok;
    float4 h[VECS], dy[VECS], ds[VECS];
    float2 s = make_float2(0.f, 0.f);  // of h^2 and of h * g
#pragma unroll
    for (int v = 0; v < VECS; ++v) {
      const int col = first + v * 4 * TG;
      const float* const at = reinterpret_cast<const float*>(from);
      h[v] = dy[v] = ds[v] = make_float4(0.f, 0.f, 0.f, 0.f);
      if constexpr (ACCESS == ACCESS_VECTOR) {
        if (col < cols) {
          h[v] = *reinterpret_cast<const float4*>(at + col);
          dy[v] = *reinterpret_cast<const float4*>(at + Ring::kArrayBytes / 4 + col);
          if (p.dsum) ds[v] = *reinterpret_cast<const float4*>(at + 2 * (Ring::kArrayBytes / 4) + col);
        }
      } else {
        h[v] = load4<ACCESS>(at + bulk_offset(h0 + row * p.ldh), col, cols);
        dy[v] = load4<ACCESS>(at + Ring::kArrayBytes / 4 + bulk_offset(dy0 + row * p.lddy), col, cols);
        if (p.dsum) ds[v] = load4<ACCESS>(at + 2 * (Ring::kArrayBytes / 4) + bulk_offset(dsum0 + row * p.ldds), col, cols);
      }
      const float2 t = sums_of_four(h[v], dy[v], w[v]);
      s.x += t.x;
      s.y += t.y;
    }
    sum_over_warp(s);
    if (TG > 32) {
      if (lane == 0) sums[turn][warp] = s;
      ok = barrier_all(1 + group, TG, ok);  // the group has read the stage; all of it goes on, or none
    } else {
      ok = __all_sync(0xffffffffu, ok);
    }
    if (!ok) {
      ended = true;
      break;
    }
    if constexpr (WIDE) {
      // A block sends its sums of the next row when all its threads have read those of this one, so that those of the row after that may be
      // written over them; its exact sums come between two of these.  Who gives up does so at the block's next barrier, with the whole block.
      if (warp == 3) {
        s = lane < TG / 32 ? sums[turn][lane] : make_float2(0.f, 0.f);
        sum_over_warp(s);
        const uint32_t bar = smem_u32(&sent[turn]);
        if (lane == 0) mbar_arrive_expect_tx(bar, blocks * 8);
        if (lane < blocks) st_async_pair(map_to_cta(smem_u32(&of_blocks[turn][rank]), lane), s, map_to_cta(bar, lane));
      }
      ok = __all_sync(0xffffffffu, mbar_wait_cluster(smem_u32(&sent[turn]), sent_phase, &abort_word));
      s = make_float2(0.f, 0.f);
      for (int k = 0; k < blocks; ++k) {
        s.x += of_blocks[turn][k].x;
        s.y += of_blocks[turn][k].y;
      }
      sent_phase ^= turn;
    } else if (TG > 32) {
      s = make_float2(0.f, 0.f);
#pragma unroll
      for (int k = 0; k < TG / 32; ++k) {
        s.x += sums[turn][group * (TG / 32) + k].x;
        s.y += sums[turn][group * (TG / 32) + k].y;
      }
    }
    turn ^= 1;
    bool hold = sums_hold(p, s) || (WIDE && !ok);
    if (TG == 32) hold = __all_sync(0xffffffffu, hold);  // a branch of the whole warp: 16384 x 200 13.36 -> 13.16 us
    if (hold) {
      const float r = refined_root(s.x * inv_cols + eps);
      const float2 of_row = make_float2(r, s.y * inv_cols * r);
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
        if (kFetchWithin && v == 1) fetch_next();
        const float4 n = normed(h[v], of_row.x);
        if (p.dx) store4<ACCESS>(p.dx + col0 + row * p.lddx, first + v * 4 * TG, cols, backward_of(n, dy[v], w[v], ds[v], of_row));
        part[v] = added(part[v], dy[v], n);
      }
    } else {
      // All of the group, which has the same sums, does them over.  A warp that gave up is not here but at the next row's barrier, or behind the
      // loop: there it brings its false, and all of them end.  Small loops over the row as it lies in global memory: held in registers
      // throughout it made the kernel spill (8192 x 8191 160 -> 173 us).
      double2 exact = make_double2(0.0, 0.0);
#pragma unroll 1
      for (int k = 0; k < 4 * VECS; ++k) {
        const int col = column_of<ACCESS>(first + (k >> 2) * 4 * TG, k & 3);
        if (col >= cols) continue;
        add_exactly(exact, h0[row * p.ldh + col], dy0[row * p.lddy + col], weight[col]);
      }
      sum_over_warp(exact);
      if (TG > 32) {
        if (lane == 0) exact_sums[warp] = exact;
        ok = barrier_all(1 + group, TG, ok);
        if (!ok) {
          ended = true;
          break;
        }
        exact = make_double2(0.0, 0.0);
        if constexpr (WIDE) {
          if (warp == 3) {
            if (lane < TG / 32) exact = exact_sums[lane];
            sum_over_warp(exact);
            const uint32_t bar = smem_u32(&sent[2]);
            if (lane == 0) mbar_arrive_expect_tx(bar, blocks * 16);
            if (lane < blocks) st_async_pair(map_to_cta(smem_u32(&exact_of_blocks[rank]), lane), exact, map_to_cta(bar, lane));
            exact = make_double2(0.0, 0.0);
          }
          ok = __all_sync(0xffffffffu, mbar_wait_cluster(smem_u32(&sent[2]), exact_phase, &abort_word));
          exact_phase ^= 1u;
        }
        const double2* const parts = WIDE ? exact_of_blocks : exact_sums + group * (TG / 32);
        const int count = WIDE ? blocks : TG / 32;
#pragma unroll 1
        for (int k = 0; k < count; ++k) {
          exact.x += parts[k].x;
          exact.y += parts[k].y;
        }
      }
      const float2 of_row = backward_row(p, exact);
#pragma unroll 1
      for (int k = 0; k < 4 * VECS; ++k) {
        const int col = column_of<ACCESS>(first + (k >> 2) * 4 * TG, k & 3);
        if (col >= cols) continue;
        const float n = h0[row * p.ldh + col] * of_row.x, d = dy0[row * p.lddy + col];
#pragma unroll
        for (int u = 0; u < VECS; ++u) {
          if (k == 4 * u) part[u].x = fmaf(d, n, part[u].x);
          if (k == 4 * u + 1) part[u].y = fmaf(d, n, part[u].y);
          if (k == 4 * u + 2) part[u].z = fmaf(d, n, part[u].z);
          if (k == 4 * u + 3) part[u].w = fmaf(d, n, part[u].w);
        }
        if (p.dx) p.dx[col0 + row * p.lddx + col] = of_row.x * fmaf(-n, of_row.y, d * weight[col]) + (p.dsum ? dsum0[row * p.ldds + col] : 0.0f);
      }
    }
    if (!kFetchWithin || !hold) fetch_next();
    if (++stage == STAGES) {
      stage = 0;
      phase ^= 1u;
    }
  }
  if (WIDE && !ended) ok = barrier_all(1, TG, ok);
  if (!ok) {
    atomicCAS(p.status, 0, 0x5100 | group);
    wait_for_copies();
  }
  if (WIDE) {  // no block retires while another can still send to it
    __syncwarp();
    cluster_arrive_relaxed();
    cluster_wait();
  }
  if (!p.dweight) return;
  float* const to = p.workspace + static_cast<long long>(unit) * p.cols + col0;
  if (G == 1) {
#pragma unroll
    for (int v = 0; v < VECS; ++v) store4<PART>(to, first + v * 4 * TG, cols, part[v]);
    return;
  }
  __syncthreads();  // no copy is in flight: every group has waited for all that it asked for
  float* const shared_part = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int v = 0; v < VECS; ++v) store4<ACCESS>(shared_part + group * Ring::kCols, first + v * 4 * TG, Ring::kCols, part[v]);
  __syncthreads();
  for (int c = threadIdx.x; c < cols; c += TG * G) {
    float s = 0.0f;
#pragma unroll
    for (int g = 0; g < G; ++g) s += shared_part[g * Ring::kCols + c];
    to[c] = s;
  }
}

// dweight[c] = sum over the blocks of their parts: eight threads a column take every eighth part, whose sums are added in a fixed order.
__global__ void __launch_bounds__(256) rmsnorm_dweight_kernel(const float* workspace, int parts, float* dweight, long long cols) {
  __shared__ float shared[8][32];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (long long c0 = blockIdx.x * 32ll; c0 < cols; c0 += gridDim.x * 32ll) {
    float s = 0.0f;
    if (c0 + lane < cols) {
#pragma unroll 8
      for (int k = warp; k < parts; k += 8) s += workspace[k * cols + c0 + lane];
    }
    shared[warp][lane] = s;
    __syncthreads();
    if (warp == 0 && c0 + lane < cols) {
#pragma unroll
      for (int w = 1; w < 8; ++w) s += shared[w][lane];
      dweight[c0 + lane] = s;
    }
    __syncthreads();
  }
}

}  // namespace sb200
