// rmsnorm.cuh — root-mean-square norm with the residual's addition, its result in float32 or microscaled, and its gradient.
//
//   h = x + residual (rounded to float32: it is stored, and the next layer adds to it),  y = h * weight / sqrt(mean(h^2) + eps)
//
// y is computed in 64 bits from the h that is stored and rounded once.  A code of 8 or 4 bits is then the rounding of the exact y: next to a rounding
// border 32 bits would fall on one side or the other depending on the order of the sum, one value in a million by a whole step, and so
// would all that is computed from it.
//
// One block a row, the row in registers (VECS float4 a thread; thread t has columns 4 (v * threads + t)), so that x and residual are read
// once.  Rows too long for that (32768 columns on) are read twice.  Bound by HBM: 8 bytes read, 5 written a value with 8-bit codes.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "microscale.cuh"

namespace sb200 {

struct RmsNorm {
  const float *x, *residual, *weight;  // residual may be null
  long long ldx, ldr, ldh, ldy;
  float *h, *y;                        // either may be null
  uint8_t *codes, *scales;             // null: no microscaled result
  long long rows, cols, chunks;
  double eps;
};

// Sum over the block of a value a thread, the same in all threads and in every launch.
template <int THREADS, class T>
__device__ __forceinline__ T block_sum(T v, T* shared) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if (THREADS == 32) return v;
  if ((threadIdx.x & 31) == 0) shared[threadIdx.x >> 5] = v;
  __syncthreads();
  T s = 0;
#pragma unroll
  for (int w = 0; w < THREADS / 32; ++w) s += shared[w];
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

__device__ __forceinline__ double normed(float h, float w, double scale) { return static_cast<double>(h) * scale * static_cast<double>(w); }

// What is done with four values of the normed row.  FORMAT: 0 float32 only, 4, 8.
template <int FORMAT, bool VEC>
__device__ __forceinline__ void rmsnorm_emit(const RmsNorm& p, long long row, long long col, const float4& h, double scale, int lane) {
  float4 w = make_float4(0.f, 0.f, 0.f, 0.f);
  if (col < p.cols) w = load4<VEC>(p.weight, col, p.cols);
  const double y[4] = {normed(h.x, w.x, scale), normed(h.y, w.y, scale), normed(h.z, w.z, scale), normed(h.w, w.w, scale)};
  if (p.y)
    store4<VEC>(p.y + row * p.ldy, col, p.cols,
                make_float4(static_cast<float>(y[0]), static_cast<float>(y[1]), static_cast<float>(y[2]), static_cast<float>(y[3])));
  if constexpr (FORMAT != 0) {
    constexpr bool FP4 = FORMAT == 4;
    const long long chunk = col / MX_CHUNK;  // the same in a whole warp
    if (chunk < p.chunks)
      mx_store_chunk<FP4>(make_float4(round_to_odd(y[0]), round_to_odd(y[1]), round_to_odd(y[2]), round_to_odd(y[3])),
                          p.codes + (row * p.chunks + chunk) * MxFormat<FP4>::kChunkBytes, p.scales + mx_scale_offset(row, chunk, p.chunks), lane);
  }
}
__device__ __forceinline__ double squares(const float4& h) {
  return fma(static_cast<double>(h.x), static_cast<double>(h.x), static_cast<double>(h.y) * h.y) +
         fma(static_cast<double>(h.z), static_cast<double>(h.z), static_cast<double>(h.w) * h.w);
}
template <bool VEC>
__device__ __forceinline__ float4 rmsnorm_input(const RmsNorm& p, long long row, long long col) {
  float4 h = load4<VEC>(p.x + row * p.ldx, col, p.cols);
  if (p.residual) {
    const float4 r = load4<VEC>(p.residual + row * p.ldr, col, p.cols);
    h = make_float4(__fadd_rn(h.x, r.x), __fadd_rn(h.y, r.y), __fadd_rn(h.z, r.z), __fadd_rn(h.w, r.w));
  }
  return h;
}
// VECS = 0: rows of any length, read twice (h may be x or residual itself: then the second reading takes h, which was stored).
template <int FORMAT, int THREADS, int VECS, bool VEC>
__global__ void __launch_bounds__(THREADS) rmsnorm_kernel(const RmsNorm p) {
  __shared__ double shared[2][THREADS / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const int lane = threadIdx.x & 31;
  const long long rows = FORMAT ? (p.rows + 127) / 128 * 128 : p.rows;
  int turn = 0;
  for (long long row = blockIdx.x; row < rows; row += gridDim.x, turn ^= 1) {
    if (FORMAT && row >= p.rows) {  // the scales' padding
      for (long long c = threadIdx.x; c < p.chunks; c += THREADS) *reinterpret_cast<uint32_t*>(p.scales + mx_scale_offset(row, c, p.chunks)) = 0u;
      continue;
    }
    if constexpr (VECS > 0) {
      float4 h[VECS];
#pragma unroll
      for (int v = 0; v < VECS; ++v) h[v] = rmsnorm_input<VEC>(p, row, 4ll * (v * THREADS + threadIdx.x));
      double s = 0.0;
#pragma unroll
      for (int v = 0; v < VECS; ++v) s += squares(h[v]);
      if (p.h) {
#pragma unroll
        for (int v = 0; v < VECS; ++v) store4<VEC>(p.h + row * p.ldh, 4ll * (v * THREADS + threadIdx.x), p.cols, h[v]);
      }
      const double scale = 1.0 / sqrt(block_sum<THREADS>(s, shared[turn]) / static_cast<double>(p.cols) + p.eps);
#pragma unroll
      for (int v = 0; v < VECS; ++v) rmsnorm_emit<FORMAT, VEC>(p, row, 4ll * (v * THREADS + threadIdx.x), h[v], scale, lane);
    } else {
      const long long padded = (p.cols + MX_CHUNK - 1) / MX_CHUNK * MX_CHUNK;
      double s = 0.0;
      for (long long col = 4ll * threadIdx.x; col < p.cols; col += 4 * THREADS) {
        const float4 h = rmsnorm_input<VEC>(p, row, col);
        s += squares(h);
        if (p.h) store4<VEC>(p.h + row * p.ldh, col, p.cols, h);
      }
      const double scale = 1.0 / sqrt(block_sum<THREADS>(s, shared[turn]) / static_cast<double>(p.cols) + p.eps);
      for (long long col = 4ll * threadIdx.x; col < padded; col += 4 * THREADS) {
        float4 h;
        if (p.h) {  // this thread's own stores; not through the read-only path
          const float* src = p.h + row * p.ldh;
          h = make_float4(col < p.cols ? src[col] : 0.f, col + 1 < p.cols ? src[col + 1] : 0.f, col + 2 < p.cols ? src[col + 2] : 0.f,
                          col + 3 < p.cols ? src[col + 3] : 0.f);
        } else {
          h = rmsnorm_input<VEC>(p, row, col);
        }
        rmsnorm_emit<FORMAT, VEC>(p, row, col, h, scale, lane);
      }
    }
  }
}

// The gradient: with r = 1 / sqrt(mean(h^2) + eps), n = h r and g = dy * weight,
//   dx = dsum + r (g - n mean(g n)),   dweight = sum over the rows of dy n.
// A block takes rows blockIdx.x, + gridDim.x, ... and keeps its part of dweight in registers (VECS = 0: in its row of the workspace); a second
// kernel adds the parts in the order of the blocks.  h and dy are read once.  Bound by HBM: 12 bytes read and 4 written a value.
struct RmsNormBackward {
  const float *h, *weight, *dy, *dsum;  // dsum may be null
  long long ldh, lddy, ldds, lddx;
  float *dx, *dweight, *workspace;      // either of dx and dweight may be null
  long long rows, cols;
  double eps;
};
template <int THREADS, int VECS, bool VEC>
__global__ void __launch_bounds__(THREADS) rmsnorm_backward_kernel(const RmsNormBackward p) {
  __shared__ float2 shared[2][THREADS / 32];
  grid_launch_dependents();
  grid_dependency_wait();
  const float inv_cols = 1.0f / static_cast<float>(p.cols), eps = static_cast<float>(p.eps);
  constexpr int HELD = VECS > 0 ? VECS : 1;
  float4 part[HELD];
#pragma unroll
  for (int v = 0; v < HELD; ++v) part[v] = make_float4(0.f, 0.f, 0.f, 0.f);
  float* const mine = p.workspace + blockIdx.x * p.cols;
  int turn = 0;
  for (long long row = blockIdx.x; row < p.rows; row += gridDim.x, turn ^= 1) {
    const float *hr = p.h + row * p.ldh, *dyr = p.dy + row * p.lddy;
    float4 h[HELD], dy[HELD];
    float2 s = make_float2(0.f, 0.f);  // of h^2 and of h * g
    auto count = [&](const float4& a, const float4& d, const float4& w) {
      s.x += fmaf(a.x, a.x, a.y * a.y) + fmaf(a.z, a.z, a.w * a.w);
      s.y += fmaf(a.x, d.x * w.x, a.y * (d.y * w.y)) + fmaf(a.z, d.z * w.z, a.w * (d.w * w.w));
    };
    if constexpr (VECS > 0) {
#pragma unroll
      for (int v = 0; v < VECS; ++v) {
        h[v] = load4<VEC>(hr, 4ll * (v * THREADS + threadIdx.x), p.cols);
        dy[v] = load4<VEC>(dyr, 4ll * (v * THREADS + threadIdx.x), p.cols);
      }
#pragma unroll
      for (int v = 0; v < VECS; ++v) count(h[v], dy[v], load4<VEC>(p.weight, 4ll * (v * THREADS + threadIdx.x), p.cols));
    } else {
      for (long long col = 4ll * threadIdx.x; col < p.cols; col += 4 * THREADS)
        count(load4<VEC>(hr, col, p.cols), load4<VEC>(dyr, col, p.cols), load4<VEC>(p.weight, col, p.cols));
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      s.x += __shfl_xor_sync(0xffffffffu, s.x, o);
      s.y += __shfl_xor_sync(0xffffffffu, s.y, o);
    }
    if ((threadIdx.x & 31) == 0) shared[turn][threadIdx.x >> 5] = s;
    __syncthreads();
    s = make_float2(0.f, 0.f);
#pragma unroll
    for (int w = 0; w < THREADS / 32; ++w) {
      s.x += shared[turn][w].x;
      s.y += shared[turn][w].y;
    }
    const float r = 1.0f / sqrtf(s.x * inv_cols + eps);
    const float along = s.y * inv_cols * r * r;  // mean(g n) r: what h is multiplied by
    auto finish = [&](long long col, const float4& a, const float4& d, float4& w_part) {
      if (p.dx) {
        const float4 w = load4<VEC>(p.weight, col, p.cols);
        float4 o = make_float4(r * fmaf(-a.x, along, d.x * w.x), r * fmaf(-a.y, along, d.y * w.y), r * fmaf(-a.z, along, d.z * w.z),
                               r * fmaf(-a.w, along, d.w * w.w));
        if (p.dsum) {
          const float4 t = load4<VEC>(p.dsum + row * p.ldds, col, p.cols);
          o = make_float4(o.x + t.x, o.y + t.y, o.z + t.z, o.w + t.w);
        }
        store4<VEC>(p.dx + row * p.lddx, col, p.cols, o);
      }
      w_part.x = fmaf(d.x, a.x * r, w_part.x);
      w_part.y = fmaf(d.y, a.y * r, w_part.y);
      w_part.z = fmaf(d.z, a.z * r, w_part.z);
      w_part.w = fmaf(d.w, a.w * r, w_part.w);
    };
    if constexpr (VECS > 0) {
#pragma unroll
      for (int v = 0; v < VECS; ++v) finish(4ll * (v * THREADS + threadIdx.x), h[v], dy[v], part[v]);
    } else {
      for (long long col = 4ll * threadIdx.x; col < p.cols; col += 4 * THREADS) {
        float4 w_part = make_float4(0.f, 0.f, 0.f, 0.f);
        if (p.dweight && row != blockIdx.x)
          w_part = make_float4(mine[col], col + 1 < p.cols ? mine[col + 1] : 0.f, col + 2 < p.cols ? mine[col + 2] : 0.f,
                               col + 3 < p.cols ? mine[col + 3] : 0.f);
        const float4 a = load4<VEC>(hr, col, p.cols), d = load4<VEC>(dyr, col, p.cols);
        finish(col, a, d, w_part);
        if (p.dweight) store4<false>(mine, col, p.cols, w_part);
      }
    }
  }
  if constexpr (VECS > 0) {
    if (p.dweight) {
#pragma unroll
      for (int v = 0; v < VECS; ++v) store4<false>(mine, 4ll * (v * THREADS + threadIdx.x), p.cols, part[v]);
    }
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
