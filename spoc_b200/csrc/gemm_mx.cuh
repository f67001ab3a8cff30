// gemm_mx.cuh — products of microscaled matrices: D = act(alpha * A.B^T + beta * C + bias), A (M x K) and B (N x K) of 8 or 4 bits with a scale
// for every 32 values of a row (microscale.cuh), D, C and bias float32.
//
// The tensor core multiplies the codes and applies both scales while it adds to the float32 accumulator (tcgen05.mma block_scale): e4m3 and e2m1
// in any combination 32 values deep an instruction (kind::mxf8f6f4), e2m1 by e2m1 64 deep at twice the rate (kind::mxf4).  The rows of B, D's
// columns, are the instruction's M (128 a block) and the rows of A its N, so that a lane of the accumulator is a column of D: a warp's store
// of one row of D is 128 consecutive bytes at any alignment, and few rows of A make a narrow accumulator instead of idle lanes.
//
// Roles of a block: warp 0 loads codes and scale tiles with TMA into a ring of stages, warp 1 copies the scales of a stage into tensor memory
// (two slots in turn) and issues its MMAs, warps 2-5 run the epilogue.  CTAS = 2: a pair of blocks on one tile of 256 columns of D; each loads its
// own 128 rows of B, half of A's rows and all of A's scales.  A stage is 128 bytes of codes of every row: 128 values, 256 where both are e2m1;
// e2m1 beside e4m3 is spread to a byte a value on the way into shared memory (by TMA: 16 values a 16-byte unit).
#pragma once
#include "microscale.cuh"

namespace sb200 {

constexpr int MXG_THREADS = 192;
constexpr uint32_t MXG_W_BYTES = 128 * 128;   // a block's rows of B
constexpr int MXG_CTRL_BYTES = 1024;
constexpr int MXG_RING_BYTES = 216 * 1024;
constexpr int MXG_MAX_STAGES = 12;
constexpr int MXG_TMEM_COLS = 512;

struct MxGemm {
  float* D;
  const float *C, *bias;
  long long ldd, ldc;
  int M, N;
  float alpha, beta;
  int act;
  int chunks;         // Kp / 128
  int num_k_blocks;   // stages of a whole k-loop
  int bt;             // rows of A a tile: the MMA's N
  int tiles_f, tiles_t;
  int groups;         // tiles of 128 rows of A's scales that a tile touches
  int stages, stage_bytes, tx_bytes;
  int accs;           // accumulators: 2 where they fit beside the scales
  int splits, split_k_blocks;
  uint32_t idesc;
  int* status;
};

// ------------------------------------------------------------------- PTX
// Shared memory -> tensor memory, 32 lanes x 128 bits, the same into all four quarters of the lanes: a tile of scales.
template <int CTAS>
__device__ __forceinline__ void tmem_copy_scales(uint32_t taddr, uint64_t desc) {
  if constexpr (CTAS == 2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}
// A tile of scales in shared memory: 32 rows of 16 bytes, unswizzled, 8 rows (128 bytes) a core matrix.
__device__ __forceinline__ uint64_t scales_desc(uint32_t smem_addr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(1) << 16;
  d |= static_cast<uint64_t>(128 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  return d;
}
#define SB200_UMMA_MX(FORM)                                                                                                          \
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %6, 0;\ntcgen05.mma." FORM " [%0], %1, %2, %3, [%4], [%5], p;\n}\n" ::"r"(tmem_d),   \
               "l"(adesc), "l"(bdesc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)                                               \
               : "memory")
template <bool FP4, int CTAS>
__device__ __forceinline__ void umma_mx(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t sfa, uint32_t sfb,
                                        uint32_t accumulate) {
  if constexpr (FP4 && CTAS == 2) SB200_UMMA_MX("cta_group::2.kind::mxf4.block_scale.scale_vec::2X");
  else if constexpr (FP4) SB200_UMMA_MX("cta_group::1.kind::mxf4.block_scale.scale_vec::2X");
  else if constexpr (CTAS == 2) SB200_UMMA_MX("cta_group::2.kind::mxf8f6f4.block_scale.scale_vec::1X");
  else SB200_UMMA_MX("cta_group::1.kind::mxf8f6f4.block_scale.scale_vec::1X");
}
// Instruction descriptor of the block-scaled forms: B's scale id at bit 4, formats at 7 and 10, N >> 3 at 17, scales of type ue8m0 at 23, M >> 7
// at 27, A's scale id at 29.  Formats: mxf4: e2m1 1; mxf8f6f4: e4m3 0, e2m1 5.  The ids say which bytes of a 32-bit column hold the scales: a
// k-step's own byte (pair of bytes).
constexpr uint32_t umma_idesc_mx(uint32_t m, uint32_t n, uint32_t a_format, uint32_t b_format) {
  return (a_format << 7) | (b_format << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 7) << 27);
}
__device__ __forceinline__ uint32_t umma_scale_ids(uint32_t id) { return (id << 4) | (id << 29); }

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) { return __uint_as_float(ld_cluster_u32(addr)); }

__device__ __forceinline__ float mx_finish(const MxGemm& p, float sum, float c, float bias) {
  float x = __fmul_rn(p.alpha, sum);
  if (p.C) x = fmaf(p.beta, c, x);
  x = __fadd_rn(x, bias);
  return p.act == 1 && !(x > 0.0f) ? 0.0f : x;
}

// Tile `item`: bands of eight tiles of D's columns, so that the rows of B and A that the blocks work on stay in L2.
__device__ __forceinline__ void mx_tile(int item, const MxGemm& p, int& tf, int& tt) {
  constexpr int BAND = 8;
  const unsigned int band_tiles = BAND * p.tiles_t;
  const unsigned int band = static_cast<unsigned int>(item) / band_tiles, within = item - band * band_tiles;
  const unsigned int width = min(BAND, p.tiles_f - static_cast<int>(band) * BAND);
  tt = within / width;
  tf = band * BAND + within - tt * width;
}

// FP4: both operands e2m1.  map_w, map_x: codes of B and A; map_sw, map_sx: their scale tiles, 512 bytes a row.
// p.splits > 1 (single blocks only): the k-loop of a tile is divided among the blocks of a cluster, each of which leaves its partial sums in
// its ring; they are added in order of k, a share of A's rows a block.
template <bool FP4, int CTAS>
__global__ void __launch_bounds__(MXG_THREADS, 1)
gemm_mx_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_sw,
               const __grid_constant__ CUtensorMap map_sx, const MxGemm p) {
  constexpr int TILES = FP4 ? 2 : 1;          // scale tiles of 128 rows and a stage
  constexpr int K_STEP = FP4 ? 256 : 128;     // values of a stage (x coordinates of the code maps are bytes where FP4, values otherwise)
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + MXG_CTRL_BYTES;
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem);            // used in the leader only
  uint64_t* empty_bar = full_bar + MXG_MAX_STAGES;                   // one set per block
  uint64_t* tmem_full_bar = full_bar + 2 * MXG_MAX_STAGES;           // one set per block
  uint64_t* tmem_empty_bar = full_bar + 2 * MXG_MAX_STAGES + 2;      // used in the leader only
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(full_bar + 2 * MXG_MAX_STAGES + 4);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = blockIdx.x & (CTAS - 1u);
  const bool in_cluster = CTAS == 1 && p.splits > 1;
  const int split = in_cluster ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = in_cluster ? static_cast<int>(blockIdx.x) / p.splits : static_cast<int>(blockIdx.x) / CTAS;
  const int units = in_cluster ? 1 << 30 : static_cast<int>(gridDim.x) / CTAS;
  const int num_tiles = p.tiles_f * p.tiles_t;
  const int k0 = split * p.split_k_blocks, k_blocks = min(p.num_k_blocks - k0, p.split_k_blocks);

  if (warp == 0) {
    constexpr int BARS = 2 * MXG_MAX_STAGES + 4;
    if (lane < BARS) mbar_init(smem_u32(&full_bar[lane]), lane >= BARS - 2 ? 4 * CTAS : 1);
    if (lane == 0) *abort_flag = 0;
    mbar_fence_init();
  }
  if (threadIdx.x == 64) {
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_sw);
    tma_prefetch_desc(&map_sx);
  }
  if (warp == 1) {
    tmem_alloc_for<CTAS>(smem_u32(tmem_slot), MXG_TMEM_COLS);
    tmem_relinquish_for<CTAS>();
    tc_fence_before_sync();
  }
  __syncthreads();
  if (CTAS == 2) {
    cluster_arrive_relaxed();
    cluster_wait();
  }
  tc_fence_after_sync();
  const uint32_t tmem_base = *tmem_slot;
  grid_launch_dependents();
  grid_dependency_wait();

  bool ok = true;
  if (warp == 0) {
    // ------------------------------------------------------ TMA producer
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      const uint64_t pol = l2_policy(0);
      const int part_t = p.bt / CTAS;
      const uint32_t x_bytes = static_cast<uint32_t>(part_t) * 128;
      for (int item = unit; item < num_tiles && ok; item += units) {
        int tf, tt;
        mx_tile(item, p, tf, tt);
        const int f0 = (tf * CTAS + static_cast<int>(rank)) * 128, t0 = tt * p.bt;
        for (int it = 0; it < k_blocks; ++it) {
          const int kb = k0 + it;
          if (!mbar_wait_bounded(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag)) {
            atomicCAS(p.status, 0, 0x2100 | (rank << 4) | stage);
            ok = false;
            break;
          }
          if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full_bar[stage]), p.tx_bytes);
          const uint32_t bar = CTAS == 2 ? map_to_cta(smem_u32(&full_bar[stage]), 0) : smem_u32(&full_bar[stage]);
          const uint32_t sp = smem_u32(ring) + stage * p.stage_bytes, ss = sp + MXG_W_BYTES + x_bytes;
          const int x = FP4 ? kb * (K_STEP / 2) : kb * K_STEP;
          tma_load_for<CTAS>(sp, &map_w, bar, x, f0, pol);
          tma_load_for<CTAS>(sp + MXG_W_BYTES, &map_x, bar, x, t0 + static_cast<int>(rank) * part_t, pol);
          tma_load_for<CTAS>(ss, &map_sw, bar, 0, (f0 >> 7) * p.chunks + kb * TILES, pol);
          for (int g = 0; g < p.groups; ++g)
            tma_load_for<CTAS>(ss + (1 + g) * TILES * MX_TILE_BYTES, &map_sx, bar, 0, ((t0 >> 7) + g) * p.chunks + kb * TILES, pol);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) wait_for_copies();
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------- MMA issuer (leader block)
    if (rank == 0 && elect_one()) {
      int stage = 0, before = 0;          // before: the stage of two k-blocks ago
      uint32_t phase = 0, before_phase = 0;
      int n_tiles = 0;
      uint32_t count = 0;                 // k-blocks so far
      const uint32_t x_bytes = static_cast<uint32_t>(p.bt / CTAS) * 128;
      const int sf_cols = 4 * TILES * (1 + p.groups);   // of a slot
      const uint32_t sf_base = tmem_base + MXG_TMEM_COLS - 2 * sf_cols;
      for (int item = unit; item < num_tiles && ok; item += units, ++n_tiles) {
        const int acc = p.accs == 2 ? n_tiles & 1 : 0;
        const uint32_t acc_phase = (p.accs == 2 ? n_tiles >> 1 : n_tiles) & 1;
        int tf, tt;
        mx_tile(item, p, tf, tt);
        const uint32_t x_shift = (tt * p.bt & 127) >> 5;  // where the tile's first row lies in its first scale tile
        const uint32_t acc_free = smem_u32(&tmem_empty_bar[acc]);
        if (!(CTAS == 2 ? mbar_wait_cluster(acc_free, acc_phase ^ 1u, abort_flag) : mbar_wait_bounded(acc_free, acc_phase ^ 1u, abort_flag))) {
          atomicCAS(p.status, 0, 0x2200 | acc);
          ok = false;
          break;
        }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + acc * p.bt;
        for (int it = 0; it < k_blocks; ++it, ++count) {
          bool ready = mbar_wait_bounded(smem_u32(&full_bar[stage]), phase, abort_flag);
          if (ready && count >= 2) {
            // the scales' slot is free once the MMAs of two k-blocks ago have read it
            ready = mbar_wait_bounded(smem_u32(&empty_bar[before]), before_phase, abort_flag);
            if (++before == p.stages) {
              before = 0;
              before_phase ^= 1u;
            }
          }
          if (!ready) {
            atomicCAS(p.status, 0, 0x2300 | stage);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint32_t sw = smem_u32(ring) + stage * p.stage_bytes, sx = sw + MXG_W_BYTES, ss = sx + x_bytes;
          const uint32_t sfw = sf_base + (count & 1u) * sf_cols, sfx = sfw + 4 * TILES;
#pragma unroll
          for (int a = 0; a < TILES; ++a) {
            tmem_copy_scales<CTAS>(sfw + 4 * a, scales_desc(ss + a * MX_TILE_BYTES));
            for (int g = 0; g < p.groups; ++g)
              tmem_copy_scales<CTAS>(sfx + 4 * (a * p.groups + g), scales_desc(ss + ((1 + g) * TILES + a) * MX_TILE_BYTES));
          }
          const bool half = FP4 && 2 * (k0 + it) + 1 == p.chunks;  // the last 128 of an odd number of chunks
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if (FP4 && k == 2 && half) break;
            const int a = FP4 ? k / 2 : 0;
            const uint32_t id = FP4 ? (k & 1) * 2 : k;
            umma_mx<FP4, CTAS>(tmem_d, umma_desc_k_sw128(sw + k * 32), umma_desc_k_sw128(sx + k * 32), p.idesc | umma_scale_ids(id), sfw + 4 * a,
                               sfx + 4 * a * p.groups + x_shift, (it | k) ? 1u : 0u);
          }
          umma_commit_for<CTAS>(smem_u32(&empty_bar[stage]), 0);
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (ok) umma_commit_for<CTAS>(smem_u32(&tmem_full_bar[acc]), 0);
      }
    }
    __syncwarp();
  } else {
    // --------------------------------------------------------- epilogue
    const int quarter = warp & 3;
    int n_tiles = 0;
    for (int item = unit; item < num_tiles && ok; item += units, ++n_tiles) {
      const int acc = p.accs == 2 ? n_tiles & 1 : 0;
      const uint32_t acc_phase = (p.accs == 2 ? n_tiles >> 1 : n_tiles) & 1;
      int tf, tt;
      mx_tile(item, p, tf, tt);
      const int f = (tf * CTAS + static_cast<int>(rank)) * 128 + quarter * 32 + lane, t0 = tt * p.bt;
      const bool landed = mbar_wait_bounded(smem_u32(&tmem_full_bar[acc]), acc_phase, abort_flag);
      if (!__all_sync(0xffffffffu, landed)) {
        if (lane == 0) atomicCAS(p.status, 0, 0x2400 | (rank << 4) | acc);
        ok = false;
        break;
      }
      tc_fence_after_sync();
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * p.bt;
      const int rows = min(p.bt, p.M - t0);
      const float bias = p.bias && f < p.N ? p.bias[f] : 0.0f;
      float* part = reinterpret_cast<float*>(ring) + quarter * 32 + lane;  // in_cluster: row t at t * 128
      for (int c = 0; c < rows; c += 32) {
        uint32_t r[32];
        tmem_ld_32x32b_x32(taddr + c, r);
        tmem_ld_wait_x32(r);
        if (in_cluster) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < rows) part[(c + j) * 128] = __uint_as_float(r[j]);
        } else if (f < p.N) {
          float* d = p.D + static_cast<long long>(t0 + c) * p.ldd + f;
          if (p.C) {
            const float* cp = p.C + static_cast<long long>(t0 + c) * p.ldc + f;
            float cv[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) cv[j] = c + j < rows ? cp[j * p.ldc] : 0.0f;
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < rows) d[j * p.ldd] = mx_finish(p, __uint_as_float(r[j]), cv[j], bias);
          } else {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (c + j < rows) d[j * p.ldd] = mx_finish(p, __uint_as_float(r[j]), 0.0f, bias);
          }
        }
        __syncwarp();  // the next load takes the whole warp
      }
      tc_fence_before_sync();
      __syncwarp();
      if (lane == 0) {
        if (CTAS == 2)
          mbar_arrive_peer(map_to_cta(smem_u32(&tmem_empty_bar[acc]), 0));
        else
          mbar_arrive(smem_u32(&tmem_empty_bar[acc]));
      }
      if (in_cluster) break;
    }
    __syncwarp();
  }

  if (in_cluster) {
    // all partial sums are written before any is read; a block that gave up says so on its own status word, and D holds no result then
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    int tf, tt;
    mx_tile(unit, p, tf, tt);
    const int t0 = tt * p.bt, rows = min(p.bt, p.M - t0);
    const int first = rows * split / p.splits, last = rows * (split + 1) / p.splits;
    const uint32_t part = smem_u32(ring);
    for (int i = threadIdx.x; i < (last - first) * 128; i += MXG_THREADS) {
      const int t = first + i / 128, f = tf * 128 + i % 128;
      if (f >= p.N) continue;
      float s = ld_cluster_f32(map_to_cta(part + (t * 128 + i % 128) * 4, 0));
      for (int k = 1; k < p.splits; ++k) s += ld_cluster_f32(map_to_cta(part + (t * 128 + i % 128) * 4, k));
      const long long row = t0 + t;
      p.D[row * p.ldd + f] = mx_finish(p, s, p.C ? p.C[row * p.ldc + f] : 0.0f, p.bias ? p.bias[f] : 0.0f);
    }
  }

  // Neither block may retire, or free tensor memory, while another can still signal its barriers, read its shared memory or write its
  // accumulators.
  tc_fence_before_sync();
  __syncthreads();
  if (CTAS == 2 || in_cluster) {
    cluster_arrive_relaxed();
    cluster_wait();
  }
  if (warp == 1) {
    tc_fence_after_sync();
    tmem_dealloc_for<CTAS>(tmem_base, MXG_TMEM_COLS);
  }
}

// An empty sum: D = act(beta * C + bias).
__global__ void __launch_bounds__(256) gemm_mx_empty_kernel(const MxGemm p) {
  grid_launch_dependents();
  grid_dependency_wait();
  const long long total = static_cast<long long>(p.M) * p.N;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < total; i += gridDim.x * 256ll) {
    const long long row = i / p.N;
    const int col = static_cast<int>(i - row * p.N);
    p.D[row * p.ldd + col] = mx_finish(p, 0.0f, p.C ? p.C[row * p.ldc + col] : 0.0f, p.bias ? p.bias[col] : 0.0f);
  }
}

}  // namespace sb200
