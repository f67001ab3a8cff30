// gemm_mx.cuh — products of microscaled matrices: D = act(alpha * A.B^T + beta * C + bias), A (M x K) and B (N x K) of 8 or 4 bits with a scale
// for every 32 values of a row (microscale.cuh), D, C and bias float32.
//
// The tensor core multiplies the codes and applies both scales while it adds to the float32 accumulator (tcgen05.mma block_scale): e4m3 and e2m1
// in any combination 32 values deep an instruction (kind::mxf8f6f4), e2m1 by e2m1 64 deep at twice the rate (kind::mxf4).  The rows of B, D's
// columns, are the instruction's M (128 a block) and the rows of A its N, so that a lane of the accumulator is a column of D: a warp's store
// of one row of D is 128 consecutive bytes at any alignment, and few rows of A make a narrow accumulator instead of idle lanes.
//
// Roles of a block: warps 0, 10 and 11 load B's codes, A's codes and the scale tiles with TMA into a ring of stages (a load takes a thread 80 cycles,
// and a k-block of a narrow tile no more than its five loads: 16 x 2048 x 16384 in 8 bits took 27.2 us with one thread), warp 1 copies the scales of
// a stage into tensor memory (p.slots in turn) and issues its MMAs, warps 2-9 run the epilogue in two groups, which take every other 32 rows of A's tile.  Beside the scales
// there is not room for two accumulators of 256 columns: they overlap, the epilogue drains the columns in common first, and the next tile's MMAs
// begin when those are drained.  CTAS = 2: a pair of blocks on one tile of 256 columns of D; each loads its
// own 128 rows of B, half of A's rows and all of A's scales.  A stage is 128 bytes of codes of every row: 128 values, 256 where both are e2m1;
// e2m1 beside e4m3 is spread to a byte a value on the way into shared memory (by TMA: 16 values a 16-byte unit).
//
// Large products are bound by the tensor core's clock under the power cap and by the way from L2 (8192^3 alone: 4 bits 203 to 218 us, 5.0 to 5.4 PFLOP/s, and 244
// to 254 among seconds of such products; 8 bits 393 to 430, 2.6 to 2.8), products with few rows of A by B's bytes (16 x 16384 x 16384 in 8 bits
// 47.8 us, 5.8 TB/s) and small ones by latency (1 x 4096 x 4096 8 by 4 bits 5.8 us).
#pragma once
#include <type_traits>

#include "microscale.cuh"

namespace sb200 {

constexpr int MXG_THREADS = 384;
constexpr uint32_t MXG_W_BYTES = 128 * 128;   // a block's rows of B
constexpr int MXG_CTRL_BYTES = 1024;
constexpr int MXG_RING_BYTES = 216 * 1024;
constexpr int MXG_MAX_STAGES = 12;
constexpr int MXG_MAX_SPLITS = 8;   // blocks of a cluster
constexpr int MXG_TMEM_COLS = 512;       // all there are

struct MxGemm {
  float* D;
  const float *C, *bias;
  long long ldd, ldc;
  int M, N;
  float alpha, beta;
  int act;
  int chunks;         // Kp / 128
  int num_k_blocks;   // stages of a whole k-loop
  int bt;             // rows of A a tile: the MMA's N; a multiple of 128 unless one tile has them all (tiles start where tiles of scales do)
  int tiles_f, tiles_t;
  int stages, stage_bytes;
  int w_tail, x_tail;            // rows of the tail maps' boxes
  int w_row_bytes, x_row_bytes;  // what a barrier counts for a row of codes of B and A: 128, or 64 where TMA spreads 4 bits to 8
  int tmem_cols;      // a power of two that holds the accumulators and, at its end, the slots of scales
  int slots;          // as many as stages where they fit: a slot is then free when its stage was; otherwise its MMAs are waited for
  int acc1;           // first column of the second accumulator; below bt: the two overlap, by 64 columns at most
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

// 128-bit load from the shared memory of a block of the cluster (address from map_to_cta)
__device__ __forceinline__ float4 ld_cluster_v4(uint32_t cluster_addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(cluster_addr));
  return v;
}

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

// FP4: both operands e2m1.  map_w, map_x: codes of B and A; the tails: the same with boxes of the last, partial rows alone, for TMA takes up to 15 ns
// for every row past the end (1 x 4096 x 4096: 8.8 us with a box of 32 rows of A, 6.7 with 16); what no row was loaded for is not stored.
// map_sw, map_sx: the scale tiles, 512 bytes a row.
// IN_CLUSTER (single blocks only): the k-loop of a tile is divided among the p.splits blocks of a cluster, each of which leaves its partial
// sums in its ring; they are added in order of k, a share of A's rows a block.
template <bool FP4, int CTAS, int GROUPS, bool IN_CLUSTER>
__global__ void __launch_bounds__(MXG_THREADS, 1)
gemm_mx_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_w_tail,
               const __grid_constant__ CUtensorMap map_x_tail, const __grid_constant__ CUtensorMap map_sw, const __grid_constant__ CUtensorMap map_sx,
               const MxGemm p) {
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
  constexpr bool in_cluster = IN_CLUSTER;
  static_assert(!IN_CLUSTER || CTAS == 1, "single blocks divide their k-loop");
  const int split = in_cluster ? static_cast<int>(cluster_ctarank()) : 0;
  const int unit = in_cluster ? static_cast<int>(blockIdx.x) / p.splits : static_cast<int>(blockIdx.x) / CTAS;
  const int units = in_cluster ? 1 << 30 : static_cast<int>(gridDim.x) / CTAS;
  const int num_tiles = p.tiles_f * p.tiles_t;
  const int k0 = split * p.split_k_blocks, k_blocks = min(p.num_k_blocks - k0, p.split_k_blocks);

  if (warp == 0) {
    constexpr int BARS = 2 * MXG_MAX_STAGES + 4;
    if (lane < BARS) mbar_init(smem_u32(&full_bar[lane]), lane >= BARS - 2 ? 8 * CTAS : 1);
    if (lane == 0) *abort_flag = 0;
    mbar_fence_init();
  }
  if (threadIdx.x == 64) {
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
    tma_prefetch_desc(&map_w_tail);
    tma_prefetch_desc(&map_x_tail);
    tma_prefetch_desc(&map_sw);
    tma_prefetch_desc(&map_sx);
  }
  if (warp == 1) {
    tmem_alloc_for<CTAS>(smem_u32(tmem_slot), p.tmem_cols);
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
  if (warp == 0 || warp >= 10) {
    // ----------------------------------------------------- TMA producers
    auto produce = [&](auto role) {
      constexpr int ROLE = decltype(role)::value;
      int stage = 0;
      uint32_t phase = 0;
      const uint64_t pol = l2_policy(0);
      const int part_t = p.bt / CTAS;
      const uint32_t x_bytes = static_cast<uint32_t>(part_t) * 128;
      for (int item = unit; item < num_tiles && ok; item += units) {
        int tf, tt;
        mx_tile(item, p, tf, tt);
        const int f0 = (tf * CTAS + static_cast<int>(rank)) * 128, t0 = tt * p.bt, x0 = t0 + static_cast<int>(rank) * part_t;
        // The maps are chosen here, so that the loads are the same straight line for every tile: behind branches each takes 100 cycles more.  A block
        // of a pair that is past the end altogether asks for a tail box there, which is zeros.
        auto rows_in = [](int first, int box, int end, int tail) { return first + box <= end ? box : tail; };
        const CUtensorMap* const pw = rows_in(f0, 128, p.N, 0) ? &map_w : &map_w_tail;
        const CUtensorMap* const px = rows_in(x0, part_t, p.M, 0) ? &map_x : &map_x_tail;
        int tx_bytes = CTAS * TILES * MX_TILE_BYTES * (1 + GROUPS);  // of all blocks of the tile
        for (int r = 0; r < CTAS; ++r)
          tx_bytes += rows_in((tf * CTAS + r) * 128, 128, p.N, p.w_tail) * p.w_row_bytes + rows_in(t0 + r * part_t, part_t, p.M, p.x_tail) * p.x_row_bytes;
        for (int it = 0; it < k_blocks; ++it) {
          const int kb = k0 + it;
          if (!mbar_wait_bounded(smem_u32(&empty_bar[stage]), phase ^ 1u, abort_flag)) {
            atomicCAS(p.status, 0, 0x4100 | (rank << 4) | stage);
            ok = false;
            break;
          }
          const uint32_t bar = CTAS == 2 ? map_to_cta(smem_u32(&full_bar[stage]), 0) : smem_u32(&full_bar[stage]);
          const uint32_t sp = smem_u32(ring) + stage * p.stage_bytes, ss = sp + MXG_W_BYTES + x_bytes;
          const int x = FP4 ? kb * (K_STEP / 2) : kb * K_STEP;
          if constexpr (ROLE == 0) {
            // the leader counts the bytes of all loads of both blocks; until it has, its barrier's phase cannot end
            if (rank == 0) mbar_arrive_expect_tx(smem_u32(&full_bar[stage]), tx_bytes);
            tma_load_for<CTAS>(sp, pw, bar, x, f0, pol);
          } else if constexpr (ROLE == 1) {
            tma_load_for<CTAS>(sp + MXG_W_BYTES, px, bar, x, x0, pol);
          } else {
            tma_load_for<CTAS>(ss, &map_sw, bar, 0, (f0 >> 7) * p.chunks + kb * TILES, pol);
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
              tma_load_for<CTAS>(ss + (1 + g) * TILES * MX_TILE_BYTES, &map_sx, bar, 0, ((t0 >> 7) + g) * p.chunks + kb * TILES, pol);
          }
          if (++stage == p.stages) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (!ok) wait_for_copies();
    };
    if (elect_one()) {
      if (warp == 0)
        produce(std::integral_constant<int, 0>());
      else if (warp == 10)
        produce(std::integral_constant<int, 1>());
      else
        produce(std::integral_constant<int, 2>());
    }
    __syncwarp();
  } else if (warp == 1) {
    // ------------------------------------------- MMA issuer (leader block)
    if (rank == 0 && elect_one()) {
      int stage = 0, before = 0;          // before: the stage that had the slot last
      uint32_t phase = 0, before_phase = 0;
      int slot = 0;
      int n_tiles = 0;
      uint32_t count = 0;                 // k-blocks so far
      const uint32_t x_bytes = static_cast<uint32_t>(p.bt / CTAS) * 128;
      constexpr int sf_cols = 4 * TILES * (1 + GROUPS);   // of a slot
      const uint32_t stage0 = smem_u32(ring);
      const uint64_t w0 = umma_desc_k_sw128(stage0), x0 = umma_desc_k_sw128(stage0 + MXG_W_BYTES);
      const uint64_t s0 = scales_desc(stage0 + MXG_W_BYTES + x_bytes);
      const uint32_t sf_base = tmem_base + p.tmem_cols - p.slots * sf_cols;
      for (int item = unit; item < num_tiles && ok; item += units, ++n_tiles) {
        const int acc = n_tiles & 1;
        // where the accumulators overlap, the tile before has to have handed its columns back, otherwise the one before that
        const int behind = p.acc1 < p.bt ? 1 : 2;
        if (n_tiles >= behind) {
          const uint32_t free = smem_u32(&tmem_empty_bar[(n_tiles - behind) & 1]), phase_of = ((n_tiles - behind) >> 1) & 1;
          if (!(CTAS == 2 ? mbar_wait_cluster(free, phase_of, abort_flag) : mbar_wait_bounded(free, phase_of, abort_flag))) {
            atomicCAS(p.status, 0, 0x4200 | acc);
            ok = false;
            break;
          }
        }
        tc_fence_after_sync();
        const uint32_t tmem_d = tmem_base + acc * p.acc1;
        for (int it = 0; it < k_blocks; ++it, ++count) {
          bool ready = mbar_wait_bounded(smem_u32(&full_bar[stage]), phase, abort_flag);
          if (ready && p.slots < p.stages && count >= static_cast<uint32_t>(p.slots)) {
            ready = mbar_wait_bounded(smem_u32(&empty_bar[before]), before_phase, abort_flag);
            if (++before == p.stages) {
              before = 0;
              before_phase ^= 1u;
            }
          }
          if (!ready) {
            atomicCAS(p.status, 0, 0x4300 | stage);
            ok = false;
            break;
          }
          tc_fence_after_sync();
          const uint64_t at = static_cast<uint64_t>(static_cast<uint32_t>(stage * p.stage_bytes) >> 4);  // descriptors count in 16 bytes
          const uint32_t sfw = sf_base + slot * sf_cols, sfx = sfw + 4 * TILES;
          slot = slot + 1 == p.slots ? 0 : slot + 1;
#pragma unroll
          for (int a = 0; a < TILES; ++a) {
            tmem_copy_scales<CTAS>(sfw + 4 * a, s0 + at + a * (MX_TILE_BYTES / 16));
#pragma unroll
            for (int g = 0; g < GROUPS; ++g)
              tmem_copy_scales<CTAS>(sfx + 4 * (a * GROUPS + g), s0 + at + ((1 + g) * TILES + a) * (MX_TILE_BYTES / 16));
          }
          // FP4, the last 128 of an odd number of chunks: the codes beside them are zeros and take the same scales, for what was loaded as theirs is
          // another row's
          const uint32_t second = FP4 && 2 * (k0 + it) + 1 == p.chunks ? 0u : 1u;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t a = FP4 && k >= 2 ? second : 0u;
            const uint32_t id = FP4 ? (k & 1) * 2 : k;
            umma_mx<FP4, CTAS>(tmem_d, w0 + at + k * 2, x0 + at + k * 2, p.idesc | umma_scale_ids(id), sfw + 4 * a, sfx + 4 * GROUPS * a,
                               (it | k) ? 1u : 0u);
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
    const int quarter = warp & 3, group = warp >= 6 ? 1 : 0;
    int n_tiles = 0;
    for (int item = unit; item < num_tiles && ok; item += units, ++n_tiles) {
      const int acc = n_tiles & 1;
      const uint32_t acc_phase = (n_tiles >> 1) & 1;
      int tf, tt;
      mx_tile(item, p, tf, tt);
      const int f = (tf * CTAS + static_cast<int>(rank)) * 128 + quarter * 32 + lane, t0 = tt * p.bt;
      const int rows = min(p.bt, p.M - t0);
      // The first accumulator is drained from its end, the second from its start: what the two have in common comes first.  A group's chunks
      // are numbers group, group + 2, ... in that order.
      const int all = (p.bt + 31) >> 5;
      auto chunk_of = [&](int n) { return (acc == 0 ? all - 1 - n : n) * 32; };
      const bool inside = f < p.N;
      const float bias = p.bias && inside ? p.bias[f] : 0.0f;
      const float* c_col = p.C ? p.C + static_cast<long long>(t0) * p.ldc + f : nullptr;
      float* d_col = p.D + static_cast<long long>(t0) * p.ldd + f;
      float cv[32];
      auto load_c = [&](int c) {
        const float* cp = c_col + c * p.ldc;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
          cv[j] = inside && c + j < rows ? *cp : 0.0f;
          cp += p.ldc;
        }
      };
      if (!in_cluster && p.C) {
        if (group < all) load_c(chunk_of(group));
        // the lines of C that the chunks behind the first will read, into L2 under the k-loop: a lane a row
        const float* ahead = p.C + static_cast<long long>(t0 + lane) * p.ldc + (f - lane);
        if (f - lane < p.N) {
          for (int n = group + 2; n < all; n += 2) {
            const int c = chunk_of(n);
            if (c + lane < rows) {
              asm volatile("prefetch.global.L2 [%0];" ::"l"(ahead + c * p.ldc));
              if (f - lane + 31 < p.N) asm volatile("prefetch.global.L2 [%0];" ::"l"(ahead + c * p.ldc + 31));
            }
          }
        }
      }
      const bool landed = mbar_wait_bounded(smem_u32(&tmem_full_bar[acc]), acc_phase, abort_flag);
      if (!__all_sync(0xffffffffu, landed)) {
        if (lane == 0) atomicCAS(p.status, 0, 0x4400 | (rank << 4) | acc);
        ok = false;
        break;
      }
      tc_fence_after_sync();
      auto hand_back = [&] {
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) {
          if (CTAS == 2)
            mbar_arrive_peer(map_to_cta(smem_u32(&tmem_empty_bar[acc]), 0));
          else
            mbar_arrive(smem_u32(&tmem_empty_bar[acc]));
        }
      };
      const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + acc * p.acc1;
      float* part = reinterpret_cast<float*>(ring) + quarter * 32 + lane;  // in_cluster: row t at t * 128
      if (group >= all) hand_back();
      for (int n = group; n < all; n += 2) {
        const int c = chunk_of(n);
        const bool hand = p.acc1 < p.bt ? n == group : n + 2 >= all;
        if (c >= rows) {  // past the end of A
          if (hand) hand_back();
          if (!in_cluster && p.C && n + 2 < all) load_c(chunk_of(n + 2));
          continue;
        }
        uint32_t r[32];
        tmem_ld_32x32b_x32(taddr + c, r);
        tmem_ld_wait_x32(r);
        if (hand) hand_back();
        if constexpr (in_cluster) {
#pragma unroll
          for (int j = 0; j < 32; ++j)
            if (c + j < rows) part[(c + j) * 128] = __uint_as_float(r[j]);
        } else {
          float x[32];
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = mx_finish(p, __uint_as_float(r[j]), p.C ? cv[j] : 0.0f, bias);
          if (p.C && n + 2 < all) load_c(chunk_of(n + 2));
          if (inside) {
            float* d = d_col + c * p.ldd;
            if (c + 32 <= rows) {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                *d = x[j];
                d += p.ldd;
              }
            } else {
#pragma unroll
              for (int j = 0; j < 32; ++j) {
                if (c + j < rows) *d = x[j];
                d += p.ldd;
              }
            }
          }
        }
        __syncwarp();  // the next load takes the whole warp
      }
      if (in_cluster) break;
    }
    __syncwarp();
  }

  if constexpr (in_cluster) {
    // all partial sums are written before any is read; a block that gave up says so on its own status word, and D holds no result then
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    int tf, tt;
    mx_tile(unit, p, tf, tt);
    const int t0 = tt * p.bt, rows = min(p.bt, p.M - t0);
    const int first = rows * split / p.splits, last = rows * (split + 1) / p.splits;
    // a thread takes four columns of a row, from all blocks at once: the way to another block's memory is 0.3 us long
    const int f = tf * 128 + lane * 4;
    const uint32_t part = smem_u32(ring) + lane * 16;
    for (int t = first + warp; t < last; t += MXG_THREADS / 32) {
      float4 v[MXG_MAX_SPLITS];
#pragma unroll
      for (int k = 0; k < MXG_MAX_SPLITS; ++k)
        if (k < p.splits) v[k] = ld_cluster_v4(map_to_cta(part + t * 512, k));
      float sum[4] = {v[0].x, v[0].y, v[0].z, v[0].w};
#pragma unroll
      for (int k = 1; k < MXG_MAX_SPLITS; ++k) {
        if (k >= p.splits) break;
        sum[0] += v[k].x;
        sum[1] += v[k].y;
        sum[2] += v[k].z;
        sum[3] += v[k].w;
      }
      const long long row = t0 + t;
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (f + j < p.N)
          p.D[row * p.ldd + f + j] = mx_finish(p, sum[j], p.C ? p.C[row * p.ldc + f + j] : 0.0f, p.bias ? p.bias[f + j] : 0.0f);
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
    tmem_dealloc_for<CTAS>(tmem_base, p.tmem_cols);
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
