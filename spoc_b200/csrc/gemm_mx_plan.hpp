// gemm_mx_plan.hpp — how a product of microscaled matrices is run (gemm_mx.cuh): tiles, k-loops, stages, tensor memory.  Host code without a call to a
// device, so that the forms that sizes take can be listed anywhere.
#pragma once
#include <stdint.h>

#include <algorithm>

#include "gemm_mx.cuh"
#include "internal.hpp"

namespace sb200 {

// Tiles: 128 (256: pairs) columns of D by bt rows.
struct MxShape {
  int ctas = 1, bt = 128, splits = 1;
};
inline int64_t mx_tiles(const MxShape& s, int64_t M, int64_t N) { return (N + 128 * s.ctas - 1) / (128 * s.ctas) * ((M + s.bt - 1) / s.bt); }

// The shape with the least estimated time.  Measured on one B200, operands from L2 and HBM, in us: a launch with one k-block 3.3; a k-block 0.165 and
// 0.4 ns a row of A in a block's tile (4 loads, 4 MMAs and a round of barriers, whatever the width up to 64 rows), half as much again where all
// SMs load at once (128 x 2048 x 16384 0.21, 2048 x 4096 x 4096 0.29); in pairs 0.22 to 0.28 for 128 rows and 0.31 to 0.42 for 256; the last
// epilogue 6 ns a row; a k-loop divided within a cluster 1.1 and 30 ns for every row a block sends (1 x 4096 x 4096 8.6 -> 5.7 us in four,
// 64 x 4096 x 4096 9.3 -> 7.3).
template <class Consider>
void mx_candidates(int64_t M, int64_t k_blocks, Consider consider) {
  const int narrow = M <= 16 ? 16 : M <= 32 ? 32 : M <= 64 ? 64 : 128;
  for (int splits = 1; splits <= MXG_MAX_SPLITS; ++splits)
    if (k_blocks >= 2 * splits || splits == 1) consider(MxShape{1, narrow, splits});
  if (M > 64) consider(MxShape{2, 128, 1});  // of 64 rows a k-block costs no less in a pair than in a block
  if (M > 128) consider(MxShape{2, 256, 1});
}
inline MxShape choose_mx_shape(int64_t M, int64_t N, int64_t k_blocks, int sm_count) {
  MxShape best;
  double best_us = 0.0;
  mx_candidates(M, k_blocks, [&](const MxShape& s) {
    const int ctas = s.ctas, bt = s.bt, splits = s.splits;
    const int64_t tiles = mx_tiles(s, M, N), units = std::max(1, sm_count / ctas);
    if (splits > 1 && tiles > cluster_capacity(splits, sm_count)) return;  // all clusters at once
    const int64_t per_item = (k_blocks + splits - 1) / splits, waves = splits > 1 ? 1 : (tiles + units - 1) / units;
    const double busy = std::min(1.0, static_cast<double>(tiles) * splits / units);
    const double k_block = ctas == 1 ? (0.165 + 0.0004 * bt) * (bt == 128 ? 1.0 + 0.4 * busy : 1.0) : bt == 256 ? 0.31 + 0.11 * busy : 0.19 + 0.0003 * bt + 0.06 * busy;
    double us = 3.3 + static_cast<double>(waves * per_item) * k_block + 0.006 * bt + 0.5 * static_cast<double>(waves - 1);
    if (splits > 1) us += 1.1 + 0.03 * bt * (splits - 1) / splits;
    if (best_us == 0.0 || us < 0.97 * best_us) {
      best = s;
      best_us = us;
    }
  });
  return best;
}

struct MxPlan : MxShape {
  int64_t tiles;
  int chunks, num_k_blocks, split_k_blocks;
  int groups;  // tiles of 128 rows of A's scales that a tile touches
  int stages, stage_bytes, slots, tmem_cols, acc1;
};
inline MxPlan plan_gemm_mx(bool fp4, int64_t M, int64_t N, int64_t K, int sm_count) {
  MxPlan p;
  p.chunks = static_cast<int>((K + MX_CHUNK - 1) / MX_CHUNK);
  p.num_k_blocks = fp4 ? (p.chunks + 1) / 2 : p.chunks;
  static_cast<MxShape&>(p) = choose_mx_shape(M, N, p.num_k_blocks, sm_count);
  p.tiles = mx_tiles(p, M, N);
  p.groups = p.bt > 128 ? 2 : 1;
  p.split_k_blocks = (p.num_k_blocks + p.splits - 1) / p.splits;
  p.splits = (p.num_k_blocks + p.split_k_blocks - 1) / p.split_k_blocks;  // the last one has something to do
  const int scale_tiles = fp4 ? 2 : 1;
  const int x_bytes = p.bt / p.ctas * 128, sf_bytes = scale_tiles * MX_TILE_BYTES * (1 + p.groups);
  p.stage_bytes = (static_cast<int>(MXG_W_BYTES) + x_bytes + sf_bytes + 1023) / 1024 * 1024;
  p.stages = std::min(MXG_MAX_STAGES, MXG_RING_BYTES / p.stage_bytes);
  const int sf_cols = 4 * scale_tiles * (1 + p.groups);
  if (p.tiles <= sm_count / p.ctas || p.splits > 1) {
    // A tile a block: no more stages than k-blocks, one accumulator, and no more tensor memory than that takes, so that the blocks of the
    // launch behind this one can set themselves up beside these.
    p.stages = std::max(1, std::min(p.stages, p.split_k_blocks));
    const int held = std::max(32, p.bt);
    p.slots = std::min(p.stages, (MXG_TMEM_COLS - held) / sf_cols);
    p.tmem_cols = 32;
    while (p.tmem_cols < held + p.slots * sf_cols) p.tmem_cols *= 2;
    p.acc1 = p.bt;
  } else {
    // two accumulators, which overlap by 64 columns at most
    p.slots = std::min(p.stages, (MXG_TMEM_COLS - 2 * p.bt + (p.bt == 256 ? 64 : 0)) / sf_cols);
    p.tmem_cols = MXG_TMEM_COLS;
    p.acc1 = std::min(256, MXG_TMEM_COLS - p.slots * sf_cols - p.bt);
  }
  return p;
}

}  // namespace sb200
