// Lists how products of microscaled matrices are run: for every "fp4 M N K" on the standard input the plan on `sm_count` SMs (first argument),
// and the candidates that it was chosen from.
#include <stdio.h>
#include <stdlib.h>

#include "gemm_mx_plan.hpp"

int main(int, char** argv) {
  const int sm_count = atoi(argv[1]);
  int fp4;
  long long M, N, K;
  while (scanf("%d %lld %lld %lld", &fp4, &M, &N, &K) == 4) {
    const sb200::MxPlan p = sb200::plan_gemm_mx(fp4 != 0, M, N, K, sm_count);
    printf("ctas=%d bt=%d splits=%d tiles=%lld chunks=%d num_k_blocks=%d split_k_blocks=%d groups=%d stages=%d stage_bytes=%d slots=%d tmem_cols=%d acc1=%d candidates=",
           p.ctas, p.bt, p.splits, static_cast<long long>(p.tiles), p.chunks, p.num_k_blocks, p.split_k_blocks, p.groups, p.stages, p.stage_bytes, p.slots,
           p.tmem_cols, p.acc1);
    sb200::mx_candidates(M, p.num_k_blocks, [](const sb200::MxShape& s) { printf("%d:%d:%d,", s.ctas, s.bt, s.splits); });
    printf("\n");
  }
}
