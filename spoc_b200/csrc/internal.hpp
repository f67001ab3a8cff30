// internal.hpp — what the library's translation units share besides the public C ABI.
#pragma once
#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>
#include <string.h>

#include <utility>

#include "../../include/sb200.h"

namespace sb200 {

// Records a failure for sb200_last_error_string() on the calling thread and returns `code`.
int set_error(int code, const char* fmt, ...) __attribute__((format(printf, 2, 3)));

// A failed CUDA call, as a status.
int set_cuda_error(cudaError_t e, const char* what);

// The kernel that a wait's number in the status word is from: the numbers of each begin with a digit of its own.
inline const char* waiting_kernel(int site) {
  switch (site >> 12) {
    case 0: return "wait_timeout_probe_kernel";
    case 1: return "gemm_pair_kernel";
    case 2: return "gemm_convert_kernel";
    case 3: return "gemm_split_kernel";
    case 4: return "gemm_mx_kernel";
    case 5: return "rmsnorm_backward_ring_kernel";
    default: return "a kernel";
  }
}

// What an operator outside sb200_shim.cu needs of a device.
struct OperatorDevice {
  int index, sm_count;
  int* status;  // device word for kernels whose bounded waits expire; operator_waits() before such a launch
};
int operator_device(int dev, OperatorDevice* out);  // makes it the calling thread's current device
void operator_waits(int dev);                       // a synchronise has the status word to read from now on
int operator_extent(int dev, uint64_t ptr, uint64_t bytes, const char* what);  // SB200_ERR_BOUNDS past the end of a buffer of the library
int operator_launched(const char* what);            // counts a launch, or reports that it failed
int encode_tensor_map_2d(CUtensorMap* map, CUtensorMapDataType type, const void* base, uint64_t inner, uint64_t rows, uint64_t row_bytes,
                         uint32_t box_inner, uint32_t box_rows, CUtensorMapSwizzle swizzle);

// Launches a kernel with programmatic stream serialization: it may set itself up while the kernel before it in the stream
// still runs.  Every kernel launched this way passes griddepcontrol.wait before it touches global memory.  The launch call
// itself is cheaper too (2.3 against 2.8 us).  shared_percent: the share of an SM's L1 that should be shared memory, -1 as the driver sees fit.
template <class... Params, class... Args>
cudaError_t launch_pdl_sharing(int shared_percent, void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, Args&&... args) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof cfg);
  cfg.gridDim = grid;
  cfg.blockDim = block;
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cudaLaunchAttribute attr[3];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.numAttrs = 1;
  if (cluster > 1) {
    cudaLaunchAttribute& a = attr[cfg.numAttrs++];
    a.id = cudaLaunchAttributeClusterDimension;
    a.val.clusterDim.x = static_cast<unsigned>(cluster);
    a.val.clusterDim.y = 1;
    a.val.clusterDim.z = 1;
  }
  if (shared_percent >= 0) {
    cudaLaunchAttribute& a = attr[cfg.numAttrs++];
    a.id = cudaLaunchAttributePreferredSharedMemoryCarveout;
    a.val.sharedMemCarveout = static_cast<unsigned>(shared_percent);
  }
  cfg.attrs = attr;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}
template <class... Params, class... Args>
cudaError_t launch_pdl(void (*kernel)(Params...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, int cluster, Args&&... args) {
  return launch_pdl_sharing(-1, kernel, grid, block, smem, st, cluster, std::forward<Args>(args)...);
}

// Clusters of `blocks` (at most 8) blocks that are resident at once when every block has an SM to itself.  A cluster lies within a
// GPC, whose SMs it may not divide evenly: the runtime counts 148, 74, 45, 33, 26, 22, 15 and 15 on a 148-SM B200.  One less from
// three blocks on, because chips differ in the SMs that are switched off and one cluster too many is a second wave.
inline long long cluster_capacity(int blocks, int sm_count) {
  static const int resident[9] = {0, 148, 74, 44, 32, 25, 21, 14, 14};
  return static_cast<long long>(resident[blocks]) * sm_count / 148;
}
// The numeric modes every GEMM entry point takes.
inline bool valid_mode(int mode) {
  return mode == SB200_MODE_3XTF32 || mode == SB200_MODE_TF32 || mode == SB200_MODE_3XF16 || mode == SB200_MODE_F16 ||
         mode == SB200_MODE_3XMIXED;
}

// While one of these lives, the products its thread launches are parts (rows, columns or both) of one of `rows` rows and `cols`
// columns: a k-loop is then divided, or not, as it would be for the whole, and the parts have the bits of the whole.
class PartsOf {
 public:
  PartsOf(long long rows, long long cols);
  ~PartsOf();
  PartsOf(const PartsOf&) = delete;
  PartsOf& operator=(const PartsOf&) = delete;

 private:
  long long rows_before_, cols_before_;
};

}  // namespace sb200
