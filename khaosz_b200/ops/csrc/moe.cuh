// Passes of moe.cu that gemm_grouped.cu runs around its products.
#pragma once
#include <cuda_runtime.h>

namespace kb {
namespace moe {

// The kernels of a pass follow one another with programmatic launch: a kernel may start while its predecessor
// still drains and waits here for the predecessor's results, before it touches memory that others write.  The
// successor is let in behind that wait, so a kernel that runs knows that everything before its direct
// predecessor has completed.
__device__ __forceinline__ void await_predecessor() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}
template <int CLUSTER = 1, typename... KArgs, typename... Args>
cudaError_t launch_after(void (*kernel)(KArgs...), dim3 grid, int threads, size_t smem, cudaStream_t st, Args&&... args) {
  cudaLaunchAttribute attr[2] = {};
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CLUSTER;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = CLUSTER > 1 ? 2 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, static_cast<KArgs>(args)...);
}

// dst[r] = src[rows[r] / k] for the first offsets[E] rows (zero where rows[r] < 0); rw[r]: the row's routing weight (may be
// null); order (may be null): the experts by falling number of rows.
int launch_gather(const void* src, long ld, const int* rows, const int* offsets, int E, int* order, const void* w, int w_f32, float* rw, void* dst, int k, int D, int R, int sms,
                  cudaStream_t st);
// out[t] = res[t] + sum_j y[slots[t][j]] (out may be null); dw[t][j] = sum_i part[slots[t][j]][i] (dw may be null).
int launch_combine(const void* y, const int* slots, const void* res, long ldr, void* out, const float* part, int n_part, void* dw, int w_f32, int T, int k,
                   int D, cudaStream_t st);

}  // namespace moe
}  // namespace kb
