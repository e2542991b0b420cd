// Passes of moe.cu that gemm_grouped.cu runs around its products.
#pragma once
#include <cuda_runtime.h>

namespace kb {
namespace moe {

// dst[r] = src[rows[r] / k] for the first *end rows (zero where rows[r] < 0); rw[r]: the row's routing weight.
int launch_gather(const void* src, long ld, const int* rows, const int* end, const void* w, int w_f32, float* rw, void* dst, int k, int D, int R, int sms,
                  cudaStream_t st);
// out[t] = res[t] + sum_j y[slots[t][j]] (out may be null); dw[t][j] = sum_i part[slots[t][j]][i] (dw may be null).
int launch_combine(const void* y, const int* slots, const void* res, long ldr, void* out, const float* part, int n_part, void* dw, int w_f32, int T, int k,
                   int D, cudaStream_t st);

}  // namespace moe
}  // namespace kb
