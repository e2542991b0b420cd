// The experts' products of a few assignments (decoding a handful of sequences), forward only.
//
// Bound by the chosen experts' weights, which pass through once: two kernels of CUDA-core dot products, one warp
// per weight row, without grouping, gather or combine passes.  In the first a warp keeps its pieces of a gate and
// an up row in registers for all tokens of that expert; the hidden activations stay in fp32.  In the second a
// block's warps share an output feature over the token's experts and add in a fixed order.
#include "common.cuh"
#include "kb_api.h"
#include "moe.cuh"

namespace kb {
namespace moe_small {

constexpr unsigned FULL = 0xffffffffu;
constexpr int WARPS = 8;
constexpr int PIECES = 4;   // 16-byte pieces of each row that a lane has in flight
constexpr int ROWS = 2;     // rows of the down projection that a warp takes, so that h is read half as often

struct Params {
  const __nv_bfloat16 *x, *wg, *wu, *wd, *res;
  const void *w, *ids;
  __nv_bfloat16* out;
  float* h;  // [n, F]
  long ldx, ldg, sg, ldu, su, ldd, sd, ldr;
  int w_f32, ids64, T, k, D, F, E;
};

__device__ __forceinline__ int expert_of(const Params& p, int a) {
  const long long e = p.ids64 ? static_cast<const long long*>(p.ids)[a] : (long long)static_cast<const int*>(p.ids)[a];
  return e < 0 || e >= p.E ? -1 : (int)e;
}
__device__ __forceinline__ float dot8(const uint4& a, const uint4& b, float s) {
  const uint32_t u[4] = {a.x, a.y, a.z, a.w}, v[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = unpack_bf16x2(u[i]), g = unpack_bf16x2(v[i]);
    s = fmaf(f.x, g.x, s);
    s = fmaf(f.y, g.y, s);
  }
  return s;
}
__device__ __forceinline__ uint4 stream_load(const uint4* p) {  // weights are read once: they need not stay in L1
  uint4 v;
  asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}

// h[a][f] = w[a] * silu(x[t] . gate[e][f]) * (x[t] . up[e][f]); the first assignment of an expert does them all,
// MEMBERS tokens in one pass over its rows (1 for a single token: half the registers, twice the warps in flight).
template <int MEMBERS>
__global__ void __launch_bounds__(WARPS * 32) up_kernel(const Params p) {
  const int lane = threadIdx.x & 31, n = p.T * p.k;
  kb::moe::await_predecessor();
  const int mine = lane < n ? expert_of(p, lane) : -1;
  const int e = __shfl_sync(FULL, mine, blockIdx.y);
  if (e < 0) return;
  unsigned members = __ballot_sync(FULL, mine == e);
  if (__ffs(members) - 1 != (int)blockIdx.y) return;
  const int f = blockIdx.x * WARPS + (threadIdx.x >> 5);
  if (f >= p.F) return;
  const uint4* g = reinterpret_cast<const uint4*>(p.wg + e * p.sg + f * p.ldg);
  const uint4* u = reinterpret_cast<const uint4*>(p.wu + e * p.su + f * p.ldu);
  const int pieces = p.D / 8;
  while (members) {
    int a[MEMBERS];
    const uint4* x[MEMBERS];
    int cnt = 0;
#pragma unroll
    for (int i = 0; i < MEMBERS; ++i) {
      a[i] = members ? __ffs(members) - 1 : a[0];
      cnt += members != 0;
      members &= members - 1;
      x[i] = reinterpret_cast<const uint4*>(p.x + (a[i] / p.k) * p.ldx);
    }
    float sg[MEMBERS], su[MEMBERS];
#pragma unroll
    for (int i = 0; i < MEMBERS; ++i) sg[i] = su[i] = 0.f;
    for (int c0 = lane; c0 < pieces; c0 += 32 * PIECES) {
      uint4 vg[PIECES], vu[PIECES];
#pragma unroll
      for (int q = 0; q < PIECES; ++q) {
        const int c = c0 + q * 32;
        vg[q] = c < pieces ? stream_load(g + c) : make_uint4(0u, 0u, 0u, 0u);
        vu[q] = c < pieces ? stream_load(u + c) : make_uint4(0u, 0u, 0u, 0u);
      }
#pragma unroll
      for (int q = 0; q < PIECES; ++q) {
        const int c = c0 + q * 32;
        if (c >= pieces) break;
#pragma unroll
        for (int i = 0; i < MEMBERS; ++i) {
          if (i >= cnt) break;
          const uint4 xv = __ldg(x[i] + c);
          sg[i] = dot8(vg[q], xv, sg[i]);
          su[i] = dot8(vu[q], xv, su[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < MEMBERS; ++i) {
      if (i >= cnt) break;
      const float gate = warp_sum(sg[i]), up = warp_sum(su[i]);
      if (lane == 0) {
        const float w = p.w_f32 ? static_cast<const float*>(p.w)[a[i]] : __bfloat162float(static_cast<const __nv_bfloat16*>(p.w)[a[i]]);
        p.h[(size_t)a[i] * p.F + f] = w * __fdividef(gate, 1.f + __expf(-gate)) * up;
      }
    }
  }
}

// out[t][d] = res[t][d] + sum_j h[t][j] . down[e_j][d]; `split` warps of the block share ROWS features.
__global__ void __launch_bounds__(WARPS * 32) down_kernel(const Params p, int split) {
  __shared__ float part[WARPS][ROWS];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int d0 = (blockIdx.x * (WARPS / split) + warp / split) * ROWS;
  const int t = blockIdx.y;
  float s[ROWS];
#pragma unroll
  for (int r = 0; r < ROWS; ++r) s[r] = 0.f;
  bool waited = false;
  if (d0 < p.D) {  // D is a multiple of 8
    const int pieces = p.F / 8;
    for (int j = warp % split; j < p.k; j += split) {
      const int a = t * p.k + j;
      const int e = expert_of(p, a);
      if (e < 0) continue;
      const __nv_bfloat16* w0 = p.wd + e * p.sd + d0 * p.ldd;
      const float4* hrow = reinterpret_cast<const float4*>(p.h + (size_t)a * p.F);
      for (int c0 = lane; c0 < pieces; c0 += 32 * PIECES) {
        uint4 v[ROWS][PIECES];
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
          for (int q = 0; q < PIECES; ++q)
            v[r][q] = c0 + q * 32 < pieces ? stream_load(reinterpret_cast<const uint4*>(w0 + r * p.ldd) + c0 + q * 32) : make_uint4(0u, 0u, 0u, 0u);
        if (!waited) {  // the first weights are under way while the hidden activations are still computed
          kb::moe::await_predecessor();
          waited = true;
        }
#pragma unroll
        for (int q = 0; q < PIECES; ++q) {
          const int c = c0 + q * 32;
          if (c >= pieces) break;
          const float4 a0 = hrow[2 * c], a1 = hrow[2 * c + 1];
#pragma unroll
          for (int r = 0; r < ROWS; ++r) {
            const float2 x0 = unpack_bf16x2(v[r][q].x), x1 = unpack_bf16x2(v[r][q].y), x2 = unpack_bf16x2(v[r][q].z), x3 = unpack_bf16x2(v[r][q].w);
            s[r] = fmaf(a0.x, x0.x, s[r]); s[r] = fmaf(a0.y, x0.y, s[r]); s[r] = fmaf(a0.z, x1.x, s[r]); s[r] = fmaf(a0.w, x1.y, s[r]);
            s[r] = fmaf(a1.x, x2.x, s[r]); s[r] = fmaf(a1.y, x2.y, s[r]); s[r] = fmaf(a1.z, x3.x, s[r]); s[r] = fmaf(a1.w, x3.y, s[r]);
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r) s[r] = warp_sum(s[r]);
  }
  if (!waited) kb::moe::await_predecessor();
  if (lane < ROWS) part[warp][lane] = lane ? s[ROWS - 1] : s[0];
  __syncthreads();
  if (lane < ROWS && d0 < p.D && warp % split == 0) {
    const int d = d0 + lane;
    float total = p.res ? __bfloat162float(p.res[t * p.ldr + d]) : 0.f;
    for (int i = 0; i < split; ++i) total += part[warp + i][lane];
    p.out[(size_t)t * p.D + d] = __float2bfloat16(total);
  }
}
static_assert(ROWS == 2, "part[] is filled by two lanes");

}  // namespace moe_small
}  // namespace kb

extern "C" int kb_moe_experts_small(const void* x, long ldx, const void* weights, int w_f32, const void* ids, int ids64, const void* wg, long ldg, long sg,
                                    const void* wu, long ldu, long su, const void* wd, long ldd, long sd, const void* res, long ldr, void* out, float* h,
                                    int T, int k, int D, int F, int E, void* stream) {
  using namespace kb::moe_small;
  if (T < 1 || k < 1 || D < 8 || F < 8 || E < 1 || (D & 7) || (F & 7)) return KB_STATUS_BAD_ARG;
  if ((long long)T * k > KB_MOE_SMALL_MAX) return KB_STATUS_TOO_LARGE;
  const uintptr_t any = reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(wg) | reinterpret_cast<uintptr_t>(wu) |
                        reinterpret_cast<uintptr_t>(wd) | reinterpret_cast<uintptr_t>(h);
  if ((any & 15) || ((ldx | ldg | sg | ldu | su | ldd | sd) & 7)) return KB_STATUS_BAD_ARG;
  using bf = const __nv_bfloat16*;
  const Params p{static_cast<bf>(x), static_cast<bf>(wg), static_cast<bf>(wu), static_cast<bf>(wd), static_cast<bf>(res), weights, ids,
                 static_cast<__nv_bfloat16*>(out), h, ldx, ldg, sg, ldu, su, ldd, sd, ldr, w_f32, ids64, T, k, D, F, E};
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  kb::moe::launch_after(T == 1 ? up_kernel<1> : up_kernel<4>, dim3((F + WARPS - 1) / WARPS, T * k), WARPS * 32, 0, st, p);
  const int split = k >= 8 ? 8 : k >= 4 ? 4 : k >= 2 ? 2 : 1;
  kb::moe::launch_after(down_kernel, dim3((D / ROWS + WARPS / split - 1) / (WARPS / split), T), WARPS * 32, 0, st, p, split);
  return cudaGetLastError() == cudaSuccess ? KB_STATUS_OK : KB_STATUS_CUDA_ERROR;
}
