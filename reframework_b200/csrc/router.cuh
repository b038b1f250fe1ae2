// What the two router entry points (router.cu, router_grouped.cu) share: the
// logits stage and the device helpers that read its partial sums.
#pragma once

#include "gemm.cuh"

namespace rf {

constexpr int ROUTER_KMAX = 16;   // a warp's lane k holds choice k
constexpr int ROUTER_EMAX = 1024;

// Where the logits stage left its sums: fp32 partials [slices][T][ld], the
// shared-expert gate's column (if any) right after the E experts'.
struct RouterLogits {
  const float *partial;
  int slices;
  int64_t ld;
};

// Launches x . gate^T (and the shared gate's column) into `workspace`
// (rf_moe_router_workspace_size bytes); `what` names the caller in messages.
int router_logits(const char *what, const void *x, int x_dtype, const void *gate, int gate_dtype,
                  const void *shared_gate, int64_t T, int64_t H, int64_t E, void *workspace,
                  size_t workspace_bytes, cudaStream_t st, RouterLogits *out);

__device__ __forceinline__ float round_dt(int dtype, float v) {
  if (dtype == RF_BF16) return __bfloat162float(__float2bfloat16_rn(v));
  if (dtype == RF_F16) return __half2float(__float2half_rn(v));
  return v;
}

// 0 + p[0] + p[stride] + ... in slice order, eight loads in flight at a time.
__device__ __forceinline__ float sum_slices(const float *p, int64_t stride, int n) {
  float v = 0.f;
  int z = 0;
  for (; z + 8 <= n; z += 8) {
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = p[(int64_t)(z + i) * stride];
#pragma unroll
    for (int i = 0; i < 8; ++i) v += q[i];
  }
  for (; z < n; ++z) v += p[(int64_t)z * stride];
  return v;
}

}  // namespace rf
