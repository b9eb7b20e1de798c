// Activations and the single-pass form shared by the group normalisation translation units.
#pragma once
#include "vc_common.h"

enum { ACT_NONE = 0, ACT_RELU = 1, ACT_SILU = 2, ACT_GELU = 3 };

template <int ACT>
static __device__ __forceinline__ float act_fwd(float z) {
  if (ACT == ACT_RELU) return z < 0.f ? 0.f : z;  // NaN stays NaN
  if (ACT == ACT_SILU) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  if (ACT == ACT_GELU) return vc_gelu(z);
  return z;
}
template <int ACT>
static __device__ __forceinline__ float act_slope(float z) {
  if (ACT == ACT_RELU) return z > 0.f ? 1.f : 0.f;
  if (ACT == ACT_SILU) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return s * fmaf(z, 1.f - s, 1.f);
  }
  if (ACT == ACT_GELU) return vc_gelu_grad(z);
  return 1.f;
}

// Single-pass form (vc_group_slab.hip): a workgroup keeps whole groups of a sample in registers.
bool vc_gn_slab_fwd(int dtype, const void* x, const void* res, const float* gamma, const float* beta, void* y, float* mean,
                    float* rstd, int N, int S, int C, int G, float eps, int act, hipStream_t stream);
bool vc_gn_slab_bwd(int dtype, const void* x, const void* dy, const void* res, const float* gamma, const float* beta,
                    const float* mean, const float* rstd, void* dx, void* dres, float* ab, int N, int S, int C, int G,
                    int act, hipStream_t stream);
