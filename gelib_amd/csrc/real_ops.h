// The operators on real channels around the equivariant layers -- group norm with an activation, the linear layer with its
// epilogue, the AdamW step -- as the C entry points (cabi_real.cpp) see them, and what their kernels share.
#pragma once

#include <algorithm>
#include <cstddef>

#include "cg_common.h"

namespace gelib_hip {

// GELIB_HIP_F32 / _BF16 / _F16 and GELIB_HIP_ACT_* of gelib_hip.h
inline size_t dtype_bytes(int dtype) { return dtype == GELIB_HIP_F32 ? 4 : 2; }

// ---- group norm (group_norm.hip) ----
struct NormArgs {
  void *y;               // forward: the result; backward: the gradient of x
  const void *x, *gy;    // x has strides, everything else is packed
  const void *w, *b;     // either may be null: 1 and 0
  const int *lengths;    // positions of every sample that count; null: all
  float *mean, *rstd;    // [samples][groups]; forward: null where nobody wants them
  void *gw, *gb;         // backward: either may be null
  long long N, S, xs, xp;  // samples, positions, strides of x in elements
  int C, G, act;
  float eps;
  void *ws;
};
size_t norm_workspace(bool backward, int dtype, long long N, long long S, int C, int G);
int launch_norm(bool backward, int dtype, const NormArgs &a, hipStream_t s);

// ---- linear layer (linear_act.hip) ----
struct LinearArgs {
  void *y;              // (rows, N)
  void *slope;          // act'(z), (rows, N): float32 for float32 layers, float16 for the 16-bit ones; null: not wanted
  const void *x, *w, *b, *r;
  const void *gy;
  void *gx, *gw, *gb;
  long long rows, xs;   // xs: elements from one row of x to the next
  int K, N, act;
  void *ws;
};
size_t linear_workspace(int backward, int dtype, long long rows, int K, int N);   // backward: bits 1 gx, 2 gw, 4 gb, 8 slope; 0 forward
int launch_linear_fwd(int dtype, const LinearArgs &a, hipStream_t s);
int launch_linear_bwd(int dtype, const LinearArgs &a, hipStream_t s);

// ---- AdamW (adamw.hip) ----
constexpr int kAdamBlock = 256;   // elements that share a scale of 8-bit moments; parameters start at multiples of it
struct AdamArgs {
  void *m, *v;               // moments of all parameters: float32, or one byte each
  short *m_top, *v_top;      // 8 bits: scale of every block
  int dtype, bits;
  float decay, b1, c1, b2, c2, eps;   // lr weight_decay, beta1, 1 - beta1, ...
};
struct AdamTensor {
  void *p;
  const void *g;
  long long n, first;
  float step_size, inv_sqrt_bc2;   // lr / (1 - b1^t), (1 - b2^t)^-1/2
  unsigned key;                    // of the random bits
};
int launch_adamw(int n, const AdamTensor *t, const AdamArgs &a, hipStream_t s);
int launch_adamw_moments(void *mv, void *vv, const void *m, const void *v, const short *mt, const short *vt, long long n, hipStream_t s);
int launch_adamw_set_moments(void *m, void *v, short *mt, short *vt, const float *mv, const float *vv, long long n, hipStream_t s);

#ifdef __HIPCC__
typedef _Float16 half_t;
typedef __bf16 bhalf_t;

template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }   // round to nearest even

enum Act { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

// act(z) and act'(z).  exp and the reciprocal are the hardware's (1 ulp): the sums in front of them are the coarser part.
template <int ACT>
__device__ __forceinline__ float act_value(float z) {
  if (ACT == kActRelu) return z < 0.f ? 0.f : z;   // (a NaN stays one)
  if (ACT == kActSilu) return z * __builtin_amdgcn_rcpf(1.f + __expf(-z));
  if (ACT == kActGelu) return 0.5f * z * (1.f + erff(z * 0.70710678118654752f));
  return z;
}
template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if (ACT == kActRelu) return z > 0.f ? 1.f : z == z ? 0.f : z;
  if (ACT == kActSilu) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    return s * (1.f + z * (1.f - s));
  }
  if (ACT == kActGelu) return 0.5f * (1.f + erff(z * 0.70710678118654752f)) + z * 0.39894228040143268f * __expf(-0.5f * z * z);
  return 1.f;
}
#endif

}  // namespace gelib_hip
