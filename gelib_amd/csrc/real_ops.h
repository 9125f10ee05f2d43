// The operators on real channels around the equivariant layers -- group norm with an activation, the linear layer with its
// epilogue, the AdamW step -- and those of a network over points -- embedding, attention, cross entropy of a linear layer's classes -- as the C entry
// points (cabi_real.cpp, cabi_points.cpp) see them, and what their kernels share.
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
  void *slope;          // act'(z), (rows, N): float32 for float32 layers, 16 bits for the others (SlopeOf); null: not wanted
  const void *x, *w, *b, *r;
  const void *gy;
  void *gx, *gw, *gb;
  long long rows, xs;   // xs: elements from one row of x to the next
  int K, N, act;
  void *ws;
};
constexpr int kLinearMostChannels = 0x7fffff00;   // of either side: rounded up to whole tiles and vectors they stay below 2^31, and a row of tiles below 2^32 threads
size_t linear_workspace(int backward, int dtype, long long rows, int K, int N);   // backward: bits 1 gx, 2 gw, 4 gb, 8 slope; 0 forward
int launch_linear_fwd(int dtype, const LinearArgs &a, hipStream_t s);
int launch_linear_bwd(int dtype, const LinearArgs &a, hipStream_t s);
int linear_act_set_option(const char *name, int value);

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

// ---- a linear layer's classes and their loss (linear_loss.hip) ----
struct LossArgs {
  float *loss, *lse_out;          // forward; lse_out may be null
  void *gx, *gw, *gb;             // backward; any may be null
  const void *x, *w, *b;
  const long long *targets;
  const float *g, *lse;
  long long rows, xs;
  int K, N;
  void *ws;
};
size_t loss_workspace(int what, int dtype, long long rows, int K, int N);   // what: bits 1 gx, 2 gw, 4 gb; 0 forward
int launch_loss(int dtype, const LossArgs &a, hipStream_t s);
int launch_loss_bwd(int dtype, const LossArgs &a, hipStream_t s);

// ---- embedding (embedding.hip) ----
struct EmbeddingArgs {
  void *y, *gtable;
  const void *table, *gy, *tokens;
  long long n, rows;
  int wide, channels;   // wide: tokens of 64 bits
  float scale;
  void *ws;
};
size_t embedding_workspace(long long n, int channels);
int launch_embedding(int dtype, const EmbeddingArgs &a, hipStream_t s);
int launch_embedding_bwd(int dtype, const EmbeddingArgs &a, hipStream_t s);

// ---- attention (attention.hip) ----
struct AttnCall {
  const void *q, *k, *v;
  const float *x, *xk, *slopes;    // null: no distances
  const int *q_marks, *k_marks;    // padded: lengths or null; packed: starts, docs + 1 of them
  long long docs, nq, nk;          // padded: samples and rows of one; packed: documents and all rows
  long long qs[3], ks[3], vs[3];   // strides of samples, positions, heads, in elements
  int dtype, packed, heads, kv_heads, dim;
  float scale;
};
struct AttnGrads {
  const void *y, *gy;
  const float *lse;
  void *gq, *gk, *gv;              // any may be null
  float *gx, *gxk, *gslopes;
  bool same_points;                // gx takes the sums over queries and keys
};
constexpr int kAttnMostDim = 128;
inline int attention_dims(int dtype, int dim) { return dim <= 16 && dtype == GELIB_HIP_F32 ? 16 : dim <= 32 ? 32 : dim <= 64 ? 64 : 128; }
size_t attention_workspace(const AttnCall &c, bool backward, bool geometry);
int launch_attention(const AttnCall &c, void *y, float *lse, void *ws, hipStream_t s);
int launch_attention_bwd(const AttnCall &c, const AttnGrads &g, void *ws, hipStream_t s);

#ifdef __HIPCC__
typedef _Float16 half_t;
typedef __bf16 bhalf_t;

template <typename T>
__device__ __forceinline__ float to_f(T v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f(float v) { return (T)v; }   // round to nearest even

// act'(z) in 16 bits for float16 layers: steps of 2^-15 from 2^-5 on and float16 below.  In float16 alone its rounding is as large as
// the layer's own, and gw, which is rounded twice besides (gz, and itself), came out 1.54 to 1.73 times as far off as with one
// rounding; these steps are 1/16 of float16's over [0.5, 1), where most slopes are.  All of [-0.18, 1.14] has a code, which silu'
// (-0.10 to 1.10) and gelu' (-0.13 to 1.13) stay within; what is not a number has its own.  16384 x 2048 -> 8192, forward and both
// directions, on one card: silu 588 and 1792 us, gelu 622 and 1824, without an activation 580 and 1630; in bfloat16, whose products draw
// less power, 521 and 1700, 547 and 1728, 517 and 1539: the codes take about 5 to 10 us forward and nothing that shows in gz.
struct slope16_t {
  static constexpr int kFloats = 0x2800, kNan = 50000;   // the float16 codes below 2^-5; positive codes end at 46572, negative ones begin at 50421
  unsigned short code;
  slope16_t() = default;
  __device__ explicit slope16_t(float s) {
    const float a = fabsf(s);
    const int small = __builtin_bit_cast(unsigned short, (half_t)a), large = (int)rintf(a * 32768.f) - 1024 + kFloats;
    const int n = a < 0.03125f ? small : large;
    code = !(s >= -0.18f && s <= 1.14f) ? kNan : s < 0.f ? 65535 - n : n;
  }
  __device__ operator float() const {
    const int n = code > kNan ? 65535 - code : code;
    const float a = n < kFloats ? (float)__builtin_bit_cast(half_t, (unsigned short)n) : (float)(n - kFloats + 1024) * 0x1p-15f;
    return code == kNan ? __builtin_nanf("") : code > kNan ? -a : a;
  }
};

enum Act { kActNone = 0, kActRelu = 1, kActSilu = 2, kActGelu = 3 };

// Phi(z), the normal distribution, given e = exp(-z^2 / 2): 1/2 erfc(|z| / sqrt 2) as e times a polynomial in t = 1 / (1 + p |z| / sqrt 2),
// reflected for z > 0.  (The form is Abramowitz & Stegun's, Handbook of Mathematical Functions, 7.1.25 to 28; p and seven coefficients are
// fitted here, for the least largest error of erfc over 0..6: 4e-10, so that what is left is the roundings of float32.)  The exponential
// serves the density in gelu' too.  Root mean square errors of gelu and gelu' over normally distributed z, in units of 2^-24: 0.41 and 0.63;
// with the handbook's five coefficients (1.5e-7) 0.93 and 1.10, in the same time (to 1 %); with the library's erff 0.42 and 0.46, at 4 % more
// time for a float32 layer (32768 x 256 -> 512, both directions) and 11 % for a norm (64 x 1024 x 256).
__device__ __forceinline__ float normal_cdf(float z, float e) {
  const float t = __builtin_amdgcn_rcpf(1.f + 0.47f * 0.70710678118654752f * __builtin_fabsf(z));
  const float tail = e * (t * (0.13292666f + t * (0.12584779f + t * (0.16198763f + t * (-0.05227607f + t * (0.29318786f + t * (-0.20470048f + t * 0.04302663f)))))));
  return z > 0.f ? 1.f - tail : tail;
}

// act(z) and act'(z).  exp and the reciprocal are the hardware's (1 ulp).  Over normally distributed z silu is 0.47 units of 2^-24 off and
// silu' 0.49, 0.39 and 0.48 in torch's float32 operations; with the library's expf and a division 0.45 and 0.48, at 2 and 11 % more time for the same two.
// kActNone stands for relu too where a flag says so.
template <int ACT>
__device__ __forceinline__ void act_both(float z, float &value, float &slope, bool relu = false) {
  if (ACT == kActSilu) {
    const float s = __builtin_amdgcn_rcpf(1.f + __expf(-z));
    value = z * s, slope = s * (1.f + z * (1.f - s));
  } else if (ACT == kActGelu) {
    const float e = __expf(-0.5f * z * z), cdf = normal_cdf(z, e);
    value = z * cdf, slope = cdf + z * 0.39894228040143268f * e;
  } else if (ACT == kActRelu || relu) {
    value = z < 0.f ? 0.f : z, slope = z > 0.f ? 1.f : z == z ? 0.f : z;   // (a NaN stays one)
  } else {
    value = z, slope = 1.f;
  }
}
#endif

}  // namespace gelib_hip
