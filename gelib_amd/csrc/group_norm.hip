// Group norm with an activation, channels last: a group is C / G neighbouring channels over the positions of a sample that count,
//     xh = (x - mean) rstd,  y = act(xh w + b);   gz = gy act'(z), q = gz w, gx = rstd (q - mean(q) - xh mean(q xh)),
//     gw = sum gz xh, gb = sum gz over samples and positions.
// Positions behind a sample's length are zero in y and gx and are never read.
#include "real_ops.h"

namespace gelib_hip {

namespace {

__device__ __forceinline__ float block_sum(float v, float *lds) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = v;
  __syncthreads();
  return (lds[0] + lds[1]) + (lds[2] + lds[3]);
}

__device__ __forceinline__ long long length_of(const NormArgs &a, long long n) {
  return a.lengths ? (long long)max(0, (int)min((long long)a.lengths[n], a.S)) : a.S;
}

// a block per (sample, group)
template <typename T, int ACT>
__global__ void __launch_bounds__(256) norm_fwd_kernel(const NormArgs a) {
  __shared__ float lds[4];
  const long long n = blockIdx.x / a.G;
  const int g = (int)(blockIdx.x % a.G), cg = a.C / a.G, c0 = g * cg;
  const long long len = length_of(a, n), cnt = len * cg;
  const T *x = (const T *)a.x + n * a.xs + c0;
  T *y = (T *)a.y + n * a.S * a.C + c0;
  float sum = 0.f;
  for (long long i = threadIdx.x; i < cnt; i += 256) sum += to_f(x[i / cg * a.xp + i % cg]);
  const float mean = cnt ? block_sum(sum, lds) / (float)cnt : 0.f;
  sum = 0.f;
  for (long long i = threadIdx.x; i < cnt; i += 256) {
    const float d = to_f(x[i / cg * a.xp + i % cg]) - mean;
    sum += d * d;
  }
  const float rstd = 1.f / sqrtf((cnt ? block_sum(sum, lds) / (float)cnt : 0.f) + a.eps);
  if (a.mean && threadIdx.x == 0) a.mean[blockIdx.x] = mean, a.rstd[blockIdx.x] = rstd;
  for (long long i = threadIdx.x; i < a.S * cg; i += 256) {
    const long long s = i / cg;
    const int c = (int)(i % cg);
    float r = 0.f;
    if (s < len) {
      const float z = (to_f(x[s * a.xp + c]) - mean) * rstd * (a.w ? to_f(((const T *)a.w)[c0 + c]) : 1.f) + (a.b ? to_f(((const T *)a.b)[c0 + c]) : 0.f);
      r = act_value<ACT>(z);
    }
    y[s * a.C + c] = from_f<T>(r);
  }
}

template <typename T, int ACT>
__global__ void __launch_bounds__(256) norm_gx_kernel(const NormArgs a) {
  __shared__ float lds[4];
  const long long n = blockIdx.x / a.G;
  const int g = (int)(blockIdx.x % a.G), cg = a.C / a.G, c0 = g * cg;
  const long long len = length_of(a, n), cnt = len * cg;
  const T *x = (const T *)a.x + n * a.xs + c0, *gy = (const T *)a.gy + n * a.S * a.C + c0;
  T *gx = (T *)a.y + n * a.S * a.C + c0;
  const float mean = a.mean[blockIdx.x], rstd = a.rstd[blockIdx.x];
  auto at = [&](long long i, float &q, float &xh) {
    const long long s = i / cg;
    const int c = (int)(i % cg);
    const float w = a.w ? to_f(((const T *)a.w)[c0 + c]) : 1.f;
    xh = (to_f(x[s * a.xp + c]) - mean) * rstd;
    q = w * to_f(gy[s * a.C + c]) * act_slope<ACT>(xh * w + (a.b ? to_f(((const T *)a.b)[c0 + c]) : 0.f));
  };
  float s1 = 0.f, s2 = 0.f, q, xh;
  for (long long i = threadIdx.x; i < cnt; i += 256) {
    at(i, q, xh);
    s1 += q, s2 += q * xh;
  }
  const float m1 = cnt ? block_sum(s1, lds) / (float)cnt : 0.f, m2 = cnt ? block_sum(s2, lds) / (float)cnt : 0.f;
  for (long long i = threadIdx.x; i < a.S * cg; i += 256) {
    float r = 0.f;
    if (i < cnt) {
      at(i, q, xh);
      r = rstd * (q - m1 - xh * m2);
    }
    gx[i / cg * a.C + i % cg] = from_f<T>(r);
  }
}

// a block per channel
template <typename T, int ACT>
__global__ void __launch_bounds__(256) norm_gw_kernel(const NormArgs a) {
  __shared__ float lds[4];
  const int c = blockIdx.x, g = c / (a.C / a.G);
  const float w = a.w ? to_f(((const T *)a.w)[c]) : 1.f, b = a.b ? to_f(((const T *)a.b)[c]) : 0.f;
  float sw = 0.f, sb = 0.f;
  for (long long i = threadIdx.x; i < a.N * a.S; i += 256) {
    const long long n = i / a.S, s = i % a.S;
    if (s >= length_of(a, n)) continue;
    const float xh = (to_f(((const T *)a.x)[n * a.xs + s * a.xp + c]) - a.mean[n * a.G + g]) * a.rstd[n * a.G + g];
    const float gz = to_f(((const T *)a.gy)[i * a.C + c]) * act_slope<ACT>(xh * w + b);
    sw += gz * xh, sb += gz;
  }
  sw = block_sum(sw, lds), sb = block_sum(sb, lds);
  if (threadIdx.x == 0) {
    if (a.gw) ((T *)a.gw)[c] = from_f<T>(sw);
    if (a.gb) ((T *)a.gb)[c] = from_f<T>(sb);
  }
}

template <typename T, int ACT>
int run(bool backward, const NormArgs &a, hipStream_t s) {
  const long long tiles = a.S ? a.N * a.G : 0;
  if (!tiles && !a.gw && !a.gb) return 0;
  if (!backward) {
    if (tiles) hipLaunchKernelGGL((norm_fwd_kernel<T, ACT>), dim3((unsigned)tiles), dim3(256), 0, s, a);
  } else {
    if (tiles && a.y) hipLaunchKernelGGL((norm_gx_kernel<T, ACT>), dim3((unsigned)tiles), dim3(256), 0, s, a);
    if (a.gw || a.gb) hipLaunchKernelGGL((norm_gw_kernel<T, ACT>), dim3(a.C), dim3(256), 0, s, a);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "group norm launch");
}

template <typename T>
int run_act(bool backward, const NormArgs &a, hipStream_t s) {
  switch (a.act) {
    case kActRelu: return run<T, kActRelu>(backward, a, s);
    case kActSilu: return run<T, kActSilu>(backward, a, s);
    case kActGelu: return run<T, kActGelu>(backward, a, s);
  }
  return run<T, kActNone>(backward, a, s);
}

}  // namespace

size_t norm_workspace(bool, int, long long, long long, int, int) { return 0; }

int launch_norm(bool backward, int dtype, const NormArgs &a, hipStream_t s) {
  if (dtype == GELIB_HIP_F32) return run_act<float>(backward, a, s);
  if (dtype == GELIB_HIP_BF16) return run_act<bhalf_t>(backward, a, s);
  return run_act<half_t>(backward, a, s);
}

}  // namespace gelib_hip
