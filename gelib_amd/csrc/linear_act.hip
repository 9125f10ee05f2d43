// The linear layer with its epilogue, z = x w + b, y = act(z) + r, and its gradients: gz = gy act'(z), gx = gz w^T, gw = x^T gz,
// gb = sum of gz over the rows.  act'(z) is what the forward pass leaves for the backward pass, not z: it lies between
// -0.2 and 1.2, so 16-bit layers keep it in float16 (11 bits) at no loss beside the 8 bits of a bfloat16 z.
#include "real_ops.h"

namespace gelib_hip {

namespace {

template <int ACT>
__device__ __forceinline__ void act_both(float z, float &value, float &slope) { value = act_value<ACT>(z), slope = act_slope<ACT>(z); }

__device__ __forceinline__ void act_both(int act, float z, float &value, float &slope) {
  if (act == kActRelu) act_both<kActRelu>(z, value, slope);
  else if (act == kActSilu) act_both<kActSilu>(z, value, slope);
  else if (act == kActGelu) act_both<kActGelu>(z, value, slope);
  else act_both<kActNone>(z, value, slope);
}

template <typename T>
struct SlopeOf { typedef half_t type; };
template <>
struct SlopeOf<float> { typedef float type; };

// C[m, n] = sum_k A[m, k] B[k, n] with any strides of A and B, 64 x 64 of it per block; gz factors on either side
template <typename T>
struct Operand {
  const T *p;
  const typename SlopeOf<T>::type *slope;   // multiplied in, at the same place
  long long sr, sc;
  __device__ float at(long long r, long long c) const {
    const long long i = r * sr + c * sc;
    const float v = to_f(p[i]);
    return slope ? to_f(from_f<T>(v * to_f(slope[i]))) : v;
  }
};

template <typename T>
__global__ void __launch_bounds__(256) gemm_kernel(const Operand<T> A, const Operand<T> B, long long M, long long N, long long K, T *C,
                                                   const T *bias, const T *res, typename SlopeOf<T>::type *slope, int act) {
  __shared__ float as[16][65], bs[16][65];
  const long long tiles = (N + 63) / 64, m0 = blockIdx.x / tiles * 64, n0 = blockIdx.x % tiles * 64;
  const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
  float acc[4][4] = {};
  for (long long k0 = 0; k0 < K; k0 += 16) {
    __syncthreads();
    for (int e = threadIdx.x; e < 1024; e += 256) {
      const int i = e / 16, k = e % 16;
      as[k][i] = m0 + i < M && k0 + k < K ? A.at(m0 + i, k0 + k) : 0.f;
      bs[k][i] = n0 + i < N && k0 + k < K ? B.at(k0 + k, n0 + i) : 0.f;
    }
    __syncthreads();
    for (int k = 0; k < 16; k++)
      for (int i = 0; i < 4; i++)
        for (int j = 0; j < 4; j++) acc[i][j] += as[k][tr * 4 + i] * bs[k][tc * 4 + j];
  }
  for (int i = 0; i < 4; i++)
    for (int j = 0; j < 4; j++) {
      const long long m = m0 + tr * 4 + i, n = n0 + tc * 4 + j;
      if (m >= M || n >= N) continue;
      float v = acc[i][j] + (bias ? to_f(bias[n]) : 0.f), d;
      act_both(act, v, v, d);
      if (slope) slope[m * N + n] = from_f<typename SlopeOf<T>::type>(d);
      C[m * N + n] = from_f<T>(v + (res ? to_f(res[m * N + n]) : 0.f));
    }
}

template <typename T>
__global__ void __launch_bounds__(256) column_sum_kernel(const T *g, const typename SlopeOf<T>::type *slope, long long M, long long N, T *out) {
  const long long n = (long long)blockIdx.x * 256 + threadIdx.x;
  if (n >= N) return;
  float s = 0.f;
  for (long long m = 0; m < M; m++) s += to_f(g[m * N + n]) * (slope ? to_f(slope[m * N + n]) : 1.f);
  out[n] = from_f<T>(s);
}

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "linear layer launch");
}

dim3 tiles(long long m, long long n) { return dim3((unsigned)(((m + 63) / 64) * ((n + 63) / 64))); }

template <typename T>
int fwd(const LinearArgs &a, hipStream_t s) {
  typedef typename SlopeOf<T>::type D;
  if (!a.rows || !a.N) return 0;
    hipLaunchKernelGGL(gemm_kernel<T>, tiles(a.rows, a.N), dim3(256), 0, s, Operand<T>{(const T *)a.x, nullptr, a.xs, 1},
                       Operand<T>{(const T *)a.w, nullptr, a.N, 1}, a.rows, a.N, a.K, (T *)a.y, (const T *)a.b, (const T *)a.r, (D *)a.slope, a.act);
  return launched();
}

template <typename T>
int bwd(const LinearArgs &a, hipStream_t s) {
  typedef typename SlopeOf<T>::type D;
  if (a.gx && a.rows && a.K)
    hipLaunchKernelGGL(gemm_kernel<T>, tiles(a.rows, a.K), dim3(256), 0, s, Operand<T>{(const T *)a.gy, (const D *)a.slope, a.N, 1},
                       Operand<T>{(const T *)a.w, nullptr, 1, a.N}, a.rows, a.K, a.N, (T *)a.gx, (const T *)nullptr, (const T *)nullptr, (D *)nullptr, 0);
  if (a.gw && a.K && a.N)
    hipLaunchKernelGGL(gemm_kernel<T>, tiles(a.K, a.N), dim3(256), 0, s, Operand<T>{(const T *)a.x, nullptr, 1, a.xs},
                       Operand<T>{(const T *)a.gy, (const D *)a.slope, a.N, 1}, a.K, a.N, a.rows, (T *)a.gw, (const T *)nullptr, (const T *)nullptr, (D *)nullptr, 0);
  if (a.gb && a.N)
    hipLaunchKernelGGL(column_sum_kernel<T>, dim3((unsigned)((a.N + 255) / 256)), dim3(256), 0, s, (const T *)a.gy, (const D *)a.slope, a.rows, (long long)a.N, (T *)a.gb);
  return launched();
}

}  // namespace

size_t linear_workspace(int, int, long long, int, int) { return 0; }

int launch_linear_fwd(int dtype, const LinearArgs &a, hipStream_t s) {
  return dtype == GELIB_HIP_F32 ? fwd<float>(a, s) : dtype == GELIB_HIP_BF16 ? fwd<bhalf_t>(a, s) : fwd<half_t>(a, s);
}

int launch_linear_bwd(int dtype, const LinearArgs &a, hipStream_t s) {
  return dtype == GELIB_HIP_F32 ? bwd<float>(a, s) : dtype == GELIB_HIP_BF16 ? bwd<bhalf_t>(a, s) : bwd<half_t>(a, s);
}

}  // namespace gelib_hip
