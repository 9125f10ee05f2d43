// One AdamW step over all parameters of an optimizer, moments in 32 or in 8 bits:
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p - lr decay p - step_size m / (sqrt(v) inv_sqrt_bc2 + eps)
// with step_size = lr / (1 - b1^t), inv_sqrt_bc2 = (1 - b2^t)^-1/2; complex parameters are twice as many reals.
//
// Every parameter owns a run of the moment arrays that starts at a multiple of 256 elements; a block of 256 elements is what
// one scale is kept for in 8 bits.  A wave owns such a block (4 elements a lane) and needs no other wave: the maximum is a
// wavefront reduction.
//
// The 8-bit form works on the bits of float32 numbers.  u = (bits without the sign + r) >> 20 are the exponent and three bits of
// the mantissa: eight steps an octave, and integers in the order of the values.  top = the largest u of a block (16 bits are
// kept of it); a value's code is u - top + 254 (v: 1..254, which are 31.6 octaves; 0 is zero, 255 is not finite) or u - top + 126
// (m: 1..126, 15.6 octaves, and the sign; below that zero, 127 is not finite).  What is not finite reads as infinity in v and as
// NaN in m: a gradient whose square overflows stops its parameter, as in 32 bits, and any other makes it NaN, as there.  A v above zero never falls to code 0: a step
// divided by its root would be as large as m / eps.  One element that is not finite leaves its neighbours' scale alone.
// r is random (20 of 32 bits of a mixed counter of seed, step and element): b2 = 0.999 changes v by a tenth of a percent of
// itself, a code step is 6 to 12, so rounding to the nearest would leave v where it is for ever.  bfloat16 parameters are
// rounded at random too (a step is mostly below half a unit in their last place).
// Every operation is rounded by itself (no contraction), so codes are a function of the inputs that a host can repeat.
#pragma clang fp contract(off)
#include <cstring>

#include "real_ops.h"

namespace gelib_hip {

namespace {

constexpr int kAdamTensors = 64;   // parameters of one launch: their table is 3 of the 4 KB of its arguments

struct AdamTable {
  struct {
    void *p;
    const void *g;
    long long n;
    unsigned first, blocks_before;  // first block of moments, blocks of the launch before this parameter
    float step_size, inv_sqrt_bc2;
    unsigned key;
  } t[kAdamTensors];
  int count;
  unsigned blocks;
};

__device__ __forceinline__ unsigned mixed(unsigned index, unsigned key) {
  unsigned h = (index + key) * 2654435769u;
  h = (h ^ (h >> 15)) * 3144134277u;
  h = (h ^ (h >> 13)) * 1779033703u;
  return h ^ (h >> 16);
}
__device__ __forceinline__ unsigned mixed_more(unsigned h) {
  h *= 2654435769u;
  return (h ^ (h >> 15)) & 0xffffu;
}

__device__ __forceinline__ int wave_max(int v) {
#pragma unroll
  for (int d = 32; d >= 1; d >>= 1) v = max(v, __shfl_xor(v, d));
  return v;
}

constexpr unsigned kInf = 0x7f800000u;
constexpr int kTopOfFinite = 2039;   // u of the largest finite float; rounding up past it stays there

constexpr unsigned kNan = 0x7fc00000u;

__device__ __forceinline__ float decoded(int code, int top, int steps, unsigned not_finite) {
  return __uint_as_float(code == 0 ? 0u : code > steps ? not_finite : (unsigned)max(code + top - steps, 0) << 20);
}
// u of a value (0 for zero, -1 where it is not finite)
__device__ __forceinline__ int upper(float x, unsigned r) {
  const unsigned b = __float_as_uint(x) & 0x7fffffffu;
  return b >= kInf ? -1 : min((int)((b + r) >> 20), kTopOfFinite);
}
template <bool ABOVE>
__device__ __forceinline__ int coded(float x, int u, int top, int steps) {
  if (u < 0) return steps + 1;
  const int c = u - top + steps;
  return c >= 1 ? ((__float_as_uint(x) & 0x7fffffffu) ? c : 0) : ABOVE && (__float_as_uint(x) & 0x7fffffffu) ? 1 : 0;
}

template <typename T, int BITS>
__global__ void __launch_bounds__(256) adamw_kernel(const AdamTable tab, const AdamArgs a) {
  const unsigned wave = blockIdx.x * 4 + threadIdx.x / 64, lane = threadIdx.x % 64;
  if (wave >= tab.blocks) return;
  int k = 0;
  while (k + 1 < tab.count && wave >= tab.t[k + 1].blocks_before) k++;
  const unsigned at = wave - tab.t[k].blocks_before;           // block of the parameter
  const long long e0 = (long long)at * kAdamBlock + lane * 4;  // element of the parameter
  const long long s0 = ((long long)tab.t[k].first + at) * kAdamBlock + lane * 4;
  T *p = (T *)tab.t[k].p;
  const T *g = (const T *)tab.t[k].g;
  const long long n = tab.t[k].n;
  const float step_size = tab.t[k].step_size, inv_sqrt_bc2 = tab.t[k].inv_sqrt_bc2;
  const unsigned key = tab.t[k].key;
  float m[4], v[4];
  if (BITS == 32) {
    for (int i = 0; i < 4; i++) m[i] = ((const float *)a.m)[s0 + i], v[i] = ((const float *)a.v)[s0 + i];
  } else {
    const int mt = a.m_top[s0 / kAdamBlock], vt = a.v_top[s0 / kAdamBlock];
    for (int i = 0; i < 4; i++) {
      const int cm = ((const unsigned char *)a.m)[s0 + i], cv = ((const unsigned char *)a.v)[s0 + i];
      m[i] = decoded(cm & 127, mt, 126, kNan);
      if (cm & 128) m[i] = -m[i];
      v[i] = decoded(cv, vt, 254, kInf);
    }
  }
  unsigned h[4];
  for (int i = 0; i < 4; i++) {
    const bool in = e0 + i < n;
    const float gi = in ? to_f(g[e0 + i]) : 0.f;
    m[i] = m[i] * a.b1 + gi * a.c1;
    v[i] = v[i] * a.b2 + (gi * gi) * a.c2;
    if (BITS == 8 || sizeof(T) == 2) h[i] = mixed((unsigned)(s0 + i), key + (unsigned)((s0 + i) >> 32) * 3144134277u);
    if (in) {
      const float denom = sqrtf(v[i]) * inv_sqrt_bc2 + a.eps;
      const float was = to_f(p[e0 + i]);
      const float np = (was - was * a.decay) - (m[i] * step_size) / denom;
      if (sizeof(T) == 2) {
        const unsigned b = __float_as_uint(np);
        ((unsigned short *)p)[e0 + i] = (b & 0x7fffffffu) > kInf ? 0x7fc0 : (b & 0x7fffffffu) == kInf ? b >> 16 : (b + mixed_more(h[i])) >> 16;
      } else {
        p[e0 + i] = from_f<T>(np);
      }
    }
  }
  if (BITS == 32) {
    for (int i = 0; i < 4; i++) ((float *)a.m)[s0 + i] = m[i], ((float *)a.v)[s0 + i] = v[i];
  } else {
    int um[4], uv[4], mt = 0, vt = 0;
    for (int i = 0; i < 4; i++) {
      um[i] = upper(m[i], h[i] & 0xfffffu), uv[i] = upper(v[i], h[i] >> 12);
      if (uv[i] < 0 && um[i] >= 0) m[i] = 0.f, um[i] = 0;   // v is infinite: its steps are zero whatever m is, and m as large as that
                                                            // would push the block's others below the smallest code
      mt = max(mt, um[i]), vt = max(vt, uv[i]);
    }
    mt = wave_max(mt), vt = wave_max(vt);
    for (int i = 0; i < 4; i++) {
      const int c = coded<false>(m[i], um[i], mt, 126);
      ((unsigned char *)a.m)[s0 + i] = c | (c && __float_as_uint(m[i]) >> 31 ? 128 : 0);
      ((unsigned char *)a.v)[s0 + i] = coded<true>(v[i], uv[i], vt, 254);
    }
    if (lane == 0) a.m_top[s0 / kAdamBlock] = mt, a.v_top[s0 / kAdamBlock] = vt;
  }
}

// what 8-bit moments stand for, in bfloat16 (four significant bits: exact); n is a multiple of 256
__global__ void __launch_bounds__(256) adamw_moments_kernel(unsigned short *mv, unsigned short *vv, const unsigned char *m, const unsigned char *v,
                                                            const short *mt, const short *vt, long long n) {
  const long long i = (long long)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;
  const float a = decoded(m[i] & 127, mt[i / kAdamBlock], 126, kNan), b = decoded(v[i], vt[i / kAdamBlock], 254, kInf);
  mv[i] = __float_as_uint(m[i] & 128 ? -a : a) >> 16;
  vv[i] = __float_as_uint(b) >> 16;
}

// 8-bit moments nearest to given values
__global__ void __launch_bounds__(256) adamw_set_moments_kernel(unsigned char *m, unsigned char *v, short *m_top, short *v_top, const float *mv,
                                                                const float *vv, long long n) {
  const long long wave = (long long)blockIdx.x * 4 + threadIdx.x / 64, s0 = wave * kAdamBlock + threadIdx.x % 64 * 4;
  if (s0 >= n) return;
  int um[4], uv[4], mt = 0, vt = 0;
  for (int i = 0; i < 4; i++) {
    um[i] = upper(mv[s0 + i], 1u << 19), uv[i] = upper(vv[s0 + i], 1u << 19);
    mt = max(mt, um[i]), vt = max(vt, uv[i]);
  }
  mt = wave_max(mt), vt = wave_max(vt);
  for (int i = 0; i < 4; i++) {
    const int c = coded<false>(mv[s0 + i], um[i], mt, 126);
    m[s0 + i] = c | (c && __float_as_uint(mv[s0 + i]) >> 31 ? 128 : 0);
    v[s0 + i] = coded<true>(vv[s0 + i], uv[i], vt, 254);
  }
  if (threadIdx.x % 64 == 0) m_top[wave] = mt, v_top[wave] = vt;
}

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "AdamW launch");
}

}  // namespace

int launch_adamw(int n, const AdamTensor *tensors, const AdamArgs &a, hipStream_t s) {
  AdamTable tab;
  std::memset(&tab, 0, sizeof(tab));
  auto flush = [&]() {
    if (tab.count == 0) return 0;
    const dim3 grid((tab.blocks + 3) / 4);
    if (a.dtype == GELIB_HIP_F32) {
      if (a.bits == 32) hipLaunchKernelGGL((adamw_kernel<float, 32>), grid, dim3(256), 0, s, tab, a);
      else hipLaunchKernelGGL((adamw_kernel<float, 8>), grid, dim3(256), 0, s, tab, a);
    } else {
      if (a.bits == 32) hipLaunchKernelGGL((adamw_kernel<bhalf_t, 32>), grid, dim3(256), 0, s, tab, a);
      else hipLaunchKernelGGL((adamw_kernel<bhalf_t, 8>), grid, dim3(256), 0, s, tab, a);
    }
    tab.count = 0, tab.blocks = 0;
    return launched();
  };
  // A launch has at most 2^26 waves (2^32 threads are HIP's limit), a larger parameter several.
  const long long most = 1LL << 25;
  const size_t elem = dtype_bytes(a.dtype);
  for (int k = 0; k < n; k++)
    for (long long done = 0; done < tensors[k].n;) {
      const AdamTensor &from = tensors[k];
      const long long left = from.n - done, now = std::min(left, most * kAdamBlock), blocks = (now + kAdamBlock - 1) / kAdamBlock;
      if (tab.count == kAdamTensors || tab.blocks + blocks > most)
        if (int rc = flush()) return rc;
      auto &t = tab.t[tab.count];
      t.p = (char *)from.p + done * elem, t.g = (const char *)from.g + done * elem, t.n = now;
      t.first = (unsigned)((from.first + done) / kAdamBlock), t.blocks_before = tab.blocks;
      t.step_size = from.step_size, t.inv_sqrt_bc2 = from.inv_sqrt_bc2, t.key = from.key;
      tab.blocks += (unsigned)blocks;
      tab.count++;
      done += now;
    }
  return flush();
}

int launch_adamw_moments(void *mv, void *vv, const void *m, const void *v, const short *mt, const short *vt, long long n, hipStream_t s) {
  const long long most = 1LL << 31;   // elements of a launch
  for (long long i = 0; i < n; i += most)
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)((std::min(n - i, most) + 255) / 256)), dim3(256), 0, s, (unsigned short *)mv + i,
                       (unsigned short *)vv + i, (const unsigned char *)m + i, (const unsigned char *)v + i, mt + i / kAdamBlock,
                       vt + i / kAdamBlock, std::min(n - i, most));
  return launched();
}

int launch_adamw_set_moments(void *m, void *v, short *mt, short *vt, const float *mv, const float *vv, long long n, hipStream_t s) {
  const long long most = 1LL << 31;
  for (long long i = 0; i < n; i += most)
    hipLaunchKernelGGL(adamw_set_moments_kernel, dim3((unsigned)((std::min(n - i, most) / kAdamBlock + 3) / 4)), dim3(256), 0, s,
                       (unsigned char *)m + i, (unsigned char *)v + i, mt + i / kAdamBlock, vt + i / kAdamBlock, mv + i, vv + i, std::min(n - i, most));
  return launched();
}

}  // namespace gelib_hip
