// One AdamW step over all parameters of an optimizer, moments in 32 or in 8 bits:
//     m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2,   p = p - lr decay p - step_size m / (sqrt(v) inv_sqrt_bc2 + eps)
// with step_size = lr / (1 - b1^t), inv_sqrt_bc2 = (1 - b2^t)^-1/2; complex parameters are twice as many reals.
//
// Every parameter owns a run of the moment arrays that starts at a multiple of 256 elements; a block of 256 elements is what
// one scale is kept for in 8 bits.  Half a wave owns such a block, 8 elements a lane in loads of up to 16 bytes, and needs nobody
// else: the maximum is a reduction over 32 lanes.  The parameter that a wave works on is found by all lanes at once (one entry
// of the table each).
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
//
// What bounds it: HBM.  40 M float32 parameters in 300 tensors, moments in 32 bits: 28 bytes an element in 240 us, 4.7 TB/s (a copy of
// 1 GiB reaches 4.8); 128 M bfloat16 parameters, moments in 32 bits: 22 bytes an element in 527 us, 5.3 TB/s.  128 M bfloat16 parameters,
// moments in 8 bits: 10 bytes an element in .33 ms, 3.9 TB/s (a pass with the moments told 441 us, 115 of it for telling them), where the
// vector unit is close behind: about 100 instructions an element, of which 3 multiplications of whole numbers at a quarter of the
// rate (with every test for what is not finite made for every element, and a fourth multiplication, 128 and .35 ms).  40 M float32
// or complex64's reals, moments in 8 bits: 164 us with the moments told.
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
    unsigned first, waves_before;  // first block of moments, waves of the launch before this parameter
    int aligned;                   // p and g start at multiples of 16 bytes
    float step_size, inv_sqrt_bc2;
    unsigned key;
  } t[kAdamTensors];
  int count;
  unsigned waves;
};

constexpr unsigned kMixA = 2654435769u, kMixB = 3144134277u, kMixC = 1779033703u;   // 2^32 / golden ratio, 2^32 (sqrt 3 - 1) and the like: odd numbers
// of h = (index + key) kMixA, which a lane forms once for its eight neighbouring elements
__device__ __forceinline__ unsigned mixed(unsigned h) {
  h = (h ^ (h >> 15)) * kMixB;
  h = (h ^ (h >> 13)) * kMixC;
  return h ^ (h >> 16);
}
__device__ __forceinline__ unsigned mixed_more(unsigned h) {
  h *= kMixA;
  return (h ^ (h >> 15)) & 0xffffu;
}

__device__ __forceinline__ int half_wave_max(int v) {
#pragma unroll
  for (int d = 16; d >= 1; d >>= 1) v = max(v, __shfl_xor(v, d));
  return v;
}

constexpr unsigned kInf = 0x7f800000u;
constexpr unsigned kNan = 0x7fc00000u;
constexpr int kTopOfFinite = 2039;   // u of the largest finite float; rounding up past it stays there

// A block's top is at least steps + 1 (2^-111 for m, 2^-95 for v: what is below is as good as zero), so codes are only ever zero for
// values that round to it.
__device__ __forceinline__ unsigned decoded(int code, int top, int steps, unsigned not_finite) {
  return code == 0 ? 0u : code > steps ? not_finite : (unsigned)(code + top - steps) << 20;
}
// the same where the lane has no code for what is not finite: base = (top - steps) << 20
__device__ __forceinline__ unsigned decoded_finite(unsigned code, unsigned base) { return code ? (code << 20) + base : 0u; }

// u of a value, -1 where it is not finite
__device__ __forceinline__ int upper(float x, unsigned r) {
  const unsigned b = __float_as_uint(x) & 0x7fffffffu;
  return b >= kInf ? -1 : min((int)((b + r) >> 20), kTopOfFinite);
}
template <bool ABOVE, bool FINITE = false>
__device__ __forceinline__ unsigned coded(int u, int top, int steps) {
  return !FINITE && u < 0 ? steps + 1 : max(u - top + steps, ABOVE ? min(u, 1) : 0);
}
// the bytes of a lane's eight elements; x: m, whose signs they keep
template <bool FINITE>
__device__ __forceinline__ void coded8(const float *x, const int *um, const int *uv, int mt, int vt, uint2 &cm, uint2 &cv) {
  cm = cv = make_uint2(0, 0);
#pragma unroll
  for (int i = 0; i < 8; i++) {
    const unsigned c = coded<false, FINITE>(um[i], mt, 126);
    (i < 4 ? cm.x : cm.y) |= (c | (__float_as_uint(x[i]) >> 24 & (c ? 128u : 0u))) << (i % 4 * 8);
    (i < 4 ? cv.x : cv.y) |= coded<true, FINITE>(uv[i], vt, 254) << (i % 4 * 8);
  }
}
__device__ __forceinline__ unsigned code_of(uint2 w, int i) { return (i < 4 ? w.x : w.y) >> (i % 4 * 8) & 255u; }

constexpr int kAdamLane = 8;   // elements of a lane: 32 lanes a block

template <typename T>
__device__ __forceinline__ void load8(const T *p, bool whole, long long n, float *v) {
  if (whole) {
    T t[kAdamLane];
    __builtin_memcpy(t, __builtin_assume_aligned(p, 16), sizeof(t));
#pragma unroll
    for (int i = 0; i < kAdamLane; i++) v[i] = to_f(t[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kAdamLane; i++) v[i] = i < n ? to_f(p[i]) : 0.f;
  }
}

template <typename T, int BITS>
__global__ void __launch_bounds__(256) adamw_kernel(const AdamTable tab, const AdamArgs a) {
  const unsigned lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + threadIdx.x / 64);
  if (wave >= tab.waves) return;
  const auto *t = (const AdamTable *)__builtin_amdgcn_kernarg_segment_ptr();
  const int k = __popcll(__ballot((int)lane < tab.count && t->t[lane].waves_before <= wave)) - 1;
  const auto &e = t->t[k];
  const long long at = ((long long)(wave - e.waves_before) * 64 + lane) * kAdamLane;   // element of the parameter
  const long long s0 = (long long)e.first * kAdamBlock + at;
  const long long left = e.n - at;             // may be below zero: a lane whose elements pad the last block, or lie behind it
  const bool own = at < (e.n + kAdamBlock - 1) / kAdamBlock * kAdamBlock;   // the moments are this parameter's
  const bool whole = left >= kAdamLane && e.aligned;
  T *p = (T *)e.p + at;
  const T *g = (const T *)e.g + at;
  float m[kAdamLane], v[kAdamLane], gr[kAdamLane], was[kAdamLane];
  load8(g, whole, left, gr);
  load8((const T *)p, whole, left, was);
  int mt = 0, vt = 0;
  if (BITS == 32) {
    load8((const float *)a.m + s0, own, 0, m);
    load8((const float *)a.v + s0, own, 0, v);
  } else {
    uint2 cm = {}, cv = {};
    if (own) {
      cm = *(const uint2 *)((const char *)a.m + s0), cv = *(const uint2 *)((const char *)a.v + s0);
      mt = a.m_top[s0 / kAdamBlock], vt = a.v_top[s0 / kAdamBlock];
    }
    // a byte of seven set bits (m), of eight (v): adding one to the seven carries into the eighth
    const unsigned ones = 0x01010101u, low = 0x7f7f7f7fu;
    const bool odd = ((((cm.x & low) + ones) | ((cm.y & low) + ones) | (((cv.x & low) + ones) & cv.x) | (((cv.y & low) + ones) & cv.y)) & ~low) != 0;
    if (__builtin_expect(__any(odd), 0)) {
#pragma unroll
      for (int i = 0; i < kAdamLane; i++) {
        const unsigned c = code_of(cm, i);
        m[i] = __uint_as_float(decoded(c & 127, mt, 126, kNan) | (c & 128) << 24);
        v[i] = __uint_as_float(decoded(code_of(cv, i), vt, 254, kInf));
      }
    } else {
      const unsigned mbase = (unsigned)(mt - 126) << 20, vbase = (unsigned)(vt - 254) << 20;
#pragma unroll
      for (int i = 0; i < kAdamLane; i++) {
        const unsigned c = code_of(cm, i);
        m[i] = __uint_as_float(decoded_finite(c & 127, mbase) | (c & 128) << 24);
        v[i] = __uint_as_float(decoded_finite(code_of(cv, i), vbase));
      }
    }
  }
  unsigned h[kAdamLane];
  // (a lane's eight elements share the upper half of their index)
  const unsigned h0 = ((unsigned)s0 + e.key + (unsigned)(s0 >> 32) * kMixB) * kMixA;
  float now[kAdamLane], odd = 0.f;
#pragma unroll
  for (int i = 0; i < kAdamLane; i++) {
    m[i] = m[i] * a.b1 + gr[i] * a.c1;
    v[i] = v[i] * a.b2 + (gr[i] * gr[i]) * a.c2;
    if (BITS == 8 || sizeof(T) == 2) h[i] = mixed(h0 + i * kMixA);
    const float denom = sqrtf(v[i]) * e.inv_sqrt_bc2 + a.eps;
    now[i] = (was[i] - was[i] * a.decay) - (m[i] * e.step_size) / denom;
    if (sizeof(T) == 2) odd = __builtin_fmaf(now[i], 0.f, odd);   // NaN once one of them is not finite
  }
  T out[kAdamLane];
  if constexpr (sizeof(T) == 2) {
    unsigned short r[kAdamLane];
    if (__builtin_expect(__any(odd != 0.f), 0)) {
#pragma unroll
      for (int i = 0; i < kAdamLane; i++) {
        const unsigned b = __float_as_uint(now[i]), u = b & 0x7fffffffu;
        r[i] = u > kInf ? 0x7fc0 : u == kInf ? b >> 16 : (b + mixed_more(h[i])) >> 16;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kAdamLane; i++) r[i] = (__float_as_uint(now[i]) + mixed_more(h[i])) >> 16;
    }
    __builtin_memcpy(out, r, sizeof(out));
  } else {
    __builtin_memcpy(out, now, sizeof(out));
  }
  if (whole) {
    __builtin_memcpy(__builtin_assume_aligned(p, 16), out, sizeof(out));
  } else {
#pragma unroll
    for (int i = 0; i < kAdamLane; i++)
      if (i < left) p[i] = out[i];
  }
  if (BITS == 32) {
    if (own) {
      __builtin_memcpy(__builtin_assume_aligned((float *)a.m + s0, 16), m, sizeof(m));
      __builtin_memcpy(__builtin_assume_aligned((float *)a.v + s0, 16), v, sizeof(v));
    }
  } else {
    int um[kAdamLane], uv[kAdamLane];
    uint2 cm, cv;
    mt = 127, vt = 255;
#pragma unroll
    for (int i = 0; i < kAdamLane; i++) {
      um[i] = ((__float_as_uint(m[i]) & 0x7fffffffu) + (h[i] & 0xfffffu)) >> 20, uv[i] = (__float_as_uint(v[i]) + (h[i] >> 12)) >> 20;
      mt = max(mt, um[i]), vt = max(vt, uv[i]);
    }
    mt = half_wave_max(mt), vt = half_wave_max(vt);
    if (__builtin_expect(__any(mt > kTopOfFinite || vt > kTopOfFinite), 0)) {   // something is not finite, or rounds up to it
      mt = 127, vt = 255;
#pragma unroll
      for (int i = 0; i < kAdamLane; i++) {
        um[i] = upper(m[i], h[i] & 0xfffffu), uv[i] = upper(v[i], h[i] >> 12);
        if (uv[i] < 0 && um[i] >= 0) um[i] = 0;   // v is infinite: its steps are zero whatever m is, and m as large as that would push
                                                  // the block's others below the smallest code
        mt = max(mt, um[i]), vt = max(vt, uv[i]);
      }
      mt = half_wave_max(mt), vt = half_wave_max(vt);
      coded8<false>(m, um, uv, mt, vt, cm, cv);
    } else {
      coded8<true>(m, um, uv, mt, vt, cm, cv);
    }
    if (own) {
      *(uint2 *)((char *)a.m + s0) = cm, *(uint2 *)((char *)a.v + s0) = cv;
      if (lane % 32 == 0) a.m_top[s0 / kAdamBlock] = mt, a.v_top[s0 / kAdamBlock] = vt;
    }
  }
}

// what 8-bit moments stand for, in bfloat16 (four significant bits: exact); n is a multiple of 256
__global__ void __launch_bounds__(256) adamw_moments_kernel(unsigned short *mv, unsigned short *vv, const unsigned char *m, const unsigned char *v,
                                                            const short *mt, const short *vt, long long n) {
  const long long s0 = ((long long)blockIdx.x * 256 + threadIdx.x) * kAdamLane;
  if (s0 >= n) return;
  const uint2 cm = *(const uint2 *)(m + s0), cv = *(const uint2 *)(v + s0);
  const int tm = mt[s0 / kAdamBlock], tv = vt[s0 / kAdamBlock];
  unsigned short a[kAdamLane], b[kAdamLane];
#pragma unroll
  for (int i = 0; i < kAdamLane; i++) {
    const unsigned c = code_of(cm, i);
    a[i] = decoded(c & 127, tm, 126, kNan) >> 16 | (c & 128) << 8;
    b[i] = decoded(code_of(cv, i), tv, 254, kInf) >> 16;
  }
  __builtin_memcpy(__builtin_assume_aligned(mv + s0, 16), a, 16);
  __builtin_memcpy(__builtin_assume_aligned(vv + s0, 16), b, 16);
}

// 8-bit moments nearest to given values (128 M elements .26 ms)
__global__ void __launch_bounds__(256) adamw_set_moments_kernel(unsigned char *m, unsigned char *v, short *m_top, short *v_top, const float *mv,
                                                                const float *vv, long long n) {
  const long long s0 = ((long long)blockIdx.x * 256 + threadIdx.x) * kAdamLane;
  if (s0 >= n) return;   // (half waves: n is a multiple of 256)
  int um[kAdamLane], uv[kAdamLane], mt = 127, vt = 255;
  float x[kAdamLane], y[kAdamLane];
  load8(mv + s0, true, 0, x);
  load8(vv + s0, true, 0, y);
#pragma unroll
  for (int i = 0; i < kAdamLane; i++) {
    um[i] = upper(x[i], 1u << 19), uv[i] = upper(y[i], 1u << 19);
    mt = max(mt, um[i]), vt = max(vt, uv[i]);
  }
  mt = half_wave_max(mt), vt = half_wave_max(vt);
  uint2 cm, cv;
  coded8<false>(x, um, uv, mt, vt, cm, cv);
  *(uint2 *)(m + s0) = cm, *(uint2 *)(v + s0) = cv;
  if (threadIdx.x % 32 == 0) m_top[s0 / kAdamBlock] = mt, v_top[s0 / kAdamBlock] = vt;
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
    const dim3 grid((tab.waves + 3) / 4);
    if (a.dtype == GELIB_HIP_F32) {
      if (a.bits == 32) hipLaunchKernelGGL((adamw_kernel<float, 32>), grid, dim3(256), 0, s, tab, a);
      else hipLaunchKernelGGL((adamw_kernel<float, 8>), grid, dim3(256), 0, s, tab, a);
    } else {
      if (a.bits == 32) hipLaunchKernelGGL((adamw_kernel<bhalf_t, 32>), grid, dim3(256), 0, s, tab, a);
      else hipLaunchKernelGGL((adamw_kernel<bhalf_t, 8>), grid, dim3(256), 0, s, tab, a);
    }
    tab.count = 0, tab.waves = 0;
    return launched();
  };
  // A launch has at most 2^25 waves, a larger parameter several (from 2^32 threads on HIP runs what is left after that many, and reports nothing).
  const long long most = 1LL << 25;
  const size_t elem = dtype_bytes(a.dtype);
  for (int k = 0; k < n; k++)
    for (long long done = 0; done < tensors[k].n;) {
      const AdamTensor &from = tensors[k];
      const long long left = from.n - done, now = std::min(left, most * 64 * kAdamLane), waves = (now + 64 * kAdamLane - 1) / (64 * kAdamLane);
      if (tab.count == kAdamTensors || tab.waves + waves > most)
        if (int rc = flush()) return rc;
      auto &t = tab.t[tab.count];
      t.p = (char *)from.p + done * elem, t.g = (const char *)from.g + done * elem, t.n = now;
      t.first = (unsigned)((from.first + done) / kAdamBlock), t.waves_before = tab.waves;
      t.step_size = from.step_size, t.inv_sqrt_bc2 = from.inv_sqrt_bc2, t.key = from.key;
      t.aligned = ((uintptr_t)t.p | (uintptr_t)t.g) % 16 == 0;
      tab.waves += (unsigned)waves;
      tab.count++;
      done += now;
    }
  return flush();
}

int launch_adamw_moments(void *mv, void *vv, const void *m, const void *v, const short *mt, const short *vt, long long n, hipStream_t s) {
  const long long most = 1LL << 31;   // elements of a launch
  for (long long i = 0; i < n; i += most)
    hipLaunchKernelGGL(adamw_moments_kernel, dim3((unsigned)((std::min(n - i, most) / kAdamLane + 255) / 256)), dim3(256), 0, s, (unsigned short *)mv + i,
                       (unsigned short *)vv + i, (const unsigned char *)m + i, (const unsigned char *)v + i, mt + i / kAdamBlock,
                       vt + i / kAdamBlock, std::min(n - i, most));
  return launched();
}

int launch_adamw_set_moments(void *m, void *v, short *mt, short *vt, const float *mv, const float *vv, long long n, hipStream_t s) {
  const long long most = 1LL << 31;
  for (long long i = 0; i < n; i += most)
    hipLaunchKernelGGL(adamw_set_moments_kernel, dim3((unsigned)((std::min(n - i, most) / kAdamLane + 255) / 256)), dim3(256), 0, s,
                       (unsigned char *)m + i, (unsigned char *)v + i, mt + i / kAdamBlock, vt + i / kAdamBlock, mv + i, vv + i, std::min(n - i, most));
  return launched();
}

}  // namespace gelib_hip
