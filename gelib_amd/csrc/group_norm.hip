// Group norm with an activation (group_norm_impl.h): how a call's tensors are cut into blocks, and simple kernels for what those do
// not take (one block cannot hold a row of the channels that a group and the loads' alignment ask for: groups of more than 256
// loads, 2048 bfloat16 channels; 512 where samples are short).
#include "group_norm_impl.h"

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

// a block per (sample, group)
template <typename T, int ACT>
__global__ void __launch_bounds__(256) norm_wide_fwd(const NormArgs a, long long base) {
  __shared__ float lds[4];
  const long long tile = base + blockIdx.x, n = tile / a.G;
  const int g = (int)(tile % a.G), cg = a.C / a.G, c0 = g * cg;
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
  if (a.mean && threadIdx.x == 0) a.mean[tile] = mean, a.rstd[tile] = rstd;
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
__global__ void __launch_bounds__(256) norm_wide_gx(const NormArgs a, long long base) {
  __shared__ float lds[4];
  const long long tile = base + blockIdx.x, n = tile / a.G;
  const int g = (int)(tile % a.G), cg = a.C / a.G, c0 = g * cg;
  const long long len = length_of(a, n), cnt = len * cg;
  const T *x = (const T *)a.x + n * a.xs + c0, *gy = (const T *)a.gy + n * a.S * a.C + c0;
  T *gx = (T *)a.y + n * a.S * a.C + c0;
  const float mean = a.mean[tile], rstd = a.rstd[tile];
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

// a block per 64 channels: four rows at a time
template <typename T, int ACT>
__global__ void __launch_bounds__(256) norm_wide_gw(const NormArgs a) {
  __shared__ float lds[2][4][64];
  const int c = blockIdx.x * 64 + threadIdx.x % 64, row = threadIdx.x / 64;
  float sw = 0.f, sb = 0.f;
  if (c < a.C) {
    const int g = c / (a.C / a.G);
    const float w = a.w ? to_f(((const T *)a.w)[c]) : 1.f, b = a.b ? to_f(((const T *)a.b)[c]) : 0.f;
    for (long long n = 0; n < a.N; n++) {
      const long long len = length_of(a, n);
      const float mean = a.mean[n * a.G + g], rstd = a.rstd[n * a.G + g];
      const T *x = (const T *)a.x + n * a.xs + c, *gy = (const T *)a.gy + n * a.S * a.C + c;
      // (samples of one position go to the rows in turn, the positions of longer ones)
      const long long first = a.S == 1 ? (n % 4 == row ? 0 : len) : row;
#pragma unroll 4
      for (long long s = first; s < len; s += 4) {
        const float xh = (to_f(x[s * a.xp]) - mean) * rstd, gz = to_f(gy[s * a.C]) * act_slope<ACT>(xh * w + b);
        sw += gz * xh, sb += gz;
      }
    }
  }
  lds[0][row][threadIdx.x % 64] = sw, lds[1][row][threadIdx.x % 64] = sb;
  __syncthreads();
  if (row == 0 && c < a.C) {
    const int t = threadIdx.x;
    if (a.gw) ((T *)a.gw)[c] = from_f<T>((lds[0][0][t] + lds[0][1][t]) + (lds[0][2][t] + lds[0][3][t]));
    if (a.gb) ((T *)a.gb)[c] = from_f<T>((lds[1][0][t] + lds[1][1][t]) + (lds[1][2][t] + lds[1][3][t]));
  }
}

template <typename T, int ACT>
int run_wide(bool backward, const NormArgs &a, hipStream_t s) {
  const long long tiles = a.N * a.G, most = 1LL << 23;   // blocks of a launch
  for (long long t = 0; t < tiles; t += most) {
    const dim3 grid((unsigned)std::min(most, tiles - t));
    if (!backward) hipLaunchKernelGGL((norm_wide_fwd<T, ACT>), grid, dim3(256), 0, s, a, t);
    else if (a.y) hipLaunchKernelGGL((norm_wide_gx<T, ACT>), grid, dim3(256), 0, s, a, t);
  }
  if (backward && (a.gw || a.gb)) hipLaunchKernelGGL((norm_wide_gw<T, ACT>), dim3((a.C + 63) / 64), dim3(256), 0, s, a);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "group norm launch");
}

template <typename T>
int run_wide_act(bool backward, const NormArgs &a, hipStream_t s) {
  switch (a.act) {
    case kActRelu: return run_wide<T, kActRelu>(backward, a, s);
    case kActSilu: return run_wide<T, kActSilu>(backward, a, s);
    case kActGelu: return run_wide<T, kActGelu>(backward, a, s);
  }
  return run_wide<T, kActNone>(backward, a, s);
}

// How a call is cut; false where one block cannot hold a row of the channels that belong together.
bool plan_norm(bool backward, int V, int e, long long N, long long S, int C, int G, NormPlan *out) {
  NormPlan p = {};
  const int cg = C / G, Cq = V / std::gcd(V, cg) * cg, quanta = C / Cq;   // Cq: whole groups and whole loads
  if (Cq / V > kNormMostT) return false;
  p.V = V;
  auto stripes_of = [&](int per) {   // stripes of about `per` quanta, as even as they can be
    per = std::max(1, std::min(per, quanta));
    p.stripes = (quanta + per - 1) / per;
    p.Cw = (quanta + p.stripes - 1) / p.stripes * Cq;
    p.stripes = (C + p.Cw - 1) / p.Cw;
    p.TX = p.Cw / V;
  };
  stripes_of((128 / e + Cq - 1) / Cq);
  const int down = std::max(1, kNormMostT / p.TX);
  p.NS = 1;
  if (S <= (long long)down * (backward ? kNormMostRBack : kNormMostR)) {
    p.TY = (int)std::min<long long>(S, down);
    p.R = (int)((S + p.TY - 1) / p.TY);
    // several small samples a block, as long as 512 blocks are left
    p.NS = (int)std::max<long long>(1, std::min<long long>(256 / (p.TX * p.TY), N * p.stripes / 512));
    const long long sets = (N + p.NS - 1) / p.NS;
    // forward: a block a set; backward: about a thousand blocks walk over the sets, each with one row of sums for gw and gb
    p.blocks = std::min<long long>(sets, backward ? std::max(1, 1024 / p.stripes) : 1 << 22);
  } else {
    stripes_of(std::min(256, std::max(64, Cq / V)) * V / Cq);
    p.TY = kNormChunkT / p.TX;
    if (p.TY == 0) return false;
    int r = kNormMostR;
    while (r > 1 && N * ((S + (long long)r * p.TY - 1) / ((long long)r * p.TY)) * p.stripes < 512) r /= 2;
    p.rows = (long long)r * p.TY;
    p.chunks = (S + p.rows - 1) / p.rows;
    if (p.chunks > 1 << 22) return false;
  }
  p.T = (p.TX * p.TY * p.NS + 63) / 64 * 64;
  *out = p;
  return p.stripes <= 65535;
}

struct NormSpace {
  size_t stats = 0, sums = 0, means = 0, total = 0;   // offsets of the last two in front of them
};
NormSpace space_of(bool backward, const NormPlan &p, long long N, int C, int G) {
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  NormSpace r;
  const size_t stats = p.R ? 0 : up((size_t)N * p.chunks * 8 * (backward ? C : G));
  r.sums = stats;
  const size_t sums = !backward ? 0 : up((size_t)(p.R ? p.blocks : N) * C * 8);
  r.means = r.sums + sums;
  r.total = r.means + (p.R ? 0 : up((size_t)N * G * 8));   // (forward: means and rstds of a call that keeps none)
  return r;
}

// the widest load that every row of a call allows
int load_width(const NormArgs &a, int e) {
  const uintptr_t p = (uintptr_t)a.x | (uintptr_t)a.y | (uintptr_t)a.gy;
  for (int V : {16 / e, 2})
    if (a.C % V == 0 && a.xs % V == 0 && a.xp % V == 0 && p % (V * e) == 0) return V;
  return 1;
}

template <typename T>
int run_empty(const NormArgs &a, hipStream_t s) {
  hipLaunchKernelGGL((norm_join<T>), dim3((2 * a.C + 31) / 32), dim3(256), 0, s, (const float *)nullptr, (T *)a.gw, (T *)a.gb, 0LL, a.C);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "group norm launch");
}

}  // namespace

size_t norm_workspace(bool backward, int dtype, long long N, long long S, int C, int G) {
  if (N == 0 || S == 0) return 0;
  const int e = (int)dtype_bytes(dtype);
  size_t most = 0;
  for (int V : {16 / e, 2, 1}) {
    NormPlan p;
    if (C % V == 0 && plan_norm(backward, V, e, N, S, C, G, &p)) most = std::max(most, space_of(backward, p, N, C, G).total);
  }
  return most;
}

int launch_norm(bool backward, int dtype, const NormArgs &a, hipStream_t s) {
  const bool sums = backward && (a.gw || a.gb);
  if (a.N == 0 || a.S == 0) {
    if (!sums) return 0;
    return dtype == GELIB_HIP_F32 ? run_empty<float>(a, s) : dtype == GELIB_HIP_BF16 ? run_empty<bhalf_t>(a, s) : run_empty<half_t>(a, s);
  }
  if (backward && !sums && !a.y) return 0;
  const int e = (int)dtype_bytes(dtype);
  NormDev d = {};
  d.a = a;
  if (!plan_norm(backward, load_width(a, e), e, a.N, a.S, a.C, a.G, &d.p))
    return dtype == GELIB_HIP_F32 ? run_wide_act<float>(backward, a, s) : dtype == GELIB_HIP_BF16 ? run_wide_act<bhalf_t>(backward, a, s) : run_wide_act<half_t>(backward, a, s);
  const NormSpace sp = space_of(backward, d.p, a.N, a.C, a.G);
  char *ws = (char *)a.ws;
  if (!d.p.R) d.stats = (float *)ws;
  if (sums || (backward && !d.p.R)) d.sums = (float *)(ws + sp.sums);
  if (!d.p.R && backward) d.means = (float *)(ws + sp.means);
  if (!d.p.R && !backward && !a.mean) d.a.mean = (float *)(ws + sp.means), d.a.rstd = d.a.mean + a.N * a.G;
  return dtype == GELIB_HIP_F32 ? launch_norm_typed<float>(backward, d, s) : dtype == GELIB_HIP_BF16 ? launch_norm_typed<bhalf_t>(backward, d, s)
                                                                                                     : launch_norm_typed<half_t>(backward, d, s);
}

}  // namespace gelib_hip
