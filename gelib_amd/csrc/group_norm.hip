// Group norm with an activation (group_norm_impl.h): how a call's tensors are cut into blocks.
#include "group_norm_impl.h"

namespace gelib_hip {

namespace {

// How a call is cut.
NormPlan plan_norm(bool backward, int V, int e, long long N, long long S, int C, int G) {
  NormPlan p = {};
  p.V = V, p.NS = 1, p.pieces = 1;
  // per: channels a stripe; cg: channels that have to be in one
  auto stripes_of = [&](int per, int cg) {
    const int Cq = V / std::gcd(V, cg) * cg, quanta = C / Cq;   // whole groups (or pieces of them) and whole loads
    const int wanted = std::max(1, std::min((per + Cq - 1) / Cq, quanta));
    p.stripes = (quanta + wanted - 1) / wanted;
    p.Cw = (quanta + p.stripes - 1) / p.stripes * Cq;   // as even as they can be
    p.stripes = (C + p.Cw - 1) / p.Cw;
    p.TX = p.Cw / V;
  };
  stripes_of(128 / e, C / G);
  const int down = kNormMostT / p.TX;
  if (p.TX <= kNormMostT && p.stripes <= 65535 && S <= (long long)down * (backward ? kNormMostRBack : kNormMostR)) {
    p.TY = (int)std::min<long long>(S, down);
    p.R = (int)((S + p.TY - 1) / p.TY);
    // several small samples a block, as long as 512 blocks are left
    p.NS = (int)std::max<long long>(1, std::min<long long>(256 / (p.TX * p.TY), N * p.stripes / 512));
    const long long sets = (N + p.NS - 1) / p.NS;
    // forward: a block a set; backward: about a thousand blocks walk over the sets, each with one row of sums for gw and gb
    p.blocks = std::min<long long>(sets, backward ? std::max(1, 1024 / p.stripes) : 1 << 22);
  } else {
    // groups that a block of 256 loads cannot hold are summed in pieces of as many channels as it can
    const int cg = C / G;
    while (V / std::gcd(V, cg / p.pieces) * (cg / p.pieces) > kNormChunkT * V) {
      do p.pieces++;
      while (cg % p.pieces);
    }
    const int Cq = V / std::gcd(V, cg / p.pieces) * (cg / p.pieces);
    stripes_of(std::max(1, kNormChunkT * V / Cq) * Cq, cg / p.pieces);
    p.TY = kNormChunkT / p.TX;
    int r = kNormMostR;
    while (r > 1 && N * ((S + (long long)r * p.TY - 1) / ((long long)r * p.TY)) * p.stripes < 512) r /= 2;
    p.rows = (long long)r * p.TY;
    p.chunks = (S + p.rows - 1) / p.rows;
  }
  p.T = (p.TX * p.TY * p.NS + 63) / 64 * 64;
  return p;
}

struct NormSpace {
  size_t stats = 0, sums = 0, means = 0, total = 0;   // offsets of the last two in front of them
};
NormSpace space_of(bool backward, const NormPlan &p, long long N, int C, int G) {
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  NormSpace r;
  const size_t stats = p.R ? 0 : up((size_t)N * p.chunks * 8 * (backward ? C : G * p.pieces));
  r.sums = stats;
  const size_t sums = !backward ? 0 : up((size_t)(p.R ? p.blocks : N) * C * 8);
  r.means = r.sums + sums;
  r.total = r.means + (p.R ? 0 : up((size_t)N * G * p.pieces * 8));   // (forward: means and rstds of a call that keeps none)
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
  for (int V : {16 / e, 2, 1})
    if (C % V == 0) most = std::max(most, space_of(backward, plan_norm(backward, V, e, N, S, C, G), N, C, G).total);
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
  d.p = plan_norm(backward, load_width(a, e), e, a.N, a.S, a.C, a.G);
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
