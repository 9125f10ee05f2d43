// Group norm with an activation, channels last: a group is C / G neighbouring channels over the positions of a sample that count,
//     xh = (x - mean) rstd,  y = act(xh w + b);   gz = gy act'(z), q = gz w, gx = rstd (q - mean(q) - xh mean(q xh)),
//     gw = sum gz xh, gb = sum gz over samples and positions.
// Positions behind a sample's length are zero in y and gx and are never read.
//
// A block owns whole groups of one sample (or of several small ones): a stripe of Cw channels, at least 128 bytes of a row, by all
// positions, TX threads of V channels (one load) side by side and TY of them down the positions.  Where a stripe fits a block's
// registers (16 loads a thread, 512 threads: 128 KB) it is read once, and the statistics are formed around the mean from registers;
// the backward pass forms gz twice from what it holds.  Larger samples are cut into chunks of positions: every chunk's mean and sum of
// squares around it (backward: its channel sums), joined by the parallel form of the variance, then a second pass over x, which the
// memory-side cache still holds up to its 256 MB; groups wider than a chunk's block (256 loads a position) are summed in pieces of as
// many channels each, joined like chunks.  What bounds either is HBM; sums go over channels first and groups after, so any channels a
// group will do, and the channel sums are the gradients of w and b.
// No atomics: sums have one order.
//
// Measured (us, bfloat16 unless said; a copy of 1 GiB reaches 4.8 TB/s): 64 x 1024 x 256, whole forward 27 (67 MB: 2.5 TB/s, one block a
// compute unit, so that its loads, two reductions and stores follow one another), backward in chunks 18 + 20 and 9 for the two
// joins; held whole backward it was 180 (410 registers spilled).  24 samples of up to 9216 x 320: statistics 22, y 34, sums 42, gx 52
// (141 MB written by each of y and gx: 4.2 and 2.7 TB/s, the second beside 25 instructions an element and two exponentials'
// worth of silu'), joins 18.  One group of 4096 channels, silu, with the host's part: 64 x 512 forward 168, both 528 (a block a group
// alone: 11900 and 28600); 8192 x 1 forward 148, both 462 (202 and 594).  8192 x 1 x 8192, chunks of one position: 257 and 978.
// 64 x 512 x 4099, loads of one channel: 383 and 910.  32768 x 1 x 64 float32: 14 forward, 18 + 4 backward: six barriers of a block
// one after the other.
#pragma once

#include <numeric>

#include "real_ops.h"

namespace gelib_hip {

struct NormPlan {
  int V, TX, TY, NS, R;       // channels a load; threads across and down; samples of a block; loads a thread holds (0: in chunks)
  int Cw, stripes;            // channels of a block
  int T;                      // threads
  long long rows, chunks;     // positions of a chunk, chunks of a sample (in chunks)
  long long blocks;           // along the samples (whole: they walk over the groups of NS samples)
  int pieces;                 // in chunks: parts of a group that are summed by themselves (groups wider than a block), as many channels each
};

struct NormDev {
  NormArgs a;
  NormPlan p;
  float *stats;   // in chunks, forward: [n][chunk][G pieces] mean and sum of squares; backward: [n][chunk][2][C]
  float *sums;    // backward: [blocks or n][2][C] channel sums of gz xh and of gz
  float *means;   // in chunks, backward: [n][G pieces][2] mean of q and of q xh
  long long first[3];   // in chunks: chunk, stripe and sample of the launch's first block
};

template <typename T>
int launch_norm_typed(bool backward, const NormDev &d, hipStream_t s);

#ifdef __HIPCC__

namespace {

// Most threads of a block, and loads that a thread holds: more than 8 of x and 8 of gy beside the channels' numbers do not fit 256
// registers.  Chunks take 256 threads, three to five blocks a compute unit, so that loads are under way while others reduce.
constexpr int kNormMostT = 512, kNormMostR = 16, kNormMostRBack = 8, kNormChunkT = 256;
constexpr int kNormBatch = 4;   // positions whose loads a thread has under way together in the passes over chunks

template <typename T>
struct Short { typedef T type; };
template <>
struct Short<float> { typedef half_t type; };   // (never converted to)

// A load of V values as the 32-bit words that it is: values are unpacked where they are used, two instructions for two of them.
template <typename T, int V>
struct Pack {
  static constexpr int N = (V * (int)sizeof(T) + 3) / 4;
  unsigned w[N];
  __device__ __forceinline__ float at(int i) const {
    if (sizeof(T) == 4) return __uint_as_float(w[i]);
    const unsigned h = w[i / 2];
    if (__is_same(T, bhalf_t)) return __uint_as_float(i % 2 ? h & 0xffff0000u : h << 16);
    return (float)__builtin_bit_cast(half_t, (unsigned short)(i % 2 ? h >> 16 : h));
  }
  __device__ __forceinline__ void set(const float *v) {
#pragma unroll
    for (int k = 0; k < N; k++) {
      if (sizeof(T) == 4) w[k] = __float_as_uint(v[k]);
      else w[k] = bits(v[2 * k]) | (V > 1 ? (unsigned)bits(v[2 * k + (V > 1)]) << 16 : 0u);
    }
  }
  // Hides where the words come from: the compiler unpacks them again where they are used next, instead of keeping every value in a
  // register of its own from one use to the other (16 loads of 8 values: 128 registers more, and 218 spilled)
  __device__ __forceinline__ void forget() {
#pragma unroll
    for (int k = 0; k < N; k++) asm volatile("" : "+v"(w[k]));
  }

 private:
  static __device__ __forceinline__ unsigned short bits(float v) { return __builtin_bit_cast(unsigned short, from_f<typename Short<T>::type>(v)); }
};
template <typename T, int V>
__device__ __forceinline__ Pack<T, V> load_pack(const T *p) {
  Pack<T, V> r;
  if constexpr (V * sizeof(T) < 4) r.w[0] = *(const unsigned short *)p;
  else __builtin_memcpy(r.w, __builtin_assume_aligned(p, V * sizeof(T)), V * sizeof(T));
  return r;
}
template <typename T, int V>
__device__ __forceinline__ void store_pack(T *p, const Pack<T, V> &r) {
  if constexpr (V * sizeof(T) < 4) *(unsigned short *)p = (unsigned short)r.w[0];
  else __builtin_memcpy(__builtin_assume_aligned(p, V * sizeof(T)), r.w, V * sizeof(T));
}

__device__ __forceinline__ long long length_of(const NormArgs &a, long long n) {
  return a.lengths ? max(0LL, min((long long)a.lengths[n], a.S)) : a.S;
}

// Where a thread stands: its first channel in the stripe and in the row, its place down the positions
struct Place {
  int tx, ns, ty, col, c0, cw;   // col: first of its V columns among the block's NS * Cw; cw: channels of this stripe
  bool on;
};
__device__ __forceinline__ Place place_of(const NormDev &d) {
  Place w;
  const int t = threadIdx.x, rest = t / d.p.TX;
  w.tx = t - rest * d.p.TX;
  w.ty = rest / d.p.NS;
  w.ns = rest - w.ty * d.p.NS;
  w.c0 = ((int)d.first[1] + blockIdx.y) * d.p.Cw;
  w.cw = min(d.p.Cw, d.a.C - w.c0);
  w.col = w.ns * d.p.Cw + w.tx * d.p.V;
  w.on = w.ty < d.p.TY && w.tx * d.p.V < w.cw;
  return w;
}

// Sums of v over the threads down the positions, one for every column, into out[column] (out and scratch: columns * TY floats and
// columns * parts).  All threads take part.
template <int V>
__device__ __forceinline__ void column_sums(const NormDev &d, const Place &w, const float *v, float *lds, float *out) {
  const int cols = d.p.NS * d.p.Cw, t = threadIdx.x;
  __syncthreads();
  if (d.p.TY == 1) {
    if (w.ty == 0) {
#pragma unroll
      for (int i = 0; i < V; i++) out[w.col + i] = v[i];
    }
    __syncthreads();
    return;
  }
  if (w.ty < d.p.TY) {
#pragma unroll
    for (int i = 0; i < V; i++) lds[w.ty * cols + w.col + i] = v[i];
  }
  __syncthreads();
  const int parts = max(1, min(d.p.TY, d.p.T / cols));
  if (parts == 1) {
    for (int c = t; c < cols; c += d.p.T) {
      float s = 0.f;
      for (int k = 0; k < d.p.TY; k++) s += lds[k * cols + c];
      out[c] = s;
    }
    __syncthreads();
    return;
  }
  const int c = t % cols, part = t / cols;
  float s = 0.f;
  if (part < parts) {
    for (int k = part; k < d.p.TY; k += parts) s += lds[k * cols + c];
  }
  __syncthreads();
  if (part < parts) lds[part * cols + c] = s;
  __syncthreads();
  if (t < cols) {
    for (int k = 1; k < parts; k++) s += lds[k * cols + t];
    out[t] = s;
  }
  __syncthreads();
}

// of[g] = f(sum over the columns of group g of in), for the NS * groups of the block; f(group, sum)
template <typename F>
__device__ __forceinline__ void group_sums(const NormDev &d, const Place &w, const float *in, F f) {
  const int cg = d.a.C / d.a.G, gs = w.cw / cg, groups = d.p.NS * gs;
  if (cg <= 16) {
    for (int g = threadIdx.x; g < groups; g += d.p.T) {
      const float *p = in + g / gs * d.p.Cw + g % gs * cg;
      float s = 0.f;
      for (int i = 0; i < cg; i++) s += p[i];
      f(g, s);
    }
  } else if (groups < d.p.T / 64) {   // fewer groups than waves: all of them at every group (one wave took 3 us for 4096 channels)
    __shared__ float part[kNormMostT / 64];
    for (int g = 0; g < groups; g++) {
      const float *p = in + g / gs * d.p.Cw + g % gs * cg;
      float s = 0.f;
      for (int i = threadIdx.x; i < cg; i += d.p.T) s += p[i];
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m);
      if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = s;
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int k = 1; k < d.p.T / 64; k++) s += part[k];
        f(g, s);
      }
      __syncthreads();
    }
  } else {
    const int waves = d.p.T / 64, lane = threadIdx.x % 64;
    for (int g = threadIdx.x / 64; g < groups && (int)threadIdx.x / 64 < waves; g += waves) {
      const float *p = in + g / gs * d.p.Cw + g % gs * cg;
      float s = 0.f;
      for (int i = lane; i < cg; i += 64) s += p[i];
#pragma unroll
      for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m);
      if (lane == 0) f(g, s);
    }
  }
  __syncthreads();
}

// a thread's channels of w or b: one load where the array is aligned for it
template <typename T, int V>
__device__ __forceinline__ void load_channels(const void *from, const Place &w, float otherwise, float *v) {
#pragma unroll
  for (int i = 0; i < V; i++) v[i] = otherwise;
  if (!from) return;
  const T *p = (const T *)from + w.c0 + (w.on ? w.tx * V : 0);
  if ((uintptr_t)from % (V * sizeof(T)) == 0) {
    const Pack<T, V> k = load_pack<T, V>(p);
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = k.at(i);
  } else {
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = to_f(p[i]);
  }
}
// the group of each of a thread's channels, counted from the stripe's first (0 for threads without channels): one division
template <int V>
__device__ __forceinline__ void groups_of(const NormDev &d, const Place &w, int *g) {
  const int cg = d.a.C / d.a.G, first = w.on ? w.tx * V : 0;
  int at = first / cg, left = cg - (first - at * cg);
#pragma unroll
  for (int i = 0; i < V; i++) {
    g[i] = at;
    if (--left == 0) at++, left = cg;
  }
}

// the group of each of a thread's channels, of the sample's: stripes may begin inside a group in the passes that only look groups up
template <int V>
__device__ __forceinline__ void groups_in_row(const NormDev &d, const Place &w, int *g) {
  const int cg = d.a.C / d.a.G, first = w.on ? w.c0 + w.tx * V : 0;
  int at = first / cg, left = cg - (first - at * cg);
#pragma unroll
  for (int i = 0; i < V; i++) {
    g[i] = at;
    if (--left == 0) at++, left = cg;
  }
}

extern __shared__ float norm_lds[];

// Statistics of what the threads hold in xr (R loads each, those at positions below len count): mean and sum of squares around it of
// every group of the block, in mean[] and square[].
template <typename T, int V, int R>
__device__ __forceinline__ void block_stats(const NormDev &d, const Place &w, const int *g, Pack<T, V> *xr, long long len, float *scratch, float *chan, float *mean,
                                            float *square) {
  float s[V] = {};
#pragma unroll
  for (int r = 0; r < R; r++)
    if (w.on && w.ty + (long long)r * d.p.TY < len) {
#pragma unroll
      for (int i = 0; i < V; i++) s[i] += xr[r].at(i);
    }
  // (a sample's length: every group of it has the same count)
  float *lens = square + d.p.NS * (d.p.Cw / (d.a.C / d.a.G));
  if (w.tx == 0 && w.ty == 0) lens[w.ns] = (float)len;
  column_sums<V>(d, w, s, scratch, chan);
  const int cg = d.a.C / d.a.G, gs = w.cw / cg;
  group_sums(d, w, chan, [&](int k, float sum) { mean[k] = lens[k / gs] > 0.f ? sum / (lens[k / gs] * (float)cg) : 0.f; });
#pragma unroll
  for (int i = 0; i < V; i++) s[i] = 0.f;
#pragma unroll
  for (int r = 0; r < R; r++) xr[r].forget();
  float mu[V];
#pragma unroll
  for (int i = 0; i < V; i++) mu[i] = mean[w.ns * gs + g[i]];
#pragma unroll
  for (int r = 0; r < R; r++)
    if (w.on && w.ty + (long long)r * d.p.TY < len) {
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float e = xr[r].at(i) - mu[i];
        s[i] += e * e;
      }
    }
  column_sums<V>(d, w, s, scratch, chan);
  group_sums(d, w, chan, [&](int k, float sum) { square[k] = sum; });
}

// LDS of a block: partial column sums, two sets of column sums, two numbers a group, a length a sample
inline size_t norm_lds_bytes(const NormPlan &p, int cg) {
  const size_t cols = (size_t)p.NS * p.Cw;
  return (cols * p.TY + 2 * cols + 2 * (size_t)p.NS * (p.Cw / cg) + p.NS) * 4;
}
struct Lds {
  float *scratch, *chan, *chan2, *first, *second;
};
__device__ __forceinline__ Lds lds_of(const NormDev &d) {
  const int cols = d.p.NS * d.p.Cw;
  Lds l;
  l.scratch = norm_lds, l.chan = l.scratch + cols * d.p.TY, l.chan2 = l.chan + cols, l.first = l.chan2 + cols;
  l.second = l.first + d.p.NS * (d.p.Cw / (d.a.C / d.a.G));
  return l;
}

template <typename T, int V, int ACT, int R>
__global__ void __launch_bounds__(kNormMostT) norm_whole_fwd(const NormDev d) {
  const Place w = place_of(d);
  const Lds l = lds_of(d);
  const NormArgs &a = d.a;
  const int cg = a.C / a.G, gs = w.cw / cg;
  float W[V], B[V];
  int g[V];
  load_channels<T, V>(a.w, w, 1.f, W);
  load_channels<T, V>(a.b, w, 0.f, B);
  groups_of<V>(d, w, g);
  for (long long n0 = (long long)blockIdx.x * d.p.NS; n0 < a.N; n0 += (long long)gridDim.x * d.p.NS) {
    const long long n = n0 + w.ns;
    const bool on = w.on && n < a.N;
    const long long len = n < a.N ? length_of(a, n) : 0;
    const T *x = (const T *)a.x + n * a.xs + w.c0 + w.tx * V;
    Pack<T, V> xr[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      const long long s = w.ty + (long long)r * d.p.TY;
      if (on && s < len) xr[r] = load_pack<T, V>(x + s * a.xp);
    }
    block_stats<T, V, R>(d, w, g, xr, len, l.scratch, l.chan, l.first, l.second);
    float mu[V], k[V];
#pragma unroll
    for (int i = 0; i < V; i++) {
      const int at_g = w.ns * gs + g[i];
      mu[i] = l.first[at_g];
      const float cnt = (float)len * (float)cg;
      k[i] = 1.f / sqrtf((cnt > 0.f ? l.second[at_g] / cnt : 0.f) + a.eps);
      if (a.mean && on && w.ty == 0 && (i ? g[i] != g[i - 1] : w.tx * V == g[0] * cg)) {
        const long long at = n * a.G + w.c0 / cg + g[i];
        a.mean[at] = mu[i], a.rstd[at] = k[i];
      }
      k[i] *= W[i];
    }
    T *y = (T *)a.y + n * a.S * a.C + w.c0 + w.tx * V;
#pragma unroll
    for (int r = 0; r < R; r++) {
      const long long s = w.ty + (long long)r * d.p.TY;
      if (!on || s >= a.S) continue;
      float o[V];
      xr[r].forget();
#pragma unroll
      for (int i = 0; i < V; i++) {
        float v, e;
        act_both<ACT>((xr[r].at(i) - mu[i]) * k[i] + B[i], v, e, a.act == kActRelu);
        o[i] = s < len ? v : 0.f;
      }
      xr[r].set(o);
      store_pack<T, V>(y + s * a.C, xr[r]);
    }
    __syncthreads();
  }
}

// xh and gz of one load
template <typename T, int V, int ACT>
__device__ __forceinline__ void gz_of(const Pack<T, V> &x, const Pack<T, V> &gy, const float *mu, const float *k, const float *W, const float *B, bool relu,
                                      float *xh, float *gz) {
#pragma unroll
  for (int i = 0; i < V; i++) {
    float v, e;
    xh[i] = (x.at(i) - mu[i]) * k[i];
    act_both<ACT>(xh[i] * W[i] + B[i], v, e, relu);
    gz[i] = gy.at(i) * e;
  }
}

// adds the NS samples' column sums to a thread's running ones (channel threadIdx.x + j T of the stripe)
template <int J>
__device__ __forceinline__ void keep_sums(const NormDev &d, const Place &w, const float *chan, float *acc) {
#pragma unroll
  for (int j = 0; j < J; j++) {
    const int c = threadIdx.x + j * d.p.T;
    if (c < w.cw) {
      float s = 0.f;   // (a chain of its own: one over all samples rounds as often as it has terms)
      for (int k = 0; k < d.p.NS; k++) s += chan[k * d.p.Cw + c];
      acc[j] += s;
    }
  }
}
// sums of q = gz w and of q xh of the groups, divided by their count, from the column sums of gz and gz xh
template <typename T>
__device__ __forceinline__ void group_means(const NormDev &d, const Place &w, float *chan, float *chan2, const float *lens, float *m1, float *m2) {
  const int cg = d.a.C / d.a.G, gs = w.cw / cg, cols = d.p.NS * d.p.Cw;
  if (d.a.w) {
    for (int c = threadIdx.x; c < cols; c += d.p.T)
      if (c % d.p.Cw < w.cw) {
        const float W = to_f(((const T *)d.a.w)[w.c0 + c % d.p.Cw]);
        chan[c] *= W, chan2[c] *= W;
      }
    __syncthreads();
  }
  auto mean = [&](float *m) { return [=](int k, float sum) { m[k] = lens[k / gs] > 0.f ? sum / (lens[k / gs] * (float)cg) : 0.f; }; };
  group_sums(d, w, chan, mean(m1));
  group_sums(d, w, chan2, mean(m2));
}

template <typename T, int V, int ACT, int R>
__global__ void __launch_bounds__(kNormMostT) norm_whole_bwd(const NormDev d) {
  const Place w = place_of(d);
  const Lds l = lds_of(d);
  const NormArgs &a = d.a;
  const int cg = a.C / a.G, gs = w.cw / cg;
  float W[V], B[V], accw[V] = {}, accb[V] = {};
  int g[V];
  load_channels<T, V>(a.w, w, 1.f, W);
  load_channels<T, V>(a.b, w, 0.f, B);
  groups_of<V>(d, w, g);
  float *lens = l.second + d.p.NS * (d.p.Cw / cg);
  for (long long n0 = (long long)blockIdx.x * d.p.NS; n0 < a.N; n0 += (long long)gridDim.x * d.p.NS) {
    const long long n = n0 + w.ns;
    const bool on = w.on && n < a.N;
    const long long len = n < a.N ? length_of(a, n) : 0;
    const T *x = (const T *)a.x + n * a.xs + w.c0 + w.tx * V, *gy = (const T *)a.gy + n * a.S * a.C + w.c0 + w.tx * V;
    Pack<T, V> xr[R], gr[R];
    float mu[V], k[V], s1[V] = {}, s2[V] = {};
#pragma unroll
    for (int r = 0; r < R; r++) {
      const long long s = w.ty + (long long)r * d.p.TY;
      if (on && s < len) xr[r] = load_pack<T, V>(x + s * a.xp), gr[r] = load_pack<T, V>(gy + s * a.C);
    }
#pragma unroll
    for (int i = 0; i < V; i++) {
      const long long at = n * a.G + w.c0 / cg + g[i];
      mu[i] = on ? a.mean[at] : 0.f, k[i] = on ? a.rstd[at] : 0.f;
    }
#pragma unroll
    for (int r = 0; r < R; r++)
      if (on && w.ty + (long long)r * d.p.TY < len) {
        float xh[V], gz[V];
        gz_of<T, V, ACT>(xr[r], gr[r], mu, k, W, B, a.act == kActRelu, xh, gz);
#pragma unroll
        for (int i = 0; i < V; i++) s1[i] += gz[i], s2[i] += gz[i] * xh[i];
      }
    if (w.tx == 0 && w.ty == 0) lens[w.ns] = (float)len;
    column_sums<V>(d, w, s1, l.scratch, l.chan);
    column_sums<V>(d, w, s2, l.scratch, l.chan2);
    if (d.sums) {
      keep_sums<V>(d, w, l.chan2, accw);
      keep_sums<V>(d, w, l.chan, accb);
      __syncthreads();
    }
    if (a.y) {
      group_means<T>(d, w, l.chan, l.chan2, lens, l.first, l.second);
      float m1[V], m2[V];
#pragma unroll
      for (int i = 0; i < V; i++) m1[i] = l.first[w.ns * gs + g[i]], m2[i] = l.second[w.ns * gs + g[i]];
      T *gx = (T *)a.y + n * a.S * a.C + w.c0 + w.tx * V;
#pragma unroll
      for (int r = 0; r < R; r++) {
        const long long s = w.ty + (long long)r * d.p.TY;
        if (!on || s >= a.S) continue;
        // (gz once more, rather than in registers from above: 128 of them where a thread holds 16 loads)
        float xh[V], gz[V], o[V];
        xr[r].forget(), gr[r].forget();
        gz_of<T, V, ACT>(xr[r], gr[r], mu, k, W, B, a.act == kActRelu, xh, gz);
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = s < len ? k[i] * (gz[i] * W[i] - m1[i] - xh[i] * m2[i]) : 0.f;
        xr[r].set(o);
        store_pack<T, V>(gx + s * a.C, xr[r]);
      }
    }
    __syncthreads();
  }
  if (d.sums) {
    float *to = d.sums + (long long)blockIdx.x * 2 * a.C + w.c0;
#pragma unroll
    for (int j = 0; j < V; j++) {
      const int c = threadIdx.x + j * d.p.T;
      if (c < w.cw) to[c] = accw[j], to[a.C + c] = accb[j];
    }
  }
}

// ---- samples in chunks ----

// mean and sum of squares of a chunk's groups: a block a chunk, stripe and sample
template <typename T, int V>
__global__ void __launch_bounds__(kNormChunkT) norm_chunk_stats(const NormDev d) {
  const Place w = place_of(d);
  const Lds l = lds_of(d);
  const NormArgs &a = d.a;
  const int cg = a.C / a.G;
  const long long n = d.first[2] + blockIdx.z, chunk = d.first[0] + blockIdx.x, s0 = chunk * d.p.rows, len = max(0LL, min(d.p.rows, length_of(a, n) - s0));
  const T *x = (const T *)a.x + n * a.xs + s0 * a.xp + w.c0 + w.tx * V;
  Pack<T, V> xr[kNormMostR];
#pragma unroll
  for (int r = 0; r < kNormMostR; r++) {
    const long long s = w.ty + (long long)r * d.p.TY;
    if (w.on && s < len) xr[r] = load_pack<T, V>(x + s * a.xp);
  }
  int g[V];
  groups_of<V>(d, w, g);
  block_stats<T, V, kNormMostR>(d, w, g, xr, len, l.scratch, l.chan, l.first, l.second);
  float *to = d.stats + ((n * d.p.chunks + chunk) * a.G + w.c0 / cg) * 2;
  for (int k = threadIdx.x; k < w.cw / cg; k += d.p.T) to[2 * k] = l.first[k], to[2 * k + 1] = l.second[k];
}

// The chunks of a sample joined, and the pieces of a group: W waves a group, of the groups from `base` on.  One where they are few; 16
// from 1024 entries on, which groups in many pieces have (64 x 512 x 4099, 131 k entries a group: forward 2280 us with one wave and a
// division an entry, 384 so) and very long samples.
template <int W>
static __global__ void __launch_bounds__(W == 1 ? 256 : 64 * W) norm_stats_join(const NormDev d, long long base) {
  const NormArgs &a = d.a;
  constexpr int kGroups = W == 1 ? 4 : 1, kStep = 64 * W;
  const long long at = base + (long long)blockIdx.x * kGroups + threadIdx.x / kStep, n = at / a.G;
  const int g = (int)(at - n * a.G), t = threadIdx.x % kStep;
  if (n >= a.N) return;   // (whole waves; whole blocks where W is more than one)
  const long long len = length_of(a, n), stride = (long long)a.G * d.p.pieces * 2;
  const int pieces = d.p.pieces, piece = a.C / a.G / pieces;   // channels of a piece
  const float *p = d.stats + n * d.p.chunks * stride + (long long)g * pieces * 2;
  const long long chunks = (len + d.p.rows - 1) / d.p.rows;
  auto all = [](float s) {
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) s += __shfl_xor(s, m);
    if (W > 1) {
      __shared__ float part[W];
      __syncthreads();
      if (threadIdx.x % 64 == 0) part[threadIdx.x / 64] = s;
      __syncthreads();
      s = part[0];
      for (int k = 1; k < W; k++) s += part[k];
    }
    return s;
  };
  // f(count, mean and sum of squares) of every kStep-th entry from t on
  const int down = kStep / pieces, across = kStep - down * pieces;
  auto each = [&](auto f) {
    int q = t % pieces;
    for (long long k = t / pieces; k < chunks;) {
      f((float)min(d.p.rows, len - k * d.p.rows), p + k * stride + 2 * q);
      k += down, q += across;
      if (q >= pieces) q -= pieces, k++;
    }
  };
  // (means around the first one: their sum is as exact as they are)
  const float first = len ? p[0] : 0.f;
  float s = 0.f, q = 0.f;
  each([&](float count, const float *e) { s += count * (e[0] - first); });
  s = all(s);
  const float mean = first + (len ? s / ((float)len * (float)pieces) : 0.f);
  each([&](float count, const float *e) {
    const float off = e[0] - mean;
    q += e[1] + count * (float)piece * off * off;
  });
  q = all(q);
  if (t == 0) a.mean[at] = mean, a.rstd[at] = 1.f / sqrtf((len ? q / ((float)len * (float)(a.C / a.G)) : 0.f) + a.eps);
}

// second pass: y of a chunk
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormChunkT) norm_apply_fwd(const NormDev d) {
  const Place w = place_of(d);
  if (!w.on) return;
  const NormArgs &a = d.a;
  const long long n = d.first[2] + blockIdx.z, chunk = d.first[0] + blockIdx.x, s0 = chunk * d.p.rows, len = length_of(a, n), end = min(s0 + d.p.rows, a.S);
  float B[V], mu[V], k[V];
  int g[V];
  load_channels<T, V>(a.w, w, 1.f, k);
  load_channels<T, V>(a.b, w, 0.f, B);
  groups_in_row<V>(d, w, g);
#pragma unroll
  for (int i = 0; i < V; i++) {
    const long long at = n * a.G + g[i];
    mu[i] = a.mean[at], k[i] *= a.rstd[at];
  }
  const T *x = (const T *)a.x + n * a.xs + w.c0 + w.tx * V;
  T *y = (T *)a.y + n * a.S * a.C + w.c0 + w.tx * V;
  for (long long s = s0 + w.ty; s < end; s += kNormBatch * d.p.TY) {
    Pack<T, V> p[kNormBatch] = {};
#pragma unroll
    for (int u = 0; u < kNormBatch; u++)
      if (s + u * d.p.TY < min(len, end)) p[u] = load_pack<T, V>(x + (s + u * d.p.TY) * a.xp);
#pragma unroll
    for (int u = 0; u < kNormBatch; u++) {
      if (s + u * d.p.TY >= end) break;
      if (s + u * d.p.TY < len) {
        float o[V];
#pragma unroll
        for (int i = 0; i < V; i++) {
          float e;
          act_both<ACT>((p[u].at(i) - mu[i]) * k[i] + B[i], o[i], e, a.act == kActRelu);
        }
        p[u].set(o);
      }
      store_pack<T, V>(y + (s + u * d.p.TY) * a.C, p[u]);
    }
  }
}

// channel sums of gz and gz xh of a chunk
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormChunkT) norm_chunk_sums(const NormDev d) {
  const Place w = place_of(d);
  const Lds l = lds_of(d);
  const NormArgs &a = d.a;
  const int cg = a.C / a.G;
  const long long n = d.first[2] + blockIdx.z, chunk = d.first[0] + blockIdx.x, s0 = chunk * d.p.rows, end = min(s0 + d.p.rows, length_of(a, n));
  float W[V], B[V], mu[V], k[V], s1[V] = {}, s2[V] = {};
  int g[V];
  load_channels<T, V>(a.w, w, 1.f, W);
  load_channels<T, V>(a.b, w, 0.f, B);
  groups_in_row<V>(d, w, g);
  if (w.on) {
#pragma unroll
    for (int i = 0; i < V; i++) {
      const long long at = n * a.G + g[i];
      mu[i] = a.mean[at], k[i] = a.rstd[at];
    }
    const T *x = (const T *)a.x + n * a.xs + w.c0 + w.tx * V, *gy = (const T *)a.gy + n * a.S * a.C + w.c0 + w.tx * V;
    for (long long s = s0 + w.ty; s < end; s += kNormBatch * d.p.TY) {
      Pack<T, V> p[kNormBatch], q[kNormBatch];
#pragma unroll
      for (int u = 0; u < kNormBatch; u++) {
        const long long at = min(s + u * d.p.TY, end - 1);   // (the last ones repeat and are not added)
        p[u] = load_pack<T, V>(x + at * a.xp), q[u] = load_pack<T, V>(gy + at * a.C);
      }
#pragma unroll
      for (int u = 0; u < kNormBatch; u++) {
        if (s + u * d.p.TY >= end) break;
        float xh[V], gz[V];
        gz_of<T, V, ACT>(p[u], q[u], mu, k, W, B, a.act == kActRelu, xh, gz);
#pragma unroll
        for (int i = 0; i < V; i++) s1[i] += gz[i], s2[i] += gz[i] * xh[i];
      }
    }
  }
  column_sums<V>(d, w, s1, l.scratch, l.chan);
  column_sums<V>(d, w, s2, l.scratch, l.chan2);
  float *to = d.stats + (n * d.p.chunks + chunk) * 2 * a.C + w.c0;
  for (int c = threadIdx.x; c < w.cw; c += d.p.T) to[c] = l.chan2[c], to[a.C + c] = l.chan[c];
}

// the chunks of a sample joined: a block a stripe and sample.  32 channels at a time by T / 32 runs of chunks.
template <typename T>
__global__ void __launch_bounds__(kNormChunkT) norm_sums_join(const NormDev d) {
  const Place w = place_of(d);
  const Lds l = lds_of(d);
  const NormArgs &a = d.a;
  const int cg = a.C / a.G, gs = w.cw / cg, runs = d.p.T / 32, run = threadIdx.x / 32;
  const long long n = d.first[2] + blockIdx.z, len = length_of(a, n);
  const long long chunks = (len + d.p.rows - 1) / d.p.rows;
  __shared__ float part[kNormChunkT / 32][2][33];
  float *lens = l.second + d.p.Cw / cg;
  if (threadIdx.x == 0) lens[0] = (float)len;
  if (chunks < runs) {   // few to sum: a thread a channel (8192 x 1 x 8192, one chunk: both directions 1970 us in runs, 990 so)
    const float *p = d.stats + n * d.p.chunks * 2 * a.C + w.c0;
    for (int c = threadIdx.x; c < w.cw; c += d.p.T) {
      float s1 = 0.f, s2 = 0.f;
      for (long long k = 0; k < chunks; k++) s2 += p[k * 2 * a.C + c], s1 += p[k * 2 * a.C + a.C + c];
      l.chan[c] = s1, l.chan2[c] = s2;
    }
    __syncthreads();
  }
  for (int base = chunks < runs ? w.cw : 0; base < w.cw; base += 32) {
    const int c = base + threadIdx.x % 32;
    float s1 = 0.f, s2 = 0.f;
    if (c < w.cw) {
      const float *p = d.stats + n * d.p.chunks * 2 * a.C + w.c0 + c;
#pragma unroll 4
      for (long long k = run; k < chunks; k += runs) s2 += p[k * 2 * a.C], s1 += p[k * 2 * a.C + a.C];
    }
    part[run][0][threadIdx.x % 32] = s1, part[run][1][threadIdx.x % 32] = s2;
    __syncthreads();
    if (threadIdx.x < 64 && base + (int)threadIdx.x % 32 < w.cw) {
      const int which = threadIdx.x / 32;
      float s = 0.f;
      for (int k = 0; k < runs; k++) s += part[k][which][threadIdx.x % 32];
      (which ? l.chan2 : l.chan)[base + threadIdx.x % 32] = s;
    }
    __syncthreads();
  }
  float *to = d.sums + n * 2 * a.C + w.c0;
  for (int c = threadIdx.x; c < w.cw; c += d.p.T) to[c] = l.chan2[c], to[a.C + c] = l.chan[c];
  __syncthreads();
  group_means<T>(d, w, l.chan, l.chan2, lens, l.first, l.second);
  float *m = d.means + (n * a.G + w.c0 / cg) * 2;
  for (int k = threadIdx.x; k < gs; k += d.p.T) m[2 * k] = l.first[k], m[2 * k + 1] = l.second[k];
}

// the means of a group's pieces averaged into the first one's place: a wave a group, of the groups from `base` on
static __global__ void __launch_bounds__(256) norm_means_join(const NormDev d, long long base) {
  const long long at = base + (long long)blockIdx.x * 4 + threadIdx.x / 64;
  if (at >= d.a.N * d.a.G) return;
  float *m = d.means + at * d.p.pieces * 2, s = 0.f;
  for (int k = threadIdx.x % 64; k < 2 * d.p.pieces; k += 64) s += m[k];   // (even lanes the first kind, odd ones the second)
#pragma unroll
  for (int j = 32; j >= 2; j >>= 1) s += __shfl_xor(s, j);
  if (threadIdx.x % 64 < 2) m[threadIdx.x % 64] = s / (float)d.p.pieces;
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kNormChunkT) norm_apply_bwd(const NormDev d) {
  const Place w = place_of(d);
  if (!w.on) return;
  const NormArgs &a = d.a;
  const long long n = d.first[2] + blockIdx.z, chunk = d.first[0] + blockIdx.x, s0 = chunk * d.p.rows, len = length_of(a, n), end = min(s0 + d.p.rows, a.S);
  float W[V], B[V], mu[V], k[V], m1[V], m2[V];
  int g[V];
  load_channels<T, V>(a.w, w, 1.f, W);
  load_channels<T, V>(a.b, w, 0.f, B);
  groups_in_row<V>(d, w, g);
#pragma unroll
  for (int i = 0; i < V; i++) {
    const long long at = n * a.G + g[i];
    mu[i] = a.mean[at], k[i] = a.rstd[at];
    m1[i] = d.means[2 * at * d.p.pieces], m2[i] = d.means[2 * at * d.p.pieces + 1];
  }
  const T *x = (const T *)a.x + n * a.xs + w.c0 + w.tx * V, *gy = (const T *)a.gy + n * a.S * a.C + w.c0 + w.tx * V;
  T *gx = (T *)a.y + n * a.S * a.C + w.c0 + w.tx * V;
  for (long long s = s0 + w.ty; s < end; s += kNormBatch * d.p.TY) {
    Pack<T, V> p[kNormBatch] = {}, q[kNormBatch] = {};
#pragma unroll
    for (int u = 0; u < kNormBatch; u++) {
      const long long at = s + u * d.p.TY;
      if (at < min(len, end)) p[u] = load_pack<T, V>(x + at * a.xp), q[u] = load_pack<T, V>(gy + at * a.C);
    }
#pragma unroll
    for (int u = 0; u < kNormBatch; u++) {
      if (s + u * d.p.TY >= end) break;
      if (s + u * d.p.TY < len) {
        float xh[V], gz[V], o[V];
        gz_of<T, V, ACT>(p[u], q[u], mu, k, W, B, a.act == kActRelu, xh, gz);
#pragma unroll
        for (int i = 0; i < V; i++) o[i] = k[i] * (gz[i] * W[i] - m1[i] - xh[i] * m2[i]);
        p[u].set(o);
      }
      store_pack<T, V>(gx + (s + u * d.p.TY) * a.C, p[u]);
    }
  }
}

// gw and gb: sums of `rows` rows of [2][C]; 32 columns by 8 runs of rows a block, a run in four chains
template <typename T>
__global__ void __launch_bounds__(256) norm_join(const float *sums, T *gw, T *gb, long long rows, int C) {
  __shared__ float lds[8][32];
  const long long c = (long long)blockIdx.x * 32 + threadIdx.x % 32;
  const int run = threadIdx.x / 32;
  float chain[4] = {};
  if (c < 2LL * C) {
    long long k = run;
#pragma unroll 2
    for (; k + 24 < rows; k += 32) {
#pragma unroll
      for (int u = 0; u < 4; u++) chain[u] += sums[(k + 8 * u) * 2 * C + c];
    }
    for (; k < rows; k += 8) chain[0] += sums[k * 2 * C + c];
  }
  float s = (chain[0] + chain[1]) + (chain[2] + chain[3]);
  lds[run][threadIdx.x % 32] = s;
  __syncthreads();
  if (run == 0 && c < 2LL * C) {
    for (int k = 1; k < 8; k++) s += lds[k][threadIdx.x];
    if (c < C && gw) gw[c] = from_f<T>(s);
    if (c >= C && gb) gb[c - C] = from_f<T>(s);
  }
}

template <typename T, int V, int ACT>
int run_norm(bool backward, const NormDev &d, hipStream_t s) {
  const NormArgs &a = d.a;
  const NormPlan &p = d.p;
  const dim3 block(p.T);
  if (p.R) {
    const size_t lds = norm_lds_bytes(p, a.C / a.G);
    const dim3 grid((unsigned)p.blocks, p.stripes);
#define GELIB_NORM(R)                                                                                              \
  do {                                                                                                             \
    if (backward) hipLaunchKernelGGL((norm_whole_bwd<T, V, ACT, R>), grid, block, lds, s, d);                      \
    else hipLaunchKernelGGL((norm_whole_fwd<T, V, ACT, R>), grid, block, lds, s, d);                               \
  } while (0)
    if (p.R == 1) GELIB_NORM(1);
    else if (p.R <= 4) GELIB_NORM(4);
    else if (p.R <= 8) GELIB_NORM(8);
    else hipLaunchKernelGGL((norm_whole_fwd<T, V, ACT, kNormMostR>), grid, block, lds, s, d);
#undef GELIB_NORM
    if (backward && d.sums)
      hipLaunchKernelGGL((norm_join<T>), dim3((2 * a.C + 31) / 32), dim3(256), 0, s, (const float *)d.sums, (T *)a.gw, (T *)a.gb, p.blocks, a.C);
  } else {
    // A launch takes 2^22 chunks, 32768 stripes and as many samples at most, a join 2^21 groups: from 2^32 threads on HIP runs what is
    // left after that many, and reports nothing.
    auto each = [&](auto kernel, NormDev v, long long chunks, size_t bytes) {
      const long long count[3] = {chunks, v.p.stripes, a.N}, most[3] = {1LL << 22, 32768, 32768};
      for (v.first[2] = 0; v.first[2] < a.N; v.first[2] += most[2])
        for (v.first[1] = 0; v.first[1] < count[1]; v.first[1] += most[1])
          for (v.first[0] = 0; v.first[0] < count[0]; v.first[0] += most[0]) {
            unsigned n[3];
            for (int k = 0; k < 3; k++) n[k] = (unsigned)std::min(most[k], count[k] - v.first[k]);
            hipLaunchKernelGGL(kernel, dim3(n[0], n[1], n[2]), dim3(v.p.T), bytes, s, v);
          }
    };
    auto join = [&](auto kernel, int groups, int threads) {   // groups of a block
      const long long all = a.N * a.G, most = 1LL << 21;
      for (long long g = 0; g < all; g += most)
        hipLaunchKernelGGL(kernel, dim3((unsigned)((std::min(most, all - g) + groups - 1) / groups)), dim3(threads), 0, s, d, g);
    };
    NormDev j = d;   // the kernels that sum groups sum the pieces of them
    j.a.G = a.G * p.pieces;
    const size_t lds = norm_lds_bytes(p, a.C / j.a.G);
    if (!backward) {
      each(norm_chunk_stats<T, V>, j, p.chunks, lds);
      if (p.chunks * p.pieces >= 1024) join(norm_stats_join<16>, 1, 1024);
      else join(norm_stats_join<1>, 4, 256);
      each(norm_apply_fwd<T, V, ACT>, d, p.chunks, 0);
    } else {
      each(norm_chunk_sums<T, V, ACT>, d, p.chunks, lds);
      // (stripes of about 32 channels: their sums are short, blocks are wanted)
      const int cg = a.C / j.a.G, Cq = V / std::gcd(V, cg) * cg;
      j.p.Cw = std::min(p.Cw, std::max(1, 32 / Cq) * Cq), j.p.stripes = (a.C + j.p.Cw - 1) / j.p.Cw, j.p.TX = 1, j.p.TY = 1, j.p.T = kNormChunkT;
      each(norm_sums_join<T>, j, 1, norm_lds_bytes(j.p, cg));
      if (a.y && p.pieces > 1) join(norm_means_join, 4, 256);
      if (a.y) each(norm_apply_bwd<T, V, ACT>, d, p.chunks, 0);
      if (a.gw || a.gb)
        hipLaunchKernelGGL((norm_join<T>), dim3((2 * a.C + 31) / 32), dim3(256), 0, s, (const float *)d.sums, (T *)a.gw, (T *)a.gb, a.N, a.C);
    }
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "group norm launch");
}

template <typename T, int V>
int run_norm_act(bool backward, const NormDev &d, hipStream_t s) {
  if (d.a.act == kActSilu) return run_norm<T, V, kActSilu>(backward, d, s);
  if (d.a.act == kActGelu) return run_norm<T, V, kActGelu>(backward, d, s);
  return run_norm<T, V, kActNone>(backward, d, s);
}

}  // namespace

template <typename T>
int launch_norm_typed(bool backward, const NormDev &d, hipStream_t s) {
  if (d.p.V == 16 / (int)sizeof(T)) return run_norm_act<T, 16 / sizeof(T)>(backward, d, s);
  if (d.p.V == 2) return run_norm_act<T, 2>(backward, d, s);
  return run_norm_act<T, 1>(backward, d, s);
}

#endif

}  // namespace gelib_hip
