// The linear layer with its epilogue, z = x w + b, y = act(z) + r, and its gradients: gz = gy act'(z), gx = gz w^T, gw = x^T gz,
// gb = sum of gz over the rows.  act'(z) is what the forward pass leaves for the backward pass, not z: it lies between
// -0.2 and 1.2, so 16-bit layers keep it in float16 (11 bits), at a fraction of the error that a rounded z would leave.
// The products are linear_gemm.h's; here: which tile and how many pieces of k a product takes, the sum of the pieces, and gz with
// its column sums, which is formed once for both products (one pass over gy and act'(z)).
#include <cmath>
#include <cstring>

#include "linear_gemm.h"

namespace gelib_hip {

namespace {
int g_linear_tile = -1, g_linear_splits = 0;   // options: -1 and 0 leave the choice to plan_of
}

int linear_act_set_option(const char *name, int value) {
  if (!std::strcmp(name, "linear_act_tile") && value >= -1 && value < kGemmTiles) g_linear_tile = value;
  else if (!std::strcmp(name, "linear_act_splits") && value >= 0 && value <= 64) g_linear_splits = value;
  else return GELIB_HIP_ERR_ARG;
  return GELIB_HIP_OK;
}

namespace {

constexpr int kColChunk = 128;   // rows whose column sum one block forms

struct Plan {
  int tile, splits;
  long long kper;
};

// The tile of a product and the pieces that its k is cut into: the least of an estimate of the time, in us.  A block's step of k takes
// `alone` while it has its compute unit to itself and `full` times the blocks there when they fill it (measured on 512 x 32768 x 256 and
// 2048 x 2048 x 8192; as many as `fit` at once); results are written, `out` bytes each, while other blocks of the unit compute, if it
// holds more than one; pieces are written and read once more by a further launch.
// bfloat16, chosen / other tiles and pieces: 8192 x 512 x 256 9.9 (64 x 128) / 12.7 (128 x 128) / 22 (256 x 256); 32768 x 256 -> 512 20 (256 x
// 256) / 22 / 22; 64 x 4096 x 4096 17 (8 pieces) / 45 (1) / 20 (16); 512 x 32768 x 256 29 (32) / 321 (1) us.
struct TileCost {
  double alone, full;
  int fit;
};
constexpr TileCost kCost16[kGemmTiles] = {{1.55, 2.0, 1}, {0.83, 0.57, 2}, {0.6, 0.34, 2}, {0.68, 0.34, 2}};
constexpr TileCost kCost32[kGemmTiles] = {{7.5, 8.2, 1}, {2.2, 2.08, 2}, {1.2, 1.09, 2}, {0.94, 0.7, 2}};

Plan plan_of(int dtype, long long M, long long N, long long K, int out) {
  const int bk = dtype == GELIB_HIP_F32 ? 32 : 64;
  const long long steps = std::max(1LL, (K + bk - 1) / bk);
  const double results = (double)M * N;
  Plan best = {};
  double least = 0;
  for (int t = 0; t < kGemmTiles; t++) {
    if (g_linear_tile >= 0 && t != g_linear_tile) continue;
    const TileCost &c = dtype == GELIB_HIP_F32 ? kCost32[t] : kCost16[t];
    const double tiles = std::ceil((double)M / kGemmBM[t]) * std::ceil((double)N / kGemmBN[t]);
    for (long long want = g_linear_splits > 0 ? std::min<long long>(g_linear_splits, steps) : 1; want <= 64 && want <= steps; want *= 2) {
      const long long per = (steps + want - 1) / want, pieces = (steps + per - 1) / per;
      const double blocks = std::ceil(tiles * pieces / 256), rounds = std::floor(blocks / c.fit), rest = blocks - rounds * c.fit;
      double us = per * (rounds * std::max(c.alone, c.fit * c.full) + (rest > 0 ? std::max(c.alone, rest * c.full) : 0)) + 1.5 * (rounds + (rest > 0));
      const double write = pieces > 1 ? results * 4.0 * pieces / 2.5e6 : results * out / 4.5e6;
      us = c.fit > 1 ? std::max(us, write) + 0.3 * write : us + write;
      if (pieces > 1) us += 4 + results * (4.0 * pieces + out) / 2.5e6;
      if (best.splits == 0 || us < least) least = us, best = {t, (int)pieces, per * bk};
      if (g_linear_splits > 0) break;
    }
  }
  return best;
}

size_t part_bytes(int dtype, long long M, long long N, long long K, int out) {
  if (M == 0 || N == 0) return 0;
  const Plan p = plan_of(dtype, M, N, K, out);
  return p.splits > 1 ? (size_t)p.splits * M * ((N + 3) & ~3LL) * 4 : 0;
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "linear layer launch");
}

// sum of the pieces of k, in their order, and the epilogue: four neighbouring results (or one, where rows do not allow) a thread
template <typename T, int ACT>
__global__ void __launch_bounds__(256) join_kernel(const GemmArgs a, unsigned per_row) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x, m = at / per_row;
  if (m >= a.M) return;
  const int n = (int)(at - m * per_row) * 4;
  const long long all = a.M * per_row * 4;
  const float *p = a.part + at * 4;
  f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
  for (int k = 0; k < a.splits; k++) s += *(const f32x4 *)(p + k * all);
  const float v[1][4] = {{s[0], s[1], s[2], s[3]}};
  epilogue<T, ACT, 1>(a, m, n, 0, v);
}

// bytes written for a result: the workspace is sized without knowing whether act' is kept, so it counts in every forward product
int out_bytes(GemmForm form, int dtype) { return (int)dtype_bytes(dtype) * (form == kFormXW ? 2 : 1); }

template <typename T>
int product(GemmForm form, int dtype, GemmArgs a, float *part, hipStream_t s) {
  const Plan p = plan_of(dtype, a.M, a.N, a.K, out_bytes(form, dtype));
  const bool a_kin = form != kFormXG;
  a.vec4 = a.N % 4 == 0 && ((uintptr_t)a.c | (uintptr_t)a.res | (uintptr_t)a.slope) % (4 * sizeof(T)) == 0;
  a.splits = p.splits, a.kper = p.kper;
  a.part = p.splits > 1 ? part : nullptr;
  a.ntiles = (unsigned)((a.N + kGemmBN[p.tile] - 1) / kGemmBN[p.tile]);
  // a launch takes 2^22 tiles at most (2^31 threads); further rows go to further launches
  const long long BM = kGemmBM[p.tile], most = std::max(1LL, (1LL << 22) / a.ntiles) * BM;
  for (long long m = 0; m < a.M; m += most) {
    GemmArgs b = a;
    b.M = std::min(most, a.M - m);
    b.mtiles = (unsigned)((b.M + BM - 1) / BM);
    b.a = (const T *)a.a + m * (a_kin ? a.lda : 1);
    b.c = (T *)a.c + m * a.N;
    if (a.res) b.res = (const T *)a.res + m * a.N;
    if (a.slope) b.slope = (T *)a.slope + m * a.N;   // (as wide as T)
    if (int rc = launch_gemm<T>(form, p.tile, b, s)) return rc;
  }
  if (!a.part) return 0;
  const unsigned per_row = (a.N + 3) / 4;
  const dim3 grid((unsigned)((a.M * per_row + 255) / 256));
  if (a.act == kActSilu) hipLaunchKernelGGL((join_kernel<T, kActSilu>), grid, dim3(256), 0, s, a, per_row);
  else if (a.act == kActGelu) hipLaunchKernelGGL((join_kernel<T, kActGelu>), grid, dim3(256), 0, s, a, per_row);
  else hipLaunchKernelGGL((join_kernel<T, kActNone>), grid, dim3(256), 0, s, a, per_row);
  return launched();
}

// Rows that are no multiple of 16 bytes, copied to ones that are, zeros at their ends: up to three matrices a launch, a thread 16
// bytes of the copy.
struct CopyArgs {
  struct {
    const void *from;
    void *to;
    long long stride, rows, first;   // elements between rows; first thread
    int cols;
  } m[3];
  int count;
  long long threads;
};
template <typename T>
__global__ void __launch_bounds__(256) copy_rows_kernel(const CopyArgs a) {
  constexpr int V = 16 / sizeof(T);
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < a.threads; t += (long long)gridDim.x * 256) {
    int k = 0;
    while (k + 1 < a.count && t >= a.m[k + 1].first) k++;
    const int per_row = (a.m[k].cols + V - 1) / V;
    const long long at = t - a.m[k].first, row = at / per_row;
    const int c = (int)(at - row * per_row) * V;
    const T *p = (const T *)a.m[k].from + row * a.m[k].stride + c;
    T v[V];
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = c + i < a.m[k].cols ? p[i] : (T)0.f;
    __builtin_memcpy(__builtin_assume_aligned((T *)a.m[k].to + at * V, 16), v, 16);
  }
}

// Takes the copies that a call needs, each at its place in the workspace, and makes them in one launch.
template <typename T>
struct Copies {
  static constexpr int V = 16 / sizeof(T);
  CopyArgs a = {};
  char *ws;
  explicit Copies(void *w) : ws((char *)w) {}
  // p and its row stride, where rows of `cols` elements are a multiple of 16 bytes, else those of a copy
  const void *rows(const void *p, long long &stride, long long rows, int cols) {
    if (cols % V == 0 || rows == 0 || cols == 0) return p;
    auto &m = a.m[a.count++];
    m = {p, ws, stride, rows, a.threads, cols};
    stride = (cols + V - 1) / V * V;
    a.threads += rows * (stride / V);
    ws += up((size_t)rows * stride * sizeof(T));
    return m.to;
  }
  void run(hipStream_t s) {
    if (a.count) hipLaunchKernelGGL((copy_rows_kernel<T>), dim3((unsigned)std::min((a.threads + 255) / 256, 1LL << 22)), dim3(256), 0, s, a);
  }
};
size_t copy_bytes(int dtype, long long rows, int cols) {
  const int V = 16 / (int)dtype_bytes(dtype);
  return cols % V ? up((size_t)rows * ((cols + V - 1) / V * 16)) : 0;
}

// gz = gy slope (slope null: gy), rounded to T, into gz unless that is null (rows of ldz, zeros behind N), and its unrounded column sums over kColChunk rows
// into sums[chunk][N] unless that is null.  A block: 64 threads of V columns by 4 rows at a time.
template <typename T, int V>
__global__ void __launch_bounds__(256) gz_kernel(const T *gy, const typename SlopeOf<T>::type *slope, T *gz, float *sums, long long rows, int N, int ldz, unsigned colblocks) {
  typedef typename SlopeOf<T>::type D;
  __shared__ float lds[4][64 * V];
  const long long chunk = blockIdx.x / colblocks;
  const long long n = ((long long)(blockIdx.x % colblocks) * 64 + threadIdx.x % 64) * V;
  const int tr = threadIdx.x / 64;
  float sum[V] = {};
  if (V == 1 && gz && n >= N && n < ldz)
    for (long long m = chunk * kColChunk + tr, end = min(rows, (chunk + 1) * kColChunk); m < end; m += 4) gz[m * ldz + n] = (T)0.f;
  if (n < N) {
    const long long end = min(rows, (chunk + 1) * kColChunk);
#pragma unroll 4
    for (long long m = chunk * kColChunk + tr; m < end; m += 4) {
      T g[V];
      D d[V];
      __builtin_memcpy(g, __builtin_assume_aligned(gy + m * N + n, V * sizeof(T)), sizeof(g));
      if (slope) __builtin_memcpy(d, __builtin_assume_aligned(slope + m * N + n, V * sizeof(T)), sizeof(d));
#pragma unroll
      for (int i = 0; i < V; i++) {
        const float v = slope ? to_f(g[i]) * to_f(d[i]) : to_f(g[i]);
        sum[i] += v;
        g[i] = from_f<T>(v);
      }
      if (gz) __builtin_memcpy(__builtin_assume_aligned(gz + m * ldz + n, V * sizeof(T)), g, sizeof(g));
    }
  }
  if (!sums) return;
#pragma unroll
  for (int i = 0; i < V; i++) lds[tr][i * 64 + threadIdx.x % 64] = sum[i];
  __syncthreads();
  if (tr == 0 && n < N)
#pragma unroll
    for (int i = 0; i < V; i++) sums[chunk * N + n + i] = (lds[0][i * 64 + threadIdx.x] + lds[1][i * 64 + threadIdx.x]) + (lds[2][i * 64 + threadIdx.x] + lds[3][i * 64 + threadIdx.x]);
}

// out[n] = sum over the chunks: 32 columns by 8 runs of chunks a block
template <typename T>
__global__ void __launch_bounds__(256) column_join_kernel(const float *sums, T *out, long long chunks, int N) {
  __shared__ float lds[8][32];
  const int n = blockIdx.x * 32 + threadIdx.x % 32, run = threadIdx.x / 32;
  float s = 0.f;
  if (n < N) {
#pragma unroll 8
    for (long long k = run; k < chunks; k += 8) s += sums[k * N + n];
  }
  lds[run][threadIdx.x % 32] = s;
  __syncthreads();
  if (run == 0 && n < N) {
    for (int k = 1; k < 8; k++) s += lds[k][threadIdx.x];
    out[n] = from_f<T>(s);
  }
}

template <typename T>
int fwd(int dtype, const LinearArgs &l, hipStream_t s) {
  if (!l.rows || !l.N) return 0;
  GemmArgs a = {};
  a.lda = l.xs, a.ldb = l.N;
  Copies<T> copies(l.ws);
  a.a = copies.rows(l.x, a.lda, l.rows, l.K);
  a.b = copies.rows(l.w, a.ldb, l.K, l.N);
  copies.run(s);
  a.c = l.y, a.bias = l.b, a.res = l.r, a.slope = l.slope, a.act = l.act;
  a.M = l.rows, a.N = l.N, a.K = l.K;
  return product<T>(kFormXW, dtype, a, (float *)copies.ws, s);
}

long long chunks_of(long long rows) { return (rows + kColChunk - 1) / kColChunk; }

template <typename T>
int bwd(int dtype, const LinearArgs &l, hipStream_t s) {
  typedef typename SlopeOf<T>::type D;
  if (!l.gx && !l.gw && !l.gb) return 0;
  const bool gx = l.gx && l.rows && l.K, gw = l.gw && l.K && l.N, products = (gx || gw) && l.rows && l.N;
  Copies<T> copies(l.ws);
  const void *x = l.x, *w = l.w;
  long long ldx = l.xs, ldw = l.N, ldz = l.N;
  if (gx) w = copies.rows(l.w, ldw, l.K, l.N);
  if (gw) x = copies.rows(l.x, ldx, l.rows, l.K);
  copies.run(s);
  char *ws = copies.ws;
  // gz in memory of its own: where act' is multiplied in, and where the rows of gy are no multiple of 16 bytes
  constexpr int V = 16 / sizeof(T);
  const bool keep = products && (l.slope || l.N % V);
  const T *gz = (const T *)l.gy;
  if (keep) {
    gz = (const T *)ws;
    ldz = (l.N + V - 1) / V * V;
    ws += up((size_t)l.rows * ldz * sizeof(T));
  }
  float *sums = nullptr;
  if (l.gb) {
    sums = (float *)ws;
    ws += up((size_t)chunks_of(l.rows) * l.N * 4);
  }
  const long long chunks = chunks_of(l.rows);
  if ((keep || l.gb) && chunks && l.N) {
    const bool wide = l.N % V == 0 && ((uintptr_t)l.gy | (uintptr_t)l.slope) % 16 == 0;
    const int columns = wide ? 64 * V : 64;
    const unsigned colblocks = (unsigned)((ldz + columns - 1) / columns);
    const long long most = std::max(1LL, (1LL << 23) / colblocks);   // chunks of a launch
    for (long long c = 0; c < chunks; c += most) {
      const long long m = c * kColChunk, now = std::min(most, chunks - c), rows = std::min(now * kColChunk, l.rows - m);
      const dim3 grid((unsigned)(now * colblocks));
      const T *gy = (const T *)l.gy + m * l.N;
      const D *d = l.slope ? (const D *)l.slope + m * l.N : nullptr;
      T *to = keep ? (T *)gz + m * ldz : nullptr;
      float *su = sums ? sums + c * l.N : nullptr;
      if (wide) hipLaunchKernelGGL((gz_kernel<T, V>), grid, dim3(256), 0, s, gy, d, to, su, rows, l.N, (int)ldz, colblocks);
      else hipLaunchKernelGGL((gz_kernel<T, 1>), grid, dim3(256), 0, s, gy, d, to, su, rows, l.N, (int)ldz, colblocks);
    }
  }
  if (l.gb && l.N)
    hipLaunchKernelGGL((column_join_kernel<T>), dim3((l.N + 31) / 32), dim3(256), 0, s, (const float *)sums, (T *)l.gb, chunks, l.N);
  GemmArgs a = {};
  if (gx) {
    a.a = gz, a.lda = ldz, a.b = w, a.ldb = ldw, a.c = l.gx;
    a.M = l.rows, a.N = l.K, a.K = l.N;
    if (int rc = product<T>(kFormGW, dtype, a, (float *)ws, s)) return rc;
  }
  if (gw) {
    a.a = x, a.lda = ldx, a.b = gz, a.ldb = ldz, a.c = l.gw;
    a.M = l.K, a.N = l.N, a.K = l.rows;
    if (int rc = product<T>(kFormXG, dtype, a, (float *)ws, s)) return rc;
  }
  return launched();
}

}  // namespace

size_t linear_workspace(int what, int dtype, long long rows, int K, int N) {
  if (what == 0) return copy_bytes(dtype, rows, K) + copy_bytes(dtype, K, N) + part_bytes(dtype, rows, N, K, out_bytes(kFormXW, dtype));
  size_t n = 0, parts = 0;
  const int V = 16 / (int)dtype_bytes(dtype);
  if ((what & 3) && K && (what & 8 || N % V)) n += up((size_t)rows * ((N + V - 1) / V * 16));
  if (what & 4) n += up((size_t)chunks_of(rows) * N * 4);
  if (what & 1) n += copy_bytes(dtype, K, N), parts = std::max(parts, part_bytes(dtype, rows, K, N, out_bytes(kFormGW, dtype)));
  if (what & 2) n += copy_bytes(dtype, rows, K), parts = std::max(parts, part_bytes(dtype, K, N, rows, out_bytes(kFormXG, dtype)));
  return n + parts;
}

int launch_linear_fwd(int dtype, const LinearArgs &a, hipStream_t s) {
  return dtype == GELIB_HIP_F32 ? fwd<float>(dtype, a, s) : dtype == GELIB_HIP_BF16 ? fwd<bhalf_t>(dtype, a, s) : fwd<half_t>(dtype, a, s);
}

int launch_linear_bwd(int dtype, const LinearArgs &a, hipStream_t s) {
  return dtype == GELIB_HIP_F32 ? bwd<float>(dtype, a, s) : dtype == GELIB_HIP_BF16 ? bwd<bhalf_t>(dtype, a, s) : bwd<half_t>(dtype, a, s);
}

}  // namespace gelib_hip
