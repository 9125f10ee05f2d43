// The linear layer with its epilogue, z = x w + b, y = act(z) + r, and its gradients: gz = gy act'(z), gx = gz w^T, gw = x^T gz,
// gb = sum of gz over the rows.  act'(z) is what the forward pass leaves for the backward pass, not z: it lies between
// -0.2 and 1.2, so bfloat16 layers keep it in float16 (11 bits) and float16 ones in finer codes (slope16_t), at a fraction of the error
// that a rounded z would leave.
// gz is rounded to the layer's type for the two products: the matrix cores multiply values of one type, and x and w have it.  With the
// rounding of the results gx and gw are then 1.4 times as far from float64 as with that one alone (bfloat16 16384 x 2048 -> 8192 with gelu:
// .0024 and .0017 of their norm), as far as those of a layer whose operations leave their results in 16 bits.  A second pair of products, with what
// the rounding takes from gz, would undo that for another 950 us beside the 1740 of both directions.  gb is the sum of unrounded values.
// The products are linear_gemm.h's; here: which tile and how many pieces of k a product takes, the sum of the pieces, and gz with
// its column sums, which is formed once for both products (one pass over gy and act'(z)).
#include <cmath>
#include <cstring>

#include "linear_products.h"

namespace gelib_hip {

int g_linear_tile = -1, g_linear_splits = 0;

int linear_act_set_option(const char *name, int value) {
  if (!std::strcmp(name, "linear_act_tile") && value >= -1 && value < kGemmTiles) g_linear_tile = value;
  else if (!std::strcmp(name, "linear_act_splits") && value >= 0 && value <= 64) g_linear_splits = value;
  else return GELIB_HIP_ERR_ARG;
  return GELIB_HIP_OK;
}

namespace {

// Rows whose column sum one block forms: fewer where blocks would be few (4099 x 517: 14.7 us with 128 rows, 7.5 with 32).
int rows_of_chunk(long long rows, int N) { return rows * N < (1LL << 25) ? 32 : 128; }

// gz = gy slope (slope null: gy), rounded to T, into gz unless that is null (rows of ldz, zeros behind N), and its unrounded column sums over chunks of rows
// into sums[chunk][N] unless that is null (col_chunk rows a chunk).  A block: 64 threads of V columns by 4 rows at a time; `colblocks` of
// them side by side from the `first` on.
template <typename T, int V>
__global__ void __launch_bounds__(256) gz_kernel(const T *gy, const typename SlopeOf<T>::type *slope, T *gz, float *sums, long long rows, int N, int ldz, unsigned colblocks, unsigned first, int col_chunk) {
  typedef typename SlopeOf<T>::type D;
  __shared__ float lds[4][64 * V];
  const long long chunk = blockIdx.x / colblocks;
  const long long n = ((long long)(first + blockIdx.x % colblocks) * 64 + threadIdx.x % 64) * V;
  const int tr = threadIdx.x / 64;
  float sum[V] = {};
  if (V == 1 && gz && n >= N && n < ldz)
    for (long long m = chunk * col_chunk + tr, end = min(rows, (chunk + 1) * col_chunk); m < end; m += 4) gz[m * ldz + n] = (T)0.f;
  if (n < N) {
    const long long end = min(rows, (chunk + 1) * col_chunk);
#pragma unroll 4
    for (long long m = chunk * col_chunk + tr; m < end; m += 4) {
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

// Up to four rows: what counts is w, read once, and how soon.  A block of 1024 threads takes 64 columns (fewer where that leaves few
// blocks): groups of threads side by side on V columns each (one load), the groups spread over k, all of a thread's loads under
// way together; the groups' sums are added in LDS.  One launch and no copies, whatever the rows' alignment (V = 1 where it is none).
// 1 x 1024 -> 4096 bfloat16: 4.4 us between calls (4.9 in the trace: 1.7 TB/s; tiles and pieces, two launches, 7.4): the latency of one
// batch of loads, one reduction and the launch.
template <typename T, int V, int M, int ACT>
__global__ void __launch_bounds__(1024) few_rows_kernel(const LinearArgs l, int side) {
  typedef typename SlopeOf<T>::type D;
  constexpr int BATCH = M == 4 && V == 8 ? 4 : 8;
  __shared__ float few_lds[1024 * V];   // [groups][side * V]
  const int groups = 1024 / side, group = threadIdx.x / side, cols = side * V;
  const long long n0 = (long long)blockIdx.x * cols;
  const int mine = threadIdx.x % side * V;
  const T *w = (const T *)l.w + min(n0 + mine, (long long)l.N - V), *x = (const T *)l.x;   // (behind the row: read once more, not written)
  float sum[M][V] = {};
  for (int k0 = group; k0 < l.K; k0 += groups * BATCH) {
    T t[BATCH][V], xv[BATCH][M];
#pragma unroll
    for (int u = 0; u < BATCH; u++) {
      const long long k = min(k0 + u * groups, l.K - 1);
      if constexpr (V == 1) t[u][0] = w[k * l.N];
      else __builtin_memcpy(t[u], __builtin_assume_aligned(w + k * l.N, 16), 16);
#pragma unroll
      for (int m = 0; m < M; m++) xv[u][m] = x[(m < l.rows ? m : 0) * l.xs + k];
    }
#pragma unroll
    for (int u = 0; u < BATCH; u++) {
      if (k0 + u * groups >= l.K) break;
#pragma unroll
      for (int m = 0; m < M; m++)
#pragma unroll
        for (int i = 0; i < V; i++) sum[m][i] += to_f(xv[u][m]) * to_f(t[u][i]);
    }
  }
#pragma unroll
  for (int m = 0; m < M; m++) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < V; i++) few_lds[group * cols + mine + i] = sum[m][i];
    // halves of the groups are added to the others until eight are left
    int left = groups;
    while (left > 8) {
      left /= 2;
      __syncthreads();
      for (int e = threadIdx.x; e < left * cols; e += 1024) few_lds[e] += few_lds[e + left * cols];
    }
    __syncthreads();
    const long long n = n0 + threadIdx.x, at = (long long)m * l.N + n;
    if (m >= l.rows || (int)threadIdx.x >= cols || n >= l.N) continue;
    float z = 0.f, y, slope;
    for (int g = 0; g < left; g++) z += few_lds[g * cols + threadIdx.x];
    if (l.b) z += to_f(((const T *)l.b)[n]);
    act_both<ACT>(z, y, slope, l.act == kActRelu);
    if (l.r) y += to_f(((const T *)l.r)[at]);
    ((T *)l.y)[at] = from_f<T>(y);
    if (l.slope) ((D *)l.slope)[at] = from_f<D>(slope);
  }
}

// Which forward products go there: up to four rows, while a thread's loads are one or two batches.  bfloat16, here / tiles: 1 x 1024 -> 4096
// 4.4 / 7.4, 2 x 1024 -> 4096 6.0 / 7.6, 4 x 1024 -> 4096 9.3 / 7.6, 1 x 4096 -> 4096 13.4 / 8.2, 1 x 333 -> 517 4.0 / 9.0, 4 x 333 -> 517
// 5.7 / 9.1 us; float32: 4 x 1024 -> 4096 7.8 / 8.0, 1 x 4096 -> 4096 15.0 / 16.3, 3 x 4096 -> 64 8.8 / 9.0, 1 x 32768 -> 256 71 / 23 us.
// (1024 threads for 64 columns: from 2^28 columns on a launch has 2^32 threads, of which HIP runs what is left after that many, and
// reports nothing.)
bool few_rows_case(int dtype, long long rows, int K, int N) {
  return rows <= 4 && K > 0 && rows * K <= 1024 * (long long)dtype_bytes(dtype) && N <= 1 << 27 && g_linear_tile < 0;
}

template <typename T, int V, int M>
void launch_few(const LinearArgs &l, hipStream_t s) {
  int side = 64 / V;   // threads side by side
  while (side > 1 && (l.N + side * V - 1) / (side * V) < 128) side /= 2;
  const dim3 grid((unsigned)((l.N + side * V - 1) / (side * V)));
  if (l.act == kActSilu) hipLaunchKernelGGL((few_rows_kernel<T, V, M, kActSilu>), grid, dim3(1024), 0, s, l, side);
  else if (l.act == kActGelu) hipLaunchKernelGGL((few_rows_kernel<T, V, M, kActGelu>), grid, dim3(1024), 0, s, l, side);
  else hipLaunchKernelGGL((few_rows_kernel<T, V, M, kActNone>), grid, dim3(1024), 0, s, l, side);
}

template <typename T>
int few_rows(const LinearArgs &l, hipStream_t s) {
  constexpr int V = 16 / sizeof(T);
  const bool wide = l.N % V == 0 && (uintptr_t)l.w % 16 == 0;
  if (wide) {
    if (l.rows == 1) launch_few<T, V, 1>(l, s);
    else if (l.rows == 2) launch_few<T, V, 2>(l, s);
    else launch_few<T, V, 4>(l, s);
  } else {
    if (l.rows == 1) launch_few<T, 1, 1>(l, s);
    else if (l.rows == 2) launch_few<T, 1, 2>(l, s);
    else launch_few<T, 1, 4>(l, s);
  }
  return launched();
}

template <typename T>
int fwd(int dtype, const LinearArgs &l, hipStream_t s) {
  if (!l.rows || !l.N) return 0;
  if (few_rows_case(dtype, l.rows, l.K, l.N)) return few_rows<T>(l, s);
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

long long chunks_of(long long rows, int N) { return (rows + rows_of_chunk(rows, N) - 1) / rows_of_chunk(rows, N); }

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
    ws += up((size_t)chunks_of(l.rows, l.N) * l.N * 4);
  }
  const long long chunks = chunks_of(l.rows, l.N);
  if ((keep || l.gb) && chunks && l.N) {
    const int col_chunk = rows_of_chunk(l.rows, l.N);
    const bool wide = l.N % V == 0 && ((uintptr_t)l.gy | (uintptr_t)l.slope) % 16 == 0;
    const int columns = wide ? 64 * V : 64;
    const unsigned all = (unsigned)((ldz + columns - 1) / columns), side = std::min(all, 1u << 23);   // blocks side by side, in one launch
    const long long most = (1LL << 23) / side;   // chunks of a launch
    for (unsigned first = 0; first < all; first += side)
      for (long long c = 0; c < chunks; c += most) {
        const unsigned colblocks = std::min(side, all - first);
        const long long m = c * col_chunk, now = std::min(most, chunks - c), rows = std::min(now * col_chunk, l.rows - m);
        const dim3 grid((unsigned)(now * colblocks));
        const T *gy = (const T *)l.gy + m * l.N;
        const D *d = l.slope ? (const D *)l.slope + m * l.N : nullptr;
        T *to = keep ? (T *)gz + m * ldz : nullptr;
        float *su = sums ? sums + c * l.N : nullptr;
        if (wide) hipLaunchKernelGGL((gz_kernel<T, V>), grid, dim3(256), 0, s, gy, d, to, su, rows, l.N, (int)ldz, colblocks, first, col_chunk);
        else hipLaunchKernelGGL((gz_kernel<T, 1>), grid, dim3(256), 0, s, gy, d, to, su, rows, l.N, (int)ldz, colblocks, first, col_chunk);
      }
  }
  if (l.gb && l.N)
    hipLaunchKernelGGL((column_join_kernel<T>), dim3((unsigned)std::min((l.N + 31LL) / 32, 1LL << 22)), dim3(256), 0, s, (const float *)sums, (T *)l.gb, chunks, l.N, (const float *)nullptr);
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
  if (what == 0 && few_rows_case(dtype, rows, K, N)) return 0;
  if (what == 0) return copy_bytes(dtype, rows, K) + copy_bytes(dtype, K, N) + part_bytes(dtype, rows, N, K, out_bytes(kFormXW, dtype));
  size_t n = 0, parts = 0;
  const int V = 16 / (int)dtype_bytes(dtype);
  if ((what & 3) && K && (what & 8 || N % V)) n += up((size_t)rows * ((N + V - 1LL) / V * 16));
  if (what & 4) n += up((size_t)chunks_of(rows, N) * N * 4);
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
