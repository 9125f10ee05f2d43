// Softmax cross entropy of a linear layer's classes: z = x w + b, loss_i = log sum_c exp z_ic - z_i,t.  The logits leave the matrix product
// as a largest value and a sum of exp for each row of a tile, and the logit of the row's own class: (rows, classes / 256) pairs instead of
// (rows, classes) logits.
// The gradient of the logits, gz = g (exp(z - lse) - onehot), needs them again: the product is formed a second time, and what leaves it is
// gz, for as many classes at a time as kMostGradients bytes hold; each such piece goes through the two products gx += gz w^T and gw = x^T gz
// while the next level of memory still has it.  Eight operations a weight and row instead of six, for rows * classes values that are
// neither kept nor read and written once more in between.
// bfloat16 8192 x 2048 -> 65536, both directions: 7.9 ms (forward 2.0, 1.1 PFLOP/s; four pieces of gz .56, gx .45, gw .46 each), at the library's rate for
// a large product (1335 TFLOP/s) 6.6.
// gz is rounded to the layer's type for the two products, as in the layer itself (linear_act.hip); gb sums unrounded values.
// float16: gz is scaled by a power of two that brings the largest |g| to 2^13 (gz stays below 2^14), so that probabilities down to
// 2^-27 are float16 values of full precision; results are scaled back before they are rounded.
#include <algorithm>

#include "linear_products.h"

namespace gelib_hip {

namespace {

constexpr size_t kMostGradients = 256u << 20;   // bytes of gz formed at a time

// A row's pairs -> the log of its sum, its loss.  `lanes` lanes a row (a power of two)
__global__ void __launch_bounds__(256) loss_join_kernel(float *loss, float *lse, const float2 *tops, const float *picked, const long long *targets, long long rows,
                                                        int ntiles, int N, int lanes) {
  const long long row = ((long long)blockIdx.x * 256 + threadIdx.x) / lanes;
  const int lane = threadIdx.x % lanes;
  float top = -INFINITY, sum = 0.f;
  if (row < rows)
    for (int k = lane; k < ntiles; k += lanes) {
      const float2 v = tops[row * ntiles + k];
      const float to = fmaxf(top, v.x), from = finite_or_zero(to);
      sum = sum * __builtin_amdgcn_exp2f((top - from) * 1.44269504088896341f) + v.y * __builtin_amdgcn_exp2f((v.x - from) * 1.44269504088896341f);
      top = to;
    }
  for (int d = 1; d < lanes; d *= 2) {
    const float otop = __shfl_xor(top, d), osum = __shfl_xor(sum, d);
    const float to = fmaxf(top, otop), from = finite_or_zero(to);
    sum = sum * __builtin_amdgcn_exp2f((top - from) * 1.44269504088896341f) + osum * __builtin_amdgcn_exp2f((otop - from) * 1.44269504088896341f);
    top = to;
  }
  if (row >= rows || lane) return;
  const float l = top + logf(sum);
  const long long t = targets[row];
  if (lse) lse[row] = l;
  loss[row] = t < 0 ? 0.f : t < N ? l - picked[row] : __builtin_nanf("");
}

// norm[0]: the power of two that brings the largest |g| of a row with a class to 2^13, norm[1]: one over it.  Many rows: largest values of blocks first
// (behind norm[1]; targets null: of these)
constexpr int kNormBlocks = 256, kNormRows = 8192;   // of a block
constexpr size_t kNormBytes = (2 + kNormBlocks) * 4;
__global__ void __launch_bounds__(1024) loss_norm_kernel(float *norm, const float *g, const long long *targets, long long rows) {
  __shared__ float lds[16];
  float top = 0.f;
#pragma unroll 4
  for (long long i = blockIdx.x * 1024LL + threadIdx.x; i < rows; i += gridDim.x * 1024LL) {
    const float v = fabsf(g[i]);
    if ((!targets || targets[i] >= 0) && v < INFINITY) top = fmaxf(top, v);
  }
#pragma unroll
  for (int d = 1; d < 64; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = top;
  __syncthreads();
  if (threadIdx.x) return;
  for (int k = 0; k < 16; k++) top = fmaxf(top, lds[k]);
  if (gridDim.x > 1) {
    norm[2 + blockIdx.x] = top;
    return;
  }
  const int e = top > 0.f ? max(-100, min(100, 13 - ilogbf(top))) : 0;
  norm[0] = ldexpf(1.f, e), norm[1] = ldexpf(1.f, -e);
}

// gx from the sums over all pieces (rows of K up to a multiple of 4), zeros in rows that are left out
template <typename T>
__global__ void __launch_bounds__(256) loss_finish_kernel(T *gx, const float *sums, const long long *targets, long long n, int K, const float *norm) {
  const long long stride = (K + 3) & ~3;
  const float by = norm ? *norm : 1.f;
  if (K % 4 == 0 && (uintptr_t)gx % (4 * sizeof(T)) == 0) {   // (as they lie)
    for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n / 4; at += (long long)gridDim.x * 256) {
      const f32x4 v = ((const f32x4 *)sums)[at];
      const bool out = targets[at / (K / 4)] < 0;
      T t[4];
#pragma unroll
      for (int i = 0; i < 4; i++) t[i] = from_f<T>(out ? 0.f : v[i] * by);
      __builtin_memcpy(__builtin_assume_aligned(gx + at * 4, 4 * sizeof(T)), t, sizeof(t));
    }
    return;
  }
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) {
    const long long row = at / K;
    gx[at] = from_f<T>(targets[row] < 0 ? 0.f : sums[row * stride + (at - row * K)] * by);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) loss_zero_kernel(T *to, long long n) {
  for (long long at = (long long)blockIdx.x * 256 + threadIdx.x; at < n; at += (long long)gridDim.x * 256) to[at] = (T)0.f;
}
template <typename T>
void zero(void *to, long long n, hipStream_t s) {
  if (to && n) hipLaunchKernelGGL(loss_zero_kernel<T>, dim3((unsigned)std::min((n + 255) / 256, 1LL << 16)), dim3(256), 0, s, (T *)to, n);
}

// ---- few rows and classes ----
// Where a product's tiles leave compute units idle and its sums are long, it is cut along k as any other: its pieces hold all logits then (they
// are few), and the loss is taken of their sum (logits_plan).

__device__ __forceinline__ void sum_exp(float &top, float &sum, float otop, float osum) {
  const float to = fmaxf(top, otop), from = finite_or_zero(to);
  sum = sum * __builtin_amdgcn_exp2f((top - from) * 1.44269504088896341f) + osum * __builtin_amdgcn_exp2f((otop - from) * 1.44269504088896341f);
  top = to;
}

// top and sum of 256 threads' pairs, in every thread
__device__ __forceinline__ void block_sum_exp(float &top, float &sum, float2 *lds) {
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const float otop = __shfl_xor(top, d), osum = __shfl_xor(sum, d);
    sum_exp(top, sum, otop, osum);
  }
  if (threadIdx.x % 64 == 0) lds[threadIdx.x / 64] = make_float2(top, sum);
  __syncthreads();
  top = lds[0].x, sum = lds[0].y;
  for (int k = 1; k < 4; k++) sum_exp(top, sum, lds[k].x, lds[k].y);
}

// A block a row
__global__ void __launch_bounds__(256) loss_rows_kernel(float *loss, float *lse, const float *logits, const long long *targets, int N) {
  __shared__ float2 lds[4];
  const long long row = blockIdx.x;
  const float *z = logits + row * ((N + 3) & ~3);
  float top = -INFINITY, sum = 0.f;
  for (int n = threadIdx.x; n < N; n += 256) sum_exp(top, sum, z[n], 1.f);
  block_sum_exp(top, sum, lds);
  if (threadIdx.x) return;
  const float l = top + logf(sum);
  const long long t = targets[row];
  if (lse) lse[row] = l;
  loss[row] = t < 0 ? 0.f : t < N ? l - z[t] : __builtin_nanf("");
}

// gz of one logit
__device__ __forceinline__ float gradient_of(float z, float lse, long long t, int n, int N, float g) {
  const float p = __builtin_amdgcn_exp2f((z - lse) * 1.44269504088896341f) - (n == t ? 1.f : 0.f);
  return t < 0 ? 0.f : p * (t < N ? g : __builtin_nanf(""));
}

constexpr int kGzRows = 8;   // of a block

// gz (rows of ldz, zeros behind N) and its column sums over kGzRows rows: a thread a column
template <typename T>
__global__ void __launch_bounds__(256) loss_gz_kernel(T *gz, float *columns, const float *logits, const float *lse, const float *g, const long long *targets,
                                                      const float *norm, long long rows, int N, int ldz) {
  const int n = blockIdx.y * 256 + threadIdx.x;
  if (n >= ldz) return;
  const long long r0 = (long long)blockIdx.x * kGzRows, stride = (N + 3) & ~3;
  const float scale = norm ? *norm : 1.f;
  float sum = 0.f;
#pragma unroll
  for (int k = 0; k < kGzRows; k++) {
    const long long r = r0 + k;
    if (r >= rows) break;
    const float v = n < N ? gradient_of(logits[r * stride + n], lse[r], targets[r], n, N, g[r] * scale) : 0.f;
    sum += v;
    gz[r * ldz + n] = from_f<T>(v);
  }
  if (columns && n < N) columns[(long long)blockIdx.x * N + n] = sum;
}

// ---- a handful of rows and classes: one launch forward, two backward, no matrix cores ----
// What counts there is launches: 19 x 64 -> 118 float32, both directions: 60 us a pass, nearly all of them the host's; through the tiles (nine
// launches) 80.  128 x 128 -> 128, here / through the tiles: 59 / 70.
constexpr long long kSmallWork = 1 << 21;   // rows * n_in * n_out
constexpr int kSmallSide = 2048;            // n_in and n_out (LDS)
// A value of gw is one thread's sum over the rows, here / through the tiles, float32, both directions: 256 x 64 -> 128 53 / 63, 512 x 64 -> 64 59 / 58,
// 1024 x 64 -> 32 98 / 59, 8192 x 16 -> 16 619 / 59.
constexpr int kSmallRows = 256;
bool small_case(long long rows, int K, int N) { return K > 0 && rows <= kSmallRows && K <= kSmallSide && N <= kSmallSide && rows * K * N <= kSmallWork; }

// z of a row's classes threadIdx.x, threadIdx.x + 256, ... into LDS; x in LDS
template <typename T>
__device__ __forceinline__ void small_logits(float *z, const float *x, const T *w, const T *b, int K, int N) {
  for (int n = threadIdx.x; n < N; n += 256) {
    float v = b ? to_f(b[n]) : 0.f;
    const T *p = w + n;
#pragma unroll 8
    for (int k = 0; k < K; k++) v = __builtin_fmaf(x[k], to_f(p[(long long)k * N]), v);
    z[n] = v;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) loss_small_kernel(const LossArgs l) {
  __shared__ float x[kSmallSide], z[kSmallSide];
  __shared__ float2 lds[4];
  const long long row = blockIdx.x;
  for (int k = threadIdx.x; k < l.K; k += 256) x[k] = to_f(((const T *)l.x)[row * l.xs + k]);
  __syncthreads();
  small_logits<T>(z, x, (const T *)l.w, (const T *)l.b, l.K, l.N);
  float top = -INFINITY, sum = 0.f;
  for (int n = threadIdx.x; n < l.N; n += 256) sum_exp(top, sum, z[n], 1.f);
  block_sum_exp(top, sum, lds);   // (and z is there)
  if (threadIdx.x) return;
  const float lse = top + logf(sum);
  const long long t = l.targets[row];
  if (l.lse_out) l.lse_out[row] = lse;
  l.loss[row] = t < 0 ? 0.f : t < l.N ? lse - z[t] : __builtin_nanf("");
}

// gz of a row, as float32 values rounded to the layer's type as for the tiles' products (float16: with norm), and gx: a wave a value of it at a time
template <typename T>
__global__ void __launch_bounds__(256) loss_small_rows_kernel(const LossArgs l, float *gz, const float *norm) {
  __shared__ float x[kSmallSide], z[kSmallSide];
  const long long row = blockIdx.x, t = l.targets[row];
  for (int k = threadIdx.x; k < l.K; k += 256) x[k] = to_f(((const T *)l.x)[row * l.xs + k]);
  __syncthreads();
  small_logits<T>(z, x, (const T *)l.w, (const T *)l.b, l.K, l.N);
  const float g = l.g[row] * (norm ? norm[0] : 1.f), lse = l.lse[row];
  for (int n = threadIdx.x; n < l.N; n += 256) {   // (its own)
    const float v = gradient_of(z[n], lse, t, n, l.N, g);
    gz[row * l.N + n] = v;
    z[n] = to_f(from_f<T>(v));
  }
  __syncthreads();
  if (!l.gx) return;
  const float back = norm ? norm[1] : 1.f;
  for (int k = threadIdx.x / 64; k < l.K; k += 4) {
    const T *w = (const T *)l.w + (long long)k * l.N;
    float v = 0.f;
    if (t >= 0)   // (what is left out gives nothing, whatever w holds)
      for (int n = threadIdx.x % 64; n < l.N; n += 64) v = __builtin_fmaf(z[n], to_f(w[n]), v);
#pragma unroll
    for (int d = 1; d < 64; d *= 2) v += __shfl_xor(v, d);
    if (threadIdx.x % 64 == 0) ((T *)l.gx)[row * l.K + k] = from_f<T>(v * back);
  }
}

// gw, a thread a value, and gb (row K)
template <typename T>
__global__ void __launch_bounds__(256) loss_small_columns_kernel(const LossArgs l, const float *gz, const float *norm) {
  const long long at = (long long)blockIdx.x * 256 + threadIdx.x;
  const int k = (int)(at / l.N), n = (int)(at - (long long)k * l.N);
  if (k > l.K || (k < l.K ? !l.gw : !l.gb)) return;
  const float back = norm ? norm[1] : 1.f;
  float v = 0.f;
  if (k < l.K) {
#pragma unroll 4
    for (long long r = 0; r < l.rows; r++) {
      const float x = to_f(((const T *)l.x)[r * l.xs + k]), g = to_f(from_f<T>(gz[r * l.N + n]));
      if (l.targets[r] >= 0) v = __builtin_fmaf(x, g, v);
    }
    ((T *)l.gw)[at] = from_f<T>(v * back);
  } else {
    for (long long r = 0; r < l.rows; r++) v += gz[r * l.N + n];
    ((T *)l.gb)[n] = from_f<T>(v * back);
  }
}

long long tiles_of(long long n, int b) { return (n + b - 1) / b; }

// x w and one of the loss's epilogues, in launches of at most 2^22 tiles
template <typename T>
int logits(int epilogue, int dtype, const GemmArgs &g, hipStream_t s) {
  const Plan p = plan_of(dtype, g.M, g.N, g.K, epilogue == kLossGrad ? (int)dtype_bytes(dtype) : 0, true);
  const long long BM = kGemmBM[p.tile];
  GemmArgs a = g;
  a.splits = 1, a.kper = p.kper, a.part = nullptr;
  a.ntiles = (unsigned)tiles_of(a.N, kGemmBN[p.tile]);
  const long long most = std::max(1LL, (1LL << 22) / a.ntiles) * BM;
  for (long long m = 0; m < g.M; m += most) {
    GemmArgs b = a;
    b.M = std::min(most, g.M - m);
    b.mtiles = (unsigned)tiles_of(b.M, (int)BM);
    b.a = (const T *)a.a + m * a.lda;
    if (a.c) b.c = (T *)a.c + m * a.ldc;
    b.targets += m;
    if (a.lse) b.lse += m, b.weight += m;
    if (a.tops) b.tops += m * a.ntiles, b.picked += m;
    if (a.columns) b.columns += m / kGemmWM[p.tile] * a.N;
    if (int rc = launch_loss_gemm<T>(epilogue, p.tile, b, s)) return rc;
  }
  return 0;
}
// the tile that logits() takes
int tile_of(int dtype, long long M, long long N, long long K, int epilogue) {
  return plan_of(dtype, M, N, K, epilogue == kLossGrad ? (int)dtype_bytes(dtype) : 0, true).tile;
}

// Pieces of k that the logits' product is cut into (1: it has the loss's epilogue): where the kernels behind them fit one launch and the sums are long
// enough for the launches more.  Both directions, in pieces / whole, us: float32 512 x 256 -> 118 110 / 94, x 512 107 / 94, 4096 x 512 -> 64 87 / 182,
// 512 x 2048 -> 118 90 / 171, 256 x 1024 -> 4096 129 / 220; bfloat16 64 x 2048 -> 1000 106 / 89, x 4096 102 / 109, x 8192 101 / 180.
Plan logits_plan(int dtype, long long rows, int K, int N) {
  return plan_of(dtype, rows, N, K, 4, rows > 1 << 20 || N > 1 << 20 || K < (dtype == GELIB_HIP_F32 ? 512 : 4096));
}
int logit_pieces(int dtype, long long rows, int K, int N) { return logits_plan(dtype, rows, K, N).splits; }

size_t logits_bytes(int dtype, long long rows, int K, int N) { return up(part_bytes(dtype, rows, N, K, 4)) + up((size_t)rows * ((N + 3) & ~3LL) * 4); }

// the logits of all classes from pieces of k, rows of N up to a multiple of 4
template <typename T>
int logits_in_pieces(int dtype, GemmArgs a, void *space, const float *&logits, hipStream_t s) {
  const Plan p = logits_plan(dtype, a.M, (int)a.K, a.N);
  a.splits = p.splits, a.kper = p.kper, a.part = (float *)space, a.act = kActNone;
  a.mtiles = (unsigned)tiles_of(a.M, kGemmBM[p.tile]), a.ntiles = (unsigned)tiles_of(a.N, kGemmBN[p.tile]);
  if (int rc = launch_gemm<T>(kFormXW, p.tile, a, s)) return rc;
  a.c = (char *)space + up(part_bytes(dtype, a.M, a.N, a.K, 4)), a.ldc = (a.N + 3) & ~3, a.vec4 = a.N % 4 == 0;
  a.bias = a.norm = nullptr;   // (in the first piece; of the gradients)
  const unsigned per_row = (a.N + 3) / 4;
  hipLaunchKernelGGL((join_kernel<float, kActNone>), dim3((unsigned)((a.M * per_row + 255) / 256)), dim3(256), 0, s, a, per_row);
  logits = (const float *)a.c;
  return launched();
}

struct Forward {
  size_t tops, picked, part, bytes;
  int ntiles, splits;
};
Forward forward_space(int dtype, long long rows, int K, int N) {
  Forward f = {};
  if (small_case(rows, K, N)) return f;
  f.splits = logit_pieces(dtype, rows, K, N);
  if (f.splits > 1) {
    f.part = copy_bytes(dtype, rows, K) + copy_bytes(dtype, K, N);
    f.bytes = f.part + logits_bytes(dtype, rows, K, N);
    return f;
  }
  f.ntiles = (int)tiles_of(N, kGemmBN[tile_of(dtype, rows, N, K, kLossSums)]);
  size_t at = copy_bytes(dtype, rows, K) + copy_bytes(dtype, K, N);
  f.tops = at, at += up((size_t)rows * f.ntiles * 8);
  f.picked = at, at += up((size_t)rows * 4);
  f.bytes = at;
  return f;
}

// Classes of a piece of gz, and where everything lies
struct Backward {
  long long piece, ldz;
  int pieces, splits;   // splits: of the logits' product
  size_t gz, norm, columns, part, bytes;
};
Backward backward_space(int what, int dtype, long long rows, int K, int N) {
  Backward b = {};
  if (small_case(rows, K, N)) {
    b.norm = up((size_t)rows * N * 4), b.bytes = b.norm + up(kNormBytes);
    return b;
  }
  const long long e = dtype_bytes(dtype), V = 16 / e;
  const long long most = std::max(256LL, (long long)(kMostGradients / (size_t)(rows * e)) / 256 * 256);
  b.pieces = (int)tiles_of(N, (int)std::min<long long>(most, 1 << 30));
  b.piece = b.pieces == 1 ? N : (tiles_of(N, b.pieces) + 255) / 256 * 256;
  b.pieces = (int)((N + b.piece - 1) / b.piece);
  b.ldz = (b.piece + V - 1) / V * V;
  b.splits = b.pieces == 1 ? logit_pieces(dtype, rows, K, N) : 1;
  const long long last = N - (b.pieces - 1) * b.piece;
  size_t at = copy_bytes(dtype, rows, K, what & 2) + copy_bytes(dtype, K, N);
  b.gz = at, at += up((size_t)rows * b.ldz * e);
  b.norm = at, at += up(kNormBytes);
  b.columns = at;
  if (what & 4 && b.splits > 1) at += up((size_t)tiles_of(rows, kGzRows) * N * 4);
  else if (what & 4)
    for (long long n : {b.piece, last}) at = std::max(at, b.columns + up((size_t)tiles_of(rows, kGemmWM[tile_of(dtype, rows, n, K, kLossGrad)]) * n * 4));
  b.part = at;
  size_t part = 0;
  if (what & 1) part = b.pieces > 1 ? up((size_t)rows * ((K + 3) & ~3LL) * 4) : part_bytes(dtype, rows, K, N, out_bytes(kFormGW, dtype));
  size_t part_w = 0;
  if (what & 2)
    for (long long n : {b.piece, last}) part_w = std::max(part_w, part_bytes(dtype, K, n, rows, out_bytes(kFormXG, dtype)));
  if (b.splits > 1) part = std::max(part, logits_bytes(dtype, rows, K, N));
  // (sums over pieces of classes live through all of them; pieces of a product only until they are joined)
  b.bytes = at + (b.pieces > 1 ? part + part_w : std::max(part, part_w));
  return b;
}

template <typename T>
int fwd(int dtype, const LossArgs &l, hipStream_t s) {
  if (small_case(l.rows, l.K, l.N)) {
    hipLaunchKernelGGL(loss_small_kernel<T>, dim3((unsigned)l.rows), dim3(256), 0, s, l);
    return launched();
  }
  const Forward at = forward_space(dtype, l.rows, l.K, l.N);
  GemmArgs a = {};
  a.lda = l.xs, a.ldb = l.N;
  Copies<T> copies(l.ws);
  a.a = copies.rows(l.x, a.lda, l.rows, l.K);
  a.b = copies.rows(l.w, a.ldb, l.K, l.N);
  copies.run(s);
  a.bias = l.b, a.M = l.rows, a.N = l.N, a.K = l.K;
  a.targets = l.targets, a.N_all = l.N;
  if (at.splits > 1) {
    const float *logits;
    if (int rc = logits_in_pieces<T>(dtype, a, (char *)l.ws + at.part, logits, s)) return rc;
    hipLaunchKernelGGL(loss_rows_kernel, dim3((unsigned)l.rows), dim3(256), 0, s, l.loss, l.lse_out, logits, l.targets, l.N);
    return launched();
  }
  a.tops = (float2 *)((char *)l.ws + at.tops), a.picked = (float *)((char *)l.ws + at.picked);
  if (int rc = logits<T>(kLossSums, dtype, a, s)) return rc;
  int lanes = 1;
  while (lanes < 64 && lanes < at.ntiles) lanes *= 2;
  const long long most = (1LL << 30) / lanes;   // rows of a launch
  for (long long m = 0; m < l.rows; m += most) {
    const long long now = std::min(most, l.rows - m);
    hipLaunchKernelGGL(loss_join_kernel, dim3((unsigned)((now * lanes + 255) / 256)), dim3(256), 0, s, l.loss + m, l.lse_out ? l.lse_out + m : nullptr,
                       a.tops + m * at.ntiles, a.picked + m, l.targets + m, now, at.ntiles, l.N, lanes);
  }
  return launched();
}

template <typename T>
int bwd(int dtype, const LossArgs &l, hipStream_t s) {
  const int what = (l.gx ? 1 : 0) | (l.gw ? 2 : 0) | (l.gb ? 4 : 0);
  if (l.rows == 0) {
    zero<T>(l.gw, (long long)l.K * l.N, s);
    zero<T>(l.gb, l.N, s);
    return launched();
  }
  const Backward at = backward_space(what, dtype, l.rows, l.K, l.N);
  char *ws = (char *)l.ws;
  float *norm = nullptr;
  if (dtype == GELIB_HIP_F16) {
    norm = (float *)(ws + at.norm);
    const unsigned blocks = (unsigned)std::max(1LL, std::min((long long)kNormBlocks, l.rows / kNormRows));
    hipLaunchKernelGGL(loss_norm_kernel, dim3(blocks), dim3(1024), 0, s, norm, l.g, l.targets, l.rows);
    if (blocks > 1) hipLaunchKernelGGL(loss_norm_kernel, dim3(1), dim3(1024), 0, s, norm, (const float *)(norm + 2), (const long long *)nullptr, (long long)blocks);
  }
  if (small_case(l.rows, l.K, l.N)) {
    float *gz = (float *)ws;
    hipLaunchKernelGGL(loss_small_rows_kernel<T>, dim3((unsigned)l.rows), dim3(256), 0, s, l, gz, (const float *)norm);
    if (l.gw || l.gb)
      hipLaunchKernelGGL(loss_small_columns_kernel<T>, dim3((unsigned)(((l.K + 1LL) * l.N + 255) / 256)), dim3(256), 0, s, l, (const float *)gz, (const float *)norm);
    return launched();
  }
  long long ldx = l.xs, ldw = l.N;
  Copies<T> copies(ws);
  // (a row that is left out may hold anything; times a gradient of zero it would still be something in gw)
  const T *x = (const T *)copies.rows(l.x, ldx, l.rows, l.K, l.gw ? l.targets : nullptr), *w = (const T *)copies.rows(l.w, ldw, l.K, l.N);
  copies.run(s);
  const float *back = norm ? norm + 1 : nullptr;
  T *gz = (T *)(ws + at.gz);
  const bool gx = l.gx && l.K, gw = l.gw && l.K;
  float *part = (float *)(ws + at.part), *part_w = part;
  if (at.pieces > 1 && (what & 1)) part_w = (float *)((char *)part + up((size_t)l.rows * ((l.K + 3) & ~3LL) * 4));
  for (int k = 0; k < at.pieces; k++) {
    const long long n0 = k * at.piece;
    const int n = (int)std::min(at.piece, l.N - n0);
    GemmArgs a = {};
    a.a = x, a.lda = ldx, a.b = w + n0, a.ldb = ldw, a.bias = l.b ? (const T *)l.b + n0 : nullptr;
    a.c = gz, a.ldc = at.ldz, a.M = l.rows, a.N = n, a.K = l.K;
    a.targets = l.targets, a.n_first = n0, a.N_all = l.N, a.lse = l.lse, a.weight = l.g, a.norm = norm;
    if (l.gb) a.columns = (float *)(ws + at.columns);
    if (at.splits > 1) {
      const float *logits;
      if (int rc = logits_in_pieces<T>(dtype, a, part, logits, s)) return rc;
      hipLaunchKernelGGL(loss_gz_kernel<T>, dim3((unsigned)tiles_of(l.rows, kGzRows), (unsigned)tiles_of(at.ldz, 256)), dim3(256), 0, s, gz, a.columns, logits, l.lse, l.g, l.targets, (const float *)norm, l.rows, n, (int)at.ldz);
    } else if (int rc = logits<T>(kLossGrad, dtype, a, s)) return rc;
    if (l.gb) {
      const long long chunks = at.splits > 1 ? tiles_of(l.rows, kGzRows) : tiles_of(l.rows, kGemmWM[tile_of(dtype, l.rows, n, l.K, kLossGrad)]);
      hipLaunchKernelGGL(column_join_kernel<T>, dim3((unsigned)std::min((n + 31LL) / 32, 1LL << 22)), dim3(256), 0, s, (const float *)a.columns, (T *)l.gb + n0, chunks, n, back);
    }
    if (gx) {
      GemmArgs p = {};
      p.a = gz, p.lda = at.ldz, p.b = w + n0, p.ldb = ldw, p.c = l.gx, p.M = l.rows, p.N = l.K, p.K = n, p.norm = back, p.left_out = l.targets;
      if (at.pieces == 1) {
        if (int rc = product<T>(kFormGW, dtype, p, part, s)) return rc;
      } else {
        const Plan plan = plan_of(dtype, p.M, p.N, p.K, 4, true);
        p.splits = 1, p.kper = plan.kper, p.add = k > 0;
        p.ntiles = (unsigned)tiles_of(p.N, kGemmBN[plan.tile]);
        const long long BM = kGemmBM[plan.tile], most = std::max(1LL, (1LL << 22) / p.ntiles) * BM;
        for (long long m = 0; m < l.rows; m += most) {
          GemmArgs b = p;
          b.M = std::min(most, l.rows - m), b.mtiles = (unsigned)tiles_of(b.M, (int)BM);
          b.a = gz + m * at.ldz, b.part = part + m * ((l.K + 3) & ~3LL);
          if (int rc = launch_gemm<T>(kFormGW, plan.tile, b, s)) return rc;
        }
      }
    }
    if (gw) {
      GemmArgs p = {};
      p.a = x, p.lda = ldx, p.b = gz, p.ldb = at.ldz, p.c = (T *)l.gw + n0, p.ldc = l.N, p.M = l.K, p.N = n, p.K = l.rows, p.norm = back;
      if (int rc = product<T>(kFormXG, dtype, p, part_w, s)) return rc;
    }
  }
  if (gx && at.pieces > 1) {
    const long long all = l.rows * l.K;
    hipLaunchKernelGGL(loss_finish_kernel<T>, dim3((unsigned)std::min((all + 255) / 256, 1LL << 20)), dim3(256), 0, s, (T *)l.gx, (const float *)part, l.targets, all, l.K, back);
  }
  return launched();
}

}  // namespace

size_t loss_workspace(int what, int dtype, long long rows, int K, int N) {
  if (rows == 0) return 0;
  return what ? backward_space(what, dtype, rows, K, N).bytes : forward_space(dtype, rows, K, N).bytes;
}

int launch_loss(int dtype, const LossArgs &a, hipStream_t s) {
  if (a.rows == 0) return 0;
  return dtype == GELIB_HIP_F32 ? fwd<float>(dtype, a, s) : dtype == GELIB_HIP_BF16 ? fwd<bhalf_t>(dtype, a, s) : fwd<half_t>(dtype, a, s);
}

int launch_loss_bwd(int dtype, const LossArgs &a, hipStream_t s) {
  if (!a.gx && !a.gw && !a.gb) return 0;
  return dtype == GELIB_HIP_F32 ? bwd<float>(dtype, a, s) : dtype == GELIB_HIP_BF16 ? bwd<bhalf_t>(dtype, a, s) : bwd<half_t>(dtype, a, s);
}

}  // namespace gelib_hip
