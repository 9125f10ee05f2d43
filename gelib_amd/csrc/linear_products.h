// A product of linear_gemm.h as its callers want it: which tile and how many pieces of k it takes, the sum of the pieces, copies of
// operands whose rows are no multiple of 16 bytes.
#pragma once

#include <cmath>

#include "linear_gemm.h"

namespace gelib_hip {

extern int g_linear_tile, g_linear_splits;   // options: -1 and 0 leave the choice to plan_of

namespace {

struct Plan {
  int tile, splits;
  long long kper;
};

// The tile of a product and the pieces that its k is cut into: the least of an estimate of the time, in us.  A block's step of k takes
// `alone` while it has its compute unit to itself and `full` times the blocks there when they fill it (measured on 512 x 32768 x 256 and
// 2048 x 2048 x 8192; as many as `fit` at once); results are written, `out` bytes each, while other blocks of the unit compute, if it
// holds more than one; pieces are written and read once more by a further launch.
// whole: in one piece.
// bfloat16, chosen / other tiles and pieces: 8192 x 512 x 256 9.9 (64 x 128) / 12.7 (128 x 128) / 22 (256 x 256); 32768 x 256 -> 512 20 (256 x
// 256) / 22 / 22; 64 x 4096 x 4096 17 (8 pieces) / 45 (1) / 20 (16); 512 x 32768 x 256 29 (32) / 321 (1) us.
struct TileCost {
  double alone, full;
  int fit;
};
constexpr TileCost kCost16[kGemmTiles] = {{1.55, 2.0, 1}, {0.83, 0.57, 2}, {0.6, 0.34, 2}, {0.68, 0.34, 2}};
constexpr TileCost kCost32[kGemmTiles] = {{7.5, 8.2, 1}, {2.2, 2.08, 2}, {1.2, 1.09, 2}, {0.94, 0.7, 2}};

Plan plan_of(int dtype, long long M, long long N, long long K, int out, bool whole = false) {
  const int bk = dtype == GELIB_HIP_F32 ? 32 : 64;
  const long long steps = std::max(1LL, (K + bk - 1) / bk);
  const double results = (double)M * N;
  Plan best = {};
  double least = 0;
  for (int t = 0; t < kGemmTiles; t++) {
    if (g_linear_tile >= 0 && t != g_linear_tile) continue;
    const TileCost &c = dtype == GELIB_HIP_F32 ? kCost32[t] : kCost16[t];
    const double tiles = std::ceil((double)M / kGemmBM[t]) * std::ceil((double)N / kGemmBN[t]);
    // pieces only where all tiles go into one launch (the rows of a piece begin at its first), and the threads of the join
    const int forced = whole || tiles > (1 << 22) || results > 0x1p32 ? 1 : g_linear_splits;
    for (long long want = forced > 0 ? std::min<long long>(forced, steps) : 1; want <= 64 && want <= steps; want *= 2) {
      const long long per = (steps + want - 1) / want, pieces = (steps + per - 1) / per;
      const double blocks = std::ceil(tiles * pieces / 256), rounds = std::floor(blocks / c.fit), rest = blocks - rounds * c.fit;
      double us = per * (rounds * std::max(c.alone, c.fit * c.full) + (rest > 0 ? std::max(c.alone, rest * c.full) : 0)) + 1.5 * (rounds + (rest > 0));
      const double write = pieces > 1 ? results * 4.0 * pieces / 2.5e6 : results * out / 4.5e6;
      us = c.fit > 1 ? std::max(us, write) + 0.3 * write : us + write;
      if (pieces > 1) us += 4 + results * (4.0 * pieces + out) / 2.5e6;
      if (best.splits == 0 || us < least) least = us, best = {t, (int)pieces, per * bk};
      if (forced > 0) break;
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
  a.vec4 = a.N % 4 == 0 && a.ldc % 4 == 0 && ((uintptr_t)a.c | (uintptr_t)a.res | (uintptr_t)a.slope) % (4 * sizeof(T)) == 0;
  a.splits = p.splits, a.kper = p.kper;
  if (a.ldc == 0) a.ldc = a.N;
  a.part = p.splits > 1 ? part : nullptr;
  a.ntiles = (unsigned)((a.N + kGemmBN[p.tile] - 1) / kGemmBN[p.tile]);
  // a launch takes 2^22 tiles at most (2^31 threads); further rows go to further launches
  const long long BM = kGemmBM[p.tile], most = std::max(1LL, (1LL << 22) / a.ntiles) * BM;
  for (long long m = 0; m < a.M; m += most) {
    GemmArgs b = a;
    b.M = std::min(most, a.M - m);
    b.mtiles = (unsigned)((b.M + BM - 1) / BM);
    b.a = (const T *)a.a + m * (a_kin ? a.lda : 1);
    b.c = (T *)a.c + m * a.ldc;
    if (a.left_out) b.left_out = a.left_out + m;
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

// Rows that are no multiple of 16 bytes, copied to ones that are, zeros at their ends, and rows without the ones that a loss leaves out:
// up to three matrices a launch, a thread 16 bytes of the copy.
struct CopyArgs {
  struct {
    const void *from;
    void *to;
    long long stride, rows, first;   // elements between rows; first thread
    int cols;
    const long long *classes;        // rows whose class is below zero become zeros; null: none
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
    T v[V] = {};
    if (!a.m[k].classes || a.m[k].classes[row] >= 0) {
      if (a.m[k].cols % V == 0) {   // (whole rows are aligned, and copied for what they leave out)
        __builtin_memcpy(v, __builtin_assume_aligned(p, 16), 16);
      } else {
#pragma unroll
        for (int i = 0; i < V; i++) v[i] = c + i < a.m[k].cols ? p[i] : (T)0.f;
      }
    }
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
  const void *rows(const void *p, long long &stride, long long rows, int cols, const long long *classes = nullptr) {
    if ((cols % V == 0 && !classes) || rows == 0 || cols == 0) return p;
    auto &m = a.m[a.count++];
    m = {p, ws, stride, rows, a.threads, cols, classes};
    stride = (cols + V - 1LL) / V * V;
    a.threads += rows * (stride / V);
    ws += up((size_t)rows * stride * sizeof(T));
    return m.to;
  }
  void run(hipStream_t s) {
    if (a.count) hipLaunchKernelGGL((copy_rows_kernel<T>), dim3((unsigned)std::min((a.threads + 255) / 256, 1LL << 22)), dim3(256), 0, s, a);
  }
};
size_t copy_bytes(int dtype, long long rows, int cols, bool always = false) {
  const int V = 16 / (int)dtype_bytes(dtype);
  return cols % V || always ? up((size_t)rows * ((cols + V - 1LL) / V * 16)) : 0;
}

// out[n] = norm (null: 1) times the sum over the chunks: 32 columns at a time by 8 runs of chunks a block
template <typename T>
__global__ void __launch_bounds__(256) column_join_kernel(const float *sums, T *out, long long chunks, int N, const float *norm) {
  __shared__ float lds[8][32];
  const int run = threadIdx.x / 32;
  for (long long n0 = blockIdx.x * 32LL; n0 < N; n0 += gridDim.x * 32LL) {
    const long long n = n0 + threadIdx.x % 32;
    float s = 0.f;
    if (n < N) {
#pragma unroll 8
      for (long long k = run; k < chunks; k += 8) s += sums[k * N + n];
    }
    lds[run][threadIdx.x % 32] = s;
    __syncthreads();
    if (run == 0 && n < N) {
      for (int k = 1; k < 8; k++) s += lds[k][threadIdx.x];
      out[n] = from_f<T>(norm ? s * *norm : s);
    }
    __syncthreads();
  }
}

}  // namespace

}  // namespace gelib_hip
