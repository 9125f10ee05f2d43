// The linear layer with its epilogue, z = x w + b, y = act(z) + r, and its gradients: gz = gy act'(z), gx = gz w^T, gw = x^T gz,
// gb = sum of gz over the rows.  act'(z) is what the forward pass leaves for the backward pass, not z: it lies between
// -0.2 and 1.2, so 16-bit layers keep it in float16 (11 bits), at a fraction of the error that a rounded z would leave.
// The products are linear_gemm.h's; here: which tile and how many pieces of k a product takes, the sum of the pieces, and gz with
// its column sums, which is formed once for both products (one pass over gy and act'(z)).
#include "linear_gemm.h"

namespace gelib_hip {

namespace {

constexpr int kColChunk = 128;   // rows whose column sum one block forms

struct Plan {
  int tile, splits;
  long long kper;
};

// The tile of a product and the pieces that its k is cut into.
Plan plan_of(int dtype, long long M, long long N, long long K) {
  const int bk = dtype == GELIB_HIP_F32 ? 32 : 64;
  const long long steps = std::max(1LL, (K + bk - 1) / bk);
  auto tiles = [&](int t) { return ((M + kGemmBM[t] - 1) / kGemmBM[t]) * ((N + kGemmBN[t] - 1) / kGemmBN[t]); };
  Plan p;
  if (M <= 16) p.tile = 3;
  else if (tiles(0) >= 192) p.tile = 0;
  else if (M > 64) p.tile = 1;
  else p.tile = 2;
  const long long t = tiles(p.tile);
  long long want = t >= 192 ? 1 : std::min(steps / 4, 512 / t);
  want = std::max(1LL, std::min(want, 64LL));
  const long long per = (steps + want - 1) / want;
  p.splits = (int)((steps + per - 1) / per);
  p.kper = per * bk;
  return p;
}

size_t part_bytes(int dtype, long long M, long long N, long long K) {
  if (M == 0 || N == 0) return 0;
  const Plan p = plan_of(dtype, M, N, K);
  return p.splits > 1 ? (size_t)p.splits * M * N * 4 : 0;
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
  const long long all = a.M * a.N;
  const float *p = a.part + m * a.N + n;
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  if (a.N % 4 == 0) {
    f32x4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (int k = 0; k < a.splits; k++) s += *(const f32x4 *)(p + k * all);
#pragma unroll
    for (int i = 0; i < 4; i++) v[i] = s[i];
  } else {
    for (int k = 0; k < a.splits; k++)
#pragma unroll
      for (int i = 0; i < 4; i++)
        if (n + i < a.N) v[i] += p[k * all + i];
  }
  epilogue4<T, ACT>(a, m, n, v);
}

template <typename T>
int product(GemmForm form, int dtype, GemmArgs a, float *part, hipStream_t s) {
  const Plan p = plan_of(dtype, a.M, a.N, a.K);
  const unsigned V = 16 / sizeof(T);
  const bool a_kin = form != kFormXG, b_kin = form == kFormGW;
  const bool fast = ((uintptr_t)a.a | (uintptr_t)a.b) % 16 == 0 && a.lda % V == 0 && a.ldb % V == 0 && (a_kin ? a.K : a.M) % V == 0 &&
                    (b_kin ? a.K : (long long)a.N) % V == 0;
  const bool vec4 = a.N % 4 == 0 && ((uintptr_t)a.c | (uintptr_t)a.res | (uintptr_t)a.slope) % (4 * sizeof(T)) == 0;
  a.splits = p.splits, a.kper = p.kper;
  a.part = p.splits > 1 ? part : nullptr;
  a.vec4 = a.part ? a.N % 4 == 0 : vec4;
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
    if (int rc = launch_gemm<T>(form, p.tile, fast, b, s)) return rc;
  }
  if (!a.part) return 0;
  a.vec4 = vec4;
  const unsigned per_row = (a.N + 3) / 4;
  const dim3 grid((unsigned)((a.M * per_row + 255) / 256));
  if (a.act == kActSilu) hipLaunchKernelGGL((join_kernel<T, kActSilu>), grid, dim3(256), 0, s, a, per_row);
  else if (a.act == kActGelu) hipLaunchKernelGGL((join_kernel<T, kActGelu>), grid, dim3(256), 0, s, a, per_row);
  else hipLaunchKernelGGL((join_kernel<T, kActNone>), grid, dim3(256), 0, s, a, per_row);
  return launched();
}

// gz = gy slope (slope null: gy), rounded to T, into gz unless that is null, and its unrounded column sums over kColChunk rows
// into sums[chunk][N] unless that is null.  A block: 64 threads of V columns by 4 rows at a time.
template <typename T, int V>
__global__ void __launch_bounds__(256) gz_kernel(const T *gy, const typename SlopeOf<T>::type *slope, T *gz, float *sums, long long rows, int N, unsigned colblocks) {
  typedef typename SlopeOf<T>::type D;
  __shared__ float lds[4][64 * V];
  const long long chunk = blockIdx.x / colblocks;
  const long long n = ((long long)(blockIdx.x % colblocks) * 64 + threadIdx.x % 64) * V;
  const int tr = threadIdx.x / 64;
  float sum[V] = {};
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
      if (gz) __builtin_memcpy(__builtin_assume_aligned(gz + m * N + n, V * sizeof(T)), g, sizeof(g));
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
  a.a = l.x, a.lda = l.xs, a.b = l.w, a.ldb = l.N, a.c = l.y, a.bias = l.b, a.res = l.r, a.slope = l.slope, a.act = l.act;
  a.M = l.rows, a.N = l.N, a.K = l.K;
  return product<T>(kFormXW, dtype, a, (float *)l.ws, s);
}

long long chunks_of(long long rows) { return (rows + kColChunk - 1) / kColChunk; }

template <typename T>
int bwd(int dtype, const LinearArgs &l, hipStream_t s) {
  typedef typename SlopeOf<T>::type D;
  if (!l.gx && !l.gw && !l.gb) return 0;
  const bool products = (l.gx && l.K) || (l.gw && l.K);
  char *ws = (char *)l.ws;
  const T *gz = (const T *)l.gy;
  const bool keep = l.slope && products && l.rows && l.N;
  if (keep) {
    gz = (const T *)ws;
    ws += up((size_t)l.rows * l.N * sizeof(T));
  }
  float *sums = nullptr;
  if (l.gb) {
    sums = (float *)ws;
    ws += up((size_t)chunks_of(l.rows) * l.N * 4);
  }
  const long long chunks = chunks_of(l.rows);
  if ((keep || l.gb) && chunks && l.N) {
    constexpr int V = 16 / sizeof(T);
    const bool wide = l.N % V == 0 && ((uintptr_t)l.gy | (uintptr_t)l.slope) % 16 == 0;
    const unsigned columns = wide ? 64 * V : 64, colblocks = (l.N + columns - 1) / columns;
    const long long most = std::max(1LL, (1LL << 23) / colblocks);   // chunks of a launch
    for (long long c = 0; c < chunks; c += most) {
      const long long m = c * kColChunk, off = m * l.N, now = std::min(most, chunks - c);
      const dim3 grid((unsigned)(now * colblocks));
      const T *gy = (const T *)l.gy + off;
      const D *d = l.slope ? (const D *)l.slope + off : nullptr;
      T *to = keep ? (T *)gz + off : nullptr;
      float *su = sums ? sums + c * l.N : nullptr;
      const long long rows = std::min(now * kColChunk, l.rows - m);
      if (wide) hipLaunchKernelGGL((gz_kernel<T, V>), grid, dim3(256), 0, s, gy, d, to, su, rows, l.N, colblocks);
      else hipLaunchKernelGGL((gz_kernel<T, 1>), grid, dim3(256), 0, s, gy, d, to, su, rows, l.N, colblocks);
    }
  }
  if (l.gb && l.N)
    hipLaunchKernelGGL((column_join_kernel<T>), dim3((l.N + 31) / 32), dim3(256), 0, s, (const float *)sums, (T *)l.gb, chunks, l.N);
  GemmArgs a = {};
  if (l.gx && l.rows && l.K) {
    a.a = gz, a.lda = l.N, a.b = l.w, a.ldb = l.N, a.c = l.gx;
    a.M = l.rows, a.N = l.K, a.K = l.N;
    if (int rc = product<T>(kFormGW, dtype, a, (float *)ws, s)) return rc;
  }
  if (l.gw && l.K && l.N) {
    a.a = l.x, a.lda = l.xs, a.b = gz, a.ldb = l.N, a.c = l.gw;
    a.M = l.K, a.N = l.N, a.K = l.rows;
    if (int rc = product<T>(kFormXG, dtype, a, (float *)ws, s)) return rc;
  }
  return launched();
}

}  // namespace

size_t linear_workspace(int what, int dtype, long long rows, int K, int N) {
  if (what == 0) return part_bytes(dtype, rows, N, K);
  size_t n = 0;
  if ((what & 8) && (what & 3) && K) n += up((size_t)rows * N * dtype_bytes(dtype));
  if (what & 4) n += up((size_t)chunks_of(rows) * N * 4);
  size_t parts = 0;
  if (what & 1) parts = std::max(parts, part_bytes(dtype, rows, K, N));
  if (what & 2) parts = std::max(parts, part_bytes(dtype, K, N, rows));
  return n + parts;
}

int launch_linear_fwd(int dtype, const LinearArgs &a, hipStream_t s) {
  return dtype == GELIB_HIP_F32 ? fwd<float>(dtype, a, s) : dtype == GELIB_HIP_BF16 ? fwd<bhalf_t>(dtype, a, s) : fwd<half_t>(dtype, a, s);
}

int launch_linear_bwd(int dtype, const LinearArgs &a, hipStream_t s) {
  return dtype == GELIB_HIP_F32 ? bwd<float>(dtype, a, s) : dtype == GELIB_HIP_BF16 ? bwd<bhalf_t>(dtype, a, s) : bwd<half_t>(dtype, a, s);
}

}  // namespace gelib_hip
