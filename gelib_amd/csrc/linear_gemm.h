// The matrix products of the linear layer on the matrix cores: C[m, n] = sum_k A[m, k] B[k, n] for the three forms that a layer
// and its gradients need -- x w, gz w^T, x^T gz -- without a copy of any operand.
//
// An operand lies in memory either with k innermost (x in x w, gz and w in gz w^T) or with its own index innermost (w in x w, both
// in x^T gz); the tile that a block stages is 128 bytes of k by R rows, or its transpose, either way R * 128 bytes of LDS, copied as
// it lies in memory, 16 bytes a lane, straight into LDS: rows start at multiples of 16 bytes and end in zeros up to the next one
// (operands that do not are copied first, linear_act.hip).  What is outside the matrix is staged as zero, so no tile needs a special
// case behind this.  Transposing happens on the way from LDS into registers: 16-bit types with the LDS unit's transposing reads (a group of 16
// lanes reads 4 rows of 16 values and each lane gets a column of 4), float32 by giving a lane the 4 neighbouring columns that one
// 16-byte read delivers: fragment j of a lane belongs to column 4 r + j, and the epilogue goes by that.
// The order of 16-byte pieces in a row of LDS is permuted (exclusive or with the row) so that the lanes of a read spread over the banks.
// Two or three buffers, one barrier a step, fragments read half a step ahead (below).
//
// The products are formed with B's fragment as the first operand, so that a lane's four results lie side by side in a row of C.
//
// What bounds it: the matrix cores, and below about 2000 rows the latency of the steps.  bfloat16 16384 x 2048 -> 8192: x w 515 to 640 us, gz w^T
// 465 to 520, x^T gz 480 to 510, by the clock that the card's power allows (0.9 to 1.2 PFLOP/s; the library's products 440 to 580, 450 and
// 590); a step of a 256 x 256 tile 1.7 us, of which the products are 1.0 at the full rate; with gelu and its slope 620 to 690 (0.54 GB written).
// float32, the same sizes: 4.1, 4.0 and 3.9 ms, 134 to 141 TFLOP/s (the library 148 to 152).
#pragma once

#include "real_ops.h"

namespace gelib_hip {

struct GemmArgs {
  const void *a, *b;
  long long lda, ldb;       // elements between the rows in memory
  void *c;                  // (M, N) packed
  const void *bias, *res;   // epilogue: c = act(bias + sum) + res, slope = act'(bias + sum); each may be null
  void *slope;
  float *part;              // [splits][M][N up to a multiple of 4] sums of the pieces of k instead of c, or null
  long long M, K, kper;     // kper: k of a piece, a multiple of the step
  int N, act, splits, vec4;  // vec4: rows of c, res and slope take vectors of 4
  unsigned mtiles, ntiles;
  long long ldc;            // elements between the rows of c
  const float *norm;        // results without an activation times this; null: 1
  int add;                  // part holds sums already: add to them
  const long long *left_out;   // rows of c whose entry is below zero are zeros, in results without an activation; null: none
  // a layer's classes and their loss (linear_loss.hip), instead of c = act(..) + res
  const long long *targets; // class of every row
  long long n_first, N_all; // the first of these classes, all of them (bias begins with these)
  const float *lse, *weight;   // kLossGrad: log of the sum of exp, the loss's gradient
  float2 *tops;             // kLossSums: [rows][ntiles] largest logit of a tile and sum of exp(logit - it)
  float *picked;            // kLossSums: logit of the row's class, where it has one
  float *columns;           // kLossGrad: [rows / WM][N] sums of gz over rows, or null
};

// epilogues beside enum Act's
constexpr int kLossSums = 16, kLossGrad = 17;

enum GemmForm { kFormXW = 0, kFormGW = 1, kFormXG = 2 };   // x w, gz w^T, x^T gz

// tiles: 0: 256 x 256, 1: 128 x 128, 2: 64 x 128, 3: 16 x 256
constexpr int kGemmTiles = 4;
constexpr int kGemmBM[kGemmTiles] = {256, 128, 64, 16}, kGemmBN[kGemmTiles] = {256, 128, 128, 256};

constexpr int kGemmWM[kGemmTiles] = {128, 64, 64, 16};   // rows of a wave

template <typename T>
int launch_gemm(GemmForm form, int tile, const GemmArgs &a, hipStream_t s);
// x w with the epilogue kLossSums or kLossGrad (one launch: up to 2^22 tiles)
template <typename T>
int launch_loss_gemm(int epilogue, int tile, const GemmArgs &a, hipStream_t s);

#ifdef __HIPCC__

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bhalf_t bf16x8 __attribute__((ext_vector_type(8)));
typedef half_t f16x8 __attribute__((ext_vector_type(8)));

// what act'(z) is kept in: float16 is 1/8 of a bfloat16 layer's rounding
template <typename T>
struct SlopeOf { typedef half_t type; };
template <>
struct SlopeOf<half_t> { typedef slope16_t type; };
template <>
struct SlopeOf<float> { typedef float type; };

__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c, bhalf_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma(s16x8 a, s16x8 b, f32x4 c, half_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

typedef __attribute__((address_space(3))) char *LdsPtr;

// 16 bytes of every lane to LDS, lane after lane from `to` (the same for the whole wave) on.  Written out because the compiler,
// which cannot tell the two buffers apart, would wait for the builtin's copy before the next read of either; the wave waits by
// itself (vmcnt) before the barrier that opens the buffer.  No register is written.
__device__ __forceinline__ void load_to_lds(const char *from, char *to) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(LdsPtr)to);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(at), "v"(from) : "memory");   // (m0 holds nothing of the compiler's between two statements)
}

static __device__ const float4 gemm_zeros[1] = {};   // what lanes outside a matrix stage

// One operand's tile.  R: its extent (BM or BN), KIN: k innermost in memory, G: neighbouring rows that fragments share in float32
template <typename T, int R, bool KIN, int THREADS, int G>
struct Stage {
  static constexpr int VEC = 16 / sizeof(T), BK = 128 / sizeof(T);
  static constexpr int CPR = KIN ? 8 : R * (int)sizeof(T) / 16;          // 16-byte pieces of a row in LDS
  static constexpr int PIECES = R * 8, NL = (PIECES + THREADS - 1) / THREADS, DOWN = THREADS / CPR;   // DOWN: rows between a thread's pieces
  // a thread's pieces lie in one column of the permuted tile
  static_assert(NL == 1 || (KIN ? DOWN / G % 8 == 0 && DOWN % G == 0 : DOWN % 4 == 0), "");
  const char *p;       // its first piece of the tile to come
  long long down, step;
  int k, mn;           // k of that piece in the tile; rows (KIN) or columns of the matrix from it on
  static __device__ __forceinline__ int swizzle(int row) {
    if (KIN) return (row / G) & 7;
    // 16 lanes read 32 bytes of four neighbouring k, and the next 16 of the four k that are 8 further on: eight places of 256 bytes
    // (without the second term every transposing read took twice its time: 25 % more LDS cycles in x w, 100 % in x^T gz)
    return sizeof(T) == 2 ? ((row & 3) << 1 | (CPR >= 16 && DOWN % 16 == 0 ? (row & 8) : 0)) & (CPR - 1) : 0;
  }
  __device__ __forceinline__ void init(const void *base, long long ld, long long mn0, long long MN, long long k0) {
    const int row = threadIdx.x / CPR, c = (threadIdx.x % CPR) ^ swizzle(row);
    const long long at = mn0 + (KIN ? row : c * VEC);
    k = KIN ? c * VEC : row;
    mn = (int)max(0LL, min(MN - at, 1LL << 30));
    p = (const char *)((const T *)base + (KIN ? at * ld + k0 + k : (k0 + k) * ld + at));
    down = DOWN * ld * (long long)sizeof(T);
    step = (KIN ? BK : BK * ld) * (long long)sizeof(T);
  }
  // the next tile, of which `left` k are there
  __device__ __forceinline__ void issue(char *lds, long long left) {
    const int have = (int)min(left, (long long)BK);
#pragma unroll
    for (int u = 0; u < NL; u++) {
      if (PIECES % THREADS != 0 && u * THREADS + threadIdx.x >= PIECES) continue;   // (whole waves)
      const bool in = KIN ? u * DOWN < mn && k < have : mn > 0 && k + u * DOWN < have;
      load_to_lds(in ? p + u * down : (const char *)gemm_zeros, lds + (u * THREADS + (threadIdx.x & ~63)) * 16);
    }
    p += step;
  }
  // 16-bit: the fragment of 16 rows from row0 on, k = ks * 32 + (lane / 16) * 8 + 0..7
  static __device__ __forceinline__ s16x8 frag16(const char *lds, int row0, int ks) {
    const int lane = threadIdx.x % 64, c = lane % 16, q = lane / 16;
    if (KIN) {
      const int row = row0 + c;
      return *(const s16x8 *)(lds + row * 128 + (((ks * 4 + q) ^ swizzle(row)) << 4));
    }
    s16x4 h[2];
#pragma unroll
    for (int i = 0; i < 2; i++) {
      const int kk = ks * 32 + q * 8 + i * 4 + c / 4, col = row0 + c % 4 * 4;
      const char *at = lds + kk * (R * 2) + (((col / 8) ^ swizzle(kk)) << 4) + col % 8 * 2;
      h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at);
    }
    return __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
  }
  // float32: fragments f = 0..G-1 of the rows row0 + lane % 16 * G + f, k = ks * 16 + (lane / 16) * 4 + 0..3
  static __device__ __forceinline__ void frag32(const char *lds, int row0, int ks, float out[G][4]) {
    const int lane = threadIdx.x % 64, c = lane % 16, q = lane / 16;
    if (KIN) {
#pragma unroll
      for (int f = 0; f < G; f++) {
        const int row = row0 + c * G + f;
        *(float4 *)out[f] = *(const float4 *)(lds + row * 128 + (((ks * 4 + q) ^ swizzle(row)) << 4));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float v[G];
        __builtin_memcpy(v, lds + (ks * 16 + q * 4 + i) * (R * 4) + (row0 + c * G) * 4, G * 4);
#pragma unroll
        for (int f = 0; f < G; f++) out[f][i] = v[f];
      }
    }
  }
};

// What a row's exponentials are formed less: its largest logit, where infinity less infinity is not what that would come to
__device__ __forceinline__ float finite_or_zero(float top) { return fabsf(top) == INFINITY ? 0.f : top; }

// `count` vectors of four neighbouring results, `apart` columns from one to the next.  All of y is written before all of the
// slopes: a line of either is then whole in the L2 when it leaves (written in turn, 16384 x 8192 results and slopes were 1.01 GB of
// writes instead of 0.54).
template <typename T, int ACT, int COUNT>
__device__ __forceinline__ void epilogue(const GemmArgs &a, long long m, long long n0, int apart, const float (*v)[4]) {
  typedef typename SlopeOf<T>::type D;
  const long long row = m * a.N, row_c = m * a.ldc;
  const float norm = ACT == kActNone && a.norm ? *a.norm : 1.f;
  const bool out = ACT == kActNone && a.left_out && a.left_out[m] < 0;   // (gradients of zero times a weight that is no number)
  if (a.vec4) {
    if (n0 >= a.N) return;
    T t[COUNT][4];
    D d[COUNT][4];
    if (a.res) {
#pragma unroll
      for (int k = 0; k < COUNT; k++) {   // (a vector behind the row reads the first one again)
        const long long n = n0 + k * apart < a.N ? n0 + k * apart : n0;
        __builtin_memcpy(t[k], __builtin_assume_aligned((const T *)a.res + row + n, 4 * sizeof(T)), 4 * sizeof(T));
      }
    } else {
#pragma unroll
      for (int k = 0; k < COUNT; k++)
#pragma unroll
        for (int i = 0; i < 4; i++) t[k][i] = (T)0.f;
    }
#pragma unroll
    for (int k = 0; k < COUNT; k++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        float y, s;
        act_both<ACT>(ACT == kActNone ? (out ? 0.f : v[k][i] * norm) : v[k][i], y, s, a.act == kActRelu);
        t[k][i] = from_f<T>(y + to_f(t[k][i]));
        d[k][i] = from_f<D>(s);
      }
#pragma unroll
    for (int k = 0; k < COUNT; k++)
      if (n0 + k * apart < a.N) __builtin_memcpy(__builtin_assume_aligned((T *)a.c + row_c + n0 + k * apart, 4 * sizeof(T)), t[k], 4 * sizeof(T));
    if (a.slope)
#pragma unroll
      for (int k = 0; k < COUNT; k++)
        if (n0 + k * apart < a.N) __builtin_memcpy(__builtin_assume_aligned((D *)a.slope + row + n0 + k * apart, 4 * sizeof(D)), d[k], 4 * sizeof(D));
    return;
  }
#pragma unroll
  for (int k = 0; k < COUNT; k++)
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const long long n = n0 + k * apart + i;
      if (n >= a.N) break;
      float y, s;
      act_both<ACT>(ACT == kActNone ? (out ? 0.f : v[k][i] * norm) : v[k][i], y, s, a.act == kActRelu);
      ((T *)a.c)[row_c + n] = from_f<T>(y + (a.res ? to_f(((const T *)a.res)[row + n]) : 0.f));
      if (a.slope) ((D *)a.slope)[row + n] = from_f<D>(s);
    }
}

template <typename T, bool AK, bool BKIN, int BM, int BN, int WM, int WN, int BUFS, int ACT>
__global__ void __launch_bounds__(64 * (BM / WM) * (BN / WN)) gemm_kernel(const GemmArgs a) {
  constexpr int THREADS = 64 * (BM / WM) * (BN / WN), BK = 128 / sizeof(T), FM = WM / 16, FN = WN / 16;
  constexpr int GM = sizeof(T) == 4 ? (FM < 4 ? FM : 4) : 1, GN = sizeof(T) == 4 ? (FN < 4 ? FN : 4) : 1;
  typedef Stage<T, BM, AK, THREADS, GM> SA;
  typedef Stage<T, BN, BKIN, THREADS, GN> SB;
  __shared__ __align__(16) char lds[BUFS][(BM + BN) * 128];
  // Blocks go round the eight XCDs in turn: each XCD gets a run of neighbouring tiles, so that its L2 holds what they share;
  // in a run, eight row tiles by all columns before the next eight.
  unsigned tile = blockIdx.x;
  const unsigned tiles = a.mtiles * a.ntiles, even = tiles / 8 * 8;
  if (tile < even) tile = tile % 8 * (even / 8) + tile / 8;
  const unsigned band = tile / (8 * a.ntiles), in_band = tile - band * 8 * a.ntiles, high = min(8u, a.mtiles - band * 8);
  const long long m0 = (long long)(band * 8 + in_band % high) * BM;
  const long long n0 = (long long)(in_band / high) * BN;
  const long long k0 = blockIdx.y * a.kper, k1 = min(k0 + a.kper, a.K);
  const int wave = threadIdx.x / 64, wm = wave % (BM / WM) * WM, wn = wave / (BM / WM) * WN;

  // sums begin with the bias (of the first piece of k)
  f32x4 acc[FM][FN];
  const int lane = threadIdx.x % 64, c = lane % 16, q = lane / 16;
#pragma unroll
  for (int j = 0; j < FN; j++) {
    f32x4 b = {0.f, 0.f, 0.f, 0.f};
    if (a.bias && blockIdx.y == 0) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const long long n = n0 + wn + j / GN * GN * 16 + (q * 4 + e) * GN + j % GN;
        b[e] = to_f(((const T *)a.bias)[n < a.N ? n : a.N - 1]);
      }
    }
#pragma unroll
    for (int i = 0; i < FM; i++) acc[i][j] = b;
  }

  SA sa;
  SB sb;
  sa.init(a.a, a.lda, m0, a.M, k0);
  sb.init(a.b, a.ldb, n0, a.N, k0);
  long long left = k1 - k0;
  auto issue = [&](int buf) __attribute__((always_inline)) {
    sa.issue(lds[buf], left);
    sb.issue(lds[buf] + BM * 128, left);
    left -= BK;
  };
  // the fragments of half a step, and their products
  struct Half {
    s16x8 a16[sizeof(T) == 2 ? FM : 1], b16[sizeof(T) == 2 ? FN : 1];
    float a32[sizeof(T) == 4 ? FM : 1][4], b32[sizeof(T) == 4 ? FN : 1][4];
  };
  auto read = [&](Half &h, int buf, int ks) __attribute__((always_inline)) {
    const char *la = lds[buf], *lb = lds[buf] + BM * 128;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int j = 0; j < FN; j++) h.b16[j] = SB::frag16(lb, wn + j * 16, ks);
#pragma unroll
      for (int i = 0; i < FM; i++) h.a16[i] = SA::frag16(la, wm + i * 16, ks);
    } else {
#pragma unroll
      for (int j = 0; j < FN; j += GN) SB::frag32(lb, wn + j * 16, ks, h.b32 + j);
#pragma unroll
      for (int i = 0; i < FM; i += GM) SA::frag32(la, wm + i * 16, ks, h.a32 + i);
    }
    if (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);   // (asked for before the products that they are read beside)
  };
  auto multiply = [&](const Half &h) __attribute__((always_inline)) {
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int i = 0; i < FM; i++)
#pragma unroll
        for (int j = 0; j < FN; j++) acc[i][j] = mfma(h.b16[j], h.a16[i], acc[i][j], T());
    } else {
#pragma unroll
      for (int k = 0; k < 4; k++)
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
          for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(h.b32[j][k], h.a32[i][k], acc[i][j], 0, 0, 0);
    }
    if (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
  };
  // What this wave has copied into LDS is there, but for the copies of `behind` tiles asked for last; what it reads from there it has.
  static_assert(BUFS == 2 || (SA::PIECES % THREADS == 0 && SB::PIECES % THREADS == 0), "every wave makes as many copies of a tile");
  auto arrive = [&](bool behind) __attribute__((always_inline)) {
    if (BUFS > 2 && behind) asm volatile("s_waitcnt vmcnt(%0)" : : "n"((BUFS - 2) * (SA::NL + SB::NL)) : "memory");
    else asm volatile("s_waitcnt vmcnt(0)" : : : "memory");
    __syncthreads();
  };
  // Half a step is multiplied while the fragments of the next half are on their way from LDS.  The barrier of a step lies between
  // its halves: everybody holds all of this tile then, so its buffer is free for the tile BUFS steps on, and the next tile, asked for
  // BUFS - 1 steps ago, is there.  (Three buffers for the tiles of small products, whose time is how soon their data come.)
  const int steps = left > 0 ? (int)((left + BK - 1) / BK) : 0;
  if (steps) {
    issue(0);
    if (BUFS > 2 && steps > 1) issue(1);
    arrive(steps > 1);
  }
  // (float32: a half is 1024 cycles of products to one LDS latency; the compiler's own order of reads and products is better there by
  // 2 to 40 %.)
  if constexpr (sizeof(T) == 4) {
    Half h;
    for (int t = 0, buf = 0; t < steps; t++, buf = buf + 1 == BUFS ? 0 : buf + 1) {
      if (t + BUFS - 1 < steps) issue(buf == 0 ? BUFS - 1 : buf - 1);
      read(h, buf, 0);
      multiply(h);
      read(h, buf, 1);
      multiply(h);
      if (t + 1 < steps) arrive(t + 2 < steps);
    }
  } else if (steps) {
    Half h0, h1;
    if (steps > BUFS - 1) issue(BUFS - 1);
    read(h0, 0, 0);
    for (int t = 0, buf = 0; t < steps; t++) {
      const int next = buf + 1 == BUFS ? 0 : buf + 1;
      read(h1, buf, 1);
      multiply(h0);
      if (t + 1 < steps) {
        arrive(t + 2 < steps);
        if (t + BUFS < steps) issue(buf);
        read(h0, next, 0);
      }
      multiply(h1);
      buf = next;
    }
  }

  if constexpr (ACT >= kLossSums) {
    // a lane holds FN vectors of four neighbouring logits of FM rows
    constexpr int apart = GN == 1 ? 16 : 4;
    const int nl = wn + (GN == 1 ? q * 4 : q * 4 * GN), left = (int)min((long long)BN, a.N - n0);   // columns of the tile: the first one's, how many there are
    auto logit = [&](int i, int k, int e) __attribute__((always_inline)) { return GN == 1 ? acc[i][k][e] : acc[i][(4 * k + e) % GN][(4 * k + e) / GN]; };
    // the class of a row as a column of the tile, -1: in another tile, or none
    auto column_of = [&](long long t) __attribute__((always_inline)) {
      const long long at = t - a.n_first - n0;
      return t >= 0 && at >= 0 && at < left ? (int)at : -1;
    };
    static_assert(FN <= 4, "");
    if constexpr (ACT == kLossSums) {
      __shared__ float2 tops[BN / WN][BM];
      const bool whole = left == BN;
#pragma unroll
      for (int i = 0; i < FM; i++) {
        const int r = wm + (i / GM * GM) * 16 + c * GM + i % GM;
        const int t = m0 + r < a.M ? column_of(a.targets[m0 + r]) : -1;
        float top = -INFINITY, sum = 0.f, own = 0.f;
#pragma unroll
        for (int k = 0; k < FN; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int n = nl + k * apart + e;
            const float z = logit(i, k, e);
            top = fmaxf(top, whole || n < left ? z : -INFINITY);
            own = n == t ? z : own;
          }
        // (only the lane that has column t writes)
        if (t >= 0 && t >= nl && (GN == 1 ? (t - nl) % 16 < 4 && t - nl < 16 * FN : t - nl < 4 * GN)) a.picked[m0 + r] = own;
        top = fmaxf(top, __shfl_xor(top, 16));
        top = fmaxf(top, __shfl_xor(top, 32));
        const float from = finite_or_zero(top);
#pragma unroll
        for (int k = 0; k < FN; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            // (the difference first: a product with log2(e) that is rounded before it loses what the logits differ by)
            const float p = __builtin_amdgcn_exp2f((logit(i, k, e) - from) * 1.44269504088896341f);
            sum += whole || nl + k * apart + e < left ? p : 0.f;
          }
        sum += __shfl_xor(sum, 16);
        sum += __shfl_xor(sum, 32);
        if (q == 0) tops[wn / WN][r] = make_float2(top, sum);
        __builtin_amdgcn_sched_barrier(0);   // (row by row: all of them at once do not fit the registers)
      }
      __syncthreads();
      for (int r = threadIdx.x; r < BM; r += THREADS) {
        if (m0 + r >= a.M) continue;
        float2 v = tops[0][r];
#pragma unroll
        for (int k = 1; k < BN / WN; k++) {
          const float2 o = tops[k][r];
          const float top = fmaxf(v.x, o.x), from = finite_or_zero(top);
          v = make_float2(top, v.y * __builtin_amdgcn_exp2f((v.x - from) * 1.44269504088896341f) + o.y * __builtin_amdgcn_exp2f((o.x - from) * 1.44269504088896341f));
        }
        a.tops[(m0 + r) * a.ntiles + n0 / BN] = v;
      }
    } else {
      float column[FN][4] = {};
      const float norm = a.norm ? *a.norm : 1.f;
      const int stored = (int)min((long long)BN, a.ldc - n0);
#pragma unroll
      for (int i = 0; i < FM; i++) {
        const long long m = m0 + wm + (i / GM * GM) * 16 + c * GM + i % GM;
        if (m < a.M) {
          const long long class_ = a.targets[m];
          const int t = column_of(class_);
          const float from = a.lse[m], g = class_ < a.N_all ? a.weight[m] * norm : __builtin_nanf("");
          T *to = (T *)a.c + m * a.ldc + n0 + nl;
#pragma unroll
          for (int k = 0; k < FN; k++) {
            T v[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int n = nl + k * apart + e;
              const float p = __builtin_amdgcn_exp2f((logit(i, k, e) - from) * 1.44269504088896341f) - (n == t ? 1.f : 0.f);
              const float gz = n < left && class_ >= 0 ? p * g : 0.f;
              column[k][e] += gz;
              v[e] = from_f<T>(gz);
            }
            if (nl + k * apart < stored) __builtin_memcpy(__builtin_assume_aligned(to + k * apart, 4 * sizeof(T)), v, 4 * sizeof(T));
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (a.columns) {
#pragma unroll
        for (int k = 0; k < FN; k++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float v = column[k][e];
#pragma unroll
            for (int d = 1; d < 16; d *= 2) v += __shfl_xor(v, d);
            const int n = nl + k * apart + e;
            if (c == 0 && n < left && m0 + wm < a.M) a.columns[(m0 + wm) / WM * a.N + n0 + n] = v;
          }
      }
    }
    return;
  }
  const long long part_row = (a.N + 3) & ~3;
  float *part = a.part ? a.part + (long long)blockIdx.y * a.M * part_row : nullptr;
#pragma unroll
  for (int i = 0; i < FM; i++) {
    const long long m = m0 + wm + (i / GM * GM) * 16 + c * GM + i % GM;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < FN; j += 4 < FN ? 4 : FN) {
      // the vectors that a lane holds of four fragments (or of all): 4 q + 0..3 of each (16 bits), or columns G e + 0..G - 1, e = 4 q + 0..3,
      // of the columns that they share
      constexpr int COUNT = FN < 4 ? FN : 4;
      float v[COUNT][4];
      const int apart = GN == 1 ? 16 : 4;
      const long long n = n0 + wn + j * 16 + (GN == 1 ? q * 4 : q * 4 * GN);
#pragma unroll
      for (int k = 0; k < COUNT; k++)
#pragma unroll
        for (int e = 0; e < 4; e++) v[k][e] = GN == 1 ? acc[i][j + k][e] : acc[i][j + (4 * k + e) % GN][(4 * k + e) / GN];
      if (part) {
#pragma unroll
        for (int k = 0; k < COUNT; k++)
          if (n + k * apart < a.N) {
            f32x4 *to = (f32x4 *)(part + m * part_row + n + k * apart);
            const f32x4 now = {v[k][0], v[k][1], v[k][2], v[k][3]};
            *to = a.add ? *to + now : now;
          }
      } else {
        epilogue<T, ACT, COUNT>(a, m, n, apart, v);
      }
    }
  }
}

template <typename T, bool AK, bool BKIN, int ACT>
void launch_tile(int tile, const GemmArgs &a, hipStream_t s) {
  const dim3 grid(a.mtiles * a.ntiles, a.splits);
#define GELIB_GEMM(BM, BN, WM, WN, BUFS)                                                                                                                 \
  do {                                                                                                                                             \
    const dim3 block(64 * (BM / WM) * (BN / WN));                                                                                                  \
    hipLaunchKernelGGL((gemm_kernel<T, AK, BKIN, BM, BN, WM, WN, BUFS, ACT>), grid, block, 0, s, a);                                                     \
  } while (0)
  switch (tile) {
    case 0: GELIB_GEMM(256, 256, 128, 64, 2); break;
    case 1: GELIB_GEMM(128, 128, 64, 64, 2); break;
    case 2: GELIB_GEMM(64, 128, 64, 32, 3); break;
    default: GELIB_GEMM(16, 256, 16, 64, 2); break;
  }
#undef GELIB_GEMM
}

template <typename T>
int launch_gemm(GemmForm form, int tile, const GemmArgs &a, hipStream_t s) {
  if (form == kFormXW) {
    if (a.act == kActSilu) launch_tile<T, true, false, kActSilu>(tile, a, s);
    else if (a.act == kActGelu) launch_tile<T, true, false, kActGelu>(tile, a, s);
    else launch_tile<T, true, false, kActNone>(tile, a, s);
  } else if (form == kFormGW) {
    launch_tile<T, true, true, kActNone>(tile, a, s);
  } else {
    launch_tile<T, false, false, kActNone>(tile, a, s);
  }
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "linear layer launch");
}

#endif

}  // namespace gelib_hip
