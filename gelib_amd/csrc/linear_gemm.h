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
// Two buffers: the next tile is on its way while this one is multiplied; one barrier a step.
//
// The products are formed with B's fragment as the first operand, so that a lane's four results lie side by side in a row of C.
#pragma once

#include "real_ops.h"

namespace gelib_hip {

struct GemmArgs {
  const void *a, *b;
  long long lda, ldb;       // elements between the rows in memory
  void *c;                  // (M, N) packed
  const void *bias, *res;   // epilogue: c = act(sum + bias) + res, slope = act'(sum + bias); each may be null
  void *slope;
  float *part;              // [splits][M][N up to a multiple of 4] sums of the pieces of k instead of c, or null
  long long M, K, kper;     // kper: k of a piece, a multiple of the step
  int N, act, splits, vec4;  // vec4: rows of c, res and slope take vectors of 4
  unsigned mtiles, ntiles;
};

enum GemmForm { kFormXW = 0, kFormGW = 1, kFormXG = 2 };   // x w, gz w^T, x^T gz

// tiles: 0: 256 x 256, 1: 128 x 128, 2: 64 x 128, 3: 16 x 256
constexpr int kGemmTiles = 4;
constexpr int kGemmBM[kGemmTiles] = {256, 128, 64, 16}, kGemmBN[kGemmTiles] = {256, 128, 128, 256};

template <typename T>
int launch_gemm(GemmForm form, int tile, const GemmArgs &a, hipStream_t s);

#ifdef __HIPCC__

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bhalf_t bf16x8 __attribute__((ext_vector_type(8)));
typedef half_t f16x8 __attribute__((ext_vector_type(8)));

template <typename T>
struct SlopeOf { typedef half_t type; };
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
  static constexpr int NL = (R * 8 + THREADS - 1) / THREADS;
  const T *p[NL];
  long long mn[NL];
  int k[NL];
  long long step;

  static __device__ __forceinline__ int swizzle(int row) {
    if (KIN) return (row / G) & 7;
    return sizeof(T) == 2 ? ((row & 3) << 1) & (CPR - 1) : 0;
  }
  __device__ __forceinline__ void init(const void *base, long long ld, long long mn0, long long MN, long long k0) {
#pragma unroll
    for (int u = 0; u < NL; u++) {
      const int L = u * THREADS + threadIdx.x, row = L / CPR, c = (L % CPR) ^ swizzle(row);
      mn[u] = mn0 + (KIN ? row : c * VEC);
      k[u] = KIN ? c * VEC : row;
      if (mn[u] >= MN) mn[u] = -1;
      p[u] = (const T *)base + (KIN ? mn[u] * ld + k0 + k[u] : (k0 + k[u]) * ld + mn[u]);
    }
    step = KIN ? BK : BK * ld;
  }
  // the tile whose first k has `left` more of it behind (k0 .. k0 + left)
  __device__ __forceinline__ void issue(char *lds, long long left) {
#pragma unroll
    for (int u = 0; u < NL; u++) {
      if (R * 8 % THREADS != 0 && u * THREADS + threadIdx.x >= R * 8) continue;   // (whole waves)
      const bool in = mn[u] >= 0 && k[u] < left;
      load_to_lds(in ? (const char *)p[u] : (const char *)gemm_zeros, lds + (u * THREADS + (threadIdx.x & ~63)) * 16);
      p[u] += step;
    }
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

// four neighbouring results of a row
template <typename T, int ACT>
__device__ __forceinline__ void epilogue4(const GemmArgs &a, long long m, int n, const float *v) {
  typedef typename SlopeOf<T>::type D;
  const long long at = m * a.N + n;
  if (a.vec4) {
    T t[4];
    D d[4];
    float b[4] = {0.f, 0.f, 0.f, 0.f}, r[4] = {0.f, 0.f, 0.f, 0.f};
    if (a.bias) {
      __builtin_memcpy(t, (const T *)a.bias + n, sizeof(t));
#pragma unroll
      for (int i = 0; i < 4; i++) b[i] = to_f(t[i]);
    }
    if (a.res) {
      __builtin_memcpy(t, __builtin_assume_aligned((const T *)a.res + at, sizeof(t)), sizeof(t));
#pragma unroll
      for (int i = 0; i < 4; i++) r[i] = to_f(t[i]);
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float y, s;
      act_both<ACT>(v[i] + b[i], y, s, a.act == kActRelu);
      t[i] = from_f<T>(y + r[i]);
      d[i] = from_f<D>(s);
    }
    __builtin_memcpy(__builtin_assume_aligned((T *)a.c + at, sizeof(t)), t, sizeof(t));
    if (a.slope) __builtin_memcpy(__builtin_assume_aligned((D *)a.slope + at, sizeof(d)), d, sizeof(d));
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; i++) {
    if (n + i >= a.N) break;
    float y, s;
    act_both<ACT>(v[i] + (a.bias ? to_f(((const T *)a.bias)[n + i]) : 0.f), y, s, a.act == kActRelu);
    ((T *)a.c)[at + i] = from_f<T>(y + (a.res ? to_f(((const T *)a.res)[at + i]) : 0.f));
    if (a.slope) ((D *)a.slope)[at + i] = from_f<D>(s);
  }
}

template <typename T, bool AK, bool BKIN, int BM, int BN, int WM, int WN, int ACT>
__global__ void __launch_bounds__(64 * (BM / WM) * (BN / WN)) gemm_kernel(const GemmArgs a) {
  constexpr int THREADS = 64 * (BM / WM) * (BN / WN), BK = 128 / sizeof(T), FM = WM / 16, FN = WN / 16;
  constexpr int GM = sizeof(T) == 4 ? (FM < 4 ? FM : 4) : 1, GN = sizeof(T) == 4 ? (FN < 4 ? FN : 4) : 1;
  typedef Stage<T, BM, AK, THREADS, GM> SA;
  typedef Stage<T, BN, BKIN, THREADS, GN> SB;
  __shared__ __align__(16) char lds[2][(BM + BN) * 128];
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

  f32x4 acc[FM][FN];
#pragma unroll
  for (int i = 0; i < FM; i++)
#pragma unroll
    for (int j = 0; j < FN; j++) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

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
  auto arrive = [&]() __attribute__((always_inline)) {
    asm volatile("s_waitcnt vmcnt(0)" : : : "memory");   // what this wave has copied into LDS is there
    __syncthreads();
  };
  const int steps = left > 0 ? (int)((left + BK - 1) / BK) : 0;
  if (steps) {
    issue(0);
    arrive();
  }
  for (int t = 0, buf = 0; t < steps; t++, buf ^= 1) {
    const bool more = t + 1 < steps;
    if (more) issue(buf ^ 1);
    const char *la = lds[buf], *lb = lds[buf] + BM * 128;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        s16x8 fa[FM], fb[FN];
#pragma unroll
        for (int i = 0; i < FM; i++) fa[i] = SA::frag16(la, wm + i * 16, ks);
#pragma unroll
        for (int j = 0; j < FN; j++) fb[j] = SB::frag16(lb, wn + j * 16, ks);
#pragma unroll
        for (int i = 0; i < FM; i++)
#pragma unroll
          for (int j = 0; j < FN; j++) acc[i][j] = mfma(fb[j], fa[i], acc[i][j], T());
      }
    } else {
#pragma unroll
      for (int ks = 0; ks < 2; ks++) {
        float fa[FM][4], fb[FN][4];
#pragma unroll
        for (int i = 0; i < FM; i += GM) SA::frag32(la, wm + i * 16, ks, fa + i);
#pragma unroll
        for (int j = 0; j < FN; j += GN) SB::frag32(lb, wn + j * 16, ks, fb + j);
#pragma unroll
        for (int k = 0; k < 4; k++)
#pragma unroll
          for (int i = 0; i < FM; i++)
#pragma unroll
            for (int j = 0; j < FN; j++) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(fb[j][k], fa[i][k], acc[i][j], 0, 0, 0);
      }
    }
    if (more) arrive();
  }

  const int lane = threadIdx.x % 64, c = lane % 16, q = lane / 16;
  const long long part_row = (a.N + 3) & ~3;
  float *part = a.part ? a.part + (long long)blockIdx.y * a.M * part_row : nullptr;
  auto out = [&](long long m, long long n, const float *v) __attribute__((always_inline)) {
    if (m >= a.M || n >= a.N) return;
    if (part) {
      *(f32x4 *)(part + m * part_row + n) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
      epilogue4<T, ACT>(a, m, (int)n, v);
    }
  };
#pragma unroll
  for (int i = 0; i < FM; i++) {
    const long long m = m0 + wm + (i / GM * GM) * 16 + c * GM + i % GM;
    if (sizeof(T) == 2 || GN == 1) {
#pragma unroll
      for (int j = 0; j < FN; j++) {
        const float v[4] = {acc[i][j][0], acc[i][j][1], acc[i][j][2], acc[i][j][3]};
        out(m, n0 + wn + j * 16 + q * 4, v);
      }
    } else if constexpr (GN == 4) {
#pragma unroll
      for (int j = 0; j < FN; j += GN)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const float v[4] = {acc[i][j][e], acc[i][(j + 1) % FN][e], acc[i][(j + 2) % FN][e], acc[i][(j + 3) % FN][e]};
          out(m, n0 + wn + j * 16 + q * 16 + e * 4, v);
        }
    } else {   // two columns a lane: elements 2 e, 2 e + 1
#pragma unroll
      for (int j = 0; j < FN; j += GN)
#pragma unroll
        for (int e = 0; e < 4; e += 2) {
          const float v[4] = {acc[i][j][e], acc[i][(j + 1) % FN][e], acc[i][j][e + 1], acc[i][(j + 1) % FN][e + 1]};
          out(m, n0 + wn + j * 16 + q * 8 + e * 2, v);
        }
    }
  }
}

template <typename T, bool AK, bool BKIN, int ACT>
void launch_tile(int tile, const GemmArgs &a, hipStream_t s) {
  const dim3 grid(a.mtiles * a.ntiles, a.splits);
#define GELIB_GEMM(BM, BN, WM, WN)                                                                                                                 \
  do {                                                                                                                                             \
    const dim3 block(64 * (BM / WM) * (BN / WN));                                                                                                  \
    hipLaunchKernelGGL((gemm_kernel<T, AK, BKIN, BM, BN, WM, WN, ACT>), grid, block, 0, s, a);                                                     \
  } while (0)
  switch (tile) {
    case 0: GELIB_GEMM(256, 256, 128, 64); break;
    case 1: GELIB_GEMM(128, 128, 64, 64); break;
    case 2: GELIB_GEMM(64, 128, 64, 32); break;
    default: GELIB_GEMM(16, 256, 16, 64); break;
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
