// Attention over the points of a document, s_ij = scale q_i . k_j - slope_h |x_i - y_j|, y_i = sum_j softmax_j(s_ij) v_j, in one pass over
// the keys with the running maximum and sum of each row, and its gradients in two passes, one by query rows and one by keys:
//   p_ij = exp(s_ij - lse_i),  D_i = gy_i . y_i,  ds_ij = p_ij (gy_i . v_j - D_i),
//   gq_i = scale sum_j ds_ij k_j,  gk_j = scale sum_i ds_ij q_i,  gv_j = sum_i p_ij gy_i,
//   gslope_h = - sum ds_ij d_ij,  gx_i = - slope sum_j ds_ij (x_i - y_j) / d_ij,  gy_j the same with the other sign.
// Sums, maxima and statistics are float32 throughout.  16-bit types round p and ds to the type of the operands that the matrix
// cores multiply them with; l and D are sums of unrounded values.
//
// Every pass has rows of its own, 16 QS a wave, whose operands and results stay in registers, and streams the other side through LDS
// in tiles of BN rows.  Scores are formed as (streamed) x (own)^T: a lane then holds four neighbouring streamed rows of ONE own row, so
// that maximum, sum and rescaling are a lane's own business but for two shuffles a tile, and the four values are, as they stand, the operand of
// the product with the transposed tile that follows (16 bits: two tiles of 16 rows side by side, the order of k being free; the
// transposed fragments are read by the LDS unit's transposing loads.  float32: each of the four is one step of k).
// A document's query rows are its (position, head of the group) pairs: heads that share keys stand in one tile.
//
// What bounds it: the vector unit, 70 to 75 % busy with the distances, exponentials and sums between the products.  8192 points, 16 heads of 64
// on 4, bfloat16, with points: forward 556 us (495 TFLOP/s), by rows 931, by keys 915; 16 on 16, without points: forward 411 us (669), both
// directions 1630 (590); 2 x 8192, 8 heads of 128 on 2, without points: forward 618 (890).  float16 scales its weights and their gradients
// (kHalfTop): forward 577, both directions 2693 where bfloat16 has 556 and 2430.  Short documents: the instructions around the
// products (addresses, rows, results): 2048 packed documents of up to 60 rows, 8 heads of 32, bfloat16: 63, 96 and 101 us.
#pragma once

#include <type_traits>

#include "real_ops.h"

namespace gelib_hip {

struct AttnArgs {
  const void *q, *k, *v, *gy;   // backward: gy and y at a stride of ldy from one (row, head) to the next
  void *y, *gq, *gk, *gv;       // packed: (rows, heads, dim)
  long long qs, ks, vs;          // strides of samples in elements
  int qp, qh, kp, kh, vp, vh;    // of positions and heads: operands with larger ones are copied (a multiplication instead of five)
  const float *x, *xk, *slopes;   // points of queries and keys (rows, 3), heads
  const int *q_marks, *k_marks;   // padded: lengths or null (all rows); packed: starts, docs + 1 of them
  float *lse, *delta;           // (query rows, heads): log2 of the sum of exp; D
  float *part_q, *part_k, *part_v;   // sums of the pieces of the streamed side: [splits][rows][heads][dim], or null
  float *part_p, *part_d;       // 16-bit types' gradients by query rows: sums of p k and of ds besides (see there)
  float2 *part_ml;              // forward: maximum and sum of every piece
  float4 *geo_q, *geo_k, *geo_p;   // [splits][rows][heads]: gradients of points, of the slope; what goes with part_p
  long long docs, nq, nk;       // padded: rows of a sample; packed: all rows
  long long rows_q, rows_k;     // all of them
  long long slots, first;       // blocks of the whole call (one piece, one head), the first of this launch
  int packed, H, KV, G, dim, ldy, splits, g_shift, blocked, heads;   // blocked: row order (RowAt); heads of keys, one after the other in a block
  unsigned g_magic;   // division of row numbers by G (group_of)
  int head_major, vec_y;   // vec_y: results take vectors of four
  float scale, scale2;          // scale2: times log2(e)
};

enum AttnBias { kBiasNone = 0, kBiasPoints = 1, kBiasGradients = 2 };

// what a launch is made for; dims: 16 (float32 only: a step of the 16-bit products is 32), 32, 64 or 128 values of a head in LDS
struct AttnPlan {
  int dims, bias;
  bool wide;   // four waves a block
};
enum AttnPass { kAttnForward, kAttnRows, kAttnKeys };
// 16 QS own rows a wave: four waves a block take two tiles each, which share every fragment of the streamed side, where registers hold
// their operands and results (share: and their distances, see RowAt); a wave alone one, since the documents are short.
constexpr int attention_qs(AttnPass pass, int element, int dims, bool wide, bool share) {
  return !wide || (dims == 128 && (pass != kAttnForward || element == 4)) || (dims == 64 && pass == kAttnRows && element == 2 && !share) ? 1 : 2;
}
constexpr int attention_rows(AttnPass pass, int element, int dims, bool wide, bool share) { return 16 * attention_qs(pass, element, dims, wide, share) * (wide ? 4 : 1); }
template <AttnPass PASS, typename T>
int launch_attention_kernels(const AttnPlan &p, const AttnArgs &a, hipStream_t s);

#ifdef __HIPCC__

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef bhalf_t bf16x8 __attribute__((ext_vector_type(8)));
typedef half_t f16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ f32x4 attn_mfma(s16x8 a, s16x8 b, f32x4 c, bhalf_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 attn_mfma(s16x8 a, s16x8 b, f32x4 c, half_t) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

constexpr float kLowest = -3.0e38f;

// float16's least normal value is 2^-14, and what the second products take as float16 values may lie anywhere below: weights, one over the number
// of keys, and their scores' gradients, which are as small or large as the loss's.  Powers of two bring them into its range, and the float32
// results are scaled back.
//   Forward: the largest weight of the first keys stands at 2^7 (kHalfTop), and the largest at 2^15 before the maximum is moved.
//   Gradients of values: weights, at most one, stand at 2^12 (kHalfUp: 2^4 to spare for scores so large that exp(s - lse) is off by that).
//   Both are multiplied after the exponential: 12 more in front of it would round s - lse, and gradients of points, three times as coarsely.
//   ds: each own row has a power of two of its own, which is chosen when its first ds come so that the largest is 2^11 to 2^12, and again when
//   one is beyond 2^15 (Lift).
template <typename T>
constexpr bool kIsHalf = std::is_same<T, half_t>::value;
constexpr float kHalfTop = 0x1p7f, kHalfUp = 0x1p12f;

// A document as a block sees it: where its rows begin in the strided operands and in packed results, how many exist, and how many there
// are to write (rows that do not exist get zeros).
struct AttnDoc {
  long long sample, q0, k0, out_q, out_k;   // q0, k0: positions within the sample (packed: of all)
  int qn, kn, own_all, tile;                // tile: of own rows, in the document
};

// row / G for rows below 2^31
__device__ __forceinline__ int group_of(const AttnArgs &a, int row) { return a.G == 1 ? row : (int)(__umulhi((unsigned)row, a.g_magic) >> a.g_shift); }

// Row of a document -> position and head of the group: heads side by side, or (blocked; the group is 2, 4 or 8) 16 positions of one head behind
// 16 of the next, so that neighbouring tiles of a wave have the same positions and share their distances.
struct RowAt {
  int pos, head;
};
__device__ __forceinline__ RowAt row_at(const AttnArgs &a, int row) {
  if (a.blocked) {
    const int tile = row >> 4, shift = 31 - __clz(a.G);
    return {((tile >> shift) << 4) + (row & 15), tile & (a.G - 1)};
  }
  const int pos = group_of(a, row);
  return {pos, row - pos * a.G};
}
__device__ __forceinline__ long long rows_in(const AttnArgs &a, int positions) { return (long long)(a.blocked ? (positions + 15) & ~15 : positions) * a.G; }

__device__ __forceinline__ int held(int v, long long lo, long long hi) { return (int)max(lo, min((long long)v, hi)); }

// Packed documents: starts are held to 0..all and to one another's order pair by pair; 0 and the number of rows stand before and behind
// them, so that rows outside of all documents belong to two that see nothing.  Document j's tiles have the numbers from
// starts[j] per / rows + j on: at least as many as it needs, without a sum over the documents before it.
__device__ __forceinline__ int start_of(const int *starts, long long docs, long long all, long long j) {
  return j == 0 ? 0 : j == docs + 2 ? (int)all : held(starts[j - 1], 0, all);
}

template <bool OWN_Q>
__device__ __forceinline__ AttnDoc find_doc(const AttnArgs &a, long long slot, int rows) {
  AttnDoc d;
  const int per = OWN_Q ? a.G : 1;
  const long long all = OWN_Q ? a.nq : a.nk;
  if (!a.packed) {
    const long long tiles = (all * per + rows - 1) / rows;
    d.sample = slot / tiles, d.tile = (int)(slot - d.sample * tiles);
    d.q0 = d.k0 = 0, d.out_q = d.sample * a.nq, d.out_k = d.sample * a.nk;
    d.qn = a.q_marks ? held(a.q_marks[d.sample], 0, a.nq) : (int)a.nq;
    d.kn = a.k_marks ? held(a.k_marks[d.sample], 0, a.nk) : (int)a.nk;
    d.own_all = (int)all;
    return d;
  }
  const int *own = OWN_Q ? a.q_marks : a.k_marks, *other = OWN_Q ? a.k_marks : a.q_marks;
  // the last document whose first slot is not behind this one: every lane asks for one of 64 borders at a time
  long long lo = 0, hi = a.docs + 2;
  while (hi - lo > 1) {
    const long long step = (hi - lo + 63) / 64, mid = lo + step * (threadIdx.x % 64 + 1);
    const bool not_behind = mid < hi && (long long)start_of(own, a.docs, all, mid) * per / rows + mid <= slot;
    // (starts that are in no order: the first border that is behind counts)
    const unsigned long long no = ~__ballot(not_behind);
    const int n = no ? __ffsll(no) - 1 : 64;
    hi = min(hi, lo + step * (n + 1)), lo += step * n;
  }
  const int b = start_of(own, a.docs, all, lo), e = max(b, start_of(own, a.docs, all, lo + 1));
  const bool real = lo >= 1 && lo <= a.docs;
  const long long other_all = OWN_Q ? a.nk : a.nq;
  const int ob = real ? start_of(other, a.docs, other_all, lo) : 0, oe = real ? max(ob, start_of(other, a.docs, other_all, lo + 1)) : 0;
  d.sample = 0, d.tile = (int)(slot - ((long long)b * per / rows + lo));
  d.q0 = OWN_Q ? b : ob, d.k0 = OWN_Q ? ob : b;
  d.out_q = d.q0, d.out_k = d.k0;
  d.own_all = e - b;
  d.qn = OWN_Q ? (real ? e - b : 0) : oe - ob, d.kn = OWN_Q ? oe - ob : (real ? e - b : 0);
  return d;
}

// 16 bytes of a row from its element c * (16 / sizeof(T)) on, zeros behind its end.  Rows lie at multiples of 16 bytes and end in zeros up to
// the next one: the host copies operands that do not (attention.hip).
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T *row, int c, int dim, bool live) {
  const int d = c * (16 / (int)sizeof(T));
  uint4 r = {0, 0, 0, 0};
  if (live && d < dim) r = *(const uint4 *)__builtin_assume_aligned(row + d, 16);
  return r;
}

// Tiles in LDS: rows of DP values in pieces of 16 bytes, whose order in a row is permuted (exclusive or) so that both kinds of reads spread
// over the banks: 16 rows of one piece (a fragment), and 8 rows of the 32 bytes that a transposing read takes of each.
template <typename T, int DP>
struct AttnTile {
  static constexpr int W = DP * (int)sizeof(T), PPR = W / 16, RP = W >= 256 ? 1 : 256 / W, EP = 16 / (int)sizeof(T);
  static constexpr int KS = sizeof(T) == 2 ? DP / 32 : DP / 16;   // steps of k of a row product
  static constexpr int NF = DP / 16;                              // fragments of a result row
  typedef typename std::conditional<sizeof(T) == 2, s16x8, f32x4>::type Frag;
  static __device__ __forceinline__ int swizzle(int row) {
    if (sizeof(T) == 2) return ((row / RP & (PPR / 2 - 1)) << 1) | (row >> 3 & 1);
    return row / RP & (PPR < 16 ? PPR - 1 : 15);
  }
  // of row row0 + lane % 16: k = ks * 32 + lane / 16 * 8 + 0..7, or ks * 16 + lane / 16 * 4 + 0..3
  static __device__ __forceinline__ Frag frag(const char *lds, int row0, int ks) {
    const int lane = threadIdx.x % 64, row = row0 + lane % 16;
    return *(const Frag *)(lds + row * W + (((ks * 4 + lane / 16) ^ swizzle(row)) << 4));
  }
  // of a row in global memory, the same
  static __device__ __forceinline__ Frag frag_of(const T *row, int ks, int dim, bool live) {
    return __builtin_bit_cast(Frag, load_piece(row, ks * 4 + (threadIdx.x % 64) / 16, dim, live));
  }
  static __device__ __forceinline__ f32x4 product(Frag a, Frag b, f32x4 c) {
    if constexpr (sizeof(T) == 2) {
      return attn_mfma(a, b, c, T());
    } else {
#pragma unroll
      for (int i = 0; i < 4; i++) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
      return c;
    }
  }
  // acc += (rows row0 .. row0 + 31 of the tile)^T p; p0, p1: a lane's values of rows row0 + 4 (lane / 16) + 0..3 and of the 16 rows on
  // Result fragments: 16 bits: f holds values 16 f + 4 (lane / 16) + 0..3 of own row lane % 16; float32: below (place).
  template <int QS>
  static __device__ __forceinline__ void transposed(f32x4 (*acc)[NF], const char *lds, int row0, const f32x4 (*p0), const f32x4 (*p1)) {
    const int lane = threadIdx.x % 64, c = lane % 16, q = lane / 16;
    if constexpr (sizeof(T) == 2) {
      s16x8 b[QS];
#pragma unroll
      for (int s = 0; s < QS; s++) {
        T t[8];
#pragma unroll
        for (int i = 0; i < 4; i++) t[i] = (T)p0[s][i], t[4 + i] = (T)p1[s][i];
        __builtin_memcpy(&b[s], t, 16);
      }
#pragma unroll
      for (int f = 0; f < NF; f++) {
        s16x4 h[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          const int row = row0 + 16 * i + 4 * q + c / 4, col = f * 16 + c % 4 * 4;
          const char *at = lds + row * W + (((col / 8) ^ swizzle(row)) << 4) + col % 8 * 2;
          h[i] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)at);
        }
        const s16x8 v = __builtin_shufflevector(h[0], h[1], 0, 1, 2, 3, 4, 5, 6, 7);
#pragma unroll
        for (int s = 0; s < QS; s++) acc[s][f] = attn_mfma(v, b[s], acc[s][f], T());
      }
    } else {
      constexpr int GV = NF < 4 ? NF : 4;   // neighbouring values of a lane: one read serves GV fragments
#pragma unroll
      for (int i = 0; i < 8; i++) {
        const int row = row0 + 16 * (i / 4) + 4 * q + i % 4;
#pragma unroll
        for (int f0 = 0; f0 < NF; f0 += GV) {
          float v[GV];
          const int at = (f0 * 16 + c * GV) * 4;
          __builtin_memcpy(v, __builtin_assume_aligned(lds + row * W + (((at >> 4) ^ swizzle(row)) << 4) + (at & 15), GV * 4), GV * 4);
#pragma unroll
          for (int g = 0; g < GV; g++)
#pragma unroll
            for (int s = 0; s < QS; s++)
              acc[s][f0 + g] = __builtin_amdgcn_mfma_f32_16x16x4f32(v[g], i < 4 ? p0[s][i % 4] : p1[s][i % 4], acc[s][f0 + g], 0, 0, 0);
        }
      }
    }
  }
  // Writes a lane's results of one own row: f(d, four neighbouring values from d on)
  template <typename F>
  static __device__ __forceinline__ void results(const f32x4 *acc, F f) {
    const int q = threadIdx.x % 64 / 16;
    if constexpr (sizeof(T) == 2) {
#pragma unroll
      for (int k = 0; k < NF; k++) f(k * 16 + 4 * q, acc[k]);
    } else {
      constexpr int GV = NF < 4 ? NF : 4;
#pragma unroll
      for (int f0 = 0; f0 < NF; f0 += GV)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          // vector e of the four: values 4 e .. 4 e + 3 of the 4 GV that the lane holds, value n in fragment n % GV at n / GV
          if (e >= GV) break;
          f32x4 v;
#pragma unroll
          for (int i = 0; i < 4; i++) v[i] = acc[f0 + (4 * e + i) % GV][(4 * e + i) / GV];
          f(f0 * 16 + q * 4 * GV + 4 * e, v);
        }
    }
  }
};

// four values of a packed row at d, what is behind its end left out
template <typename T>
__device__ __forceinline__ void store4(T *row, int d, int dim, bool vec, f32x4 v) {
  if (vec) {
    if (d >= dim) return;
    T t[4];
#pragma unroll
    for (int i = 0; i < 4; i++) t[i] = from_f<T>(v[i]);
    __builtin_memcpy(__builtin_assume_aligned(row + d, 4 * sizeof(T)), t, 4 * sizeof(T));
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++)
      if (d + i < dim) row[d + i] = from_f<T>(v[i]);
  }
}

// the other three lanes of an own row
__device__ __forceinline__ float over_row_max(float v) {
  v = fmaxf(v, __shfl_xor(v, 16));
  return fmaxf(v, __shfl_xor(v, 32));
}
__device__ __forceinline__ float over_row_sum(float v) {
  v += __shfl_xor(v, 16);
  return v + __shfl_xor(v, 32);
}

// The kernels that have no register to spare for Lift: float16, 64 values, gradients of points, four waves
template <typename T, int DP, int BIAS, int WAVES>
constexpr bool kFrugal = kIsHalf<T> && DP == 64 && BIAS == kBiasGradients && WAVES > 1;
// They do one thing after the other (what the compiler would begin early takes registers)
template <bool FRUGAL>
__device__ __forceinline__ void in_turn() {
  if constexpr (FRUGAL) __builtin_amdgcn_sched_barrier(0);
}

// Powers of two of the gradients of scores (float16 only)
template <typename T, int QS>
struct Lift {
  float by[QS];   // zero: not chosen yet
  __device__ __forceinline__ Lift() {
#pragma unroll
    for (int s = 0; s < QS; s++) by[s] = 0.f;
  }
  // d[u][s], of 32 streamed rows: times their powers of two, which acc, the sums so far, follow
  template <int SETS, int NF>
  __device__ __forceinline__ void apply(f32x4 (*d)[SETS], f32x4 (*acc)[NF]) {
    if constexpr (!kIsHalf<T>) return;
#pragma unroll
    for (int s = 0; s < QS; s++) {
      float top = 0.f;
#pragma unroll
      for (int u = 0; u < 2; u++)
#pragma unroll
        for (int i = 0; i < 4; i++) top = fmaxf(top, fabsf(d[u][s][i]));
      // (a lane's own values tell whether there is anything to do: the row's other lanes are asked then only)
      if (__any(by[s] == 0.f ? top > 0.f : top * by[s] > 0x1p15f)) {
        top = over_row_max(top);
        const bool grown = by[s] == 0.f ? top > 0.f : top * by[s] > 0x1p15f;
        // (frexp's exponent of a value from 1/2 to 1 is zero, that of 2^n is n + 1)
        const int to = max(-120, min(120, 12 - __builtin_amdgcn_frexp_expf(top))), more = grown ? to - (__builtin_amdgcn_frexp_expf(by[s]) - 1) : 0;
#pragma unroll
        for (int f = 0; f < NF; f++)
#pragma unroll
          for (int i = 0; i < 4; i++) acc[s][f][i] = ldexpf(acc[s][f][i], more);   // (zeros if nothing was chosen yet)
        by[s] = grown ? ldexpf(1.f, to) : by[s];
      }
#pragma unroll
      for (int u = 0; u < 2; u++) d[u][s] *= by[s];
    }
  }
  // the sums as they are
  template <int NF>
  __device__ __forceinline__ void down(f32x4 (*acc)[NF]) const {
    if constexpr (!kIsHalf<T>) return;
#pragma unroll
    for (int s = 0; s < QS; s++) {
      const int less = by[s] == 0.f ? 0 : 1 - __builtin_amdgcn_frexp_expf(by[s]);
#pragma unroll
      for (int f = 0; f < NF; f++)
#pragma unroll
        for (int i = 0; i < 4; i++) acc[s][f][i] = ldexpf(acc[s][f][i], less);
    }
  }
};

typedef __attribute__((address_space(3))) char *AttnLds;

// 16 (or 4) bytes of every lane to LDS, lane after lane from `to` (the same for the whole wave) on.  Written out because the compiler, which
// cannot tell two buffers apart, would wait for the builtin's copy before the next read of either; the wave waits by itself (arrive()).  No
// register is written but m0, which is reserved: the compiler keeps nothing there, and cannot be told of it as clobbered (nothing but these
// copies names it in the kernels).
__device__ __forceinline__ void attn_copy16(const void *from, char *to) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(AttnLds)to);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" : : "s"(at), "v"(from) : "memory");
}
__device__ __forceinline__ void attn_copy4(const void *from, char *to) {
  const unsigned at = __builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)(AttnLds)to);
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dword %1, off" : : "s"(at), "v"(from) : "memory");
}

static __device__ const float4 attn_zeros[1] = {};                                       // what stands for rows that do not exist
static __device__ const float attn_infinity[1] = {__builtin_inff()};                     // and for their lse: no key has a share

// Copies of the tile `buf` ago have arrived, and nobody reads the buffer that is filled next.  (One wave alone: its reads are done.)
template <int WAVES>
__device__ __forceinline__ void arrive() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" : : : "memory");
  if (WAVES > 1) __syncthreads();
}

// A tile of the streamed side straight into LDS, as far as whole pairs of 16 rows exist: row_of(row) is a row's address, null where it does
// not exist (from `left` on none does).
// FRUGAL: rows and places are formed for each tile again, which frees registers.
template <typename T, int DP, int BN, int THREADS, bool FRUGAL, typename F>
__device__ __forceinline__ void copy_tile(char *lds, F row_of, int left, int dim) {
  typedef AttnTile<T, DP> Tile;
  constexpr int NL = BN * Tile::PPR / THREADS, DOWN = THREADS / Tile::PPR;
  static_assert(BN * Tile::PPR % THREADS == 0 && THREADS % Tile::PPR == 0, "");
  int id = threadIdx.x;
  if constexpr (FRUGAL) asm volatile("" : "+v"(id));   // (as far as the compiler knows another number each time)
  const int row0 = id / Tile::PPR, slot = id % Tile::PPR, wave0 = threadIdx.x & ~63;
#pragma unroll 4
  for (int u = 0; u < NL; u++) {
    if (u * DOWN >= ((left + 31) & ~31)) break;
    const int row = row0 + u * DOWN, c = slot ^ Tile::swizzle(row);
    const T *at = row < left && c * Tile::EP < dim ? row_of(row) : nullptr;
    attn_copy16(at ? (const void *)(at + c * Tile::EP) : (const void *)attn_zeros, lds + (u * THREADS + wave0) * 16);
  }
}
// One number a row, row after row (64 of them are written): at(row) is its address.
template <typename F>
__device__ __forceinline__ void copy_numbers(float *lds, F at) { attn_copy4(at(threadIdx.x % 64), (char *)lds); }

// f(t, buffer) for the tiles from t0 to t1, each copied while the one before it is at work (four waves, two buffers) or right before
// (one wave: the others of its compute unit work meanwhile)
template <int WAVES, typename B, typename C, typename F>
__device__ __forceinline__ void each_tile(B *b, int t0, int t1, C copy, F f) {
  if constexpr (WAVES > 1) {
    if (t0 < t1) copy(t0, b[0]);
    for (int t = t0, buf = 0; t < t1; t++, buf ^= 1) {
      arrive<WAVES>();
      if (t + 1 < t1) copy(t + 1, b[buf ^ 1]);
      f(t, b[buf]);
    }
  } else {
    for (int t = t0; t < t1; t++) {
      asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
      copy(t, b[0]);
      arrive<WAVES>();
      f(t, b[0]);
    }
  }
}

// streamed rows of a tile: 64, half as many where a row is 512 bytes
template <typename T, int DP>
constexpr int kAttnBN = DP * sizeof(T) >= 512 ? 32 : 64;

// Block -> slot, head of keys, piece.  Blocks go round the eight XCDs in turn: each gets a run of neighbours, which share keys (one head's
// tiles) or, where documents are a tile or two, memory lines (a row's heads).
struct AttnWork {
  long long slot;
  int kv, split;
};
// (w.kv: the block's first head of keys)
__device__ __forceinline__ AttnWork work_of(const AttnArgs &a) {
  AttnWork w;
  const unsigned even = gridDim.x / 8 * 8;
  unsigned id = blockIdx.x;
  if (id < even) id = id % 8 * (even / 8) + id / 8;
  const int groups = (a.KV + a.heads - 1) / a.heads;
  const long long at = a.first + id, all = a.slots * groups;
  w.split = (int)(at / all);
  const long long r = at - w.split * all;
  if (a.head_major) w.kv = (int)(r / a.slots), w.slot = r - w.kv * a.slots;   // (one head a block)
  else w.slot = r / groups, w.kv = (int)(r - w.slot * groups) * a.heads;
  return w;
}

// the part of `tiles` that a piece of the streamed side takes
__device__ __forceinline__ void piece_of(int tiles, int split, int splits, int &from, int &to) {
  const int per = (tiles + splits - 1) / splits;
  from = min(tiles, split * per), to = min(tiles, from + per);
}

// Distance of an own row from one point of the streamed side, and what its gradients take of it.
template <int BIAS>
struct Distance {
  float far, inv, d[3];
  __device__ __forceinline__ void form(const float *x, const f32x4 *p, int i) {
    if constexpr (BIAS != kBiasNone) {
#pragma unroll
      for (int k = 0; k < 3; k++) d[k] = x[k] - p[k][i];
      // (a square beyond float32 counts as its largest: infinity would meet slopes, shares and inverses of zero.  NaN stays NaN)
      const float sq = __builtin_elementwise_minimum(d[0] * d[0] + d[1] * d[1] + d[2] * d[2], 0x1.fffffep127f);
      if constexpr (BIAS == kBiasGradients) inv = __builtin_amdgcn_rsqf(fmaxf(sq, 1e-37f)), far = sq * inv;   // (in one place: d and far are zero)
      else far = __builtin_amdgcn_sqrtf(sq);
    }
  }
  // sums of g d / |d|
  __device__ __forceinline__ void add(float *sums, float g) const {
    const float w = g * inv;
#pragma unroll
    for (int k = 0; k < 3; k++) sums[k] = __builtin_fmaf(w, d[k], sums[k]);
  }
};

// What own rows of queries are in the first two passes
template <typename T, int DP, int QS, int BIAS>
struct QueryRows {
  typedef AttnTile<T, DP> Tile;
  typename Tile::Frag q[QS][Tile::KS];
  float x[QS][3], slope[QS];   // slope: of log2 units, negative
  bool there[QS], mine[QS];    // it exists; it is this document's to write
  // row of the results: position * heads + head (formed where it is wanted: registers)
  static __device__ __forceinline__ long long out(const AttnArgs &a, const AttnDoc &doc, int kv, int row0, int s) {
    const RowAt r = row_at(a, row0 + 16 * s + threadIdx.x % 16);
    return (doc.out_q + r.pos) * a.H + kv * a.G + r.head;
  }
  __device__ __forceinline__ void negate() {
    typedef unsigned u32x4 __attribute__((ext_vector_type(4)));
    const unsigned sign = sizeof(T) == 2 ? 0x80008000u : 0x80000000u;
#pragma unroll
    for (int s = 0; s < QS; s++)
#pragma unroll
      for (int k = 0; k < Tile::KS; k++) q[s][k] = __builtin_bit_cast(typename Tile::Frag, __builtin_bit_cast(u32x4, q[s][k]) ^ sign);
  }
  __device__ __forceinline__ void load(const AttnArgs &a, const AttnDoc &doc, int kv, int row0, int live) {
#pragma unroll
    for (int s = 0; s < QS; s++) {
      const RowAt r = row_at(a, row0 + 16 * s + threadIdx.x % 16);
      const int h = kv * a.G + r.head;
      mine[s] = r.pos < doc.own_all, there[s] = r.pos < live;
      const T *row = (const T *)a.q + doc.sample * a.qs + (doc.q0 + r.pos) * a.qp + (long long)h * a.qh;
#pragma unroll
      for (int k = 0; k < Tile::KS; k++) q[s][k] = Tile::frag_of(row, k, a.dim, there[s]);
      if (BIAS) {
#pragma unroll
        for (int e = 0; e < 3; e++) x[s][e] = there[s] ? a.x[(doc.out_q + r.pos) * 3 + e] : 0.f;
        slope[s] = there[s] ? a.slopes[h] * -1.44269504088896341f : 0.f;
      }
    }
  }
};

// Tiles of keys, values and points on their way through LDS
template <typename T, int DP, int WAVES, int BIAS>
struct KeyTiles {
  typedef AttnTile<T, DP> Tile;
  static constexpr int THREADS = 64 * WAVES, BUFS = WAVES > 1 ? 2 : 1, BN = kAttnBN<T, DP>;
  struct Buffer {
    __align__(16) char k[BN * Tile::W], v[BN * Tile::W];
    __align__(16) float x[BIAS ? 3 : 1][64];
  };
  const T *k, *v;
  const float *x;
  int kp, vp, dim, rows;
  __device__ __forceinline__ KeyTiles(const AttnArgs &a, const AttnDoc &doc, int kv)
      : k((const T *)a.k + doc.sample * a.ks + doc.k0 * a.kp + (long long)kv * a.kh), v((const T *)a.v + doc.sample * a.vs + doc.k0 * a.vp + (long long)kv * a.vh), x(BIAS ? a.xk + doc.out_k * 3 : nullptr),
        kp(a.kp), vp(a.vp), dim(a.dim), rows(doc.kn) {}
  __device__ __forceinline__ void copy(int t, Buffer &b) const {
    const int left = rows - t * BN;
    const T *kt = k + (long long)t * BN * kp, *vt = v + (long long)t * BN * vp;
    copy_tile<T, DP, BN, THREADS, kFrugal<T, DP, BIAS, WAVES>>(b.k, [&](int row) { return kt + (long long)row * kp; }, left, dim);
    copy_tile<T, DP, BN, THREADS, kFrugal<T, DP, BIAS, WAVES>>(b.v, [&](int row) { return vt + (long long)row * vp; }, left, dim);
    if (BIAS) {
      const float *xt = x + (long long)t * BN * 3;
#pragma unroll
      for (int e = 0; e < 3; e++)
        if (WAVES == 1 || (int)threadIdx.x / 64 == e) copy_numbers(b.x[BIAS ? e : 0], [&](int row) { return row < left ? xt + row * 3 + e : (const float *)attn_zeros; });
    }
  }
  // f(tile, buffer) for the tiles from t0 to t1, each copied while the one before it is at work
  template <typename F>
  __device__ __forceinline__ void each(Buffer *b, int t0, int t1, F f) const {
    each_tile<WAVES>(b, t0, t1, [&](int t, Buffer &to) __attribute__((always_inline)) { copy(t, to); }, f);
  }
};

template <typename T, int DP, int WAVES, int QS, int BIAS, bool SHARE>
__device__ __forceinline__ void attention_fwd_head(const AttnArgs &a, const AttnWork &w, const AttnDoc &doc, typename KeyTiles<T, DP, WAVES, BIAS>::Buffer *lds) {
  typedef AttnTile<T, DP> Tile;
  typedef KeyTiles<T, DP, WAVES, BIAS> Keys;
  constexpr int BN = Keys::BN, SUB = BN / 16, BM = 16 * QS * WAVES;
  const int q4 = threadIdx.x % 64 / 16 * 4, live = doc.kn > 0 ? doc.qn : 0;
  const int row0 = doc.tile * BM + threadIdx.x / 64 * (16 * QS);
  QueryRows<T, DP, QS, BIAS> own;
  own.load(a, doc, w.kv, row0, live);

  // Exponentials are formed less the maximum so far, m (log2), which is that of the first tile with a score above -infinity (begun: a row
  // has had one).  It moves only when a score is more than 8 above it: values are then at most 2^8 times what they would be, and
  // rescaling is rare.  Scores themselves are kept whole until then: less a maximum far below them they would lose digits.
  // Without distances what is kept are products that the scale, which is above zero then, has not met yet (q takes its sign): it and the
  // maximum are one instruction in front of the exponential.  8192 x 8192, 16 heads of 64, bfloat16: 411 us, with scores scaled at once 423, less the
  // maximum from the start 397; with points (8192, 16 heads on 4) an instruction more than that, 540 and 506.
  const float unit = BIAS ? 1.f : fmaxf(fabsf(a.scale2), 0x1p-149f);   // (not zero: times -infinity)
  if (!BIAS && a.scale2 < 0.f) own.negate();
  float m[QS], l[QS];
  bool begun[QS];
  f32x4 acc[QS][Tile::NF];
#pragma unroll
  for (int s = 0; s < QS; s++) {
    m[s] = 0.f, l[s] = 0.f, begun[s] = false;
#pragma unroll
    for (int f = 0; f < Tile::NF; f++) acc[s][f] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  int t0, t1;
  piece_of((long long)doc.tile * BM < rows_in(a, live) ? (doc.kn + BN - 1) / BN : 0, w.split, a.splits, t0, t1);
  const Keys keys(a, doc, w.kv);
  keys.each(lds, t0, t1, [&](int t, const typename Keys::Buffer &b) __attribute__((always_inline)) {
    const int left = doc.kn - t * BN, subs = min(SUB, (left + 15) / 16);
    f32x4 sc[QS][SUB];
#pragma unroll
    for (int j = 0; j < SUB; j++) {
      if (j >= subs) {
#pragma unroll
        for (int s = 0; s < QS; s++) sc[s][j] = f32x4{-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        continue;
      }
      f32x4 z[QS];
#pragma unroll
      for (int s = 0; s < QS; s++) z[s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < Tile::KS; k++) {
        const typename Tile::Frag fk = Tile::frag(b.k, j * 16, k);
#pragma unroll
        for (int s = 0; s < QS; s++) z[s] = Tile::product(fk, own.q[s][k], z[s]);
      }
      if constexpr (BIAS != kBiasNone) {
        f32x4 p[3];
#pragma unroll
        for (int e = 0; e < 3; e++) p[e] = *(const f32x4 *)&b.x[e][j * 16 + q4];
#pragma unroll
        for (int i = 0; i < 4; i++) {
          Distance<kBiasPoints> far;
#pragma unroll
          for (int s = 0; s < QS; s++) {
            if (!SHARE || s == 0) far.form(own.x[s], p, i);   // (the wave's tiles have the same positions)
            sc[s][j][i] = __builtin_fmaf(z[s][i], a.scale2, far.far * own.slope[s]);
          }
        }
      } else {
#pragma unroll
        for (int s = 0; s < QS; s++)
#pragma unroll
          for (int i = 0; i < 4; i++) sc[s][j][i] = z[s][i];
      }
      if (left < j * 16 + 16)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (j * 16 + q4 + i >= left)
#pragma unroll
            for (int s = 0; s < QS; s++) sc[s][j][i] = -INFINITY;
    }
    float top[QS];
    bool grown = false;
#pragma unroll
    for (int s = 0; s < QS; s++) {
      float v = kLowest;
#pragma unroll
      for (int j = 0; j < SUB; j++) v = fmaxf(v, fmaxf(fmaxf(sc[s][j][0], sc[s][j][1]), fmaxf(sc[s][j][2], sc[s][j][3])));
      top[s] = over_row_max(v);
      grown |= begun[s] ? top[s] * unit > m[s] + 8.f : top[s] > kLowest;
    }
    if (__any(grown)) {
#pragma unroll
      for (int s = 0; s < QS; s++) {
        const bool first = !begun[s] && top[s] > kLowest;
        const float to = first || (begun[s] && top[s] * unit > m[s]) ? top[s] * unit : m[s], by = first ? 0.f : __builtin_amdgcn_exp2f(m[s] - to);
        m[s] = to, l[s] *= by, begun[s] |= first;
#pragma unroll
        for (int f = 0; f < Tile::NF; f++) acc[s][f] *= by;
      }
    }
#pragma unroll
    for (int j = 0; j < SUB; j += 2) {
      if (j >= subs) break;
      f32x4 p0[QS], p1[QS];
#pragma unroll
      for (int s = 0; s < QS; s++) {
#pragma unroll
        for (int i = 0; i < 4; i++) p0[s][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s][j][i], unit, -m[s])), p1[s][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s][j + 1][i], unit, -m[s]));
        if constexpr (kIsHalf<T>) p0[s] *= kHalfTop, p1[s] *= kHalfTop;
        const f32x4 both = p0[s] + p1[s];
        l[s] += (both[0] + both[1]) + (both[2] + both[3]);
      }
      Tile::template transposed<QS>(acc, b.v, j * 16, p0, p1);
    }
  });

#pragma unroll
  for (int s = 0; s < QS; s++) {
    if constexpr (kIsHalf<T>)
#pragma unroll
      for (int f = 0; f < Tile::NF; f++) acc[s][f] *= 1.f / kHalfTop;
    const float all = over_row_sum(l[s]) * (kIsHalf<T> ? 1.f / kHalfTop : 1.f), sum = own.there[s] ? all : 0.f;
    if (!own.mine[s]) continue;
    const long long at = own.out(a, doc, w.kv, row0, s);
    if (a.part_q) {
      const long long in_part = w.split * a.rows_q * a.H + at;
      if (q4 == 0) a.part_ml[in_part] = make_float2(sum == 0.f ? kLowest : m[s], sum);
      float *to = a.part_q + in_part * a.dim;
      Tile::results(acc[s], [&](int d, f32x4 v) { store4<float>(to, d, a.dim, a.dim % 4 == 0, v); });
      continue;
    }
    const float by = sum == 0.f ? 0.f : 1.f / sum;
    if (a.lse && q4 == 0) a.lse[at] = sum == 0.f ? INFINITY : m[s] + __builtin_amdgcn_logf(sum);   // (log2; infinity: no key has a share)
    if (sum == 0.f) {   // (zero, whatever values there are)
#pragma unroll
      for (int f = 0; f < Tile::NF; f++) acc[s][f] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    T *to = (T *)a.y + at * a.dim;
    Tile::results(acc[s], [&](int d, f32x4 v) { store4<T>(to, d, a.dim, a.vec_y, v * by); });
  }
}

template <typename T, int DP, int WAVES, int QS, int BIAS, bool SHARE>
__global__ void __launch_bounds__(64 * WAVES, sizeof(T) == 2 && DP <= 64 ? 3 : 2) attention_fwd_kernel(const AttnArgs a) {
  constexpr int BM = 16 * QS * WAVES;
  __shared__ typename KeyTiles<T, DP, WAVES, BIAS>::Buffer lds[WAVES > 1 ? 2 : 1];
  AttnWork w = work_of(a);
  const AttnDoc doc = find_doc<true>(a, w.slot, BM);
  if ((long long)doc.tile * BM >= rows_in(a, doc.own_all)) return;
  if constexpr (WAVES > 1) {
    attention_fwd_head<T, DP, WAVES, QS, BIAS, SHARE>(a, w, doc, lds);
  } else {
    for (const int end = min(w.kv + a.heads, a.KV); w.kv < end; w.kv++) attention_fwd_head<T, DP, WAVES, QS, BIAS, SHARE>(a, w, doc, lds);
  }
}

// ---- gradients by query rows: gq, the points and slopes of queries, D ----
//
// D from a y that was rounded to 16 bits, and formed from p that were, is off by 2^-9 of itself, and so would be every ds and, worse, the
// float32 gradients of points and slopes.  But the p of a row sum to one, so what D0 = gy . y lacks is the sum of the row's p (gy . v - D0): the
// sums with p in the place of ds are formed beside the sums proper, and times that are what has to be taken away.  (cloud of 8192 points, 16
// heads of 64, bfloat16: errors of the gradients of points and slopes .004 without it.)  The pass by keys has the D that is right.

template <typename T, int DP, int WAVES, int QS, int BIAS, bool SHARE>
__device__ __forceinline__ void attention_rows_head(const AttnArgs &a, const AttnWork &w, const AttnDoc &doc, typename KeyTiles<T, DP, WAVES, BIAS>::Buffer *lds) {
  typedef AttnTile<T, DP> Tile;
  typedef KeyTiles<T, DP, WAVES, BIAS> Keys;
  constexpr int BN = Keys::BN, SUB = BN / 16, BM = 16 * QS * WAVES;
  constexpr bool MEND = sizeof(T) == 2;
  constexpr int SETS = MEND ? 2 * QS : QS;   // ds, p
  const int q4 = threadIdx.x % 64 / 16 * 4, live = doc.kn > 0 ? doc.qn : 0;
  const int row0 = doc.tile * BM + threadIdx.x / 64 * (16 * QS);
  QueryRows<T, DP, QS, BIAS> own;
  own.load(a, doc, w.kv, row0, live);

  typename Tile::Frag fg[QS][Tile::KS];
  float nlse[QS], delta[QS], rest[QS];   // -lse, D0, the sum of ds
#pragma unroll
  for (int s = 0; s < QS; s++) {
    delta[s] = 0.f, rest[s] = 0.f;
    const long long at = own.out(a, doc, w.kv, row0, s);
#pragma unroll
    for (int k = 0; k < Tile::KS; k++) {
      fg[s][k] = Tile::frag_of((const T *)a.gy + at * a.ldy, k, a.dim, own.there[s]);
      const typename Tile::Frag fy = Tile::frag_of((const T *)a.y + at * a.ldy, k, a.dim, own.there[s]);
      T gv[Tile::EP], yv[Tile::EP];
      __builtin_memcpy(gv, &fg[s][k], 16);
      __builtin_memcpy(yv, &fy, 16);
#pragma unroll
      for (int e = 0; e < Tile::EP; e++) delta[s] += to_f(gv[e]) * to_f(yv[e]);
    }
    delta[s] = over_row_sum(delta[s]);
    nlse[s] = own.there[s] ? -a.lse[at] : -INFINITY;
  }
  Lift<T, QS> lift;
  f32x4 acc[SETS][Tile::NF];
  float geo[SETS][4];
#pragma unroll
  for (int s = 0; s < SETS; s++) {
#pragma unroll
    for (int f = 0; f < Tile::NF; f++) acc[s][f] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < 4; e++) geo[s][e] = 0.f;
  }
  int t0, t1;
  piece_of((long long)doc.tile * BM < rows_in(a, live) ? (doc.kn + BN - 1) / BN : 0, w.split, a.splits, t0, t1);
  const Keys keys(a, doc, w.kv);
  keys.each(lds, t0, t1, [&](int t, const typename Keys::Buffer &b) __attribute__((always_inline)) {
    const int left = doc.kn - t * BN, subs = min(SUB, (left + 15) / 16);
#pragma unroll 1
    for (int j0 = 0; j0 < SUB; j0 += 2) {
      if (j0 >= subs) break;
      f32x4 ds[2][SETS];
      float part[QS][4] = {}, part_rest[QS] = {};   // (of 32 keys: sums over thousands of them one after the other would lose two digits)
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int j = j0 + u;
        f32x4 z[QS], dp[QS];
#pragma unroll
        for (int s = 0; s < QS; s++) z[s] = f32x4{0.f, 0.f, 0.f, 0.f}, dp[s] = f32x4{-delta[s], -delta[s], -delta[s], -delta[s]};
#pragma unroll
        for (int k = 0; k < Tile::KS; k++) {
          const typename Tile::Frag fk = Tile::frag(b.k, j * 16, k), fv = Tile::frag(b.v, j * 16, k);
#pragma unroll
          for (int s = 0; s < QS; s++) z[s] = Tile::product(fk, own.q[s][k], z[s]), dp[s] = Tile::product(fv, fg[s][k], dp[s]);
        }
        f32x4 point[3];
        if (BIAS)
#pragma unroll
          for (int e = 0; e < 3; e++) point[e] = *(const f32x4 *)&b.x[BIAS ? e : 0][j * 16 + q4];
        // (everything of one key before the next one's: registers)
        auto elements = [&](auto masked) __attribute__((always_inline)) {
#pragma unroll
          for (int i = 0; i < 4; i++) {
            const bool in = !masked.value || j * 16 + q4 + i < left;
            Distance<BIAS> far;
            float both = 0.f;
#pragma unroll
            for (int s = 0; s < QS; s++) {
              if (!SHARE || s == 0) far.form(own.x[s], point, i);
              float v = BIAS ? __builtin_fmaf(far.far, own.slope[s], nlse[s]) : nlse[s];
              v = __builtin_fmaf(z[s][i], a.scale2, v);
              if (masked.value) v = in ? v : -INFINITY;
              const float p = __builtin_amdgcn_exp2f(v), g = p * dp[s][i];
              ds[u][s][i] = g;
              if constexpr (MEND) ds[u][QS + s][i] = p, part_rest[s] += g;
              if constexpr (BIAS == kBiasGradients) {
                // (heads of one position: their gradients of the point are one sum, kept with the first)
                both = SHARE && s > 0 ? __builtin_fmaf(g, own.slope[s], both) : g * own.slope[s];
                if (!SHARE || s == QS - 1) far.add(part[SHARE ? 0 : s], both);
                part[s][3] = __builtin_fmaf(g, far.far, part[s][3]);
                if constexpr (MEND) far.add(geo[QS + s], p), geo[QS + s][3] = __builtin_fmaf(p, far.far, geo[QS + s][3]);
              }
            }
          }
        };
        if (left < j * 16 + 16) elements(std::true_type());
        else elements(std::false_type());
      }
      if constexpr (BIAS == kBiasGradients)
#pragma unroll
        for (int s = 0; s < QS; s++)
#pragma unroll
          for (int e = 0; e < 4; e++) geo[s][e] += part[s][e];
      if constexpr (MEND)
#pragma unroll
        for (int s = 0; s < QS; s++) rest[s] += part_rest[s];
      lift.apply(ds, acc);
      Tile::template transposed<SETS>(acc, b.k, j0 * 16, ds[0], ds[1]);
    }
  });

  lift.down(acc);
#pragma unroll
  for (int s = 0; s < QS; s++) {
    const bool pieces = MEND && a.part_d;   // (what is lacking is known when all pieces are there)
    const float lacks = MEND ? over_row_sum(rest[s]) : 0.f;
    const long long at = own.out(a, doc, w.kv, row0, s), in_part = w.split * a.rows_q * a.H + at;
    if (BIAS == kBiasGradients) {
#pragma unroll
      for (int e = 0; e < 4; e++) {
        geo[s][e] = over_row_sum(geo[s][e]) * (e < 3 ? 0.69314718055994531f : -1.f);
        if (MEND) geo[QS * MEND + s][e] = over_row_sum(geo[QS * MEND + s][e]) * (e < 3 ? own.slope[s] * 0.69314718055994531f : -1.f);
        if (MEND && !pieces) geo[s][e] -= lacks * geo[QS * MEND + s][e];
      }
      if (own.mine[s] && q4 == 0) {
        a.geo_q[in_part] = make_float4(geo[s][0], geo[s][1], geo[s][2], geo[s][3]);
        if (pieces) a.geo_p[in_part] = make_float4(geo[QS * MEND + s][0], geo[QS * MEND + s][1], geo[QS * MEND + s][2], geo[QS * MEND + s][3]);
      }
    }
    if (!own.mine[s]) continue;
    if (q4 == 0) {
      if (pieces) a.part_d[in_part] = lacks;
      if (w.split == 0) a.delta[at] = pieces ? delta[s] : delta[s] + lacks;
    }
    if (a.part_q) {
      float *to = a.part_q + in_part * a.dim;
      Tile::results(acc[s], [&](int d, f32x4 v) { store4<float>(to, d, a.dim, a.dim % 4 == 0, v * a.scale); });
      if constexpr (MEND) {
        float *too = a.part_p + in_part * a.dim;
        Tile::results(acc[QS + s], [&](int d, f32x4 v) { store4<float>(too, d, a.dim, a.dim % 4 == 0, v * a.scale); });
      }
    } else if (a.gq) {
      if constexpr (MEND)
#pragma unroll
        for (int f = 0; f < Tile::NF; f++) acc[s][f] -= acc[QS + s][f] * lacks;
      T *to = (T *)a.gq + at * a.dim;
      Tile::results(acc[s], [&](int d, f32x4 v) { store4<T>(to, d, a.dim, a.vec_y, v * a.scale); });
    }
  }
}

template <typename T, int DP, int WAVES, int QS, int BIAS, bool SHARE>
__global__ void __launch_bounds__(64 * WAVES, 2) attention_rows_kernel(const AttnArgs a) {
  constexpr int BM = 16 * QS * WAVES;
  __shared__ typename KeyTiles<T, DP, WAVES, BIAS>::Buffer lds[WAVES > 1 ? 2 : 1];
  AttnWork w = work_of(a);
  const AttnDoc doc = find_doc<true>(a, w.slot, BM);
  if ((long long)doc.tile * BM >= rows_in(a, doc.own_all)) return;
  if constexpr (WAVES > 1) {
    attention_rows_head<T, DP, WAVES, QS, BIAS, SHARE>(a, w, doc, lds);
  } else {
    for (const int end = min(w.kv + a.heads, a.KV); w.kv < end; w.kv++) attention_rows_head<T, DP, WAVES, QS, BIAS, SHARE>(a, w, doc, lds);
  }
}

// ---- gradients by keys: gk, gv, the points of keys ----

// Tiles of query rows, gradients and what belongs to the rows on their way through LDS
template <typename T, int DP, int BIAS>
struct RowBuffer {
  static constexpr int BN = kAttnBN<T, DP>;
  __align__(16) char q[BN * AttnTile<T, DP>::W], g[BN * AttnTile<T, DP>::W];
  __align__(16) float r[BIAS ? 6 : 2][64];   // lse, D, slope, points of the rows
};

template <typename T, int DP, int WAVES, int QS, int BIAS, bool SHARE>
__device__ __forceinline__ void attention_keys_head(const AttnArgs &a, const AttnWork &w, const AttnDoc &doc, RowBuffer<T, DP, BIAS> *lds) {
  typedef AttnTile<T, DP> Tile;
  constexpr int THREADS = 64 * WAVES, BN = kAttnBN<T, DP>, SUB = BN / 16, BM = 16 * QS * WAVES, ROW = BIAS ? 6 : 2;
  typedef RowBuffer<T, DP, BIAS> Buffer;
  const int lane = threadIdx.x % 64, c = lane % 16, q4 = lane / 16 * 4;
  const int key0 = doc.tile * BM + threadIdx.x / 64 * (16 * QS);

  typename Tile::Frag fk[QS][Tile::KS], fv[QS][Tile::KS];
  float x[QS][3];
  bool mine[QS], exists[QS];
#pragma unroll
  for (int s = 0; s < QS; s++) {
    const int key = key0 + 16 * s + c;
    exists[s] = key < doc.kn, mine[s] = key < doc.own_all;
    const T *rk = (const T *)a.k + doc.sample * a.ks + (doc.k0 + key) * a.kp + (long long)w.kv * a.kh;
    const T *rv = (const T *)a.v + doc.sample * a.vs + (doc.k0 + key) * a.vp + (long long)w.kv * a.vh;
#pragma unroll
    for (int k = 0; k < Tile::KS; k++) fk[s][k] = Tile::frag_of(rk, k, a.dim, exists[s]), fv[s][k] = Tile::frag_of(rv, k, a.dim, exists[s]);
    if (BIAS)
#pragma unroll
      for (int e = 0; e < 3; e++) x[s][e] = exists[s] ? a.xk[(doc.out_k + key) * 3 + e] : 0.f;
  }
  Lift<T, QS> lift;
  f32x4 ak[QS][Tile::NF], av[QS][Tile::NF];
  float geo[QS][3];
#pragma unroll
  for (int s = 0; s < QS; s++) {
#pragma unroll
    for (int f = 0; f < Tile::NF; f++) ak[s][f] = f32x4{0.f, 0.f, 0.f, 0.f}, av[s][f] = ak[s][f];
#pragma unroll
    for (int e = 0; e < 3; e++) geo[s][e] = 0.f;
  }

  const int rows = doc.tile * BM < doc.kn ? (int)rows_in(a, doc.qn) : 0;
  int t0, t1;
  piece_of((int)(((long long)rows + BN - 1) / BN), w.split, a.splits, t0, t1);
  const T *q0 = (const T *)a.q + doc.sample * a.qs + doc.q0 * a.qp + (long long)w.kv * a.G * a.qh;
  const long long o0 = doc.out_q * a.H + w.kv * a.G;
  auto copy = [&](int t, Buffer &b) __attribute__((always_inline)) {
    const int left = rows - t * BN, whole = (left + 31) & ~31;
    // (a row that does not exist is the last that does, whose lse, infinity, leaves it without a share: zeros times a key or value of infinity would be
    // no number.  Testing for that in the loop cost the kernel for 128 values without points 11 %.)
    auto row_of = [&](int row) __attribute__((always_inline)) { const RowAt r = row_at(a, t * BN + row); return RowAt{min(r.pos, doc.qn - 1), r.head}; };
    copy_tile<T, DP, BN, THREADS, kFrugal<T, DP, BIAS, WAVES>>(b.q, [&](int row) { const RowAt r = row_of(row); return q0 + (long long)r.pos * a.qp + (long long)r.head * a.qh; }, whole, a.dim);
    copy_tile<T, DP, BN, THREADS, kFrugal<T, DP, BIAS, WAVES>>(b.g, [&](int row) { const RowAt r = row_of(row); return (const T *)a.gy + (o0 + (long long)r.pos * a.H + r.head) * a.ldy; }, whole, a.dim);
#pragma unroll
    for (int e = 0; e < ROW; e++)
      if (WAVES == 1 || (int)threadIdx.x / 64 == e % 4)
        copy_numbers(b.r[e], [&](int row) {
          const RowAt r = row_at(a, t * BN + row);
          const long long o = o0 + (long long)r.pos * a.H + r.head;
          const float *at = e == 0 ? a.lse + o : e == 1 ? a.delta + o : e == 2 ? a.slopes + w.kv * a.G + r.head : a.x + (doc.out_q + r.pos) * 3 + (e - 3);
          return row < left && r.pos < doc.qn ? at : e == 0 ? attn_infinity : (const float *)attn_zeros;
        });
  };
  each_tile<WAVES>(lds, t0, t1, copy, [&](int t, const Buffer &b) __attribute__((always_inline)) {
    const int subs = min(SUB, (rows - t * BN + 15) / 16);
#pragma unroll 1
    for (int j0 = 0; j0 < SUB; j0 += 2) {
      if (j0 >= subs) break;
      f32x4 p[2][QS], ds[2][QS];   // scores and gy . v - D, then p and ds
#pragma unroll
      for (int u = 0; u < 2; u++) {
        const int j = j0 + u;
        const f32x4 delta = *(const f32x4 *)&b.r[1][j * 16 + q4];
#pragma unroll
        for (int s = 0; s < QS; s++) p[u][s] = f32x4{0.f, 0.f, 0.f, 0.f}, ds[u][s] = -delta;
#pragma unroll
        for (int k = 0; k < Tile::KS; k++) {
          const typename Tile::Frag fq = Tile::frag(b.q, j * 16, k), fg = Tile::frag(b.g, j * 16, k);
#pragma unroll
          for (int s = 0; s < QS; s++) p[u][s] = Tile::product(fq, fk[s][k], p[u][s]), ds[u][s] = Tile::product(fg, fv[s][k], ds[u][s]);
        }
      }
      float part[QS][3] = {};
      // 16 rows after the other, or, where SHARE, all: the second 16 have the positions of the first
#pragma unroll
      for (int u0 = 0; u0 < (SHARE ? 1 : 2); u0++) {
        in_turn<kFrugal<T, DP, BIAS, WAVES>>();
        constexpr int U = SHARE ? 2 : 1;
        f32x4 nlse[U], slope[U], point[3];   // what rows are
#pragma unroll
        for (int v = 0; v < U; v++) {
          nlse[v] = -*(const f32x4 *)&b.r[0][(j0 + u0 + v) * 16 + q4];
          if constexpr (BIAS != kBiasNone) slope[v] = *(const f32x4 *)&b.r[2][(j0 + u0 + v) * 16 + q4];
        }
        if constexpr (BIAS != kBiasNone)
#pragma unroll
          for (int e = 0; e < 3; e++) point[e] = *(const f32x4 *)&b.r[3 + e][(j0 + u0) * 16 + q4];
#pragma unroll
        for (int s = 0; s < QS; s++)
#pragma unroll
          for (int i = 0; i < 4; i++) {
            Distance<BIAS> far;
            far.form(x[s], point, i);   // (from the key: the sign that its gradient takes)
            float both = 0.f;           // gradients of rows of one position, times their slopes
#pragma unroll
            for (int v = 0; v < U; v++) {
              const int u = u0 + v;
              float less = nlse[v][i];
              if constexpr (BIAS != kBiasNone) less = __builtin_fmaf(far.far, slope[v][i] * -1.44269504088896341f, less);
              const float prob = __builtin_amdgcn_exp2f(__builtin_fmaf(p[u][s][i], a.scale2, less)), g = prob * ds[u][s][i];
              p[u][s][i] = kIsHalf<T> ? prob * kHalfUp : prob, ds[u][s][i] = g;
              if constexpr (BIAS == kBiasGradients) both = __builtin_fmaf(g, slope[v][i], both);
            }
            if constexpr (BIAS == kBiasGradients) far.add(part[s], both);
          }
      }
      if constexpr (BIAS == kBiasGradients)
#pragma unroll
        for (int s = 0; s < QS; s++)
#pragma unroll
          for (int e = 0; e < 3; e++) geo[s][e] -= part[s][e];
      in_turn<kFrugal<T, DP, BIAS, WAVES>>();
      Tile::template transposed<QS>(av, b.g, j0 * 16, p[0], p[1]);
      in_turn<kFrugal<T, DP, BIAS, WAVES>>();
      lift.apply(ds, ak);
      in_turn<kFrugal<T, DP, BIAS, WAVES>>();
      Tile::template transposed<QS>(ak, b.q, j0 * 16, ds[0], ds[1]);
    }
  });

  lift.down(ak);
#pragma unroll
  for (int s = 0; s < QS; s++) {
    const long long out = (doc.out_k + key0 + 16 * s + c) * a.KV + w.kv, at = w.split * a.rows_k * a.KV + out;
    if constexpr (kIsHalf<T>)
#pragma unroll
      for (int f = 0; f < Tile::NF; f++) av[s][f] *= 1.f / kHalfUp;
    if (!exists[s]) {   // (its score is no -infinity above: its values and gradients are zeros here)
#pragma unroll
      for (int f = 0; f < Tile::NF; f++) ak[s][f] = f32x4{0.f, 0.f, 0.f, 0.f}, av[s][f] = ak[s][f];
    }
    if (BIAS == kBiasGradients) {
#pragma unroll
      for (int e = 0; e < 3; e++) {
        const float all = over_row_sum(geo[s][e]);
        geo[s][e] = exists[s] ? all : 0.f;
      }
      if (mine[s] && q4 == 0) a.geo_k[at] = make_float4(geo[s][0], geo[s][1], geo[s][2], 0.f);
    }
    if (!mine[s]) continue;
    if (a.part_k) {
      float *tk = a.part_k + at * a.dim, *tv = a.part_v + at * a.dim;
      Tile::results(ak[s], [&](int d, f32x4 v) { store4<float>(tk, d, a.dim, a.dim % 4 == 0, v * a.scale); });
      Tile::results(av[s], [&](int d, f32x4 v) { store4<float>(tv, d, a.dim, a.dim % 4 == 0, v); });
    } else {
      if (a.gk) {
        T *to = (T *)a.gk + out * a.dim;
        Tile::results(ak[s], [&](int d, f32x4 v) { store4<T>(to, d, a.dim, a.vec_y, v * a.scale); });
      }
      if (a.gv) {
        T *to = (T *)a.gv + out * a.dim;
        Tile::results(av[s], [&](int d, f32x4 v) { store4<T>(to, d, a.dim, a.vec_y, v); });
      }
    }
  }
}

template <typename T, int DP, int WAVES, int QS, int BIAS, bool SHARE>
__global__ void __launch_bounds__(64 * WAVES, sizeof(T) == 4 && DP >= 64 ? 1 : 2) attention_keys_kernel(const AttnArgs a) {
  constexpr int BM = 16 * QS * WAVES;
  __shared__ RowBuffer<T, DP, BIAS> lds[WAVES > 1 ? 2 : 1];
  AttnWork w = work_of(a);
  const AttnDoc doc = find_doc<false>(a, w.slot, BM);
  if ((long long)doc.tile * BM >= doc.own_all) return;
  if constexpr (WAVES > 1) {
    attention_keys_head<T, DP, WAVES, QS, BIAS, SHARE>(a, w, doc, lds);
  } else {
    for (const int end = min(w.kv + a.heads, a.KV); w.kv < end; w.kv++) attention_keys_head<T, DP, WAVES, QS, BIAS, SHARE>(a, w, doc, lds);
  }
}

// Launches of at most 2^22 blocks (2^30 threads) each.
constexpr long long kAttnMostBlocks = 1 << 22;

template <AttnPass PASS, typename T, int DP, int WAVES, int BIAS, bool SHARE>
void launch_attention_pass(AttnArgs a, hipStream_t s) {
  constexpr int QS = attention_qs(PASS, sizeof(T), DP, WAVES > 1, SHARE);
  const long long blocks = a.slots * ((a.KV + a.heads - 1) / a.heads) * a.splits;
  for (a.first = 0; a.first < blocks; a.first += kAttnMostBlocks) {
    const dim3 grid((unsigned)std::min(kAttnMostBlocks, blocks - a.first)), block(64 * WAVES);
    if constexpr (PASS == kAttnForward) hipLaunchKernelGGL((attention_fwd_kernel<T, DP, WAVES, QS, BIAS, SHARE>), grid, block, 0, s, a);
    else if constexpr (PASS == kAttnRows) hipLaunchKernelGGL((attention_rows_kernel<T, DP, WAVES, QS, BIAS, SHARE>), grid, block, 0, s, a);
    else hipLaunchKernelGGL((attention_keys_kernel<T, DP, WAVES, QS, BIAS, SHARE>), grid, block, 0, s, a);
  }
}

template <AttnPass PASS, typename T, int DP, int BIAS>
void launch_attention_bias(const AttnPlan &p, const AttnArgs &a, hipStream_t s) {
  // (own rows share where a wave has two tiles of them, streamed ones always)
  constexpr bool SHARES = BIAS != kBiasNone && (PASS == kAttnKeys || attention_qs(PASS, sizeof(T), DP, true, true) == 2);
  if (!p.wide) launch_attention_pass<PASS, T, DP, 1, BIAS, false>(a, s);
  else if (!SHARES || !a.blocked) launch_attention_pass<PASS, T, DP, 4, BIAS, false>(a, s);
  else if constexpr (SHARES) launch_attention_pass<PASS, T, DP, 4, BIAS, true>(a, s);
}

template <AttnPass PASS, typename T, int DP>
void launch_attention_dims(const AttnPlan &p, const AttnArgs &a, hipStream_t s) {
  if (p.bias == kBiasNone) launch_attention_bias<PASS, T, DP, kBiasNone>(p, a, s);
  else if (PASS == kAttnForward || p.bias == kBiasPoints) launch_attention_bias<PASS, T, DP, kBiasPoints>(p, a, s);
  else if constexpr (PASS != kAttnForward) launch_attention_bias<PASS, T, DP, kBiasGradients>(p, a, s);
}

template <AttnPass PASS, typename T>
int launch_attention_kernels(const AttnPlan &p, const AttnArgs &a, hipStream_t s) {
  if constexpr (sizeof(T) == 4)
    if (p.dims == 16) launch_attention_dims<PASS, T, 16>(p, a, s);
  if (p.dims == 32) launch_attention_dims<PASS, T, 32>(p, a, s);
  else if (p.dims == 64) launch_attention_dims<PASS, T, 64>(p, a, s);
  else if (p.dims == 128) launch_attention_dims<PASS, T, 128>(p, a, s);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "attention launch");
}
#endif

}  // namespace gelib_hip
