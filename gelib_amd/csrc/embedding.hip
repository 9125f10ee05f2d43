// Rows of a table by tokens, y[i] = scale table[t_i], and the gradient of the table, gtable[r] = scale sum over t_i = r of gy[i], in an
// order that does not depend on timing: the tokens are sorted (stably, so that a row's gradients are added in the order of the tokens)
// and sums are formed over pieces of the sorted list.
//
// Sort: least significant digits of 8 bits first, three launches a digit: how often each digit stands in a block's 2048 tokens, the sums
// over the blocks before, the places.  A token below zero or behind the table is left out by the first digit.
// Sums: a wave takes a piece of the sorted list and some channels; a run of equal tokens that lies inside its piece is a finished row.  What
// the ends of a piece share with their neighbours goes to a list of two entries a piece, whose entries are in order again: the same kernel
// sums that list, and so on until one piece is left.  Adding to rows in memory as they come would be one launch, but atomic additions are
// in no order, and take turns where tokens are few (a million atoms of a dozen elements).
// (A table of sums in the LDS of every block instead of the sort, for 118 rows: 285 us with read, add and write, 670 with LDS's own additions.)
// What bounds it: memory.  1048576 x 128 float32 of 118 rows: forward 132 us (4.1 TB/s), sort 24, sums 152 (rows of 512 bytes in sorted order, 3.5 TB/s) + 3
// joins of 8; 65536 x 2048 bfloat16 of 65536 rows: forward 84, zeros 34, sort 36, sums 110 (4.9 TB/s) + 20.
#include "real_ops.h"

namespace gelib_hip {

namespace {

typedef unsigned int u32;

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "embedding launch");
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

constexpr long long kMostThreads = 1LL << 30;   // of a launch

template <typename T, int V>
struct alignas(sizeof(T) * V) Some {
  T v[V];
};

__device__ __forceinline__ long long token_at(const void *tokens, int wide, long long i) { return wide ? ((const long long *)tokens)[i] : ((const int *)tokens)[i]; }

// ---- forward: a thread writes V neighbouring values ----
template <typename T, int V>
__global__ void __launch_bounds__(256) embedding_kernel(T *y, const T *table, const void *tokens, int wide, long long rows, int per_row, float scale, long long first, long long all) {
  const long long at = first + (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= all) return;
  const long long i = at / per_row;
  const long long c = at - i * per_row, t = token_at(tokens, wide, i);
  Some<T, V> r;
  if (t >= 0 && t < rows) {
    r = ((const Some<T, V> *)table)[t * per_row + c];
#pragma unroll
    for (int k = 0; k < V; k++) r.v[k] = from_f<T>(to_f(r.v[k]) * scale);
  } else {
#pragma unroll
    for (int k = 0; k < V; k++) r.v[k] = from_f<T>(t < 0 ? 0.f : __builtin_nanf(""));
  }
  ((Some<T, V> *)y)[at] = r;
}

// ---- sort ----

constexpr int kSortTokens = 2048;   // a block's

struct Sorted {   // tokens and where they stood
  u32 *key, *at;
};

// Token i of the list that is sorted by a digit: the caller's in the first pass, else those sorted by the digits before.  -1: not in the table.
struct Source {
  const void *tokens;
  int wide;
  long long n, rows;
  Sorted from;         // key null: the first pass
  const u32 *count;    // of tokens in the table, from the second pass on
  __device__ __forceinline__ long long size() const { return from.key ? (long long)*count : n; }
  __device__ __forceinline__ int key(long long i) const {
    if (from.key) return (int)from.key[i];
    const long long t = token_at(tokens, wide, i);
    return t >= 0 && t < rows ? (int)t : -1;
  }
  __device__ __forceinline__ u32 place(long long i) const { return from.key ? from.at[i] : (u32)i; }
};

// counts[digit][block]
__global__ void __launch_bounds__(256) sort_count_kernel(const Source s, int shift, u32 *counts, u32 blocks) {
  __shared__ u32 lds[256];
  lds[threadIdx.x] = 0;
  __syncthreads();
  const long long b = (long long)blockIdx.x * kSortTokens, n = s.size();
#pragma unroll
  for (int u = 0; u < kSortTokens / 256; u++) {
    const long long i = b + u * 256 + threadIdx.x;
    const int k = i < n ? s.key(i) : -1;
    if (k >= 0) atomicAdd(&lds[(u32)k >> shift & 255], 1u);   // (a count: the order does not show)
  }
  __syncthreads();
  counts[(size_t)threadIdx.x * blocks + blockIdx.x] = lds[threadIdx.x];
}

// exclusive sums over 256 threads
__device__ __forceinline__ u32 sum_before(u32 v, u32 *lds, u32 &all) {
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  u32 s = v;
#pragma unroll
  for (int d = 1; d < 64; d *= 2) {
    const u32 o = __shfl_up(s, d);
    if (lane >= d) s += o;
  }
  __syncthreads();
  if (lane == 63) lds[wave] = s;
  __syncthreads();
  u32 before = 0;
  all = 0;
#pragma unroll
  for (int w = 0; w < 4; w++) {
    before += w < wave ? lds[w] : 0;
    all += lds[w];
  }
  return before + s - v;
}

// counts of one digit -> sums over the blocks before, totals[digit]
__global__ void __launch_bounds__(256) sort_scan_kernel(u32 *counts, u32 *totals, u32 blocks) {
  __shared__ u32 lds[4];
  u32 *row = counts + (size_t)blockIdx.x * blocks, carry = 0;
  for (u32 b = 0; b < blocks; b += 256) {
    const u32 i = b + threadIdx.x, v = i < blocks ? row[i] : 0;
    u32 all;
    const u32 before = sum_before(v, lds, all);
    if (i < blocks) row[i] = carry + before;
    carry += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = carry;
}

// Every wave takes its share of the block's tokens in rounds of 64: a lane's place is that of its digit so far, plus the lanes of
// the same digit before it.
__global__ void __launch_bounds__(256) sort_place_kernel(const Source s, int shift, const u32 *counts, const u32 *totals, u32 *count, Sorted to, u32 blocks) {
  __shared__ u32 base[4][256], lds[4];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const long long n = s.size(), b = (long long)blockIdx.x * kSortTokens + wave * (kSortTokens / 4);
  for (int w = 0; w < 4; w++) base[w][threadIdx.x] = 0;
  u32 all;
  const u32 first = sum_before(totals[threadIdx.x], lds, all) + counts[(size_t)threadIdx.x * blocks + blockIdx.x];
  if (blockIdx.x == 0 && threadIdx.x == 0) *count = all;
  __syncthreads();
  int key[kSortTokens / 256];
#pragma unroll
  for (int u = 0; u < kSortTokens / 256; u++) {
    const long long i = b + u * 64 + lane;
    key[u] = i < n ? s.key(i) : -1;
    if (key[u] >= 0) atomicAdd(&base[wave][(u32)key[u] >> shift & 255], 1u);
  }
  __syncthreads();
  u32 at = first;
  for (int w = 0; w < 4; w++) {   // (a thread a digit)
    const u32 c = base[w][threadIdx.x];
    base[w][threadIdx.x] = at;
    at += c;
  }
  __syncthreads();
#pragma unroll
  for (int u = 0; u < kSortTokens / 256; u++) {
    const bool there = key[u] >= 0;
    const u32 digit = (u32)key[u] >> shift & 255;
    unsigned long long same = __ballot(there);
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const unsigned long long ones = __ballot(digit >> k & 1);
      same &= digit >> k & 1 ? ones : ~ones;
    }
    const u32 before = __popcll(same & ((1ull << lane) - 1));
    u32 place = 0;
    if (there) place = base[wave][digit] + before;
    __builtin_amdgcn_wave_barrier();
    if (there && before == 0) base[wave][digit] += __popcll(same);
    __builtin_amdgcn_wave_barrier();
    if (there) to.key[place] = (u32)key[u], to.at[place] = s.place(b + u * 64 + lane);
  }
}

// ---- sums over pieces ----

// A list in order of its tokens: rows of gy (the first list) or float32 sums (the others); entries with no token are passed over.
template <typename T>
struct List {
  const u32 *key, *at;   // at null: entry i is row i
  const T *rows;
  const u32 *count;      // null: `most` of them
  long long most;
};
constexpr u32 kNoToken = 0xffffffffu;

// What the entry of an unfinished run left of a piece's border (either of the two before it) names
template <typename T>
__device__ __forceinline__ u32 token_before(const List<T> &l, long long i) {
  if (i == 0) return kNoToken;
  const u32 k = l.key[i - 1];
  return k == kNoToken && i > 1 ? l.key[i - 2] : k;
}

// A wave: `piece` entries, 64 V channels.  Two entries of the next list a piece: what of its first run continues to the left (or is the
// whole piece and continues to either side), what of its last continues to the right.
template <typename T, typename O, int V>
__global__ void __launch_bounds__(256) embedding_sum_kernel(const List<T> l, O *out, float scale, int C, int chunks, int piece, u32 *next_key, float *next_rows, long long first, long long waves) {
  const long long w = first + ((long long)blockIdx.x * 256 + threadIdx.x) / 64;
  if (w >= waves) return;
  const long long p = w / chunks, n = l.count ? (long long)*l.count : l.most;
  const int c = ((int)(w - p * chunks) * 64 + threadIdx.x % 64) * V;
  const bool names = w - p * chunks == 0 && threadIdx.x % 64 == 0;
  const long long b = p * piece, e = min(n, b + piece);
  const bool here = c < C;
  const int cc = here ? c : 0;
  float acc[V] = {};
  u32 run = kNoToken, head = kNoToken, tail = kNoToken;
  bool from_left = false;
  auto finish = [&](bool to_right) __attribute__((always_inline)) {
    if (run == kNoToken) return;
    if (from_left || to_right) {
      const int which = from_left ? 0 : 1;
      (which ? tail : head) = run;
      if (here) {
        Some<float, V> r;
#pragma unroll
        for (int k = 0; k < V; k++) r.v[k] = acc[k];
        *(Some<float, V> *)(next_rows + (p * 2 + which) * C + c) = r;
      }
    } else if (here) {
      Some<O, V> r;
#pragma unroll
      for (int k = 0; k < V; k++) r.v[k] = from_f<O>(acc[k] * scale);
      *(Some<O, V> *)(out + (long long)run * C + c) = r;
    }
  };
  if (b < e) {
    const u32 left = token_before(l, b);
    constexpr int U = 16;   // rows under way
    const int lane = threadIdx.x % 64;
    bool any = false;
    for (long long i0 = b; i0 < e; i0 += 64) {
      // 64 entries at a time, one a lane: what there is, and where its row lies
      const bool in = i0 + lane < e;
      const u32 keys = in ? l.key[i0 + lane] : kNoToken;
      const u32 rows = in && l.at ? l.at[i0 + lane] : (u32)(i0 + lane);
      unsigned long long there = __ballot(keys != kNoToken);
      while (there) {
        // (loads without a branch between them: behind the last entry it is read again)
        u32 key[U];
        Some<T, V> v[U];
        int k = 0;
#pragma unroll
        for (int u = 0; u < U; u++) {
          k = there ? __ffsll(there) - 1 : k;
          key[u] = there ? __builtin_amdgcn_readlane(keys, k) : kNoToken;
          there &= there - 1;
          v[u] = *(const Some<T, V> *)(l.rows + (long long)(u32)__builtin_amdgcn_readlane(rows, k) * C + cc);
        }
        if (key[0] == run && key[U - 1] == run) {   // (keys ascend: all of one row, summed in pairs first: smaller errors)
#pragma unroll
          for (int i = 0; i < V; i++) {
            float t[U];
#pragma unroll
            for (int u = 0; u < U; u++) t[u] = to_f(v[u].v[i]);
#pragma unroll
            for (int m = U / 2; m; m /= 2)
#pragma unroll
              for (int u = 0; u < m; u++) t[u] += t[u + m];
            acc[i] += t[0];
          }
          continue;
        }
#pragma unroll
        for (int u = 0; u < U; u++) {
          if (key[u] == kNoToken) continue;
          if (key[u] != run) {
            finish(false);
            from_left = !any && key[u] == left;
            any = true;
            run = key[u];
#pragma unroll
            for (int i = 0; i < V; i++) acc[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < V; i++) acc[i] += to_f(v[u].v[i]);
        }
      }
    }
    // the first entry of the next piece, or the one behind it, would continue the last run
    bool to_right = false;
    if (e < n) {
      const u32 k = l.key[e];
      to_right = (k == kNoToken && e + 1 < n ? l.key[e + 1] : k) == run && run != kNoToken;
    }
    finish(to_right);
  }
  if (names && next_key) next_key[p * 2] = head, next_key[p * 2 + 1] = tail;
}

template <typename T>
__global__ void __launch_bounds__(256) embedding_zero_kernel(T *out, long long first, long long all) {
  const long long at = (first + (long long)blockIdx.x * 256 + threadIdx.x) * 8;
  if (at + 8 <= all && (uintptr_t)out % 16 == 0) {
    const uint4 z = {0, 0, 0, 0};
#pragma unroll
    for (int k = 0; k < (int)sizeof(T) * 8 / 16; k++) ((uint4 *)(out + at))[k] = z;
  } else {
    for (long long i = at; i < min(all, at + 8); i++) out[i] = (T)0.f;
  }
}

template <typename F>
int in_launches(long long threads, F f) {
  for (long long first = 0; first < threads; first += kMostThreads) {
    f(first, dim3((unsigned)((std::min(kMostThreads, threads - first) + 255) / 256)));
    if (int rc = launched()) return rc;
  }
  return 0;
}

// neighbouring values that rows and their addresses allow in one load of at most 16 bytes
int width_of(int e, int C, uintptr_t address) {
  int v = 16 / e;
  while (v > 1 && (C % v || address % (v * e))) v /= 2;
  return v;
}

#define GELIB_BY_WIDTH(V, CALL)             \
  switch (V) {                              \
    case 8: CALL(8); break;                 \
    case 4: CALL(4); break;                 \
    case 2: CALL(2); break;                 \
    default: CALL(1);                       \
  }

template <typename T>
int forward(const EmbeddingArgs &a, hipStream_t s) {
  const int v = width_of(sizeof(T), a.channels, (uintptr_t)a.y | (uintptr_t)a.table), per_row = a.channels / v;
  const long long all = a.n * per_row;
  return in_launches(all, [&](long long first, dim3 grid) {
#define GELIB_CALL(V) hipLaunchKernelGGL((embedding_kernel<T, (V) * sizeof(T) <= 16 ? (V) : 1>), grid, dim3(256), 0, s, (T *)a.y, (const T *)a.table, a.tokens, a.wide, a.rows, per_row, a.scale, first, all)
    GELIB_BY_WIDTH(v, GELIB_CALL)
#undef GELIB_CALL
  });
}

// entries of a piece
int piece_of(long long n) { return n >= 1 << 18 ? 256 : 64; }

struct Space {
  size_t key[2], at[2], counts, totals, count, keys[2], rows[2], bytes = 0;
};
Space space_of(long long n, int C) {
  Space s = {};
  auto take = [&](size_t &at, size_t bytes) { at = s.bytes, s.bytes += up(bytes); };
  const long long blocks = (n + kSortTokens - 1) / kSortTokens;
  for (int k = 0; k < 2; k++) take(s.key[k], (size_t)n * 4), take(s.at[k], (size_t)n * 4);
  take(s.counts, (size_t)blocks * 256 * 4), take(s.totals, 256 * 4), take(s.count, 4);
  long long left = n;
  for (int k = 0; k < 2; k++) {   // (the lists after these two are shorter, and take their places in turn)
    left = (left + piece_of(left) - 1) / piece_of(left) * 2;
    take(s.keys[k], (size_t)left * 4), take(s.rows[k], (size_t)left * C * 4);
  }
  return s;
}

template <typename T, typename O, int V>
int sum_list(const List<T> &l, O *out, float scale, int C, int piece, u32 *next_key, float *next_rows, hipStream_t s) {
  const int chunks = (C + 64 * V - 1) / (64 * V);
  const long long waves = (l.most + piece - 1) / piece * chunks;
  return in_launches(waves * 64, [&](long long first, dim3 grid) {
    hipLaunchKernelGGL((embedding_sum_kernel<T, O, V>), grid, dim3(256), 0, s, l, out, scale, C, chunks, piece, next_key, next_rows, first / 64, waves);
  });
}

template <typename T, int V>
int sums(const EmbeddingArgs &a, const Sorted &in, const u32 *count, const Space &at, char *ws, hipStream_t s) {
  List<T> l = {in.key, in.at, (const T *)a.gy, count, a.n};
  auto next = [&](int k, long long most) { return List<float>{(const u32 *)(ws + at.keys[k]), nullptr, (const float *)(ws + at.rows[k]), nullptr, most}; };
  // (a list of one piece has no unfinished runs and no list behind it)
  int piece = piece_of(l.most), k = 0;
  long long pieces = (l.most + piece - 1) / piece;
  if (int rc = sum_list<T, T, V>(l, (T *)a.gtable, a.scale, a.channels, piece, (u32 *)(ws + at.keys[0]), (float *)(ws + at.rows[0]), s)) return rc;
  constexpr int VF = V < 4 ? V : 4;
  for (; pieces > 1; k ^= 1) {
    const List<float> f = next(k, pieces * 2);
    piece = piece_of(f.most), pieces = (f.most + piece - 1) / piece;
    if (int rc = sum_list<float, T, VF>(f, (T *)a.gtable, a.scale, a.channels, piece, (u32 *)(ws + at.keys[k ^ 1]), (float *)(ws + at.rows[k ^ 1]), s)) return rc;
  }
  return 0;
}

template <typename T>
int backward(const EmbeddingArgs &a, hipStream_t s) {
  const long long all = a.rows * a.channels;
  if (int rc = in_launches((all + 7) / 8, [&](long long first, dim3 grid) { hipLaunchKernelGGL(embedding_zero_kernel<T>, grid, dim3(256), 0, s, (T *)a.gtable, first, all); })) return rc;
  if (a.n == 0) return 0;
  const Space at = space_of(a.n, a.channels);
  char *ws = (char *)a.ws;
  Sorted list[2];
  for (int k = 0; k < 2; k++) list[k] = {(u32 *)(ws + at.key[k]), (u32 *)(ws + at.at[k])};
  u32 *counts = (u32 *)(ws + at.counts), *totals = (u32 *)(ws + at.totals), *count = (u32 *)(ws + at.count);
  const u32 blocks = (u32)((a.n + kSortTokens - 1) / kSortTokens);
  Source src = {a.tokens, a.wide, a.n, a.rows, {nullptr, nullptr}, count};
  int k = 0;
  for (int shift = 0; shift == 0 || (shift < 32 && (a.rows - 1) >> shift); shift += 8, k ^= 1) {
    hipLaunchKernelGGL(sort_count_kernel, dim3(blocks), dim3(256), 0, s, src, shift, counts, blocks);
    hipLaunchKernelGGL(sort_scan_kernel, dim3(256), dim3(256), 0, s, counts, totals, blocks);
    hipLaunchKernelGGL(sort_place_kernel, dim3(blocks), dim3(256), 0, s, src, shift, (const u32 *)counts, (const u32 *)totals, count, list[k], blocks);
    if (int rc = launched()) return rc;
    src.from = list[k];
  }
  const Sorted in = list[k ^ 1];
  const int v = width_of(sizeof(T), a.channels, (uintptr_t)a.gy | (uintptr_t)a.gtable);
#define GELIB_CALL(V) return sums<T, (V) * sizeof(T) <= 16 ? (V) : 1>(a, in, count, at, ws, s)
  GELIB_BY_WIDTH(v, GELIB_CALL)
#undef GELIB_CALL
}

}  // namespace

size_t embedding_workspace(long long n, int channels) { return n ? space_of(n, channels).bytes : 0; }

int launch_embedding(int dtype, const EmbeddingArgs &a, hipStream_t s) {
  return dtype == GELIB_HIP_F32 ? forward<float>(a, s) : dtype == GELIB_HIP_BF16 ? forward<bhalf_t>(a, s) : forward<half_t>(a, s);
}
int launch_embedding_bwd(int dtype, const EmbeddingArgs &a, hipStream_t s) {
  return dtype == GELIB_HIP_F32 ? backward<float>(a, s) : dtype == GELIB_HIP_BF16 ? backward<bhalf_t>(a, s) : backward<half_t>(a, s);
}

}  // namespace gelib_hip
