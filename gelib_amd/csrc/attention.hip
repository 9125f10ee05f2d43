// Attention over the points of documents: which kernels a call takes (attention_impl.h has them), the joins of pieces, the sums of the
// gradients of points over heads and of slopes over rows.
#include "attention_impl.h"

namespace gelib_hip {

namespace {

constexpr int kSlopeRows = 128;   // rows whose slopes' gradients one block sums

int bn_of(int dtype, int dims) { return dims * dtype_bytes(dtype) >= 512 ? 32 : 64; }

// What one pass over `own` rows of a document (on the average) with `streamed` rows of the other side takes.
struct Pass {
  bool wide, blocked;
  long long slots;
  int splits, heads;   // heads: of keys, one after the other in a block
};
Pass pass_of(const AttnCall &c, AttnPass pass) {
  const bool own_q = pass != kAttnKeys;
  const long long G = c.heads / c.kv_heads, per = own_q ? G : 1, other = own_q ? 1 : G;
  const long long all = own_q ? c.nq : c.nk, streamed_all = (own_q ? c.nk : c.nq) * other;
  const double docs = c.packed ? (double)std::max(1LL, c.docs) : 1.0;
  const double own = all * per / docs, streamed = streamed_all / docs;
  Pass p;
  p.wide = own > 64;
  // Heads of a group by tiles, where distances are formed: both sides of a tile pair share them.  Positions are filled up to 16, which costs
  // less than it gives from two such tiles on.
  const int e = (int)dtype_bytes(c.dtype), dims = attention_dims(c.dtype, c.dim);
  const bool shares = !own_q || attention_qs(pass, e, dims, true, true) == 2;
  p.blocked = shares && c.slopes && p.wide && (G == 2 || G == 4 || G == 8) && c.nq / docs >= 32 && (!own_q || attention_rows(pass, e, dims, true, true) % (16 * G) == 0);
  const int rows = attention_rows(pass, e, dims, p.wide, p.blocked);
  const long long in_doc = own_q && p.blocked ? (all + 15) / 16 * 16 * per : all * per;
  p.slots = c.packed ? all * per / rows + c.docs + 3 : c.docs * ((in_doc + rows - 1) / rows);
  // Short documents: a wave takes several heads, which finds its document once, while there are four waves to every SIMD.
  p.heads = 1;
  while (!p.wide && p.heads * 2 <= c.kv_heads && p.slots * ((c.kv_heads + p.heads * 2 - 1) / (p.heads * 2)) >= 4096) p.heads *= 2;
  // pieces of the streamed side where blocks do not fill the compute units, two tiles each at least (8 x 1 queries of 16 heads, 4099 keys of 4,
  // kernel and join: pieces of 4 tiles 15.5 + 5.2, 2 tiles 11.6 + 7.3, 1 tile 10.7 + 10.6 us)
  const double blocks = std::max(1.0, own / rows) * (c.packed ? docs : (double)c.docs) * c.kv_heads / p.heads, want = p.wide ? 512 : 2048;
  const double most = streamed / bn_of(c.dtype, attention_dims(c.dtype, c.dim)) / 2;
  p.splits = (int)std::max(1.0, std::min({want / blocks, most, 64.0}));
  return p;
}

size_t up(size_t n) { return (n + 255) & ~(size_t)255; }

// Operands whose heads do not lie at multiples of 16 bytes, copied to (row, head, values up to a multiple of 16 bytes): a thread 16
// bytes of the copy.
struct Operand {
  const void *from;
  long long s, p, h;   // strides of samples, positions, heads
  long long docs, n;
  int heads;
};
struct AttnCopies {
  struct {
    Operand o;
    void *to;
    long long first;   // thread
  } m[5];
  int count, dim, per;   // per: pieces of a head
  long long threads;
};
template <typename T>
__global__ void __launch_bounds__(256) attention_copy_kernel(const AttnCopies a) {
  constexpr int V = 16 / sizeof(T);
  for (long long t = (long long)blockIdx.x * 256 + threadIdx.x; t < a.threads; t += (long long)gridDim.x * 256) {
    int k = 0;
    while (k + 1 < a.count && t >= a.m[k + 1].first) k++;
    const Operand &o = a.m[k].o;
    const long long at = t - a.m[k].first, rh = at / a.per, row = rh / o.heads, doc = row / o.n;
    const int c = (int)(at - rh * a.per) * V;
    const T *p = (const T *)o.from + doc * o.s + (row - doc * o.n) * o.p + (rh - row * o.heads) * o.h + c;
    T v[V];
#pragma unroll
    for (int i = 0; i < V; i++) v[i] = c + i < a.dim ? p[i] : (T)0.f;
    __builtin_memcpy(__builtin_assume_aligned((T *)a.m[k].to + at * V, 16), v, 16);
  }
}

int padded_dim(const AttnCall &c) {
  const int v = 16 / (int)dtype_bytes(c.dtype);
  return (c.dim + v - 1) / v * v;
}
bool aligned(const AttnCall &c, const void *p, const long long *s) {
  const long long e = (long long)dtype_bytes(c.dtype);
  return s[1] <= 0x7fffffff && s[2] <= 0x7fffffff && c.dim * e % 16 == 0 && ((long long)(uintptr_t)p | (c.packed ? 0 : s[0] * e) | s[1] * e | s[2] * e) % 16 == 0;
}

// Where everything lies in the workspace
struct Space {
  size_t q = 0, k = 0, v = 0, y = 0, gy = 0, part_q = 0, part_p = 0, part_d = 0, part_k = 0, part_v = 0, ml = 0, delta = 0, geo_q = 0, geo_p = 0, geo_k = 0, slopes = 0, bytes = 0;
};
long long rows_of(const AttnCall &c, bool q) { return c.packed ? (q ? c.nq : c.nk) : c.docs * (q ? c.nq : c.nk); }
Space space_of(const AttnCall &c, bool backward, bool geometry) {
  Space s;
  const long long rq = rows_of(c, true) * c.heads, rk = rows_of(c, false) * c.kv_heads;
  auto take = [&](size_t &at, size_t bytes) { at = s.bytes, s.bytes += up(bytes); };
  const size_t head = (size_t)padded_dim(c) * dtype_bytes(c.dtype);
  if (!aligned(c, c.q, c.qs)) take(s.q, rq * head);
  if (!aligned(c, c.k, c.ks)) take(s.k, rk * head);
  if (!aligned(c, c.v, c.vs)) take(s.v, rk * head);
  if (backward && padded_dim(c) != c.dim) take(s.y, rq * head), take(s.gy, rq * head);
  const Pass r = pass_of(c, backward ? kAttnRows : kAttnForward);
  if (r.splits > 1) take(s.part_q, (size_t)r.splits * rq * c.dim * 4);
  if (!backward) {
    if (r.splits > 1) take(s.ml, (size_t)r.splits * rq * 8);
    return s;
  }
  if (r.splits > 1 && c.dtype != GELIB_HIP_F32) {
    take(s.part_p, (size_t)r.splits * rq * c.dim * 4), take(s.part_d, (size_t)r.splits * rq * 4);
    if (geometry) take(s.geo_p, (size_t)r.splits * rq * 16);
  }
  const Pass k = pass_of(c, kAttnKeys);
  if (k.splits > 1) take(s.part_k, (size_t)k.splits * rk * c.dim * 4), take(s.part_v, (size_t)k.splits * rk * c.dim * 4);
  take(s.delta, (size_t)rq * 4);
  if (geometry) {
    take(s.geo_q, (size_t)r.splits * rq * 16);
    take(s.geo_k, (size_t)k.splits * rk * 16);
    take(s.slopes, (size_t)((rows_of(c, true) + kSlopeRows - 1) / kSlopeRows) * c.heads * 4);
  }
  return s;
}

int launched() {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? 0 : record_hip_error(e, "attention launch");
}

constexpr long long kMostThreads = 1LL << 30;   // of a launch

// y of a (row, head), a wave each: pieces' results to their common maximum.  Lane k has piece k's share (there are at most 64), four
// groups of 16 lanes take every fourth piece, four values a lane.
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(const AttnArgs a, long long first, long long rows) {
  const long long row = first + ((long long)blockIdx.x * 256 + threadIdx.x) / 64;
  if (row >= rows) return;
  const int lane = threadIdx.x % 64, d0 = lane % 16 * 4;
  const float2 ml = lane < a.splits ? a.part_ml[lane * rows + row] : make_float2(kLowest, 0.f);
  float top = ml.x;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) top = fmaxf(top, __shfl_xor(top, k));
  const float share = ml.y == 0.f ? 0.f : __builtin_amdgcn_exp2f(ml.x - top);
  float sum = ml.y * share;
#pragma unroll
  for (int k = 1; k < 64; k *= 2) sum += __shfl_xor(sum, k);
  const float by = sum == 0.f ? 0.f : 1.f / sum;
  const bool whole = a.dim % 4 == 0;
  for (int d = d0; d < (a.dim + 63) / 64 * 64; d += 64) {
    float4 v = {0.f, 0.f, 0.f, 0.f};
    for (int s = lane / 16; s < (a.splits + 3) / 4 * 4; s += 4) {
      const float w = __shfl(share, s);   // (all lanes: the loop is one for the wave)
      if (w == 0.f || d >= a.dim) continue;   // (a piece without a share has written nothing to speak of)
      const float *p = a.part_q + (s * rows + row) * a.dim + d;
      float4 t = {0.f, 0.f, 0.f, 0.f};
      if (whole) t = *(const float4 *)__builtin_assume_aligned(p, 16);
      else t.x = p[0], t.y = d + 1 < a.dim ? p[1] : 0.f, t.z = d + 2 < a.dim ? p[2] : 0.f, t.w = d + 3 < a.dim ? p[3] : 0.f;
      v.x += t.x * w, v.y += t.y * w, v.z += t.z * w, v.w += t.w * w;
    }
#pragma unroll
    for (int i = 0; i < 4; i++) {
      float e = i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
      e += __shfl_xor(e, 16);
      e += __shfl_xor(e, 32);
      if (lane < 16 && d + i < a.dim) ((T *)a.y)[row * a.dim + d + i] = from_f<T>(e * by);
    }
  }
  if (lane == 0 && a.lse) a.lse[row] = sum == 0.f ? INFINITY : top + __builtin_amdgcn_logf(sum);
}

// 16-bit types: gq of one (row, head) from the sums of its pieces, less what D0 lacks times the sums with p (attention_impl.h), and the same
// for the gradients of points and slopes, which are left in the first piece's place; D
template <typename T>
__global__ void __launch_bounds__(256) attention_mend_kernel(const AttnArgs a, long long first, long long all, int per_row) {
  const long long at = first + (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= all) return;
  const long long row = at / per_row, rows = a.rows_q * a.H;
  const int d = (int)(at - row * per_row) * 4, n = min(4, a.dim - d);
  float lacks = 0.f;
  for (int s = 0; s < a.splits; s++) lacks += a.part_d[s * rows + row];
  float v[4] = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; s++) {
    const long long p = (s * rows + row) * a.dim + d;
    for (int i = 0; i < n; i++) v[i] += a.part_q[p + i] - lacks * a.part_p[p + i];
  }
  if (a.gq)
    for (int i = 0; i < n; i++) ((T *)a.gq)[row * a.dim + d + i] = from_f<T>(v[i]);
  if (d) return;
  a.delta[row] += lacks;
  if (!a.geo_q) return;
  float4 g = {0.f, 0.f, 0.f, 0.f};
  for (int s = 0; s < a.splits; s++) {
    const float4 q = a.geo_q[s * rows + row], p = a.geo_p[s * rows + row];
    g.x += q.x - lacks * p.x, g.y += q.y - lacks * p.y, g.z += q.z - lacks * p.z, g.w += q.w - lacks * p.w;
  }
  a.geo_q[row] = g;
}

// out[i] = sum of the pieces' values
template <typename T>
__global__ void __launch_bounds__(256) attention_sum_kernel(T *out, const float *part, long long first, long long n, int splits) {
  const long long at = first + (long long)blockIdx.x * 256 + threadIdx.x;
  if (at >= n) return;
  float v = 0.f;
  for (int s = 0; s < splits; s++) v += part[s * n + at];
  out[at] = from_f<T>(v);
}

// gradients of points: sums over heads and pieces, of queries (geo_q), keys (geo_k) or, where they are the same points, both.  2^SHIFT lanes a row
// (up to 16; known to the compiler, which has four loads under way then: with a number that it does not know 732 instead of 609 us), neighbouring heads side by side: one query of 128 heads on 65536 keys in 64 pieces, both directions of the call:
// 609 us, with a thread a row 1411; 16 heads on 4: 371 / 471.  No more lanes than terms (4 heads on 2, 65536 points: 16
// lanes 5.9 us, four 3.8; one head of 2048 points: 3.5 with one as with 16).
template <int SHIFT>
__global__ void __launch_bounds__(256) attention_points_kernel(float *out, const float4 *gq, int splits_q, int H, const float4 *gk, int splits_k, int KV,
                                                               long long first, long long rows) {
  const long long row = (first + (long long)blockIdx.x * 256 + threadIdx.x) >> SHIFT;
  constexpr int lanes = 1 << SHIFT;
  const int lane = threadIdx.x & (lanes - 1);
  float sum[3] = {0.f, 0.f, 0.f};
  auto add = [&](const float4 *g, int splits, int heads) {
#pragma unroll 4
    for (int i = lane; i < splits * heads; i += lanes) {
      const int s = splits == 1 ? 0 : i / heads;
      const float4 v = g[(s * rows + row) * heads + (i - s * heads)];
      sum[0] += v.x, sum[1] += v.y, sum[2] += v.z;
    }
  };
  if (row < rows) {
    if (gq) add(gq, splits_q, H);
    if (gk) add(gk, splits_k, KV);
  }
#pragma unroll
  for (int d = 1; d < lanes; d *= 2)
#pragma unroll
    for (int e = 0; e < 3; e++) sum[e] += __shfl_xor(sum[e], d);
  if (row < rows)
#pragma unroll
    for (int e = 0; e < 3; e++)
      if ((e & (lanes - 1)) == lane) out[row * 3 + e] = sum[e];
}

// gradients of slopes: of kSlopeRows rows and up to 64 heads, a block (side: threads side by side on heads, a power of two); then of all blocks
__global__ void __launch_bounds__(256) attention_slopes_kernel(float *part, const float4 *geo, int splits, long long rows, int H, int side, long long blocks) {
  __shared__ float lds[256];
  const int h = blockIdx.y * side + threadIdx.x % side, down = 256 / side;
  for (long long b = blockIdx.x; b < blocks; b += gridDim.x) {
    const long long r0 = b * kSlopeRows;
    const int n = (int)min((long long)kSlopeRows, rows - r0);
    float v = 0.f;
    if (h < H)
#pragma unroll 4
      for (int i = threadIdx.x / side; i < n * splits; i += down) {
        const int s = splits == 1 ? 0 : i / n;
        v += geo[(s * rows + r0 + (i - s * n)) * H + h].w;
      }
    lds[threadIdx.x] = v;
    __syncthreads();
    for (int k = 128; k >= side; k /= 2) {
      if ((int)threadIdx.x < k) lds[threadIdx.x] += lds[threadIdx.x + k];
      __syncthreads();
    }
    if ((int)threadIdx.x < side && h < H) part[b * H + h] = lds[threadIdx.x];
    __syncthreads();
  }
}
__global__ void __launch_bounds__(256) attention_slopes_join_kernel(float *out, const float *part, long long blocks, int H) {
  __shared__ float lds[256];
  float v = 0.f;
  for (long long b = threadIdx.x; b < blocks; b += 256) v += part[b * H + blockIdx.x];
  lds[threadIdx.x] = v;
  __syncthreads();
  for (int k = 128; k; k /= 2) {
    if ((int)threadIdx.x < k) lds[threadIdx.x] += lds[threadIdx.x + k];
    __syncthreads();
  }
  if (threadIdx.x == 0) out[blockIdx.x] = lds[0];
}

template <typename F>
int in_launches(long long threads, F f) {
  for (long long first = 0; first < threads; first += kMostThreads) {
    f(first, dim3((unsigned)((std::min(kMostThreads, threads - first) + 255) / 256)));
    if (int rc = launched()) return rc;
  }
  return 0;
}

template <typename T>
int sum_pieces(void *out, const float *part, long long n, int splits, hipStream_t s) {
  return in_launches(n, [&](long long first, dim3 grid) { hipLaunchKernelGGL(attention_sum_kernel<T>, grid, dim3(256), 0, s, (T *)out, part, first, n, splits); });
}

// The call's operands, copied where they have to be (y and gy: of the backward pass).
template <typename T>
AttnArgs args_of(const AttnCall &c, const void *y, const void *gy, const Space &at, char *ws, hipStream_t s) {
  AttnArgs a = {};
  const int dim = padded_dim(c), H = c.heads, KV = c.kv_heads;
  a.q = c.q, a.k = c.k, a.v = c.v, a.y = (void *)y, a.gy = gy;
  a.qs = c.qs[0], a.ks = c.ks[0], a.vs = c.vs[0];
  long long qp = c.qs[1], qh = c.qs[2], kp = c.ks[1], kh = c.ks[2], vp = c.vs[1], vh = c.vs[2];
  if (c.packed) a.qs = a.ks = a.vs = 0;
  a.x = c.x, a.xk = c.xk, a.slopes = c.slopes, a.q_marks = c.q_marks, a.k_marks = c.k_marks;
  a.docs = c.docs, a.nq = c.nq, a.nk = c.nk, a.rows_q = rows_of(c, true), a.rows_k = rows_of(c, false);
  a.packed = c.packed, a.H = H, a.KV = KV, a.G = H / KV, a.dim = c.dim, a.ldy = c.dim;
  if (a.G > 1) {   // n / G = n magic >> (31 + bits) for n < 2^31
    int bits = 1;
    while (1LL << bits < a.G) bits++;
    a.g_magic = (unsigned)((1ULL << (31 + bits)) / a.G + 1), a.g_shift = bits - 1;
  }
  a.scale = c.scale, a.scale2 = (float)(c.scale * 1.4426950408889634);
  AttnCopies copies = {};
  copies.dim = c.dim, copies.per = dim * (int)sizeof(T) / 16;
  const long long docs = c.packed ? 1 : c.docs;
  auto copy = [&](const void *&p, long long &ss, long long &sp, long long &sh, size_t where, long long n, int heads) {
    if (docs * n == 0) return;
    auto &m = copies.m[copies.count++];
    m.o = {p, ss, sp, sh, docs, n, heads}, m.to = ws + where, m.first = copies.threads;
    copies.threads += docs * n * heads * copies.per;
    p = m.to, ss = n * heads * dim, sp = (long long)heads * dim, sh = dim;
    if (c.packed) ss = 0;
  };
  if (!aligned(c, c.q, c.qs)) copy(a.q, a.qs, qp, qh, at.q, c.nq, H);
  if (!aligned(c, c.k, c.ks)) copy(a.k, a.ks, kp, kh, at.k, c.nk, KV);
  if (!aligned(c, c.v, c.vs)) copy(a.v, a.vs, vp, vh, at.v, c.nk, KV);
  if (gy && dim != c.dim) {
    const void *yp = y;
    for (auto *p : {&yp, &a.gy}) {
      long long ss = c.nq * H * c.dim, sp = (long long)H * c.dim, sh = c.dim;
      copy(*p, ss, sp, sh, p == &yp ? at.y : at.gy, c.nq, H);
    }
    a.y = (void *)yp, a.ldy = dim;
  }
  a.qp = (int)qp, a.qh = (int)qh, a.kp = (int)kp, a.kh = (int)kh, a.vp = (int)vp, a.vh = (int)vh;
  if (copies.threads) hipLaunchKernelGGL(attention_copy_kernel<T>, dim3((unsigned)std::min((copies.threads + 255) / 256, 1LL << 22)), dim3(256), 0, s, copies);
  return a;
}

// whether rows of results take vectors of four values
bool whole4(const AttnCall &c, std::initializer_list<const void *> results) {
  uintptr_t all = 0;
  for (const void *p : results) all |= (uintptr_t)p;
  return c.dim % 4 == 0 && all % (4 * dtype_bytes(c.dtype)) == 0;
}

AttnArgs pass_args(AttnArgs a, const Pass &p) {
  a.slots = p.slots, a.splits = p.splits, a.head_major = p.wide, a.blocked = p.blocked, a.heads = p.heads;
  return a;
}

template <typename T>
int forward(const AttnCall &c, void *y, float *lse, void *ws, hipStream_t s) {
  const Space at = space_of(c, false, false);
  const Pass p = pass_of(c, kAttnForward);
  AttnArgs a = pass_args(args_of<T>(c, y, nullptr, at, (char *)ws, s), p);
  a.lse = lse, a.vec_y = whole4(c, {y});
  if (p.splits > 1) a.part_q = (float *)((char *)ws + at.part_q), a.part_ml = (float2 *)((char *)ws + at.ml);
  if (int rc = launch_attention_kernels<kAttnForward, T>({attention_dims(c.dtype, c.dim), c.slopes ? kBiasPoints : kBiasNone, p.wide}, a, s)) return rc;
  if (p.splits == 1) return 0;
  const long long rows = a.rows_q * a.H;
  return in_launches(rows * 64, [&](long long first, dim3 grid) { hipLaunchKernelGGL(attention_join_kernel<T>, grid, dim3(256), 0, s, a, first / 64, rows); });
}

template <typename T>
int backward(const AttnCall &c, const AttnGrads &g, void *ws, hipStream_t s) {
  const bool geometry = c.slopes && (g.gx || g.gxk || g.gslopes);
  const Space at = space_of(c, true, geometry);
  auto in_ws = [&](size_t where) { return (char *)ws + where; };
  AttnArgs a = args_of<T>(c, g.y, g.gy, at, (char *)ws, s);
  a.lse = (float *)g.lse, a.delta = (float *)in_ws(at.delta), a.vec_y = whole4(c, {g.gq, g.gk, g.gv});
  a.gq = g.gq, a.gk = g.gk, a.gv = g.gv;
  if (geometry) a.geo_q = (float4 *)in_ws(at.geo_q), a.geo_k = (float4 *)in_ws(at.geo_k);
  const int bias = geometry ? kBiasGradients : c.slopes ? kBiasPoints : kBiasNone, dims = attention_dims(c.dtype, c.dim);
  Pass pr = pass_of(c, kAttnRows);
  const Pass pk = pass_of(c, kAttnKeys);
  AttnArgs r = pass_args(a, pr), k = pass_args(a, pk);
  const bool mend = pr.splits > 1 && sizeof(T) == 2;
  if (pr.splits > 1) r.part_q = (float *)in_ws(at.part_q);
  if (mend) {
    r.part_p = (float *)in_ws(at.part_p), r.part_d = (float *)in_ws(at.part_d);
    if (geometry) r.geo_p = (float4 *)in_ws(at.geo_p);
  }
  if (int rc = launch_attention_kernels<kAttnRows, T>({dims, bias, pr.wide}, r, s)) return rc;
  if (mend) {
    const int per_row = (c.dim + 3) / 4;
    const long long all = a.rows_q * a.H * per_row;
    if (int rc = in_launches(all, [&](long long first, dim3 grid) { hipLaunchKernelGGL(attention_mend_kernel<T>, grid, dim3(256), 0, s, r, first, all, per_row); })) return rc;
    pr.splits = 1;   // (of the gradients of points, from here on)
  } else if (pr.splits > 1 && g.gq)
    if (int rc = sum_pieces<T>(g.gq, r.part_q, a.rows_q * a.H * a.dim, pr.splits, s)) return rc;
  if (g.gk || g.gv || geometry) {
    if (pk.splits > 1) k.part_k = (float *)in_ws(at.part_k), k.part_v = (float *)in_ws(at.part_v);
    if (int rc = launch_attention_kernels<kAttnKeys, T>({dims, bias, pk.wide}, k, s)) return rc;
    if (pk.splits > 1) {
      const long long n = a.rows_k * a.KV * a.dim;
      if (g.gk)
        if (int rc = sum_pieces<T>(g.gk, k.part_k, n, pk.splits, s)) return rc;
      if (g.gv)
        if (int rc = sum_pieces<T>(g.gv, k.part_v, n, pk.splits, s)) return rc;
    }
  }
  if (!geometry) return 0;
  auto points = [&](float *out, bool of_q, bool of_k, long long rows) {
    const int terms = std::max(of_q ? pr.splits * a.H : 0, of_k ? pk.splits * a.KV : 0);
    int shift = 0;
    while (shift < 4 && 1 << shift < terms) shift++;
    auto launch = [&](auto lanes_log2) {
      constexpr int S = decltype(lanes_log2)::value;
      return in_launches(rows << S, [&](long long first, dim3 grid) {
        hipLaunchKernelGGL(attention_points_kernel<S>, grid, dim3(256), 0, s, out, of_q ? a.geo_q : nullptr, pr.splits, a.H, of_k ? a.geo_k : nullptr, pk.splits, a.KV, first, rows);
      });
    };
    switch (shift) {
      case 0: return launch(std::integral_constant<int, 0>());
      case 1: return launch(std::integral_constant<int, 1>());
      case 2: return launch(std::integral_constant<int, 2>());
      case 3: return launch(std::integral_constant<int, 3>());
      default: return launch(std::integral_constant<int, 4>());
    }
  };
  if (g.gx)
    if (int rc = points(g.gx, true, g.same_points, a.rows_q)) return rc;
  if (g.gxk)
    if (int rc = points(g.gxk, false, true, a.rows_k)) return rc;
  if (g.gslopes) {
    float *part = (float *)in_ws(at.slopes);
    const long long blocks = (a.rows_q + kSlopeRows - 1) / kSlopeRows;
    if (blocks) {
      int side = 1;
      while (side < 64 && side < a.H) side *= 2;
      const long long beside = (a.H + side - 1) / side, most = std::max(1LL, (1LL << 22) / beside);   // (blocks of a launch)
      hipLaunchKernelGGL(attention_slopes_kernel, dim3((unsigned)std::min(blocks, most), (unsigned)beside), dim3(256), 0, s, part, a.geo_q, pr.splits, a.rows_q, a.H, side, blocks);
      if (int rc = launched()) return rc;
    }
    hipLaunchKernelGGL(attention_slopes_join_kernel, dim3(a.H), dim3(256), 0, s, g.gslopes, part, blocks, a.H);
    return launched();
  }
  return 0;
}

}  // namespace

size_t attention_workspace(const AttnCall &c, bool backward, bool geometry) { return space_of(c, backward, geometry).bytes; }

int launch_attention(const AttnCall &c, void *y, float *lse, void *ws, hipStream_t s) {
  if (rows_of(c, true) == 0) return 0;
  return c.dtype == GELIB_HIP_F32 ? forward<float>(c, y, lse, ws, s) : c.dtype == GELIB_HIP_BF16 ? forward<bhalf_t>(c, y, lse, ws, s) : forward<half_t>(c, y, lse, ws, s);
}

int launch_attention_bwd(const AttnCall &c, const AttnGrads &g, void *ws, hipStream_t s) {
  return c.dtype == GELIB_HIP_F32 ? backward<float>(c, g, ws, s) : c.dtype == GELIB_HIP_BF16 ? backward<bhalf_t>(c, g, ws, s) : backward<half_t>(c, g, ws, s);
}

}  // namespace gelib_hip
