// C entry points of the operators of a network over points: checks of their arguments, then one launcher each.  Nothing is launched
// unless every pointer is device memory of the current GPU and long enough.
#include <cmath>

#include "cabi_check.h"
#include "real_ops.h"

using namespace gelib_hip;

namespace {

bool dtype_ok(int dtype) { return dtype >= GELIB_HIP_F32 && dtype <= GELIB_HIP_F16; }

int embedding_shape(int dtype, int token_bytes, int64_t n, int64_t rows, int C, float scale) {
  if (!dtype_ok(dtype) || (token_bytes != 4 && token_bytes != 8) || n < 0 || rows < 0 || rows > 0x7fffffff || C < 1 || !std::isfinite(scale)) return GELIB_HIP_ERR_ARG;
  if (!product_ok(n, C) || !product_ok(rows, C)) return GELIB_HIP_ERR_ARG;
  return GELIB_HIP_OK;
}
int embedding_bwd_shape(int dtype, int token_bytes, int64_t n, int64_t rows, int C, float scale) {
  return n > 0x7fffffff ? (int)GELIB_HIP_ERR_ARG : embedding_shape(dtype, token_bytes, n, rows, C, scale);
}

int attention_shape(const gelib_attention_desc &a) {
  if (!dtype_ok(a.dtype) || (a.packed != 0 && a.packed != 1) || a.documents < 0 || a.queries < 0 || a.keys < 0 || !std::isfinite(a.scale)) return GELIB_HIP_ERR_ARG;
  if (a.heads < 1 || a.kv_heads < 1 || a.heads % a.kv_heads || a.heads > (1 << 20) || a.dim < 1 || a.dim > kAttnMostDim) return GELIB_HIP_ERR_ARG;
  // rows of a document, heads that share keys counted one by one, and starts are 32-bit numbers
  const int64_t most = 0x7fffff00;
  if (a.queries > most / (a.heads / a.kv_heads) || a.keys > most || a.documents > (1LL << 31)) return GELIB_HIP_ERR_ARG;
  const int64_t docs = a.packed ? 1 : a.documents;
  if (!product_ok(docs, a.queries) || !product_ok(docs, a.keys)) return GELIB_HIP_ERR_ARG;
  if (!product_ok(docs * a.queries, (int64_t)a.heads * a.dim) || !product_ok(docs * a.keys, (int64_t)a.kv_heads * a.dim)) return GELIB_HIP_ERR_ARG;
  for (const int64_t *s : {a.q_strides, a.k_strides, a.v_strides}) {
    for (int k = 0; k < 3; k++)
      if (s[k] < 0) return GELIB_HIP_ERR_ARG;
    const int64_t n = s == a.q_strides ? a.queries : a.keys, h = s == a.q_strides ? a.heads : a.kv_heads;
    if ((!a.packed && !product_ok(a.documents, s[0])) || !product_ok(n, s[1]) || !product_ok(h, s[2])) return GELIB_HIP_ERR_ARG;
  }
  if (!a.points != !a.slopes || !a.key_points != !a.slopes) {
    // (an empty side has no points to point to)
    const bool points = a.points || docs * a.queries == 0, key_points = a.key_points || docs * a.keys == 0;
    if (a.slopes ? !points || !key_points : a.points || a.key_points) return GELIB_HIP_ERR_ARG;
  }
  if (a.packed && (!a.query_marks || !a.key_marks)) return GELIB_HIP_ERR_NULL;
  return GELIB_HIP_OK;
}

AttnCall call_of(const gelib_attention_desc &a) {
  AttnCall c = {};
  c.q = a.q, c.k = a.k, c.v = a.v, c.x = a.points, c.xk = a.key_points, c.slopes = a.slopes, c.q_marks = a.query_marks, c.k_marks = a.key_marks;
  c.docs = a.documents, c.nq = a.queries, c.nk = a.keys;
  for (int k = 0; k < 3; k++) c.qs[k] = a.q_strides[k], c.ks[k] = a.k_strides[k], c.vs[k] = a.v_strides[k];
  c.dtype = a.dtype, c.packed = a.packed, c.heads = a.heads, c.kv_heads = a.kv_heads, c.dim = a.dim, c.scale = a.scale;
  return c;
}

// the operands' memory
void attention_operands(Memory &mem, const gelib_attention_desc &a) {
  const unsigned e = (unsigned)dtype_bytes(a.dtype);
  const int64_t docs = a.packed ? 1 : a.documents;
  auto strided = [&](const void *p, const int64_t *s, int64_t n, int64_t h) {
    if (docs && n) mem.need(p, ((a.packed ? 0 : (docs - 1) * s[0]) + (n - 1) * s[1] + (h - 1) * s[2] + a.dim) * e, e);
  };
  strided(a.q, a.q_strides, a.queries, a.heads);
  strided(a.k, a.k_strides, a.keys, a.kv_heads);
  strided(a.v, a.v_strides, a.keys, a.kv_heads);
  mem.may(a.points, docs * a.queries * 12, 4);
  mem.may(a.key_points, docs * a.keys * 12, 4);
  mem.may(a.slopes, (int64_t)a.heads * 4, 4);
  for (const int32_t *m : {a.query_marks, a.key_marks}) mem.may(m, (a.packed ? a.documents + 1 : a.documents) * 4, 4);
}

int loss_shape(int dtype, int64_t rows, int K, int N, int64_t xs) {
  if (!dtype_ok(dtype) || rows < 0 || K < 0 || N < 1 || xs < 0 || std::max(K, N) > kLinearMostChannels) return GELIB_HIP_ERR_ARG;
  if (!product_ok(rows, K) || !product_ok(rows, N) || !product_ok(rows, xs)) return GELIB_HIP_ERR_ARG;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  if (rows > 1 && xs * e % row_align(e, K) != 0) return GELIB_HIP_ERR_ARG;
  return GELIB_HIP_OK;
}

void loss_operands(Memory &mem, const void *x, const void *w, const void *bias, const int64_t *targets, int dtype, int64_t rows, int K, int N, int64_t xs) {
  const unsigned e = (unsigned)dtype_bytes(dtype);
  if (rows && K) mem.need(x, ((rows - 1) * xs + K) * e, row_align(e, K)), mem.need(w, (int64_t)K * N * e, row_align(e, N));
  mem.may(bias, (int64_t)N * e, e);
  mem.need(targets, rows * 8, 8);
}

}  // namespace

extern "C" {

int gelib_hip_embedding_fwd(void *y, const void *table, const void *tokens, int token_bytes, int dtype, int64_t ntokens, int64_t rows, int channels,
                            float scale, void *stream) {
  set_last_path(kPathNone);
  if (int rc = embedding_shape(dtype, token_bytes, ntokens, rows, channels, scale)) return rc;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  Memory mem;
  mem.need(y, ntokens * channels * e, e);
  if (ntokens) mem.need(table, rows * channels * e, e);
  mem.need(tokens, ntokens * token_bytes, (unsigned)token_bytes);
  if (int rc = mem.rc()) return rc;
  EmbeddingArgs a = {};
  a.y = y, a.table = table, a.tokens = tokens, a.wide = token_bytes == 8, a.n = ntokens, a.rows = rows, a.channels = channels, a.scale = scale;
  set_last_path(kPathReal);
  return launch_embedding(dtype, a, (hipStream_t)stream);
}

int gelib_hip_embedding_bwd(void *gtable, const void *gy, const void *tokens, int token_bytes, int dtype, int64_t ntokens, int64_t rows, int channels,
                            float scale, void *workspace, uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (int rc = embedding_bwd_shape(dtype, token_bytes, ntokens, rows, channels, scale)) return rc;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  Memory mem;
  mem.need(gtable, rows * channels * e, e);
  if (rows) mem.need(gy, ntokens * channels * e, e), mem.need(tokens, ntokens * token_bytes, (unsigned)token_bytes);
  if (int rc = mem.rc()) return rc;
  if (rows == 0) return GELIB_HIP_OK;
  if (int rc = check_workspace(workspace, workspace_bytes, embedding_workspace(ntokens, channels))) return rc;
  EmbeddingArgs a = {};
  a.gtable = gtable, a.gy = gy, a.tokens = tokens, a.wide = token_bytes == 8, a.n = ntokens, a.rows = rows, a.channels = channels, a.scale = scale;
  a.ws = workspace;
  set_last_path(kPathReal);
  return launch_embedding_bwd(dtype, a, (hipStream_t)stream);
}

uint64_t gelib_hip_embedding_workspace_bytes(int dtype, int64_t ntokens, int64_t rows, int channels) {
  if (embedding_bwd_shape(dtype, 8, ntokens, rows, channels, 1.f) || rows == 0) return 0;
  return embedding_workspace(ntokens, channels);
}

int gelib_hip_attention_fwd(const gelib_attention_desc *a, void *y, float *lse, void *workspace, uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (!a) return GELIB_HIP_ERR_NULL;
  if (int rc = attention_shape(*a)) return rc;
  const unsigned e = (unsigned)dtype_bytes(a->dtype);
  const int64_t rows = (a->packed ? 1 : a->documents) * a->queries * a->heads;
  Memory mem;
  attention_operands(mem, *a);
  mem.need(y, rows * a->dim * e, e);
  mem.may(lse, rows * 4, 4);
  if (int rc = mem.rc()) return rc;
  const AttnCall c = call_of(*a);
  if (int rc = check_workspace(workspace, workspace_bytes, attention_workspace(c, false, false))) return rc;
  set_last_path(kPathReal);
  return launch_attention(c, y, lse, workspace, (hipStream_t)stream);
}

int gelib_hip_attention_bwd(const gelib_attention_desc *a, const void *y, const float *lse, const void *gy, void *gq, void *gk, void *gv, float *gpoints,
                            float *gkey_points, float *gslopes, int same_points, void *workspace, uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (!a) return GELIB_HIP_ERR_NULL;
  if (int rc = attention_shape(*a)) return rc;
  const unsigned e = (unsigned)dtype_bytes(a->dtype);
  const int64_t docs = a->packed ? 1 : a->documents, rq = docs * a->queries, rk = docs * a->keys;
  if (!a->slopes && (gpoints || gkey_points || gslopes)) return GELIB_HIP_ERR_ARG;
  if (same_points && (gkey_points || rq != rk || a->points != a->key_points)) return GELIB_HIP_ERR_ARG;
  Memory mem;
  attention_operands(mem, *a);
  for (const void *p : {y, gy}) mem.need(p, rq * a->heads * a->dim * e, row_align(e, a->dim));
  mem.need(lse, rq * a->heads * 4, 4);
  mem.may(gq, rq * a->heads * a->dim * e, e);
  mem.may(gk, rk * a->kv_heads * a->dim * e, e);
  mem.may(gv, rk * a->kv_heads * a->dim * e, e);
  mem.may(gpoints, rq * 12, 4);
  mem.may(gkey_points, rk * 12, 4);
  mem.may(gslopes, (int64_t)a->heads * 4, 4);
  if (int rc = mem.rc()) return rc;
  const AttnCall c = call_of(*a);
  if (int rc = check_workspace(workspace, workspace_bytes, attention_workspace(c, true, gpoints || gkey_points || gslopes))) return rc;
  AttnGrads g = {};
  g.y = y, g.gy = gy, g.lse = lse, g.gq = gq, g.gk = gk, g.gv = gv, g.gx = gpoints, g.gxk = gkey_points, g.gslopes = gslopes, g.same_points = same_points != 0;
  set_last_path(kPathReal);
  return launch_attention_bwd(c, g, workspace, (hipStream_t)stream);
}

uint64_t gelib_hip_attention_workspace_bytes(const gelib_attention_desc *a, int what) {
  if (!a || what < 0 || what > 2 || attention_shape(*a)) return 0;
  return attention_workspace(call_of(*a), what > 0, what == 2);
}

int gelib_hip_linear_cross_entropy_fwd(float *loss, float *lse, const void *x, const void *w, const void *bias, const int64_t *targets, int dtype,
                                       int64_t rows, int n_in, int n_out, int64_t x_row_stride, void *workspace, uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (int rc = loss_shape(dtype, rows, n_in, n_out, x_row_stride)) return rc;
  Memory mem;
  mem.need(loss, rows * 4, 4);
  mem.may(lse, rows * 4, 4);
  loss_operands(mem, x, w, bias, targets, dtype, rows, n_in, n_out, x_row_stride);
  if (int rc = mem.rc()) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, loss_workspace(0, dtype, rows, n_in, n_out))) return rc;
  LossArgs a = {};
  a.loss = loss, a.lse_out = lse, a.x = x, a.w = w, a.b = bias, a.targets = (const long long *)targets;
  a.rows = rows, a.xs = x_row_stride, a.K = n_in, a.N = n_out, a.ws = workspace;
  set_last_path(kPathReal);
  return launch_loss(dtype, a, (hipStream_t)stream);
}

int gelib_hip_linear_cross_entropy_bwd(void *gx, void *gw, void *gb, const float *g, const float *lse, const void *x, const void *w, const void *bias,
                                       const int64_t *targets, int dtype, int64_t rows, int n_in, int n_out, int64_t x_row_stride, void *workspace,
                                       uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (int rc = loss_shape(dtype, rows, n_in, n_out, x_row_stride)) return rc;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  Memory mem;
  mem.need(g, rows * 4, 4);
  mem.need(lse, rows * 4, 4);
  loss_operands(mem, x, w, bias, targets, dtype, rows, n_in, n_out, x_row_stride);
  mem.may(gx, rows * n_in * e, e);
  mem.may(gw, (int64_t)n_in * n_out * e, e);
  mem.may(gb, (int64_t)n_out * e, e);
  if (int rc = mem.rc()) return rc;
  const int what = (gx ? 1 : 0) | (gw ? 2 : 0) | (gb ? 4 : 0);
  if (int rc = check_workspace(workspace, workspace_bytes, what ? loss_workspace(what, dtype, rows, n_in, n_out) : 0)) return rc;
  LossArgs a = {};
  a.gx = gx, a.gw = gw, a.gb = gb, a.g = g, a.lse = lse, a.x = x, a.w = w, a.b = bias, a.targets = (const long long *)targets;
  a.rows = rows, a.xs = x_row_stride, a.K = n_in, a.N = n_out, a.ws = workspace;
  set_last_path(kPathReal);
  return launch_loss_bwd(dtype, a, (hipStream_t)stream);
}

uint64_t gelib_hip_linear_cross_entropy_workspace_bytes(int backward, int dtype, int64_t rows, int n_in, int n_out) {
  if (backward < 0 || backward > 7 || loss_shape(dtype, rows, n_in, n_out, 0)) return 0;
  return loss_workspace(backward, dtype, rows, n_in, n_out);
}

}  // extern "C"
