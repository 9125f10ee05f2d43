// The operators of a network over points (embedding, attention, cross entropy of a linear layer's classes) for gelib_base: tensors are
// checked and results allocated here, one call of the C ABI does the rest on torch's current stream of the tensors' GPU.
#include <cmath>
#include <limits>

#include "real_ops.h"
#include "tensors.h"

using namespace gelib_tensors;

namespace {

void same_kind(const at::Tensor &t, const at::Tensor &x, const char *name, const char *of) {
  if (t.scalar_type() != x.scalar_type()) throw py::type_error(std::string("GElib: ") + name + " has another type than " + of);
  if (t.device() != x.device()) throw py::value_error(std::string("GElib: ") + name + " is on another device than " + of);
}

void of_type(const at::Tensor &t, at::ScalarType type, const at::Tensor &x, const char *name, const char *type_name) {
  if (t.scalar_type() != type) throw py::type_error(std::string("GElib: ") + name + " is " + type_name);
  if (t.device() != x.device()) throw py::value_error(std::string("GElib: ") + name + " is on another device than the tensors it goes with");
}

// ---- embedding ----

void embedding_check(const at::Tensor &tokens, const at::Tensor &table, double scale) {
  on_gpu(table);
  type_of(table);
  if (tokens.scalar_type() != at::kLong && tokens.scalar_type() != at::kInt) throw py::type_error("GElib: tokens are int32 or int64");
  if (tokens.device() != table.device()) throw py::value_error("GElib: tokens are on another device than the table");
  if (table.dim() != 2 || table.size(1) < 1) throw py::value_error("GElib: the table has rows and channels");
  if (table.size(0) > 0x7fffffff || table.size(1) > 0x7fffffff || tokens.numel() > 0x7fffffff) throw py::value_error("GElib: at most 2^31 - 1 tokens, rows and channels");
  if (!std::isfinite(scale)) throw py::value_error("GElib: scale is a finite number");
}

std::vector<int64_t> with_channels(const at::Tensor &tokens, int64_t channels) {
  std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
  shape.push_back(channels);
  return shape;
}

at::Tensor embedding_fwd(const at::Tensor &tokens, const at::Tensor &table, double scale) {
  OnDevice on(table);
  const at::Tensor T = tokens.contiguous(), W = plain(table);
  at::Tensor y = at::empty(with_channels(tokens, table.size(1)), table.options().memory_format(at::MemoryFormat::Contiguous));
  done(gelib_hip_embedding_fwd(ptr(y), ptr(W), ptr(T), (int)T.element_size(), type_of(table), T.numel(), W.size(0), (int)W.size(1), (float)scale, on.stream));
  return y;
}

at::Tensor embedding_bwd(const at::Tensor &gy_, const at::Tensor &tokens, const at::Tensor &table, double scale) {
  OnDevice on(table);
  const at::Tensor T = tokens.contiguous(), gy = plain(gy_);
  same_kind(gy, table, "the gradient", "the table");
  if (gy.sizes() != at::IntArrayRef(with_channels(tokens, table.size(1)))) throw py::value_error("GElib: the gradient has another shape than the result");
  at::Tensor g = at::empty(table.sizes(), table.options().memory_format(at::MemoryFormat::Contiguous));
  const uint64_t bytes = gelib_hip_embedding_workspace_bytes(type_of(table), T.numel(), table.size(0), (int)table.size(1));
  at::Tensor ws = workspace(bytes, table);
  done(gelib_hip_embedding_bwd(ptr(g), ptr(gy), ptr(T), (int)T.element_size(), type_of(table), T.numel(), table.size(0), (int)table.size(1), (float)scale, ptr(ws), bytes,
                               on.stream));
  return g;
}

at::Tensor embedding_from_torch(const at::Tensor &tokens, const at::Tensor &table, double scale) {
  AsWritten types;
  const int64_t rows = table.size(0);
  const at::Tensor t = tokens.to(at::kLong), below = t.lt(0).unsqueeze(-1), beyond = t.ge(rows).unsqueeze(-1);
  if (rows == 0) return at::zeros(with_channels(tokens, table.size(1)), table.options()).masked_fill(beyond, std::numeric_limits<double>::quiet_NaN());
  const at::Tensor y = at::index_select(table, 0, t.clamp(0, rows - 1).reshape({-1})).reshape(with_channels(tokens, table.size(1))).to(at::kFloat) * (float)scale;
  return y.masked_fill(below, 0).masked_fill(beyond, std::numeric_limits<double>::quiet_NaN()).to(table.scalar_type());
}

struct EmbeddingFn : torch::autograd::Function<EmbeddingFn> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &tokens, const at::Tensor &table, double scale) {
    ctx->save_for_backward({tokens, table});
    ctx->saved_data["scale"] = scale;
    return embedding_fwd(tokens, table, scale);
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    const double scale = ctx->saved_data["scale"].toDouble();
    variable_list grads(3);
    if (!g[0].defined()) return grads;
    if (at::GradMode::is_enabled() || left_to_torch({&g[0], &saved[0], &saved[1]})) {
      grads[1] = graph_grads([&](const variable_list &v) { return embedding_from_torch(saved[0], v[0], scale); }, {saved[1]}, g[0])[0];
      return grads;
    }
    grads[1] = embedding_bwd(g[0], saved[0], saved[1], scale);
    return grads;
  }
};

at::Tensor embedding(const at::Tensor &tokens, const at::Tensor &table, double scale) {
  embedding_check(tokens, table, scale);
  if (left_to_torch({&tokens, &table})) return embedding_from_torch(tokens, table, scale);
  if (at::GradMode::is_enabled() && table.requires_grad()) return EmbeddingFn::apply(tokens, table, scale);
  return embedding_fwd(tokens, table, scale);
}

// ---- attention ----

// What a call is made of, all but its types checked and its defaults filled in.
struct Attention {
  at::Tensor q, k, v, points, slopes, key_points;   // key_points undefined: the queries' points
  at::Tensor q_marks, k_marks;
  bool packed;
  double scale;
};

Attention attention_of(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const Maybe &points, const Maybe &slopes, const Maybe &key_points, const Maybe &lengths,
                       const Maybe &query_lengths, const Maybe &starts, const Maybe &query_starts, const std::optional<double> &scale) {
  Attention a;
  on_gpu(q);
  type_of(q);
  same_kind(k, q, "k", "q");
  same_kind(v, q, "v", "q");
  a.packed = q.dim() == 3;
  if (q.dim() != 3 && q.dim() != 4) throw py::value_error("GElib: q is (samples, positions, heads, dim), or (rows, heads, dim) of packed documents");
  if (k.dim() != q.dim() || k.sizes() != v.sizes()) throw py::value_error("GElib: k and v are of one shape, with as many dimensions as q");
  const int64_t d = q.dim(), dim = q.size(d - 1), heads = q.size(d - 2), kv = k.size(d - 2);
  if (k.size(d - 1) != dim) throw py::value_error("GElib: q and k have heads of one size");
  if (dim < 1 || dim > 128) throw py::value_error("GElib: heads have 1 to 128 channels");
  if (heads < 1 || kv < 1 || heads % kv || heads > (1 << 20)) throw py::value_error("GElib: the number of heads of k divides that of q");
  if (!a.packed && k.size(0) != q.size(0)) throw py::value_error("GElib: q and k have as many samples");
  const int64_t nq = q.size(d - 3), nk = k.size(d - 3), most = 0x7fffff00;
  if (nq > most / (heads / kv) || nk > most) throw py::value_error("GElib: too many rows");
  auto marks = [&](const Maybe &m, int64_t n, const char *name) {
    of_type(*m, at::kInt, q, name, "int32");
    if (m->dim() != 1 || (n >= 0 ? m->size(0) != n : m->size(0) < 1)) throw py::value_error(std::string("GElib: ") + name + ": one a sample, or the documents' starts and the last one's end");
    return *m;
  };
  if (a.packed) {
    if (lengths || query_lengths) throw py::value_error("GElib: lengths are of padded samples; packed documents have starts");
    if (!starts) throw py::value_error("GElib: packed documents need their starts");
    a.k_marks = marks(starts, -1, "starts");
    if (!query_starts && nq != nk) throw py::value_error("GElib: queries and keys that are not the same rows need query_starts");
    a.q_marks = query_starts ? marks(query_starts, a.k_marks.size(0), "query_starts") : a.k_marks;
  } else {
    if (starts || query_starts) throw py::value_error("GElib: starts are of packed documents (rows, heads, dim); padded samples have lengths");
    if (lengths) a.k_marks = marks(lengths, q.size(0), "lengths");
    if (query_lengths) a.q_marks = marks(query_lengths, q.size(0), "query_lengths");
  }
  if (!points != !slopes) throw py::value_error("GElib: points and slopes belong together");
  if (key_points && !points) throw py::value_error("GElib: key_points need points");
  if (points) {
    auto shaped = [&](const at::Tensor &p, const at::Tensor &of, const char *name) {
      of_type(p, at::kFloat, q, name, "float32");
      std::vector<int64_t> shape(of.sizes().begin(), of.sizes().end() - 2);
      shape.push_back(3);
      if (p.sizes() != at::IntArrayRef(shape)) throw py::value_error(std::string("GElib: ") + name + " has three coordinates a row");
    };
    a.points = *points;
    shaped(a.points, q, "points");
    if (key_points && !key_points->is_same(*points)) a.key_points = *key_points, shaped(a.key_points, k, "key_points");
    else if (nq != nk) throw py::value_error("GElib: queries and keys that are not the same rows need key_points");
    a.slopes = *slopes;
    of_type(a.slopes, at::kFloat, q, "slopes", "float32");
    if (a.slopes.dim() != 1 || a.slopes.size(0) != heads) throw py::value_error("GElib: one slope a head of q");
  }
  a.scale = scale ? *scale : 1 / std::sqrt((double)dim);
  if (!std::isfinite(a.scale)) throw py::value_error("GElib: scale is a finite number");
  a.q = q, a.k = k, a.v = v;
  return a;
}

at::Tensor heads_in_memory(const at::Tensor &t) {   // a head's channels lie side by side, rows and heads anywhere
  const at::Tensor r = t.is_neg() ? t.resolve_neg() : t;
  return r.stride(-1) == 1 || r.size(-1) == 1 ? r : r.contiguous();
}

struct Operands {
  Attention a;   // as the kernels take them
  gelib_attention_desc d = {};
  explicit Operands(const Attention &given) : a(given) {
    a.q = heads_in_memory(a.q), a.k = heads_in_memory(a.k), a.v = heads_in_memory(a.v);
    if (a.points.defined()) a.points = plain(a.points), a.slopes = plain(a.slopes);
    if (a.key_points.defined()) a.key_points = plain(a.key_points);
    if (a.q_marks.defined()) a.q_marks = a.q_marks.contiguous();
    if (a.k_marks.defined()) a.k_marks = a.k_marks.contiguous();
    const int64_t n = a.q.dim();
    d.q = ptr(a.q), d.k = ptr(a.k), d.v = ptr(a.v);
    if (a.points.defined()) {
      d.points = (const float *)ptr(a.points), d.slopes = (const float *)ptr(a.slopes);
      d.key_points = a.key_points.defined() ? (const float *)ptr(a.key_points) : d.points;
    }
    if (a.q_marks.defined()) d.query_marks = (const int32_t *)ptr(a.q_marks);
    if (a.k_marks.defined()) d.key_marks = (const int32_t *)ptr(a.k_marks);
    d.packed = a.packed;
    d.documents = a.packed ? a.k_marks.size(0) - 1 : a.q.size(0);
    d.queries = a.q.size(n - 3), d.keys = a.k.size(n - 3);
    d.heads = (int)a.q.size(n - 2), d.kv_heads = (int)a.k.size(n - 2), d.dim = (int)a.q.size(n - 1);
    d.dtype = type_of(a.q), d.scale = (float)a.scale;
    auto strides = [&](int64_t *s, const at::Tensor &t) {
      s[0] = a.packed ? 0 : t.stride(0), s[1] = t.stride(n - 3), s[2] = t.stride(n - 2);
      // (of an extent of one: any; it would count among what is not aligned)
      if (!a.packed && t.size(0) == 1) s[0] = 0;
      if (t.size(n - 3) <= 1) s[1] = 0;
      if (t.size(n - 2) == 1) s[2] = 0;
    };
    strides(d.q_strides, a.q), strides(d.k_strides, a.k), strides(d.v_strides, a.v);
  }
};

std::tuple<at::Tensor, at::Tensor> attention_fwd(const Attention &given, bool keep) {
  OnDevice on(given.q);
  const Operands o(given);
  const auto packed = given.q.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor y = at::empty(given.q.sizes(), packed), lse;
  if (keep) lse = at::empty(given.q.sizes().slice(0, given.q.dim() - 1), packed.dtype(at::kFloat));
  const uint64_t bytes = gelib_hip_attention_workspace_bytes(&o.d, 0);
  at::Tensor ws = workspace(bytes, given.q);
  done(gelib_hip_attention_fwd(&o.d, ptr(y), (float *)ptr(lse), ptr(ws), bytes, on.stream));
  return {y, lse};
}

// Gradients of q, k, v, points, slopes and key_points; those that are not wanted stay undefined.
variable_list attention_bwd(const Attention &given, const at::Tensor &y, const at::Tensor &lse, const at::Tensor &gy_, const std::vector<bool> &wanted) {
  OnDevice on(given.q);
  const Operands o(given);
  const at::Tensor gy = plain(gy_);
  same_kind(gy, given.q, "the gradient", "q");
  if (gy.sizes() != given.q.sizes()) throw py::value_error("GElib: the gradient has another shape than the result");
  const at::Tensor *like[] = {&given.q, &given.k, &given.v, &given.points, &given.slopes, &given.key_points};
  variable_list g(6);
  for (int k = 0; k < 6; k++)
    if (wanted[k]) g[k] = at::empty(like[k]->sizes(), like[k]->options().memory_format(at::MemoryFormat::Contiguous));
  const bool geometry = ptr(g[3]) || ptr(g[4]) || ptr(g[5]);
  const uint64_t bytes = gelib_hip_attention_workspace_bytes(&o.d, geometry ? 2 : 1);
  at::Tensor ws = workspace(bytes, given.q);
  const bool same = given.points.defined() && !given.key_points.defined();
  done(gelib_hip_attention_bwd(&o.d, ptr(y), (const float *)ptr(lse), ptr(gy), ptr(g[0]), ptr(g[1]), ptr(g[2]), (float *)ptr(g[3]), (float *)ptr(g[5]), (float *)ptr(g[4]),
                               same, ptr(ws), bytes, on.stream));
  return g;
}

// tensors: q, k, v, points, slopes, key_points
at::Tensor attention_from_torch(const variable_list &t, const Attention &a) {
  AsWritten types;
  auto batched = [&](const at::Tensor &x) { return a.packed && x.defined() ? x.unsqueeze(0) : x; };
  at::Tensor q = batched(t[0]).to(at::kFloat), k = batched(t[1]).to(at::kFloat), v = batched(t[2]).to(at::kFloat);
  at::Tensor points = batched(t[3]), key_points = t[5].defined() ? batched(t[5]) : points;
  const int64_t n = q.size(0), nq = q.size(1), nk = k.size(1), heads = q.size(2), kv = k.size(2), dim = q.size(3), G = heads / kv;
  // which queries see which keys
  at::Tensor sees, there_q, there_k;   // (n, nq, nk), (n, nq), (n, nk); undefined: all
  if (a.packed) {
    auto document = [&](const at::Tensor &starts, int64_t rows) {
      const at::Tensor s = starts.to(at::kLong), i = at::arange(rows, s.options());
      return i.unsqueeze(1).ge(s.unsqueeze(0)).sum(1);
    };
    const at::Tensor dq = document(a.q_marks, nq), dk = document(a.k_marks, nk);
    const int64_t docs = a.k_marks.size(0) - 1;
    there_q = (dq.ge(1) & dq.le(docs)).unsqueeze(0), there_k = (dk.ge(1) & dk.le(docs)).unsqueeze(0);
    sees = dq.unsqueeze(1).eq(dk.unsqueeze(0)).unsqueeze(0) & there_q.unsqueeze(2) & there_k.unsqueeze(1);
  } else {
    if (a.q_marks.defined()) there_q = at::arange(nq, a.q_marks.options()).unsqueeze(0).lt(a.q_marks.unsqueeze(1));
    if (a.k_marks.defined()) there_k = at::arange(nk, a.k_marks.options()).unsqueeze(0).lt(a.k_marks.unsqueeze(1)), sees = there_k.unsqueeze(1).expand({n, nq, nk});
  }
  // (what is not there may be no number, which times zero would still be none.  A row of shared points may be there on one side only)
  auto without = [&](at::Tensor &x, const at::Tensor &there) {
    if (x.defined() && there.defined()) x = x.masked_fill((x.dim() == 4 ? there.unsqueeze(2).unsqueeze(3) : there.unsqueeze(2)).logical_not(), 0);
  };
  without(q, there_q), without(points, there_q);
  without(k, there_k), without(v, there_k), without(key_points, there_k);
  const at::Tensor kt = k.permute({0, 2, 3, 1}), vt = v.permute({0, 2, 1, 3});
  const at::Tensor rows = q.reshape({n, nq, kv, G, dim}).permute({0, 2, 3, 1, 4}).reshape({n, kv, G * nq, dim});
  at::Tensor s = at::matmul(rows, kt).reshape({n, kv, G, nq, nk}) * a.scale;
  if (points.defined()) {
    const at::Tensor sq = (points.unsqueeze(2) - key_points.unsqueeze(1)).square().sum(3), zero = sq.eq(0);
    const at::Tensor far = sq.masked_fill(zero, 1).sqrt().masked_fill(zero, 0);   // (no direction where two points are one)
    s = s - t[4].view({1, kv, G, 1, 1}) * far.view({n, 1, 1, nq, nk});
  }
  if (sees.defined()) {
    const at::Tensor hidden = sees.logical_not().view({sees.size(0), 1, 1, nq, nk}), blind = sees.any(2).logical_not().view({sees.size(0), 1, 1, nq, 1});
    s = at::softmax(s.masked_fill(hidden, -std::numeric_limits<double>::infinity()).masked_fill(blind, 0), -1).masked_fill(hidden, 0);
  } else if (nk) {
    s = at::softmax(s, -1);
  }
  at::Tensor y = at::matmul(s.reshape({n, kv, G * nq, nk}), vt).reshape({n, kv, G, nq, dim}).permute({0, 3, 1, 2, 4}).reshape({n, nq, heads, dim});
  if (there_q.defined()) y = y.masked_fill(there_q.logical_not().view({there_q.size(0), nq, 1, 1}), 0);
  return (a.packed ? y.squeeze(0) : y).to(t[0].scalar_type());
}

struct AttentionFn : torch::autograd::Function<AttentionFn> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const Maybe &points, const Maybe &slopes,
                            const Maybe &key_points, const Maybe &q_marks, const Maybe &k_marks, bool packed, double scale) {
    const Attention a = {q, k, v, some(points), some(slopes), some(key_points), some(q_marks), some(k_marks), packed, scale};
    auto [y, lse] = attention_fwd(a, true);
    ctx->save_for_backward({q, k, v, a.points, a.slopes, a.key_points, a.q_marks, a.k_marks, y, lse});
    ctx->saved_data["packed"] = packed;
    ctx->saved_data["scale"] = scale;
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    variable_list grads(10);
    if (!g[0].defined()) return grads;
    const Attention a = {saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], saved[6], saved[7], ctx->saved_data["packed"].toBool(), ctx->saved_data["scale"].toDouble()};
    if (at::GradMode::is_enabled() || left_to_torch({&g[0], &saved[0], &saved[1], &saved[2], &saved[3], &saved[4], &saved[5]})) {
      const variable_list got = graph_grads([&](const variable_list &t) { return attention_from_torch(t, a); }, {saved[0], saved[1], saved[2], saved[3], saved[4], saved[5]}, g[0]);
      std::copy(got.begin(), got.end(), grads.begin());
      return grads;
    }
    std::vector<bool> wanted(6);
    size_t at = 0;   // (tensors that were given are counted)
    for (int k = 0; k < 6; k++)
      if (saved[k].defined()) wanted[k] = ctx->needs_input_grad(at++);
    if (std::find(wanted.begin(), wanted.end(), true) == wanted.end()) return grads;
    const variable_list got = attention_bwd(a, saved[8], saved[9], g[0], wanted);
    std::copy(got.begin(), got.end(), grads.begin());
    return grads;
  }
};

at::Tensor attention(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const Maybe &points, const Maybe &slopes, const Maybe &key_points, const Maybe &lengths,
                     const Maybe &query_lengths, const Maybe &starts, const Maybe &query_starts, const std::optional<double> &scale) {
  const Attention a = attention_of(q, k, v, points, slopes, key_points, lengths, query_lengths, starts, query_starts, scale);
  if (left_to_torch({&q, &k, &v, address(points), address(slopes), address(key_points), address(lengths), address(query_lengths), address(starts), address(query_starts)}))
    return attention_from_torch({a.q, a.k, a.v, a.points, a.slopes, a.key_points}, a);
  if (at::GradMode::is_enabled() && (needs(q) || needs(k) || needs(v) || needs(a.points) || needs(a.slopes) || needs(a.key_points)))
    return AttentionFn::apply(q, k, v, some(a.points), some(a.slopes), some(a.key_points), some(a.q_marks), some(a.k_marks), a.packed, a.scale);
  return std::get<0>(attention_fwd(a, false));
}

// ---- cross entropy of a linear layer's classes ----

void loss_check(const at::Tensor &x, const at::Tensor &w, const at::Tensor &targets, const Maybe &b) {
  on_gpu(x);
  type_of(x);
  same_kind(w, x, "w", "x");
  if (x.dim() < 1 || w.dim() != 2 || w.size(0) != x.size(-1)) throw py::value_error("GElib: x (..., n_in) and w (n_in, n_out) are needed");
  if (w.size(1) < 1) throw py::value_error("GElib: there is at least one class");
  if (std::max(w.size(0), w.size(1)) > 0x7fffff00) throw py::value_error("GElib: too many channels");
  of_type(targets, at::kLong, x, "targets", "int64");
  if (targets.sizes() != x.sizes().slice(0, x.dim() - 1)) throw py::value_error("GElib: one target a row of x");
  if (b) {
    same_kind(*b, x, "bias", "x");
    if (b->dim() != 1 || b->size(0) != w.size(1)) throw py::value_error("GElib: bias has one value a class");
  }
}

std::tuple<at::Tensor, at::Tensor> loss_fwd(const at::Tensor &x, const at::Tensor &w, const at::Tensor &targets, const Maybe &b, bool keep) {
  OnDevice on(x);
  const Rows X = rows_of(x);
  const at::Tensor W = plain(w), B = b ? plain(*b) : at::Tensor(), T = targets.contiguous();
  const auto f32 = x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
  at::Tensor loss = at::empty(targets.sizes(), f32), lse;
  if (keep) lse = at::empty(targets.sizes(), f32);
  const int N = (int)w.size(1);
  const uint64_t bytes = gelib_hip_linear_cross_entropy_workspace_bytes(0, type_of(x), X.rows, X.K, N);
  at::Tensor ws = workspace(bytes, x);
  done(gelib_hip_linear_cross_entropy_fwd((float *)ptr(loss), (float *)ptr(lse), ptr(X.x), ptr(W), ptr(B), (const int64_t *)ptr(T), type_of(x), X.rows, X.K, N, X.stride,
                                          ptr(ws), bytes, on.stream));
  return {loss, lse};
}

variable_list loss_bwd(const at::Tensor &g_, const at::Tensor &lse, const at::Tensor &x, const at::Tensor &w, const at::Tensor &targets, const Maybe &b, const bool wanted[3]) {
  OnDevice on(x);
  const Rows X = rows_of(x);
  const at::Tensor W = plain(w), B = b ? plain(*b) : at::Tensor(), T = targets.contiguous(), G = plain(g_);
  same_kind(G, lse, "the gradient", "the losses");
  if (G.sizes() != targets.sizes()) throw py::value_error("GElib: the gradient has another shape than the losses");
  const int N = (int)w.size(1);
  const auto packed = x.options().memory_format(at::MemoryFormat::Contiguous);
  variable_list g(3);
  if (wanted[0]) g[0] = at::empty(x.sizes(), packed);
  if (wanted[1]) g[1] = at::empty(w.sizes(), packed);
  if (wanted[2]) g[2] = at::empty({N}, packed);
  const int what = (ptr(g[0]) ? 1 : 0) | (ptr(g[1]) ? 2 : 0) | (ptr(g[2]) ? 4 : 0);
  const uint64_t bytes = what ? gelib_hip_linear_cross_entropy_workspace_bytes(what, type_of(x), X.rows, X.K, N) : 0;
  at::Tensor ws = workspace(bytes, x);
  done(gelib_hip_linear_cross_entropy_bwd(ptr(g[0]), ptr(g[1]), ptr(g[2]), (const float *)ptr(G), (const float *)ptr(lse), ptr(X.x), ptr(W), ptr(B), (const int64_t *)ptr(T),
                                          type_of(x), X.rows, X.K, N, X.stride, ptr(ws), bytes, on.stream));
  return g;
}

at::Tensor loss_from_torch(const at::Tensor &x, const at::Tensor &w, const at::Tensor &b, const at::Tensor &targets) {
  AsWritten types;
  // (a row left out may hold anything, and so may what it meets in w: zero before the product and after)
  const at::Tensor out = targets.lt(0), out_row = out.unsqueeze(-1);
  at::Tensor z = at::matmul(x.to(at::kFloat).masked_fill(out_row, 0), w.to(at::kFloat));
  if (b.defined()) z = z + b.to(at::kFloat);
  z = z.masked_fill(out_row, 0);
  const at::Tensor of = at::gather(z, -1, targets.clamp(0, w.size(1) - 1).unsqueeze(-1)).squeeze(-1);
  return (at::logsumexp(z, -1) - of).masked_fill(out, 0).masked_fill(targets.ge(w.size(1)), std::numeric_limits<double>::quiet_NaN());
}

struct LossFn : torch::autograd::Function<LossFn> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &w, const at::Tensor &targets, const Maybe &b) {
    auto [loss, lse] = loss_fwd(x, w, targets, b, true);
    ctx->save_for_backward({x, w, targets, some(b), lse});
    return loss;
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &targets = saved[2], &b = saved[3];
    variable_list grads(4);
    if (!g[0].defined()) return grads;
    if (at::GradMode::is_enabled() || left_to_torch({&g[0], &x, &w, &targets, &b})) {
      const variable_list got = graph_grads([&](const variable_list &v) { return loss_from_torch(v[0], v[1], v[2], targets); }, {x, w, b}, g[0]);
      grads[0] = got[0], grads[1] = got[1], grads[3] = got[2];
      return grads;
    }
    const bool wanted[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), b.defined() && ctx->needs_input_grad(3)};
    if (!wanted[0] && !wanted[1] && !wanted[2]) return grads;
    const variable_list got = loss_bwd(g[0], saved[4], x, w, targets, some(b), wanted);
    grads[0] = got[0], grads[1] = got[1], grads[3] = got[2];
    return grads;
  }
};

at::Tensor linear_cross_entropy(const at::Tensor &x, const at::Tensor &w, const at::Tensor &targets, const Maybe &b) {
  loss_check(x, w, targets, b);
  if (left_to_torch({&x, &w, &targets, address(b)})) return loss_from_torch(x, w, some(b), targets);
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (b && needs(*b)))) return LossFn::apply(x, w, targets, b);
  return std::get<0>(loss_fwd(x, w, targets, b, false));
}

}  // namespace

void bind_point_ops(pybind11::module_ &m) {
  m.def("embedding", &embedding);
  m.def("attention", &attention);
  m.def("linear_cross_entropy", &linear_cross_entropy);
}
