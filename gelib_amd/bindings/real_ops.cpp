// The operators on real channels (group norm with an activation, linear layer with its epilogue, AdamW) for gelib_base: tensors
// are checked and results allocated here, one call of the C ABI does the rest on torch's current stream of the tensors' GPU.
// (A step over hundreds of parameters, or a layer on a few rows, would spend longer in Python than on the GPU.)
#include "real_ops.h"
#include "tensors.h"

using namespace gelib_tensors;

namespace {

int act_of(const std::string &act) {
  if (act == "none") return GELIB_HIP_ACT_NONE;
  if (act == "relu") return GELIB_HIP_ACT_RELU;
  if (act == "silu") return GELIB_HIP_ACT_SILU;
  if (act == "gelu") return GELIB_HIP_ACT_GELU;
  throw py::value_error("GElib: act is one of 'none', 'relu', 'silu', 'gelu'");
}

// ---- group norm ----

// x as samples x positions x channels: the strides of its samples and positions, of x itself where its positions are evenly
// spaced, its channels contiguous and its rows aligned as those of a packed tensor are (16 bytes where the number of channels
// allows), else of a copy: reading and writing it once is less than narrow loads cost, and a result does not depend on the layout
struct NormShape {
  at::Tensor x;
  int64_t N, S, xs, xp;
  int C;
};
NormShape norm_shape(const at::Tensor &t) {
  NormShape r;
  r.x = t.is_neg() ? t.resolve_neg() : t;
  const int64_t d = t.dim();
  r.N = t.size(0), r.C = (int)t.size(d - 1), r.S = 1;
  for (int64_t k = 1; k < d - 1; k++) r.S *= t.size(k);
  bool even = t.stride(d - 1) == 1 || r.C == 1;
  int64_t step = -1, inner = 1;   // position stride, positions of the dimensions already seen
  for (int64_t k = d - 2; k >= 1 && even; k--) {
    if (t.size(k) == 1) continue;
    if (step < 0) step = r.x.stride(k);
    else even = r.x.stride(k) == step * inner;
    inner *= t.size(k);
  }
  const int64_t e = t.element_size(), width = r.C % (16 / e) == 0 ? 16 / e : r.C % 2 == 0 ? 2 : 1;
  if (even) even = (step < 0 || step % width == 0) && (r.N == 1 || r.x.stride(0) % width == 0) && (uintptr_t)r.x.data_ptr() % (width * e) == 0;
  if (!even || r.x.numel() == 0) {
    r.x = r.x.is_contiguous() ? r.x.clone() : r.x.contiguous();
    step = r.C;
  }
  r.xp = step < 0 ? r.C : step;
  r.xs = r.N > 1 ? r.x.stride(0) : r.S * r.C;
  return r;
}

void eps_check(double eps) {
  if (!(eps >= 0)) throw py::value_error("GElib: eps is not below zero");
}
void norm_check(const at::Tensor &x, int64_t groups, const Maybe &w, const Maybe &b, const Maybe &lengths) {
  on_gpu(x);
  type_of(x);
  if (x.dim() < 2) throw py::value_error("GElib: x has a batch dimension first and its channels last");
  const int64_t C = x.size(-1);
  if (groups < 1 || C < 1 || C % groups || C > 0x7fffffff) throw py::value_error("GElib: the number of groups divides the number of channels");
  for (auto *t : {&w, &b})
    if (*t) {
      like(**t, x, t == &w ? "weight" : "bias");
      if ((*t)->dim() != 1 || (*t)->size(0) != C) throw py::value_error("GElib: weight and bias have one value a channel");
    }
  if (lengths) {
    if (lengths->scalar_type() != at::kInt) throw py::type_error("GElib: lengths are int32");
    if (lengths->device() != x.device()) throw py::value_error("GElib: lengths are on another device than x");
    if (lengths->dim() != 1 || lengths->size(0) != x.size(0)) throw py::value_error("GElib: one length a sample");
  }
}

std::tuple<at::Tensor, at::Tensor> norm_fwd(const at::Tensor &x, int64_t groups, const Maybe &w, const Maybe &b, double eps,
                                                        const std::string &act, const Maybe &lengths, bool keep) {
  norm_check(x, groups, w, b, lengths);
  const int a = act_of(act);
  eps_check(eps);
  OnDevice on(x);
  NormShape s = norm_shape(x);
  at::Tensor W = w ? plain(*w) : at::Tensor(), B = b ? plain(*b) : at::Tensor(), L = lengths ? lengths->contiguous() : at::Tensor();
  at::Tensor y = at::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous)), stats;
  if (keep) stats = at::empty({2, s.N, groups}, x.options().dtype(at::kFloat));   // mean, rstd
  const uint64_t bytes = gelib_hip_group_norm_act_workspace_bytes(0, type_of(x), s.N, s.S, s.C, (int)groups);
  at::Tensor ws = workspace(bytes, x);
  done(gelib_hip_group_norm_act_fwd(ptr(y), (float *)ptr(stats), ptr(stats) ? (float *)ptr(stats) + s.N * groups : nullptr, ptr(s.x), ptr(W), ptr(B), (int32_t *)ptr(L), type_of(x), s.N, s.S,
                                    s.C, (int)groups, s.xs, s.xp, (float)eps, a, ptr(ws), bytes, on.stream));
  return {y, stats};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> norm_bwd(const at::Tensor &gy_, const at::Tensor &stats, const at::Tensor &x, int64_t groups,
                                         const Maybe &w, const Maybe &b, int act, const Maybe &lengths, bool need_x, bool need_w,
                                         bool need_b) {
  norm_check(x, groups, w, b, lengths);
  OnDevice on(x);
  NormShape s = norm_shape(x);
  at::Tensor gy = plain(gy_), W = w ? plain(*w) : at::Tensor(), B = b ? plain(*b) : at::Tensor(), L = lengths ? lengths->contiguous() : at::Tensor();
  like(gy, x, "the gradient");
  if (gy.sizes() != x.sizes()) throw py::value_error("GElib: the gradient has another shape than x");
  const auto packed = x.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor gx = need_x ? at::empty(x.sizes(), packed) : at::Tensor(), gw = need_w ? at::empty({s.C}, packed) : at::Tensor(),
             gb = need_b ? at::empty({s.C}, packed) : at::Tensor();
  const uint64_t bytes = gelib_hip_group_norm_act_workspace_bytes(1, type_of(x), s.N, s.S, s.C, (int)groups);
  at::Tensor ws = workspace(bytes, x);
  done(gelib_hip_group_norm_act_bwd(ptr(gx), ptr(gw), ptr(gb), ptr(gy), (float *)ptr(stats), ptr(stats) ? (float *)ptr(stats) + s.N * groups : nullptr, ptr(s.x), ptr(W), ptr(B), (int32_t *)ptr(L),
                                    type_of(x), s.N, s.S, s.C, (int)groups, s.xs, s.xp, act, ptr(ws), bytes, on.stream));
  return {gx, gw, gb};
}

// The same from torch's own operations: for gradients of gradients, and where only torch's operations will do.
// (silu as a product: the gradient of torch's silu has no forward-mode derivative)
at::Tensor activated(const at::Tensor &z, int64_t act) {
  return act == GELIB_HIP_ACT_RELU ? at::relu(z) : act == GELIB_HIP_ACT_SILU ? z * at::sigmoid(z) : act == GELIB_HIP_ACT_GELU ? at::gelu(z) : z;
}
at::Tensor norm_from_torch(const at::Tensor &x, const at::Tensor &w, const at::Tensor &b, const at::Tensor &lengths, int64_t groups, double eps, int64_t act) {
  AsWritten types;
  const int64_t n = x.size(0), c = x.size(-1);
  at::Tensor t = x.reshape({n, -1, groups, c / groups}).to(at::kFloat), live, count;
  if (lengths.defined()) {
    const at::Tensor held = lengths.clamp(0, t.size(1));
    live = at::arange(t.size(1), held.options()).lt(held.unsqueeze(1)).view({n, -1, 1, 1});
    count = (held.clamp_min(1).to(at::kLong) * t.size(3)).view({n, 1, 1, 1});   // (2^31 values and more are a large group, not a wrong one)
    t = t.masked_fill(live.logical_not(), 0);
  } else {
    count = at::full({}, (double)t.size(1) * t.size(3), t.options());
  }
  at::Tensor d = t - t.sum({1, 3}, true) / count;
  if (live.defined()) d = d.masked_fill(live.logical_not(), 0);
  t = (d * (d.square().sum({1, 3}, true) / count + eps).rsqrt()).reshape(x.sizes());
  if (w.defined()) t = t * w.to(at::kFloat);
  if (b.defined()) t = t + b.to(at::kFloat);
  t = activated(t, act);
  if (live.defined()) t = t.reshape({n, -1, groups, c / groups}).masked_fill(live.logical_not(), 0).reshape(x.sizes());
  return t.to(x.scalar_type());
}

struct NormFn : torch::autograd::Function<NormFn> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const Maybe &w, const Maybe &b, int64_t groups, double eps, const std::string &act,
                            const Maybe &lengths) {
    auto [y, stats] = norm_fwd(x, groups, w, b, eps, act, lengths, true);
    ctx->save_for_backward({x, some(w), some(b), some(lengths), stats});
    ctx->saved_data["how"] = groups * 4 + act_of(act);
    ctx->saved_data["eps"] = eps;
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &b = saved[2], &lengths = saved[3];
    const int64_t how = ctx->saved_data["how"].toInt(), groups = how / 4, act = how % 4;
    variable_list grads(7);
    if (!g[0].defined()) return grads;
    if (at::GradMode::is_enabled() || left_to_torch({&g[0], &x, &w, &b})) {   // a graph of the gradients is wanted, or their tangents
      const double eps = ctx->saved_data["eps"].toDouble();
      const variable_list got = graph_grads([&](const variable_list &v) { return norm_from_torch(v[0], v[1], v[2], lengths, groups, eps, act); }, {x, w, b}, g[0]);
      std::copy(got.begin(), got.end(), grads.begin());
      return grads;
    }
    size_t at = 0;   // (tensors that were given are counted)
    const bool need_x = ctx->needs_input_grad(at), need_w = w.defined() && ctx->needs_input_grad(++at), need_b = b.defined() && ctx->needs_input_grad(++at);
    auto [gx, gw, gb] = norm_bwd(g[0], saved[4], x, groups, some(w), some(b), (int)act, some(lengths), need_x, need_w, need_b);
    grads[0] = gx, grads[1] = gw, grads[2] = gb;
    return grads;
  }
};

at::Tensor group_norm_act(const at::Tensor &x, int64_t groups, const Maybe &w, const Maybe &b, double eps, const std::string &act, const Maybe &lengths) {
  if (left_to_torch({&x, address(w), address(b), address(lengths)})) {
    norm_check(x, groups, w, b, lengths);
    eps_check(eps);
    return norm_from_torch(x, some(w), some(b), some(lengths), groups, eps, act_of(act));
  }
  if (at::GradMode::is_enabled() && (x.requires_grad() || (w && needs(*w)) || (b && needs(*b)))) {
    norm_check(x, groups, w, b, lengths);   // (refusals come before anything is recorded)
    return NormFn::apply(x, w, b, groups, eps, act, lengths);
  }
  return std::get<0>(norm_fwd(x, groups, w, b, eps, act, lengths, false));
}

// ---- linear layer ----

void linear_check(const at::Tensor &x, const at::Tensor &w) {
  on_gpu(x);
  type_of(x);
  like(w, x, "w");
  if (x.dim() < 1 || w.dim() != 2 || w.size(0) != x.size(-1)) throw py::value_error("GElib: x (..., n_in) and w (n_in, n_out) are needed");
  if (std::max(w.size(0), w.size(1)) > 0x7fffff00) throw py::value_error("GElib: too many channels");
}

// the shape of the result, which bias and residual fit
std::vector<int64_t> linear_shape(const at::Tensor &x, const at::Tensor &w, const Maybe &b, const Maybe &r) {
  linear_check(x, w);
  std::vector<int64_t> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = w.size(1);
  if (b) {
    like(*b, x, "bias");
    if (b->dim() != 1 || b->size(0) != w.size(1)) throw py::value_error("GElib: bias has one value a column of w");
  }
  if (r) {
    like(*r, x, "residual");
    if (r->sizes() != at::IntArrayRef(shape)) throw py::value_error("GElib: residual is shaped like the result");
  }
  return shape;
}

std::tuple<at::Tensor, at::Tensor> linear_fwd(const at::Tensor &x, const at::Tensor &w, const Maybe &b, const Maybe &r, const std::string &act, bool keep) {
  const std::vector<int64_t> shape = linear_shape(x, w, b, r);
  const int a = act_of(act);
  OnDevice on(x);
  Rows X = rows_of(x);
  at::Tensor W = plain(w), B = b ? plain(*b) : at::Tensor(), R = r ? plain(*r) : at::Tensor();
  const auto packed = x.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor y = at::empty(shape, packed), slope;
  if (keep && a != GELIB_HIP_ACT_NONE) slope = at::empty(shape, packed.dtype(x.scalar_type() == at::kFloat ? at::kFloat : at::kHalf));
  const int N = (int)w.size(1);
  const uint64_t bytes = gelib_hip_linear_act_workspace_bytes(0, type_of(x), X.rows, X.K, N);
  at::Tensor ws = workspace(bytes, x);
  done(gelib_hip_linear_act_fwd(ptr(y), ptr(slope), ptr(X.x), ptr(W), ptr(B), ptr(R), type_of(x), X.rows, X.K, N, X.stride, a, ptr(ws), bytes, on.stream));
  return {y, slope};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> linear_bwd(const at::Tensor &gy_, const Maybe &slope, const at::Tensor &x, const at::Tensor &w, bool need_x, bool need_w,
                                           bool need_b) {
  linear_check(x, w);
  OnDevice on(x);
  Rows X = rows_of(x);
  at::Tensor gy = plain(gy_), W = plain(w);
  like(gy, x, "the gradient");
  const int N = (int)w.size(1);
  if (gy.numel() != X.rows * N) throw py::value_error("GElib: the gradient has another shape than the result");
  const auto packed = x.options().memory_format(at::MemoryFormat::Contiguous);
  at::Tensor gx = need_x ? at::empty(x.sizes(), packed) : at::Tensor(), gw = need_w ? at::empty(w.sizes(), packed) : at::Tensor(),
             gb = need_b ? at::empty({N}, packed) : at::Tensor();
  const int what = (ptr(gx) ? 1 : 0) | (ptr(gw) ? 2 : 0) | (ptr(gb) ? 4 : 0) | (slope && slope->numel() ? 8 : 0);
  const uint64_t bytes = gelib_hip_linear_act_workspace_bytes(what, type_of(x), X.rows, X.K, N);
  at::Tensor ws = workspace(bytes, x);
  done(gelib_hip_linear_act_bwd(ptr(gx), ptr(gw), ptr(gb), ptr(gy), slope ? ptr(*slope) : nullptr, ptr(X.x), ptr(W), type_of(x), X.rows, X.K, N, X.stride,
                                ptr(ws), bytes, on.stream));
  return {gx, gw, gb};
}

at::Tensor linear_from_torch(const at::Tensor &x, const at::Tensor &w, const at::Tensor &b, const at::Tensor &r, int64_t act) {
  AsWritten types;
  at::Tensor z = at::matmul(x.to(at::kFloat), w.to(at::kFloat));
  if (b.defined()) z = z + b.to(at::kFloat);
  z = activated(z, act);
  if (r.defined()) z = z + r.to(at::kFloat);
  return z.to(x.scalar_type());
}

// Keeps act'(x w + bias) for the backward pass: the product is not formed again, and nothing else of its size is kept.
struct LinearFn : torch::autograd::Function<LinearFn> {
  static at::Tensor forward(AutogradContext *ctx, const at::Tensor &x, const at::Tensor &w, const Maybe &b, const Maybe &r, const std::string &act) {
    auto [y, slope] = linear_fwd(x, w, b, r, act, true);
    ctx->save_for_backward({x, w, some(b), slope});
    ctx->saved_data["how"] = (int64_t)(act_of(act) * 2 + r.has_value());
    return y;
  }
  static variable_list backward(AutogradContext *ctx, variable_list g) {
    const variable_list saved = ctx->get_saved_variables();
    const at::Tensor &x = saved[0], &w = saved[1], &b = saved[2];
    const int64_t how = ctx->saved_data["how"].toInt(), act = how / 2;
    variable_list grads(5);
    if (!g[0].defined()) return grads;
    size_t at = 1;
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = b.defined() && ctx->needs_input_grad(++at),
               need_r = how % 2 && ctx->needs_input_grad(++at);
    if (need_r) grads[3] = g[0];
    if (!need_x && !need_w && !need_b) return grads;
    if (at::GradMode::is_enabled() || left_to_torch({&g[0], &x, &w, &b})) {   // a graph of the gradients is wanted, or their tangents
      const variable_list got = graph_grads([&](const variable_list &v) { return linear_from_torch(v[0], v[1], v[2], {}, act); }, {x, w, b}, g[0]);
      std::copy(got.begin(), got.end(), grads.begin());
      return grads;
    }
    auto [gx, gw, gb] = linear_bwd(g[0], some(saved[3]), x, w, need_x, need_w, need_b);
    grads[0] = gx, grads[1] = gw, grads[2] = gb;
    return grads;
  }
};

at::Tensor linear_act(const at::Tensor &x, const at::Tensor &w, const Maybe &b, const Maybe &r, const std::string &act) {
  if (left_to_torch({&x, &w, address(b), address(r)})) {
    linear_shape(x, w, b, r);
    return linear_from_torch(x, w, some(b), some(r), act_of(act));
  }
  if (at::GradMode::is_enabled() && (x.requires_grad() || w.requires_grad() || (b && needs(*b)) || (r && needs(*r)))) {
    linear_check(x, w);   // (refusals come before anything is recorded)
    return LinearFn::apply(x, w, b, r, act);
  }
  return std::get<0>(linear_fwd(x, w, b, r, act, false));
}

// ---- AdamW ----

// The parameters of an optimizer that share hyperparameters: where their moments begin in its arrays and the steps each has taken
// (one without a gradient takes none).
struct AdamWGroup {
  std::vector<at::Tensor> params;
  std::vector<int64_t> first, steps, sizes;   // sizes: bytes, which the places were made for

  AdamWGroup(std::vector<at::Tensor> p, std::vector<int64_t> f) : params(std::move(p)), first(std::move(f)), steps(params.size(), 0) {
    if (first.size() != params.size()) throw py::value_error("GElib: one place a parameter");
    for (const at::Tensor &t : params) sizes.push_back(t.nbytes());
  }

  void step(const at::Tensor &m, const at::Tensor &v, const Maybe &mt, const Maybe &vt, int bits, double lr, double beta1, double beta2, double eps,
            double decay, uint64_t seed) {
    struct Lists {
      std::vector<void *> p;
      std::vector<const void *> g;
      std::vector<int64_t> n, first, step;
    } lists[2];   // float32 and complex64, bfloat16
    std::vector<at::Tensor> copies;   // of gradients that are not contiguous
    std::vector<size_t> moved;
    at::NoGradGuard no_grad;
    OnDevice on(m);
    for (size_t k = 0; k < params.size(); k++) {
      const at::Tensor &t = params[k], &grad = t.grad();
      if (!grad.defined() || t.numel() == 0) continue;
      const auto type = t.scalar_type();
      const bool cplx = type == at::kComplexFloat;
      if (!cplx && type != at::kFloat && type != at::kBFloat16) throw py::type_error("GElib: parameters are float32, bfloat16 or complex64");
      if (grad.is_sparse() || grad.scalar_type() != type) throw py::type_error("GElib: a gradient is dense and has its parameter's type");
      if (t.device() != m.device() || grad.device() != m.device()) throw py::value_error("GElib: parameters, gradients and moments are on one GPU");
      if (!t.is_contiguous() || t.is_conj() || t.is_neg()) throw py::value_error("GElib: parameters are contiguous in memory");
      if ((int64_t)t.nbytes() != sizes[k]) throw py::value_error("GElib: a parameter has another size or type than the optimizer was made for");
      if (grad.sizes() != t.sizes()) throw py::value_error("GElib: a gradient is shaped like its parameter");
      const void *g = grad.data_ptr();
      if (!grad.is_contiguous() || grad.is_conj() || grad.is_neg()) {
        copies.push_back(grad.resolve_conj().resolve_neg().contiguous());
        g = copies.back().data_ptr();
      }
      Lists &l = lists[type == at::kBFloat16];
      l.p.push_back(t.data_ptr());
      l.g.push_back(g);
      l.n.push_back(t.numel() * (cplx ? 2 : 1));
      l.first.push_back(first[k]);
      l.step.push_back(steps[k] + 1);
      moved.push_back(k);
    }
    for (int b = 1; b >= 0; b--)   // (bfloat16 first: where it is refused nothing has been launched)
      if (Lists &l = lists[b]; !l.p.empty()) {
        const int status = gelib_hip_adamw_step((int)l.p.size(), l.p.data(), l.g.data(), l.n.data(), l.first.data(), l.step.data(), ptr(m), ptr(v),
                                  mt ? (int16_t *)ptr(*mt) : nullptr, vt ? (int16_t *)ptr(*vt) : nullptr, b ? GELIB_HIP_BF16 : GELIB_HIP_F32, bits, lr,
                                  beta1, beta2, eps, decay, seed, on.stream);
        if (status == GELIB_HIP_ERR_UNSUPPORTED)
          throw std::runtime_error("GElib: a step with moments in 8 bits or bfloat16 parameters cannot be recorded into a graph: every replay would round by the "
                                   "same random bits");
        done(status);
      }
    for (size_t k : moved) {
      steps[k]++;
      params[k].unsafeGetTensorImpl()->bump_version();   // (changed in place, as far as autograd is concerned)
    }
  }
};

std::tuple<at::Tensor, at::Tensor> adamw_moments(const at::Tensor &m, const at::Tensor &v, const at::Tensor &mt, const at::Tensor &vt) {
  OnDevice on(m);
  at::Tensor a = at::empty(m.sizes(), m.options().dtype(at::kBFloat16)), b = at::empty_like(a);
  done(gelib_hip_adamw_moments(ptr(a), ptr(b), ptr(m), ptr(v), (int16_t *)ptr(mt), (int16_t *)ptr(vt), m.numel(), on.stream));
  return {a, b};
}

void adamw_set_moments(const at::Tensor &m, const at::Tensor &v, const at::Tensor &mt, const at::Tensor &vt, const at::Tensor &a, const at::Tensor &b) {
  OnDevice on(m);
  TORCH_CHECK(a.scalar_type() == at::kFloat && b.scalar_type() == at::kFloat && a.numel() == m.numel() && b.numel() == m.numel() && a.device() == m.device() &&
              b.device() == m.device() && a.is_contiguous() && b.is_contiguous(), "GElib: moments are given as float32, one an element");
  done(gelib_hip_adamw_set_moments(ptr(m), ptr(v), (int16_t *)ptr(mt), (int16_t *)ptr(vt), (float *)ptr(a), (float *)ptr(b), m.numel(), on.stream));
}

}  // namespace

void bind_real_ops(pybind11::module_ &m) {
  m.def("group_norm_act", &group_norm_act);
  m.def("linear_act", &linear_act);
  py::class_<AdamWGroup>(m, "AdamWGroup", "Parameters of one AdamW step, with the places of their moments")
      .def(py::init<std::vector<at::Tensor>, std::vector<int64_t>>())
      .def("step", &AdamWGroup::step)
      .def_property("steps", [](const AdamWGroup &g) { return g.steps; },
                    [](AdamWGroup &g, std::vector<int64_t> s) {
                      if (s.size() != g.params.size()) throw py::value_error("GElib: one number of steps a parameter");
                      g.steps = std::move(s);
                    });
  m.def("adamw_moments", &adamw_moments);
  m.def("adamw_set_moments", &adamw_set_moments);
}
