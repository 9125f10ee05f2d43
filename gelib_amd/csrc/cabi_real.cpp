// C entry points of the operators on real channels: checks of their arguments, then one launcher each.  Nothing is launched
// unless every pointer is device memory of the current GPU and long enough.
#include <cmath>
#include <new>
#include <vector>

#include "real_ops.h"

using namespace gelib_hip;

namespace {

constexpr int64_t kMostElements = 1LL << 46;   // of one tensor: products of two extents below it do not overflow

bool types_ok(int dtype, int act) { return dtype >= GELIB_HIP_F32 && dtype <= GELIB_HIP_F16 && act >= GELIB_HIP_ACT_NONE && act <= GELIB_HIP_ACT_GELU; }

// both factors are not below zero
bool product_ok(int64_t a, int64_t b) { return a == 0 || b <= kMostElements / a; }

int check_workspace(const void *ws, uint64_t have, uint64_t need) {
  if (need == 0) return GELIB_HIP_OK;
  if (!ws || have < need || ((uintptr_t)ws & 15)) return GELIB_HIP_ERR_WORKSPACE;
  return check_memory(ws, (int64_t)need);
}

// Collects the first refusal: missing pointers before memory that is not the device's.
struct Memory {
  int missing = GELIB_HIP_OK, foreign = GELIB_HIP_OK;
  void need(const void *p, int64_t bytes, unsigned align) {
    if (bytes == 0 || missing) return;
    if (!p) missing = GELIB_HIP_ERR_NULL;
    else if ((uintptr_t)p % align) missing = GELIB_HIP_ERR_ARG;
    else if (!foreign) foreign = check_memory(p, bytes);
  }
  void may(const void *p, int64_t bytes, unsigned align) {
    if (p) need(p, bytes, align);
  }
  int rc() const { return missing ? missing : foreign; }
};

int norm_shape(int dtype, int act, int64_t N, int64_t S, int C, int G, int64_t xs, int64_t xp) {
  if (!types_ok(dtype, act) || N < 0 || S < 0 || C < 1 || C > (1 << 26) || G < 1 || C % G || xs < 0 || xp < 0) return GELIB_HIP_ERR_ARG;
  if (!product_ok(N, S) || !product_ok(N * S, C) || N > (1LL << 40) / G || !product_ok(N, xs) || !product_ok(S, xp)) return GELIB_HIP_ERR_ARG;
  return GELIB_HIP_OK;
}

// what rows of `cols` elements are aligned to: 16 bytes where they are a multiple of it long
unsigned row_align(unsigned e, int64_t cols) { return cols * e % 16 == 0 ? 16 : e; }

int linear_shape(int dtype, int act, int64_t rows, int K, int N, int64_t xs) {
  if (!types_ok(dtype, act) || rows < 0 || K < 0 || N < 0 || xs < 0 || std::max(K, N) > kLinearMostChannels) return GELIB_HIP_ERR_ARG;
  if (!product_ok(rows, K) || !product_ok(rows, N) || !product_ok(rows, xs)) return GELIB_HIP_ERR_ARG;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  if (rows > 1 && xs * e % row_align(e, K) != 0) return GELIB_HIP_ERR_ARG;
  return GELIB_HIP_OK;
}

}  // namespace

extern "C" {

uint64_t gelib_hip_group_norm_act_workspace_bytes(int backward, int dtype, int64_t samples, int64_t positions, int channels, int groups) {
  if (norm_shape(dtype, 0, samples, positions, channels, groups, 0, 0)) return 0;
  return norm_workspace(backward != 0, dtype, samples, positions, channels, groups);
}

int gelib_hip_group_norm_act_fwd(void *y, float *mean, float *rstd, const void *x, const void *weight, const void *bias, const int32_t *lengths,
                                 int dtype, int64_t samples, int64_t positions, int channels, int groups, int64_t x_sample_stride,
                                 int64_t x_position_stride, float eps, int act, void *workspace, uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (int rc = norm_shape(dtype, act, samples, positions, channels, groups, x_sample_stride, x_position_stride)) return rc;
  if (!(eps >= 0.f) || !mean != !rstd) return GELIB_HIP_ERR_ARG;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  const int64_t all = samples * positions * channels * e;
  Memory mem;
  if (all) mem.need(x, ((samples - 1) * x_sample_stride + (positions - 1) * x_position_stride + channels) * e, e);
  mem.need(y, all, e);
  mem.may(weight, (int64_t)channels * e, e);
  mem.may(bias, (int64_t)channels * e, e);
  mem.may(lengths, samples * 4, 4);
  mem.may(mean, samples * groups * 4, 4);
  mem.may(rstd, samples * groups * 4, 4);
  if (int rc = mem.rc()) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, norm_workspace(false, dtype, samples, positions, channels, groups))) return rc;
  NormArgs a = {};
  a.y = y, a.x = x, a.w = weight, a.b = bias, a.lengths = lengths, a.mean = mean, a.rstd = rstd;
  a.N = samples, a.S = positions, a.xs = x_sample_stride, a.xp = x_position_stride;
  a.C = channels, a.G = groups, a.act = act, a.eps = eps, a.ws = workspace;
  set_last_path(kPathReal);
  return launch_norm(false, dtype, a, (hipStream_t)stream);
}

int gelib_hip_group_norm_act_bwd(void *gx, void *gw, void *gb, const void *gy, const float *mean, const float *rstd, const void *x,
                                 const void *weight, const void *bias, const int32_t *lengths, int dtype, int64_t samples, int64_t positions,
                                 int channels, int groups, int64_t x_sample_stride, int64_t x_position_stride, int act, void *workspace,
                                 uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (int rc = norm_shape(dtype, act, samples, positions, channels, groups, x_sample_stride, x_position_stride)) return rc;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  const int64_t all = samples * positions * channels * e;
  Memory mem;
  if (all) mem.need(x, ((samples - 1) * x_sample_stride + (positions - 1) * x_position_stride + channels) * e, e);
  mem.need(gy, all, e);
  mem.may(gx, all, e);
  for (const void *p : {weight, bias, (const void *)gw, (const void *)gb}) mem.may(p, (int64_t)channels * e, e);
  mem.may(lengths, samples * 4, 4);
  if (all) mem.need(mean, samples * groups * 4, 4), mem.need(rstd, samples * groups * 4, 4);
  if (int rc = mem.rc()) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, norm_workspace(true, dtype, samples, positions, channels, groups))) return rc;
  NormArgs a = {};
  a.y = gx, a.x = x, a.gy = gy, a.w = weight, a.b = bias, a.lengths = lengths, a.mean = (float *)mean, a.rstd = (float *)rstd, a.gw = gw, a.gb = gb;
  a.N = samples, a.S = positions, a.xs = x_sample_stride, a.xp = x_position_stride;
  a.C = channels, a.G = groups, a.act = act, a.ws = workspace;
  set_last_path(kPathReal);
  return launch_norm(true, dtype, a, (hipStream_t)stream);
}

uint64_t gelib_hip_linear_act_workspace_bytes(int backward, int dtype, int64_t rows, int n_in, int n_out) {
  if (backward < 0 || backward > 15 || linear_shape(dtype, 0, rows, n_in, n_out, 0)) return 0;
  return linear_workspace(backward, dtype, rows, n_in, n_out);
}

int gelib_hip_linear_act_fwd(void *y, void *slope, const void *x, const void *w, const void *bias, const void *residual, int dtype, int64_t rows,
                             int n_in, int n_out, int64_t x_row_stride, int act, void *workspace, uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (int rc = linear_shape(dtype, act, rows, n_in, n_out, x_row_stride)) return rc;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  const int64_t out = rows * n_out;
  Memory mem;
  mem.need(y, out * e, e);
  if (act != GELIB_HIP_ACT_NONE) mem.may(slope, out * e, e);   // (as wide as the layer's type)
  if (out && n_in) mem.need(x, ((rows - 1) * x_row_stride + n_in) * e, row_align(e, n_in)), mem.need(w, (int64_t)n_in * n_out * e, row_align(e, n_out));
  mem.may(bias, (int64_t)n_out * e, e);
  mem.may(residual, out * e, e);
  if (int rc = mem.rc()) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, linear_workspace(0, dtype, rows, n_in, n_out))) return rc;
  LinearArgs a = {};
  a.y = y, a.slope = act == GELIB_HIP_ACT_NONE ? nullptr : slope, a.x = x, a.w = w, a.b = bias, a.r = residual;
  a.rows = rows, a.xs = x_row_stride, a.K = n_in, a.N = n_out, a.act = act, a.ws = workspace;
  set_last_path(kPathReal);
  return launch_linear_fwd(dtype, a, (hipStream_t)stream);
}

int gelib_hip_linear_act_bwd(void *gx, void *gw, void *gb, const void *gy, const void *slope, const void *x, const void *w, int dtype, int64_t rows,
                             int n_in, int n_out, int64_t x_row_stride, void *workspace, uint64_t workspace_bytes, void *stream) {
  set_last_path(kPathNone);
  if (int rc = linear_shape(dtype, 0, rows, n_in, n_out, x_row_stride)) return rc;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  const int64_t out = rows * n_out;
  Memory mem;
  mem.need(gy, out * e, row_align(e, n_out));
  mem.may(slope, out * e, e);
  mem.may(gx, rows * n_in * e, e);
  mem.may(gw, (int64_t)n_in * n_out * e, e);
  mem.may(gb, (int64_t)n_out * e, e);
  if (gx && rows && n_in) mem.need(w, (int64_t)n_in * n_out * e, row_align(e, n_out));
  if (gw && out && n_in) mem.need(x, ((rows - 1) * x_row_stride + n_in) * e, row_align(e, n_in));
  if (int rc = mem.rc()) return rc;
  const int what = (gx ? 1 : 0) | (gw ? 2 : 0) | (gb ? 4 : 0) | (slope ? 8 : 0);
  if (int rc = check_workspace(workspace, workspace_bytes, linear_workspace(what, dtype, rows, n_in, n_out))) return rc;
  LinearArgs a = {};
  a.slope = (void *)slope, a.x = x, a.w = w, a.gy = gy, a.gx = gx, a.gw = gw, a.gb = gb;
  a.rows = rows, a.xs = x_row_stride, a.K = n_in, a.N = n_out, a.ws = workspace;
  set_last_path(kPathReal);
  return launch_linear_bwd(dtype, a, (hipStream_t)stream);
}

int gelib_hip_adamw_step(int ntensors, void *const *p, const void *const *g, const int64_t *n, const int64_t *first, const int64_t *step, void *m,
                         void *v, int16_t *m_top, int16_t *v_top, int dtype, int state_bits, double lr, double beta1, double beta2, double eps,
                         double weight_decay, uint64_t seed, void *stream) {
  set_last_path(kPathNone);
  if (ntensors < 0 || (dtype != GELIB_HIP_F32 && dtype != GELIB_HIP_BF16) || (state_bits != 8 && state_bits != 32)) return GELIB_HIP_ERR_ARG;
  if (!(beta1 >= 0 && beta1 < 1 && beta2 >= 0 && beta2 < 1 && eps >= 0) || !std::isfinite(lr) || !std::isfinite(weight_decay)) return GELIB_HIP_ERR_ARG;
  if (ntensors == 0) return GELIB_HIP_OK;
  if (!p || !g || !n || !first || !step) return GELIB_HIP_ERR_NULL;
  const unsigned e = (unsigned)dtype_bytes(dtype);
  Memory mem;
  int64_t end = 0;
  for (int k = 0; k < ntensors; k++) {
    if (n[k] < 0 || first[k] < 0 || first[k] % kAdamBlock || step[k] < 1) return GELIB_HIP_ERR_ARG;
    if (n[k] > (1LL << 39) || first[k] > (1LL << 39)) return GELIB_HIP_ERR_ARG;   // (blocks of 256 are counted in 32 bits)
    mem.need(p[k], n[k] * e, e);
    mem.need(g[k], n[k] * e, e);
    if (n[k]) end = std::max(end, first[k] + (n[k] + kAdamBlock - 1) / kAdamBlock * kAdamBlock);
  }
  const unsigned s = state_bits / 8;
  mem.need(m, end * s, 16);
  mem.need(v, end * s, 16);
  if (state_bits == 8) mem.need(m_top, end / kAdamBlock * 2, 2), mem.need(v_top, end / kAdamBlock * 2, 2);
  if (int rc = mem.rc()) return rc;
  if (end == 0) return GELIB_HIP_OK;
  if (state_bits == 8 || dtype == GELIB_HIP_BF16) {
    hipStreamCaptureStatus recorded = hipStreamCaptureStatusNone;
    if (hipStreamIsCapturing((hipStream_t)stream, &recorded) != hipSuccess) (void)hipGetLastError();
    if (recorded != hipStreamCaptureStatusNone) return GELIB_HIP_ERR_UNSUPPORTED;   // every replay would round by the same random bits
  }
  AdamArgs a;
  a.m = m, a.v = v, a.m_top = m_top, a.v_top = v_top, a.dtype = dtype, a.bits = state_bits;
  a.decay = (float)(lr * weight_decay);
  a.b1 = (float)beta1, a.c1 = (float)(1 - beta1), a.b2 = (float)beta2, a.c2 = (float)(1 - beta2);
  a.eps = (float)eps;
  AdamTensor t = {};
  int64_t of = 0;   // the step that t's numbers belong to (nearly always the same for all)
  try {
    std::vector<AdamTensor> table;
    table.reserve(ntensors);
    for (int k = 0; k < ntensors; k++) {
      if (step[k] != of) {
        of = step[k];
        t.step_size = (float)(lr / (1 - std::pow(beta1, (double)of)));
        t.inv_sqrt_bc2 = (float)(1 / std::sqrt(1 - std::pow(beta2, (double)of)));
        t.key = (unsigned)seed * 3144134277u + (unsigned)(seed >> 32) * 2654435769u + (unsigned)of * 1779033703u;
      }
      t.p = p[k], t.g = g[k], t.n = n[k], t.first = first[k];
      table.push_back(t);
    }
    set_last_path(kPathReal);
    return launch_adamw(ntensors, table.data(), a, (hipStream_t)stream);
  } catch (const std::bad_alloc &) {
    return GELIB_HIP_ERR_ARG;
  }
}

static int check_moments(const void *mv, const void *vv, const void *m, const void *v, const int16_t *mt, const int16_t *vt, int64_t n, unsigned e) {
  set_last_path(kPathNone);
  if (n < 0 || n % kAdamBlock) return GELIB_HIP_ERR_ARG;
  if (n > (1LL << 40)) return GELIB_HIP_ERR_ARG;
  Memory mem;
  mem.need(mv, n * e, 16), mem.need(vv, n * e, 16);
  mem.need(m, n, 16), mem.need(v, n, 16);
  mem.need(mt, n / kAdamBlock * 2, 2), mem.need(vt, n / kAdamBlock * 2, 2);
  return mem.rc();
}

int gelib_hip_adamw_moments(void *m_values, void *v_values, const void *m, const void *v, const int16_t *m_top, const int16_t *v_top, int64_t n,
                            void *stream) {
  if (int rc = check_moments(m_values, v_values, m, v, m_top, v_top, n, 2)) return rc;
  set_last_path(kPathReal);
  return launch_adamw_moments(m_values, v_values, m, v, m_top, v_top, n, (hipStream_t)stream);
}

int gelib_hip_adamw_set_moments(void *m, void *v, int16_t *m_top, int16_t *v_top, const float *m_values, const float *v_values, int64_t n,
                                void *stream) {
  if (int rc = check_moments(m_values, v_values, m, v, m_top, v_top, n, 4)) return rc;
  set_last_path(kPathReal);
  return launch_adamw_set_moments(m, v, m_top, v_top, m_values, v_values, n, (hipStream_t)stream);
}

}  // extern "C"
