// C ABI of the operators around the attention call: argument validation and launch.
// Nothing here allocates device memory or synchronises; every launch goes to the caller's stream.
#include "../../include/xdit_amd_attn.h"

#include <algorithm>
#include <cmath>
#include <cstring>

#include "api_error.h"
#include "block_params.h"

namespace {

using xdit::api_fail;

bool multiple_of(const void* p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

bool float_dtype(int d) { return d == XDIT_DTYPE_BF16 || d == XDIT_DTYPE_FP16 || d == XDIT_DTYPE_FP32; }
int size_of(int d) { return d == XDIT_DTYPE_FP32 ? 4 : 2; }

// Whether no two rows of `C` elements share one: going from the smallest stride up, each has to step over all that those below it reach.
struct Axis { int64_t n, stride; };
template <int N>
bool rows_apart(int64_t C, Axis (&axes)[N]) {
  std::sort(axes, axes + N, [](const Axis& a, const Axis& b) { return a.stride < b.stride; });
  __int128 reach = C;
  for (const Axis& a : axes) {
    if (a.n <= 1) continue;
    if (a.stride < reach) return false;
    reach += (__int128)a.stride * (a.n - 1);
  }
  return true;
}

// A (B, S, C) tensor whose rows are read or written 8 elements at a time.  `written`: rows must not overlap.
int check_rows(const char* name, const void* p, const xdit_row_strides& st, int esize, int64_t B, int64_t S, int64_t C, bool written) {
  if (p == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "%s is NULL", name);
  const unsigned align = esize == 1 ? 8 : 16;
  const int64_t m = align / esize;
  if (!multiple_of(p, align)) return api_fail(XDIT_ERR_INVALID_ARG, "%s is not %u-byte aligned", name, align);
  if ((B > 1 && st.b % m) || (S > 1 && st.s % m))
    return api_fail(XDIT_ERR_INVALID_ARG, "%s: strides (%lld,%lld) must be multiples of %lld elements", name, (long long)st.b, (long long)st.s, (long long)m);
  if (st.b < 0 || st.s < 0) return api_fail(XDIT_ERR_INVALID_ARG, "%s: negative stride", name);
  Axis axes[] = {{B, st.b}, {S, st.s}};
  if (written && !rows_apart(C, axes))
    return api_fail(XDIT_ERR_INVALID_ARG, "%s: strides (%lld,%lld) make its rows of %lld overlap", name, (long long)st.b, (long long)st.s, (long long)C);
  return 0;
}

int check_vector(const char* name, const void* p) {
  if (p != nullptr && !multiple_of(p, 16)) return api_fail(XDIT_ERR_INVALID_ARG, "%s is not 16-byte aligned", name);
  return 0;
}

// What both directions of the gated norm share.
int check_norm_problem(int dtype, int mod_dtype, int weight_dtype, int norm, int y_norm, int B, int C, int64_t S, float alpha) {
  if (!float_dtype(dtype)) return api_fail(XDIT_ERR_INVALID_ARG, "dtype %d must be bf16, fp16 or fp32", dtype);
  if (mod_dtype != dtype && mod_dtype != XDIT_DTYPE_FP32) return api_fail(XDIT_ERR_INVALID_ARG, "mod_dtype %d must be dtype or fp32", mod_dtype);
  if (weight_dtype != dtype && weight_dtype != XDIT_DTYPE_FP32) return api_fail(XDIT_ERR_INVALID_ARG, "weight_dtype %d must be dtype or fp32", weight_dtype);
  if (norm < XDIT_ROWNORM_NONE || norm > XDIT_ROWNORM_LAYER || y_norm < XDIT_ROWNORM_NONE || y_norm > XDIT_ROWNORM_LAYER)
    return api_fail(XDIT_ERR_INVALID_ARG, "unknown norm %d or y_norm %d", norm, y_norm);
  if (B <= 0 || S <= 0 || C <= 0) return api_fail(XDIT_ERR_INVALID_ARG, "B, S, C must be positive");
  if (B > 65535 || S > (int64_t(1) << 30) || B * S > 0x7fffffffLL) return api_fail(XDIT_ERR_INVALID_ARG, "too many rows for one launch");
  if (C % 8 != 0 || C > xdit::kNormMaxC) return api_fail(XDIT_ERR_UNSUPPORTED, "C = %d: need a multiple of 8, at most %d", C, xdit::kNormMaxC);
  if (!std::isfinite(alpha)) return api_fail(XDIT_ERR_INVALID_ARG, "residual_scale must be finite");
  return 0;
}

xdit::RowStrides rs(const xdit_row_strides& s) { return {s.b, s.s}; }

}  // namespace

extern "C" {

int xdit_gated_norm(const xdit_gated_norm_args* a) {
  xdit::api_clear_error();
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_gated_norm_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_gated_norm_args));
  int rc = check_norm_problem(a->dtype, a->mod_dtype, a->weight_dtype, a->norm, a->y_norm, a->B, a->C, a->S, a->residual_scale);
  if (rc) return rc;
  const int es = size_of(a->dtype), ms = size_of(a->mod_dtype);
  const int64_t B = a->B, S = a->S, C = a->C;
  if ((rc = check_rows("x", a->x, a->x_stride, es, B, S, C, false))) return rc;
  if (a->y != nullptr && (rc = check_rows("y", a->y, a->y_stride, es, B, S, C, false))) return rc;
  if (a->h != nullptr && (rc = check_rows("h", a->h, a->h_stride, es, B, S, C, true))) return rc;
  if (a->y == nullptr && (a->gate != nullptr || a->y_weight != nullptr || a->y_norm != XDIT_ROWNORM_NONE))
    return api_fail(XDIT_ERR_INVALID_ARG, "gate, y_weight and y_norm need y");
  if (a->norm == XDIT_ROWNORM_NONE) {
    if (a->h == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "without a norm there is only h to write, and h is NULL");
    if (a->weight != nullptr || a->bias != nullptr || a->scale != nullptr || a->shift != nullptr || a->fp8)
      return api_fail(XDIT_ERR_INVALID_ARG, "weight, bias, scale, shift and fp8 need a norm");
  } else if ((rc = check_rows("n", a->n, a->n_stride, a->fp8 ? 1 : es, B, S, C, true))) {
    return rc;
  }
  if (a->fp8 && (a->n_scale == nullptr || !multiple_of(a->n_scale, 4))) return api_fail(XDIT_ERR_INVALID_ARG, "n_scale is NULL or not 4-byte aligned");
  if ((a->norm != XDIT_ROWNORM_NONE && !(a->eps >= 0.f && std::isfinite(a->eps))) || (a->y_norm != XDIT_ROWNORM_NONE && !(a->y_eps >= 0.f && std::isfinite(a->y_eps))))
    return api_fail(XDIT_ERR_INVALID_ARG, "eps must be finite and >= 0");
  if (a->gate != nullptr && (rc = check_rows("gate", a->gate, a->gate_stride, ms, B, S, C, false))) return rc;
  if (a->scale != nullptr && (rc = check_rows("scale", a->scale, a->scale_stride, ms, B, S, C, false))) return rc;
  if (a->shift != nullptr && (rc = check_rows("shift", a->shift, a->shift_stride, ms, B, S, C, false))) return rc;
  if ((rc = check_vector("weight", a->weight)) || (rc = check_vector("bias", a->bias)) || (rc = check_vector("y_weight", a->y_weight)) ||
      (rc = check_vector("stats", a->stats)))
    return rc;
  xdit::GatedNormParams p;
  std::memset(&p, 0, sizeof(p));
  p.x = a->x; p.y = a->y; p.h = a->h; p.n = a->n; p.n_scale = a->n_scale; p.stats = a->stats;
  p.gate = a->gate; p.scale = a->scale; p.shift = a->shift; p.weight = a->weight; p.bias = a->bias; p.y_weight = a->y_weight;
  p.xs = rs(a->x_stride); p.ys = rs(a->y_stride); p.hs = rs(a->h_stride); p.ns = rs(a->n_stride);
  p.gs = rs(a->gate_stride); p.ss = rs(a->scale_stride); p.fs = rs(a->shift_stride);
  p.B = a->B; p.S = (int)S; p.C = a->C; p.rows = B * S;
  p.norm = a->norm; p.y_norm = a->y_norm; p.fp8 = a->fp8 != 0;
  p.mod_wide = a->mod_dtype == XDIT_DTYPE_FP32; p.weight_wide = a->weight_dtype == XDIT_DTYPE_FP32;
  p.eps = a->eps; p.y_eps = a->y_eps; p.alpha = a->residual_scale; p.inv_c = 1.0f / (float)C;
  const hipError_t e = xdit::launch_gated_norm(p, a->dtype, (hipStream_t)a->stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "gated norm launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

static int fill_norm_backward(const xdit_gated_norm_backward_args* a, xdit::GatedNormBwdParams& p, bool pointers) {
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_gated_norm_backward_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_gated_norm_backward_args));
  int rc = check_norm_problem(a->dtype, a->mod_dtype, a->weight_dtype, a->norm, a->y_norm, a->B, a->C, a->S, a->residual_scale);
  if (rc) return rc;
  std::memset(&p, 0, sizeof(p));
  p.dh = a->dh; p.dn = a->dn; p.h = a->h; p.y = a->y; p.stats = a->stats;
  p.gate = a->gate; p.scale = a->scale; p.weight = a->weight; p.bias = a->bias; p.y_weight = a->y_weight;
  p.dx = a->dx; p.dy = a->dy; p.dgate = a->dgate; p.dscale = a->dscale; p.dshift = a->dshift;
  p.dweight = a->dweight; p.dbias = a->dbias; p.dy_weight = a->dy_weight;
  p.dhs = rs(a->dh_stride); p.dns = rs(a->dn_stride); p.hs = rs(a->h_stride); p.ys = rs(a->y_stride);
  p.gs = rs(a->gate_stride); p.ss = rs(a->scale_stride); p.dxs = rs(a->dx_stride); p.dys = rs(a->dy_stride);
  p.B = a->B; p.S = (int)a->S; p.C = a->C;
  p.norm = a->norm; p.y_norm = a->y_norm;
  p.mod_wide = a->mod_dtype == XDIT_DTYPE_FP32; p.weight_wide = a->weight_dtype == XDIT_DTYPE_FP32;
  p.gate_per_token = a->gate_per_token != 0; p.mod_per_token = a->mod_per_token != 0;
  p.alpha = a->residual_scale; p.inv_c = 1.0f / (float)a->C;
  xdit::gated_norm_bwd_plan(p);
  if (!pointers) return 0;
  const int es = size_of(a->dtype), ms = size_of(a->mod_dtype);
  const int64_t B = a->B, S = a->S, C = a->C;
  if (a->dh == nullptr && a->dn == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "dh and dn are both NULL");
  if (a->dh != nullptr && (rc = check_rows("dh", a->dh, a->dh_stride, es, B, S, C, false))) return rc;
  if (a->stats == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "stats is NULL");
  if (a->dn != nullptr) {
    if (a->norm == XDIT_ROWNORM_NONE) return api_fail(XDIT_ERR_INVALID_ARG, "dn needs a norm");
    if ((rc = check_rows("dn", a->dn, a->dn_stride, es, B, S, C, false))) return rc;
    if ((rc = check_rows("h", a->h, a->h_stride, es, B, S, C, false))) return rc;
  } else if (a->dscale != nullptr || a->dshift != nullptr || a->dweight != nullptr || a->dbias != nullptr) {
    return api_fail(XDIT_ERR_INVALID_ARG, "dscale, dshift, dweight and dbias need dn");
  }
  if (a->y != nullptr) {
    if ((rc = check_rows("y", a->y, a->y_stride, es, B, S, C, false))) return rc;
  } else if (a->dy != nullptr || a->dgate != nullptr || a->dy_weight != nullptr) {
    return api_fail(XDIT_ERR_INVALID_ARG, "dy, dgate and dy_weight need y");
  }
  if (a->dx != nullptr && (rc = check_rows("dx", a->dx, a->dx_stride, es, B, S, C, true))) return rc;
  if (a->dy != nullptr && (rc = check_rows("dy", a->dy, a->dy_stride, es, B, S, C, true))) return rc;
  if (a->gate != nullptr && (rc = check_rows("gate", a->gate, a->gate_stride, ms, B, a->gate_per_token ? S : 1, C, false))) return rc;
  if (a->scale != nullptr && (rc = check_rows("scale", a->scale, a->scale_stride, ms, B, a->mod_per_token ? S : 1, C, false))) return rc;
  if (!a->gate_per_token) p.gs.s = 0;
  if (!a->mod_per_token) p.ss.s = 0;
  const struct { const char* name; const void* p; } vec[] = {{"weight", a->weight}, {"bias", a->bias}, {"y_weight", a->y_weight}, {"stats", a->stats},
      {"dgate", a->dgate}, {"dscale", a->dscale}, {"dshift", a->dshift}, {"dweight", a->dweight}, {"dbias", a->dbias}, {"dy_weight", a->dy_weight}};
  for (const auto& v : vec)
    if ((rc = check_vector(v.name, v.p))) return rc;
  return 0;
}

static int64_t norm_backward_bytes(const xdit::GatedNormBwdParams& p) { return p.sums ? (int64_t)p.B * p.parts * 3 * p.C * 4 : 0; }

int64_t xdit_gated_norm_backward_workspace_bytes(const xdit_gated_norm_backward_args* a) {
  xdit::api_clear_error();
  xdit::GatedNormBwdParams p;
  const int rc = fill_norm_backward(a, p, false);
  return rc ? rc : norm_backward_bytes(p);
}

int xdit_gated_norm_backward(const xdit_gated_norm_backward_args* a) {
  xdit::api_clear_error();
  xdit::GatedNormBwdParams p;
  if (int rc = fill_norm_backward(a, p, true)) return rc;
  const int64_t need = norm_backward_bytes(p);
  if (need > 0 && (a->workspace == nullptr || !multiple_of(a->workspace, 16) || a->workspace_bytes < need))
    return api_fail(XDIT_ERR_INVALID_ARG, "workspace of %lld bytes (16-byte aligned) is needed, %lld given", (long long)need, (long long)a->workspace_bytes);
  p.partial = (float*)a->workspace;
  const hipError_t e = xdit::launch_gated_norm_bwd(p, a->dtype, (hipStream_t)a->stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "gated norm backward launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

static int fill_axes_rope(const xdit_axes_rope_args* a, xdit::AxesRopeParams& p, bool backward, bool pointers) {
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_axes_rope_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_axes_rope_args));
  if (!float_dtype(a->dtype)) return api_fail(XDIT_ERR_INVALID_ARG, "dtype %d must be bf16, fp16 or fp32", a->dtype);
  if (a->weight_dtype != a->dtype && a->weight_dtype != XDIT_DTYPE_FP32) return api_fail(XDIT_ERR_INVALID_ARG, "weight_dtype %d must be dtype or fp32", a->weight_dtype);
  if (a->rope != XDIT_ROPE_INTERLEAVED && a->rope != XDIT_ROPE_SPLIT_HALF) return api_fail(XDIT_ERR_INVALID_ARG, "rope %d must be interleaved or split_half", a->rope);
  if (a->pos_bits != -32 && a->pos_bits != 32 && a->pos_bits != 64) return api_fail(XDIT_ERR_INVALID_ARG, "pos_bits %d must be -32 (fp32), 32 or 64", a->pos_bits);
  if (a->freq_bits != 32 && a->freq_bits != 64) return api_fail(XDIT_ERR_INVALID_ARG, "freq_bits %d must be 32 or 64", a->freq_bits);
  if (a->B <= 0 || a->S <= 0) return api_fail(XDIT_ERR_INVALID_ARG, "B and S must be positive");
  if (a->S > (int64_t(1) << 30) || (int64_t)a->B * a->S > 0x7fffffffLL) return api_fail(XDIT_ERR_INVALID_ARG, "too many tokens for one launch");
  if (a->D <= 0 || a->D % 8 != 0 || a->D > 512) return api_fail(XDIT_ERR_UNSUPPORTED, "head_dim %d: need a multiple of 8, at most 512", a->D);
  if (a->tensors != 1 && a->tensors != 2) return api_fail(XDIT_ERR_INVALID_ARG, "tensors %d must be 1 or 2", a->tensors);
  if (a->axes < 1 || a->axes > XDIT_ROPE_MAX_AXES) return api_fail(XDIT_ERR_INVALID_ARG, "axes %d must be between 1 and %d", a->axes, XDIT_ROPE_MAX_AXES);
  if (a->norm && !(a->eps >= 0.f && std::isfinite(a->eps))) return api_fail(XDIT_ERR_INVALID_ARG, "eps must be finite and >= 0");
  std::memset(&p, 0, sizeof(p));
  int64_t P = 0;
  for (int i = 0; i < XDIT_ROPE_MAX_AXES; i++) {
    if (i < a->axes) {
      if (a->pairs[i] < 0 || a->pairs[i] > a->D) return api_fail(XDIT_ERR_INVALID_ARG, "pairs[%d] = %d is out of range", i, a->pairs[i]);
      P += a->pairs[i];
    }
    p.axis_end[i] = (int)P;
  }
  if (2 * P > a->D) return api_fail(XDIT_ERR_INVALID_ARG, "%lld pairs do not fit head_dim %d", (long long)P, a->D);
  if (P % 4 != 0) return api_fail(XDIT_ERR_UNSUPPORTED, "%lld rotated pairs: need a multiple of 4", (long long)P);
  p.P = (int)P;
  p.tensors = a->tensors; p.B = a->B; p.S = (int)a->S; p.D = a->D; p.axes = a->axes;
  p.split_half = a->rope == XDIT_ROPE_SPLIT_HALF; p.norm = a->norm != 0;
  p.pos_bits = a->pos_bits; p.freq_wide = a->freq_bits == 64; p.weight_wide = a->weight_dtype == XDIT_DTYPE_FP32;
  p.positions = a->positions; p.ps_b = a->pos_stride_b; p.ps_s = a->pos_stride_s; p.inv_freq = a->inv_freq;
  p.eps = a->eps; p.inv_d = 1.0f / (float)a->D;
  const int es = size_of(a->dtype);
  int rc;
  for (int i = 0; i < a->tensors; i++) {
    const xdit_axes_rope_tensor& t = a->t[i];
    xdit::RopeTensor& o = p.t[i];
    if (t.H <= 0 || t.H > 65535) return api_fail(XDIT_ERR_INVALID_ARG, "t[%d]: H = %d must be between 1 and 65535", i, t.H);
    o.x = t.x; o.dy = t.dy; o.y = t.y; o.weight = t.weight; o.dweight = backward && p.norm ? t.dweight : nullptr; o.H = t.H;
    o.xs_b = t.x_stride.b; o.xs_h = t.x_stride.h; o.xs_s = t.x_stride.s;
    o.ds_b = t.dy_stride.b; o.ds_h = t.dy_stride.h; o.ds_s = t.dy_stride.s;
    o.ys_b = t.y_stride.b; o.ys_h = t.y_stride.h; o.ys_s = t.y_stride.s;
    p.sums |= o.dweight != nullptr;
    if (!pointers) continue;
    const struct { const char* name; const void* ptr; const xdit_strides* st; bool used, written; } rows[] = {
        {"x", t.x, &t.x_stride, !backward || p.norm, false}, {"dy", t.dy, &t.dy_stride, backward, false}, {"y", t.y, &t.y_stride, true, true}};
    for (const auto& r : rows) {
      if (!r.used) continue;
      const xdit_row_strides bs = {r.st->b, r.st->s}, bh = {r.st->b, r.st->h};
      if ((rc = check_rows(r.name, r.ptr, bs, es, a->B, a->S, a->D, r.written)) || (rc = check_rows(r.name, r.ptr, bh, es, a->B, t.H, a->D, r.written))) return rc;
      Axis axes[] = {{a->B, r.st->b}, {t.H, r.st->h}, {a->S, r.st->s}};
      if (r.written && !rows_apart(a->D, axes))
        return api_fail(XDIT_ERR_INVALID_ARG, "%s: strides (%lld,%lld,%lld) make its rows of %d overlap", r.name, (long long)r.st->b, (long long)r.st->h, (long long)r.st->s, a->D);
    }
    if (t.weight != nullptr && !p.norm) return api_fail(XDIT_ERR_INVALID_ARG, "a weight needs the norm");
    if ((rc = check_vector("weight", t.weight))) return rc;
    if (o.dweight != nullptr && t.weight == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "dweight needs weight");
  }
  if (pointers && P > 0) {   // without a rotated pair neither is read
    if (a->positions == nullptr || !multiple_of(a->positions, a->pos_bits == 64 ? 8 : 4)) return api_fail(XDIT_ERR_INVALID_ARG, "positions is NULL or not aligned to its elements");
    if (a->inv_freq == nullptr || !multiple_of(a->inv_freq, a->freq_bits / 8)) return api_fail(XDIT_ERR_INVALID_ARG, "inv_freq is NULL or not aligned to its elements");
    if (a->pos_stride_b < 0 || a->pos_stride_s < 0) return api_fail(XDIT_ERR_INVALID_ARG, "positions: negative stride");
  }
  xdit::axes_rope_plan(p, backward);
  return 0;
}

int xdit_axes_rope(const xdit_axes_rope_args* a) {
  xdit::api_clear_error();
  xdit::AxesRopeParams p;
  if (int rc = fill_axes_rope(a, p, false, true)) return rc;
  const hipError_t e = xdit::launch_axes_rope(p, a->dtype, false, (hipStream_t)a->stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "rotation launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

static int64_t rope_backward_bytes(const xdit::AxesRopeParams& p) { return p.sums ? (int64_t)p.head_groups * p.token_groups * 2 * p.D * 4 : 0; }

int64_t xdit_axes_rope_backward_workspace_bytes(const xdit_axes_rope_args* a) {
  xdit::api_clear_error();
  xdit::AxesRopeParams p;
  const int rc = fill_axes_rope(a, p, true, false);
  return rc ? rc : rope_backward_bytes(p);
}

int xdit_axes_rope_backward(const xdit_axes_rope_args* a) {
  xdit::api_clear_error();
  xdit::AxesRopeParams p;
  if (int rc = fill_axes_rope(a, p, true, true)) return rc;
  const int64_t need = rope_backward_bytes(p);
  if (need > 0 && (a->workspace == nullptr || !multiple_of(a->workspace, 16) || a->workspace_bytes < need))
    return api_fail(XDIT_ERR_INVALID_ARG, "workspace of %lld bytes (16-byte aligned) is needed, %lld given", (long long)need, (long long)a->workspace_bytes);
  p.partial = (float*)a->workspace;
  const hipError_t e = xdit::launch_axes_rope(p, a->dtype, true, (hipStream_t)a->stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "rotation backward launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

int xdit_fp8_block_quant(const xdit_block_quant_args* a) {
  xdit::api_clear_error();
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_block_quant_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_block_quant_args));
  if (!float_dtype(a->dtype)) return api_fail(XDIT_ERR_INVALID_ARG, "dtype %d must be bf16, fp16 or fp32", a->dtype);
  if (a->block_rows != 1 && a->block_rows != 128) return api_fail(XDIT_ERR_INVALID_ARG, "block_rows %d must be 1 or 128", a->block_rows);
  if (a->B <= 0 || a->S <= 0 || a->K <= 0) return api_fail(XDIT_ERR_INVALID_ARG, "B, S, K must be positive");
  if (a->S > (int64_t(1) << 30) || a->B * a->S > 0x7fffffffLL || a->K > (int64_t(1) << 30)) return api_fail(XDIT_ERR_INVALID_ARG, "tensor too large for one launch");
  if (a->K % 8 != 0) return api_fail(XDIT_ERR_UNSUPPORTED, "K = %lld: need a multiple of 8", (long long)a->K);
  if (a->block_rows == 128 && a->B != 1) return api_fail(XDIT_ERR_INVALID_ARG, "blocks of 128 rows need B = 1");
  int rc;
  if ((rc = check_rows("x", a->x, a->x_stride, size_of(a->dtype), a->B, a->S, a->K, false))) return rc;
  if ((rc = check_rows("y", a->y, a->y_stride, 1, a->B, a->S, a->K, true))) return rc;
  if (a->scale == nullptr || !multiple_of(a->scale, 4)) return api_fail(XDIT_ERR_INVALID_ARG, "scale is NULL or not 4-byte aligned");
  xdit::BlockQuantParams p;
  std::memset(&p, 0, sizeof(p));
  p.x = a->x; p.y = (unsigned char*)a->y; p.scale = a->scale; p.xs = rs(a->x_stride); p.ys = rs(a->y_stride);
  p.rows = a->B * a->S; p.S = (int)a->S; p.K = (int)a->K; p.kblocks = (p.K + 127) / 128;
  const hipError_t e = xdit::launch_fp8_block_quant(p, a->dtype, a->block_rows, (hipStream_t)a->stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "block quantiser launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

static int fill_block_matmul(const xdit_block_matmul_args* a, xdit::BlockMatmulParams& p, bool pointers) {
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_block_matmul_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_block_matmul_args));
  if (!float_dtype(a->out_dtype)) return api_fail(XDIT_ERR_INVALID_ARG, "out_dtype %d must be bf16, fp16 or fp32", a->out_dtype);
  if (a->bias_dtype != a->out_dtype && a->bias_dtype != XDIT_DTYPE_FP32) return api_fail(XDIT_ERR_INVALID_ARG, "bias_dtype %d must be out_dtype or fp32", a->bias_dtype);
  if (a->M <= 0 || a->N <= 0 || a->K <= 0) return api_fail(XDIT_ERR_INVALID_ARG, "M, N, K must be positive");
  if (a->M > (1 << 30) || a->N > (1 << 24) || a->K > (1 << 24)) return api_fail(XDIT_ERR_INVALID_ARG, "M is limited to 2^30, N and K to 2^24");
  if (a->K % 16 != 0) return api_fail(XDIT_ERR_UNSUPPORTED, "K = %lld: need a multiple of 16", (long long)a->K);
  if (a->cu_count < 0 || a->cu_count > 4096) return api_fail(XDIT_ERR_INVALID_ARG, "cu_count %d must be between 0 and 4096", a->cu_count);
  std::memset(&p, 0, sizeof(p));
  p.x = (const unsigned char*)a->x; p.xsc = a->x_scale; p.w = (const unsigned char*)a->w; p.wsc = a->w_scale; p.bias = a->bias; p.out = a->out;
  p.xs = a->x_stride; p.ws = a->w_stride; p.os = a->out_stride;
  p.xsc_m = a->x_scale_stride_m; p.xsc_k = a->x_scale_stride_k; p.wsc_n = a->w_scale_stride_n; p.wsc_k = a->w_scale_stride_k;
  p.M = (int)a->M; p.N = (int)a->N; p.K = (int)a->K; p.kblocks = (p.K + 127) / 128;
  p.bias_wide = a->bias_dtype == XDIT_DTYPE_FP32;
  p.cu_count = a->cu_count;
  p.exact = a->exact_sums != 0;
  if (!pointers) return 0;
  if (a->x == nullptr || a->w == nullptr || a->x_scale == nullptr || a->w_scale == nullptr || a->out == nullptr)
    return api_fail(XDIT_ERR_INVALID_ARG, "x, x_scale, w, w_scale or out is NULL");
  if (!multiple_of(a->x_scale, 4) || !multiple_of(a->w_scale, 4)) return api_fail(XDIT_ERR_INVALID_ARG, "x_scale and w_scale must be 4-byte aligned");
  if (!multiple_of(a->x, 16) || !multiple_of(a->w, 16)) return api_fail(XDIT_ERR_INVALID_ARG, "x and w must be 16-byte aligned");
  if ((a->M > 1 && (a->x_stride % 16 || a->x_stride < a->K)) || (a->N > 1 && (a->w_stride % 16 || a->w_stride < a->K)))
    return api_fail(XDIT_ERR_INVALID_ARG, "rows of x and w must be multiples of 16 bytes apart, at least K = %lld", (long long)a->K);
  if ((a->M > 1 && a->x_stride >= (1 << 24)) || (a->N > 1 && a->w_stride >= (1 << 24))) return api_fail(XDIT_ERR_INVALID_ARG, "row strides of 2^24 bytes or more are not supported");
  if (!multiple_of(a->out, size_of(a->out_dtype)) || (a->M > 1 && a->out_stride < a->N))
    return api_fail(XDIT_ERR_INVALID_ARG, "out is not aligned to its elements or its rows overlap");
  if (a->x_scale_stride_m < 0 || a->x_scale_stride_k < 0 || a->w_scale_stride_n < 0 || a->w_scale_stride_k < 0)
    return api_fail(XDIT_ERR_INVALID_ARG, "negative scale stride");
  if (a->bias != nullptr && !multiple_of(a->bias, size_of(a->bias_dtype))) return api_fail(XDIT_ERR_INVALID_ARG, "bias is not aligned to its elements");
  if (a->workspace != nullptr && (!multiple_of(a->workspace, 16) || a->workspace_bytes < 0)) return api_fail(XDIT_ERR_INVALID_ARG, "workspace is not 16-byte aligned");
  p.partial = (float*)a->workspace;
  return 0;
}

int64_t xdit_fp8_block_matmul_workspace_bytes(const xdit_block_matmul_args* a) {
  xdit::api_clear_error();
  xdit::BlockMatmulParams p;
  const int rc = fill_block_matmul(a, p, false);
  return rc ? rc : (int64_t)xdit::fp8_block_matmul_workspace(p);
}

int xdit_fp8_block_matmul(const xdit_block_matmul_args* a) {
  xdit::api_clear_error();
  xdit::BlockMatmulParams p;
  if (int rc = fill_block_matmul(a, p, true)) return rc;
  const hipError_t e = xdit::launch_fp8_block_matmul(p, a->out_dtype, a->workspace != nullptr ? (size_t)a->workspace_bytes : 0, (hipStream_t)a->stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "block-scaled product launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

}  // extern "C"
