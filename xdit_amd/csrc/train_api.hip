// C ABI of what a training step adds to the forward pass: argument validation, launch plans and launch.
// Nothing here allocates device memory or synchronises; every launch goes to the caller's stream.
#include "../../include/xdit_amd_attn.h"

#include <algorithm>
#include <cmath>
#include <cstring>
#include <vector>

#include "api_error.h"
#include "attn_bwd.h"
#include "attn_split.h"
#include "grad_norm.h"

namespace {

using xdit::api_fail;

int64_t align256(int64_t n) { return (n + 255) & ~int64_t(255); }

// A compute unit's workgroups over time: how many of an XCD's places become free when.  Units are dealt out in the order of the launch,
// each to the place that is free first, as the hardware does it.
struct Places {
  struct Group { double time; int64_t n; } g[8];
  int used;
  explicit Places(int64_t places) : used(1) { g[0] = {0.0, places}; }
  void run(int64_t units, double each) {
    int64_t all = 0;
    for (int i = 0; i < used; i++) all += g[i].n;
    if (units > 4 * all) {   // whole rounds shift every place alike
      const int64_t rounds = (units - 3 * all) / all;
      for (int i = 0; i < used; i++) g[i].time += rounds * each;
      units -= rounds * all;
    }
    while (units > 0) {
      const Group first = g[0];   // kept in order of time
      const int64_t n = first.n < units ? first.n : units;
      units -= n;
      if (n < first.n) g[0].n -= n;
      else std::copy(g + 1, g + used--, g);
      int at = 0;
      while (at < used && g[at].time < first.time + each) at++;
      if (at < used && g[at].time < first.time + each + 1e-9) { g[at].n += n; continue; }
      if (used == 8) { g[7].n += n; continue; }   // (an estimate: the latest of them takes it)
      std::copy_backward(g + at, g + used, g + used + 1);
      g[at] = {first.time + each, n};
      used++;
    }
  }
  double end() const { return g[used - 1].time; }
};

// Microseconds that a launch takes.  A unit's step (64 streamed rows; fp32: 32) takes `shared` beside the others that a compute unit holds
// and `alone` where no compute unit has more than one; `fixed` are its operands, first tile and results.  Partial results are read back at
// 5 TB/s by a launch of 4 us (they are written while other units compute).
struct StepCost {
  double alone[2], shared[2];   // keys, queries
  double fixed[2];
  double part;                  // of a tensor's partial tile
};

// Where every unit has a place at once: the units of a compute unit are those whose numbers differ by the number of compute units, and what
// they do adds up, less what they gain by running beside each other.
double one_round_us(const xdit::BwdRole& k, const xdit::BwdRole& q, int64_t cus, int per_cu, const StepCost& c) {
  struct Group { int64_t end; double work, fixed; } g[4];
  int n = 0;
  int64_t units = 0;
  for (int i = 0; i < 2; i++) {
    const xdit::BwdRole& r = i ? q : k;
    if (r.total == 0) continue;
    if (r.whole) g[n++] = {units += r.whole, r.steps * c.alone[i], c.fixed[i]};
    if (r.per_xcd > r.whole) g[n++] = {units += r.units - r.whole, r.len * c.alone[i], c.fixed[i]};
  }
  double longest = 0.0;
  for (int s = -1; s < n - 1; s++) {   // the compute units at which a group begins have the longest lists
    double work = 0.0, fixed = 0.0, gain = 0.0;
    int on = 0, at = 0;
    for (int64_t u = (s < 0 ? 0 : g[s].end) % cus; u < units; u += cus, on++) {
      while (u >= g[at].end) at++;
      work += g[at].work;
      fixed = std::max(fixed, g[at].fixed);
      gain = (1.0 - c.shared[0] / (per_cu * c.alone[0])) * on / std::max(per_cu - 1, 1);
    }
    longest = std::max(longest, work * (1.0 - gain) + fixed);
  }
  return longest;
}

double launch_us(const xdit::BwdRole& k, const xdit::BwdRole& q, int64_t cus, int per_cu, const StepCost& c) {
  const bool one_round = k.units + q.units <= cus * per_cu;
  Places p(cus * per_cu);
  double us = 0.0;
  for (int i = 0; i < 2; i++) {
    const xdit::BwdRole& r = i ? q : k;
    if (r.total == 0) continue;
    if (!one_round) {
      if (r.whole) p.run(r.whole, r.steps * c.shared[i] + c.fixed[i]);
      if (r.per_xcd > r.whole) p.run(r.units - r.whole, r.len * c.shared[i] + c.fixed[i]);
    }
    us += (double)xdit::bwd_cut_tiles(r) * r.parts * (2 - i) * c.part;
  }
  return (one_round ? one_round_us(k, q, cus, per_cu, c) : p.end()) + us + (k.parts > 1 || q.parts > 1 ? 4.0 : 0.0);
}

void set_parts(xdit::BwdRole& r, int whole, int parts) {
  r.whole = whole < r.per_xcd ? whole : r.per_xcd;
  r.len = (r.steps + parts - 1) / parts;
  r.parts = r.whole == r.per_xcd ? 1 : (r.steps + r.len - 1) / r.len;
  if (r.parts == 1) { r.whole = r.per_xcd; r.len = r.steps; }
  r.units = r.total == 0 ? 0 : r.whole == 0 ? (r.total * r.parts + 7) / 8 : r.whole + (r.per_xcd - r.whole) * r.parts;
}

constexpr int kParts[] = {2, 3, 4, 6, 8, 12, 16, 24, 32, 48, 64};

// Which tiles of a role are cut into parts, and into how many: all of them, or (`last`: the role's units are the last of the launch) the last ones of
// every XCD's tiles; kept where the estimate of the launch gets shorter by it.
void plan_role(xdit::BwdRole& r, const xdit::BwdRole& k, const xdit::BwdRole& q, int64_t cus, int per_cu, const StepCost& c, bool last) {
  if (r.total == 0) return;
  xdit::BwdRole best = r;
  double best_us = launch_us(k, q, cus, per_cu, c);
  for (int parts : kParts) {
    if (parts > r.steps) break;
    int64_t cut = r.per_xcd;
    for (int round = 0; cut > 0 && round < (last ? 4 : 1); round++) {
      if ((cut == r.per_xcd ? (int64_t)r.total * parts / 8 : cut * parts) <= 4 * cus * per_cu) {
        set_parts(r, r.per_xcd - (int)cut, parts);
        const double us = launch_us(k, q, cus, per_cu, c);
        if (us < best_us * 0.99) { best_us = us; best = r; }
      }
      cut = round == 0 ? std::min<int64_t>(cut - 1, cus * per_cu) : cut / 2;
    }
  }
  r = best;
}

void plan_roles(xdit::AttnBwdParams& p, int64_t cus, int per_cu, const StepCost& c) {
  xdit::BwdRole &k = p.keys, &q = p.queries;
  if (k.total && q.total && k.units + q.units <= cus * per_cu) {   // few tiles: the roles run side by side, so that both have to be cut for either to matter
    double best_us = launch_us(k, q, cus, per_cu, c);
    xdit::BwdRole best_k = k, best_q = q;
    for (int parts : kParts) {
      if (parts > k.steps && parts > q.steps) break;
      set_parts(k, 0, std::min(parts, k.steps));
      set_parts(q, 0, std::min(parts, q.steps));
      const double us = launch_us(k, q, cus, per_cu, c);
      if (us < best_us * (best_k.parts == 1 && best_q.parts == 1 ? 0.95 : 0.99)) { best_us = us; best_k = k; best_q = q; }   // the estimates are off by as much
    }
    k = best_k;
    q = best_q;
  }
  plan_role(k, k, q, cus, per_cu, c, q.total == 0);
  plan_role(q, k, q, cus, per_cu, c, true);
}

struct BwdPlan {
  int64_t stats, norms, keys, queries;   // bytes
  int64_t need() const { return stats + norms + keys + queries; }
  int64_t workgroups;                    // of the largest launch
};

// A launch has less than 2^32 threads, 256 of them in a workgroup.
int check_launches(const BwdPlan& plan) {
  return plan.workgroups >= (int64_t(1) << 24) ? api_fail(XDIT_ERR_INVALID_ARG, "B*H times the sequence length is too large for one launch") : 0;
}

BwdPlan plan_bwd(const xdit_attn_bwd_args* a, xdit::AttnBwdParams& p) {
  BwdPlan plan;
  const bool f32 = a->dtype == XDIT_DTYPE_FP32;
  const int rows = xdit::kBwdRows, step = f32 ? 32 : 64;
  const int dc = f32 ? (xdit::bwd_f32_groups(a->D) + 1) / 2 * 16 : (a->D + 31) / 32 * 32;   // computed columns of the gradients
  const int64_t bh = (int64_t)a->B * a->H;
  const int per_cu = f32 ? (a->D <= 96 ? 2 : 1) : a->D <= 64 ? 3 : 2;   // workgroups on a compute unit
  const int64_t cus = (xdit::resident_cus(a->cu_count) + 7) / 8;   // of an XCD
  p.Sq = (int)a->Sq; p.Sk = (int)a->Sk; p.Sk2 = (int)a->Sk2;
  p.tiles1 = (int)((a->Sk + rows - 1) / rows);
  p.keys.tiles = p.tiles1 + (int)((a->Sk2 + rows - 1) / rows);
  p.keys.steps = (int)((a->Sq + step - 1) / step);
  p.queries.tiles = (int)((a->Sq + rows - 1) / rows);
  p.step1 = (int)((a->Sk + step - 1) / step);
  p.queries.steps = p.step1 + (int)((a->Sk2 + step - 1) / step);
  p.keys.total = a->dk != nullptr ? (int)(bh * p.keys.tiles) : 0;
  p.queries.total = a->dq != nullptr ? (int)(bh * p.queries.tiles) : 0;
  for (xdit::BwdRole* r : {&p.keys, &p.queries}) {
    r->per_xcd = (r->total + 7) / 8;
    set_parts(*r, r->per_xcd, 1);
  }
  // measured: 8 and 16 heads of 16384 rows on 4096 and of 4096 on 16384, 8 to 48 of 2048 on 2048 and 4096, 3 of 1536 on 1536; fp32: 8 and
  // 16 of 4096 at head_dims 64, 72 and 128, whose steps take what their matrix instructions do (over the columns that are contracted and
  // those of the gradients)
  StepCost cost = a->D <= 64 ? StepCost{{1.15, 1.0}, {2.99, 2.35}, {6.0, 5.0}, 0.0} : StepCost{{1.95, 1.62}, {3.56, 2.8}, {7.0, 5.5}, 0.0};
  if (f32) {
    const int contracted = 8 * xdit::bwd_f32_groups(a->D);
    const double k = 0.0158 * (2 * contracted + 2 * dc), q = 0.017 * (2 * contracted + dc);
    cost = StepCost{{k, q}, {per_cu * 0.94 * k, per_cu * 0.94 * q}, {8.0, 6.0}, 0.0};
  }
  cost.part = rows * dc * 4 / 5e6;
  plan_roles(p, cus, per_cu, cost);
  p.sq_pad = (int)((a->Sq + xdit::kBwdStatRows - 1) / xdit::kBwdStatRows * xdit::kBwdStatRows);
  plan.stats = align256(bh * 2 * p.sq_pad * 4);
  plan.norms = a->dtype == XDIT_DTYPE_FP16 ? align256(bh * xdit::bwd_value_blocks(p) * 4) : 0;
  auto partial = [&](const xdit::BwdRole& r, int tensors) { return (int64_t)xdit::bwd_cut_tiles(r) * r.parts * tensors * rows * dc * 4; };
  plan.keys = partial(p.keys, 2);
  plan.queries = partial(p.queries, 1);
  const int64_t stats = bh * (p.sq_pad / xdit::kBwdStatRows + (a->dtype == XDIT_DTYPE_FP16 ? xdit::bwd_value_blocks(p) : 0));
  const int64_t fold = (int64_t)(2 * xdit::bwd_cut_tiles(p.keys) + xdit::bwd_cut_tiles(p.queries)) * (rows * dc / 1024);
  plan.workgroups = std::max({stats, fold, 8 * (int64_t)(p.keys.units + p.queries.units)});
  return plan;
}

// What can be checked without looking at a pointer's target; the size of the workspace depends on nothing else.
int check_bwd_shape(const xdit_attn_bwd_args* a) {
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_attn_bwd_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_attn_bwd_args));
  if (a->dtype != XDIT_DTYPE_BF16 && a->dtype != XDIT_DTYPE_FP16 && a->dtype != XDIT_DTYPE_FP32)
    return api_fail(a->dtype == XDIT_DTYPE_FP8_E4M3FN ? XDIT_ERR_UNSUPPORTED : XDIT_ERR_INVALID_ARG, "dtype %d must be bf16, fp16 or fp32", a->dtype);
  if (a->B <= 0 || a->H <= 0) return api_fail(XDIT_ERR_INVALID_ARG, "B=%d H=%d must be positive", a->B, a->H);
  if (a->Sq <= 0 || a->Sk <= 0 || a->Sk2 < 0)
    return api_fail(XDIT_ERR_INVALID_ARG, "Sq=%lld Sk=%lld Sk2=%lld: need Sq>0, Sk>0, Sk2>=0", (long long)a->Sq, (long long)a->Sk, (long long)a->Sk2);
  if (a->Sq > (int64_t(1) << 29) || a->Sk > (int64_t(1) << 29) || a->Sk2 > (int64_t(1) << 29))
    return api_fail(XDIT_ERR_INVALID_ARG, "sequence length above 2^29");
  if ((int64_t)a->B * a->H * ((a->Sq + 31) / 32) > (int64_t(1) << 24) || (int64_t)a->B * a->H * ((a->Sk + 31) / 32 + (a->Sk2 + 31) / 32) > (int64_t(1) << 24))
    return api_fail(XDIT_ERR_INVALID_ARG, "B*H times the sequence length is too large for one launch");
  if (!(a->softmax_scale > 0.f) || !std::isfinite(a->softmax_scale))
    return api_fail(XDIT_ERR_INVALID_ARG, "softmax_scale must be finite and > 0");
  if (a->D <= 0 || a->D % 8 != 0 || a->D > 128) return api_fail(XDIT_ERR_UNSUPPORTED, "head_dim %d: need a multiple of 8, at most 128", a->D);
  if (a->cu_count < 0 || a->cu_count > 4096) return api_fail(XDIT_ERR_INVALID_ARG, "cu_count %d must be between 0 and 4096", a->cu_count);
  if (a->reserved0 != 0) return api_fail(XDIT_ERR_INVALID_ARG, "reserved0 must be 0");
  if (a->dq == nullptr && a->dk == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "dq and dk are both NULL");
  const bool k = a->dk != nullptr, s2 = a->Sk2 > 0;
  if ((a->dv != nullptr) != k || (s2 && ((a->dk2 != nullptr) != k || (a->dv2 != nullptr) != k)))
    return api_fail(XDIT_ERR_INVALID_ARG, "dk and dv (with Sk2 also dk2 and dv2) are given together or not at all");
  return 0;
}

int check_grad(const char* name, const void* p, const xdit_strides& st, int es, int64_t B, int64_t H, int64_t S, int D) {
  if (int rc = xdit::api_check_tensor(name, p, st, es, D)) return rc;
  xdit::Axis axes[3] = {{B, st.b}, {H, st.h}, {S, st.s}};
  if (!xdit::rows_apart(D, axes)) return api_fail(XDIT_ERR_INVALID_ARG, "%s: rows overlap", name);
  return 0;
}

// The bytes of a (B, H, S) tensor of rows, from its first one on.
struct Rows {
  uintptr_t at;
  int64_t width;
  struct { int64_t n, stride; } axis[3];   // bytes
  __int128 end() const {
    __int128 e = (__int128)at + width;
    for (const auto& a : axis) e += (__int128)a.stride * (a.n - 1);
    return e;
  }
};

Rows rows_of(const void* p, int64_t B, int64_t H, int64_t S, const xdit_strides& st, int64_t width, int es) {
  return {reinterpret_cast<uintptr_t>(p), width * es, {{B, st.b * es}, {H, st.h * es}, {S, st.s * es}}};
}

// Whether a row of x and one of y share a byte: whether a sum of steps, at most those between two rows of either, leads from x to within a
// row of y.  Steps are taken from the largest stride down, those only from which the smaller ones still reach: one or two a stride where
// rows lie as those of views of one buffer do. Where they lie otherwise and 4096 sums were looked at, the answer is that they may.
bool share_bytes(const Rows& x, const Rows& y) {
  if ((__int128)x.at >= y.end() || (__int128)y.at >= x.end()) return false;
  struct Step { __int128 stride; int64_t least, most; } step[6];
  int n = 0;
  for (int i = 0; i < 6; i++) {
    const auto& a = i < 3 ? x.axis[i] : y.axis[i - 3];
    if (a.n <= 1 || a.stride == 0) continue;
    int k = 0;
    while (k < n && step[k].stride != a.stride) k++;
    if (k == n) step[n++] = {a.stride, 0, 0};
    if (i < 3) step[k].least -= a.n - 1;
    else step[k].most += a.n - 1;
  }
  std::sort(step, step + n, [](const Step& a, const Step& b) { return a.stride > b.stride; });
  __int128 below[7], above[7];   // how far the steps from the k-th on lead back and forth
  below[n] = above[n] = 0;
  for (int k = n - 1; k >= 0; k--) {
    below[k] = below[k + 1] + step[k].stride * step[k].least;
    above[k] = above[k + 1] + step[k].stride * step[k].most;
  }
  int budget = 4096;
  auto meet = [&](auto& self, int k, __int128 d) -> bool {   // d: from a row of x to one of y
    if (--budget < 0) return true;
    if (k == n) return d < x.width && -d < y.width;
    const __int128 st = step[k].stride;
    for (__int128 c = std::max<__int128>(step[k].least, (-y.width - d - above[k + 1]) / st - 1); c <= step[k].most; c++) {
      const __int128 at = d + c * st;
      if (at + above[k + 1] <= -y.width) continue;
      if (at + below[k + 1] >= x.width) break;
      if (self(self, k + 1, at)) return true;
    }
    return false;
  };
  return meet(meet, 0, (__int128)y.at - x.at);
}

// The same of all gradients and inputs, whatever part of them it is.
int check_overlaps(const xdit_attn_bwd_args* a) {
  const int es = a->dtype == XDIT_DTYPE_FP32 ? 4 : 2;
  Rows in[9], out[5];
  int inputs = 0, outputs = 0;
  auto add = [&](Rows* list, int& n, const void* p, int64_t S, const xdit_strides& st) {
    if (p != nullptr && S > 0) list[n++] = rows_of(p, a->B, a->H, S, st, a->D, es);
  };
  add(in, inputs, a->dout, a->Sq, a->dout_stride);
  add(in, inputs, a->q, a->Sq, a->q_stride);
  add(in, inputs, a->k, a->Sk, a->k_stride);
  add(in, inputs, a->v, a->Sk, a->v_stride);
  add(in, inputs, a->k2, a->Sk2, a->k2_stride);
  add(in, inputs, a->v2, a->Sk2, a->v2_stride);
  add(in, inputs, a->out, a->Sq, a->out_stride);
  in[inputs++] = rows_of(a->lse, a->B, a->H, a->Sq, a->lse_stride, 1, 4);
  if (a->dlse != nullptr) in[inputs++] = rows_of(a->dlse, a->B, a->H, a->Sq, a->dlse_stride, 1, 4);
  add(out, outputs, a->dq, a->Sq, a->dq_stride);
  add(out, outputs, a->dk, a->Sk, a->dk_stride);
  add(out, outputs, a->dv, a->Sk, a->dv_stride);
  add(out, outputs, a->dk2, a->Sk2, a->dk2_stride);
  add(out, outputs, a->dv2, a->Sk2, a->dv2_stride);
  for (int i = 0; i < outputs; i++) {
    for (int j = 0; j < inputs; j++)
      if (share_bytes(out[i], in[j])) return api_fail(XDIT_ERR_INVALID_ARG, "a gradient overlaps an input");
    for (int j = 0; j < i; j++)
      if (share_bytes(out[i], out[j])) return api_fail(XDIT_ERR_INVALID_ARG, "two gradients overlap");
  }
  return 0;
}

// A gradient in the place of an input, or two in one place: other workgroups still read what a workgroup writes.
int check_places(const xdit_attn_bwd_args* a) {
  const void* in[] = {a->dout, a->q, a->k, a->v, a->out, a->lse, a->dlse, a->Sk2 > 0 ? a->k2 : nullptr, a->Sk2 > 0 ? a->v2 : nullptr};
  const void* out[] = {a->dq, a->dk, a->dv, a->Sk2 > 0 ? a->dk2 : nullptr, a->Sk2 > 0 ? a->dv2 : nullptr};
  for (int i = 0; i < 5; i++) {
    if (out[i] == nullptr) continue;
    for (const void* p : in)
      if (p == out[i]) return api_fail(XDIT_ERR_INVALID_ARG, "a gradient lies in the place of an input");
    for (int j = 0; j < i; j++)
      if (out[j] == out[i]) return api_fail(XDIT_ERR_INVALID_ARG, "two gradients lie in one place");
  }
  return 0;
}

xdit::BwdTensor tensor(const void* p, const xdit_strides& st) { return {const_cast<void*>(p), st.b, st.h, st.s}; }

// ---- norm and clipping of a list of gradients ----

int size_of(int dtype) { return dtype == XDIT_DTYPE_FP32 ? 4 : 2; }
bool float_dtype(int d) { return d == XDIT_DTYPE_BF16 || d == XDIT_DTYPE_FP16 || d == XDIT_DTYPE_FP32; }

int check_list(const char* name, int64_t count, void* const* data, const int64_t* numel, const int32_t* dtype) {
  if (data == nullptr || numel == nullptr || dtype == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "%s: a table is NULL", name);
  for (int64_t i = 0; i < count; i++) {
    if (!float_dtype(dtype[i])) return api_fail(XDIT_ERR_INVALID_ARG, "%s %lld: dtype %d must be bf16, fp16 or fp32", name, (long long)i, dtype[i]);
    if (numel[i] < 0 || numel[i] > (int64_t(1) << 40)) return api_fail(XDIT_ERR_INVALID_ARG, "%s %lld: %lld elements", name, (long long)i, (long long)numel[i]);
    if (numel[i] == 0) continue;
    if (data[i] == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "%s %lld is NULL", name, (long long)i);
    if (reinterpret_cast<uintptr_t>(data[i]) % size_of(dtype[i])) return api_fail(XDIT_ERR_INVALID_ARG, "%s %lld is not aligned to its elements", name, (long long)i);
  }
  return 0;
}

int check_norm_list(const xdit_grad_norm_args* a) {
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_grad_norm_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_grad_norm_args));
  if (a->kind < XDIT_GRADNORM_MAX || a->kind > XDIT_GRADNORM_L2) return api_fail(XDIT_ERR_INVALID_ARG, "unknown norm %d", a->kind);
  if (a->count < 0 || a->count > (1 << 24)) return api_fail(XDIT_ERR_INVALID_ARG, "count %lld must lie between 0 and 2^24", (long long)a->count);
  return a->count ? check_list("gradient", a->count, const_cast<void* const*>(a->data), a->numel, a->dtype) : 0;
}

// Elements of a workgroup: the list over about 2048 workgroups, eight for a compute unit, between one pass of 256 threads and 32.
int64_t chunk_elements(int64_t count, const int64_t* numel) {
  int64_t total = 0, chunk = 2048;
  for (int64_t i = 0; i < count; i++) total += numel[i];
  while (chunk < 65536 && chunk * 2048 < total) chunk *= 2;
  return chunk;
}
int64_t chunks_of(int64_t numel, int64_t chunk) { return numel == 0 ? 0 : (numel + 7 + chunk - 1) / chunk; }   // up to 7 elements before its aligned start

// The launches that leave a partial value of every chunk; their count, or a negative status.  With a counter and a norm there is one
// launch, which leaves the norm too.
int64_t launch_partials(int64_t count, const void* const* data, const int64_t* numel, const int32_t* dtypes, int kind, double* partial, hipStream_t stream,
                        unsigned* counter = nullptr, float* norm = nullptr) {
  const int64_t chunk = chunk_elements(count, numel);
  const double* const start = partial;
  xdit::NormParams p;
  p.chunk = (int)chunk;
  p.kind = kind;
  p.counter = counter;
  p.norm = norm;
  for (int dtype = XDIT_DTYPE_BF16; dtype <= XDIT_DTYPE_FP32; dtype++) {   // a launch holds tensors of one dtype
    int n = 0;
    int64_t chunks = 0;
    for (int64_t i = 0; i <= count; i++) {
      const bool takes = i < count && dtypes[i] == dtype && numel[i] != 0;
      const int64_t more = takes ? chunks_of(numel[i], chunk) : 0;
      if (n && (i == count || (takes && (n == xdit::kNormTensors || chunks + more > (1 << 30))))) {
        std::fill(p.t.first + n, p.t.first + xdit::kNormTensors, 0xffffffffu);
        p.partial = partial;
        const hipError_t e = xdit::launch_grad_norm(p, dtype, (unsigned)chunks, stream);
        if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "gradient norm launch failed: %s", hipGetErrorString(e));
        partial += chunks;
        n = 0;
        chunks = 0;
      }
      if (takes) {
        p.t.first[n] = (uint32_t)chunks;
        p.t.numel[n] = numel[i];
        p.t.src[n++] = data[i];
        chunks += more;
      }
    }
  }
  return partial - start;
}

int64_t partials_of(int64_t count, const int64_t* numel) {
  const int64_t chunk = chunk_elements(count, numel);
  int64_t n = 0;
  for (int64_t i = 0; i < count; i++) n += chunks_of(numel[i], chunk);
  return n;
}

// Whether the norm of a list is one launch's, and its last workgroup can add the partial sums up: tensors of one dtype, as many as a launch
// takes, few chunks.
bool one_launch(int64_t count, const int64_t* numel, const int32_t* dtypes, int64_t partials) {
  int64_t tensors = 0;
  int dtype = -1;
  for (int64_t i = 0; i < count; i++) {
    if (numel[i] == 0) continue;
    if (tensors++ && dtypes[i] != dtype) return false;
    dtype = dtypes[i];
  }
  return tensors > 0 && tensors <= xdit::kNormTensors && partials <= xdit::kClipPartials;
}

int check_partials(int64_t n, const void* workspace, int64_t bytes) {
  if (n && (workspace == nullptr || (reinterpret_cast<uintptr_t>(workspace) & 7u) || bytes < n * (int64_t)sizeof(double)))
    return api_fail(XDIT_ERR_INVALID_ARG, "workspace must be 8-byte aligned and hold %lld bytes", (long long)(n * sizeof(double)));
  return 0;
}

// Whether no destination overlaps another one, a source other than itself, or the norm, and a norm that is written no source.
bool destinations_apart(const xdit_clip_grads_args* a) {
  struct Span { uintptr_t begin, end; int64_t i; };
  std::vector<Span> dst;
  dst.reserve(a->count);
  for (int64_t i = 0; i < a->count; i++)
    if (a->numel[i]) dst.push_back({reinterpret_cast<uintptr_t>(a->dst[i]), reinterpret_cast<uintptr_t>(a->dst[i]) + a->numel[i] * size_of(a->dst_dtype[i]), i});
  std::sort(dst.begin(), dst.end(), [](const Span& x, const Span& y) { return x.begin < y.begin; });
  for (size_t n = 1; n < dst.size(); n++)
    if (dst[n].begin < dst[n - 1].end) return false;
  const uintptr_t norm = reinterpret_cast<uintptr_t>(a->norm != nullptr ? a->norm : a->norm_out);   // every workgroup reads it, or one writes it while others read gradients
  for (int64_t i = 0; i < a->count; i++) {
    if (a->numel[i] == 0) continue;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(a->src[i]), end = begin + a->numel[i] * size_of(a->src_dtype[i]);
    if (a->norm == nullptr && norm < end && norm + sizeof(float) > begin) return false;
    auto at = std::upper_bound(dst.begin(), dst.end(), begin, [](uintptr_t x, const Span& s) { return x < s.end; });   // the first that ends behind the source's start
    for (; at != dst.end() && at->begin < end; ++at)
      if (at->i != i || at->begin != begin || a->src_dtype[i] != a->dst_dtype[i]) return false;
  }
  auto at = std::upper_bound(dst.begin(), dst.end(), norm, [](uintptr_t x, const Span& s) { return x < s.end; });
  return at == dst.end() || at->begin >= norm + sizeof(float);
}

}  // namespace

extern "C" {

int64_t xdit_grad_norm_workspace_bytes(const xdit_grad_norm_args* a) {
  xdit::api_clear_error();
  if (int rc = check_norm_list(a)) return rc;
  return partials_of(a->count, a->numel) * (int64_t)sizeof(double);
}

int xdit_grad_norm(const xdit_grad_norm_args* a) {
  xdit::api_clear_error();
  if (int rc = check_norm_list(a)) return rc;
  if (a->norm == nullptr || reinterpret_cast<uintptr_t>(a->norm) & 3u) return api_fail(XDIT_ERR_INVALID_ARG, "norm is NULL or not 4-byte aligned");
  if (reinterpret_cast<uintptr_t>(a->counter) & 3u) return api_fail(XDIT_ERR_INVALID_ARG, "counter is not 4-byte aligned");
  const int64_t partials = partials_of(a->count, a->numel);
  if (int rc = check_partials(partials, a->workspace, a->workspace_bytes)) return rc;
  hipStream_t stream = (hipStream_t)a->stream;
  const bool one = a->counter != nullptr && one_launch(a->count, a->numel, a->dtype, partials);
  const int64_t n = launch_partials(a->count, a->data, a->numel, a->dtype, a->kind, (double*)a->workspace, stream, one ? a->counter : nullptr, a->norm);
  if (n < 0 || one) return n < 0 ? (int)n : XDIT_OK;
  const hipError_t e = xdit::launch_grad_norm_total((const double*)a->workspace, n, a->kind, a->norm, stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "gradient norm launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

int xdit_clip_grads(const xdit_clip_grads_args* a) {
  xdit::api_clear_error();
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_clip_grads_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_clip_grads_args));
  if (a->count < 0 || a->count > (1 << 24)) return api_fail(XDIT_ERR_INVALID_ARG, "count %lld must lie between 0 and 2^24", (long long)a->count);
  if (a->reserved0 != 0) return api_fail(XDIT_ERR_INVALID_ARG, "reserved0 must be 0");
  if (!(a->max_norm >= 0.f) || !std::isfinite(a->max_norm)) return api_fail(XDIT_ERR_INVALID_ARG, "max_norm must be finite and >= 0");
  const bool given = a->norm != nullptr;
  if (given ? reinterpret_cast<uintptr_t>(a->norm) & 3u : a->norm_out == nullptr || reinterpret_cast<uintptr_t>(a->norm_out) & 3u)
    return api_fail(XDIT_ERR_INVALID_ARG, "norm and norm_out are NULL, or one is not 4-byte aligned");
  if (!given && (a->kind < XDIT_GRADNORM_MAX || a->kind > XDIT_GRADNORM_L2)) return api_fail(XDIT_ERR_INVALID_ARG, "unknown norm %d", a->kind);
  int rc;
  if (a->count) {
    if ((rc = check_list("gradient", a->count, const_cast<void* const*>(a->src), a->numel, a->src_dtype))) return rc;
    if ((rc = check_list("result", a->count, a->dst, a->numel, a->dst_dtype))) return rc;
  }
  if (!given && (rc = check_partials(partials_of(a->count, a->numel), a->workspace, a->workspace_bytes))) return rc;
  try {
    if (!destinations_apart(a)) return api_fail(XDIT_ERR_INVALID_ARG, "a result overlaps another one, a gradient other than its own, or the norm");
  } catch (const std::bad_alloc&) {
    return api_fail(XDIT_ERR_INVALID_ARG, "no host memory for %lld tensors", (long long)a->count);
  }
  hipStream_t stream = (hipStream_t)a->stream;
  const int64_t chunk = chunk_elements(a->count, a->numel);
  xdit::ClipParams p;
  p.chunk = (int)chunk;
  p.max_norm = a->max_norm;
  p.norm = a->norm;
  p.partial = nullptr;
  p.norm_out = nullptr;
  p.partials = 0;
  p.kind = a->kind;
  if (!given) {
    const int64_t n = launch_partials(a->count, a->src, a->numel, a->src_dtype, a->kind, (double*)a->workspace, stream);
    if (n < 0) return (int)n;
    if (n == 0 || n > xdit::kClipPartials) {
      const hipError_t e = xdit::launch_grad_norm_total((const double*)a->workspace, n, a->kind, a->norm_out, stream);
      if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "gradient norm launch failed: %s", hipGetErrorString(e));
      p.norm = a->norm_out;
    } else {
      p.partial = (const double*)a->workspace;
      p.partials = (int)n;
      p.norm_out = a->norm_out;   // of the first launch
    }
  }
  for (int pair = 0; pair < 9; pair++) {   // a launch holds tensors of one dtype and results of one
    const int sd = pair / 3, dd = pair % 3;
    int n = 0;
    int64_t chunks = 0;
    for (int64_t i = 0; i <= a->count; i++) {
      const bool takes = i < a->count && a->src_dtype[i] == sd && a->dst_dtype[i] == dd && a->numel[i] != 0;
      const int64_t more = takes ? chunks_of(a->numel[i], chunk) : 0;
      if (n && (i == a->count || (takes && (n == xdit::kClipTensors || chunks + more > (1 << 30))))) {
        std::fill(p.t.first + n, p.t.first + xdit::kClipTensors, 0xffffffffu);
        const hipError_t e = xdit::launch_grad_clip(p, sd, dd, (unsigned)chunks, stream);
        if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "clipping launch failed: %s", hipGetErrorString(e));
        p.norm_out = nullptr;
        n = 0;
        chunks = 0;
      }
      if (takes) {
        p.t.first[n] = (uint32_t)chunks;
        p.t.numel[n] = a->numel[i];
        p.t.src[n] = a->src[i];
        p.dst[n++] = a->dst[i];
        chunks += more;
      }
    }
  }
  return XDIT_OK;
}

int64_t xdit_attn_bwd_workspace_bytes(const xdit_attn_bwd_args* a) {
  xdit::api_clear_error();
  if (int rc = check_bwd_shape(a)) return rc;
  xdit::AttnBwdParams p;
  std::memset(&p, 0, sizeof(p));
  const BwdPlan plan = plan_bwd(a, p);
  if (int rc = check_launches(plan)) return rc;
  return plan.need();
}

int xdit_attn_bwd(const xdit_attn_bwd_args* a) {
  xdit::api_clear_error();
  if (int rc = check_bwd_shape(a)) return rc;
  const int es = a->dtype == XDIT_DTYPE_FP32 ? 4 : 2;
  int rc;
  if ((rc = xdit::api_check_tensor("dout", a->dout, a->dout_stride, es, a->D))) return rc;
  if ((rc = xdit::api_check_tensor("q", a->q, a->q_stride, es, a->D))) return rc;
  if ((rc = xdit::api_check_tensor("k", a->k, a->k_stride, es, a->D))) return rc;
  if ((rc = xdit::api_check_tensor("v", a->v, a->v_stride, es, a->D))) return rc;
  if ((rc = xdit::api_check_tensor("out", a->out, a->out_stride, es, a->D))) return rc;
  if (a->Sk2 > 0) {
    if ((rc = xdit::api_check_tensor("k2", a->k2, a->k2_stride, es, a->D))) return rc;
    if ((rc = xdit::api_check_tensor("v2", a->v2, a->v2_stride, es, a->D))) return rc;
  }
  if (a->dq != nullptr && (rc = check_grad("dq", a->dq, a->dq_stride, es, a->B, a->H, a->Sq, a->D))) return rc;
  if (a->dk != nullptr) {
    if ((rc = check_grad("dk", a->dk, a->dk_stride, es, a->B, a->H, a->Sk, a->D))) return rc;
    if ((rc = check_grad("dv", a->dv, a->dv_stride, es, a->B, a->H, a->Sk, a->D))) return rc;
    if (a->Sk2 > 0) {
      if ((rc = check_grad("dk2", a->dk2, a->dk2_stride, es, a->B, a->H, a->Sk2, a->D))) return rc;
      if ((rc = check_grad("dv2", a->dv2, a->dv2_stride, es, a->B, a->H, a->Sk2, a->D))) return rc;
    }
  }
  if (a->lse == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "lse is NULL");
  if ((rc = check_places(a))) return rc;
  if (reinterpret_cast<uintptr_t>(a->lse) & 3u || reinterpret_cast<uintptr_t>(a->dlse) & 3u)
    return api_fail(XDIT_ERR_INVALID_ARG, "lse and dlse must be 4-byte aligned");
  if (a->lse_stride.b < 0 || a->lse_stride.h < 0 || a->lse_stride.s < 0 || a->dlse_stride.b < 0 || a->dlse_stride.h < 0 || a->dlse_stride.s < 0)
    return api_fail(XDIT_ERR_INVALID_ARG, "lse and dlse: negative stride");

  xdit::AttnBwdParams p;
  std::memset(&p, 0, sizeof(p));
  const BwdPlan plan = plan_bwd(a, p);
  if ((rc = check_launches(plan))) return rc;
  const int64_t need = plan.need();
  if (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 15u) || a->workspace_bytes < need)
    return api_fail(XDIT_ERR_INVALID_ARG, "workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
  if ((rc = check_overlaps(a))) return rc;
  p.q = tensor(a->q, a->q_stride);
  p.k = tensor(a->k, a->k_stride);
  p.v = tensor(a->v, a->v_stride);
  p.out = tensor(a->out, a->out_stride);
  p.dout = tensor(a->dout, a->dout_stride);
  p.dq = tensor(a->dq, a->dq_stride);
  p.dk = tensor(a->dk, a->dk_stride);
  p.dv = tensor(a->dv, a->dv_stride);
  if (a->Sk2 > 0) {
    p.k2 = tensor(a->k2, a->k2_stride);
    p.v2 = tensor(a->v2, a->v2_stride);
    p.dk2 = tensor(a->dk2, a->dk2_stride);
    p.dv2 = tensor(a->dv2, a->dv2_stride);
  }
  p.lse = a->lse;
  p.ls_b = a->lse_stride.b; p.ls_h = a->lse_stride.h; p.ls_s = a->lse_stride.s;
  p.dlse = a->dlse;
  p.dl_b = a->dlse_stride.b; p.dl_h = a->dlse_stride.h; p.dl_s = a->dlse_stride.s;
  p.B = a->B; p.H = a->H; p.D = a->D;
  p.scale = a->softmax_scale;
  unsigned char* ws = (unsigned char*)a->workspace;
  p.stats = (float*)ws;
  if (plan.norms) p.value_norms = (float*)(ws + plan.stats);
  p.keys.partial = (float*)(ws + plan.stats + plan.norms);
  p.queries.partial = (float*)(ws + plan.stats + plan.norms + plan.keys);
  hipStream_t stream = (hipStream_t)a->stream;
  const hipError_t e = a->dtype == XDIT_DTYPE_FP32 ? xdit::launch_attn_bwd_f32(p, stream)
                                                   : xdit::launch_attn_bwd_16(p, a->dtype == XDIT_DTYPE_FP16, stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "attention backward launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

}  // extern "C"
