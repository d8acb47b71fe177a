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

// Cuts the streamed steps of every row tile into parts so that the units fill the compute units.  A unit costs its steps and about
// two more (operands, first tile, results); a call in parts also writes and reads fp32 partial results, `fold` steps' time a unit for a
// compute unit, and has one launch more.  The cheapest number of parts, at most four units per compute unit.
void plan_role(xdit::BwdRole& r, int64_t bh, int cus, double fold) {
  const int64_t base = bh * r.tiles;
  double best = -1;
  for (int parts = 1; parts <= r.steps && parts <= 64 && (parts == 1 || base * parts <= 4 * (int64_t)cus); parts++) {
    const int len = (r.steps + parts - 1) / parts;
    const int n = (r.steps + len - 1) / len;
    if (n != parts) continue;
    const double rounds = (double)((base * n + cus - 1) / cus);
    const double cost = rounds * (len + 2.0) + (n > 1 ? rounds * fold + 1.0 : 0.0);
    if (best < 0 || cost < best) { best = cost; r.parts = n; r.len = len; }
  }
}

struct BwdPlan {
  int waves;
  int64_t stats, amax, partial;   // bytes
};

BwdPlan plan_bwd(const xdit_attn_bwd_args* a, xdit::AttnBwdParams& p) {
  BwdPlan plan;
  const bool f32 = a->dtype == XDIT_DTYPE_FP32;
  plan.waves = f32 ? 4 : 8;
  const int rows = 32 * plan.waves, step = f32 ? 32 : 64;
  const int dc = (a->D + 31) / 32 * 32;
  const int64_t bh = (int64_t)a->B * a->H;
  const int cus = xdit::resident_cus(a->cu_count);
  p.tiles1 = (int)((a->Sk + rows - 1) / rows);
  p.keys.tiles = p.tiles1 + (int)((a->Sk2 + rows - 1) / rows);
  p.keys.steps = (int)((a->Sq + step - 1) / step);
  p.queries.tiles = (int)((a->Sq + rows - 1) / rows);
  p.step1 = (int)((a->Sk + step - 1) / step);
  p.queries.steps = p.step1 + (int)((a->Sk2 + step - 1) / step);
  plan_role(p.keys, bh, cus, 4.0);
  plan_role(p.queries, bh, cus, 2.0);
  p.sq_pad = (int)((a->Sq + xdit::kBwdStatRows - 1) / xdit::kBwdStatRows * xdit::kBwdStatRows);
  plan.stats = align256(bh * 2 * p.sq_pad * 4);
  plan.amax = a->dtype == XDIT_DTYPE_FP16 ? align256(bh * (p.sq_pad / xdit::kBwdStatRows) * 4) : 0;
  const int64_t pk = a->dk != nullptr && p.keys.parts > 1 ? bh * p.keys.tiles * p.keys.parts * 2 * rows * dc * 4 : 0;
  const int64_t pq = a->dq != nullptr && p.queries.parts > 1 ? bh * p.queries.tiles * p.queries.parts * rows * dc * 4 : 0;
  plan.partial = pk > pq ? pk : pq;   // the roles run one after the other
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

// Whether no destination overlaps another one, or a source other than itself.
bool destinations_apart(const xdit_clip_grads_args* a) {
  struct Span { uintptr_t begin, end; int64_t i; };
  std::vector<Span> dst;
  dst.reserve(a->count);
  for (int64_t i = 0; i < a->count; i++)
    if (a->numel[i]) dst.push_back({reinterpret_cast<uintptr_t>(a->dst[i]), reinterpret_cast<uintptr_t>(a->dst[i]) + a->numel[i] * size_of(a->dst_dtype[i]), i});
  std::sort(dst.begin(), dst.end(), [](const Span& x, const Span& y) { return x.begin < y.begin; });
  for (size_t n = 1; n < dst.size(); n++)
    if (dst[n].begin < dst[n - 1].end) return false;
  for (int64_t i = 0; i < a->count; i++) {
    if (a->numel[i] == 0) continue;
    const uintptr_t begin = reinterpret_cast<uintptr_t>(a->src[i]), end = begin + a->numel[i] * size_of(a->src_dtype[i]);
    auto at = std::upper_bound(dst.begin(), dst.end(), begin, [](uintptr_t x, const Span& s) { return x < s.end; });   // the first that ends behind the source's start
    for (; at != dst.end() && at->begin < end; ++at)
      if (at->i != i || at->begin != begin || a->src_dtype[i] != a->dst_dtype[i]) return false;
  }
  return true;
}

}  // namespace

extern "C" {

int64_t xdit_grad_norm_workspace_bytes(const xdit_grad_norm_args* a) {
  xdit::api_clear_error();
  if (int rc = check_norm_list(a)) return rc;
  const int64_t chunk = chunk_elements(a->count, a->numel);
  int64_t n = 0;
  for (int64_t i = 0; i < a->count; i++) n += chunks_of(a->numel[i], chunk);
  return n * (int64_t)sizeof(double);
}

int xdit_grad_norm(const xdit_grad_norm_args* a) {
  xdit::api_clear_error();
  if (int rc = check_norm_list(a)) return rc;
  if (a->norm == nullptr || reinterpret_cast<uintptr_t>(a->norm) & 3u) return api_fail(XDIT_ERR_INVALID_ARG, "norm is NULL or not 4-byte aligned");
  const int64_t chunk = chunk_elements(a->count, a->numel);
  int64_t need = 0;
  for (int64_t i = 0; i < a->count; i++) need += chunks_of(a->numel[i], chunk);
  if (need && (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 7u) || a->workspace_bytes < need * (int64_t)sizeof(double)))
    return api_fail(XDIT_ERR_INVALID_ARG, "workspace must be 8-byte aligned and hold %lld bytes", (long long)(need * sizeof(double)));
  hipStream_t stream = (hipStream_t)a->stream;
  hipError_t e = hipSuccess;
  double* partial = (double*)a->workspace;
  xdit::NormParams p;
  p.chunk = (int)chunk;
  p.kind = a->kind;
  for (int dtype = XDIT_DTYPE_BF16; dtype <= XDIT_DTYPE_FP32; dtype++) {   // a launch holds tensors of one dtype
    int n = 0;
    int64_t chunks = 0;
    for (int64_t i = 0; i <= a->count; i++) {
      const bool takes = i < a->count && a->dtype[i] == dtype && a->numel[i] != 0;
      const int64_t more = takes ? chunks_of(a->numel[i], chunk) : 0;
      if (n && (i == a->count || (takes && (n == xdit::kNormTensors || chunks + more > (1 << 30))))) {
        std::fill(p.t.first + n, p.t.first + xdit::kNormTensors, 0xffffffffu);
        p.partial = partial;
        if ((e = xdit::launch_grad_norm(p, dtype, (unsigned)chunks, stream)) != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "gradient norm launch failed: %s", hipGetErrorString(e));
        partial += chunks;
        n = 0;
        chunks = 0;
      }
      if (takes) {
        p.t.first[n] = (uint32_t)chunks;
        p.t.numel[n] = a->numel[i];
        p.t.src[n++] = a->data[i];
        chunks += more;
      }
    }
  }
  if ((e = xdit::launch_grad_norm_total((const double*)a->workspace, need, a->kind, a->norm, stream)) != hipSuccess)
    return api_fail(XDIT_ERR_LAUNCH, "gradient norm launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

int xdit_clip_grads(const xdit_clip_grads_args* a) {
  xdit::api_clear_error();
  if (a == nullptr) return api_fail(XDIT_ERR_INVALID_ARG, "args is NULL");
  if (a->struct_size != sizeof(xdit_clip_grads_args))
    return api_fail(XDIT_ERR_INVALID_ARG, "struct_size %u != %zu (ABI mismatch)", a->struct_size, sizeof(xdit_clip_grads_args));
  if (a->count < 0 || a->count > (1 << 24)) return api_fail(XDIT_ERR_INVALID_ARG, "count %lld must lie between 0 and 2^24", (long long)a->count);
  if (!(a->max_norm >= 0.f) || !std::isfinite(a->max_norm)) return api_fail(XDIT_ERR_INVALID_ARG, "max_norm must be finite and >= 0");
  if (a->norm == nullptr || reinterpret_cast<uintptr_t>(a->norm) & 3u) return api_fail(XDIT_ERR_INVALID_ARG, "norm is NULL or not 4-byte aligned");
  if (a->count == 0) return XDIT_OK;
  int rc;
  if ((rc = check_list("gradient", a->count, const_cast<void* const*>(a->src), a->numel, a->src_dtype))) return rc;
  if ((rc = check_list("result", a->count, a->dst, a->numel, a->dst_dtype))) return rc;
  try {
    if (!destinations_apart(a)) return api_fail(XDIT_ERR_INVALID_ARG, "a result overlaps another one, or a gradient other than its own");
  } catch (const std::bad_alloc&) {
    return api_fail(XDIT_ERR_INVALID_ARG, "no host memory for %lld tensors", (long long)a->count);
  }
  hipStream_t stream = (hipStream_t)a->stream;
  const int64_t chunk = chunk_elements(a->count, a->numel);
  xdit::ClipParams p;
  p.chunk = (int)chunk;
  p.max_norm = a->max_norm;
  p.norm = a->norm;
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
  return plan.stats + plan.amax + plan.partial;
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
  if (reinterpret_cast<uintptr_t>(a->lse) & 3u || reinterpret_cast<uintptr_t>(a->dlse) & 3u)
    return api_fail(XDIT_ERR_INVALID_ARG, "lse and dlse must be 4-byte aligned");
  if (a->lse_stride.b < 0 || a->lse_stride.h < 0 || a->lse_stride.s < 0 || a->dlse_stride.b < 0 || a->dlse_stride.h < 0 || a->dlse_stride.s < 0)
    return api_fail(XDIT_ERR_INVALID_ARG, "lse and dlse: negative stride");

  xdit::AttnBwdParams p;
  std::memset(&p, 0, sizeof(p));
  const BwdPlan plan = plan_bwd(a, p);
  const int64_t need = plan.stats + plan.amax + plan.partial;
  if (a->workspace == nullptr || (reinterpret_cast<uintptr_t>(a->workspace) & 15u) || a->workspace_bytes < need)
    return api_fail(XDIT_ERR_INVALID_ARG, "workspace must be 16-byte aligned and hold %lld bytes", (long long)need);
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
  p.Sq = (int)a->Sq; p.Sk = (int)a->Sk; p.Sk2 = (int)a->Sk2;
  p.scale = a->softmax_scale;
  unsigned char* ws = (unsigned char*)a->workspace;
  p.stats = (float*)ws;
  if (plan.amax) p.amax = (float*)(ws + plan.stats);
  p.keys.partial = p.queries.partial = (float*)(ws + plan.stats + plan.amax);
  hipStream_t stream = (hipStream_t)a->stream;
  const hipError_t e = a->dtype == XDIT_DTYPE_FP32 ? xdit::launch_attn_bwd_f32(p, stream)
                                                   : xdit::launch_attn_bwd_16(p, a->dtype == XDIT_DTYPE_FP16, plan.waves, stream);
  if (e != hipSuccess) return api_fail(XDIT_ERR_LAUNCH, "attention backward launch failed: %s", hipGetErrorString(e));
  return XDIT_OK;
}

}  // extern "C"
