// The C entries of a training step with launchers that launch nothing, for tests without a GPU: which calls are taken, and what their rows share.
// Compiled for the host alone, together with the entries' own source.
#include "../xdit_amd/csrc/train_api.hip"

#include <cstdarg>
#include <cstdio>

static char message[256];

namespace xdit {
void api_clear_error() { message[0] = 0; }
int api_fail(int code, const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  std::vsnprintf(message, sizeof(message), fmt, ap);
  va_end(ap);
  return code;
}
int api_check_tensor(const char*, const void*, const xdit_strides&, int, int) { return 0; }
hipError_t launch_attn_bwd_16(const AttnBwdParams&, int, hipStream_t) { return hipSuccess; }
hipError_t launch_attn_bwd_f32(const AttnBwdParams&, hipStream_t) { return hipSuccess; }
hipError_t launch_grad_norm(const NormParams&, int, unsigned, hipStream_t) { return hipSuccess; }
hipError_t launch_grad_norm_total(const double*, int64_t, int, float*, hipStream_t) { return hipSuccess; }
hipError_t launch_grad_clip(const ClipParams&, int, int, unsigned, hipStream_t) { return hipSuccess; }
}  // namespace xdit

extern "C" {

const char* host_message() { return message; }

// Whether two tensors, each told by address, bytes of a row, and count and stride of three axes, share a byte.
int host_share_bytes(const int64_t* x, const int64_t* y) {
  auto rows = [](const int64_t* v) { return Rows{(uintptr_t)v[0], v[1], {{v[2], v[3]}, {v[4], v[5]}, {v[6], v[7]}}}; };
  return share_bytes(rows(x), rows(y));
}

// Groups of 8 columns that an fp32 call of this head_dim is computed with.
int host_f32_groups(int D) { return xdit::bwd_f32_groups(D); }

// How a call of attention's backward pass is cut up: for either role tiles of a (batch, head), steps, all tiles, tiles of an XCD, of those whole ones, parts, their
// length, units of an XCD; then the workspace's bytes of partial results of either role.
void host_plan(const xdit_attn_bwd_args* a, int64_t* out) {
  xdit::AttnBwdParams p;
  std::memset(&p, 0, sizeof(p));
  const BwdPlan plan = plan_bwd(a, p);
  for (const xdit::BwdRole* r : {&p.keys, &p.queries})
    for (int64_t x : {r->tiles, r->steps, r->total, r->per_xcd, r->whole, r->parts, r->len, r->units}) *out++ = x;
  *out++ = plan.keys;
  *out++ = plan.queries;
}

// Walks through the units of a plan as the kernels do -> 0, or what is wrong with it first.
int host_walk(const xdit_attn_bwd_args* a) {
  xdit::AttnBwdParams p;
  std::memset(&p, 0, sizeof(p));
  const BwdPlan plan = plan_bwd(a, p);
  const int dc = a->dtype == XDIT_DTYPE_FP32 ? (xdit::bwd_f32_groups(a->D) + 1) / 2 * 16 : (a->D + 31) / 32 * 32;
  for (int role = 0; role < 2; role++) {
    const xdit::BwdRole& r = role ? p.queries : p.keys;
    if (r.total == 0) {
      if (r.units) return 1;   // units of a role that is not asked for
      continue;
    }
    const int64_t cut = xdit::bwd_cut_tiles(r), slots = cut * r.parts;
    if ((role ? plan.queries : plan.keys) != slots * (2 - role) * xdit::kBwdRows * dc * 4) return 2;   // other than the slots take
    std::vector<char> steps((size_t)r.total * r.steps, 0), written((size_t)slots, 0);
    // the tile that the sum of the parts takes a cut one for
    auto tile_of = [&](int64_t c) { return r.whole == 0 ? c : c / (r.per_xcd - r.whole) * r.per_xcd + r.whole + c % (r.per_xcd - r.whole); };
    for (int xcd = 0; xcd < 8; xcd++)
      for (int n = 0; n < r.units; n++) {
        xdit::BwdUnit u;
        if (!xdit::bwd_unit(r, xcd, n, u)) continue;
        const int first = u.slot < 0 ? 0 : u.part * r.len, last = u.slot < 0 || first + r.len > r.steps ? r.steps : first + r.len;
        if (u.tile < 0 || u.tile >= r.total || first >= last) return 3;   // nothing to do, or no such tile
        if (u.slot >= slots || (u.slot >= 0 && written[u.slot]++)) return 4;   // a slot outside the workspace, or one twice
        if (u.slot >= 0 && (tile_of(u.slot / r.parts) != u.tile || u.slot % r.parts != u.part)) return 5;   // added up as another's
        for (int t = first; t < last; t++)
          if (steps[(size_t)u.tile * r.steps + t]++) return 6;   // a step twice
      }
    for (char c : steps)
      if (c != 1) return 7;   // a step left out
    for (int64_t c = 0; c < cut; c++)
      for (int k = 0; k < r.parts; k++)
        if (tile_of(c) < r.total && !written[c * r.parts + k]) return 8;   // a part that is added up and that no unit writes
  }
  return 0;
}

}  // extern "C"
