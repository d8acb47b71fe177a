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

}  // extern "C"
