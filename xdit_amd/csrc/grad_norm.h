// Parameters of the gradient norm and of clipping, shared between their kernels and the C ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace xdit {

// A launch takes its tensors in the kernel arguments (below 4 KiB of them), so that a captured call needs no table in memory.
constexpr int kNormTensors = 184;
constexpr int kClipTensors = 136;

template <int N> struct GradTable {
  uint32_t first[N];   // first chunk of every tensor; unused entries 0xffffffff
  int64_t numel[N];
  const void* src[N];
};

struct NormParams {
  GradTable<kNormTensors> t;
  int chunk;           // elements of a workgroup
  int kind;            // 0 maximum, 1 sum of sizes, 2 sum of squares
  double* partial;     // one per workgroup, from this launch's first on
  unsigned* counter;   // not null: the launch's last workgroup to finish adds all partial sums up (there are no others), writes the norm and clears it
  float* norm;
};

constexpr int kClipPartials = 1024;  // partial sums that the workgroups of a clipping launch, or the last one of a norm's, add up by themselves

struct ClipParams {
  GradTable<kClipTensors> t;
  void* dst[kClipTensors];
  int chunk;
  float max_norm;
  const float* norm;      // given, or written by an earlier launch; nullptr: of `partial`
  const double* partial;  // at most kClipPartials partial sums
  int partials, kind;
  float* norm_out;        // receives the norm of `partial` (nullptr: another launch writes it)
};

hipError_t launch_grad_norm(const NormParams& p, int dtype, unsigned workgroups, hipStream_t stream);
hipError_t launch_grad_norm_total(const double* partial, int64_t n, int kind, float* norm, hipStream_t stream);
hipError_t launch_grad_clip(const ClipParams& p, int src_dtype, int dst_dtype, unsigned workgroups, hipStream_t stream);

}  // namespace xdit
