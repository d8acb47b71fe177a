// Parameters of attention's backward pass, shared between its kernels and the C ABI.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "common.h"

namespace xdit {

struct BwdTensor {  // a logical (B, H, S, D) tensor with a unit stride over D
  void* p;
  int64_t b, h, s;
};

// The work of one role (see attn_bwd_16.hip): every (batch, head) has `tiles` row tiles, whose streamed range of
// `steps` tiles is cut into `parts` parts of `len` tiles.
struct BwdRole {
  int tiles, steps, parts, len;
  float* partial;  // parts > 1: [(bh, tile)][part][tensor][row][column] in fp32, folded by a launch of its own
};

struct AttnBwdParams {
  BwdTensor q, k, v, k2, v2, out, dout;
  BwdTensor dq, dk, dv, dk2, dv2;  // p == nullptr: not asked for
  const float* lse;
  const float* dlse;               // may be null
  int64_t ls_b, ls_h, ls_s;
  int64_t dl_b, dl_h, dl_s;
  int B, H, Sq, Sk, Sk2, D;
  float scale;
  int sq_pad;         // Sq rounded up to whole tiles
  float* stats;       // workspace: per (batch, head) lse / ln 2 of every row, then -delta of every row, sq_pad of each
  float* amax;        // workspace, fp16: largest |dout| of every block of kBwdStatRows rows of a (batch, head)
  int tiles1;         // row tiles of the first segment of keys
  int step1;          // streamed tiles of the first segment of keys
  BwdRole keys;       // row tiles of keys, queries streamed: dk and dv
  BwdRole queries;    // row tiles of queries, keys streamed: dq
};

constexpr int kBwdStatRows = 64;  // rows of a workgroup of the statistics kernel

hipError_t launch_attn_bwd_16(const AttnBwdParams& p, int dtype_is_fp16, int waves, hipStream_t stream);
hipError_t launch_attn_bwd_f32(const AttnBwdParams& p, hipStream_t stream);

}  // namespace xdit
