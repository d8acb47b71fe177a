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

// The work of one role (see attn_bwd_16.hip).  Every (batch, head) has `tiles` row tiles that stream `steps` tiles each.  An XCD takes
// `per_xcd` consecutive tiles of all (batch, head)s: the first `whole` of them are one unit each, the ranges of the others are cut into
// `parts` units of `len` steps, whose fp32 results a launch of its own adds up.  Where all tiles are cut (`whole` 0), an XCD takes consecutive
// units of them instead, so that a few tiles occupy all XCDs.
struct BwdRole {
  int tiles, steps;
  int total;            // tiles of all (batch, head)s; 0: the role's gradients are not asked for
  int per_xcd, whole, parts, len;
  int units;            // per XCD
  float* partial;       // [cut tile][part][tensor][128 rows of computed columns (PartLayout)]
};

// Tiles that are cut: all of them, or those behind every XCD's `whole` (some of the last XCD's may not exist).
__host__ __device__ __forceinline__ int bwd_cut_tiles(const BwdRole& r) { return r.parts == 1 ? 0 : r.whole == 0 ? r.total : 8 * (r.per_xcd - r.whole); }

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
  float* stats;       // workspace: per (batch, head) lse / ln 2 of every row (fp16: less kFp16Exponent), then -delta of every row, sq_pad of each
  float* value_norms; // workspace, fp16: of every block of kBwdStatRows keys of every (batch, head) the largest norm of a row of v
  int tiles1;         // row tiles of the first segment of keys
  int step1;          // streamed tiles of the first segment of keys
  BwdRole keys;       // row tiles of keys, queries streamed: dk and dv
  BwdRole queries;    // row tiles of queries, keys streamed: dq
};

// fp16's numbers end at 2^-24, and P is small: it is computed times 2^15 (it stays below 65504, fp16's last number, up to 1.999) where it
// is rounded (attn_bwd_16.hip).
constexpr int kFp16Exponent = 15;
constexpr int kBwdStatRows = 64;  // rows of a workgroup of the statistics kernel
constexpr int kBwdWaves = 4;      // wavefronts of a workgroup, 32 owned rows each
constexpr int kBwdRows = 32 * kBwdWaves;

// fp32: groups of 8 columns that a head_dim is computed with, those that it has (up to 32: four, whose others are zeros); its gradients
// have blocks of 16.  An odd number of them against the even one above it, 16 heads of 4096: head_dim 40 1225 against 1342 us, 56 1643
// against 1756, 72 2053 against 2169, 88 2475 against 2600, 104 3165 against 3255, 120 3570 against 3677.
inline int bwd_f32_groups(int D) { return D <= 32 ? 4 : D / 8; }

// Blocks of kBwdStatRows rows of a (batch, head)'s values, both segments.
__host__ __device__ __forceinline__ int bwd_value_blocks(const AttnBwdParams& p) {
  return (p.Sk + kBwdStatRows - 1) / kBwdStatRows + (p.Sk2 + kBwdStatRows - 1) / kBwdStatRows;
}

// A unit's tile (of all), part and slot of its partial result; false for the units that an XCD's last tiles do not have.
struct BwdUnit {
  int tile, part;
  int64_t slot;   // < 0: a whole tile
};
__host__ __device__ __forceinline__ bool bwd_unit(const BwdRole& r, int xcd, int n, BwdUnit& u) {
  int t = n;
  u.part = 0;
  u.slot = -1;
  if (r.whole == 0 && r.parts > 1) {
    const int id = xcd * r.units + n;
    u.tile = id / r.parts;
    u.part = id - u.tile * r.parts;
    u.slot = id;
    return u.tile < r.total;
  }
  if (n >= r.whole) {
    const int i = (n - r.whole) / r.parts;
    t = r.whole + i;
    u.part = n - r.whole - i * r.parts;
    if (r.parts > 1) u.slot = ((int64_t)xcd * (r.per_xcd - r.whole) + i) * r.parts + u.part;
  }
  u.tile = xcd * r.per_xcd + t;
  return u.tile < r.total;
}

hipError_t launch_attn_bwd_16(const AttnBwdParams& p, int dtype_is_fp16, hipStream_t stream);
hipError_t launch_attn_bwd_f32(const AttnBwdParams& p, hipStream_t stream);

}  // namespace xdit
