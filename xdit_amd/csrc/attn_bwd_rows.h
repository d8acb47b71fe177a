// Row-wise kernels of attention's backward pass, before and behind its products.
#pragma once
#include "attn_bwd.h"
#include "row_ops.h"

namespace xdit {
namespace {

// lse / ln 2 and -delta of every row; rows up to the padded count get (infinity, 0), whose probabilities are zeros.  A row whose
// log-sum-exp is -infinity attended nothing: the same.  fp16: also the largest |dout| of the block's rows.
template <typename T>
__global__ __launch_bounds__(256) void bwd_stats_kernel(const AttnBwdParams p) {
  const int lpr = p.D > 64 ? 16 : 8;   // lanes per row, 8 columns each
  const int blocks = p.sq_pad / kBwdStatRows;
  const int bh = blockIdx.x / blocks, block = blockIdx.x - bh * blocks;
  const int b = bh / p.H, h = bh - b * p.H;
  const int sub = threadIdx.x & (lpr - 1);
  float top = 0.f;
  for (int r = threadIdx.x / lpr; r < kBwdStatRows; r += 256 / lpr) {
    const int row = block * kBwdStatRows + r;
    float dot = 0.f;
    if (row < p.Sq && sub * 8 < p.D) {
      const Raw8<T> o = load_raw8<T>(p.out.p, b * p.out.b + h * p.out.h + (int64_t)row * p.out.s + sub * 8);
      const Raw8<T> g = load_raw8<T>(p.dout.p, b * p.dout.b + h * p.dout.h + (int64_t)row * p.dout.s + sub * 8);
#pragma unroll
      for (int e = 0; e < 8; e++) {
        dot = __builtin_fmaf(o[e], g[e], dot);
        top = fmaxf(top, __builtin_fabsf(g[e]));
      }
    }
    for (int m = 1; m < lpr; m <<= 1) dot += __shfl_xor(dot, m);
    if (sub == 0) {
      float lse2 = INFINITY, nd = 0.f;
      if (row < p.Sq) {
        const float l = p.lse[b * p.ls_b + h * p.ls_h + row * p.ls_s];
        if (l != -INFINITY) {
          lse2 = l * kLog2e;
          nd = (p.dlse != nullptr ? p.dlse[b * p.dl_b + h * p.dl_h + row * p.dl_s] : 0.f) - dot;
        }
      }
      float* st = p.stats + (int64_t)bh * 2 * p.sq_pad + row;
      st[0] = lse2;
      st[p.sq_pad] = nd;
    }
  }
  if (p.amax != nullptr) {
    __shared__ float tops[4];
    for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
    if (threadIdx.x == 0) p.amax[(int64_t)bh * blocks + block] = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
  }
}

// Adds the parts of every row up, in their order, and rounds.
template <typename T, int DC, bool KEYS>
__global__ __launch_bounds__(256) void bwd_fold_kernel(const AttnBwdParams p, int rows_per_tile) {
  typedef __attribute__((ext_vector_type(4))) T vec4;
  const BwdRole& R = KEYS ? p.keys : p.queries;
  const int per_tile = (rows_per_tile * (DC / 4) + 255) / 256;
  const int bt = blockIdx.x / per_tile;
  const int bh = bt / R.tiles;
  int tile = bt - bh * R.tiles;
  const int b = bh / p.H, h = bh - b * p.H;
  const int which = blockIdx.y;
  const int i = (blockIdx.x - bt * per_tile) * 256 + threadIdx.x;
  const int row = i / (DC / 4), col = (i % (DC / 4)) * 4;
  const bool second = KEYS && tile >= p.tiles1;
  if (second) tile -= p.tiles1;
  const int rows = KEYS ? (second ? p.Sk2 : p.Sk) : p.Sq;
  const int own = tile * rows_per_tile + row;
  if (row >= rows_per_tile || own >= rows || col >= p.D) return;
  const int tensors = KEYS ? 2 : 1;
  const float* src = R.partial + ((int64_t)bt * R.parts * tensors + which) * rows_per_tile * DC + (int64_t)row * DC + col;
  f32x4 x = *(const f32x4*)src;
  for (int n = 1; n < R.parts; n++) x += *(const f32x4*)(src + (int64_t)n * tensors * rows_per_tile * DC);
  const BwdTensor& O = KEYS ? (which ? (second ? p.dv2 : p.dv) : (second ? p.dk2 : p.dk)) : p.dq;
  *(vec4*)((T*)O.p + b * O.b + h * O.h + (int64_t)own * O.s + col) = __builtin_convertvector(x, vec4);
}

}  // namespace
}  // namespace xdit
