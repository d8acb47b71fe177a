// Row-wise kernels of attention's backward pass, before and behind its products.
#pragma once
#include "attn_bwd.h"
#include "row_ops.h"

namespace xdit {
namespace {

// The largest norm of a row of block n of all (batch, head)s' values.
template <typename T, int LPR>
__device__ __forceinline__ void value_norm(const AttnBwdParams& p, int n) {
  constexpr int STEP = 256 / LPR, PASSES = kBwdStatRows / STEP;
  const int blocks = bwd_value_blocks(p), heads = p.B * p.H;
  const bool by_token = p.v.h < p.v.s;
  const int bh = by_token ? n % heads : n / blocks;
  int block = by_token ? n / heads : n - bh * blocks;
  const int b = bh / p.H, h = bh - b * p.H;
  float* const dst = p.value_norms + (int64_t)bh * blocks + block;
  const int blocks1 = (p.Sk + kBwdStatRows - 1) / kBwdStatRows;
  const bool second = block >= blocks1;
  if (second) block -= blocks1;
  const BwdTensor& V = second ? p.v2 : p.v;
  const int rows = second ? p.Sk2 : p.Sk, sub = threadIdx.x & (LPR - 1);
  const T* const vp = (const T*)V.p + b * V.b + h * V.h + sub * 8;
  float squares[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; i++) squares[i] = 0.f;
  if (sub * 8 < p.D) {
    Raw8<T> v[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; i++) {
      int row = block * kBwdStatRows + threadIdx.x / LPR + i * STEP;
      row = row < rows ? row : rows - 1;
      v[i] = load_raw8<T>(vp, (int64_t)row * V.s);
    }
#pragma unroll
    for (int i = 0; i < PASSES; i++)
#pragma unroll
      for (int e = 0; e < 8; e++) squares[i] = __builtin_fmaf(v[i][e], v[i][e], squares[i]);
  }
  float top = 0.f;
#pragma unroll
  for (int i = 0; i < PASSES; i++) {
    for (int m = 1; m < LPR; m <<= 1) squares[i] += __shfl_xor(squares[i], m);
    top = fmaxf(top, squares[i]);
  }
  __shared__ float tops[4];
  for (int m = LPR; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  if (threadIdx.x == 0) *dst = __builtin_sqrtf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
}

// lse / ln 2 and -delta of every row; rows up to the padded count get (infinity, 0), whose probabilities are zeros.  A row whose
// log-sum-exp is -infinity attended nothing: the same.  fp16: further blocks look at the values (value_norm). Reading out and dout bounds
// it: all loads of a thread are asked for at once, `out`, which nothing reads again, past the caches' replacement order, and where the
// heads of a token lie side by side, blocks that run together take all heads of their tokens (40 heads of 32760 x 128, BSHD: 139 us with
// two loads at a time and head by head, 126 so).  LPR: lanes per row, 8 columns each.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void bwd_stats_kernel(const AttnBwdParams p) {
  constexpr int STEP = 256 / LPR, PASSES = kBwdStatRows / STEP;
  const int blocks = p.sq_pad / kBwdStatRows, heads = p.B * p.H;
  constexpr bool FP16 = __is_same(T, _Float16);
  if constexpr (FP16) {
    if ((int)blockIdx.x >= heads * blocks) return value_norm<T, LPR>(p, blockIdx.x - heads * blocks);
  }
  const bool by_token = p.dout.h < p.dout.s;
  const int bh = by_token ? blockIdx.x % heads : blockIdx.x / blocks;
  const int block = by_token ? blockIdx.x / heads : blockIdx.x - bh * blocks;
  const int b = bh / p.H, h = bh - b * p.H;
  const int sub = threadIdx.x & (LPR - 1);
  const int row0 = block * kBwdStatRows + threadIdx.x / LPR;
  const T* const op = (const T*)p.out.p + b * p.out.b + h * p.out.h + sub * 8;
  const T* const gp = (const T*)p.dout.p + b * p.dout.b + h * p.dout.h + sub * 8;
  Raw8<T> o[PASSES], g[PASSES];
  float lse[PASSES], dlse[PASSES];
#pragma unroll
  for (int i = 0; i < PASSES; i++) {
    int row = row0 + i * STEP;
    row = row < p.Sq ? row : p.Sq - 1;
    if (sub * 8 < p.D) {
#pragma unroll
      for (int n = 0; n < Raw8<T>::N; n++) o[i].x[n] = __builtin_nontemporal_load((const typename Raw8<T>::vec*)(op + (int64_t)row * p.out.s) + n);
      g[i] = load_raw8<T>(gp, (int64_t)row * p.dout.s);
    } else {
#pragma unroll
      for (int n = 0; n < Raw8<T>::N; n++) o[i].x[n] = g[i].x[n] = (typename Raw8<T>::vec)(T)0.f;
    }
    lse[i] = p.lse[b * p.ls_b + h * p.ls_h + row * p.ls_s];
    dlse[i] = p.dlse != nullptr ? p.dlse[b * p.dl_b + h * p.dl_h + row * p.dl_s] : 0.f;
  }
#pragma unroll
  for (int i = 0; i < PASSES; i++) {
    const int row = row0 + i * STEP;
    float dot = 0.f;
#pragma unroll
    for (int e = 0; e < 8; e++) dot = __builtin_fmaf(o[i][e], g[i][e], dot);
    for (int m = 1; m < LPR; m <<= 1) dot += __shfl_xor(dot, m);
    const bool live = row < p.Sq && lse[i] != -INFINITY;
    if (sub == 0) {
      float* st = p.stats + (int64_t)bh * 2 * p.sq_pad + row;
      st[0] = live ? lse[i] * kLog2e - (FP16 ? (float)kFp16Exponent : 0.f) : INFINITY;
      st[p.sq_pad] = live ? dlse[i] - dot : 0.f;
    }
  }
}

template <typename T>
void launch_bwd_stats(const AttnBwdParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)(p.B * p.H) * (p.sq_pad / kBwdStatRows + (__is_same(T, _Float16) ? bwd_value_blocks(p) : 0)));
  if (p.D > 64) hipLaunchKernelGGL((bwd_stats_kernel<T, 16>), grid, dim3(256), 0, stream, p);
  else hipLaunchKernelGGL((bwd_stats_kernel<T, 8>), grid, dim3(256), 0, stream, p);
}

// A part's result for 128 rows of DC columns, in units of four columns as the accumulators of its wavefronts hold them, so that a store
// covers 1 KiB (as rows, in pieces of 32 bytes: 4 heads of 1024 32.1 us a call, so 31.2; 24 of 4608 772, so 770).  BLOCK: the columns and
// rows of an accumulator.
template <int DC, int BLOCK> struct PartLayout {
  static __device__ __forceinline__ void place(int i, int& row, int& col) {
    constexpr int BLOCKS = DC / BLOCK;
    const int lane = i & 63, m = i >> 6;
    if (BLOCK == 32) {
      row = m / (4 * BLOCKS) * 32 + (lane & 31);
      col = m / 4 % BLOCKS * 32 + m % 4 * 8 + (lane >> 5) * 4;
    } else {
      row = m / BLOCKS * 16 + (lane & 15);
      col = m % BLOCKS * 16 + (lane >> 4) * 4;
    }
  }
};

// Adds the parts of every row of the tiles that were cut up, in their order, and rounds.  Blocks of the keys role first, dk and dv of a
// tile side by side, then those of the queries role.  The parts' reading bounds it: 63 MB (40 heads of 32760 on 512) 15.6 us, 38 MB (fp32,
// 16 heads of 1024 at head_dim 72) 8.2.
template <typename T, int DC, int BLOCK>
__global__ __launch_bounds__(256) void bwd_fold_kernel(const AttnBwdParams p) {
  typedef __attribute__((ext_vector_type(4))) T vec4;
  constexpr int BLOCKS = kBwdRows * (DC / 4) / 256;   // of a tile's gradient
  int n = blockIdx.x / BLOCKS;
  const int i = (blockIdx.x - n * BLOCKS) * 256 + threadIdx.x;
  int row, col;
  PartLayout<DC, BLOCK>::place(i, row, col);
  const int from_keys = bwd_cut_tiles(p.keys) * 2;
  const bool keys = n < from_keys;
  const BwdRole& R = keys ? p.keys : p.queries;
  const int tensors = keys ? 2 : 1;
  if (!keys) n -= from_keys;
  const int which = n % tensors, cut = n / tensors;
  const int xcd = cut / (R.per_xcd - R.whole), t = cut - xcd * (R.per_xcd - R.whole);
  const int bt = R.whole == 0 ? cut : xcd * R.per_xcd + R.whole + t;
  if (bt >= R.total) return;
  const int bh = bt / R.tiles;
  int tile = bt - bh * R.tiles;
  const int b = bh / p.H, h = bh - b * p.H;
  const bool second = keys && tile >= p.tiles1;
  if (second) tile -= p.tiles1;
  const int rows = keys ? (second ? p.Sk2 : p.Sk) : p.Sq;
  const int own = tile * kBwdRows + row;
  if (own >= rows || col >= p.D) return;
  const float* src = R.partial + ((int64_t)cut * R.parts * tensors + which) * kBwdRows * DC + i * 4;
  f32x4 x = *(const f32x4*)src;
#pragma unroll 4
  for (int k = 1; k < R.parts; k++) x += *(const f32x4*)(src + (int64_t)k * tensors * kBwdRows * DC);
  const BwdTensor& O = keys ? (which ? (second ? p.dv2 : p.dv) : (second ? p.dk2 : p.dk)) : p.dq;
  *(vec4*)((T*)O.p + b * O.b + h * O.h + (int64_t)own * O.s + col) = __builtin_convertvector(x, vec4);
}

template <typename T, int DC, int BLOCK>
hipError_t launch_bwd_fold(const AttnBwdParams& p, hipStream_t stream) {
  const int tiles = bwd_cut_tiles(p.keys) * 2 + bwd_cut_tiles(p.queries);
  if (tiles) hipLaunchKernelGGL((bwd_fold_kernel<T, DC, BLOCK>), dim3((unsigned)tiles * (kBwdRows * (DC / 4) / 256)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace
}  // namespace xdit
