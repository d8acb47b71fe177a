// Backward pass of the attention forward for fp32 tensors: the formulas, roles and partial results of the 16-bit kernel
// (attn_bwd_16.hip) on v_mfma_f32_32x32x2_f32, with everything in fp32.
//
// Lane l of that instruction holds row/column l%32 and ONE contraction element, l/32; its result has the layout of the 16-bit
// one.  Contraction over head_dim takes the columns 8j + 4*(l/32) + 0..3 in four steps, so that a lane reads 16 bytes of its row at a
// time; contraction over streamed rows takes rows 8*(i/4) + 4*(l/32) + i%4 in step i, which is where accumulator register i of P or dS
// has them.
//
// The instruction takes 64 clocks, which bounds the kernel; two workgroups of four wavefronts on a compute unit keep the matrix pipe fed (one at head_dims above 96, whose
// operands and accumulators take more than 256 registers).
#include "attn_bwd_rows.h"
#include "attn_split.h"
#include "attn_tiles.h"

namespace xdit {
namespace {

constexpr int kRows32 = 32;   // streamed rows per LDS tile

// LDS layout of a streamed tile, filled by 1 KiB pieces (a direct load writes lane i at 16 i) that lie 16 bytes more apart: rows that are read together (one
// 16-byte column of 16 consecutive rows) sit in different pieces, on other banks.  KG: groups of 8 columns that hold the
// tensors' head_dim; DB: blocks of 32 columns of the gradients.
template <int KG, int DB> struct Geom32 {
  static constexpr int ROW_BYTES = KG <= 8 && DB <= 2 ? 256 : 512;
  static constexpr int NG = kRows32 * ROW_BYTES / 1024;
  static constexpr int PITCH = 1024 + 16;
  static constexpr int TENSOR_BYTES = NG * PITCH;
  static constexpr int BUF_BYTES = 2 * TENSOR_BYTES + 2 * kRows32 * 4;
  static constexpr int LANES_PER_ROW = ROW_BYTES / 16;
  static __device__ __forceinline__ int at(int r) { return r % NG * PITCH + r / NG * ROW_BYTES; }   // byte offset of a row
};

template <int KG, int DB, bool KEYS>
__device__ __forceinline__ void bwd_role_f32(const AttnBwdParams& p, int xcd, int n, unsigned char* smem) {
  typedef Geom32<KG, DB> G;
  constexpr int ROWS = kBwdRows;

  const BwdRole& R = KEYS ? p.keys : p.queries;
  BwdUnit unit;
  if (!bwd_unit(R, xcd, n, unit)) return;
  const int bh = unit.tile / R.tiles;
  int tile = unit.tile - bh * R.tiles;
  const int b = bh / p.H, h = bh - b * p.H;
  const int first = unit.slot < 0 ? 0 : unit.part * R.len;
  const int last = unit.slot < 0 || first + R.len > R.steps ? R.steps : first + R.len;

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
  const bool second = KEYS && tile >= p.tiles1;
  if (second) tile -= p.tiles1;
  const BwdTensor& F = KEYS ? (second ? p.k2 : p.k) : p.q;
  const BwdTensor& Gt = KEYS ? (second ? p.v2 : p.v) : p.dout;
  const int own_rows = KEYS ? (second ? p.Sk2 : p.Sk) : p.Sq;
  const int own = tile * ROWS + wave * 32 + l32;
  f32x4 f[KG], g[KG];
  {
    const int r = own < own_rows ? own : own_rows - 1;
    const float* fp = (const float*)F.p + b * F.b + h * F.h + (int64_t)r * F.s + hh * 4;
    const float* gp = (const float*)Gt.p + b * Gt.b + h * Gt.h + (int64_t)r * Gt.s + hh * 4;
#pragma unroll
    for (int j = 0; j < KG; j++) {
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      f[j] = g[j] = zero;
      if (8 * j < p.D) {
        f[j] = *(const f32x4*)(fp + 8 * j);
        g[j] = *(const f32x4*)(gp + 8 * j);
      }
    }
  }
  const float c = p.scale * kLog2e;
  const float* stats = p.stats + (int64_t)bh * 2 * p.sq_pad;
  float own_lse = 0.f, own_nd = 0.f;
  if (!KEYS && own < p.sq_pad) { own_lse = stats[own]; own_nd = stats[p.sq_pad + own]; }

  // Columns of the LDS tiles that the tensors do not have (never written by the loads): zeros.
  XDIT_LDS unsigned char* const tiles = (XDIT_LDS unsigned char*)smem;
  constexpr int WIDE = (8 * KG > 32 * DB ? 8 * KG : 32 * DB) / 4;   // 16-byte columns that are read
  if (4 * WIDE > p.D) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int c0 = p.D / 4, n0 = WIDE - c0;
    for (int i = threadIdx.x; i < 4 * kRows32 * n0; i += 64 * kBwdWaves) {
      const int which = i / (kRows32 * n0), j = i % (kRows32 * n0);
      *(XDIT_LDS f32x4*)(tiles + (which >> 1) * G::BUF_BYTES + (which & 1) * G::TENSOR_BYTES + G::at(j % kRows32) + (c0 + j / kRows32) * 16) = zero;
    }
  }

  const unsigned lds_base = (unsigned)(uintptr_t)tiles;
  const bool ld_on = (lane % G::LANES_PER_ROW) * 4 < p.D;
  auto issue = [&](int t, unsigned bo) {
    const bool s2 = !KEYS && t >= p.step1;
    const BwdTensor& X = KEYS ? p.q : s2 ? p.k2 : p.k;
    const BwdTensor& Y = KEYS ? p.dout : s2 ? p.v2 : p.v;
    const int rows = KEYS ? p.Sq : s2 ? p.Sk2 : p.Sk;
    const int row0 = (s2 ? t - p.step1 : t) * kRows32;
    const int left = rows - row0 < kRows32 ? rows - row0 : kRows32;
    const float* xb = (const float*)X.p + b * X.b + h * X.h + (int64_t)row0 * X.s;
    const float* yb = (const float*)Y.p + b * Y.b + h * Y.h + (int64_t)row0 * Y.s;
    const unsigned xs = (unsigned)X.s * 4, ys = (unsigned)Y.s * 4;
    if (ld_on) {
#pragma unroll
      for (int i = 0; i < G::NG / kBwdWaves; i++) {
        const int piece = wave + i * kBwdWaves;
        int r = piece + lane / G::LANES_PER_ROW * G::NG;
        r = r < left ? r : left - 1;   // rows past the end re-read the last one
        const unsigned col = (lane % G::LANES_PER_ROW) * 16;
        load_lds_16(xb, __umul24((unsigned)r, xs) + col, lds_base + bo + piece * G::PITCH);
        load_lds_16(yb, __umul24((unsigned)r, ys) + col, lds_base + bo + G::TENSOR_BYTES + piece * G::PITCH);
      }
    }
    if (KEYS && wave == 0)   // 32 of lse / ln 2, then 32 of -delta
      load_lds_4(stats + row0, ((lane >> 5) * p.sq_pad + l32) * 4u, lds_base + bo + 2 * G::TENSOR_BYTES);
  };

  f32x16 acc_f[DB], acc_g[KEYS ? DB : 1];
#pragma unroll
  for (int db = 0; db < DB; db++)
#pragma unroll
    for (int e = 0; e < 16; e++) {
      acc_f[db][e] = 0.f;
      if (KEYS) acc_g[KEYS ? db : 0][e] = 0.f;
    }

  issue(first, 0);
  // The compiler accounts for the loads of the owned rows here: any wait for them inside the loop would be one for the tile loads too.
#pragma unroll
  for (int j = 0; j < KG; j++) asm volatile("" : "+v"(f[j]), "+v"(g[j]));

  for (int t = first; t < last; t++) {
    const unsigned bo = ((t - first) & 1) * G::BUF_BYTES;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < last) issue(t + 1, G::BUF_BYTES - bo);
    int left = kRows32;
    if (!KEYS) {
      const int l = t >= p.step1 ? p.Sk2 - (t - p.step1) * kRows32 : p.Sk - t * kRows32;
      left = l < kRows32 ? l : kRows32;
    }
    const XDIT_LDS unsigned char* const buf = tiles + bo;
    const XDIT_LDS float* const st = (const XDIT_LDS float*)(buf + 2 * G::TENSOR_BYTES);
    f32x16 s, dp;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      s[i] = 0.f;
      dp[i] = KEYS ? st[kRows32 + 8 * (i >> 2) + 4 * hh + (i & 3)] : own_nd;
    }
    const XDIT_LDS unsigned char* const xr = buf + G::at(l32) + 16 * hh;
#pragma unroll
    for (int j = 0; j < KG; j++) {
      const f32x4 x = *(const XDIT_LDS f32x4*)(xr + 32 * j);
      const f32x4 y = *(const XDIT_LDS f32x4*)(xr + G::TENSOR_BYTES + 32 * j);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s = __builtin_amdgcn_mfma_f32_32x32x2f32(x[e], f[j][e], s, 0, 0, 0);
        dp = __builtin_amdgcn_mfma_f32_32x32x2f32(y[e], g[j][e], dp, 0, 0, 0);
      }
    }
    float pr[16], ds[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = 8 * (i >> 2) + 4 * hh + (i & 3);
      const float l = KEYS ? st[r] : own_lse;
      pr[i] = fast_exp2(__builtin_fmaf(s[i], c, -l));
    }
    if (!KEYS && left < kRows32) {   // only a segment's last tile: keys behind its end
#pragma unroll
      for (int i = 0; i < 16; i++)
        if (8 * (i >> 2) + 4 * hh + (i & 3) >= left) pr[i] = 0.f;
    }
#pragma unroll
    for (int i = 0; i < 16; i++) ds[i] = pr[i] * dp[i];
    const XDIT_LDS unsigned char* const columns = buf + 4 * hh * G::PITCH + 4 * l32;   // row 4 hh, column l32
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const XDIT_LDS float* const xc = (const XDIT_LDS float*)(columns + G::at(8 * (i >> 2) + (i & 3)));
#pragma unroll
      for (int db = 0; db < DB; db++) {
        if constexpr (KEYS) acc_g[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(xc[G::TENSOR_BYTES / 4 + 32 * db], pr[i], acc_g[db], 0, 0, 0);
        acc_f[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(xc[32 * db], ds[i], acc_f[db], 0, 0, 0);
      }
    }
  }

#pragma unroll
  for (int which = 0; which < (KEYS ? 2 : 1); which++) {   // 0: gradient of F, 1: of G
    const float w = which ? 1.f : p.scale;
    const BwdTensor& O = KEYS ? (which ? (second ? p.dv2 : p.dv) : (second ? p.dk2 : p.dk)) : p.dq;
    float* orow = (float*)O.p + b * O.b + h * O.h + (int64_t)own * O.s;
    float* prow = R.partial + ((unit.slot * (KEYS ? 2 : 1) + which) * ROWS + wave * 32 + l32) * 32 * DB;
#pragma unroll
    for (int db = 0; db < DB; db++)
#pragma unroll
      for (int a = 0; a < 4; a++) {
        const int col = 32 * db + 8 * a + 4 * hh;
        f32x4 x;
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] = (which ? acc_g[KEYS ? db : 0] : acc_f[db])[4 * a + e] * w;
        if (unit.slot >= 0) *(f32x4*)(prow + col) = x;
        else if (own < own_rows && col < p.D) *(f32x4*)(orow + col) = x;
      }
  }
}

template <int KG, int DB>
__global__ __launch_bounds__(64 * kBwdWaves, DB <= 3 ? 2 : 1) void attn_bwd_f32_kernel(const AttnBwdParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds32[];
  const int xcd = blockIdx.x % 8, n = blockIdx.x / 8;   // as in the 16-bit kernel
  if (n < p.keys.units) bwd_role_f32<KG, DB, true>(p, xcd, n, lds32);
  else bwd_role_f32<KG, DB, false>(p, xcd, n - p.keys.units, lds32);
}

template <int KG, int DB>
hipError_t launch_kernels(const AttnBwdParams& p, hipStream_t stream) {
  static std::atomic<bool> lds_ready[kMaxDevices];
  constexpr int lds = 2 * Geom32<KG, DB>::BUF_BYTES;
  const int slot = current_device_slot();
  if (!lds_ready[slot].load(std::memory_order_relaxed)) {
    hipError_t e = hipFuncSetAttribute((const void*)attn_bwd_f32_kernel<KG, DB>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    lds_ready[slot].store(true, std::memory_order_relaxed);
  }
  launch_bwd_stats<float>(p, stream);
  hipLaunchKernelGGL((attn_bwd_f32_kernel<KG, DB>), dim3(8u * (unsigned)(p.keys.units + p.queries.units)), dim3(64 * kBwdWaves), lds, stream, p);
  return launch_bwd_fold<float, 32 * DB>(p, stream);
}

}  // namespace

// head_dims up to 80 of the 96-column form contract over 80 columns (72 is a model's own).
hipError_t launch_attn_bwd_f32(const AttnBwdParams& p, hipStream_t stream) {
  if (p.D <= 32) return launch_kernels<4, 1>(p, stream);
  if (p.D <= 64) return launch_kernels<8, 2>(p, stream);
  if (p.D <= 80) return launch_kernels<10, 3>(p, stream);
  if (p.D <= 96) return launch_kernels<12, 3>(p, stream);
  return launch_kernels<16, 4>(p, stream);
}

}  // namespace xdit
