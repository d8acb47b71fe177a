// Backward pass of the attention forward for fp32 tensors: the formulas, roles and partial results of the 16-bit kernel
// (attn_bwd_16.hip) on v_mfma_f32_16x16x4_f32, with everything in fp32.
//
// Lane l of that instruction holds row/column l%16 and ONE contraction element, l/16; its result has column l%16 and rows 4*(l/16)..+3 in
// lane l.  A wavefront's 32 owned rows are two groups of 16, a tile's 32 rows two groups as well.  Contraction over head_dim takes the
// columns 16j + 4*(l/16) + 0..3 in four steps, so that a lane reads 16 bytes of its row at a time (8 at the end of an odd number of
// 8-column groups); contraction over streamed rows takes rows 4*(l/16) + i in step i, which is where accumulator register i of P or dS has
// them.  (Blocks of 16 columns rather than the 32 of v_mfma_f32_32x32x2_f32: head_dim 72 is 72 contracted columns and 80 of the gradients
// instead of 80 and 96, 16 heads of 4096 take 2055 us instead of 2340; at head_dim 64 both take 1745 us, at 128 3650 and 3615.)
//
// The instruction takes 32 clocks, which bounds the kernel; two workgroups of four wavefronts on a compute unit keep the matrix pipe fed
// (one at head_dims above 96, whose operands and accumulators take more than 256 registers).
#include "attn_bwd_rows.h"
#include "attn_split.h"
#include "attn_tiles.h"

namespace xdit {
namespace {

constexpr int kRows32 = 32;   // streamed rows per LDS tile

// LDS layout of a streamed tile, filled by 1 KiB pieces (a direct load writes lane i at 16 i) that lie 16 bytes more apart: rows that are
// read together (one 16-byte column of 8 consecutive rows, one 64-byte column of rows 4 apart) sit in different pieces, on other banks.
// N8: groups of 8 columns.
template <int N8> struct Geom32 {
  static constexpr int ROW_BYTES = N8 <= 8 ? 256 : 512;
  static constexpr int NG = kRows32 * ROW_BYTES / 1024;
  static constexpr int PITCH = 1024 + 16;
  static constexpr int TENSOR_BYTES = NG * PITCH;
  static constexpr int BUF_BYTES = 2 * TENSOR_BYTES + 2 * kRows32 * 4;
  static constexpr int LANES_PER_ROW = ROW_BYTES / 16;
  static __device__ __forceinline__ int at(int r) { return r % NG * PITCH + r / NG * ROW_BYTES; }   // byte offset of a row
};

template <int N8, bool KEYS>
__device__ __forceinline__ void bwd_role_f32(const AttnBwdParams& p, int xcd, int n, unsigned char* smem) {
  typedef Geom32<N8> G;
  typedef __attribute__((ext_vector_type(2))) float f32x2;
  constexpr int ROWS = kBwdRows, WIDE = N8 / 2, TAIL = N8 % 2, CB = WIDE + TAIL;   // 16-column groups, an 8-column one behind them; blocks of the gradients

  const BwdRole& R = KEYS ? p.keys : p.queries;
  BwdUnit unit;
  if (!bwd_unit(R, xcd, n, unit)) return;
  const int bh = unit.tile / R.tiles;
  int tile = unit.tile - bh * R.tiles;
  const int b = bh / p.H, h = bh - b * p.H;
  const int first = unit.slot < 0 ? 0 : unit.part * R.len;
  const int last = unit.slot < 0 || first + R.len > R.steps ? R.steps : first + R.len;

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6), lane = threadIdx.x & 63, l16 = lane & 15, qq = lane >> 4;
  const bool second = KEYS && tile >= p.tiles1;
  if (second) tile -= p.tiles1;
  const BwdTensor& F = KEYS ? (second ? p.k2 : p.k) : p.q;
  const BwdTensor& Gt = KEYS ? (second ? p.v2 : p.v) : p.dout;
  const int own_rows = KEYS ? (second ? p.Sk2 : p.Sk) : p.Sq;
  const int own0 = tile * ROWS + wave * 32 + l16;   // and 16 rows behind it
  f32x4 f[2][WIDE], g[2][WIDE];
  f32x2 f_tail[2], g_tail[2];
#pragma unroll
  for (int o = 0; o < 2; o++) {
    const int r = own0 + 16 * o < own_rows ? own0 + 16 * o : own_rows - 1;
    const float* fp = (const float*)F.p + b * F.b + h * F.h + (int64_t)r * F.s;
    const float* gp = (const float*)Gt.p + b * Gt.b + h * Gt.h + (int64_t)r * Gt.s;
#pragma unroll
    for (int j = 0; j < WIDE; j++) {
      const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
      const int col = 16 * j + 4 * qq;
      f[o][j] = g[o][j] = zero;
      if (col < p.D) {
        f[o][j] = *(const f32x4*)(fp + col);
        g[o][j] = *(const f32x4*)(gp + col);
      }
    }
    if (TAIL) {   // a head_dim of exactly 8 N8
      f_tail[o] = *(const f32x2*)(fp + 16 * WIDE + 2 * qq);
      g_tail[o] = *(const f32x2*)(gp + 16 * WIDE + 2 * qq);
    }
  }
  const float c = p.scale * kLog2e;
  const float* stats = p.stats + (int64_t)bh * 2 * p.sq_pad;
  float own_lse[2] = {0.f, 0.f}, own_nd[2] = {0.f, 0.f};
#pragma unroll
  for (int o = 0; o < 2; o++)
    if (!KEYS && own0 + 16 * o < p.sq_pad) { own_lse[o] = stats[own0 + 16 * o]; own_nd[o] = stats[p.sq_pad + own0 + 16 * o]; }

  // Columns of the LDS tiles that the tensors do not have (never written by the loads): zeros.
  XDIT_LDS unsigned char* const tiles = (XDIT_LDS unsigned char*)smem;
  if (16 * CB > p.D) {
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int c0 = p.D / 4, n0 = 4 * CB - c0;
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
      load_lds_4(stats + row0, ((lane >> 5) * p.sq_pad + (lane & 31)) * 4u, lds_base + bo + 2 * G::TENSOR_BYTES);
  };

  f32x4 acc_f[CB][2], acc_g[KEYS ? CB : 1][2];
#pragma unroll
  for (int cb = 0; cb < CB; cb++)
#pragma unroll
    for (int e = 0; e < 8; e++) {
      acc_f[cb][e >> 2][e & 3] = 0.f;
      if (KEYS) acc_g[KEYS ? cb : 0][e >> 2][e & 3] = 0.f;
    }

  issue(first, 0);
  // The compiler accounts for the loads of the owned rows here: any wait for them inside the loop would be one for the tile loads too.
#pragma unroll
  for (int o = 0; o < 2; o++) {
#pragma unroll
    for (int j = 0; j < WIDE; j++) asm volatile("" : "+v"(f[o][j]), "+v"(g[o][j]));
    if (TAIL) asm volatile("" : "+v"(f_tail[o]), "+v"(g_tail[o]));
    if (!KEYS) asm volatile("" : "+v"(own_lse[o]), "+v"(own_nd[o]));
  }

  for (int t = first; t < last; t++) {
    const unsigned bo = ((t - first) & 1) * G::BUF_BYTES;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    if (t + 1 < last) issue(t + 1, G::BUF_BYTES - bo);
    if constexpr (KEYS) {   // queries that attended nothing, as in the 16-bit kernel
      XDIT_LDS unsigned char* const buf = tiles + bo;
      const int rows = p.Sq - t * kRows32;   // of the tensors, from this tile on
      const unsigned none = (unsigned)__builtin_amdgcn_ballot_w64(((const XDIT_LDS float*)(buf + 2 * G::TENSOR_BYTES))[lane_now() & 31] == INFINITY);
      if (none << (rows < kRows32 ? kRows32 - rows : 0)) {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
        for (unsigned rest = none; rest != 0; rest &= rest - 1) {
          const int r = __builtin_ctz(rest), n = lane_now();
          if (n < G::LANES_PER_ROW)
            *(XDIT_LDS f32x4*)(buf + G::at(r) + n * 16) = *(XDIT_LDS f32x4*)(buf + G::at(r) + G::TENSOR_BYTES + n * 16) = zero;
        }
        __syncthreads();
      }
    }
    if (N8 <= 12 && tile * ROWS + wave * 32 >= own_rows) continue;   // a wavefront without rows leaves its SIMD to the other workgroup's (80 heads of 3291 on 3: 209 -> 155 us)
    int left = kRows32;
    if (!KEYS) {
      const int l = t >= p.step1 ? p.Sk2 - (t - p.step1) * kRows32 : p.Sk - t * kRows32;
      left = l < kRows32 ? l : kRows32;
    }
    const XDIT_LDS unsigned char* const buf = tiles + bo;
    const XDIT_LDS f32x4* const st = (const XDIT_LDS f32x4*)(buf + 2 * G::TENSOR_BYTES);
    f32x4 s[2][2], dp[2][2];   // [streamed group][owned group]
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int o = 0; o < 2; o++) {
        const f32x4 zero = {0.f, 0.f, 0.f, 0.f}, own = {own_nd[o], own_nd[o], own_nd[o], own_nd[o]};
        s[r][o] = zero;
        dp[r][o] = KEYS ? st[kRows32 / 4 + 4 * r + qq] : own;
      }
    const XDIT_LDS unsigned char* const row0 = buf + G::at(l16) + 16 * qq;
    constexpr int GROUP = 16 % G::NG * G::PITCH + 16 / G::NG * G::ROW_BYTES;   // from a row to the one 16 behind it
#pragma unroll
    for (int j = 0; j < WIDE; j++) {
      f32x4 x[2], y[2];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        x[r] = *(const XDIT_LDS f32x4*)(row0 + r * GROUP + 64 * j);
        y[r] = *(const XDIT_LDS f32x4*)(row0 + r * GROUP + G::TENSOR_BYTES + 64 * j);
      }
#pragma unroll
      for (int e = 0; e < 4; e++)
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
          for (int o = 0; o < 2; o++) {
            s[r][o] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r][e], f[o][j][e], s[r][o], 0, 0, 0);
            dp[r][o] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[r][e], g[o][j][e], dp[r][o], 0, 0, 0);
          }
      // (Wide heads: reads of later groups, taken ahead, spill 100 registers at head_dims 88 and 96 and cost 1 % at 128.)
      if (N8 >= 11) __builtin_amdgcn_sched_barrier(0);
    }
    if (TAIL) {
      const XDIT_LDS unsigned char* const end = buf + G::at(l16) + 64 * WIDE + 8 * qq;
      f32x2 x[2], y[2];
#pragma unroll
      for (int r = 0; r < 2; r++) {
        x[r] = *(const XDIT_LDS f32x2*)(end + r * GROUP);
        y[r] = *(const XDIT_LDS f32x2*)(end + r * GROUP + G::TENSOR_BYTES);
      }
#pragma unroll
      for (int e = 0; e < 2; e++)
#pragma unroll
        for (int r = 0; r < 2; r++)
#pragma unroll
          for (int o = 0; o < 2; o++) {
            s[r][o] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[r][e], f_tail[o][e], s[r][o], 0, 0, 0);
            dp[r][o] = __builtin_amdgcn_mfma_f32_16x16x4f32(y[r][e], g_tail[o][e], dp[r][o], 0, 0, 0);
          }
    }
#pragma unroll
    for (int r = 0; r < 2; r++) {
      f32x4 lse = {0.f, 0.f, 0.f, 0.f};
      if (KEYS) lse = st[4 * r + qq];
#pragma unroll
      for (int o = 0; o < 2; o++)
#pragma unroll
        for (int i = 0; i < 4; i++) s[r][o][i] = fast_exp2(__builtin_fmaf(s[r][o][i], c, -(KEYS ? lse[i] : own_lse[o])));
    }
    if (!KEYS && left < kRows32) {   // only a segment's last tile: keys behind its end
#pragma unroll
      for (int r = 0; r < 2; r++)
#pragma unroll
        for (int i = 0; i < 4; i++)
          if (16 * r + 4 * qq + i >= left) s[r][0][i] = s[r][1][i] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int o = 0; o < 2; o++)
#pragma unroll
        for (int i = 0; i < 4; i++) dp[r][o][i] *= s[r][o][i];
    const XDIT_LDS unsigned char* const columns = buf + G::at(4 * qq) + 4 * l16;   // row 4 qq, column l16; the three rows behind it lie a piece apart each
#pragma unroll
    for (int r = 0; r < 2; r++)
#pragma unroll
      for (int i = 0; i < 4; i++) {
        const XDIT_LDS float* const xc = (const XDIT_LDS float*)(columns + r * GROUP + i * G::PITCH);
#pragma unroll
        for (int cb = 0; cb < CB; cb++)
#pragma unroll
          for (int o = 0; o < 2; o++) {
            if constexpr (KEYS) acc_g[cb][o] = __builtin_amdgcn_mfma_f32_16x16x4f32(xc[G::TENSOR_BYTES / 4 + 16 * cb], s[r][o][i], acc_g[cb][o], 0, 0, 0);
            acc_f[cb][o] = __builtin_amdgcn_mfma_f32_16x16x4f32(xc[16 * cb], dp[r][o][i], acc_f[cb][o], 0, 0, 0);
          }
        if (N8 >= 11) __builtin_amdgcn_sched_barrier(0);
      }
  }

#pragma unroll
  for (int which = 0; which < (KEYS ? 2 : 1); which++) {   // 0: gradient of F, 1: of G
    const float w = which ? 1.f : p.scale;
    const BwdTensor& O = KEYS ? (which ? (second ? p.dv2 : p.dv) : (second ? p.dk2 : p.dk)) : p.dq;
#pragma unroll
    for (int o = 0; o < 2; o++) {
      const int own = own0 + 16 * o;
      float* orow = (float*)O.p + b * O.b + h * O.h + (int64_t)own * O.s;
      f32x4* to = (f32x4*)(R.partial + (unit.slot * (KEYS ? 2 : 1) + which) * ROWS * 16 * CB) + (wave * 2 + o) * (64 * CB) + lane;   // register by register: PartLayout
#pragma unroll
      for (int cb = 0; cb < CB; cb++) {
        const int col = 16 * cb + 4 * qq;
        f32x4 x = (which ? acc_g[KEYS ? cb : 0][o] : acc_f[cb][o]) * w;
        if (!KEYS && own_lse[o] == INFINITY) x = f32x4{0.f, 0.f, 0.f, 0.f};   // a query that attended nothing
        if (unit.slot >= 0) to[cb * 64] = x;
        else if (own < own_rows && col < p.D) *(f32x4*)(orow + col) = x;
      }
    }
  }
}

template <int N8>
__global__ __launch_bounds__(64 * kBwdWaves, N8 <= 12 ? 2 : 1) void attn_bwd_f32_kernel(const AttnBwdParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char lds32[];
  const int xcd = blockIdx.x % 8, n = blockIdx.x / 8;   // as in the 16-bit kernel
  if (n < p.keys.units) bwd_role_f32<N8, true>(p, xcd, n, lds32);
  else bwd_role_f32<N8, false>(p, xcd, n - p.keys.units, lds32);
}

template <int N8>
hipError_t launch_kernels(const AttnBwdParams& p, hipStream_t stream) {
  static std::atomic<bool> lds_ready[kMaxDevices];
  constexpr int lds = 2 * Geom32<N8>::BUF_BYTES;
  const int slot = current_device_slot();
  if (!lds_ready[slot].load(std::memory_order_relaxed)) {
    hipError_t e = hipFuncSetAttribute((const void*)attn_bwd_f32_kernel<N8>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    lds_ready[slot].store(true, std::memory_order_relaxed);
  }
  launch_bwd_stats<float>(p, stream);
  hipLaunchKernelGGL((attn_bwd_f32_kernel<N8>), dim3(8u * (unsigned)(p.keys.units + p.queries.units)), dim3(64 * kBwdWaves), lds, stream, p);
  return launch_bwd_fold<float, (N8 + 1) / 2 * 16, 16>(p, stream);
}

}  // namespace

hipError_t launch_attn_bwd_f32(const AttnBwdParams& p, hipStream_t stream) {
  switch (bwd_f32_groups(p.D)) {
    case 4: return launch_kernels<4>(p, stream);
    case 5: return launch_kernels<5>(p, stream);
    case 6: return launch_kernels<6>(p, stream);
    case 7: return launch_kernels<7>(p, stream);
    case 8: return launch_kernels<8>(p, stream);
    case 9: return launch_kernels<9>(p, stream);
    case 10: return launch_kernels<10>(p, stream);
    case 11: return launch_kernels<11>(p, stream);
    case 12: return launch_kernels<12>(p, stream);
    case 13: return launch_kernels<13>(p, stream);
    case 14: return launch_kernels<14>(p, stream);
    case 15: return launch_kernels<15>(p, stream);
    default: return launch_kernels<16>(p, stream);
  }
}

}  // namespace xdit
