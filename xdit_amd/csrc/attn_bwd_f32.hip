// Backward pass of the attention forward for fp32 tensors: the formulas, roles and partial results of the 16-bit kernel
// (attn_bwd_16.hip) on v_mfma_f32_32x32x2_f32, with everything in fp32.
//
// Lane l of that instruction holds row/column l%32 and ONE contraction element, l/32; its result has the layout of the 16-bit
// one.  Contraction over head_dim takes the columns 8j + 4*(l/32) + 0..3 in four steps, so that a lane reads 16 bytes of its row at a
// time; contraction over streamed rows takes rows 8*(i/4) + 4*(l/32) + i%4 in step i, which is where accumulator register i of P or dS
// has them.
//
// The instruction takes 64 clocks, so one wavefront per SIMD (four of 32 owned rows, whose operands and accumulators then have
// 512 registers) keeps the matrix pipe fed; it bounds the kernel.
#include "attn_bwd_rows.h"
#include "attn_split.h"

namespace xdit {
namespace {

constexpr int kRows32 = 32;   // streamed rows per LDS tile

// KG: groups of 8 columns that hold the tensors' head_dim; DB: blocks of 32 columns of the gradients.
template <int KG, int DB>
constexpr int pitch_f32() { return (32 * DB > 8 * KG ? 32 * DB : 8 * KG) + 4; }   // floats; 16 bytes more: rows on other banks
template <int KG, int DB>
constexpr int buf_f32() { return 2 * kRows32 * pitch_f32<KG, DB>() + 2 * kRows32; }

template <int KG, int DB, bool KEYS>
__device__ __forceinline__ void bwd_role_f32(const AttnBwdParams& p, int xcd, int n, float* lds32) {
  constexpr int ROWS = kBwdRows, PITCH = pitch_f32<KG, DB>(), BUF = buf_f32<KG, DB>(), THREADS = 64 * kBwdWaves;
  constexpr int CHUNKS = kRows32 * KG * 2;                      // 16-byte pieces of a tensor's tile
  constexpr int LOADS = (CHUNKS + THREADS - 1) / THREADS;

  const BwdRole& R = KEYS ? p.keys : p.queries;
  BwdUnit unit;
  if (!bwd_unit(R, xcd, n, unit)) return;
  const int bh = unit.tile / R.tiles;
  int tile = unit.tile - bh * R.tiles;
  const int b = bh / p.H, h = bh - b * p.H;
  const int first = unit.slot < 0 ? 0 : unit.part * R.len;
  const int last = unit.slot < 0 || first + R.len > R.steps ? R.steps : first + R.len;

  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;
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
  for (int i = threadIdx.x; i < 2 * BUF; i += THREADS) lds32[i] = 0.f;
  __syncthreads();

  f32x4 rx[LOADS], ry[LOADS];
  float rs = 0.f;
  auto fetch = [&](int t) {
    const bool s2 = !KEYS && t >= p.step1;
    const BwdTensor& X = KEYS ? p.q : s2 ? p.k2 : p.k;
    const BwdTensor& Y = KEYS ? p.dout : s2 ? p.v2 : p.v;
    const int rows = KEYS ? p.Sq : s2 ? p.Sk2 : p.Sk;
    const int row0 = (s2 ? t - p.step1 : t) * kRows32;
    const float* xb = (const float*)X.p + b * X.b + h * X.h;
    const float* yb = (const float*)Y.p + b * Y.b + h * Y.h;
#pragma unroll
    for (int n = 0; n < LOADS; n++) {
      const int i = threadIdx.x + n * THREADS;
      int r = row0 + i / (2 * KG);
      const int col = i % (2 * KG) * 4;
      if (i < CHUNKS && col < p.D) {
        r = r < rows ? r : rows - 1;   // rows past the end re-read the last one
        rx[n] = *(const f32x4*)(xb + (int64_t)r * X.s + col);
        ry[n] = *(const f32x4*)(yb + (int64_t)r * Y.s + col);
      }
    }
    if (KEYS && threadIdx.x < 2 * kRows32) rs = stats[(threadIdx.x / kRows32) * (int64_t)p.sq_pad + row0 + threadIdx.x % kRows32];
  };
  auto put = [&](float* buf) {
#pragma unroll
    for (int n = 0; n < LOADS; n++) {
      const int i = threadIdx.x + n * THREADS;
      const int r = i / (2 * KG), col = i % (2 * KG) * 4;
      if (i < CHUNKS && col < p.D) {
        *(f32x4*)(buf + r * PITCH + col) = rx[n];
        *(f32x4*)(buf + (kRows32 + r) * PITCH + col) = ry[n];
      }
    }
    if (KEYS && threadIdx.x < 2 * kRows32) buf[2 * kRows32 * PITCH + threadIdx.x] = rs;
  };

  f32x16 acc_f[DB], acc_g[KEYS ? DB : 1];
#pragma unroll
  for (int db = 0; db < DB; db++)
#pragma unroll
    for (int e = 0; e < 16; e++) {
      acc_f[db][e] = 0.f;
      if (KEYS) acc_g[KEYS ? db : 0][e] = 0.f;
    }

  fetch(first);
  put(lds32);
  for (int t = first; t < last; t++) {
    float* buf = lds32 + ((t - first) & 1) * BUF;
    __syncthreads();
    if (t + 1 < last) fetch(t + 1);
    int left = kRows32;
    if (!KEYS) {
      const int l = t >= p.step1 ? p.Sk2 - (t - p.step1) * kRows32 : p.Sk - t * kRows32;
      left = l < kRows32 ? l : kRows32;
    }
    f32x16 s, dp;
#pragma unroll
    for (int i = 0; i < 4; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) {
        s[4 * i + e] = 0.f;
        dp[4 * i + e] = KEYS ? buf[2 * kRows32 * PITCH + kRows32 + 8 * i + 4 * hh + e] : own_nd;
      }
    const float* xr = buf + l32 * PITCH + 4 * hh;
#pragma unroll
    for (int j = 0; j < KG; j++) {
      const f32x4 x = *(const f32x4*)(xr + 8 * j);
      const f32x4 y = *(const f32x4*)(xr + kRows32 * PITCH + 8 * j);
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
      const float l = KEYS ? buf[2 * kRows32 * PITCH + r] : own_lse;
      pr[i] = fast_exp2(__builtin_fmaf(s[i], c, -l));
      if (!KEYS && r >= left) pr[i] = 0.f;
      ds[i] = pr[i] * dp[i];
    }
    const float* xc = buf + 4 * hh * PITCH + l32;
#pragma unroll
    for (int i = 0; i < 16; i++) {
      const int r = 8 * (i >> 2) + (i & 3);
#pragma unroll
      for (int db = 0; db < DB; db++) {
        if constexpr (KEYS) acc_g[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(xc[(kRows32 + r) * PITCH + 32 * db], pr[i], acc_g[db], 0, 0, 0);
        acc_f[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(xc[r * PITCH + 32 * db], ds[i], acc_f[db], 0, 0, 0);
      }
    }
    if (t + 1 < last) put(lds32 + ((t + 1 - first) & 1) * BUF);   // the buffer of the tile before this one
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
__global__ __launch_bounds__(64 * kBwdWaves, 1) void attn_bwd_f32_kernel(const AttnBwdParams p) {
  extern __shared__ __attribute__((aligned(16))) float lds32[];
  const int xcd = blockIdx.x % 8, n = blockIdx.x / 8;   // as in the 16-bit kernel
  if (n < p.keys.units) bwd_role_f32<KG, DB, true>(p, xcd, n, lds32);
  else bwd_role_f32<KG, DB, false>(p, xcd, n - p.keys.units, lds32);
}

template <int KG, int DB>
hipError_t launch_kernels(const AttnBwdParams& p, hipStream_t stream) {
  static std::atomic<bool> lds_ready[kMaxDevices];
  constexpr int lds = 2 * buf_f32<KG, DB>() * 4;
  const int slot = current_device_slot();
  if (!lds_ready[slot].load(std::memory_order_relaxed)) {
    hipError_t e = hipFuncSetAttribute((const void*)attn_bwd_f32_kernel<KG, DB>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    lds_ready[slot].store(true, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL((bwd_stats_kernel<float>), dim3((unsigned)(p.B * p.H) * (p.sq_pad / kBwdStatRows)), dim3(256), 0, stream, p);
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
