// Norms before and after a block fused with its gate and residual scale, forward and backward, for gfx950.
//
//     v = N_y(y) w_y ;  h = x + alpha gate v ;  n = (N(h) w + b)(1 + scale) + shift
// Everything between the loads and the stores is fp32; h and n are rounded once, and n comes from the unrounded h
// (a rounded one would add its 2^-9 to every element of n in bf16).  A norm's variance is taken from the differences
// to the mean, in registers, so large means cost no digits.
//
// Backward, from h, (mean, r) of h and of y, and the gradients dh, dn; u = (h - mean) r, z likewise from y:
//     du = dn (1 + scale) w ;  t = dh + r (du - [layer] mean(du) - u mean(du u))         dx = t
//     e = alpha gate t w_y ;   dy = r_y (e - [layer] mean(e) - z mean(e z)), or e
// and over rows  A = sum dn u, F = sum dn, G = sum t z, from which every parameter's gradient follows:
//     dshift = F, dscale = w A + b F, dw = sum_b (1 + scale) A, db = sum_b (1 + scale) F,
//     dgate = alpha w_y G, dw_y = sum_b alpha gate G
// (with a scale or a gate per token the factor goes into the sum, and dscale, dshift, dgate are elementwise).
// HBM-bound: forward one read of x and y and one write of h and n, backward one read of dh, dn, h, y and one
// write of dx and dy.
#include "attn_split.h"
#include "block_params.h"
#include "row_ops.h"

namespace xdit {

namespace gnorm {

// A row is held by as many wavefronts as it has 512 columns, eight columns a thread, and a workgroup goes over the rows of one
// part of one batch entry: modulation and gains stay in registers, folded to three vectors (gate alpha w_y, (1 + scale) w and
// b (1 + scale) + shift), where fetching them for every row was two thirds of all traffic from the L2.  The next rows are on their
// way while these are worked on.

// Sums over the wavefronts of a workgroup of up to four values (k = 0 .. K-1) a wavefront has posted at part[k][wave]: sixteen
// lanes read a value's entries, a DPP row adds them, and the total is broadcast from there.
constexpr int kMaxWaves = 16;
struct Posted { float v[4][kMaxWaves]; };

__device__ __forceinline__ float from_lane(float x, int lane) { return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane)); }

// Mean and reciprocal deviation of R rows of C elements, of which a thread holds eight of each (zeros beyond the row).  One
// barrier: a wavefront sums its 512 elements and the squares of their differences to ITS mean, and the squares about the
// row's mean follow from those and the means (Chan, Golub and LeVeque, 1979), so that no digits cancel.
template <int R>
__device__ __forceinline__ void row_stats(const float (&v)[R][8], bool layer, bool live, int waves, int wave, int lane, float inv_c, float eps, Posted& sums,
                                          Posted& squares, float (&mean)[R], float (&rstd)[R], int chunks) {
  const float inv_mine = 1.f / (float)(min(64, chunks - 64 * wave) * 8);   // of this wavefront's elements
  float s[R], q[R];
#pragma unroll
  for (int r = 0; r < R; r++) {
    float x = 0.f;
    if (layer) {
#pragma unroll
      for (int i = 0; i < 8; i++) x += v[r][i];
      x = wave_sum(x);
    }
    s[r] = x;
    const float m = x * inv_mine;
    float y = 0.f;
#pragma unroll
    for (int i = 0; i < 8; i++) { const float d = v[r][i] - m; y += d * d; }
    q[r] = wave_sum(live ? y : 0.f);
  }
  if (waves > 1) {
    if (lane == 0) {
#pragma unroll
      for (int r = 0; r < R; r++) { sums.v[r][wave] = s[r]; squares.v[r][wave] = q[r]; }
    }
    __syncthreads();
    const int r = lane >> 4, w = lane & 15;
    const bool there = w < waves && r < R;
    const float ws = there ? sums.v[r][w] : 0.f, wq = there ? squares.v[r][w] : 0.f;
    const float total = row16_sum(ws);
    const float n = (float)(min(64, chunks - 64 * w) * 8);
    const float d = there && layer ? ws * __builtin_amdgcn_rcpf(n) - total * inv_c : 0.f;
    const float all = row16_sum(there ? wq + n * d * d : 0.f);
#pragma unroll
    for (int k = 0; k < R; k++) { s[k] = from_lane(total, 16 * k); q[k] = from_lane(all, 16 * k); }
  }
#pragma unroll
  for (int r = 0; r < R; r++) {
    mean[r] = s[r] * inv_c;
    rstd[r] = inv_sqrt(q[r] * inv_c + eps);
  }
}

// Eight columns of a row of n as T or as part of an fp8 block, whose scale is returned: 16 lanes, a DPP row, hold its 128 columns.
template <typename T>
__device__ __forceinline__ float put_row8(const GatedNormParams& p, float (&n)[8], void* to, bool live) {
  if (!p.fp8) {
    if (live) store8<T>(to, 0, n);
    return 0.f;
  }
  // n has no bits of its own to keep (it is not stored): products with 1 / 448 and with the scale's reciprocal in place of the quantiser's
  // divisions, which took 40 % of the time (VALU instructions).  The scale is within 3 * 2^-24 of the quantiser's and a quotient within
  // 7 * 2^-24, so only one that close to the middle of two e4m3 numbers can come out as the other.
  const float top = __uint_as_float(row16_max(live ? absmax8(n) : 0));
  float scale = top * (1.f / kFp8Max);
  scale = top == 0.f ? 1.f : (scale < 0x1p-126f ? 0x1p-126f : scale);
  const float inv = __builtin_amdgcn_rcpf(scale);
#pragma unroll
  for (int i = 0; i < 8; i++) n[i] *= inv;
  if (live) *(i32x2*)to = to_fp8(n);
  return scale;
}

// 32760 x 5120 bf16 with y to fp8: 252 us, 4.7 TB/s; without y 141 us.  TOKEN: modulation has a row per token and is fetched when it is
// needed, nothing ahead: the same call to bf16 601 us, 3.9 TB/s.  The bound of six wavefronts a SIMD is that of 16-bit rows; fp32 rows spill 22
// registers under it (32760 x 5120: 637 us, 4.2 TB/s).
template <typename T, bool TOKEN>
__global__ __launch_bounds__(1024, TOKEN ? 4 : 6) void gated_norm_kernel(const GatedNormParams p) {
  constexpr int R = 1;   // rows at a time; written for one row without the arrays, the 16-bit kernel spills 22 registers
  __shared__ Posted post[2][4];   // by turns: [y sums, y squares, h sums, h squares]
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int chunks = p.C >> 3, waves = (int)blockDim.x >> 6;
  const bool live = (int)threadIdx.x < chunks;
  const int col = (live ? (int)threadIdx.x : 0) * 8;
  const int b = blockIdx.y;
  const int s0 = blockIdx.x * p.rows_per_part, s1 = min(p.S, s0 + p.rows_per_part);
  const bool has_y = p.y != nullptr;
  Raw8<T> x[R], y[R];
  auto load = [&](int s) {
#pragma unroll
    for (int r = 0; r < R; r++) {
      const int sr = min(s + r, s1 - 1);   // rows past the part re-read its last
      x[r] = load_raw8<T>(p.x, b * p.xs.b + sr * p.xs.s + col);
      if (has_y) y[r] = load_raw8<T>(p.y, b * p.ys.b + sr * p.ys.s + col);
    }
  };
  load(s0);
  float g[8], sc[8], sh[8];
  auto fill = [](float (&v)[8], float c) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = c;
  };
  auto fold_gate = [&](int s) {   // g = gate alpha w_y
    float yw[8];
    fill(g, 1.f); fill(yw, 1.f);
    if (p.gate != nullptr) load_param8<T>(p.gate, b * p.gs.b + s * p.gs.s + col, p.mod_wide, g);
    if (p.y_weight != nullptr) load_param8<T>(p.y_weight, col, p.weight_wide, yw);
#pragma unroll
    for (int i = 0; i < 8; i++) g[i] *= p.alpha * yw[i];
  };
  auto fold_scale = [&](int s) {   // sc = (1 + scale) w, sh = b (1 + scale) + shift
    float w[8], bi[8];
    fill(sc, 0.f); fill(sh, 0.f); fill(w, 1.f); fill(bi, 0.f);
    if (p.scale != nullptr) load_param8<T>(p.scale, b * p.ss.b + s * p.ss.s + col, p.mod_wide, sc);
    if (p.shift != nullptr) load_param8<T>(p.shift, b * p.fs.b + s * p.fs.s + col, p.mod_wide, sh);
    if (p.weight != nullptr) load_param8<T>(p.weight, col, p.weight_wide, w);
    if (p.bias != nullptr) load_param8<T>(p.bias, col, p.weight_wide, bi);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      sh[i] = __builtin_fmaf(bi[i], 1.f + sc[i], sh[i]);
      sc[i] = w[i] * (1.f + sc[i]);
    }
  };
  if constexpr (!TOKEN) {
    fold_gate(0);
    fold_scale(0);
  }
  float kept = 0.f;
  for (int s = s0, turn = 0; s < s1; s += R, turn ^= 1) {
    float h[R][8], v[R][8];
    float ym[R], yr[R], m[R], rs[R];
#pragma unroll
    for (int r = 0; r < R; r++) {
      get8(x[r], h[r]);
      if (has_y) get8(y[r], v[r]);
      ym[r] = m[r] = 0.f;
      yr[r] = rs[r] = 1.f;
      if (!live) { fill(h[r], 0.f); fill(v[r], 0.f); }
    }
    if (s + R < s1) load(s + R);
    if (has_y) {
      if (p.y_norm != 0) {
        row_stats<R>(v, p.y_norm == 2, live, waves, wave, lane, p.inv_c, p.y_eps, post[turn][0], post[turn][1], ym, yr, chunks);
#pragma unroll
        for (int r = 0; r < R; r++)
#pragma unroll
          for (int i = 0; i < 8; i++) v[r][i] = (v[r][i] - ym[r]) * yr[r];
      }
#pragma unroll
      for (int r = 0; r < R; r++) {
        if constexpr (TOKEN) fold_gate(min(s + r, s1 - 1));
#pragma unroll
        for (int i = 0; i < 8; i++) h[r][i] = live ? __builtin_fmaf(g[i], v[r][i], h[r][i]) : 0.f;
      }
    }
    if (p.h != nullptr) {
#pragma unroll
      for (int r = 0; r < R; r++)
        if (live && s + r < s1) store8<T>(p.h, b * p.hs.b + (s + r) * p.hs.s + col, h[r]);
    }
    if (p.norm != 0) row_stats<R>(h, p.norm == 2, live, waves, wave, lane, p.inv_c, p.eps, post[turn][2], post[turn][3], m, rs, chunks);
#pragma unroll
    for (int r = 0; r < R; r++) {
      if (s + r >= s1) continue;   // uniform
      const int64_t row = (int64_t)b * p.S + s + r;
      if (p.stats != nullptr && threadIdx.x == 0) *(f32x4*)(p.stats + row * 4) = (f32x4){m[r], rs[r], ym[r], yr[r]};
      if (p.norm == 0) continue;
      if constexpr (TOKEN) fold_scale(s + r);
      float n[8];
#pragma unroll
      for (int i = 0; i < 8; i++) n[i] = __builtin_fmaf((h[r][i] - m[r]) * rs[r], sc[i], sh[i]);
      const int64_t at = b * p.ns.b + (s + r) * p.ns.s + col;
      const float scale = put_row8<T>(p, n, p.fp8 ? (void*)((unsigned char*)p.n + at) : (void*)((T*)p.n + at), live);
      if (p.fp8) {   // a block's 16 lanes keep the scales of 16 rows and store them side by side (one at a time they cost 42 MB of partial lines there)
        const int k = (s + r - s0) & 15, mine = lane & 15;
        if (k == mine) kept = scale;
        if ((k == 15 || s + r + 1 == s1) && mine <= k && (int)(threadIdx.x & ~15u) < chunks) p.n_scale[(int64_t)(threadIdx.x >> 4) * p.rows + row - k + mine] = kept;
      }
    }
  }
}

// Many rows: a wavefront to a row of more than 64 (N - 1) and up to 64 N chunks of 8 columns; the three parameter vectors of the batch entry lie in LDS, as
// halves of chunks so that a lane's 16-byte reads are consecutive.  Nothing is exchanged between wavefronts, so twelve to
// thirty-two of them on a compute unit keep 150 KB of rows on their way.
template <typename T, int N>
__global__ __launch_bounds__(256, N >= 6 ? 3 : 4) void gated_norm_wave_kernel(const GatedNormParams p) {
  extern __shared__ __align__(16) f32x4 vectors[];   // [vector][N][2][64]: sc, sh and, with y, g
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int chunks = p.C >> 3, b = blockIdx.y;
  const bool has_y = p.y != nullptr;
  for (int c = threadIdx.x; c < 64 * N; c += 256) {
    const int col = (c < chunks ? c : 0) * 8;
    float v[8], sc[8], sh[8], w[8];
    auto fill = [](float (&v)[8], float c) {
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] = c;
    };
    auto put = [&](int vec, const float (&v)[8]) {
#pragma unroll
      for (int q = 0; q < 2; q++) vectors[((vec * N + (c >> 6)) * 2 + q) * 64 + (c & 63)] = (f32x4){v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
    };
    fill(sc, 0.f); fill(sh, 0.f); fill(w, 1.f); fill(v, 0.f);
    if (p.scale != nullptr) load_param8<T>(p.scale, b * p.ss.b + col, p.mod_wide, sc);
    if (p.shift != nullptr) load_param8<T>(p.shift, b * p.fs.b + col, p.mod_wide, sh);
    if (p.weight != nullptr) load_param8<T>(p.weight, col, p.weight_wide, w);
    if (p.bias != nullptr) load_param8<T>(p.bias, col, p.weight_wide, v);
#pragma unroll
    for (int i = 0; i < 8; i++) {
      sh[i] = __builtin_fmaf(v[i], 1.f + sc[i], sh[i]);
      sc[i] = w[i] * (1.f + sc[i]);
    }
    put(0, sc);
    put(1, sh);
    if (!has_y) continue;
    fill(v, 1.f); fill(w, 1.f);
    if (p.gate != nullptr) load_param8<T>(p.gate, b * p.gs.b + col, p.mod_wide, v);
    if (p.y_weight != nullptr) load_param8<T>(p.y_weight, col, p.weight_wide, w);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] *= p.alpha * w[i];
    put(2, v);
  }
  __syncthreads();
  auto vec8 = [&](int vec, int k, float (&v)[8]) {
#pragma unroll
    for (int q = 0; q < 2; q++) {
      const f32x4 t = vectors[((vec * N + k) * 2 + q) * 64 + lane];
#pragma unroll
      for (int i = 0; i < 4; i++) v[4 * q + i] = t[i];
    }
  };
  const bool last = lane + 64 * (N - 1) < chunks;   // the chunks before the last are whole
  const int col_last = last ? (lane + 64 * (N - 1)) * 8 : 0;
  auto col = [&](int k) { return (unsigned)(k < N - 1 ? lane * 8 + 512 * k : col_last); };   // 32-bit offsets from a row's uniform start
  for (int s = blockIdx.x * 4 + wave; s < p.S; s += gridDim.x * 4) {
    Raw8<T> x[N], y[N];
    auto row_of = [&](const void* p, const RowStrides& st) { return (const char*)((const T*)p + b * st.b + s * st.s); };
    const char* xrow = row_of(p.x, p.xs);
#pragma unroll
    for (int k = 0; k < N; k++) x[k] = *(const Raw8<T>*)(xrow + col(k) * (unsigned)sizeof(T));
    if (has_y) {
      const char* yrow = row_of(p.y, p.ys);
#pragma unroll
      for (int k = 0; k < N; k++) y[k] = *(const Raw8<T>*)(yrow + col(k) * (unsigned)sizeof(T));
    }
    float h[N][8];
    float ym = 0.f, yr = 1.f, m = 0.f, rs = 1.f;
    if (has_y) {
      if (p.y_norm != 0) {
        if (p.y_norm == 2) {
          float a = 0.f;
#pragma unroll
          for (int k = 0; k < N; k++) {
            float c = 0.f;
#pragma unroll
            for (int i = 0; i < 8; i++) c += y[k][i];
            a += k < N - 1 || last ? c : 0.f;
          }
          ym = wave_sum(a) * p.inv_c;
        }
        float a = 0.f;
#pragma unroll
        for (int k = 0; k < N; k++) {
          float c = 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++) { const float d = y[k][i] - ym; c = __builtin_fmaf(d, d, c); }
          a += k < N - 1 || last ? c : 0.f;
        }
        yr = inv_sqrt(wave_sum(a) * p.inv_c + p.y_eps);
      }
#pragma unroll
      for (int k = 0; k < N; k++) {
        float g[8];
        vec8(2, k, g);
        asm volatile("" : "+v"(x[k].x[0]), "+v"(y[k].x[0]));   // as loaded: no conversion is kept from the sums above
#pragma unroll
        for (int i = 0; i < 8; i++) h[k][i] = __builtin_fmaf(g[i], (y[k][i] - ym) * yr, x[k][i]);
        __builtin_amdgcn_sched_barrier(0);   // chunk by chunk: h takes the registers that x and y leave
      }
    } else {
#pragma unroll
      for (int k = 0; k < N; k++) get8(x[k], h[k]);
    }
    if (p.h != nullptr) {
      char* hrow = (char*)row_of(p.h, p.hs);
#pragma unroll
      for (int k = 0; k < N; k++)
        if (k < N - 1 || last) store8<T>(hrow + col(k) * (unsigned)sizeof(T), 0, h[k]);
    }
    if (p.norm == 2) {
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < N; k++) {
        float c = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) c += h[k][i];
        a += k < N - 1 || last ? c : 0.f;
      }
      m = wave_sum(a) * p.inv_c;
    }
    if (p.norm != 0) {
      float a = 0.f;
#pragma unroll
      for (int k = 0; k < N; k++) {
        float c = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) { const float d = h[k][i] - m; c = __builtin_fmaf(d, d, c); }
        a += k < N - 1 || last ? c : 0.f;
      }
      rs = inv_sqrt(wave_sum(a) * p.inv_c + p.eps);
    }
    const int64_t row = (int64_t)b * p.S + s;
    if (p.stats != nullptr && lane == 0) *(f32x4*)(p.stats + row * 4) = (f32x4){m, rs, ym, yr};
    if (p.norm == 0) continue;
    char* nrow = p.fp8 ? (char*)p.n + b * p.ns.b + s * p.ns.s : (char*)row_of(p.n, p.ns);
#pragma unroll
    for (int k = 0; k < N; k++) {
      float n[8], sc[8], sh[8];
      vec8(0, k, sc);
      vec8(1, k, sh);
#pragma unroll
      for (int i = 0; i < 8; i++) n[i] = __builtin_fmaf((h[k][i] - m) * rs, sc[i], sh[i]);
      const bool in = k < N - 1 || last;
      const float scale = put_row8<T>(p, n, nrow + col(k) * (p.fp8 ? 1u : (unsigned)sizeof(T)), in);
      if (p.fp8 && in && (lane & 15) == 0) p.n_scale[(int64_t)(col(k) >> 7) * p.rows + row] = scale;
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// Rows are spread over wavefronts (a workgroup to a row) where there are fewer rows than four for a compute unit, where the modulation changes
// with the row, and where a row does not fit a wavefront's registers (six chunks of 512 columns).  Both ways, bf16 with y, gate, scale
// and shift, us, workgroup and wavefront to a row: 240 x 1152 3.6 4.0, 1024 x 1152 5.0 4.6, 3000 x 1152 8.9 8.2,
// 4608 x 2560 17.4 17.4, 35552 x 1920 114 105 (5.2 TB/s), 32760 x 2560 138 130.
template <typename T, int N>
static hipError_t launch_wave(const GatedNormParams& p, hipStream_t stream) {
  static std::atomic<int> residency[kMaxDevices];
  const int lds = (p.y != nullptr ? 3 : 2) * N * 2048;
  std::atomic<int>& known = residency[current_device_slot()];
  int n = known.load(std::memory_order_relaxed);
  if (n == 0) {   // asked with the three vectors of a call with y
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&n, (const void*)gated_norm_wave_kernel<T, N>, 256, 3 * N * 2048) != hipSuccess || n <= 0) n = 1;
    known.store(n, std::memory_order_relaxed);
  }
  int64_t groups = ((int64_t)resident_cus() * n + p.B - 1) / p.B;
  if (groups > (p.S + 3) / 4) groups = (p.S + 3) / 4;
  hipLaunchKernelGGL((gated_norm_wave_kernel<T, N>), dim3((unsigned)groups, (unsigned)p.B), dim3(256), lds, stream, p);
  return hipGetLastError();
}

template <typename T>
static hipError_t run(GatedNormParams p, hipStream_t stream) {
  const bool token = (p.gate != nullptr && p.gs.s != 0) || (p.scale != nullptr && p.ss.s != 0) || (p.shift != nullptr && p.fs.s != 0);
  const int waves = (p.C + 511) / 512;
  if (!token && waves <= 6 && p.rows >= (int64_t)resident_cus() * 4) {
    if (waves <= 1) return launch_wave<T, 1>(p, stream);
    if (waves <= 2) return launch_wave<T, 2>(p, stream);
    if (waves <= 3) return launch_wave<T, 3>(p, stream);
    if (waves <= 4) return launch_wave<T, 4>(p, stream);
    if (waves <= 5) return launch_wave<T, 5>(p, stream);
    return launch_wave<T, 6>(p, stream);
  }
  const int per_simd = (waves + 3) / 4;   // of the six wavefronts (with modulation per token four) that fit a SIMD by registers
  const int64_t at_once = (int64_t)resident_cus() * ((token ? 4 : 6) / per_simd);
  p.rows_per_part = (int)((p.rows + at_once - 1) / at_once);
  const dim3 grid((unsigned)((p.S + p.rows_per_part - 1) / p.rows_per_part), (unsigned)p.B), block(64 * waves);
  if (token) hipLaunchKernelGGL((gated_norm_kernel<T, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((gated_norm_kernel<T, false>), grid, block, 0, stream, p);
  return hipGetLastError();
}

// ---- backward --------------------------------------------------------------------------------

// The two totals over a workgroup of values x, one barrier.
__device__ __forceinline__ void two_sums(float& a, float& b, int waves, int wave, int lane, Posted& post) {
  a = wave_sum(a);
  b = wave_sum(b);
  if (waves == 1) return;
  if (lane == 0) { post.v[0][wave] = a; post.v[1][wave] = b; }
  __syncthreads();
  const int k = lane >> 4, w = lane & 15;
  const float t = row16_sum(w < waves && k < 2 ? post.v[k][w] : 0.f);
  a = from_lane(t, 0);
  b = from_lane(t, 16);
}

// A workgroup runs over the rows of one part of one batch entry, as many at a time as it has teams of wavefronts (short rows
// leave room for several); a thread keeps the sums of its eight columns, and the teams' sums are added in LDS at the end.
// 8500 x 1536 fp16: 35 us, 4.5 TB/s (one team to a workgroup 44); 32760 x 5120 bf16 with the sums, a call, 458 us, 4.4 TB/s.
// The other forms spill: fp32 rows 5 registers (811 us, 5.0 TB/s), modulation per token 9, in fp32 36 (bf16 976 us, 3.8 TB/s).
template <typename T, bool TOKEN>
__global__ __launch_bounds__(1024) void gated_norm_bwd_kernel(const GatedNormBwdParams p) {
  __shared__ Posted posts[kMaxWaves][2][2];
  extern __shared__ __align__(16) float joined[];   // [3][C] where there are several teams
  const int lane = threadIdx.x & 63, waves = (p.C + 511) >> 9;
  const int team = __builtin_amdgcn_readfirstlane((int)threadIdx.x / (64 * waves)), wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6) - team * waves;
  const int chunks = p.C >> 3, place = 64 * wave + lane;   // of this thread's chunk
  Posted (&post)[2][2] = posts[team];
  const int col = (place < chunks ? place : 0) * 8;
  const int b = blockIdx.y;
  const int s0 = blockIdx.x * p.rows_per_part, s1 = min(p.S, s0 + p.rows_per_part);
  const bool has_n = p.dn != nullptr, has_y = p.y != nullptr;
  Raw8<T> rdh, rdn, rh, ry;
  f32x4 st;
  auto load = [&](int s) {
    st = *(const f32x4*)(p.stats + ((int64_t)b * p.S + s) * 4);
    if (p.dh != nullptr) rdh = load_raw8<T>(p.dh, b * p.dhs.b + s * p.dhs.s + col);
    if (has_n) {
      rdn = load_raw8<T>(p.dn, b * p.dns.b + s * p.dns.s + col);
      rh = load_raw8<T>(p.h, b * p.hs.b + s * p.hs.s + col);
    }
    if (has_y) ry = load_raw8<T>(p.y, b * p.ys.b + s * p.ys.s + col);
  };
  constexpr bool AHEAD = sizeof(T) == 2 && !TOKEN;   // the next row is requested ahead where the registers allow it (the other forms spill as it is)
  if constexpr (AHEAD) load(min(s0 + team, s1 - 1));
  float scw[8], gyw[8], sa[8] = {}, sf[8] = {}, sg[8] = {};   // (1 + scale) w, alpha gate w_y, column sums
  auto fill = [](float (&v)[8], float c) {
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = c;
  };
  auto times = [&](const void* q, int64_t off, bool wide, float plus, float (&v)[8]) {   // v *= plus + q
    if (q == nullptr) return;
    float w[8];
    load_param8<T>(q, off, wide, w);
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] *= plus + w[i];
  };
  if constexpr (!TOKEN) {
    fill(scw, 1.f);
    times(p.scale, b * p.ss.b + col, p.mod_wide, 1.f, scw);
    times(p.weight, col, p.weight_wide, 0.f, scw);
    fill(gyw, p.alpha);
    times(p.gate, b * p.gs.b + col, p.mod_wide, 0.f, gyw);
    times(p.y_weight, col, p.weight_wide, 0.f, gyw);
  }
  for (int first = s0, turn = 0; first < s1; first += p.teams, turn ^= 1) {
    const bool there = first + team < s1;            // a team without a row goes through the motions: the barriers are everybody's
    const bool live = there && place < chunks;
    const int s = min(first + team, s1 - 1);
    const int64_t row = (int64_t)b * p.S + s;
    if constexpr (!AHEAD) load(s);
    const f32x4 now = st;
    float t[8], du[8], u[8];
    fill(t, 0.f);
    if (p.dh != nullptr) get8(rdh, t);
    if (has_n) { get8(rdn, du); get8(rh, u); }
    const Raw8<T> y_now = ry;
    if (AHEAD && first + p.teams < s1) load(min(first + p.teams + team, s1 - 1));
    if (has_n) {
#pragma unroll
      for (int i = 0; i < 8; i++) u[i] = (u[i] - now[0]) * now[1];
      if constexpr (!TOKEN) {
#pragma unroll
        for (int i = 0; i < 8; i++) { sa[i] += there ? du[i] * u[i] : 0.f; sf[i] += there ? du[i] : 0.f; du[i] *= scw[i]; }
      } else {
        if (p.mod_per_token && live && p.dshift != nullptr) store_param8<T>(p.dshift, row * p.C + col, p.mod_wide, du);
        if (p.mod_per_token && live && p.dscale != nullptr) {
          float d[8], bi[8];
#pragma unroll
          for (int i = 0; i < 8; i++) d[i] = u[i];
          times(p.weight, col, p.weight_wide, 0.f, d);
          fill(bi, 0.f);
          if (p.bias != nullptr) load_param8<T>(p.bias, col, p.weight_wide, bi);
#pragma unroll
          for (int i = 0; i < 8; i++) d[i] = du[i] * (d[i] + bi[i]);
          store_param8<T>(p.dscale, row * p.C + col, p.mod_wide, d);
        }
        if (p.mod_per_token) times(p.scale, b * p.ss.b + s * p.ss.s + col, p.mod_wide, 1.f, du);
#pragma unroll
        for (int i = 0; i < 8; i++) { sa[i] += there ? du[i] * u[i] : 0.f; sf[i] += there ? du[i] : 0.f; }
        if (!p.mod_per_token) times(p.scale, b * p.ss.b + col, p.mod_wide, 1.f, du);
        times(p.weight, col, p.weight_wide, 0.f, du);
      }
      float a = 0.f, d = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) { a += du[i]; d += du[i] * u[i]; }
      a = live ? a : 0.f;
      d = live ? d : 0.f;
      two_sums(a, d, waves, wave, lane, post[turn][0]);
      const float mean = p.norm == 2 ? a * p.inv_c : 0.f, dot = d * p.inv_c;
#pragma unroll
      for (int i = 0; i < 8; i++) t[i] += now[1] * (du[i] - mean - u[i] * dot);
    }
    if (p.dx != nullptr && live) store8<T>(p.dx, b * p.dxs.b + s * p.dxs.s + col, t);
    if (!has_y) continue;
    float z[8];   // t becomes e
    get8(y_now, z);
#pragma unroll
    for (int i = 0; i < 8; i++) z[i] = (z[i] - now[2]) * now[3];
    if constexpr (!TOKEN) {
#pragma unroll
      for (int i = 0; i < 8; i++) { sg[i] += there ? t[i] * z[i] : 0.f; t[i] *= gyw[i]; }
    } else {
      if (p.gate_per_token && live && p.dgate != nullptr) {
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; i++) d[i] = p.alpha * t[i] * z[i];
        times(p.y_weight, col, p.weight_wide, 0.f, d);
        store_param8<T>(p.dgate, row * p.C + col, p.mod_wide, d);
      }
      if (!p.gate_per_token) {
#pragma unroll
        for (int i = 0; i < 8; i++) sg[i] += there ? t[i] * z[i] : 0.f;
      }
#pragma unroll
      for (int i = 0; i < 8; i++) t[i] *= p.alpha;
      times(p.gate, b * p.gs.b + s * p.gs.s + col, p.mod_wide, 0.f, t);
      if (p.gate_per_token) {
#pragma unroll
        for (int i = 0; i < 8; i++) sg[i] += there ? t[i] * z[i] : 0.f;
      }
      times(p.y_weight, col, p.weight_wide, 0.f, t);
    }
    if (p.y_norm != 0) {
      float a = 0.f, d = 0.f;
#pragma unroll
      for (int i = 0; i < 8; i++) { a += t[i]; d += t[i] * z[i]; }
      a = live ? a : 0.f;
      d = live ? d : 0.f;
      two_sums(a, d, waves, wave, lane, post[turn][1]);
      const float mean = p.y_norm == 2 ? a * p.inv_c : 0.f, dot = d * p.inv_c;
#pragma unroll
      for (int i = 0; i < 8; i++) t[i] = now[3] * (t[i] - mean - z[i] * dot);
    }
    if (p.dy != nullptr && live) store8<T>(p.dy, b * p.dys.b + s * p.dys.s + col, t);
  }
  if (!p.sums) return;
  for (int t = 1; t < p.teams; t++) {   // the last team's sums, plus the one's before, and so on
    if (t > 1) __syncthreads();
    if (team == p.teams - t && place < chunks) {
      store8<float>(joined, col, sa);
      store8<float>(joined, p.C + col, sf);
      store8<float>(joined, 2 * p.C + col, sg);
    }
    __syncthreads();
    if (team == p.teams - t - 1 && place < chunks) {
      float v[8];
      auto add = [&](int vec, float (&sum)[8]) {
        get8(load_raw8<float>(joined, vec * p.C + col), v);
#pragma unroll
        for (int i = 0; i < 8; i++) sum[i] += v[i];
      };
      add(0, sa);
      add(1, sf);
      add(2, sg);
    }
  }
  if (team != 0 || place >= chunks) return;
  float* out = p.partial + ((int64_t)b * p.parts + blockIdx.x) * 3 * p.C;
  store8<float>(out, col, sa);
  store8<float>(out, p.C + col, sf);
  store8<float>(out, 2 * (int64_t)p.C + col, sg);
}

template <typename T>
__device__ __forceinline__ float param_at(const void* p, int64_t i, bool wide) { return wide ? ((const float*)p)[i] : (float)((const T*)p)[i]; }
template <typename T>
__device__ __forceinline__ void put_param(void* p, int64_t i, bool wide, float v) {
  if (wide) ((float*)p)[i] = v;
  else ((T*)p)[i] = (T)v;
}

// The parts' sums, added in a fixed order (64 runs of every 64th part, then the runs), and from them the parameters'
// gradients; 16 columns per workgroup, one batch entry after the other: 2 entries of 1536 columns 7 us, 1024 entries 1.7 ms.
template <typename T>
__global__ __launch_bounds__(1024) void gated_norm_bwd_finish_kernel(const GatedNormBwdParams p) {
  constexpr int RUNS = 64;
  __shared__ float runs[3][RUNS][17], totals[3][16];
  const int k = threadIdx.x & 15, run = threadIdx.x >> 4;
  const int c = blockIdx.x * 16 + k;
  const bool live = c < p.C;
  const int cc = live ? c : 0;
  // parameters are requested ahead of the sums that they are multiplied with
  const float w = p.weight != nullptr ? param_at<T>(p.weight, cc, p.weight_wide) : 1.f, bi = p.bias != nullptr ? param_at<T>(p.bias, cc, p.weight_wide) : 0.f;
  const float yw = p.y_weight != nullptr ? param_at<T>(p.y_weight, cc, p.weight_wide) : 1.f;
  float dw = 0.f, db = 0.f, dyw = 0.f;
  for (int b = 0; b < p.B; b++) {
    const float sc = p.scale != nullptr && !p.mod_per_token ? 1.f + param_at<T>(p.scale, b * p.ss.b + cc, p.mod_wide) : 1.f;
    const float ga = p.alpha * (p.gate != nullptr && !p.gate_per_token ? param_at<T>(p.gate, b * p.gs.b + cc, p.mod_wide) : 1.f);
    float a = 0.f, f = 0.f, g = 0.f;
    const float* in = p.partial + ((int64_t)b * p.parts + run) * 3 * p.C + cc;
#pragma unroll 8
    for (int i = run; i < p.parts; i += RUNS, in += RUNS * 3 * (int64_t)p.C) { a += in[0]; f += in[p.C]; g += in[2 * (int64_t)p.C]; }
    __syncthreads();   // the sums of the batch entry before have been read
    runs[0][run][k] = a;
    runs[1][run][k] = f;
    runs[2][run][k] = g;
    __syncthreads();
    for (int i = threadIdx.x >> 6; i < 48; i += 16) {   // a wavefront adds the 64 runs of a column
      const float t = wave_sum(runs[i >> 4][threadIdx.x & 63][i & 15]);
      if ((threadIdx.x & 63) == 0) totals[i >> 4][i & 15] = t;
    }
    __syncthreads();
    if (run != 0 || !live) continue;
    a = totals[0][k];
    f = totals[1][k];
    g = totals[2][k];
    if (p.mod_per_token) {
      dw += a;
      db += f;
    } else {
      if (p.dshift != nullptr) put_param<T>(p.dshift, (int64_t)b * p.C + c, p.mod_wide, f);
      if (p.dscale != nullptr) put_param<T>(p.dscale, (int64_t)b * p.C + c, p.mod_wide, w * a + bi * f);
      dw += sc * a;
      db += sc * f;
    }
    if (p.gate_per_token) {
      dyw += g;
    } else {
      if (p.dgate != nullptr) put_param<T>(p.dgate, (int64_t)b * p.C + c, p.mod_wide, p.alpha * yw * g);
      dyw += ga * g;
    }
  }
  if (run != 0 || !live) return;
  if (p.dweight != nullptr) put_param<T>(p.dweight, c, p.weight_wide, dw);
  if (p.dbias != nullptr) put_param<T>(p.dbias, c, p.weight_wide, db);
  if (p.dy_weight != nullptr) put_param<T>(p.dy_weight, c, p.weight_wide, dyw);
}

template <typename T>
static hipError_t run_bwd(const GatedNormBwdParams& p, hipStream_t stream) {
  const dim3 grid((unsigned)p.parts, (unsigned)p.B), block(64 * ((p.C + 511) / 512) * p.teams);
  const int lds = p.teams > 1 ? 12 * p.C : 0;   // several teams: rows of up to 4096 columns
  if (p.mod_per_token || p.gate_per_token) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, true>), grid, block, lds, stream, p);
  else hipLaunchKernelGGL((gated_norm_bwd_kernel<T, false>), grid, block, lds, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.sums) return e;
  hipLaunchKernelGGL((gated_norm_bwd_finish_kernel<T>), dim3((unsigned)((p.C + 15) / 16)), dim3(1024), 0, stream, p);
  return hipGetLastError();
}

}  // namespace gnorm

hipError_t launch_gated_norm(const GatedNormParams& p, int dtype, hipStream_t stream) {
  if (dtype == 0) return gnorm::run<__bf16>(p, stream);
  if (dtype == 1) return gnorm::run<_Float16>(p, stream);
  if (dtype == 2) return gnorm::run<float>(p, stream);
  return hipErrorInvalidValue;
}

// Workgroups of up to 16 wavefronts, one on a compute unit (by registers), each with as many teams as fit; a part has two rows
// for every team at least, so that writing and reading a part's sums (24 C bytes) stays beside the rows' 12 C and more.
void gated_norm_bwd_plan(GatedNormBwdParams& p) {
  const bool mods = !p.mod_per_token && (p.dscale != nullptr || p.dshift != nullptr);
  p.sums = mods || (!p.gate_per_token && p.dgate != nullptr) || p.dweight != nullptr || p.dbias != nullptr || p.dy_weight != nullptr;
  const int waves = (p.C + 511) / 512;
  p.teams = 16 / waves;
  const int64_t cus = resident_cus();
  int64_t per = ((int64_t)p.B * p.S + cus - 1) / cus;
  while (p.teams > 1 && p.teams > per) p.teams /= 2;   // few rows: smaller workgroups, more of them
  if (p.sums && per < 2 * p.teams) per = 2 * p.teams;
  if (per > p.S) per = p.S;
  p.rows_per_part = (int)per;
  p.parts = (int)((p.S + per - 1) / per);
}

hipError_t launch_gated_norm_bwd(const GatedNormBwdParams& p, int dtype, hipStream_t stream) {
  if (dtype == 0) return gnorm::run_bwd<__bf16>(p, stream);
  if (dtype == 1) return gnorm::run_bwd<_Float16>(p, stream);
  if (dtype == 2) return gnorm::run_bwd<float>(p, stream);
  return hipErrorInvalidValue;
}

}  // namespace xdit
