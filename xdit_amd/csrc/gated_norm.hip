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
#include "block_params.h"
#include "row_ops.h"

namespace xdit {

namespace gnorm {

// One workgroup of four wavefronts per row; a thread holds up to N chunks of 8 columns (thread, thread + 256, ...).
template <typename T, int N>
__global__ __launch_bounds__(256) void gated_norm_row_kernel(const GatedNormParams p) {
  __shared__ float part[4][8];
  const int64_t row = blockIdx.x;
  const int b = (int)(row / p.S);
  const int s = (int)(row - (int64_t)b * p.S);
  const int chunks = p.C >> 3;
  float h[N][8];
  float ym = 0.f, yr = 1.f, m = 0.f, r = 1.f;
  bool live[N];
  int col[N];
#pragma unroll
  for (int k = 0; k < N; k++) {
    const int c = threadIdx.x + 256 * k;
    live[k] = c < chunks;
    col[k] = (live[k] ? c : 0) * 8;
    get8(load_raw8<T>(p.x, b * p.xs.b + s * p.xs.s + col[k]), h[k]);
  }
  if (p.y != nullptr) {
    float v[N][8];
#pragma unroll
    for (int k = 0; k < N; k++) get8(load_raw8<T>(p.y, b * p.ys.b + s * p.ys.s + col[k]), v[k]);
    if (p.y_norm == 2) {
      float a[1] = {0.f};
#pragma unroll
      for (int k = 0; k < N; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) a[0] += live[k] ? v[k][i] : 0.f;
      block_sums<1, 4>(a, part[0]);
      ym = a[0] * p.inv_c;
    }
    if (p.y_norm != 0) {
      float a[1] = {0.f};
#pragma unroll
      for (int k = 0; k < N; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) { const float d = v[k][i] - ym; a[0] += live[k] ? d * d : 0.f; }
      block_sums<1, 4>(a, part[1]);
      yr = 1.0f / sqrtf(a[0] * p.inv_c + p.y_eps);
    }
#pragma unroll
    for (int k = 0; k < N; k++) {
      float g[8], w[8];
      if (p.y_norm != 0) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[k][i] = (v[k][i] - ym) * yr;
      }
      if (p.y_weight != nullptr) {
        load_param8<T>(p.y_weight, col[k], p.weight_wide, w);
#pragma unroll
        for (int i = 0; i < 8; i++) v[k][i] *= w[i];
      }
      if (p.gate != nullptr) {
        load_param8<T>(p.gate, b * p.gs.b + s * p.gs.s + col[k], p.mod_wide, g);
#pragma unroll
        for (int i = 0; i < 8; i++) v[k][i] *= g[i];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) h[k][i] += p.alpha * v[k][i];
    }
  }
  if (p.h != nullptr) {
#pragma unroll
    for (int k = 0; k < N; k++)
      if (live[k]) store8<T>(p.h, b * p.hs.b + s * p.hs.s + col[k], h[k]);
  }
  if (p.norm == 2) {
    float a[1] = {0.f};
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
      for (int i = 0; i < 8; i++) a[0] += live[k] ? h[k][i] : 0.f;
    block_sums<1, 4>(a, part[2]);
    m = a[0] * p.inv_c;
  }
  if (p.norm != 0) {
    float a[1] = {0.f};
#pragma unroll
    for (int k = 0; k < N; k++)
#pragma unroll
      for (int i = 0; i < 8; i++) { const float d = h[k][i] - m; a[0] += live[k] ? d * d : 0.f; }
    block_sums<1, 4>(a, part[3]);
    r = 1.0f / sqrtf(a[0] * p.inv_c + p.eps);
  }
  if (p.stats != nullptr && threadIdx.x == 0) *(f32x4*)(p.stats + row * 4) = (f32x4){m, r, ym, yr};
  if (p.norm == 0) return;
#pragma unroll
  for (int k = 0; k < N; k++) {
    float v[8], w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) v[i] = (h[k][i] - m) * r;
    if (p.weight != nullptr) {
      load_param8<T>(p.weight, col[k], p.weight_wide, w);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] *= w[i];
    }
    if (p.bias != nullptr) {
      load_param8<T>(p.bias, col[k], p.weight_wide, w);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += w[i];
    }
    if (p.scale != nullptr) {
      load_param8<T>(p.scale, b * p.ss.b + s * p.ss.s + col[k], p.mod_wide, w);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] *= 1.0f + w[i];
    }
    if (p.shift != nullptr) {
      load_param8<T>(p.shift, b * p.fs.b + s * p.fs.s + col[k], p.mod_wide, w);
#pragma unroll
      for (int i = 0; i < 8; i++) v[i] += w[i];
    }
    if (!p.fp8) {
      if (live[k]) store8<T>(p.n, b * p.ns.b + s * p.ns.s + col[k], v);
    } else {  // a block of 128 columns is a DPP row: 16 lanes of 8 columns
      const Divider div(block_scale(row16_max(live[k] ? absmax8(v) : 0)));
      const i32x2 q = cast8(v, div);
      if (live[k]) {
        *(i32x2*)((unsigned char*)p.n + b * p.ns.b + s * p.ns.s + col[k]) = q;
        if ((threadIdx.x & 15) == 0) p.n_scale[(int64_t)(col[k] >> 7) * p.rows + row] = div.scale;
      }
    }
  }
}

template <typename T>
static hipError_t run(const GatedNormParams& p, hipStream_t stream) {
  const int n = (p.C + 2047) / 2048;
  const dim3 grid((unsigned)p.rows), block(256);
  if (n <= 1) hipLaunchKernelGGL((gated_norm_row_kernel<T, 1>), grid, block, 0, stream, p);
  else if (n <= 2) hipLaunchKernelGGL((gated_norm_row_kernel<T, 2>), grid, block, 0, stream, p);
  else if (n <= 3) hipLaunchKernelGGL((gated_norm_row_kernel<T, 3>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((gated_norm_row_kernel<T, 4>), grid, block, 0, stream, p);
  return hipGetLastError();
}

// ---- backward --------------------------------------------------------------------------------

// A workgroup runs over the rows of one part of one batch entry; a thread keeps the column sums of its chunks.
template <typename T, int N>
__global__ __launch_bounds__(256) void gated_norm_bwd_kernel(const GatedNormBwdParams p) {
  __shared__ float part[4][8];
  const int b = blockIdx.y;
  const int s0 = blockIdx.x * p.rows_per_part;
  const int s1 = min(p.S, s0 + p.rows_per_part);
  const int chunks = p.C >> 3;
  float sa[N][8] = {}, sf[N][8] = {}, sg[N][8] = {};
  bool live[N];
  int col[N];
#pragma unroll
  for (int k = 0; k < N; k++) {
    const int c = threadIdx.x + 256 * k;
    live[k] = c < chunks;
    col[k] = (live[k] ? c : 0) * 8;
  }
  for (int s = s0; s < s1; s++) {
    const int64_t row = (int64_t)b * p.S + s;
    const f32x4 st = *(const f32x4*)(p.stats + row * 4);
    float t[N][8], du[N][8], u[N][8];
    float a[2] = {0.f, 0.f};
#pragma unroll
    for (int k = 0; k < N; k++) {
#pragma unroll
      for (int i = 0; i < 8; i++) t[k][i] = 0.f;
      if (p.dh != nullptr) get8(load_raw8<T>(p.dh, b * p.dhs.b + s * p.dhs.s + col[k]), t[k]);
      if (p.dn != nullptr) {
        float w[8], bi[8];
        get8(load_raw8<T>(p.dn, b * p.dns.b + s * p.dns.s + col[k]), du[k]);
        get8(load_raw8<T>(p.h, b * p.hs.b + s * p.hs.s + col[k]), u[k]);
#pragma unroll
        for (int i = 0; i < 8; i++) u[k][i] = (u[k][i] - st[0]) * st[1];
        if (p.mod_per_token) {
          if (live[k] && p.dshift != nullptr) store_param8<T>(p.dshift, row * p.C + col[k], p.mod_wide, du[k]);
          if (live[k] && p.dscale != nullptr) {
            float d[8];
#pragma unroll
            for (int i = 0; i < 8; i++) d[i] = u[k][i];
            if (p.weight != nullptr) {
              load_param8<T>(p.weight, col[k], p.weight_wide, w);
#pragma unroll
              for (int i = 0; i < 8; i++) d[i] *= w[i];
            }
            if (p.bias != nullptr) {
              load_param8<T>(p.bias, col[k], p.weight_wide, bi);
#pragma unroll
              for (int i = 0; i < 8; i++) d[i] += bi[i];
            }
#pragma unroll
            for (int i = 0; i < 8; i++) d[i] *= du[k][i];
            store_param8<T>(p.dscale, row * p.C + col[k], p.mod_wide, d);
          }
        }
        float sc[8];
        if (p.scale != nullptr) load_param8<T>(p.scale, b * p.ss.b + s * p.ss.s + col[k], p.mod_wide, sc);
        if (p.scale != nullptr && p.mod_per_token) {
#pragma unroll
          for (int i = 0; i < 8; i++) du[k][i] *= 1.0f + sc[i];
        }
#pragma unroll
        for (int i = 0; i < 8; i++) { sa[k][i] += du[k][i] * u[k][i]; sf[k][i] += du[k][i]; }
        if (p.scale != nullptr && !p.mod_per_token) {
#pragma unroll
          for (int i = 0; i < 8; i++) du[k][i] *= 1.0f + sc[i];
        }
        if (p.weight != nullptr) {
          load_param8<T>(p.weight, col[k], p.weight_wide, w);
#pragma unroll
          for (int i = 0; i < 8; i++) du[k][i] *= w[i];
        }
        if (live[k]) {
#pragma unroll
          for (int i = 0; i < 8; i++) { a[0] += du[k][i]; a[1] += du[k][i] * u[k][i]; }
        }
      }
    }
    if (p.dn != nullptr) {
      block_sums<2, 4>(a, part[(s - s0) & 1]);
      const float mean = p.norm == 2 ? a[0] * p.inv_c : 0.f, dot = a[1] * p.inv_c;
#pragma unroll
      for (int k = 0; k < N; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) t[k][i] += st[1] * (du[k][i] - mean - u[k][i] * dot);
    }
    if (p.dx != nullptr) {
#pragma unroll
      for (int k = 0; k < N; k++)
        if (live[k]) store8<T>(p.dx, b * p.dxs.b + s * p.dxs.s + col[k], t[k]);
    }
    if (p.y == nullptr) continue;
    // t becomes e, u becomes z
    a[0] = a[1] = 0.f;
#pragma unroll
    for (int k = 0; k < N; k++) {
      float g[8], w[8];
      get8(load_raw8<T>(p.y, b * p.ys.b + s * p.ys.s + col[k]), u[k]);
#pragma unroll
      for (int i = 0; i < 8; i++) u[k][i] = (u[k][i] - st[2]) * st[3];
      if (p.y_weight != nullptr) load_param8<T>(p.y_weight, col[k], p.weight_wide, w);
      if (p.gate_per_token && p.dgate != nullptr && live[k]) {
        float d[8];
#pragma unroll
        for (int i = 0; i < 8; i++) d[i] = p.alpha * t[k][i] * (p.y_weight != nullptr ? u[k][i] * w[i] : u[k][i]);
        store_param8<T>(p.dgate, row * p.C + col[k], p.mod_wide, d);
      }
      if (p.gate != nullptr) load_param8<T>(p.gate, b * p.gs.b + s * p.gs.s + col[k], p.mod_wide, g);
      if (!p.gate_per_token) {
#pragma unroll
        for (int i = 0; i < 8; i++) sg[k][i] += t[k][i] * u[k][i];
      }
#pragma unroll
      for (int i = 0; i < 8; i++) t[k][i] *= p.gate != nullptr ? p.alpha * g[i] : p.alpha;
      if (p.gate_per_token) {
#pragma unroll
        for (int i = 0; i < 8; i++) sg[k][i] += t[k][i] * u[k][i];
      }
      if (p.y_weight != nullptr) {
#pragma unroll
        for (int i = 0; i < 8; i++) t[k][i] *= w[i];
      }
      if (live[k]) {
#pragma unroll
        for (int i = 0; i < 8; i++) { a[0] += t[k][i]; a[1] += t[k][i] * u[k][i]; }
      }
    }
    if (p.y_norm != 0) {
      block_sums<2, 4>(a, part[2 + ((s - s0) & 1)]);
      const float mean = p.y_norm == 2 ? a[0] * p.inv_c : 0.f, dot = a[1] * p.inv_c;
#pragma unroll
      for (int k = 0; k < N; k++)
#pragma unroll
        for (int i = 0; i < 8; i++) t[k][i] = st[3] * (t[k][i] - mean - u[k][i] * dot);
    }
    if (p.dy != nullptr) {
#pragma unroll
      for (int k = 0; k < N; k++)
        if (live[k]) store8<T>(p.dy, b * p.dys.b + s * p.dys.s + col[k], t[k]);
    }
  }
  if (!p.sums) return;
  float* out = p.partial + ((int64_t)b * p.parts + blockIdx.x) * 3 * p.C;
#pragma unroll
  for (int k = 0; k < N; k++) {
    if (!live[k]) continue;
    store8<float>(out, col[k], sa[k]);
    store8<float>(out, p.C + col[k], sf[k]);
    store8<float>(out, 2 * (int64_t)p.C + col[k], sg[k]);
  }
}

template <typename T>
__device__ __forceinline__ float param_at(const void* p, int64_t i, bool wide) { return wide ? ((const float*)p)[i] : (float)((const T*)p)[i]; }
template <typename T>
__device__ __forceinline__ void put_param(void* p, int64_t i, bool wide, float v) {
  if (wide) ((float*)p)[i] = v;
  else ((T*)p)[i] = (T)v;
}

// The parts' sums, added in their order, and from them the parameters' gradients; one thread per column.
template <typename T>
__global__ __launch_bounds__(256) void gated_norm_bwd_finish_kernel(const GatedNormBwdParams p) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= p.C) return;
  const float w = p.weight != nullptr ? param_at<T>(p.weight, c, p.weight_wide) : 1.f;
  const float bi = p.bias != nullptr ? param_at<T>(p.bias, c, p.weight_wide) : 0.f;
  const float yw = p.y_weight != nullptr ? param_at<T>(p.y_weight, c, p.weight_wide) : 1.f;
  float dw = 0.f, db = 0.f, dyw = 0.f;
  for (int b = 0; b < p.B; b++) {
    float a = 0.f, f = 0.f, g = 0.f;
    const float* in = p.partial + (int64_t)b * p.parts * 3 * p.C + c;
    for (int i = 0; i < p.parts; i++, in += 3 * (int64_t)p.C) { a += in[0]; f += in[p.C]; g += in[2 * (int64_t)p.C]; }
    if (p.mod_per_token) {
      dw += a;
      db += f;
    } else {
      const float sc = p.scale != nullptr ? 1.f + param_at<T>(p.scale, b * p.ss.b + c, p.mod_wide) : 1.f;
      if (p.dshift != nullptr) put_param<T>(p.dshift, (int64_t)b * p.C + c, p.mod_wide, f);
      if (p.dscale != nullptr) put_param<T>(p.dscale, (int64_t)b * p.C + c, p.mod_wide, w * a + bi * f);
      dw += sc * a;
      db += sc * f;
    }
    if (p.gate_per_token) {
      dyw += g;
    } else {
      const float ga = p.gate != nullptr ? param_at<T>(p.gate, b * p.gs.b + c, p.mod_wide) : 1.f;
      if (p.dgate != nullptr) put_param<T>(p.dgate, (int64_t)b * p.C + c, p.mod_wide, p.alpha * yw * g);
      dyw += p.alpha * ga * g;
    }
  }
  if (p.dweight != nullptr) put_param<T>(p.dweight, c, p.weight_wide, dw);
  if (p.dbias != nullptr) put_param<T>(p.dbias, c, p.weight_wide, db);
  if (p.dy_weight != nullptr) put_param<T>(p.dy_weight, c, p.weight_wide, dyw);
}

template <typename T>
static hipError_t run_bwd(const GatedNormBwdParams& p, hipStream_t stream) {
  const int n = (p.C + 2047) / 2048;
  const dim3 grid((unsigned)p.parts, (unsigned)p.B), block(256);
  if (n <= 1) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, 1>), grid, block, 0, stream, p);
  else if (n <= 2) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, 2>), grid, block, 0, stream, p);
  else if (n <= 3) hipLaunchKernelGGL((gated_norm_bwd_kernel<T, 3>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((gated_norm_bwd_kernel<T, 4>), grid, block, 0, stream, p);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.sums) return e;
  hipLaunchKernelGGL((gated_norm_bwd_finish_kernel<T>), dim3((unsigned)((p.C + 255) / 256)), dim3(256), 0, stream, p);
  return hipGetLastError();
}

}  // namespace gnorm

hipError_t launch_gated_norm(const GatedNormParams& p, int dtype, hipStream_t stream) {
  if (dtype == 0) return gnorm::run<__bf16>(p, stream);
  if (dtype == 1) return gnorm::run<_Float16>(p, stream);
  if (dtype == 2) return gnorm::run<float>(p, stream);
  return hipErrorInvalidValue;
}

// Parts: enough workgroups to fill the chip (4 per compute unit), at least 16 rows each where there are that many.
void gated_norm_bwd_plan(GatedNormBwdParams& p) {
  const bool mods = !p.mod_per_token && (p.dscale != nullptr || p.dshift != nullptr);
  p.sums = mods || (!p.gate_per_token && p.dgate != nullptr) || p.dweight != nullptr || p.dbias != nullptr || p.dy_weight != nullptr;
  int per = (int)(((int64_t)p.B * p.S + 1023) / 1024);
  if (p.sums && per < 16) per = 16;
  if (per > p.S) per = p.S;
  p.rows_per_part = per;
  p.parts = (p.S + per - 1) / per;
}

hipError_t launch_gated_norm_bwd(const GatedNormBwdParams& p, int dtype, hipStream_t stream) {
  if (dtype == 0) return gnorm::run_bwd<__bf16>(p, stream);
  if (dtype == 1) return gnorm::run_bwd<_Float16>(p, stream);
  if (dtype == 2) return gnorm::run_bwd<float>(p, stream);
  return hipErrorInvalidValue;
}

}  // namespace xdit
