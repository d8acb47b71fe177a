// Rotary positions on several axes, after an optional RMSNorm over head_dim, forward and backward, for gfx950.
//
//     phi = position[token, axis(p)] * inv_freq[p] ;  (x1, x2) -> (x1 cos phi - x2 sin phi, x1 sin phi + x2 cos phi)
// Backward: the rotation by -phi gives d; with the norm x^ = x r, y = x^ w before the rotation,
//     dx = r (w d - x^ mean(w d x^)) ,  dw = sum over rows of d x^ .
// The angle is brought into [-1/2, 1/2] turns in fp64 (a position of 10^5 would cost an fp32 angle five digits); the
// rest is fp32 and the result is rounded once.  HBM-bound: every row is read and written once (backward with the norm:
// two reads); a token's sines and cosines are computed once, by the wavefront that goes over all of its heads, where
// tables would be 8 bytes per element of a head and token.
#include "block_params.h"
#include "row_ops.h"

namespace xdit {

namespace axrope {

template <typename T> struct Four { typedef __attribute__((ext_vector_type(4))) T vec; };
template <typename T> struct Pair { typename Four<T>::vec lo, hi; };

// What a lane holds of a row: four pairs, as two groups of four consecutive elements at columns `a` and `b` (one group
// of eight where they touch: interleaved pairs, and the columns behind the rotated ones).
template <typename T, bool SPLIT> struct RowPart {   // as loaded
  typename Four<T>::vec lo, hi;
  __device__ __forceinline__ void load(const void* p, int64_t off, int a, int b) {
    if constexpr (SPLIT) {
      lo = *(const typename Four<T>::vec*)((const T*)p + off + a);
      hi = *(const typename Four<T>::vec*)((const T*)p + off + b);
    } else {
      const Raw8<T> r = load_raw8<T>(p, off + a);
      lo = __builtin_bit_cast(Pair<T>, r).lo;
      hi = __builtin_bit_cast(Pair<T>, r).hi;
    }
  }
  __device__ __forceinline__ void get(float (&v)[8]) const {
#pragma unroll
    for (int i = 0; i < 4; i++) { v[i] = (float)lo[i]; v[4 + i] = (float)hi[i]; }
  }
};
template <typename T, bool SPLIT>
__device__ __forceinline__ void load_row(const void* p, int64_t off, int a, int b, float (&v)[8]) {
  RowPart<T, SPLIT> r;
  r.load(p, off, a, b);
  r.get(v);
}
template <typename T, bool SPLIT>
__device__ __forceinline__ void store_row(void* p, int64_t off, int a, int b, const float (&v)[8]) {
  if constexpr (SPLIT) {
    typename Four<T>::vec lo, hi;
#pragma unroll
    for (int i = 0; i < 4; i++) { lo[i] = (T)v[i]; hi[i] = (T)v[4 + i]; }
    *(typename Four<T>::vec*)((T*)p + off + a) = lo;
    *(typename Four<T>::vec*)((T*)p + off + b) = hi;
  } else {
    store8<T>(p, off + a, v);
  }
}
template <typename T, bool SPLIT>
__device__ __forceinline__ void load_gain(const void* p, bool wide, int a, int b, float (&v)[8]) {
  if (wide) load_row<float, SPLIT>(p, 0, a, b, v);
  else load_row<T, SPLIT>(p, 0, a, b, v);
}

template <bool SPLIT>
__device__ __forceinline__ void rotate(float (&v)[8], const float (&cs)[4], const float (&sn)[4]) {
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int i1 = SPLIT ? j : 2 * j, i2 = SPLIT ? 4 + j : 2 * j + 1;
    const float x1 = v[i1], x2 = v[i2];
    v[i1] = x1 * cs[j] - x2 * sn[j];
    v[i2] = x1 * sn[j] + x2 * cs[j];
  }
}

// Sum over the `lpr` consecutive lanes (a power of two, uniform) that hold a row, to all of them.
__device__ __forceinline__ float row_sum(float x, int lpr) {
  if (lpr >= 2) x = dpp_plus<0xB1>(x);    // quad_perm [1,0,3,2]
  if (lpr >= 4) x = dpp_plus<0x4E>(x);    // quad_perm [2,3,0,1]
  if (lpr >= 8) x = dpp_plus<0x141>(x);   // row_half_mirror
  if (lpr >= 16) x = dpp_plus<0x140>(x);  // row_mirror
  if (lpr >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  if (lpr >= 64) x = sum_halves(x);
  return x;
}

// Sines and cosines of the four pairs of lane chunk c at token (b, s); sign -1 turns back.  16-bit tensors take the hardware's
// sine and cosine of a part of a turn (off by at most 1.3e-7, against the 2^-9 or 2^-12 of the result's rounding).
template <bool EXACT>
__device__ __forceinline__ void turn(const AxesRopeParams& p, int b, int s, int c, float sign, float (&cs)[4], float (&sn)[4]) {
#pragma unroll
  for (int j = 0; j < 4; j++) { cs[j] = 1.f; sn[j] = 0.f; }
  if (4 * c >= p.P) return;  // P is a multiple of 4: a lane's pairs are rotated together
#pragma unroll
  for (int j = 0; j < 4; j++) {
    const int q = 4 * c + j;
    const int axis = (q >= p.axis_end[0]) + (q >= p.axis_end[1]) + (q >= p.axis_end[2]);
    const int64_t at = b * p.ps_b + s * p.ps_s + axis;
    const double pos = p.pos_bits == -32 ? (double)((const float*)p.positions)[at] : p.pos_bits == 32 ? (double)((const int*)p.positions)[at] : (double)((const int64_t*)p.positions)[at];
    const double f = p.freq_wide ? ((const double*)p.inv_freq)[q] : (double)((const float*)p.inv_freq)[q];
    const double turns = pos * (f * 0.15915494309189533577);  // 1 / (2 pi)
    const float r = (float)(turns - rint(turns));
    if constexpr (EXACT) {
      sincospif(2.f * r, &sn[j], &cs[j]);
    } else {
      sn[j] = __builtin_amdgcn_sinf(r);
      cs[j] = __builtin_amdgcn_cosf(r);
    }
    sn[j] *= sign;
  }
}

// One wavefront per token and head group: `lpr` lanes per row, 64 / lpr heads at a time.  32760 tokens of 40 + 40 heads of 128: 264 us, 5.1 TB/s
// (fp32, a call, 549 us, 4.9 TB/s).
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256) void axes_rope_kernel(const AxesRopeParams p) {
  const unsigned tok = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // uniform, as everything of the token
  if (tok >= (unsigned)p.B * (unsigned)p.S) return;
  const int lane = threadIdx.x & 63;
  const int c = lane & (p.lpr - 1), slot = lane / p.lpr, slots = 64 / p.lpr;
  const bool live = c * 8 < p.D;
  const int cc = live ? c : 0;
  const bool apart = SPLIT && 4 * cc < p.P;
  const int ca = apart ? 4 * cc : 8 * cc, cb = apart ? p.P + 4 * cc : 8 * cc + 4;
  const int b = (int)(tok / (unsigned)p.S), s = (int)(tok - (unsigned)b * (unsigned)p.S);
  float cs[4], sn[4];
  turn<sizeof(T) == 4>(p, b, s, cc, 1.f, cs, sn);
  const int g0 = blockIdx.y * p.heads_per_wave, g1 = g0 + p.heads_per_wave;
  int base = 0;
  for (int t = 0; t < p.tensors; t++) {
    const RopeTensor& q = p.t[t];
    const int h_begin = max(0, g0 - base), h_end = min(q.H, g1 - base);
    base += q.H;
    float w[8];
#pragma unroll
    for (int i = 0; i < 8; i++) w[i] = 1.f;
    if (q.weight != nullptr && h_begin < h_end) load_gain<T, SPLIT>(q.weight, p.weight_wide, ca, cb, w);
    for (int h0 = h_begin; h0 < h_end; h0 += slots) {
      const int h = h0 + slot;
      const int hc = h < h_end ? h : h_end - 1;
      float v[8];
      load_row<T, SPLIT>(q.x, b * q.xs_b + hc * q.xs_h + s * q.xs_s, ca, cb, v);
      if (p.norm) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; i++) ss += v[i] * v[i];
        const float r = inv_sqrt(row_sum(live ? ss : 0.f, p.lpr) * p.inv_d + p.eps);
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] *= r * w[i];
      }
      rotate<SPLIT>(v, cs, sn);
      if (live && h < h_end) store_row<T, SPLIT>(q.y, b * q.ys_b + hc * q.ys_h + s * q.ys_s, ca, cb, v);
    }
  }
}

// Backward: a workgroup's wavefronts go over the tokens (token group, token group + groups, ...), four at a time, and
// keep the sums of d x^ of their lanes' columns.  8500 tokens of 24 + 24 heads of 64, fp16, split halves: 37 us, 4.2 TB/s;
// 32760 of 40 + 40 of 128 in fp32, a call, 792 us, 5.1 TB/s (of the fp32 forms split halves spill 4 registers).
template <typename T, bool SPLIT>
__global__ __launch_bounds__(256, 4) void axes_rope_bwd_kernel(const AxesRopeParams p) {
  __shared__ float part[4][2][512];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int c = lane & (p.lpr - 1), slot = lane / p.lpr, slots = 64 / p.lpr;
  const bool live = c * 8 < p.D;
  const int cc = live ? c : 0;
  const bool apart = SPLIT && 4 * cc < p.P;
  const int ca = apart ? 4 * cc : 8 * cc, cb = apart ? p.P + 4 * cc : 8 * cc + 4;
  const int g0 = blockIdx.y * p.heads_per_wave, g1 = g0 + p.heads_per_wave, first = p.t[0].H;
  const int begin[2] = {min(g0, first), max(0, g0 - first)}, end[2] = {min(first, g1), p.tensors == 2 ? min(p.t[1].H, g1 - first) : 0};   // heads of q and k
  float sum[2][8] = {};
  for (int64_t tok = (int64_t)blockIdx.x * 4 + wave; tok < (int64_t)p.B * p.S; tok += (int64_t)p.token_groups * 4) {   // uniform
    const int b = (int)((unsigned)tok / (unsigned)p.S), s = (int)((unsigned)tok - (unsigned)b * (unsigned)p.S);
    RowPart<T, SPLIT> next_d, next_x;   // the heads after these, k's first too, are on their way while these are worked on
    auto request = [&](const RopeTensor& q, int h0, int h_end) __attribute__((always_inline)) {
      const int h = min(h0 + slot, h_end - 1);
      next_d.load(q.dy, b * q.ds_b + h * q.ds_h + s * q.ds_s, ca, cb);
      if (p.norm) next_x.load(q.x, b * q.xs_b + h * q.xs_h + s * q.xs_s, ca, cb);
    };
    if (begin[0] < end[0]) request(p.t[0], begin[0], end[0]);
    else request(p.t[1], begin[1], end[1]);
    float cs[4], sn[4];
    turn<sizeof(T) == 4>(p, b, s, cc, -1.f, cs, sn);
#pragma unroll
    for (int t = 0; t < 2; t++) {
      if (begin[t] >= end[t]) continue;
      const RopeTensor& q = p.t[t];
      const int h_begin = begin[t], h_end = end[t];
      float w[8];
#pragma unroll
      for (int i = 0; i < 8; i++) w[i] = 1.f;
      if (q.weight != nullptr) load_gain<T, SPLIT>(q.weight, p.weight_wide, ca, cb, w);
      for (int h0 = h_begin; h0 < h_end; h0 += slots) {
        const int h = h0 + slot;
        const bool there = live && h < h_end;
        const int hc = h < h_end ? h : h_end - 1;
        float d[8], x[8];
        next_d.get(d);
        if (p.norm) next_x.get(x);
        if (h0 + slots < h_end) request(q, h0 + slots, h_end);
        else if (t == 0 && begin[1] < end[1]) request(p.t[1], begin[1], end[1]);
        rotate<SPLIT>(d, cs, sn);
        if (p.norm) {
          float ss = 0.f, dot = 0.f;
#pragma unroll
          for (int i = 0; i < 8; i++) ss += x[i] * x[i];
          const float r = inv_sqrt(row_sum(live ? ss : 0.f, p.lpr) * p.inv_d + p.eps);
#pragma unroll
          for (int i = 0; i < 8; i++) {
            x[i] *= r;
            sum[t][i] += there ? d[i] * x[i] : 0.f;
            d[i] *= w[i];
            dot += d[i] * x[i];
          }
          dot = row_sum(live ? dot : 0.f, p.lpr) * p.inv_d;
#pragma unroll
          for (int i = 0; i < 8; i++) d[i] = r * (d[i] - x[i] * dot);
        }
        if (there) store_row<T, SPLIT>(q.y, b * q.ys_b + hc * q.ys_h + s * q.ys_s, ca, cb, d);
      }
    }
  }
  if (!p.sums) return;  // uniform
#pragma unroll
  for (int t = 0; t < 2; t++)
#pragma unroll
    for (int i = 0; i < 8; i++) {
      for (int m = p.lpr; m < 64; m <<= 1) sum[t][i] += __shfl_xor(sum[t][i], m);
      if (slot == 0 && live) part[wave][t][(i < 4 ? ca : cb - 4) + i] = sum[t][i];
    }
  __syncthreads();
  float* out = p.partial + ((int64_t)blockIdx.y * p.token_groups + blockIdx.x) * 2 * p.D;
  for (int i = threadIdx.x; i < 2 * p.D; i += 256) {
    const int t = i >= p.D, col = i - t * p.D;
    out[i] = part[0][t][col] + part[1][t][col] + part[2][t][col] + part[3][t][col];
  }
}

// The workgroups' sums in a fixed order, 256 runs of every 256th and then the runs; 4 columns per workgroup.
template <typename T>
__global__ __launch_bounds__(1024) void axes_rope_bwd_finish_kernel(const AxesRopeParams p) {
  __shared__ float part[256][5];
  const int t = blockIdx.y;
  const RopeTensor& q = p.t[t];
  if (q.dweight == nullptr) return;
  const int run = threadIdx.x >> 2;
  const int n = p.head_groups * p.token_groups;
  float s = 0.f;
#pragma unroll 4
  for (int i = run; i < n; i += 256) s += p.partial[((int64_t)i * 2 + t) * p.D + blockIdx.x * 4 + (threadIdx.x & 3)];
  part[run][threadIdx.x & 3] = s;
  __syncthreads();
  if (threadIdx.x >= 256) return;
  const int lane = threadIdx.x & 63, of = threadIdx.x >> 6;   // a wavefront adds the runs of a column
  s = wave_sum((part[lane][of] + part[lane + 64][of]) + (part[lane + 128][of] + part[lane + 192][of]));
  if (lane != 0) return;
  const int col = blockIdx.x * 4 + (threadIdx.x >> 6);
  if (p.weight_wide) ((float*)q.dweight)[col] = s;
  else ((T*)q.dweight)[col] = (T)s;
}

template <typename T>
static hipError_t run(const AxesRopeParams& p, bool backward, hipStream_t stream) {
  const dim3 block(256);
  if (!backward) {
    const dim3 grid((unsigned)(((int64_t)p.B * p.S + 3) / 4), (unsigned)p.head_groups);
    if (p.split_half) hipLaunchKernelGGL((axes_rope_kernel<T, true>), grid, block, 0, stream, p);
    else hipLaunchKernelGGL((axes_rope_kernel<T, false>), grid, block, 0, stream, p);
    return hipGetLastError();
  }
  const dim3 grid((unsigned)p.token_groups, (unsigned)p.head_groups);
  if (p.split_half) hipLaunchKernelGGL((axes_rope_bwd_kernel<T, true>), grid, block, 0, stream, p);
  else hipLaunchKernelGGL((axes_rope_bwd_kernel<T, false>), grid, block, 0, stream, p);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || !p.sums) return e;
  hipLaunchKernelGGL((axes_rope_bwd_finish_kernel<T>), dim3((unsigned)(p.D / 4), (unsigned)p.tensors), dim3(1024), 0, stream, p);
  return hipGetLastError();
}

}  // namespace axrope

// A wavefront takes all heads of its token where that leaves the chip some 4096 wavefronts, fewer heads otherwise
// (one instruction's worth at least): the sines are computed again by each of them (512 tokens of 24 heads of 128: 5.9 us, 7.5 with 1024
// wavefronts, 6.7 with 16384; 4096 tokens of 16 heads of 72: 13.2, with 16384 16.2).  Backward: at most the 1024 workgroups that
// the chip holds at once, each going over its tokens, so that there are few sums to add up (8500 tokens of 24 heads of 64: 36.6 us,
// 48.6 with 512, 43.0 with 2048; 17776 of 48: 138, 208, 145).
void axes_rope_plan(AxesRopeParams& p, bool backward) {
  int lpr = 1;
  while (lpr * 8 < p.D) lpr <<= 1;
  p.lpr = lpr;
  const int64_t tokens = (int64_t)p.B * p.S;
  const int slots = 64 / lpr;
  int total = 0;
  for (int t = 0; t < p.tensors; t++) total += p.t[t].H;
  int groups = (int)((4096 + tokens - 1) / tokens);
  const int most = (total + slots - 1) / slots;
  if (groups > most) groups = most;
  p.heads_per_wave = ((total + groups - 1) / groups + slots - 1) / slots * slots;
  p.head_groups = (total + p.heads_per_wave - 1) / p.heads_per_wave;
  const int64_t wgs = (tokens + 3) / 4;
  p.token_groups = (int)(backward && wgs * p.head_groups > 1024 ? (1024 + p.head_groups - 1) / p.head_groups : wgs);
}

hipError_t launch_axes_rope(const AxesRopeParams& p, int dtype, bool backward, hipStream_t stream) {
  if (dtype == 0) return axrope::run<__bf16>(p, backward, stream);
  if (dtype == 1) return axrope::run<_Float16>(p, backward, stream);
  if (dtype == 2) return axrope::run<float>(p, backward, stream);
  return hipErrorInvalidValue;
}

}  // namespace xdit
