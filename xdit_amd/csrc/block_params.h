// Parameters and host-side launch functions of the operators around the attention call.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace xdit {

struct RowStrides { int64_t b, s; };

// dtype codes are the C ABI's (0 bf16, 1 fp16, 2 fp32); norms 0 none, 1 RMS, 2 layer.
struct GatedNormParams {
  const void* x;
  const void* y;
  void* h;
  void* n;
  float* n_scale;
  float* stats;
  const void* gate;
  const void* scale;
  const void* shift;
  const void* weight;
  const void* bias;
  const void* y_weight;
  RowStrides xs, ys, hs, ns, gs, ss, fs;  // gs: gate, ss: scale, fs: shift
  int B, S, C;
  int64_t rows;  // B * S
  int norm, y_norm, fp8;
  int mod_wide, weight_wide;  // those parameters are fp32 beside 16-bit tensors
  float eps, y_eps, alpha, inv_c;
  int rows_per_part;  // filled by the launcher
};

struct GatedNormBwdParams {
  const void* dh;
  const void* dn;
  const void* h;
  const void* y;
  const float* stats;
  const void* gate;
  const void* scale;
  const void* weight;
  const void* bias;
  const void* y_weight;
  void* dx;
  void* dy;
  void* dgate;
  void* dscale;
  void* dshift;
  void* dweight;
  void* dbias;
  void* dy_weight;
  RowStrides dhs, dns, hs, ys, gs, ss, dxs, dys;
  int B, S, C;
  int norm, y_norm;
  int mod_wide, weight_wide;
  int gate_per_token, mod_per_token;
  float alpha, inv_c;
  float* partial;     // [B][parts][3][C]: sums over the rows of a part (dn u, dn, t z), see the kernel
  int parts;          // parts the rows of a batch entry are cut into
  int rows_per_part;
  int teams;          // rows a workgroup works on at a time
  int sums;           // column sums are asked for
};

constexpr int kNormMaxC = 8192;

hipError_t launch_gated_norm(const GatedNormParams& p, int dtype, hipStream_t stream);
hipError_t launch_gated_norm_bwd(const GatedNormBwdParams& p, int dtype, hipStream_t stream);
void gated_norm_bwd_plan(GatedNormBwdParams& p);  // fills parts, rows_per_part and sums

// Rotation of q and k by positions on several axes.
struct RopeTensor {
  const void* x;
  const void* dy;
  void* y;
  const void* weight;
  void* dweight;
  int64_t xs_b, xs_h, xs_s;
  int64_t ds_b, ds_h, ds_s;
  int64_t ys_b, ys_h, ys_s;
  int H;
};

struct AxesRopeParams {
  RopeTensor t[2];
  int tensors;
  int B, S, D;
  int P;              // rotated pairs
  int axis_end[4];    // first pair behind the axis' range (P for the axes that are not there)
  int axes;
  int split_half, norm;
  int pos_bits, freq_wide, weight_wide;
  const void* positions;
  int64_t ps_b, ps_s;
  const void* inv_freq;
  float eps, inv_d;
  int lpr;             // lanes per row: smallest power of two >= D / 8
  int heads_per_wave;  // of the heads of q and k, laid end to end
  int head_groups;
  int token_groups;    // workgroups the tokens are dealt to (backward; forward: four tokens each)
  float* partial;      // backward: [head group][token group][2][D]
  int sums;
};

hipError_t launch_axes_rope(const AxesRopeParams& p, int dtype, bool backward, hipStream_t stream);
void axes_rope_plan(AxesRopeParams& p, bool backward);  // fills lpr, heads_per_wave, head_groups, token_groups

// Block-wise fp8 quantiser and the block-scaled product.
struct BlockQuantParams {
  const void* x;
  unsigned char* y;
  float* scale;
  RowStrides xs, ys;
  int64_t rows;  // B * S
  int S, K, kblocks;
};

hipError_t launch_fp8_block_quant(const BlockQuantParams& p, int dtype, int block_rows, hipStream_t stream);

struct BlockMatmulParams {
  const unsigned char* x;
  const float* xsc;
  const unsigned char* w;
  const float* wsc;
  const void* bias;
  void* out;
  int64_t xs, ws, os;            // row strides of x, w and out
  int64_t xsc_m, xsc_k, wsc_n, wsc_k;
  int M, N, K, kblocks;
  int bias_wide;
  int exact;
  int cu_count;
  float* partial;                // split K: [split][M][N] sums
  int splits;                    // parts K is cut into
  int blocks_per_split;
};

size_t fp8_block_matmul_workspace(const BlockMatmulParams& p);
hipError_t launch_fp8_block_matmul(const BlockMatmulParams& p, int out_dtype, size_t workspace_bytes, hipStream_t stream);

}  // namespace xdit
