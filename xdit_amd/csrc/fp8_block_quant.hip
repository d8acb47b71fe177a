// fp8 (e4m3) quantiser with an fp32 scale per 1 x 128 or 128 x 128 block, for gfx950.
//
//     scale = absmax / 448 ;  y = e4m3(x / scale)
// HBM-bound: one read of x, one byte per element and a scale per block written.  A block of a row is 16 lanes of 8
// elements, one DPP row, so its abs-max needs no LDS; a 128 x 128 block stays in the registers of its workgroup
// between the abs-max and the cast (13824 x 5120 bf16: 37 us, 5.7 TB/s).
#include "block_params.h"
#include "row_ops.h"

namespace xdit {

namespace bquant {

// Few blocks: 16 lanes each, laid end to end row by row (4250 x 1480 bf16: 6.9 us, 2.8 TB/s; the kernel below 7.5).
template <typename T>
__global__ __launch_bounds__(256) void quant_rows_kernel(const BlockQuantParams p) {
  const int64_t unit = (int64_t)blockIdx.x * 16 + (threadIdx.x >> 4);
  const int64_t row = unit / p.kblocks;
  const int kb = (int)(unit - row * p.kblocks);
  const int col = kb * 128 + (threadIdx.x & 15) * 8;
  const bool live = row < p.rows && col < p.K;
  const int64_t r = row < p.rows ? row : p.rows - 1;
  const int64_t b = r / p.S, s = r - b * p.S;
  float v[8] = {};
  if (live) get8(load_raw8<T>(p.x, b * p.xs.b + s * p.xs.s + col), v);
  const Divider div(block_scale(row16_max(absmax8(v))));
  if (!live) return;
  *(i32x2*)(p.y + b * p.ys.b + s * p.ys.s + col) = cast8(v, div);
  if ((threadIdx.x & 15) == 0) p.scale[kb * p.rows + row] = div.scale;
}

// Many blocks: a workgroup takes 16 rows and two blocks of each, both loads under way at once, and stores the 16 scales of a column of blocks
// side by side (32760 x 5120 bf16: 95 us, 5.3 TB/s, the kernel above 105; 4608 x 5120: 15.2 and 16.2).
constexpr int kTogether = 2;
template <typename T>
__global__ __launch_bounds__(256) void quant_many_kernel(const BlockQuantParams p) {
  const unsigned across = (p.kblocks + kTogether - 1) / kTogether, group = blockIdx.x / across, part = blockIdx.x - group * across;
  const int64_t row = (int64_t)group * 16 + (threadIdx.x >> 4);
  const bool there = row < p.rows;
  const unsigned r = (unsigned)min(row, p.rows - 1), b = r / (unsigned)p.S, s = r - b * (unsigned)p.S;
  const int col = part * (128 * kTogether) + (threadIdx.x & 15) * 8;
  const int64_t from = b * p.xs.b + s * p.xs.s, to = b * p.ys.b + s * p.ys.s;
  Raw8<T> raw[kTogether];
#pragma unroll
  for (int k = 0; k < kTogether; k++) raw[k] = load_raw8<T>(p.x, from + min(col + 128 * k, p.K - 8));
#pragma unroll
  for (int k = 0; k < kTogether; k++) {
    const int kb = part * kTogether + k;
    if (kb >= p.kblocks) return;   // uniform
    const bool live = there && col + 128 * k < p.K;
    float v[8] = {};
    if (live) get8(raw[k], v);
    const Divider div(block_scale(row16_max(absmax8(v))));
    if (live) *(i32x2*)(p.y + to + col + 128 * k) = cast8(v, div);
    if (there && (threadIdx.x & 15) == 0) p.scale[kb * p.rows + row] = div.scale;
  }
}

// A workgroup per 128 x 128 block; a thread holds 8 columns of rows r, r + 16, ..., r + 112.
template <typename T>
__global__ __launch_bounds__(256) void quant_tiles_kernel(const BlockQuantParams p) {
  __shared__ unsigned part[4];
  const int col = blockIdx.x * 128 + (threadIdx.x & 15) * 8;
  const int64_t row0 = (int64_t)blockIdx.y * 128 + (threadIdx.x >> 4);
  float v[8][8];
  unsigned m = 0;
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const bool live = col < p.K && row0 + 16 * k < p.rows;
#pragma unroll
    for (int i = 0; i < 8; i++) v[k][i] = 0.f;
    if (live) get8(load_raw8<T>(p.x, (row0 + 16 * k) * p.xs.s + col), v[k]);
    m = max(m, absmax8(v[k]));
  }
  m = row16_max(m);
  m = max(m, (unsigned)__shfl_xor((int)m, 16));
  m = max(m, (unsigned)__shfl_xor((int)m, 32));
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = m;
  __syncthreads();
  const Divider div(block_scale(max(max(part[0], part[1]), max(part[2], part[3]))));
#pragma unroll
  for (int k = 0; k < 8; k++)
    if (col < p.K && row0 + 16 * k < p.rows) *(i32x2*)(p.y + (row0 + 16 * k) * p.ys.s + col) = cast8(v[k], div);
  if (threadIdx.x == 0) p.scale[(int64_t)blockIdx.y * p.kblocks + blockIdx.x] = div.scale;
}

template <typename T>
static hipError_t run(const BlockQuantParams& p, int block_rows, hipStream_t stream) {
  if (block_rows == 1) {
    // equal at about 160000 blocks, where the chip is filled five times over with 16 lanes each
    const bool many = p.rows * p.kblocks >= 160000;
    const int64_t groups = many ? (p.rows + 15) / 16 * ((p.kblocks + kTogether - 1) / kTogether) : (p.rows * p.kblocks + 15) / 16;
    if (groups > 0x7fffffffLL) return hipErrorInvalidValue;
    if (many) hipLaunchKernelGGL((quant_many_kernel<T>), dim3((unsigned)groups), dim3(256), 0, stream, p);
    else hipLaunchKernelGGL((quant_rows_kernel<T>), dim3((unsigned)groups), dim3(256), 0, stream, p);
  } else {
    const int64_t down = (p.rows + 127) / 128;
    if (down > 65535) return hipErrorInvalidValue;
    hipLaunchKernelGGL((quant_tiles_kernel<T>), dim3((unsigned)p.kblocks, (unsigned)down), dim3(256), 0, stream, p);
  }
  return hipGetLastError();
}

}  // namespace bquant

hipError_t launch_fp8_block_quant(const BlockQuantParams& p, int dtype, int block_rows, hipStream_t stream) {
  if (dtype == 0) return bquant::run<__bf16>(p, block_rows, stream);
  if (dtype == 1) return bquant::run<_Float16>(p, block_rows, stream);
  if (dtype == 2) return bquant::run<float>(p, block_rows, stream);
  return hipErrorInvalidValue;
}

}  // namespace xdit
