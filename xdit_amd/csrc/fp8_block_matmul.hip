// Product of fp8 (e4m3) matrices with a scale per block of 128, out = x w^T + bias, for gfx950.
//
//     out[m, n] = sum_kb xs[m, kb] ws[n / 128, kb] (sum over the block's k of x[m, k] w[n, k])
// One v_mfma_f32_16x16x128_f8f6f4 contracts exactly one block: the instruction starts from zero and its 16 x 16 sums go
// into the fp32 accumulators with one multiply-add each by xs ws.  The weights are the A operand and the activations the
// B operand, so a lane holds four consecutive n of one m: one scale per lane and block, and neighbouring outputs.
// A and B have the same lane -> k map, so which 32 of a row's k a lane holds is free as long as both agree.
//
// The fp8 matrix instructions of this chip add the products of eight consecutive k at a time and cut each at 2^-13 of the largest
// one's binade (a product of 2^16 beside seven of 2^2 gives 2^16; beside products of other eights it loses nothing; the older
// 16x16x32 form does the same, at a third of the rate): on random bytes a block's sum is off by 305 units of 2^-24 of its terms'
// sizes on average, 2900 at most.  That leaves a result 1.4e-5 to 3.3e-5 of its size off: nothing beside bf16's
// rounding (1.66e-3 with and without), 0.2 to 1.2 % more error beside fp16's (2.07e-4 to 2.08e-4 .. 2.10e-4).  For fp32 results, or where the
// caller asks for it, both operands are widened to fp16, which is exact, and the fp16 instructions sum within 5 units.
#include <atomic>
#include <cmath>
#include <type_traits>

#include "attn_split.h"
#include "attn_tiles.h"
#include "block_params.h"
#include "row_ops.h"

namespace xdit {

namespace bmm {

// Eight bytes as fp16, exactly.
__device__ __forceinline__ f16x8 widen8(int lo, int hi) {
  const f16x2 a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true);
  const f16x2 c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true);
  return (f16x8){a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
// `half`: a bias that is not fp32 is fp16, otherwise bf16.
__device__ __forceinline__ float bias_at(const BlockMatmulParams& p, int half, int n) {
  if (p.bias_wide) return ((const float*)p.bias)[n];
  return half == 0 ? (float)((const __bf16*)p.bias)[n] : (float)((const _Float16*)p.bias)[n];
}
template <typename T> constexpr int kIsHalf = __is_same(T, _Float16) ? 1 : 0;

// ---- the tiled kernel --------------------------------------------------------------------------------
// A workgroup of WN x WM wavefronts computes BN x BM outputs (n x m), a wavefront 16 TN x 16 TM of them.  The operands'
// 128-byte row pieces of a block of K stream through LDS in STAGES buffers, filled by direct global -> LDS loads of 16 bytes
// a lane; the scales of the block (BM of x, one or two of w) travel with them.  A buffer is a plain array of 128-byte
// rows whose eight 16-byte chunks are stored in the order chunk ^ (row / 2 % 8): sixteen consecutive rows' equal chunks, what a
// fragment read fetches at a time, then lie in sixteen different places of the 256 bytes that LDS serves per clock.
template <int BN_, int BM_, int WN_, int WM_, int STAGES_>
struct Shape {
  static constexpr int BN = BN_, BM = BM_, WN = WN_, WM = WM_, STAGES = STAGES_;
  static constexpr int NW = WN * WM;                  // wavefronts
  static constexpr int TN = BN / WN / 16, TM = BM / WM / 16;
  static constexpr int W_LOADS = BN / 8 / NW;         // 1 KiB pieces of 8 rows per stage and wavefront, of w
  static constexpr int X_LOADS = BM / 8 > NW ? BM / 8 / NW : 1;   // ... and of x (few rows: some pieces are fetched twice)
  static constexpr int LOADS = W_LOADS + X_LOADS + 1; // ... and a load of scales
  static constexpr int W_BYTES = BN * 128, X_BYTES = BM * 128;
  static constexpr int SC_X = W_BYTES + X_BYTES;      // scales of x
  static constexpr int SC_W = SC_X + (BM > 64 ? BM : 64) * 4;   // scales of w, 64 of them (lane % (BN / 128))
  static constexpr int STAGE_BYTES = SC_W + 256;
  static constexpr int LDS = STAGES * STAGE_BYTES;
  static constexpr int SC_PIECES = BM > 64 ? BM / 64 : 1;
  static_assert(BN % (16 * WN) == 0 && BM % (16 * WM) == 0 && (BN / 8) % NW == 0 && (BM / 8 % NW == 0 || NW % (BM / 8) == 0), "pieces");
  static_assert(NW % 2 == 0 && (BM / 8) % 2 == 0, "a wavefront's pieces have one parity");
  static_assert(SC_PIECES < NW, "the wavefronts behind the first fetch the scales of w");
  static_assert(BN / WN <= 128 && 128 % (BN / WN) == 0, "a wavefront's n lie in one block of 128");
};

// What x holds beyond K in the last block (w re-reads its row's last chunk there).
static __device__ const __align__(16) unsigned char kZeros[16] = {};

// 16 bytes a lane from 64-bit addresses straight into LDS at lds + 16 lane.
__device__ __forceinline__ void load_lds_16_at(const void* p, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dwordx4 %1, off"
      :
      : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p)
      : "memory", "m0");
}
// The same with 4 bytes a lane, to lds + 4 lane.
__device__ __forceinline__ void load_lds_4(const void* p, unsigned lds) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "global_load_lds_dword %1, off"
      :
      : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(p)
      : "memory", "m0");
}
// At most N of this wavefront's loads are under way, and all of its LDS reads are done.
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(N) : "memory"); }

// The 128 k of 16 rows as a matrix instruction takes them: bytes, or widened to fp16.
template <bool EXACT> struct Operand;
template <> struct Operand<false> {
  i32x8 v;
  __device__ __forceinline__ void set(const i32x8& x) { v = x; }
};
template <> struct Operand<true> {
  f16x8 v[4];
  __device__ __forceinline__ void set(const i32x8& x) {
#pragma unroll
    for (int t = 0; t < 4; t++) v[t] = widen8(x[2 * t], x[2 * t + 1]);
  }
};
// 16 x 16 outputs summed over a block.
__device__ __forceinline__ f32x4 block_sum(const Operand<false>& a, const Operand<false>& b) {
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a.v, b.v, (f32x4){0.f, 0.f, 0.f, 0.f}, 0, 0, 0, 0, 0, 0);
}
__device__ __forceinline__ f32x4 block_sum(const Operand<true>& a, const Operand<true>& b) {
  f32x4 d = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int t = 0; t < 4; t++) d = __builtin_amdgcn_mfma_f32_16x16x32_f16(a.v[t], b.v[t], d, 0, 0, 0);
  return d;
}

// Tile of the problem that workgroup `w` computes.  Workgroups go round-robin to the 8 XCDs; each XCD takes a contiguous
// range of an order in which 32 consecutive tiles, what it runs at once, are a patch of 8 x 4 tiles (m x n), so that its L2
// serves every row panel to 4 and every column panel to 8 of them.
__device__ __forceinline__ bool tile_of(int w, int tiles_n, int tiles_m, int& tn, int& tm) {
  const int total = tiles_n * tiles_m;
  const int i = xcd_tile_index(w, (total + 7) / 8);
  if (i >= total) return false;
  const int band = i / (8 * tiles_n);
  const int height = min(8, tiles_m - 8 * band);
  const int r = i - band * 8 * tiles_n;
  tn = r / height;
  tm = 8 * band + r - tn * height;
  return true;
}

// A wavefront's 16 TN x 16 TM sums, plus bias, as rows m of `out`, sixteen rows at a time through LDS that is free
// for every wavefront.
template <typename T, typename S>
__device__ __forceinline__ void put_rows(const f32x4 (&acc)[S::TN][S::TM], unsigned char* smem, T* out, int64_t os, const void* bias, int half,
                                         const BlockMatmulParams& p, int n0, int m0, int wave, int lane) {
  typedef __attribute__((ext_vector_type(4))) T vec4;
  constexpr int WIDE = 16 * S::TN, PITCH = WIDE * sizeof(T) + 16;   // rows 16 bytes apart from a multiple of 256
  static_assert(S::NW * 16 * PITCH <= S::LDS && WIDE * 4 <= 16 * PITCH, "staging rows");
  unsigned char* mine = smem + wave * 16 * PITCH;
  const int l16 = lane & 15, quad = lane >> 4;
  const int width = min(WIDE, p.N - n0);
  float add[S::TN][4] = {};
  if (bias != nullptr) {   // uniform
    for (int n = lane; n < WIDE; n += 64) ((float*)mine)[n] = n < width ? bias_at(p, half, n0 + n) : 0.f;
    asm volatile("" ::: "memory");   // LDS operations of a wavefront stay in order; other lanes' entries are read below
    __builtin_amdgcn_wave_barrier();
#pragma unroll
    for (int i = 0; i < S::TN; i++) {
      const f32x4 v = *(const f32x4*)(mine + (16 * i + 4 * quad) * 4);
#pragma unroll
      for (int e = 0; e < 4; e++) add[i][e] = v[e];
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
  const bool lines = ((uintptr_t)out | (uintptr_t)(os * sizeof(T))) % 16 == 0 && width == WIDE;   // whole rows that start on 16 bytes
#pragma unroll
  for (int j = 0; j < S::TM; j++) {
#pragma unroll
    for (int i = 0; i < S::TN; i++) {
      vec4 v;
#pragma unroll
      for (int e = 0; e < 4; e++) v[e] = (T)(acc[i][j][e] + add[i][e]);
      *(vec4*)(mine + l16 * PITCH + (16 * i + 4 * quad) * sizeof(T)) = v;
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    const int rows = min(16, p.M - m0 - 16 * j);
    T* dst = out + (int64_t)(m0 + 16 * j) * os + n0;
    if (lines) {
      constexpr int E = 16 / sizeof(T), PER_ROW = WIDE / E;   // 16-byte pieces
#pragma unroll
      for (int k = 0; k < (16 * PER_ROW + 63) / 64; k++) {
        const int r = (64 * k + lane) / PER_ROW, n = (64 * k + lane) % PER_ROW * E;
        if (r < rows) *(i32x4*)(dst + r * os + n) = *(const i32x4*)(mine + r * PITCH + n * sizeof(T));
      }
    } else {
#pragma unroll 16
      for (int i = lane; i < 16 * WIDE; i += 64) {
        const int r = i / WIDE, n = i % WIDE;
        if (r < rows && n < width) dst[r * os + n] = ((const T*)(mine + r * PITCH))[n];
      }
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
  }
}

// RAGGED: K is not a multiple of 128.  Bound by the matrix pipe and the loop around it where there are many rows: 32760 x 13824 x 5120 to bf16
// takes 2046 to 2117 us, 2.19 to 2.27 PFLOP/s; a loop of nothing but this instruction from zero and its scaled adds reaches 2.39 on the chip.
// The large tile is what feeds it: 256 x 256 outputs of a block take a compute unit 1.41 us, four tiles of 128 x 128 take it 2.1.
// One row is the weights' reading: 1 x 30720 x 5120 takes 27.5 us, 5.7 TB/s (part of it out of the memory-side cache).
template <typename T, bool EXACT, bool RAGGED, typename S>
__global__ __launch_bounds__(64 * S::NW) void matmul_tiled_kernel(const BlockMatmulParams p) {
  extern __shared__ __align__(16) unsigned char smem[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int l16 = lane & 15, quad = lane >> 4;
  const int kb0 = blockIdx.y * p.blocks_per_split, kb1 = min(p.kblocks, kb0 + p.blocks_per_split);

  // ---- loads of a stage: piece g = wave + NW i holds rows 8 g .. 8 g + 7 of the tile of w (x)
  const unsigned lds0 = (unsigned)(uintptr_t)(XDIT_LDS unsigned char*)smem;
  const int piece_row = lane >> 3;
  const unsigned chunk = (unsigned)((lane & 7) ^ ((4 * wave + (lane >> 4)) & 7)) * 16;   // NW is even: a wavefront's pieces have one parity
  const bool xscale = wave < S::SC_PIECES;
  const int64_t sc_step = xscale ? p.xsc_k : p.wsc_k;
  const unsigned sc_dst = xscale ? S::SC_X + 256 * wave : S::SC_W;
  int tile_n, tile_m;
  if (!tile_of(blockIdx.x, (p.N + S::BN - 1) / S::BN, (p.M + S::BM - 1) / S::BM, tile_n, tile_m)) return;
  const int n0 = tile_n * S::BN, m0 = tile_m * S::BM;
  const int wlast = min(S::BN, p.N - n0) - 1, xlast = min(S::BM, p.M - m0) - 1;   // rows beyond the matrix re-read its last one
  int coming = kb0;   // the block that is requested next
  const unsigned char* wbase = p.w + (int64_t)n0 * p.ws + (int64_t)kb0 * 128;
  const unsigned char* xbase = p.x + (int64_t)m0 * p.xs + (int64_t)kb0 * 128;
  const float* sc = xscale ? p.xsc + (int64_t)(m0 + min(64 * wave + lane, xlast)) * p.xsc_m + (int64_t)kb0 * p.xsc_k
                           : p.wsc + (int64_t)min((n0 >> 7) + (lane % (S::BN > 128 ? S::BN / 128 : 1)), (p.N - 1) >> 7) * p.wsc_n + (int64_t)kb0 * p.wsc_k;
  auto request = [&](int stage) {
    const unsigned dst = lds0 + stage * S::STAGE_BYTES;
    const int k_left = p.K - coming * 128;
    const unsigned c = RAGGED ? min((int)chunk, k_left - 16) : chunk;   // w re-reads its row's last chunk beyond K
#pragma unroll
    for (int i = 0; i < S::W_LOADS; i++) {
      const int g = wave + S::NW * i;
      load_lds_16(wbase, __umul24((unsigned)min(8 * g + piece_row, wlast), (unsigned)p.ws) + c, dst + g * 1024);
    }
#pragma unroll
    for (int i = 0; i < S::X_LOADS; i++) {
      const int g = S::BM / 8 >= S::NW ? wave + S::NW * i : wave % (S::BM / 8);
      const unsigned off = __umul24((unsigned)min(8 * g + piece_row, xlast), (unsigned)p.xs) + chunk;
      if constexpr (RAGGED) load_lds_16_at((int)chunk < k_left ? xbase + off : kZeros, dst + S::W_BYTES + g * 1024);
      else load_lds_16(xbase, off, dst + S::W_BYTES + g * 1024);
    }
    load_lds_4(sc, dst + sc_dst);
    coming++;
    wbase += 128;
    xbase += 128;
    sc += sc_step;
  };

  // ---- fragments: lane (l16, quad) holds chunks quad and quad + 4 of its row.  LDS serves a 16-byte read in groups of lanes such as
  // {0-3, 12-15, 20-23, 24-27}; with chunks 2 quad and 2 quad + 1 those met in pairs (half of all LDS clocks), with these they do not.
  const int wn = wave % S::WN, wm = wave / S::WN;
  const int swz = (l16 >> 1) & 7;
  const int off0 = l16 * 128 + ((quad ^ swz) << 4), off1 = l16 * 128 + (((quad + 4) ^ swz) << 4);
  const int a_row = wn * S::TN * 16 * 128, b_row = S::W_BYTES + wm * S::TM * 16 * 128;
  auto fragment = [&](const unsigned char* rows) {
    const i32x4 lo = *(const i32x4*)(rows + off0), hi = *(const i32x4*)(rows + off1);
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
  };

  f32x4 acc[S::TN][S::TM] = {};
  // The sums of row i + 1 of the tile are under way while those of row i are scaled and added: a wavefront issues in order, and
  // a result is there some ten instructions after its matrix instruction.
  auto compute = [&](const unsigned char* buf, int into) {
    Operand<EXACT> b[S::TM], a;
    float s[S::TM];
    f32x4 d[2][S::TM];
    a.set(fragment(buf + a_row));
    const float ws = *(const float*)(buf + S::SC_W + 4 * (S::BN > 128 ? (wn * S::TN * 16) >> 7 : 0));
#pragma unroll
    for (int j = 0; j < S::TM; j++) b[j].set(fragment(buf + b_row + j * 2048));
#pragma unroll
    for (int j = 0; j < S::TM; j++) s[j] = *(const float*)(buf + S::SC_X + 4 * ((wm * S::TM + j) * 16 + l16)) * ws;
#pragma unroll
    for (int i = 0; i <= S::TN; i++) {
      i32x8 next;
      if (i + 1 < S::TN) next = fragment(buf + a_row + (i + 1) * 2048);
      if (i == 0 && into >= 0) request(into);   // uniform
#pragma unroll
      for (int j = 0; j < S::TM; j++) {
        if (i < S::TN) d[i & 1][j] = block_sum(a, b[j]);
        if (i > 0) {
#pragma unroll
          for (int e = 0; e < 4; e++) acc[i - 1][j][e] = __builtin_fmaf(d[(i - 1) & 1][j][e], s[j], acc[i - 1][j][e]);
        }
        __builtin_amdgcn_sched_barrier(0);
      }
      if (i + 1 < S::TN) a.set(next);
    }
  };
#pragma unroll
  for (int i = 0; i < S::STAGES - 1; i++)
    if (kb0 + i < kb1) request(i);
  int stage = 0;
  for (int kb = kb0; kb < kb1; kb++) {
    if (S::STAGES > 2 && kb + S::STAGES - 2 < kb1) wait_loads<S::LOADS * (S::STAGES - 2)>();
    else wait_loads<0>();
    __builtin_amdgcn_s_barrier();   // block kb is in its buffer for every wavefront, the buffer before it is no longer read
    asm volatile("" ::: "memory");
    compute(smem + stage * S::STAGE_BYTES, kb + S::STAGES - 1 < kb1 ? (stage == 0 ? S::STAGES - 1 : stage - 1) : -1);
    stage = stage + 1 == S::STAGES ? 0 : stage + 1;
  }
  // accumulator element e of lane (l16, quad): m = l16, n = 4 quad + e; the rows leave through LDS as whole lines (element by element
  // this end took a third of a 5120-deep product)
  wait_loads<0>();
  __builtin_amdgcn_s_barrier();   // no wavefront reads its buffers any more
  asm volatile("" ::: "memory");
  const int n_out = n0 + wn * S::TN * 16, m_out = m0 + wm * S::TM * 16;
  if (p.splits > 1) put_rows<float, S>(acc, smem, p.partial + (int64_t)blockIdx.y * p.M * p.N, p.N, nullptr, 0, p, n_out, m_out, wave, lane);
  else put_rows<T, S>(acc, smem, (T*)p.out, p.os, p.bias, kIsHalf<T>, p, n_out, m_out, wave, lane);
}

template <typename T, bool EXACT, bool RAGGED, typename S>
static hipError_t launch_kernel(const BlockMatmulParams& p, hipStream_t stream) {
  const int64_t tiles = (int64_t)((p.N + S::BN - 1) / S::BN) * ((p.M + S::BM - 1) / S::BM);
  if (tiles > 0x3fffffff) return hipErrorInvalidValue;
  static std::atomic<bool> lds_ready[kMaxDevices];
  const int slot = current_device_slot();
  if (S::LDS > 65536 && !lds_ready[slot].load(std::memory_order_relaxed)) {  // > 64 KiB of dynamic LDS must be enabled once per kernel and device
    const hipError_t e = hipFuncSetAttribute((const void*)matmul_tiled_kernel<T, EXACT, RAGGED, S>, hipFuncAttributeMaxDynamicSharedMemorySize, S::LDS);
    if (e != hipSuccess) return e;
    lds_ready[slot].store(true, std::memory_order_relaxed);
  }
  hipLaunchKernelGGL((matmul_tiled_kernel<T, EXACT, RAGGED, S>), dim3((unsigned)((tiles + 7) / 8 * 8), (unsigned)p.splits), dim3(64 * S::NW), S::LDS, stream, p);
  return hipGetLastError();
}

template <typename T, bool EXACT, typename S>
static hipError_t launch_tiled(const BlockMatmulParams& p, hipStream_t stream) {
  return p.K % 128 != 0 ? launch_kernel<T, EXACT, true, S>(p, stream) : launch_kernel<T, EXACT, false, S>(p, stream);
}

// The parts' sums in their order, plus bias.
template <typename T>
__global__ __launch_bounds__(256) void matmul_join_kernel(const BlockMatmulParams p) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, count = (int64_t)p.M * p.N;
  if (i >= count) return;
  const int64_t m = i / p.N;
  const int n = (int)(i - m * p.N);
  const float* in = p.partial + i;
  float v = 0.f;
#pragma unroll 4
  for (int k = 0; k < p.splits; k++) v += in[k * count];
  ((T*)p.out)[m * p.os + n] = (T)(v + (p.bias != nullptr ? bias_at(p, kIsHalf<T>, n) : 0.f));
}

// ---- how a product is run ---------------------------------------------------------------------------
// Seven shapes (with exact sums the first four and 128 x 128 in two buffers), each with K uncut or cut into some parts;
// the one with the shortest estimated time is taken:
//     start + sum over the rounds of workgroups [fix + blocks of K a workgroup * max(lat, workgroups on a compute unit * busy)],
//     at least the bytes of x, w and out at the memory's rate, and for a cut K the second kernel's launch and its traffic.
// lat is what a block takes a workgroup alone (its loads' way), busy what it costs a compute unit (its products), both in us.  The
// constants are fitted to 4009 times of every option at 190 problems (1 to 12000 rows, 64 to 30720 columns, K 320 to
// 13824; 16-bit results) and 1161 at 70 (exact sums); there the choice is 1.4 % (0.9 %) slower than the fastest option on
// average, 14 % (10 %) at worst.  Nothing was fitted above 12000 rows, where the estimate is short (32760 x 13824 x 5120: 1594 us) and only
// serves to rank.  Shapes of 128 x 16, 128 x 32 and 128 x 256 would give another 0.2 %.
struct Option { int bn, bm, per_cu; double lat, busy, fix; };
static const Option kFast[] = {{64, 16, 3, 0.181, 0.118, 1.162}, {64, 32, 3, 0.226, 0.222, 1.044}, {64, 64, 2, 0.122, 0.231, 1.054}, {128, 64, 2, 0.393, 0.472, 0.935},
                               {128, 128, 2, 0.763, 0.524, 0.328}, {128, 128, 1, 0.702, 0.400, 1.060}, {256, 256, 1, 0.559, 1.410, 2.624}};
static const Option kExact[] = {{64, 16, 3, 0.201, 0.160, 0.962}, {64, 32, 3, 0.277, 0.305, 1.192}, {64, 64, 2, 0.363, 0.341, 0.898}, {128, 64, 2, 0.653, 0.594, 0.924},
                                {128, 128, 2, 1.187, 0.938, 1.506}};
struct Part { int rows, shape, splits; double us; };

static double estimate(const BlockMatmulParams& p, const Option& o, int64_t M, int splits) {
  const int64_t cus = resident_cus(p.cu_count);
  const double rate = p.exact ? 7.3e6 : 8.4e6, join = p.exact ? 4.0 : 4.6, join_bytes = p.exact ? 0.67e-6 : 1.2e-6;   // bytes per us; us; us per sum
  const int blocks = (p.kblocks + splits - 1) / splits;
  const int64_t groups = ((p.N + o.bn - 1) / o.bn) * ((M + o.bm - 1) / o.bm) * splits, round = cus * o.per_cu, rest = groups % round;
  const double moved = ((double)p.N + M) * p.K, written = (double)M * p.N;
  double us = (double)(groups / round) * (o.fix + blocks * fmax(o.lat, o.per_cu * o.busy));
  if (rest > 0) us += o.fix + blocks * fmax(o.lat, (double)((rest + cus - 1) / cus) * o.busy);
  us = fmax(us, (moved + (splits == 1 ? 2.0 * written : 0.0)) / rate + o.fix);
  if (splits > 1) us += join + join_bytes * splits * written;
  return us;
}

static Part plan_rows(const BlockMatmulParams& p, int M) {
  const Option* options = p.exact ? kExact : kFast;
  const int64_t cus = resident_cus(p.cu_count);
  Part best = {M, 0, 1, 0.0};
  for (int i = 0; i < (p.exact ? 5 : 7); i++) {
    const Option& o = options[i];
    const int64_t tiles = (int64_t)((p.N + o.bn - 1) / o.bn) * ((M + o.bm - 1) / o.bm);
    static const int kCuts[] = {1, 2, 3, 4, 6, 8, 12, 16};
    for (int cut : kCuts) {
      if (cut > 1 && (cut > p.kblocks / 2 || tiles * cut > 6 * cus)) break;   // two blocks a part at least, and no cut where the chip is full
      const int blocks = (p.kblocks + cut - 1) / cut, splits = (p.kblocks + blocks - 1) / blocks;
      const double us = estimate(p, o, M, splits);
      if (best.us == 0.0 || us < best.us) best = {M, i, splits, us};
    }
  }
  return best;
}

// Many rows: where the largest tiles' last round leaves compute units idle, only the rows of its full rounds are run with them,
// and those behind as a product of their own (4250 x 5120 x 5120: 340 tiles of 256 x 256 are 1.33 rounds and took 130 us; twelve of
// the 17 rows of tiles as one round, and the rest as another product, take 114).
struct Plan { Part part[2]; int parts; };
static Plan plan_of(const BlockMatmulParams& p) {
  Plan r = {{plan_rows(p, p.M)}, 1};
  const int large = p.exact ? 4 : 6;
  const Option& o = (p.exact ? kExact : kFast)[large];
  const int64_t across = (p.N + o.bn - 1) / o.bn, round = (int64_t)resident_cus(p.cu_count) * o.per_cu;
  const int64_t rounds = across * ((p.M + o.bm - 1) / o.bm) / round;
  const int64_t rows = rounds * round / across * o.bm;
  if (rows > 0 && rows < p.M) {
    const Part first = {(int)rows, large, 1, estimate(p, o, rows, 1)}, rest = plan_rows(p, (int)(p.M - rows));
    if (first.us + rest.us + 1.0 < r.part[0].us) r = {{first, rest}, 2};
  }
  return r;
}

template <typename T, bool EXACT>
static hipError_t launch_shape(const BlockMatmulParams& p, int shape, hipStream_t stream) {
  switch (shape) {
    case 0: return launch_tiled<T, EXACT, Shape<64, 16, 4, 1, 4>>(p, stream);
    case 1: return launch_tiled<T, EXACT, Shape<64, 32, 4, 1, 4>>(p, stream);
    case 2: return launch_tiled<T, EXACT, Shape<64, 64, 2, 2, 4>>(p, stream);
    case 3: return launch_tiled<T, EXACT, Shape<128, 64, 4, 1, 3>>(p, stream);
    case 4: return launch_tiled<T, EXACT, Shape<128, 128, 2, 2, 2>>(p, stream);
  }
  if constexpr (!EXACT) {
    if (shape == 5) return launch_tiled<T, EXACT, Shape<128, 128, 2, 2, 4>>(p, stream);
    if (shape == 6) return launch_tiled<T, EXACT, Shape<256, 256, 2, 4, 2>>(p, stream);
  }
  return hipErrorInvalidValue;
}

static size_t part_bytes(const Part& part, int N) { return part.splits > 1 ? (size_t)part.splits * part.rows * N * 4 : 0; }

template <typename T>
static hipError_t run(BlockMatmulParams p, size_t workspace_bytes, hipStream_t stream) {
  const Plan plan = plan_of(p);
  for (int i = 0; i < plan.parts; i++) {
    const Part& part = plan.part[i];
    p.M = part.rows;
    p.splits = part_bytes(part, p.N) <= workspace_bytes ? part.splits : 1;
    p.blocks_per_split = (p.kblocks + p.splits - 1) / p.splits;
    hipError_t e = p.exact ? launch_shape<T, true>(p, part.shape, stream) : launch_shape<T, false>(p, part.shape, stream);
    if (e == hipSuccess && p.splits > 1) {
      hipLaunchKernelGGL((matmul_join_kernel<T>), dim3((unsigned)(((int64_t)p.M * p.N + 255) / 256)), dim3(256), 0, stream, p);
      e = hipGetLastError();
    }
    if (e != hipSuccess) return e;
    p.x += (int64_t)part.rows * p.xs;
    p.xsc += (int64_t)part.rows * p.xsc_m;
    p.out = (T*)p.out + (int64_t)part.rows * p.os;
  }
  return hipSuccess;
}

}  // namespace bmm

size_t fp8_block_matmul_workspace(const BlockMatmulParams& p) {
  const bmm::Plan plan = bmm::plan_of(p);
  size_t most = 0;
  for (int i = 0; i < plan.parts; i++) {
    const size_t bytes = bmm::part_bytes(plan.part[i], p.N);   // the parts run one after the other
    if (bytes > most) most = bytes;
  }
  return most;
}

hipError_t launch_fp8_block_matmul(const BlockMatmulParams& p, int out_dtype, size_t workspace_bytes, hipStream_t stream) {
  if (out_dtype == 0) return bmm::run<__bf16>(p, workspace_bytes, stream);
  if (out_dtype == 1) return bmm::run<_Float16>(p, workspace_bytes, stream);
  if (out_dtype == 2) return bmm::run<float>(p, workspace_bytes, stream);
  return hipErrorInvalidValue;
}

}  // namespace xdit
