// Backward pass of the non-causal attention forward for 16-bit tensors on gfx950.
//
//   P_ij = exp(scale q_i.k_j - lse_i)      delta_i = dout_i.out_i - dlse_i
//   dV_j = sum_i P_ij dout_i               dS_ij = P_ij (dout_i.v_j - delta_i)
//   dK_j = scale sum_i dS_ij q_i           dQ_i = scale sum_j dS_ij k_j
//
// P is recomputed from the forward's log-sum-exp, so nothing of size Sq x Sk is ever in memory.
//
// Work decomposition: bwd_stats_kernel writes lse / ln 2 and -delta of every row, then one launch has the units of two roles:
//   keys     a workgroup owns 128 keys, wavefront w keys [32w, 32w+32); it streams the queries: dK and dV (four products)
//   queries  a workgroup owns 128 queries; it streams the keys: dQ (three products)
// Seven products instead of the five of a single pass: that one adds every workgroup's share of dQ up in memory, by atomics (whose order
// changes the result) or through Sk / 128 fp32 copies of dQ (5 heads of 32760: 21.5 GB written and read again, 8.5 ms at a copy's rate,
// where the two products more take 2.1). The longer units, those of the keys, start first; the last units may be parts of tiles, which even
// out the end of the launch and let few tiles fill the chip (BwdRole; the parts are added up by bwd_fold_kernel). Workgroups have four
// wavefronts, two of them share a compute unit (three at head_dim 64): with eight wavefronts in step 5 heads of 32760 tokens took 3939 us
// in the queries role, with four 3596, 24 heads of 4250 x 2 at head_dim 64 1010 and 877 us in both.
//
// The matrix rate under the power limit bounds long rows: bf16, 5 heads of 32760 at head_dim 128 take 7.6 to 7.8 ms, 1.23 to 1.27 PFLOP/s
// over the seven products where a library product of 8192^3 reaches 1.33 (matrix pipe busy 65 % at 1.7 GHz, no LDS bank conflicts); 24
// heads of 4608 769 to 800 us, 1.14 to 1.19. fp16, 48 heads of 4250 at head_dim 64: 778 to 805 us.
//
// MFMA orientation (v_mfma_f32_32x32x16; A is 32x16, B is 16x32, lane l holds row/column l%32 and contraction elements
// 8*(l/32)..+7; the result puts column l%32 and rows 8*(i/4) + 4*(l/32) + i%4, i = 0..15, in lane l).  X, Y: the streamed tensors
// (keys role: q, dout; queries role: k, v); F, G: the owned rows (k, v; q, dout), in registers for the whole kernel:
//   S  = X F^T, dP = Y G^T   A = rows of X, Y from LDS, B = F^T, G^T: a lane owns ONE row of F, and P, dS of it in its accumulators
//   dV^T += Y^T P (keys role), dF^T += X^T dS   A = X^T, Y^T read transposed from LDS; B = P, dS: the accumulators, converted, are the operand
// P and dS are rounded to the tensors' type for their products; all sums are fp32.
#include "attn_bwd_rows.h"
#include "attn_split.h"
#include "attn_tiles.h"

namespace xdit {
namespace {

constexpr int kTileRows = 64;   // streamed rows per LDS tile

// LDS layout of a streamed tile: 64 rows, filled by 1 KiB pieces (a direct load writes lane i at 16 i), pieces 16 bytes more apart.
// It is read in two ways: 16 consecutive rows at one 16-byte column (contraction over head_dim) and 4 consecutive rows at 64 bytes of
// columns (transposed).  Rows r sit 16 * (4 (r % 4) + (r / 4) % 4) bytes apart modulo 256, which spreads either over all banks.
template <int D> struct BwdGeom {
  static constexpr int ROW_BYTES = 2 * D;
  static constexpr int NG = kTileRows * ROW_BYTES / 1024;   // pieces
  static constexpr int PITCH = 1024 + 16;
  static constexpr int TENSOR_BYTES = NG * PITCH;
  static constexpr int STAT_BYTES = 2 * kTileRows * 4;
  static constexpr int BUF_BYTES = 2 * TENSOR_BYTES + STAT_BYTES;
  static constexpr int LANES_PER_ROW = ROW_BYTES / 16;
  static __device__ __forceinline__ int piece(int r) { return D == 128 ? 4 * (r & 3) + ((r >> 2) & 3) : 4 * (r & 1) + ((r >> 2) & 3); }
  static __device__ __forceinline__ int slot(int r) { return D == 128 ? r >> 4 : ((r >> 1) & 1) + 2 * (r >> 4); }
  static __device__ __forceinline__ int row(int g, int s) {
    return D == 128 ? ((g >> 2) & 3) + 4 * (g & 3) + 16 * s : (g >> 2) + 2 * (s & 1) + 4 * (g & 3) + 16 * (s >> 1);
  }
  static constexpr int STEP32 = (D == 128 ? 2 : 4) * ROW_BYTES;  // +32 rows
  static constexpr int STEP16 = STEP32 / 2;                      // +16 rows
  static constexpr int STEP8 = 2 * PITCH;                        // +8 rows where bit 3 of the row is clear
};

// fp16: numbers end at 2^-24 and 65504, and P and dS span more than that.  P is computed times 2^15 in the keys role, which is free: the
// exponent gets it.  dS is computed times 2^m, and a lane owns one row of the result, so that m is the lane's own:
//   queries role  the row's largest possible dS stays below 2^15, by
//                 |dS_ij| = P_ij |dP_ij - delta_i| <= |dout_i| max_j |v_j| + |delta_i|      (norms; of a chunk of a ring P_ij <= 1 too)
//   keys role     a key's dS are those of many queries, of any sizes, and P_ij may be far below 1: m starts at kFp16Most and is lowered (lower_exponent)
//                 where a dS of the key would come to 2^15, so that this one comes to 2^2 .. 2^3.  What is off by a
//                 denormal's 2^-25 afterwards is so by 2^-27 of the largest, whose own rounding is 2^-11.
// (One m for a whole (batch, head), from a bound over all of its rows: 16384 keys at head_dim 128, a row of dout 4000 times the others and
// a value of 50, the error of the other rows' dq was 1.2e-2 of them, 2.8e-4 with a row's own.  The maximum costs 48 heads of
// 4250 at head_dim 64 805 us instead of 798.)
constexpr int kFp16Most = 40;   // a dS of less than 2^-38 at most is below every fp16 result

// The largest norm of a row of v.
__device__ __forceinline__ float value_norm_of(const AttnBwdParams& p, int bh) {
  __shared__ float tops[kBwdWaves];
  const int n = bwd_value_blocks(p);
  float top = 0.f;   // of the values' norms
  for (int i = threadIdx.x; i < n; i += 64 * kBwdWaves) top = fmaxf(top, p.value_norms[(int64_t)bh * n + i]);
  for (int m = 1; m < 64; m <<= 1) top = fmaxf(top, __shfl_xor(top, m));
  if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
  __syncthreads();
  for (int i = 0; i < kBwdWaves; i++) top = fmaxf(top, tops[i]);
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(top)));
}

// The queries role's m of a row whose dS stay at or below `most`.
__device__ __forceinline__ int fp16_exponent(float most) {
  const int e = (int)(__float_as_uint(most) >> 23 & 255);   // below 2^(e - 126)
  const int m = e == 255 ? 0 : 141 - e;                     // (not finite: nor is the row)
  return m > kFp16Most ? kFp16Most : m;
}

// Where a lane's dS come to 2^15: lowers the exponent of its key, whose other rows the lane 32 away has, and what has been added up.
template <int DBLOCKS>
__device__ __forceinline__ void lower_exponent(float top, float& p_to_ds, f32x16& ds, f32x16 (&acc)[DBLOCKS]) {
  const int e = (int)(__float_as_uint(max_halves(top)) >> 23) - 127;
  const float less = __builtin_ldexpf(1.f, e >= 15 && e < 128 ? 2 - e : 0);   // (an infinity stays one)
  p_to_ds *= less;
#pragma unroll
  for (int i = 0; i < 16; i++) ds[i] *= less;
#pragma unroll
  for (int db = 0; db < DBLOCKS; db++)
#pragma unroll
    for (int i = 0; i < 16; i++) acc[db][i] *= less;
}

constexpr int kAhead = 4;  // LDS fragment reads in flight

// Staging block of a wavefront for its results: 32 rows of 64 columns, rows 8 bytes apart from a multiple of 128.
constexpr int kBwdStagePitch = 64 * 2 + 8;
constexpr int kBwdStageBytes = 32 * kBwdStagePitch;

// S += X_half F^T, then dP += Y_half G^T (contraction over head_dim, KSTEPS steps of 16 each): one sequence of fragment reads, so that
// the second product does not wait for its first ones.  Y lies Y_OFF bytes behind X.
template <typename T, int KSTEPS, int Y_OFF>
__device__ __forceinline__ void rows_products(f32x16& s, f32x16& dp, const typename Mfma16<T>::vec8 (&f)[KSTEPS], const typename Mfma16<T>::vec8 (&g)[KSTEPS], unsigned addr) {
  constexpr int N = 2 * KSTEPS;
  typename Mfma16<T>::vec8 x[N];
  auto read = [&](auto I) {
    constexpr int i = I;
    lds_read_b128<(i < KSTEPS ? 32 * i : Y_OFF + 32 * (i - KSTEPS))>(x[i], addr);
  };
  static_for<kAhead>([&](auto I) { read(I); });
  static_for<N>([&](auto I) {
    constexpr int i = I;
    constexpr int younger = (i + kAhead <= N ? kAhead : N - i) - 1;
    lds_wait<younger>(x[i]);
    if constexpr (i < KSTEPS) s = Mfma16<T>::mma(x[i], f[i], s);
    else dp = Mfma16<T>::mma(x[i], g[i - KSTEPS], dp);
    if constexpr (i + kAhead < N) read(std::integral_constant<int, i + kAhead>{});
  });
}

// Transposed products over the half's 32 rows, a sequence of fragment reads again: G_PRODUCTS: acc_g[db] += Y_half^T P, then acc_f[db] +=
// X_half^T dS (pf, df: two steps of 16 rows).  The first reads are started by `start`, ahead of the arithmetic that makes P and dS.
template <typename T, int D, int DBLOCKS, bool G_PRODUCTS, int Y_OFF>
struct ColumnsProducts {
  typedef typename Mfma16<T>::vec8 vec8;
  typedef BwdGeom<D> G;
  typedef __attribute__((ext_vector_type(8))) short s16x8;
  static constexpr int NM = 2 * DBLOCKS, N = G_PRODUCTS ? 2 * NM : NM;
  static constexpr int PD = kAhead / 2 < N ? kAhead / 2 : N;   // products whose two reads are in flight
  s16x4 v0[N], v1[N];
  template <int i> __device__ __forceinline__ void read(unsigned addr) {
    constexpr int j = G_PRODUCTS && i >= NM ? i - NM : i;
    constexpr int off = (G_PRODUCTS && i < NM ? Y_OFF : 0) + (j / DBLOCKS) * G::STEP16 + (j % DBLOCKS) * 64;
    lds_read_tr16_b64<off>(v0[i], addr);
    lds_read_tr16_b64<off + G::STEP8>(v1[i], addr);
  }
  __device__ __forceinline__ void start(unsigned addr) {
    static_for<PD>([&](auto I) { this->template read<decltype(I)::value>(addr); });
  }
  template <int NG>
  __device__ __forceinline__ void run(f32x16 (&acc_g)[NG], f32x16 (&acc_f)[DBLOCKS], const vec8 (&pf)[2], const vec8 (&df)[2], unsigned addr) {
    static_for<N>([&](auto I) {
      constexpr int i = decltype(I)::value;
      constexpr int younger = 2 * ((i + PD <= N ? PD : N - i) - 1);
      lds_wait2<younger>(v0[i], v1[i]);
      const s16x8 vv = __builtin_shufflevector(v0[i], v1[i], 0, 1, 2, 3, 4, 5, 6, 7);
      constexpr int j = G_PRODUCTS && i >= NM ? i - NM : i;
      if constexpr (G_PRODUCTS && i < NM) acc_g[j % DBLOCKS] = Mfma16<T>::mma(__builtin_bit_cast(vec8, vv), pf[j / DBLOCKS], acc_g[j % DBLOCKS]);
      else acc_f[j % DBLOCKS] = Mfma16<T>::mma(__builtin_bit_cast(vec8, vv), df[j / DBLOCKS], acc_f[j % DBLOCKS]);
      if constexpr (i + PD < N) this->template read<i + PD>(addr);
    });
  }
};

// One unit of a role.  D: the head_dim of the LDS geometry, DC (a multiple of 32) that of the gradients, DK (a multiple of 16) the
// contracted one; columns between the tensors' head_dim and those are zeros in F and G and in the LDS tiles.
template <typename T, int D, int DC, int DK, bool KEYS>
__device__ __forceinline__ void bwd_role(const AttnBwdParams& p, int xcd, int n, unsigned char* smem) {
  typedef typename Mfma16<T>::vec8 vec8;
  typedef __attribute__((ext_vector_type(4))) T vec4;
  typedef BwdGeom<D> G;
  constexpr int NW = kBwdWaves, KSTEPS = DK / 16, DBLOCKS = DC / 32, ROWS = kBwdRows;

  const BwdRole& R = KEYS ? p.keys : p.queries;
  BwdUnit unit;
  if (!bwd_unit(R, xcd, n, unit)) return;
  const int bh = unit.tile / R.tiles;
  int tile = unit.tile - bh * R.tiles;
  const int b = bh / p.H, h = bh - b * p.H;
  const int first = unit.slot < 0 ? 0 : unit.part * R.len;
  const int last = unit.slot < 0 || first + R.len > R.steps ? R.steps : first + R.len;

  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x >> 6);
  const int lane = threadIdx.x & 63, l32 = lane & 31, hh = lane >> 5;

  // ---- owned rows ----
  const bool second = KEYS && tile >= p.tiles1;
  if (second) tile -= p.tiles1;
  const BwdTensor& F = KEYS ? (second ? p.k2 : p.k) : p.q;
  const BwdTensor& Gt = KEYS ? (second ? p.v2 : p.v) : p.dout;
  const int own_rows = KEYS ? (second ? p.Sk2 : p.Sk) : p.Sq;
  const int own0 = tile * ROWS + wave * 32;
  const int own = own0 + l32;
  // Whole rows side by side in a load; through LDS (below) every lane gets its own row.  (Each lane's own row by loads of 32 bytes a row: a
  // unit of 40 heads of 32760 on 512 keys took 5.3 us to issue them, so 3.3; the call 1265 us, so 1240.)
  constexpr int OWN_LOADS = D / 16;
  vec8 raw_f[OWN_LOADS], raw_g[OWN_LOADS];
  {
    const int chunk = lane % G::LANES_PER_ROW;
    const T* fp = (const T*)F.p + b * F.b + h * F.h + chunk * 8;
    const T* gp = (const T*)Gt.p + b * Gt.b + h * Gt.h + chunk * 8;
#pragma unroll
    for (int i = 0; i < OWN_LOADS; i++) {
#pragma unroll
      for (int e = 0; e < 8; e++) raw_f[i][e] = raw_g[i][e] = (T)0.f;
      int r = own0 + (i * 64 + lane) / G::LANES_PER_ROW;
      r = r < own_rows ? r : own_rows - 1;
      if (chunk * 8 < p.D) {
        raw_f[i] = *(const vec8*)(fp + (int64_t)r * F.s);
        raw_g[i] = *(const vec8*)(gp + (int64_t)r * Gt.s);
      }
    }
  }
  const float c = p.scale * kLog2e;
  const float* stats = p.stats + (int64_t)bh * 2 * p.sq_pad;
  constexpr bool FP16 = __is_same(T, _Float16);
  const float value_norm = FP16 && !KEYS ? value_norm_of(p, bh) : 0.f;
  int m = 0;   // fp16, queries role
  float p_to_ds = FP16 && KEYS ? __builtin_ldexpf(1.f, kFp16Most - kFp16Exponent) : 1.f;
  float own_lse = 0.f, own_nd = 0.f;
  if constexpr (!KEYS) {
    if (own < p.sq_pad) { own_lse = stats[own]; own_nd = stats[p.sq_pad + own]; }
  }

  // ---- tile loads ----
  const unsigned lds_base = (unsigned)(uintptr_t)(XDIT_LDS unsigned char*)smem;
  // Wavefront w loads pieces w, w + 4, ...: piece w + 4 i holds the rows i + ld_row of its lanes.
  const bool ld_on = (lane % G::LANES_PER_ROW) * 8 < p.D;
  // (Lane numbers are asked for again where they are needed: two registers more through the loop would spill at head_dim 128.)
  auto ld_row = [&] { return G::row(wave, lane_now() / G::LANES_PER_ROW); };
  auto ld_col = [&] { return (unsigned)(lane_now() % G::LANES_PER_ROW) * 16; };
  const unsigned char* ld_x;   // first rows of the tile to be loaded next
  const unsigned char* ld_y;
  const float* ld_stats = stats;
  unsigned ld_xs, ld_ys, ld_vx, ld_vy;   // row strides, the lane's offsets in bytes
  int ld_left;                 // rows of the segment from that tile on
  auto aim = [&](int t) {
    const bool s2 = !KEYS && t >= p.step1;
    const BwdTensor& X = KEYS ? p.q : s2 ? p.k2 : p.k;
    const BwdTensor& Y = KEYS ? p.dout : s2 ? p.v2 : p.v;
    const int row0 = (s2 ? t - p.step1 : t) * kTileRows;
    ld_left = (KEYS ? p.Sq : s2 ? p.Sk2 : p.Sk) - row0;
    ld_xs = (unsigned)X.s * 2;
    ld_ys = (unsigned)Y.s * 2;
    ld_x = (const unsigned char*)((const T*)X.p + b * X.b + h * X.h + (int64_t)row0 * X.s);
    ld_y = (const unsigned char*)((const T*)Y.p + b * Y.b + h * Y.h + (int64_t)row0 * Y.s);
    if (KEYS) ld_stats = stats + row0;
    ld_vx = __umul24((unsigned)ld_row(), ld_xs) + ld_col();
    ld_vy = __umul24((unsigned)ld_row(), ld_ys) + ld_col();
  };
  // Loads that tile and moves on to the one behind it.
  auto issue = [&](unsigned bo) {
    if (ld_on) {
      const unsigned dst = lds_base + bo + wave * G::PITCH;
      if (ld_left >= kTileRows) {
#pragma unroll
        for (int i = 0; i < G::NG / NW; i++) {
          load_lds_16(ld_x + (uint64_t)i * ld_xs, ld_vx, dst + i * NW * G::PITCH);
          load_lds_16(ld_y + (uint64_t)i * ld_ys, ld_vy, dst + G::TENSOR_BYTES + i * NW * G::PITCH);
        }
      } else {   // a segment's last tile: rows past its end re-read the last one
#pragma unroll
        for (int i = 0; i < G::NG / NW; i++) {
          int r = ld_row() + i;
          r = r < ld_left ? r : ld_left - 1;
          load_lds_16(ld_x, __umul24((unsigned)r, ld_xs) + ld_col(), dst + i * NW * G::PITCH);
          load_lds_16(ld_y, __umul24((unsigned)r, ld_ys) + ld_col(), dst + G::TENSOR_BYTES + i * NW * G::PITCH);
        }
      }
    }
    if (KEYS && wave < 2) load_lds_4(ld_stats + wave * p.sq_pad, lane_now() * 4, lds_base + bo + 2 * G::TENSOR_BYTES + wave * kTileRows * 4);
    ld_x += (uint64_t)ld_xs * kTileRows;
    ld_y += (uint64_t)ld_ys * kTileRows;
    ld_left -= kTileRows;
    if (KEYS) ld_stats += kTileRows;
  };
  aim(first);
  issue(0);
  // The owned rows through the second buffer, which is free until the first step: a wavefront's 32 rows in a block of its own, 16-byte
  // columns exchanged by the row's number, so that neither the writes nor the reads meet a bank twice.
  vec8 f[KSTEPS], g[KSTEPS];
  {
    XDIT_LDS unsigned char* const stage = (XDIT_LDS unsigned char*)smem + G::BUF_BYTES + wave * 32 * G::ROW_BYTES;
    static_assert(NW * 32 * G::ROW_BYTES <= G::BUF_BYTES, "owned rows");
#pragma unroll
    for (int which = 0; which < 2; which++) {
#pragma unroll
      for (int i = 0; i < OWN_LOADS; i++) {
        const int row = (i * 64 + lane) / G::LANES_PER_ROW, chunk = lane % G::LANES_PER_ROW;
        *(XDIT_LDS vec8*)(stage + row * G::ROW_BYTES + (chunk ^ (row % G::LANES_PER_ROW)) * 16) = which ? raw_g[i] : raw_f[i];
      }
      __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
      __builtin_amdgcn_wave_barrier();
#pragma unroll
      for (int ks = 0; ks < KSTEPS; ks++)
        (which ? g : f)[ks] = *(const XDIT_LDS vec8*)(stage + l32 * G::ROW_BYTES + ((2 * ks + hh) ^ (l32 % G::LANES_PER_ROW)) * 16);
      __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
      __builtin_amdgcn_wave_barrier();
    }
  }
  // Every wait for the owned rows is here: one inside the loop would be one for the tile loads too.
#pragma unroll
  for (int ks = 0; ks < KSTEPS; ks++) asm volatile("" : "+v"(f[ks]), "+v"(g[ks]));
  if constexpr (FP16 && !KEYS) {
    float squares = 0.f;
#pragma unroll
    for (int ks = 0; ks < KSTEPS; ks++)
#pragma unroll
      for (int e = 0; e < 8; e++) squares = __builtin_fmaf((float)g[ks][e], (float)g[ks][e], squares);
    m = fp16_exponent(__builtin_sqrtf(sum_halves(squares)) * value_norm + __builtin_fabsf(own_nd));
    own_lse += (float)(kFp16Exponent - m);
  }
  // Columns that the tensors do not have: zeros, once.
  if (DC > p.D) {
    __syncthreads();   // all wavefronts have their owned rows
    const i32x4 zero = {0, 0, 0, 0};
    const int c0 = p.D / 8, n = DC / 8 - c0;
    for (int i = threadIdx.x; i < 4 * kTileRows * n; i += 64 * NW) {
      const int which = i / (kTileRows * n), j = i % (kTileRows * n), r = j % kTileRows, ch = c0 + j / kTileRows;
      *(XDIT_LDS i32x4*)((XDIT_LDS unsigned char*)smem + (which >> 1) * G::BUF_BYTES + (which & 1) * G::TENSOR_BYTES + G::piece(r) * G::PITCH + G::slot(r) * G::ROW_BYTES + ch * 16) = zero;
    }
  }

  const unsigned row_addr = lds_base + G::piece(l32) * G::PITCH + G::slot(l32) * G::ROW_BYTES + hh * 16;
  const int tr_row = 4 * hh + ((lane & 15) >> 2);
  const unsigned col_addr = lds_base + G::piece(tr_row) * G::PITCH + G::slot(tr_row) * G::ROW_BYTES + (16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2;

  f32x16 acc_f[DBLOCKS], acc_g[KEYS ? DBLOCKS : 1];
#pragma unroll
  for (int db = 0; db < DBLOCKS; db++)
#pragma unroll
    for (int e = 0; e < 16; e++) {
      acc_f[db][e] = 0.f;
      if (KEYS) acc_g[KEYS ? db : 0][e] = 0.f;
    }
  for (int t = first; t < last; t++) {
    const unsigned bo = ((t - first) & 1) * G::BUF_BYTES;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __syncthreads();
    const int left = ld_left + kTileRows;   // rows of the segment from this tile on
    if (t + 1 < last) {
      if (!KEYS && t + 1 == p.step1) aim(t + 1);   // the second segment's first tile
      issue(G::BUF_BYTES - bo);
    }
    // Queries that attended nothing: zeros in place of rows that need not be finite, which a probability of zero does not undo.  (Looking
    // at 64 log-sum-exps a tile: 5 heads of 32760 7543 -> 7590 us, 24 of 4608 766 -> 769.)
    if constexpr (KEYS) {
      XDIT_LDS unsigned char* const buf = (XDIT_LDS unsigned char*)smem + bo;
      const uint64_t none = __builtin_amdgcn_ballot_w64(((const XDIT_LDS float*)(buf + 2 * G::TENSOR_BYTES))[lane_now()] == INFINITY);
      if (none << (left < kTileRows ? kTileRows - left : 0)) {   // (rows behind the last one alone are copies of it)
        for (uint64_t rest = none; rest != 0; rest &= rest - 1) {
          const int r = __builtin_ctzll(rest), n = lane_now();
          XDIT_LDS int* const row = (XDIT_LDS int*)(buf + G::piece(r) * G::PITCH + G::slot(r) * G::ROW_BYTES) + n;
          if (n * 4 < G::ROW_BYTES) row[0] = row[G::TENSOR_BYTES / 4] = 0;
        }
        __syncthreads();
      }
    }
    const int halves = own0 >= own_rows ? 0 : left > 32 ? 2 : 1;
#pragma unroll 1
    for (int hb = 0; hb < halves; hb++) {   // 32 streamed rows at a time, those that there are
      const unsigned ra = row_addr + bo + hb * G::STEP32, ca = col_addr + bo + hb * G::STEP32;
      f32x16 s, dp;
      const XDIT_LDS f32x4* st = (const XDIT_LDS f32x4*)((XDIT_LDS unsigned char*)smem + bo + 2 * G::TENSOR_BYTES + hb * 128 + hh * 16);
#pragma unroll
      for (int i = 0; i < 4; i++) {
        f32x4 x = {own_nd, own_nd, own_nd, own_nd};
        if (KEYS) x = st[kTileRows / 4 + 2 * i];
#pragma unroll
        for (int e = 0; e < 4; e++) {
          s[4 * i + e] = 0.f;
          dp[4 * i + e] = x[e];
        }
      }
      rows_products<T, KSTEPS, G::TENSOR_BYTES>(s, dp, f, g, ra);
      __builtin_amdgcn_sched_barrier(0);
      if constexpr (FP16 && KEYS) {   // ahead of the other reads: none may be in flight where accumulators change
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < 4; i++) {
          f32x4 x = st[2 * i];
#pragma unroll
          for (int e = 0; e < 4; e++) {
            s[4 * i + e] = fast_exp2(__builtin_fmaf(s[4 * i + e], c, -x[e]));
            dp[4 * i + e] *= s[4 * i + e] * p_to_ds;
            top = fmaxf(top, __builtin_fabsf(dp[4 * i + e]));
          }
        }
        if (__builtin_amdgcn_ballot_w64(top >= 32768.f)) lower_exponent(top, p_to_ds, dp, acc_f);
      }
      ColumnsProducts<T, D, DBLOCKS, KEYS, G::TENSOR_BYTES> columns;
      columns.start(ca);
      vec8 pf[2], df[2];
      if constexpr (!KEYS) {
#pragma unroll
        for (int e = 0; e < 16; e++) s[e] = fast_exp2(__builtin_fmaf(s[e], c, -own_lse));
        if (left < kTileRows) {   // only a segment's last tile: keys behind its end
#pragma unroll
          for (int e = 0; e < 16; e++)
            if (32 * hb + 8 * (e >> 2) + 4 * hh + (e & 3) >= left) s[e] = 0.f;
        }
      }
#pragma unroll
      for (int i = 0; i < 4; i++) {
        f32x4 pr, ds;
        if constexpr (KEYS && !FP16) {
          f32x4 x = st[2 * i];
#pragma unroll
          for (int e = 0; e < 4; e++) pr[e] = fast_exp2(__builtin_fmaf(s[4 * i + e], c, -x[e]));
        }
#pragma unroll
        for (int e = 0; e < 4; e++) {
          if (!KEYS || FP16) pr[e] = s[4 * i + e];
          ds[e] = FP16 && KEYS ? dp[4 * i + e] : pr[e] * dp[4 * i + e];
        }
        const vec4 a = __builtin_convertvector(pr, vec4), d = __builtin_convertvector(ds, vec4);
#pragma unroll
        for (int e = 0; e < 4; e++) {
          pf[i >> 1][4 * (i & 1) + e] = a[e];
          df[i >> 1][4 * (i & 1) + e] = d[e];
        }
      }
      __builtin_amdgcn_sched_barrier(0);
      columns.run(acc_g, acc_f, pf, df, ca);
    }
  }

  // ---- results ----
  if (!KEYS && own_lse == INFINITY) {   // a query that attended nothing: zeros, whatever its rows hold
#pragma unroll
    for (int db = 0; db < DBLOCKS; db++)
#pragma unroll
      for (int e = 0; e < 16; e++) acc_f[db][e] = 0.f;
  }
  if (unit.slot < 0) __syncthreads();   // the staging blocks lie over the tiles
#pragma unroll
  for (int which = 0; which < (KEYS ? 2 : 1); which++) {   // 0: gradient of F, 1: of G
    const float w = which ? __builtin_ldexpf(1.f, FP16 ? -kFp16Exponent : 0) : FP16 && KEYS ? p.scale * __builtin_ldexpf(1.f, -kFp16Exponent) / p_to_ds : __builtin_ldexpf(p.scale, -m);
    if (unit.slot >= 0) {
      f32x4* to = (f32x4*)(R.partial + (unit.slot * (KEYS ? 2 : 1) + which) * ROWS * DC) + wave * (8 * DC) + lane;   // register by register: PartLayout
#pragma unroll
      for (int db = 0; db < DBLOCKS; db++)
#pragma unroll
        for (int a = 0; a < 4; a++) {
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = (which ? acc_g[KEYS ? db : 0] : acc_f[db])[4 * a + e] * w;
          to[(4 * db + a) * 64] = x;
        }
    } else {
      // Through LDS, 64 columns at a time, so that a store covers whole 128-byte lines of 8 rows.
      const BwdTensor& O = KEYS ? (which ? (second ? p.dv2 : p.dv) : (second ? p.dk2 : p.dk)) : p.dq;
      T* orow = (T*)O.p + b * O.b + h * O.h + (int64_t)own0 * O.s;
      XDIT_LDS unsigned char* stage = (XDIT_LDS unsigned char*)smem + wave * kBwdStageBytes;
      const int rows_live = own_rows - own0;   // may be <= 0 or above 32
#pragma unroll
      for (int half = 0; half < (DBLOCKS + 1) / 2; half++) {
#pragma unroll
        for (int d = 0; d < 2; d++) {
          const int db = 2 * half + d;
          if (db < DBLOCKS) {
#pragma unroll
            for (int a = 0; a < 4; a++) {
              f32x4 x;
#pragma unroll
              for (int e = 0; e < 4; e++) x[e] = (which ? acc_g[KEYS ? db : 0] : acc_f[db])[4 * a + e] * w;
              *(XDIT_LDS vec4*)(stage + l32 * kBwdStagePitch + (32 * d + 8 * a + 4 * hh) * 2) = __builtin_convertvector(x, vec4);
            }
          }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
#pragma unroll
        for (int r = 0; r < 4; r++) {
          const int row = (lane >> 3) + 8 * r, col = 64 * half + (lane & 7) * 8;
          const vec8 x = *(const XDIT_LDS vec8*)(stage + row * kBwdStagePitch + (lane & 7) * 16);
          if (row < rows_live && col < p.D) *(vec8*)(orow + row * O.s + col) = x;
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        __builtin_amdgcn_wave_barrier();
      }
    }
  }
}

// Workgroup i runs on XCD i % 8: an XCD takes consecutive tiles, so that those of one (batch, head) stream the same rows through one L2.
template <typename T, int D, int DC, int DK>
__global__ __launch_bounds__(64 * kBwdWaves, D == 64 ? 3 : 2) void attn_bwd_16_kernel(const AttnBwdParams p) {
  extern __shared__ __attribute__((aligned(1024))) unsigned char smem[];
  const int xcd = blockIdx.x % 8, n = blockIdx.x / 8;
  if (n < p.keys.units) bwd_role<T, D, DC, DK, true>(p, xcd, n, smem);
  else bwd_role<T, D, DC, DK, false>(p, xcd, n - p.keys.units, smem);
}

template <typename T, int D, int DC, int DK = DC>
hipError_t launch_kernels(const AttnBwdParams& p, hipStream_t stream) {
  static std::atomic<bool> lds_ready[kMaxDevices];
  constexpr int lds = 2 * BwdGeom<D>::BUF_BYTES;
  static_assert(lds >= kBwdWaves * kBwdStageBytes, "staging blocks");
  const int slot = current_device_slot();
  if (!lds_ready[slot].load(std::memory_order_relaxed)) {  // > 64 KiB of dynamic LDS must be enabled once per kernel and device
    hipError_t e = hipFuncSetAttribute((const void*)attn_bwd_16_kernel<T, D, DC, DK>, hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
    lds_ready[slot].store(true, std::memory_order_relaxed);
  }
  launch_bwd_stats<T>(p, stream);
  hipLaunchKernelGGL((attn_bwd_16_kernel<T, D, DC, DK>), dim3(8u * (unsigned)(p.keys.units + p.queries.units)), dim3(64 * kBwdWaves), lds, stream, p);
  return launch_bwd_fold<T, DC, 32>(p, stream);
}

// (Contracting over 80 columns of 96 and 48 of 64: 16 heads of 4096 at head_dim 72 305 us instead of 318, 32 at 40 393 instead of 419.)
template <typename T>
hipError_t launch_typed(const AttnBwdParams& p, hipStream_t stream) {
  if (p.D <= 32) return launch_kernels<T, 64, 32>(p, stream);
  if (p.D <= 48) return launch_kernels<T, 64, 64, 48>(p, stream);
  if (p.D <= 64) return launch_kernels<T, 64, 64>(p, stream);
  if (p.D <= 80) return launch_kernels<T, 128, 96, 80>(p, stream);
  if (p.D <= 96) return launch_kernels<T, 128, 96>(p, stream);
  return launch_kernels<T, 128, 128>(p, stream);
}

}  // namespace

hipError_t launch_attn_bwd_16(const AttnBwdParams& p, int dtype_is_fp16, hipStream_t stream) {
  return dtype_is_fp16 ? launch_typed<_Float16>(p, stream) : launch_typed<__bf16>(p, stream);
}

}  // namespace xdit
