/*
 * xdit_amd_attn.h — C ABI of the MI355X (gfx950) attention hot path.
 *
 * One shared library (libxdit_amd_attn.so) exports the entry points below.  They are what a
 * foreign-function binding (ctypes, cffi, pybind, a C++ torch op) of xDiT's attention path would
 * bind on one GPU.  Every pointer is a DEVICE pointer owned by the caller; the library allocates
 * nothing, keeps nothing after return, never synchronises the device and launches on the stream
 * the caller passes.  All strides are in ELEMENTS of the tensor's own dtype.  The innermost
 * (head_dim) stride of every tensor is 1.
 *
 * Return value: 0 on success, a negative xdit_status otherwise; the message of the last failure
 * on the calling thread is available from xdit_attn_last_error().
 *
 * Reference interfaces replaced (paths relative to the xDiT source tree):
 *   - the `(out, lse)` vendor flash-attention forward reached by the backend registry entries
 *     xfuser/core/distributed/attention_backend.py:504-516 (SDPA_FLASH), :534-548 (SDPA_EFFICIENT),
 *     :774-823 (AITER), :887-918 (FLASH), and by the per-step kernel call of the legacy ring loop
 *     xfuser/core/long_ctx_attention/ring/ring_flash_attn.py:105-134            -> xdit_attn_fwd
 *   - the fp8 forward with per-(batch,head) descales, attention_backend.py:617-642 (FLASH_3_FP8)
 *     and :717-772 (AITER_FP8)                                                   -> xdit_attn_fwd (dtype FP8)
 *   - the ring online-softmax merge `update_out_and_lse` called at
 *     ring_flash_attn.py:138 (+ epilogue :145-148) and torch's `_SDPAMerger._merge_one`
 *     (torch/distributed/tensor/experimental/_context_parallel/_attention.py:181-182)
 *                                                                                -> xdit_lse_merge
 *   - `per_tensor_quant`, attention_backend.py:606-615                           -> xdit_fp8_quant
 */
#ifndef XDIT_AMD_ATTN_H
#define XDIT_AMD_ATTN_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define XDIT_ATTN_ABI_VERSION 11

typedef enum {
  XDIT_OK = 0,
  XDIT_ERR_INVALID_ARG = -1,   /* null pointer, bad shape/stride/alignment, unsupported option */
  XDIT_ERR_UNSUPPORTED = -2,   /* a combination this library does not implement (e.g. causal)  */
  XDIT_ERR_LAUNCH = -3         /* the HIP runtime rejected the launch                          */
} xdit_status;

typedef enum {
  XDIT_DTYPE_BF16 = 0,
  XDIT_DTYPE_FP16 = 1,
  XDIT_DTYPE_FP32 = 2,
  XDIT_DTYPE_FP8_E4M3FN = 3    /* OCP e4m3fn (max 448), the fp8 format of gfx950 */
} xdit_dtype;

/* Logical tensor (B, H, S, D) with arbitrary B/H/S element strides; D stride is 1.
 * BHSD-contiguous:                stride = {H*S*D, S*D, D}
 * BSHD-contiguous viewed as BHSD: stride = {S*H*D, D, H*D}                                   */
typedef struct {
  int64_t b, h, s;
} xdit_strides;

/*
 * Non-causal scaled-dot-product attention forward returning the output and the per-row
 * log-sum-exp (natural log, softmax scale included):
 *     s_ij = softmax_scale * sum_d q_id k_jd ,  j over Sk keys of (k,v) then Sk2 keys of (k2,v2)
 *     out_i = sum_j softmax_j(s_ij) v_j ,  lse_i = log sum_j exp(s_ij)
 * For FP8 inputs q,k,v are multiplied by q_descale[b,h], k_descale[b,h], v_descale[b,h] first.
 * head_dim: a multiple of 8; bf16 / fp16 / fp32 up to 128 (bf16 and fp16 on the 16-bit matrix
 * cores at every such head_dim, at the cost of the next of 64 / 128; fp32 on the fp32 matrix
 * cores), fp8 128 or 64.
 * Replaces: attention_backend.py:504-516/:774-823/:887-918 (+ :617-642, :717-772 for fp8) and the
 * kernel call at ring_flash_attn.py:123-134.  The optional second KV segment replaces the
 * torch.cat of joint (text) keys/values at usp.py:239-241 / ring_flash_attn.py:89-100.
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_attn_args) */
  int32_t dtype;               /* xdit_dtype of q, k, v, k2, v2 */
  int32_t out_dtype;           /* xdit_dtype of out: same as dtype for bf16/fp16/fp32; bf16 or fp16 for fp8 */
  int32_t causal;              /* must be 0 */
  int32_t B, H, D;             /* batch, heads (Hq == Hk), head_dim */
  int32_t rows_per_workgroup;  /* 0 = chosen by the library; 128, 256 or 384 = that workgroup shape
                                  (bf16 / fp16 / fp8 kernels; a tuning and testing aid) */
  int64_t Sq, Sk, Sk2;         /* query rows; keys in segment 1; keys in segment 2 (0 = none) */
  float softmax_scale;         /* > 0 */
  int32_t cu_count;            /* 0 = plan the launch for the compute units of the current device;
                                  > 0 = for that many (tuning, testing, capacity planning) */
  int32_t streamed_sharing;    /* 0 (default): the work geometry of a launch is fixed, so results are
                                  reproducible bit for bit from call to call, as those of the vendor
                                  forwards this call replaces are (the reference's `deterministic`
                                  option concerns its backward pass only: ring_flash_attn.py:190, :206,
                                  :229).  != 0 opts in to a balanced launch that hands KV iterations of
                                  a shared query tile to whichever workgroup is free: 1-2 % faster on
                                  some shapes, results then reproducible only to rounding (the last
                                  bit of some outputs) */
  int32_t workspace_preserved; /* != 0: the caller vouches that nothing but this library has written
                                  `workspace` since an earlier call of this library that was given the
                                  same pointer, returned XDIT_OK and had 0 here on the first call after
                                  allocating the buffer (any such call will do: balanced or not, any
                                  dtype; a call that is given a workspace of at least 16 KiB with 0 here
                                  clears the counters at its start with a small launch).  The counters are
                                  then still zero and that launch is spared.  0 is always valid */
  int32_t balance;             /* 0 = the library decides from its time estimate whether a launch given a
                                  workspace is balanced; 1 = never (plain launch); 2 = whenever the planner
                                  offers a balanced plan (a tuning and testing aid, like rows_per_workgroup) */
  int32_t reserved0;           /* must be 0 */
  const void* q;
  const void* k;
  const void* v;
  const void* k2;              /* may be NULL when Sk2 == 0 */
  const void* v2;
  void* out;                   /* (B,H,Sq,D) out_dtype */
  float* lse;                  /* (B,H,Sq) fp32, may be NULL */
  xdit_strides q_stride, k_stride, v_stride, k2_stride, v2_stride, out_stride;
  int64_t lse_stride_b, lse_stride_h;   /* lse stride over Sq is 1 */
  const float* q_descale;      /* FP8 only: (B,H) fp32 each; NULL means 1.0 */
  const float* k_descale;
  const float* v_descale;
  int64_t descale_stride_b, descale_stride_h;
  void* workspace;             /* optional scratch, 16-byte aligned; may be NULL (see below) */
  int64_t workspace_bytes;
  void* stream;                /* hipStream_t; NULL = the null stream */
} xdit_attn_args;

int xdit_attn_fwd(const xdit_attn_args* args);

/*
 * xdit_attn_fwd on query rows that lie in two tensors (the image and the text queries of a joint
 * attention call): of the args->Sq rows the last tail->Sq2 are read from tail->q2, those before them
 * from args->q.  Everything else, the result included, is that of xdit_attn_fwd on the rows copied
 * one behind the other; sizing and planning calls take `args` as it is.  bf16 / fp16.
 * Replaces the torch.cat of the joint query at usp.py:286-288.
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_query_tail) */
  int32_t reserved0;           /* must be 0 */
  int64_t Sq2;                 /* 0 < Sq2 < args->Sq */
  const void* q2;              /* (B,H,Sq2,D), dtype of q */
  xdit_strides q2_stride;
} xdit_query_tail;

int xdit_attn_fwd_two_queries(const xdit_attn_args* args, const xdit_query_tail* tail);

/*
 * Scratch bytes with which xdit_attn_fwd can balance this problem over the chip: when the number
 * of query tiles is not a multiple of what the GPU holds at once, the key/value range of the
 * tiles of the last, partly filled round is shared between workgroups, whose partial
 * (out, lse) pairs go through the workspace and are folded by the workgroups themselves at their
 * ends (tiles of up to 16 parts) or by a second small kernel.
 * Returns 0 when nothing would be gained, a negative xdit_status for invalid arguments
 * (pointers are not inspected).  Passing no or too small a workspace to xdit_attn_fwd is always
 * valid: the launch is then simply not balanced.  The workspace needs no initialisation and may
 * be used for anything else between calls (see workspace_preserved for what a caller gains by
 * leaving it alone).  No counterpart in the reference (its kernels are vendor code).
 */
int64_t xdit_attn_workspace_bytes(const xdit_attn_args* args);

/*
 * xdit_attn_fwd for callers that cannot allocate device memory (code under HIP graph capture,
 * tight serving loops, harnesses that forbid hipMalloc): same arguments, results and kernels, but
 * the scratch of the balanced launch is a fixed array of XDIT_ATTN_NOALLOC_SCRATCH_BYTES inside
 * the library (one copy per GPU, held until the process ends) instead of a workspace of the
 * caller; args->workspace is ignored.  Nothing is allocated or freed by the call.  A problem whose
 * xdit_attn_workspace_bytes exceeds the array is rejected with XDIT_ERR_INVALID_ARG (use
 * xdit_attn_fwd with a workspace then, or set args->balance = 1: the plain launch needs no
 * scratch); Flux-1024 (B=1, H=24, S=4608, D=128) needs 28.75 MB.
 * Every call on a GPU shares that GPU's array: calls that may overlap on one GPU (two streams,
 * two threads) race on it and must be serialised by the caller; calls on one stream are ordered.
 * The array needs no clearing between calls (the kernels of a call leave its counters at zero; after
 * a call that failed a small launch clears them first).  It costs every GPU that the process uses
 * the library on its XDIT_ATTN_NOALLOC_SCRATCH_BYTES of device memory from the moment the library is
 * loaded, whether or not this entry point is ever called.  The first call on a device looks up the
 * array's device address and sets a kernel attribute: make it outside any stream capture; later
 * calls only launch kernels.  No counterpart in the reference.
 */
#define XDIT_ATTN_NOALLOC_SCRATCH_BYTES (32 * 1024 * 1024)
int xdit_attn_fwd_noalloc(const xdit_attn_args* args);

/*
 * How xdit_attn_fwd (or, with plan->ring_step set, xdit_attn_fwd_accumulate) would launch this
 * problem when given the workspace it asks for (pointers of `args` are not inspected): for tests,
 * tuning and capacity planning.  The query rows are cut
 * into `query_tiles` tiles of `rows_per_workgroup` rows, each with `kv_iterations` tiles of 64
 * keys.  `whole_tiles` of them are run by one workgroup each; with ranges > 0 the KV iterations
 * of the other tiles, laid end to end, are cut into `ranges` ranges of `range_len` iterations
 * (the last one shorter) that go to `claimers` workgroups: workgroup ids first_claimer ..
 * first_claimer + claimers - 1, of which those below whole_tiles run a whole tile first; claimer
 * c starts with range c and, with counter != 0, takes further ranges from a counter in the
 * workspace.  A query tile's partial results occupy at most `slots_per_tile` workspace slots.
 * bf16 / fp16 (head_dim up to 128; the geometry is that of head_dim 64 or 128, whichever is
 * the next one up) and fp8 (head_dim 128 or 64).  fp32 (head_dim up to 128): whole tiles only, of 128
 * rows with `kv_iterations` tiles of 32 keys, or, when those would leave more than a quarter of
 * the compute units without a workgroup, of 64 rows with tiles of 64 keys.  No counterpart in the
 * reference.
 * A 16-bit forward over few keys can run on another kernel instead (resident_parts > 0): the other fields then still
 * describe the launch it takes the place of.
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_launch_plan), set by the caller (or its size without resident_parts) */
  int32_t rows_per_workgroup;
  int32_t query_tiles;
  int32_t kv_iterations;
  int64_t workspace_bytes;     /* = xdit_attn_workspace_bytes(args); with ring_step: what xdit_attn_fwd_accumulate asks for */
  int32_t whole_tiles;
  int32_t ranges;
  int32_t range_len;
  int32_t slots_per_tile;
  int32_t claimers;
  int32_t first_claimer;
  int32_t counter;
  int32_t workgroups;          /* workgroups the attention kernel's work is cut into; all of them are launched,
                                  except in a plain launch (ranges == 0) of more than there are compute units
                                  whose workgroups fill a compute unit alone: one per compute unit is then
                                  started and runs the others one after the other */
  int32_t streamed;            /* != 0: streamed sharing instead of ranges: the `claimers` workgroups are dealt
                                  out over the shared tiles in contiguous groups; every member owns
                                  `range_len` KV iterations of its tile and draws the others one at a
                                  time from the tile's counter (only with streamed_sharing != 0) */
  int32_t fold_in_kernel;      /* != 0: the parts of a shared tile are folded by the workgroups of the attention
                                  kernel themselves (the ring step; tiles of at most 16 parts); 0: by a second
                                  small kernel */
  int32_t parts_first;         /* != 0: a claimer processes its range BEFORE its whole tile, and the workgroups
                                  fold the shared tiles at their ends, a slice of rows each */
  int32_t ring_step;           /* INPUT, set by the caller like struct_size: != 0 plans the launch of
                                  xdit_attn_fwd_accumulate for these arguments, 0 that of xdit_attn_fwd */
  int32_t resident_parts;      /* > 0: the call runs on the kernel that holds the keys of a (batch, head) in LDS (16-bit, at most
                                  four tiles of 64 keys at head_dim above 64, eight up to 64, both segments together;
                                  rows_per_workgroup and balance 0; where it is expected to take less time): the query
                                  rows of every (batch, head) are cut into this many parts, a workgroup each.  The result
                                  has the bits of the launch it takes the place of, which is always a plain one (ranges == 0) */
  int32_t reserved0;           /* 0 */
} xdit_launch_plan;

int xdit_attn_launch_plan(const xdit_attn_args* args, xdit_launch_plan* plan);

/*
 * One fold of the ring online-softmax merge, in fp32:
 *     acc_out <- acc_out - sigmoid(block_lse - acc_lse) * (acc_out - block_out)
 *     acc_lse <- acc_lse - logsigmoid(acc_lse - block_lse)
 * `first != 0` initialises instead: acc_out <- float(block_out), acc_lse <- block_lse.
 * If final_out != NULL the merged row is also written there in final_dtype (the epilogue cast
 * `out.to(q.dtype)`).  acc_out/block_out/final_out are logical (B,H,S,D); acc_lse/block_lse are
 * logical (B,H,S) with their own B/H/S strides, so the (B,S,H,1) accumulator layout of the legacy
 * ring and the (B,H,S) layout a kernel returns both map without copies.  head_dim: a multiple of
 * 8 up to 512.
 * Replaces: update_out_and_lse at ring_flash_attn.py:138, the epilogue at :145, and
 * torch _SDPAMerger._merge_one (…/_context_parallel/_attention.py:161-163, :181-182).
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_merge_args) */
  int32_t block_dtype;         /* xdit_dtype of block_out: bf16, fp16 or fp32 */
  int32_t final_dtype;         /* xdit_dtype of final_out (ignored when final_out == NULL) */
  int32_t first;               /* != 0: initialise the accumulator from the block */
  int32_t B, H, D;
  int32_t reserved0;
  int64_t S;
  float* acc_out;              /* fp32 */
  float* acc_lse;              /* fp32 */
  const void* block_out;
  const float* block_lse;      /* fp32 */
  void* final_out;             /* may be NULL */
  xdit_strides acc_out_stride, block_out_stride, final_out_stride;
  xdit_strides acc_lse_stride, block_lse_stride;
  void* stream;
} xdit_merge_args;

int xdit_lse_merge(const xdit_merge_args* args);

/*
 * One ring step in one launch: the forward of xdit_attn_fwd on this step's keys/values, folded
 * into the fp32 accumulator (acc_out, acc_lse) in the kernel's epilogue with the arithmetic of
 * xdit_lse_merge.  The block's rows are rounded to `out_dtype` before the fold, as if they had gone
 * through a block_out tensor, so the result equals xdit_attn_fwd + xdit_lse_merge bit for bit
 * (when neither launch is balanced, or both cut the KV iterations of their shared query tiles the
 * same way, which xdit_attn_launch_plan shows; to rounding of the block otherwise)
 * while the block is never written to memory and the accumulator is touched once.
 *   first != 0            initialise the accumulator from this block (acc_out is not read)
 *   args->out  (or NULL)  receives the merged rows in out_dtype: the final step's cast
 *   args->lse  (or NULL)  receives the merged log-sum-exp, (B,H,Sq) with args' lse strides
 *   discard_acc_out != 0  acc_out is read but not written back (last step: `out` and acc_lse
 *                         carry the result); needs args->out
 * acc_out is logical (B,H,Sq,D) fp32, acc_lse logical (B,H,Sq) fp32 with its own strides (the
 * (B,S,H,1) accumulator of the legacy ring maps without a copy).  bf16 / fp16 / fp32 inputs with
 * head_dim a multiple of 8 up to 128, fp8 inputs with head_dim 128 or 64; XDIT_ERR_UNSUPPORTED
 * otherwise (use the two calls).
 * args->workspace (optional, as for xdit_attn_fwd; the size this call asks for is the
 * workspace_bytes of xdit_attn_launch_plan with ring_step = 1, which can differ from
 * xdit_attn_workspace_bytes because the ring step is planned on its own; a smaller buffer is
 * valid, the launch is then not balanced) lets the launch be balanced: the parts of the shared
 * query tiles are then folded, and folded on into the accumulator, by the attention kernel's own
 * workgroups, and the result still equals a balanced xdit_attn_fwd with the same ranges +
 * xdit_lse_merge bit for bit.
 * Replaces, per ring step: the kernel call at ring_flash_attn.py:123-134, update_out_and_lse at
 * :138 and, on the last step, the cast at :145.
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_ring_acc) */
  int32_t first;
  int32_t discard_acc_out;
  int32_t reserved0;
  float* acc_out;
  float* acc_lse;
  xdit_strides acc_out_stride, acc_lse_stride;
} xdit_ring_acc;

int xdit_attn_fwd_accumulate(const xdit_attn_args* args, const xdit_ring_acc* acc);

/*
 * Abs-max fp8 quantiser, the step in front of the fp8 forward:
 *     scale = absmax(x) / 448 (1.0 if x is all zero) ;  y = fp8_e4m3fn(x / scale) ;  descale = scale
 * `per_tensor != 0`: one abs-max over the whole tensor, broadcast to every (b,h) entry of
 * `descale` — the reference's per_tensor_quant (attention_backend.py:606-615), whose descale is
 * `scale.expand(B, H)`.  `per_tensor == 0`: one abs-max per (batch, head) slice.
 * `scale_in != NULL` (device pointer to one float) supplies a static scale instead of the abs-max
 * (the `scale=` argument of per_tensor_quant).  Values whose quotient exceeds 448 saturate.
 * `x2` / `y2` (S2 > 0): a second tensor (B,H,S2,D) quantised with the scales of the first, the
 * abs-max taken over both (the joint keys, or values, that a caller would otherwise torch.cat onto
 * the first tensor before quantising: usp.py:239-241 in front of attention_backend.py:606-615).
 * `scratch`: optional device memory of at least XDIT_FP8_QUANT_SCRATCH_BYTES(B, H) bytes, private
 * to the stream until the call's kernels finish, no initialisation needed.  With it the call is
 * two launches (abs-max with one scratch slot per workgroup; cast), one with a static scale.
 * Without it `descale` (B*H contiguous fp32) doubles as the reduction buffer and the call is four
 * launches (clear, abs-max through atomics, cast, descales); results are the same.
 * `hadamard_block` (0 or 1 = off; else a power of two <= 128 that divides D) first rotates every
 * row along head_dim, block by block, by the orthonormal Sylvester-Hadamard matrix R of that size
 * with entries +-r, r = 1/sqrt(block) rounded to in_dtype, and rounds the result to in_dtype:
 * `torch.matmul(x.unflatten(-1, (D/block, block)), R).flatten(-2)` of the reference's
 * _fp8_hadamard_rotate (attention_backend.py:703-714; matrix :71-94).  Applied to both q and k
 * it leaves q.k unchanged and spreads outliers before the fp8 cast (:725-728).
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_quant_args) */
  int32_t in_dtype;            /* bf16, fp16 or fp32 */
  int32_t per_tensor;
  int32_t B, H, D;
  int64_t S;
  const void* x;               /* (B,H,S,D) in_dtype */
  void* y;                     /* (B,H,S,D) fp8 e4m3fn bytes */
  float* descale;              /* (B,H) fp32, contiguous */
  const float* scale_in;       /* optional static scale, may be NULL */
  xdit_strides x_stride, y_stride;
  void* stream;
  int32_t hadamard_block;
  int32_t reserved0;
  int64_t S2;                  /* rows of the second tensor (0 = none) */
  const void* x2;              /* (B,H,S2,D) in_dtype */
  void* y2;                    /* (B,H,S2,D) fp8 e4m3fn bytes */
  xdit_strides x2_stride, y2_stride;
  void* scratch;               /* optional, may be NULL */
  int64_t scratch_bytes;
} xdit_quant_args;

#define XDIT_FP8_QUANT_SCRATCH_BYTES(B, H) (4 * ((int64_t)(B) * (H) > 4096 ? (int64_t)(B) * (H) : 4096))

int xdit_fp8_quant(const xdit_quant_args* args);

/*
 * Up to four quantiser calls (the q, k and v of one attention call) in the same launches: `jobs` is an
 * array of `count` structs of one in_dtype and one stream, each as for xdit_fp8_quant.  Jobs with
 * scratch must not share it.  The results are those of `count` single calls, bit for bit.
 */
int xdit_fp8_quant_batch(const xdit_quant_args* jobs, int32_t count);

/*
 * Pre-attention prologue of an xDiT attention processor, fused into one pass over Q (or K):
 *     y = rotary(norm(x)), written through its own strides (e.g. BSHD in, BHSD-contiguous out)
 * replacing `attn.norm_q(query)`, `apply_rotary_emb(query, image_rotary_emb)` and the later
 * `.transpose(1, 2)` + contiguous copy (transformer_flux.py:116-147,
 * transformer_hunyuan_video.py:48-83, transformer_wan.py:99-122 under
 * xfuser/model_executor/models/transformers/).  With norm and rotation off it is a strided
 * re-layout (what V needs).  x and y are logical (B,H,S,D) with element strides.
 *   norm   XDIT_NORM_NONE; XDIT_NORM_HEAD: RMSNorm over head_dim of every (b,h,s) row, `weight`
 *          has D entries; XDIT_NORM_TOKEN: over all H*D elements of a token, `weight` has H*D
 *          entries indexed h*D+d (Wan's norm over the un-split projection).  Statistics in fp32:
 *          x * rsqrt(mean(x^2) + eps), rounded to dtype, times weight (same dtype; NULL = no
 *          gain), rounded again: the roundings of diffusers' RMSNorm with a 16-bit gain.
 *   rope   XDIT_ROPE_NONE; XDIT_ROPE_INTERLEAVED: pairs (2i, 2i+1),
 *          out[j] = x[j] cos[j] + rot[j] sin[j] with rot = (-x[2i+1], x[2i]) (diffusers
 *          apply_rotary_emb, use_real_unbind_dim=-1); XDIT_ROPE_SPLIT_HALF: pairs (j, j + D/2)
 *          (use_real_unbind_dim=-2); XDIT_ROPE_WAN: out[2i] = x[2i] cos[2i] - x[2i+1] sin[2i+1],
 *          out[2i+1] = x[2i] sin[2i+1] + x[2i+1] cos[2i] (transformer_wan.py:108-120).
 *          cos / sin are fp32, `rope_stride` elements from row to row, D values per row, shared
 *          by batch and heads.  Only sequence rows [rope_row0, rope_row0 + rope_rows) are
 *          rotated, with table row s - rope_row0 (HunyuanVideo rotates the video tokens and not
 *          the text tokens behind them); products in fp32, result rounded to dtype.
 */
enum xdit_norm_mode { XDIT_NORM_NONE = 0, XDIT_NORM_HEAD = 1, XDIT_NORM_TOKEN = 2 };
enum xdit_rope_mode { XDIT_ROPE_NONE = 0, XDIT_ROPE_INTERLEAVED = 1, XDIT_ROPE_SPLIT_HALF = 2, XDIT_ROPE_WAN = 3 };

typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_prologue_args) */
  int32_t dtype;               /* bf16, fp16 or fp32: x, y and weight */
  int32_t norm;                /* xdit_norm_mode */
  int32_t rope;                /* xdit_rope_mode */
  int32_t B, H, D;
  float eps;
  int64_t S;
  const void* x;
  void* y;
  const void* weight;          /* may be NULL */
  const float* cos;            /* NULL when rope == XDIT_ROPE_NONE */
  const float* sin;
  int64_t rope_stride;
  int64_t rope_row0, rope_rows;
  xdit_strides x_stride, y_stride;
  void* stream;
} xdit_prologue_args;

int xdit_qk_prologue(const xdit_prologue_args* args);

/*
 * `count` (1..8) prologue jobs in ONE launch: the Q, K and V tensors of the text and image streams
 * of an attention block (what transformer_flux.py:116-147 handles with some ten separate torch
 * kernels).  All jobs share dtype and stream; XDIT_NORM_TOKEN jobs cannot be batched.
 */
int xdit_qk_prologue_batch(const xdit_prologue_args* jobs, int32_t count);

/* ---- training ------------------------------------------------------------------------------------ */

/*
 * Backward pass of xdit_attn_fwd: gradients of q, k, v (and of the second segment k2, v2) from those of its results.
 *     P_ij = exp(softmax_scale q_i.k_j - lse_i)          delta_i = dout_i.out_i - dlse_i
 *     dv_j = sum_i P_ij dout_i                            dS_ij = P_ij (dout_i.v_j - delta_i)
 *     dk_j = softmax_scale sum_i dS_ij q_i                dq_i = softmax_scale sum_j dS_ij k_j
 * `out` and `lse` are what the forward call gave for the same q, k, v and scale; `dlse` (may be NULL: zeros) is the gradient of lse.
 * With the out, lse and dout of a whole ring it gives one chunk's dk and dv, and that chunk's share of dq.  A row whose lse is
 * -infinity attended nothing: it gives and gets no gradient, whatever its q, dout and out hold.
 * bf16, fp16 or fp32, head_dim a multiple of 8 up to 128.  P and dS are rounded to dtype for the products, everything else is fp32, each gradient is
 * rounded once.  fp16: scaled by powers of two, dS by one of every query's own for dq and of every key's own for dk, so that neither a large row of dout nor a
 * large value takes bits of other rows; P by 2^15 (a probability below 2^-29 is off by up to 2^-40).  The same call gives the same bits.  dq, or dk and dv (then dk2 and dv2 too where Sk2 > 0), may be NULL: not computed.
 * Gradients must not overlap each other or an input, which is checked (rows that interleave, as those of views of one buffer, are told apart; where
 * strides are such that telling would take thousands of steps the call is refused).
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_attn_bwd_args) */
  int32_t dtype;               /* of every tensor but lse and dlse: bf16, fp16 or fp32 */
  int32_t B, H, D;
  int32_t cu_count;            /* 0 = plan the launch for the compute units of the current device; > 0 = for that many */
  int64_t Sq, Sk, Sk2;
  float softmax_scale;         /* > 0 */
  int32_t reserved0;           /* must be 0 */
  const void* dout;            /* (B,H,Sq,D) */
  const void* q;
  const void* k;               /* (B,H,Sk,D) */
  const void* v;
  const void* k2;              /* (B,H,Sk2,D); may be NULL when Sk2 == 0 */
  const void* v2;
  const void* out;             /* (B,H,Sq,D) */
  const float* lse;            /* (B,H,Sq), any strides, as dlse */
  const float* dlse;           /* (B,H,Sq); may be NULL */
  void* dq;
  void* dk;
  void* dv;
  void* dk2;
  void* dv2;
  xdit_strides dout_stride, q_stride, k_stride, v_stride, k2_stride, v2_stride, out_stride;
  xdit_strides dq_stride, dk_stride, dv_stride, dk2_stride, dv2_stride;
  xdit_strides lse_stride, dlse_stride;
  void* workspace;             /* 16-byte aligned, of the size below, private to the call until its kernels finish */
  int64_t workspace_bytes;
  void* stream;
} xdit_attn_bwd_args;

int xdit_attn_bwd(const xdit_attn_bwd_args* args);
int64_t xdit_attn_bwd_workspace_bytes(const xdit_attn_bwd_args* args);  /* which gradients are asked for counts, no pointer is followed */

/*
 * Norm of a list of gradients, as if they were one vector: the largest size of an element, the sum of sizes or the root of
 * the sum of squares.  Sums are in 64 bits, in a fixed order; the result is rounded to fp32.  An element that is not a number makes the norm one.
 * The tables are HOST arrays of `count` entries; they are read before the call returns.
 */
enum xdit_grad_norm_kind { XDIT_GRADNORM_MAX = 0, XDIT_GRADNORM_L1 = 1, XDIT_GRADNORM_L2 = 2 };

typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_grad_norm_args) */
  int32_t kind;                /* xdit_grad_norm_kind */
  int64_t count;               /* 0: the norm is 0 */
  const void* const* data;     /* device pointers, aligned to their elements; contiguous tensors */
  const int64_t* numel;        /* 0 is allowed */
  const int32_t* dtype;        /* xdit_dtype: bf16, fp16 or fp32, any mixture */
  float* norm;                 /* device: one fp32 */
  void* workspace;             /* 8-byte aligned, of the size below, private to the call until its kernels finish */
  int64_t workspace_bytes;
  void* stream;
  uint32_t* counter;           /* device, 0 before the first call that is given it and left 0 by every one; as private as the workspace.  With it a
                                  list of one dtype and few elements takes one launch, not two.  May be NULL */
} xdit_grad_norm_args;

int xdit_grad_norm(const xdit_grad_norm_args* args);
int64_t xdit_grad_norm_workspace_bytes(const xdit_grad_norm_args* args);  /* from count and numel */

/*
 * Clipping by the gradients' own norm, or by one that is in device memory (e.g. of those of every rank):
 *     dst = src * min(1, max_norm / (norm + 1e-6))
 * in fp32, rounded once.  dst may be src itself; otherwise no dst may overlap another dst, a src or the norm, nor norm_out a src.  Where the factor is 1 a dst
 * that is its src is left as it is.  The tables are HOST arrays, read before the call returns.
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_clip_grads_args) */
  float max_norm;              /* finite, >= 0 */
  int64_t count;
  const void* const* src;
  void* const* dst;
  const int64_t* numel;
  const int32_t* src_dtype;    /* bf16, fp16 or fp32 */
  const int32_t* dst_dtype;
  const float* norm;           /* device: one fp32; NULL: the norm of src, as xdit_grad_norm computes it */
  float* norm_out;             /* device: one fp32, receives the norm where `norm` is NULL */
  int32_t kind;                /* xdit_grad_norm_kind of that norm */
  int32_t reserved0;           /* must be 0 */
  void* workspace;             /* for that norm, of the size that xdit_grad_norm_workspace_bytes gives for src */
  int64_t workspace_bytes;
  void* stream;
} xdit_clip_grads_args;

int xdit_clip_grads(const xdit_clip_grads_args* args);

/* ---- around the attention call: the rest of a DiT block ------------------------------------------ */

/*
 * Norms before and after a block fused with its gate and residual scale.  Rows are (b, s), columns C:
 *     v = y | rms(y) | layer(y), times y_weight                    (y_norm)
 *     h = x + residual_scale * gate * v                            (y == NULL: h = x)
 *     n = (rms(h) | layer(h)) * weight + bias, times (1 + scale), plus shift   (norm)
 * with layer(h) = (h - mean) / sqrt(var + eps) and rms(h) = h / sqrt(mean(h^2) + eps) over C.  What is NULL is
 * left out.  Everything is computed in fp32 from the inputs; h and n are rounded once, n from the unrounded h.
 * A row whose mean square is beyond fp32 (elements of some 2^63 and more) has an infinite deviation: its norm is zero.
 * `fp8 != 0`: n is written as e4m3 bytes with one fp32 scale per block of 128 columns of a row, quantised from the unrounded n
 * as by xdit_fp8_block_quant but with products by reciprocals for its divisions: a scale may differ from that call's by 3 * 2^-24 of
 * itself, and a value whose quotient is within 7 * 2^-24 of the middle of two e4m3 numbers may become the other one.  What
 * xdit_fp8_block_matmul takes where C is a multiple of 16.  n_scale[kb * B*S + b*S + s] holds the scale of columns
 * [128 kb, 128 kb + 128).  `stats` (optional) receives (mean, 1/deviation) of h and of y, four floats a row
 * (0 and 1 for a norm that is absent; an RMS norm's mean is 0): what the backward call reads.
 * gate, scale and shift are (B, 1 or S, C): s stride 0 for one row per batch entry.  C: a multiple of 8, at most 8192.
 * h may be NULL (not wanted) and may be x or y themselves; n may be x or y.  norm == XDIT_ROWNORM_NONE: n is not written.
 * Replaces: the AdaLayerNormZero modulation, the gated residual addition and the sandwich norms that diffusers'
 * transformer blocks run around the processors of xfuser/model_executor/models/transformers/ as separate kernels.
 */
enum xdit_rownorm { XDIT_ROWNORM_NONE = 0, XDIT_ROWNORM_RMS = 1, XDIT_ROWNORM_LAYER = 2 };

typedef struct {
  int64_t b, s;                /* element strides of a (B, S, C) tensor; the C stride is 1 */
} xdit_row_strides;

typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_gated_norm_args) */
  int32_t dtype;               /* x, y, h, n: bf16, fp16 or fp32 */
  int32_t mod_dtype;           /* gate, scale, shift: dtype or fp32 */
  int32_t weight_dtype;        /* weight, bias, y_weight: dtype or fp32 */
  int32_t norm, y_norm;        /* xdit_rownorm */
  int32_t fp8;
  int32_t B, C;
  float eps, y_eps, residual_scale;
  int64_t S;
  const void* x;
  const void* y;               /* may be NULL */
  void* h;                     /* may be NULL */
  void* n;
  float* n_scale;              /* fp8 only */
  float* stats;                /* (B,S,4) contiguous, may be NULL */
  const void* gate;            /* each may be NULL */
  const void* scale;
  const void* shift;
  const void* weight;
  const void* bias;
  const void* y_weight;
  xdit_row_strides x_stride, y_stride, h_stride, n_stride, gate_stride, scale_stride, shift_stride;
  void* stream;
} xdit_gated_norm_args;

int xdit_gated_norm(const xdit_gated_norm_args* args);

/*
 * Gradients of xdit_gated_norm from dh and dn (either may be NULL), the h, y and stats of the forward call and its
 * parameters.  dx is the gradient of x (and the running gradient of the residual stream).  dgate / dscale / dshift have the
 * forms of gate / scale / shift (contiguous, one row per batch entry or per token; scale and shift must agree in that),
 * dweight, dbias and dy_weight have C entries; each output may be NULL.  Column sums are taken in fp32 in a fixed order.
 * `workspace`: xdit_gated_norm_backward_workspace_bytes(args) bytes, 16-byte aligned, private to the stream until the
 * call's kernels finish (0 bytes where no column sum is asked for).
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_gated_norm_backward_args) */
  int32_t dtype, mod_dtype, weight_dtype;
  int32_t norm, y_norm;
  int32_t gate_per_token, mod_per_token;   /* != 0: gate (scale and shift) have a row per token */
  int32_t B, C;
  float residual_scale;
  int32_t reserved0;
  int64_t S;
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
  xdit_row_strides dh_stride, dn_stride, h_stride, y_stride, gate_stride, scale_stride, dx_stride, dy_stride;
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} xdit_gated_norm_backward_args;

int64_t xdit_gated_norm_backward_workspace_bytes(const xdit_gated_norm_backward_args* args);
int xdit_gated_norm_backward(const xdit_gated_norm_backward_args* args);

/*
 * Rotary positions on several axes (time, height, width, ...) for q and k in one launch, after an optional RMSNorm over
 * head_dim.  Pair p of the P = pairs[0] + pairs[1] + ... rotated pairs belongs to the axis whose range of `pairs` it lies in:
 *     phi = positions[b, s, axis(p)] * inv_freq[p]
 *     (y1, y2) = (x1 cos phi - x2 sin phi, x1 sin phi + x2 cos phi)
 * with the pair's elements 2p and 2p + 1 (XDIT_ROPE_INTERLEAVED) or p and p + P (XDIT_ROPE_SPLIT_HALF); columns from 2P on
 * are not rotated.  norm != 0: x is first divided by sqrt(mean(x^2) + eps) over head_dim and multiplied by `weight`.
 * Angles are reduced in fp64, everything else is fp32, the result is rounded once.  No tables: a token's sines and cosines
 * are computed once for all of its heads.  head_dim: a multiple of 8 up to 512; P a multiple of 4 (0: the norm alone).
 * Replaces: the position embedding modules that build (cos, sin) tables and the rotation of the processors
 * (transformer_flux.py:146-147, transformer_hunyuan_video.py:60-83, transformer_wan.py:108-120).
 *
 * xdit_axes_rope_backward: dy is the gradient of the rotated tensor, y receives that of x; x (the forward call's
 * input) is read only where norm != 0.  `dweight` (norm != 0; D entries, may be NULL) receives the sum over rows, taken in
 * fp32 in a fixed order through `workspace` (xdit_axes_rope_backward_workspace_bytes, 16-byte aligned, private to the
 * stream until the call's kernels finish).
 */
#define XDIT_ROPE_MAX_AXES 4

typedef struct {
  const void* x;               /* (B,H,S,D) */
  const void* dy;              /* backward only */
  void* y;                     /* may be x (forward) or dy (backward) with the same strides */
  const void* weight;          /* may be NULL */
  void* dweight;               /* backward only, may be NULL */
  xdit_strides x_stride, dy_stride, y_stride;
  int32_t H, reserved0;
} xdit_axes_rope_tensor;

typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_axes_rope_args) */
  int32_t dtype;               /* bf16, fp16 or fp32 */
  int32_t weight_dtype;        /* weight, dweight: dtype or fp32 */
  int32_t rope;                /* XDIT_ROPE_INTERLEAVED or XDIT_ROPE_SPLIT_HALF */
  int32_t norm;
  int32_t pos_bits;            /* positions: -32 fp32, 32 int32, 64 int64 */
  int32_t freq_bits;           /* inv_freq: 32 fp32, 64 fp64 */
  int32_t B, D;
  int32_t tensors;             /* 1 or 2 of `t` are there */
  int32_t axes;
  int32_t pairs[XDIT_ROPE_MAX_AXES];
  float eps;
  int64_t S;
  const void* positions;       /* (B, S, axes), axis stride 1 */
  int64_t pos_stride_b, pos_stride_s;
  const void* inv_freq;        /* P entries, radians per unit of position */
  xdit_axes_rope_tensor t[2];  /* q and k */
  void* workspace;             /* backward only */
  int64_t workspace_bytes;
  void* stream;
} xdit_axes_rope_args;

int xdit_axes_rope(const xdit_axes_rope_args* args);
int64_t xdit_axes_rope_backward_workspace_bytes(const xdit_axes_rope_args* args);
int xdit_axes_rope_backward(const xdit_axes_rope_args* args);

/*
 * fp8 (e4m3) quantiser with an fp32 scale per block of 1 x 128 (block_rows 1: activations) or 128 x 128 elements (block_rows
 * 128: weights), the blocks at the end cut off by the tensor:
 *     scale = absmax / 448, at least 2^-126, 1 for a block of zeros ;  y = e4m3(x / scale)
 * y has the bytes of a true fp32 division.  A block that holds a NaN is NaN, one with an infinity has an infinite scale.
 * scale: block_rows 1: scale[kb * B*S + b*S + s]; 128 (B must be 1): scale[(s / 128) * ceil(K / 128) + kb].
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_block_quant_args) */
  int32_t dtype;               /* x: bf16, fp16 or fp32 */
  int32_t block_rows;          /* 1 or 128 */
  int32_t B;
  int64_t S, K;                /* x is (B, S, K); K a multiple of 8 */
  const void* x;
  void* y;                     /* (B, S, K) e4m3 bytes */
  float* scale;
  xdit_row_strides x_stride, y_stride;
  void* stream;
} xdit_block_quant_args;

int xdit_fp8_block_quant(const xdit_block_quant_args* args);

/*
 * Product of block-scaled fp8 (e4m3) matrices, out = x w^T + bias:
 *     out[m, n] = sum_kb x_scale[m, kb] w_scale[n / 128, kb] sum_{k in block kb} x[m, k] w[n, k]  + bias[n]
 * x (M, K) with a scale per 1 x 128 block, w (N, K) with one per 128 x 128 block (what xdit_fp8_block_quant makes), K a
 * multiple of 16, rows 16-byte aligned.  The scaled sums of the blocks are held in fp32 and the result is rounded once to
 * out_dtype.  Within a block, exact_sums != 0: products are exact and summed in fp32 (the operands are widened to fp16 on their
 * way into the matrix cores); 0: the fp8 matrix instructions, twice as fast, which add eight consecutive k at a time and cut
 * every product of those at 2^-13 of the largest one's binade (an error of 1.4e-5 to 3.3e-5 of the result's size: beside a rounding to
 * bf16 nothing, beside one to fp16 0.2 to 1.2 % more).  `workspace` (optional, xdit_fp8_block_matmul_workspace_bytes, 16-byte
 * aligned, private to the stream until the call's kernels finish) lets a product of few rows cut K over the chip; without it
 * K is not cut.  Results are reproducible bit for bit for the same arguments and workspace.
 */
typedef struct {
  uint32_t struct_size;        /* = sizeof(xdit_block_matmul_args) */
  int32_t out_dtype;           /* bf16, fp16 or fp32 */
  int32_t bias_dtype;          /* out_dtype or fp32 */
  int32_t cu_count;            /* 0 = plan for the compute units of the current device; > 0 = for that many (tests, tuning) */
  int32_t exact_sums;
  int32_t reserved0;
  int64_t M, N, K;
  const void* x;
  const float* x_scale;
  const void* w;
  const float* w_scale;
  const void* bias;            /* N entries, may be NULL */
  void* out;                   /* (M, N) */
  int64_t x_stride, w_stride, out_stride;       /* elements from row to row */
  int64_t x_scale_stride_m, x_scale_stride_k;   /* of (M, ceil(K / 128)) */
  int64_t w_scale_stride_n, w_scale_stride_k;   /* of (ceil(N / 128), ceil(K / 128)) */
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} xdit_block_matmul_args;

int64_t xdit_fp8_block_matmul_workspace_bytes(const xdit_block_matmul_args* args);
int xdit_fp8_block_matmul(const xdit_block_matmul_args* args);

/*
 * Number of the capture that `stream` is under, 0 if it is under none.  A captured call keeps the address of its workspace,
 * and its graph may be replayed on any stream: give the calls of one capture a workspace that no eager call and no other
 * capture is given, with `workspace_preserved` 0 on the first of them.
 */
uint64_t xdit_stream_capture_id(void* stream);

/* Message of the last error on the calling thread ("" if none). Never NULL. */
const char* xdit_attn_last_error(void);

/* XDIT_ATTN_ABI_VERSION the library was built with. */
int xdit_attn_abi_version(void);

#ifdef __cplusplus
}
#endif
#endif /* XDIT_AMD_ATTN_H */
