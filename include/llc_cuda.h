/* C ABI of the sm_100a kernel library ("ops/cuda", the sibling of the reference's empty
 * ops/cpu/ops.h).  One entry point per kernel family; each is the CUDA replacement for
 * the code the reference generates for the named LLH ops.  Pointers are device pointers,
 * extents and strides are in elements, `stream` is a cudaStream_t (NULL = legacy default
 * stream).  Every function returns 0 or an LlcStatus (llc_runtime.h) and records a message
 * readable with llc_last_error().  Nothing here allocates device memory.
 */
#ifndef LLC_CUDA_H_
#define LLC_CUDA_H_

#include <stdint.h>

#include "llc_runtime.h"

#ifdef __cplusplus
extern "C" {
#endif

typedef enum LlcAct { LLC_ACT_NONE = 0, LLC_ACT_RELU = 1, LLC_ACT_GELU = 2 } LlcAct;
typedef enum LlcPrecision { LLC_PREC_FP32 = 0, LLC_PREC_TF32 = 1, LLC_PREC_TF32X3 = 2, LLC_PREC_BF16 = 3 } LlcPrecision;

/* out[b0,b1,m,n] = act(alpha * scale[n] * sum_k A[b0,b1,m,k] * B[b0,b1,k,n] + shift[n] + res[b0,b1,m,n])
 * Replaces llh.matmul / llh.batch_matmul (-> stablehlo.dot / dot_general,
 * src/Conversion/LLHToHLO/LLHToHLO.cpp:363-382, :485) together with the elementwise ops that
 * follow it in the graph (bias add, ReLU = max(x,0) LLHPreprocessingForHLO.cpp:76-101, residual).
 * A must have unit stride along k.  B has unit stride along k (b_sk == 1, weights stored [n][k])
 * or along n (b_sn == 1).  scale/shift/res may be NULL.  Accumulation is fp32. */
typedef struct LlcGemmParams {
  const void* a; const void* b; void* out;
  const float* scale; const float* shift; const void* res;
  int32_t in_dtype;    /* LLC_FLOAT32 or LLC_BFLOAT16, both operands */
  int32_t out_dtype;   /* LLC_FLOAT32 or LLC_BFLOAT16 */
  int32_t res_dtype;
  int32_t precision;   /* LlcPrecision; LLC_PREC_FP32 = FMA path */
  int64_t m, n, k, b0, b1;
  int64_t a_s0, a_s1, a_sm;            /* strides of A: batch0, batch1, row (k stride is 1) */
  int64_t b_s0, b_s1, b_sk, b_sn;
  int64_t o_s0, o_s1, o_sm;            /* n stride is 1 */
  int64_t r_s0, r_s1, r_sm, r_sn;
  float alpha;
  int32_t act;         /* LlcAct */
  /* Optional scratch for K slices (few output tiles, long K): device memory, 16-byte
   * aligned, whose first 4096 bytes are zero before the first use (the kernel leaves them zero).
   * NULL disables them.  Launches that share one workspace must not overlap on the GPU. */
  void* workspace;
  int64_t workspace_bytes;
  /* Optional, precision tf32x3 only: B - truncate_to_tf32(B), laid out exactly like b (same strides).  When given, the
   * kernel loads it instead of splitting every B tile itself; weights are split once at load time this way. */
  const void* b_lo;
} LlcGemmParams;
int llc_cuda_gemm(const LlcGemmParams* p, void* stream);

/* llc_cuda_gemm on the FMA path for callers that must not allocate device memory (a process whose
 * own pool already owns the GPU, a loop that cannot take the synchronisation an allocation
 * implies).  No counterpart in the reference.  The split-K scratch is a 1 MiB array built into the
 * library (each GPU that loads the library holds it until exit); `workspace` in the parameter block
 * is ignored.  A shape whose split needs more than 1 MiB is refused with LLC_ERR_ARGUMENT.  The
 * first call on a device looks up the array's device address (cudaGetSymbolAddress); make that
 * first call before starting any stream capture.  All calls share the one array: launches that
 * overlap on the GPU (different streams or threads of one process on one device) race.
 * Calls no cudaMalloc / cudaFree. */
int llc_cuda_gemm_static_scratch(const LlcGemmParams* p, void* stream);

/* out[b0,b1,m,:] = softmax_n(scale * sum_d Q[b0,b1,m,d] K[b0,b1,n,d] + mask[b0,b1,m,n]) V[b0,b1,n,:] in one kernel: the
 * scores stay in tensor memory, the probabilities in shared memory (keys in blocks of 128, running softmax).  Replaces the chain llh.batch_matmul -> llh.div /
 * llh.add (scale, mask) -> softmax (decomposed by llcompiler/compiler/torch_compile_config.py:24) -> llh.batch_matmul that
 * the reference lowers op by op (src/Conversion/LLHToHLO/LLHToHLO.cpp:363-382).  bf16 operands and output with unit
 * stride along d, d == 64, 1 <= n <= 512; every other stride a non-negative multiple of 8 elements (0 = broadcast for
 * batch strides), pointers 16-byte aligned.  mask may be NULL; it has unit stride along n and may broadcast over
 * b0, b1 and m (stride 0).  Anything else returns LLC_ERR_UNSUPPORTED. */
typedef struct LlcAttentionParams {
  const void* q; const void* k; const void* v; const void* mask; void* out;
  int32_t dtype;        /* LLC_BFLOAT16 */
  int32_t mask_dtype;   /* LLC_FLOAT32 or LLC_BFLOAT16 */
  int64_t b0, b1, m, n, d;
  int64_t q_s0, q_s1, q_sm;
  int64_t k_s0, k_s1, k_sn;
  int64_t v_s0, v_s1, v_sn;
  int64_t o_s0, o_s1, o_sm;
  int64_t mask_s0, mask_s1, mask_sm;
  float scale;
} LlcAttentionParams;
int llc_cuda_attention(const LlcAttentionParams* p, void* stream);

/* Health word of the tensor-core kernels.  Their waits on memory barriers are bounded; a wait that
 * gives up records 1 (producer), 2 (issuer), 3 (operand split), 4 (epilogue), 5 (gather), 6 or 7 (attention), 8 to 12 (paged attention) and the launch's
 * result is then invalid.  Returns the recorded code (0 = healthy) and clears it; -1 if the device
 * cannot be read.  Synchronises the device.  No counterpart in the reference. */
int llc_cuda_status(void);

/* NHWC implicit-GEMM convolution with the same epilogue; replaces llh.conv
 * (-> stablehlo.convolution, LLHToHLO.cpp:214-270), the decomposed batch-norm inference that
 * follows it (src/Dialect/LLH/Transforms/DecomposeOps.cpp:125-144, folded to scale/shift),
 * the residual add and the ReLU.  x is [N,H,W,C], w is [F,KH,KW,C], out and res are [N,OH,OW,F]. */
typedef struct LlcConvParams {
  const void* x; const void* w; void* out;
  const float* scale; const float* shift; const void* res;
  int32_t in_dtype, out_dtype, res_dtype, precision;
  int64_t n, h, w_in, c, f, kh, kw, oh, ow;
  int32_t stride_h, stride_w, pad_h, pad_w, dil_h, dil_w;
  float alpha;
  int32_t act;
  const void* w_lo;   /* optional, precision tf32x3: w - truncate_to_tf32(w), same layout as w (see LlcGemmParams.b_lo) */
  /* Optional element strides of x along n, h and w (the channel stride is 1); all 0 = dense [N,H,W,C].  The strides may
   * describe an overlapping view: with x_sw < c every "pixel" is a window of c consecutive elements that advances by x_sw,
   * which turns a filter row of a narrow-channel convolution into the channels of a 1-wide kernel.  Tensor-core precisions
   * only (bf16, tf32, tf32x3); c * element size must then be a multiple of 16 bytes and so must the strides. */
  int64_t x_sn, x_sh, x_sw;
  /* Optional scratch for K slices (few output tiles, long K), as in LlcGemmParams: device memory, 16-byte aligned, first
   * 4096 bytes zero before the first use (left zero).  NULL disables them. */
  void* workspace;
  int64_t workspace_bytes;
} LlcConvParams;
int llc_cuda_conv2d(const LlcConvParams* p, void* stream);

/* NHWC max pooling; replaces llh.max_pool (-> stablehlo.reduce_window, LLHToHLO.cpp:295-339).
 * Padding taps are skipped (equivalent to a -inf initial value; the reference initialises
 * with 0, :313-314). */
typedef struct LlcPoolParams {
  const void* x; void* out;
  int32_t in_dtype, out_dtype;
  int64_t n, h, w, c, oh, ow;
  int32_t kh, kw, stride_h, stride_w, pad_h, pad_w, dil_h, dil_w;
} LlcPoolParams;
int llc_cuda_maxpool2d(const LlcPoolParams* p, void* stream);

/* out[o,i] = reduce_r x[o,r,i]; x dense [outer,R,inner].  op: 0 sum, 1 max, 2 min, 3 mean.
 * Replaces llh.reduce_sum/max/min (-> stablehlo.reduce, LLHToHLO.cpp:81-171) and the global
 * average pool (llh.adaptive_average_pool, declared without a lowering, LLHOps.td:337-339). */
int llc_cuda_reduce(const void* x, void* out, int32_t in_dtype, int32_t out_dtype, int64_t outer,
                    int64_t r, int64_t inner, int32_t op, void* stream);

/* Row softmax over dense [rows, len]; replaces the amax/sub/exp/sum/div chain of the
 * reference's decomposition (llcompiler/compiler/torch_compile_config.py:24). */
int llc_cuda_softmax(const void* x, void* out, int32_t in_dtype, int32_t out_dtype, int64_t rows,
                     int64_t len, void* stream);

/* Row LayerNorm over dense [rows, d] with fp32 statistics; llh.layer_norm is declared by the
 * reference (LLHOps.td:454-463) without a lowering. */
int llc_cuda_layernorm(const void* x, const void* gamma, const void* beta, void* out, int32_t in_dtype,
                       int32_t param_dtype, int32_t out_dtype, int64_t rows, int64_t d, float eps, void* stream);

/* out[r,:] = table[ids[r],:]; ids are int64.  Rows with an id outside [0, vocab) are written
 * as zeros and counted in *bad_ids when bad_ids is not NULL (a device int32). */
int llc_cuda_gather(const void* table, const int64_t* ids, void* out, int32_t table_dtype, int32_t out_dtype,
                    int64_t rows, int64_t d, int64_t vocab, int32_t* bad_ids, void* stream);

/* out[r,:] = LayerNorm(table[ids[r],:] + add[(r / period) * add_s0 + (r % period) * add_s1 + (0..d-1)]) * gamma + beta in one
 * pass: llc_cuda_gather, the elementwise add (rounded to the storage type, as that step stores it) and llc_cuda_layernorm
 * where nothing else reads what is between them.  All tensors of one type, f32 or bf16.  add may be NULL.  Rows with an id outside [0, vocab) use zeros for the
 * table row and are counted in *bad_ids when it is not NULL. */
typedef struct LlcEmbedNormParams {
  const void* table; const int64_t* ids; const void* add; const void* gamma; const void* beta; void* out;
  int32_t dtype;
  int64_t rows, d, vocab, period, add_s0, add_s1;
  float eps;
  int32_t* bad_ids;
} LlcEmbedNormParams;
int llc_cuda_embed_norm(const LlcEmbedNormParams* p, void* stream);

/* Rotary positions: out[t,h,:] is x[t,h,:] with `pairs` pairs of its elements turned, pair i by the angle
 * a = positions[axis(i)][t] * inv_freq[i]:  (x, y) -> (x cos a - y sin a, x sin a + y cos a).  Pair i is elements
 * (i, i + pairs), or (2 i, 2 i + 1) when interleaved; elements from 2 * pairs on are copied.  The pairs are dealt out to the
 * axes in order, sections[0] to axis 0 and so on (time, height and width of a video, say); the sections add up to pairs.
 * Angles are computed in 64 bits, the turn in 32, one rounding at the store.  x and out have unit stride along d; out may
 * be x itself (same address, same strides), any other overlap is the caller's error.  No counterpart in the reference. */
#define LLC_ROTARY_MAX_AXES 4
typedef struct LlcRotaryParams {
  const void* x; void* out;
  const void* positions;       /* [axes, tokens], unit stride along tokens */
  const double* inv_freq;      /* [pairs] */
  int32_t dtype;               /* LLC_FLOAT32, LLC_BFLOAT16 or LLC_FLOAT16 */
  int32_t pos_dtype;           /* LLC_INT32 or LLC_INT64 */
  int64_t tokens, heads, d, pairs;
  int64_t x_st, x_sh, o_st, o_sh;   /* strides of a token and of a head */
  int64_t pos_sa;                   /* stride of an axis of positions */
  int32_t axes;                     /* 1 to LLC_ROTARY_MAX_AXES */
  int32_t interleaved;
  int32_t sections[LLC_ROTARY_MAX_AXES];
} LlcRotaryParams;
int llc_cuda_rotary(const LlcRotaryParams* p, void* stream);

/* ---- Paged key / value cache ----------------------------------------------------------------------------------------
 * A cache is a pool of pages of page_size token slots, k_cache and v_cache of logical shape
 * [num_pages, page_size, kv_heads, d] with any strides along the first three dims.  A batch of sequences is described by
 * three int32 arrays on the device, so that a captured graph can be replayed with other lengths:
 *   page_table [batch, table_width]  slot j of sequence b is slot j % page_size of page page_table[b][j / page_size]
 *   q_start    [batch + 1]           rows q_start[b] .. q_start[b+1]-1 of q, k and v are sequence b's new tokens
 *   kv_len     [batch]               tokens of sequence b in the cache, its new ones included: the i-th of n new tokens
 *                                    has place kv_len[b] - n + i
 * Rows from q_start[batch] on belong to nobody and are left as they were.  A length beyond the table's reach counts as the
 * reach, a negative one as 0.  Page numbers outside [0, num_pages) are never followed.
 *
 * llc_cuda_kv_append writes the new tokens' keys and values into their slots, the keys turned by their rotary angles when
 * inv_freq is not NULL, and writes the queries, turned the same way, to q_out when q is not NULL.  positions NULL: every
 * axis is the token's place.  A token whose page number is outside [0, num_pages) or whose place is outside the table
 * (or negative) is not stored and is counted in *bad_pages when that is not NULL (a device int32); its query is turned
 * all the same.  Two tokens of a call must not have the same slot.  No counterpart in the reference. */
typedef struct LlcKvAppendParams {
  const void* k; const void* v; void* k_cache; void* v_cache;
  const void* q; void* q_out;          /* optional */
  const int32_t* page_table; const int32_t* q_start; const int32_t* kv_len;
  const void* positions;               /* optional: [axes, tokens], unit stride along tokens */
  const double* inv_freq;              /* optional: [pairs] */
  int32_t* bad_pages;                  /* optional */
  int32_t dtype;                       /* all tensors: LLC_FLOAT32, LLC_BFLOAT16 or LLC_FLOAT16 */
  int32_t pos_dtype;                   /* LLC_INT32 or LLC_INT64 */
  int64_t tokens, batch, heads, kv_heads, d, pairs;
  int64_t num_pages, page_size, table_width, table_s0;
  int64_t q_st, q_sh, qo_st, qo_sh, k_st, k_sh, v_st, v_sh;
  int64_t kc_sp, kc_sn, kc_sh, vc_sp, vc_sn, vc_sh;   /* strides of a page, a slot and a head */
  int64_t pos_sa;
  int32_t axes, interleaved;
  int32_t sections[LLC_ROTARY_MAX_AXES];
} LlcKvAppendParams;
int llc_cuda_kv_append(const LlcKvAppendParams* p, void* stream);

/* out[t,h,:] = sum_j w_j v_j, w = softmax over the visible j of scale * q[t,h,:] . k_j, for the new tokens t of a ragged
 * batch over a paged cache that holds their keys and values already (llc_cuda_kv_append); query head h reads key head
 * h / (heads / kv_heads).  A token at place p sees the keys j <= p; with window > 0 only those with p - j < window, and the
 * first `sinks` keys of the sequence besides.  A token that sees nothing (kv_len smaller than its place asks for) gets zeros; one
 * whose visible scores are all -inf gets NaN, which is what softmax makes of them.  A visible value that is infinite makes its element of the
 * result infinite, or NaN where its weight is too small for the type it is held in (below about 2^-31 of the largest in f16, 2^-126 otherwise).
 * A slot whose page number is outside [0, num_pages) reads as zeros (key and value) and each such page that a query sees is
 * counted in *bad_pages (at least once, or more often) when that is not NULL.  Nothing else of the cache is read into the
 * result: slots past kv_len, pages before the window and unused pages may hold anything.
 * out may be q itself (same address, same strides).
 * max_q: at least the largest number of new tokens of a sequence; a sequence that has more is left out.
 * f32, bf16 and f16, all tensors alike, unit stride along d, d <= 256.  bf16 and f16 with d 64 or 128, page_size a power of
 * two >= 16, strides of 16 bytes' multiples and 16-byte aligned pointers run on the tensor cores, everything else
 * (f32, other head sizes, pages and strides) on a kernel of plain multiply-adds.
 * workspace: scratch for joining sums over parts of the keys, llc_cuda_paged_attention_workspace bytes, 16-byte aligned,
 * contents arbitrary; NULL (or too small) disables the split.  Launches that share one must not overlap on the GPU. */
typedef struct LlcPagedAttentionParams {
  const void* q; const void* k_cache; const void* v_cache; void* out;
  const int32_t* page_table; const int32_t* q_start; const int32_t* kv_len;
  int32_t* bad_pages;                  /* optional */
  int32_t dtype;
  float scale;
  int64_t tokens, batch, heads, kv_heads, d, max_q;
  int64_t num_pages, page_size, table_width, table_s0;
  int64_t q_st, q_sh, o_st, o_sh;
  int64_t kc_sp, kc_sn, kc_sh, vc_sp, vc_sn, vc_sh;
  int64_t window, sinks;               /* window 0: every earlier key is visible */
  void* workspace; int64_t workspace_bytes;
} LlcPagedAttentionParams;
int llc_cuda_paged_attention(const LlcPagedAttentionParams* p, void* stream);
/* Bytes of workspace that the call can use (it depends on shapes and types alone); 0 when it uses none. */
int64_t llc_cuda_paged_attention_workspace(const LlcPagedAttentionParams* p);

/* x [n, c, hw] (NCHW planes) -> out [n, hw, c_pad] (NHWC pixels), channels c..c_pad-1 written as
 * zeros.  The layout change the reference expresses as llh.transpose perms [0,2,3,1] around conv
 * (src/Dialect/LLH/Transforms/TransformLayout.cpp:141-198), with the channel padding the
 * tensor-core convolution wants for a 3-channel stem. */
int llc_cuda_nchw_to_nhwc(const void* x, void* out, int32_t dtype, int64_t n, int64_t c, int64_t hw, int64_t c_pad, void* stream);

/* The same re-layout into rows of w_total pixels: the image starts at column w_left, the columns left and right of it are
 * zeros.  out is [n, h, w_total, c_pad]; f32 with c_pad 4 or bf16 with c_pad 8 (16 bytes per pixel).  With the halo in
 * memory, eight neighbouring pixels of a narrow-channel input are one contiguous 128-byte run, which is what lets the stem
 * convolution read a whole filter row per K block (see LlcConvParams.x_sw). */
int llc_cuda_nchw_to_nhwc_wide(const void* x, void* out, int32_t dtype, int64_t n, int64_t c, int64_t h, int64_t w, int64_t c_pad, int64_t w_left,
                               int64_t w_total, void* stream);

/* Multi-destination copy: `bytes` bytes at `src` are stored at byte offset `dst_offset_bytes` of each of the `n_dst`
 * (at most 8) buffers in `dst` (a host array of device pointers); each source vector is read once.  The destinations may
 * be peer memory of other GPUs (plain stores over NVLink): this is the gather step of batch-sharded inference, every rank
 * pushing its slice of the output into every rank's copy of the full batch; the caller synchronises the ranks before
 * (the destinations are free) and after (every slice has arrived).  No counterpart in the reference, which runs on one
 * device; it stands where its Execution::run results (src/Compiler/Execution.cpp:21-66) of several GPUs are put together. */
int llc_cuda_push_rows(const void* src, void* const* dst, int32_t n_dst, int64_t dst_offset_bytes, int64_t bytes, void* stream);

/* Fused elementwise chain: one coalesced pass that evaluates a small register program per
 * output element.  Replaces chains of llh.add/sub/mul/div/max/min/abs/sqrt/exp/where/compare/
 * convert_to/broadcast_to (-> stablehlo elementwise ops, LLHToHLO.cpp:479-490) and strided
 * copies (llh.transpose -> stablehlo.transpose).  `prog` is ';'-separated instructions, the
 * i-th defines register i: "ld<k>" loads input k, "#<v>" is a constant, "<op>,<a>[,<b>[,<c>]]"
 * applies an op to earlier registers.  All arithmetic is fp32.  Up to 8 inputs, rank <= 6. */
typedef struct LlcEltwiseOperand { const void* data; int32_t dtype; int64_t strides[6]; } LlcEltwiseOperand;
typedef struct LlcEltwiseParams {
  void* out; int32_t out_dtype; int32_t rank;
  int64_t shape[6]; int64_t out_strides[6];
  int32_t n_in; LlcEltwiseOperand in[8];
  const char* prog;
} LlcEltwiseParams;
int llc_cuda_eltwise(const LlcEltwiseParams* p, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* LLC_CUDA_H_ */
