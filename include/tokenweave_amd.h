/*
 * tokenweave_amd — C ABI of the MI355X (gfx950) fused
 * P-partial reduce + residual-add + RMSNorm path.
 *
 * One rank, one GPU.  Every pointer is a DEVICE pointer to row-major,
 * row-contiguous memory ([num_tokens, hidden_size], element stride 1, row
 * stride hidden_size) unless stated otherwise.  Every call only ENQUEUES work
 * on `stream` (a hipStream_t; NULL = the default stream) of the device that is
 * current on the calling thread: no allocation, no host synchronisation, safe
 * under stream capture.  Return value: TW_OK, or a negative TW_ERR_* code with
 * a message retrievable from tw_last_error() on the same thread.  Nothing
 * throws across this boundary.
 *
 * Arithmetic (identical for every entry point; the reference's CPU path,
 * csrc/cpu/layernorm.cpp:44-88, with round-to-nearest-even stores):
 *   S   = sum_{p=0}^{P-1} f32(partial_p)        fp32, fixed order p = 0..P-1
 *   s   = S + f32(residual)                      fp32
 *   r'  = bf16_rne(s)                            -> residual (in place)
 *   inv = 1 / sqrt( sum_j s_j^2 / H + eps )      fp32, unrounded s
 *   y   = bf16_rne( f32(r') * inv * f32(w) )     -> output
 * Row results do not depend on num_tokens, on max_ctas or on which other rows
 * are in the call.
 */
#ifndef TOKENWEAVE_AMD_H
#define TOKENWEAVE_AMD_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Exported from the shared library.  (A build that compiles the sources into another
 * library may define TW_API beforehand to keep these names out of its own exports.) */
#ifndef TW_API
#define TW_API __attribute__((visibility("default")))
#endif

#define TW_OK 0
#define TW_ERR_INVALID_ARGUMENT (-1) /* null pointer, negative size, bad P / rank */
#define TW_ERR_ALIGNMENT (-2)        /* 16-byte alignment or H % 8 violated      */
#define TW_ERR_DTYPE (-3)            /* dtype not supported by this entry point   */
#define TW_ERR_LAUNCH (-4)           /* the HIP runtime refused the launch        */

/* Element types of the baseline ops (the reference dispatches them with
 * VLLM_DISPATCH_FLOATING_TYPES, csrc/dispatch_utils.h:14-21).  The *_cta and
 * reduce entry points are bf16 only, like the reference's
 * VLLM_BF16_DISPATCH_FLOATING_TYPES (csrc/dispatch_utils.h:23-27). */
#define TW_DTYPE_BF16 0
#define TW_DTYPE_F16 1
#define TW_DTYPE_F32 2

/* Output kinds of the dynamic per-token quantisation ops. */
#define TW_QUANT_FP8_E4M3FN 0
#define TW_QUANT_INT8 1

#define TW_MAX_PARTIALS 16

/* Library version (major*10000 + minor*100 + patch). */
TW_API int tw_version(void);

/* Message for the last non-TW_OK return on this thread ("" if none). */
TW_API const char* tw_last_error(void);

/* Number of compute units of the current device (<0 on error). */
TW_API int tw_num_compute_units(void);

/* input <- RMSNorm(input + residual) * weight ; residual <- input + residual.
 * Replaces ::fused_add_rms_norm (csrc/layernorm_kernels.cu:194-231, schema at
 * csrc/torch_bindings.cpp:141-144; CPU twin csrc/cpu/layernorm.cpp:105-117).
 * Any hidden_size and alignment are accepted: rows that are not 16-byte
 * aligned or hidden_size % 8 != 0 take an element-wise kernel, as the
 * reference's launcher does (layernorm_kernels.cu:223-230). */
TW_API int tw_fused_add_rms_norm(void* input, void* residual, const void* weight,
                          int64_t num_tokens, int64_t hidden_size,
                          float epsilon, int dtype, void* stream);

/* out <- RMSNorm(input) * weight.
 * Replaces ::rms_norm (csrc/layernorm_kernels.cu:165-181, schema at
 * csrc/torch_bindings.cpp:135-138; CPU twin csrc/cpu/layernorm.cpp:91-103). */
TW_API int tw_rms_norm(void* out, const void* input, const void* weight,
                int64_t num_tokens, int64_t hidden_size, float epsilon,
                int dtype, void* stream);

/* out <- input (the copy becomes the residual stream) ;
 * input <- RMSNorm(input) * weight.
 * Replaces ::rms_norm_inplace (csrc/tokenweave_fused_kernels.cu:186-202,
 * schema at csrc/torch_bindings.cpp:147-150). */
TW_API int tw_rms_norm_inplace(void* out, void* input, const void* weight,
                        int64_t num_tokens, int64_t hidden_size, float epsilon,
                        int dtype, void* stream);

/* tw_fused_add_rms_norm on a grid capped at max_ctas workgroups that walk the
 * rows with stride max_ctas (max_ctas <= 0: library default).  bf16 only;
 * pointers must be 16-byte aligned and hidden_size % 8 == 0, else
 * TW_ERR_ALIGNMENT.
 * Replaces ::fused_add_rms_norm_cta (csrc/tokenweave_artifact_kernels.cu:
 * 717-754, schema at csrc/torch_bindings.cpp:160-164). */
TW_API int tw_fused_add_rms_norm_cta(void* input, void* residual, const void* weight,
                              int64_t num_tokens, int64_t hidden_size,
                              int max_ctas, float epsilon, void* stream);

/* The fused op restricted to one GPU, general form.
 *   partials : HOST array of P device pointers, each [num_tokens, hidden_size]
 *              bf16 (this rank's row shard of every tensor-parallel partial sum)
 *   y        : [num_tokens, hidden_size] bf16 output; may alias any partials[p]
 *   residual : read and overwritten with r'
 * 1 <= P <= TW_MAX_PARTIALS.  bf16; 16-byte alignment and H % 8 == 0 required.
 * This is the body of fused_rs_ln_ag_cta_kernel
 * (csrc/tokenweave_fused_kernels.cu:106-152) with the switch-side
 * multimem.ld_reduce replaced by P loads from local HBM. */
TW_API int tw_reduce_add_rms_norm(const void* const* partials, int num_partials,
                           void* y, void* residual, const void* weight,
                           int64_t num_tokens, int64_t hidden_size,
                           int max_ctas, float epsilon, void* stream);

/* Same op with the reference's argument list.  `mcptr` is the device address
 * of this rank's row shard inside partial buffer 0; partial p lives at
 * mcptr + p * peer_stride_bytes (the one-GPU stand-in for "the same offset in
 * every peer's symmetric buffer").  y is written to `input`, which normally is
 * the shard of partial `rank` (mcptr + rank * peer_stride_bytes), as the
 * reference stores y over its own staging rows.  signal pads do not exist on
 * one GPU and are not part of this ABI.
 * Replaces ::fused_rs_ln_cta (csrc/tokenweave_artifact_kernels.cu:772-813,
 * schema at csrc/torch_bindings.cpp:166-171). */
TW_API int tw_fused_rs_ln_cta(void* input, void* residual, const void* weight,
                       uint64_t mcptr, int64_t peer_stride_bytes, int rank,
                       int world_size, int max_ctas, float epsilon,
                       int64_t num_tokens, int64_t hidden_size, void* stream);

/* Identical to tw_fused_rs_ln_cta on one GPU: the all-gather that distinguishes
 * the reference op is the store of y to the peers, and there are none.
 * Replaces ::fused_rs_ln_ag_cta (csrc/tokenweave_fused_kernels.cu:220-261,
 * schema at csrc/torch_bindings.cpp:152-157). */
TW_API int tw_fused_rs_ln_ag_cta(void* input, void* residual, const void* weight,
                          uint64_t mcptr, int64_t peer_stride_bytes, int rank,
                          int world_size, int max_ctas, float epsilon,
                          int64_t num_tokens, int64_t hidden_size,
                          void* stream);

/* Workspace of the *_ws entry points: TW_SPLIT_WORKSPACE_BYTES of device memory,
 * 256-byte aligned, all zeros before the first call that uses it.  Every call
 * leaves it ready for the next one (its arrival counters back at zero) when its
 * kernel has finished.  Calls that share a workspace must not overlap in time
 * (same stream, or ordered by events).  It holds the hand-over slots of
 * TW_SPLIT_MAX_TOKENS rows that are cut into segments. */
#define TW_SPLIT_MAX_TOKENS 256
#define TW_SPLIT_WORKSPACE_BYTES (TW_SPLIT_MAX_TOKENS * 384)

/* tw_reduce_add_rms_norm for decode-size batches.  With few token rows and many
 * compute units a row is cut into segments of whole 64-vector chunks, one
 * workgroup per segment; the segments leave their partial sums of squares in
 * `workspace`, and the workgroup that arrives last normalises the row.  Results
 * are bit-identical to tw_reduce_add_rms_norm.  The split is used when
 * max_ctas <= 0, num_tokens <= TW_SPLIT_MAX_TOKENS and tw_split_segments() says
 * more than one segment.  The workspace also serves batches of a few more rows
 * than the device has compute units (C < num_tokens <= C + C/4): one workgroup
 * per row would give some units two rows and the others one, so the first C rows
 * get a workgroup each and the excess rows are cut into quarters, a workgroup
 * each, handed over the same way (bit-identical again).  Otherwise, or
 * with workspace == NULL, the call IS tw_reduce_add_rms_norm.
 * workspace_bytes < TW_SPLIT_WORKSPACE_BYTES is an error.
 * The reference sizes its persistent grids per batch so that its kernels are not
 * starved of CTAs (grid = min(MAX_CTAS, rows), block = hidden_size / 8:
 * csrc/tokenweave_fused_kernels.cu:241-244, vllm/model_executor/models/
 * tokenweave_utils.py:86); on 256 compute units a decode batch of 1-32 rows needs
 * more than one workgroup per row to do the same. */
TW_API int tw_reduce_add_rms_norm_ws(const void* const* partials, int num_partials,
                              void* y, void* residual, const void* weight,
                              int64_t num_tokens, int64_t hidden_size,
                              int max_ctas, float epsilon, void* workspace,
                              int64_t workspace_bytes, void* stream);

/* tw_fused_rs_ln_ag_cta (= tw_fused_rs_ln_cta on one GPU) with the workspace of
 * tw_reduce_add_rms_norm_ws: the reference's argument list for decode-size
 * batches.  Replaces ::fused_rs_ln_ag_cta / ::fused_rs_ln_cta as above. */
TW_API int tw_fused_rs_ln_ag_cta_ws(void* input, void* residual, const void* weight,
                             uint64_t mcptr, int64_t peer_stride_bytes, int rank,
                             int world_size, int max_ctas, float epsilon,
                             int64_t num_tokens, int64_t hidden_size,
                             void* workspace, int64_t workspace_bytes,
                             void* stream);

/* tw_reduce_add_rms_norm_ws without a workspace argument and without any
 * allocation: the workspace is a static array in the library's device code
 * (TW_SPLIT_WORKSPACE_BYTES = 96 KiB on every GPU the library is used on, held
 * until the process ends).  No counterpart in the reference; it is for callers
 * that cannot allocate device memory — code under HIP graph capture, tight
 * serving loops, harnesses that forbid hipMalloc.  num_tokens above
 * TW_SPLIT_MAX_TOKENS is refused with TW_ERR_INVALID_ARGUMENT (such batches need
 * no workspace: use tw_reduce_add_rms_norm).  The first call on a device resolves
 * the array's address (not a stream operation: make it before capturing).  All
 * calls on one GPU share the one array: calls that overlap in time on the same GPU
 * (different streams, no ordering) race; order them or use the *_ws form with a
 * workspace per stream. */
TW_API int tw_reduce_add_rms_norm_noalloc(const void* const* partials, int num_partials,
                                   void* y, void* residual, const void* weight,
                                   int64_t num_tokens, int64_t hidden_size,
                                   int max_ctas, float epsilon, void* stream);

/* Segments per row the *_ws entry points use for this shape on the current
 * device: 1 = one workgroup per row (no workspace traffic).  For a batch of a few
 * more rows than compute units it is the number of segments of each excess row. */
TW_API int tw_split_segments(int64_t num_tokens, int64_t hidden_size, int max_ctas);

/* out[M, N] = a[M, K] * b[N, K]^T, bf16 in, fp32 accumulate on MFMA, bf16 out.
 * `ldc` is the row stride of out in elements (>= N), so the result can land in
 * a row slice of a wider staging buffer.  Required: K % 8 == 0, N % 4 == 0,
 * ldc % 4 == 0, 16-byte aligned a and b, 8-byte aligned out.  max_cus > 0
 * limits the grid to that many workgroups so a concurrent kernel keeps the
 * remaining compute units.
 * Replaces UnquantizedLinearMethod.apply_inplace = torch.matmul(x, W.t(), out=)
 * (vllm/model_executor/layers/linear.py:203-228) for the row-parallel o_proj /
 * down_proj that produces one rank's partial sum. */
TW_API int tw_gemm_bf16_nt(void* out, const void* a, const void* b, int64_t M,
                    int64_t N, int64_t K, int64_t ldc, int max_cus,
                    void* stream);

/* tw_gemm_bf16_nt with the linear layer's optional bias: bias is [N] bf16 in device
 * memory (8-byte aligned) or NULL.  It is added as the reference adds it — to the
 * product already rounded to bf16, in fp32, rounded again:
 *   out = bf16_rne( f32(bf16_rne(a * b^T)) + f32(bias) )
 * (torch.matmul(x, W.t(), out=output); output += bias,
 * vllm/model_executor/layers/linear.py:224-228).  In a tensor-parallel layer only
 * rank 0 passes its bias (linear.py:1306-1308), so the P-way sum holds it once. */
TW_API int tw_gemm_bf16_nt_bias(void* out, const void* a, const void* b, const void* bias,
                         int64_t M, int64_t N, int64_t K, int64_t ldc, int max_cus,
                         void* stream);

/* The producer of the fused op's input: the P row-parallel partial sums of one
 * token split in ONE launch, outs[p][M, N] = as[p][M, K] * bs[p][N, K]^T for
 * p < num_partials, each written straight into its rank's staging rows (outs[p] =
 * slot p of the staging buffer at the split's first row, ldc = the slot's row
 * stride in elements) — the layout tw_reduce_add_rms_norm / tw_fused_rs_ln_ag_cta
 * read, with no copy in between.  outs, as, bs are HOST arrays of num_partials
 * device pointers; shapes, alignment and max_cus as for tw_gemm_bf16_nt; results are
 * bit-identical to num_partials calls of tw_gemm_bf16_nt.  Workgroups walk
 * num_partials x tiles; with eight partials every XCD computes one of them.
 * Replaces the row-parallel o_proj / down_proj writing in place into the symmetric
 * staging buffer: UnquantizedLinearMethod.apply_inplace and
 * RowParallelLinear.forward_inplace (vllm/model_executor/layers/linear.py:203-228,
 * 1310-1321), called from vllm/model_executor/models/llama.py:99-103,248-249 —
 * there one GEMM per rank, here (one GPU standing in for the ranks) all of them. */
TW_API int tw_gemm_bf16_nt_partials(void* const* outs, const void* const* as,
                             const void* const* bs, int num_partials, int64_t M,
                             int64_t N, int64_t K, int64_t ldc, int max_cus,
                             void* stream);

/* Norm with static-scale fp8 output.  out is [num_tokens, hidden_size] of OCP
 * float8 e4m3fn (1 byte per element): out = fp8_rne(clamp(y / *scale, +-448)),
 * where y is the bf16 (or `dtype`) result the unquantised op would store, and
 * `scale` points to ONE fp32 value in device memory.  input is not modified.
 * Replaces ::rms_norm_static_fp8_quant (csrc/layernorm_quant_kernels.cu:165-190,
 * schema at csrc/torch_bindings.cpp:199-205). */
TW_API int tw_rms_norm_static_fp8_quant(void* out, const void* input, const void* weight,
                                        const float* scale, int64_t num_tokens,
                                        int64_t hidden_size, float epsilon, int dtype,
                                        void* stream);

/* residual <- input + residual ; out <- fp8 quantisation (as above) of
 * RMSNorm(residual) * weight.  input is not modified.
 * Replaces ::fused_add_rms_norm_static_fp8_quant
 * (csrc/layernorm_quant_kernels.cu:203-245, schema at
 * csrc/torch_bindings.cpp:207-213). */
TW_API int tw_fused_add_rms_norm_static_fp8_quant(void* out, const void* input, void* residual,
                                                  const void* weight, const float* scale,
                                                  int64_t num_tokens, int64_t hidden_size,
                                                  float epsilon, int dtype, void* stream);

/* tw_reduce_add_rms_norm with the fp8 output above: the fused P-partial op
 * feeding an fp8 GEMM.  bf16 in; 16-byte alignment and hidden_size % 16 == 0
 * required.  No counterpart in the reference (its TokenWeave kernels emit bf16);
 * it composes the two reference ops it is named after. */
TW_API int tw_reduce_add_rms_norm_static_fp8_quant(const void* const* partials, int num_partials,
                                                   void* out, void* residual, const void* weight,
                                                   const float* scale, int64_t num_tokens,
                                                   int64_t hidden_size, int max_ctas,
                                                   float epsilon, void* stream);

/* Residual-add (optional) + RMSNorm + dynamic per-token quantisation:
 *   x = input + residual (fp32) ; residual <- x ; rms = 1/sqrt(mean(x^2) + epsilon)
 *   n = round(round(x * rms) * weight)            (both roundings to the input type)
 *   scales[t] = max(min(max_j |n[t][j]|, *scale_ub) / qmax, floor)
 *   out = fp8_e4m3fn(clamp(n / scales[t], +-448))     qmax 448, floor 1/(448 * 512)
 *       | int8(saturate(rint(n * (1 / scales[t]))))   qmax 127, floor FLT_EPSILON
 * out: [num_tokens, hidden_size] bytes; scales: num_tokens floats (device);
 * scale_ub: NULL or one device float (fp8 only); residual: NULL or
 * [num_tokens, hidden_size], updated in place.  input is not modified.  Any
 * hidden_size / alignment (vector kernel for bf16 and fp16, 16-byte aligned, hidden_size % 16 == 0).
 * Replaces ::rms_norm_dynamic_per_token_quant
 * (csrc/quantization/fused_kernels/fused_layernorm_dynamic_per_token_quant.cu:131-155,
 * schema at csrc/torch_bindings.cpp:216-221). */
TW_API int tw_rms_norm_dynamic_per_token_quant(void* out, const void* input, const void* weight,
                                               float* scales, const float* scale_ub,
                                               void* residual, int64_t num_tokens,
                                               int64_t hidden_size, float epsilon, int dtype,
                                               int out_kind, void* stream);

/* The op above over P partial buffers: x = sum_p partials[p] + residual in fp32,
 * fixed order.  bf16 in; 16-byte alignment and hidden_size % 16 == 0 required;
 * residual may be NULL.  No counterpart in the reference (its TokenWeave kernels
 * emit bf16); it fuses the reference's all-reduce + the op above. */
TW_API int tw_reduce_add_rms_norm_dynamic_per_token_quant(
    const void* const* partials, int num_partials, void* out, float* scales, void* residual,
    const void* weight, const float* scale_ub, int64_t num_tokens, int64_t hidden_size,
    int max_ctas, float epsilon, int out_kind, void* stream);

/* tw_gemm_bf16_nt_partials with a bias per product: biases is NULL or a HOST array of
 * num_partials device pointers, each [N] bf16 or NULL (one GPU standing in for the ranks
 * passes rank 0's bias in biases[0] and NULL elsewhere, linear.py:1306-1308).  Same
 * arithmetic as tw_gemm_bf16_nt_bias; bit-identical to num_partials calls of it. */
TW_API int tw_gemm_bf16_nt_partials_bias(void* const* outs, const void* const* as,
                                  const void* const* bs, const void* const* biases,
                                  int num_partials, int64_t M, int64_t N, int64_t K,
                                  int64_t ldc, int max_cus, void* stream);

/* ---------------------------------------------------------------------------
 * Between a decoder layer's projections: rotation of queries and keys by their
 * positions, a paged cache of keys and values in 4 bits, attention over it.  (No
 * counterpart on the reference's path; head counts and lengths are the caller's.)
 *
 * tw_heads: a tensor [num_tokens, heads, head_size] whose channels are contiguous; the
 * strides are in elements (views of a wider projection output are fine).  Rows of an output
 * must not share memory: TW_ERR_INVALID_ARGUMENT.
 * ------------------------------------------------------------------------- */
typedef struct tw_heads {
  void* data;
  int64_t heads;
  int64_t token_stride;
  int64_t head_stride;
} tw_heads;

#define TW_ROTARY_INTERLEAVED 1 /* pairs are neighbours (2j, 2j+1), not (j, j + rotary_dim/2) */
#define TW_ROTARY_INVERSE 2     /* turn back: the gradient of a rotation, or a key's move     */

/* For every pair (x1, x2) of the first rotary_dim channels of every head:
 *   y1 = x1 * cos - x2 * sin ;  y2 = x2 * cos + x1 * sin      (fp32, rounded once)
 * cos_sin: [max_positions, rotary_dim] fp32, a row holding the cosines of its
 * rotary_dim/2 pairs and then the sines; row positions[t] serves token t.  The channels
 * behind rotary_dim are copied.  out may be the input.  A position outside
 * [0, max_positions) makes the turned channels NaN.  k_out / k may both be NULL.
 * dtype: TW_DTYPE_*; any head_size, rotary_dim even, 2 <= rotary_dim <= head_size. */
TW_API int tw_rotary_positions(const tw_heads* q_out, const tw_heads* q, const tw_heads* k_out,
                               const tw_heads* k, const int64_t* positions, const float* cos_sin,
                               int64_t max_positions, int64_t num_tokens, int head_size,
                               int rotary_dim, int flags, int dtype, void* stream);

/* The cache: num_pages pages, [num_pages][kv_heads][page_size * (D + D/16)] bytes, 16-byte
 * aligned; D = head_size in {64, 128, 256}, page_size a power of two, 16 to 256.  A value is
 * 4 bits (sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6: e2m1) times 2^e, one e for 32
 * channels of a token: 4.25 bits a value.  e is the smallest with |x| <= 7 * 2^e for all
 * 32, in [-23, 13] (so that every value is exact in fp16; larger magnitudes saturate at
 * 6 * 2^13); ties go to the even code; a block with an infinity or a NaN reads as NaN.
 * Of one head in one page, P = page_size:
 *   keys    [P][D/2]              two channels a byte, the lower in the low nibble
 *   values  [P/4][16][4][D/32]    of four tokens each sixteenth of the channels together
 *   scales  [D/32][P] of the keys, then [D/32][P] of the values: e + 127, or 255 for NaN */
#define TW_KV4_MIN_PAGE 16
#define TW_KV4_MAX_PAGE 256

/* Writes the tokens' keys and values to their slots (slot = page * page_size + place;
 * int64; a slot outside the cache, -1 for instance, is skipped; two tokens of a call with
 * one slot are an error that is not found).  With cos_sin the keys are turned on the way, as
 * tw_rotary_positions does and rounded to `dtype` before they are coded, and the queries
 * (q -> q_out; both may be NULL) are turned in the same launch.  Without cos_sin
 * (NULL; positions is not read) the keys are coded as they are and q must be NULL. */
TW_API int tw_kv4_append(void* pages, int64_t num_pages, int page_size, const tw_heads* k,
                         const tw_heads* v, const int64_t* slots, const tw_heads* q_out,
                         const tw_heads* q, const int64_t* positions, const float* cos_sin,
                         int64_t max_positions, int64_t num_tokens, int head_size, int rotary_dim,
                         int flags, int dtype, void* stream);

/* k_out, v_out <- the values that the slots hold; zeros where a slot is outside the cache. */
TW_API int tw_kv4_read(const tw_heads* k_out, const tw_heads* v_out, const void* pages,
                       int64_t num_pages, int page_size, const int64_t* slots, int64_t num_tokens,
                       int head_size, int dtype, void* stream);

/* out = softmax(scale * q k^T) v over a sequence's cached tokens, for every query head; query
 * heads g * G .. g * G + G - 1 share key head g (G = q->heads / kv_heads).
 *   block_table  [num_seqs][table_stride] int32, the first table_width of a row are read:
 *                page of tokens 0 .. P-1, P .. 2P-1, ... of the sequence; tokens of a page
 *                outside [0, num_pages) are as if masked
 *   seq_lens     [num_seqs] int32: cached tokens, the new ones among them (appended before)
 *   query_starts [num_seqs + 1] int32: sequence s has the tokens query_starts[s] ..
 *                query_starts[s+1] - 1 of q and out, the last of its cached tokens; NULL:
 *                num_tokens / num_seqs tokens each.  A batch may be attended in parts: tokens
 *                below 0 are an earlier call's, those from num_tokens on a later one's (and
 *                not seen here, though seq_lens counts them)
 * Query i of n sees the tokens up to its own, seq_len - n + i, and of these the last
 * `window` where window > 0.  A query that sees none gives zeros, and so do tokens of q before
 * query_starts[0] and from query_starts[num_seqs] on, which no sequence has (padding).
 * max_queries: at least the largest number of new tokens of a sequence (tokens of a sequence
 * behind that many are not computed, and their rows of out are left as they were).
 * bf16 or fp16; scores and sums in fp32.  seq_lens may change between the replays of a
 * captured call.
 * workspace: tw_kv4_attention_workspace() bytes, 16-byte aligned, contents of no meaning
 * before and after; calls that may run at the same time need one each. */
TW_API int64_t tw_kv4_attention_workspace(int q_heads, int kv_heads, int head_size, int64_t num_seqs,
                                          int64_t num_tokens, int64_t max_queries, int64_t table_width,
                                          int page_size);
TW_API int tw_kv4_attention(const tw_heads* out, const tw_heads* q, const void* pages,
                            int64_t num_pages, int page_size, int kv_heads,
                            const int32_t* block_table, int64_t table_stride, int64_t table_width,
                            const int32_t* seq_lens, const int32_t* query_starts, int64_t num_seqs,
                            int64_t num_tokens, int64_t max_queries, int head_size, float scale,
                            int64_t window, int dtype, void* workspace, int64_t workspace_bytes,
                            void* stream);

/* ---------------------------------------------------------------------------
 * The feed-forward half of a decoder layer: a gated product with its gradients, rows to
 * 8-bit codes with a scale for 128 channels, the product of such codes.  (No counterpart on
 * the reference's path; every size is the caller's.)
 * ------------------------------------------------------------------------- */
#define TW_ACT_SILU 0      /* x / (1 + e^-x)                                        */
#define TW_ACT_GELU 1      /* x (1 + erf(x / sqrt 2)) / 2                           */
#define TW_ACT_GELU_TANH 2 /* x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))) / 2       */
/* They are evaluated in fp32 with the exponential and reciprocal instructions.  For x >= -1 the value
 * is off by 5 * 2^-24 of itself or less; below, where it is x times a small exponential e^-z, by about
 * (z + 6) * 2^-24 (silu, z = -x) and (3 z + 20) * 2^-24 (the gelus: what the rounding of their
 * arguments to fp32 does to it). */

/* out[M, I] = act(G) * U,  G = a[M, K] b[0:I, K]^T,  U = a b[I:2I, K]^T:  bf16, both sums in
 * fp32, the result rounded once.  b is one contiguous [2 I, K] (gate rows, then up rows), out has
 * rows of stride ldc.  gate_up, where not NULL, takes G and U, rounded, as [M, 2 I] (stride
 * ld_gate_up): what the gradient needs.  K % 8 == 0, K <= 2^24, I % 4 == 0, strides % 4 == 0; a, b
 * 16-byte, out, gate_up 8-byte aligned; max_cus as for tw_gemm_bf16_nt.
 * workspace: tw_gated_gemm_bf16_nt_workspace() bytes (asked with the same device current; 0 for
 * most sizes: fp32 sums where some hundred rows are divided along K), 256-byte aligned, contents of
 * no meaning before and after; calls that may run at the same time need one each. */
TW_API int64_t tw_gated_gemm_bf16_nt_workspace(int64_t M, int64_t I, int64_t K);
TW_API int tw_gated_gemm_bf16_nt(void* out, void* gate_up, const void* a, const void* b, int64_t M,
                                 int64_t I, int64_t K, int64_t ldc, int64_t ld_gate_up,
                                 int activation, int max_cus, void* workspace,
                                 int64_t workspace_bytes, void* stream);

/* Its gradients, with D = [grad_out * U * act'(G), grad_out * act(G)] rounded to bf16:
 *   grad_a[M, K] = D b,  grad_b[2 I, K] = D^T a     (either may be NULL; contiguous)
 * K and, for grad_a, 2 I and, for grad_b, M at most 2^21.
 * workspace: tw_gated_gemm_bf16_nt_backward_workspace() bytes (asked with the same device current,
 * for the gradients that are wanted), 256-byte aligned, contents of no meaning before and after;
 * calls that may run at the same time need one each. */
TW_API int64_t tw_gated_gemm_bf16_nt_backward_workspace(int64_t M, int64_t I, int64_t K, int want_a,
                                                        int want_b);
TW_API int tw_gated_gemm_bf16_nt_backward(void* grad_a, void* grad_b, const void* grad_out,
                                          int64_t ld_grad_out, const void* a, const void* b,
                                          const void* gate_up, int64_t ld_gate_up, int64_t M,
                                          int64_t I, int64_t K, int activation, int max_cus,
                                          void* workspace, int64_t workspace_bytes, void* stream);

#define TW_FP8_GROUP 128 /* channels of a scale; the last group of a row holds what is left */

/* Rows to OCP float8 e4m3fn codes with one fp32 scale for TW_FP8_GROUP channels of a row:
 *   scale = max(max |y|, 1e-10) / 448, rounded to fp32 ;  code = the e4m3 value next to y / scale
 * (the exact quotient: ties to the even code).  y is the input's row (activation < 0), or, of an
 * input of 2 K channels, act(first half) * second half in fp32, not rounded in between.  A group that
 * holds an infinity or a NaN gives NaN codes.  out is [num_rows, K] contiguous; the scale of
 * row t, group g is scales[t * scale_row_stride + g * scale_group_stride] (the product below reads
 * scale_row_stride == 1 fastest).  dtype TW_DTYPE_*; any K, any alignment of whole elements. */
TW_API int tw_quant_fp8_groups(void* out, float* scales, int64_t scale_row_stride,
                               int64_t scale_group_stride, const void* input, int64_t ld_input,
                               int64_t num_rows, int64_t K, int activation, int dtype, void* stream);

/* out[M, N] = sum over blocks k of 128:  a_scale[m, k] * b_scale[n / 128, k] * (a b^T over the block)
 * a [M, K] and b [N, K] e4m3fn codes, contiguous; a's scales at the given strides (elements), b's
 * [ceil(N / 128), ceil(K / 128)] contiguous; rounded once to dtype (TW_DTYPE_BF16 or TW_DTYPE_F16),
 * rows of out at stride ldc.  The matrix instruction adds aligned eights of products first, at 13 bits
 * below the exponent of the largest of the eight; the sums of those, and of the blocks with their
 * scales, are fp32's.  K % 16 == 0, K <= 2^22, N % 4 == 0, ldc % 4 == 0, scales of two rows 0 to 2^20
 * elements apart; a, b 16-byte, out 8-byte aligned; max_cus as for tw_gemm_bf16_nt.
 * workspace: tw_gemm_fp8_block_nt_workspace() bytes, as for tw_gated_gemm_bf16_nt. */
TW_API int64_t tw_gemm_fp8_block_nt_workspace(int64_t M, int64_t N, int64_t K);
TW_API int tw_gemm_fp8_block_nt(void* out, const void* a, const float* a_scales,
                                int64_t scale_row_stride, int64_t scale_block_stride, const void* b,
                                const float* b_scales, int64_t M, int64_t N, int64_t K, int64_t ldc,
                                int dtype, int max_cus, void* workspace, int64_t workspace_bytes,
                                void* stream);

#ifdef __cplusplus
}
#endif
#endif /* TOKENWEAVE_AMD_H */
