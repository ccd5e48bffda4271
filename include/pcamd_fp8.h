/*
 * pcamd_fp8.h - C ABI of the MI355X (gfx950) FP8 hot path.
 *
 * One shared library, libpcamd_fp8.so, exports these functions. They take raw
 * device pointers, element strides (in elements, not bytes) and sizes, launch
 * asynchronously on the given hipStream_t (passed as void*), never allocate
 * device memory, keep no mutable global state and are reentrant. Every
 * function returns PCAMD_OK (0) or a negative status; pcamd_last_error()
 * returns a thread-local description of the most recent failure.
 *
 * Reference interfaces replaced (paths relative to xuOAO/practice_cuda):
 *   pcamd_quant_block   <- fp8_training/fp8_bench/impls/triton_per_block.py:60-150
 *                          (launches kernels/quant/per_block.py:6-48)
 *   pcamd_quant_block_dual <- no single counterpart: the block_m = 1 and
 *                          block_n = 1 calls of pcamd_quant_block on one tensor
 *   pcamd_quant_block_ex, pcamd_quant_block_dual_ex <- the two above with an
 *                          output store policy (flags)
 *   pcamd_quant_channel <- fp8_training/fp8_bench/impls/triton_per_channel.py:90-219
 *                          (launches kernels/quant/per_channel.py:35-102, :105-267)
 *   pcamd_quant_tensor  <- fp8_training/fp8_bench/impls/triton_per_tensor.py:28-95
 *                          and kernels/fp8_bmm/fp8_warper.py:9-77
 *   pcamd_bmm_quant_a   <- kernels/fp8_bmm/kernel/fp8_quant_bmm_fused_kernel.py:30-146
 *                          (its intent: the activation quantized inside the GEMM)
 *   pcamd_repack_fp8    <- the `.contiguous()` copies of the do_transpose_a /
 *                          do_transpose_b BMM variants
 *                          (impls/triton_per_block.py:254-272)
 *   pcamd_bmm_scaled    <- impls/triton_per_block.py:232-420 (block scales),
 *                          impls/triton_per_channel.py:271-427 (channel scales),
 *                          impls/triton_per_tensor.py:140-306 and
 *                          kernels/fp8_bmm/fp8_warper.py:79-129 (tensor scale)
 *   pcamd_bmm_scaled_mixed <- the same GEMM with an e5m2 and an e4m3fn operand:
 *                          fp8_training/fp8_bench/modules/bmm_linear.py:121-227
 *                          (custom op fp8_bench::bmm_linear_tma, called for
 *                          dgrad / wgrad at :402-410, :441-446 with torchao's
 *                          e5m2 grad_output and e4m3fn input / weight, :43-46)
 */
#ifndef PCAMD_FP8_H
#define PCAMD_FP8_H

#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

#define PCAMD_ABI_VERSION 7 /* 2: pcamd_bmm_scaled_mixed; 3: pcamd_quant_block_ex, pcamd_quant_block_dual_ex;
                              4: PCAMD_F64 scale arithmetic of pcamd_quant_tensor;
                              5: pcamd_quant_channel_ws, pcamd_quant_tensor_ws;
                              6: pcamd_rms_norm_quant and the pcamd_latent_ functions;
                              7: the int8 functions and the pcamd_expert_ ones */

/* status codes */
#define PCAMD_OK 0
#define PCAMD_ERR_INVALID (-1)     /* bad argument (shape, stride, pointer, code) */
#define PCAMD_ERR_UNSUPPORTED (-2) /* valid but not implemented combination */
#define PCAMD_ERR_LAUNCH (-3)      /* hipGetLastError() after launch */

/* element type codes */
#define PCAMD_F32 0
#define PCAMD_BF16 1
#define PCAMD_F16 2
#define PCAMD_E4M3FN 3 /* OCP fp8 e4m3fn: max 448, no inf, NaN = 0x7f/0xff */
#define PCAMD_E5M2 4   /* OCP fp8 e5m2: max 57344, inf = 0x7c */
#define PCAMD_F64 5    /* scale arithmetic only (pcamd_quant_tensor) */

/* BMM scale modes */
#define PCAMD_SCALE_BLOCK 0   /* sa[b, m/qbm, k/qbk], sb[b, k/qbk, n/qbn] */
#define PCAMD_SCALE_CHANNEL 1 /* sa[b, m], sb[b, n] */
#define PCAMD_SCALE_TENSOR 2  /* sa[0] (and sb[0] when scales_are_quant) */

/* quantizer flags (the _ex entry points) */
#define PCAMD_QUANT_CACHED_OUTPUT 1 /* write y and the scales with ordinary, cache-allocating stores */

/* BMM epilogue activations */
#define PCAMD_ACT_NONE 0
#define PCAMD_ACT_GELU 1 /* exact: 0.5 x (1 + erf(x / sqrt 2)) */
#define PCAMD_ACT_SWIGLU 2 /* int8 products only: silu(gate) * other, over halves of b's rows */

int pcamd_abi_version(void);
const char *pcamd_last_error(void);

/*
 * Per-block quantization of x[batch, m, n] into fp8 y with one fp32 dequant
 * scale per block_m x block_n tile (block sizes are powers of two).
 * Per block: amax = max|x|; s = max(amax, eps); qs = fp8_max / s;
 * scale[b, i, j] = 1 / qs; y = fp8_rne(clamp(x * qs, -fp8_max, fp8_max)).
 * Replaces fp8_training/fp8_bench/impls/triton_per_block.py:60-150.
 */
int pcamd_quant_block(const void *x, int x_dtype, int64_t batch, int64_t m,
                      int64_t n, int64_t sxb, int64_t sxm, int64_t sxn,
                      void *y, int y_dtype, int64_t syb, int64_t sym,
                      int64_t syn, float *scale, int64_t ssb, int64_t ssm,
                      int64_t ssn, int64_t block_m, int64_t block_n,
                      float fp8_max, float eps, void *stream);

/*
 * Both block quantizations the block-scaled training recipe applies to one
 * tensor, from a single read of x: y_row / scale_row are exactly
 * pcamd_quant_block(block_m = 1, block_n = block) and y_col / scale_col
 * exactly pcamd_quant_block(block_m = block, block_n = 1). y_row has strides
 * syb, sym, syn and y_col its own ycb, ycm, ycn: the same layout, or stored
 * transposed (ycm = 1, element (r, c) at c * ycn + r), which makes it the
 * K-major operand of a GEMM reducing over m. scale_row is
 * [batch, m, ceil(n / block)] and scale_col [batch, ceil(m / block), n]
 * (strides in elements). One kernel serves row-contiguous x with block = 128
 * (transposed y_col: m and n multiples of 128, 16-byte aligned rows); other
 * layouts and block sizes run the two quantizers in turn. The reference has no
 * single counterpart: its per-block training module is unfinished
 * (fp8_training/fp8_bench/modules/per_block.py:13-67), and this pairs the
 * act/grad 1x128 quantization (impls/triton_per_block.py:60-150, block_m = 1)
 * with the wgrad re-quantization along the reduction dimension.
 */
int pcamd_quant_block_dual(const void *x, int x_dtype, int64_t batch,
                           int64_t m, int64_t n, int64_t sxb, int64_t sxm,
                           int64_t sxn, void *y_row, int64_t syb, int64_t sym,
                           int64_t syn, void *y_col, int64_t ycb, int64_t ycm,
                           int64_t ycn, int y_dtype, float *scale_row,
                           int64_t srb, int64_t srm, int64_t srn,
                           float *scale_col, int64_t scb, int64_t scm,
                           int64_t scn, int64_t block, float fp8_max, float eps,
                           void *stream);

/*
 * pcamd_quant_block and pcamd_quant_block_dual with flags. By default the
 * quantizers write their fp8 outputs and scales with non-temporal stores
 * (the fastest for a quantization on its own); PCAMD_QUANT_CACHED_OUTPUT
 * writes them with ordinary stores, which leave them in the GPU's caches
 * (the 256 MB memory-side cache included) for a kernel that reads them next,
 * e.g. the GEMM after the training layer's quantization. Bytes and scales
 * are the same either way; flags = 0 is exactly the call without _ex; other
 * bits return PCAMD_ERR_INVALID. The reference interfaces are those of
 * pcamd_quant_block / pcamd_quant_block_dual (the Triton kernels there pick
 * their own cache policy). Available from PCAMD_ABI_VERSION 3.
 */
int pcamd_quant_block_ex(const void *x, int x_dtype, int64_t batch, int64_t m,
                         int64_t n, int64_t sxb, int64_t sxm, int64_t sxn,
                         void *y, int y_dtype, int64_t syb, int64_t sym,
                         int64_t syn, float *scale, int64_t ssb, int64_t ssm,
                         int64_t ssn, int64_t block_m, int64_t block_n,
                         float fp8_max, float eps, int flags, void *stream);
int pcamd_quant_block_dual_ex(const void *x, int x_dtype, int64_t batch,
                              int64_t m, int64_t n, int64_t sxb, int64_t sxm,
                              int64_t sxn, void *y_row, int64_t syb,
                              int64_t sym, int64_t syn, void *y_col,
                              int64_t ycb, int64_t ycm, int64_t ycn,
                              int y_dtype, float *scale_row, int64_t srb,
                              int64_t srm, int64_t srn, float *scale_col,
                              int64_t scb, int64_t scm, int64_t scn,
                              int64_t block, float fp8_max, float eps,
                              int flags, void *stream);

/*
 * Per-channel quantization. channel_axis = -2: one scale per row (reduce over
 * n); channel_axis = -1: one scale per column (reduce over m).
 * s = max(amax, eps); qs = fp8_max / s; scale[b, c] = s / fp8_max;
 * y = fp8_rne(clamp(x * qs, -fp8_max, fp8_max)).
 * Replaces fp8_training/fp8_bench/impls/triton_per_channel.py:90-219.
 */
int pcamd_quant_channel(const void *x, int x_dtype, int64_t batch, int64_t m,
                        int64_t n, int64_t sxb, int64_t sxm, int64_t sxn,
                        void *y, int y_dtype, int64_t syb, int64_t sym,
                        int64_t syn, float *scale, int64_t ssb, int64_t ssc,
                        int channel_axis, float fp8_max, float eps,
                        void *stream);

/*
 * pcamd_quant_channel with a workspace of pcamd_quant_channel_workspace()
 * bytes (device memory, 4-byte aligned, contents ignored and overwritten; it
 * may be NULL, and is not needed where the size is 0). With it the per-column
 * scales of a tall tensor take two launches (three if it is narrow as well)
 * instead of four. Same bytes.
 * Available from PCAMD_ABI_VERSION 5.
 */
int64_t pcamd_quant_channel_workspace(int64_t batch, int64_t m, int64_t n,
                                      int channel_axis);
int pcamd_quant_channel_ws(const void *x, int x_dtype, int64_t batch,
                           int64_t m, int64_t n, int64_t sxb, int64_t sxm,
                           int64_t sxn, void *y, int y_dtype, int64_t syb,
                           int64_t sym, int64_t syn, float *scale,
                           int64_t ssb, int64_t ssc, int channel_axis,
                           float fp8_max, float eps, void *workspace,
                           int64_t workspace_bytes, void *stream);

/*
 * Per-tensor quantization: amax over the whole tensor, s = max(amax, eps),
 * qs = reciprocal(s) * fp8_max, scale[0] = reciprocal(qs),
 * y = fp8_rne(clamp(x * qs)). quant_scale_out (may be NULL) receives qs. Both
 * scalars are device fp32. scale_dtype (PCAMD_F32 / PCAMD_BF16 / PCAMD_F16) is
 * the dtype the scalar steps are rounded to: PCAMD_F32 for
 * fp8_training/fp8_bench/impls/triton_per_tensor.py:28-95; the input's dtype
 * for the legacy kernels/fp8_bmm/fp8_warper.py:9-77, whose torch ops on 0-d
 * tensors of the input's dtype round every step (the results are then
 * exactly representable in that dtype). PCAMD_F64 (from PCAMD_ABI_VERSION 4)
 * is torchao's tensorwise scale, which the reference's Float8BMMLinear
 * quantizes with (fp8_training/fp8_bench/modules/float8/float8_utils.py:
 * 45-48, used through float8_scaling_utils.py): qs = fp32(fp8_max /
 * max(fp64(amax), eps)) with the division in fp64, scale[0] = reciprocal(qs)
 * in fp32 (the reciprocal its scaled GEMMs take), then the same
 * fp8_rne(clamp(x * qs)) (float8_training_tensor.py:153-154).
 */
int pcamd_quant_tensor(const void *x, int x_dtype, int64_t batch, int64_t m,
                       int64_t n, int64_t sxb, int64_t sxm, int64_t sxn,
                       void *y, int y_dtype, int64_t syb, int64_t sym,
                       int64_t syn, float *scale, float *quant_scale_out,
                       float fp8_max, float eps, int scale_dtype,
                       void *stream);

/*
 * pcamd_quant_tensor with a workspace of at least 1024 bytes (device memory,
 * 16-byte aligned, contents ignored and overwritten; may be NULL): contiguous
 * tensors then take two launches instead of four. scale_cast (may be NULL)
 * receives the dequant scale in x's dtype. Same bytes. Available from
 * PCAMD_ABI_VERSION 5.
 */
int pcamd_quant_tensor_ws(const void *x, int x_dtype, int64_t batch,
                          int64_t m, int64_t n, int64_t sxb, int64_t sxm,
                          int64_t sxn, void *y, int y_dtype, int64_t syb,
                          int64_t sym, int64_t syn, float *scale,
                          float *quant_scale_out, float fp8_max, float eps,
                          int scale_dtype, void *scale_cast, void *workspace,
                          int64_t workspace_bytes, void *stream);

/*
 * Scaled FP8 batched GEMM: c[b, m, n] = act(sum_k a[b, m, k] b[b, k, n] *
 * scale + bias[b, m, n]) with fp32 accumulation, a/b fp8 of the same code.
 * Block mode applies sa[b, m/qbm, kq] * sb[b, kq, n/qbn] to each qbk-wide
 * partial sum (qbk a multiple of 128); channel mode multiplies the full sum by
 * sa[b, m] * sb[b, n]; tensor mode by sa[0]. scales_are_quant = 1 means the
 * scales are quant scales and the product is inverted (1 / (sa * sb)).
 * bias may be NULL. Strides are in elements; a must be contiguous along k or
 * m, b along n or k, c and bias along n.
 */
int pcamd_bmm_scaled(const void *a, const void *b, int ab_dtype,
                     int64_t batch, int64_t m, int64_t n, int64_t k,
                     int64_t sab, int64_t sam, int64_t sak, int64_t sbb,
                     int64_t sbk, int64_t sbn, void *c, int c_dtype,
                     int64_t scb, int64_t scm, int64_t scn, const void *bias,
                     int bias_dtype, int64_t sbiasb, int64_t sbiasm,
                     int64_t sbiasn, const float *sa, int64_t ssab,
                     int64_t ssa1, int64_t ssa2, const float *sb,
                     int64_t ssbb, int64_t ssb1, int64_t ssb2, int scale_mode,
                     int scales_are_quant, int64_t qbm, int64_t qbk,
                     int64_t qbn, int activation, void *stream);

/*
 * pcamd_bmm_scaled with a format code per operand (a_dtype, b_dtype:
 * PCAMD_E4M3FN or PCAMD_E5M2, equal or not): the training recipe's e5m2
 * gradient times an e4m3fn weight or activation. Every other argument and
 * the math are those of pcamd_bmm_scaled, which is this call with a_dtype ==
 * b_dtype. Available from PCAMD_ABI_VERSION 2.
 */
int pcamd_bmm_scaled_mixed(const void *a, int a_dtype, const void *b,
                           int b_dtype, int64_t batch, int64_t m, int64_t n,
                           int64_t k, int64_t sab, int64_t sam, int64_t sak,
                           int64_t sbb, int64_t sbk, int64_t sbn, void *c,
                           int c_dtype, int64_t scb, int64_t scm, int64_t scn,
                           const void *bias, int bias_dtype, int64_t sbiasb,
                           int64_t sbiasm, int64_t sbiasn, const float *sa,
                           int64_t ssab, int64_t ssa1, int64_t ssa2,
                           const float *sb, int64_t ssbb, int64_t ssb1,
                           int64_t ssb2, int scale_mode, int scales_are_quant,
                           int64_t qbm, int64_t qbk, int64_t qbn,
                           int activation, void *stream);

/*
 * Block-scaled FP8 GEMM with the activation quantization fused into the K
 * loop: a (bf16 or fp16, [batch, m, k], contiguous along k with 16-byte
 * aligned rows) is quantized in 1 x 128 groups along k inside the kernel -
 * bytes and dequant scales exactly those of pcamd_quant_block(block_m = 1,
 * block_n = 128, fp8_max, eps) into ab_dtype - and multiplied by the fp8 b
 * (block scales sb[b, k/128, n/qbn], quant-K block 128) as pcamd_bmm_scaled
 * would with those A scales. qa_out / sa_out (both or neither; qa_out
 * contiguous along k, 8-byte aligned rows) receive the quantized A and its
 * scales [batch, m, k/128]. k must be a positive multiple of 128; other
 * layouts return PCAMD_ERR_UNSUPPORTED (quantize, then pcamd_bmm_scaled).
 * The call pays off for n <= 256 (with n a multiple of 16, k a multiple of
 * 256 and quant-N blocks of at least 128, one workgroup holds every column
 * and reads a once; any bias, activation and output type); wider products quantize each 128-row block of a once per
 * 256-column tile of c, where quantizing first and then multiplying is
 * faster. Replaces the intent of the reference's fused quant + BMM kernel
 * (kernels/fp8_bmm/kernel/fp8_quant_bmm_fused_kernel.py:30-146), whose
 * per-tile scale helper is unfinished there, with the per-block recipe of
 * fp8_training/fp8_bench/impls/triton_per_block.py:60-150 (A) and :232-420
 * (GEMM).
 */
int pcamd_bmm_quant_a(const void *a, int a_dtype, const void *b, int ab_dtype,
                      int64_t batch, int64_t m, int64_t n, int64_t k,
                      int64_t sab, int64_t sam, int64_t sak, int64_t sbb,
                      int64_t sbk, int64_t sbn, void *c, int c_dtype,
                      int64_t scb, int64_t scm, int64_t scn, const void *bias,
                      int bias_dtype, int64_t sbiasb, int64_t sbiasm,
                      int64_t sbiasn, const float *sb, int64_t ssbb,
                      int64_t ssb1, int64_t ssb2, int64_t qbn, void *qa_out,
                      int64_t sqab, int64_t sqam, int64_t sqak, float *sa_out,
                      int64_t soab, int64_t soam, int64_t soak, float fp8_max,
                      float eps, int activation, void *stream);

/*
 * Transposing byte copy of an fp8 tensor: y[b, r, c] = x[b, r, c] for a
 * view x contiguous along rows (sxr == 1) into a view y contiguous along
 * columns (syc == 1); strides in elements (= bytes). This is the copy of the
 * BMM wrappers' transpose variants - an M-major A made K-major, or an
 * N-major B made K-major - that the reference makes with `.contiguous()`
 * on the strided view (fp8_training/fp8_bench/impls/triton_per_block.py:
 * 254-272). Other stride patterns return PCAMD_ERR_UNSUPPORTED.
 */
int pcamd_repack_fp8(const void *x, int64_t batch, int64_t rows,
                     int64_t cols, int64_t sxb, int64_t sxr, int64_t sxc,
                     void *y, int64_t syb, int64_t syr, int64_t syc,
                     void *stream);

/*
 * Root-mean-square norm with the residual's addition, quantized in 1 x 128
 * groups: r = x + residual in fp32 (residual may be NULL; otherwise
 * residual_out, which may be residual or x, receives r in x's type),
 * v = r * rsqrt(mean(r^2) + norm_eps) * weight over rows of n, and y, scale
 * as pcamd_quant_block(block_m = 1, block_n = 128) gives for the fp32 v. x,
 * residual, residual_out, y: [batch, m, n], contiguous along n, any row
 * strides and alignment; weight: [n] (w_dtype: PCAMD_F32, PCAMD_BF16 or
 * PCAMD_F16, like x_dtype); scale: [batch, m, ceil(n / 128)]. A NaN stays a
 * NaN code and does not count in its group's maximum. Available from
 * PCAMD_ABI_VERSION 6, as the functions below.
 */
int pcamd_rms_norm_quant(const void *x, int x_dtype, int64_t batch, int64_t m,
                         int64_t n, int64_t sxb, int64_t sxm,
                         const void *residual, int64_t srb, int64_t srm,
                         const void *weight, int w_dtype, void *y, int y_dtype,
                         int64_t syb, int64_t sym, float *scale, int64_t ssb,
                         int64_t ssm, void *residual_out, int64_t sob,
                         int64_t som, float norm_eps, float fp8_max, float eps,
                         void *stream);

/*
 * Writes new tokens into the pages of a latent cache: latent[tokens,
 * latent_dim], normed as above where weight is given, in the tokens' type
 * (bf16 or fp16) or as e4m3fn codes with one fp32 scale per 128 columns, and
 * rope[tokens, rope_dim] as it is. slots (slot_bytes 4 or 8: int32, int64)
 * holds page * page_size + place per token; a token whose slot is negative or
 * past pages * page_size is skipped. Tokens of one slot are written in no order
 * and may leave parts of each there; other slots are not touched. The cache
 * arrays have a stride per page (clp, crp, csp) and per token (clt, crt, cst),
 * in elements. latent_dim is a multiple of 128 up to 512, rope_dim one of 8 up
 * to 512.
 */
int pcamd_latent_append(const void *latent, const void *rope, int dtype,
                        int64_t tokens, int64_t latent_dim, int64_t rope_dim,
                        int64_t slt, int64_t srt, const void *weight,
                        int w_dtype, const void *slots, int slot_bytes,
                        void *cache_latent, int cache_dtype, int64_t clp,
                        int64_t clt, void *cache_rope, int64_t crp, int64_t crt,
                        float *cache_scale, int64_t csp, int64_t cst,
                        int64_t pages, int64_t page_size, float norm_eps,
                        float eps, void *stream);

/*
 * Attention of absorbed queries over a latent cache: for new token i of S and
 * head h, s[t] = softmax_scale * (q_latent . latent[t] + q_rope . rope[t]) over
 * the tokens t < len - S + i + 1 of the sequence, out = sum_t softmax(s)[t]
 * latent[t], lse (may be NULL) = log sum_t exp(s[t]); a row that sees no token
 * gives zeros and -inf. q_latent [batch, S, heads, latent_dim], q_rope
 * [batch, S, heads, rope_dim], out like q_latent (strides per batch, token and
 * head); token t of sequence b is place t % page_size of page table[b, t /
 * page_size]; lens[batch] counts a sequence's tokens. Lengths are cut to
 * max_pages * page_size, at most 2^31 - 1024, and page numbers to the pool.
 * latent_dim and rope_dim are 512 and 64, or 256 and 32. Rows of queries and cache are 16-byte aligned,
 * of out 8-byte; a cache stride may be up to 2^31 - 1 elements (offsets are 64
 * bits wide). The workspace (16-byte aligned, contents
 * ignored and overwritten) has at least pcamd_latent_decode_workspace() bytes;
 * a negative result of that call is a status.
 */
int64_t pcamd_latent_decode_workspace(int64_t batch, int64_t new_tokens,
                                      int64_t heads, int64_t latent_dim,
                                      int64_t page_size, int64_t max_pages);
int pcamd_latent_decode(const void *q_latent, const void *q_rope, int dtype,
                        int64_t batch, int64_t new_tokens, int64_t heads,
                        int64_t latent_dim, int64_t rope_dim, int64_t qlb,
                        int64_t qls, int64_t qlh, int64_t qrb, int64_t qrs,
                        int64_t qrh, const void *cache_latent, int cache_dtype,
                        int64_t clp, int64_t clt, const void *cache_rope,
                        int64_t crp, int64_t crt, const float *cache_scale,
                        int64_t csp, int64_t cst, int64_t pages,
                        int64_t page_size, const int32_t *table,
                        int64_t table_stride, int64_t max_pages,
                        const int32_t *lens, void *out, int64_t ob, int64_t os,
                        int64_t oh, float *lse, int64_t lb, int64_t ls,
                        int64_t lh, float softmax_scale, void *workspace,
                        int64_t workspace_bytes, void *stream);

/*
 * Attention of packed sequences with expanded keys: head h of key token t has
 * the key [k_nope[t, h] | k_rope[t]] and the value v[t, h]; sequence i holds
 * the queries cu_q[i] .. cu_q[i + 1] - 1 and the keys cu_k[i] .. cu_k[i + 1] -
 * 1 (offsets beyond the tensors are cut to them). causal: query i of nq sees
 * the first nk - nq + i + 1 keys of nk. out [total_q, heads, v_dim], lse
 * [total_q, heads] (may be NULL); queries that see no key, and those ahead of
 * the first sequence or behind the last, give zeros and -inf. nope_dim,
 * rope_dim and v_dim are 128, 64 and 128, or 64, 32 and 64. Rows of q, k_nope,
 * k_rope and v are 16-byte aligned, of out 8-byte; up to 2^30 tokens, and up to
 * 2^30 elements from one key's (value's) token to the next.
 */
int pcamd_latent_prefill(const void *q, const void *k_nope, const void *k_rope,
                         const void *v, int dtype, int64_t total_q,
                         int64_t total_k, int64_t heads, int64_t nope_dim,
                         int64_t rope_dim, int64_t v_dim, int64_t sqt,
                         int64_t sqh, int64_t skt, int64_t skh, int64_t srt,
                         int64_t svt, int64_t svh, const int32_t *cu_q,
                         const int32_t *cu_k, int64_t sequences, void *out,
                         int64_t sot, int64_t soh, float *lse, int64_t slt,
                         int64_t slh, float softmax_scale, int causal,
                         void *stream);

/*
 * Int8 codes of x[batch, m, n] (fp32, bf16 or fp16, contiguous along n, any
 * row strides and alignment) with one scale a row: top = max(max|x|, eps),
 * scale[b, i] = top / 127 (fp32 division), y = rint(127 x / top) of the real
 * quotient, ties to even. A row with a NaN or an infinity gets the scale NaN
 * and codes of zero. Rows of y are 16-byte aligned and written up to the next
 * multiple of 16 bytes, with zeros behind n. n is at most 2^31 - 16385.
 * Available from PCAMD_ABI_VERSION 7, as the functions below. No counterpart in
 * the reference, whose quantizers are fp8
 * (fp8_training/fp8_bench/impls/triton_per_channel.py:90-219).
 */
int pcamd_quant_int8(const void *x, int x_dtype, int64_t batch, int64_t m,
                     int64_t n, int64_t sxb, int64_t sxm, void *y, int64_t syb,
                     int64_t sym, float *scale, int64_t ssb, int64_t ssm,
                     float eps, void *stream);

/*
 * c[b, i, j] = act(sum_k a[b, i, k] b[b, j, k] * (sa[b, i] * sb[b, j]) +
 * bias[b, i, j]) for int8 a[batch, m, k] and b[batch, n, k], both contiguous
 * along k with 16-byte aligned rows; c is fp32, bf16 or fp16, contiguous along
 * its columns. Sums are exact (int32), k goes up to 131071. PCAMD_ACT_SWIGLU:
 * b has 2 n rows (and sb and bias as many columns), c[.., j] = silu(column j)
 * * column n + j. Bytes of a row up to the next multiple of 16 may be read and
 * do not count.
 */
int pcamd_bmm_int8(const void *a, const void *b, int64_t batch, int64_t m,
                   int64_t n, int64_t k, int64_t sab, int64_t sam, int64_t sbb,
                   int64_t sbn, void *c, int c_dtype, int64_t scb, int64_t scm,
                   const void *bias, int bias_dtype, int64_t sbiasb,
                   int64_t sbiasm, int64_t sbiasn, const float *sa,
                   int64_t ssab, int64_t ssam, const float *sb, int64_t ssbb,
                   int64_t ssbn, int activation, void *stream);

/*
 * Pairs (token, choice) sorted by expert, stable: ids[pairs] (id_bytes 4 or 8:
 * int32, int64), order[place] = pair, place[pair] = its place, starts[experts
 * + 1] the first place of each expert and the end of the last. Pairs whose id
 * is negative or not below experts come last, in their own order, and have
 * place -1 - place. Up to 1024 experts and 2^31 - 1 pairs. The workspace has
 * at least pcamd_expert_sort_workspace() bytes; a negative result of that call
 * is a status.
 */
int64_t pcamd_expert_sort_workspace(int64_t pairs, int64_t experts);
int pcamd_expert_sort(const void *ids, int id_bytes, int64_t pairs,
                      int64_t experts, int32_t *order, int32_t *place,
                      int32_t *starts, void *workspace, int64_t workspace_bytes,
                      void *stream);

/*
 * Rows to the order of experts and back (place[tokens, choices] as above;
 * fp32, bf16 or fp16, contiguous along width, up to 128 choices):
 *   dispatch: out[place] = x[token], zeros at the places of pairs without one;
 *   combine: out[t] = sum_j weights[t, j] rows[place[t, j]] in fp32, choices
 *     ascending, pairs without an expert left out; weights [tokens, choices]
 *     contiguous (w_dtype), or NULL for ones (the gradient of dispatch);
 *   combine_backward: grad_rows[place] = weights[t, j] grad[t] (zeros for
 *     pairs without an expert) and grad_weights[t, j] = rows[place] . grad[t]
 *     (fp32; 0 for those); either may be NULL.
 */
int pcamd_expert_dispatch(const void *x, int dtype, int64_t tokens,
                          int64_t choices, int64_t width, int64_t sxt,
                          const int32_t *place, void *out, int64_t sos,
                          void *stream);
int pcamd_expert_combine(const void *rows, int dtype, int64_t tokens,
                         int64_t choices, int64_t width, int64_t srs,
                         const int32_t *place, const void *weights, int w_dtype,
                         void *out, int64_t sot, void *stream);
int pcamd_expert_combine_backward(const void *grad, const void *rows, int dtype,
                                  int64_t tokens, int64_t choices,
                                  int64_t width, int64_t sgt, int64_t srs,
                                  const int32_t *place, const void *weights,
                                  int w_dtype, void *grad_rows, int64_t sos,
                                  float *grad_weights, void *stream);

/*
 * The int8 product grouped by expert: rows starts[e] .. starts[e + 1] - 1 of
 * c[pairs, n] are rows of a times b[e] (b[experts, n, k]; 2 n rows each with
 * PCAMD_ACT_SWIGLU), with sa[row of a], sb[e, column] and bias[e, column].
 * Row s of c takes row s of a, or where order is given row order[s] / choices
 * (a then holds pairs / choices tokens; any number where both are 0). Rows
 * behind starts[experts] are written as zeros.
 */
int pcamd_expert_bmm_int8(const void *a, int64_t a_rows, const void *b,
                          int64_t experts, int64_t n, int64_t k, int64_t sam,
                          int64_t sbe, int64_t sbn, void *c, int c_dtype,
                          int64_t scm, const void *bias, int bias_dtype,
                          int64_t sbiase, int64_t sbiasn, const float *sa,
                          int64_t ssam, const float *sb, int64_t ssbe,
                          int64_t ssbn, const int32_t *starts,
                          const int32_t *order, int64_t pairs, int64_t choices,
                          int activation, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* PCAMD_FP8_H */
