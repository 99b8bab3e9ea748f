/*
 * xent_sm100.h: C ABI of the B200 (sm_100a) cross-entropy kernels (the loss over the vocabulary
 * projection at the end of gpt.c's transformer).  Same library and conventions as attn_sm100.h
 * (device pointers on the current device, row-major fp32, any 4-byte alignment, work only enqueued on
 * `stream`, ATTN_OK / negative ATTN_ERR_* / positive cudaError_t).
 *
 * Reference interfaces these entry points replace (paths relative to the gpt.c project root):
 *
 *   xent_sm100_forward    cross_entropy_forward_cuda_kernel    kernels/src/cuda/CrossEntropyLoss.cu:136-156 (kernel :8-79)
 *   xent_sm100_backward   cross_entropy_backward_cuda_kernel   kernels/src/cuda/CrossEntropyLoss.cu:158-178 (kernel :82-129)
 *   (declared kernels/src/cuda/CrossEntropyLoss.h:9-20); CPU counterparts: kernels/src/cpu/CrossEntropyLoss.c
 */
#ifndef XENT_SM100_H
#define XENT_SM100_H

#include "attn_sm100.h"
#include "tensor_sm100.h" /* types of elements and indices */

#ifdef __cplusplus
extern "C" {
#endif

/*
 * logsm[r, :] = log_softmax(logits[r, :]);  *loss += sum_r -logsm[r, (int)targets[r]] / rows.
 * targets holds class indices as floats (the reference's convention); *loss must be initialised by the
 * caller (the reference's layer hands in zeros).  rows = B*T, C = classes.
 */
int xent_sm100_forward(const float *logits, const float *targets, float *logsm, float *loss, int rows, int C, void *stream);

/*
 * What the forward does when rows never arrive, without a fault: the same kernel, for rows of 30000 to 53248 classes, fetches only
 * the first `loaded` rows.  Its waits for the others run out after limit_us microseconds (at most 0.1 s), attn_sm100_device_status
 * reports 1252, and the rows before them are complete.  (The reference has no counterpart.)
 */
int xent_sm100_selftest_wait_limit(const float *logits, const float *targets, float *logsm, float *loss, int rows, int C, int loaded,
                                   unsigned limit_us, void *stream);

/*
 * dout[r, target_r] = -g[r] / rows;  s = sum_j dout[r, j];  dout[r, j] -= exp(logsm[r, j]) * s.
 * Works on what dout holds (read-modify-write), like the reference, whose layer hands in zeros; g has one
 * value per row.
 */
int xent_sm100_backward(const float *g, const float *targets, const float *logsm, float *dout, int rows, int C, void *stream);

/*
 * Draws a class from each row of logits with given random numbers.  (The reference's infer_gpt.c:341-408 divides by the temperature,
 * takes the softmax on the GPU and draws on the host; it has no top-k, top-p or min-p.)  Row r, with classes in the order of falling
 * logits, equal ones by index:
 *     w_i = exp((x_i - max x) / temperature[r])
 *     kept: the first top_k[r] classes; of these the shortest run from the front with at least top_p[r] of their weight, one at
 *           least; of these the ones with w_i >= min_p[r]
 *     tokens[r] = the first class, in the order of the index, at which the running sum of the kept weights exceeds u[r] times their sum
 * Each of temperature, top_k, top_p and min_p has one value a row, or is NULL (1, all, all, all).  temperature <= 0 or NaN: the
 * largest logit, the first of equal ones.  top_k outside 1 .. C - 1, top_p >= 1 and min_p <= 0, or NaN, restrict nothing; top_p <= 0 and
 * min_p >= 1 keep the classes of the largest logit only, the first of them and all of them.  u is in [0, 1) (outside: the nearest
 * number inside; NaN: 0).  A logit of +inf has all the weight, one of -inf none; a row with a NaN, or of -inf alone, has no
 * class to draw: its token is -1.
 * Weights are 64-bit whole numbers, 2^-44 of the largest one each, so that every sum is exact and the token does not depend on the order in
 * which they are added; C is at most 425984.  Rows are `ld` elements apart (any number from C on).
 */
int xent_sm100_sample(const float *logits, const float *u, const float *temperature, const int *top_k, const float *top_p,
                      const float *min_p, int *tokens, long long ld, int rows, int C, void *stream);

/*
 * The vocabulary projection and the loss in one: z = x . w^T is never in memory.  (The reference keeps the logits, their log-softmax and
 * their gradient: src/transformer.c:107-108, kernels/src/cuda/CrossEntropyLoss.cu.)
 *
 *   x [rows, K], w [V, K]   `type` TENSOR_F32 or TENSOR_BF16, rows ldx and ldw elements apart, any alignment of whole elements
 *   targets [rows]          `target_type` TENSOR_INT32, TENSOR_INT64 or TENSOR_IDS_F32 (the reference's); a row whose target is not in 0 .. V - 1
 *                           has no loss and no part in the gradients, whatever its x holds
 *   lse[r]    = log sum_v exp z[r, v]
 *   losses[r] = lse[r] - z[r, targets[r]], 0 for a row without a target
 *
 * The products of bf16 tensors are exact, those of fp32 tensors are made of two bf16 terms of each factor (16 bits of it; values
 * above 3.38e38 in size have none); sums are fp32.  The tensor cores cut sums off: logits are multiplied by what that takes on average, 1 + 0.28 2^-24 for each
 * 16 features (fp32 tensors: three times that), so where nothing is cut off, as with one feature that is not zero, they are too large by it (768 bf16 features: 8e-7
 * of themselves; 4096 of fp32: 1.3e-5).  rows may be 0.  Outputs overlap no input and not each other.
 * Up to 2^30 rows and classes and 2^24 features, rows of x and w up to 2^34 elements apart; ATTN_ERR_UNSUPPORTED beyond.
 * scratch: xent_sm100_linear_forward_scratch_bytes bytes for the same arguments on the same device, 256-byte aligned.  (Of the tensors their
 * alignment matters there: bf16 ones on 16-byte boundaries are read where they are, others copied.)
 */
size_t xent_sm100_linear_forward_scratch_bytes(const void *x, const void *w, long long ldx, long long ldw, int type, int rows, int V, int K);
int xent_sm100_linear_forward(const void *x, const void *w, const void *targets, float *losses, float *lse, void *scratch,
                              long long ldx, long long ldw, int type, int target_type, int rows, int V, int K, void *stream);

/*
 * What that call does when operands never arrive, without a fault: the same kernels, for more than 48 rows, ask only for the operands of the first `loaded` tiles
 * (256 rows by up to 256 classes).  The waits for the others run out after their second, attn_sm100_device_status reports 1302 or 1304, whichever
 * wait was first, and losses and lse are not defined.
 */
int xent_sm100_selftest_linear_wait_limit(const void *x, const void *w, const void *targets, float *losses, float *lse, void *scratch,
                                          long long ldx, long long ldw, int type, int target_type, int rows, int V, int K, int loaded,
                                          void *stream);

/*
 * Its gradients, with lse from the forward call on the same x, w and targets:
 *     G[r, v]  = g[r] (exp(z[r, v] - lse[r]) - [v = targets[r]])    g has one value per row, or one in all (one_g); 0 without a target
 *     dx[r, :] = sum_v G[r, v] w[v, :]      overwritten, rows K elements apart, of `type`; may be NULL
 *     dw[v, :] += sum_r G[r, v] x[r, :]     rows lddw elements apart, of `type`, one rounding a call (fp32: one for every 1024 rows; values below 2^-126 in size
 *                                           may become 0, L2 adds); may be NULL, but not both
 * With bf16 tensors G is rounded to bf16 before these products (above 8 rows; without the significand of the largest |g| of a row that has a target, which the
 * sums are multiplied by: one factor for all rows costs no accuracy), with fp32 tensors it is two bf16 terms like the others, and above 16 rows dx and dw are multiplied by
 * what the tensor cores cut off of them on average, up to 1 + 2.9e-6.  The results
 * have the same bits in every call on GPUs of as many SMs.
 * G is in memory for two pieces of the vocabulary at a time, up to 256 MB each, or 16384 bytes a row (fp32 32768) where that is more:
 * scratch of xent_sm100_linear_backward_scratch_bytes bytes, which also has room for dx in fp32 and for copies of x and, if fp32, of w;
 * 256-byte aligned.  Up to 2^20 rows.  dx and dw overlap each other and the inputs in no byte (rows of one inside the gaps of another count as that).
 */
size_t xent_sm100_linear_backward_scratch_bytes(const void *x, const void *w, long long ldx, long long ldw, int type, int rows, int V, int K);
int xent_sm100_linear_backward(const float *g, const void *x, const void *w, const void *targets, const float *lse, void *dx, void *dw,
                               void *scratch, long long ldx, long long ldw, long long lddw, int one_g, int type, int target_type, int rows,
                               int V, int K, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* XENT_SM100_H */
