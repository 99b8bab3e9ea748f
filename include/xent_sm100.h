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

#ifdef __cplusplus
}
#endif

#endif /* XENT_SM100_H */
