/*
 * tensor_sm100.h: C ABI of the B200 (sm_100a) element-wise tensor helpers: the fills, copies and
 * residual adds around the attention layer in every gpt.c block.  Same library and conventions as
 * attn_sm100.h (device pointers on the current device, work only enqueued on `stream`, ATTN_OK /
 * negative ATTN_ERR_* / positive cudaError_t); any alignment is accepted, 16-byte aligned pointers
 * take the vectorised path.  n == 0 is a no-op.
 *
 * Reference interfaces these entry points replace (paths relative to the gpt.c project root):
 *
 *   tensor_sm100_fill     zeros/ones/fill_tensor_data_cuda   kernels/src/cuda/Tensor.cu:79-107 (kernel :8-13)
 *   tensor_sm100_arange   arange_tensor_data_cuda            kernels/src/cuda/Tensor.cu:109-117 (kernel :15-20)
 *   tensor_sm100_copy     copy_tensor_data_cuda              kernels/src/cuda/Tensor.cu:119-130 (kernel :22-27)
 *   tensor_sm100_axpy     saxpy_cuda with unit strides       kernels/src/cuda/Tensor.cu:132-141 (cublasSaxpy)
 *   tensor_sm100_gelu_forward / _backward   gelu_forward/backward_cuda_kernel   kernels/src/cuda/GeLU.cu:40-64 (kernels :5-38)
 */
#ifndef TENSOR_SM100_H
#define TENSOR_SM100_H

#include "attn_sm100.h"

#ifdef __cplusplus
extern "C" {
#endif

/* p[i] = value for i < n. */
int tensor_sm100_fill(float *p, size_t n, float value, void *stream);
/* p[i] = (float)(start + step * i), the integer expression of the reference. */
int tensor_sm100_arange(float *p, size_t n, int start, int step, void *stream);
/* dst[i] = src[i]; the ranges must not overlap. */
int tensor_sm100_copy(float *dst, const float *src, size_t n, void *stream);
/* y[i] = alpha * x[i] + y[i], one fused multiply-add per element. */
int tensor_sm100_axpy(size_t n, float alpha, const float *x, float *y, void *stream);
/* y[i] = 0.5 x (1 + tanh(sqrt(2/pi) (x + 0.044715 x^3))): the tanh approximation of GELU the reference uses. */
int tensor_sm100_gelu_forward(const float *x, float *y, size_t n, void *stream);
/* dx[i] = g[i] * d/dx of the above at x[i] (overwritten, like the reference). */
int tensor_sm100_gelu_backward(const float *g, const float *x, float *dx, size_t n, void *stream);

/* Types of elements, and of tokens, positions and targets (the reference's dataloader.c:67-70 makes them fp32). */
#define TENSOR_F32 0
#define TENSOR_BF16 1
#define TENSOR_INT32 0
#define TENSOR_INT64 1
#define TENSOR_IDS_F32 2

/*
 * y[t, :] = scale * table[tokens[t], :] + pos_table[positions[t], :] for t < n, computed in fp32 and rounded once.
 *   table [V, C], pos_table [P, C]   of `type`, rows ld and pos_ld elements apart; pos_table may be NULL
 *   tokens, positions [n]            of `id_type`; positions NULL: t % T, a token's place in its sequence of T
 *   y [n, C]                         of `type`, contiguous
 * A token outside 0 .. V - 1 (padding), or a position outside 0 .. P - 1, brings zeros.
 * Up to 2^20 columns, and 2^40 values of y; ATTN_ERR_UNSUPPORTED beyond.  y overlaps no input.
 * The reference's counterpart is embedding_forward_cuda_kernel (kernels/src/cuda/Embedding.cu:46-58), without scale and positions.
 */
int tensor_sm100_embedding_forward(const void *tokens, const void *table, const void *positions, const void *pos_table, void *y, long long n,
                                   long long ld, long long pos_ld, float scale, int type, int id_type, int T, int C, int V, int P, void *stream);

/*
 * dtable[v, :]     += scale * sum of dy[t, :] over tokens[t] = v
 * dpos_table[p, :] += sum of dy[t, :] over positions[t] = p
 *   dy [n, C] of `type`, rows ld_dy elements apart; dtable [V, C], dpos_table [P, C] of `grad_type`, rows ld and pos_ld elements apart; one of
 *   them may be NULL.  None of the three may overlap another (rows of one inside the gaps of another count as that), nor the gradients tokens or positions.
 * Sums are fp32 in an order that the sizes fix, rounded once where grad_type is TENSOR_BF16: the same bits in every call.  Tokens and positions
 * outside their table have no part.  Rows that no token names are neither read nor written.
 * An fp32 gradient, what it holds or becomes, that is below 2^-126 in size may become 0 (L2 adds).
 * scratch: tensor_sm100_embedding_backward_scratch_bytes bytes with P = 0 unless positions are given and V = 0 without dtable,
 * 256-byte aligned (may be NULL if that is 0).
 * Up to 2^30 places, 2^20 columns and 2^30 rows of a table; ATTN_ERR_UNSUPPORTED beyond.
 * The reference's counterpart is embedding_backward_cuda_kernel (kernels/src/cuda/Embedding.cu:60-74): an atomic addition a value.
 */
size_t tensor_sm100_embedding_backward_scratch_bytes(long long n, int C, int V, int P);
int tensor_sm100_embedding_backward(const void *dy, const void *tokens, void *dtable, const void *positions, void *dpos_table, void *scratch,
                                    long long n, long long ld_dy, long long ld, long long pos_ld, float scale, int type, int grad_type,
                                    int id_type, int T, int C, int V, int P, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* TENSOR_SM100_H */
