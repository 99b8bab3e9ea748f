// What the kernels of projection and loss share.
#pragma once

#include "attn_internal.h"
#include "ids.cuh"

namespace head {

// The tensor cores cut every sum of 16 products and what was there off to fp32: a sum of n such steps that grows evenly is on average n / 4 half
// units too small, and so were the logits (K = 1600: by 28 2^-24 of themselves in bf16 and 86 in fp32, which has three products; 4096: by 68
// and 212).  z as the tensor cores leave it times fix_of() is z.  (Without it the log-sum-exp of logits of standard deviation 30 is 1.6e-6 off, with it 5e-7.)
// That is an average over values of many bits, which activations and weights are.  Where nothing is cut off (one feature that is not zero, small whole numbers, rows filled
// up with zeros) logits are too large by it: 13 2^-24 of themselves for 768 bf16 features, 215 (1.3e-5) for 4096 of fp32, as far off as they would be too small otherwise.  Sums that
// end every few steps would need no such factor; the warps that would add them up have no registers for 128 of them a thread.
constexpr double kCut = 0.28 / 16777216.0;  // of a step
inline double fix_of(int K, int type) { return 1.0 + kCut * ((K + 15) / 16 * (type == TENSOR_F32 ? 3 : 1)); }

// Up to kFewRows rows (xent_few_sm100.cu).  The forward: maxima and sums of each row over the classes of each CTA.  The backward of up to 16 rows, where grad_g
// is given: G, then the products.
constexpr int kFewRows = 48;
struct FewRows {
    const void *x, *w;
    long long ldx, ldw;
    Ids targets;
    float2 *part;  // [few_rows_parts, M]
    float *zt;     // the targets' logits
    int M, V, K;
    const float *grad_g, *lse;
    int one_g;
    float *G;      // [V, few_rows_stride]
    float fix;
};
bool few_rows_fit(const void *x, const void *w, long long ldx, long long ldw, int type, int M, int V, int K, int sms);
int few_rows_parts(int V, int sms);
cudaError_t launch_few_rows(const FewRows &a, int type, int sms, cudaStream_t s);
cudaError_t few_rows_set_attributes();
int few_rows_stride(int M);
bool few_rows_gradients_fit(const void *x, const void *w, const void *dw, long long ldx, long long ldw, long long lddw, int type, int M, int V, int K);
int few_rows_pieces(int M, int V, int K, int sms);  // of dx, to be added up
cudaError_t launch_few_rows_products(const FewRows &a, int type, void *dw, long long lddw, float *dxp, int dx_pitch, int sms, cudaStream_t s);

}  // namespace head
