// What the kernels of projection and loss share.
#pragma once

#include "attn_internal.h"
#include "ids.cuh"

namespace head {

// Up to kFewRows rows (xent_few_sm100.cu).  The forward: maxima and sums of each row over the classes of each CTA.  The backward of up to 16 rows, where grad_g
// is given: G, then the products.
constexpr int kFewRows = 64;
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
