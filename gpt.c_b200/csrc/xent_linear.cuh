// What the kernels of projection and loss share.
#pragma once

#include "attn_internal.h"
#include "ids.cuh"

namespace head {

// The forward of up to kFewRows rows (xent_few_sm100.cu): maxima and sums of each row over the classes of each CTA.
constexpr int kFewRows = 64;
struct FewRows {
    const void *x, *w;
    long long ldx, ldw;
    Ids targets;
    float2 *part;  // [few_rows_parts, M]
    float *zt;     // the targets' logits
    int M, V, K;
};
bool few_rows_fit(const void *x, const void *w, long long ldx, long long ldw, int type, int M, int V, int K, int sms);
int few_rows_parts(int V, int sms);
cudaError_t launch_few_rows(const FewRows &a, int type, int sms, cudaStream_t s);
cudaError_t few_rows_set_attributes();

}  // namespace head
