// The call that the two attention kernels over a paged cache share (paged_attn_sm100.cu, paged_tile_sm100.cu).
#pragma once

#include "paged.cuh"

namespace paged {

struct Call {
    Cache c;
    const float *q;
    float *out;
    long long ld;
    int heads, max_new, type;
    float scale_log2;
    int *status;
    cudaStream_t s;
};

// Sequences with more than `few` rows (new tokens x query heads of a group), D <= 128.
cudaError_t launch_tiles(const Call &a, int few);
cudaError_t tiles_set_attributes();
cudaError_t few_rows_set_attributes();

}  // namespace paged
