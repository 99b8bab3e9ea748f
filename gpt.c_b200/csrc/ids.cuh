// Tokens, positions and targets: int32, int64, or fp32 as gpt.c's data loader makes them.
#pragma once

#include "../../include/tensor_sm100.h"

struct Ids {
    const void *p;
    int type;
    // The i-th one; -1 where it is none of 0 .. V - 1 (fp32: of its whole part, as the reference casts it).
    __device__ __forceinline__ int at(long long i, int V) const {
        if (type == TENSOR_INT64) {
            const long long t = static_cast<const long long *>(p)[i];
            return t >= 0 && t < V ? (int)t : -1;
        }
        if (type == TENSOR_INT32) {
            const int t = static_cast<const int *>(p)[i];
            return t >= 0 && t < V ? t : -1;
        }
        const float t = static_cast<const float *>(p)[i];
        return t > -1.f && t < (float)V && (int)t < V ? (int)t : -1;
    }
    // The ones at i, i + step, .. (from the one at end - 1 on, that one): asked for together.
    template <int kN>
    __device__ __forceinline__ void many(int (&out)[kN], int V, long long i, int step, long long end) const {
        if (type == TENSOR_INT64) {
            long long t[kN];
#pragma unroll
            for (int r = 0; r < kN; r++) t[r] = static_cast<const long long *>(p)[min(i + (long long)r * step, end - 1)];
#pragma unroll
            for (int r = 0; r < kN; r++) out[r] = t[r] >= 0 && t[r] < V ? (int)t[r] : -1;
        } else {
            int t[kN];
#pragma unroll
            for (int r = 0; r < kN; r++) t[r] = static_cast<const int *>(p)[min(i + (long long)r * step, end - 1)];
#pragma unroll
            for (int r = 0; r < kN; r++) {
                const float f = __int_as_float(t[r]);
                if (type == TENSOR_IDS_F32) t[r] = f > -1.f && f < (float)V ? (int)f : -1;
                out[r] = t[r] >= 0 && t[r] < V ? t[r] : -1;
            }
        }
    }
};
