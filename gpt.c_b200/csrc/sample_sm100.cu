// The draw of a class from each row of logits, by temperature, top-k, top-p and min-p, for sm_100a.
//
// With the classes ordered by falling logit, equal ones by index, what each restriction keeps is a run from the front of
// that order, so the classes kept are those above one logit and the first few that equal it.  A weight is a whole number,
// round(2^44 exp((x - max) / T)): sums of up to 2^18 of them fit 64 bits and are exact in any order.
//
// One block per row.  The logit that ends the run is found bit by bit from the top of its order-preserving 32-bit key: 32 passes over the
// row, which stays in L2, each counting the classes (or adding up the weights) at and above a key.
#include "attn_internal.h"
#include "tc05.cuh"

#include "../../include/xent_sm100.h"

namespace sample {
namespace {

constexpr int kThreads = 1024, kWarps = kThreads / 32;
constexpr int kMaxC = 425984;
typedef unsigned long long u64;

// The order of fp32 numbers as that of 32-bit ones (-0 counts as +0).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

struct Row {
    const float *x;
    int C;
    float max;
    double inv_t;
};

__device__ __forceinline__ u64 weight(const Row &r, float x) {
    if (x == r.max) return 1ull << 44;
    if (x == -INFINITY || r.max == INFINITY) return 0;
    return __double2ull_rn(exp(((double)x - (double)r.max) * r.inv_t) * 17592186044416.0);
}

template <class T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The same total for every thread.  `at` is free again for the call after the next.
__device__ u64 block_sum(u64 v, u64 *at) {
    v = warp_sum(v);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) at[threadIdx.x >> 5] = v;
    __syncthreads();
    return warp_sum(at[threadIdx.x & 31]);
}

// Index of the first class, in the order of the index, at which the running sum of f exceeds `above` (which the sum of all does).
template <class F>
__device__ int first_above(const Row &r, F f, u64 above, u64 *at, int *found) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, each = ((r.C + kWarps - 1) / kWarps + 31) / 32 * 32;
    const int begin = min(warp * each, r.C), end = min(begin + each, r.C);
    u64 sum = 0;
    for (int i = begin + lane; i < end; i += 32) sum += f(i);
    sum = warp_sum(sum);
    __syncthreads();
    if (lane == 0) at[warp] = sum;
    __syncthreads();
    u64 before = 0;
    for (int w = 0; w < warp; w++) before += at[w];
    if (before <= above && before + sum > above) {  // one warp
        for (int i = begin + lane; i - lane < end; i += 32) {
            u64 run = i < end ? f(i) : 0;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const u64 left = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += left;
            }
            const uint32_t hit = __ballot_sync(0xffffffffu, before + run > above);
            if (hit) {
                if (lane == __ffs(hit) - 1) *found = i;
                break;
            }
            before += __shfl_sync(0xffffffffu, run, 31);
        }
    }
    __syncthreads();
    return *found;
}

__global__ void __launch_bounds__(kThreads) sample_kernel(const float *logits, const float *u, const float *temperature, const int *top_k,
                                                          const float *top_p, const float *min_p, int *tokens, long long ld, int C) {
    __shared__ u64 at[32];
    __shared__ int found;
    tc05::pdl_launch_dependents();
    tc05::pdl_wait();
    const int row = blockIdx.x;
    Row r{logits + row * ld, C, -INFINITY, 1.0};
    bool bad = false;
    for (int i = threadIdx.x; i < C; i += kThreads) {
        const float x = r.x[i];
        r.max = fmaxf(r.max, x);
        bad |= x != x;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.max = fmaxf(r.max, __shfl_xor_sync(0xffffffffu, r.max, o));
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) tokens[row] = -1;
        return;
    }
    float *most = reinterpret_cast<float *>(at);
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = r.max;
    __syncthreads();
    r.max = most[threadIdx.x & 31];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) r.max = fmaxf(r.max, __shfl_xor_sync(0xffffffffu, r.max, o));
    if (r.max == -INFINITY) {
        if (threadIdx.x == 0) tokens[row] = -1;
        return;
    }
    const float T = temperature ? temperature[row] : 1.f;
    if (!(T > 0.f)) {
        const int first = first_above(r, [&](int i) { return (u64)(r.x[i] == r.max); }, 0, at, &found);
        if (threadIdx.x == 0) tokens[row] = first;
        return;
    }
    r.inv_t = 1.0 / (double)T;

    // the classes kept: keys above `edge`, and those equal to it up to class `upto`
    uint32_t edge = 0;
    int upto = C - 1;
    const int k = top_k ? top_k[row] : 0;
    const float p = top_p ? top_p[row] : 1.f, least = min_p ? min_p[row] : 0.f;
    const bool by_k = k >= 1 && k < C, by_p = p < 1.f;
    u64 ties = 0;  // of them kept
    if (by_k) {
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t key = edge | (1u << bit);
            u64 n = 0;
            for (int i = threadIdx.x; i < C; i += kThreads) n += key_of(r.x[i]) >= key;
            if (block_sum(n, at) >= (u64)k) edge = key;
        }
        u64 n = 0;
        for (int i = threadIdx.x; i < C; i += kThreads) n += key_of(r.x[i]) > edge;
        ties = (u64)k - block_sum(n, at);
    }
    if (by_p) {
        const float last = __uint_as_float(edge & 0x80000000u ? edge & 0x7fffffffu : ~edge);
        const u64 tied = by_k ? ties * weight(r, last) : 0;
        u64 n = 0;
        for (int i = threadIdx.x; i < C; i += kThreads) n += (!by_k || key_of(r.x[i]) > edge) ? weight(r, r.x[i]) : 0;
        const u64 mass = block_sum(n, at) + tied;
        // the smallest whole number that is at least p * mass
        const u64 share = p > 0.f ? (u64)((double)p * 18446744073709551616.0) : 0;
        u64 need = __umul64hi(share, mass) + (share * mass != 0);
        if (need == 0) need = 1;
        uint32_t cut = 0;
        for (int bit = 31; bit >= 0; bit--) {
            const uint32_t key = cut | (1u << bit);
            if (by_k && key <= edge) {  // all of them
                cut = key;
                continue;
            }
            u64 sum = 0;
            for (int i = threadIdx.x; i < C; i += kThreads) sum += key_of(r.x[i]) >= key ? weight(r, r.x[i]) : 0;
            if (block_sum(sum, at) >= need) cut = key;
        }
        u64 sum = 0;
        for (int i = threadIdx.x; i < C; i += kThreads) sum += key_of(r.x[i]) > cut ? weight(r, r.x[i]) : 0;
        sum = block_sum(sum, at);
        const u64 one = weight(r, __uint_as_float(cut & 0x80000000u ? cut & 0x7fffffffu : ~cut));
        const u64 some = one ? (need - sum + one - 1) / one : 0;
        ties = by_k && cut == edge && ties < some ? ties : some;
        edge = cut;
    }
    if (by_k || by_p) {
        upto = first_above(r, [&](int i) { return (u64)(key_of(r.x[i]) == edge); }, ties - 1, at, &found);
        __syncthreads();
    }
    const u64 lowest = least > 0.f ? (least < 1.f ? (u64)ceil((double)least * 17592186044416.0) : 1ull << 44) : 0;
    auto kept = [&](int i) -> u64 {
        const uint32_t key = key_of(r.x[i]);
        if (key < edge || (key == edge && i > upto)) return 0;
        const u64 w = weight(r, r.x[i]);
        return w >= lowest ? w : 0;
    };
    u64 sum = 0;
    for (int i = threadIdx.x; i < C; i += kThreads) sum += kept(i);
    sum = block_sum(sum, at);
    const float v = u[row];
    const u64 part = v >= 1.f ? ~0ull : v > 0.f ? (u64)((double)v * 18446744073709551616.0) : 0;
    const int token = first_above(r, kept, __umul64hi(part, sum), at, &found);
    if (threadIdx.x == 0) tokens[row] = token;
}

}  // namespace
}  // namespace sample

extern "C" int xent_sm100_sample(const float *logits, const float *u, const float *temperature, const int *top_k, const float *top_p,
                                 const float *min_p, int *tokens, long long ld, int rows, int C, void *stream) {
    if (!logits || !u || !tokens) return ATTN_ERR_NULL;
    if (rows < 0 || C <= 0 || ld < C) return ATTN_ERR_ARGUMENT;
    if (C > sample::kMaxC) return ATTN_ERR_UNSUPPORTED;
    int *status = nullptr;
    const int rc = attn::device_status_word(&status);
    if (rc != ATTN_OK) return rc;
    if (rows == 0) return ATTN_OK;
    return (int)attn::launch_after_previous(sample::sample_kernel, dim3((unsigned)rows), dim3(sample::kThreads), 0, static_cast<cudaStream_t>(stream), logits, u,
                                            temperature, top_k, top_p, min_p, tokens, ld, C);
}
