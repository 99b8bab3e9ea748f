// What the attention kernels over a paged cache share (paged_attn_sm100.cu, paged_decode_sm100.cu, paged_tile_sm100.cu).
#pragma once

#include "attn24.cuh"
#include "attn_internal.h"
#include "paged.cuh"

namespace paged {

using namespace attn24;

__device__ __forceinline__ void cp16(uint32_t dst, const void *src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
// One of the arrivals that `bar` waits for, once this thread's copies so far are there.
__device__ __forceinline__ void arrive_when_copied(uint64_t *bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int kN>
__device__ __forceinline__ void cp_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(kN) : "memory"); }

// A warp's arrival after what its lanes did to tensor memory.
__device__ __forceinline__ void arrive_tmem(uint64_t *bar, int lane) {
    tc_fence_before_sync();
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
}

// x - hi for both halves of a pair of bf16 values, exact where hi is the upper half of x.
__device__ __forceinline__ float2 less(float2 x, uint32_t hi) {
    float2 r;
    asm("{\n\t.reg .b16 a, b, m;\n\tmov.b32 {a, b}, %2;\n\tmov.b16 m, 0xbf80;\n\tfma.rn.f32.bf16 %0, a, m, %3;\n\tfma.rn.f32.bf16 %1, b, m, %4;\n\t}"
        : "=f"(r.x), "=f"(r.y)
        : "r"(hi), "f"(x.x), "f"(x.y));
    return r;
}
// p = hi + mid + lo, each the next eight bits cut off: exact.
__device__ __forceinline__ void cut3(float2 p, uint32_t &hi, uint32_t &mid, uint32_t &lo) {
    hi = __byte_perm(__float_as_uint(p.x), __float_as_uint(p.y), 0x7632);
    const float2 r = less(p, hi);
    mid = __byte_perm(__float_as_uint(r.x), __float_as_uint(r.y), 0x7632);
    const float2 s = less(r, mid);
    lo = __byte_perm(__float_as_uint(s.x), __float_as_uint(s.y), 0x7632);
}

// Element offset of key j's row from that of its head, -1 where it has no page.
__device__ __forceinline__ long long place(const Cache &c, const int *table, int j, int end, bool &missing) {
    if (j >= end) return -1;
    const int slot = j / c.page_size, page = table[slot];
    if (page < 0 || page >= c.pages) {
        missing = true;
        return -1;
    }
    return page * c.page_stride + (long long)(j - slot * c.page_size) * c.D;
}

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// One row over again in fp32 arithmetic, by a warp: keys from .. to - 1.
template <class T, int kDP>
__device__ __noinline__ void exact_row(const Cache &c, const float *q, const int *table, int kvh, int from, int to, float scale_log2, float *o, float *m_out,
                                       float *l_out) {
    constexpr int kE = kDP / 32, kAhead = 4;
    const int lane = threadIdx.x & 31;
    const T *kp = static_cast<const T *>(c.k) + (long long)kvh * c.page_size * c.D, *vp = static_cast<const T *>(c.v) + (long long)kvh * c.page_size * c.D;
    float x[kE], acc[kE], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < kE; e++) x[e] = lane + 32 * e < c.D ? q[lane + 32 * e] * scale_log2 : 0.f, acc[e] = 0.f;
    bool missing = false, is_nan = false;
#pragma unroll 1
    for (int j = from; j < to && !is_nan; j += kAhead) {
        float s[kAhead], v[kAhead][kE];
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const long long at = place(c, table, j + u, to, missing);
            s[u] = 0.f;
#pragma unroll
            for (int e = 0; e < kE; e++) {
                const bool in = at >= 0 && lane + 32 * e < c.D;
                s[u] = fmaf(x[e], in ? as_float(kp[at + lane + 32 * e]) : 0.f, s[u]);
                v[u][e] = in ? as_float(vp[at + lane + 32 * e]) : 0.f;
            }
#pragma unroll
            for (int w = 16; w > 0; w >>= 1) s[u] += __shfl_xor_sync(0xffffffffu, s[u], w);
            if (at < 0) s[u] = -INFINITY;
            is_nan = is_nan || !(s[u] < INFINITY);  // an infinite maximum is subtracted from itself
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            const float top = fmaxf(m, s[u]);
            if (top == -INFINITY || s[u] == -INFINITY) continue;  // no weight
            const float keep = ex2f(m - top), p = ex2f(s[u] - top);
            l = l * keep + p;
#pragma unroll
            for (int e = 0; e < kE; e++) acc[e] = acc[e] * keep + p * v[u][e];
            m = top;
        }
    }
#pragma unroll
    for (int e = 0; e < kE; e++) o[lane + 32 * e] = is_nan ? NAN : acc[e];
    if (lane == 0) *m_out = is_nan ? 0.f : m, *l_out = is_nan ? NAN : l;
}


// One value of a row from the parts of a cluster's CTAs: with(k) gives part k's maximum, sum and value.  All are asked for before the
// first is used: one after the other they took longer than the keys of a short context.
struct Part {
    float m, l, o;
};
template <class F>
__device__ __forceinline__ float joined_value(int ranks, F with) {
    Part p[8];
    float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
    for (int k = 0; k < 8; k++) p[k] = k < ranks ? with(k) : Part{-INFINITY, 0.f, 0.f};
#pragma unroll
    for (int k = 0; k < 8; k++) top = fmaxf(top, p[k].m);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int k = 0; k < 8; k++) {
        const float by = ex2f(p[k].m - base);
        sum = fmaf(p[k].l, by, sum), o = fmaf(p[k].o, by, o);
    }
    return sum == 0.f ? 0.f : o / sum;
}

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
// Sequences with up to `few` rows, 8 at most; bf16 pages, D <= 128.
cudaError_t launch_decode(const Call &a, int few);
cudaError_t decode_set_attributes();
// CTAs of one of `units`, which share its keys: as many as fit the GPU at a time, two an SM and a few more (160 units of up to 2000 keys, 4
// rows: 50 us with one, 36 with two each), and enough for no more than 4096 keys each.
inline unsigned ranks_of(const Call &a, long long units) {
    const int sms = attn::sm_count();
    unsigned ranks = 1;
    while (ranks < 8 && units * ranks * 2 <= 5 * sms / 2) ranks *= 2;
    const long long keys = (long long)a.c.width * a.c.page_size;
    while (ranks < 8 && keys / ranks > 4096) ranks *= 2;
    return ranks;
}
cudaError_t tiles_set_attributes();
cudaError_t few_rows_set_attributes();

}  // namespace paged
