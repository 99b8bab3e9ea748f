// Keys and values of new tokens into a paged cache, with the position rotation on the way, for sm_100a.
//
// Token t of sequence s, the i-th of its new ones, has position p = past[s] + i and goes to row p % page_size of page
// table[s, p / page_size].  With a table of angles, columns (a, b) of a pair become
// (a cos - b sin, b cos + a sin), fp32, of q and k; pages of bf16 take each value rounded once, after the rotation.
//
// Bound by HBM for a prefill step and by the chain of loads cu -> past -> table -> store for a decoding step.  A warp
// takes 32 * kUnits units of 8 columns of one token: it asks for its part of the row before it looks for the sequence, so
// that chain and data travel together.  10920 tokens of 20 + 2 x 5 heads of 128, rotated, bf16 pages: 54 to 57 us, 5.5 to 5.8 TB/s of reads
// and writes, from GPU to GPU; 24 tokens of 3 x 12 heads of 64: 3.3 to 3.7 us, little more than a launch.
#include "attn_internal.h"
#include "paged.cuh"
#include "tc05.cuh"

#include "../../include/attn_sm100.h"

namespace paged {
namespace {

constexpr int kThreads = 256;
constexpr int kUnits = 4;  // per lane

// How the 8 columns of a unit are taken.  kHalves: pairs (i, i + R/2), a unit is 4 columns and their 4 partners; kPairs:
// neighbours (2i, 2i + 1); both where R is a multiple of 8, so that a unit lies wholly inside the rotated columns or
// outside.  kAny: any even R, each column with its partner by itself.
enum Turn : int { kNone, kHalves, kPairs, kAny };

struct Row {
    const float *qkv;
    float *q_out;
    const float *rotary;  // [positions, R]: R/2 cosines, R/2 sines
    long long ld;
    int heads, R, positions, pairs;
};

__device__ __forceinline__ float4 ld4(const float *p) { return __ldcs(reinterpret_cast<const float4 *>(p)); }

__device__ __forceinline__ void put4(float *p, float4 v) { *reinterpret_cast<float4 *>(p) = v; }
__device__ __forceinline__ void put4(__nv_bfloat16 *p, float4 v) {
    *reinterpret_cast<uint2 *>(p) = make_uint2(tc05::pack_bf16x2(v.x, v.y), tc05::pack_bf16x2(v.z, v.w));
}
template <class T>
__device__ __forceinline__ void put8(T *p, int a, int b, float4 x, float4 y) {
    put4(p + a, x);
    put4(p + b, y);
}
__device__ __forceinline__ void put8(__nv_bfloat16 *p, int a, int b, float4 x, float4 y) {
    if (b == a + 4) {
        *reinterpret_cast<uint4 *>(p + a) = make_uint4(tc05::pack_bf16x2(x.x, x.y), tc05::pack_bf16x2(x.z, x.w),
                                                       tc05::pack_bf16x2(y.x, y.y), tc05::pack_bf16x2(y.z, y.w));
    } else {
        put4(p + a, x);
        put4(p + b, y);
    }
}

// a, b: the columns of a unit's two words inside their head.
template <int kTurn>
__device__ __forceinline__ void columns(int u, int R, int &a, int &b) {
    if (kTurn == kHalves && u < R / 8) a = 4 * u, b = R / 2 + 4 * u;
    else a = 8 * u, b = a + 4;
}

__device__ __forceinline__ void turn(float &a, float &b, float c, float s) {
    const float x = a * c - b * s;
    b = b * c + a * s;
    a = x;
}

template <class T, int kTurn>
__global__ void __launch_bounds__(kThreads) append_kernel(Cache c, Row r, int parts, int *status) {
    const int lane = threadIdx.x & 31;
    const long long w = (long long)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5);
    const int t = (int)(w / parts), part = (int)(w % parts);
    tc05::pdl_launch_dependents();
    tc05::pdl_wait();
    if (t >= c.tokens) return;
    const int each = c.D / 8, from = kTurn == kNone ? r.heads : 0;  // units of a head; heads that only rotation looks at
    const int units = (r.heads + 2 * c.kv_heads - from) * each;
    const float *row = r.qkv + t * r.ld + (long long)from * c.D;
    float4 x[kUnits], y[kUnits];
    int at[kUnits];
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
        const int n = (part * kUnits + i) * 32 + lane, h = n / each;
        int a, b;
        columns<kTurn>(n - h * each, r.R, a, b);
        at[i] = n < units ? h : -1;
        if (n < units) {
            x[i] = ld4(row + h * c.D + a);
            y[i] = ld4(row + h * c.D + b);
        }
    }
    const int s = sequence_of(c.cu, c.seqs, t);
    const Span span = span_of(c, s);
    const int i_new = t - span.first;
    if (i_new < 0 || i_new >= span.count) return;  // a row that belongs to no sequence
    const long long pos = (long long)span.past + i_new;
    const long long slot = pos / c.page_size;
    int page = -1;
    if (span.past >= 0 && slot < c.width) page = c.table[(long long)s * c.width + slot];
    if (page < 0 || page >= c.pages || (kTurn != kNone && pos >= r.positions)) {
        if (lane == 0) report(status, ST_APPEND);
        return;
    }
    const long long base = page * c.page_stride + (pos - slot * c.page_size) * c.D;
    const float *angles = kTurn == kNone ? nullptr : r.rotary + pos * r.R;
#pragma unroll
    for (int i = 0; i < kUnits; i++) {
        if (at[i] < 0) continue;
        const int h = from + at[i], u = (part * kUnits + i) * 32 + lane - at[i] * each;
        const bool turned = h < r.heads + c.kv_heads;  // q and k
        int a, b;
        columns<kTurn>(u, r.R, a, b);
        if (kTurn != kNone && turned) {
            if (kTurn == kHalves && u < r.R / 8) {
                const float4 cs = *reinterpret_cast<const float4 *>(angles + a), sn = *reinterpret_cast<const float4 *>(angles + b);
                turn(x[i].x, y[i].x, cs.x, sn.x);
                turn(x[i].y, y[i].y, cs.y, sn.y);
                turn(x[i].z, y[i].z, cs.z, sn.z);
                turn(x[i].w, y[i].w, cs.w, sn.w);
            } else if (kTurn == kPairs && a < r.R) {
                const float4 cs = *reinterpret_cast<const float4 *>(angles + a / 2), sn = *reinterpret_cast<const float4 *>(angles + (r.R + a) / 2);
                turn(x[i].x, x[i].y, cs.x, sn.x);
                turn(x[i].z, x[i].w, cs.y, sn.y);
                turn(y[i].x, y[i].y, cs.z, sn.z);
                turn(y[i].z, y[i].w, cs.w, sn.w);
            } else if (kTurn == kAny) {
                float v[8] = {x[i].x, x[i].y, x[i].z, x[i].w, y[i].x, y[i].y, y[i].z, y[i].w};
                const float *head = r.qkv + t * r.ld + (long long)h * c.D;
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int d = a + e, half = r.R / 2;
                    if (d >= r.R) continue;
                    const bool second = r.pairs ? (d & 1) : d >= half;
                    const int pair = r.pairs ? d >> 1 : (second ? d - half : d);
                    const float other = head[r.pairs ? d ^ 1 : (second ? d - half : d + half)];
                    const float cs = angles[pair], sn = angles[half + pair];
                    v[e] = second ? v[e] * cs + other * sn : v[e] * cs - other * sn;
                }
                x[i] = make_float4(v[0], v[1], v[2], v[3]);
                y[i] = make_float4(v[4], v[5], v[6], v[7]);
            }
        }
        if (h < r.heads) {
            float *q = r.q_out + ((long long)t * r.heads + h) * c.D;
            put8(q, a, b, x[i], y[i]);
        } else {
            const int kv = h - r.heads, hk = kv < c.kv_heads ? kv : kv - c.kv_heads;
            T *dst = static_cast<T *>(kv < c.kv_heads ? c.k : c.v) + base + (long long)hk * c.page_size * c.D;
            put8(dst, a, b, x[i], y[i]);
        }
    }
}

template <class T>
cudaError_t launch(const Cache &c, const Row &r, int *status, cudaStream_t s) {
    const bool eight = r.R % 8 == 0 && (reinterpret_cast<uintptr_t>(r.rotary) & 15) == 0;
    const int turn = r.rotary == nullptr ? kNone : !eight ? kAny : r.pairs ? kPairs : kHalves;
    const int units = ((r.rotary ? r.heads : 0) + 2 * c.kv_heads) * (c.D / 8), parts = (units + 32 * kUnits - 1) / (32 * kUnits);
    const long long blocks = ((long long)c.tokens * parts + kThreads / 32 - 1) / (kThreads / 32);
    if (blocks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    auto kernel = turn == kNone ? append_kernel<T, kNone> : turn == kHalves ? append_kernel<T, kHalves> : turn == kPairs ? append_kernel<T, kPairs> : append_kernel<T, kAny>;
    return attn::launch_after_previous(kernel, dim3((unsigned)blocks), dim3(kThreads), 0, s, c, r, parts, status);
}

}  // namespace
}  // namespace paged

extern "C" int attn_sm100_paged_append(const float *qkv, float *q_out, void *k_pages, void *v_pages, const int *page_table,
                                       const int *cu_seqlens, const int *past, const float *rotary, long long ld, long long page_stride,
                                       int cache_type, int tokens, int seqs, int n_heads, int kv_heads, int D, int page_size, int pages,
                                       int table_width, int positions, int rotary_dim, int rotary_pairs, void *stream) {
    if (!qkv || !k_pages || !v_pages || !page_table || !cu_seqlens || !past || (rotary && !q_out)) return ATTN_ERR_NULL;
    int rc = paged::check_cache(tokens, seqs, n_heads, kv_heads, D, page_size, pages, table_width, cache_type, k_pages, v_pages, page_stride);
    if (rc != ATTN_OK) return rc;
    if (rotary && (rotary_dim <= 0 || rotary_dim % 2 || rotary_dim > D || positions <= 0)) return ATTN_ERR_ARGUMENT;
    if (ld < (long long)(n_heads + 2 * kv_heads) * D) return ATTN_ERR_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(qkv) & 15) || (reinterpret_cast<uintptr_t>(q_out) & 15) || ld % 4 || (reinterpret_cast<uintptr_t>(rotary) & 3))
        return ATTN_ERR_ALIGN;
    int *status = nullptr;
    if ((rc = attn::device_status_word(&status)) != ATTN_OK) return rc;
    if (tokens == 0) return ATTN_OK;
    const paged::Cache c{k_pages, v_pages, page_table, cu_seqlens, past, page_stride, seqs, kv_heads, D, page_size, pages, table_width, tokens};
    const paged::Row r{qkv, q_out, rotary, ld, n_heads, rotary ? rotary_dim : 0, positions, rotary_pairs != 0};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    return (int)(cache_type == ATTN_CACHE_BF16 ? paged::launch<__nv_bfloat16>(c, r, status, s) : paged::launch<float>(c, r, status, s));
}
