// Attention of new tokens over a paged key/value cache for sm_100a: few rows, bound by HBM.
//
//   out[t, h] = sum_j p_j v[j] / sum_j p_j,   p_j = exp(scale q[t, h] . k[j] - m),   j = 0 .. position of t
//
// A unit is one sequence, one key/value head and up to kRows of its rows (row = new token x query head of the group); a
// cluster of 1 to 8 CTAs takes it, each CTA one run of the keys, each warp every fourth batch of that run.  LPR lanes hold
// one key (16 bytes each, twice that for the widest heads), so a warp reads 32 / LPR keys in one request; every such group
// of lanes keeps a running maximum, sum and output of its own for its keys, in fp32 and in registers, and they are joined
// only at the end: over the lanes by shuffles, over the warps in shared memory, over the cluster through distributed shared
// memory.  No atomics, no scratch buffer, one launch; the order of every sum is fixed.
#include <cooperative_groups.h>

#include "attn_internal.h"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "tc05.cuh"

#include "../../include/attn_sm100.h"

namespace paged {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;
constexpr int kThreads = 32 * kWarps;

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// exp2(a - b) where b is the larger of the two or both are -inf (then 0: nothing has weight yet)
__device__ __forceinline__ float weight(float a, float b) { return a == -INFINITY ? 0.f : ex2(a - b); }

template <class T>
struct Words;  // 16 bytes of the cache as floats
template <>
struct Words<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void open(const uint4 &w, float (&f)[4]) {
        f[0] = __uint_as_float(w.x), f[1] = __uint_as_float(w.y), f[2] = __uint_as_float(w.z), f[3] = __uint_as_float(w.w);
    }
};
template <>
struct Words<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void open(const uint4 &w, float (&f)[8]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) f[2 * i] = __uint_as_float(v[i] << 16), f[2 * i + 1] = __uint_as_float(v[i] & 0xffff0000u);
    }
};

template <int kRows, int kWidth>
struct Partial {
    float m[kRows], l[kRows];
    float o[kRows][kWidth];
};

__device__ __forceinline__ uint4 load16(const void *p) {
    uint4 v;
    asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
    return v;
}

// kLanes: lanes of a key; kChunks: 16-byte words of a lane
template <class T, int kLanes, int kChunks, int kRows>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(Cache c, const float *q, float *out, long long ld, int heads,
                                                            int groups, int few, int max_new, float scale_log2,
                                                            int *status) {
    constexpr int kN = Words<T>::kN, kWidth = kLanes * kChunks * kN, kKeys = 32 / kLanes, kBatch = 4 / kChunks;
    __shared__ Partial<kRows, kWidth> part[kWarps];
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = lane % kLanes, mine = lane / kLanes;
    const int unit = blockIdx.x / ranks, s = unit / groups, row0 = (unit % groups) * kRows, kvh = blockIdx.y;
    const int G = heads / c.kv_heads;
    tc05::pdl_launch_dependents();
    tc05::pdl_wait();
    const Span w = span_of(c, s);
    const int rows = w.count * G;
    if (unit % groups == 0 && kvh == 0 && rank == 0 && threadIdx.x == 0 && (w.count > max_new || (w.count > 0 && w.past < 0))) report(status, ST_ATTEND);
    if (row0 >= rows || rows > few || w.past < 0 || w.count > max_new) return;  // the whole cluster
    const int last = min(row0 + kRows, rows) - 1;
    const long long room = (long long)c.width * c.page_size;
    const int keys = (int)min((long long)w.past + last / G + 1, room);
    if (w.past + (long long)w.count > room && row0 == 0 && threadIdx.x == 0) report(status, ST_ATTEND);
    const int *table = c.table + (long long)s * c.width;

    float qv[kRows][kChunks][kN], m[kRows], l[kRows], o[kRows][kChunks][kN];
    int seen[kRows];  // keys that the row sees
#pragma unroll
    for (int r = 0; r < kRows; r++) {
        const int at = min(row0 + r, last), t = at / G;
        seen[r] = row0 + r <= last ? w.past + t + 1 : 0;
        m[r] = -INFINITY, l[r] = 0.f;
        const float *src = q + (w.first + t) * ld + (long long)(kvh * G + at % G) * c.D;
#pragma unroll
        for (int ch = 0; ch < kChunks; ch++) {
            const int d = (ch * kLanes + sub) * kN;
#pragma unroll
            for (int e = 0; e < kN; e += 4) {
                const float4 v = d < c.D ? *reinterpret_cast<const float4 *>(src + d + e) : make_float4(0.f, 0.f, 0.f, 0.f);
                qv[r][ch][e] = v.x * scale_log2, qv[r][ch][e + 1] = v.y * scale_log2;
                qv[r][ch][e + 2] = v.z * scale_log2, qv[r][ch][e + 3] = v.w * scale_log2;
            }
#pragma unroll
            for (int e = 0; e < kN; e++) o[r][ch][e] = 0.f;
        }
    }

    // this CTA's run of keys, in whole batches of all its warps
    constexpr int kRound = kKeys * kBatch * kWarps;
    const int rounds = (keys + kRound - 1) / kRound, each = (rounds + ranks - 1) / ranks;
    const int begin = rank * each * kRound, end = min(keys, begin + each * kRound);
    const T *kp = static_cast<const T *>(c.k) + (long long)kvh * c.page_size * c.D, *vp = static_cast<const T *>(c.v) + (long long)kvh * c.page_size * c.D;
    bool missing = false;
    // the first element of a key's row, -1 where there is no such key
    auto place = [&](int j) -> long long {
        if (j >= end) return -1;
        const int slot = j / c.page_size, page = table[slot];
        if (page < 0 || page >= c.pages) {
            missing = true;
            return -1;
        }
        return page * c.page_stride + (long long)(j - slot * c.page_size) * c.D;
    };
    long long where[kBatch];
#pragma unroll
    for (int u = 0; u < kBatch; u++) where[u] = place(begin + warp * kKeys * kBatch + u * kKeys + mine);
    for (int j0 = begin + warp * kKeys * kBatch; j0 < end; j0 += kRound) {
        uint4 kw[kBatch][kChunks], vw[kBatch][kChunks];
        bool there[kBatch];
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
            there[u] = where[u] >= 0;
#pragma unroll
            for (int ch = 0; ch < kChunks; ch++) {
                const int d = (ch * kLanes + sub) * kN;
                const bool ok = there[u] && d < c.D;
                kw[u][ch] = ok ? load16(kp + where[u] + d) : make_uint4(0, 0, 0, 0);
                vw[u][ch] = ok ? load16(vp + where[u] + d) : make_uint4(0, 0, 0, 0);
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; u++) where[u] = place(j0 + kRound + u * kKeys + mine);
        float sc[kBatch][kRows];
#pragma unroll
        for (int u = 0; u < kBatch; u++) {
#pragma unroll
            for (int r = 0; r < kRows; r++) sc[u][r] = 0.f;
#pragma unroll
            for (int ch = 0; ch < kChunks; ch++) {
                float f[kN];
                Words<T>::open(kw[u][ch], f);
#pragma unroll
                for (int r = 0; r < kRows; r++)
#pragma unroll
                    for (int e = 0; e < kN; e++) sc[u][r] = fmaf(qv[r][ch][e], f[e], sc[u][r]);
            }
#pragma unroll
            for (int r = 0; r < kRows; r++)
#pragma unroll
                for (int x = kLanes / 2; x > 0; x >>= 1) sc[u][r] += __shfl_xor_sync(0xffffffffu, sc[u][r], x);
        }
#pragma unroll
        for (int r = 0; r < kRows; r++) {
            bool ok[kBatch];
            float top = m[r];
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                ok[u] = there[u] && j0 + u * kKeys + mine < seen[r];
                if (ok[u]) top = fmaxf(top, sc[u][r]);
            }
            const float keep = weight(m[r], top);
            m[r] = top;
            l[r] *= keep;
#pragma unroll
            for (int ch = 0; ch < kChunks; ch++)
#pragma unroll
                for (int e = 0; e < kN; e++) o[r][ch][e] *= keep;
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                sc[u][r] = ok[u] ? weight(sc[u][r], top) : 0.f;
                l[r] += sc[u][r];
            }
        }
#pragma unroll
        for (int u = 0; u < kBatch; u++)
#pragma unroll
            for (int ch = 0; ch < kChunks; ch++) {
                float f[kN];
                Words<T>::open(vw[u][ch], f);
#pragma unroll
                for (int r = 0; r < kRows; r++) {
                    // a value that the row does not see may be anything, and 0 times it not 0
                    if (kRows > 1 && sc[u][r] == 0.f) continue;
#pragma unroll
                    for (int e = 0; e < kN; e++) o[r][ch][e] = fmaf(sc[u][r], f[e], o[r][ch][e]);
                }
            }
    }
    if (missing) report(status, ST_ATTEND);

    // join the groups of lanes, then the warps, then the CTAs
#pragma unroll
    for (int r = 0; r < kRows; r++) {
#pragma unroll
        for (int x = kLanes; x < 32; x <<= 1) {
            const float mo = __shfl_xor_sync(0xffffffffu, m[r], x), top = fmaxf(m[r], mo);
            const float a = weight(m[r], top), b = weight(mo, top);
            l[r] = l[r] * a + __shfl_xor_sync(0xffffffffu, l[r], x) * b;
#pragma unroll
            for (int ch = 0; ch < kChunks; ch++)
#pragma unroll
                for (int e = 0; e < kN; e++) o[r][ch][e] = o[r][ch][e] * a + __shfl_xor_sync(0xffffffffu, o[r][ch][e], x) * b;
            m[r] = top;
        }
        if (mine == 0) {
            if (sub == 0) part[warp].m[r] = m[r], part[warp].l[r] = l[r];
#pragma unroll
            for (int ch = 0; ch < kChunks; ch++)
#pragma unroll
                for (int e = 0; e < kN; e++) part[warp].o[r][(ch * kLanes + sub) * kN + e] = o[r][ch][e];
        }
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    if (rank == 0) {
        for (int i = threadIdx.x; i < kRows * c.D; i += kThreads) {
            const int r = i / c.D, d = i - r * c.D;
            if (row0 + r > last) break;
            float top = -INFINITY, sum = 0.f, acc = 0.f;
            for (int k = 0; k < ranks; k++) {
                const Partial<kRows, kWidth> *p = ranks > 1 ? cluster.map_shared_rank(&part[0], k) : part;
                for (int x = 0; x < kWarps; x++) {
                    const float mo = p[x].m[r], t2 = fmaxf(top, mo), a = weight(top, t2), b = weight(mo, t2);
                    sum = sum * a + p[x].l[r] * b;
                    acc = acc * a + p[x].o[r][d] * b;
                    top = t2;
                }
            }
            const int at = row0 + r;
            out[((long long)(w.first + at / G) * heads + kvh * G + at % G) * c.D + d] = sum == 0.f ? 0.f : acc / sum;
        }
    }
    if (ranks > 1) cluster.sync();  // shared memory of the others is read until here
}

// ------------------------------------------------------------------------------------------
// launch
// ------------------------------------------------------------------------------------------
template <class T, int kLanes, int kChunks, int kRows>
cudaError_t launch_few(const Call &a, int few) {
    const int G = a.heads / a.c.kv_heads, groups = (int)((min((long long)a.max_new * G, (long long)few) + kRows - 1) / kRows);
    const long long units = (long long)a.c.seqs * groups, all = units * a.c.kv_heads;
    const int sms = attn::sm_count();
    unsigned ranks = 1;
    while (ranks < 8 && all * ranks < 2 * sms) ranks *= 2;
    const long long keys = (long long)a.c.width * a.c.page_size;
    while (ranks < 8 && keys / ranks > 4096) ranks *= 2;
    if (units * ranks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    return attn::launch_clusters_after_previous(few_rows_kernel<T, kLanes, kChunks, kRows>, dim3((unsigned)(units * ranks), (unsigned)a.c.kv_heads), dim3(kThreads),
                                                0, ranks, a.s, a.c, a.q, a.out, a.ld, a.heads, groups, few, a.max_new, a.scale_log2, a.status);
}

template <class T, int kLanes, int kChunks>
cudaError_t launch_rows(const Call &a, int few) {
    const long long rows = min((long long)a.max_new * (a.heads / a.c.kv_heads), (long long)few);
    if (rows == 1) return launch_few<T, kLanes, kChunks, 1>(a, few);
    if (rows == 2) return launch_few<T, kLanes, kChunks, 2>(a, few);
    return launch_few<T, kLanes, kChunks, 4>(a, few);
}

template <class T>
cudaError_t launch(const Call &a, int few) {
    const int words = a.c.D / Words<T>::kN;  // of 16 bytes
    if (words <= 4) return launch_rows<T, 4, 1>(a, few);
    if (words <= 8) return launch_rows<T, 8, 1>(a, few);
    if (words <= 16) return launch_rows<T, 16, 1>(a, few);
    if (words <= 32) return launch_rows<T, 32, 1>(a, few);
    return launch_rows<T, 32, 2>(a, few);
}

// Sequences of up to kFewRows rows go to the kernel above, which reads their keys at the HBM rate, the others to the tensor
// cores; both kernels find their own sequences on the device, so a step that mixes them takes two launches.
constexpr int kFewRows = 4;
constexpr int kMeanRows = 128;  // from this many rows a sequence on, on average, the tensor cores take all of them in one launch

cudaError_t forward(const Call &a) {
    const long long G = a.heads / a.c.kv_heads, most = a.max_new * G;
    if (most <= kFewRows || a.c.D > 128) return a.type == ATTN_CACHE_BF16 ? launch<__nv_bfloat16>(a, 0x7fffffff) : launch<float>(a, 0x7fffffff);
    const bool both = G <= kFewRows && a.c.tokens * G < (long long)kMeanRows * a.c.seqs;
    const int few = both ? kFewRows : 0;
    const cudaError_t e = launch_tiles(a, few);
    if (e != cudaSuccess || !both) return e;
    return a.type == ATTN_CACHE_BF16 ? launch<__nv_bfloat16>(a, few) : launch<float>(a, few);
}

}  // namespace
}  // namespace paged

extern "C" int attn_sm100_paged_forward(const float *q, const void *k_pages, const void *v_pages, const int *page_table, const int *cu_seqlens,
                                        const int *past, float *out, long long ld, long long page_stride, int cache_type, int tokens, int seqs,
                                        int n_heads, int kv_heads, int D, int page_size, int pages, int table_width, int max_new, float scale,
                                        void *stream) {
    if (!q || !k_pages || !v_pages || !page_table || !cu_seqlens || !past || !out) return ATTN_ERR_NULL;
    int rc = paged::check_cache(tokens, seqs, n_heads, kv_heads, D, page_size, pages, table_width, cache_type, k_pages, v_pages, page_stride);
    if (rc != ATTN_OK) return rc;
    if (ld < (long long)n_heads * D || max_new < 0 || !(scale == scale)) return ATTN_ERR_ARGUMENT;
    if (kv_heads > 65535) return ATTN_ERR_UNSUPPORTED;
    if ((reinterpret_cast<uintptr_t>(q) & 15) || (reinterpret_cast<uintptr_t>(out) & 15) || ld % 4) return ATTN_ERR_ALIGN;
    int *status = nullptr;
    if ((rc = attn::device_status_word(&status)) != ATTN_OK) return rc;
    if (tokens == 0) return ATTN_OK;
    const int most = max_new == 0 || max_new > tokens ? tokens : max_new;
    if ((long long)tokens * (n_heads / kv_heads) > 0x3fffffffll) return ATTN_ERR_UNSUPPORTED;
    const paged::Call a{{const_cast<void *>(k_pages), const_cast<void *>(v_pages), page_table, cu_seqlens, past, page_stride, seqs, kv_heads, D, page_size, pages,
                         table_width, tokens},
                        q, out, ld, n_heads, most, cache_type, scale * 1.4426950408889634f, status, static_cast<cudaStream_t>(stream)};
    return (int)paged::forward(a);
}
