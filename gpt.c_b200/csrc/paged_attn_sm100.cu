// Attention of new tokens over a paged key/value cache for sm_100a: few rows, bound by HBM.
//
//   out[t, h] = sum_j p_j v[j] / sum_j p_j,   p_j = exp(scale q[t, h] . k[j] - m),   j = 0 .. position of t
//
// A unit is one sequence, one key/value head and up to kRows of its rows (row = new token x query head of the group); a
// cluster of 1 to 8 CTAs takes it, each CTA one run of the keys.  One warp brings them: pages are contiguous for a head, so it asks
// the copy engine for whole runs of a page at a time, four stages ahead.  Four warps compute: kLanes lanes hold
// one key (16 bytes each, twice that for the widest heads), so a warp reads 32 / kLanes keys at a time; every such group
// of lanes keeps a running maximum, sum and output of its own for its keys, in fp32 and in registers, and they are joined
// only at the end: over the lanes by shuffles, over the warps in shared memory, over the cluster through distributed shared
// memory.  No atomics, no scratch buffer; the order of every sum is fixed.  One sequence of
// 1001 positions, 12 heads of 64: 6.5 us, the chain past -> page table -> page -> sums -> join; its 6 MB alone would take 0.9.
//
// Stages in which a key has no weight for one of the rows (not seen, no page, a score of -inf) leave such keys out one by one, in code of
// their own; with the checks among the other stages' instructions six contexts of 20000 and more, 4 rows, heads of 128, took 185 us, so 177.
#include <cooperative_groups.h>

#include <type_traits>

#include "attn24.cuh"
#include "attn_internal.h"
#include "paged.cuh"
#include "paged_attn.cuh"
#include "tc05.cuh"

#include "../../include/attn_sm100.h"

namespace paged {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4;  // that compute, and one that brings keys and values
constexpr int kThreads = 32 * (kWarps + 1);
constexpr int kStages = 4;

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
    static __device__ __forceinline__ void open(const uint4 &w, float2 (&f)[2]) {
        f[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y)), f[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
    }
};
template <>
struct Words<__nv_bfloat16> {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void open(const uint4 &w, float2 (&f)[4]) {
        const uint32_t v[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = make_float2(__uint_as_float(v[i] << 16), __uint_as_float(v[i] & 0xffff0000u));
    }
};

template <int kRows, int kWidth>
struct Partial {
    float m[kRows], l[kRows];
    float o[kRows][kWidth];
};

enum Site : int { SITE_FULL = 451, SITE_EMPTY };

// kLanes: lanes of a key; kChunks: 16-byte words of a lane
template <class T, int kLanes, int kChunks, int kRows>
struct FewSmem {
    static constexpr int kWidth = kLanes * kChunks * Words<T>::kN;
    static constexpr int kKeys = 32 / kLanes, kBatch = 4 / kChunks;  // keys of a warp at a time, and how often in a stage
    static constexpr int kStep = kKeys * kBatch * kWarps;            // keys of a stage
    uint8_t k[kStages][kStep * kWidth * sizeof(T)], v[kStages][kStep * kWidth * sizeof(T)];  // rows of D elements, one behind the other
    Partial<kRows, kWidth> part[kWarps], all;
    uint64_t full[kStages], empty[kStages];
    int holes[kStages];  // whether a key of the stage has no page
    int abort_flag;
};

__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(smem_u32(dst)), "l"(src), "r"(bytes),
                 "r"(smem_u32(bar))
                 : "memory");
}

template <class T, int kLanes, int kChunks, int kRows>
__global__ void __launch_bounds__(kThreads) few_rows_kernel(Cache c, const float *q, float *out, long long ld, int heads, int groups, int few, int max_new,
                                                            float scale_log2, int *status) {
    using Smem = FewSmem<T, kLanes, kChunks, kRows>;
    constexpr int kN = Words<T>::kN, kPairs = kN / 2, kKeys = Smem::kKeys, kBatch = Smem::kBatch, kStep = Smem::kStep;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, sub = lane % kLanes, mine = lane / kLanes;
    const int unit = blockIdx.x / ranks, s = unit / groups, row0 = (unit % groups) * kRows, kvh = blockIdx.y;
    const int G = heads / c.kv_heads;
    WaitCtx ctx{&sm.abort_flag, status};
    if (threadIdx.x == 0) {
        sm.abort_flag = 0;
        for (int i = 0; i < kStages; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], kWarps);
        }
        fence_barrier_init();
    }
    pdl_wait();
    const Span w = span_of(c, s);
    const int rows = w.count * G;
    if (unit % groups == 0 && kvh == 0 && rank == 0 && threadIdx.x == 0 && (w.count > max_new || (w.count > 0 && w.past < 0))) report(status, ST_ATTEND);
    if (row0 >= rows || rows > few || w.past < 0 || w.count > max_new) return;  // the whole cluster
    const int last = min(row0 + kRows, rows) - 1;
    const long long room = (long long)c.width * c.page_size;
    const int keys = (int)min((long long)w.past + last / G + 1, room);
    if (w.past + (long long)w.count > room && row0 == 0 && threadIdx.x == 0) report(status, ST_ATTEND);
    const int *table = c.table + (long long)s * c.width;
    // this CTA's run of keys, in whole stages
    const int all = (keys + kStep - 1) / kStep, each = (all + ranks - 1) / ranks;
    const int begin = rank * each * kStep, end = min(keys, begin + each * kStep), steps = max(0, (end - begin + kStep - 1) / kStep);
    const int row_bytes = c.D * (int)sizeof(T);
    __syncthreads();

    if (warp == kWarps) {
        // ------------------------------ keys and values ------------------------------
        const T *kp = static_cast<const T *>(c.k) + (long long)kvh * c.page_size * c.D, *vp = static_cast<const T *>(c.v) + (long long)kvh * c.page_size * c.D;
        for (int n = 0; n < steps; n++) {
            const int st = n % kStages, from = begin + n * kStep, to = min(end, from + kStep);
            const int first = from / c.page_size, runs = (to - 1) / c.page_size - first + 1;  // runs of keys within a page, one a lane
            if (n >= kStages) attn24::await(&sm.empty[st], (n / kStages - 1) & 1, ctx, SITE_EMPTY);
            if (lane == 0) sm.holes[st] = 0;
            __syncwarp();
            int missing = 0;
            for (int i = lane; i < runs; i += 32) {
                const int slot = first + i, page = table[slot], j0 = max(from, slot * c.page_size), j1 = min(to, (slot + 1) * c.page_size);
                const bool there = page >= 0 && page < c.pages;
                if (!there) missing += j1 - j0;
            }
            const int lost = __reduce_add_sync(0xffffffffu, missing);
            if (lane == 0) {
                if (lost) sm.holes[st] = 1, report(status, ST_ATTEND);
                mbar_expect_tx(&sm.full[st], 2u * (uint32_t)((to - from - lost) * row_bytes));
            }
            __syncwarp();
            for (int i = lane; i < runs; i += 32) {
                const int slot = first + i, page = table[slot], j0 = max(from, slot * c.page_size), j1 = min(to, (slot + 1) * c.page_size);
                if (page < 0 || page >= c.pages) continue;
                const long long at = page * c.page_stride + (long long)(j0 - slot * c.page_size) * c.D;
                const uint32_t bytes = (uint32_t)((j1 - j0) * row_bytes);
                bulk_load(sm.k[st] + (j0 - from) * row_bytes, kp + at, bytes, &sm.full[st]);
                bulk_load(sm.v[st] + (j0 - from) * row_bytes, vp + at, bytes, &sm.full[st]);
            }
            __syncwarp();
        }
    } else {
        // ------------------------------ softmax and sums ------------------------------
        float2 qv[kRows][kChunks][kPairs], o[kRows][kChunks][kPairs];
        float m[kRows], l[kRows];
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
                for (int e = 0; e < kPairs; e += 2) {
                    const float4 v = d < c.D ? *reinterpret_cast<const float4 *>(src + d + 2 * e) : make_float4(0.f, 0.f, 0.f, 0.f);
                    qv[r][ch][e] = make_float2(v.x * scale_log2, v.y * scale_log2);
                    qv[r][ch][e + 1] = make_float2(v.z * scale_log2, v.w * scale_log2);
                }
#pragma unroll
                for (int e = 0; e < kPairs; e++) o[r][ch][e] = make_float2(0.f, 0.f);
            }
        }
        const int most = min(end, w.past + row0 / G + 1);  // keys that every row sees
        for (int n = 0; n < steps; n++) {
            const int st = n % kStages, j0 = begin + n * kStep + warp * (kKeys * kBatch) + mine;
            attn24::await(&sm.full[st], (n / kStages) & 1, ctx, SITE_FULL);
            const bool whole = begin + (n + 1) * kStep <= most && !sm.holes[st];
            bool there[kBatch];
#pragma unroll
            for (int u = 0; u < kBatch; u++) there[u] = whole || j0 + u * kKeys < end;
            if (!whole && sm.holes[st]) {
#pragma unroll
                for (int u = 0; u < kBatch; u++)
                    if (there[u]) {
                        const int page = table[(j0 + u * kKeys) / c.page_size];
                        there[u] = page >= 0 && page < c.pages;
                    }
            }
            const int at = (warp * (kKeys * kBatch) + mine) * row_bytes;
            float sc[kBatch][kRows];
#pragma unroll
            for (int u = 0; u < kBatch; u++) {
                float2 sum[kRows];
#pragma unroll
                for (int r = 0; r < kRows; r++) sum[r] = make_float2(0.f, 0.f);
#pragma unroll
                for (int ch = 0; ch < kChunks; ch++) {
                    const int d = (ch * kLanes + sub) * kN;
                    uint4 word = make_uint4(0, 0, 0, 0);
                    if (there[u] && d < c.D) word = *reinterpret_cast<const uint4 *>(sm.k[st] + at + u * kKeys * row_bytes + d * (int)sizeof(T));
                    float2 f[kPairs];
                    Words<T>::open(word, f);
#pragma unroll
                    for (int r = 0; r < kRows; r++)
#pragma unroll
                        for (int e = 0; e < kPairs; e++) sum[r] = fma2(qv[r][ch][e], f[e], sum[r]);
                }
#pragma unroll
                for (int r = 0; r < kRows; r++) {
                    sc[u][r] = sum[r].x + sum[r].y;
#pragma unroll
                    for (int x = kLanes / 2; x > 0; x >>= 1) sc[u][r] += __shfl_xor_sync(0xffffffffu, sc[u][r], x);
                }
            }
            // A key without weight (not there, not seen, or with a score of -inf) may have any value, and 0 times that need not be 0.
            auto add_up = [&](auto careful) {
                uint32_t without = 0;  // bit kBatch r + u
#pragma unroll
                for (int r = 0; r < kRows; r++) {
                    if (careful) {
#pragma unroll
                        for (int u = 0; u < kBatch; u++) {
                            if (!there[u] || j0 + u * kKeys >= seen[r]) sc[u][r] = -INFINITY;
                            without |= (sc[u][r] == -INFINITY ? 1u : 0u) << (kBatch * r + u);
                        }
                    }
                    float top = m[r];
#pragma unroll
                    for (int u = 0; u < kBatch; u++) top = fmaxf(top, sc[u][r]);
                    const float base = top == -INFINITY ? 0.f : top, keep = ex2(m[r] - base);  // nothing has weight yet
                    m[r] = top;
                    l[r] *= keep;
#pragma unroll
                    for (int ch = 0; ch < kChunks; ch++)
#pragma unroll
                        for (int e = 0; e < kPairs; e++) o[r][ch][e] = mul2(o[r][ch][e], make_float2(keep, keep));
#pragma unroll
                    for (int u = 0; u < kBatch; u++) {
                        sc[u][r] = ex2(sc[u][r] - base);
                        l[r] += sc[u][r];
                    }
                }
#pragma unroll
                for (int u = 0; u < kBatch; u++)
#pragma unroll
                    for (int ch = 0; ch < kChunks; ch++) {
                        const int d = (ch * kLanes + sub) * kN;
                        uint4 word = make_uint4(0, 0, 0, 0);
                        if ((!careful || there[u]) && d < c.D) word = *reinterpret_cast<const uint4 *>(sm.v[st] + at + u * kKeys * row_bytes + d * (int)sizeof(T));
                        float2 f[kPairs];
                        Words<T>::open(word, f);
#pragma unroll
                        for (int r = 0; r < kRows; r++) {
                            if (careful && (without >> (kBatch * r + u) & 1u)) continue;
#pragma unroll
                            for (int e = 0; e < kPairs; e++) o[r][ch][e] = fma2(make_float2(sc[u][r], sc[u][r]), f[e], o[r][ch][e]);
                        }
                    }
            };
            float low = INFINITY;
#pragma unroll
            for (int u = 0; u < kBatch; u++)
#pragma unroll
                for (int r = 0; r < kRows; r++) low = fminf(low, sc[u][r]);
            if (whole && low > -INFINITY) add_up(std::false_type{});
            else add_up(std::true_type{});
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[st]);
        }

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
                    for (int e = 0; e < kPairs; e++) {
                        o[r][ch][e].x = o[r][ch][e].x * a + __shfl_xor_sync(0xffffffffu, o[r][ch][e].x, x) * b;
                        o[r][ch][e].y = o[r][ch][e].y * a + __shfl_xor_sync(0xffffffffu, o[r][ch][e].y, x) * b;
                    }
                m[r] = top;
            }
            if (mine == 0) {
                if (sub == 0) sm.part[warp].m[r] = m[r], sm.part[warp].l[r] = l[r];
#pragma unroll
                for (int ch = 0; ch < kChunks; ch++)
#pragma unroll
                    for (int e = 0; e < kPairs; e++) *reinterpret_cast<float2 *>(&sm.part[warp].o[r][(ch * kLanes + sub) * kN + 2 * e]) = o[r][ch][e];
            }
        }
    }
    // Let the next kernel start only now: beside this one's loads its CTAs made one sequence of 1001 positions take 8.5 instead of 7.8 us.
    pdl_launch_dependents();
    if (sm.abort_flag) __nanosleep(50000);  // let copies that are still in flight land
    __syncthreads();
    const int count = last - row0 + 1;
    for (int i = threadIdx.x; i < count * c.D; i += kThreads) {
        const int r = i / c.D, d = i - r * c.D;
        float top = -INFINITY, sum = 0.f, o_all = 0.f;
#pragma unroll
        for (int x = 0; x < kWarps; x++) top = fmaxf(top, sm.part[x].m[r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int x = 0; x < kWarps; x++) {
            const float by = ex2(sm.part[x].m[r] - base);
            sum = fmaf(sm.part[x].l[r], by, sum), o_all = fmaf(sm.part[x].o[r][d], by, o_all);
        }
        sm.all.o[r][d] = o_all;
        if (d == 0) sm.all.m[r] = top, sm.all.l[r] = sum;
    }
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    // every CTA of the cluster writes some of the values
    for (int i = rank * kThreads + threadIdx.x; i < count * c.D; i += ranks * kThreads) {
        const int r = i / c.D, d = i - r * c.D, at = row0 + r;
        out[((long long)(w.first + at / G) * heads + kvh * G + at % G) * c.D + d] = joined_value(ranks, [&](int k) {
            const auto &p = ranks > 1 ? *cluster.map_shared_rank(&sm.all, k) : sm.all;
            return Part{p.m[r], p.l[r], p.o[r][d]};
        });
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
    const unsigned ranks = ranks_of(a, all);
    if (units * ranks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    return attn::launch_clusters_after_previous(few_rows_kernel<T, kLanes, kChunks, kRows>, dim3((unsigned)(units * ranks), (unsigned)a.c.kv_heads), dim3(kThreads),
                                                sizeof(FewSmem<T, kLanes, kChunks, kRows>), ranks, a.s, a.c, a.q, a.out, a.ld, a.heads, groups, few, a.max_new, a.scale_log2, a.status);
}

template <class T, int kLanes, int kChunks>
cudaError_t launch_rows(const Call &a, int few) {
    const long long rows = min((long long)a.max_new * (a.heads / a.c.kv_heads), (long long)few);
    if (rows == 1) return launch_few<T, kLanes, kChunks, 1>(a, few);
    if (rows == 2) return launch_few<T, kLanes, kChunks, 2>(a, few);
    return launch_few<T, kLanes, kChunks, 4>(a, few);
}

cudaError_t launch(const Call &a, int few) {
    if (a.type == ATTN_CACHE_BF16) return launch_rows<__nv_bfloat16, 32, 1>(a, few);  // D > 128
    const int words = a.c.D / Words<float>::kN;  // of 16 bytes
    if (words <= 4) return launch_rows<float, 4, 1>(a, few);
    if (words <= 8) return launch_rows<float, 8, 1>(a, few);
    if (words <= 16) return launch_rows<float, 16, 1>(a, few);
    if (words <= 32) return launch_rows<float, 32, 1>(a, few);
    return launch_rows<float, 32, 2>(a, few);
}

template <class T, int kLanes, int kChunks>
cudaError_t set_rows() {
    const cudaFuncAttribute at = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaError_t e = cudaFuncSetAttribute(few_rows_kernel<T, kLanes, kChunks, 1>, at, (int)sizeof(FewSmem<T, kLanes, kChunks, 1>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(few_rows_kernel<T, kLanes, kChunks, 2>, at, (int)sizeof(FewSmem<T, kLanes, kChunks, 2>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(few_rows_kernel<T, kLanes, kChunks, 4>, at, (int)sizeof(FewSmem<T, kLanes, kChunks, 4>));
    return e;
}
// Sequences of few rows go to the kernels that read their keys at the HBM rate, the others to the tile kernel; all find
// their own sequences on the device, so a step may mix them.  Two launches, one behind the other, for such a step only where there are more
// sequences x key/value heads than the tile kernel takes in two rounds or so, or long contexts, which it would walk with one CTA each:
// 32 single tokens and two pieces of up to 500, 5 heads of 128 for 20, short bursts: 71 us with the tile kernel alone, 86 with both; 64 single tokens
// 115 / 137, 128 of them 165 / 163; 32 of them with 12 heads of 64 76 / 74, 24 55 / 72, 64 125 / 110; fp32, 170 units 178 / 222, 330 319 / 298.
// And where there are few rows on average: a step of single tokens whose program does not give max_new.
constexpr int kFewRows16 = 8, kFewRows32 = 4;
constexpr int kMeanRows = 128;             // from this many rows a sequence on, on average, the tile kernel takes all of them in any case
constexpr int kUnits16 = 5, kUnits32 = 4;  // halves of a round of the SMs
constexpr long long kShort = 8192;         // positions that the page table has room for

cudaError_t forward(const Call &a) {
    const bool narrow = a.type == ATTN_CACHE_BF16 && a.c.D <= 128;
    const long long G = a.heads / a.c.kv_heads, most = a.max_new * G;
    const int limit = narrow ? kFewRows16 : kFewRows32;
    auto launch_few_rows = [&](int few) { return narrow ? launch_decode(a, few) : launch(a, few); };
    if (a.c.D > 128) return launch_few_rows(0x7fffffff);
    const bool far = narrow && a.c.pages * a.c.page_stride > 1ll << 34;  // beyond that kernel's 32-bit places: the tile kernel takes all
    if (most <= limit && !far) return launch_few_rows(limit);
    const bool one = a.c.tokens * G > (long long)limit * a.c.seqs && (long long)a.c.width * a.c.page_size <= kShort &&
                     2ll * a.c.seqs * a.c.kv_heads <= (narrow ? kUnits16 : kUnits32) * attn::sm_count();
    const bool both = !far && !one && G <= limit && a.c.tokens * G < (long long)kMeanRows * a.c.seqs;
    if (both) {
        const cudaError_t e = launch_few_rows(limit);
        if (e != cudaSuccess) return e;
    }
    return launch_tiles(a, both ? limit : 0);
}

}  // namespace

cudaError_t few_rows_set_attributes() {
    cudaError_t e = set_rows<float, 4, 1>();
    if (e == cudaSuccess) e = set_rows<float, 8, 1>();
    if (e == cudaSuccess) e = set_rows<float, 16, 1>();
    if (e == cudaSuccess) e = set_rows<float, 32, 1>();
    if (e == cudaSuccess) e = set_rows<float, 32, 2>();
    return e != cudaSuccess ? e : set_rows<__nv_bfloat16, 32, 1>();
}

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
