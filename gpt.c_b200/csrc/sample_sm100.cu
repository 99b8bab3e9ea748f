// The draw of a class from each row of logits, by temperature, top-k, top-p and min-p, for sm_100a.
//
// With the classes ordered by falling logit, equal ones by index, what each restriction keeps is a run from the front of
// that order, so the classes kept are those above one logit and, of those equal to it, the ones up to an index.  A weight is a
// whole number, round(2^44 exp((x - max) / T)): sums of up to 2^19 of them fit 64 bits and are exact in any order.
//
// A cluster of 1 to 8 CTAs holds a row in shared memory, each CTA a piece, and reads it once.  Where a run ends (the k-th class, or the
// one at which the weight reaches p of all) is found by a histogram over 2048 steps of max - x: counts or weights are added up in shared
// memory, the step in which the run ends is taken from their sums over the cluster, and the classes of that step, some dozens,
// are put in order by comparing each with each.  Where they are more than that (equal logits, outliers that stretch the steps)
// the histogram is taken again over their order-preserving 32-bit keys, 2048 times finer each time.  Then one pass adds up what is kept, in
// the order of the index, and one warp walks the stretch in which the draw falls.
#include <cooperative_groups.h>

#include "attn_internal.h"
#include "tc05.cuh"

#include "../../include/xent_sm100.h"

namespace sample {
namespace {

namespace cg = cooperative_groups;

constexpr int kThreads = 512, kWarps = kThreads / 32;
constexpr int kRanks = 8;      // CTAs of a row at most
constexpr int kBins = 2048;    // of a histogram
constexpr int kList = 512;     // classes that are compared each with each
constexpr int kMaxC = 425984;  // a piece of kMaxC / kRanks logits fits shared memory beside the rest
typedef unsigned long long u64;

struct Smem {
    union {
        struct {
            uint32_t lo[kBins], hi[kBins];  // a histogram's sums, the two halves of each
        };
        struct {  // rank 0, once the sums have been read: the classes of one step
            uint32_t key[kList];
            int index[kList];
            u64 weight[kList];
        };
    };
    u64 sums[kRanks];               // of the CTAs, in the order of their pieces
    u64 at[kWarps];
    u64 before;                     // what lies in front of `bin`
    float2 range[kRanks];           // each CTA's largest logit and smallest finite one
    int nan[kRanks];
    int bin;
    uint32_t count, kmin, kmax;     // rank 0: classes of the step, and the range of their keys
    uint32_t edge;                  // the last class kept
    int upto;
    int found;
};

// The order of fp32 numbers as that of 32-bit ones (-0 counts as +0).
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) { return __uint_as_float(key & 0x80000000u ? key & 0x7fffffffu : ~key); }

template <class T>
__device__ __forceinline__ T warp_sum(T v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan(u64 v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 left = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += left;
    }
    return v;
}

// One row as its cluster sees it.
struct Row {
    Smem &sm;
    const float *x;  // this CTA's piece, in shared memory
    int n, base;     // its length, and its first class
    int ranks, rank;
    float max;
    double inv_t;

    __device__ __forceinline__ void sync() const {
        if (ranks > 1) cg::this_cluster().sync();
        else __syncthreads();
    }
    // The same variable in the CTA of rank r.
    template <class V>
    __device__ __forceinline__ V *there(V *p, int r) const {
        return ranks > 1 ? cg::this_cluster().map_shared_rank(p, r) : p;
    }

    __device__ __forceinline__ u64 weight(float v) const {
        if (v == max) return 1ull << 44;
        if (v == -INFINITY || max == INFINITY) return 0;
        return __double2ull_rn(exp(((double)v - (double)max) * inv_t) * 17592186044416.0);
    }

    // f(i) of the classes of all pieces in the order of the index: the class at which their running sum exceeds above(total of
    // all).  The thread that finds it calls then(class).
    template <class F, class A, class Then>
    __device__ void first_above(F f, A above, Then then) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, each = ((n + kWarps - 1) / kWarps + 31) / 32 * 32;
        const int begin = min(warp * each, n), end = min(begin + each, n);
        u64 sum = 0;
        for (int i = begin + lane; i < end; i += 32) sum += f(i);
        sum = warp_sum(sum);
        if (lane == 0) sm.at[warp] = sum;
        __syncthreads();
        if (warp == 0) {
            const u64 all = warp_sum(lane < kWarps ? sm.at[lane] : 0);
            if (lane < ranks) *there(&sm.sums[rank], lane) = all;
        }
        sync();
        u64 before = 0, total = 0;
        for (int r = 0; r < ranks; r++) {
            if (r < rank) before += sm.sums[r];
            total += sm.sums[r];
        }
        for (int w = 0; w < warp; w++) before += sm.at[w];
        const u64 target = above(total);
        if (before <= target && before + sum > target) {  // one warp of the cluster
            for (int i = begin + lane; i - lane < end; i += 32) {
                const u64 run = before + warp_scan(i < end ? f(i) : 0, lane);
                const uint32_t hit = __ballot_sync(0xffffffffu, run > target);
                if (hit) {
                    if (lane == __ffs(hit) - 1) then(base + i);
                    break;
                }
                before = __shfl_sync(0xffffffffu, run, 31);
            }
        }
    }

    // The end of the run in which what `value` gives adds up to `need` (at most the total over what `in` lets through), the first
    // class first: edge and upto are set.  kMass: values are weights, else every class counts 1.  s: steps of the first histogram
    // in units of the logits.
    template <bool kMass, class In, class Need>
    __device__ void find_end(In in, Need need_of, float s) const {
        u64 need = 0, before = 0;
        uint32_t klo = 0, khi = 0xffffffffu;
        int shift = -1;  // of keys; the first histogram goes by values
#pragma unroll 1
        while (true) {
            auto bin_of = [&](float v, uint32_t key) { return shift < 0 ? (int)fminf((max - v) * s, (float)(kBins - 1)) : (int)((khi - key) >> shift); };
            for (int b = threadIdx.x; b < kBins; b += kThreads) sm.lo[b] = sm.hi[b] = 0;
            __syncthreads();
            for (int i = threadIdx.x; i < n; i += kThreads) {
                const float v = x[i];
                const uint32_t key = key_of(v);
                if (key < klo || key > khi || !in(key, i)) continue;
                const int b = bin_of(v, key);
                if (kMass) {
                    const u64 w = weight(v);
                    if (w == 0) continue;
                    const uint32_t low = (uint32_t)w, old = atomicAdd(&sm.lo[b], low), up = (uint32_t)(w >> 32) + (old + low < low);
                    if (up) atomicAdd(&sm.hi[b], up);
                } else {
                    atomicAdd(&sm.lo[b], 1u);
                }
            }
            sync();
            // every CTA adds up its share of the steps over the cluster
            const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share = kBins / ranks, per = share / kWarps >= 32 ? share / kWarps : 32;
            const int from = rank * share + warp * per, to = min(from + per, (rank + 1) * share);
            u64 part[kBins / kThreads] = {}, mine = 0;  // of steps from + 32 j + lane
#pragma unroll
            for (int j = 0; j < kBins / kThreads; j++) {
                const int b = from + 32 * j + lane;
                if (b < to)
                    for (int r = 0; r < ranks; r++) {
                        part[j] += *there(&sm.lo[b], r);
                        if (kMass) part[j] += (u64)*there(&sm.hi[b], r) << 32;
                    }
                mine += part[j];
            }
            mine = warp_sum(mine);
            if (lane == 0) sm.at[warp] = mine;
            __syncthreads();
            if (warp == 0) {
                const u64 all = warp_sum(lane < kWarps ? sm.at[lane] : 0);
                if (lane < ranks) *there(&sm.sums[rank], lane) = all;
            }
            if (rank == 0 && threadIdx.x == 0) sm.count = 0, sm.kmin = 0xffffffffu, sm.kmax = 0;
            sync();
            u64 run = before, total = 0;
            for (int r = 0; r < ranks; r++) {
                if (r < rank) run += sm.sums[r];
                total += sm.sums[r];
            }
            if (shift < 0) need = need_of(total);
            for (int w = 0; w < warp; w++) run += sm.at[w];
            if (run < need && run + mine >= need) {  // one warp of the cluster
#pragma unroll
                for (int j = 0; j < kBins / kThreads; j++) {
                    const u64 sum = run + warp_scan(part[j], lane);
                    const uint32_t hit = __ballot_sync(0xffffffffu, sum >= need);
                    if (hit) {
                        if (lane == __ffs(hit) - 1)
                            for (int r = 0; r < ranks; r++) *there(&sm.bin, r) = from + 32 * j + lane, *there(&sm.before, r) = sum - part[j];
                        break;
                    }
                    run = __shfl_sync(0xffffffffu, sum, 31);
                }
            }
            sync();
            const int bin = sm.bin;
            before = sm.before;
            // the classes of that step, at rank 0
            uint32_t *count = there(&sm.count, 0), *keys = there(&sm.key[0], 0), kmin = 0xffffffffu, kmax = 0;
            int *indexes = there(&sm.index[0], 0);
            for (int i = threadIdx.x; i - lane < n; i += kThreads) {
                const float v = i < n ? x[i] : 0.f;
                const uint32_t key = key_of(v);
                const bool hit = i < n && key >= klo && key <= khi && in(key, i) && bin_of(v, key) == bin;
                const uint32_t hits = __ballot_sync(0xffffffffu, hit);
                if (hits == 0) continue;
                uint32_t slot = 0;
                if (lane == 0) slot = atomicAdd(count, (uint32_t)__popc(hits));
                slot = __shfl_sync(0xffffffffu, slot, 0) + __popc(hits & ((1u << lane) - 1u));
                if (hit) {
                    kmin = min(kmin, key), kmax = ::max(kmax, key);
                    if (slot < kList) keys[slot] = key, indexes[slot] = base + i;
                }
            }
            kmin = __reduce_min_sync(0xffffffffu, kmin), kmax = __reduce_max_sync(0xffffffffu, kmax);
            if (lane == 0 && kmin <= kmax) atomicMin(there(&sm.kmin, 0), kmin), atomicMax(there(&sm.kmax, 0), kmax);
            sync();
            const uint32_t classes = *there(&sm.count, 0);
            klo = *there(&sm.kmin, 0), khi = *there(&sm.kmax, 0);
            if (classes <= kList) {
                if (rank == 0) {
                    if (kMass) {
                        for (int i = threadIdx.x; i < (int)classes; i += kThreads) sm.weight[i] = weight(value_of(sm.key[i]));
                        __syncthreads();
                    }
                    for (int i = threadIdx.x; i < (int)classes; i += kThreads) {
                        const uint32_t key = sm.key[i];
                        const int index = sm.index[i];
                        u64 sum = before;
                        for (int j = 0; j < (int)classes; j++) {
                            const uint32_t other = sm.key[j];
                            if (other > key || (other == key && sm.index[j] < index)) sum += kMass ? sm.weight[j] : 1;
                        }
                        const u64 own = kMass ? sm.weight[i] : 1;
                        if (sum < need && sum + own >= need)
                            for (int r = 0; r < ranks; r++) *there(&sm.edge, r) = key, *there(&sm.upto, r) = index;
                    }
                }
                sync();
                return;
            }
            if (klo == khi) {  // equal logits: so many of them, by the index
                const u64 own = kMass ? weight(value_of(klo)) : 1, some = (need - before + own - 1) / own;
                if (threadIdx.x == 0) sm.edge = klo;
                first_above([&](int i) { return (u64)(key_of(x[i]) == klo && in(klo, i)); }, [&](u64) { return some - 1; },
                            [&](int index) {
                                for (int r = 0; r < ranks; r++) *there(&sm.upto, r) = index;
                            });
                sync();
                return;
            }
            shift = ::max(0, 32 - __clz(khi - klo) - 11);
            sync();  // before the lists are used again
        }
    }
};

__global__ void __launch_bounds__(kThreads) sample_kernel(const float *logits, const float *u, const float *temperature, const int *top_k,
                                                          const float *top_p, const float *min_p, int *tokens, long long ld, int C, int piece) {
    extern __shared__ __align__(16) uint8_t raw[];
    Smem &sm = *reinterpret_cast<Smem *>(raw);
    float *x = reinterpret_cast<float *>(raw + sizeof(Smem));
    const int ranks = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank(), row = blockIdx.x / ranks;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    tc05::pdl_launch_dependents();
    tc05::pdl_wait();
    Row r{sm, x, max(0, min(piece, C - rank * piece)), rank * piece, ranks, rank, -INFINITY, 1.0};
    const float *src = logits + row * ld + r.base;
    float top = -INFINITY, low = INFINITY;
    bool bad = false;
#pragma unroll 8
    for (int i = threadIdx.x; i < r.n; i += kThreads) {
        const float v = src[i];
        x[i] = v;
        top = fmaxf(top, v);
        if (v > -INFINITY) low = fminf(low, v);
        bad |= v != v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
    }
    float2 *most = reinterpret_cast<float2 *>(sm.at);
    if (lane == 0) most[warp] = make_float2(top, low);
    bad = __syncthreads_or(bad);
    if (warp == 0) {
        const float2 v = most[lane % kWarps];
        top = v.x, low = v.y;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, o));
        }
        if (lane < ranks) *r.there(&sm.range[rank], lane) = make_float2(top, low), *r.there(&sm.nan[rank], lane) = bad;
    }
    const float T = temperature ? temperature[row] : 1.f, p = top_p ? top_p[row] : 1.f, least = min_p ? min_p[row] : 0.f, v = u[row];
    const int k = top_k ? top_k[row] : 0;
    r.sync();
    low = INFINITY, bad = false;
    for (int i = 0; i < ranks; i++) r.max = fmaxf(r.max, sm.range[i].x), low = fminf(low, sm.range[i].y), bad |= sm.nan[i] != 0;
    if (bad || r.max == -INFINITY) {  // the whole cluster; nobody looks at another CTA's memory any more
        if (rank == 0 && threadIdx.x == 0) tokens[row] = -1;
        return;
    }
    auto write = [&](int i) { tokens[row] = i; };
    if (!(T > 0.f)) {
        r.first_above([&](int i) { return (u64)(x[i] == r.max); }, [](u64) { return 0ull; }, write);
        return;
    }
    r.inv_t = 1.0 / (double)T;

    // the classes kept: keys above `edge`, and those equal to it up to class `upto`
    uint32_t edge = 0;
    int upto = C;
    auto in = [&](uint32_t key, int i) { return key > edge || (key == edge && r.base + i <= upto); };
    if (k >= 1 && k < C) {
        r.find_end<false>([](uint32_t, int) { return true; }, [&](u64) { return (u64)k; }, (float)(kBins - 1) / (r.max - low));
        edge = sm.edge, upto = sm.upto;
    }
    if (p < 1.f) {
        const u64 share = p > 0.f ? (u64)((double)p * 18446744073709551616.0) : 0;
        r.find_end<true>(in,
                         [&](u64 mass) {  // the smallest whole number that is at least p * mass
                             const u64 need = __umul64hi(share, mass) + (share * mass != 0);
                             return need ? need : 1;
                         },
                         64.f / T);
        edge = sm.edge, upto = sm.upto;
    }
    const u64 lowest = least > 0.f ? (least < 1.f ? (u64)ceil((double)least * 17592186044416.0) : 1ull << 44) : 0;
    const u64 part = v >= 1.f ? ~0ull : v > 0.f ? (u64)((double)v * 18446744073709551616.0) : 0;
    r.first_above(
        [&](int i) -> u64 {
            if (!in(key_of(x[i]), i)) return 0;
            const u64 w = r.weight(x[i]);
            return w >= lowest ? w : 0;
        },
        [&](u64 total) { return __umul64hi(part, total); }, write);
}

// CTAs of a row: as many as keep the SMs busy, with at least 2048 logits each, and enough for several to share an SM's memory.
int ranks_of(int rows, int C) {
    const int sms = attn::sm_count();
    int ranks = 1;
    while (ranks < kRanks && ((long long)rows * ranks < 2 * sms || C / ranks > 12800) && C / (2 * ranks) >= 2048) ranks *= 2;
    return ranks;
}

size_t smem_bytes(int piece) { return sizeof(Smem) + sizeof(float) * (size_t)piece; }

}  // namespace

cudaError_t set_attributes() {
    return cudaFuncSetAttribute(sample_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem_bytes(kMaxC / kRanks));
}

}  // namespace sample

extern "C" int xent_sm100_sample(const float *logits, const float *u, const float *temperature, const int *top_k, const float *top_p,
                                 const float *min_p, int *tokens, long long ld, int rows, int C, void *stream) {
    if (!logits || !u || !tokens) return ATTN_ERR_NULL;
    if (rows < 0 || C <= 0 || ld < C) return ATTN_ERR_ARGUMENT;
    if (C > sample::kMaxC || rows > 0x7fffffff / sample::kRanks) return ATTN_ERR_UNSUPPORTED;
    int *status = nullptr;
    const int rc = attn::device_status_word(&status);
    if (rc != ATTN_OK) return rc;
    if (rows == 0) return ATTN_OK;
    const int ranks = sample::ranks_of(rows, C), piece = (C + ranks - 1) / ranks;
    return (int)attn::launch_clusters_after_previous(sample::sample_kernel, dim3((unsigned)rows * ranks), dim3(sample::kThreads), sample::smem_bytes(piece),
                                                     (unsigned)ranks, static_cast<cudaStream_t>(stream), logits, u, temperature, top_k, top_p, min_p, tokens, ld,
                                                     C, piece);
}
