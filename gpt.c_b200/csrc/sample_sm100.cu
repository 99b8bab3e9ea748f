// The draw of a class from each row of logits, by temperature, top-k, top-p and min-p, for sm_100a.
//
// With the classes ordered by falling logit, equal ones by index, what each restriction keeps is a run from the front of
// that order, so the classes kept are those above one logit and, of those equal to it, the ones up to an index.  A weight is a
// whole number, round(2^44 exp((x - max) / T)): sums of up to 2^19 of them fit 64 bits and are exact in any order.
//
// A cluster of 1 to 8 CTAs holds a row in shared memory, each CTA a piece, and reads it once, 16 bytes at a time.
//
// Few classes matter where top-k or min-p is given: min-p leaves those within T ln(1 / min_p) of the largest logit; and no
// fewer than k logits lie at or above the k-th largest of the maxima of four neighbours each, which a histogram over a quarter as
// many values finds.  They go to a list in one CTA (up to 2048, most often little more than k), which ends the runs and draws.
// Otherwise, and where the list is too short, the cluster looks through the row: where a run ends is found by a histogram of counts or
// weights over 2048 steps of max - x, and the classes of the step in which it ends are put in order by comparing
// each with each; where they are too many for that, the histogram is taken again over their keys, 2048 times finer each time.
//
// Bound by the joins of a row's phases, not by HBM: 1 row of 50257, top-k 40, 10.1 us; 96 rows, top-p and min-p, 20.9 us; 500 rows, top-k 1000 and
// top-p, 94 us (three rounds of a row an SM), where reading takes 15.
#include <cooperative_groups.h>

#include <type_traits>

#include "attn_internal.h"
#include "tc05.cuh"

#include "../../include/xent_sm100.h"

namespace sample {
namespace {

namespace cg = cooperative_groups;

constexpr int kRanks = 8;      // CTAs of a row at most
constexpr int kBins = 2048;    // of a histogram
constexpr int kList = 512;     // classes that are compared each with each
constexpr int kMost = 2048;    // classes of the list
constexpr int kFew = 128;      // classes of a list that one thread each compares with all others
constexpr int kListThreads = 512, kEach = kMost / kListThreads;  // who works on it, and the classes of each
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
        struct {  // the same, of the list
            u64 order[kList], value[kList];
        };
        struct {
            uint32_t list_key[kMost];
            int list_index[kMost];
        };
    };
    double powers[64];              // 2^(i / 64)
    u64 sums[kRanks];               // of the CTAs, in the order of their pieces
    u64 at[32];                     // of this CTA's warps
    u64 before;                     // what lies in front of `bin`
    u64 end, omin, omax;            // in the list
    u64 front;                      // what lies in front of a stretch of the piece
    int stretch[2];
    float2 range[kRanks];           // each CTA's largest logit, NaN if one is, and its smallest maximum of four
    int bin;
    uint32_t count, kmin, kmax;     // rank 0: classes of the step, and the range of their keys
    uint32_t edge;                  // the last class kept
    int upto;
    int taken, counts[kRanks];      // classes that this CTA, each CTA has put in the list
    int first;                      // rank 0: the first class with the largest logit
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
template <class T>
__device__ __forceinline__ T warp_scan(T v, int lane) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const T left = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += left;
    }
    return v;
}

// For the threads that work on the list.
__device__ __forceinline__ void list_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kListThreads) : "memory"); }

__device__ __forceinline__ void few_sync() { asm volatile("bar.sync 1, %0;" ::"n"(kFew) : "memory"); }

// One row as its cluster sees it.
template <int kThreads>
struct Row {
    static constexpr int kWarps = kThreads / 32;
    Smem &sm;
    const float *x;    // this CTA's piece, in shared memory, from a 16-byte boundary of the row's memory on
    int begin, end;    // the logits in it; class of the first place: base
    int base, ranks, rank;
    float max;
    double by;         // 64 log2(e) / T

    // What the warps before this one have in `at`.
    __device__ __forceinline__ u64 in_front(int warps) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        return warp_sum(lane < warp && lane < warps ? sm.at[lane] : 0);
    }
    __device__ __forceinline__ void sync() const {
        if (ranks > 1) cg::this_cluster().sync();
        else __syncthreads();
    }
    // The same variable in the CTA of rank r.
    template <class V>
    __device__ __forceinline__ V *there(V *p, int r) const {
        return ranks > 1 ? cg::this_cluster().map_shared_rank(p, r) : p;
    }

    // 2^44 exp((v - max) / T) by 2^(n / 64) from a table and the series of exp for what is left, |r| <= ln(2) / 128: the first term
    // left out is 2^-44 of the result.  Adding 2^52 rounds it to a whole number.  max is finite.
    __device__ __forceinline__ u64 weight(float v) const {
        constexpr double kWhole = 6755399441055744.0, kLn = 0.010830424696249145;  // 1.5 * 2^52, ln(2) / 64
        const double d = (double)v - (double)max, k = fma(d, by, kWhole);
        const int n = __double2loint(k);
        const double r = fma(d, by, kWhole - k);
        const double s = r * fma(r, fma(r, fma(r, kLn * kLn * kLn * kLn / 24, kLn * kLn * kLn / 6), kLn * kLn / 2), kLn);
        const double p = sm.powers[n & 63], w = fma(p, s, p);
        const double whole = __hiloint2double(__double2hiint(w) + (((n >> 6) + 44) << 20), __double2loint(w)) + 4503599627370496.0;
        const bool some = k >= kWhole - 46.0 * 64;  // not where v is -inf
        return some ? (u64)(__double2hiint(whole) & 0xfffff) << 32 | (uint32_t)__double2loint(whole) : 0;
    }

    // f(i) of the classes of all pieces in the order of the index: the class at which their running sum exceeds above(total of
    // all).  The thread that finds it calls then(class).
    template <class F, class A, class Then>
    __device__ void first_above(F f, A above, Then then) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        // a stretch of the piece for each warp, added up; what lies in front of this warp's, and its own
        auto stretch = [&](int lo, int hi, int &from, int &to) {
            const int each = ((hi - lo + kWarps - 1) / kWarps + 31) / 32 * 32;
            from = min(lo + warp * each, hi), to = min(from + each, hi);
            u64 sum = 0;
#pragma unroll 4
            for (int i = from + lane; i < to; i += 32) sum += f(i);
            sum = warp_sum(sum);
            if (lane == 0) sm.at[warp] = sum;
            __syncthreads();
            return sum;
        };
        int from, to;
        u64 sum = stretch(begin, end, from, to);
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
        const u64 target = above(total);
        if (before > target || before + sm.sums[rank] <= target) return;  // not in this CTA's piece
        // the stretch in which it is, once more, by all warps
        before += in_front(kWarps);
        if (before <= target && before + sum > target && lane == 0) sm.stretch[0] = from, sm.stretch[1] = to, sm.front = before;
        __syncthreads();
        before = sm.front;
        sum = stretch(sm.stretch[0], sm.stretch[1], from, to);
        before += in_front(kWarps);
        if (before <= target && before + sum > target) {  // one warp
            for (int i = from + lane; i - lane < to; i += 32) {
                const u64 run = before + warp_scan(i < to ? f(i) : 0, lane);
                const uint32_t hit = __ballot_sync(0xffffffffu, run > target);
                if (hit) {
                    if (lane == __ffs(hit) - 1) then(base + i);
                    break;
                }
                before = __shfl_sync(0xffffffffu, run, 31);
            }
        }
    }

    // The cluster's histograms are there: the first step at which their running sum, from `before` on, reaches need_of(total); bin
    // and before (what lies in front of it) are set in every CTA.  Returns what was needed.
    template <bool kMass, class Need>
    __device__ u64 find_bin(u64 before, Need need_of) const {
        sync();
        // every CTA adds up its share of the steps over the cluster
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, share = kBins / ranks, per = share / kWarps >= 32 ? share / kWarps : 32;
        const int from = rank * share + warp * per, to = min(from + per, (rank + 1) * share);
        using Sum = std::conditional_t<kMass, u64, uint32_t>;
        Sum part[kBins / kThreads] = {}, mine = 0;  // of steps from + 32 j + lane
#pragma unroll
        for (int j = 0; j < kBins / kThreads; j++) {
            const int b = from + 32 * j + lane;
            if (b < to)
                for (int r = 0; r < ranks; r++) {
                    part[j] += *there(&sm.lo[b], r);
                    if constexpr (kMass) part[j] += (u64)*there(&sm.hi[b], r) << 32;
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
        sync();
        u64 run = before, total = 0;
        for (int r = 0; r < ranks; r++) {
            if (r < rank) run += sm.sums[r];
            total += sm.sums[r];
        }
        const u64 need = need_of(total);
        run += in_front(kWarps);
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
        return need;
    }
    __device__ __forceinline__ void clear() const {
        for (int b = threadIdx.x; b < kBins / 2; b += kThreads) reinterpret_cast<uint4 *>(sm.lo)[b] = make_uint4(0, 0, 0, 0);
        __syncthreads();
    }
    __device__ __forceinline__ void add(int b, u64 w) const {
        const uint32_t low = (uint32_t)w, old = atomicAdd(&sm.lo[b], low), up = (uint32_t)(w >> 32) + (old + low < low);
        if (up) atomicAdd(&sm.hi[b], up);
    }
    __device__ __forceinline__ int step_of(float v, float s) const { return (int)fminf((max - v) * s, (float)(kBins - 1)); }

    // The classes with logits of `least` (finite) and more to the list at rank 0.  Returns their number; those above kMost are not there.
    __device__ int gather(float least) const {
        if (threadIdx.x == 0) sm.count = 0, sm.taken = 0;
        sync();
        uint32_t *count = there(&sm.count, 0), *keys = there(&sm.list_key[0], 0), words = 0;
        int *indexes = there(&sm.list_index[0], 0);
        const int lane = threadIdx.x & 31;
        // a bit for each of this thread's words of four that has one; few have
        int j = 0;
#pragma unroll 4
        for (int i = 4 * threadIdx.x; i < end; i += 4 * kThreads, j++) {
            const float4 v = *reinterpret_cast<const float4 *>(x + i);
            words |= (uint32_t)(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) >= least) << j;
        }
        int mine = 0;
        for (uint32_t left = words; left; left &= left - 1) {
            const float4 v = *reinterpret_cast<const float4 *>(x + 4 * (threadIdx.x + (__ffs(left) - 1) * kThreads));
            mine += (v.x >= least) + (v.y >= least) + (v.z >= least) + (v.w >= least);
        }
        int run = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += left;
        }
        uint32_t slot = 0;
        if (lane == 31 && run) slot = atomicAdd(count, (uint32_t)run), atomicAdd(&sm.taken, run);
        slot = __shfl_sync(0xffffffffu, slot, 31) + run - mine;
        for (uint32_t left = words; left; left &= left - 1) {
            const int i = 4 * (threadIdx.x + (__ffs(left) - 1) * kThreads);
            const float4 v = *reinterpret_cast<const float4 *>(x + i);
            const float f[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (f[e] >= least) {
                    if (slot < kMost) keys[slot] = key_of(f[e]), indexes[slot] = base + i + e;
                    slot++;
                }
        }
        __syncthreads();
        if (threadIdx.x < ranks) *there(&sm.counts[rank], threadIdx.x) = sm.taken;
        sync();  // from here on rank 0 may go on alone
        int all = 0;
        for (int r = 0; r < ranks; r++) all += sm.counts[r];
        return all;
    }

    // In the list: the class at which the values, in rising order, add up to `need` (at most their sum).  Values of 0 take no part, orders
    // differ from each other; bins: steps of the first histogram, rising with the order.
    __device__ u64 cut(const u64 (&order)[kEach], const u64 (&value)[kEach], const int (&bins)[kEach], u64 need) const {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
        u64 before = 0, omin = 0, omax = ~0ull;
        int shift = -1;
#pragma unroll 1
        while (true) {
            auto step = [&](int j) { return value[j] == 0 || order[j] < omin || order[j] > omax ? -1 : shift < 0 ? bins[j] : (int)((order[j] - omin) >> shift); };
            list_sync();
            for (int b = threadIdx.x; b < kBins / 2; b += kListThreads) reinterpret_cast<uint4 *>(sm.lo)[b] = make_uint4(0, 0, 0, 0);
            list_sync();
#pragma unroll
            for (int j = 0; j < kEach; j++)
                if (step(j) >= 0) add(step(j), value[j]);
            if (threadIdx.x == 0) sm.count = 0, sm.omin = ~0ull, sm.omax = 0;
            list_sync();
            u64 part[kBins / kListThreads], mine = 0;
#pragma unroll
            for (int j = 0; j < kBins / kListThreads; j++) {
                const int b = threadIdx.x * (kBins / kListThreads) + j;
                part[j] = (u64)sm.hi[b] << 32 | sm.lo[b];
                mine += part[j];
            }
            const u64 scan = warp_scan(mine, lane);
            if (lane == 31) sm.at[warp] = scan;
            list_sync();
            u64 run = before + scan - mine + in_front(kListThreads / 32);
#pragma unroll
            for (int j = 0; j < kBins / kListThreads; j++) {
                if (run < need && run + part[j] >= need) sm.bin = threadIdx.x * (kBins / kListThreads) + j, sm.before = run;
                run += part[j];
            }
            list_sync();
            const int bin = sm.bin;
            before = sm.before;
#pragma unroll
            for (int j = 0; j < kEach; j++)
                if (step(j) == bin) {
                    const uint32_t slot = atomicAdd(&sm.count, 1u);
                    if (slot < kList) sm.order[slot] = order[j], sm.value[slot] = value[j];
                }
            list_sync();
            const int n = (int)sm.count;
            if (n <= kList) {
                for (int i = threadIdx.x; i < n; i += kListThreads) {
                    const u64 own = sm.order[i];
                    u64 sum = before;
                    for (int j = 0; j < n; j++) sum += sm.order[j] < own ? sm.value[j] : 0;
                    if (sum < need && sum + sm.value[i] >= need) sm.end = own;
                }
                list_sync();
                return sm.end;
            }
#pragma unroll
            for (int j = 0; j < kEach; j++)
                if (step(j) == bin) atomicMin(&sm.omin, order[j]), atomicMax(&sm.omax, order[j]);
            list_sync();
            omin = sm.omin, omax = sm.omax;
            shift = ::max(0, 64 - __clzll((long long)(omax - omin)) - 11);
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
            auto bin_of = [&](float v) { return shift < 0 ? step_of(v, s) : (int)((khi - key_of(v)) >> shift); };
            auto there_is = [&](float v, int i) { return in(v, i) && (shift < 0 || (key_of(v) >= klo && key_of(v) <= khi)); };
            clear();
#pragma unroll 4
            for (int i = begin + threadIdx.x; i < end; i += kThreads) {
                const float v = x[i];
                if (!there_is(v, i)) continue;
                const int b = bin_of(v);
                if (kMass) {
                    const u64 w = weight(v);
                    if (w) add(b, w);
                } else {
                    atomicAdd(&sm.lo[b], 1u);
                }
            }
            sync();
            if (rank == 0 && threadIdx.x == 0) sm.count = 0, sm.kmin = 0xffffffffu, sm.kmax = 0;
            need = find_bin<kMass>(before, [&](u64 total) { return shift < 0 ? need_of(total) : need; });
            const int bin = sm.bin, lane = threadIdx.x & 31;
            before = sm.before;
            // the classes of that step, at rank 0
            uint32_t *count = there(&sm.count, 0), *keys = there(&sm.key[0], 0), kmin = 0xffffffffu, kmax = 0;
            int *indexes = there(&sm.index[0], 0);
            for (int i = begin + threadIdx.x; i - lane < end; i += kThreads) {
                const float v = i < end ? x[i] : 0.f;
                const bool hit = i < end && there_is(v, i) && bin_of(v) == bin;
                const uint32_t hits = __ballot_sync(0xffffffffu, hit);
                if (hits == 0) continue;
                const uint32_t key = key_of(v);
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
                first_above([&](int i) { return (u64)(key_of(x[i]) == klo && in(x[i], i)); }, [&](u64) { return some - 1; },
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

__device__ __forceinline__ float max_nan(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// The smallest whole number that is at least p * mass, 1 at least.
__device__ __forceinline__ u64 part_of(float p, u64 mass) {
    const u64 share = p > 0.f ? (u64)((double)p * 18446744073709551616.0) : 0;
    const u64 need = __umul64hi(share, mass) + (share * mass != 0);
    return need ? need : 1;
}

template <int kThreads>
__global__ void __launch_bounds__(kThreads) sample_kernel(const float *logits, const float *u, const float *temperature, const int *top_k,
                                                          const float *top_p, const float *min_p, int *tokens, long long ld, int rows, int C, int words, int ahead) {
    extern __shared__ __align__(16) uint8_t raw[];
    Smem &sm = *reinterpret_cast<Smem *>(raw);
    float *x = reinterpret_cast<float *>(raw + sizeof(Smem));
    const int ranks = (int)cg::this_cluster().num_blocks(), rank = (int)cg::this_cluster().block_rank(), row = blockIdx.x / ranks;
    constexpr int kWarps = kThreads / 32;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (ranks > 1) tc05::cluster_arrive();  // waited for behind the loads
    if (threadIdx.x < 64) sm.powers[threadIdx.x] = exp2((double)threadIdx.x / 64);
    tc05::pdl_launch_dependents();
    tc05::pdl_wait();
    // the row in words of 16 bytes as they lie in memory, `words` of them a CTA; what is not in the row is -inf
    const float *src = logits + row * ld;
    const int skip = (int)((reinterpret_cast<uintptr_t>(src) >> 2) & 3), base = 4 * rank * words - skip;
    Row<kThreads> r{sm, x, max(0, -base), max(0, min(4 * words, C - base)), base, ranks, rank, -INFINITY, 1.0};
    float top = -INFINITY, low = INFINITY;
    if (ahead > 0 && threadIdx.x == 0 && row + ahead < rows) {  // the row that this SM takes next, to L2
        const char *from = reinterpret_cast<const char *>((reinterpret_cast<uintptr_t>(src + ahead * ld) + 15) & ~(uintptr_t)15);
        const int bytes = (4 * (C - 3)) & ~15;
        for (int i = 0; i < bytes; i += 16384)
            asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(from + i), "r"(min(16384, bytes - i)) : "memory");
    }
#pragma unroll 4
    for (int i = 4 * threadIdx.x; i < r.end; i += 4 * kThreads) {
        float4 v;
        if (i >= r.begin && i + 4 <= r.end) {
            v = *reinterpret_cast<const float4 *>(src + base + i);
        } else {
            float f[4];
            for (int e = 0; e < 4; e++) f[e] = i + e >= r.begin && i + e < r.end ? src[base + i + e] : -INFINITY;
            v = make_float4(f[0], f[1], f[2], f[3]);
        }
        *reinterpret_cast<float4 *>(x + i) = v;
        const float most = max_nan(max_nan(v.x, v.y), max_nan(v.z, v.w));
        top = max_nan(top, most);
        if (most > -INFINITY) low = fminf(low, most);
    }
    auto both = [&](float2 v) {  // over the warp
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            v.x = max_nan(v.x, __shfl_xor_sync(0xffffffffu, v.x, o));
            v.y = fminf(v.y, __shfl_xor_sync(0xffffffffu, v.y, o));
        }
        return v;
    };
    float2 *most = reinterpret_cast<float2 *>(sm.at);
    const float2 own = both(make_float2(top, low));
    if (lane == 0) most[warp] = own;
    if (threadIdx.x == 0) sm.first = 0x7fffffff;
    __syncthreads();
    if (ranks > 1) tc05::cluster_wait();  // the other CTAs have begun: their shared memory is there
    if (warp == 0) {
        const float2 all = both(most[lane % kWarps]);
        if (lane < ranks) *r.there(&sm.range[rank], lane) = all;
    }
    const float T = temperature ? temperature[row] : 1.f, p = top_p ? top_p[row] : 1.f, least = min_p ? min_p[row] : 0.f, draw = u[row];
    const int k = top_k ? top_k[row] : 0;
    r.sync();
    low = INFINITY;
    for (int i = 0; i < ranks; i++) r.max = max_nan(r.max, sm.range[i].x), low = fminf(low, sm.range[i].y);
    if (!(r.max > -INFINITY)) {  // the whole cluster; nobody looks at another CTA's memory any more
        if (rank == 0 && threadIdx.x == 0) tokens[row] = -1;
        return;
    }
    if (r.max == INFINITY) {  // it has all the weight
        for (int i = threadIdx.x; i < r.end; i += kThreads) x[i] = x[i] == INFINITY ? 0.f : -INFINITY;
        r.max = low = 0.f;
        top = top == INFINITY ? 0.f : -INFINITY;
        __syncthreads();
    }
    if (!(T > 0.f) || k == 1 || p <= 0.f) {  // the first of the largest
        int first = 0x7fffffff;
        for (int i = 4 * threadIdx.x; i < r.end; i += 4 * kThreads) {
            const float4 v = *reinterpret_cast<const float4 *>(x + i);
            if (first < 0x7fffffff || !(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)) == r.max)) continue;
            first = base + i + (v.x == r.max ? 0 : v.y == r.max ? 1 : v.z == r.max ? 2 : 3);
        }
        first = __reduce_min_sync(0xffffffffu, first);
        if (lane == 0 && first < 0x7fffffff) atomicMin(r.there(&sm.first, 0), first);
        r.sync();
        if (rank == 0 && threadIdx.x == 0) tokens[row] = sm.first;
        return;
    }
    r.by = 64 * 1.4426950408889634 / (double)T;
    const u64 lowest = least > 0.f ? (least < 1.f ? (u64)ceil((double)least * 17592186044416.0) : 1ull << 44) : 0;
    const u64 part = draw >= 1.f ? ~0ull : draw > 0.f ? (u64)((double)draw * 18446744073709551616.0) : 0;
    const bool by_k = k > 1 && k < C, by_p = p < 1.f;

    // the list of classes that matter, if it is a short one
    const float s = (float)(kBins - 1) / (r.max - low);
    u64 mass = 0;
    int listed = kMost + 1;
    if (by_k && k <= kMost) {
        r.clear();
        u64 words_in_all = 0;
        if (3 * k <= kThreads * ranks) {  // few: the largest of each thread are enough of them
            atomicAdd(&sm.lo[r.step_of(top, s)], 1u);
        } else {
            for (int i = 4 * threadIdx.x; i < r.end; i += 4 * kThreads) {
                const float4 v = *reinterpret_cast<const float4 *>(x + i);
                atomicAdd(&sm.lo[r.step_of(fmaxf(fmaxf(v.x, v.y), fmaxf(v.z, v.w)), s)], 1u);
            }
        }
        r.find_bin<false>(0, [&](u64 total) { return words_in_all = total, min((u64)k, total); });
        // the logits at the end of that step, and what its rounding may hide; the last step has no end
        const float least_of_them = sm.bin == kBins - 1 ? -INFINITY : r.max - (float)(sm.bin + 1) / s * 1.00001f - 1e-6f * fabsf(r.max);
        if (words_in_all >= (u64)k) listed = r.gather(fmaxf(least_of_them, -3.402823466e38f));
    } else if (!by_k && lowest) {
        if (by_p) {
            u64 sum = 0;
#pragma unroll 4
            for (int i = r.begin + threadIdx.x; i < r.end; i += kThreads) sum += r.weight(x[i]);
            sum = warp_sum(sum);
            if (lane == 0) sm.at[warp] = sum;
            __syncthreads();
            if (warp == 0) {
                sum = warp_sum(lane < kWarps ? sm.at[lane] : 0);
                if (lane < ranks) *r.there(&sm.sums[rank], lane) = sum;
            }
        }
        // T ln(1 / min_p) below the largest, and a little more than rounding, to 2^-44 too, may hide: the list is looked through by weight
        const float reach = T * (1e-5f - 1.00001f * logf(fmaxf(fminf(least, 1.f) - 1.2e-13f, 1.4e-14f)));
        listed = r.gather(fmaxf(r.max - reach - 1e-6f * fabsf(r.max), -3.402823466e38f));
        for (int i = 0; i < ranks; i++) mass += sm.sums[i];
    }
    if (listed <= kFew) {
        // every class against each other, one a thread
        if (rank > 0 || threadIdx.x >= kFew) return;
        const int i = threadIdx.x;
        const bool in = i < listed;
        const uint32_t key = in ? sm.list_key[i] : 0, index = in ? sm.list_index[i] : 0;
        const u64 order = (u64)~key << 32 | index;
        u64 weight = in ? r.weight(value_of(key)) : 0;
        few_sync();
        sm.order[i] = order, sm.value[i] = weight;
        few_sync();
        u64 front = 0, all = 0;  // the weight of the classes before this one
        int place = 0;           // their number
        for (int j = 0; j < listed; j++) {
            const bool before = sm.order[j] < order;
            place += before;
            front += before ? sm.value[j] : 0;
        }
        if (by_k && place >= k) weight = 0;
        auto total = [&] {  // of the weights left
            const u64 v = warp_sum(weight);
            if (lane == 0) sm.at[warp] = v;
            few_sync();
            return warp_sum(lane < kFew / 32 ? sm.at[lane] : 0);
        };
        all = total();
        if (by_p && front >= part_of(p, by_k ? all : mass)) weight = 0;
        if (weight < lowest) weight = 0;
        sm.order[i] = index, sm.value[i] = weight;
        few_sync();
        const u64 target = __umul64hi(part, total());
        front = 0;
        for (int j = 0; j < listed; j++) front += sm.order[j] < index ? sm.value[j] : 0;
        if (front <= target && front + weight > target) tokens[row] = (int)index;
        return;
    }
    if (listed <= kMost) {
        if (rank > 0 || threadIdx.x >= kListThreads) return;
        u64 order[kEach], weight[kEach], value[kEach];
        int bins[kEach], index[kEach];
        const float per = 64.f / T;
#pragma unroll
        for (int j = 0; j < kEach; j++) {
            const int i = threadIdx.x + j * kListThreads;
            const bool in = i < listed;
            const uint32_t key = in ? sm.list_key[i] : 0;
            index[j] = in ? sm.list_index[i] : 0;
            order[j] = (u64)~key << 32 | (uint32_t)index[j];
            weight[j] = in ? r.weight(value_of(key)) : 0;
            value[j] = in;
            bins[j] = by_k ? r.step_of(value_of(key), s) : r.step_of(value_of(key), per);
        }
        u64 end = ~0ull;
        if (by_k && listed > k) end = r.cut(order, value, bins, (u64)k);  // fewer than k: the others are at -inf
        u64 sum = 0;
        auto total = [&] {  // of the weights up to the end
            u64 v = 0;
#pragma unroll
            for (int j = 0; j < kEach; j++) v += value[j] = order[j] <= end ? weight[j] : 0;
            v = warp_sum(v);
            list_sync();
            if (lane == 0) sm.at[warp] = v;
            list_sync();
            return warp_sum(lane < kListThreads / 32 ? sm.at[lane] : 0);
        };
        sum = total();
        if (by_p) {
            const u64 need = part_of(p, by_k ? sum : mass);
            if (need <= sum) {  // else all of the list is within it
#pragma unroll
                for (int j = 0; j < kEach; j++) bins[j] = r.step_of(value_of(~(uint32_t)(order[j] >> 32)), per);
                end = r.cut(order, value, bins, need);
            }
        }
#pragma unroll
        for (int j = 0; j < kEach; j++)
            if (weight[j] < lowest) weight[j] = 0;
        sum = total();
        int step = 0;
        while ((C - 1) >> step >= kBins) step++;
#pragma unroll
        for (int j = 0; j < kEach; j++) order[j] = (uint32_t)index[j], bins[j] = index[j] >> step;
        const u64 token = r.cut(order, value, bins, __umul64hi(part, sum) + 1);
        if (threadIdx.x == 0) tokens[row] = (int)token;
        return;
    }

    // the classes kept: logits above `edge`, and those equal to it up to class `upto`
    float edge = -INFINITY;
    int upto = C;
    auto in = [&](float v, int i) { return v > edge || (v == edge && r.base + i <= upto); };
    if (by_k) {
        r.find_end<false>([](float, int) { return true; }, [&](u64) { return (u64)k; }, s);
        edge = value_of(sm.edge), upto = sm.upto;
    }
    if (by_p) {
        r.find_end<true>(in, [&](u64 total) { return part_of(p, total); }, 64.f / T);
        edge = value_of(sm.edge), upto = sm.upto;
    }
    auto target = [&](u64 total) { return __umul64hi(part, total); };
    auto write = [&](int i) { tokens[row] = i; };
    if (!by_k && !by_p && !lowest)
        r.first_above([&](int i) { return r.weight(x[i]); }, target, write);
    else
        r.first_above(
            [&](int i) -> u64 {
                if (!in(x[i], i)) return 0;
                const u64 w = r.weight(x[i]);
                return w >= lowest ? w : 0;
            },
            target, write);
}

// CTAs of a row: one, of 1024 threads, where there are enough rows to fill the SMs or a row is short, else as many, of 512,
// as give each SM one, with at least 2048 logits each; and enough for a row to fit.
constexpr int kAlone = 53000;  // logits that one CTA can hold
int ranks_of(int rows, int C) {
    const int sms = attn::sm_count();
    int ranks = 1;
    while (ranks < kRanks && (C / ranks > kAlone || ((long long)rows * ranks * 2 <= sms - 20 && C / (2 * ranks) >= 2048))) ranks *= 2;
    return ranks;
}

size_t smem_bytes(int words) { return sizeof(Smem) + 16 * (size_t)words; }
int words_of(int C, int ranks) { return (C + 3 + 4 * ranks - 1) / (4 * ranks); }  // of 16 bytes, wherever the row begins

}  // namespace

cudaError_t set_attributes() {
    const cudaFuncAttribute at = cudaFuncAttributeMaxDynamicSharedMemorySize;
    const cudaError_t e = cudaFuncSetAttribute(sample_kernel<512>, at, (int)smem_bytes(words_of(kMaxC, kRanks)));
    return e != cudaSuccess ? e : cudaFuncSetAttribute(sample_kernel<1024>, at, (int)smem_bytes(words_of(kAlone, 1)));
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
    const int ranks = sample::ranks_of(rows, C), words = sample::words_of(C, ranks);
    const bool alone = ranks == 1;
    return (int)attn::launch_clusters_after_previous(alone ? sample::sample_kernel<1024> : sample::sample_kernel<512>, dim3((unsigned)rows * ranks),
                                                     dim3(alone ? 1024 : 512), sample::smem_bytes(words), (unsigned)ranks, static_cast<cudaStream_t>(stream),
                                                     logits, u, temperature, top_k, top_p, min_p, tokens, ld, rows, C, words,
                                                     alone && C > 3 ? attn::sm_count() : 0);  // 1024 threads of 64 registers: one CTA an SM
}
