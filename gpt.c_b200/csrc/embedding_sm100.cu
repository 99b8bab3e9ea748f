// Rows of the token table, scaled, with rows of the position table added; and the gradients of both tables, for sm_100a.
//
//     y[t] = scale table[tokens[t]] + pos_table[positions[t]]
//     dtable[v] += scale sum over tokens[t] = v of dy[t]          dpos_table[p] += sum over positions[t] = p of dy[t]
//
// Lookup: a copy, bound by HBM where the rows are many and by a launch where they are few.
//
// Gradient: the places t are put in the order of their tokens (equal tokens by t), and the sorted list is cut into ranges of the same
// number of places, whatever the tokens are.  A thread keeps the sum of a few columns over a run of equal tokens and adds it to the table
// where the run ends; the parts of runs that cross a border of a range are kept, and a last kernel adds them up in the order of the
// list.  So every sum has a fixed order, and a token that takes half of the batch is spread over the GPU.
//
// Three ways to the order, by the number of places: up to 512 no list at all (few_kernel); up to 8192 one CTA for each of 128 buckets of tokens
// (bucket_kernel), since the GPU is empty meanwhile; above, one cluster (sort_kernel), next to which the other CTAs of that launch make the
// gradient of positions that are a token's place in its sequence, where no list is needed.
#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "attn_internal.h"
#include "ids.cuh"
#include "tc05.cuh"

#include "../../include/tensor_sm100.h"

namespace embed {
namespace {

namespace cg = cooperative_groups;
using tc05::pack_bf16x2;
using tc05::pdl_launch_dependents;
using tc05::pdl_wait;

constexpr int kThreads = 256, kUnits = 4;
constexpr int kSortThreads = 1024, kSortCtas = 8, kSortWarps = kSortThreads / 32;
constexpr int kBits = 9, kBins = 1 << kBits;  // of a pass of the sort, at most
constexpr int kItems = 8;                     // places of a lane in a round of the sort
constexpr int kAhead = 8;                     // places whose rows a thread asks for together
// CTAs that sort without a cluster, and the longest list they take, which is what their shared memory holds.  (8192 places of 768 fp32 columns, the whole
// gradient: 16.5 us, by the cluster 30.)
constexpr int kBucketBits = 7, kBucketed = 8192;
// Places of a bucket that are compared each with each, by numbers of 32 bits: no token's own, V, has to have 30 bits as well, so a table of 2^30 rows takes the other way.
constexpr int kComparedBits = 9, kCompared = 1 << kComparedBits, kComparedRows = (1 << 30) - 1;
static_assert((kComparedRows >> kBucketBits) < 1 << (32 - kComparedBits), "a token's digits above its bucket's, V's among them, fit above a place");
// Where each place can look at all others.  (768 fp32 columns, by buckets in brackets: 16 places 3.4 us (10.5), 512 places 6.8 (11.2); its time grows with
// the square.)
constexpr int kFewTokens = 512;

// kN columns of a row as they are in memory: one value, or 8, 16 or 32 bytes.  A thread asks for several before it looks at one: turned into fp32 where it
// arrives, under a condition, each load was waited for by itself (runs of 49152 rows of 1600 bf16 values: 230 us).
template <class T, int kN>
struct Raw {
    static constexpr int kWords = kN * sizeof(T) / 4;
    uint32_t w[kWords ? kWords : 1];

    // sum += these
    __device__ __forceinline__ void add_to(float (&sum)[kN]) const {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kN; i++) sum[i] += __uint_as_float(w[i]);
        } else if constexpr (kN == 1) {
            sum[0] += __uint_as_float(w[0] << 16);
        } else {
#pragma unroll
            for (int i = 0; i < kN / 2; i++) sum[2 * i] += __uint_as_float(w[i] << 16), sum[2 * i + 1] += __uint_as_float(w[i] & 0xffff0000u);
        }
    }
    // these += scale * sum, rounded once
    __device__ __forceinline__ void add(const float (&sum)[kN], float scale) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int i = 0; i < kN; i++) w[i] = __float_as_uint(fmaf(sum[i], scale, __uint_as_float(w[i])));
        } else if constexpr (kN == 1) {
            w[0] = pack_bf16x2(fmaf(sum[0], scale, __uint_as_float(w[0] << 16)), 0.f);
        } else {
#pragma unroll
            for (int i = 0; i < kN / 2; i++)
                w[i] = pack_bf16x2(fmaf(sum[2 * i], scale, __uint_as_float(w[i] << 16)), fmaf(sum[2 * i + 1], scale, __uint_as_float(w[i] & 0xffff0000u)));
        }
    }

    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < (kWords ? kWords : 1); i++) w[i] = 0;
    }
    __device__ __forceinline__ void load(const T *p) {
        if constexpr (kWords == 8)
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(p));
        else if constexpr (kWords == 4) *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(p);
        else if constexpr (kWords == 2) *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(p);
        else if constexpr (sizeof(T) == 4) w[0] = __float_as_uint(*p);
        else w[0] = *reinterpret_cast<const unsigned short *>(p);
    }
    __device__ __forceinline__ void store(T *p) const {
        if constexpr (kWords == 8)
            asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]),
                         "r"(w[6]), "r"(w[7])
                         : "memory");
        else if constexpr (kWords == 4) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<const uint4 *>(w);
        else if constexpr (kWords == 2) *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<const uint2 *>(w);
        else if constexpr (sizeof(T) == 4) *p = __uint_as_float(w[0]);
        else *reinterpret_cast<unsigned short *>(p) = (unsigned short)w[0];
    }
    // scale * this + y, rounded once to fp32, and to bf16 where the values are that
    __device__ __forceinline__ void multiply_add(float scale, const Raw &y) {
#pragma unroll
        for (int i = 0; i < (kWords ? kWords : 1); i++) {
            if constexpr (sizeof(T) == 4)
                w[i] = __float_as_uint(fmaf(__uint_as_float(w[i]), scale, __uint_as_float(y.w[i])));
            else
                w[i] = pack_bf16x2(fmaf(__uint_as_float(w[i] << 16), scale, __uint_as_float(y.w[i] << 16)),
                                   fmaf(__uint_as_float(w[i] & 0xffff0000u), scale, __uint_as_float(y.w[i] & 0xffff0000u)));
        }
    }
};

struct Lookup {
    const void *table, *pos_table;  // pos_table NULL: none
    void *y;
    long long ld, pos_ld, n;
    Ids tokens, positions;          // positions NULL: a token's place in its sequence of T
    int T, C, V, P;
    float scale;
};

// kN columns at a time; a block takes `rows` rows of `words` such pieces.  i / words for i < 2^16 is the upper half of i * magic.
// Pieces of a thread: two where they are 32 bytes of two tables, whose four take too many registers.
// 8192 rows of 768 fp32 values with positions 6.5 us with everything in L2, 8.9 from HBM (4500 GB/s): two loads that wait for each other, 2.8 rounds of blocks, and 97 MB from
// L2, a quarter of them rows of positions that each sequence reads again; 49152 of 1600 bf16 values without positions 46 to 48 us (5500 GB/s, HBM).  Rows that start anywhere go a
// value at a time: 8192 x 767 28 us (fp32) and 35 (bf16), 49152 x 1599 bf16 350.
constexpr int units_of(int bytes, bool places) { return bytes == 32 && places ? 2 : kUnits; }
template <class E, int kN, bool kPlaces>
__global__ void __launch_bounds__(kThreads, 4) lookup_kernel(Lookup a, int rows, int words, unsigned magic) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kUnits = units_of(kN * sizeof(E), kPlaces);
    const long long row0 = (long long)blockIdx.x * rows;
    const int here = (int)min((long long)rows, a.n - row0) * words;
    const unsigned place0 = kPlaces && !a.positions.p ? (unsigned)(row0 % a.T) : 0;
    for (int i0 = threadIdx.x; i0 < here; i0 += kThreads * kUnits) {
        int row[kUnits], col[kUnits], token[kUnits], place[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            const int i = i0 + u * kThreads;
            row[u] = rows == 1 ? 0 : words == 1 ? i : (int)__umulhi((unsigned)i, magic);
            col[u] = (i - row[u] * words) * kN;
            token[u] = place[u] = -1;
            if (i >= here) continue;
            token[u] = a.tokens.at(row0 + row[u], a.V);
            if (kPlaces) {
                const int p = a.positions.p ? a.positions.at(row0 + row[u], a.P) : (int)((place0 + (unsigned)row[u]) % (unsigned)a.T);
                place[u] = p < a.P ? p : -1;
            }
        }
        Raw<E, kN> x[kUnits], y[kPlaces ? kUnits : 1];
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            x[u].clear(), y[kPlaces ? u : 0].clear();
            if (token[u] >= 0) x[u].load(static_cast<const E *>(a.table) + token[u] * a.ld + col[u]);
            if (kPlaces && place[u] >= 0) y[u].load(static_cast<const E *>(a.pos_table) + place[u] * a.pos_ld + col[u]);
        }
#pragma unroll
        for (int u = 0; u < kUnits; u++) {
            if (i0 + u * kThreads >= here) continue;
            x[u].multiply_add(a.scale, y[kPlaces ? u : 0]);
            x[u].store(static_cast<E *>(a.y) + (row0 + row[u]) * a.C + col[u]);
        }
    }
}

// One table's gradient.
struct List {
    Ids ids;
    void *grad;
    long long ld;
    int V, n;
    float scale;
    int2 *places[2];      // tokens and their places, as the passes of the sort take turns
    const int2 *sorted;   // the one that holds the result
    int passes, bits;     // of a pass
    int length, ranges;   // places of a range
    float *head, *tail;   // [ranges, C]: parts of the run that came into a range, and of the one that leaves it
};
struct Gradient {
    const void *dy;
    long long ld;
    List list[2];
    int lists, C;
    int T, P;             // positions that are a token's place: sequences of T, table of P (T 0: none)
    int place_width;      // pieces of rows of that table that a block has at a time, a power of two
    long long n;
    void *pos_grad;
    long long pos_ld;
};

constexpr int kPitch = kBins + 1;  // four threads that add up a digit's counts read four rows of `warp` in different banks

struct SortSmem {
    int2 sorted[kSortThreads * kItems];  // a round's places by digit, so that they leave in runs
    int warp[kSortWarps][kPitch];
    int count[kBins], base[kBins], first[kBins], scan[kSortWarps];
};

// Running sums over the threads of a block: what is in front of `v`.
__device__ __forceinline__ int in_front(int v, int *scan) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int sum = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int left = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += left;
    }
    if (lane == 31) scan[warp] = sum;
    __syncthreads();
    const int other = lane < warp ? scan[lane] : 0;
    __syncthreads();
    return __reduce_add_sync(0xffffffffu, other) + sum - v;
}

// A block's round of a stable sort by one digit: up to kItems places a lane, all of a warp's next to each other.  Of places with the same digit, a
// warp's own order is kept by votes on the digit's bits, that of the warps by running sums of their counts.
struct Round {
    int k[kItems], place[kItems], in_warp[kItems];  // k < 0: none
    int items, bits, shift;

    __device__ __forceinline__ int digit(int key) const { return key >> shift & ((1 << bits) - 1); }
    __device__ __forceinline__ int first(int begin) const { return begin + (int)(threadIdx.x >> 5) * items * 32 + (int)(threadIdx.x & 31); }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int r = 0; r < kItems; r++) k[r] = -1;
    }
    // places[begin] to places[end - 1] (begin < end)
    __device__ __forceinline__ void read(const int2 *places, int begin, int end) {
        const int i0 = first(begin);
        int2 e[kItems];
#pragma unroll
        for (int r = 0; r < kItems; r++) e[r] = __ldcg(places + min(i0 + 32 * r, end - 1));
#pragma unroll
        for (int r = 0; r < kItems; r++) k[r] = r < items && i0 + 32 * r < end ? e[r].x : -1, place[r] = e[r].y;
    }
    __device__ __forceinline__ void read(const Ids &ids, int V, int begin, int end) {
        const int i0 = first(begin);
        ids.many<kItems>(k, V, i0, 32, end);
#pragma unroll
        for (int r = 0; r < kItems; r++) {
            place[r] = i0 + 32 * r;
            if (r >= items || place[r] >= end) k[r] = -1;
            else if (k[r] < 0) k[r] = V;
        }
    }
    // What sm.warp and sm.count hold then: of each digit, places of the warps before each; of them all.
    __device__ __forceinline__ void rank(SortSmem &sm) {
        const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, bins = 1 << bits;
        for (int i = lane; i < bins; i += 32) sm.warp[warp][i] = 0;
        __syncwarp();
#pragma unroll
        for (int r = 0; r < kItems; r++) {
            if (r >= items) break;
            const int d = digit(k[r]);
            unsigned same = __ballot_sync(0xffffffffu, k[r] >= 0);  // lanes with this digit
#pragma unroll
            for (int b = 0; b < kBits; b++) {
                if (b >= bits) break;
                const bool set = d >> b & 1;
                const unsigned vote = __ballot_sync(0xffffffffu, set);
                same &= set ? vote : ~vote;
            }
            const int seen = k[r] < 0 ? 0 : sm.warp[warp][d];
            __syncwarp();
            if (k[r] >= 0 && lane == __ffs(same) - 1) sm.warp[warp][d] = seen + __popc(same);
            __syncwarp();
            in_warp[r] = seen + __popc(same & ((1u << lane) - 1));
        }
        __syncthreads();
        for (int d0 = 0; d0 < bins; d0 += kSortThreads / 4) {  // two rounds of threads where there are 512 digits
            const int d = d0 + (int)(threadIdx.x >> 2), q = threadIdx.x & 3;
            int c[kSortWarps / 4], sum = 0;
            if (d < bins) {
#pragma unroll
                for (int w = 0; w < kSortWarps / 4; w++) c[w] = sm.warp[q * (kSortWarps / 4) + w][d], sum += c[w];
            }
            int before = sum;
            const int one = __shfl_up_sync(0xffffffffu, before, 1);
            if (q >= 1) before += one;
            const int two = __shfl_up_sync(0xffffffffu, before, 2);
            if (q >= 2) before += two;
            if (d < bins) {
                if (q == 3) sm.count[d] = before;
                before -= sum;
#pragma unroll
                for (int w = 0; w < kSortWarps / 4; w++) sm.warp[q * (kSortWarps / 4) + w][d] = before, before += c[w];
            }
        }
        __syncthreads();
    }
    // The round's `count` places leave for out[sm.base[digit]] and on, by way of shared memory: stored there one by one each took a sector
    // (49152 places: 14 us of 20 a pass).
    __device__ __forceinline__ void scatter(SortSmem &sm, int2 *out, int count) {
        const int d = threadIdx.x;
        const int front = in_front(d < 1 << bits ? sm.count[d] : 0, sm.scan);
        if (d < 1 << bits) sm.first[d] = front;
        __syncthreads();
#pragma unroll
        for (int r = 0; r < kItems; r++) {
            if (k[r] < 0) continue;
            const int digit_r = digit(k[r]);
            sm.sorted[sm.first[digit_r] + sm.warp[threadIdx.x >> 5][digit_r] + in_warp[r]] = make_int2(k[r], place[r]);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < count; i += kSortThreads) {
            const int2 e = sm.sorted[i];
            out[sm.base[digit(e.x)] + i - sm.first[digit(e.x)]] = e;
        }
    }
};

// The places of a list in the order of their tokens, 2^bits tokens a pass, from the lowest digit on.  A cluster; each CTA has a piece.
__device__ void sort_list(const List &l, SortSmem &sm) {
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), bins = 1 << l.bits;
    const int piece = ((l.n + kSortCtas - 1) / kSortCtas + 31) / 32 * 32;
    const int from = (int)min((long long)l.n, (long long)rank * piece), to = (int)min((long long)l.n, (long long)from + piece);
    Round r;
    r.items = min(kItems, (piece + kSortThreads - 1) / kSortThreads), r.bits = l.bits;
    const int round = r.items * kSortThreads;
    for (int pass = 0; pass < l.passes; pass++) {
        r.shift = pass * l.bits;
        const int2 *in = l.places[pass & 1];
        int2 *out = l.places[(pass & 1) ^ 1];
        auto read = [&](int begin) {
            if (begin >= to) r.clear();
            else if (pass == 0) r.read(l.ids, l.V, begin, to);
            else r.read(in, begin, to);
        };
        const bool once = piece <= round;
        const int d = threadIdx.x;
        if (once) {  // the whole piece is in registers
            read(from);
            r.rank(sm);
        } else {
            if (d < bins) sm.count[d] = 0;
            __syncthreads();
            for (int begin = from; begin < to; begin += round) {
                read(begin);
#pragma unroll
                for (int i = 0; i < kItems; i++)
                    if (r.k[i] >= 0) atomicAdd(&sm.count[r.digit(r.k[i])], 1);
            }
        }
        cluster.sync();
        // where this CTA's places of each digit go
        int all = 0, before = 0;
        if (d < bins) {
            int v[kSortCtas];
#pragma unroll
            for (int c = 0; c < kSortCtas; c++) v[c] = cluster.map_shared_rank(sm.count, c)[d];
#pragma unroll
            for (int c = 0; c < kSortCtas; c++) {
                if (c < rank) before += v[c];
                all += v[c];
            }
        }
        const int front = in_front(all, sm.scan);
        if (d < bins) sm.base[d] = front + before;
        if (once) {
            r.scatter(sm, out, to - from);
        } else {
            cluster.sync();  // the counts have been read
            for (int begin = from; begin < to; begin += round) {
                read(begin);
                r.rank(sm);
                r.scatter(sm, out, min(round, to - begin));
                __syncthreads();
                if (d < bins) sm.base[d] += sm.count[d];
                __syncthreads();
            }
        }
        cluster.sync();  // what the others have written is there for the next pass, and nobody reads the counts any more
    }
}

// The same for lists of up to kBucketed places, by CTAs that need not wait for each other: each looks through all tokens and takes those with its
// lowest digit, whose order among each other it then makes by comparing each with each, or by the digits above.
struct BucketSmem {
    SortSmem sort;
    int2 mine[kBucketed];
};
__device__ void sort_bucket(const List &l, int bucket, BucketSmem &sm) {
    constexpr int kMost = kBucketed / kSortThreads;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int items = (l.n + kSortThreads - 1) / kSortThreads, i0 = warp * items * 32 + lane;
    int less = 0, mine = 0;  // of this warp
    unsigned votes[kMost];
    int k[kMost];
    l.ids.many<kMost>(k, l.V, i0, 32, l.n);
#pragma unroll
    for (int r = 0; r < kMost; r++) {
        const bool there = r < items && i0 + 32 * r < l.n;
        if (k[r] < 0) k[r] = l.V;
        const int d = k[r] & ((1 << kBucketBits) - 1);
        less += __popc(__ballot_sync(0xffffffffu, there && d < bucket));
        votes[r] = __ballot_sync(0xffffffffu, there && d == bucket);
        mine += __popc(votes[r]);
    }
    int at = in_front(lane == 0 ? mine : 0, sm.sort.scan);
    if (lane == 31) sm.sort.count[warp] = less, sm.sort.count[32 + warp] = mine;
    at = __shfl_sync(0xffffffffu, at, 0);
    __syncthreads();
    const int base = __reduce_add_sync(0xffffffffu, sm.sort.count[lane]), count = __reduce_add_sync(0xffffffffu, sm.sort.count[32 + lane]);
#pragma unroll
    for (int r = 0; r < kMost; r++) {
        if (votes[r] >> lane & 1) sm.mine[at + __popc(votes[r] & ((1u << lane) - 1))] = make_int2(k[r], i0 + 32 * r);
        at += __popc(votes[r]);
    }
    __syncthreads();
    if (count == 0) return;
    if (count <= kCompared && l.V <= kComparedRows) {  // each with each: a token's other digits and its place in the bucket as one number
        uint32_t *all = reinterpret_cast<uint32_t *>(sm.sort.sorted);
        const int i = threadIdx.x, fours = (count + 3) / 4;
        uint32_t own = 0xffffffffu;
        if (i < count) own = (uint32_t)(sm.mine[i].x >> kBucketBits) << kComparedBits | (uint32_t)i;
        if (i < 4 * fours) all[i] = own;
        __syncthreads();
        if (i >= count) return;
        int rank = 0;
        for (int j = 0; j < fours; j++) {
            const uint4 o = reinterpret_cast<const uint4 *>(all)[j];
            rank += (o.x < own) + (o.y < own) + (o.z < own) + (o.w < own);
        }
        const_cast<int2 *>(l.sorted)[base + rank] = sm.mine[i];
        return;
    }
    static_assert(kBucketed <= kItems * kSortThreads, "a bucket is one round");
    Round r;
    r.items = min(kItems, (count + kSortThreads - 1) / kSortThreads), r.bits = l.bits;
    const int d = threadIdx.x;
    for (int pass = 0; pass < l.passes; pass++) {
        r.shift = kBucketBits + pass * l.bits;
        int2 *out = l.places[(l.passes - 1 - pass) & 1] + base;
        const int2 *in = l.places[(l.passes - pass) & 1] + base;
        if (pass > 0) {
            r.read(in, 0, count);
        } else {
            const int first = r.first(0);
#pragma unroll
            for (int i = 0; i < kItems; i++) {
                const int2 e = sm.mine[min(first + 32 * i, count - 1)];
                r.k[i] = i < r.items && first + 32 * i < count ? e.x : -1, r.place[i] = e.y;
            }
        }
        r.rank(sm.sort);
        const int front = in_front(d < 1 << r.bits ? sm.sort.count[d] : 0, sm.sort.scan);
        if (d < 1 << r.bits) sm.sort.base[d] = front;
        __syncthreads();
        r.scatter(sm.sort, out, count);
        __syncthreads();
    }
}

// What a gradient holds, to which a sum is added: fp32 values where they are, by L2, so that nobody waits for them (one thread of a call adds to a
// place, so the order is fixed); bf16 values are asked for ahead and rounded once.
template <class G, int kN>
struct Held {
    Raw<G, sizeof(G) == 2 ? kN : 1> old;
    __device__ __forceinline__ void ask(const G *p) {
        if constexpr (sizeof(G) == 2) old.load(p);
    }
    __device__ __forceinline__ void add(G *p, const float (&sum)[kN], float scale) {
        if constexpr (sizeof(G) == 2) {
            old.add(sum, scale);
            old.store(p);
        } else if constexpr (kN == 1) {
            asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(p), "f"(sum[0] * scale) : "memory");
        } else {
#pragma unroll
            for (int i = 0; i < kN; i += 4)
                asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(p + i), "f"(sum[i] * scale), "f"(sum[i + 1] * scale), "f"(sum[i + 2] * scale),
                             "f"(sum[i + 3] * scale)
                             : "memory");
        }
    }
};

template <int kN>
__device__ __forceinline__ void put(float *p, const float (&sum)[kN]) {
    Raw<float, kN> r;
#pragma unroll
    for (int e = 0; e < kN; e++) r.w[e] = __float_as_uint(sum[e]);
    r.store(p);
}
template <int kN>
__device__ __forceinline__ void clear(float (&v)[kN]) {
#pragma unroll
    for (int e = 0; e < kN; e++) v[e] = 0.f;
}

// Rows t, t + step, .. of dy, eight at a time.
template <class E, int kN>
__device__ __forceinline__ void add_rows(const Gradient &a, long long t, long long step, int col, float (&sum)[kN]) {
    for (; t < a.n; t += kAhead * step) {
        Raw<E, kN> v[kAhead];
#pragma unroll
        for (int u = 0; u < kAhead; u++) v[u].load(static_cast<const E *>(a.dy) + min(t + u * step, a.n - 1) * a.ld + col);
        float part[kN] = {};  // (a sum of every term behind the other loses bits where they are many)
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (t + u * step < a.n) v[u].add_to(part);
#pragma unroll
        for (int e = 0; e < kN; e++) sum[e] += part[e];
    }
}

// The positions that are a token's place: dpos[t] += dy[t] + dy[t + T] + .., by block `block` of `blocks`, of which all threads come here and `threads` work.
// a.place_width of them have a piece of a row of the table each (place_width() says how many); `threads` / place_width share its sequences, each taking every so many-th, and
// their sums are added up in pairs.  `shared`: threads / 2 * kN values, unless every thread has a piece of its own.
template <class E, class G, int kN>
__device__ __forceinline__ void add_places(const Gradient &a, int block, int blocks, int threads, float *shared) {
    const int words = a.C / kN, width = a.place_width;
    const long long total = min(min((long long)a.T, a.n), (long long)a.P) * words;
    Held<G, kN> old;
    if (width == threads) {  // (the loop below with one group: 4 % slower in the largest case)
        for (long long i = (long long)block * width + threadIdx.x; i < total && (int)threadIdx.x < threads; i += (long long)blocks * width) {
            const long long t = i / words;
            const int col = (int)(i - t * words) * kN;
            G *grad = static_cast<G *>(a.pos_grad) + t * a.pos_ld + col;
            float sum[kN] = {};
            old.ask(grad);
            add_rows<E, kN>(a, t, a.T, col, sum);
            old.add(grad, sum, 1.f);
        }
        return;
    }
    const int groups = threads / width, group = (int)threadIdx.x / width, own = (int)threadIdx.x & (width - 1);
    for (long long i0 = (long long)block * width; i0 < total; i0 += (long long)blocks * width) {
        const long long i = i0 + own, t = i / words;
        const int col = (int)(i - t * words) * kN;
        const bool inside = i < total && group < groups;
        G *grad = static_cast<G *>(a.pos_grad) + t * a.pos_ld + col;
        float sum[kN] = {};
        if (inside && group == 0) old.ask(grad);
        if (inside) add_rows<E, kN>(a, t + (long long)group * a.T, (long long)groups * a.T, col, sum);
        for (int half = groups / 2; half > 0; half /= 2) {
            if (inside && group >= half && group < 2 * half) {
#pragma unroll
                for (int e = 0; e < kN; e++) shared[e * (threads / 2) + (group - half) * width + own] = sum[e];
            }
            __syncthreads();
            if (inside && group < half) {
#pragma unroll
                for (int e = 0; e < kN; e++) sum[e] += shared[e * (threads / 2) + group * width + own];
            }
            __syncthreads();
        }
        if (inside && group == 0) old.add(grad, sum, 1.f);
    }
}

// Clusters 0 .. lists - 1 sort; the others add up the positions that are a token's place.  Bound by the passes, two of
// 8 bits for 50257 tokens, whose CTAs wait for each other; it hides the 157 MB of dy that the others read.  49152 places of 1600 bf16 columns, half of them one
// token: 99 us, of which sort, runs and joins have 31, 48 and 21 %.
template <class E, class G, int kN>
__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(const __grid_constant__ Gradient a) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    pdl_launch_dependents();
    pdl_wait();
    const int cluster = blockIdx.x / kSortCtas, others = a.lists * kSortCtas;
    if (cluster < a.lists) sort_list(a.list[cluster], *reinterpret_cast<SortSmem *>(smem_raw));
    else add_places<E, G, kN>(a, (int)blockIdx.x - others, (int)gridDim.x - others, kSortThreads, reinterpret_cast<float *>(smem_raw));
}

// A CTA for each bucket of each list.  Bound by latency: no more than 4 MB are moved, most of them from L2.  8192 places of 768 fp32
// columns: 18.5 us with positions, of which this, runs and joins have 27, 46 and 27 %.
__global__ void __launch_bounds__(kSortThreads, 1) bucket_kernel(const __grid_constant__ Gradient a) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    pdl_launch_dependents();
    pdl_wait();
    const int which = blockIdx.x >> kBucketBits;
    sort_bucket(a.list[which], blockIdx.x & ((1 << kBucketBits) - 1), *reinterpret_cast<BucketSmem *>(smem_raw));
}

// A warp takes a range of a sorted list, and 32 kN columns (blockIdx.y).  Blocks behind the ranges add up the positions that are a token's place
// where the sort was not a launch of few CTAs, which leaves room for that.
// Bound by what 16 warps an SM have on their way, since a thread takes 113 or 114 registers: sums and two batches of rows where the table is fp32 (which ranges of up to 8192
// places, one batch long, do not use), sums, one batch and what the table holds where it is bf16.  Half of the memory's rate for 49152 rows of 1600 bf16 columns.
template <class E, class G, int kN>
__global__ void __launch_bounds__(kThreads) runs_kernel(const __grid_constant__ Gradient a, int blocks) {
    pdl_launch_dependents();
    pdl_wait();
    if ((int)blockIdx.x >= blocks) {
        __shared__ float shared[kThreads / 2 * kN];
        add_places<E, G, kN>(a, (int)((blockIdx.x - blocks) * gridDim.y + blockIdx.y), (int)((gridDim.x - blocks) * gridDim.y), kThreads, shared);
        return;
    }
    const int lane = threadIdx.x & 31, unit = (int)blockIdx.x * (kThreads / 32) + (int)(threadIdx.x >> 5);
    const int which = unit < a.list[0].ranges ? 0 : 1;
    const List &l = a.list[which];
    const int range = unit - (which ? a.list[0].ranges : 0);
    if (range >= l.ranges || which >= a.lists) return;
    const int2 *places = l.sorted;
    const int col = ((int)blockIdx.y * 32 + lane) * kN;
    const bool inside = col < a.C;
    const int from = range * l.length, count = min(l.n - from, l.length);  // up to 32
    const int2 place = lane < count ? places[from + lane] : make_int2(-1, 0);
    const int mine = place.x, row = place.y;
    const int outer = lane == 0 ? (from > 0 ? places[from - 1].x : -1) : lane == 1 && from + count < l.n ? places[from + count].x : -1;
    const int in_front = __shfl_sync(0xffffffffu, outer, 0), behind = __shfl_sync(0xffffffffu, outer, 1);
    const int first = __shfl_sync(0xffffffffu, mine, 0), last = __shfl_sync(0xffffffffu, mine, count - 1);
    bool began = in_front != first;  // the run began in this range
    const bool goes_on = behind == last;
    float sum[kN] = {};
    const E *dy = static_cast<const E *>(a.dy) + (inside ? col : 0);
    G *grad = static_cast<G *>(l.grad) + (inside ? col : 0);
    struct Batch {
        Raw<E, kN> v[kAhead];
        Held<G, kN> old[kAhead];
        int k[kAhead + 1];
    };
    auto ask = [&](Batch &b, int i0) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) b.v[u].load(dy + __shfl_sync(0xffffffffu, row, (i0 + u) & 31) * a.ld);  // (behind the range: the row of place 0)
#pragma unroll
        for (int u = 0; u <= kAhead; u++) {
            const int next = __shfl_sync(0xffffffffu, mine, (i0 + u) & 31);
            b.k[u] = i0 + u < 32 ? next : -1;
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++)
            if (b.k[u + 1] != b.k[u] && b.k[u] < l.V && b.k[u] >= 0) b.old[u].ask(grad + b.k[u] * l.ld);
    };
    auto take = [&](Batch &b, int i0) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (b.k[u] < 0) break;
            if (b.k[u] >= l.V) {  // no token
                began = true;
                continue;
            }
            b.v[u].add_to(sum);
            if (b.k[u + 1] == b.k[u]) continue;
            if (inside) {
                if (!began) put<kN>(l.head + (long long)range * a.C + col, sum);
                else if (i0 + u == count - 1 && goes_on) put<kN>(l.tail + (long long)range * a.C + col, sum);
                else b.old[u].add(grad + b.k[u] * l.ld, sum, l.scale);
            }
            began = true;
            clear(sum);
        }
    };
    if constexpr (sizeof(G) == 2) {
        for (int i0 = 0; i0 < count; i0 += kAhead) {
            Batch b;
            ask(b, i0);
            take(b, i0);
        }
    } else {  // what fp32 gradients hold takes no registers: one batch is on its way while the other is added up
        Batch even, odd;
        ask(even, 0);
        for (int i0 = 0; i0 < count; i0 += 2 * kAhead) {
            if (i0 + kAhead < count) ask(odd, i0 + kAhead);
            take(even, i0);
            if (i0 + kAhead >= count) break;
            if (i0 + 2 * kAhead < count) ask(even, i0 + 2 * kAhead);
            take(odd, i0 + kAhead);
        }
    }
}

// Runs that leave the range in which they began: the sum of their parts, in the order of the list.  A warp looks at a range and takes runs of
// up to kFew parts itself; a block takes the longer ones of its 16 ranges one by one, its warps every 16th part.
// Bound by the longest run, whose parts are read by one block of each 128 columns (one token has half of the places in the case above).
constexpr int kFew = 8, kJoinWarps = 16;
template <class G, int kN>
__global__ void __launch_bounds__(32 * kJoinWarps) join_kernel(const __grid_constant__ Gradient a) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float part[kJoinWarps][32 * kN];
    __shared__ int last_of[kJoinWarps];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = ((int)blockIdx.y * 32 + lane) * kN;
    const bool inside = col < a.C;
    const int blocks0 = (a.list[0].ranges + kJoinWarps - 1) / kJoinWarps, which = blockIdx.x < (unsigned)blocks0 ? 0 : 1;
    const List &l = a.list[which];
    const int range0 = ((int)blockIdx.x - (which ? blocks0 : 0)) * kJoinWarps, range = range0 + warp;
    const int2 *places = l.sorted;
    int parts = 0, k = -1;  // of the run that begins in this range and goes on: behind this one
    if (range < l.ranges) {
        const int from = range * l.length, to = min(l.n, from + l.length);
        // lane 0: the last place, lanes 1 to 30: the first ones of the next ranges, lane 31: the place in front of this one
        const int at = lane == 0 ? to - 1 : lane < 31 ? to + (lane - 1) * l.length : from - 1;
        const int seen = at >= 0 && at < l.n ? places[at].x : -1;
        k = __shfl_sync(0xffffffffu, seen, 0);
        const unsigned same = __ballot_sync(0xffffffffu, seen == k);
        if (k < l.V && !(same >> 31)) parts = __ffs(~(same >> 1)) - 1;  // (a range's last place has its token: sorted)
        if (parts == 30) {  // more: where the run ends is sought 32 ranges at a time
            int lo = range + 30, hi = l.ranges;  // range lo begins with k
            while (hi - lo > 1) {
                const int step = (hi - lo + 31) / 32, probe = lo + (lane + 1) * step;
                const int more = __popc(__ballot_sync(0xffffffffu, probe < hi && places[(long long)min(probe, hi - 1) * l.length].x == k));
                lo += more * step;
                hi = min(hi, lo + step);
            }
            parts = lo - range;
        }
    }
    if (lane == 0) last_of[warp] = parts > kFew ? range + parts : -1;
    G *const grad = static_cast<G *>(l.grad) + col;
    auto sum_of = [&](int first, int end, int step, float(&sum)[kN]) {  // parts first, first + step, .. up to end
        for (int r0 = first; r0 <= end; r0 += step * kAhead) {
            Raw<float, kN> v[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++) v[u].load(l.head + (long long)min(r0 + step * u, end) * a.C + col);
#pragma unroll
            for (int u = 0; u < kAhead; u++)
                if (r0 + step * u <= end) v[u].add_to(sum);
        }
    };
    Raw<float, kN> tail;
    Held<G, kN> old;
    if (parts > 0 && inside) {
        old.ask(grad + k * l.ld);
        tail.load(l.tail + (long long)range * a.C + col);
        if (parts <= kFew) {
            float sum[kN] = {};
            tail.add_to(sum);
            sum_of(range + 1, range + parts, 1, sum);
            old.add(grad + k * l.ld, sum, l.scale);
        }
    }
    __syncthreads();
    for (int w = 0; w < kJoinWarps; w++) {
        const int end = last_of[w];
        if (end < 0) continue;
        float sum[kN] = {};
        if (inside) sum_of(range0 + w + 1 + warp, end, kJoinWarps, sum);
#pragma unroll
        for (int e = 0; e < kN; e++) part[warp][lane * kN + e] = sum[e];
        __syncthreads();
        if (warp == w && inside) {
            clear(sum);
            tail.add_to(sum);
            for (int i = 0; i < kJoinWarps; i++)
#pragma unroll
                for (int e = 0; e < kN; e++) sum[e] += part[i][lane * kN + e];
            old.add(grad + k * l.ld, sum, l.scale);
        }
        __syncthreads();
    }
}

// Few tokens: a block for each place t of each list.  The first place of a token adds up the rows of all; `groups` threads share a column's
// rows, each taking every groups-th.  The blocks behind them add up the positions that are a token's place.  Bound by the launch and two loads that wait for
// each other: 3.4 us from 1 to 128 places.
template <class E, class G, int kN>
__global__ void __launch_bounds__(kSortThreads) few_kernel(const __grid_constant__ Gradient a, int width, int groups) {
    pdl_launch_dependents();
    pdl_wait();
    extern __shared__ __align__(16) float shared[];
    __shared__ int list[kFewTokens], counts[kFewTokens / 32], of[1];
    const int n = (int)a.n, which = blockIdx.x / n;
    if (which >= a.lists) {
        add_places<E, G, kN>(a, (int)blockIdx.x - a.lists * n, (int)gridDim.x - a.lists * n, kFewTokens, shared);
        return;
    }
    const List &l = a.list[which];
    const int t = blockIdx.x - which * n, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    // every warp but the last ones looks at 32 places; places in front of t with its token: nothing to do here
    if (threadIdx.x == 0) of[0] = l.ids.at(t, l.V);
    const int mine = (int)threadIdx.x < n ? l.ids.at(threadIdx.x, l.V) : -1;
    __syncthreads();
    const int k = of[0];
    const unsigned same = __ballot_sync(0xffffffffu, mine == k && (int)threadIdx.x < n);
    if (lane == 0 && warp < kFewTokens / 32) counts[warp] = __popc(same);
    const bool before = mine == k && (int)threadIdx.x < t;
    if (__syncthreads_or(before) || k < 0) return;
    int front = 0, all = 0;
    for (int w = 0; w < (n + 31) / 32; w++) {
        if (w < warp) front += counts[w];
        all += counts[w];
    }
    if (same >> lane & 1) list[front + __popc(same & ((1u << lane) - 1))] = threadIdx.x;
    __syncthreads();
    const int group = threadIdx.x / width, column = threadIdx.x - group * width;
    for (int c0 = 0; c0 < a.C; c0 += width * kN) {
        const int col = c0 + column * kN;
        const bool inside = col < a.C && group < groups;
        float sum[kN] = {};
        Raw<G, kN> old;
        G *grad = static_cast<G *>(l.grad) + k * l.ld + col;
        if (inside && group == 0) old.load(grad);
        if (inside) {
            for (int i = group; i < all; i += groups * kAhead) {
                Raw<E, kN> v[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; u++) v[u].load(static_cast<const E *>(a.dy) + list[min(i + u * groups, all - 1)] * a.ld + col);
#pragma unroll
                for (int u = 0; u < kAhead; u++)
                    if (i + u * groups < all) v[u].add_to(sum);
            }
        }
        if (all > 1 && groups > 1) {
            if (group > 0 && group < groups) {
#pragma unroll
                for (int e = 0; e < kN; e++) shared[((group - 1) * width + column) * kN + e] = sum[e];
            }
            __syncthreads();
            if (group == 0) {
                for (int g = 1; g < groups; g++)
#pragma unroll
                    for (int e = 0; e < kN; e++) sum[e] += shared[((g - 1) * width + column) * kN + e];
            }
            __syncthreads();
        }
        if (inside && group == 0) {
            old.add(sum, l.scale);
            old.store(grad);
        }
    }
}

// ---- host side ----

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

bool float_type(int t) { return t == TENSOR_F32 || t == TENSOR_BF16; }
bool id_type(int t) { return t >= TENSOR_INT32 && t <= TENSOR_IDS_F32; }
uintptr_t id_mask(int t) { return t == TENSOR_INT64 ? 7 : 3; }
uintptr_t each_of(int t) { return t == TENSOR_F32 ? 4 : 2; }
uintptr_t bits(const void *p) { return reinterpret_cast<uintptr_t>(p); }

// The memory from a matrix's first row to its last; NULL: none.
struct Span {
    uintptr_t from, to;
    Span(const void *p, long long rows, long long ld, long long columns, uintptr_t each) : from(bits(p)), to(p ? bits(p) + ((rows - 1) * ld + columns) * each : 0) {}
    bool meets(const Span &o) const { return from && o.from && from < o.to && o.from < to; }
};

// Places of a range, which a warp takes: 32 at most.  Short ranges make more warps, long ones fewer parts of runs.  (768 fp32 columns: 8192 places
// 16.5 us by 8, 17.8 by 16; 16384 places 40 by 8, 36.6 by 16; 32768 places 72 by 16, 69 by 32; 49152 places 93.6 by 16, 90 by 32.)
int range_length(long long n) { return n <= 8192 ? 8 : n <= 16384 ? 16 : 32; }

template <class E>
cudaError_t launch_lookup(const Lookup &a, int bytes, int rows, int words, cudaStream_t s) {
    const unsigned magic = words > 1 ? (unsigned)(((1ull << 32) + words - 1) / words) : 0;
    const dim3 grid((unsigned)((a.n + rows - 1) / rows)), block(kThreads);
    auto kernel = a.pos_table ? (bytes == 32 ? lookup_kernel<E, 32 / sizeof(E), true> : bytes == 16 ? lookup_kernel<E, 16 / sizeof(E), true> : lookup_kernel<E, 1, true>)
                              : (bytes == 32 ? lookup_kernel<E, 32 / sizeof(E), false> : bytes == 16 ? lookup_kernel<E, 16 / sizeof(E), false> : lookup_kernel<E, 1, false>);
    return attn::launch_after_previous(kernel, grid, block, 0, s, a, rows, words, magic);
}

// Scratch of one list; where it is set up if `base` is given.
size_t list_bytes(long long n, int C, int V, List *l, char *base) {
    size_t at = 0;
    auto take = [&](size_t bytes) {
        char *here = base + at;
        at += up256(bytes);
        return here;
    };
    const int length = range_length(n);
    const long long ranges = (n + length - 1) / length;
    int need = 1;
    while (need < 31 && (1ll << need) <= V) need++;  // V itself stands for no token
    if (n <= kBucketed) need = std::max(1, need - kBucketBits);
    const int passes = (need + kBits - 1) / kBits;
    if (l) {
        l->length = length, l->ranges = (int)ranges;
        l->passes = passes, l->bits = (need + passes - 1) / passes;
    }
    for (int i = 0; i < 2; i++) {
        int2 *places = reinterpret_cast<int2 *>(take((size_t)n * sizeof(int2)));
        if (l) l->places[i] = places;
    }
    if (l) l->sorted = l->places[n <= kBucketed ? 0 : passes & 1];
    float *head = reinterpret_cast<float *>(take((size_t)ranges * C * 4)), *tail = reinterpret_cast<float *>(take((size_t)ranges * C * 4));
    if (l) l->head = head, l->tail = tail;
    return at;
}

// How many pieces of rows of the position table a block of `threads` takes at a time: one a thread, but fewer, whose sequences threads share, where that makes fewer than `blocks`
// blocks, there are eight sequences for each thread, and a row is still read 32 bytes at a time.  us of the whole gradient of 768 fp32 columns with one a thread, in brackets by
// this rule: 8192 places in sequences of 1 518 (46), of 8 88 (34), of 64 35 (29); 65536 in sequences of 1 5983 (148), of 16 584 (123).  Halved once more where blocks are
// enough, 48 sequences of 1024 x 1600 bf16 columns took 119 instead of 100.
int place_width(long long places, const Gradient &a, int threads, int blocks) {
    const long long sequences = a.T > 0 ? (a.n + a.T - 1) / a.T : 0;
    int width = threads;
    while (width > 2 && sequences * width > 8ll * threads && (places + width - 1) / width < blocks) width /= 2;
    return width;
}

template <class E, class G, int kN>
cudaError_t launch_gradient(Gradient a, cudaStream_t s) {
    const int words = a.C / kN;
    const long long places = a.T > 0 ? std::min(std::min((long long)a.T, a.n), (long long)a.P) * words : 0;
    if (a.n <= kFewTokens) {
        const int width = std::min(256, (words + 31) / 32 * 32), groups = std::max(1, std::min(4, kSortThreads / width));
        const int threads = std::max(width * groups, kFewTokens);
        a.place_width = place_width(places, a, kFewTokens, 148);
        const long long blocks = a.lists * a.n + std::min(600ll, (places + a.place_width - 1) / a.place_width);
        const int shared = std::max(width * (groups - 1), a.place_width < kFewTokens ? kFewTokens / 2 : 0);
        return attn::launch_after_previous(few_kernel<E, G, kN>, dim3((unsigned)blocks), dim3((unsigned)threads), sizeof(float) * kN * shared, s, a, width, groups);
    }
    cudaError_t e;
    a.place_width = a.n <= kBucketed ? place_width(places, a, kThreads, 296) : place_width(places, a, kSortThreads, 136);
    const long long all = (places + a.place_width - 1) / a.place_width;  // blocks for the positions that are a token's place
    if (a.n <= kBucketed) {
        e = a.lists == 0 ? cudaSuccess : attn::launch_after_previous(bucket_kernel, dim3((unsigned)(a.lists << kBucketBits)), dim3(kSortThreads), sizeof(BucketSmem), s, a);
    } else {
        const long long clusters = a.lists + std::min((all + kSortCtas - 1) / kSortCtas, 17ll);
        e = attn::launch_clusters_after_previous(sort_kernel<E, G, kN>, dim3((unsigned)(clusters * kSortCtas)), dim3(kSortThreads), sizeof(SortSmem), kSortCtas, s, a);
    }
    if (e != cudaSuccess || (a.lists == 0 && a.n > kBucketed)) return e;
    const unsigned slices = (unsigned)((words + 31) / 32);
    const int ranges = a.list[0].ranges + (a.lists > 1 ? a.list[1].ranges : 0);
    const int groups = (ranges + kThreads / 32 - 1) / (kThreads / 32);
    const long long others = a.n <= kBucketed ? (std::min(all, 1184ll) + slices - 1) / slices : 0;
    e = attn::launch_after_previous(runs_kernel<E, G, kN>, dim3((unsigned)(groups + others), slices), dim3(kThreads), 0, s, a, groups);
    if (e != cudaSuccess || a.lists == 0) return e;
    const int joins = (a.list[0].ranges + kJoinWarps - 1) / kJoinWarps + (a.lists > 1 ? (a.list[1].ranges + kJoinWarps - 1) / kJoinWarps : 0);
    constexpr int kJoined = kN > 4 ? 4 : kN;  // narrower, since one run may be all that there is to do
    return attn::launch_after_previous(join_kernel<G, kJoined>, dim3((unsigned)joins, (unsigned)((a.C / kJoined + 31) / 32)), dim3(32 * kJoinWarps), 0, s, a);
}

template <class E, class G>
cudaError_t launch_gradient(const Gradient &a, bool wide, cudaStream_t s) {
    return wide ? launch_gradient<E, G, 16 / sizeof(E)>(a, s) : launch_gradient<E, G, 1>(a, s);
}

template <class E>
cudaError_t set(cudaError_t e) {
    auto one = [&](auto *kernel, size_t bytes) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    };
    constexpr int kN = 16 / sizeof(E);
    one(sort_kernel<E, float, kN>, sizeof(SortSmem)), one(sort_kernel<E, float, 1>, sizeof(SortSmem));
    one(sort_kernel<E, __nv_bfloat16, kN>, sizeof(SortSmem)), one(sort_kernel<E, __nv_bfloat16, 1>, sizeof(SortSmem));
    one(bucket_kernel, sizeof(BucketSmem));
    return e;
}

}  // namespace

cudaError_t set_attributes() { return set<__nv_bfloat16>(set<float>(cudaSuccess)); }

}  // namespace embed

extern "C" {

int tensor_sm100_embedding_forward(const void *tokens, const void *table, const void *positions, const void *pos_table, void *y, long long n,
                                   long long ld, long long pos_ld, float scale, int type, int id_type, int T, int C, int V, int P, void *stream) {
    if (!tokens || !table || !y) return ATTN_ERR_NULL;
    if (n < 0 || C <= 0 || V <= 0 || ld < C || !embed::float_type(type) || !embed::id_type(id_type)) return ATTN_ERR_ARGUMENT;
    if (pos_table && (P <= 0 || pos_ld < C || (!positions && T <= 0))) return ATTN_ERR_ARGUMENT;
    const uintptr_t each = embed::each_of(type);
    if ((embed::bits(table) | embed::bits(pos_table) | embed::bits(y)) % each || ((embed::bits(tokens) | embed::bits(positions)) & embed::id_mask(id_type))) return ATTN_ERR_ALIGN;
    if (n > 0) {
        if (n > (1ll << 40) / C || C > (1 << 20)) return ATTN_ERR_UNSUPPORTED;
        const uintptr_t id_bytes = embed::id_mask(id_type) + 1;
        const embed::Span out(y, n, C, C, each);
        for (const embed::Span &in : {embed::Span(table, V, ld, C, each), embed::Span(pos_table, P, pos_ld, C, each), embed::Span(tokens, 1, n, n, id_bytes), embed::Span(positions, 1, n, n, id_bytes)})
            if (out.meets(in)) return ATTN_ERR_ARGUMENT;
    }
    int *status = nullptr;
    const int rc = attn::device_status_word(&status);
    if (rc != ATTN_OK) return rc;
    if (n == 0) return ATTN_OK;
    // 32 bytes at a time where every row allows it, else 16, else a value
    const uintptr_t all = embed::bits(table) | embed::bits(pos_table) | embed::bits(y) | C * each | (uintptr_t)ld * each | (pos_table ? (uintptr_t)pos_ld * each : 0);
    const int bytes = all % 32 == 0 ? 32 : all % 16 == 0 ? 16 : (int)each, words = (int)(C * each / bytes);
    // a block has a piece for each thread, or all that one takes where that leaves blocks enough
    const int units = embed::units_of(bytes, pos_table != nullptr);
    const long long pieces = n * words, per = pieces >= embed::kThreads * units * 600ll ? embed::kThreads * units : embed::kThreads;
    const int rows = (int)std::max(1ll, per / words);
    if ((n + rows - 1) / rows > 0x7fffffffll) return ATTN_ERR_UNSUPPORTED;
    const embed::Lookup a{table, pos_table, y, ld, pos_ld, n, Ids{tokens, id_type}, Ids{positions, id_type}, T, C, V, P, scale};
    return (int)(type == TENSOR_F32 ? embed::launch_lookup<float>(a, bytes, rows, words, static_cast<cudaStream_t>(stream))
                                    : embed::launch_lookup<__nv_bfloat16>(a, bytes, rows, words, static_cast<cudaStream_t>(stream)));
}

size_t tensor_sm100_embedding_backward_scratch_bytes(long long n, int C, int V, int P) {
    if (n <= 0 || n > (1 << 30) || C <= 0 || C > (1 << 20) || V < 0 || V > (1 << 30) || P < 0 || P > (1 << 30)) return 0;
    return (V ? embed::list_bytes(n, C, V, nullptr, nullptr) : 0) + (P ? embed::list_bytes(n, C, P, nullptr, nullptr) : 0);
}

int tensor_sm100_embedding_backward(const void *dy, const void *tokens, void *dtable, const void *positions, void *dpos_table, void *scratch, long long n,
                                    long long ld_dy, long long ld, long long pos_ld, float scale, int type, int grad_type, int id_type, int T, int C, int V, int P,
                                    void *stream) {
    if (!dy || (!dtable && !dpos_table) || (dtable && !tokens)) return ATTN_ERR_NULL;
    if (n < 0 || C <= 0 || ld_dy < C || !embed::float_type(type) || !embed::float_type(grad_type) || !embed::id_type(id_type)) return ATTN_ERR_ARGUMENT;
    if ((dtable && (V <= 0 || ld < C)) || (dpos_table && (P <= 0 || pos_ld < C || (!positions && T <= 0)))) return ATTN_ERR_ARGUMENT;
    const uintptr_t each = embed::each_of(type), grad_each = embed::each_of(grad_type);
    if (embed::bits(dy) % each || (embed::bits(dtable) | embed::bits(dpos_table)) % grad_each || (embed::bits(scratch) & 255) ||
        ((embed::bits(tokens) | embed::bits(positions)) & embed::id_mask(id_type)))
        return ATTN_ERR_ALIGN;
    if (n > (1 << 30) || C > (1 << 20) || V > (1 << 30) || P > (1 << 30)) return ATTN_ERR_UNSUPPORTED;
    if (n > 0 && (dtable || positions) && !scratch) return ATTN_ERR_NULL;  // (behind the sizes that have none)
    const embed::Span table_at(dtable, V, ld, C, grad_each), pos_at(dpos_table, P, pos_ld, C, grad_each);
    if (n > 0) {
        const uintptr_t id_bytes = embed::id_mask(id_type) + 1;
        for (const embed::Span &in : {embed::Span(dy, n, ld_dy, C, each), embed::Span(tokens, 1, n, n, id_bytes), embed::Span(positions, 1, n, n, id_bytes)})
            if (table_at.meets(in) || pos_at.meets(in)) return ATTN_ERR_ARGUMENT;
    }
    if (table_at.meets(pos_at)) return ATTN_ERR_ARGUMENT;
    int *status = nullptr;
    const int rc = attn::device_status_word(&status);
    if (rc != ATTN_OK) return rc;
    if (n == 0) return ATTN_OK;
    embed::Gradient a = {};
    a.dy = dy, a.ld = ld_dy, a.C = C, a.n = n;
    char *base = static_cast<char *>(scratch);
    auto add = [&](const void *ids, void *grad, long long ld_grad, int rows, float by) {
        embed::List &l = a.list[a.lists++];
        l.ids = Ids{ids, id_type};
        l.grad = grad, l.ld = ld_grad, l.V = rows, l.n = (int)n, l.scale = by;
        base += embed::list_bytes(n, C, rows, &l, base);
    };
    if (dtable) add(tokens, dtable, ld, V, scale);
    if (dpos_table && positions) add(positions, dpos_table, pos_ld, P, 1.f);
    if (dpos_table && !positions) a.T = T, a.P = P, a.pos_grad = dpos_table, a.pos_ld = pos_ld;
    // 16 bytes of dy at a time, and as many columns of the gradients
    const uintptr_t columns = 16 / each;
    const bool wide = C % columns == 0 && (embed::bits(dy) | (uintptr_t)ld_dy * each) % 16 == 0 &&
                      (embed::bits(dtable) | embed::bits(dpos_table) | (dtable ? (uintptr_t)ld * grad_each : 0) | (dpos_table ? (uintptr_t)pos_ld * grad_each : 0)) %
                              (columns * grad_each) == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == TENSOR_F32)
        return (int)(grad_type == TENSOR_F32 ? embed::launch_gradient<float, float>(a, wide, s) : embed::launch_gradient<float, __nv_bfloat16>(a, wide, s));
    return (int)(grad_type == TENSOR_F32 ? embed::launch_gradient<__nv_bfloat16, float>(a, wide, s) : embed::launch_gradient<__nv_bfloat16, __nv_bfloat16>(a, wide, s));
}

}  // extern "C"
