// Rows of the token table, scaled, with rows of the position table added; and the gradients of both tables, for sm_100a.
//
//     y[t] = scale table[tokens[t]] + pos_table[positions[t]]
//     dtable[v] += scale sum over tokens[t] = v of dy[t]          dpos_table[p] += sum over positions[t] = p of dy[t]
//
// Lookup: bound by HBM, a thread takes four words of 16 bytes, whose rows it asks for together.
//
// Gradient: the places t are put in the order of their tokens (equal tokens by t), and the sorted list is cut into ranges of the same
// number of places, whatever the tokens are.  A thread keeps the sum of a few columns over a run of equal tokens and adds it to the table
// where the run ends; the parts of runs that cross a border of a range are kept, and a last kernel adds them up in the order of the
// list.  So every sum has a fixed order, and a token that takes half of the batch is spread over the GPU.  The list is sorted by one
// cluster, while the other CTAs of that launch make the gradient of positions that are a token's place in its sequence, where no list is
// needed.
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
constexpr int kAhead = 4;                     // places whose rows a thread asks for together

// kN columns of a row, as fp32.
template <class T, int kN>
__device__ __forceinline__ void load(float (&v)[kN], const T *p) {
    if constexpr (kN == 1) {
        v[0] = (float)*p;
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < kN; i += 4) {
            const float4 f = *reinterpret_cast<const float4 *>(p + i);
            v[i] = f.x, v[i + 1] = f.y, v[i + 2] = f.z, v[i + 3] = f.w;
        }
    } else {
        uint32_t w[kN / 2];
        if constexpr (kN == 8) *reinterpret_cast<uint4 *>(w) = *reinterpret_cast<const uint4 *>(p);
        else *reinterpret_cast<uint2 *>(w) = *reinterpret_cast<const uint2 *>(p);
#pragma unroll
        for (int i = 0; i < kN / 2; i++) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
}
template <class T, int kN>
__device__ __forceinline__ void store(T *p, const float (&v)[kN]) {
    if constexpr (kN == 1) {
        *p = (T)v[0];
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < kN; i += 4) *reinterpret_cast<float4 *>(p + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
        uint32_t w[kN / 2];
#pragma unroll
        for (int i = 0; i < kN / 2; i++) w[i] = pack_bf16x2(v[2 * i], v[2 * i + 1]);
        if constexpr (kN == 8) *reinterpret_cast<uint4 *>(p) = *reinterpret_cast<uint4 *>(w);
        else *reinterpret_cast<uint2 *>(p) = *reinterpret_cast<uint2 *>(w);
    }
}

struct Lookup {
    const void *table, *pos_table;  // pos_table NULL: none
    void *y;
    long long ld, pos_ld, n;
    Ids tokens, positions;          // positions NULL: a token's place in its sequence of T
    int T, C, V, P;
    float scale;
};

// kN columns at a time.
template <class E, int kN>
__global__ void __launch_bounds__(kThreads) lookup_kernel(Lookup a, int words) {
    pdl_launch_dependents();
    pdl_wait();
    const long long total = a.n * words;
    const long long first = (long long)blockIdx.x * (kThreads * kUnits) + threadIdx.x;
    long long row[kUnits];
    int col[kUnits], token[kUnits], place[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
        const long long i = first + u * kThreads;
        row[u] = i / words;
        col[u] = (int)(i - row[u] * words) * kN;
        token[u] = place[u] = -1;
        if (i >= total) {
            row[u] = -1;
            continue;
        }
        token[u] = a.tokens.at(row[u], a.V);
        if (a.pos_table) {
            const long long p = a.positions.p ? a.positions.at(row[u], a.P) : row[u] % a.T;
            place[u] = p < a.P ? (int)p : -1;
        }
    }
    float x[kUnits][kN], y[kUnits][kN];
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
#pragma unroll
        for (int e = 0; e < kN; e++) x[u][e] = y[u][e] = 0.f;
        if (token[u] >= 0) load<E, kN>(x[u], static_cast<const E *>(a.table) + token[u] * a.ld + col[u]);
        if (place[u] >= 0) load<E, kN>(y[u], static_cast<const E *>(a.pos_table) + place[u] * a.pos_ld + col[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnits; u++) {
        if (row[u] < 0) continue;
#pragma unroll
        for (int e = 0; e < kN; e++) x[u][e] = fmaf(x[u][e], a.scale, y[u][e]);
        store<E, kN>(static_cast<E *>(a.y) + row[u] * a.C + col[u], x[u]);
    }
}

// One table's gradient.
struct List {
    Ids ids;
    void *grad;
    long long ld;
    int V, n;
    float scale;
    int *key[2], *at[2];  // tokens and their places, as the passes of the sort take turns
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
    long long n;
    void *pos_grad;
    long long pos_ld;
};

struct SortSmem {
    int warp[kSortWarps][kBins];
    int count[kBins], base[kBins], scan[kBins / 32];
};

// The places of a list in the order of their tokens, 2^bits tokens a pass, from the lowest digit on.  A cluster; each CTA has a piece.
__device__ void sort_list(const List &l, SortSmem &sm) {
    cg::cluster_group cluster = cg::this_cluster();
    const int rank = (int)cluster.block_rank(), warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int bins = 1 << l.bits;
    const int piece = ((l.n + kSortCtas - 1) / kSortCtas + 31) / 32 * 32;
    const int from = min((long long)l.n, (long long)rank * piece), to = min((long long)l.n, (long long)from + piece);
    for (int pass = 0; pass < l.passes; pass++) {
        const int shift = pass * l.bits;
        const volatile int *key = l.key[pass & 1], *at = l.at[pass & 1];
        int *key_out = l.key[(pass & 1) ^ 1], *at_out = l.at[(pass & 1) ^ 1];
        auto key_of = [&](int i) {
            if (pass > 0) return (int)key[i];
            const int k = l.ids.at(i, l.V);
            return k < 0 ? l.V : k;
        };
        for (int d = threadIdx.x; d < bins; d += kSortThreads) sm.count[d] = 0;
        __syncthreads();
        for (int i = from + threadIdx.x; i < to; i += kSortThreads) atomicAdd(&sm.count[key_of(i) >> shift & (bins - 1)], 1);
        cluster.sync();
        // where this CTA's places of each digit go
        int all = 0, before = 0;
        const int d = threadIdx.x;
        if (d < bins) {
            for (int c = 0; c < kSortCtas; c++) {
                const int v = cluster.map_shared_rank(sm.count, c)[d];
                if (c < rank) before += v;
                all += v;
            }
        }
        int sum = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += left;
        }
        if (d < kBins && lane == 31) sm.scan[warp] = sum;
        __syncthreads();
        if (d < bins) {
            int front = 0;
            for (int k = 0; k < warp; k++) front += sm.scan[k];
            sm.base[d] = front + sum - all + before;
        }
        for (int begin = from; begin < to; begin += kSortThreads * kItems) {
            for (int i = lane; i < bins; i += 32) sm.warp[warp][i] = 0;
            __syncwarp();
            int k[kItems], place[kItems], in_warp[kItems];
#pragma unroll
            for (int r = 0; r < kItems; r++) {
                const int i = begin + (warp * kItems + r) * 32 + lane;
                k[r] = i < to ? key_of(i) : -1;
                place[r] = i < to ? (pass > 0 ? at[i] : i) : 0;
            }
#pragma unroll
            for (int r = 0; r < kItems; r++) {
                const int digit = k[r] < 0 ? -1 : k[r] >> shift & (bins - 1);
                const unsigned same = __match_any_sync(0xffffffffu, digit);
                const int seen = digit < 0 ? 0 : sm.warp[warp][digit];
                __syncwarp();
                if (digit >= 0 && lane == __ffs(same) - 1) sm.warp[warp][digit] = seen + __popc(same);
                __syncwarp();
                in_warp[r] = seen + __popc(same & ((1u << lane) - 1));
            }
            __syncthreads();
            if (d < bins) {
                int running = sm.base[d];
                for (int w = 0; w < kSortWarps; w++) {
                    const int c = sm.warp[w][d];
                    sm.warp[w][d] = running;
                    running += c;
                }
                sm.base[d] = running;
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < kItems; r++) {
                if (k[r] < 0) continue;
                const int dst = sm.warp[warp][k[r] >> shift & (bins - 1)] + in_warp[r];
                key_out[dst] = k[r];
                at_out[dst] = place[r];
            }
            __syncthreads();
        }
        cluster.sync();  // what the others have written is there for the next pass, and nobody reads the counts any more
    }
}

// kN columns of grad += scale * sum.
template <class G, int kN>
__device__ __forceinline__ void add_to(G *p, const float (&old)[kN], const float (&sum)[kN], float scale) {
    float v[kN];
#pragma unroll
    for (int e = 0; e < kN; e++) v[e] = fmaf(sum[e], scale, old[e]);
    store<G, kN>(p, v);
}

// Clusters 0 .. lists - 1 sort; the others add up the positions that are a token's place.
template <class E, class G, int kN>
__global__ void __launch_bounds__(kSortThreads, 1) sort_kernel(const __grid_constant__ Gradient a) {
    extern __shared__ __align__(16) uint8_t smem_raw[];
    pdl_launch_dependents();
    pdl_wait();
    const int cluster = blockIdx.x / kSortCtas;
    if (cluster < a.lists) {
        sort_list(a.list[cluster], *reinterpret_cast<SortSmem *>(smem_raw));
        return;
    }
    const int words = a.C / kN;
    const long long T = min((long long)a.T, a.n), total = min(T, (long long)a.P) * words;
    const long long step = (long long)(gridDim.x - a.lists * kSortCtas) * kSortThreads;
    for (long long i = (long long)(blockIdx.x - a.lists * kSortCtas) * kSortThreads + threadIdx.x; i < total; i += step) {
        const long long t = i / words;
        const int col = (int)(i - t * words) * kN;
        float sum[kN] = {}, old[kN];
        G *grad = static_cast<G *>(a.pos_grad) + t * a.pos_ld + col;
        load<G, kN>(old, grad);
        for (long long r = t; r < a.n; r += (long long)kAhead * a.T) {
            float v[kAhead][kN];
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
#pragma unroll
                for (int e = 0; e < kN; e++) v[u][e] = 0.f;
                if (r + (long long)u * a.T < a.n) load<E, kN>(v[u], static_cast<const E *>(a.dy) + (r + (long long)u * a.T) * a.ld + col);
            }
#pragma unroll
            for (int u = 0; u < kAhead; u++)
#pragma unroll
                for (int e = 0; e < kN; e++) sum[e] += v[u][e];
        }
        add_to<G, kN>(grad, old, sum, 1.f);
    }
}

// A range of a sorted list: blockIdx.x; columns: threads of blockIdx.y.
template <class E, class G, int kN>
__global__ void __launch_bounds__(kThreads) runs_kernel(const __grid_constant__ Gradient a) {
    pdl_launch_dependents();
    pdl_wait();
    const int which = blockIdx.x < (unsigned)a.list[0].ranges ? 0 : 1;
    const List &l = a.list[which];
    const int range = blockIdx.x - (which ? a.list[0].ranges : 0);
    const int *key = l.key[l.passes & 1], *at = l.at[l.passes & 1];
    const int col = (blockIdx.y * blockDim.x + threadIdx.x) * kN;
    if (col >= a.C) return;
    const int from = range * l.length, to = min(l.n, from + l.length);
    const bool from_before = from > 0 && key[from - 1] == key[from], goes_on = to < l.n && key[to] == key[to - 1];
    float sum[kN] = {};
    bool began = !from_before;  // the run began in this range
    for (int i0 = from; i0 < to; i0 += kAhead) {
        int k[kAhead + 1];
        float v[kAhead][kN], old[kAhead][kN];
#pragma unroll
        for (int u = 0; u <= kAhead; u++) k[u] = i0 + u < to ? key[i0 + u] : -1;
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (k[u] < 0 || k[u] >= l.V) continue;
            load<E, kN>(v[u], static_cast<const E *>(a.dy) + at[i0 + u] * a.ld + col);
            if (k[u + 1] != k[u]) load<G, kN>(old[u], static_cast<G *>(l.grad) + k[u] * l.ld + col);
        }
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (k[u] < 0 || k[u] >= l.V) continue;
#pragma unroll
            for (int e = 0; e < kN; e++) sum[e] += v[u][e];
            if (k[u + 1] == k[u]) continue;
            if (!began) store<float, kN>(l.head + (long long)range * a.C + col, sum);
            else if (i0 + u == to - 1 && goes_on) store<float, kN>(l.tail + (long long)range * a.C + col, sum);
            else add_to<G, kN>(static_cast<G *>(l.grad) + k[u] * l.ld + col, old[u], sum, l.scale);
            began = true;
#pragma unroll
            for (int e = 0; e < kN; e++) sum[e] = 0.f;
        }
    }
}

// Runs that leave the range blockIdx.x in which they began: their parts, warps taking every eighth.
template <class G, int kN>
__global__ void __launch_bounds__(256) join_kernel(const __grid_constant__ Gradient a) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ float part[8][32 * kN];
    const int which = blockIdx.x < (unsigned)a.list[0].ranges ? 0 : 1;
    const List &l = a.list[which];
    const int range = blockIdx.x - (which ? a.list[0].ranges : 0);
    const int *key = l.key[l.passes & 1];
    const int from = range * l.length, to = min(l.n, from + l.length);
    const int k = key[to - 1];
    if (to >= l.n || k >= l.V || key[to] != k || (from > 0 && key[from - 1] == k)) return;
    int lo = to, hi = l.n;  // the run ends in front of the first place behind `to` with another token
    while (lo < hi) {
        const int mid = lo + (hi - lo) / 2;
        if (key[mid] == k) lo = mid + 1;
        else hi = mid;
    }
    const int last = (lo - 1) / l.length;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, col = (blockIdx.y * 32 + lane) * kN;
    float sum[kN] = {};
    if (col < a.C) {
        for (int r0 = range + 1 + warp; r0 <= last; r0 += 8 * kAhead) {
            float v[kAhead][kN];
#pragma unroll
            for (int u = 0; u < kAhead; u++) {
#pragma unroll
                for (int e = 0; e < kN; e++) v[u][e] = 0.f;
                if (r0 + 8 * u <= last) load<float, kN>(v[u], l.head + (long long)(r0 + 8 * u) * a.C + col);
            }
#pragma unroll
            for (int u = 0; u < kAhead; u++)
#pragma unroll
                for (int e = 0; e < kN; e++) sum[e] += v[u][e];
        }
    }
#pragma unroll
    for (int e = 0; e < kN; e++) part[warp][lane * kN + e] = sum[e];
    __syncthreads();
    if (warp != 0 || col >= a.C) return;
    float old[kN], first[kN];
    G *grad = static_cast<G *>(l.grad) + k * l.ld + col;
    load<G, kN>(old, grad);
    load<float, kN>(first, l.tail + (long long)range * a.C + col);
#pragma unroll
    for (int e = 0; e < kN; e++) {
        sum[e] = first[e];
#pragma unroll
        for (int w = 0; w < 8; w++) sum[e] += part[w][lane * kN + e];
    }
    add_to<G, kN>(grad, old, sum, l.scale);
}

// ---- host side ----

size_t up256(size_t v) { return (v + 255) / 256 * 256; }

bool float_type(int t) { return t == TENSOR_F32 || t == TENSOR_BF16; }
bool id_type(int t) { return t >= TENSOR_INT32 && t <= TENSOR_IDS_F32; }
uintptr_t id_mask(int t) { return t == TENSOR_INT64 ? 7 : 3; }
uintptr_t each_of(int t) { return t == TENSOR_F32 ? 4 : 2; }
uintptr_t bits(const void *p) { return reinterpret_cast<uintptr_t>(p); }

bool overlap(const void *a, long long rows_a, long long ld_a, uintptr_t each_a, const void *b, long long rows_b, long long ld_b, uintptr_t each_b, int C) {
    const uintptr_t end_a = bits(a) + ((rows_a - 1) * ld_a + C) * each_a, end_b = bits(b) + ((rows_b - 1) * ld_b + C) * each_b;
    return bits(a) < end_b && bits(b) < end_a;
}

// Places of a range: short ones where there are few, so that every SM has some.
int range_length(long long n) { return n <= 2048 ? 4 : n <= 16384 ? 8 : n <= 32768 ? 16 : n <= 65536 ? 32 : 64; }

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
    const int passes = (need + kBits - 1) / kBits;
    if (l) {
        l->length = length, l->ranges = (int)ranges;
        l->passes = passes, l->bits = (need + passes - 1) / passes;
    }
    for (int i = 0; i < 2; i++) {
        int *k = reinterpret_cast<int *>(take((size_t)n * 4)), *p = reinterpret_cast<int *>(take((size_t)n * 4));
        if (l) l->key[i] = k, l->at[i] = p;
    }
    float *head = reinterpret_cast<float *>(take((size_t)ranges * C * 4)), *tail = reinterpret_cast<float *>(take((size_t)ranges * C * 4));
    if (l) l->head = head, l->tail = tail;
    return at;
}

template <class E, class G, int kN>
cudaError_t launch_gradient(const Gradient &a, cudaStream_t s) {
    const int words = a.C / kN;
    long long clusters = a.lists;
    if (a.T > 0) {
        const long long work = std::min(std::min((long long)a.T, a.n), (long long)a.P) * words;
        clusters += std::max(1ll, std::min((work + kSortThreads * kSortCtas - 1) / (kSortThreads * kSortCtas), 17ll));
    }
    if (a.lists == 0 && a.T == 0) return cudaSuccess;
    cudaError_t e = attn::launch_clusters_after_previous(sort_kernel<E, G, kN>, dim3((unsigned)(clusters * kSortCtas)), dim3(kSortThreads), sizeof(SortSmem), kSortCtas, s, a);
    if (e != cudaSuccess || a.lists == 0) return e;
    const int ranges = a.list[0].ranges + (a.lists > 1 ? a.list[1].ranges : 0);
    const int threads = std::min(kThreads, (words + 31) / 32 * 32), slices = (words + threads - 1) / threads;
    e = attn::launch_after_previous(runs_kernel<E, G, kN>, dim3((unsigned)ranges, (unsigned)slices), dim3((unsigned)threads), 0, s, a);
    if (e != cudaSuccess) return e;
    return attn::launch_after_previous(join_kernel<G, kN>, dim3((unsigned)ranges, (unsigned)((words + 31) / 32)), dim3(256), 0, s, a);
}

template <class E, class G>
cudaError_t launch_gradient(const Gradient &a, bool wide, cudaStream_t s) {
    return wide ? launch_gradient<E, G, 4>(a, s) : launch_gradient<E, G, 1>(a, s);
}

template <class E>
cudaError_t set(cudaError_t e) {
    auto one = [&](auto *kernel) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(SortSmem));
    };
    one(sort_kernel<E, float, 4>), one(sort_kernel<E, float, 1>), one(sort_kernel<E, __nv_bfloat16, 4>), one(sort_kernel<E, __nv_bfloat16, 1>);
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
    int *status = nullptr;
    const int rc = attn::device_status_word(&status);
    if (rc != ATTN_OK) return rc;
    if (n == 0) return ATTN_OK;
    const bool wide = ((embed::bits(table) | embed::bits(pos_table) | embed::bits(y)) & 15) == 0 && C * each % 16 == 0 && ld * each % 16 == 0 &&
                      (!pos_table || pos_ld * each % 16 == 0);
    const int words = wide ? (int)(C * each / 16) : C;
    const long long per = embed::kThreads * embed::kUnits;
    if (n > (1ll << 40) / C || (n * words + per - 1) / per > 0x7fffffffll) return ATTN_ERR_UNSUPPORTED;
    const embed::Lookup a{table, pos_table, y, ld, pos_ld, n, Ids{tokens, id_type}, Ids{positions, id_type}, T, C, V, P, scale};
    const dim3 grid((unsigned)((n * words + per - 1) / per)), block(embed::kThreads);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == TENSOR_F32)
        return (int)(wide ? attn::launch_after_previous(embed::lookup_kernel<float, 4>, grid, block, 0, s, a, words)
                          : attn::launch_after_previous(embed::lookup_kernel<float, 1>, grid, block, 0, s, a, words));
    return (int)(wide ? attn::launch_after_previous(embed::lookup_kernel<__nv_bfloat16, 8>, grid, block, 0, s, a, words)
                      : attn::launch_after_previous(embed::lookup_kernel<__nv_bfloat16, 1>, grid, block, 0, s, a, words));
}

size_t tensor_sm100_embedding_backward_scratch_bytes(long long n, int C, int V, int P) {
    if (n <= 0 || n > (1 << 30) || C <= 0 || V < 0 || P < 0) return 0;
    return (V ? embed::list_bytes(n, C, V, nullptr, nullptr) : 0) + (P ? embed::list_bytes(n, C, P, nullptr, nullptr) : 0);
}

int tensor_sm100_embedding_backward(const void *dy, const void *tokens, void *dtable, const void *positions, void *dpos_table, void *scratch, long long n,
                                    long long ld_dy, long long ld, long long pos_ld, float scale, int type, int grad_type, int id_type, int T, int C, int V, int P,
                                    void *stream) {
    if (!dy || (!dtable && !dpos_table) || (dtable && !tokens)) return ATTN_ERR_NULL;
    if (n < 0 || C <= 0 || ld_dy < C || !embed::float_type(type) || !embed::float_type(grad_type) || !embed::id_type(id_type)) return ATTN_ERR_ARGUMENT;
    if ((dtable && (V <= 0 || ld < C)) || (dpos_table && (P <= 0 || pos_ld < C || (!positions && T <= 0)))) return ATTN_ERR_ARGUMENT;
    const bool listed = dtable || positions;
    if (n > 0 && listed && !scratch) return ATTN_ERR_NULL;
    const uintptr_t each = embed::each_of(type), grad_each = embed::each_of(grad_type);
    if (embed::bits(dy) % each || (embed::bits(dtable) | embed::bits(dpos_table)) % grad_each || (embed::bits(scratch) & 255) ||
        ((embed::bits(tokens) | embed::bits(positions)) & embed::id_mask(id_type)))
        return ATTN_ERR_ALIGN;
    if (n > (1 << 30) || C > (1 << 20)) return ATTN_ERR_UNSUPPORTED;
    if ((n && dtable && embed::overlap(dy, n, ld_dy, each, dtable, V, ld, grad_each, C)) || (n && dpos_table && embed::overlap(dy, n, ld_dy, each, dpos_table, P, pos_ld, grad_each, C)) ||
        (dtable && dpos_table && embed::overlap(dtable, V, ld, grad_each, dpos_table, P, pos_ld, grad_each, C)))
        return ATTN_ERR_ARGUMENT;
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
    // four columns at a time
    const bool wide = C % 4 == 0 && (embed::bits(dy) | (uintptr_t)(ld_dy * each)) % (4 * each) == 0 &&
                      (embed::bits(dtable) | embed::bits(dpos_table) | (uintptr_t)(dtable ? ld * grad_each : 0) | (uintptr_t)(dpos_table ? pos_ld * grad_each : 0)) %
                              (4 * grad_each) == 0;
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (type == TENSOR_F32)
        return (int)(grad_type == TENSOR_F32 ? embed::launch_gradient<float, float>(a, wide, s) : embed::launch_gradient<float, __nv_bfloat16>(a, wide, s));
    return (int)(grad_type == TENSOR_F32 ? embed::launch_gradient<__nv_bfloat16, float>(a, wide, s) : embed::launch_gradient<__nv_bfloat16, __nv_bfloat16>(a, wide, s));
}

}  // extern "C"
