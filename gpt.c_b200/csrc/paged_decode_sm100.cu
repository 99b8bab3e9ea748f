// Attention of new tokens over a paged key/value cache of bf16 for sm_100a: up to 8 rows, bound by HBM.
//
//   out[t, h] = sum_j p_j v[j] / sum_j p_j,   p_j = exp2(s_j - m),   s_j = (scale log2(e) q[t, h]) . k[j]
//
// A unit is one sequence, one key/value head and its rows (row = new token x query head of the group), 8 at most.  32 keys, a
// stage, are S^T = K Q^T and O^T += V^T P^T with mma.m16n8k16, rows in its smallest dimension: tcgen05.mma would compute 128
// rows, of which 120 are not there, and its results would have to come back through tensor memory.  q and p are three bf16
// terms each, so they take part exactly; sums over 32 keys start at zero and are added to the output with ordinary additions.
// K and V come by asynchronous 16-byte copies from wherever their pages are, V transposed by the load from shared memory.
//
// Up to 2 rows (packed_kernel): the terms of q, and of p, are columns of one product.  Each warp works by itself: it brings its stages,
// one ahead, and keeps a maximum, a sum and an output of its own.  Where there are many units a warp takes one; else four
// warps of a CTA, and the CTAs of a cluster, share it and are joined at the end.
// Up to 8 rows (rows_kernel): a product for each term; one warp of a CTA brings the stages, four take every fourth.
//
// 96 sequences of up to 1023 positions, 12 heads of 64: 40 us, 4.0 TB/s, CTAs that begin and end by themselves (30 % of issue
// slots used).  6 of up to 40001, 20 heads of 128 over 5: 103 us, 5.2 TB/s.
//
// A row whose result is not finite is computed again in fp32 arithmetic (0 times an infinite value that it does not see is NaN).
#include <cooperative_groups.h>

#include "attn_internal.h"
#include "paged_attn.cuh"

namespace paged {
namespace {

namespace cg = cooperative_groups;

constexpr int kWarps = 4, kThreads = 32 * (kWarps + 1);  // of the second kernel: that compute, and one that brings keys and values
constexpr int kRows = 8, kKeys = 32;                     // its rows; keys of a stage

enum Site : int { SITE_FULL = 461, SITE_EMPTY };

__device__ __forceinline__ void ldsm(uint32_t (&a)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm_t(uint32_t (&a)[4], uint32_t at) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(a[0]), "=r"(a[1]), "=r"(a[2]), "=r"(a[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ uint32_t transposed(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ void mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Where key j's row begins, in 16-byte words behind the first of its head: 32 bits reach 32 GB.  -1 where it has no page.
__device__ __forceinline__ int word_of(const Cache &c, const int *table, int j, int end, bool &missing) {
    const long long at = place(c, table, j, end, missing);
    return at < 0 ? -1 : (int)(at >> 3);
}

// ------------------------------------------------------------------------------------------
// up to eight rows
// ------------------------------------------------------------------------------------------
template <int kDP>
struct __align__(128) RowsSmem {
    static constexpr int kPitch = 2 * kDP, kTile = kKeys * kPitch, kStages = kDP == 64 ? 8 : 6;
    union {
        uint8_t kv[kStages][2][kTile];  // rows of kDP elements, their 16-byte words swizzled
        struct {                        // at the end
            float o[kWarps][kRows][kDP];
            float joined[kRows][kDP];
        };
    };
    float m[kWarps][kRows], l[kWarps][kRows], m_all[kRows], l_all[kRows];
    uint64_t full[kStages], empty[kStages];
    uint32_t there[kStages];  // a bit for each key of the stage that has a page
    int odd[kRows];
    int abort_flag;
};

template <int kDP>
__global__ void __launch_bounds__(kThreads, kDP == 64 ? 3 : 2) rows_kernel(Cache c, const float *q, float *out, long long ld, int heads, int few, int max_new,
                                                                            float scale_log2, int *status) {
    using Smem = RowsSmem<kDP>;
    constexpr int kStages = Smem::kStages, kPitch = Smem::kPitch, kK = kDP / 16;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int s = blockIdx.x / ranks, kvh = blockIdx.y, G = heads / c.kv_heads;
    WaitCtx ctx{&sm.abort_flag, status};
    if (threadIdx.x == 0) {
        sm.abort_flag = 0;
        for (int i = 0; i < kStages; i++) {
            mbar_init(&sm.full[i], 33);
            mbar_init(&sm.empty[i], 1);
        }
        fence_barrier_init();
    }
    if (threadIdx.x < kRows) sm.odd[threadIdx.x] = 0;
    pdl_launch_dependents();
    pdl_wait();
    const Span w = span_of(c, s);
    const int rows = w.count * G;
    const long long room = (long long)c.width * c.page_size;
    if (kvh == 0 && rank == 0 && threadIdx.x == 0 && w.count > 0 && (w.count > max_new || w.past < 0 || w.past + (long long)w.count > room)) report(status, ST_ATTEND);
    if (rows == 0 || rows > few || w.past < 0 || w.count > max_new) return;  // the whole cluster
    const int keys = (int)min((long long)w.past + w.count, room);
    const int *table = c.table + (long long)s * c.width;
    // this CTA's run of keys, in whole stages
    const int all = (keys + kKeys - 1) / kKeys, each = (all + ranks - 1) / ranks;
    const int begin = min(rank * each, all) * kKeys, steps = max(0, min(each, all - rank * each)), end = min(keys, begin + steps * kKeys);
    __syncthreads();

    // two rows of this lane: 2 (lane % 4) and the next; `group` is a key, or a column, of the eight that it has
    const int group = lane >> 2, pair = 2 * (lane & 3);
    float acc[kK][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
    if (warp == kWarps) {
        // ------------------------------ keys and values ------------------------------
        constexpr int kChunks = kDP / 8, kPer = 32 / kChunks;  // words of a row; rows that the warp takes at once
        const long long head = (long long)kvh * c.page_size * c.D;
        const int mine = lane / kChunks, ch = lane % kChunks;
        const bool col = 8 * ch < c.D;
        const long long at = col ? head + 8 * ch : 0;
        const __nv_bfloat16 *kp = static_cast<const __nv_bfloat16 *>(c.k) + at, *vp = static_cast<const __nv_bfloat16 *>(c.v) + at;
        bool missing = false;
        int next = steps > 0 ? word_of(c, table, begin + lane, end, missing) : -1;
        for (int n = 0; n < steps; n++) {
            const int st = n % kStages;
            const int here = next;
            next = word_of(c, table, begin + (n + 1) * kKeys + lane, end, missing);
            const uint32_t there = __ballot_sync(0xffffffffu, here >= 0);
            if (n >= kStages) await(&sm.empty[st], (n / kStages - 1) & 1, ctx, SITE_EMPTY);
            if (lane == 0) {
                sm.there[st] = there;
                mbar_arrive(&sm.full[st]);
            }
            const uint32_t kt = smem_u32(sm.kv[st][0]), vt = smem_u32(sm.kv[st][1]);
#pragma unroll
            for (int i = 0; i < kKeys / kPer; i++) {
                const int r = i * kPer + mine, off = __shfl_sync(0xffffffffu, here, r);
                const uint32_t to = r * kPitch + ((ch ^ (r & 7)) << 4);
                const bool in = off >= 0 && col;
                cp16(kt + to, kp + (long long)max(off, 0) * 8, in);
                cp16(vt + to, vp + (long long)max(off, 0) * 8, in);
            }
            arrive_when_copied(&sm.full[st]);
        }
        cp_wait<0>();
        if (missing) report(status, ST_ATTEND);
    } else {
        // ------------------------------ products and softmax ------------------------------
        uint32_t qt[3][kK][2];
        {
            const int at = min(group, rows - 1);
            const float *src = q + (w.first + at / G) * ld + (long long)(kvh * G + at % G) * c.D + pair;
#pragma unroll
            for (int kk = 0; kk < kK; kk++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const int d = 16 * kk + 8 * i;
                    const float2 v = group < rows && d < c.D ? *reinterpret_cast<const float2 *>(src + d) : make_float2(0.f, 0.f);
                    cut3(make_float2(v.x * scale_log2, v.y * scale_log2), qt[0][kk][i], qt[1][kk][i], qt[2][kk][i]);
                }
        }
#pragma unroll
        for (int kk = 0; kk < kK; kk++)
#pragma unroll
            for (int e = 0; e < 4; e++) acc[kk][e] = 0.f;
        int seen[2];  // keys that the rows see
#pragma unroll
        for (int i = 0; i < 2; i++) seen[i] = pair + i < rows ? w.past + (pair + i) / G + 1 : 0x7fffffff;
        // where this lane's part of a 16 x 16 block lies: K as rows of keys, V transposed
        const int k_row = (lane & 7) + 8 * ((lane >> 3) & 1), k_word = lane >> 4, v_row = (lane & 7) + 8 * (lane >> 4), v_word = (lane >> 3) & 1;
        for (int n = warp; n < steps; n += kWarps) {
            const int st = n % kStages, key0 = begin + n * kKeys;
            await(&sm.full[st], (n / kStages) & 1, ctx, SITE_FULL);
            const uint32_t kt = smem_u32(sm.kv[st][0]), vt = smem_u32(sm.kv[st][1]), there = sm.there[st];
            float sc[2][4];
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t a[kK][4];
#pragma unroll
                for (int kk = 0; kk < kK; kk++) ldsm(a[kk], kt + (16 * b + k_row) * kPitch + (((2 * kk + k_word) ^ (k_row & 7)) << 4));
                sc[b][0] = sc[b][1] = sc[b][2] = sc[b][3] = 0.f;
#pragma unroll
                for (int term = 2; term >= 0; term--)
#pragma unroll
                    for (int kk = 0; kk < kK; kk++) mma(sc[b], a[kk], qt[term][kk][0], qt[term][kk][1]);
            }
            if (there != 0xffffffffu || __any_sync(0xffffffffu, key0 + kKeys > min(seen[0], seen[1]))) {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int j = 16 * b + 8 * (e >> 1) + group;
                        if (!(there >> j & 1u) || key0 + j >= seen[e & 1]) sc[b][e] = -INFINITY;
                    }
            }
            float alpha[2], minus[2];
#pragma unroll
            for (int i = 0; i < 2; i++) {
                float top = fmaxf(max3(sc[0][i], sc[0][2 + i], sc[1][i]), sc[1][2 + i]);
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
                top = fmaxf(top, m[i]);
                const float base = top == -INFINITY ? 0.f : top;  // nothing but -inf so far
                alpha[i] = ex2f(m[i] - base);
                minus[i] = -base;
                m[i] = top;
                l[i] *= alpha[i];
            }
            float step[kK][4];
            uint32_t p[3][2][2];
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int h = 0; h < 2; h++) {  // keys 0 to 7, 8 to 15 of the block
                    const float2 x = add2(make_float2(sc[b][2 * h], sc[b][2 * h + 1]), make_float2(minus[0], minus[1]));
                    const float2 e = make_float2(ex2f(x.x), ex2f(x.y));
                    l[0] += e.x, l[1] += e.y;
                    uint32_t t[3];
                    cut3(e, t[0], t[1], t[2]);
#pragma unroll
                    for (int i = 0; i < 3; i++) p[i][b][h] = transposed(t[i]);
                }
#pragma unroll
            for (int kk = 0; kk < kK; kk++) {
                uint32_t a[2][4];
#pragma unroll
                for (int b = 0; b < 2; b++) ldsm_t(a[b], vt + (16 * b + v_row) * kPitch + (((2 * kk + v_word) ^ (v_row & 7)) << 4));
                step[kk][0] = step[kk][1] = step[kk][2] = step[kk][3] = 0.f;
#pragma unroll
                for (int term = 2; term >= 0; term--)
#pragma unroll
                    for (int b = 0; b < 2; b++) mma(step[kk], a[b], p[term][b][0], p[term][b][1]);
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.empty[st]);
#pragma unroll
            for (int kk = 0; kk < kK; kk++)
#pragma unroll
                for (int e = 0; e < 4; e++) acc[kk][e] = fmaf(acc[kk][e], alpha[e & 1], step[kk][e]);
        }
#pragma unroll
        for (int i = 0; i < 2; i++)
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l[i] += __shfl_xor_sync(0xffffffffu, l[i], x);
    }
    if (sm.abort_flag) __nanosleep(50000);  // let copies that are still in flight land
    __syncthreads();                        // the results take the place of keys and values
    if (warp < kWarps) {
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (group == 0) sm.m[warp][pair + i] = m[i], sm.l[warp][pair + i] = l[i];
#pragma unroll
            for (int kk = 0; kk < kK; kk++) sm.o[warp][pair + i][16 * kk + group] = acc[kk][i], sm.o[warp][pair + i][16 * kk + 8 + group] = acc[kk][2 + i];
        }
    }
    __syncthreads();
    // the warps of this CTA
    for (int i = threadIdx.x; i < rows * kDP; i += kThreads) {
        const int r = i / kDP, d = i % kDP;
        float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
        for (int x = 0; x < kWarps; x++) top = fmaxf(top, sm.m[x][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int x = 0; x < kWarps; x++) {
            const float by = ex2f(sm.m[x][r] - base);
            sum = fmaf(sm.l[x][r], by, sum), o = fmaf(sm.o[x][r][d], by, o);
        }
        sm.joined[r][d] = o;
        if (d == 0) sm.m_all[r] = top, sm.l_all[r] = sum;
        if (!(fmaf(o, 0.f, sum * 0.f) == 0.f)) sm.odd[r] = 1;  // what is finite times zero is zero
    }
    __syncthreads();
    for (int r = warp; r < rows; r += kWarps + 1)
        if (sm.odd[r])
            exact_row<__nv_bfloat16, kDP>(c, q + (w.first + r / G) * ld + (long long)(kvh * G + r % G) * c.D, table, kvh, begin, min(end, w.past + r / G + 1), scale_log2,
                                          sm.joined[r], &sm.m_all[r], &sm.l_all[r]);
    if (ranks > 1) cluster.sync();
    else __syncthreads();
    // every CTA of the cluster writes some of the values
    for (int i = rank * kThreads + threadIdx.x; i < rows * c.D; i += ranks * kThreads) {
        const int r = i / c.D, d = i - r * c.D;
        out[((long long)(w.first + r / G) * heads + kvh * G + r % G) * c.D + d] = joined_value(ranks, [&](int k) {
            const Smem &p = ranks > 1 ? *cluster.map_shared_rank(&sm, k) : sm;
            return Part{p.m_all[r], p.l_all[r], p.joined[r][d]};
        });
    }
    if (ranks > 1) cluster.sync();  // shared memory of the others is read until here
}

// ------------------------------------------------------------------------------------------
// one or two rows
// ------------------------------------------------------------------------------------------
constexpr int kAhead = 2;  // stages of a warp: with 3, fewer warps fit an SM (96 sequences, 12 heads of 64: 40 us with 2, 51 with 3)

template <int kDP, int kW>
struct __align__(128) PackedSmem {
    static constexpr int kPitch = 2 * kDP, kTile = kKeys * kPitch;
    union {
        uint8_t kv[kW][kAhead][2][kTile];  // rows of kDP elements, their 16-byte words swizzled
        struct {                           // at the end
            float o[kW][2][kDP];
            float joined[2][kDP];
        };
    };
    float m[kW][2], l[kW][2], m_all[2], l_all[2];
    uint32_t there[kW][kAhead];  // a bit for each key of the stage that has a page
    int odd[2];
};

// Column n of a product is term n / kR of row n % kR; columns from 3 kR on are zero.
//
// S^T in the accumulators: lane 4 g + t has columns 2 t and 2 t + 1 of rows g and g + 8 of a block of 16 keys, which are keys 2 g and 2 g + 1
// (the rows of K are taken in that order), so that the sums over t leave every lane of a group the scores of four keys,
// 2 g, 2 g + 1, 16 + 2 g, 17 + 2 g.  P^T as an operand: lane 4 n + t has column n of keys 2 t, 2 t + 1, 2 t + 8, 2 t + 9 of a block.  With
// keys 8 b .. 8 b + 7 and 16 + 8 b .. as the block b of that product, these are the four keys of group 4 b + t.
template <int kDP, int kW, int kR>
__global__ void __launch_bounds__(32 * kW) packed_kernel(Cache c, const float *q, float *out, long long ld, int heads, int few, int max_new, float scale_log2, int *status) {
    using Smem = PackedSmem<kDP, kW>;
    constexpr int kT = 32 * kW, kPitch = Smem::kPitch, kK = kDP / 16;
    extern __shared__ __align__(128) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int s = blockIdx.x / ranks, kvh = blockIdx.y, G = heads / c.kv_heads;
    auto sync = [] {
        if (kW == 1) __syncwarp();
        else __syncthreads();
    };
    pdl_launch_dependents();
    pdl_wait();
    const Span w = span_of(c, s);
    const int rows = w.count * G;
    const long long room = (long long)c.width * c.page_size;
    if (kvh == 0 && rank == 0 && threadIdx.x == 0 && w.count > 0 && (w.count > max_new || w.past < 0 || w.past + (long long)w.count > room)) report(status, ST_ATTEND);
    if (rows == 0 || rows > few || w.past < 0 || w.count > max_new) return;  // the whole cluster
    const int keys = (int)min((long long)w.past + w.count, room);
    const int *table = c.table + (long long)s * c.width;
    // this CTA's run of keys, in whole stages, of which this warp takes every kW-th
    const int all = (keys + kKeys - 1) / kKeys, each = (all + ranks - 1) / ranks;
    const int begin = min(rank * each, all) * kKeys, stages = max(0, min(each, all - rank * each)), end = min(keys, begin + stages * kKeys);
    const int steps = (stages - warp + kW - 1) / kW;

    constexpr int kChunks = kDP / 8, kPer = 32 / kChunks;  // words of a row; rows that the warp brings at once
    const int mine = lane / kChunks, ch = lane % kChunks;
    const bool col = 8 * ch < c.D;
    const long long from = (long long)kvh * c.page_size * c.D + (col ? 8 * ch : 0);
    const __nv_bfloat16 *kp = static_cast<const __nv_bfloat16 *>(c.k) + from, *vp = static_cast<const __nv_bfloat16 *>(c.v) + from;
    bool missing = false;
    auto first_key = [&](int n) { return begin + (warp + n * kW) * kKeys; };
    int next = word_of(c, table, first_key(0) + lane, end, missing);
    auto bring = [&](int n) {
        const int st = n % kAhead, here = next;
        next = word_of(c, table, first_key(n + 1) + lane, end, missing);
        const uint32_t there = __ballot_sync(0xffffffffu, here >= 0);
        if (lane == 0) sm.there[warp][st] = there;
        const uint32_t kt = smem_u32(sm.kv[warp][st][0]), vt = smem_u32(sm.kv[warp][st][1]);
#pragma unroll
        for (int i = 0; i < kKeys / kPer; i++) {
            const int r = i * kPer + mine, off = __shfl_sync(0xffffffffu, here, r);
            const bool in = off >= 0 && col;
            cp16(kt + r * kPitch + ((ch ^ (r >> 1 & 7)) << 4), kp + (long long)max(off, 0) * 8, in);
            cp16(vt + r * kPitch + ((ch ^ (r & 7)) << 4), vp + (long long)max(off, 0) * 8, in);
        }
    };
#pragma unroll
    for (int n = 0; n < kAhead - 1; n++) {
        if (n < steps) bring(n);
        cp_commit();
    }

    const int g = lane >> 2, t = lane & 3;
    float acc[kK][4], m[kR], l[kR];
    uint32_t qt[kK][2];
    {
        const int row = g % kR, term = g / kR;
        const float *src = q + (w.first + min(row, rows - 1) / G) * ld + (long long)(kvh * G + min(row, rows - 1) % G) * c.D + 2 * t;
#pragma unroll
        for (int kk = 0; kk < kK; kk++)
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const int d = 16 * kk + 8 * i;
                const float2 v = d < c.D ? *reinterpret_cast<const float2 *>(src + d) : make_float2(0.f, 0.f);
                uint32_t x[3];
                cut3(make_float2(v.x * scale_log2, v.y * scale_log2), x[0], x[1], x[2]);
                qt[kk][i] = term == 0 ? x[0] : term == 1 ? x[1] : term == 2 && g < 3 * kR ? x[2] : 0u;
            }
    }
#pragma unroll
    for (int kk = 0; kk < kK; kk++)
#pragma unroll
        for (int e = 0; e < 4; e++) acc[kk][e] = 0.f;
    int seen[kR];  // keys that the rows see
#pragma unroll
    for (int r = 0; r < kR; r++) seen[r] = r < rows ? w.past + r / G + 1 : 0x7fffffff, m[r] = -INFINITY, l[r] = 0.f;
    // where this lane's part of a block lies: K as rows of keys in the order above, V transposed
    const int k_row = 2 * (lane & 7) + (lane >> 3 & 1), k_word = lane >> 4, v_row = (lane & 7) + 16 * (lane >> 4), v_word = lane >> 3 & 1;
    for (int n = 0; n < steps; n++) {
        const int st = n % kAhead, key0 = first_key(n);
        if (n + kAhead - 1 < steps) bring(n + kAhead - 1);
        cp_commit();
        cp_wait<kAhead - 1>();
        __syncwarp();
        const uint32_t kt = smem_u32(sm.kv[warp][st][0]), vt = smem_u32(sm.kv[warp][st][1]), there = sm.there[warp][st];
        float sc[2][4];
#pragma unroll
        for (int b = 0; b < 2; b++) sc[b][0] = sc[b][1] = sc[b][2] = sc[b][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < kK; kk++)
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t a[4];
                ldsm(a, kt + (16 * b + k_row) * kPitch + (((2 * kk + k_word) ^ (lane & 7)) << 4));
                mma(sc[b], a, qt[kk][0], qt[kk][1]);
            }
        // scores of keys 16 b + 2 g + h, over the columns of a row
        float x[kR][2][2];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                if (kR == 1) {
                    float v = sc[b][2 * h] + sc[b][2 * h + 1];
                    v += __shfl_xor_sync(0xffffffffu, v, 1);
                    x[0][b][h] = __shfl_sync(0xffffffffu, v, lane & 28);  // columns 0 to 2 are with lanes 0 and 1 of the group
                } else {
#pragma unroll
                    for (int r = 0; r < kR; r++) {  // columns r, r + 2 and r + 4
                        const float v = sc[b][2 * h + r];
                        const float one = __shfl_sync(0xffffffffu, v, (lane & 28) + 2), two = __shfl_sync(0xffffffffu, v, (lane & 28) + 1);
                        x[r][b][h] = one + two + __shfl_sync(0xffffffffu, v, lane & 28);
                    }
                }
            }
        float alpha[kR];
        uint32_t mine_of[kR][2];  // this lane's term (t) of p, keys 2 g and 2 g + 1 of each half
#pragma unroll
        for (int r = 0; r < kR; r++) {
            if (there != 0xffffffffu || key0 + kKeys > seen[r]) {
#pragma unroll
                for (int b = 0; b < 2; b++)
#pragma unroll
                    for (int h = 0; h < 2; h++) {
                        const int j = 16 * b + 2 * g + h;
                        if (!(there >> j & 1u) || key0 + j >= seen[r]) x[r][b][h] = -INFINITY;
                    }
            }
            float top = fmaxf(max3(x[r][0][0], x[r][0][1], x[r][1][0]), x[r][1][1]);
#pragma unroll
            for (int y = 4; y < 32; y <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, y));
            top = fmaxf(top, m[r]);
            const float base = top == -INFINITY ? 0.f : top;  // nothing but -inf so far
            alpha[r] = ex2f(m[r] - base);
            m[r] = top;
            float sum = 0.f;
#pragma unroll
            for (int b = 0; b < 2; b++) {
                const float2 p = make_float2(ex2f(x[r][b][0] - base), ex2f(x[r][b][1] - base));
                sum += p.x + p.y;
                uint32_t cut[3];
                cut3(p, cut[0], cut[1], cut[2]);
                mine_of[r][b] = t == 0 ? cut[0] : t == 1 ? cut[1] : cut[2];
            }
            l[r] = l[r] * alpha[r] + sum;
        }
        uint32_t pt[2][2];
#pragma unroll
        for (int b = 0; b < 2; b++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
                const int there_is = 4 * (4 * b + t) + (g / kR < 3 ? g / kR : 0);
                uint32_t v = __shfl_sync(0xffffffffu, mine_of[0][h], there_is);
                if (kR == 2) {
                    const uint32_t other = __shfl_sync(0xffffffffu, mine_of[kR - 1][h], there_is);
                    v = g & 1 ? other : v;
                }
                pt[b][h] = g < 3 * kR ? v : 0u;
            }
#pragma unroll
        for (int kk = 0; kk < kK; kk++) {
            float step[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int b = 0; b < 2; b++) {
                uint32_t a[4];
                ldsm_t(a, vt + (8 * b + v_row) * kPitch + (((2 * kk + v_word) ^ (lane & 7)) << 4));
                mma(step, a, pt[b][0], pt[b][1]);
            }
            // columns 2 t and 2 t + 1: rows 0 and 1 where there are two
#pragma unroll
            for (int e = 0; e < 4; e++) acc[kk][e] = fmaf(acc[kk][e], alpha[kR == 2 ? e & 1 : 0], step[e]);
        }
        __syncwarp();  // the stage may be brought again
    }
    if (missing) report(status, ST_ATTEND);
    cp_wait<0>();
    // sums over the groups; every lane of a group has the same
#pragma unroll
    for (int r = 0; r < kR; r++)
#pragma unroll
        for (int y = 4; y < 32; y <<= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], y);
    sync();  // the results take the place of keys and values
    if (threadIdx.x < 2) sm.odd[threadIdx.x] = 0;
#pragma unroll
    for (int kk = 0; kk < kK; kk++)
#pragma unroll
        for (int h = 0; h < 2; h++)
#pragma unroll
            for (int r = 0; r < kR; r++) {
                float v = kR == 1 ? acc[kk][2 * h] + acc[kk][2 * h + 1] : acc[kk][2 * h + r];  // the terms' columns
                v += __shfl_xor_sync(0xffffffffu, v, 1);
                v += __shfl_xor_sync(0xffffffffu, v, 2);
                if (t == 0) sm.o[warp][r][16 * kk + 8 * h + g] = v;
            }
    if (lane == 0)
#pragma unroll
        for (int r = 0; r < kR; r++) sm.m[warp][r] = m[r], sm.l[warp][r] = l[r];
    sync();
    // the warps of this CTA
    for (int i = threadIdx.x; i < rows * kDP; i += kT) {
        const int r = i / kDP, d = i % kDP;
        float top = -INFINITY, sum = 0.f, o = 0.f;
#pragma unroll
        for (int x = 0; x < kW; x++) top = fmaxf(top, sm.m[x][r]);
        const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
        for (int x = 0; x < kW; x++) {
            const float by = ex2f(sm.m[x][r] - base);
            sum = fmaf(sm.l[x][r], by, sum), o = fmaf(sm.o[x][r][d], by, o);
        }
        sm.joined[r][d] = o;
        if (d == 0) sm.m_all[r] = top, sm.l_all[r] = sum;
        if (!(fmaf(o, 0.f, sum * 0.f) == 0.f)) sm.odd[r] = 1;  // what is finite times zero is zero
    }
    sync();
    for (int r = warp; r < rows; r += kW)
        if (sm.odd[r])
            exact_row<__nv_bfloat16, kDP>(c, q + (w.first + r / G) * ld + (long long)(kvh * G + r % G) * c.D, table, kvh, begin, min(end, w.past + r / G + 1), scale_log2,
                                          sm.joined[r], &sm.m_all[r], &sm.l_all[r]);
    if (ranks > 1) cluster.sync();
    else sync();
    // every CTA of the cluster writes some of the values
    for (int i = rank * kT + threadIdx.x; i < rows * c.D; i += ranks * kT) {
        const int r = i / c.D, d = i - r * c.D;
        out[((long long)(w.first + r / G) * heads + kvh * G + r % G) * c.D + d] = joined_value(ranks, [&](int k) {
            const Smem &p = ranks > 1 ? *cluster.map_shared_rank(&sm, k) : sm;
            return Part{p.m_all[r], p.l_all[r], p.joined[r][d]};
        });
    }
    if (ranks > 1) cluster.sync();  // shared memory of the others is read until here
}

template <int kDP, int kW, int kR>
cudaError_t launch_packed(const Call &a, int few, unsigned ranks) {
    if ((long long)a.c.seqs * ranks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    return attn::launch_clusters_after_previous(packed_kernel<kDP, kW, kR>, dim3((unsigned)a.c.seqs * ranks, (unsigned)a.c.kv_heads), dim3(32 * kW),
                                                sizeof(PackedSmem<kDP, kW>), ranks, a.s, a.c, a.q, a.out, a.ld, a.heads, few, a.max_new, a.scale_log2, a.status);
}

// One warp a unit where that leaves each SM enough of them and no sequence can be long; else four warps and as many CTAs as fit the
// GPU at a time, and enough for 2048 keys a warp.  Lengths up to 1022 positions, one warp / four, us: 12 heads of 64, 30 sequences 34 / 17,
// 96 43 / 40, 400 119 / 130; heads of 128, 96 sequences 80 / 115.
template <int kDP, int kR>
cudaError_t launch_packed_width(const Call &a, int few) {
    constexpr int kFull = kDP == 64 ? 8 : 2, kResident = kDP == 64 ? 3 : 1;
    const long long units = (long long)a.c.seqs * a.c.kv_heads, keys = (long long)a.c.width * a.c.page_size;
    const int sms = attn::sm_count();
    if (units >= (long long)kFull * sms && keys <= 2048) return launch_packed<kDP, 1, kR>(a, few, 1);
    unsigned ranks = 1;
    while (ranks < 8 && (units * ranks * 2 <= (long long)kResident * sms || keys > 4 * 2048ll * ranks)) ranks *= 2;
    return launch_packed<kDP, 4, kR>(a, few, ranks);
}

template <int kDP>
cudaError_t launch_rows(const Call &a, int few) {
    const unsigned ranks = ranks_of(a, (long long)a.c.seqs * a.c.kv_heads);
    if ((long long)a.c.seqs * ranks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    return attn::launch_clusters_after_previous(rows_kernel<kDP>, dim3((unsigned)a.c.seqs * ranks, (unsigned)a.c.kv_heads), dim3(kThreads), sizeof(RowsSmem<kDP>), ranks,
                                                a.s, a.c, a.q, a.out, a.ld, a.heads, few, a.max_new, a.scale_log2, a.status);
}

template <int kDP>
cudaError_t launch_width(const Call &a, int few) {
    const long long most = min((long long)few, (long long)a.max_new * (a.heads / a.c.kv_heads));
    if (most == 1) return launch_packed_width<kDP, 1>(a, few);
    return most == 2 ? launch_packed_width<kDP, 2>(a, few) : launch_rows<kDP>(a, few);
}

template <int kDP>
cudaError_t set_width() {
    const cudaFuncAttribute at = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaError_t e = cudaFuncSetAttribute(rows_kernel<kDP>, at, (int)sizeof(RowsSmem<kDP>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(packed_kernel<kDP, 1, 1>, at, (int)sizeof(PackedSmem<kDP, 1>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(packed_kernel<kDP, 1, 2>, at, (int)sizeof(PackedSmem<kDP, 1>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(packed_kernel<kDP, 4, 1>, at, (int)sizeof(PackedSmem<kDP, 4>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(packed_kernel<kDP, 4, 2>, at, (int)sizeof(PackedSmem<kDP, 4>));
    return e;
}

}  // namespace

cudaError_t launch_decode(const Call &a, int few) { return a.c.D <= 64 ? launch_width<64>(a, few) : launch_width<128>(a, few); }

cudaError_t decode_set_attributes() {
    const cudaError_t e = set_width<64>();
    return e != cudaSuccess ? e : set_width<128>();
}

}  // namespace paged
