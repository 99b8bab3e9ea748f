// Attention of new tokens over a paged key/value cache for sm_100a: many rows, on the tensor cores.
//
//   out[t, h] = sum_j p_j v[j] / sum_j p_j,   p_j = exp2(s_j - m),   s_j = (scale log2(e) q[t, h]) . k[j]
//
// A unit is one sequence, one key/value head and 128 of its rows (row = new token x query head of the group); a CTA takes it,
// or a cluster of CTAs with a run of the keys each, and walks the keys in steps of 64.  fp32 values are three bf16 terms
// (attn24.cuh), so q and p take part exactly; bf16 pages are one term, fp32 pages three: 3 or 6 passes a product.  The tensor
// cores truncate their sums, so the P V of each step starts at zero and is added to the output in registers.
//
// Warps: one issues the tensor-core instructions, a few bring keys and values (bf16 by asynchronous 16-byte copies, fp32
// through registers, split on the way) from wherever their pages are into a ring, eight per group do the softmax, two
// threads a row.  Two score buffers alternate, S of step n+2 is issued behind P V of step n.  Where a step takes the tensor
// cores less time than a softmax step (bf16, head size up to 64: 768 cycles), two groups take every other step each, with a
// maximum, sum and output of their own that are joined at the end.
//
// A row whose result is not finite is computed again in fp32 arithmetic: 0 times an infinite value that the row does
// not see is NaN on the tensor cores, and so are the terms of an infinity.
#include <cooperative_groups.h>

#include "attn24.cuh"
#include "attn_internal.h"
#include "paged.cuh"
#include "paged_attn.cuh"

namespace paged {
namespace {

namespace cg = cooperative_groups;
using namespace attn24;

constexpr int kRowsTile = 128;

template <class T, int kDP>
struct Shape {
    static constexpr bool kWide = sizeof(T) == 4;          // fp32 pages
    static constexpr int kTerms = kWide ? 3 : 1;           // of K and V
    static constexpr int kGroups = !kWide && kDP == 64 ? 2 : 1;
    static constexpr int kProducers = kWide ? 7 : 3;       // warps 1 .. ; warp 0 issues
    static constexpr int kFirst = kProducers + 1;          // first softmax warp, a multiple of four
    static constexpr int kThreads = 32 * (kFirst + 8 * kGroups);
    static constexpr int kPlane = kStep * kDP * 2;         // one term of 64 keys
    static constexpr int kStage = 2 * kTerms * kPlane;     // K terms, V terms
    static constexpr int kStages = kWide ? (kDP == 64 ? 4 : 2) : (kDP == 64 ? 8 : 6);
    static constexpr int kLag = kWide ? 0 : (kDP == 64 ? 4 : 2);  // steps between the request of a stage and its hand-over
    static constexpr uint32_t kColO = 192, kColQ = 192 + kDP;     // scores: twice 96 columns before them
    static_assert(kColQ + 3 * kDP / 2 <= 512, "tensor memory");
    static_assert(kLag <= kStages - 2 || kLag == 0, "a step is consumed only when the next one is there");
};

template <class T, int kDP>
struct __align__(1024) TileSmem {
    using S = Shape<T, kDP>;
    union {
        uint8_t ring[S::kStages][S::kStage];
        struct {  // at the end
            float o[kRowsTile][kDP + 4];
            float o1[kRowsTile][kDP + 4];
        } fin;
    };
    uint64_t kv_full[S::kStages], kv_empty[S::kStages], s_full[2], p_full[2], o_full[2], o_free, q_ready;
    uint32_t valid[S::kStages][2];          // keys of the stage that are there
    float xmax[S::kGroups][2][2][kRowsTile];  // [group][step parity][half][row]
    float m[kRowsTile], l[kRowsTile], m1[kRowsTile], l1[kRowsTile], half_l[S::kGroups][kRowsTile];
    uint32_t odd[kRowsTile / 32];           // rows to be computed again
    int seq, tile;
    uint32_t tmem_base;
    int abort_flag;
};

enum Site : int { SITE_KV_EMPTY = 401, SITE_KV_FULL, SITE_S_FULL, SITE_P_FULL, SITE_O_FULL, SITE_O_FREE, SITE_Q_READY, SITE_ALIGN };

// The sequence and tile of unit `u`, tiles counted over the sequences with more than `few` rows and no more new tokens than max_new;
// tile -1 past the last.  A whole warp.  check: reports lengths that the call does not allow.
__device__ __forceinline__ void find_tile(const Cache &c, int G, int few, int max_new, int u, bool check, int *status, int &seq, int &tile) {
    const int lane = threadIdx.x & 31;
    seq = 0, tile = -1;
    for (int base = 0; base < c.seqs; base += 32) {
        const int s = base + lane;
        int tiles = 0;
        if (s < c.seqs) {
            const Span w = span_of(c, s);
            const bool good = w.count <= max_new && w.past >= 0;
            if (check && w.count > 0 && (!good || w.past + (long long)w.count > (long long)c.width * c.page_size)) report(status, ST_ATTEND);
            const long long rows = (long long)w.count * G;
            tiles = good && rows > few ? (int)((rows + kRowsTile - 1) / kRowsTile) : 0;
        }
        int run = tiles;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int left = __shfl_up_sync(0xffffffffu, run, o);
            if (lane >= o) run += left;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, run > u);
        if (past != 0 && tile < 0) {
            const int at = __ffs(past) - 1;
            seq = base + at;
            tile = u - __shfl_sync(0xffffffffu, run - tiles, at);
            if (!check) return;
        }
        u -= __shfl_sync(0xffffffffu, run, 31);
        if (tile >= 0) u = 0x7fffffff;  // only the check goes on
    }
}

template <class T, int kDP>
__global__ void __launch_bounds__(Shape<T, kDP>::kThreads, 1) tile_kernel(Cache c, const float *q, float *out, long long ld, int heads, int few, int max_new,
                                                                         float scale_log2, int *status) {
    using Sh = Shape<T, kDP>;
    using Smem = TileSmem<T, kDP>;
    constexpr int kK = kDP / 16, kStages = Sh::kStages, kPlane = Sh::kPlane, kGroups = Sh::kGroups, kTerms = Sh::kTerms, kHalf = kDP / 2;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int ranks = (int)cluster.num_blocks(), rank = (int)cluster.block_rank();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31, kvh = blockIdx.y, G = heads / c.kv_heads;
    WaitCtx ctx{&sm.abort_flag, status};
    if (threadIdx.x == 0) {
        if ((smem_u32(smem_raw) & 1023u) != 0) report(status, ST_TIMEOUT_BASE + SITE_ALIGN);
        sm.abort_flag = 0;
        for (int i = 0; i < kStages; i++) {
            mbar_init(&sm.kv_full[i], Sh::kProducers);
            mbar_init(&sm.kv_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.s_full[i], 1);
            mbar_init(&sm.p_full[i], 8);
            mbar_init(&sm.o_full[i], 1);
        }
        mbar_init(&sm.o_free, 8);
        mbar_init(&sm.q_ready, 8);
        fence_barrier_init();
    }
    if (warp == 1) tmem_alloc_then_launch_dependents(&sm.tmem_base, 512);
    pdl_wait();
    if (warp == 0) {
        int seq, tile;
        const int units = gridDim.x / ranks, u = units - 1 - (int)(blockIdx.x / ranks);  // the last tiles of a sequence are its longest
        find_tile(c, G, few, max_new, u, u == 0 && kvh == 0 && rank == 0, status, seq, tile);
        if (lane == 0) sm.seq = seq, sm.tile = tile;
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem_base, 0);
    const int seq = __shfl_sync(0xffffffffu, sm.seq, 0), tile = __shfl_sync(0xffffffffu, sm.tile, 0);
    const Span w = span_of(c, seq);
    const int rows = w.count * G, row0 = tile * kRowsTile;
    const int *table = c.table + (long long)seq * c.width;
    // this CTA's run of keys: steps first .. first + nsteps - 1
    const int last = (min(row0 + kRowsTile, rows) - 1) / G;
    const int keys = tile < 0 ? 0 : (int)min((long long)w.past + last + 1, (long long)c.width * c.page_size);
    const int all = (keys + kStep - 1) / kStep, each = (all + ranks - 1) / ranks;
    const int first = min(rank * each, all), nsteps = min(each, all - first);
    const long long head = (long long)kvh * c.page_size * c.D;

    if (nsteps > 0 && warp == 0) {
        // ------------------------------ MMA issuer ------------------------------
        constexpr uint32_t idesc_s = idesc_bf16_f32(kRowsTile, kStep, 0, 0), idesc_o = idesc_bf16_f32(kRowsTile, kDP, 0, 1);
        constexpr int kPasses = kTerms == 3 ? 6 : 3;
        constexpr int kTermA[6] = {2, 1, 0, 1, 0, 0}, kTermB[6] = {0, 1, 2, 0, 1, 0};  // smallest first
        const uint32_t leader = elect_leader();
        const uint64_t kd = smem_desc_sw128(smem_u32(sm.ring[0]), 16, 1024);
        const uint64_t vd = smem_desc_sw128(smem_u32(sm.ring[0]) + kTerms * kPlane, kStep * 128, 1024);
        auto term_a = [&](int i) { return kTerms == 3 ? kTermA[i] : 2 - i; };
        auto term_b = [&](int i) { return kTerms == 3 ? kTermB[i] : 0; };
        auto issue_s = [&](int n) {
            const int st = n % kStages;
            await(&sm.kv_full[st], (n / kStages) & 1, ctx, SITE_KV_FULL);
            const uint64_t at = desc_advance(kd, st * Sh::kStage);
#pragma unroll
            for (int i = 0; i < kPasses; i++)
#pragma unroll
                for (int kk = 0; kk < kK; kk++)
                    mma_ts_lead(leader, tmem + (n & 1) * 96, tmem + Sh::kColQ + kHalf * term_a(i) + 8 * kk,
                                desc_advance(at, term_b(i) * kPlane + (kk >> 2) * (kStep * 128) + (kk & 3) * 32), idesc_s, i > 0 || kk > 0 ? 1u : 0u);
            tc_commit_lead(leader, &sm.s_full[n & 1]);
        };
        await(&sm.q_ready, 0, ctx, SITE_Q_READY);
        issue_s(0);
        if (nsteps > 1) issue_s(1);
        for (int n = 0; n < nsteps; n++) {
            const int st = n % kStages;
            await(&sm.p_full[n & 1], (n >> 1) & 1, ctx, SITE_P_FULL);
            if (kGroups == 2 && n > 0) await(&sm.o_free, (n - 1) & 1, ctx, SITE_O_FREE);
            const uint64_t at = desc_advance(vd, st * Sh::kStage);
#pragma unroll
            for (int i = 0; i < kPasses; i++)
#pragma unroll
                for (int kk = 0; kk < kStep / 16; kk++)
                    mma_ts_lead(leader, tmem + Sh::kColO, tmem + (n & 1) * 96 + term_column(term_a(i), kk), desc_advance(at, term_b(i) * kPlane + kk * 2048),
                                idesc_o, i > 0 || kk > 0 ? 1u : 0u);
            tc_commit_lead(leader, &sm.o_full[n & 1]);
            tc_commit_lead(leader, &sm.kv_empty[st]);
            if (n + 2 < nsteps) issue_s(n + 2);  // where P_n was, which P V of step n, earlier in the pipe, has read by then
        }
    } else if (nsteps > 0 && warp < Sh::kFirst) {
        // ------------------------------ producers ------------------------------
        constexpr int kChunks = kDP / 8, kPer = 32 / kChunks;  // pieces of 8 columns of a row; rows that a warp takes at once
        const int mine = lane / kChunks, ch = lane % kChunks, from = warp - 1;
        const T *kp = static_cast<const T *>(c.k) + head, *vp = static_cast<const T *>(c.v) + head;
        const bool col = 8 * ch < c.D;
        bool missing = false;
        for (int n = 0; n < nsteps; n++) {
            const int st = n % kStages, key0 = (first + n) * kStep;
            const long long lo = place(c, table, key0 + lane, keys, missing), hi = place(c, table, key0 + 32 + lane, keys, missing);
            const uint32_t there0 = __ballot_sync(0xffffffffu, lo >= 0), there1 = __ballot_sync(0xffffffffu, hi >= 0);
            if (n >= kStages) await(&sm.kv_empty[st], (n / kStages - 1) & 1, ctx, SITE_KV_EMPTY);
            if (from == 0 && lane == 0) sm.valid[st][0] = there0, sm.valid[st][1] = there1;
            uint8_t *kt = sm.ring[st], *vt = kt + kTerms * kPlane;
            if constexpr (!Sh::kWide) {
#pragma unroll
                for (int i = 0; i < (64 / kPer + Sh::kProducers - 1) / Sh::kProducers; i++) {
                    const int it = i * Sh::kProducers + from;
                    if (it >= 64 / kPer) break;
                    const int r = it * kPer + mine;
                    const long long off = __shfl_sync(0xffffffffu, it * kPer < 32 ? lo : hi, r & 31);
                    const bool in = off >= 0 && col;
                    const long long at = in ? off + 8 * ch : 0;
                    const uint32_t to = (ch >> 3) * (kStep * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4);
                    cp16(smem_u32(kt) + to, kp + at, in);
                    cp16(smem_u32(vt) + to, vp + at, in);
                }
                cp_commit();
                if (n >= Sh::kLag) {
                    cp_wait<Sh::kLag>();
                    warp_arrive(&sm.kv_full[(n - Sh::kLag) % kStages], lane);
                }
            } else {
                constexpr int kEach = (64 / kPer + Sh::kProducers - 1) / Sh::kProducers;
#pragma unroll 1
                for (int kv = 0; kv < 2; kv++) {
                    const float *src = reinterpret_cast<const float *>(kv ? vp : kp);
                    float4 f[kEach][2];
#pragma unroll
                    for (int i = 0; i < kEach; i++) {
                        const int it = i * Sh::kProducers + from, r = it * kPer + mine;
                        const long long off = __shfl_sync(0xffffffffu, it * kPer < 32 ? lo : hi, r & 31);
                        f[i][0] = f[i][1] = make_float4(0.f, 0.f, 0.f, 0.f);
                        if (it < 64 / kPer && off >= 0 && col) {
                            f[i][0] = *reinterpret_cast<const float4 *>(src + off + 8 * ch);
                            f[i][1] = *reinterpret_cast<const float4 *>(src + off + 8 * ch + 4);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < kEach; i++) {
                        const int it = i * Sh::kProducers + from, r = it * kPer + mine;
                        if (it >= 64 / kPer) break;
                        const float g[8] = {f[i][0].x, f[i][0].y, f[i][0].z, f[i][0].w, f[i][1].x, f[i][1].y, f[i][1].z, f[i][1].w};
                        store_split3<true>(kv ? vt : kt, kPlane, (ch >> 3) * (kStep * 128) + r * 128 + (((ch & 7) ^ (r & 7)) << 4), g);
                    }
                }
                warp_arrive(&sm.kv_full[st], lane);
            }
        }
        if constexpr (!Sh::kWide) {
            cp_wait<0>();
            for (int n = max(0, nsteps - Sh::kLag); n < nsteps; n++) warp_arrive(&sm.kv_full[n % kStages], lane);
        }
        if (missing) report(status, ST_ATTEND);
    }
    float o[kHalf], m = -INFINITY, l = 0.f;
    const int group = (warp - Sh::kFirst) >> 3, half = ((warp - Sh::kFirst) >> 2) & 1, quarter = warp & 3, row = 32 * quarter + lane;
    const uint32_t lane_addr = (uint32_t)(quarter << 5) << 16;
    const bool softmax = warp >= Sh::kFirst;
    if (softmax) {
        // ------------------------------ softmax ------------------------------
        const int at = row0 + row;
        const int seen = tile >= 0 && at < rows ? w.past + at / G + 1 : 0;  // keys that this row sees
#pragma unroll
        for (int e = 0; e < kHalf; e++) o[e] = 0.f;
        if (nsteps > 0 && group == 0) {
            const float *src = q + (w.first + at / G) * ld + (long long)(kvh * G + at % G) * c.D + half * kHalf;
#pragma unroll
            for (int b = 0; b < kHalf; b += 32) {
                uint32_t t[3][16];
#pragma unroll
                for (int e = 0; e < 32; e += 4) {
                    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                    if (at < rows && half * kHalf + b + e < c.D) v = *reinterpret_cast<const float4 *>(src + b + e);
                    cut3(make_float2(v.x * scale_log2, v.y * scale_log2), t[0][e / 2], t[1][e / 2], t[2][e / 2]);
                    cut3(make_float2(v.z * scale_log2, v.w * scale_log2), t[0][e / 2 + 1], t[1][e / 2 + 1], t[2][e / 2 + 1]);
                }
#pragma unroll
                for (int i = 0; i < 3; i++) tmem_st16(tmem + lane_addr + Sh::kColQ + kHalf * i + (half * kHalf + b) / 2, t[i]);
            }
            tmem_wait_st();
            arrive_tmem(&sm.q_ready, lane);
        }
        const uint32_t t_o = tmem + lane_addr + Sh::kColO + half * kHalf;
        auto add_output = [&](int n, float by) {
            await(&sm.o_full[n & 1], (n >> 1) & 1, ctx, SITE_O_FULL);
#pragma unroll
            for (int b = 0; b < kHalf; b += 16) {
                uint32_t r[16];
                tmem_ld16(t_o + b, r);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e++) o[b + e] = fmaf(o[b + e], by, __uint_as_float(r[e]));
            }
        };
        float alpha_before = 1.f;
        for (int n = group; n < nsteps; n += kGroups) {
            const int st = n % kStages, key0 = (first + n) * kStep + 32 * half;
            const uint32_t t_s = tmem + lane_addr + (n & 1) * 96;
            await(&sm.kv_full[st], (n / kStages) & 1, ctx, SITE_KV_FULL);  // for what it says of the keys
            const int lim = seen - key0;
            const uint32_t bits = sm.valid[st][half] & (lim >= 32 ? 0xffffffffu : lim <= 0 ? 0u : (1u << lim) - 1u);
            await(&sm.s_full[n & 1], (n >> 1) & 1, ctx, SITE_S_FULL);
            uint32_t s[32];
            tmem_ld32(t_s + 32 * half, s);
            tmem_wait_ld();
            if (__any_sync(0xffffffffu, bits != 0xffffffffu)) {
#pragma unroll
                for (int e = 0; e < 32; e++)
                    if (!(bits >> e & 1u)) s[e] = 0xff800000u;  // -inf
            }
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < 32; e += 2) mx = max3(mx, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
            const int par = (n / kGroups) & 1;
            sm.xmax[group][par][half][row] = mx;
            named_sync(1 + 4 * group + quarter, 64);
            mx = max3(m, mx, sm.xmax[group][par][half ^ 1][row]);
            const float base = mx == -INFINITY ? 0.f : mx;  // nothing but -inf so far
            const float alpha = ex2f(m - base);
            m = mx;
            const float2 minus = make_float2(-base, -base);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int b = 0; b < 2; b++) {  // 16 columns make 8 of each term
                uint32_t hi[8], mid[8], lo[8];
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float2 x = add2(make_float2(__uint_as_float(s[16 * b + 2 * e]), __uint_as_float(s[16 * b + 2 * e + 1])), minus);
                    const float2 p = make_float2(ex2f(x.x), ex2f(x.y));
                    sum = add2(sum, p);
                    cut3(p, hi[e], mid[e], lo[e]);
                }
                tmem_st8(t_s + term_column(0, 2 * half + b), hi);
                tmem_st8(t_s + term_column(1, 2 * half + b), mid);
                tmem_st8(t_s + term_column(2, 2 * half + b), lo);
            }
            l = l * alpha + (sum.x + sum.y);
            tmem_wait_st();
            if (kGroups == 1 && n > 0) add_output(n - 1, alpha_before);
            alpha_before = alpha;
            arrive_tmem(&sm.p_full[n & 1], lane);
            if (kGroups == 2) {
                add_output(n, alpha);
                arrive_tmem(&sm.o_free, lane);
            }
        }
        if (kGroups == 1 && nsteps > 0) add_output(nsteps - 1, alpha_before);
        if (half == 1) sm.half_l[group][row] = l;
    }
    if (sm.abort_flag) __nanosleep(50000);  // let products that are still in flight end
    if (threadIdx.x < kRowsTile / 32) sm.odd[threadIdx.x] = 0;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc(tmem, 512);  // before anything that waits for the other CTAs of the cluster
    if (tile >= 0) {
        if (softmax) {
            if (half == 0) l += sm.half_l[group][row];
            if (kGroups == 2 && group == 1) {
#pragma unroll
                for (int e = 0; e < kHalf; e += 4)
                    *reinterpret_cast<float4 *>(&sm.fin.o1[row][half * kHalf + e]) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                if (half == 0) sm.m1[row] = m, sm.l1[row] = l;
            }
        }
        if (kGroups == 2) __syncthreads();
        if (softmax && group == 0) {
            if (kGroups == 2) {
                const float mo = sm.m1[row], top = fmaxf(m, mo), base = top == -INFINITY ? 0.f : top, a = ex2f(m - base), b = ex2f(mo - base);
#pragma unroll
                for (int e = 0; e < kHalf; e++) o[e] = o[e] * a + sm.fin.o1[row][half * kHalf + e] * b;
                l = l * a + sm.l1[row] * b;  // of the first half
                m = top;
            }
            float zero = half == 0 ? l * 0.f : 0.f;  // what is finite times zero is zero
#pragma unroll
            for (int e = 0; e < kHalf; e++) zero = fmaf(o[e], 0.f, zero);
#pragma unroll
            for (int e = 0; e < kHalf; e += 4)
                *reinterpret_cast<float4 *>(&sm.fin.o[row][half * kHalf + e]) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            if (half == 0) sm.m[row] = m, sm.l[row] = l;
            const uint32_t odd = __ballot_sync(0xffffffffu, !(zero == 0.f) && row0 + row < rows);
            if (lane == 0 && odd) atomicOr(&sm.odd[quarter], odd);
        }
        __syncthreads();
        if (sm.odd[0] | sm.odd[1] | sm.odd[2] | sm.odd[3]) {
            for (int r = warp; r < kRowsTile; r += Sh::kThreads / 32) {
                if (!(sm.odd[r >> 5] >> (r & 31) & 1u)) continue;
                const int at = row0 + r;
                exact_row<T, kDP>(c, q + (w.first + at / G) * ld + (long long)(kvh * G + at % G) * c.D, table, kvh, first * kStep,
                                  min(min((first + nsteps) * kStep, keys), w.past + at / G + 1), scale_log2, sm.fin.o[r], &sm.m[r], &sm.l[r]);
            }
        }
        if (ranks > 1) cluster.sync();
        else __syncthreads();
        // rows rank, rank + ranks, .. of all CTAs' parts; 16 or 32 threads a row
        constexpr int kWords = kDP / 4;
        const int per = Sh::kThreads / kWords, word = threadIdx.x % kWords;
        for (int r = rank + ranks * (int)(threadIdx.x / kWords); r < kRowsTile && row0 + r < rows; r += ranks * per) {
            float top = -INFINITY, sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            for (int k = 0; k < ranks; k++) {
                const Smem &p = ranks > 1 ? *cluster.map_shared_rank(&sm, k) : sm;
                const float mo = p.m[r], t2 = fmaxf(top, mo), base = t2 == -INFINITY ? 0.f : t2, a = ex2f(top - base), b = ex2f(mo - base);
                const float4 v = *reinterpret_cast<const float4 *>(&p.fin.o[r][4 * word]);
                sum = sum * a + p.l[r] * b;
                acc = make_float4(acc.x * a + v.x * b, acc.y * a + v.y * b, acc.z * a + v.z * b, acc.w * a + v.w * b);
                top = t2;
            }
            const int at = row0 + r;
            const float by = sum == 0.f ? 0.f : 1.f / sum;
            if (4 * word < c.D)
                *reinterpret_cast<float4 *>(out + ((long long)(w.first + at / G) * heads + kvh * G + at % G) * c.D + 4 * word) =
                    make_float4(acc.x * by, acc.y * by, acc.z * by, acc.w * by);
        }
        if (ranks > 1) cluster.sync();  // shared memory of the others is read until here
    }
}

template <class T, int kDP>
cudaError_t launch_tile(const Call &a, int few) {
    using Sh = Shape<T, kDP>;
    const int G = a.heads / a.c.kv_heads, sms = attn::sm_count();
    const long long units = (long long)a.c.tokens * G / kRowsTile + a.c.seqs;
    unsigned ranks = 1;
    while (ranks < 8 && units * a.c.kv_heads * ranks * 2 <= sms) ranks *= 2;
    if (units * ranks > 0x7fffffffll) return cudaErrorInvalidConfiguration;
    return attn::launch_clusters_after_previous(tile_kernel<T, kDP>, dim3((unsigned)(units * ranks), (unsigned)a.c.kv_heads), dim3(Sh::kThreads),
                                                sizeof(TileSmem<T, kDP>), ranks, a.s, a.c, a.q, a.out, a.ld, a.heads, few, a.max_new, a.scale_log2, a.status);
}

}  // namespace

cudaError_t launch_tiles(const Call &a, int few) {
    if (a.type == ATTN_CACHE_BF16) return a.c.D <= 64 ? launch_tile<__nv_bfloat16, 64>(a, few) : launch_tile<__nv_bfloat16, 128>(a, few);
    return a.c.D <= 64 ? launch_tile<float, 64>(a, few) : launch_tile<float, 128>(a, few);
}

cudaError_t tiles_set_attributes() {
    const cudaFuncAttribute at = cudaFuncAttributeMaxDynamicSharedMemorySize;
    cudaError_t e = cudaFuncSetAttribute(tile_kernel<__nv_bfloat16, 64>, at, (int)sizeof(TileSmem<__nv_bfloat16, 64>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tile_kernel<__nv_bfloat16, 128>, at, (int)sizeof(TileSmem<__nv_bfloat16, 128>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tile_kernel<float, 64>, at, (int)sizeof(TileSmem<float, 64>));
    if (e == cudaSuccess) e = cudaFuncSetAttribute(tile_kernel<float, 128>, at, (int)sizeof(TileSmem<float, 128>));
    return e;
}

}  // namespace paged
