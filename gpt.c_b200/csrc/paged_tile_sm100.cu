// Attention of new tokens over a paged key/value cache for sm_100a: many rows, on the tensor cores.
//
//   out[t, h] = sum_j p_j v[j] / sum_j p_j,   p_j = exp2(s_j - m),   s_j = (scale log2(e) q[t, h]) . k[j]
//
// A unit is one sequence, one key/value head and 128 of its rows (row = new token x query head of the group); a CTA takes it,
// or a cluster of CTAs with a run of the keys each, and walks the keys in steps of 64.  fp32 values are three bf16 terms
// (attn24.cuh), so q and p take part exactly; bf16 pages are one term, fp32 pages three: 3 or 6 passes a product.  The tensor
// cores truncate their sums, so the P V of each step starts at zero and is added to the output in registers.
//
// Warps: one issues the tensor-core instructions, two or three bring keys and values of bf16 from wherever their pages are into a ring
// (the copy engine, boxes of 8 to 64 rows that lie in one page; asynchronous 16-byte copies where pages are not a multiple of 8 rows),
// sixteen do the softmax and, of fp32 pages, bring keys and values through registers, split on the way (three warps for that alone took
// 4000 cycles a step).  Where a step takes the tensor cores as long as a softmax step or
// longer (1536 cycles and more: fp32, or head sizes above 64) four threads share a row and two score buffers alternate; else (768
// cycles) two threads do, and two groups of eight warps take every other step each, with a maximum, sum and output of their own that
// are joined at the end, and three score buffers, so that a group finds its next scores when it has done with one step (with two
// buffers S of step n+2 had to wait for P V of step n, and a step took 1430 cycles).
//
// 3380 new tokens of sequences of up to 8024 positions, 12 heads of 64, bf16: 213 us, a step 1200 cycles, bound by the softmax warps'
// instructions (61 % of issue slots; tensor pipe 62 %).  2048 new tokens, 25 heads of 64, fp32: 60 us, short units, start and end.
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

template <class T, int kDP, bool kTma>
struct Shape {
    static constexpr bool kWide = sizeof(T) == 4;          // fp32 pages
    static constexpr int kTerms = kWide ? 3 : 1;           // of K and V
    static constexpr int kGroups = !kWide && kDP == 64 ? 2 : 1;
    static constexpr int kSplit = 4 / kGroups;             // threads of a row
    static constexpr int kGroupWarps = 4 * kSplit;
    static constexpr int kProducers = 3;                   // warps 1 to 3; warp 0 issues
    static constexpr int kFirst = kProducers + 1;          // first softmax warp, a multiple of four
    static constexpr int kThreads = 32 * (kFirst + 16);
    static constexpr int kPlane = kStep * kDP * 2;         // one term of 64 keys
    static constexpr int kStage = 2 * kTerms * kPlane;     // K terms, V terms
    static constexpr int kStages = kWide ? (kDP == 64 ? 4 : 2) : (kDP == 64 ? 8 : 6);
    static constexpr int kLead = kWide ? kStages / 2 : 0;  // steps that the softmax warps are ahead with fp32 keys and values
    static constexpr int kBuffers = kGroups + 1;           // of scores, 96 columns each
    static constexpr uint32_t kColO = 96 * kBuffers, kColQ = kColO + kGroups * kDP;  // an output for each group
    static_assert(kColQ + 3 * kDP / 2 <= 512, "tensor memory");
};

template <class T, int kDP, bool kTma>
struct __align__(1024) TileSmem {
    using S = Shape<T, kDP, kTma>;
    union {
        uint8_t ring[S::kStages][S::kStage];
        struct {  // at the end
            float o[kRowsTile][kDP + 4];
            float o1[kRowsTile][kDP + 4];
        } fin;
    };
    uint64_t kv_full[S::kStages], kv_empty[S::kStages], s_full[3], p_full[2], o_full[2], q_ready, tail[2];
    uint32_t valid[S::kStages][2];          // keys of the stage that are there
    uint8_t nibble[S::kStages][16];         // fp32 pages: of the four rows of each warp
    float xmax[S::kGroups][2][S::kSplit][kRowsTile];  // [group][step parity][part][row]: maxima, at the end sums
    float m[kRowsTile], l[kRowsTile], m1[kRowsTile], l1[kRowsTile];
    uint32_t odd[kRowsTile / 32];           // rows to be computed again
    int seq, tile;
    Span span;
    uint32_t tmem_base;
    int abort_flag;
};

enum Site : int { SITE_KV_EMPTY = 401, SITE_KV_FULL, SITE_S_FULL, SITE_P_FULL, SITE_O_FULL, SITE_Q_READY, SITE_ALIGN, SITE_TAIL };

// The sequence and tile of unit `u`, tiles counted over the sequences with more than `few` rows and no more new tokens than max_new;
// tile -1 past the last.  Up to 64 sequences are taken in the order of falling length (32 at a time), and the tiles of each from its last, so
// that the longest units begin first and the shortest fill the end.  A whole warp.  check: reports lengths that the call does not allow.
__device__ __forceinline__ void find_tile(const Cache &c, int G, int few, int max_new, int u, bool check, int *status, int &seq, int &tile) {
    const int lane = threadIdx.x & 31;
    seq = 0, tile = -1;
    for (int base = 0; base < c.seqs; base += 32) {
        const int s = base + lane;
        int tiles = 0, length = 0;
        if (s < c.seqs) {
            const Span w = span_of(c, s);
            const bool good = w.count <= max_new && w.past >= 0;
            if (check && w.count > 0 && (!good || w.past + (long long)w.count > (long long)c.width * c.page_size)) report(status, ST_ATTEND);
            const long long rows = (long long)w.count * G;
            tiles = good && rows > few ? (int)((rows + kRowsTile - 1) / kRowsTile) : 0;
            length = w.past + w.count;
        }
        int before = 0, all = 0;  // tiles in front of this lane's
        if (c.seqs <= 64) {
            for (int j = 0; j < min(32, c.seqs - base); j++) {
                const int other = __shfl_sync(0xffffffffu, tiles, j), longer = __shfl_sync(0xffffffffu, length, j);
                before += longer > length || (longer == length && j < lane) ? other : 0;
                all += other;
            }
        } else {
            int run = tiles;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int left = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += left;
            }
            before = run - tiles, all = __shfl_sync(0xffffffffu, run, 31);
        }
        const uint32_t mine = __ballot_sync(0xffffffffu, u >= before && u < before + tiles);
        if (mine != 0) {
            const int at = __ffs(mine) - 1;
            seq = base + at;
            tile = __shfl_sync(0xffffffffu, before + tiles, at) - 1 - u;
            if (!check) return;
            u = 0x7fffffff;  // only the check goes on
        }
        u -= all;
    }
}

template <class T, int kDP, bool kTma>
__global__ void __launch_bounds__(Shape<T, kDP, kTma>::kThreads, 1)
tile_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, int box, Cache c, const float *q, float *out, long long ld, int heads,
            int few, int max_new, float scale_log2, int whole, int *status) {
    using Sh = Shape<T, kDP, kTma>;
    using Smem = TileSmem<T, kDP, kTma>;
    constexpr int kK = kDP / 16, kStages = Sh::kStages, kPlane = Sh::kPlane, kGroups = Sh::kGroups;
    constexpr int kBuffers = Sh::kBuffers, kTerms = Sh::kTerms, kSplit = Sh::kSplit, kPart = kDP / kSplit;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Smem &sm = *reinterpret_cast<Smem *>(smem_raw);
    cg::cluster_group cluster = cg::this_cluster();
    const int size = (int)cluster.num_blocks(), which = (int)blockIdx.x / size;
    const bool alone = which * size < whole;  // the first `whole` units have a CTA each, the others a cluster
    const int ranks = alone ? 1 : size, rank = alone ? 0 : (int)cluster.block_rank();
    const int warp = __shfl_sync(0xffffffffu, (int)(threadIdx.x >> 5), 0), lane = threadIdx.x & 31;
    const int unit = alone ? (int)blockIdx.x : whole + which - whole / size, kvh = unit % c.kv_heads, G = heads / c.kv_heads;
    WaitCtx ctx{&sm.abort_flag, status};
    if (threadIdx.x == 0) {
        if ((smem_u32(smem_raw) & 1023u) != 0) report(status, ST_TIMEOUT_BASE + SITE_ALIGN);
        sm.abort_flag = 0;
        for (int i = 0; i < kStages; i++) {
            mbar_init(&sm.kv_full[i], kTma ? 4 : Sh::kWide ? 16 : 32 * Sh::kProducers + 1);
            mbar_init(&sm.kv_empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.p_full[i], Sh::kGroupWarps);
            mbar_init(&sm.o_full[i], 1);
            mbar_init(&sm.tail[i], 1);
        }
        for (int i = 0; i < 3; i++) mbar_init(&sm.s_full[i], 1);
        mbar_init(&sm.q_ready, 16);
        fence_barrier_init();
    }
    if (kTma && threadIdx.x == 64) {
        tma_prefetch_desc(&map_k);
        tma_prefetch_desc(&map_v);
    }
    if (warp == 1) tmem_alloc_then_launch_dependents(&sm.tmem_base, 512);
    pdl_wait();
    if (warp == 0) {
        int seq, tile;
        const int u = unit / c.kv_heads;
        find_tile(c, G, few, max_new, u, u == 0 && kvh == 0 && rank == 0, status, seq, tile);
        const Span span = span_of(c, seq);
        if (lane == 0) sm.seq = seq, sm.tile = tile, sm.span = span;
    }
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem_base, 0);
    const int seq = __shfl_sync(0xffffffffu, sm.seq, 0), tile = __shfl_sync(0xffffffffu, sm.tile, 0);
    const Span w = sm.span;
    const int rows = w.count * G, row0 = tile * kRowsTile;
    const int *table = c.table + (long long)seq * c.width;
    // this CTA's run of keys: steps first .. first + nsteps - 1
    const int last = (min(row0 + kRowsTile, rows) - 1) / G;
    const int keys = tile < 0 ? 0 : (int)min((long long)w.past + last + 1, (long long)c.width * c.page_size);
    const int all = (keys + kStep - 1) / kStep, each = (all + ranks - 1) / ranks, first = min(rank * each, all), nsteps = min(each, all - first);
    // new token and head of a row
    auto token_of = [&](int at) { return G == 1 ? at : at / G; };
    auto head_of = [&](int at) { return kvh * G + (G == 1 ? 0 : at % G); };
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
            fence_proxy_async_smem();  // here, not where they are written: there it would wait for everything that is on its way
            const uint64_t at = desc_advance(kd, st * Sh::kStage);
#pragma unroll
            for (int i = 0; i < kPasses; i++)
#pragma unroll
                for (int kk = 0; kk < kK; kk++)
                    mma_ts_lead(leader, tmem + n % kBuffers * 96, tmem + Sh::kColQ + kDP / 2 * term_a(i) + 8 * kk,
                                desc_advance(at, term_b(i) * kPlane + (kk >> 2) * (kStep * 128) + (kk & 3) * 32), idesc_s, i > 0 || kk > 0 ? 1u : 0u);
            tc_commit_lead(leader, &sm.s_full[n % kBuffers]);
        };
        await(&sm.q_ready, 0, ctx, SITE_Q_READY);
        for (int n = 0; n < min(kBuffers, nsteps); n++) issue_s(n);
        for (int n = 0; n < nsteps; n++) {
            const int st = n % kStages;
            await(&sm.p_full[n & 1], (n >> 1) & 1, ctx, SITE_P_FULL);
            const uint64_t at = desc_advance(vd, st * Sh::kStage);
#pragma unroll
            for (int i = 0; i < kPasses; i++)
#pragma unroll
                for (int kk = 0; kk < kStep / 16; kk++)
                    mma_ts_lead(leader, tmem + Sh::kColO + n % kGroups * kDP, tmem + n % kBuffers * 96 + term_column(term_a(i), kk), desc_advance(at, term_b(i) * kPlane + kk * 2048),
                                idesc_o, i > 0 || kk > 0 ? 1u : 0u);
            tc_commit_lead(leader, &sm.o_full[n & 1]);
            tc_commit_lead(leader, &sm.kv_empty[st]);
            if (n + kBuffers < nsteps) issue_s(n + kBuffers);  // where P_n was, which P V of step n, earlier in the pipe, has read by then
        }
    } else if (kTma && nsteps > 0 && (warp == 2 || warp == 3)) {
        // ------------------------------ producers of K and of V: boxes, one a lane ------------------------------
        // Few instructions a step: beside sixteen busy warps each of them takes this one about six cycles.
        const int boxes = kStep / box, slots = kStep / c.page_size, row_step = kStep % c.page_size;
        const uint32_t all_boxes = boxes == 32 ? 0xffffffffu : (1u << boxes) - 1u;
        bool missing = false;
        int j = first * kStep + lane * box, slot = j / c.page_size, row = j % c.page_size, row_here = row;
        auto page_of = [&] {  // of key j; -1 where there is no key
            const int page = lane < boxes && j < keys ? table[slot] : -1;
            row_here = row;
            j += kStep, slot += slots, row += row_step;
            if (row >= c.page_size) row -= c.page_size, slot++;
            return page;
        };
        int page = page_of(), at_row = row_here;  // looked up a step ahead
        const int kv = warp - 2;
        const CUtensorMap *map = kv ? &map_v : &map_k;
        uint8_t *const tile_at = sm.ring[0] + kv * kPlane, *const to = tile_at + (lane < boxes ? lane : 0) * box * 128;
        for (int n = 0; n < nsteps; n++) {
            const int st = n % kStages, here_row = at_row;
            // past the last page where there is none: that reads as zeros
            const bool wanted = lane < boxes && (first + n) * kStep + lane * box < keys, there_is = wanted && (unsigned)page < (unsigned)c.pages;
            const int here = there_is ? page : c.pages;
            missing |= wanted && !there_is;
            page = page_of(), at_row = row_here;
            if (n >= kStages) await(&sm.kv_empty[st], (n / kStages - 1) & 1, ctx, SITE_KV_EMPTY);
            const int key0 = (first + n) * kStep;
            const bool last_part = key0 + kStep > keys;
            uint64_t *bar = last_part ? &sm.tail[kv] : &sm.kv_full[st];
            const uint32_t found = __ballot_sync(0xffffffffu, there_is);
            if (lane == 0) mbar_expect_tx(bar, kPlane);
            __syncwarp();
            if (lane < boxes) {
#pragma unroll
                for (int b = 0; b < kDP / 64; b++) tma_load_4d(to + st * Sh::kStage + b * (kStep * 128), map, bar, 64 * b, here_row, kvh, here);
            }
            uint32_t there[2] = {0xffffffffu, 0xffffffffu};  // the keys of the stage that have a page
            if (found != all_boxes) {
                const uint32_t row_bits = box >= 32 ? 0xffffffffu : (1u << box) - 1u;
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    there[i] = 0;
                    for (int b = 32 * i / box; b * box < 32 * (i + 1); b++)
                        if (found >> b & 1u) there[i] |= row_bits << (b * box & 31);
                }
            }
            if (lane == 0 && kv == 0) sm.valid[st][0] = there[0], sm.valid[st][1] = there[1];
            if (last_part) {  // rows of the last page that nothing has been stored in: 0 times what they hold need not be 0
                await(&sm.tail[kv], 0, ctx, SITE_TAIL);
                for (int r = keys - key0; r < kStep; r++)
                    for (int i = lane; i < (kDP / 64) * 8; i += 32)
                        *reinterpret_cast<uint4 *>(tile_at + st * Sh::kStage + (i >> 3) * (kStep * 128) + r * 128 + ((i & 7) << 4)) = make_uint4(0, 0, 0, 0);
                fence_proxy_async_smem();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sm.kv_full[st]);  // in the place of the copies' arrival
            }
            if (lane == 0) mbar_arrive(&sm.kv_full[st]);
        }
        if (missing) report(status, ST_ATTEND);
    } else if (!kTma && !Sh::kWide && nsteps > 0 && warp < Sh::kFirst) {
        // ------------------------------ producers ------------------------------
        constexpr int kChunks = kDP / 8, kPer = 32 / kChunks;  // pieces of 8 columns of a row; rows that a warp takes at once
        constexpr int kIts = 64 / kPer;                        // of a tile
        const int mine = lane / kChunks, ch = lane % kChunks, from = warp - 1;
        const bool col = 8 * ch < c.D;
        const T *kp = static_cast<const T *>(c.k) + head + (col ? 8 * ch : 0), *vp = static_cast<const T *>(c.v) + head + (col ? 8 * ch : 0);
        const uint32_t column = (ch >> 3) * (kStep * 128);
        auto spot = [&](int r) { return column + r * 128 + (((ch & 7) ^ (r & 7)) << 4); };
        bool missing = false;
        // of keys `lane` and 32 + `lane` of a step, looked up a step ahead
        long long lo = place(c, table, first * kStep + lane, keys, missing), hi = place(c, table, first * kStep + 32 + lane, keys, missing);
        if constexpr (!Sh::kWide) {
            for (int n = 0; n < nsteps; n++) {
                const int st = n % kStages, next0 = (first + n + 1) * kStep;
                const long long lo1 = place(c, table, next0 + lane, keys, missing), hi1 = place(c, table, next0 + 32 + lane, keys, missing);
                const uint32_t there0 = __ballot_sync(0xffffffffu, lo >= 0), there1 = __ballot_sync(0xffffffffu, hi >= 0);
                if (n >= kStages) await(&sm.kv_empty[st], (n / kStages - 1) & 1, ctx, SITE_KV_EMPTY);
                if (from == 0 && lane == 0) {
                    sm.valid[st][0] = there0, sm.valid[st][1] = there1;
                    mbar_arrive(&sm.kv_full[st]);
                }
                const uint32_t kt = smem_u32(sm.ring[st]), vt = kt + kPlane;
#pragma unroll
                for (int i = 0; i < (kIts + 2) / 3; i++) {
                    const int it = 3 * i + from;
                    if (it >= kIts) break;
                    const int r = it * kPer + mine;
                    const long long off = __shfl_sync(0xffffffffu, it * kPer < 32 ? lo : hi, r & 31);
                    const bool in = off >= 0 && col;
                    const uint32_t to = spot(r);
                    cp16(kt + to, kp + max(off, 0ll), in);
                    cp16(vt + to, vp + max(off, 0ll), in);
                }
                arrive_when_copied(&sm.kv_full[st]);
                lo = lo1, hi = hi1;
            }
            cp_wait<0>();
        }
        if (missing) report(status, ST_ATTEND);
    }
    float o[kPart], m = -INFINITY, l = 0.f;
    const int group = (warp - Sh::kFirst) / Sh::kGroupWarps, part = ((warp - Sh::kFirst) >> 2) % kSplit, quarter = warp & 3, row = 32 * quarter + lane;
    const uint32_t lane_addr = (uint32_t)(quarter << 5) << 16;
    const bool softmax = warp >= Sh::kFirst;
    if (softmax) {
        // ------------------------------ softmax ------------------------------
        constexpr int kCols = kStep / kSplit;  // scores of this thread
        const int at = row0 + row;
        const int seen = tile >= 0 && at < rows ? w.past + token_of(at) + 1 : 0;  // keys that this row sees
        const int all_see = __reduce_min_sync(0xffffffffu, seen);           // and every row of this warp
#pragma unroll
        for (int e = 0; e < kPart; e++) o[e] = 0.f;
        // fp32 pages: eight threads a row, each with 8 columns of every 64 of K and of V; loads of a step are under way while the one
        // before is split
        constexpr int kBlocks = kDP / 64, kLead = Sh::kLead;
        const int mine = (int)threadIdx.x - 32 * Sh::kFirst, k_row = mine >> 3, k_ch = mine & 7;
        float4 kf[Sh::kWide ? kBlocks : 1][2], vf[Sh::kWide ? kBlocks : 1][2];
        bool have = false, missing = false;
        int j = first * kStep + k_row, slot = 0, in_page = 0, page = -1;
        const int end_key = min(keys, (first + nsteps) * kStep), slots = kStep / c.page_size, page_step = kStep % c.page_size;
        auto look_up = [&] { page = j < end_key ? table[slot] : -1; };
        auto fetch = [&] {
            const bool wanted = j < end_key;
            have = wanted && (unsigned)page < (unsigned)c.pages;
            missing |= wanted && !have;
            const long long at = have ? page * c.page_stride + (long long)in_page * c.D + head + 8 * k_ch : 0;
#pragma unroll
            for (int i = 0; i < kBlocks; i++) {
                const bool in = have && 64 * i + 8 * k_ch < c.D;
                const float4 zero = make_float4(0.f, 0.f, 0.f, 0.f);
                const float4 *kp = reinterpret_cast<const float4 *>(static_cast<const float *>(c.k) + at + 64 * i);
                const float4 *vp = reinterpret_cast<const float4 *>(static_cast<const float *>(c.v) + at + 64 * i);
                kf[i][0] = in ? kp[0] : zero, kf[i][1] = in ? kp[1] : zero;
                vf[i][0] = in ? vp[0] : zero, vf[i][1] = in ? vp[1] : zero;
            }
            j += kStep, slot += slots, in_page += page_step;
            if (in_page >= c.page_size) in_page -= c.page_size, slot++;
            look_up();
        };
        auto put = [&](int n) {  // into the stage of step n
            uint8_t *to = sm.ring[n % kStages] + k_row * 128 + ((k_ch ^ (k_row & 7)) << 4);
#pragma unroll
            for (int i = 0; i < kBlocks; i++)
#pragma unroll
                for (int kv = 0; kv < 2; kv++) {
                    const float4 x = kv ? vf[i][0] : kf[i][0], y = kv ? vf[i][1] : kf[i][1];
                    uint32_t h[4], m[4], l[4];
                    cut3(make_float2(x.x, x.y), h[0], m[0], l[0]);
                    cut3(make_float2(x.z, x.w), h[1], m[1], l[1]);
                    cut3(make_float2(y.x, y.y), h[2], m[2], l[2]);
                    cut3(make_float2(y.z, y.w), h[3], m[3], l[3]);
                    uint8_t *at = to + kv * kTerms * kPlane + i * (kStep * 128);
                    *reinterpret_cast<uint4 *>(at) = make_uint4(h[0], h[1], h[2], h[3]);
                    *reinterpret_cast<uint4 *>(at + kPlane) = make_uint4(m[0], m[1], m[2], m[3]);
                    *reinterpret_cast<uint4 *>(at + 2 * kPlane) = make_uint4(l[0], l[1], l[2], l[3]);
                }
            const uint32_t rows4 = __ballot_sync(0xffffffffu, have);
            __syncwarp();  // lane 0 arrives for what all lanes have stored
            if (lane == 0) {
                sm.nibble[n % kStages][mine >> 5] = (uint8_t)((rows4 & 1) | (rows4 >> 7 & 2) | (rows4 >> 14 & 4) | (rows4 >> 21 & 8));
                mbar_arrive(&sm.kv_full[n % kStages]);
            }
        };
        if (Sh::kWide && nsteps > 0) {
            slot = j / c.page_size, in_page = j % c.page_size;
            look_up();
            fetch();
        }
        if (nsteps > 0) {
            constexpr int kShare = kDP / 4;  // columns of Q for each thread of a row, of both groups
            const int from = (group * kSplit + part) * kShare;
            const float *src = q + (w.first + token_of(at)) * ld + (long long)head_of(at) * c.D + from;
            uint32_t x[3][kShare / 2];
#pragma unroll
            for (int e = 0; e < kShare; e += 4) {
                float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
                if (at < rows && from + e < c.D) v = *reinterpret_cast<const float4 *>(src + e);
                cut3(make_float2(v.x * scale_log2, v.y * scale_log2), x[0][e / 2], x[1][e / 2], x[2][e / 2]);
                cut3(make_float2(v.z * scale_log2, v.w * scale_log2), x[0][e / 2 + 1], x[1][e / 2 + 1], x[2][e / 2 + 1]);
            }
#pragma unroll
            for (int i = 0; i < 3; i++) {
                const uint32_t to = tmem + lane_addr + Sh::kColQ + kDP / 2 * i + from / 2;
                if constexpr (kShare == 16) tmem_st8(to, x[i]);
                else tmem_st16(to, x[i]);
            }
            tmem_wait_st();
            arrive_tmem(&sm.q_ready, lane);
        }
        if (Sh::kWide) {
            for (int n = 0; n < min(kLead, nsteps); n++) {
                put(n);
                fetch();
            }
        }
        const uint32_t t_o = tmem + lane_addr + Sh::kColO + group * kDP + part * kPart;
        auto add_output = [&](int n, float by) {
            await(&sm.o_full[n & 1], (n >> 1) & 1, ctx, SITE_O_FULL);
            const float2 by2 = make_float2(by, by);
#pragma unroll
            for (int b = 0; b < kPart; b += 16) {
                uint32_t r[16];
                tmem_ld16(t_o + b, r);
                tmem_wait_ld();
#pragma unroll
                for (int e = 0; e < 16; e += 2) {
                    const float2 sum = fma2(make_float2(o[b + e], o[b + e + 1]), by2, make_float2(__uint_as_float(r[e]), __uint_as_float(r[e + 1])));
                    o[b + e] = sum.x, o[b + e + 1] = sum.y;
                }
            }
        };
        float alpha_before = 1.f;
        for (int n = group; n < nsteps; n += kGroups) {
            const int st = n % kStages, key0 = (first + n) * kStep + kCols * part;
            const uint32_t t_s = tmem + lane_addr + n % kBuffers * 96;
            await(&sm.s_full[n % kBuffers], (n / kBuffers) & 1, ctx, SITE_S_FULL);
            if (Sh::kWide && kLead == 1) {  // two stages: the other one is free when P V of the step before has been added up
                if (n > 0) add_output(n - 1, alpha_before);
                if (n + 1 < nsteps) {
                    __syncwarp();
                    put(n + 1);
                    fetch();
                }
            }
            uint32_t s[kCols];
            if constexpr (kCols == 32) tmem_ld32(t_s + kCols * part, s);
            else tmem_ld16(t_s + kCols * part, s);
            // what the warps that brought the keys say of them: it was there before the scores were asked for
            uint32_t there;
            if constexpr (Sh::kWide) {
                const uint32_t n4 = *reinterpret_cast<const uint32_t *>(&sm.nibble[st][4 * part]);
                there = (n4 & 0xf) | (n4 >> 4 & 0xf0) | (n4 >> 8 & 0xf00) | (n4 >> 12 & 0xf000);
            } else {
                there = sm.valid[st][part * kCols / 32] >> (part * kCols % 32);
            }
            const uint32_t full = kCols == 32 ? 0xffffffffu : (1u << (kCols & 31)) - 1u;
            tmem_wait_ld();
            if ((first + n + 1) * kStep > all_see || (there & full) != full) {
                const int lim = seen - key0;
                const uint32_t bits = there & (lim >= 32 ? 0xffffffffu : lim <= 0 ? 0u : (1u << lim) - 1u);
#pragma unroll
                for (int e = 0; e < kCols; e++)
                    if (!(bits >> e & 1u)) s[e] = 0xff800000u;  // -inf
            }
            float mx = -INFINITY;
#pragma unroll
            for (int e = 0; e < kCols; e += 2) mx = max3(mx, __uint_as_float(s[e]), __uint_as_float(s[e + 1]));
            const int par = (n / kGroups) & 1;
            sm.xmax[group][par][part][row] = mx;
            named_sync(1 + 4 * group + quarter, 32 * kSplit);
            if constexpr (kSplit == 2) mx = max3(m, mx, sm.xmax[group][par][part ^ 1][row]);
            else mx = fmaxf(m, fmaxf(max3(sm.xmax[group][par][0][row], sm.xmax[group][par][1][row], sm.xmax[group][par][2][row]), sm.xmax[group][par][kSplit - 1][row]));
            const float base = mx == -INFINITY ? 0.f : mx;  // nothing but -inf so far
            const float alpha = ex2f(m - base);
            m = mx;
            const float2 minus = make_float2(-base, -base);
            float2 sum = make_float2(0.f, 0.f);
#pragma unroll
            for (int b = 0; b < kCols / 16; b++) {  // 16 columns make 8 of each term
                uint32_t hi[8], rest[16];  // mid and lo lie side by side
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const float2 x = add2(make_float2(__uint_as_float(s[16 * b + 2 * e]), __uint_as_float(s[16 * b + 2 * e + 1])), minus);
                    const float2 p = make_float2(ex2f(x.x), ex2f(x.y));
                    sum = add2(sum, p);
                    cut3(p, hi[e], rest[e], rest[8 + e]);
                }
                tmem_st8(t_s + term_column(0, part * (kCols / 16) + b), hi);
                tmem_st16(t_s + term_column(1, part * (kCols / 16) + b), rest);
            }
            l = l * alpha + (sum.x + sum.y);
            tmem_wait_st();
            // this group's output is free for the next P V
            if (n >= kGroups && !(Sh::kWide && kLead == 1)) add_output(n - kGroups, alpha_before);
            alpha_before = alpha;
            arrive_tmem(&sm.p_full[n & 1], lane);
            if (Sh::kWide && kLead == 2 && n + 2 < nsteps) {  // four stages: that of step n - 2, which has been added up
                put(n + 2);
                fetch();
            }
        }
        if (missing) report(status, ST_ATTEND);
        if (nsteps > group) add_output(nsteps - 1 - (nsteps - 1 - group) % kGroups, alpha_before);
        // each part's share of the sum; the step that last used this parity is behind a barrier that all have passed
        named_sync(1 + 4 * group + quarter, 32 * kSplit);
        sm.xmax[group][0][part][row] = l;
    }
    if (sm.abort_flag) __nanosleep(50000);  // let products that are still in flight end
    if (threadIdx.x < kRowsTile / 32) sm.odd[threadIdx.x] = 0;
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    if (warp == 1) tmem_dealloc(tmem, 512);  // before anything that waits for the other CTAs of the cluster
    if (tile >= 0) {
        if (softmax) {
            l = 0.f;
#pragma unroll
            for (int i = 0; i < kSplit; i++) l += sm.xmax[group][0][i][row];
            if (kGroups == 2 && group == 1) {
#pragma unroll
                for (int e = 0; e < kPart; e += 4)
                    *reinterpret_cast<float4 *>(&sm.fin.o1[row][part * kPart + e]) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                if (part == 0) sm.m1[row] = m, sm.l1[row] = l;
            }
        }
        if (kGroups == 2) __syncthreads();
        if (softmax && group == 0) {
            if (kGroups == 2) {
                const float mo = sm.m1[row], top = fmaxf(m, mo), base = top == -INFINITY ? 0.f : top, a = ex2f(m - base), b = ex2f(mo - base);
#pragma unroll
                for (int e = 0; e < kPart; e++) o[e] = o[e] * a + sm.fin.o1[row][part * kPart + e] * b;
                l = l * a + sm.l1[row] * b;
                m = top;
            }
            float zero = l * 0.f;  // what is finite times zero is zero
#pragma unroll
            for (int e = 0; e < kPart; e++) zero = fmaf(o[e], 0.f, zero);
#pragma unroll
            for (int e = 0; e < kPart; e += 4)
                *reinterpret_cast<float4 *>(&sm.fin.o[row][part * kPart + e]) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
            if (part == 0) sm.m[row] = m, sm.l[row] = l;
            const uint32_t odd = __ballot_sync(0xffffffffu, !(zero == 0.f) && row0 + row < rows);
            if (lane == 0 && odd) atomicOr(&sm.odd[quarter], odd);
        }
        __syncthreads();
        if (sm.odd[0] | sm.odd[1] | sm.odd[2] | sm.odd[3]) {
            for (int r = warp; r < kRowsTile; r += Sh::kThreads / 32) {
                if (!(sm.odd[r >> 5] >> (r & 31) & 1u)) continue;
                const int at = row0 + r;
                exact_row<T, kDP>(c, q + (w.first + token_of(at)) * ld + (long long)head_of(at) * c.D, table, kvh, first * kStep,
                                  min(min((first + nsteps) * kStep, keys), w.past + token_of(at) + 1), scale_log2, sm.fin.o[r], &sm.m[r], &sm.l[r]);
            }
        }
        if (ranks > 1) cluster.sync();
        else __syncthreads();
        // rows rank, rank + ranks, .. of all CTAs' parts; 16 or 32 threads a row
        constexpr int kWords = kDP / 4;
        const int per = Sh::kThreads / kWords, word = threadIdx.x % kWords;
        for (int r = rank + ranks * (int)(threadIdx.x / kWords); r < kRowsTile && row0 + r < rows; r += ranks * per) {
            float sum = 0.f;
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
            if (ranks == 1) {
                sum = sm.l[r], acc = *reinterpret_cast<const float4 *>(&sm.fin.o[r][4 * word]);
            } else {
                float m_of[8], l_of[8], top = -INFINITY;
                float4 v[8];
#pragma unroll
                for (int k = 0; k < 8; k++) {  // all asked for before the first is used
                    m_of[k] = -INFINITY, l_of[k] = 0.f, v[k] = acc;
                    if (k < ranks) {
                        const Smem &p = *cluster.map_shared_rank(&sm, k);
                        m_of[k] = p.m[r], l_of[k] = p.l[r], v[k] = *reinterpret_cast<const float4 *>(&p.fin.o[r][4 * word]);
                    }
                }
#pragma unroll
                for (int k = 0; k < 8; k++) top = fmaxf(top, m_of[k]);
                const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const float by = ex2f(m_of[k] - base);
                    sum = fmaf(l_of[k], by, sum);
                    acc = make_float4(fmaf(v[k].x, by, acc.x), fmaf(v[k].y, by, acc.y), fmaf(v[k].z, by, acc.z), fmaf(v[k].w, by, acc.w));
                }
            }
            const int at = row0 + r;
            const float by = sum == 0.f ? 0.f : 1.f / sum;
            if (4 * word < c.D)
                *reinterpret_cast<float4 *>(out + ((long long)(w.first + token_of(at)) * heads + head_of(at)) * c.D + 4 * word) =
                    make_float4(acc.x * by, acc.y * by, acc.z * by, acc.w * by);
        }
        if (ranks > 1) cluster.sync();  // shared memory of the others is read until here
    }
}

template <class T, int kDP, bool kTma>
cudaError_t launch_tile(const Call &a, int few, const CUtensorMap &k, const CUtensorMap &v, int box) {
    using Sh = Shape<T, kDP, kTma>;
    const int G = a.heads / a.c.kv_heads, sms = attn::sm_count();
    const long long units = (long long)a.c.tokens * G / kRowsTile + a.c.seqs;
    const long long all = units * a.c.kv_heads;
    if (all > 0x7fffffffll / 8) return cudaErrorInvalidConfiguration;
    // What is left behind full rounds of one unit an SM, where that is less than half a round, would hold a few SMs for as long as a full
    // one: those units, the shortest, are shared by two CTAs each, the others taken by one (324 units of up to 126 steps: 228 us without,
    // 213 so; in short bursts of calls 204, 182, and 207 with clusters of four, of which fewer fit the GPU).
    const int rest = (int)(all % sms);
    unsigned ranks = 1;
    int whole = 0;
    if (all < sms) {
        while (ranks < 8 && all * ranks * 2 <= sms) ranks *= 2;  // few units share their keys among the SMs that are left
    } else if (rest != 0 && 2 * rest <= sms) {
        ranks = 2;
        whole = (int)all - rest;
        whole -= whole % ranks;
    }
    const long long ctas = whole + (all - whole) * ranks;
    return attn::launch_clusters_after_previous(tile_kernel<T, kDP, kTma>, dim3((unsigned)ctas), dim3(Sh::kThreads), sizeof(TileSmem<T, kDP, kTma>), ranks, a.s, k, v,
                                                box, a.c, a.q, a.out, a.ld, a.heads, few, a.max_new, a.scale_log2, whole, a.status);
}

// Pages as a map {D, rows of a page, heads, pages}, boxes of 64 columns by `box` rows; columns past the D-th read as zeros.
int pages_map(CUtensorMap *map, const Cache &c, const void *base, int box) {
    const cuuint64_t dims[4] = {(cuuint64_t)c.D, (cuuint64_t)c.page_size, (cuuint64_t)c.kv_heads, (cuuint64_t)c.pages};
    const cuuint64_t strides[3] = {(cuuint64_t)c.D * 2, (cuuint64_t)c.D * 2 * c.page_size, (cuuint64_t)c.page_stride * 2};
    const cuuint32_t boxes[4] = {64, (cuuint32_t)box, 1, 1};
    return attn::encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, base, dims, strides, boxes);
}

template <int kDP>
cudaError_t launch_narrow(const Call &a, int few) {
    const int box = kStep < (a.c.page_size & -a.c.page_size) ? kStep : a.c.page_size & -a.c.page_size;  // the largest power of two in the page size
    CUtensorMap k{}, v{};
    if (box < 8 || a.c.page_stride >= 1ll << 39 || pages_map(&k, a.c, a.c.k, box) != 0 || pages_map(&v, a.c, a.c.v, box) != 0)
        return launch_tile<__nv_bfloat16, kDP, false>(a, few, k, v, 0);
    return launch_tile<__nv_bfloat16, kDP, true>(a, few, k, v, box);
}

template <class T, int kDP, bool kTma>
cudaError_t set_one() {
    return cudaFuncSetAttribute(tile_kernel<T, kDP, kTma>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(TileSmem<T, kDP, kTma>));
}

}  // namespace

cudaError_t launch_tiles(const Call &a, int few) {
    if (a.type == ATTN_CACHE_BF16) return a.c.D <= 64 ? launch_narrow<64>(a, few) : launch_narrow<128>(a, few);
    const CUtensorMap none{};
    return a.c.D <= 64 ? launch_tile<float, 64, false>(a, few, none, none, 0) : launch_tile<float, 128, false>(a, few, none, none, 0);
}

cudaError_t tiles_set_attributes() {
    cudaError_t e = set_one<__nv_bfloat16, 64, true>();
    if (e == cudaSuccess) e = set_one<__nv_bfloat16, 64, false>();
    if (e == cudaSuccess) e = set_one<__nv_bfloat16, 128, true>();
    if (e == cudaSuccess) e = set_one<__nv_bfloat16, 128, false>();
    if (e == cudaSuccess) e = set_one<float, 64, false>();
    if (e == cudaSuccess) e = set_one<float, 128, false>();
    return e;
}

}  // namespace paged
