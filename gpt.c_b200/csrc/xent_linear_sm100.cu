// The vocabulary projection with the cross-entropy of its rows, and their gradients, without the logits in memory, for sm_100a.
//
//     z = x w^T             lse_r = log sum_v exp z_rv             loss_r = lse_r - z_r,t(r)
//     G_rv = g_r (exp(z_rv - lse_r) - [v = t(r)])        dx = G w        dw += G^T x
//
// Forward: tiles of z are made in tensor memory and read once, for a maximum and a sum of exponentials of each row of the tile; a
// second kernel joins them over the tiles of a row.
// Backward: z is made again, a piece of the vocabulary at a time, and leaves its tile as G, in bf16, to a buffer that the two products
// read.  The launch that makes the products of a piece also makes G of the next one, so its tail is filled with short tiles.
//
// All three products go through one loop over tiles of 256 x 256 and contraction blocks of 64:
//     z   A: x,  contraction contiguous    B: w, contraction contiguous
//     dx  A: G,  contraction contiguous    B: w, columns contiguous
//     dw  A: G,  rows contiguous           B: x, columns contiguous
// fp32 operands are two bf16 planes, hi and lo (16 bits, 2^-18 of a value is left), and a product is hi hi + hi lo + lo hi: four tiles of a
// contraction block serve three products.  Six products of three planes would have all 24 bits in twice the time, TF32 operands
// 11 bits in two thirds of it.  fp32 sums of dx and dw leave the tensor cores, which truncate every sum, after 16 blocks, and what that takes on average is put back (cut_of).  With bf16 operands G is rounded
// to bf16 like the activations and gradients around it, without the factor that its rows share (common_of), which the sums take; they stay fp32 until one rounding at the end.
//
// A CTA has a tile of 256 x 256 in two accumulators of 128 rows: shared memory takes in 64 KB a block and hands out 96 in 1280 cycles, against
// 1024 of the tensor cores.  (Two CTAs on a tile would take in half of B each; pairs have stopped for good on this GPU and are not used.)
//
// Warp 0 hands out items (from a counter in the backward, longest first) and asks for tiles, warp 1 issues the products, the others take the sums out.
// The waits on barriers are bounded (tc05.cuh); the allocation of tensor memory and the wait for the previous kernel end for the reasons given there.
//
// Bound by the power limit where rows are many: 8192 x 768 x 50257 bf16, forward 475 to 510 us (1240 to 1330 TFLOP/s at 1.55 GHz, 1 kW), backward 1740 to 1850
// (three products with z made again: 1025 to 1090; the GPU's sustained rate for one matrix product is 1389); 4096 rows fp32 730 and 2580 to 2740 us (three
// times the products: 1300, 1040 to 1100).  The backward moves 700 MB of G and dw a piece besides, and the launches of the first and last piece have z or products
// alone, whose tensor cores are busy for 53 % of the time instead of 66 %.  Few rows wait for their operands: 40 rows bf16 23 to 26 and 98 us, where reading and writing takes 12 and 47.
#include <cuda_bf16.h>

#include <algorithm>
#include <type_traits>

#include "tc05.cuh"
#include "xent_linear.cuh"

#include "../../include/xent_sm100.h"

namespace head {
namespace {

using namespace tc05;

constexpr int kTile = 256, kBlock = 64;
constexpr int kEpiWarps = 16, kThreads = 32 * (2 + kEpiWarps);
constexpr int kSlotBytes = kTile * kBlock * 2;
constexpr int kQueue = 4;
constexpr int kSegment = 16;           // contraction blocks of fp32 operands that one sum in tensor memory takes
constexpr float kLog2e = 1.4426950408889634f;

enum Site : int { SITE_EMPTY = 301, SITE_FULL, SITE_ACC_EMPTY, SITE_ACC_FULL, SITE_ITEM, SITE_ITEM_FREE, SITE_PART_FULL, SITE_PART_EMPTY, SITE_SMEM_ALIGN };
enum Kind : int { kLogits, kDx, kDw };

template <int kSlots, bool kBackward>
struct __align__(1024) Smem {
    uint8_t slot[kSlots][kSlotBytes];
    float2 part[kBackward ? 1 : 2][kBackward ? 1 : 3][kBackward ? 1 : 128];  // maximum and sum of a row in three quarters of a tile
    uint64_t full[kSlots], empty[kSlots];
    uint64_t acc_full[2], acc_empty[2];
    uint64_t item_full[kQueue], item_empty[kQueue];
    uint64_t part_full[2][4], part_empty[2][4];  // of each quarter of the lanes
    int item[kQueue];
    uint32_t tmem_base;
    int abort_flag;
};

struct Maps {
    CUtensorMap x, w;      // boxes of 64 contraction steps x 128 rows, x a tile's width
    CUtensorMap x_mn, w_mn;  // boxes of 64 columns x 64 contraction steps
    CUtensorMap g, g_mn;   // the piece whose products are made, like x and like x_mn
    CUtensorMap dw;        // boxes of 256 columns x 64 rows, where p.fetch_dw
};

struct Problem {
    int M, V, K;
    int tiles_m, tiles_k;         // tiles of the rows of x, of its columns
    int dx, dw, total;            // work items: dx, dw, z; those with the longest contraction of dx and dw first
    int dw_first;
    int dx_pieces, dx_blocks;     // pieces of the contraction of dx, blocks of each
    int blocks_m, blocks_k;       // contraction blocks over the rows, over the columns of x
    int v0, cols;                 // the piece of the vocabulary whose products are made
    int next_v0, next_cols;       // the piece whose z is made, in tiles of `wide` columns (a multiple of 16)
    int wide;
    int first;                    // the first piece: what dx holds is not added to
    int pitch;                    // columns of a row of G
    long long plane;              // elements from the hi to the lo plane of G
    Ids targets;
    const float *g, *lse;
    int one_g;
    __nv_bfloat16 *out;           // G of the next piece
    float *dxp;                   // [dx_pieces, M, dx_pitch]
    long long dx_pitch;
    void *dw_out;
    long long lddw;
    int fetch_dw;                 // a tile of dw is asked for into L2 when its item is handed out
    int dw_wide;                  // bytes that the rows of dw allow at a time: 32, 16, or (0) an element
    float2 *part;                 // forward: [tiles of V, M]
    float *zt;                    // forward: the target's logit
    int *counter;                 // items are handed out (else round robin)
    float fix, log2e;             // z as the tensor cores leave it times `fix` is z; fix * log2(e)
    float fix_g;                  // of G, which makes up for what the sums of dw lose
    const float *common;          // bf16: what the sums of dx and dw are multiplied by, and what G is (common_of)
    int loaded;                   // forward: items whose operands are asked for, all but in a test of the waits
};

struct Item {
    int kind, m0, n0, n, halves;   // n: columns, a multiple of 16
    int blocks, block0;            // contraction blocks, and where they begin
    int piece;
};

template <bool kBackward>
__device__ __forceinline__ Item decode(const Problem &p, int w) {
    Item it;
    int rows, cols;
    it.block0 = 0;
    it.piece = 0;
    if (kBackward && p.dw_first && w < p.dx + p.dw) w = w < p.dw ? p.dx + w : w - p.dw;
    if (kBackward && w < p.dx) {
        it.kind = kDx;
        const int t = w / p.dx_pieces;
        it.piece = w - t * p.dx_pieces;
        it.n0 = t % p.tiles_k * kTile;
        it.m0 = t / p.tiles_k * kTile;
        rows = p.M, cols = p.K;
        it.block0 = it.piece * p.dx_blocks;
        it.blocks = min(p.dx_blocks, p.cols / kBlock - it.block0);
    } else if (kBackward && w < p.dx + p.dw) {
        it.kind = kDw;
        const int t = w - p.dx;
        it.n0 = t % p.tiles_k * kTile;
        it.m0 = t / p.tiles_k * kTile;  // in the piece
        rows = min(p.cols, p.V - p.v0), cols = p.K;
        it.blocks = p.blocks_m;
    } else {
        it.kind = kLogits;
        const int t = kBackward ? w - p.dx - p.dw : w;
        it.m0 = t % p.tiles_m * kTile;
        it.n0 = t / p.tiles_m * p.wide;  // in the piece
        rows = p.M, cols = min(p.next_cols, p.V - p.next_v0);
        it.blocks = p.blocks_k;
    }
    it.halves = rows - it.m0 > 128 ? 2 : 1;
    it.n = min(it.kind == kLogits ? p.wide : kTile, max(16, (cols - it.n0 + 15) / 16 * 16));
    return it;
}

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int c0, int c1, int c2) {
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(smem_u32(dst)), "l"(map), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

// Into L2 alone.
__device__ __forceinline__ void tma_prefetch_2d(const CUtensorMap *map, int c0, int c1) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(map), "r"(c0), "r"(c1) : "memory");
}

__device__ __forceinline__ void load8(uint32_t (&r)[8], const void *p) {
    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7])
                 : "l"(p)
                 : "memory");
}
__device__ __forceinline__ void store8(void *p, const uint32_t (&r)[8]) {
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]),
                 "r"(r[5]), "r"(r[6]), "r"(r[7])
                 : "memory");
}

// 32 sums of a row, of which `left` (more than 0) are inside, stored at `at`, 32-byte aligned.
__device__ __forceinline__ void put_f32(float *at, const uint32_t (&z)[32], int left) {
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; e++) v[e] = z[i + e];
        if (i < left) store8(at + i, v);
    }
}
// A lane has 32 columns of its row as tensor memory gives them.  Four lanes exchange blocks of eight, so that each has the same eight columns, those of
// block `lane & 3`, of all four rows (z[8 t + ..]: of row t), and an instruction touches 8 rows instead of 32, 128 bytes of each.
// (fp32 gradients of 40 x 768 x 50257 238 -> 216 us, of 4096 rows 2779 -> 2744; bf16 ones were slower, by the registers it takes.)
__device__ __forceinline__ void four_rows(int lane, uint32_t (&z)[32]) {
    const bool odd = lane & 1, high = lane & 2;
#pragma unroll
    for (int b = 0; b < 32; b += 16)
#pragma unroll
        for (int e = b; e < b + 8; e++) {
            const uint32_t got = __shfl_xor_sync(0xffffffffu, odd ? z[e] : z[e + 8], 1);
            z[e] = odd ? got : z[e];
            z[e + 8] = odd ? z[e + 8] : got;
        }
#pragma unroll
    for (int e = 0; e < 16; e++) {
        const uint32_t got = __shfl_xor_sync(0xffffffffu, high ? z[e] : z[e + 16], 2);
        z[e] = high ? got : z[e];
        z[e + 16] = high ? z[e + 16] : got;
    }
}
// A lane has 32 columns of its row; afterwards it has its column of 32 rows, so that an instruction touches one row.
__device__ __forceinline__ void transpose(int lane, uint32_t (&z)[32]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const bool up = lane & o;
#pragma unroll
        for (int e = 0; e < 32; e++) {
            if (e & o) continue;
            const uint32_t got = __shfl_xor_sync(0xffffffffu, up ? z[e] : z[e + o], o);
            z[e] = up ? got : z[e];
            z[e + o] = up ? z[e + o] : got;
        }
    }
}
// kN sums of a row added to what is there, as far as `left` goes.  One thread adds to a place, so the order of the sums is fixed; L2 adds, and nobody
// waits for what was there (loaded and stored, a half of a tile took 6 us, in which the tensor cores waited for its accumulator).
template <int kN>
__device__ __forceinline__ void add_f32(float *at, const uint32_t *z, int left) {
#pragma unroll
    for (int i = 0; i < kN; i += 4)
        if (i < left)
            asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at + i), "r"(z[i]), "r"(z[i + 1]), "r"(z[i + 2]), "r"(z[i + 3]) : "memory");
}
// The same for bf16 values, which are rounded once: 32 sums, times `by`, added to what was there, 16 words of two values.
__device__ __forceinline__ uint32_t add_bf16x2(uint32_t old, uint32_t a, uint32_t b, float by) {
    return pack_bf16x2(fmaf(__uint_as_float(a), by, __uint_as_float(old << 16)), fmaf(__uint_as_float(b), by, __uint_as_float(old & 0xffff0000u)));
}
__device__ __forceinline__ void add_bf16(__nv_bfloat16 *at, const uint32_t (&old)[16], const uint32_t (&z)[32], int left, int wide, float by) {
    if (wide == 32) {
#pragma unroll
        for (int i = 0; i < 32; i += 16) {
            if (i >= left) continue;
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; e++) v[e] = add_bf16x2(old[i / 2 + e], z[i + 2 * e], z[i + 2 * e + 1], by);
            store8(at + i, v);
        }
    } else if (wide == 16) {
#pragma unroll
        for (int i = 0; i < 32; i += 8) {
            if (i >= left) continue;
            uint4 *q = reinterpret_cast<uint4 *>(at + i);
            uint4 v = *q;
            v.x = add_bf16x2(v.x, z[i], z[i + 1], by), v.y = add_bf16x2(v.y, z[i + 2], z[i + 3], by);
            v.z = add_bf16x2(v.z, z[i + 4], z[i + 5], by), v.w = add_bf16x2(v.w, z[i + 6], z[i + 7], by);
            *q = v;
        }
    }
}
// 32 x 32 sums (of bf16 rows times `by`) added to rows of dw that start anywhere, an element at a time; `z`: the lane's column, `count` rows and `left` columns are inside.
// (With the rows that lanes have from tensor memory an instruction touched 32: forward and backward of 100 x 1001 x 50257 bf16 1407 -> 316 us, fp32 611 -> 439.)
template <class T>
__device__ __forceinline__ void add_anywhere(int lane, T *at, long long ld, const uint32_t (&z)[32], int count, int left, float by) {
    if (lane >= left) return;
    at += lane;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int r = 0; r < 32; r++)
            if (r < count) asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(at + r * ld), "r"(z[r]) : "memory");
    } else {
#pragma unroll
        for (int r = 0; r < 32; r += 8) {
            uint16_t old[8];
#pragma unroll
            for (int e = 0; e < 8; e++) old[e] = r + e < count ? *reinterpret_cast<const uint16_t *>(at + (r + e) * ld) : 0;
#pragma unroll
            for (int e = 0; e < 8; e++)
                if (r + e < count) at[(r + e) * ld] = __float2bfloat16_rn(fmaf(__uint_as_float(z[r + e]), by, __uint_as_float((uint32_t)old[e] << 16)));
        }
    }
}

// kTerms 1: bf16 operands; 3: fp32 operands as two planes.  kAnywhere: the rows of dw may start anywhere (a kernel of its own: the registers of
// both ways together spill, 60 x 768 x 50257 bf16 127 -> 147 us).
template <int kTerms, bool kBackward, int kSlots, bool kAnywhere>
__global__ void __launch_bounds__(kThreads, 1) tiles_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Problem p, int *status) {
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    using S = Smem<kSlots, kBackward>;
    S &sm = *reinterpret_cast<S *>(smem_raw);
    if ((smem_u32(smem_raw) & 1023u) != 0) {
        if (threadIdx.x == 0 && status) atomicCAS(status, 0, ST_TIMEOUT_BASE + SITE_SMEM_ALIGN);
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    constexpr int kLoads = kTerms == 1 ? 2 : 4;  // slots of a contraction block: A hi, B hi, B lo, A lo
    WaitCtx ctx{&sm.abort_flag, status, 0};
    if (threadIdx.x == 0) {
        sm.abort_flag = 0;
        for (int i = 0; i < kSlots; i++) {
            mbar_init(&sm.full[i], 1);
            mbar_init(&sm.empty[i], 1);
        }
        for (int i = 0; i < 2; i++) {
            mbar_init(&sm.acc_full[i], 1);
            mbar_init(&sm.acc_empty[i], kEpiWarps);
        }
        for (int i = 0; i < kQueue; i++) {
            mbar_init(&sm.item_full[i], 1);
            mbar_init(&sm.item_empty[i], 1 + kEpiWarps);
        }
        for (int i = 0; i < 8; i++) {
            mbar_init(&sm.part_full[i / 4][i % 4], 3);
            mbar_init(&sm.part_empty[i / 4][i % 4], 1);
        }
        fence_barrier_init();
        tma_prefetch_desc(&maps.x);
        tma_prefetch_desc(&maps.w);
    }
    if (warp == 1) tmem_alloc_then_launch_dependents(&sm.tmem_base, 512);
    pdl_wait();  // every thread, before its first access to global memory
    tc_fence_before_sync();
    __syncthreads();
    tc_fence_after_sync();
    const uint32_t tmem = sm.tmem_base;

    if (warp == 0) {
        // ------------------------------ hands out items, asks for tiles ------------------------------
        if (lane == 0) {
            int n = 0;  // slots filled
            bool ok = true;
            int w = blockIdx.x;
            for (int j = 0;; j++) {
                const int at = j % kQueue;
                if (j >= kQueue && !(ok = mbar_wait(&sm.item_empty[at], (j / kQueue - 1) & 1, ctx, SITE_ITEM_FREE))) break;
                sm.item[at] = w;
                mbar_arrive(&sm.item_full[at]);
                if (w >= p.total || (!kBackward && w >= p.loaded)) break;
                const Item it = decode<kBackward>(p, w);
                w = p.counter ? (int)gridDim.x + atomicAdd(p.counter, 1) : w + (int)gridDim.x;
                if (kBackward && it.kind == kDw && p.fetch_dw)
                    for (int r = 0; r < 128 * it.halves; r += 64) tma_prefetch_2d(&maps.dw, it.n0, p.v0 + it.m0 + r);
                const int a_boxes = 2 * it.halves, b_boxes = (it.n + 63) / 64;
                for (int b = it.block0; ok && b < it.block0 + it.blocks; b++) {
#pragma unroll
                    for (int l = 0; l < kLoads; l++, n++) {
                        const int st = n % kSlots, plane = l >= 2 ? 1 : 0;
                        const bool is_a = l == 0 || l == 3;
                        if (n >= kSlots && !mbar_wait(&sm.empty[st], (n / kSlots - 1) & 1, ctx, SITE_EMPTY)) {
                            ok = false;
                            break;
                        }
                        uint8_t *dst = sm.slot[st];
                        uint64_t *bar = &sm.full[st];
                        if (it.kind == kLogits) {
                            mbar_expect_tx(bar, (is_a ? 128 * it.halves : p.wide) * (kBlock * 2));
                            if (is_a)
                                for (int h = 0; h < it.halves; h++) tma_load_3d(dst + h * 16384, &maps.x, bar, b * kBlock, it.m0 + h * 128, plane);
                            else tma_load_3d(dst, &maps.w, bar, b * kBlock, p.next_v0 + it.n0, plane);
                        } else if (it.kind == kDx && is_a) {
                            mbar_expect_tx(bar, 16384 * it.halves);
                            for (int h = 0; h < it.halves; h++) tma_load_3d(dst + h * 16384, &maps.g, bar, b * kBlock, it.m0 + h * 128, plane);
                        } else {
                            const CUtensorMap *map = it.kind == kDx ? &maps.w_mn : is_a ? &maps.g_mn : &maps.x_mn;
                            const int boxes = is_a ? a_boxes : b_boxes, c0 = is_a ? it.m0 : it.n0, row = (it.kind == kDx ? p.v0 : 0) + b * kBlock;
                            mbar_expect_tx(bar, boxes * (kBlock * 128));
                            for (int i = 0; i < boxes; i++) tma_load_3d(dst + i * (kBlock * 128), map, bar, c0 + 64 * i, row, plane);
                        }
                    }
                }
                if (!ok) break;
            }
            if (sm.abort_flag) {  // a wait has run out: shared memory is not given up before the copies that are under way have arrived
                for (int i = max(0, n - kSlots); i < n; i++) {
                    const uint64_t t0 = global_timer_ns();
                    while (!mbar_test_wait(&sm.full[i % kSlots], (i / kSlots) & 1) && global_timer_ns() - t0 < 10000000ull) {
                    }
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------ issues the products ------------------------------
        constexpr int kLead = kTerms == 1 ? 3 : 1;
        const uint32_t leader = elect_leader();
        int st = 0, half = 0;  // next slot; halves of tiles so far
        uint32_t turn = 0;     // parity of the slots' phase
        bool ok = true;
        // The products of an item, with what its operands' layout decides known to the compiler: the descriptors of an instruction are the slot's and
        // constants (with steps known at run time alone an instruction took 230 cycles to issue, where the tensor cores take 128).
        auto products = [&](const Item &it, auto a_mn_c, auto b_mn_c) {
            constexpr bool a_mn = decltype(a_mn_c)::value, b_mn = decltype(b_mn_c)::value;
            constexpr uint32_t step_a = a_mn ? 2048 / 16 : 32 / 16, step_b = b_mn ? 2048 / 16 : 32 / 16;
            const uint32_t idesc = idesc_bf16_f32(128, it.n, a_mn, b_mn);
            const uint64_t base_a = smem_desc_sw128(smem_u32(sm.slot[0]), a_mn ? kBlock * 128 : 16, 1024);
            const uint64_t base_b = smem_desc_sw128(smem_u32(sm.slot[0]), b_mn ? kBlock * 128 : 16, 1024);
            const int seg = kTerms == 3 && kBackward && b_mn ? kSegment : it.blocks;
            for (int b0 = 0; b0 < it.blocks; b0 += seg) {
                const int b1 = min(it.blocks, b0 + seg);
                // One half's products of a block, term t, from the block's slots.
                auto issue = [&](const int (&slot)[kLoads], int t, int h, int b) {
                    const uint64_t a = base_a + (uint32_t)(slot[t == 2 ? kLoads - 1 : 0] * (kSlotBytes / 16)) + h * (16384 / 16);
                    const uint64_t bb = base_b + (uint32_t)(slot[t == 1 ? 2 % kLoads : 1] * (kSlotBytes / 16));
                    const uint32_t to = tmem + (uint32_t)((half + h) & 1) * kTile;
#pragma unroll
                    for (int k = 0; k < kBlock / 16; k++) mma_ss_lead(leader, to, a + k * step_a, bb + k * step_b, idesc, b > b0 || t > 0 || k > 0);
                    if (t == kTerms - 1 && b == b1 - 1) tc_commit_lead(leader, &sm.acc_full[(half + h) & 1]);
                };
                auto wait = [&](int &slot) {
                    slot = st;
                    if (!mbar_wait_warp(&sm.full[st], turn, ctx, SITE_FULL)) return false;
                    if (++st == kSlots) st = 0, turn ^= 1;
                    return true;
                };
                auto wait_acc = [&](int h) {
                    if (half + h >= 2 && !mbar_wait_warp(&sm.acc_empty[(half + h) & 1], ((half + h) / 2 - 1) & 1, ctx, SITE_ACC_EMPTY)) return false;
                    tc_fence_after_sync();
                    return true;
                };
                if (!wait_acc(0)) return false;
                int b = b0;
                if (it.halves == 2) {
                    // The second accumulator is still being read when the first is free (the warps that read them take one after the other), so the
                    // first half's products of kLead blocks come first.
                    int slot[kLead][kLoads];
                    const int n = min(kLead, b1 - b0);
#pragma unroll
                    for (int i = 0; i < kLead; i++) {
                        if (i >= n) break;
#pragma unroll
                        for (int l = 0; l < kLoads; l++)
                            if (!wait(slot[i][l])) return false;
                        tc_fence_after_sync();
#pragma unroll
                        for (int t = 0; t < kTerms; t++) issue(slot[i], t, 0, b0 + i);
                    }
                    if (!wait_acc(1)) return false;
#pragma unroll
                    for (int i = 0; i < kLead; i++) {
                        if (i >= n) break;
#pragma unroll
                        for (int t = 0; t < kTerms; t++) issue(slot[i], t, 1, b0 + i);
#pragma unroll
                        for (int l = 0; l < kLoads; l++) tc_commit_lead(leader, &sm.empty[slot[i][l]]);
                    }
                    b += n;
                }
                for (; b < b1; b++) {
                    int slot[kLoads];
                    if (!wait(slot[0]) || !wait(slot[1])) return false;
#pragma unroll
                    for (int t = 0; t < kTerms; t++) {
                        if (t > 0 && !wait(slot[(1 + t) % kLoads])) return false;
                        tc_fence_after_sync();
                        issue(slot, t, 0, b);
                        if (it.halves == 2) issue(slot, t, 1, b);
                        // a slot is free as soon as its last product is done: hi of A and lo of B before the third one
                        if (t == 1) tc_commit_lead(leader, &sm.empty[slot[0]]), tc_commit_lead(leader, &sm.empty[slot[2 % kLoads]]);
                        if (t == 2) tc_commit_lead(leader, &sm.empty[slot[1]]), tc_commit_lead(leader, &sm.empty[slot[kLoads - 1]]);
                        if (kTerms == 1) tc_commit_lead(leader, &sm.empty[slot[0]]), tc_commit_lead(leader, &sm.empty[slot[1]]);
                    }
                }
                half += it.halves;
            }
            return true;
        };
        for (int j = 0; ok; j++) {
            const int at = j % kQueue;
            if (!mbar_wait_warp(&sm.item_full[at], (j / kQueue) & 1, ctx, SITE_ITEM)) break;
            const int w = __reduce_max_sync(0xffffffffu, sm.item[at]);  // (the same in all lanes, in a register that the compiler knows to be)
            if (lane == 0) mbar_arrive(&sm.item_empty[at]);
            if (w >= p.total) break;
            const Item it = decode<kBackward>(p, w);
            if (!kBackward || it.kind == kLogits) ok = products(it, std::false_type{}, std::false_type{});
            else if (it.kind == kDx) ok = products(it, std::false_type{}, std::true_type{});
            else ok = products(it, std::true_type{}, std::true_type{});
        }
    } else {
        // ------------------------------ takes the sums out ------------------------------
        // A warp reads 32 rows (its quarter of tensor memory's lanes) and 64 columns of each half of a tile.
        const int quarter = warp & 3, group = (warp - 2) >> 2;
        const uint32_t from = tmem + ((uint32_t)(quarter * 32) << 16) + 64 * group;
        int half = 0;
        bool ok = true;
        for (int j = 0; ok; j++) {
            const int at = j % kQueue;
            if (!mbar_wait_warp(&sm.item_full[at], (j / kQueue) & 1, ctx, SITE_ITEM)) break;
            const int w = sm.item[at];
            __syncwarp();
            if (lane == 0) mbar_arrive(&sm.item_empty[at]);
            if (w >= p.total) break;
            const Item it = decode<kBackward>(p, w);
            const int seg = kTerms == 3 && kBackward && it.kind != kLogits ? kSegment : it.blocks;
            for (int b0 = 0; ok && b0 < it.blocks; b0 += seg) {
                for (int h = 0; h < it.halves; h++, half++) {
                    const int acc = half & 1;
                    const int row = it.m0 + h * 128 + quarter * 32 + lane, off = 64 * group;
                    int target = -1;
                    float by = kBackward && kTerms == 1 && it.kind == kDw ? p.common[0] : 0.f, nl = 0.f;  // by: what G, or sums of bf16 rows of dw, are multiplied by
                    if (it.kind == kLogits && row < p.M) {
                        target = p.targets.at(row, p.V);
                        if (kBackward) {
                            by = p.g[p.one_g ? 0 : row] * (kTerms == 1 ? p.common[1] : p.fix_g);
                            nl = -p.lse[row] * kLog2e;
                        }
                    }
                    if constexpr (!kBackward) {
                        if (!mbar_wait_warp(&sm.acc_full[acc], (half / 2) & 1, ctx, SITE_ACC_FULL)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
                        uint32_t z[64];
                        tmem_ld32(from + acc * kTile, *reinterpret_cast<uint32_t(*)[32]>(z));
                        tmem_ld32(from + acc * kTile + 32, *reinterpret_cast<uint32_t(*)[32]>(z + 32));
                        tmem_wait_ld();
                        tc_fence_before_sync();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&sm.acc_empty[acc]);
                        const int left = min(p.V - it.n0, p.wide) - off, place = target - it.n0 - off;
                        const bool here = target >= 0 && place >= 0 && place < min(64, left);
                        float top = -INFINITY, sum = 0.f;
                        if (left < 64) {
#pragma unroll
                            for (int e = 0; e < 64; e++)
                                if (e >= left) z[e] = __float_as_uint(-INFINITY);
                        }
#pragma unroll
                        for (int e = 0; e < 64; e++) top = fmaxf(top, __uint_as_float(z[e]));
                        const float nt = top == -INFINITY ? 0.f : -top * p.log2e;
                        float s[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                        for (int e = 0; e < 64; e++) s[e & 3] += ex2(fmaf(__uint_as_float(z[e]), p.log2e, nt));
                        sum = (s[0] + s[1]) + (s[2] + s[3]);
                        if (__any_sync(0xffffffffu, here)) {
#pragma unroll
                            for (int e = 0; e < 64; e++)
                                if (here && e == place) p.zt[row] = __uint_as_float(z[e]) * p.fix;
                        }
                        top *= p.fix;
                        // the four quarters of the tile's columns: the first of these warps joins them
                        const int buffer = half & 1, turn = (half / 2) & 1;
                        uint64_t *const there = &sm.part_full[buffer][quarter], *const read = &sm.part_empty[buffer][quarter];
                        if (group > 0) {
                            if (half >= 2 && !mbar_wait_warp(read, turn ^ 1, ctx, SITE_PART_EMPTY)) {
                                ok = false;
                                break;
                            }
                            sm.part[buffer][group - 1][quarter * 32 + lane] = make_float2(top, sum);
                            __syncwarp();
                            if (lane == 0) mbar_arrive(there);
                        } else {
                            if (!mbar_wait_warp(there, turn, ctx, SITE_PART_FULL)) {
                                ok = false;
                                break;
                            }
                            float2 q[4] = {make_float2(top, sum)};
#pragma unroll
                            for (int i = 0; i < 3; i++) q[i + 1] = sm.part[buffer][i][quarter * 32 + lane];
                            __syncwarp();
                            if (lane == 0) mbar_arrive(read);
                            const float m = fmaxf(fmaxf(q[0].x, q[1].x), fmaxf(q[2].x, q[3].x)), nm = m == -INFINITY ? 0.f : -m * kLog2e;
                            sum = 0.f;
#pragma unroll
                            for (int i = 0; i < 4; i++) sum += q[i].y * ex2(fmaf(q[i].x, kLog2e, nm));
                            if (row < p.M) p.part[(long long)(it.n0 / p.wide) * p.M + row] = make_float2(m, sum);
                        }
                    } else {
                        // 32 columns at a time: registers that do not fit would be kept in L2, since shared memory leaves no room for L1
                        const long long v = (long long)p.v0 + row;                                        // dw: the class
                        const int left = (it.kind == kLogits ? min(p.wide, p.next_cols - it.n0) : min(it.n, p.K - it.n0)) - off;
                        const bool inside = (it.kind == kDw ? v < p.V && row < p.cols : row < p.M) && left > 0;
                        __nv_bfloat16 *dw = static_cast<__nv_bfloat16 *>(p.dw_out) + v * p.lddw + it.n0 + off;  // where it is bf16
                        uint32_t old[16];
                        auto ask = [&](int i) {  // for what dw holds, before the wait
                            if (kTerms == 1 && !kAnywhere && it.kind == kDw && inside && p.dw_wide == 32) {
                                if (i < left) load8(*reinterpret_cast<uint32_t(*)[8]>(old), dw + i);
                                if (i + 16 < left) load8(*reinterpret_cast<uint32_t(*)[8]>(old + 8), dw + i + 16);
                            }
                        };
                        ask(0);
                        if (!mbar_wait_warp(&sm.acc_full[acc], (half / 2) & 1, ctx, SITE_ACC_FULL)) {
                            ok = false;
                            break;
                        }
                        tc_fence_after_sync();
#pragma unroll 1
                        for (int i = 0; i < 64; i += 32) {
                            uint32_t z[32];
                            tmem_ld32(from + acc * kTile + i, z);
                            tmem_wait_ld();
                            if (i == 32) {
                                tc_fence_before_sync();
                                __syncwarp();
                                if (lane == 0) mbar_arrive(&sm.acc_empty[acc]);
                            }
                            if (it.kind == kLogits) {
                                if (i >= left) continue;  // (a whole warp)
                                const int known = p.V - p.next_v0 - it.n0 - off - i, place = target - p.next_v0 - it.n0 - off - i;
                                const bool here = target >= 0 && place >= 0 && place < 32;
#pragma unroll
                                for (int e = 0; e < 32; e++) z[e] = __float_as_uint(ex2(fmaf(__uint_as_float(z[e]), p.log2e, nl)));
                                if (__any_sync(0xffffffffu, here)) {
#pragma unroll
                                    for (int e = 0; e < 32; e++)
                                        if (here && e == place) z[e] = __float_as_uint(__uint_as_float(z[e]) - 1.f);
                                }
                                if (known < 32) {
#pragma unroll
                                    for (int e = 0; e < 32; e++)
                                        if (e >= known) z[e] = 0;
                                }
                                if (inside) {
                                    __nv_bfloat16 *to = p.out + (long long)row * p.pitch + it.n0 + off + i;
#pragma unroll
                                    for (int c = 0; c < 32; c += 16) {
                                        uint32_t hi[8], lo[8];
#pragma unroll
                                        for (int e = 0; e < 8; e++) {
                                            const float a = __uint_as_float(z[c + 2 * e]) * by, b = __uint_as_float(z[c + 2 * e + 1]) * by;
                                            if (kTerms == 1) hi[e] = pack_bf16x2(a, b);
                                            else split_bf16x2(a, b, hi[e], lo[e]);
                                            if (target < 0) hi[e] = lo[e] = 0;
                                        }
                                        if (i + c < left) store8(to + c, hi);
                                        if (kTerms == 3 && i + c < left) store8(to + p.plane + c, lo);
                                    }
                                }
                            } else if (kAnywhere && it.kind == kDw) {
                                using T = std::conditional_t<kTerms == 3, float, __nv_bfloat16>;
                                transpose(lane, z);
                                const int row0 = row - lane;
                                add_anywhere(lane, static_cast<T *>(p.dw_out) + ((long long)p.v0 + row0) * p.lddw + it.n0 + off + i, p.lddw, z, min(p.cols, p.V - p.v0) - row0, left - i, by);
                            } else if (kTerms == 3) {
                                four_rows(lane, z);
                                const int row4 = row - lane + (lane & ~3), column = i + 8 * (lane & 3);
                                const int rows = it.kind == kDx ? p.M : min(p.cols, p.V - p.v0);
#pragma unroll
                                for (int t = 0; t < 4; t++) {
                                    if (row4 + t >= rows || column >= left) continue;
                                    if (it.kind == kDx) {
                                        float *to = p.dxp + ((long long)it.piece * p.M + row4 + t) * p.dx_pitch + it.n0 + off + column;
                                        if (p.first && b0 == 0) store8(to, *reinterpret_cast<const uint32_t(*)[8]>(z + 8 * t));
                                        else add_f32<8>(to, z + 8 * t, 8);
                                    } else {
                                        add_f32<8>(static_cast<float *>(p.dw_out) + ((long long)p.v0 + row4 + t) * p.lddw + it.n0 + off + column, z + 8 * t, left - column);
                                    }
                                }
                            } else if (inside && i < left) {
                                if (it.kind == kDw) {
                                    add_bf16(dw + i, old, z, left - i, p.dw_wide, by);
                                } else {
                                    float *to = p.dxp + ((long long)it.piece * p.M + row) * p.dx_pitch + it.n0 + off + i;
                                    if (p.first && b0 == 0) put_f32(to, z, left - i);
                                    else add_f32<32>(to, z, left - i);
                                }
                            }
                            __syncwarp();
                            if (i == 0) ask(32);
                        }
                    }
                }
            }
        }
    }

    // ------------------------------ tear-down ------------------------------
    if (sm.abort_flag) __nanosleep(50000);  // products that have been issued end
    tc_fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        tc_fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

// Maximum and sum of each row from those of its tiles.  A block takes 32 rows, a warp every 32nd tile, eight of them at a time.
__global__ void __launch_bounds__(1024) join_kernel(const float2 *__restrict__ part, const float *__restrict__ zt, Ids targets, float *__restrict__ losses,
                                                    float *__restrict__ lse, int tiles, int M, int V) {
    pdl_launch_dependents();
    pdl_wait();
    constexpr int kAhead = 8;
    __shared__ float2 all[32][32];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row = blockIdx.x * 32 + lane;
    auto over = [](float m, float top) { return top == -INFINITY ? 0.f : ex2((m - top) * kLog2e); };  // exp(m - top); nothing there: 0
    float m = -INFINITY, s = 0.f;
    if (row < M) {
        for (int t0 = warp; t0 < tiles; t0 += 32 * kAhead) {
            float2 q[kAhead];
#pragma unroll
            for (int u = 0; u < kAhead; u++) q[u] = t0 + 32 * u < tiles ? part[(long long)(t0 + 32 * u) * M + row] : make_float2(-INFINITY, 0.f);
            float top = m;
#pragma unroll
            for (int u = 0; u < kAhead; u++) top = fmaxf(top, q[u].x);
            s *= over(m, top);
#pragma unroll
            for (int u = 0; u < kAhead; u++) s += q[u].y * over(q[u].x, top);
            m = top;
        }
    }
    all[warp][lane] = make_float2(m, s);
    __syncthreads();
    if (warp != 0 || row >= M) return;
    float top = -INFINITY, sum = 0.f;
#pragma unroll 8
    for (int i = 0; i < 32; i++) top = fmaxf(top, all[i][lane].x);
#pragma unroll 8
    for (int i = 0; i < 32; i++) sum += all[i][lane].y * over(all[i][lane].x, top);
    const float l = top + logf(sum);
    lse[row] = l;
    losses[row] = targets.at(row, V) >= 0 ? l - zt[row] : 0.f;
}

// The factor of all rows' G that bf16 gradients do not take into it: the significand c, 1 to 2, of the largest |g| of a row that has a target.  With
// g = 1 / rows, or the same g for each row, G / c is p - [v = t] times a power of two; with g in it, nearly every target's entry, -g, would be rounded to the
// same side by the same share, up to 2^-8, and so would everything that is made of it (3001 x 1600 x 50257: 1.7e-3).  Where rows have factors of
// their own each rounds its own entries.  A power of two stays in G, so that no product leaves the range it had.  out: c, 1 / c.
struct Common {
    const float *g;
    float *out;
    int one_g;
};
__device__ __forceinline__ void common_of(const Common &a, const Ids &targets, int rows, int V) {
    constexpr int kAhead = 8;
    __shared__ float most[8];
    float top = 0.f;
    if (a.one_g) {
        top = fabsf(a.g[0]);
    } else {
        for (int r0 = threadIdx.x; r0 < rows; r0 += 256 * kAhead) {
            int t[kAhead];
            float v[kAhead];
            targets.many<kAhead>(t, V, r0, 256, rows);
#pragma unroll
            for (int u = 0; u < kAhead; u++) v[u] = a.g[min(r0 + 256 * u, rows - 1)];  // (behind the last row: that one again)
#pragma unroll
            for (int u = 0; u < kAhead; u++)
                if (t[u] >= 0) top = fmaxf(top, fabsf(v[u]));
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if ((threadIdx.x & 31) == 0) most[threadIdx.x >> 5] = top;
    __syncthreads();
    if (threadIdx.x > 0) return;
#pragma unroll
    for (int i = 0; i < 8; i++) top = fmaxf(top, most[i]);
    const float c = top >= 1.1754944e-38f && top < INFINITY ? __uint_as_float((__float_as_uint(top) & 0x007fffffu) | 0x3f800000u) : 1.f;
    a.out[0] = c, a.out[1] = 1.f / c;
}

// src [R, K] as bf16 planes [R, pitch] (hi, and lo of fp32 values).  Rows without a target become zeros where targets are given.  Also
// clears the counters of work items; one more block finds the common factor where it is asked for.
template <class T>
__global__ void __launch_bounds__(256) planes_kernel(const T *__restrict__ src, long long ld, __nv_bfloat16 *__restrict__ hi, __nv_bfloat16 *__restrict__ lo,
                                                     int R, int K, int pitch, int wide, Ids targets, int V, int *counters, int count, Common common) {
    pdl_launch_dependents();
    pdl_wait();
    const int blocks = common.out ? (int)gridDim.x - 1 : (int)gridDim.x;
    if ((int)blockIdx.x == blocks) {
        common_of(common, targets, R, V);
        return;
    }
    const int words = pitch / 8;
    const long long total = (long long)R * words;
    if (blockIdx.x == 0)
        for (int i = threadIdx.x; i < count; i += 256) counters[i] = 0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)blocks * 256) {
        const long long r = i / words;
        const int c = (int)(i - r * words) * 8;
        const T *at = src + r * ld + c;
        uint32_t h[4] = {}, l[4] = {};
        const bool none = targets.p != nullptr && targets.at(r, V) < 0;
        if (!none) {
            if constexpr (sizeof(T) == 2) {
                if (wide && c + 8 <= K) {
                    const uint4 v = *reinterpret_cast<const uint4 *>(at);
                    h[0] = v.x, h[1] = v.y, h[2] = v.z, h[3] = v.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (c + e < K) h[e / 2] |= (uint32_t)reinterpret_cast<const unsigned short *>(at)[e] << (e & 1) * 16;
                }
            } else {
                float v[8] = {};
                if (wide && c + 8 <= K) {
                    const float4 a = __ldcs(reinterpret_cast<const float4 *>(at)), b = __ldcs(reinterpret_cast<const float4 *>(at) + 1);
                    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
                } else {
#pragma unroll
                    for (int e = 0; e < 8; e++)
                        if (c + e < K) v[e] = at[e];
                }
#pragma unroll
                for (int e = 0; e < 4; e++) split_bf16x2(v[2 * e], v[2 * e + 1], h[e], l[e]);
            }
        }
        *reinterpret_cast<uint4 *>(hi + r * pitch + c) = make_uint4(h[0], h[1], h[2], h[3]);
        if (sizeof(T) == 4) *reinterpret_cast<uint4 *>(lo + r * pitch + c) = make_uint4(l[0], l[1], l[2], l[3]);
    }
}

// dx from the pieces of its contraction, times `by`, and times the common factor where there is one.  kGroups threads share four columns, each taking every kGroups-th piece; their sums are added in order.
template <class T, int kGroups>
__global__ void __launch_bounds__(256) sum_kernel(T *__restrict__ dx, const float *__restrict__ pieces, int count, int M, int K, int pitch, int wide, float by, const float *__restrict__ common) {
    pdl_launch_dependents();
    pdl_wait();
    if (common) by *= common[0];
    constexpr int kWords = 256 / kGroups, kAhead = 4;
    __shared__ float4 part[kGroups > 1 ? kGroups : 1][kGroups > 1 ? kWords : 1];
    const unsigned words = pitch / 4;
    const int group = threadIdx.x / kWords, place = threadIdx.x % kWords;
    const long long total = (long long)M * words, apart = (long long)M * pitch;
    for (long long i0 = (long long)blockIdx.x * kWords; i0 < total; i0 += (long long)gridDim.x * kWords) {
        const long long i = i0 + place, r = total <= 0xffffffffll ? (unsigned)i / words : i / words;
        const int c = (int)(i - r * words) * 4;
        float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
        if (i < total) {
            for (int p0 = group; p0 < count; p0 += kGroups * kAhead) {
                float4 v[kAhead];
#pragma unroll
                for (int u = 0; u < kAhead; u++) v[u] = __ldcs(reinterpret_cast<const float4 *>(pieces + min(p0 + kGroups * u, count - 1) * apart + r * pitch + c));
#pragma unroll
                for (int u = 0; u < kAhead; u++)
                    if (p0 + kGroups * u < count) sum = make_float4(sum.x + v[u].x, sum.y + v[u].y, sum.z + v[u].z, sum.w + v[u].w);
            }
        }
        if (kGroups > 1) {
            part[group][place] = sum;
            __syncthreads();
            if (group == 0) {
#pragma unroll
                for (int g = 1; g < kGroups; g++) sum = make_float4(sum.x + part[g][place].x, sum.y + part[g][place].y, sum.z + part[g][place].z, sum.w + part[g][place].w);
            }
            __syncthreads();
        }
        if (group > 0 || i >= total) continue;
        T *at = dx + r * K + c;
        sum = make_float4(sum.x * by, sum.y * by, sum.z * by, sum.w * by);
        const float s[4] = {sum.x, sum.y, sum.z, sum.w};
        if (wide && c + 4 <= K) {
            if constexpr (sizeof(T) == 2) *reinterpret_cast<uint2 *>(at) = make_uint2(pack_bf16x2(s[0], s[1]), pack_bf16x2(s[2], s[3]));
            else *reinterpret_cast<float4 *>(at) = sum;
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c + e < K) at[e] = (T)s[e];
        }
    }
}

// ---- host side ----

// G of a piece takes 256 MB at most, but for pieces of 32 tiles of classes: below that an item of dw, whose contraction is all rows, is longer than what a
// piece gives an SM to do.  Backward of 8192 x 768 x 50257 bf16 with 64, 128, 256, 512 MB: 2154, 1820, 1787, 1744 us; 16384 rows: 6324, 4293, 3671, 3629.
constexpr size_t kPieceBytes = (size_t)256 << 20;
constexpr int kLeastTiles = 32;
constexpr int kMostRows = 1 << 20;  // of the backward: a sum of dw over more steps would be cut off by more than it is rounded
constexpr int kFetchBlocks = 8;         // of 64 rows (40 rows, bf16 107 -> 98 us)
constexpr int kForwardSlots = 6, kBackwardSlots = 7;

int up(int v, int to) { return (v + to - 1) / to * to; }
size_t up256(size_t v) { return (v + 255) / 256 * 256; }

// What a call reads in place and what it copies, and where everything lies in the scratch buffer.
struct Layout {
    bool few, copy_x, copy_w;
    int pitch, planes;
    size_t x, w, part, zt, counters, g[2], dxp, total;
    int cols, pieces;         // of the vocabulary
    int wide;                 // columns of a tile of z
    int dx_pieces, dx_blocks, dx_pitch;
    size_t plane_x, plane_w, plane_g;  // elements
};

bool in_place(const void *p, long long ld) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld % 8 == 0; }

// Columns of a tile of z: 256, but where they make few rounds of the SMs, what makes these rounds end together (200 x 768 x 50257: two rounds of 176
// instead of 256, 30.9 -> 29.8 us).  A narrow tile costs a little more, as if it had 32 columns more, and where a tile has only half of its rows
// it waits for its operands anyway: 40 rows take 25.0 us at 256 columns, 26.4 at 176.
int tile_width(int M, int V, int sms) {
    const int tiles_m = (M + kTile - 1) / kTile, extra = M > 128 ? 32 : 256;
    auto rounds = [&](int n) { return ((long long)tiles_m * ((V + n - 1) / n) + sms - 1) / sms; };
    int best = kTile;
    if (rounds(kTile) <= 8)
        for (int n = kTile - 16; n >= 64; n -= 16)
            if (rounds(n) * (n + extra) < rounds(best) * (best + extra)) best = n;
    return best;
}

Layout layout(const void *x, const void *w, long long ldx, long long ldw, int type, int M, int V, int K, bool backward, int sms) {
    Layout l = {};
    l.planes = type == TENSOR_F32 ? 2 : 1;
    l.pitch = up(K, 8);
    l.few = !backward && few_rows_fit(x, w, ldx, ldw, type, M, V, K, sms);
    if (l.few) {
        l.zt = up256((size_t)few_rows_parts(V, sms) * M * sizeof(float2));
        l.total = l.zt + up256((size_t)M * sizeof(float));
        return l;
    }
    l.copy_x = type == TENSOR_F32 || backward || !in_place(x, ldx);  // the gradients need rows of zeros where there is no target
    l.copy_w = type == TENSOR_F32 || !in_place(w, ldw);
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up256(bytes);
        return here;
    };
    l.plane_x = up256((size_t)M * l.pitch * 2) / 2;
    l.plane_w = up256((size_t)V * l.pitch * 2) / 2;
    if (l.copy_x) l.x = take(l.plane_x * 2 * l.planes);
    if (l.copy_w) l.w = take(l.plane_w * 2 * l.planes);
    const int tiles_v = (V + kTile - 1) / kTile, tiles_m = (M + kTile - 1) / kTile, tiles_k = (K + kTile - 1) / kTile;
    if (!backward) {
        l.wide = tile_width(M, V, sms);
        l.part = take((size_t)((V + l.wide - 1) / l.wide) * M * sizeof(float2));
        l.zt = take((size_t)M * sizeof(float));
        l.total = at;
        return l;
    }
    // pieces of the vocabulary: as many tiles each
    const size_t tile_bytes = (size_t)M * kTile * 2 * l.planes;
    const int most = (int)std::min<size_t>(tiles_v, std::max<size_t>(kLeastTiles, kPieceBytes / tile_bytes));
    l.pieces = (tiles_v + most - 1) / most;
    const int tiles = (tiles_v + l.pieces - 1) / l.pieces;
    l.pieces = (tiles_v + tiles - 1) / tiles;
    l.cols = l.pieces > 1 ? tiles * kTile : up(V, kBlock);
    l.wide = l.pieces > 1 ? kTile : tile_width(M, l.cols, sms);
    // Pieces of the contraction of dx: none is longer than a share of what an SM has to do for a piece of the vocabulary.  Share 0.5, 0.7, 1.0: 40 rows bf16
    // 98.6, 106, 106 us; 500 rows 187, 178, 173; 2048 x 768 x 16384 198, 198, 179; 4096 rows fp32 2661, 2609, 2705 (each more piece is 4 bytes a value of dx twice).
    const int blocks = l.cols / kBlock;
    const double load = ((double)tiles_m * tiles_k * blocks + (double)tiles * tiles_k * std::max(4, (M + kBlock - 1) / kBlock)) / sms;
    const int longest = std::max(12, (int)(load * (M <= 128 ? 0.5 : type == TENSOR_F32 ? 0.7 : 1.0)));
    l.dx_pieces = std::min(64, (blocks + longest - 1) / longest);
    l.dx_blocks = (blocks + l.dx_pieces - 1) / l.dx_pieces;
    l.dx_pieces = (blocks + l.dx_blocks - 1) / l.dx_blocks;
    l.dx_pitch = up(K, 8);
    l.counters = take(sizeof(int) * (l.pieces + 3));  // and the common factor
    l.plane_g = (size_t)M * l.cols;
    for (int i = 0; i < (l.pieces > 1 ? 2 : 1); i++) l.g[i] = take(l.plane_g * 2 * l.planes);
    l.dxp = take((size_t)l.dx_pieces * M * l.dx_pitch * sizeof(float));
    l.total = at;
    return l;
}

// The backward of up to 16 rows: G, and the pieces of dx.
struct FewLayout {
    size_t g, dxp, total;
    int pieces, dx_pitch;
};
FewLayout few_layout(int M, int V, int K, int sms) {
    FewLayout l;
    l.pieces = few_rows_pieces(M, V, K, sms), l.dx_pitch = up(K, 8);
    l.g = 0, l.dxp = up256((size_t)V * few_rows_stride(M) * sizeof(float));
    l.total = l.dxp + up256((size_t)l.pieces * M * l.dx_pitch * sizeof(float));
    return l;
}

// [rows, cols] bf16 of `planes` planes: boxes of 64 columns by box_rows rows.
int map_of(CUtensorMap *map, const void *base, long long rows, int cols, long long pitch, size_t plane, int planes, int box_rows) {
    const cuuint64_t dims[3] = {(cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)planes};
    const cuuint64_t strides[2] = {(cuuint64_t)pitch * 2, planes > 1 ? (cuuint64_t)plane * 2 : (cuuint64_t)pitch * 2};
    const cuuint32_t box[3] = {64, (cuuint32_t)box_rows, 1};
    return attn::encode_tiled(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, base, dims, strides, box);
}

void set_fix(Problem &p, int type) {
    const double fix = fix_of(p.K, type);
    p.fix = (float)fix, p.log2e = (float)(1.4426950408889634 * fix);
}

// What a gradient loses, as a share of it: sums of fp32 operands end after kSegment blocks or with the contraction of `blocks`.  dw is what G makes up for, before
// the sums, and dx the rest, behind them: neither costs anything there.  (4096 x 768 x 50257: dx and dw were 2.8e-6 too small and 4.1e-6 of their norm off, now
// 1e-7 and 3.0e-6.)  bf16 gradients are rounded to 2^-9 of themselves, next to which it is nothing.  (0.9: these sums grow less evenly.)
double cut_of(int blocks) {
    const int full = blocks / kSegment, rest = blocks % kSegment;
    return 0.9 * kCut * 3 * (kBlock / 16) * ((double)full * kSegment * kSegment + (double)rest * rest) / blocks;
}

int blocks_for(long long words) { return (int)std::max(1ll, std::min(words / 256 + 1, 148ll * 16)); }

cudaError_t launch_planes(const void *src, long long ld, int type, void *to, size_t plane, int R, int K, int pitch, Ids targets, int V, int *counters, int count,
                          Common common, cudaStream_t s) {
    __nv_bfloat16 *hi = static_cast<__nv_bfloat16 *>(to), *lo = hi + plane;
    const int grid = blocks_for((long long)R * (pitch / 8)) + (common.out != nullptr);
    const int each = type == TENSOR_F32 ? 4 : 2, wide = (reinterpret_cast<uintptr_t>(src) & 15) == 0 && ld * each % 16 == 0;
    if (type == TENSOR_F32)
        return attn::launch_after_previous(planes_kernel<float>, dim3(grid), dim3(256), 0, s, static_cast<const float *>(src), ld, hi, lo, R, K, pitch, wide, targets, V,
                                           counters, count, common);
    return attn::launch_after_previous(planes_kernel<__nv_bfloat16>, dim3(grid), dim3(256), 0, s, static_cast<const __nv_bfloat16 *>(src), ld, hi, lo, R, K, pitch, wide,
                                       targets, V, counters, count, common);
}

// Eight threads share the pieces where there are more than four and few words: 49 pieces of 40 x 768 18 -> 4.8 us, 7 of 2048 x 768 23.5 us by eight (11 by one).
template <class T>
cudaError_t launch_sum(T *dx, const float *pieces, int count, int M, int K, int pitch, int wide, float by, const float *common, cudaStream_t s) {
    const int groups = count > 4 && (long long)M * (pitch / 4) < 100000 ? 8 : 1;
    const int grid = blocks_for((long long)M * (pitch / 4) * groups);
    return groups > 1 ? attn::launch_after_previous(sum_kernel<T, 8>, dim3(grid), dim3(256), 0, s, dx, pieces, count, M, K, pitch, wide, by, common)
                      : attn::launch_after_previous(sum_kernel<T, 1>, dim3(grid), dim3(256), 0, s, dx, pieces, count, M, K, pitch, wide, by, common);
}

template <int kTerms, bool kBackward>
cudaError_t launch_tiles(const Maps &maps, const Problem &p, int sms, int *status, cudaStream_t s) {
    constexpr int kSlots = kBackward ? kBackwardSlots : kForwardSlots;
    auto kernel = tiles_kernel<kTerms, kBackward, kSlots, false>;
    if constexpr (kBackward)
        if (p.dw && p.dw_wide < 16) kernel = tiles_kernel<kTerms, kBackward, kSlots, true>;
    return attn::launch_after_previous(kernel, dim3((unsigned)std::min(p.total, sms)), dim3(kThreads), sizeof(Smem<kSlots, kBackward>),
                                       s, maps, p, status);
}

// The memory of a matrix; NULL: none.
struct Span {
    uintptr_t from, to;
    Span(const void *p, long long rows, long long ld, long long columns, size_t each)
        : from(reinterpret_cast<uintptr_t>(p)), to(p ? from + ((rows - 1) * ld + columns) * each : 0) {}
    bool meets(const Span &o) const { return from && o.from && from < o.to && o.from < to; }
};

int check(const void *x, const void *w, const void *targets, const void *scratch, long long ldx, long long ldw, int type, int target_type, int rows, int V, int K) {
    if (rows < 0 || V <= 0 || K <= 0 || ldx < K || ldw < K) return ATTN_ERR_ARGUMENT;
    if ((type != TENSOR_F32 && type != TENSOR_BF16) || target_type < TENSOR_INT32 || target_type > TENSOR_IDS_F32) return ATTN_ERR_ARGUMENT;
    const uintptr_t each = type == TENSOR_F32 ? 3 : 1, id = target_type == TENSOR_INT64 ? 7 : 3;
    if ((reinterpret_cast<uintptr_t>(x) & each) || (reinterpret_cast<uintptr_t>(w) & each) || (reinterpret_cast<uintptr_t>(targets) & id) ||
        (reinterpret_cast<uintptr_t>(scratch) & 255))
        return ATTN_ERR_ALIGN;
    // coordinates and numbers of tiles are 31-bit numbers, row strides of the copy engine 40-bit ones
    if (rows > (1 << 30) || V > (1 << 30) || K > (1 << 24) || ldx > (1ll << 34) || ldw > (1ll << 34)) return ATTN_ERR_UNSUPPORTED;
    if ((double)((rows + kTile - 1) / kTile + 1) * ((V + kTile - 1) / kTile + 1) > 1e9) return ATTN_ERR_UNSUPPORTED;
    return ATTN_OK;
}

}  // namespace

cudaError_t set_attributes() {
    cudaError_t e = few_rows_set_attributes();
    auto set = [&](const void *kernel, size_t bytes) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)bytes);
    };
    set(reinterpret_cast<const void *>(tiles_kernel<1, false, kForwardSlots, false>), sizeof(Smem<kForwardSlots, false>));
    set(reinterpret_cast<const void *>(tiles_kernel<3, false, kForwardSlots, false>), sizeof(Smem<kForwardSlots, false>));
    set(reinterpret_cast<const void *>(tiles_kernel<1, true, kBackwardSlots, false>), sizeof(Smem<kBackwardSlots, true>));
    set(reinterpret_cast<const void *>(tiles_kernel<1, true, kBackwardSlots, true>), sizeof(Smem<kBackwardSlots, true>));
    set(reinterpret_cast<const void *>(tiles_kernel<3, true, kBackwardSlots, false>), sizeof(Smem<kBackwardSlots, true>));
    set(reinterpret_cast<const void *>(tiles_kernel<3, true, kBackwardSlots, true>), sizeof(Smem<kBackwardSlots, true>));
    return e;
}

}  // namespace head

extern "C" {

size_t xent_sm100_linear_forward_scratch_bytes(const void *x, const void *w, long long ldx, long long ldw, int type, int rows, int V, int K) {
    if (head::check(x, w, nullptr, nullptr, ldx, ldw, type, TENSOR_INT32, rows, V, K) != ATTN_OK || rows == 0) return 0;
    return head::layout(x, w, ldx, ldw, type, rows, V, K, false, attn::sm_count()).total;
}

size_t xent_sm100_linear_backward_scratch_bytes(const void *x, const void *w, long long ldx, long long ldw, int type, int rows, int V, int K) {
    if (head::check(x, w, nullptr, nullptr, ldx, ldw, type, TENSOR_INT32, rows, V, K) != ATTN_OK || rows == 0 || rows > head::kMostRows) return 0;
    const size_t tiles = head::layout(x, w, ldx, ldw, type, rows, V, K, true, attn::sm_count()).total;
    return rows <= 16 ? std::max(tiles, head::few_layout(rows, V, K, attn::sm_count()).total) : tiles;  // (which of them depends on dw too)
}

// loaded < 0: all items are loaded.  Otherwise only rows that go by tiles.
static int linear_forward(const void *x, const void *w, const void *targets, float *losses, float *lse, void *scratch, long long ldx, long long ldw, int type,
                          int target_type, int rows, int V, int K, int loaded, void *stream) {
    using namespace head;
    if (!x || !w || !targets || !losses || !lse) return ATTN_ERR_NULL;
    int rc = check(x, w, targets, scratch, ldx, ldw, type, target_type, rows, V, K);
    if (rc != ATTN_OK) return rc;
    if (rows > 0 && !scratch) return ATTN_ERR_NULL;  // (behind the sizes that have none)
    if ((reinterpret_cast<uintptr_t>(losses) & 3) || (reinterpret_cast<uintptr_t>(lse) & 3)) return ATTN_ERR_ALIGN;
    if (rows > 0) {
        const size_t each = type == TENSOR_F32 ? 4 : 2;
        const Span losses_at(losses, 1, rows, rows, 4), lse_at(lse, 1, rows, rows, 4);
        for (const Span &in : {Span(x, rows, ldx, K, each), Span(w, V, ldw, K, each), Span(targets, 1, rows, rows, target_type == TENSOR_INT64 ? 8 : 4)})
            if (losses_at.meets(in) || lse_at.meets(in)) return ATTN_ERR_ARGUMENT;
        if (losses_at.meets(lse_at)) return ATTN_ERR_ARGUMENT;
    }
    int *status = nullptr;
    if ((rc = attn::device_status_word(&status)) != ATTN_OK) return rc;
    if (rows == 0) return ATTN_OK;
    const int sms = attn::sm_count();
    const Layout l = layout(x, w, ldx, ldw, type, rows, V, K, false, sms);
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    char *base = static_cast<char *>(scratch);
    cudaError_t e = cudaSuccess;
    if (l.few && loaded >= 0) return ATTN_ERR_SHAPE;
    if (l.few) {
        const FewRows a{x, w, ldx, ldw, Ids{targets, target_type}, reinterpret_cast<float2 *>(base), reinterpret_cast<float *>(base + l.zt), rows, V, K, nullptr, nullptr, 0, nullptr, (float)fix_of(K, type)};
        if ((e = launch_few_rows(a, type, sms, s)) != cudaSuccess) return (int)e;
        return (int)attn::launch_after_previous(join_kernel, dim3((rows + 31) / 32), dim3(1024), 0, s, a.part, a.zt, a.targets, losses, lse, few_rows_parts(V, sms), rows, V);
    }
    if (l.copy_w && (e = launch_planes(w, ldw, type, base + l.w, l.plane_w, V, K, l.pitch, Ids{nullptr, 0}, 0, nullptr, 0, Common{}, s)) != cudaSuccess) return (int)e;
    if (l.copy_x && (e = launch_planes(x, ldx, type, base + l.x, l.plane_x, rows, K, l.pitch, Ids{nullptr, 0}, 0, nullptr, 0, Common{}, s)) != cudaSuccess) return (int)e;
    Maps maps = {};
    if ((rc = map_of(&maps.x, l.copy_x ? base + l.x : x, rows, K, l.copy_x ? l.pitch : rows > 1 ? ldx : l.pitch, l.plane_x, l.planes, 128)) != 0) return rc;
    if ((rc = map_of(&maps.w, l.copy_w ? base + l.w : w, V, K, l.copy_w ? l.pitch : V > 1 ? ldw : l.pitch, l.plane_w, l.planes, l.wide)) != 0) return rc;
    Problem p = {};
    p.M = rows, p.V = V, p.K = K;
    set_fix(p, type);
    p.tiles_m = (rows + kTile - 1) / kTile;
    p.blocks_k = (K + kBlock - 1) / kBlock;
    p.next_cols = V, p.wide = l.wide;
    const int tiles = (V + l.wide - 1) / l.wide;
    p.total = p.tiles_m * tiles;
    p.loaded = loaded < 0 ? p.total : loaded;
    p.targets = Ids{targets, target_type};
    p.part = reinterpret_cast<float2 *>(base + l.part);
    p.zt = reinterpret_cast<float *>(base + l.zt);
    e = type == TENSOR_F32 ? launch_tiles<3, false>(maps, p, sms, status, s) : launch_tiles<1, false>(maps, p, sms, status, s);
    if (e != cudaSuccess) return (int)e;
    return (int)attn::launch_after_previous(join_kernel, dim3((rows + 31) / 32), dim3(1024), 0, s, p.part, p.zt, p.targets, losses, lse, tiles, rows, V);
}

int xent_sm100_linear_forward(const void *x, const void *w, const void *targets, float *losses, float *lse, void *scratch, long long ldx, long long ldw, int type,
                              int target_type, int rows, int V, int K, void *stream) {
    return linear_forward(x, w, targets, losses, lse, scratch, ldx, ldw, type, target_type, rows, V, K, -1, stream);
}

int xent_sm100_selftest_linear_wait_limit(const void *x, const void *w, const void *targets, float *losses, float *lse, void *scratch, long long ldx, long long ldw, int type,
                                          int target_type, int rows, int V, int K, int loaded, void *stream) {
    if (loaded < 0) return ATTN_ERR_SHAPE;
    return linear_forward(x, w, targets, losses, lse, scratch, ldx, ldw, type, target_type, rows, V, K, loaded, stream);
}

int xent_sm100_linear_backward(const float *g, const void *x, const void *w, const void *targets, const float *lse, void *dx, void *dw, void *scratch, long long ldx,
                               long long ldw, long long lddw, int one_g, int type, int target_type, int rows, int V, int K, void *stream) {
    using namespace head;
    if (!g || !x || !w || !targets || !lse || (!dx && !dw)) return ATTN_ERR_NULL;
    int rc = check(x, w, targets, scratch, ldx, ldw, type, target_type, rows, V, K);
    if (rc != ATTN_OK) return rc;
    if (dw && lddw < K) return ATTN_ERR_ARGUMENT;
    if (rows > kMostRows) return ATTN_ERR_UNSUPPORTED;
    if (rows > 0 && !scratch) return ATTN_ERR_NULL;
    const size_t each = type == TENSOR_F32 ? 4 : 2;
    if ((reinterpret_cast<uintptr_t>(g) & 3) || (reinterpret_cast<uintptr_t>(lse) & 3) || reinterpret_cast<uintptr_t>(dx) % each || reinterpret_cast<uintptr_t>(dw) % each)
        return ATTN_ERR_ALIGN;
    if (rows > 0) {
        const Span x_at(x, rows, ldx, K, each), w_at(w, V, ldw, K, each), dx_at(dx, rows, K, K, each), dw_at(dw, V, lddw, K, each);
        const Span lse_at(lse, 1, rows, rows, 4), g_at(g, 1, rows, one_g ? 1 : rows, 4), t_at(targets, 1, rows, rows, target_type == TENSOR_INT64 ? 8 : 4);
        for (const Span &out : {dx_at, dw_at})
            for (const Span &in : {x_at, w_at, lse_at, g_at, t_at})
                if (out.meets(in)) return ATTN_ERR_ARGUMENT;
        if (dx_at.meets(dw_at)) return ATTN_ERR_ARGUMENT;
    }
    int *status = nullptr;
    if ((rc = attn::device_status_word(&status)) != ATTN_OK) return rc;
    if (rows == 0) return ATTN_OK;
    const int sms = attn::sm_count();
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    char *base = static_cast<char *>(scratch);
    cudaError_t e = cudaSuccess;
    auto sum = [&](const float *pieces, int count, int pitch, double by, const float *common) {
        const int wide = (reinterpret_cast<uintptr_t>(dx) & 15) == 0 && (size_t)K * each % 16 == 0;
        return (int)(type == TENSOR_F32 ? launch_sum(static_cast<float *>(dx), pieces, count, rows, K, pitch, wide, (float)by, common, s)
                                        : launch_sum(static_cast<__nv_bfloat16 *>(dx), pieces, count, rows, K, pitch, wide, (float)by, common, s));
    };
    if (few_rows_gradients_fit(x, w, dw, ldx, ldw, lddw, type, rows, V, K)) {
        const FewLayout f = few_layout(rows, V, K, sms);
        const FewRows a{x, w, ldx, ldw, Ids{targets, target_type}, nullptr, nullptr, rows, V, K, g, lse, one_g, reinterpret_cast<float *>(base + f.g), (float)fix_of(K, type)};
        float *dxp = dx ? reinterpret_cast<float *>(base + f.dxp) : nullptr;
        if ((e = launch_few_rows(a, type, sms, s)) != cudaSuccess) return (int)e;
        if ((e = launch_few_rows_products(a, type, dw, lddw, dxp, f.dx_pitch, sms, s)) != cudaSuccess) return (int)e;
        return dx ? sum(dxp, f.pieces, f.dx_pitch, 1.0, nullptr) : ATTN_OK;
    }
    const Layout l = layout(x, w, ldx, ldw, type, rows, V, K, true, sms);
    if (l.copy_w && (e = launch_planes(w, ldw, type, base + l.w, l.plane_w, V, K, l.pitch, Ids{nullptr, 0}, 0, nullptr, 0, Common{}, s)) != cudaSuccess) return (int)e;
    int *counters = reinterpret_cast<int *>(base + l.counters);
    const Common common{g, type == TENSOR_BF16 ? reinterpret_cast<float *>(counters + l.pieces + 1) : nullptr, one_g};
    if ((e = launch_planes(x, ldx, type, base + l.x, l.plane_x, rows, K, l.pitch, Ids{targets, target_type}, V, counters, l.pieces + 1, common, s)) != cudaSuccess) return (int)e;

    const void *wp = l.copy_w ? base + l.w : w;
    const long long pitch_w = l.copy_w ? l.pitch : V > 1 ? ldw : l.pitch;
    Maps maps = {};
    if ((rc = map_of(&maps.x, base + l.x, rows, K, l.pitch, l.plane_x, l.planes, 128)) != 0) return rc;
    if ((rc = map_of(&maps.w, wp, V, K, pitch_w, l.plane_w, l.planes, l.wide)) != 0) return rc;
    if ((rc = map_of(&maps.x_mn, base + l.x, rows, K, l.pitch, l.plane_x, l.planes, kBlock)) != 0) return rc;
    if ((rc = map_of(&maps.w_mn, wp, V, K, pitch_w, l.plane_w, l.planes, kBlock)) != 0) return rc;
    Problem p = {};
    p.M = rows, p.V = V, p.K = K;
    set_fix(p, type);
    p.fix_g = 1.f, p.common = common.out;
    double fix_dx = 1.0;
    p.tiles_m = (rows + kTile - 1) / kTile;
    p.tiles_k = (K + kTile - 1) / kTile;
    p.blocks_m = (rows + kBlock - 1) / kBlock;
    p.blocks_k = (K + kBlock - 1) / kBlock;
    p.dx_pieces = l.dx_pieces, p.dx_blocks = l.dx_blocks;
    p.pitch = l.cols, p.wide = l.wide;
    if (type == TENSOR_F32) p.fix_g = (float)(1.0 + cut_of(p.blocks_m)), fix_dx = 1.0 + cut_of(p.dx_blocks) - cut_of(p.blocks_m);
    p.plane = (long long)l.plane_g;
    p.targets = Ids{targets, target_type};
    p.g = g, p.lse = lse, p.one_g = one_g;
    p.dxp = reinterpret_cast<float *>(base + l.dxp);
    p.dx_pitch = l.dx_pitch;
    p.dw_out = dw, p.lddw = lddw;
    for (int b : {32, 16})
        if (!p.dw_wide && reinterpret_cast<uintptr_t>(dw) % b == 0 && (size_t)lddw * each % b == 0 && (size_t)K * each % b == 0) p.dw_wide = b;
    // dw comes from HBM once it is added to.  Where that is soon after its item has been handed out, it is on its way by then.
    if (dw && p.dw_wide >= 16 && p.blocks_m <= kFetchBlocks) {
        const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)V}, strides[1] = {(cuuint64_t)lddw * each};
        const cuuint32_t box[2] = {kTile, 64};
        if ((rc = attn::encode_tiled(&maps.dw, type == TENSOR_F32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, dw, dims, strides, box,
                                     CU_TENSOR_MAP_SWIZZLE_NONE)) != 0)
            return rc;
        p.fetch_dw = 1;
    }
    for (int i = 0; i <= l.pieces; i++) {  // the products of piece i - 1, z of piece i
        p.dx = i > 0 && dx ? p.tiles_m * p.tiles_k * l.dx_pieces : 0;
        p.dw = 0;
        if (i > 0) {
            p.v0 = (i - 1) * l.cols;
            p.cols = std::min(l.cols, up(V - p.v0, kBlock));
            if (dw) p.dw = (p.cols + kTile - 1) / kTile * p.tiles_k;
            p.first = i == 1;
            const void *g0 = base + l.g[(i - 1) & 1];
            if ((rc = map_of(&maps.g, g0, rows, p.cols, l.cols, l.plane_g, l.planes, 128)) != 0) return rc;
            if ((rc = map_of(&maps.g_mn, g0, rows, p.cols, l.cols, l.plane_g, l.planes, kBlock)) != 0) return rc;
        }
        int z = 0;
        if (i < l.pieces) {
            p.next_v0 = i * l.cols;
            p.next_cols = std::min(l.cols, up(V - p.next_v0, kBlock));
            p.out = reinterpret_cast<__nv_bfloat16 *>(base + l.g[i & 1]);
            z = p.tiles_m * ((p.next_cols + l.wide - 1) / l.wide);
        }
        p.total = p.dx + p.dw + z;
        p.dw_first = p.blocks_m > p.dx_blocks;
        p.counter = counters + i;
        e = type == TENSOR_F32 ? launch_tiles<3, true>(maps, p, sms, status, s) : launch_tiles<1, true>(maps, p, sms, status, s);
        if (e != cudaSuccess) return (int)e;
    }
    return dx ? sum(p.dxp, l.dx_pieces, l.dx_pitch, fix_dx, common.out) : ATTN_OK;
}

}  // extern "C"
