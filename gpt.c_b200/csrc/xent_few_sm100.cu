// The forward of projection and loss (xent_linear_sm100.cu) for few rows: the weights are read once, straight into registers, for sm_100a.
//
// With up to 48 rows the products are few and the weights all that has to be moved.  The tiles of the other kernel have half of their shared memory
// for rows that are not there, and fp32 weights are written and read again as bf16 planes.  Here a warp takes 16 classes at a time: a lane reads eight
// values of a row, 32 or 16 bytes, which are the lane's part of two mma fragments if the contraction is taken in that order, and splits fp32 values into
// hi and lo on the way.  x is in shared memory, bf16 (hi and lo), its rows so far apart that eight lanes that read two of them meet no bank twice.
// Maximum and sum of each row stay in registers until the end.
//
// Bound by HBM where there are up to 16 rows, then by the products (mma.sync has a quarter of the rate) and what they wait for.  Classes of 768 features, us with the
// join, in brackets with tiles: 16 x 50257 bf16 15.6 (26), fp32 37 (110); 32 rows 20.1 (25), 46 (103); 48 rows fp32 58 (104), bf16 25.7 (22.8); 64 rows fp32 104 (104);
// 16 x 100 bf16 8.2 (11.3), fp32 11.5 (20).  Reading takes 12 us of bf16 and 24 of fp32 weights.  fp32 rows that start anywhere: 5 x 1001 x 50257 55 us (146).  All
// warps help with x, whether there are classes for them or not (16 x 2000 bf16 14.2 -> 9.0); bf16 values are asked for where the products have taken the ones before,
// since registers would be copied otherwise (16 x 1600 x 50257 45.3 -> 35.5).
#include <cuda_bf16.h>

#include <algorithm>

#include "ids.cuh"
#include "tc05.cuh"
#include "xent_linear.cuh"

namespace head {
namespace {

using namespace tc05;

constexpr int kMostWarps = 12;  // of 168 registers

__device__ __forceinline__ void mma(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float exp_of(float x) { return exp2f(x * 1.4426950408889634f); }

// 32 bytes of a row as they are in memory: 16 bf16 values, or 8 fp32 values, which make as many of hi and lo.
template <class T>
struct Piece {
    static constexpr int kValues = 32 / sizeof(T);
    uint32_t v[8];
    __device__ __forceinline__ void load(const T *p, int left) {  // `left`: values that are inside, as many as 16 bytes at a time
#pragma unroll
        for (int i = 0; i < 2; i++)
            *reinterpret_cast<uint4 *>(v + 4 * i) = left > i * kValues / 2 ? *reinterpret_cast<const uint4 *>(p + i * kValues / 2) : make_uint4(0, 0, 0, 0);
    }
    // fp32 values that start anywhere: every fourth one from the lane's on, so that four lanes read 16 bytes of a row next to each other.  (The order of the
    // contraction is free as long as both factors have the same.)
    __device__ __forceinline__ void load_fourths(const T *p, int left) {
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = left > 4 * i ? *reinterpret_cast<const uint32_t *>(p + 4 * i) : 0;
    }
    // kValues / 2 words of two bf16 values
    __device__ __forceinline__ void split(uint32_t (&hi)[kValues / 2], uint32_t (&lo)[kValues / 2]) const {
#pragma unroll
        for (int i = 0; i < kValues / 2; i++) {
            if constexpr (sizeof(T) == 2) hi[i] = v[i], lo[i] = 0;
            else split_bf16x2(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]), hi[i], lo[i]);
        }
    }
};

// What the backward makes of z: G[v, 0 .. stride - 1], of up to 16 rows.
struct ToG {
    float *out;
    const float *g, *lse;
    int one_g, stride;
};

// kTiles: of 16 rows of x.  `classes`: of a CTA, a multiple of 16.  kGradient: G instead of maxima and sums.
// kAnywhere: rows of fp32 values that do not all start on 16 bytes.
template <class T, int kTiles, bool kGradient, bool kAnywhere>
__global__ void __launch_bounds__(32 * kMostWarps) few_rows_kernel(const T *__restrict__ x, long long ldx, const T *__restrict__ w, long long ldw, Ids targets,
                                                                   float2 *__restrict__ part, float *__restrict__ zt, ToG to, float fix, int M, int V, int K, int classes, int pitch) {
    pdl_launch_dependents();
    pdl_wait();
    extern __shared__ __align__(16) uint8_t rows[];  // [plane][16 kTiles][pitch bytes]
    __shared__ float2 all[kMostWarps][16 * kTiles];
    constexpr int kAhead = sizeof(T) == 2 ? 7 - kTiles : kTiles == 1 ? 4 : 3;  // as many as there are registers for
    constexpr int kPlanes = sizeof(T) / 2, kBlock = 128 / sizeof(T), kEach = Piece<T>::kValues, kWords = kEach / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, g = lane >> 2, q = lane & 3;
    const int class0 = blockIdx.x * classes, tiles = (min(V, class0 + classes) - class0 + 15) / 16, blocks = (K + kBlock - 1) / kBlock;
    const int mine = tiles > warp ? (tiles - warp + warps - 1) / warps : 0, total = mine * blocks;

    // what is asked for next: block load_b of tile load_t
    Piece<T> ahead[kAhead][2];
    int load_b = 0, load_t = warp;
    const T *from[2];
    auto rows_of = [&](int t) {
#pragma unroll
        for (int r = 0; r < 2; r++) from[r] = w + (long long)min(class0 + 16 * t + 8 * r + g, V - 1) * ldw + (kAnywhere ? q : kEach * q);
    };
    auto ask = [&](Piece<T>(&to)[2], int n) {
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int left = n < total ? K - kBlock * load_b : 0;
            if constexpr (kAnywhere) to[r].load_fourths(from[r] + kBlock * load_b, left - q);
            else to[r].load(from[r] + kBlock * load_b, left - kEach * q);
        }
        if (++load_b == blocks) load_b = 0, load_t += warps, rows_of(load_t);
    };
    rows_of(load_t);
#pragma unroll
    for (int i = 0; i < kAhead; i++) ask(ahead[i], i);

    const int words = blocks * kBlock / kEach;  // pieces of a row
    for (int i = threadIdx.x; i < 16 * kTiles * words; i += blockDim.x) {
        const int row = i / words, c = (i - row * words) * kEach;
        uint32_t hi[kWords], lo[kWords];
        Piece<T> e;
        if constexpr (kAnywhere) {
            const int first = c / kBlock * kBlock + c / kEach % 4;
            e.load_fourths(x + row * ldx + first, row < M ? K - first : 0);
        } else {
            e.load(x + row * ldx + c, row < M ? K - c : 0);
        }
        e.split(hi, lo);
#pragma unroll
        for (int k = 0; k < kWords; k += 4) {
            *reinterpret_cast<uint4 *>(rows + row * pitch + c * 2 + 4 * k) = make_uint4(hi[k], hi[k + 1], hi[k + 2], hi[k + 3]);
            if (kPlanes == 2) *reinterpret_cast<uint4 *>(rows + (16 * kTiles + row) * pitch + c * 2 + 4 * k) = make_uint4(lo[k], lo[k + 1], lo[k + 2], lo[k + 3]);
        }
    }
    int target[kTiles][2];
    float top[kTiles][2], sum[kTiles][2];
#pragma unroll
    for (int m = 0; m < kTiles; m++)
#pragma unroll
        for (int r = 0; r < 2; r++) {
            const int row = 16 * m + 8 * r + g;
            target[m][r] = row < M ? targets.at(row, V) : -1;
            top[m][r] = -INFINITY, sum[m][r] = 0.f;
            if (kGradient && row < M) top[m][r] = to.lse[row], sum[m][r] = target[m][r] < 0 ? 0.f : to.g[to.one_g ? 0 : row];
        }
    __syncthreads();

    float z[kTiles][2][4];
    int b = 0, t = warp;
    for (int n0 = 0; n0 < total; n0 += kAhead) {
#pragma unroll
        for (int u = 0; u < kAhead; u++) {
            if (n0 + u >= total) break;
            if (b == 0) {
#pragma unroll
                for (int m = 0; m < kTiles; m++)
#pragma unroll
                    for (int i = 0; i < 8; i++) z[m][i / 4][i % 4] = 0.f;
            }
            uint32_t hi[2][kWords], lo[2][kWords];
#pragma unroll
            for (int r = 0; r < 2; r++) ahead[u][r].split(hi[r], lo[r]);
            if (sizeof(T) == 4) ask(ahead[u], n0 + u + kAhead);
#pragma unroll
            for (int m = 0; m < kTiles; m++) {
#pragma unroll
                for (int k = 0; k < kWords; k += 4) {
#pragma unroll
                    for (int p = 0; p < kPlanes; p++) {
                        uint4 a[2];
#pragma unroll
                        for (int r = 0; r < 2; r++)
                            a[r] = *reinterpret_cast<const uint4 *>(rows + (16 * (p * kTiles + m) + 8 * r + g) * pitch + 2 * (kBlock * b + kEach * q + 2 * k));
                        const uint32_t a0[4] = {a[0].x, a[1].x, a[0].y, a[1].y}, a1[4] = {a[0].z, a[1].z, a[0].w, a[1].w};
#pragma unroll
                        for (int r = 0; r < 2; r++) {
                            mma(z[m][r], a0, hi[r][k], hi[r][k + 1]);
                            mma(z[m][r], a1, hi[r][k + 2], hi[r][k + 3]);
                            if (kPlanes == 2 && p == 0) {
                                mma(z[m][r], a0, lo[r][k], lo[r][k + 1]);
                                mma(z[m][r], a1, lo[r][k + 2], lo[r][k + 3]);
                            }
                        }
                    }
                }
            }
            if (sizeof(T) == 2) ask(ahead[u], n0 + u + kAhead);  // (its values go to the products as they are)
            if (++b < blocks) continue;
            b = 0;
            // 16 classes are done: a lane has classes 8 r + 2 q and the next of rows g and 8 + g of each tile
            const int first = class0 + 16 * t + 2 * q;
            t += warps;
#pragma unroll
            for (int m = 0; m < kTiles; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    if constexpr (kGradient) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int c = first + 8 * (i / 2) + i % 2, row = 8 * h + g;
                            const float p = exp_of(fmaf(z[m][i / 2][2 * h + i % 2], fix, -top[m][h])) - (c == target[m][h] ? 1.f : 0.f);
                            if (c < V && row < to.stride) to.out[(long long)c * to.stride + row] = target[m][h] < 0 ? 0.f : p * sum[m][h];
                        }
                    } else {
                        float v[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const int c = first + 8 * (i / 2) + i % 2;
                            v[i] = c < V ? z[m][i / 2][2 * h + i % 2] * fix : -INFINITY;
                            if (c < V && c == target[m][h]) zt[16 * m + 8 * h + g] = v[i];
                        }
                        const float most = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), top[m][h]), by = most == -INFINITY ? 0.f : most;
                        sum[m][h] *= exp_of(top[m][h] - by);
#pragma unroll
                        for (int i = 0; i < 4; i++) sum[m][h] += exp_of(v[i] - by);
                        top[m][h] = most;
                    }
                }
        }
    }
    if constexpr (!kGradient) {
        // the lanes of a row, then the warps
        auto join = [](float &m, float &s, float m2, float s2) {
            const float most = fmaxf(m, m2), by = most == -INFINITY ? 0.f : most;
            s = s * exp_of(m - by) + s2 * exp_of(m2 - by);
            m = most;
        };
#pragma unroll
        for (int m = 0; m < kTiles; m++)
#pragma unroll
            for (int h = 0; h < 2; h++) {
#pragma unroll
                for (int o = 1; o < 4; o <<= 1)
                    join(top[m][h], sum[m][h], __shfl_xor_sync(0xffffffffu, top[m][h], o), __shfl_xor_sync(0xffffffffu, sum[m][h], o));
                if (q == 0) all[warp][16 * m + 8 * h + g] = make_float2(top[m][h], sum[m][h]);
            }
        __syncthreads();
        const int row = threadIdx.x;
        if (row < M) {
            float m = -INFINITY, s = 0.f;
            for (int i = 0; i < warps; i++) join(m, s, all[i][row].x, all[i][row].y);
            part[(long long)blockIdx.x * M + row] = make_float2(m, s);
        }
    }
}

// ---------------------------------------------------------------------------------------------
// The two products of the backward for up to 16 rows, in fp32 arithmetic: a thread has four columns of x and of the sums of dx for all rows, and goes through
// classes of its block: w once for dx, dw once for what is added to it.  G of a class is the same for all threads.
//
// Bound by HBM: w is read again (with the G kernel twice in all) and dw read and written, 617 MB of fp32 and 309 of bf16 at 768 x 50257: 94 and 47 us.
// Measured with G and the sum of dx, in brackets with tiles: 1 row fp32 111 us (216; 780 features 121, 371), 16 rows 166 (214), where the multiplications
// take as long; bf16, whose values come eight bytes a thread, 75 for 1 row, 80 for 4, 92 for 8 (98), but 145 for 16, which tiles keep.  With the forward: 100 to
// 4000 classes, 1 row bf16 18 to 27 (27 to 36), 16 rows fp32 31 to 44 (39 to 52); fp32 rows that start anywhere, 1 x 1001 x 50257 224 (465), 3 x 333 x 50257 87 (197).
// ---------------------------------------------------------------------------------------------
constexpr int kProductThreads = 256, kClasses = 64, kAheadClasses = 8;

// Four columns of a thread: next to each other, or (kAnywhere: rows of fp32 values that do not all start on 16 bytes) `step` apart, so that a warp's are next to
// each other; `left` of the columns from the first on are inside.
template <class T, bool kAnywhere>
struct Four {
    static constexpr int kWords = sizeof(T);  // of four values
    uint32_t v[kWords];
    __device__ __forceinline__ void load(const T *p, int step, int left) {
        if constexpr (kAnywhere) {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = e * step < left ? *reinterpret_cast<const uint32_t *>(p + e * step) : 0;
        } else if constexpr (sizeof(T) == 4) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
        else *reinterpret_cast<uint2 *>(v) = *reinterpret_cast<const uint2 *>(p);
    }
    __device__ __forceinline__ void values(float (&f)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; i++) f[i] = sizeof(T) == 4 ? __uint_as_float(v[i % kWords]) : __uint_as_float(i & 1 ? v[i / 2 % kWords] & 0xffff0000u : v[i / 2 % kWords] << 16);
    }
};

template <class T, int kRows, bool kAnywhere>
__global__ void __launch_bounds__(kProductThreads, kRows <= 8 ? 2 : 1) few_rows_products_kernel(const T *__restrict__ x, long long ldx, const T *__restrict__ w, long long ldw, Ids targets,
                                                                                                const float *__restrict__ G, T *dw, long long lddw, float *__restrict__ dxp,
                                                                                                int dx_pitch, int M, int V, int K, int classes, int width) {
    pdl_launch_dependents();
    pdl_wait();
    __shared__ __align__(16) float of_class[kClasses][kRows];
    const int groups = (int)blockDim.x / width, group = (int)threadIdx.x / width, column = (int)threadIdx.x - group * width;
    const int col = kAnywhere ? (int)blockIdx.y * width * 4 + column : ((int)blockIdx.y * width + column) * 4, step = kAnywhere ? width : 1, left = K - col;
    const bool inside = left > 0;
    const int begin = blockIdx.x * classes, end = min(V, begin + classes);
    float xs[kRows][4], sum[kRows][4];
#pragma unroll
    for (int m = 0; m < kRows; m++) {
        Four<T, kAnywhere> f;
#pragma unroll
        for (int i = 0; i < f.kWords; i++) f.v[i] = 0;
        if (dw != nullptr && inside && m < M && targets.at(m, V) >= 0) f.load(x + m * ldx + col, step, left);  // rows without a target may hold anything
        f.values(xs[m]);
#pragma unroll
        for (int e = 0; e < 4; e++) sum[m][e] = 0.f;
    }
    for (int v0 = begin; v0 < end; v0 += kClasses) {
        const int count = min(kClasses, end - v0);
        __syncthreads();
        for (int i = threadIdx.x; i < count * kRows / 4; i += (int)blockDim.x)
            reinterpret_cast<float4 *>(&of_class[0][0])[i] = reinterpret_cast<const float4 *>(G + (long long)v0 * kRows)[i];
        __syncthreads();
        for (int c0 = group * kAheadClasses; c0 < count; c0 += groups * kAheadClasses) {
            Four<T, kAnywhere> ws[kAheadClasses], old[sizeof(T) == 2 ? kAheadClasses : 1];
            if (!inside) continue;
#pragma unroll
            for (int u = 0; u < kAheadClasses; u++) {
                const long long v = v0 + min(c0 + u, count - 1);
                if (dxp) ws[u].load(w + v * ldw + col, step, left);
                if (sizeof(T) == 2 && dw) old[u % (sizeof(T) == 2 ? kAheadClasses : 1)].load(dw + v * lddw + col, step, left);
            }
#pragma unroll
            for (int u = 0; u < kAheadClasses; u++) {
                if (c0 + u >= count) break;
                float f[4], add[4] = {0.f, 0.f, 0.f, 0.f};
                ws[u].values(f);
#pragma unroll
                for (int m = 0; m < kRows; m++) {
                    const float g = of_class[c0 + u][m];
#pragma unroll
                    for (int e = 0; e < 4; e++) sum[m][e] = fmaf(g, f[e], sum[m][e]), add[e] = fmaf(g, xs[m][e], add[e]);
                }
                if (!dw) continue;
                T *at = dw + (long long)(v0 + c0 + u) * lddw + col;
                if constexpr (kAnywhere) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (e * step < left) asm volatile("red.relaxed.gpu.global.add.f32 [%0], %1;" ::"l"(at + e * step), "f"(add[e]) : "memory");
                } else if constexpr (sizeof(T) == 4) {
                    asm volatile("red.relaxed.gpu.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(at), "f"(add[0]), "f"(add[1]), "f"(add[2]), "f"(add[3]) : "memory");
                } else {
                    float h[4];
                    old[u].values(h);
                    *reinterpret_cast<uint2 *>(at) = make_uint2(pack_bf16x2(h[0] + add[0], h[1] + add[1]), pack_bf16x2(h[2] + add[2], h[3] + add[3]));
                }
            }
        }
    }
    if (!dxp) return;
    if (groups > 1) {  // their sums, in order
        __shared__ float4 part[kProductThreads];
#pragma unroll
        for (int m = 0; m < kRows; m++) {
            if (m >= M) break;
            part[threadIdx.x] = make_float4(sum[m][0], sum[m][1], sum[m][2], sum[m][3]);
            __syncthreads();
            if (group == 0) {
                for (int i = 1; i < groups; i++) {
                    const float4 other = part[i * width + column];
                    sum[m][0] += other.x, sum[m][1] += other.y, sum[m][2] += other.z, sum[m][3] += other.w;
                }
            }
            __syncthreads();
        }
    }
    if (group == 0 && inside) {
#pragma unroll
        for (int m = 0; m < kRows; m++)
            if (m < M) {
                float *to = dxp + ((long long)blockIdx.x * M + m) * dx_pitch + col;
                if constexpr (kAnywhere) {
#pragma unroll
                    for (int e = 0; e < 4; e++)
                        if (e * step < left) to[e * step] = sum[m][e];
                } else {
                    *reinterpret_cast<float4 *>(to) = make_float4(sum[m][0], sum[m][1], sum[m][2], sum[m][3]);
                }
            }
    }
}

// Eight lanes read four pieces of 16 bytes each of two rows, next to each other (fp32: hi or lo of 8 values) or 32 bytes apart: the pitch keeps them in
// different banks.
int row_pitch(int K, int planes) { return (K * 2 + 127) / 128 * 128 + (planes == 2 ? 64 : 16); }
size_t shared_bytes(int M, int K, int planes) { return (size_t)(M + 15) / 16 * 16 * row_pitch(K, planes) * planes; }
constexpr size_t kMostShared = 200 << 10;

// Tiles of a CTA, the rounds of its warps, and how many warps would do in as many.
struct Split {
    int tiles, each, rounds, warps;
};
Split split_of(int V, int sms) {
    Split p;
    p.tiles = (V + 15) / 16, p.each = (p.tiles + sms - 1) / sms;
    p.rounds = (p.each + kMostWarps - 1) / kMostWarps;
    p.warps = (p.each + p.rounds - 1) / p.rounds;
    return p;
}

// Rows that can be read by 16 bytes.
bool aligned(const void *p, long long rows, long long ld, int K, int each) { return !p || (((reinterpret_cast<uintptr_t>(p) | (uintptr_t)K * each) & 15) == 0 && (rows == 1 || ld * each % 16 == 0)); }

template <class T, bool kAnywhere>
auto kernel_of(int M, bool gradient) {
    auto kernel = gradient ? few_rows_kernel<T, 1, true, kAnywhere> : M <= 16 ? few_rows_kernel<T, 1, false, kAnywhere> : few_rows_kernel<T, 2, false, kAnywhere>;
    if constexpr (sizeof(T) == 4)
        if (M > 32) kernel = few_rows_kernel<T, 3, false, kAnywhere>;
    return kernel;
}
template <class T>
cudaError_t launch(const FewRows &a, int sms, cudaStream_t s) {
    const Split p = split_of(a.V, sms);
    auto kernel = kernel_of<T, false>(a.M, a.grad_g != nullptr);
    if constexpr (sizeof(T) == 4)
        if (!aligned(a.x, a.M, a.ldx, a.K, 4) || !aligned(a.w, a.V, a.ldw, a.K, 4)) kernel = kernel_of<T, true>(a.M, a.grad_g != nullptr);
    const ToG to{a.G, a.grad_g, a.lse, a.one_g, few_rows_stride(a.M)};
    return attn::launch_after_previous(kernel, dim3((unsigned)((p.tiles + p.each - 1) / p.each)), dim3(32 * kMostWarps), shared_bytes(a.M, a.K, sizeof(T) / 2), s, static_cast<const T *>(a.x), a.ldx,
                                       static_cast<const T *>(a.w), a.ldw, a.targets, a.part, a.zt, to, a.fix, a.M, a.V, a.K, p.each * 16, row_pitch(a.K, sizeof(T) / 2));
}

// Threads along the columns of a block of the products (as many groups of them as fit share its classes), blocks along the columns, and blocks of
// classes: as many as an SM holds, since each has a piece of dx.
int product_width(int K) { return std::min(kProductThreads, ((K + 3) / 4 + 31) / 32 * 32); }
int product_columns(int K) { return (K + 4 * product_width(K) - 1) / (4 * product_width(K)); }
int product_blocks(int M, int V, int K, int sms) { return std::min(std::max(1, sms * (M <= 8 ? 2 : 1) / product_columns(K)), (V + 7) / 8); }
template <class T>
cudaError_t launch_products(const FewRows &a, T *dw, long long lddw, float *dxp, int dx_pitch, int sms, cudaStream_t s) {
    const int blocks = product_blocks(a.M, a.V, a.K, sms), classes = (a.V + blocks - 1) / blocks, stride = few_rows_stride(a.M), width = product_width(a.K);
    auto kernel = stride == 4 ? few_rows_products_kernel<T, 4, false> : few_rows_products_kernel<T, 8, false>;
    if constexpr (sizeof(T) == 4) {
        if (!aligned(a.x, a.M, a.ldx, a.K, 4) || !aligned(a.w, a.V, a.ldw, a.K, 4) || !aligned(dw, a.V, lddw, a.K, 4))
            kernel = stride == 4 ? few_rows_products_kernel<T, 4, true> : stride == 8 ? few_rows_products_kernel<T, 8, true> : few_rows_products_kernel<T, 16, true>;
        else if (stride == 16) kernel = few_rows_products_kernel<T, 16, false>;
    }
    return attn::launch_after_previous(kernel, dim3((unsigned)few_rows_pieces(a.M, a.V, a.K, sms), (unsigned)product_columns(a.K)), dim3((unsigned)(kProductThreads / width * width)), 0, s,
                                       static_cast<const T *>(a.x), a.ldx, static_cast<const T *>(a.w), a.ldw, a.targets, a.G, dw, lddw, dxp, dx_pitch, a.M, a.V, a.K, classes, width);
}

template <class T>
cudaError_t set() {
    cudaError_t e = cudaSuccess;
    auto one = [&](auto *kernel) {
        if (e == cudaSuccess) e = cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared);
    };
    for (int M : {16, 32, 48}) {
        if (sizeof(T) == 2 && M > 32) continue;
        one(kernel_of<T, false>(M, false)), one(kernel_of<T, false>(M, true));
        if constexpr (sizeof(T) == 4) one(kernel_of<T, true>(M, false)), one(kernel_of<T, true>(M, true));
    }
    return e;
}

}  // namespace

cudaError_t few_rows_set_attributes() {
    const cudaError_t e = set<float>();
    return e != cudaSuccess ? e : set<__nv_bfloat16>();
}

// (bf16 rows that start anywhere would be read by 2 bytes: the other kernel's copy is faster.)
static bool fits(const void *x, const void *w, long long ldx, long long ldw, int type, int M, int V, int K) {
    return shared_bytes(M, K, type == TENSOR_F32 ? 2 : 1) <= kMostShared && (type == TENSOR_F32 || (aligned(x, M, ldx, K, 2) && aligned(w, V, ldw, K, 2)));
}
bool few_rows_fit(const void *x, const void *w, long long ldx, long long ldw, int type, int M, int V, int K, int sms) {
    const int tiles_m = (M + 15) / 16;
    if (M > kFewRows || !fits(x, w, ldx, ldw, type, M, V, K)) return false;
    // bf16 weights: up to 32 rows, more than 16 only where the warps end together (32 x 768 x 32000, 7 warps' work in two rounds: 17.2 us, with tiles 15.7).
    const Split p = split_of(V, sms);
    return type == TENSOR_F32 || tiles_m == 1 || (tiles_m == 2 && (p.rounds == 1 || p.warps >= 9));
}
int few_rows_stride(int M) { return M <= 4 ? 4 : M <= 8 ? 8 : 16; }
bool few_rows_gradients_fit(const void *x, const void *w, const void *dw, long long ldx, long long ldw, long long lddw, int type, int M, int V, int K) {
    return M <= (type == TENSOR_F32 ? 16 : 8) && fits(x, w, ldx, ldw, type, M, V, K) && (type == TENSOR_F32 || aligned(dw, V, lddw, K, 2));
}
int few_rows_pieces(int M, int V, int K, int sms) {
    const int blocks = product_blocks(M, V, K, sms), classes = (V + blocks - 1) / blocks;
    return (V + classes - 1) / classes;
}
cudaError_t launch_few_rows_products(const FewRows &a, int type, void *dw, long long lddw, float *dxp, int dx_pitch, int sms, cudaStream_t s) {
    return type == TENSOR_F32 ? launch_products(a, static_cast<float *>(dw), lddw, dxp, dx_pitch, sms, s)
                              : launch_products(a, static_cast<__nv_bfloat16 *>(dw), lddw, dxp, dx_pitch, sms, s);
}
int few_rows_parts(int V, int sms) {
    const Split p = split_of(V, sms);
    return (p.tiles + p.each - 1) / p.each;
}
cudaError_t launch_few_rows(const FewRows &a, int type, int sms, cudaStream_t s) { return type == TENSOR_F32 ? launch<float>(a, sms, s) : launch<__nv_bfloat16>(a, sms, s); }

}  // namespace head
