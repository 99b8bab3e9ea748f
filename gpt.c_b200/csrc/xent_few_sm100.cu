// The forward of projection and loss (xent_linear_sm100.cu) for few rows: the weights are read once, straight into registers, for sm_100a.
//
// With up to 64 rows the products are few and the weights all that has to be moved.  The tiles of the other kernel have half of their shared memory
// for rows that are not there, and fp32 weights are written and read again as bf16 planes.  Here a warp takes 16 classes at a time: a lane reads eight
// values of a row, 32 or 16 bytes, which are the lane's part of two mma fragments if the contraction is taken in that order, and splits fp32 values into
// hi and lo on the way.  x is in shared memory, bf16 (hi and lo), its rows so far apart that eight lanes that read two of them meet no bank twice.
// Maximum and sum of each row stay in registers until the end.
//
// Bound by HBM where there are up to 16 rows, then by the products (mma.sync has a quarter of the rate) and what they wait for.  Classes of 768 features, us with the
// join, in brackets with tiles: 16 x 50257 bf16 18.7 (25.4), fp32 38 (110); 32 rows 22.3 (24.9), 45 (103); 48 rows 25.7 (22.8), 57 (104); 32 x 8000 13.4 (12.5),
// 23 (25); 16 x 32000 bf16, whose CTAs have work for seven warps, 17.5 (15.8).  Reading takes 12 us of bf16 and 24 of fp32 weights.
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
    __device__ __forceinline__ void load(const T *p, int left) {  // `left`: values that are inside, a multiple of 8
        if (left >= kValues) {
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                         : "l"(p));
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = 0;
            if (sizeof(T) == 2 && left > 0) *reinterpret_cast<uint4 *>(v) = *reinterpret_cast<const uint4 *>(p);
        }
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

// kTiles: of 16 rows of x.  `classes`: of a CTA, a multiple of 16.
template <class T, int kTiles>
__global__ void __launch_bounds__(32 * kMostWarps) few_rows_kernel(const T *__restrict__ x, long long ldx, const T *__restrict__ w, long long ldw, Ids targets,
                                                                   float2 *__restrict__ part, float *__restrict__ zt, int M, int V, int K, int classes, int pitch) {
    pdl_launch_dependents();
    pdl_wait();
    extern __shared__ __align__(16) uint8_t rows[];  // [plane][16 kTiles][pitch bytes]
    __shared__ float2 all[kMostWarps][16 * kTiles];
    constexpr int kPlanes = sizeof(T) / 2, kAhead = 3, kBlock = 128 / sizeof(T), kEach = Piece<T>::kValues, kWords = kEach / 2;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5, g = lane >> 2, q = lane & 3;
    const int class0 = blockIdx.x * classes, tiles = (min(V, class0 + classes) - class0 + 15) / 16, blocks = (K + kBlock - 1) / kBlock;
    const int mine = tiles > warp ? (tiles - warp + warps - 1) / warps : 0, total = mine * blocks;

    // what is asked for next: block load_b of tile load_t
    Piece<T> ahead[kAhead][2];
    int load_b = 0, load_t = warp;
    const T *from[2];
    auto rows_of = [&](int t) {
#pragma unroll
        for (int r = 0; r < 2; r++) from[r] = w + (long long)min(class0 + 16 * t + 8 * r + g, V - 1) * ldw + kEach * q;
    };
    auto ask = [&](Piece<T>(&to)[2], int n) {
#pragma unroll
        for (int r = 0; r < 2; r++) to[r].load(from[r] + kBlock * load_b, n < total ? K - kBlock * load_b - kEach * q : 0);
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
        e.load(x + row * ldx + c, row < M ? K - c : 0);
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
            ask(ahead[u], n0 + u + kAhead);
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
            if (++b < blocks) continue;
            b = 0;
            // 16 classes are done: a lane has classes 8 r + 2 q and the next of rows g and 8 + g of each tile
            const int first = class0 + 16 * t + 2 * q;
            t += warps;
#pragma unroll
            for (int m = 0; m < kTiles; m++)
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    float v[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const int c = first + 8 * (i / 2) + i % 2;
                        v[i] = c < V ? z[m][i / 2][2 * h + i % 2] : -INFINITY;
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
    if (row >= M) return;
    float m = -INFINITY, s = 0.f;
    for (int i = 0; i < warps; i++) join(m, s, all[i][row].x, all[i][row].y);
    part[(long long)blockIdx.x * M + row] = make_float2(m, s);
}

// Eight lanes read four pieces of 16 bytes each of two rows, next to each other (fp32: hi or lo of 8 values) or 32 bytes apart.
int row_pitch(int K, int planes) { return (K * 2 + 127) / 128 * 128 + (planes == 2 ? 64 : 16); }
size_t shared_bytes(int M, int K, int planes) { return (size_t)(M + 15) / 16 * 16 * row_pitch(K, planes) * planes; }
constexpr size_t kMostShared = 200 << 10;

// Tiles of a CTA, and its warps: as many as end together.
struct Split {
    int tiles, each, rounds, warps;
};
Split split_of(int M, int V, int sms) {
    Split p;
    p.tiles = (V + 15) / 16, p.each = (p.tiles + sms - 1) / sms;
    p.rounds = (p.each + kMostWarps - 1) / kMostWarps;
    p.warps = std::max((p.each + p.rounds - 1) / p.rounds, (M + 31) / 32);
    return p;
}

template <class T>
cudaError_t launch(const FewRows &a, int sms, cudaStream_t s) {
    const auto [tiles, each, rounds, warps] = split_of(a.M, a.V, sms);
    auto kernel = a.M <= 16 ? few_rows_kernel<T, 1> : a.M <= 32 ? few_rows_kernel<T, 2> : a.M <= 48 ? few_rows_kernel<T, 3> : few_rows_kernel<T, 4>;
    return attn::launch_after_previous(kernel, dim3((unsigned)((tiles + each - 1) / each)), dim3(32 * warps), shared_bytes(a.M, a.K, sizeof(T) / 2), s, static_cast<const T *>(a.x), a.ldx,
                                       static_cast<const T *>(a.w), a.ldw, a.targets, a.part, a.zt, a.M, a.V, a.K, each * 16, row_pitch(a.K, sizeof(T) / 2));
}

template <class T>
cudaError_t set() {
    cudaError_t e = cudaSuccess;
    for (auto kernel : {few_rows_kernel<T, 1>, few_rows_kernel<T, 2>, few_rows_kernel<T, 3>, few_rows_kernel<T, 4>})
        if (e == cudaSuccess) e = cudaFuncSetAttribute(reinterpret_cast<const void *>(kernel), cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kMostShared);
    return e;
}

}  // namespace

cudaError_t few_rows_set_attributes() {
    const cudaError_t e = set<float>();
    return e != cudaSuccess ? e : set<__nv_bfloat16>();
}

bool few_rows_fit(const void *x, const void *w, long long ldx, long long ldw, int type, int M, int V, int K, int sms) {
    const int each = type == TENSOR_F32 ? 4 : 2, tiles_m = (M + 15) / 16;
    if (M > kFewRows || K % 8 || shared_bytes(M, K, each / 2) > kMostShared) return false;
    if (((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 31) || (M > 1 && ldx * each % 32) || ldw * each % 32) return false;
    // fp32 weights: from about as many classes on as the planes of the other way take time for.  bf16 ones: up to 32 rows, and warps enough.
    if (type == TENSOR_F32) return V >= 4000 * tiles_m;
    const Split p = split_of(M, V, sms);
    return tiles_m <= 2 && V >= 8000 && (p.rounds == 1 || p.warps >= 10);
}
int few_rows_parts(int V, int sms) {
    const Split p = split_of(1, V, sms);
    return (p.tiles + p.each - 1) / p.each;
}
cudaError_t launch_few_rows(const FewRows &a, int type, int sms, cudaStream_t s) { return type == TENSOR_F32 ? launch<float>(a, sms, s) : launch<__nv_bfloat16>(a, sms, s); }

}  // namespace head
