// What the kernels over a paged key/value cache share: where a token's sequence, its pages and its rows are.
#pragma once

#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/attn_sm100.h"

namespace paged {

constexpr int kMaxD = 256;

// What append and attention ask of a cache and of their sizes alike.
inline int check_cache(int tokens, int seqs, int heads, int kv_heads, int D, int page_size, int pages, int width, int type, const void *k,
                       const void *v, long long page_stride) {
    if (tokens < 0 || seqs <= 0 || heads <= 0 || kv_heads <= 0 || D <= 0 || page_size <= 0 || pages <= 0 || width <= 0) return ATTN_ERR_ARGUMENT;
    if (heads % kv_heads || (type != ATTN_CACHE_F32 && type != ATTN_CACHE_BF16)) return ATTN_ERR_ARGUMENT;
    if (D % 8 || D > kMaxD || heads > 65535 || page_size > (1 << 20)) return ATTN_ERR_UNSUPPORTED;
    if ((long long)width * page_size > 0x7fffffffll - (1 << 20)) return ATTN_ERR_UNSUPPORTED;  // positions are 32-bit numbers
    const long long each = type == ATTN_CACHE_BF16 ? 2 : 4;
    if (page_stride < (long long)kv_heads * page_size * D) return ATTN_ERR_ARGUMENT;
    if ((reinterpret_cast<uintptr_t>(k) & 15) || (reinterpret_cast<uintptr_t>(v) & 15) || page_stride * each % 16) return ATTN_ERR_ALIGN;
    return ATTN_OK;
}

enum : int {
    ST_APPEND = 2001,  // a position outside its sequence's row of the page table, a page that is not there, or no angles for it
    ST_ATTEND = 2002,  // the same among the keys of a sequence, or more new tokens than max_new
};

struct Cache {
    void *k, *v;          // [pages, kv_heads, page_size, D], pages page_stride elements apart
    const int *table;     // [seqs, width]
    const int *cu;        // [seqs + 1]
    const int *past;      // [seqs]
    long long page_stride;
    int seqs, kv_heads, D, page_size, pages, width, tokens;
};

struct Span {
    int first, count, past;  // new tokens first .. first + count - 1, past tokens before them
};

// Whatever the table of lengths holds, the span lies inside the tensors.
__device__ __forceinline__ Span span_of(const Cache &c, int s) {
    Span w;
    w.first = min(max(c.cu[s], 0), c.tokens);
    w.count = min(max(c.cu[s + 1], w.first), c.tokens) - w.first;
    w.past = min(c.past[s], 0x7ffffffe - w.count);  // positions stay 32-bit numbers, beyond any page table if they were
    return w;
}

// The last sequence that begins at or before token t.  A whole warp: 32 places are looked at in a round, so up to 32
// sequences take one trip to memory and up to 1024 two.
__device__ __forceinline__ int sequence_of(const int *cu, int seqs, int t) {
    const int lane = threadIdx.x & 31;
    int lo = 0, hi = seqs;
    while (hi - lo > 1) {
        const int step = (hi - lo + 31) / 32, at = lo + (lane + 1) * step;
        const int n = __popc(__ballot_sync(0xffffffffu, at < hi && cu[at] <= t));
        lo += n * step;
        hi = min(hi, lo + step);
    }
    return lo;
}

__device__ __forceinline__ void report(int *status, int code) {
    if (status) atomicCAS(status, 0, code);
}

}  // namespace paged
