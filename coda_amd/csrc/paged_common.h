// What the ragged-batch kernels share: packed token rows cut into sequences by seq_start [B+1], and the geometry of a paged
// key/value cache.  Everything read from device memory (starts, lengths, page numbers) is clamped or tested before it is
// used as an index: a wrong entry costs the rows it describes, never an access outside the caller's buffers.
#pragma once
#include "coda_abi_internal.h"

namespace paged {

constexpr int HEAD_DIM = 128;

// n / d for 0 <= n < 2^31 and 1 <= d < 2^31 as multiply-high, add, shift (round-up method: magic = ceil(2^(32+s) / d) - 2^32
// with s = ceil(log2 d); the sum of the high product and n stays below 2^32).  Page sizes are the caller's and need not be
// powers of two.
struct FastDiv {
    unsigned int magic, shift, d;
};

inline FastDiv make_fast_div(unsigned int d) {
    FastDiv f;
    f.d = d;
    f.shift = 0;
    while ((1ull << f.shift) < d) ++f.shift;
    f.magic = (unsigned int)(((1ull << f.shift) - d) * (1ull << 32) / d + 1);
    if (d == 1) f.magic = 0;
    return f;
}

__device__ __forceinline__ int fast_div(const FastDiv& f, int n) {
    return (int)((__umulhi((unsigned int)n, f.magic) + (unsigned int)n) >> f.shift);
}

// Pages [num_pages][n_kv][page_size][128]; K and V have the same geometry.
struct Pages {
    const int* table; long long ld_table;     // [B, max_pages] page numbers
    int max_pages, num_pages;
    FastDiv page;                             // page.d = page_size
    long long page_stride_b;                  // bytes from page to page
    long long head_stride_b;                  // bytes from head to head inside a page
    int row_b;                                // bytes of one key or value: 256 (bf16) or 128 (e4m3)
};

// Index of the last b in [0, B) with f(b) <= x, or -1: f must not decrease.  64 probes per step, so two dependent loads for
// up to 4096 sequences where a binary search would chain twelve.  Every lane of the wave gets the answer.  An f that does
// decrease (a caller's mistake) still ends with an index inside [0, B).
template <class F>
__device__ __forceinline__ int wave_search(int B, long long x, F f) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = B;
    for (;;) {
        const int step = (len + 63) >> 6;
        const long long at = (long long)lane * step;
        const bool ok = at < len && f(lo + (int)at) <= x;
        const int n = __popcll(__ballot(ok));
        if (n == 0) return -1;
        lo += (n - 1) * step;
        len = min(step, len - (n - 1) * step);
        if (step == 1) return lo;
    }
}

__device__ __forceinline__ int clamp_start(const int* seq_start, int b, int T) { return min(max(seq_start[b], 0), T); }

}  // namespace paged

// Host-side checks common to the entry points that take a paged cache; 0 or an error code (with words).
int coda_check_pages(const char* who, const void* k_cache, const void* v_cache, const int* page_table, long long ld_table, int max_pages,
                     long long page_stride, int num_pages, int page_size, int cache_type, float k_scale, float v_scale, int n_kv,
                     paged::Pages* out);
int coda_refuse(const char* who, int code, const char* why);
