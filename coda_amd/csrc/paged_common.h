// What the ragged-batch kernels share: packed token rows cut into sequences by seq_start [B+1], and the geometry of a paged
// key/value cache.  Everything read from device memory (starts, lengths, page numbers) is clamped or tested before it is
// used as an index: a wrong entry costs rows (its own; starts that decrease, also others of the call, whose tiles are counted past
// them), never an access outside the caller's buffers.
#pragma once
#include "coda_abi_internal.h"

namespace paged {

constexpr int HEAD_DIM = 128;
constexpr int MAX_HEADS = 1 << 20;

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

__device__ __forceinline__ int clamp_start(const int* seq_start, int b, int T) { return min(max(seq_start[b], 0), T); }

// A sequence as the kernels need it: its first token row, its tokens, and its entries of two arrays by sequence (kv_len and pos0,
// adapter).  All loaded in ONE round trip, by the lane that asks for the sequence, and handed to the wave from there.
struct Seq {
    int b, s0, n, x, y;
};

struct SeqArrays {
    const int* start; const int* x; const int* y;   // x, y may be null: 0
    int B, T;
};

struct SeqLane {
    int s, e, x, y;
    __device__ __forceinline__ void load(const SeqArrays& a, int i) {
        s = clamp_start(a.start, i, a.T);
        e = clamp_start(a.start, i + 1, a.T);
        x = a.x ? a.x[i] : 0;
        y = a.y ? a.y[i] : 0;
    }
    __device__ __forceinline__ Seq from(int b, int lane) const {
        const int s0 = __builtin_amdgcn_readlane(s, lane);
        return {b, s0, __builtin_amdgcn_readlane(e, lane) - s0, __builtin_amdgcn_readlane(x, lane), __builtin_amdgcn_readlane(y, lane)};
    }
};

// The sequence that owns token row t (b = -1: none).  64 probes per step, so two dependent loads for up to 4096 sequences where a
// binary search would chain twelve.  Starts that decrease (a caller's mistake) still end with an index inside [0, B).
__device__ __forceinline__ Seq seq_of_token(const SeqArrays& a, int t) {
    const int lane = threadIdx.x & 63;
    int lo = 0, len = a.B;
    for (;;) {
        const int step = (len + 63) >> 6;
        const long long at = (long long)lane * step;
        SeqLane l = {0, 0, 0, 0};
        bool ok = at < len;
        if (ok) {
            l.load(a, lo + (int)at);
            ok = l.s <= t;
        }
        const int n = __popcll(__ballot(ok));
        if (n == 0) return {-1, 0, 0, 0, 0};
        lo += (n - 1) * step;
        if (step == 1) {
            Seq q = l.from(lo, n - 1);
            if (t - q.s0 >= q.n) q.b = -1;
            return q;
        }
        len = min(step, len - (n - 1) * step);
    }
}

// inclusive running sum over the lanes of a wave
__device__ __forceinline__ int wave_running_sum(int v) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int w = __shfl_up(v, o, 64);
        if (lane >= o) v += w;
    }
    return v;
}

// 256 sequences, four per lane, all loads in flight at once
struct SeqBlock {
    SeqLane l[4];
    __device__ __forceinline__ void load(const SeqArrays& a, int c) {
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int i = c + 64 * u + (int)(threadIdx.x & 63);
            l[u] = {0, 0, 0, 0};
            if (i < a.B) l[u].load(a, i);
        }
    }
};

// rows -> tiles of R rows; rows = tokens * heads < 2^31
template <int R>
__device__ __forceinline__ int tiles_of(const SeqLane& l, int g) {
    const int rows = max(l.e - l.s, 0) * g;
    return rows / R + (rows % R != 0);
}

// Item `item` of all the sequences' items (tiles, or tiles times key ranges), sequence i having count(its SeqLane) of them: a running
// sum over the sequences.  Items are numbered without gaps: a numbering that leaves idle ones between the sequences is cheaper to
// invert, but workgroups go round the eight XCDs by number, and a pattern of idle ones then leaves whole XCDs without work (32
// sequences of one tile each on every other number: attention took 38 us where 23 do).  `k`: the item's place in its sequence.
// b = -1: there are fewer items.  `blk` holds the first 256 sequences.
template <class F>
__device__ __forceinline__ Seq seq_of_item(const SeqArrays& a, SeqBlock& blk, int item, int& k, F count) {
    int base = 0;
    for (int c = 0; c < a.B; c += 256) {
        if (c) blk.load(a, c);
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            if (c + 64 * u >= a.B) break;
            const int mine = count(blk.l[u]), sum = wave_running_sum(mine);
            const unsigned long long past = __ballot(sum > item - base);
            if (past) {
                const int w = __ffsll((long long)past) - 1;
                k = item - base - __builtin_amdgcn_readlane(sum - mine, w);
                return blk.l[u].from(c + 64 * u + w, w);
            }
            base += __builtin_amdgcn_readlane(sum, 63);         // <= item: cannot overflow
        }
    }
    k = 0;
    return {-1, 0, 0, 0, 0};
}

// A launch holds fewer than 2^32 work items: what has more is refused in words before anything is launched.
inline bool grid_fits(long long workgroups, int threads) { return workgroups * threads <= 0xffffffffLL; }

}  // namespace paged

// Host-side checks common to the entry points that take a paged cache; 0 or an error code (with words).
int coda_check_pages(const char* who, const void* k_cache, const void* v_cache, const int* page_table, long long ld_table, int max_pages,
                     long long page_stride, int num_pages, int page_size, int cache_type, float k_scale, float v_scale, int n_kv,
                     paged::Pages* out);
int coda_refuse(const char* who, int code, const char* why);
