// Attention of new tokens over a paged key/value cache, head_dim 128.
//
//     out_i = sum_j softmax_j(scale q_i . K_j) V_j over the keys j < lim(i) of the token's sequence
//
// One pass over the keys with a running maximum and sum (in log2 units).  Where there are too few rows to fill the chip, or rows of
// very different lengths, the keys are cut into ranges and a second kernel joins the ranges' (maximum, sum, unnormalised output)
// triples in fp32, in a fixed order.  How long a range is comes from the lengths on the device (see cut_of): the host knows only bounds.
//
// Rows.  The g = n_q / n_kv query heads of a key/value head read the same keys, so a sequence of n tokens is n g ROWS per
// key/value head (row r = token r / g, head r % g) and tiles are cut from those: one token of a g = 2 model is two rows of one
// tile, a block of 32 tokens is 64.
//
// Two kernels: `few` (16 or 32 rows a workgroup; waves share the KEYS) for single tokens and short blocks, `many` (128 or 256 rows; waves
// share the ROWS) for longer ones; make_plan has the rule and what both sides of it measured.  Both compute S^T[key][row] = K Q^T, so
// that a lane holds scores of one row and its accumulators are directly the B operand of O^T[d][row] += V^T P^T, whose A operand
// is read from LDS with the transposing ds_read_b64_tr_b16.
// LDS image of a K or V tile: 256 B a key (bf16 also for e4m3 pages: the conversion is exact), 16-byte chunk ch of key r at
// ch ^ swz(r): free of bank conflicts for both kinds of read.
//
// Pages come in through registers (loads of the NEXT tile fly under the current tile's products): keys of a tile may lie on different
// pages, e4m3 is converted on the way, scores of keys that a row does not see are replaced, and values of keys beyond the
// sequence or on an invalid page are zeroed on the way to LDS, so that whatever their slots hold (infinities, NaN) cannot reach the
// sums through 0 * x.  Whole bf16 tiles of the `many` kernel need none of that and are copied to LDS directly.
#include "paged_common.h"
#include <type_traits>

using namespace paged;

namespace {

constexpr float RESCALE_THR = 6.0f;            // log2 units: weights stay below 2^6 between rescales

struct AttnArgs {
    const char* q; long long ldq_b;
    char* out; long long ldo_b;
    const int* seq_start; const int* pos0; const int* kv_len;
    int B, T, max_kv;
    Pages pg;
    const char* k; const char* v;
    int n_q, n_kv, g;
    FastDiv gdiv;
    int mask_block, slanted;                   // slanted: the keys that a mask hides count in how the work is cut
    float scale_log2e, v_scale;
    int max_ranges;                            // 1: keys are not cut
    int min_keys; float per_range;             // a range: at least min_keys keys, and sum(tiles * keys) * per_range
    float* po; float* pml;                     // partial outputs [max_ranges][T n_q][128] and (maximum, sum) [max_ranges][T n_q][2]
    int* range_keys;                           // the range length that the first kernel took, for the second
};

// row bits 0..3 to the 16 chunk positions; the low two so that the transposing reads of 16 keys (few rows) fall on different banks too
__device__ __forceinline__ int swz(int row) { return ((row & 3) << 2) | ((row >> 1) & 2) | ((row >> 3) & 1); }

typedef __attribute__((ext_vector_type(8))) short s16x8_t;

// A tile of R rows of one sequence and a range of its keys; what its rows see: all of the sequence's kv keys, or those before the end
// of the row's mask block.
struct TileRows {
    int b, s0, n;        // sequence, its first token row, its tokens
    int r0, rows;        // first row of the tile, rows of the sequence
    int range, keys;     // range of keys and its length
};

struct Limits {
    int kv, pos0;
};

// Keys of a sequence of n tokens.  slanted: those that some of its tokens see under the mask, which end at most mask_block keys behind the
// last token.
__device__ __forceinline__ int kv_of(const AttnArgs& a, int kv_len, int pos0, int n) {
    const int kv = min(max(kv_len, 0), a.max_kv);
    if (!a.slanted) return kv;
    return min(kv, max(__builtin_elementwise_add_sat(__builtin_elementwise_add_sat(pos0, n), a.mask_block), 0));
}

__device__ __forceinline__ int kv_of(const AttnArgs& a, const SeqLane& l) { return kv_of(a, l.x, l.y, l.e - l.s); }

__device__ __forceinline__ Limits limits_of(const AttnArgs& a, const Seq& q) { return {kv_of(a, q.x, q.y, q.n), q.y}; }

// Length of the ranges of a sequence with kv keys: ceil(kv / range_keys) equal ones, in whole 128 keys
__device__ __forceinline__ int keys_of(int kv, int range_keys) {
    const int n = max(1, (kv + range_keys - 1) / range_keys);
    return max(((kv + n - 1) / n + 127) & ~127, 128);           // also for no keys: it is divided by
}

// Uncut calls with a mask: tiles are taken longest first, over all sequences, so that the last ones to start are short (eight causal
// sequences of 2048 tokens are 1024 tiles of 1 .. 16 lengths on 256 CUs: in sequence order the last CU ends 19 % after the average).
// Tile k of a sequence sees about min(kv, pos0 + (k + 1) R / g) keys, which grows with k, so how many of its tiles see at least `keys`
// is a formula and the order needs no sorting: lane j counts the tiles of at least the j-th of 33 thresholds.  For up to 16 sequences: the
// search walks over all of them, and tiles of one sequence that run at different times no longer find its keys in the L2 (us with / without:
// 4 x 2048 tokens 129 / 166, 8 x 2048 238 / 263, 16 x 1000 behind 500 241 / 264, but 30 x 600 131 / 126, 32 x 384 79 / 65).
constexpr int LONGEST_FIRST = 16, LEVELS = 32;

struct Cost {
    int tiles, kv, pos0;                       // of one sequence
    template <int R>
    __device__ __forceinline__ int at_least(const AttnArgs& a, int keys) const {       // tiles that see `keys` or more
        if (kv < keys) return 0;
        const long long need = max((long long)keys - pos0, 0ll) * a.g;
        return max(tiles - max((int)min((need + R - 1) / R, 0x7fffffffll) - 1, 0), 0);
    }
};

// -> the sequence, k: its tile; b = -1: none
template <int R>
__device__ __forceinline__ Seq longest_first(const AttnArgs& a, const SeqLane& l, int item, int& k) {
    const int lane = threadIdx.x & 63;
    const Cost mine = {tiles_of<R>(l, a.g), kv_of(a, l), max(l.y, 0)};
    auto of = [&](int b) {
        return Cost{__builtin_amdgcn_readlane(mine.tiles, b), __builtin_amdgcn_readlane(mine.kv, b), __builtin_amdgcn_readlane(mine.pos0, b)};
    };
    int hi = 0;
    for (int b = 0; b < a.B; ++b) hi = max(hi, of(b).kv);
    const int step = hi / LEVELS + 1;
    auto threshold = [&](int j) { return max(hi + 1 - j * step, 0); };      // none .. all
    const int keys = threshold(min(lane, LEVELS));
    int total = 0;
    for (int b = 0; b < a.B; ++b) total += of(b).template at_least<R>(a, keys);
    const unsigned long long fewer = __ballot(total <= item);               // a run of ones from lane 0
    const int j = __popcll(fewer) - 1;
    k = 0;
    if (j >= LEVELS) return {-1, 0, 0, 0, 0};
    const int before = lane < a.B ? mine.at_least<R>(a, threshold(j)) : 0;
    const int here = lane < a.B ? mine.at_least<R>(a, threshold(j + 1)) - before : 0;
    const int sum = wave_running_sum(here), left = item - __builtin_amdgcn_readlane(total, j);
    const int b = __ffsll((long long)__ballot(sum > left)) - 1;
    k = __builtin_amdgcn_readlane(mine.tiles - 1 - before, b) - (left - __builtin_amdgcn_readlane(sum - here, b));
    return l.from(b, b);
}

// Work unit -> tile and range.  The longest a range may be follows from the whole work, sum over the sequences of tiles * keys, so that
// the units come out about equal and about as many as the chip takes at once (or in a few rounds): every wave adds the lengths up for
// itself, in the same order.
template <int R, bool LONGEST>
__device__ __forceinline__ bool find_unit(const AttnArgs& a, int unit, TileRows& t, Limits& lm) {
    const SeqArrays arr = {a.seq_start, a.kv_len, a.pos0, a.B, a.T};
    SeqBlock blk;
    blk.load(arr, 0);
    int range_keys = 0x40000000;
    if (a.max_ranges > 1) {
        float work = 0.f;
        for (int c = 0; c < a.B; c += 256) {
            SeqBlock more;
            if (c) more.load(arr, c);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const SeqLane& l = c ? more.l[u] : blk.l[u];
                const int kv = kv_of(a, l);                     // slanted: the tiles see from about pos0 to all of them
                work += (float)tiles_of<R>(l, a.g) * (a.slanted ? 0.5f * ((float)kv + (float)min(kv, max(l.y, 0))) : (float)kv);
            }
        }
        work = wave_sum(work);
        range_keys = max(a.min_keys, ((int)fminf(work * a.per_range, 1.2e9f) + 128) & ~127);       // more than any kv_len: one range
        if (blockIdx.x == 0 && threadIdx.x == 0) *a.range_keys = range_keys;
    }
    int k;
    Seq q;
    if (LONGEST && a.max_ranges == 1 && a.mask_block && a.B <= LONGEST_FIRST) {
        q = longest_first<R>(a, blk.l[0], unit, k);
    } else {
        q = seq_of_item(arr, blk, unit, k, [&](const SeqLane& l) {
            const int kv = kv_of(a, l);
            return tiles_of<R>(l, a.g) * (a.max_ranges > 1 ? max(1, (kv + range_keys - 1) / range_keys) : 1);
        });
        // later tiles of a sequence see more keys under a mask: they go first
        const int ranges = max(1, (kv_of(a, q.x, q.y, q.n) + range_keys - 1) / range_keys), rows = q.n * a.g, tiles = rows / R + (rows % R != 0);
        k = (tiles - 1 - k / ranges) * ranges + k % ranges;
    }
    if (__builtin_amdgcn_readfirstlane(q.b) < 0) return false;
    lm = limits_of(a, q);
    const int rows = q.n * a.g, ranges = max(1, (lm.kv + range_keys - 1) / range_keys);
    // All of this is the same in every lane, which the compiler does not find out by itself (loops, ballots): told so, it keeps what
    // follows from it - bounds, page bases, branches - in scalar registers.
    auto u = [](int v) { return __builtin_amdgcn_readfirstlane(v); };
    t = {u(q.b), u(q.s0), u(q.n), u(k / ranges * R), u(rows), u(k % ranges), u(keys_of(lm.kv, range_keys))};
    lm = {u(lm.kv), u(lm.pos0)};
    return true;
}

__device__ __forceinline__ int limit_of(const AttnArgs& a, const Limits& l, int token) {
    if (a.mask_block == 0) return l.kv;
    const long long p = (long long)l.pos0 + token;
    if (p < 0) return 0;
    const long long end = ((long long)((unsigned int)p / (unsigned int)a.mask_block) + 1) * a.mask_block;
    return (int)min((long long)l.kv, end);
}

// byte offset of key `key` (of this sequence and head) inside the cache; ok = false for keys outside [0, end) and bad pages
struct KeyAt {
    size_t off; bool ok;
};

__device__ __forceinline__ int page_entry(const AttnArgs& a, const int* table, int key, int end) {
    return key < end ? table[fast_div(a.pg.page, key)] : -1;
}

__device__ __forceinline__ KeyAt key_at(const AttnArgs& a, int entry, int key) {
    KeyAt k;
    k.ok = (unsigned)entry < (unsigned)a.pg.num_pages;
    const int slot = key - fast_div(a.pg.page, key) * (int)a.pg.page.d;
    k.off = k.ok ? (size_t)entry * a.pg.page_stride_b + (size_t)slot * a.pg.row_b : 0;
    return k;
}

__device__ __forceinline__ size_t shfl_size(size_t v, int src) {
    const unsigned lo = __shfl((int)(unsigned)v, src, 64), hi = __shfl((int)(unsigned)(v >> 32), src, 64);
    return ((size_t)hi << 32) | lo;
}

// Where the keys of a range are, looked up ahead.
// Pages of a multiple of 16 keys (G16): 16 aligned keys lie on one page, one after the other.  Lane l holds the offset of 16-key group
// 64 w + l of window w (1024 keys), so a tile's groups come out by readlane as wave-uniform bases, their keys are whole contiguous
// KiB at constant offsets from them, and most tiles cost no look-up at all.
// Other page sizes: lane l holds the offset of key l of the tile.  On the same pages this takes a little longer: 9.8 us against 9.4 (one
// token, 1000 keys), 72.7 against 70.6 (128 single tokens, 333 MB of e4m3), 219 against 217 (prompts).
template <int KEYS, bool G16>
struct PageSource {
    static constexpr int UNIT = G16 ? 16 : 1, SPAN = G16 ? 64 : KEYS;     // keys per lane, lanes per look-up
    unsigned int lo, hi;                       // offset inside the cache
    unsigned long long there;                  // lanes whose page exists
    int entry;                                 // page number of the next look-up, on its way
    int at;                                    // next look-up (window or tile)

    __device__ __forceinline__ int key_of(int w) const { return (w * SPAN + (int)(threadIdx.x & (SPAN - 1))) * UNIT; }
    // `first`: tile
    __device__ __forceinline__ void start(const AttnArgs& a, const int* table, int k_lo, int k_hi, int first) {
        at = G16 ? first * (KEYS / 16) / 64 : first;
        entry = page_entry(a, table, k_lo + key_of(at), k_hi);
    }
    // makes tile t's keys known and sends for what a later one needs (G16: the next window; else the tile after t by `step`)
    __device__ __forceinline__ void advance(const AttnArgs& a, const int* table, int k_lo, int k_hi, int t, int step) {
        if (G16 && t * (KEYS / 16) / 64 != at) return;          // still the window before
        const KeyAt k = key_at(a, entry, k_lo + key_of(at));
        lo = (unsigned)k.off;
        hi = (unsigned)(k.off >> 32);
        there = __ballot(k.ok);
        at += G16 ? 1 : step;
        entry = page_entry(a, table, k_lo + key_of(at), k_hi);
    }
    // keys of tile t that exist, lowest bit first
    __device__ __forceinline__ unsigned long long exist(int k_lo, int k_hi, int t) const {
        constexpr unsigned long long ALL = KEYS == 64 ? ~0ull : (1ull << (KEYS & 63)) - 1;
        if (!G16) return there & ALL;
        constexpr int G = KEYS / 16;
        const unsigned int g = (unsigned int)(there >> (t * G & 63)) & ((1u << G) - 1);
        if (g == (1u << G) - 1 && k_lo + (t + 1) * KEYS <= k_hi) return ALL;
        unsigned long long ok = 0;
#pragma unroll
        for (int i = 0; i < G; ++i) {
            const int live = (g >> i) & 1 ? min(max(k_hi - k_lo - t * KEYS - 16 * i, 0), 16) : 0;
            ok |= (unsigned long long)((1u << live) - 1u) << (16 * i);
        }
        return ok;
    }
    // G16: uniform offset of group i of tile t
    __device__ __forceinline__ size_t group(int t, int i) const {
        const int l = (t * (KEYS / 16) + i) & 63;
        return ((size_t)(unsigned)__builtin_amdgcn_readlane((int)hi, l) << 32) | (unsigned)__builtin_amdgcn_readlane((int)lo, l);
    }
    // else: offset of key i (per lane)
    __device__ __forceinline__ size_t key(int i) const { return shfl_size(((size_t)hi << 32) | lo, i); }
};

// four e4m3 bytes -> four bf16 (exact: three mantissa bits, exponents within bf16's)
__device__ __forceinline__ u32x2_t bf16_of_e4m3(unsigned int w) {
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
    const auto hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    u32x2_t o;
    o[0] = pack_bf16x2(lo[0], lo[1]);
    o[1] = pack_bf16x2(hi[0], hi[1]);
    return o;
}

// bf16 infinities and NaN of a 16-byte piece set to zero; true if there were any
__device__ __forceinline__ bool drop_nonfinite(u32x4_t& v) {
    bool any = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const bool lo = (v[i] & 0x7f80u) == 0x7f80u, hi = (v[i] & 0x7f800000u) == 0x7f800000u;
        if (lo) v[i] &= 0xffff0000u;
        if (hi) v[i] &= 0x0000ffffu;
        any |= lo | hi;
    }
    return any;
}

// A tile that some row sees only in part holds values of keys that other rows must not feel, and the products cannot skip
// them: 0 * inf = NaN.  Staging such a tile drops its infinities and NaN from the LDS image; if there were any, this finds
// the outputs they belong to: those features of the rows that do see their key come out as NaN.  Bit e of the answer stands for
// feature feature(e), e < n.  Rare, and slow on purpose: a rolled loop that needs no registers.
template <bool F8, class F>
__device__ __forceinline__ unsigned long long find_nonfinite(const AttnArgs& a, const int* table, size_t head_off, int key0, int nkeys,
                                                             int end, int lim, int n, F feature) {
    unsigned long long bits = 0;
#pragma unroll 1
    for (int j = 0; j < nkeys; ++j) {
        const int key = key0 + j;
        const KeyAt at = key_at(a, page_entry(a, table, key, end), key);
        if (key >= end || !at.ok || key >= lim) continue;
        const char* p = a.v + head_off + at.off;
#pragma unroll 1
        for (int e = 0; e < n; ++e) {
            const int d = feature(e);
            const bool bad = F8 ? (((const unsigned char*)p)[d] & 0x7f) == 0x7f : (((const unsigned short*)p)[d] & 0x7f80) == 0x7f80;
            if (bad) bits |= 1ull << e;
        }
    }
    return bits;
}

// output row of a tile row: token row and head
struct RowAt {
    int token, head;
};

__device__ __forceinline__ RowAt row_at(const AttnArgs& a, const TileRows& t, int kvh, int r) {
    const int i = fast_div(a.gdiv, r);
    return {t.s0 + i, kvh * a.g + (r - i * a.g)};
}

// one row's 8 consecutive outputs (d0..): normalised bf16 to `out`, or fp32 partials
__device__ __forceinline__ u32x4_t pack8(const float (&f)[8]) {
    u32x4_t v;
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = pack_bf16x2(f[2 * i], f[2 * i + 1]);
    return v;
}

// weight of a part with maximum m in a sum with maximum mm; a part without a maximum holds zeros (or NaN): nothing to scale
__device__ __forceinline__ float part_weight(float m, float mm) { return m == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - mm); }

// Writes a lane's 16 bytes of a K or V piece (4 bf16 or 8 e4m3 keys) into a tile image: bf16 rows of 256 B, chunk ch of key r at
// ch ^ swz(r).  PART (V images): keys that do not exist become zeros, and so do infinities and NaN; true if there were any of those.
template <bool F8>
struct ImageWriter {
    int row0, at0;                             // key within the piece, and its byte offset with the swizzle's lane-dependent part
    __device__ __forceinline__ explicit ImageWriter(int lane) {
        row0 = F8 ? lane >> 3 : lane >> 4;
        const int ch = F8 ? 2 * (lane & 7) : lane & 15;
        at0 = row0 * 256 + ((ch ^ swz(row0)) << 4);
    }
    template <bool PART>
    __device__ __forceinline__ bool put(char* img, int piece, const u32x4_t& v, unsigned long long ok) const {
        bool dropped = false;
        const bool live = !PART || ((ok >> (piece * (F8 ? 8 : 4) + row0)) & 1);
        const u32x4_t zero = {0, 0, 0, 0};
        // swz(a + b) = swz(a) ^ swz(b) for parts without common bits
        if (F8) {
            const int at = piece * 2048 + (at0 ^ (swz(8 * (piece & 1)) << 4));
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const u32x2_t v0 = bf16_of_e4m3(v[2 * j]), v1 = bf16_of_e4m3(v[2 * j + 1]);
                u32x4_t w = {v0[0], v0[1], v1[0], v1[1]};
                if (PART) {
                    if (!live) w = zero;
                    dropped |= drop_nonfinite(w);
                }
                *(u32x4_t*)(img + (at ^ (j << 4))) = w;
            }
        } else {
            u32x4_t w = v;
            if (PART) {
                if (!live) w = zero;
                dropped = drop_nonfinite(w);
            }
            *(u32x4_t*)(img + piece * 1024 + (at0 ^ (swz(4 * (piece & 3)) << 4))) = w;
        }
        return dropped;
    }
};

// four keys x 16 features, transposed on the way: lane i of a group of 16 addresses 8 bytes (key i >> 2, features 4 (i & 3) ..) and
// receives feature i of the four keys
__device__ __forceinline__ s16x4_t read_transposed(const char* p) { return __builtin_amdgcn_ds_read_tr16_b64_v4i16((CODA_LDS s16x4_t*)p); }

__device__ __forceinline__ bf16x8_t join4(s16x4_t a, s16x4_t b) {
    const s16x8_t v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(bf16x8_t, v);
}

// ---------------------------------------------------------------------------------------------------------------------
// Few rows: RG groups of 16.  Four waves take tiles of 32 keys in turn, each with its own V image, maximum, sum and output; they meet
// once, at the end.  No barrier in the loop.
//
// What bounds it: the bytes of the cache (decode), or the latency of one tile after the other (short sequences).  So the next tile's
// pages are in flight under this one's products, K goes from memory straight into the A fragments of v_mfma_f32_16x16x32_bf16 (a
// quarter-wave reads 64 B of a key, the fragments of a tile are whole lines) and only V passes LDS, for its transposition.
// Measured (16 heads on 8, one token a sequence): 128 x 2000 keys bf16 181 us = 5.8 TB/s, 128 x 4000 e4m3 189 us = 5.6 TB/s, 1 x 100000 81 us =
// 5.0 TB/s with its join; 32 blocks of 32 tokens behind 2000 keys 65 us = 4.3 TB/s.  A large copy reaches 5.2 TB/s.
//   S^T[key][row]:  lane -> row lane & 15, keys 16 kt + 4 quad + i          (quad = lane >> 4)
//   P^T as B:       k index (quad, j) is key 16 (j >> 2) + 4 quad + (j & 3): the accumulators as they are
//   O^T[d][row]:    lane -> row lane & 15, features 16 dt + 4 quad + i
constexpr int FEW_TILE = 32;                                    // keys per tile
constexpr int FEW_WAVE_LDS = FEW_TILE * 256;                    // V image, then 16 rows of fp32 output: 8 KiB a wave

template <int RG, bool F8, bool G16>
__global__ __launch_bounds__(256, RG == 1 && F8 ? 3 : 2) void paged_attn_few_kernel(AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int R = 16 * RG;
    constexpr int NP = F8 ? 4 : 8;                              // 1 KiB pieces of a K or V tile
    __shared__ float ml[4][2][16 * RG];
    const int lane = threadIdx.x & 63, kw = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 15, quad = lane >> 4;
    const int kvh = blockIdx.x % a.n_kv;
    TileRows tr;
    Limits lm;
    if (!find_unit<R, false>(a, blockIdx.x / a.n_kv, tr, lm)) return;
    const int last = min(tr.r0 + R, tr.rows) - 1;               // last live row of the tile
    const int end = __builtin_amdgcn_readfirstlane(limit_of(a, lm, fast_div(a.gdiv, last)));    // keys that any row of the tile sees
    const int all = __builtin_amdgcn_readfirstlane(limit_of(a, lm, fast_div(a.gdiv, tr.r0)));   // keys that every row of it sees
    const int nsp = a.max_ranges > 1 ? max(1, (end + tr.keys - 1) / tr.keys) : 1;
    if (tr.range >= nsp) return;
    const int k_lo = tr.range * tr.keys, k_hi = min(end, k_lo + tr.keys);
    const size_t head_off = (size_t)kvh * a.pg.head_stride_b;
    const int* table = a.pg.table + (size_t)tr.b * a.pg.ld_table;
    const char* kbase = a.k + head_off;
    const char* vbase = a.v + head_off;
    const int nt = (k_hi - k_lo + FEW_TILE - 1) / FEW_TILE;     // may be <= 0: rows that see no key

    PageSource<FEW_TILE, G16> src;
    u32x4_t kr[NP], vr[NP];
    unsigned int ok = 0;                                        // keys of the fetched tile that exist
    auto fetch = [&](int t) {
        src.advance(a, table, k_lo, k_hi, t, 4);
        ok = (unsigned int)src.exist(k_lo, k_hi, t);
        constexpr int ROW = F8 ? 128 : 256, PROWS = F8 ? 8 : 4, SUB = F8 ? 8 : 16;
#pragma unroll
        for (int g = 0; g < 2; ++g) {                           // K: a lane's key of each half of the tile, 64 B of 16 keys a piece
            const size_t at = G16 ? src.group(t, g) : src.key(16 * g + c);
            const char* p = kbase + at;
            const unsigned int in = (G16 ? c * ROW : 0) + quad * 16;
#pragma unroll
            for (int ks = 0; ks < NP / 2; ++ks) kr[g * (NP / 2) + ks] = *(const u32x4_t*)(p + in + ks * 64);
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {                          // V: whole KiB, 64 / SUB keys
            const char* p = vbase + (G16 ? src.group(t, i * PROWS / 16) : src.key(i * PROWS + lane / SUB));
            const unsigned int in = G16 ? i * PROWS % 16 * ROW + lane * 16 : (lane % SUB) * 16;
            vr[i] = *(const u32x4_t*)(p + in);
        }
    };
    if (kw < nt) {
        src.start(a, table, k_lo, k_hi, kw);
        fetch(kw);
    }

    // ---- queries: lane -> row c, features as the K fragments have them
    bf16x8_t qf[RG][4];
    int lim[RG];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        const RowAt at = row_at(a, tr, kvh, min(tr.r0 + rg * 16 + c, tr.rows - 1));
        lim[rg] = limit_of(a, lm, at.token - tr.s0);
        const char* qp = a.q + (size_t)at.token * a.ldq_b + (size_t)at.head * 256;
#pragma unroll
        for (int ks = 0; ks < 4; ++ks) qf[rg][ks] = *(const bf16x8_t*)(qp + (F8 ? 8 * (ks >> 1) + 2 * quad + (ks & 1) : 4 * ks + quad) * 16);
    }

    char* vimg = lds + kw * FEW_WAVE_LDS;
    f32x4_t o[RG][8];
    float m_run[RG], l_run[RG];
    unsigned int bad[RG];
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) o[rg][dt] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
        m_run[rg] = -INFINITY;
        l_run[rg] = 0.f;
        bad[rg] = 0;
    }
    const ImageWriter<F8> img(lane);
    // V^T fragments: keys 4 quad .. + 3 and 16 + 4 quad .. + 3, features 16 dt + c
    const int v0 = (4 * quad + (c >> 2)) * 256 + ((((c >> 1) & 1) ^ swz(4 * quad + (c >> 2))) << 4) + 8 * (c & 1);

    for (int t = kw; t < nt; t += 4) {
        const unsigned int ok_t = ok;
        const int key0 = k_lo + t * FEW_TILE;
        const bool part = ok_t != 0xffffffffu || key0 + FEW_TILE > all;           // wave-uniform
        bool dropped = false;
        // ---- S^T
        f32x4_t s[RG][2];
#pragma unroll
        for (int g = 0; g < 2; ++g) {
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) s[rg][g] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < 4; ++ks) {
                bf16x8_t kf;
                if (F8) {
                    const u32x4_t w = kr[2 * g + (ks >> 1)];
                    const u32x2_t x = bf16_of_e4m3(w[2 * (ks & 1)]), y = bf16_of_e4m3(w[2 * (ks & 1) + 1]);
                    kf = __builtin_bit_cast(bf16x8_t, (u32x4_t){x[0], x[1], y[0], y[1]});
                } else {
                    kf = __builtin_bit_cast(bf16x8_t, kr[(4 * g + ks) % NP]);
                }
#pragma unroll
                for (int rg = 0; rg < RG; ++rg) s[rg][g] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[rg][ks], s[rg][g], 0, 0, 0);
            }
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            if (part) dropped |= img.template put<true>(vimg, i, vr[i], ok_t);
            else img.template put<false>(vimg, i, vr[i], ok_t);
        }
        __builtin_amdgcn_sched_barrier(0);
        if (t + 4 < nt) fetch(t + 4);
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int rg = 0; rg < RG; ++rg) {
            if (part) {                                         // uniform, and kept a branch by the empty asm
                asm volatile("" ::: "memory");
                const int left = lim[rg] - key0 - 4 * quad;
                const unsigned int okq = ok_t >> (4 * quad);
#pragma unroll
                for (int g = 0; g < 2; ++g)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (16 * g + i >= left || !((okq >> (16 * g + i)) & 1)) s[rg][g][i] = -INFINITY;
            }
            float mx = fmaxf(s[rg][0][0], s[rg][1][0]);
#pragma unroll
            for (int i = 1; i < 4; ++i) mx = fmaxf(mx, fmaxf(s[rg][0][i], s[rg][1][i]));
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale_log2e;
            if (__any(mx > m_run[rg] + RESCALE_THR)) {
                // only rows that ask for it, so that no row's bits depend on what another one sees; one that has seen no key yet keeps -inf
                // and nothing to scale
                const float m_new = mx > m_run[rg] + RESCALE_THR ? mx : m_run[rg];
                const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run[rg] - m_new);
                l_run[rg] *= alpha;
                m_run[rg] = m_new;
#pragma unroll
                for (int dt = 0; dt < 8; ++dt) o[rg][dt] *= alpha;
            }
            const float neg_m = m_run[rg] == -INFINITY ? 0.f : -m_run[rg];
            float psum = 0.f;
#pragma unroll
            for (int g = 0; g < 2; ++g)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[rg][g][i], a.scale_log2e, neg_m));
                    s[rg][g][i] = p;
                    psum += p;
                }
            l_run[rg] += psum;
        }
        // ---- O^T, the weights as a bf16 pair (value and remainder): the second product of each fragment hides under the page loads, and
        // the weights keep 16 significant bits instead of 8
        bf16x8_t ph[RG], pl[RG];
#pragma unroll
        for (int rg = 0; rg < RG; ++rg)
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = s[rg][j >> 2][j & 3];
                ph[rg][j] = (__bf16)p;
                pl[rg][j] = (__bf16)(p - (float)ph[rg][j]);
            }
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) {
            // rows + 16: the same swizzle; features 16 dt: chunk 2 dt
            const bf16x8_t vf = join4(read_transposed(vimg + (v0 ^ (dt << 5))), read_transposed(vimg + 4096 + (v0 ^ (dt << 5))));
#pragma unroll
            for (int rg = 0; rg < RG; ++rg) {
                o[rg][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pl[rg], o[rg][dt], 0, 0, 0);
                o[rg][dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, ph[rg], o[rg][dt], 0, 0, 0);
            }
        }
        if (__any(dropped)) {
#pragma unroll
            for (int rg = 0; rg < RG; ++rg)
                bad[rg] |= (unsigned int)find_nonfinite<F8>(a, table, head_off, key0, FEW_TILE, k_hi, lim[rg], 32,
                                                            [&](int e) { return 16 * (e >> 2) + 4 * quad + (e & 3); });
        }
    }

    // ---- the four key waves' triples: common maximum, scaled sums
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        if (__any(bad[rg] != 0)) {
#pragma unroll
            for (int e = 0; e < 32; ++e)
                if ((bad[rg] >> e) & 1) o[rg][e >> 2][e & 3] = __builtin_nanf("");
        }
        float l = l_run[rg] + __shfl_xor(l_run[rg], 16, 64);
        l += __shfl_xor(l, 32, 64);
        if (quad == 0) {
            ml[kw][0][rg * 16 + c] = m_run[rg];
            ml[kw][1][rg * 16 + c] = l;
        }
    }
    __syncthreads();
#pragma unroll
    for (int rg = 0; rg < RG; ++rg) {
        float m = ml[0][0][rg * 16 + c];
#pragma unroll
        for (int w = 1; w < 4; ++w) m = fmaxf(m, ml[w][0][rg * 16 + c]);
        const float f = part_weight(m_run[rg], m);
        // a wave's own image region holds its 16 x 128 fp32 block: 16-byte chunk ch of row r at ch ^ r
        if (rg > 0) __syncthreads();                            // the block of the previous row group has been read
#pragma unroll
        for (int dt = 0; dt < 8; ++dt) *(f32x4_t*)(vimg + c * 512 + (((4 * dt + quad) ^ c) << 4)) = o[rg][dt] * f;
        __syncthreads();
        // key wave w joins rows 4 w .. 4 w + 3: lane -> row, 8 features
        const int rr = kw * 4 + quad, tile_row = tr.r0 + rg * 16 + rr;
        float acc[8], ll = 0.f, mm = ml[0][0][rg * 16 + rr];
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] = 0.f;
#pragma unroll
        for (int w = 1; w < 4; ++w) mm = fmaxf(mm, ml[w][0][rg * 16 + rr]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            ll += ml[w][1][rg * 16 + rr] * part_weight(ml[w][0][rg * 16 + rr], mm);
#pragma unroll
            for (int q4 = 0; q4 < 2; ++q4) {
                const f32x4_t x = *(const f32x4_t*)(lds + w * FEW_WAVE_LDS + rr * 512 + (((2 * c + q4) ^ rr) << 4));
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[4 * q4 + j] += x[j];
            }
        }
        if (tile_row >= tr.rows) continue;
        const RowAt at = row_at(a, tr, kvh, tile_row);
        if (nsp == 1) {
            const float inv = ll == 0.f ? 0.f : a.v_scale / ll;            // no key seen: zeros
#pragma unroll
            for (int j = 0; j < 8; ++j) acc[j] *= inv;
            *(u32x4_t*)(a.out + (size_t)at.token * a.ldo_b + (size_t)at.head * 256 + c * 16) = pack8(acc);
        } else {
            const size_t row = (size_t)tr.range * a.T * a.n_q + (size_t)at.token * a.n_q + at.head;
            float* op = a.po + row * HEAD_DIM + c * 8;
            *(f32x4_t*)op = (f32x4_t){acc[0], acc[1], acc[2], acc[3]};
            *(f32x4_t*)(op + 4) = (f32x4_t){acc[4], acc[5], acc[6], acc[7]};
            if (c == 0) *(f32x2_t*)(a.pml + row * 2) = (f32x2_t){mm, ll};
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Many rows: NW waves of 32 rows each share a double-buffered stream of 64-key tiles, one barrier a tile.
//
// What bounds it: the chain products - maximum - exponentials - products of a wave, which the other wave of its SIMD only partly
// covers, and the LDS reads of every fragment for only 32 rows.  The weights are a bf16 pair, so of three matrix instructions two are the
// second product's.  Measured, 16 heads on 8: 8 x 2048 tokens, no mask 386 us = 712 TFLOP/s (with the remainders, which are not counted,
// the matrix unit does half as much again), causal 225 us; 2 x 8192 no mask 1419 us = 775 TFLOP/s; a large matrix product reaches 1257 on
// this card.  One bf16 weight in place of the pair took 291, 175 and 1025 us, with an error of 0.0022 of the result where its own rounding
// to bf16 is 0.0017: a call's rows would be less exact for being many.
// Whole bf16 tiles straight to LDS instead of through registers: 8 x 2048 no mask 399 / 403 us (another card, in turn, three times), 2 x 8192
// 1504 / 1526, 8 x 200 causal over 4000 keys 122 / 126.  Tried with one weight, and slower or no faster against 303 .. 314 us for 8 x 2048
// without mask through registers: the two halves of the workgroup one barrier apart (341), the softmax of a tile beside the scores of the
// next (311), wave priorities around the products (316).
constexpr int MANY_TILE = 64;
constexpr int MANY_BUF = 2 * MANY_TILE * 256;                   // K and V image: 32 KiB

// LDS writes done, then the barrier; global loads on their way to registers stay in flight (__syncthreads would wait for them)
__device__ __forceinline__ void lds_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// MFMA fragments out of the images (v_mfma_f32_32x32x16_bf16).
//   K (A operand of S^T, 32 keys x 16 features): lane -> key 32 k2 + (lane & 31), chunk 2 ks + (lane >> 5)
//   V^T (A operand of O^T, 32 features x 16 keys): keys 16 st + 4 h .. + 3 and + 8, features 32 db + (lane & 31)
struct ImageReader {
    int k0, v0;
    __device__ __forceinline__ explicit ImageReader(int lane) {
        const int c = lane & 31, h = lane >> 5;
        k0 = c * 256 + ((h ^ swz(c)) << 4);
        const int i16 = lane & 15, tq = i16 >> 2, tp = i16 & 3;
        const int ch = 2 * ((lane >> 4) & 1) + (tp >> 1);
        v0 = (4 * h + tq) * 256 + ((ch ^ swz(4 * h + tq)) << 4) + 8 * (tp & 1);
    }
    __device__ __forceinline__ bf16x8_t k(const char* img, int k2, int ks) const {
        return *(const bf16x8_t*)(img + 32 * k2 * 256 + (k0 ^ (ks << 5)));
    }
    __device__ __forceinline__ bf16x8_t v(const char* img, int st, int db) const {
        const char* p = img + st * 4096;
        const int at = v0 ^ (db << 6);
        return join4(read_transposed(p + at), read_transposed(p + 2048 + (at ^ (swz(8) << 4))));
    }
};

// 16 bytes a lane, from a uniform base and a lane's offset, straight to a uniform LDS address + 16 lane; vmcnt counts it.  In asm because
// the compiler waits for a copy that it knows of before every transposing read, which ends the overlap half a tile early.
__device__ __forceinline__ void to_lds(const char* base, unsigned int in, unsigned int to) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(to), "v"(in), "s"(base) : "m0", "memory");
}

template <int NW, bool F8, bool G16>
__global__ __launch_bounds__(NW * 64, NW == 4 ? 2 : 1) void paged_attn_many_kernel(AttnArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int R = 32 * NW;
    constexpr bool DMA = !F8 && G16;
    constexpr int NP = (F8 ? 8 : 16) / NW;                      // 1 KiB pieces of a K (or V) tile per wave
    __shared__ int dropped_s[4];                                // tile t & 3: non-finite values were dropped from its V image
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = lane & 31, h = lane >> 5;
    // tiles of a sequence read the same keys: with the key/value head as the fastest index, and workgroups going round the eight XCDs, a
    // head stays on few XCDs (one, for 8 heads) and its keys are found in that L2
    const int kvh = blockIdx.x % a.n_kv;
    TileRows tr;
    Limits lm;
    if (!find_unit<R, true>(a, blockIdx.x / a.n_kv, tr, lm)) return;
    const int last = min(tr.r0 + R, tr.rows) - 1;
    const int end = __builtin_amdgcn_readfirstlane(limit_of(a, lm, fast_div(a.gdiv, last)));
    const int all = __builtin_amdgcn_readfirstlane(limit_of(a, lm, fast_div(a.gdiv, tr.r0)));
    const int nsp = a.max_ranges > 1 ? max(1, (end + tr.keys - 1) / tr.keys) : 1;
    if (tr.range >= nsp) return;
    const int k_lo = tr.range * tr.keys, k_hi = min(end, k_lo + tr.keys);
    const size_t head_off = (size_t)kvh * a.pg.head_stride_b;
    const int* table = a.pg.table + (size_t)tr.b * a.pg.ld_table;
    const char* kbase = a.k + head_off;
    const char* vbase = a.v + head_off;

    const int my_row = tr.r0 + wave * 32 + c;
    const RowAt at = row_at(a, tr, kvh, min(my_row, tr.rows - 1));
    const int lim = limit_of(a, lm, at.token - tr.s0);
    // what this wave's rows see: all of them / any of them (limits do not decrease along the rows)
    const int w_all = __builtin_amdgcn_readlane(lim, 0), w_any = __builtin_amdgcn_readlane(lim, 31);
    bf16x8_t qf[8];
    {
        const char* qp = a.q + (size_t)at.token * a.ldq_b + (size_t)at.head * 256 + h * 16;
#pragma unroll
        for (int ks = 0; ks < 8; ++ks) qf[ks] = *(const bf16x8_t*)(qp + ks * 32);
    }
    f32x16_t o[4];
#pragma unroll
    for (int db = 0; db < 4; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    float m_run = -INFINITY, l_run = 0.f;
    unsigned long long bad = 0;

    u32x4_t kr[NP], vr[NP];
    PageSource<MANY_TILE, G16> src;
    auto whole = [&](int t, unsigned long long ok) { return ok == ~0ull && k_lo + (t + 1) * MANY_TILE <= all; };
    const unsigned int lds0 = (unsigned int)(uintptr_t)(CODA_LDS char*)lds;
    // sends for pieces i NW + wave of tile t; returns which of its keys exist
    auto send = [&](int t) {
        src.advance(a, table, k_lo, k_hi, t, 1);
        const unsigned long long ok = src.exist(k_lo, k_hi, t);
        constexpr int ROW = F8 ? 128 : 256, PROWS = F8 ? 8 : 4, SUB = F8 ? 8 : 16;
        if (DMA && whole(t, ok)) {
            const unsigned int to = lds0 + (t & 1) * MANY_BUF;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                const int row = (i * NW + wave) * 4;
                const size_t at = src.group(t, row >> 4) + (row & 15) * 256;
                const unsigned int in = (lane >> 4) * 256 + (((lane & 15) ^ swz(row + (lane >> 4))) << 4);
                to_lds(kbase + at, in, to + row * 256);
                to_lds(vbase + at, in, to + MANY_TILE * 256 + row * 256);
            }
            return ok;
        }
#pragma unroll
        for (int i = 0; i < NP; ++i) {
            const int key = (i * NW + wave) * PROWS;
            const size_t at = G16 ? src.group(t, key >> 4) : src.key(key + lane / SUB);
            const unsigned int in = G16 ? (key & 15) * ROW + lane * 16 : (lane % SUB) * 16;
            kr[i] = *(const u32x4_t*)(kbase + at + in);
            vr[i] = *(const u32x4_t*)(vbase + at + in);
        }
        return ok;
    };
    const ImageWriter<F8> img(lane);
    const ImageReader rd(lane);

    auto tile = [&](int t, const char* kimg, bool part, unsigned long long ok) {
        const char* vimg = kimg + MANY_TILE * 256;
        f32x16_t s[2];
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[k2][i] = 0.f;
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) s[k2] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(rd.k(kimg, k2, ks), qf[ks], s[k2], 0, 0, 0);
        }
        if (part) {                                             // uniform, and kept a branch by the empty asm
            asm volatile("" ::: "memory");
            const int left = lim - k_lo - t * MANY_TILE - 4 * h;
            const unsigned long long okh = ok >> (4 * h);
#pragma unroll
            for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int j = 32 * k2 + (i & 3) + 8 * (i >> 2);
                    if (j >= left || !((okh >> j) & 1)) s[k2][i] = -INFINITY;
                }
        }
        float mx = s[0][0];
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[k2][i]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * a.scale_log2e;
        if (__any(mx > m_run + RESCALE_THR)) {
            const float m_new = mx > m_run + RESCALE_THR ? mx : m_run;      // only rows that ask for it, as above
            const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m_run - m_new);
            l_run *= alpha;
            m_run = m_new;
#pragma unroll
            for (int db = 0; db < 4; ++db)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
        }
        const float neg_m = m_run == -INFINITY ? 0.f : -m_run;
        float psum = 0.f;
#pragma unroll
        for (int k2 = 0; k2 < 2; ++k2)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(s[k2][i], a.scale_log2e, neg_m));
                s[k2][i] = p;
                psum += p;
            }
        l_run += psum;
        // the weights as a bf16 pair, as in the `few` kernel: each V fragment that was read from LDS enters two products
#pragma unroll
        for (int st = 0; st < 4; ++st) {
            bf16x8_t ph, pl;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float p = s[st >> 1][8 * (st & 1) + j];
                ph[j] = (__bf16)p;
                pl[j] = (__bf16)(p - (float)ph[j]);
            }
            bf16x8_t vf[4];
#pragma unroll
            for (int db = 0; db < 4; ++db) vf[db] = rd.v(vimg, st, db);
#pragma unroll
            for (int db = 0; db < 4; ++db) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db], pl, o[db], 0, 0, 0);
#pragma unroll
            for (int db = 0; db < 4; ++db) o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf[db], ph, o[db], 0, 0, 0);
        }
    };

    const int nt = (k_hi - k_lo + MANY_TILE - 1) / MANY_TILE;
    if (threadIdx.x < 4) dropped_s[threadIdx.x] = 0;
    __syncthreads();
    if (nt > 0) {
        // tile t arrives in its image; partly seen by the WORKGROUP's rows: that must hold finite values and zeros only
        auto publish = [&](int t, unsigned long long ok) {
            char* kimg = lds + (t & 1) * MANY_BUF;
            char* vimg = kimg + MANY_TILE * 256;
            if (!whole(t, ok)) {
                bool dropped = false;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    img.template put<false>(kimg, i * NW + wave, kr[i], ok);
                    dropped |= img.template put<true>(vimg, i * NW + wave, vr[i], ok);
                }
                if (dropped) dropped_s[t & 3] = 1;
            } else if (DMA) {
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            } else {
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    img.template put<false>(kimg, i * NW + wave, kr[i], ok);
                    img.template put<false>(vimg, i * NW + wave, vr[i], ok);
                }
            }
        };
        src.start(a, table, k_lo, k_hi, 0);
        unsigned long long ok = send(0), ok_next = 0;
        publish(0, ok);
        for (int t = 0; t < nt; ++t) {
            // one barrier a tile: behind it tile t's image is complete and nobody reads tile t - 1's any more
            lds_barrier();
            const bool dropped = dropped_s[t & 3] != 0;
            if (threadIdx.x == 0) dropped_s[(t + 2) & 3] = 0;   // last read two barriers ago, next written behind the next one
            if (t + 1 < nt) ok_next = send(t + 1);
            __builtin_amdgcn_sched_barrier(0);
            const char* kimg = lds + (t & 1) * MANY_BUF;
            const int key0 = k_lo + t * MANY_TILE;
            if (key0 < w_any) {                                 // else none of this wave's rows sees the tile
                tile(t, kimg, ok != ~0ull || key0 + MANY_TILE > w_all, ok);
                if (dropped)
                    bad |= find_nonfinite<F8>(a, table, head_off, key0, MANY_TILE, k_hi, lim, 64,
                                              [&](int e) { return 32 * (e >> 4) + (e & 3) + 8 * ((e >> 2) & 3) + 4 * h; });
            }
            __builtin_amdgcn_sched_barrier(0);
            if (t + 1 < nt) publish(t + 1, ok_next);
            ok = ok_next;
        }
    }

    if (__any(bad != 0)) {
#pragma unroll
        for (int e = 0; e < 64; ++e)
            if ((bad >> e) & 1) o[e >> 4][e & 15] = __builtin_nanf("");
    }
    // ---- epilogue (flash_attn.hip): the halves trade groups so that a lane holds 8 consecutive features
    const float l_tot = l_run + __shfl_xor(l_run, 32, 64);
    const bool live = my_row < tr.rows;
    if (nsp == 1) {
        const float inv = l_tot == 0.f ? 0.f : a.v_scale / l_tot;      // no key seen: zeros
        char* op = a.out + (size_t)at.token * a.ldo_b + (size_t)at.head * 256;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int gA = 2 * j, gB = 2 * j + 1;
                const unsigned a0 = pack_bf16x2(o[db][4 * gA] * inv, o[db][4 * gA + 1] * inv);
                const unsigned a1 = pack_bf16x2(o[db][4 * gA + 2] * inv, o[db][4 * gA + 3] * inv);
                const unsigned b0 = pack_bf16x2(o[db][4 * gB] * inv, o[db][4 * gB + 1] * inv);
                const unsigned b1 = pack_bf16x2(o[db][4 * gB + 2] * inv, o[db][4 * gB + 3] * inv);
                const auto s0 = __builtin_amdgcn_permlane32_swap(a0, b0, false, false);
                const auto s1 = __builtin_amdgcn_permlane32_swap(a1, b1, false, false);
                if (live) *(u32x4_t*)(op + (32 * db + 8 * (2 * j + h)) * 2) = (u32x4_t){s0[0], s1[0], s0[1], s1[1]};
            }
    } else if (live) {
        const size_t row = (size_t)tr.range * a.T * a.n_q + (size_t)at.token * a.n_q + at.head;
        float* op = a.po + row * HEAD_DIM;
#pragma unroll
        for (int db = 0; db < 4; ++db)
#pragma unroll
            for (int i4 = 0; i4 < 4; ++i4)
                *(f32x4_t*)(op + 32 * db + 8 * i4 + 4 * h) = (f32x4_t){o[db][4 * i4], o[db][4 * i4 + 1], o[db][4 * i4 + 2], o[db][4 * i4 + 3]};
        if (h == 0) *(f32x2_t*)(a.pml + row * 2) = (f32x2_t){m_run, l_tot};
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// Joins the key ranges of (token, head) rows.  R: rows per tile of the kernel that wrote the ranges (the rows of a tile have the same
// number of ranges).  `rows`: half a wave per row, two heads of a token in a wave (one search), the loads of eight ranges in flight at once.
// `join`: a workgroup per row, the ranges shared out over its eight half-waves, which meet in LDS: for many ranges of few rows (us a call:
// 16 rows of 47 ranges 17.1 / 15.6, 64 rows 24.3 / 22.5, but 1600 rows of 24 ranges 40.7 / 53.7).  Bound by latency (sequence, its
// length, the parts: three dependent loads) or by the parts' bytes: 4.7 us for 2048 rows, 8.0 for 16384 rows of up to 4 ranges.
constexpr int AT_ONCE = 8;

template <int R>
__device__ __forceinline__ int ranges_of(const AttnArgs& a, int token, int head) {
    const Seq q = seq_of_token({a.seq_start, a.kv_len, a.pos0, a.B, a.T}, token);
    if (q.b < 0) return 0;                                      // a row of no sequence
    const int r = (token - q.s0) * a.g + head % a.g;
    const int last = (int)min(((long long)r / R + 1) * R, (long long)q.n * a.g) - 1;
    const Limits lm = limits_of(a, q);
    const int end = limit_of(a, lm, fast_div(a.gdiv, last)), keys = keys_of(lm.kv, *a.range_keys);
    return (end + keys - 1) / keys;
}

template <int R>
__global__ __launch_bounds__(256) void paged_attn_join_rows_kernel(AttnArgs a) {
    const int lane = threadIdx.x & 63, l = lane & 31;
    const int unit = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    const int pairs = (a.n_q + 1) / 2, token = unit / pairs;
    if (token >= a.T) return;
    const int head = unit % pairs * 2 + (lane >> 5);
    int nsp = ranges_of<R>(a, token, head);
    if (nsp <= 1 || head >= a.n_q) nsp = 0;                     // written by the first kernel
    const size_t rows = (size_t)a.T * a.n_q, row = (size_t)token * a.n_q + min(head, a.n_q - 1);
    float m = -INFINITY, tot = 0.f;
    f32x4_t y = {0.f, 0.f, 0.f, 0.f};
    auto some = [&](int i0) {
        f32x2_t e[AT_ONCE];
        f32x4_t x[AT_ONCE];
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (!__any(i0 + i < nsp)) break;
            const size_t at = (size_t)max(min(i0 + i, nsp - 1), 0) * rows + row;
            e[i] = *(const f32x2_t*)(a.pml + at * 2);
            x[i] = *(const f32x4_t*)(a.po + at * HEAD_DIM + 4 * l);
        }
        float mn = m;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i)
            if (i0 + i < nsp) mn = fmaxf(mn, e[i][0]);
        const float fo = part_weight(m, mn);
        tot *= fo;
        y = y * fo;
#pragma unroll
        for (int i = 0; i < AT_ONCE; ++i) {
            if (i0 + i >= nsp) break;
            const float f = part_weight(e[i][0], mn);
            tot += e[i][1] * f;
            y = y + x[i] * f;
        }
        m = mn;
    };
    some(0);                                                    // apart: nothing to rescale
    for (int i0 = AT_ONCE; __any(i0 < nsp); i0 += AT_ONCE) some(i0);
    if (nsp == 0) return;
    const float inv = tot == 0.f ? 0.f : a.v_scale / tot;
    *(u32x2_t*)(a.out + (size_t)token * a.ldo_b + (size_t)head * 256 + l * 8) =
        (u32x2_t){pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv)};
}

template <int R>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(AttnArgs a) {
    __shared__ float sm[8], sl[8];
    __shared__ f32x4_t so[8][32];
    const int token = blockIdx.x / a.n_q, head = blockIdx.x % a.n_q;
    const int nsp = ranges_of<R>(a, token, head);
    if (nsp <= 1) return;
    const int grp = threadIdx.x >> 5, l = threadIdx.x & 31;
    const size_t rows = (size_t)a.T * a.n_q, row = (size_t)blockIdx.x;
    float m = -INFINITY, sum = 0.f;
    f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
    for (int s0 = grp; s0 < nsp; s0 += 32) {                    // four ranges in flight
        f32x2_t e[4];
        f32x4_t x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const size_t at = (size_t)min(s0 + 8 * i, nsp - 1) * rows + row;
            e[i] = *(const f32x2_t*)(a.pml + at * 2);
            x[i] = *(const f32x4_t*)(a.po + at * HEAD_DIM + 4 * l);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (s0 + 8 * i >= nsp) break;
            const float mn = fmaxf(m, e[i][0]);
            const float fo = part_weight(m, mn), fn = part_weight(e[i][0], mn);
            sum = sum * fo + e[i][1] * fn;
            acc = acc * fo + x[i] * fn;
            m = mn;
        }
    }
    if (l == 0) { sm[grp] = m; sl[grp] = sum; }
    so[grp][l] = acc;
    __syncthreads();
    if (grp) return;
    float mm = sm[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mm = fmaxf(mm, sm[i]);
    float tot = 0.f;
    f32x4_t y = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float f = part_weight(sm[i], mm);
        tot += sl[i] * f;
        y = y + so[i][l] * f;
    }
    const float inv = tot == 0.f ? 0.f : a.v_scale / tot;
    *(u32x2_t*)(a.out + (size_t)token * a.ldo_b + (size_t)head * 256 + l * 8) =
        (u32x2_t){pack_bf16x2(y[0] * inv, y[1] * inv), pack_bf16x2(y[2] * inv, y[3] * inv)};
}

// How a call is cut: rows per tile, workgroups, the bounds of the key ranges.  A function of the call's sizes alone.
struct Plan {
    int R; long long wgs; int max_ranges, min_keys; float per_range;
};

constexpr int WS_HEAD = 256;                    // bytes in front of the partial outputs: the range length

Plan make_plan(int T, int B, int max_kv, int n_q, int n_kv, bool slanted, int cus) {
    const int g = n_q / n_kv;
    const double rho = (double)T * g / B;                       // rows per sequence and key/value head, on average
    Plan p;
    // tiles per key/value head, at least, where no sequence is empty
    auto tiles = [&](int R) {
        const long long t = ((long long)T * g + R - 1) / R;
        return t > B ? t : B;
    };
    const long long two = 2LL * cus;                            // workgroups of 256 threads that are resident at once
    // us with tiles of so many rows, 16 heads on 8, bf16:
    //   16 / 32      32 sequences x 2000 keys: rho 8 51 / 53, rho 16 51 / 53, rho 24 58 / 53
    //   32 / 128     32 x 1000: rho 48 38 / 44, rho 64 41 / 50, rho 80 58 / 53; 128 x 1500: 182 / 224, 183 / 190, 246 / 200; 8 x 4000:
    //                43 / 45, 50 / 47, 62 / 49; all tiles resident and keys short, 8 x 300: rho 64 14.1 / 20.1, rho 128 14.9 / 21.0
    //   128 / 256    16 x 2000: rho 256 84 / 102; 4 x 1000: rho 768 52.6 / 50.7, rho 1024 57.6 / 56.9; 8 x 2048 new: 403 / 402, 2 x 8192
    //                new 1547 / 1522, behind 8000 keys 1 x 1000 128 / 123, but 2 x 2048 new 74 / 88 (too few tiles for the chip)
    // (64 rows on eight waves lost to 32 or 128 everywhere.)
    if (rho <= 16) p.R = 16;
    else if (rho <= 64 || (rho <= 128 && max_kv < 2048 && tiles(32) * n_kv <= two)) p.R = 32;
    else p.R = rho > 1536 && tiles(256) * n_kv * (max_kv < 2048 ? 1 : max_kv / 2048) >= cus ? 256 : 128;
    const long long bound = (long long)T * g / p.R + B;         // tiles per key/value head, at most
    const long long some = tiles(p.R);
    const long long slots = p.R == 256 ? cus : two;
    // The shortest range.  Tiles on less than a quarter of the chip wait for latency, and the chain of a range's tiles is what they wait
    // for: 128 keys, once there are enough of them to pay for the second kernel (us uncut / cut into 128 ..: one token on 8 heads, 700 keys
    // 13.4 / 13.8, 1000 15.9 / 14.7, 1500 19.8 / 14.8, 5000 50 / 15.6; a block of 32 700 17.7 / 16.5, 1500 26 / 17.7; 100 tokens 500 22.1 / 19.8,
    // 1500 50 / 22.4).  Otherwise eight steps of a workgroup, 1024 or 512 keys (us at half / at it / at twice: 32 single tokens x 2000 keys
    // 54.2 / 50.7 / 50.6, 8 blocks of 128 tokens x 2000 55.3 / 54.2 / 67.7, 8 of 200 x 4000 123 / 122 / 130).  No more partial outputs than
    // 64 MiB.
    const bool idle = some * n_kv * 4 < slots;
    const int least = idle ? 128 : p.R <= 32 ? 1024 : 512;
    const long long row_bytes = (long long)T * n_q * (HEAD_DIM + 2) * 4;
    long long most = idle && max_kv < (p.R <= 32 ? 768 : 512) ? 1 : max_kv / least;
    if (most > (64LL << 20) / row_bytes) most = (64LL << 20) / row_bytes;
    if (most > 256) most = 256;
    // few tiles: one round of equal units.  Many: about four rounds, so that sequences of unequal length even out
    const long long units = some * n_kv * 2 <= slots ? slots - some * n_kv : 4 * slots;
    p.max_ranges = most < 2 || some * n_kv >= 2 * units ? 1 : (int)most;
    p.min_keys = p.max_ranges > 1 ? ((max_kv + p.max_ranges - 1) / p.max_ranges + 127) / 128 * 128 : 0;
    if (p.max_ranges > 1 && p.min_keys < least) p.min_keys = least;
    p.per_range = (float)((double)n_kv / units);
    // every tile's first range, and the further ones: at most work / range length <= units / n_kv of them (1/64 for the sum's rounding), or
    // twice as many where the work is slanted: it is then at least half a sequence's tiles times its keys
    p.wgs = bound * n_kv + (p.max_ranges > 1 ? (1 + slanted) * (units + units / 64 + n_kv) : 0);
    return p;
}

long long plan_bytes(const Plan& p, int T, int n_q) {
    return p.max_ranges > 1 ? WS_HEAD + (long long)p.max_ranges * T * n_q * (HEAD_DIM + 2) * 4 : 0;
}

}  // namespace

extern "C" long long coda_paged_attn_workspace_bytes(int T, int B, int max_kv, int n_q, int n_kv) {
    if (T <= 0 || B <= 0 || max_kv < 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv) return 0;
    if ((long long)T * n_q > 0x7fffffffLL) return 0;            // the call refuses these too
    return plan_bytes(make_plan(T, B, max_kv, n_q, n_kv, false, coda_device_cus()), T, n_q);
}

extern "C" int coda_paged_attn(const void* q, long long ld_q, void* out, long long ld_out, const int* seq_start, const int* pos0,
                               const int* kv_len, int B, int T, const int* page_table, long long ld_table, int max_pages,
                               const void* k_cache, const void* v_cache, long long page_stride, int num_pages, int page_size,
                               int cache_type, float k_scale, float v_scale, int max_kv, int n_q, int n_kv, float scale, int mask_block,
                               void* workspace, long long workspace_bytes, void* stream) {
    const char* who = "coda_paged_attn";
    if (B <= 0 || T <= 0 || n_q <= 0 || n_kv <= 0 || n_q % n_kv) return coda_refuse(who, CODA_ERR_SHAPE, "a size is not positive, or n_q % n_kv");
    if ((long long)T * n_q > 0x7fffffffLL) return coda_refuse(who, CODA_ERR_SHAPE, "T * n_q exceeds 2^31 - 1");
    // running sums over 64 sequences of tiles stay below 2^31 even for starts that make every sequence T rows long
    if ((long long)T * (n_q / n_kv) > 1 << 28) return coda_refuse(who, CODA_ERR_SHAPE, "T * n_q / n_kv exceeds 2^28");
    if (max_kv < 0 || (long long)max_kv > (long long)max_pages * page_size || max_kv > 1 << 30)
        return coda_refuse(who, CODA_ERR_SHAPE, "max_kv is not within max_pages * page_size and 2^30");
    if (ld_q < (long long)n_q * HEAD_DIM || ld_out < (long long)n_q * HEAD_DIM) return coda_refuse(who, CODA_ERR_SHAPE, "a row stride is shorter than a row");
    if (!q || !out || !seq_start || !pos0 || !kv_len) return coda_refuse(who, CODA_ERR_ARG, "null pointer");
    if (!(scale > 0.f)) return coda_refuse(who, CODA_ERR_ARG, "scale must be positive");
    if (mask_block < 0) return coda_refuse(who, CODA_ERR_ARG, "mask_block is negative");
    if (((uintptr_t)q | (uintptr_t)out) & 15 || (ld_q * 2) % 16 || (ld_out * 2) % 16) return coda_refuse(who, CODA_ERR_ALIGN, "rows start on 16 bytes");
    AttnArgs a;
    const int rc = coda_check_pages(who, k_cache, v_cache, page_table, ld_table, max_pages, page_stride, num_pages, page_size, cache_type,
                                    k_scale, v_scale, n_kv, &a.pg);
    if (rc != CODA_OK) return rc;
    const bool f8 = cache_type == CODA_CACHE_E4M3;
    a.scale_log2e = scale * (f8 ? k_scale : 1.0f) * 1.4426950408889634f;
    if (!(a.scale_log2e >= 1e-30f && a.scale_log2e <= 1e30f)) return coda_refuse(who, CODA_ERR_ARG, "scale times k_scale is not within [1e-30, 1e30]");
    // With some tokens a sequence, a mask hides up to half of what its tiles would see: us with / without counting that, causal: 1 x 2048 tokens
    // 66 / 73, 1 x 2048 behind 2000 keys 112 / 130, 2 x 900 behind 1000 equal.  Single tokens have nothing to gain, and the grid for the
    // shorter ranges costs them (128 x 1 over e4m3 81 / 75).
    a.slanted = mask_block > 0 && T > 4LL * B;
    const Plan p = make_plan(T, B, max_kv, n_q, n_kv, a.slanted, coda_device_cus());
    const long long need = plan_bytes(p, T, n_q);
    if (need > 0 && (!workspace || workspace_bytes < need)) return coda_refuse(who, CODA_ERR_ARG, "workspace is smaller than coda_paged_attn_workspace_bytes");
    if ((uintptr_t)workspace & 15) return coda_refuse(who, CODA_ERR_ALIGN, "the workspace starts on 16 bytes");
    if (!grid_fits(p.wgs, p.R == 256 ? 512 : 256)) return coda_refuse(who, CODA_ERR_SHAPE, "too many tiles for one launch");
    a.q = (const char*)q; a.ldq_b = ld_q * 2;
    a.out = (char*)out; a.ldo_b = ld_out * 2;
    a.seq_start = seq_start; a.pos0 = pos0; a.kv_len = kv_len;
    a.B = B; a.T = T; a.max_kv = max_kv;
    a.k = (const char*)k_cache; a.v = (const char*)v_cache;
    a.n_q = n_q; a.n_kv = n_kv; a.g = n_q / n_kv; a.gdiv = make_fast_div((unsigned)a.g);
    a.mask_block = mask_block;
    a.v_scale = f8 ? v_scale : 1.0f;
    a.max_ranges = p.max_ranges; a.min_keys = p.min_keys; a.per_range = p.per_range;
    a.range_keys = p.max_ranges > 1 ? (int*)workspace : nullptr;
    a.po = p.max_ranges > 1 ? (float*)((char*)workspace + WS_HEAD) : nullptr;
    a.pml = p.max_ranges > 1 ? a.po + (long long)p.max_ranges * T * n_q * HEAD_DIM : nullptr;
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto kernel, int threads, int lds) -> int {
        if (coda_ensure_dyn_lds((const void*)kernel, lds) != CODA_OK) return CODA_ERR_LAUNCH;
        hipLaunchKernelGGL(kernel, dim3((unsigned)p.wgs), dim3(threads), lds, st, a);
        CODA_CHECK_LAUNCH("paged_attn");
        return CODA_OK;
    };
    // pages of a multiple of 16 keys take the kernels that address 16 keys at a time
    auto pick = [&](auto f8c, auto g16c) -> int {
        constexpr bool F8 = decltype(f8c)::value, G16 = decltype(g16c)::value;
        if (p.R == 16) return go(paged_attn_few_kernel<1, F8, G16>, 256, 4 * FEW_WAVE_LDS);
        if (p.R == 32) return go(paged_attn_few_kernel<2, F8, G16>, 256, 4 * FEW_WAVE_LDS);
        if (p.R == 128) return go(paged_attn_many_kernel<4, F8, G16>, 256, 2 * MANY_BUF);
        return go(paged_attn_many_kernel<8, F8, G16>, 512, 2 * MANY_BUF);
    };
    const bool g16 = page_size % 16 == 0;
    const std::true_type yes{};
    const std::false_type no{};
    const int r2 = f8 ? (g16 ? pick(yes, yes) : pick(yes, no)) : (g16 ? pick(no, yes) : pick(no, no));
    if (r2 != CODA_OK || p.max_ranges == 1) return r2;
    const long long rows = (long long)T * n_q;
    auto join = [&](auto tile_rows) {
        constexpr int R = decltype(tile_rows)::value;
        if (p.max_ranges <= AT_ONCE || rows > 4LL * coda_device_cus()) hipLaunchKernelGGL(paged_attn_join_rows_kernel<R>, dim3((unsigned)(((long long)T * ((n_q + 1) / 2) + 3) / 4)), dim3(256), 0, st, a);
        else hipLaunchKernelGGL(paged_attn_join_kernel<R>, dim3((unsigned)rows), dim3(256), 0, st, a);
    };
    if (p.R == 16) join(std::integral_constant<int, 16>{});
    else if (p.R == 32) join(std::integral_constant<int, 32>{});
    else if (p.R == 128) join(std::integral_constant<int, 128>{});
    else join(std::integral_constant<int, 256>{});
    CODA_CHECK_LAUNCH("paged_attn join");
    return CODA_OK;
}
