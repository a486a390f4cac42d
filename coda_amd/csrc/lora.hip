// Low-rank adapters of many requests beside a shared projection, on a ragged batch:
//
//     C[t] = R[t] + s[a] (X[t] A[a]^T) B[a]^T,     a = the adapter of t's sequence;  no adapter: C[t] = R[t]
//
// Two launches (one for small batches, lora_one_kernel).  `down` computes U = X A^T for tiles of one sequence's tokens, K cut over the
// waves of a workgroup and, where there are few tiles, over workgroups (fp32 slabs in the workspace, summed in a fixed order by their
// readers).  `up` sums the slabs, scales, computes U B^T in fp32 and adds R to it, so that the result is rounded once.
//
// v_mfma_f32_16x16x32_bf16 in both, weights as the A operand: a lane then holds four consecutive outputs (ranks, features) of one
// token.  Both are bound by memory at serving ranks (8 .. 128).  X, A, R and C move as contiguous 512 bytes of a row, through LDS:
// fragments straight from memory (16 rows x 64 B an instruction) took 27 + 120 us where this took 22 + 95 (17.9 k tokens, rank 32,
// 2048 -> 6144; later steps took the second to 82).  U enters the second product as a bf16 pair (value and remainder): the extra matrix instructions are free in a
// kernel that waits for memory, and U keeps 16 bits.
// Measured: 17.9 k tokens of 32 sequences, rank 32, 2048 -> 6144: down 22 us, up 82, a call 102: 508 MB at 5.0 TB/s (a large copy: 5.1); 32
// blocks of 32 tokens, rank 64, 6144 -> 2048: 8.1 + 7.6 us, bound by the latency of one tile's chain (tile, slabs, products, result);
// 32 single tokens, rank 16, 2048 -> 4096, in one launch: 6.8 us.
#include "paged_common.h"
#include <type_traits>

using namespace paged;

namespace {

struct Tile {
    int row0, n;                                // first token row, tokens (0: there is no such tile)
    int adapter;                                // -1: none
    int pad;                                    // 16 bytes each
};

struct LoraArgs {
    const char* x; long long ldx_b;
    const char* a; const char* b;
    const float* scale;
    const int* seq_start; const int* adapter;
    int B, T, n_adapters, rank;
    const char* r; long long ldr_b;
    char* c; long long ldc_b;
    int N, K;
    int nslots, ksplit, kchunk, nslice;
    float* u;                                   // [ksplit][T][rank]
    Tile* tiles;                                // [nslots]: what the first launch found, for the second
};

template <int TM>
__device__ __forceinline__ Tile find_tile(const LoraArgs& a, int slot) {
    const SeqArrays arr = {a.seq_start, a.adapter, nullptr, a.B, a.T};
    SeqBlock blk;
    blk.load(arr, 0);
    int k;
    const Seq q = seq_of_item(arr, blk, slot, k, [](const SeqLane& l) { return tiles_of<TM>(l, 1); });
    if (q.b < 0) return {0, 0, -1, 0};
    return {q.s0 + k * TM, min(q.n - k * TM, TM), (unsigned)q.x < (unsigned)a.n_adapters ? q.x : -1, 0};
}

// x as a bf16 value and its bf16 remainder.  bf16 rounds to infinity a little before fp32 ends: such an x is bf16's largest value and the
// rest; an infinity has no remainder (inf - inf would make it a NaN).
__device__ __forceinline__ void bf16_pair(float x, __bf16& h, __bf16& l) {
    float f = round_bf16(x);
    if (fabsf(f) == INFINITY && fabsf(x) != INFINITY) f = copysignf(0x1.fep127f, x);
    h = (__bf16)f;
    l = (__bf16)(fabsf(f) == INFINITY ? 0.f : x - f);
}

// U of 16 MT tokens, 16 RT ranks (those beyond the adapter's are computed from its last row and dropped).
// Steps of 256 elements: rows of X and A come in as contiguous 512 bytes through registers (those of the next two steps fly under this
// one's products: 7.7 us, one step ahead 8.4, 32 blocks of 32 tokens, rank 64, K 6144) into an LDS image, 16-byte chunk ch of row r at ch ^ (r & 15), and the four waves take 64 elements of each step.
template <int MT, int RT>
struct Down {
    static constexpr int ROWS = 16 * (MT + RT);
    static constexpr int NL = ROWS / 8;                         // 16-byte loads per thread and step (8 rows per pass of 256 threads)
    static constexpr int LDS = ROWS * 512 > 4 * MT * RT * 1024 ? ROWS * 512 : 4 * MT * RT * 1024;
};

template <int MT, int RT>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    extern __shared__ __attribute__((aligned(16))) char lds[];
    constexpr int NL = Down<MT, RT>::NL;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Two workgroups share the ranks beyond 64, eight apart, so that they run on one XCD and find X in its L2.  (One with all 128 has a CU to
    // itself and nothing to run beside its waits: 17.9 k tokens, rank 128, 6144 -> 2048 227 us against 196, 2048 -> 2048 137 against 123.)
    const bool two = a.rank > 16 * RT;
    const int half = two ? (blockIdx.x >> 3) & 1 : 0, unit = two ? (int)(blockIdx.x >> 4) * 8 + (int)(blockIdx.x & 7) : (int)blockIdx.x;
    const int slot = unit / a.ksplit, ks = unit % a.ksplit, rank0 = half * 16 * RT;
    if (slot >= a.nslots) return;
    const Tile t = find_tile<16 * MT>(a, slot);
    if (ks == 0 && half == 0 && threadIdx.x == 0) a.tiles[slot] = t;
    if (t.n == 0 || t.adapter < 0) return;
    const int lr = threadIdx.x >> 5, lc = threadIdx.x & 31;     // this thread's row (of 8) and chunk in a pass
    const char* src[NL];
#pragma unroll
    for (int i = 0; i < NL; ++i) {
        const int r = 8 * i + lr;
        src[i] = (i < 2 * MT ? a.x + (size_t)(t.row0 + min(r, t.n - 1)) * a.ldx_b
                             : a.a + ((size_t)t.adapter * a.rank + min(rank0 + r - 16 * MT, a.rank - 1)) * a.K * 2);
    }
    const int k0 = ks * a.kchunk, k1 = min(a.K, k0 + a.kchunk);
    u32x4_t va[NL], vb[NL];
    auto fetch = [&](u32x4_t (&v)[NL], int k) {
        const size_t at = (size_t)min(k + 8 * lc, a.K - 8) * 2; // past K: something that exists; the products stop at k1
#pragma unroll
        for (int i = 0; i < NL; ++i) v[i] = *(const u32x4_t*)(src[i] + at);
    };
    f32x4_t acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[m][r] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    const int row = lane & 15, quad = lane >> 4;
    fetch(va, k0);
    if (k0 + 256 < k1) fetch(vb, k0 + 256);
    auto step = [&](u32x4_t (&v)[NL], int k) {
#pragma unroll
        for (int i = 0; i < NL; ++i) *(u32x4_t*)(lds + (8 * i + lr) * 512 + ((lc ^ ((8 * i + lr) & 15)) << 4)) = v[i];
        __syncthreads();
        if (k + 512 < k1) fetch(v, k + 512);
        if (k + 64 * wave < k1) {
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const int at = row * 512 + (((8 * wave + 4 * s + quad) ^ row) << 4);
                bf16x8_t xf[MT], af[RT];
#pragma unroll
                for (int m = 0; m < MT; ++m) xf[m] = *(const bf16x8_t*)(lds + m * 8192 + at);
#pragma unroll
                for (int r = 0; r < RT; ++r) af[r] = *(const bf16x8_t*)(lds + (MT + r) * 8192 + at);
#pragma unroll
                for (int m = 0; m < MT; ++m)
#pragma unroll
                    for (int r = 0; r < RT; ++r) acc[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[r], xf[m], acc[m][r], 0, 0, 0);
            }
        }
        __syncthreads();
    };
    for (int k = k0; k < k1; k += 512) {
        step(va, k);
        if (k + 256 < k1) step(vb, k + 256);
    }
    f32x4_t* part = (f32x4_t*)lds;                              // [4][MT RT][64]
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) part[(wave * MT * RT + m * RT + r) * 64 + lane] = acc[m][r];
    __syncthreads();
    float* u = a.u + (size_t)ks * a.T * a.rank;
#pragma unroll
    for (int i0 = 0; i0 < MT * RT; i0 += 4) {
        const int i = i0 + wave;
        if (i >= MT * RT) break;
        const f32x4_t* p = part + i * 64 + lane;
        const f32x4_t sum = (p[0] + p[MT * RT * 64]) + (p[2 * MT * RT * 64] + p[3 * MT * RT * 64]);
        const int tok = 16 * (i / RT) + row, r0 = rank0 + 16 * (i % RT) + 4 * quad;
        if (tok < t.n && r0 < a.rank) *(f32x4_t*)(u + (size_t)(t.row0 + tok) * a.rank + r0) = sum;       // rank % 8 == 0
    }
}

// 16 MT tokens x nslice features; KS steps of 32 ranks.  Two workgroups a CU also at KS = 4, by the launch bound: rank 128 as in `down` 171 us
// where one took 196; three or four at smaller KS spill (118 us against 103 at rank 32).
template <int MT, int KS>
__global__ __launch_bounds__(256, 2) void lora_up_kernel(LoraArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nsl = (a.N + a.nslice - 1) / a.nslice;
    const int slot = blockIdx.x / nsl, n0 = (blockIdx.x % nsl) * a.nslice, n1 = min(a.N, n0 + a.nslice);
    const Tile t = a.tiles[slot];
    if (t.n == 0) return;
    const int col = lane & 15, quad = lane >> 4;
    const int lr = threadIdx.x >> 5, lc = threadIdx.x & 31;     // row (of 8) and 16-byte chunk of a pass over 256 features
    if (t.adapter < 0) {
        if (a.r == a.c && a.ldr_b == a.ldc_b) return;
        for (int f0 = n0; f0 < n1; f0 += 256) {                 // all rows of a step in flight: row after row took twice the kernel's time
            u32x4_t v[2 * MT];
            const int f = f0 + 8 * lc;
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)
                v[i] = *(const u32x4_t*)(a.r + (size_t)(t.row0 + min(8 * i + lr, t.n - 1)) * a.ldr_b + (size_t)min(f, a.N - 8) * 2);
#pragma unroll
            for (int i = 0; i < 2 * MT; ++i)
                if (8 * i + lr < t.n && f < n1) *(u32x4_t*)(a.c + (size_t)(t.row0 + 8 * i + lr) * a.ldc_b + (size_t)f * 2) = v[i];
        }
        return;
    }
    const char* bp = a.b + (size_t)t.adapter * a.N * a.rank * 2;
    // Steps of 256 features, 64 a wave.  R comes in and C goes out as contiguous 512 bytes of a row; the products meet them in an fp32
    // LDS image [token][256] (a token's 16-byte chunks ch at ch ^ (token & 15)).
    __shared__ __attribute__((aligned(16))) char delta[16 * MT * 1024];
    bf16x8_t w[4][KS];
    u32x4_t rr[2 * MT];
    auto load = [&](int f0) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int f = min(f0 + 64 * wave + 16 * j + col, a.N - 1);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const int r0 = 32 * k + 8 * quad;
                bf16x8_t z;
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = (__bf16)0.f;
                w[j][k] = r0 < a.rank ? *(const bf16x8_t*)(bp + ((size_t)f * a.rank + r0) * 2) : z;
            }
        }
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i)
            rr[i] = *(const u32x4_t*)(a.r + (size_t)(t.row0 + min(8 * i + lr, t.n - 1)) * a.ldr_b + (size_t)min(f0 + 8 * lc, a.N - 8) * 2);
    };
    load(n0);                                   // flies while U is put together
    // U of the tile as bf16 pairs in LDS: the workgroup's threads sum the slabs of four ranks each (loads of eight slabs in
    // flight), ranks beyond the adapter's are zero
    constexpr int UC = 32 * KS + 8;             // padded row: the fragment reads of 16 tokens fall on different banks
    __shared__ __attribute__((aligned(16))) __bf16 us[2][16 * MT][UC];
    const float s = a.scale ? a.scale[t.adapter] : 1.0f;
    const size_t slab = (size_t)a.T * a.rank;
    for (int e = threadIdx.x; e < 16 * MT * 8 * KS; e += 256) {
        const int m = e / (8 * KS), r0 = 4 * (e % (8 * KS));
        f32x4_t v = {0.f, 0.f, 0.f, 0.f};
        if (r0 < a.rank) {
            const float* up = a.u + (size_t)(t.row0 + min(m, t.n - 1)) * a.rank + r0;
            for (int p = 0; p < a.ksplit; p += 8) {
                f32x4_t w[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) w[i] = *(const f32x4_t*)(up + (size_t)min(p + i, a.ksplit - 1) * slab);
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (p + i < a.ksplit) v += w[i];
            }
        }
        bf16x4_t h4, l4;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            __bf16 h, l;
            bf16_pair(s * v[j], h, l);
            h4[j] = h;
            l4[j] = l;
        }
        *(bf16x4_t*)&us[0][m][r0] = h4;
        *(bf16x4_t*)&us[1][m][r0] = l4;
    }
    __syncthreads();
    bf16x8_t hi[MT][KS], lo[MT][KS];            // U^T fragments: lane -> token col, ranks 32 k + 8 quad .. + 7
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            hi[m][k] = *(const bf16x8_t*)&us[0][16 * m + col][32 * k + 8 * quad];
            lo[m][k] = *(const bf16x8_t*)&us[1][16 * m + col][32 * k + 8 * quad];
        }
    for (int f0 = n0; f0 < n1; f0 += 256) {
#pragma unroll
        for (int m = 0; m < MT; ++m)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                f32x4_t acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j][k], lo[m][k], acc, 0, 0, 0);
                    acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j][k], hi[m][k], acc, 0, 0, 0);
                }
                // features 64 wave + 16 j + 4 quad .. + 3 of token col
                *(f32x4_t*)(delta + (16 * m + col) * 1024 + (((16 * wave + 4 * j + quad) ^ col) << 4)) = acc;
            }
        __syncthreads();
        u32x4_t out[2 * MT];
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const int tok = 8 * i + lr;
            const f32x4_t d0 = *(const f32x4_t*)(delta + tok * 1024 + (((2 * lc) ^ (tok & 15)) << 4));
            const f32x4_t d1 = *(const f32x4_t*)(delta + tok * 1024 + (((2 * lc + 1) ^ (tok & 15)) << 4));
            float x[8];
            unpack8(rr[i], x);
            out[i] = (u32x4_t){pack_bf16x2(x[0] + d0[0], x[1] + d0[1]), pack_bf16x2(x[2] + d0[2], x[3] + d0[3]),
                               pack_bf16x2(x[4] + d1[0], x[5] + d1[1]), pack_bf16x2(x[6] + d1[2], x[7] + d1[3])};
        }
        if (f0 + 256 < n1) load(f0 + 256);
#pragma unroll
        for (int i = 0; i < 2 * MT; ++i) {
            const int tok = 8 * i + lr;
            if (tok < t.n && f0 + 8 * lc < n1) *(u32x4_t*)(a.c + (size_t)(t.row0 + tok) * a.ldc_b + (size_t)(f0 + 8 * lc) * 2) = out[i];
        }
        __syncthreads();
    }
}

// Both products of 16 tokens in one launch, for batches that wait for latency and not for bytes (single tokens of some requests): a
// workgroup of 16 waves takes 1024 features of a tile and computes the tile's U for itself, K cut over the waves, fragments straight from
// memory with everything in flight at once: weights and R of the second product while the first one runs.
template <int RT>
__global__ __launch_bounds__(1024) void lora_one_kernel(LoraArgs a) {
    __shared__ f32x4_t part[16][RT][64];
    __shared__ __attribute__((aligned(16))) __bf16 us[2][16][40];        // rows of 32 ranks, padded
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int col = lane & 15, quad = lane >> 4;
    const int nsl = (a.N + 1023) / 1024, n0 = (int)(blockIdx.x % nsl) * 1024;
    const Tile t = find_tile<16>(a, blockIdx.x / nsl);
    if (t.n == 0) return;
    const int f0 = n0 + 64 * wave;
    const size_t row = t.row0 + min(col, t.n - 1);
    // R, and the weights of the second product: row m of block j is feature 32 (j >> 1) + 8 (m >> 2) + 4 (j & 1) + (m & 3), so that a
    // lane's accumulators of two blocks are 8 consecutive features of its token
    u32x4_t rr[2];
    bf16x8_t w[4];
    const char* bp = a.b + (size_t)max(t.adapter, 0) * a.N * a.rank * 2;
#pragma unroll
    for (int q = 0; q < 2; ++q) rr[q] = *(const u32x4_t*)(a.r + row * a.ldr_b + (size_t)min(f0 + 32 * q + 8 * quad, a.N - 8) * 2);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const int f = min(f0 + 32 * (j >> 1) + 8 * (col >> 2) + 4 * (j & 1) + (col & 3), a.N - 1);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[j][e] = (__bf16)0.f;
        if (8 * quad < a.rank) w[j] = *(const bf16x8_t*)(bp + ((size_t)f * a.rank + 8 * quad) * 2);
    }
    f32x4_t acc[4];
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        float x[8];
        unpack8(rr[q], x);
        acc[2 * q] = (f32x4_t){x[0], x[1], x[2], x[3]};
        acc[2 * q + 1] = (f32x4_t){x[4], x[5], x[6], x[7]};
    }
    if (t.adapter >= 0) {
        const char* xp = a.x + row * a.ldx_b + quad * 16;
        f32x4_t u[RT];
        const char* ap[RT];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            u[r] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
            ap[r] = a.a + ((size_t)t.adapter * a.rank + min(16 * r + col, a.rank - 1)) * a.K * 2 + quad * 16;
        }
        for (int k = 64 * wave; k < a.K; k += 2048) {                    // two 128-byte lines of every row per wave and step
            bf16x8_t xf[4], af[4][RT];
#pragma unroll
            for (int s = 0; s < 4; ++s) {
                const size_t at = (size_t)min(k + 1024 * (s >> 1), a.K - 64) * 2 + (s & 1) * 64;
                xf[s] = *(const bf16x8_t*)(xp + at);
#pragma unroll
                for (int r = 0; r < RT; ++r) af[s][r] = *(const bf16x8_t*)(ap[r] + at);
            }
#pragma unroll
            for (int s = 0; s < 4; ++s)
                if (k + 1024 * (s >> 1) < a.K) {
#pragma unroll
                    for (int r = 0; r < RT; ++r) u[r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(af[s][r], xf[s], u[r], 0, 0, 0);
                }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) part[wave][r][lane] = u[r];
        __syncthreads();
        if (wave < 2) {                                                  // ranks 16 wave + 4 quad .. + 3 of token col
            f32x4_t v = {0.f, 0.f, 0.f, 0.f};
            if (wave < RT && 16 * wave + 4 * quad < a.rank) {
#pragma unroll
                for (int i = 0; i < 16; ++i) v += part[i][wave < RT ? wave : 0][lane];
            }
            const float s = a.scale ? a.scale[t.adapter] : 1.0f;
            bf16x4_t h4, l4;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                __bf16 h, l;
                bf16_pair(s * v[j], h, l);
                h4[j] = h;
                l4[j] = l;
            }
            *(bf16x4_t*)&us[0][col][16 * wave + 4 * quad] = h4;
            *(bf16x4_t*)&us[1][col][16 * wave + 4 * quad] = l4;
        }
        __syncthreads();
        const bf16x8_t hi = *(const bf16x8_t*)&us[0][col][8 * quad], lo = *(const bf16x8_t*)&us[1][col][8 * quad];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j], lo, acc[j], 0, 0, 0);
            acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j], hi, acc[j], 0, 0, 0);
        }
    } else if (a.r == a.c && a.ldr_b == a.ldc_b) {
        return;
    }
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const int f = f0 + 32 * q + 8 * quad;
        const u32x4_t v = {pack_bf16x2(acc[2 * q][0], acc[2 * q][1]), pack_bf16x2(acc[2 * q][2], acc[2 * q][3]),
                           pack_bf16x2(acc[2 * q + 1][0], acc[2 * q + 1][1]), pack_bf16x2(acc[2 * q + 1][2], acc[2 * q + 1][3])};
        if (col < t.n && f < a.N) *(u32x4_t*)(a.c + row * a.ldc_b + (size_t)f * 2) = v;
    }
}

struct Plan {
    bool one;                                   // one launch
    int mt, ksplit, kchunk, nslice;             // mt: 16-token blocks per tile
    long long nslots;
};

Plan make_plan(int T, int B, int N, int K, int rank, int cus) {
    Plan p;
    // 16 tokens a tile where sequences have no more on average, else 32 (us with 16 / 32: 32 x 16 tokens, rank 64, 2048 -> 4096 13.2 / 14.5,
    // 32 x 20 15.5 / 15.0, 32 x 32, 6144 -> 2048 16.7 / 16.0, prompts as above 118 / 103).  64 a tile, with fewer
    // workgroups on a CU: prompts, rank 64, 6144 -> 2048 108 against 106, rank 128 184 against 171
    p.mt = (double)T / B <= 16 ? 1 : 2;
    p.nslots = (long long)T / (16 * p.mt) + B;
    const long long tiles = ((long long)T + 16 * p.mt - 1) / (16 * p.mt) > B ? ((long long)T + 16 * p.mt - 1) / (16 * p.mt) : B;
    // One launch where a CU gets at most one workgroup of it and the A that each of them reads is small: us a call one / two launches, rank 16,
    // 2048 -> 4096: 9.3 / 12.4 with 32 single tokens, 9.6 / 12.4 with 64 (256 workgroups), 13.7 / 13.6 with 128; rank 16, 6144 -> 2048 (A of
    // 98 k values): equal
    p.one = p.mt == 1 && rank <= 32 && (long long)rank * K <= 65536 && tiles * ((N + 1023) / 1024) <= cus;
    // features of a workgroup: two steps where that leaves a workgroup per CU (U is put together once for both: prompts 103 us against 110
    // with one step, and 104 with four), else one (32 blocks as above 15.4 us, 16.3 with two)
    p.nslice = tiles * ((N + 511) / 512) >= cus ? 512 : 256;
    // K ranges: one workgroup per CU; up to four where the slabs of U, written once and read by every slice of the second launch, stay under
    // an eighth of X, R and C.  us with 1 / 2 / 4 / 8 / 16 ranges: prompts 108 / 103 / 105 / 115 / 148 (two taken), 32 blocks 34 / 24 / 18 / 16.3
    // / 19 (eight taken), 64 x 64 tokens, rank 64, 2048 -> 4096 34 / 30.5 / 30.7 / 37 / 52.  No range under one step of the four waves.
    const long long slab = 4LL * rank * (1 + (N + p.nslice - 1) / p.nslice), most = (2LL * K + 4LL * N) / 8 / slab;
    long long ks = (4LL * cus + tiles - 1) / tiles;
    if (ks > most) ks = most;
    if (ks < (cus + tiles - 1) / tiles) ks = (cus + tiles - 1) / tiles;
    if (ks > K / 256) ks = K / 256;
    if (ks < 1) ks = 1;
    p.kchunk = (int)(((K + ks - 1) / ks + 63) / 64 * 64);
    p.ksplit = (K + p.kchunk - 1) / p.kchunk;
    return p;
}

long long plan_bytes(const Plan& p, int T, int rank) { return p.one ? 0 : p.nslots * (long long)sizeof(Tile) + (long long)p.ksplit * T * rank * 4; }

}  // namespace

extern "C" long long coda_lora_workspace_bytes(int T, int B, int N, int K, int rank) {
    if (T <= 0 || B <= 0 || N <= 0 || K <= 0 || rank <= 0 || T > 1 << 28 || N > 1 << 30 || K > 1 << 30 || rank > 128) return 0;
    return plan_bytes(make_plan(T, B, N, K, rank, coda_device_cus()), T, rank);
}

extern "C" int coda_lora_bf16(const void* X, long long ldx, const void* A, const void* Bw, const float* scale, const int* seq_start,
                              const int* adapter, int B, int T, int n_adapters, int rank, const void* R, long long ldr, void* C,
                              long long ldc, int N, int K, void* workspace, long long workspace_bytes, void* stream) {
    const char* who = "coda_lora_bf16";
    if (B <= 0 || T <= 0 || n_adapters <= 0 || N <= 0 || K <= 0) return coda_refuse(who, CODA_ERR_SHAPE, "a size is not positive");
    // running sums over 64 sequences of tiles stay below 2^31 even for starts that make every sequence T rows long
    if (T > 1 << 28) return coda_refuse(who, CODA_ERR_SHAPE, "T exceeds 2^28");
    if (N > 1 << 30 || K > 1 << 30) return coda_refuse(who, CODA_ERR_SHAPE, "N or K exceeds 2^30");       // sums with tile sizes would wrap
    if (rank <= 0 || rank % 8 || rank > 128) return coda_refuse(who, CODA_ERR_SHAPE, "rank is a multiple of 8 up to 128");
    if (K % 64 || N % 8) return coda_refuse(who, CODA_ERR_SHAPE, "K % 64 or N % 8");
    if (ldx < K || ldr < N || ldc < N) return coda_refuse(who, CODA_ERR_SHAPE, "a row stride is shorter than a row");
    if (!X || !A || !Bw || !seq_start || !adapter || !R || !C) return coda_refuse(who, CODA_ERR_ARG, "null pointer");
    if (((uintptr_t)X | (uintptr_t)A | (uintptr_t)Bw | (uintptr_t)R | (uintptr_t)C) & 15 || (ldx * 2) % 16 || (ldr * 2) % 16 || (ldc * 2) % 16)
        return coda_refuse(who, CODA_ERR_ALIGN, "rows start on 16 bytes");
    const Plan p = make_plan(T, B, N, K, rank, coda_device_cus());
    if (!p.one && (!workspace || workspace_bytes < plan_bytes(p, T, rank)))
        return coda_refuse(who, CODA_ERR_ARG, "workspace is smaller than coda_lora_workspace_bytes");
    if ((uintptr_t)workspace & 15) return coda_refuse(who, CODA_ERR_ALIGN, "the workspace starts on 16 bytes");
    const long long downs = rank > 64 ? (p.nslots * p.ksplit + 7) / 8 * 16 : p.nslots * p.ksplit, ups = p.nslots * ((N + p.nslice - 1) / p.nslice);
    if (!p.one && (!grid_fits(downs, 256) || !grid_fits(ups, 256))) return coda_refuse(who, CODA_ERR_SHAPE, "too many tiles for one launch");
    LoraArgs a;
    a.x = (const char*)X; a.ldx_b = ldx * 2;
    a.a = (const char*)A; a.b = (const char*)Bw; a.scale = scale;
    a.seq_start = seq_start; a.adapter = adapter; a.B = B; a.T = T; a.n_adapters = n_adapters; a.rank = rank;
    a.r = (const char*)R; a.ldr_b = ldr * 2;
    a.c = (char*)C; a.ldc_b = ldc * 2;
    a.N = N; a.K = K;
    a.nslots = (int)p.nslots; a.ksplit = p.ksplit; a.kchunk = p.kchunk; a.nslice = p.nslice;
    a.tiles = (Tile*)workspace;
    a.u = (float*)(a.tiles + p.nslots);
    hipStream_t st = (hipStream_t)stream;
    const dim3 gd((unsigned)downs), gu((unsigned)ups), block(256);
    if (p.one) {
        const dim3 g1((unsigned)(p.nslots * ((N + 1023) / 1024)));
        if (rank <= 16) hipLaunchKernelGGL(lora_one_kernel<1>, g1, dim3(1024), 0, st, a);
        else hipLaunchKernelGGL(lora_one_kernel<2>, g1, dim3(1024), 0, st, a);
        CODA_CHECK_LAUNCH("lora");
        return CODA_OK;
    }
    auto down = [&](auto kernel, int lds) -> int {
        if (coda_ensure_dyn_lds((const void*)kernel, lds) != CODA_OK) return CODA_ERR_LAUNCH;
        hipLaunchKernelGGL(kernel, gd, block, lds, st, a);
        CODA_CHECK_LAUNCH("lora down");
        return CODA_OK;
    };
    // ranks in blocks of 16 (down) and 32 (up)
    auto go = [&](auto mt) -> int {
        constexpr int MT = decltype(mt)::value;
        int rc;
        if (rank <= 16) rc = down(lora_down_kernel<MT, 1>, Down<MT, 1>::LDS);
        else if (rank <= 32) rc = down(lora_down_kernel<MT, 2>, Down<MT, 2>::LDS);
        else rc = down(lora_down_kernel<MT, 4>, Down<MT, 4>::LDS);
        if (rc != CODA_OK) return rc;
        if (rank <= 32) hipLaunchKernelGGL((lora_up_kernel<MT, 1>), gu, block, 0, st, a);
        else if (rank <= 64) hipLaunchKernelGGL((lora_up_kernel<MT, 2>), gu, block, 0, st, a);
        else hipLaunchKernelGGL((lora_up_kernel<MT, 4>), gu, block, 0, st, a);
        CODA_CHECK_LAUNCH("lora up");
        return CODA_OK;
    };
    return p.mt == 1 ? go(std::integral_constant<int, 1>{}) : go(std::integral_constant<int, 2>{});
}
