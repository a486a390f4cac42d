// Low-rank adapters of many requests beside a shared projection, on a ragged batch:
//
//     C[t] = R[t] + s[a] (X[t] A[a]^T) B[a]^T,     a = the adapter of t's sequence;  no adapter: C[t] = R[t]
//
// Two launches.  `down` computes U = X A^T for tiles of one sequence's tokens, K cut over the waves of a workgroup and, where there
// are few tiles, over workgroups (fp32 slabs in the workspace, summed in a fixed order by their readers).  `up` sums the slabs, scales, and
// adds U B^T to R with R as the start value of the accumulators, so that the result is rounded once.
//
// v_mfma_f32_16x16x32_bf16 in both, weights as the A operand: a lane then holds four consecutive outputs (ranks, features) of one
// token.  Both products read each weight and activation once per tile straight into fragments, 64 B of a row a quarter-wave: there is
// too little reuse at serving ranks (8 .. 128) for a detour through LDS to pay.  U enters the second product as a bf16 pair
// (value and remainder): the extra matrix instructions are free in a kernel that waits for memory, and U keeps 16 bits.
#include "paged_common.h"

using namespace paged;

namespace {

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
};

struct Tile {
    int b, s0, n, t0, adapter;                  // sequence, its first row, its tokens; the tile's first token; -1: no adapter
};

// tile slots of sequence b start at floor(start_b / TM) + b (paged_attn.hip numbers its tiles the same way)
template <int TM>
__device__ __forceinline__ bool find_tile(const LoraArgs& a, int slot, Tile& t) {
    auto first = [&](int i) { return (long long)(clamp_start(a.seq_start, i, a.T) / TM + i); };
    t.b = wave_search(a.B, slot, first);
    if (t.b < 0) return false;
    t.s0 = clamp_start(a.seq_start, t.b, a.T);
    t.n = clamp_start(a.seq_start, t.b + 1, a.T) - t.s0;
    const long long t0 = (slot - first(t.b)) * TM;
    t.t0 = (int)t0;
    const int ad = a.adapter[t.b];
    t.adapter = (unsigned)ad < (unsigned)a.n_adapters ? ad : -1;
    return t0 < t.n;
}

// U of 16 MT tokens, 16 RT ranks (those beyond the adapter's are computed from its last row and dropped)
template <int MT, int RT>
__global__ __launch_bounds__(256) void lora_down_kernel(LoraArgs a) {
    __shared__ f32x4_t part[4][MT * RT][64];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int slot = blockIdx.x / a.ksplit, ks = blockIdx.x % a.ksplit;
    Tile t;
    if (!find_tile<16 * MT>(a, slot, t) || t.adapter < 0) return;
    const int row = lane & 15, quad = lane >> 4;
    const char* xp[MT];
    const char* ap[RT];
#pragma unroll
    for (int m = 0; m < MT; ++m) xp[m] = a.x + (size_t)(t.s0 + min(t.t0 + 16 * m + row, t.n - 1)) * a.ldx_b + quad * 16;
#pragma unroll
    for (int r = 0; r < RT; ++r)
        ap[r] = a.a + ((size_t)t.adapter * a.rank + min(16 * r + row, a.rank - 1)) * a.K * 2 + quad * 16;
    f32x4_t acc[MT][RT];
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) acc[m][r] = (f32x4_t){0.f, 0.f, 0.f, 0.f};
    const int k1 = min(a.K, (ks + 1) * a.kchunk);
    // 64 elements (one 128-byte line of every row) a step, the four waves in turn; the next step's fragments fly under this one's
    bf16x8_t xf[2][MT], af[2][RT];
    auto load = [&](int k) {
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int m = 0; m < MT; ++m) xf[s][m] = *(const bf16x8_t*)(xp[m] + (size_t)k * 2 + s * 64);
#pragma unroll
            for (int r = 0; r < RT; ++r) af[s][r] = *(const bf16x8_t*)(ap[r] + (size_t)k * 2 + s * 64);
        }
    };
    int k = ks * a.kchunk + 64 * wave;
    if (k < k1) load(k);
    for (; k < k1; k += 256) {
        bf16x8_t xc[2][MT], ac[2][RT];
#pragma unroll
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int m = 0; m < MT; ++m) xc[s][m] = xf[s][m];
#pragma unroll
            for (int r = 0; r < RT; ++r) ac[s][r] = af[s][r];
        }
        load(min(k + 256, a.K - 64));          // past the range: a line that exists, not used
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int m = 0; m < MT; ++m)
#pragma unroll
                for (int r = 0; r < RT; ++r) acc[m][r] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ac[s][r], xc[s][m], acc[m][r], 0, 0, 0);
    }
#pragma unroll
    for (int m = 0; m < MT; ++m)
#pragma unroll
        for (int r = 0; r < RT; ++r) part[wave][m * RT + r][lane] = acc[m][r];
    __syncthreads();
    float* u = a.u + (size_t)ks * a.T * a.rank;
#pragma unroll
    for (int i0 = 0; i0 < MT * RT; i0 += 4) {
        const int i = i0 + wave;
        if (i >= MT * RT) break;
        const f32x4_t sum = (part[0][i][lane] + part[1][i][lane]) + (part[2][i][lane] + part[3][i][lane]);
        const int tok = t.t0 + 16 * (i / RT) + row, r0 = 16 * (i % RT) + 4 * quad;
        if (tok < t.n && r0 < a.rank) *(f32x4_t*)(u + (size_t)(t.s0 + tok) * a.rank + r0) = sum;       // rank % 8 == 0
    }
}

// 16 MT tokens x nslice features; KS steps of 32 ranks
template <int MT, int KS>
__global__ __launch_bounds__(256) void lora_up_kernel(LoraArgs a) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nsl = (a.N + a.nslice - 1) / a.nslice;
    const int slot = blockIdx.x / nsl, n0 = (blockIdx.x % nsl) * a.nslice, n1 = min(a.N, n0 + a.nslice);
    Tile t;
    if (!find_tile<16 * MT>(a, slot, t)) return;
    const int col = lane & 15, quad = lane >> 4;
    if (t.adapter < 0) {
        if (a.r == a.c && a.ldr_b == a.ldc_b) return;
        for (int m = 0; m < 16 * MT && t.t0 + m < t.n; ++m) {
            const size_t row = t.s0 + t.t0 + m;
            for (int f = n0 + 8 * (int)threadIdx.x; f < n1; f += 2048)
                *(u32x4_t*)(a.c + row * a.ldc_b + (size_t)f * 2) = *(const u32x4_t*)(a.r + row * a.ldr_b + (size_t)f * 2);
        }
        return;
    }
    // U^T fragments: lane -> token col, ranks 32 k + 8 quad .. + 7
    bf16x8_t hi[MT][KS], lo[MT][KS];
    const float s = a.scale ? a.scale[t.adapter] : 1.0f;
#pragma unroll
    for (int m = 0; m < MT; ++m) {
        const float* up = a.u + (size_t)(t.s0 + min(t.t0 + 16 * m + col, t.n - 1)) * a.rank;
#pragma unroll
        for (int k = 0; k < KS; ++k) {
            const int r0 = 32 * k + 8 * quad;
            f32x4_t v0 = {0.f, 0.f, 0.f, 0.f}, v1 = v0;
            if (r0 < a.rank)
                for (int p = 0; p < a.ksplit; ++p) {
                    const f32x4_t* q = (const f32x4_t*)(up + (size_t)p * a.T * a.rank + r0);
                    v0 += q[0];
                    v1 += q[1];
                }
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float v = s * (j < 4 ? v0[j & 3] : v1[j & 3]);
                hi[m][k][j] = (__bf16)v;
                lo[m][k][j] = (__bf16)(v - (float)hi[m][k][j]);
            }
        }
    }
    const char* bp = a.b + (size_t)t.adapter * a.N * a.rank * 2;
    // 64 features a step, the four waves in turn.  Row m of weight block j is feature 16 (m >> 2) + 4 j + (m & 3): the accumulators
    // of the four blocks then are 16 CONSECUTIVE features of a lane's token, two 16-byte pieces of R and C
    for (int f0 = n0 + 64 * wave; f0 < n1; f0 += 256) {
        bf16x8_t w[4][KS];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int f = min(f0 + 16 * (col >> 2) + 4 * j + (col & 3), a.N - 1);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
                const int r0 = 32 * k + 8 * quad;
                bf16x8_t z;
#pragma unroll
                for (int e = 0; e < 8; ++e) z[e] = (__bf16)0.f;
                w[j][k] = r0 < a.rank ? *(const bf16x8_t*)(bp + ((size_t)f * a.rank + r0) * 2) : z;
            }
        }
        const int f = f0 + 16 * quad;
#pragma unroll
        for (int m = 0; m < MT; ++m) {
            const int tok = t.t0 + 16 * m + col;
            const bool live = tok < t.n;
            const size_t row = t.s0 + min(tok, t.n - 1);
            f32x4_t acc[4];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                float x[8];
                unpack8(*(const u32x4_t*)(a.r + row * a.ldr_b + (size_t)min(f + 8 * q, a.N - 8) * 2), x);
                acc[2 * q] = (f32x4_t){x[0], x[1], x[2], x[3]};
                acc[2 * q + 1] = (f32x4_t){x[4], x[5], x[6], x[7]};
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
#pragma unroll
                for (int k = 0; k < KS; ++k) {
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j][k], lo[m][k], acc[j], 0, 0, 0);
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(w[j][k], hi[m][k], acc[j], 0, 0, 0);
                }
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const u32x4_t v = {pack_bf16x2(acc[2 * q][0], acc[2 * q][1]), pack_bf16x2(acc[2 * q][2], acc[2 * q][3]),
                                   pack_bf16x2(acc[2 * q + 1][0], acc[2 * q + 1][1]), pack_bf16x2(acc[2 * q + 1][2], acc[2 * q + 1][3])};
                if (live && f + 8 * q < n1) *(u32x4_t*)(a.c + row * a.ldc_b + (size_t)(f + 8 * q) * 2) = v;
            }
        }
    }
}

struct Plan {
    int mt, ksplit, kchunk, nslice;
    long long nslots;
};

Plan make_plan(int T, int B, int N, int K, int rank, int cus) {
    Plan p;
    const double rho = (double)T / B;                           // tokens per sequence, on average
    p.mt = rho <= 16 ? 1 : rho <= 32 || rank > 64 ? 2 : 4;
    p.nslots = (long long)T / (16 * p.mt) + B;
    const long long tiles = ((long long)T + 16 * p.mt - 1) / (16 * p.mt) > B ? ((long long)T + 16 * p.mt - 1) / (16 * p.mt) : B;
    // two workgroups per CU, no K range shorter than the four waves' steps
    long long ks = (2LL * cus + tiles - 1) / tiles;
    if (ks > K / 256) ks = K / 256;
    if (ks < 1) ks = 1;
    p.kchunk = (int)(((K + ks - 1) / ks + 63) / 64 * 64);
    p.ksplit = (K + p.kchunk - 1) / p.kchunk;
    // features of a workgroup: 256 (one step of each wave), more when that still makes eight workgroups per CU
    p.nslice = 256;
    while (p.nslice < 1024 && p.nslice < N && tiles * ((N + 2 * p.nslice - 1) / (2 * p.nslice)) >= 8LL * cus) p.nslice *= 2;
    return p;
}

}  // namespace

extern "C" long long coda_lora_workspace_bytes(int T, int B, int N, int K, int rank) {
    if (T <= 0 || B <= 0 || N <= 0 || K <= 0 || rank <= 0) return 0;
    return (long long)make_plan(T, B, N, K, rank, coda_device_cus()).ksplit * T * rank * 4;
}

extern "C" int coda_lora_bf16(const void* X, long long ldx, const void* A, const void* Bw, const float* scale, const int* seq_start,
                              const int* adapter, int B, int T, int n_adapters, int rank, const void* R, long long ldr, void* C,
                              long long ldc, int N, int K, void* workspace, long long workspace_bytes, void* stream) {
    const char* who = "coda_lora_bf16";
    if (B <= 0 || T <= 0 || n_adapters <= 0 || N <= 0 || K <= 0) return coda_refuse(who, CODA_ERR_SHAPE, "a size is not positive");
    if (rank <= 0 || rank % 8 || rank > 128) return coda_refuse(who, CODA_ERR_SHAPE, "rank is a multiple of 8 up to 128");
    if (K % 64 || N % 8) return coda_refuse(who, CODA_ERR_SHAPE, "K % 64 or N % 8");
    if (ldx < K || ldr < N || ldc < N) return coda_refuse(who, CODA_ERR_SHAPE, "a row stride is shorter than a row");
    if (!X || !A || !Bw || !seq_start || !adapter || !R || !C) return coda_refuse(who, CODA_ERR_ARG, "null pointer");
    if (((uintptr_t)X | (uintptr_t)A | (uintptr_t)Bw | (uintptr_t)R | (uintptr_t)C) & 15 || (ldx * 2) % 16 || (ldr * 2) % 16 || (ldc * 2) % 16)
        return coda_refuse(who, CODA_ERR_ALIGN, "rows start on 16 bytes");
    const Plan p = make_plan(T, B, N, K, rank, coda_device_cus());
    if (!workspace || workspace_bytes < (long long)p.ksplit * T * rank * 4)
        return coda_refuse(who, CODA_ERR_ARG, "workspace is smaller than coda_lora_workspace_bytes");
    if ((uintptr_t)workspace & 15) return coda_refuse(who, CODA_ERR_ALIGN, "the workspace starts on 16 bytes");
    const long long downs = p.nslots * p.ksplit, ups = p.nslots * ((N + p.nslice - 1) / p.nslice);
    if (downs > 0x7fffffffLL || ups > 0x7fffffffLL) return coda_refuse(who, CODA_ERR_SHAPE, "too many tiles for one launch");
    LoraArgs a;
    a.x = (const char*)X; a.ldx_b = ldx * 2;
    a.a = (const char*)A; a.b = (const char*)Bw; a.scale = scale;
    a.seq_start = seq_start; a.adapter = adapter; a.B = B; a.T = T; a.n_adapters = n_adapters; a.rank = rank;
    a.r = (const char*)R; a.ldr_b = ldr * 2;
    a.c = (char*)C; a.ldc_b = ldc * 2;
    a.N = N; a.K = K;
    a.nslots = (int)p.nslots; a.ksplit = p.ksplit; a.kchunk = p.kchunk; a.nslice = p.nslice;
    a.u = (float*)workspace;
    hipStream_t st = (hipStream_t)stream;
    const dim3 gd((unsigned)downs), gu((unsigned)ups), block(256);
    const int rt = rank <= 16 ? 1 : rank <= 32 ? 2 : rank <= 64 ? 4 : 8;
#define CODA_LORA_RANKS(MT)                                                                             \
    do {                                                                                                \
        if (rt == 1) hipLaunchKernelGGL((lora_down_kernel<MT, 1>), gd, block, 0, st, a);                \
        else if (rt == 2) hipLaunchKernelGGL((lora_down_kernel<MT, 2>), gd, block, 0, st, a);           \
        else if (rt == 4) hipLaunchKernelGGL((lora_down_kernel<MT, 4>), gd, block, 0, st, a);           \
        else hipLaunchKernelGGL((lora_down_kernel<(MT > 2 ? 2 : MT), 8>), gd, block, 0, st, a);         \
        CODA_CHECK_LAUNCH("lora down");                                                                 \
        if (rt <= 2) hipLaunchKernelGGL((lora_up_kernel<MT, 1>), gu, block, 0, st, a);                  \
        else if (rt == 4) hipLaunchKernelGGL((lora_up_kernel<MT, 2>), gu, block, 0, st, a);             \
        else hipLaunchKernelGGL((lora_up_kernel<(MT > 2 ? 2 : MT), 4>), gu, block, 0, st, a);           \
        CODA_CHECK_LAUNCH("lora up");                                                                   \
    } while (0)
    if (p.mt == 1) CODA_LORA_RANKS(1);
    else if (p.mt == 2) CODA_LORA_RANKS(2);
    else CODA_LORA_RANKS(4);                    // rank <= 64: make_plan gives larger ranks at most 32 tokens a tile
#undef CODA_LORA_RANKS
    return CODA_OK;
}
