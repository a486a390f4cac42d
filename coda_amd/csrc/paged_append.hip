// Keys and values of new tokens into a paged cache, with q/k RMSNorm and the rotary embedding on the way.
//
// For token i of sequence b at position p = pos0[b] + i, every q and k head row x of 128 becomes
//     n = w x / sqrt(mean(x^2) + eps),      y_j = n_j cos_pj - n_{j+64} sin_pj (j < 64),  n_j cos_pj + n_{j-64} sin_pj (j >= 64)
// q rows go to q_out, k rows (y) and v rows (x) to slot p % page_size of page page_table[b, p / page_size].
//
// Memory-bound: a token moves (n_q + 2 n_kv) rows in and as many out, about ten operations an element.  A row of 256 B is 16
// lanes of 16 B (the rotary partner j ^ 64 is lane ^ 8), a wave works on ONE token, four rows at a time, so the sequence
// search, the cos / sin rows and the page lookup are paid once per wave.  `parts` waves share a token: all its rows at
// once when there are few tokens (latency), a wave per sixteen rows when there are many.
// Measured (16 q and 8 k/v heads): 15.6 k tokens to bf16 pages 51 us = 5.2 TB/s, the rate of a large copy; 4096 to e4m3 pages 16.5 us =
// 3.7 TB/s; 32 single tokens 3.8 us.  More waves in flight by fewer registers (launch bounds 8) took 105 us where this takes 51: rows
// are then no longer loaded ahead.
#include "paged_common.h"
#include <stdio.h>

using namespace paged;

int coda_refuse(const char* who, int code, const char* why) {
    char msg[240];
    snprintf(msg, sizeof(msg), "%s: %s", who, why);
    coda_set_last_error_msg(msg);
    return code;
}

int coda_check_pages(const char* who, const void* k_cache, const void* v_cache, const int* page_table, long long ld_table, int max_pages,
                     long long page_stride, int num_pages, int page_size, int cache_type, float k_scale, float v_scale, int n_kv, Pages* out) {
    if (!k_cache || !v_cache || !page_table) return coda_refuse(who, CODA_ERR_ARG, "null cache or page table");
    if (cache_type != CODA_CACHE_BF16 && cache_type != CODA_CACHE_E4M3) return coda_refuse(who, CODA_ERR_ARG, "unknown cache type");
    // !(s > 0) also catches NaN; an infinite scale would store zeros and read NaN
    if (cache_type == CODA_CACHE_E4M3 && (!(k_scale > 0.f) || !(v_scale > 0.f) || k_scale > 1e30f || v_scale > 1e30f || k_scale < 1e-30f || v_scale < 1e-30f))
        return coda_refuse(who, CODA_ERR_ARG, "scales of an e4m3 cache lie in [1e-30, 1e30]");
    if (max_pages <= 0 || num_pages <= 0 || page_size <= 0 || ld_table < max_pages) return coda_refuse(who, CODA_ERR_SHAPE, "page table or page size");
    if (n_kv > MAX_HEADS) return coda_refuse(who, CODA_ERR_SHAPE, "too many heads");        // the size of a page would wrap
    if ((long long)max_pages * page_size > 0x7fffffffLL) return coda_refuse(who, CODA_ERR_SHAPE, "max_pages * page_size exceeds 2^31 - 1");
    const int elt = cache_type == CODA_CACHE_E4M3 ? 1 : 2;
    if (page_stride < (long long)n_kv * page_size * HEAD_DIM) return coda_refuse(who, CODA_ERR_SHAPE, "page_stride is smaller than a page");
    if (((uintptr_t)k_cache | (uintptr_t)v_cache) & 15 || (page_stride * elt) % 16) return coda_refuse(who, CODA_ERR_ALIGN, "pages start on 16 bytes");
    out->table = page_table; out->ld_table = ld_table; out->max_pages = max_pages; out->num_pages = num_pages;
    out->page = make_fast_div((unsigned int)page_size);
    out->row_b = HEAD_DIM * elt;
    out->page_stride_b = page_stride * elt;
    out->head_stride_b = (long long)page_size * out->row_b;
    return CODA_OK;
}

namespace {

struct AppendArgs {
    const char* qkv; long long ld_b;
    char* q_out; long long ldq_b;
    const u32x4_t* qw; const u32x4_t* kw;     // null: no norm
    const u32x4_t* cos; const u32x4_t* sin; int max_pos;
    const int* seq_start; const int* pos0; int B, T;
    Pages pg;
    char* k; char* v;
    float k_inv, v_inv;
    int n_q, n_kv, parts;
    float eps;
};

// Eight values as e4m3 (round to nearest even), clamped to the type's largest value 448 like every saturating conversion to
// it; a NaN stays a NaN (min / max alone would drop it).
__device__ __forceinline__ u32x2_t pack_e4m3(const float (&f)[8]) {
    float c[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) c[j] = f[j] != f[j] ? f[j] : fminf(fmaxf(f[j], -448.f), 448.f);
    u32x2_t o;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        int w = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * i], c[4 * i + 1], 0, false);
        w = __builtin_amdgcn_cvt_pk_fp8_f32(c[4 * i + 2], c[4 * i + 3], w, true);
        o[i] = (unsigned int)w;
    }
    return o;
}

// lane -> the lane `N` further on, round its group of 16: a register move, where __shfl_xor goes through LDS
template <int N>
__device__ __forceinline__ float rotate16(float v) {
    return __uint_as_float(__builtin_amdgcn_update_dpp(0, (int)__float_as_uint(v), 0x120 + N, 0xf, 0xf, false));
}

// sum over the 16 lanes of a row, in the pairs (and with the bits) of a butterfly of 8, 4, 2, 1
__device__ __forceinline__ float row_sum(float v) {
    v += rotate16<8>(v);
    v += rotate16<4>(v);
    v += rotate16<2>(v);
    return v + rotate16<1>(v);
}

// F8: e4m3 cache.  STEPWISE: bf16 after every operation, the rounding points (and bits) of coda_qknorm_rope; otherwise
// everything stays in fp32 and is rounded once, to the type it is stored in.
template <bool F8, bool STEPWISE>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
    const int lane = threadIdx.x & 63, sub = lane & 15, grp = lane >> 4;
    const long long wave = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long tl = wave / a.parts;
    if (tl >= a.T) return;
    const int t = __builtin_amdgcn_readfirstlane((int)tl), part = __builtin_amdgcn_readfirstlane((int)(wave - tl * a.parts));
    const char* row = a.qkv + (size_t)t * a.ld_b + sub * 16;
    const int n_heads = a.n_q + 2 * a.n_kv, step = 4 * a.parts;
    // four rows of loads in flight per lane, the first before anything is known about the token; a row beyond the last head re-reads the
    // last one and stores nothing
    u32x4_t raw[4];
    auto load = [&](int h0) {
#pragma unroll
        for (int u = 0; u < 4; ++u) raw[u] = *(const u32x4_t*)(row + (size_t)min(h0 + u * step, n_heads - 1) * 256);
    };
    load(part * 4 + grp);
    const Seq q = seq_of_token({a.seq_start, a.pos0, nullptr, a.B, a.T}, t);
    if (q.b < 0) return;                                        // a row of no sequence: left alone
    const int b = q.b;
    const long long p64 = (long long)q.x + (t - q.s0);
    if (p64 < 0 || p64 >= a.max_pos) return;                    // no rotary row: nothing is written for this token
    const int pos = (int)p64;
    const int lp = fast_div(a.pg.page, pos), slot = pos - lp * (int)a.pg.page.d;
    const int page = lp < a.pg.max_pages ? a.pg.table[(size_t)b * a.pg.ld_table + lp] : -1;
    const bool store = (unsigned)page < (unsigned)a.pg.num_pages;
    const size_t at = store ? (size_t)page * a.pg.page_stride_b + (size_t)slot * a.pg.row_b + (size_t)sub * (F8 ? 8 : 16) : 0;

    float c[8], s[8];
    unpack8(a.cos[(size_t)pos * 16 + sub], c);
    unpack8(a.sin[(size_t)pos * 16 + sub], s);
    if (sub < 8) {                                              // the first half takes -x2, the second half x1
#pragma unroll
        for (int j = 0; j < 8; ++j) s[j] = -s[j];
    }
    char* qrow = a.q_out + (size_t)t * a.ldq_b + sub * 16;

    auto put = [&](char* cache, int h, const float (&y)[8], float inv) {
        char* dst = cache + at + (size_t)h * a.pg.head_stride_b;
        if (F8) {
            float z[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) z[j] = y[j] * inv;
            *(u32x2_t*)dst = pack_e4m3(z);
        } else {
            u32x4_t o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
            *(u32x4_t*)dst = o;
        }
    };
    auto one = [&](int h, const u32x4_t raw) {
        float f[8];
        unpack8(raw, f);
        if (h - grp >= a.n_q + a.n_kv) {                        // four v rows: wave-uniform
            if (h < n_heads && store) put(a.v, h - a.n_q - a.n_kv, f, a.v_inv);
            return;
        }
        // the four rows of a wave can be of different kinds, and the exchanges below need every lane: v rows run along
        const bool is_q = h < a.n_q, is_v = h >= a.n_q + a.n_kv;
        float n[8], other[8], y[8];
        if (a.qw) {
            float ss = 0.f, w[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) ss += f[j] * f[j];
            const float ms = row_sum(ss) * (1.0f / 128.0f) + a.eps;
            // the reciprocal root instruction is off by one last place, far below the stored type's; the stepwise form keeps the exact one
            const float inv = STEPWISE ? 1.0f / sqrtf(ms) : __builtin_amdgcn_rsqf(ms);
            unpack8((is_q ? a.qw : a.kw)[sub], w);
#pragma unroll
            for (int j = 0; j < 8; ++j) n[j] = STEPWISE ? round_bf16(w[j] * round_bf16(f[j] * inv)) : w[j] * (f[j] * inv);
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) n[j] = f[j];
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) other[j] = rotate16<8>(n[j]);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            if (STEPWISE) y[j] = round_bf16(round_bf16(n[j] * c[j]) + round_bf16(other[j] * s[j]));
            else y[j] = n[j] * c[j] + other[j] * s[j];
        }
        if (h >= n_heads) return;
        if (is_q) {
            u32x4_t o;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[i] = pack_bf16x2(y[2 * i], y[2 * i + 1]);
            *(u32x4_t*)(qrow + (size_t)h * 256) = o;
        } else if (store) {
            if (is_v) put(a.v, h - a.n_q - a.n_kv, f, a.v_inv);
            else put(a.k, h - a.n_q, y, a.k_inv);
        }
    };
    for (int h0 = part * 4 + grp; h0 - grp < n_heads; h0 += 4 * step) {
        if (h0 - grp != part * 4) load(h0);
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (h0 - grp + u * step < n_heads) one(h0 + u * step, raw[u]);        // wave-uniform
    }
}

}  // namespace

extern "C" int coda_paged_append(const void* qkv, long long ld_qkv, void* q_out, long long ld_q, const void* q_weight,
                                 const void* k_weight, const void* cos, const void* sin, int max_pos, const int* seq_start,
                                 const int* pos0, int B, int T, const int* page_table, long long ld_table, int max_pages, void* k_cache,
                                 void* v_cache, long long page_stride, int num_pages, int page_size, int cache_type, float k_scale,
                                 float v_scale, int n_q, int n_kv, float eps, int flags, void* stream) {
    const char* who = "coda_paged_append";
    if (B <= 0 || T <= 0 || n_q <= 0 || n_kv <= 0 || max_pos <= 0) return coda_refuse(who, CODA_ERR_SHAPE, "a size is not positive");
    if (B > 1 << 30) return coda_refuse(who, CODA_ERR_SHAPE, "B exceeds 2^30");     // the other two have a workgroup per sequence: fewer
    if ((long long)n_q + 2LL * n_kv > MAX_HEADS) return coda_refuse(who, CODA_ERR_SHAPE, "too many heads");
    if (ld_qkv < ((long long)n_q + 2LL * n_kv) * HEAD_DIM || ld_q < (long long)n_q * HEAD_DIM) return coda_refuse(who, CODA_ERR_SHAPE, "a row stride is shorter than a row");
    if (!qkv || !q_out || !cos || !sin || !seq_start || !pos0) return coda_refuse(who, CODA_ERR_ARG, "null pointer");
    if (!q_weight != !k_weight) return coda_refuse(who, CODA_ERR_ARG, "q_weight and k_weight come together or not at all");
    if (flags & ~CODA_APPEND_STEPWISE) return coda_refuse(who, CODA_ERR_ARG, "unknown flag");
    if (((uintptr_t)qkv | (uintptr_t)q_out | (uintptr_t)cos | (uintptr_t)sin | (uintptr_t)q_weight | (uintptr_t)k_weight) & 15 ||
        (ld_qkv * 2) % 16 || (ld_q * 2) % 16)
        return coda_refuse(who, CODA_ERR_ALIGN, "rows start on 16 bytes");
    AppendArgs a;
    const int rc = coda_check_pages(who, k_cache, v_cache, page_table, ld_table, max_pages, page_stride, num_pages, page_size, cache_type,
                                    k_scale, v_scale, n_kv, &a.pg);
    if (rc != CODA_OK) return rc;
    a.qkv = (const char*)qkv; a.ld_b = ld_qkv * 2;
    a.q_out = (char*)q_out; a.ldq_b = ld_q * 2;
    a.qw = (const u32x4_t*)q_weight; a.kw = (const u32x4_t*)k_weight;
    a.cos = (const u32x4_t*)cos; a.sin = (const u32x4_t*)sin; a.max_pos = max_pos;
    a.seq_start = seq_start; a.pos0 = pos0; a.B = B; a.T = T;
    a.k = (char*)k_cache; a.v = (char*)v_cache;
    const bool f8 = cache_type == CODA_CACHE_E4M3, stepwise = flags & CODA_APPEND_STEPWISE;
    a.k_inv = f8 ? 1.0f / k_scale : 1.0f;
    a.v_inv = f8 ? 1.0f / v_scale : 1.0f;
    a.n_q = n_q; a.n_kv = n_kv; a.eps = eps;
    const int n_heads = n_q + 2 * n_kv;
    // waves per token: as many as there are groups of four rows while that leaves the chip unfilled, else one wave per
    // sixteen rows (its four loads in flight).  us with 2 / 4 / 8 waves of a token of 32 rows: 32 tokens 4.8 / 4.2 / 3.8, 4096 tokens 16.5 /
    // 18.2 / 23.7, 15.6 k tokens 51.6 / 59.4 / 87.3
    const long long fill = 16LL * coda_device_cus();
    a.parts = (n_heads + 15) / 16;
    while (a.parts * 4 < n_heads && (long long)T * a.parts * 2 <= fill) a.parts *= 2;
    const long long wgs = ((long long)T * a.parts + 3) / 4;
    if (!grid_fits(wgs, 256)) return coda_refuse(who, CODA_ERR_SHAPE, "too many rows for one launch");
    const dim3 grid((unsigned)wgs), block(256);
    hipStream_t st = (hipStream_t)stream;
    if (f8 && stepwise) hipLaunchKernelGGL((paged_append_kernel<true, true>), grid, block, 0, st, a);
    else if (f8) hipLaunchKernelGGL((paged_append_kernel<true, false>), grid, block, 0, st, a);
    else if (stepwise) hipLaunchKernelGGL((paged_append_kernel<false, true>), grid, block, 0, st, a);
    else hipLaunchKernelGGL((paged_append_kernel<false, false>), grid, block, 0, st, a);
    CODA_CHECK_LAUNCH("paged_append");
    return CODA_OK;
}
