// paged_store.cuh -- K and V rows of new tokens into their pages, with the
// pages' key bounds.
#pragma once

#include <cuda_bf16.h>

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"

namespace b200 {

// Two f32 values as 16-bit values of the cache type, rounded to nearest even.
template <bool BF16>
__device__ __forceinline__ uint32_t pack16(float x, float y) {
    if (BF16) {
        const __nv_bfloat162 h = __floats2bfloat162_rn(x, y);
        return *reinterpret_cast<const uint32_t*>(&h);
    }
    const __half2 h = __floats2half2_rn(x, y);
    return *reinterpret_cast<const uint32_t*>(&h);
}

template <bool BF16>
__device__ __forceinline__ float2 unpack16(uint32_t w) {
    if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
    return __half22float2(*reinterpret_cast<const __half2*>(&w));
}

struct PagedStoreArgs {
    b200_paged_kv kv;
    const float *k, *v;
    int64_t k_ld, v_ld;
    const int64_t* slots;
    int64_t n_tokens;
};

constexpr int kStoreThreads = 128;
constexpr int kStoreTile = 64;  // tokens whose runs one CTA looks for, at most
constexpr int kStoreRows = 2;   // rows a thread has in flight

// CTA (tile of `tile` tokens, head): the runs of tokens of one page that begin
// in its tile, wherever they end.  D / 8 lanes take a row of the head, 16 bytes
// of the page each, and the CTA's groups of lanes every kStoreThreads / (D / 8)-th
// row; a page's bounds are theirs alone, so they meet in shared memory once per
// run, without atomics.  12 bytes per element; bound by the latency of slots,
// then rows: with two rows a thread and 80 registers 8192 tokens x 8 x 128 take
// 24.3 us (4.2 TB/s), 64 decode tokens 3.85 us; four rows a thread (126
// registers, half the CTAs) took 31 and 6.0 us.  Meant for pages of 16 to 64
// rows: with pages of 1 the same tokens take 220 us (most lanes idle), with
// pages of 2048 207 us (one CTA per page and head).
template <bool BF16, int D>
__global__ void __launch_bounds__(kStoreThreads, 6) paged_store_kernel(PagedStoreArgs a, int tile) {
    constexpr int LPR = D / 8;                // lanes per row, 8 values each
    constexpr int RPP = kStoreThreads / LPR;  // rows per pass
    constexpr int W = kStoreThreads / 32;
    __shared__ float s_lo[W][D], s_hi[W][D];
    const int64_t n_slots = a.kv.n_pages * a.kv.page_size;
    const int ps = a.kv.page_size, head = blockIdx.y, tid = threadIdx.x, lane = tid & 31;
    const int g = tid / LPR, d = (tid % LPR) * 8;
    auto slot_of = [&](int64_t t) -> int64_t { return t >= 0 && t < a.n_tokens ? a.slots[t] : -1; };
    auto page_of = [&](int64_t s) -> int { return s >= 0 && s < n_slots ? (int)((unsigned)s / (unsigned)ps) : -1; };
    const int64_t first = (int64_t)blockIdx.x * tile;
    unsigned long long starts = 0;
    for (int base = 0; base < tile; base += 32) {
        const int x = base + lane;
        const int64_t s = x < tile ? slot_of(first + x) : -1;
        if (s >= n_slots) record_status(B200_DEVSTATUS_BOUNDS);
        const int page = page_of(s), before = page_of(slot_of(first + x - 1));
        starts |= (unsigned long long)__ballot_sync(0xffffffffu, page >= 0 && page != before) << base;
    }
    for (; starts != 0; starts &= starts - 1) {
        const int64_t t0 = first + __ffsll(starts) - 1;
        const int page = page_of(slot_of(t0));
        float lo[8], hi[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) lo[e] = INFINITY, hi[e] = -INFINITY;
        bool opens = false;  // row 0 of the page is among the rows
        const float* ks = a.k + head * D + d;
        const float* vs = a.v + head * D + d;
        // the page's bounds so far, on their way while the rows are read
        static_assert(D <= 2 * kStoreThreads, "a thread keeps two channels");
        const int64_t bounds_at = (((int64_t)page * a.kv.n_head_kv + head) * D + 2 * tid) / 2;
        uint32_t* pl = static_cast<uint32_t*>(a.kv.k_lo) + bounds_at;
        uint32_t* ph = static_cast<uint32_t*>(a.kv.k_hi) + bounds_at;
        const bool keeps = a.kv.k_lo != nullptr && 2 * tid < D;
        uint32_t old_lo = 0, old_hi = 0;
        if (keeps) old_lo = *pl, old_hi = *ph;
        uint8_t* kd = static_cast<uint8_t*>(a.kv.k) + page * a.kv.k_page + head * a.kv.k_head + 2 * d;
        uint8_t* vd = static_cast<uint8_t*>(a.kv.v) + page * a.kv.v_page + head * a.kv.v_head + 2 * d;
        for (int j = g; j < ps; j += RPP * kStoreRows) {
            int row[kStoreRows];  // -1: not of this run
            float4 x[kStoreRows][2], y[kStoreRows][2];
#pragma unroll
            for (int r = 0; r < kStoreRows; ++r) {
                const int64_t s = j + r * RPP < ps ? slot_of(t0 + j + r * RPP) : -1;
                row[r] = page_of(s) == page ? (int)(s - (int64_t)page * ps) : -1;
            }
#pragma unroll
            for (int r = 0; r < kStoreRows; ++r)
                if (row[r] >= 0) {
                    const int64_t t = t0 + j + r * RPP;
                    const float4* kp = reinterpret_cast<const float4*>(ks + t * a.k_ld);
                    const float4* vp = reinterpret_cast<const float4*>(vs + t * a.v_ld);
                    x[r][0] = __ldcs(kp), x[r][1] = __ldcs(kp + 1), y[r][0] = __ldcs(vp), y[r][1] = __ldcs(vp + 1);
                }
#pragma unroll
            for (int r = 0; r < kStoreRows; ++r) {
                if (row[r] < 0) continue;
                opens |= row[r] == 0;
                const uint4 w = make_uint4(pack16<BF16>(x[r][0].x, x[r][0].y), pack16<BF16>(x[r][0].z, x[r][0].w),
                                           pack16<BF16>(x[r][1].x, x[r][1].y), pack16<BF16>(x[r][1].z, x[r][1].w));
                const uint4 u = make_uint4(pack16<BF16>(y[r][0].x, y[r][0].y), pack16<BF16>(y[r][0].z, y[r][0].w),
                                           pack16<BF16>(y[r][1].x, y[r][1].y), pack16<BF16>(y[r][1].z, y[r][1].w));
                *reinterpret_cast<uint4*>(kd + row[r] * a.kv.k_row) = w;
                *reinterpret_cast<uint4*>(vd + row[r] * a.kv.v_row) = u;
                const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float2 f = unpack16<BF16>(ws[e]);
                    lo[2 * e] = fminf(lo[2 * e], f.x), hi[2 * e] = fmaxf(hi[2 * e], f.x);
                    lo[2 * e + 1] = fminf(lo[2 * e + 1], f.y), hi[2 * e + 1] = fmaxf(hi[2 * e + 1], f.y);
                }
            }
            if (row[kStoreRows - 1] < 0) break;  // the run is consecutive: it ends before this row
        }
        if (a.kv.k_lo == nullptr) continue;
#pragma unroll
        for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                lo[e] = fminf(lo[e], __shfl_xor_sync(0xffffffffu, lo[e], o));
                hi[e] = fmaxf(hi[e], __shfl_xor_sync(0xffffffffu, hi[e], o));
            }
        if (lane < LPR)
#pragma unroll
            for (int e = 0; e < 8; ++e) s_lo[tid >> 5][d + e] = lo[e], s_hi[tid >> 5][d + e] = hi[e];
        const bool fresh = __syncthreads_or(opens);
        if (keeps) {
            const int c = 2 * tid;
            float2 l = make_float2(INFINITY, INFINITY), h = make_float2(-INFINITY, -INFINITY);
            if (!fresh) l = unpack16<BF16>(old_lo), h = unpack16<BF16>(old_hi);
#pragma unroll
            for (int r = 0; r < W; ++r) {
                l.x = fminf(l.x, s_lo[r][c]), l.y = fminf(l.y, s_lo[r][c + 1]);
                h.x = fmaxf(h.x, s_hi[r][c]), h.y = fmaxf(h.y, s_hi[r][c + 1]);
            }
            *pl = pack16<BF16>(l.x, l.y);
            *ph = pack16<BF16>(h.x, h.y);
        }
        __syncthreads();  // the next run's rows may replace s_lo, s_hi
    }
}

}  // namespace b200
