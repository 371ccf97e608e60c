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

// CTA (t, head): active where token t opens a run of tokens of one page; it
// stores the run's rows of that head.
template <bool BF16, int D>
__global__ void __launch_bounds__(kStoreThreads) paged_store_kernel(PagedStoreArgs a) {
    constexpr int LPR = D / 8;                  // lanes per row, 8 values each
    constexpr int RPP = kStoreThreads / LPR;    // rows per pass
    __shared__ float s_lo[RPP][D], s_hi[RPP][D];
    __shared__ int s_first;
    const int64_t n_slots = a.kv.n_pages * a.kv.page_size;
    const int ps = a.kv.page_size, head = blockIdx.y, tid = threadIdx.x;
    const int g = tid / LPR, d = (tid % LPR) * 8;
    auto page_of = [&](int64_t t) -> int {
        if (t < 0 || t >= a.n_tokens) return -1;
        const int64_t s = a.slots[t];
        return s >= 0 && s < n_slots ? (int)((unsigned)s / (unsigned)ps) : -1;
    };
    const int64_t t0 = blockIdx.x;
    const int page = page_of(t0);
    if (page < 0) {
        if (tid == 0 && a.slots[t0] >= n_slots) record_status(B200_DEVSTATUS_BOUNDS);
        return;
    }
    if (page_of(t0 - 1) == page) return;
    if (tid == 0) s_first = 0;
    float lo[8], hi[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) lo[e] = INFINITY, hi[e] = -INFINITY;
    bool first = false;
    for (int j = g; j < ps; j += RPP) {
        const int64_t t = t0 + j;
        if (page_of(t) != page) break;
        const int row = (int)(a.slots[t] - (int64_t)page * ps);
        first |= row == 0;
        const float4* src = reinterpret_cast<const float4*>(a.k + t * a.k_ld + head * D + d);
        const float4 x = src[0], y = src[1];
        const float4* vs = reinterpret_cast<const float4*>(a.v + t * a.v_ld + head * D + d);
        const float4 vx = vs[0], vy = vs[1];
        const uint4 w = make_uint4(pack16<BF16>(x.x, x.y), pack16<BF16>(x.z, x.w), pack16<BF16>(y.x, y.y),
                                   pack16<BF16>(y.z, y.w));
        const uint4 u = make_uint4(pack16<BF16>(vx.x, vx.y), pack16<BF16>(vx.z, vx.w), pack16<BF16>(vy.x, vy.y),
                                   pack16<BF16>(vy.z, vy.w));
        uint8_t* kd = static_cast<uint8_t*>(a.kv.k) + page * a.kv.k_page + row * a.kv.k_row + head * a.kv.k_head;
        uint8_t* vd = static_cast<uint8_t*>(a.kv.v) + page * a.kv.v_page + row * a.kv.v_row + head * a.kv.v_head;
        *reinterpret_cast<uint4*>(kd + 2 * d) = w;
        *reinterpret_cast<uint4*>(vd + 2 * d) = u;
        const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float2 f = unpack16<BF16>(ws[e]);
            lo[2 * e] = fminf(lo[2 * e], f.x), hi[2 * e] = fmaxf(hi[2 * e], f.x);
            lo[2 * e + 1] = fminf(lo[2 * e + 1], f.y), hi[2 * e + 1] = fmaxf(hi[2 * e + 1], f.y);
        }
    }
    if (a.kv.k_lo == nullptr) return;
#pragma unroll
    for (int e = 0; e < 8; ++e) s_lo[g][d + e] = lo[e], s_hi[g][d + e] = hi[e];
    __syncthreads();
    if (first) s_first = 1;
    __syncthreads();
    for (int c = 2 * tid; c < D; c += 2 * kStoreThreads) {
        float2 l = make_float2(INFINITY, INFINITY), h = make_float2(-INFINITY, -INFINITY);
        uint32_t* pl = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.kv.k_lo) +
                                                   ((int64_t)page * a.kv.n_head_kv + head) * D + c);
        uint32_t* ph = reinterpret_cast<uint32_t*>(static_cast<uint16_t*>(a.kv.k_hi) +
                                                   ((int64_t)page * a.kv.n_head_kv + head) * D + c);
        if (!s_first) l = unpack16<BF16>(*pl), h = unpack16<BF16>(*ph);
        for (int r = 0; r < RPP; ++r) {
            l.x = fminf(l.x, s_lo[r][c]), l.y = fminf(l.y, s_lo[r][c + 1]);
            h.x = fmaxf(h.x, s_hi[r][c]), h.y = fmaxf(h.y, s_hi[r][c + 1]);
        }
        *pl = pack16<BF16>(l.x, l.y);
        *ph = pack16<BF16>(h.x, h.y);
    }
}

}  // namespace b200
