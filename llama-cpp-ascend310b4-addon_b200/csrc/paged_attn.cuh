// paged_attn.cuh -- attention of one new token per sequence over a paged
// key-value cache.
#pragma once

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"
#include "paged_select.cuh"

namespace b200 {

constexpr int kPaHeads = 8;  // query heads of one KV head handled together
constexpr int kPaThreads = 128;

struct PagedAttnArgs {
    b200_paged_kv kv;
    const float* q;
    int64_t q_stride;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_lens;
    const uint16_t* mask;
    int64_t mask_stride;
    const int32_t* sel;
    float* out;
    float scale;
    int n_seq, n_head, n_sel, max_blocks;
};

// CTA (KV head and chunk of 8 query heads, sequence); each warp takes every
// fourth position and keeps the running maximum as a pair (score, mask), so
// that a row of equal large negative mask values keeps its scores' bits.
template <bool BF16, int D>
__global__ void __launch_bounds__(kPaThreads) paged_attn_kernel(PagedAttnArgs a) {
    constexpr int E = D / 32, W = kPaThreads / 32;
    __shared__ float s_o[W][kPaHeads][D];
    __shared__ float s_m[W][kPaHeads], s_k[W][kPaHeads], s_l[W][kPaHeads];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int G = a.n_head / a.kv.n_head_kv, chunks = (G + kPaHeads - 1) / kPaHeads;
    const int h = blockIdx.x / chunks, j0 = (blockIdx.x % chunks) * kPaHeads, gn = min(kPaHeads, G - j0);
    const int64_t s = blockIdx.y;
    const int ps = a.kv.page_size;
    int len = a.seq_lens[s];
    const int cap = (int)min((int64_t)a.max_blocks * ps, (int64_t)INT32_MAX);
    if (len < 0 || len > cap) {
        if (tid == 0) record_status(B200_DEVSTATUS_BOUNDS);
        len = len < 0 ? 0 : cap;
    }
    float q[kPaHeads][E], o[kPaHeads][E], m[kPaHeads], l[kPaHeads];
    float mk = -INFINITY;
    for (int j = 0; j < kPaHeads; ++j) {
        m[j] = -INFINITY, l[j] = 0.f;
        for (int e = 0; e < E; ++e) {
            q[j][e] = j < gn ? a.q[s * a.q_stride + (int64_t)(h * G + j0 + j) * D + lane * E + e] : 0.f;
            o[j][e] = 0.f;
        }
    }
    const int32_t* sel = a.sel ? a.sel + (s * a.kv.n_head_kv + h) * (int64_t)a.n_sel : nullptr;
    const int64_t n_tok = sel ? (int64_t)a.n_sel * ps : len;
    for (int64_t i = warp; i < n_tok; i += W) {
        int b = (int)(i / ps);
        const int row = (int)(i % ps);
        if (sel) b = sel[b];
        if (b < 0 || (int64_t)b * ps + row >= len) continue;
        const int64_t pos = (int64_t)b * ps + row;
        float bias = 0.f;
        if (a.mask) bias = h2f(a.mask[s * a.mask_stride + pos]);
        if (bias == -INFINITY) continue;
        const int page = a.table[s * a.table_stride + b];
        if ((unsigned)page >= (unsigned)a.kv.n_pages) {
            if (lane == 0) record_status(B200_DEVSTATUS_BOUNDS);
            continue;
        }
        const uint32_t* kp = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.kv.k) + page * a.kv.k_page +
                                                               row * a.kv.k_row + h * a.kv.k_head) + lane * (E / 2);
        const uint32_t* vp = reinterpret_cast<const uint32_t*>(static_cast<const uint8_t*>(a.kv.v) + page * a.kv.v_page +
                                                               row * a.kv.v_row + h * a.kv.v_head) + lane * (E / 2);
        float k[E], v[E];
        for (int e = 0; e < E / 2; ++e) {
            const float2 x = unpack16<BF16>(kp[e]), y = unpack16<BF16>(vp[e]);
            k[2 * e] = x.x, k[2 * e + 1] = x.y, v[2 * e] = y.x, v[2 * e + 1] = y.y;
        }
        const float nk = fmaxf(mk, bias);
        for (int j = 0; j < gn; ++j) {
            float x = 0.f;
            for (int e = 0; e < E; ++e) x += q[j][e] * k[e];
            x = warp_sum(x) * a.scale + (bias - nk);
            const float mo = m[j] == -INFINITY ? -INFINITY : m[j] + (mk - nk);
            const float mn = fmaxf(mo, x), c = expf(mo - mn), p = expf(x - mn);
            l[j] = l[j] * c + p;
            for (int e = 0; e < E; ++e) o[j][e] = o[j][e] * c + p * v[e];
            m[j] = mn;
        }
        mk = nk;
    }
    for (int j = 0; j < gn; ++j) {
        for (int e = 0; e < E; ++e) s_o[warp][j][lane * E + e] = o[j][e];
        if (lane == 0) s_m[warp][j] = m[j], s_k[warp][j] = mk, s_l[warp][j] = l[j];
    }
    __syncthreads();
    for (int j = 0; j < gn; ++j) {
        float nk = -INFINITY, mx = -INFINITY, sum = 0.f, w[W];
        for (int x = 0; x < W; ++x) nk = fmaxf(nk, s_k[x][j]);
        for (int x = 0; x < W; ++x) w[x] = s_m[x][j] == -INFINITY ? -INFINITY : s_m[x][j] + (s_k[x][j] - nk);
        for (int x = 0; x < W; ++x) mx = fmaxf(mx, w[x]);
        for (int x = 0; x < W; ++x) {
            w[x] = w[x] == -INFINITY ? 0.f : expf(w[x] - mx);
            sum += w[x] * s_l[x][j];
        }
        for (int d = tid; d < D; d += kPaThreads) {
            float y = 0.f;
            for (int x = 0; x < W; ++x) y += w[x] * s_o[x][j][d];
            a.out[(s * a.n_head + h * G + j0 + j) * (int64_t)D + d] = sum > 0.f ? y / sum : 0.f;
        }
    }
}

}  // namespace b200
