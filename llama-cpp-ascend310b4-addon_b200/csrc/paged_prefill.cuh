// paged_prefill.cuh -- attention of a chunk of new tokens per sequence over the
// paged cache.
#pragma once

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"
#include "paged_store.cuh"

namespace b200 {

struct PagedPrefillArgs {
    b200_paged_kv kv;
    const uint16_t* q;
    int64_t q_stride;
    const int32_t* table;
    int64_t table_stride;
    const int32_t *seq_lens, *cu;
    const uint16_t* mask;
    int64_t mask_stride;
    uint16_t* out;
    int n_tokens, n_head, group, n_seq, max_blocks, window;
    float scale;
};

// The tokens of sequence s: rows first .. first + n - 1 of q, the last of them
// at position len - 1.
struct PfSeq {
    int first, n, len;
};
__device__ __forceinline__ PfSeq pf_seq(const PagedPrefillArgs& a, int s, bool record) {
    const int64_t cap = min((int64_t)a.max_blocks * a.kv.page_size, (int64_t)INT32_MAX);
    const int c0 = a.cu[s], c1 = a.cu[s + 1], l = a.seq_lens[s];
    PfSeq q;
    q.first = max(0, min(c0, a.n_tokens));
    q.n = max(0, min(c1, a.n_tokens) - q.first);
    q.len = max(0, (int)min((int64_t)l, cap));
    if (record && (q.first != c0 || c1 < c0 || c1 > a.n_tokens || q.len != l)) record_status(B200_DEVSTATUS_BOUNDS);
    return q;
}

// One row of one head by a warp, in f32 products of whole values: what the formula
// says whatever infinities and NaN meet.  Lane l owns channels l * D / 32 on.
template <bool BF16, int D>
__device__ void pf_row(const PagedPrefillArgs& a, int s, const PfSeq& sq, int i, int head) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, h = head / a.group, ps = a.kv.page_size;
    const int64_t t = sq.first + i;
    const uint16_t* qp = a.q + t * a.q_stride + head * D + lane * E;
    float q[E], o[E];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const float2 f = unpack16<BF16>(*reinterpret_cast<const uint32_t*>(qp + e));
        q[e] = f.x, q[e + 1] = f.y, o[e] = o[e + 1] = 0.f;
    }
    const int at = sq.len - sq.n + i;  // may be negative: sees nothing
    const int p0 = a.window > 0 ? max(0, at - a.window + 1) : 0;
    double m = -INFINITY;
    float sum = 0.f;
    for (int p = p0; p <= at; ++p) {
        float bias = 0.f;
        if (a.mask) {
            bias = h2f(a.mask[s * a.mask_stride + p]);
            if (bias == -INFINITY) continue;
        }
        const int page = a.table[s * a.table_stride + p / ps], r = p % ps;
        if ((unsigned)page >= (unsigned)a.kv.n_pages) {
            if (lane == 0) record_status(B200_DEVSTATUS_BOUNDS);
            continue;
        }
        const uint8_t* kp = static_cast<const uint8_t*>(a.kv.k) + page * a.kv.k_page + r * a.kv.k_row + h * a.kv.k_head;
        const uint8_t* vp = static_cast<const uint8_t*>(a.kv.v) + page * a.kv.v_page + r * a.kv.v_row + h * a.kv.v_head;
        float x = 0.f, v[E];
#pragma unroll
        for (int e = 0; e < E; e += 2) {
            const float2 k = unpack16<BF16>(*reinterpret_cast<const uint32_t*>(kp + 2 * (lane * E + e)));
            const float2 w = unpack16<BF16>(*reinterpret_cast<const uint32_t*>(vp + 2 * (lane * E + e)));
            x = fmaf(q[e + 1], k.y, fmaf(q[e], k.x, x));
            v[e] = w.x, v[e + 1] = w.y;
        }
        x = warp_sum(x);
        const double y = (double)(x * a.scale) + (double)bias;  // a mask of the lowest value keeps the score's bits
        if (y > m) {
            const float f = exp2f((float)((m - y) * 1.4426950408889634));
            if (m != -INFINITY) {
                sum *= f;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] *= f;
            }
            m = y;
        }
        const float w = y == -INFINITY ? 0.f : exp2f((float)((y - m) * 1.4426950408889634));
        sum += w;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = fmaf(w, v[e], o[e]);
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* op = a.out + (t * a.n_head + head) * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2)
        *reinterpret_cast<uint32_t*>(op + e) =
            sum == 0.f ? 0u : pack16<BF16>(o[e] * inv, o[e + 1] * inv);
}

// A warp per (row, head).
template <bool BF16, int D>
__global__ void __launch_bounds__(256) paged_prefill_rows_kernel(const __grid_constant__ PagedPrefillArgs a) {
    const int64_t task = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    const int64_t t = task / a.n_head;
    const int head = (int)(task - t * a.n_head);
    if (t >= a.n_tokens) return;
    int lo = 0, hi = a.n_seq;  // the sequence of row t: cu[lo] <= t < cu[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t) lo = mid;
        else hi = mid;
    }
    const PfSeq sq = pf_seq(a, lo, head == 0 && (threadIdx.x & 31) == 0);
    if (t < sq.first || t >= sq.first + sq.n) return;
    pf_row<BF16, D>(a, lo, sq, (int)(t - sq.first), head);
}

}  // namespace b200
