// paged_plan.cuh -- page allocation and slot maps from request lengths.
//
// Everything follows from three prefix sums over the sequences (token rows,
// pages needed, pages given back): a token's sequence, a new page's block and
// a popped stack entry are then found by binary search in shared memory, so
// the writes are spread over threads by output element, however uneven the
// sequences are.  The call is bound by latency (a few hundred KB at most): one
// cluster of up to 8 CTAs, each with the sums of all sequences, so nothing but
// one barrier separates reading the lengths from replacing them in place.
// Measured: 64 sequences with one token each 3.65 us, 1024 mixed ones with 25000
// tokens 15.7 us (60 us on one CTA).  The launch is sized by the token rows, so a
// small batch in which a long sequence ends gives its pages back with few
// threads: 8192 pages beside 7 tokens 49 us.
#pragma once

#include <cooperative_groups.h>

#include "args.h"
#include "common.cuh"

namespace b200 {

struct PagedPlanArgs {
    const int32_t* new_lens;
    const int32_t* seq_lens;
    int32_t* table;
    int64_t table_stride;
    int32_t* free_pages;
    const int32_t* n_free;
    int64_t* slots;
    int32_t* positions;
    int32_t* cu;
    int32_t* seq_lens_out;
    int32_t* n_free_out;
    int n_seq, max_blocks, page_size, n_pages, max_tokens;
};

constexpr int kPlanThreads = 1024;
constexpr int kPlanCtas = 8;

B200_HD inline size_t plan_smem_bytes(int n_seq) { return (size_t)(4 * n_seq + 3) * sizeof(int); }

// Inclusive sums of a and b over the CTA's threads; `part` has 2 * 32 entries.
__device__ __forceinline__ void block_scan2(long long& a, long long& b, long long* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, o), y = __shfl_up_sync(0xffffffffu, b, o);
        if (lane >= o) a += x, b += y;
    }
    __syncthreads();  // the previous scan's readers are done with part
    if (lane == 31) part[warp] = a, part[32 + warp] = b;
    __syncthreads();
    long long x = lane < warp ? part[lane] : 0, y = lane < warp ? part[32 + lane] : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        x += __shfl_xor_sync(0xffffffffu, x, o);
        y += __shfl_xor_sync(0xffffffffu, y, o);
    }
    a += x;
    b += y;
}

// Largest i with v[i] <= x, for v[0] = 0 <= x < v[n], v ascending.
__device__ __forceinline__ int find_segment(const int* v, int n, int x) {
    int lo = 0, hi = n;  // v[lo] <= x < v[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (v[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) paged_plan_kernel(PagedPlanArgs a) {
    extern __shared__ int plan_smem[];
    __shared__ long long part[64];
    __shared__ int s_got;
    const int n = a.n_seq, ps = a.page_size, tid = threadIdx.x;
    int* s_cu = plan_smem;          // [n + 1] first token row (at most max_tokens)
    int* s_need = s_cu + n + 1;     // [n + 1] pages needed by the sequences before
    int* s_back = s_need + n + 1;   // [n + 1] pages given back by the sequences before
    int* s_old = s_back + n + 1;    // [n] cached tokens, ~tokens where the request does not fit
    const int cap = (int)min((long long)a.max_blocks * ps, (long long)INT32_MAX);
    int n0 = a.n_free[0];
    if (n0 < 0 || n0 > a.n_pages) {
        if (tid == 0 && blockIdx.x == 0) record_status(B200_DEVSTATUS_BOUNDS);
        n0 = n0 < 0 ? 0 : a.n_pages;
    }
    if (tid == 0) s_got = 0, s_cu[0] = 0, s_need[0] = 0, s_back[0] = 0;

    long long rows = 0, need_sum = 0, back_sum = 0;  // totals of the tiles before
    for (int base = 0; base < n; base += blockDim.x) {
        const int i = base + tid;
        int old = 0, add = 0;
        bool ends = false;
        if (i < n) {
            const int nl = a.new_lens[i];
            old = a.seq_lens[i];
            if (old < 0 || old > cap) {
                record_status(B200_DEVSTATUS_BOUNDS);
                old = old < 0 ? 0 : cap;
            }
            ends = nl < 0;
            add = max(nl, 0);
        }
        const long long old_b = ((long long)old + ps - 1) / ps;
        long long cu = add, back = ends ? old_b : 0;
        block_scan2(cu, back, part);
        cu += rows;
        back += back_sum;
        const long long end_b = ((long long)old + add + ps - 1) / ps;
        const bool fits = i < n && !ends && cu <= a.max_tokens && end_b <= a.max_blocks;
        long long need = fits ? end_b - old_b : 0, unused = 0;
        block_scan2(need, unused, part);
        need += need_sum;
        if (i < n) {
            s_cu[i + 1] = (int)min(cu, (long long)a.max_tokens);
            s_need[i + 1] = (int)min(need, (long long)INT32_MAX);
            s_back[i + 1] = (int)min(back, (long long)INT32_MAX);
            s_old[i] = fits ? old : ~old;
        }
        // the tile's last thread holds the new totals
        __syncthreads();
        if (tid == (int)blockDim.x - 1) part[0] = cu, part[1] = back, part[2] = need;
        __syncthreads();
        rows = part[0];
        back_sum = part[1];
        need_sum = part[2];
    }
    __syncthreads();
    long long top = n0 + back_sum;
    if (top > a.n_pages) {  // more pages given back than exist: the surplus is dropped
        if (tid == 0 && blockIdx.x == 0) record_status(B200_DEVSTATUS_BOUNDS);
        top = a.n_pages;
    }
    const int pool = (int)top, n_back = pool - n0;
    // pages handed out: the largest prefix of needs that the pool covers
    for (int i = tid; i < n; i += blockDim.x)
        if (s_need[i + 1] <= pool && (i + 1 == n || s_need[i + 2] > pool)) s_got = s_need[i + 1];
    __syncthreads();
    const int got = s_got;

    auto given_back = [&](int r) {  // r-th page of the ending sequences
        const int i = find_segment(s_back, n, r);
        return a.table[i * a.table_stride + (r - s_back[i])];
    };
    auto popped = [&](int r) {
        const int p = pool - 1 - r;
        return p >= n0 ? given_back(p - n0) : a.free_pages[p];
    };
    auto blocks_of = [&](int tokens) { return (int)(((unsigned)tokens + (unsigned)ps - 1u) / (unsigned)ps); };

    // unsigned: a step past the last of 2^31 - 2 rows or pages must not wrap around
    const unsigned at = blockIdx.x * blockDim.x + tid, step = gridDim.x * blockDim.x;
    for (unsigned u = at; u < (unsigned)a.max_tokens; u += step) {
        const int t = (int)u;
        int64_t slot = -1;
        int pos = -1;
        if (t < s_cu[n]) {
            const int i = find_segment(s_cu, n, t);
            const int old = s_old[i];
            if (old >= 0 && (s_need[i + 1] == s_need[i] || s_need[i + 1] <= pool)) {
                pos = old + (t - s_cu[i]);
                const int b = pos / ps, old_b = blocks_of(old);
                const int page =
                    b < old_b ? a.table[i * a.table_stride + b] : popped(s_need[i] + (b - old_b));
                if ((unsigned)page < (unsigned)a.n_pages) {
                    slot = (int64_t)page * ps + (pos - b * ps);
                } else {
                    record_status(B200_DEVSTATUS_BOUNDS);
                    pos = -1;
                }
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
    for (unsigned u = at; u < (unsigned)got; u += step) {
        const int r = (int)u;
        const int i = find_segment(s_need, n, r);
        a.table[i * a.table_stride + blocks_of(s_old[i]) + (r - s_need[i])] = popped(r);
    }
    for (unsigned u = at; u < (unsigned)n_back; u += step) {
        const int r = (int)u;
        const int page = given_back(r);
        if ((unsigned)page >= (unsigned)a.n_pages) record_status(B200_DEVSTATUS_BOUNDS);
        a.free_pages[n0 + r] = page;
    }
    // every CTA has read the lengths and the page count
    if (gridDim.x > 1) cooperative_groups::this_cluster().sync();
    else __syncthreads();
    for (int i = (int)at; i < n; i += (int)step) {
        const int old = s_old[i];
        int len = old >= 0 ? old : ~old;
        if (a.new_lens[i] < 0) len = 0;
        else if (old >= 0 && (s_need[i + 1] == s_need[i] || s_need[i + 1] <= pool)) len += a.new_lens[i];
        a.seq_lens_out[i] = len;
        a.cu[i] = s_cu[i];
    }
    if (at == 0) {
        a.cu[n] = s_cu[n];
        a.n_free_out[0] = pool - got;
    }
}

}  // namespace b200
