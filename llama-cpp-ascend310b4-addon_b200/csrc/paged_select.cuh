// paged_select.cuh -- block selection for sparse attention: an upper bound of
// q . k per block from the page's key bounds, and the n_sel best blocks.
//
// Scores are summed in 64 bits: f32 sums of 64 to 256 products are off by
// some 1e-6 of a score, and with thousands of blocks per head the scores
// around the last place of the selection lie that close together, so 32 bits
// would pick blocks by rounding.
#pragma once

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"
#include "paged_store.cuh"

namespace b200 {

struct PagedSelectArgs {
    const uint16_t *lo, *hi;
    const float* q;
    int64_t q_stride;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_lens;
    int32_t* sel;
    unsigned long long* keys;  // [n_seq][n_head_kv][max_blocks] ordered scores
    int n_seq, n_head, n_head_kv, max_blocks, page_size, n_pages, n_sel;
};

// Blocks of sequence s; a length outside the table is clamped.
__device__ __forceinline__ int paged_blocks(int len, int max_blocks, int page_size) {
    const unsigned b = len <= 0 ? 0u : ((unsigned)len + (unsigned)page_size - 1u) / (unsigned)page_size;
    return (int)min(b, (unsigned)max_blocks);
}

// Order-preserving 64-bit key of a double; NaN below everything.
__device__ __forceinline__ unsigned long long order_key(double x) {
    if (x != x) return 0ull;
    const long long b = __double_as_longlong(x + 0.0);  // -0 -> +0
    return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}

constexpr int kSelectThreads = 256;

// One warp per (sequence, block, KV head).
template <bool BF16, int D>
__global__ void __launch_bounds__(kSelectThreads) paged_score_kernel(PagedSelectArgs a) {
    constexpr int E = D / 32;
    const int64_t item = (int64_t)blockIdx.x * (kSelectThreads / 32) + threadIdx.x / 32;
    const int lane = threadIdx.x & 31;
    const int h = (int)(item % a.n_head_kv);
    const int64_t sb = item / a.n_head_kv;
    const int b = (int)(sb % a.max_blocks);
    const int64_t s = sb / a.max_blocks;
    if (s >= a.n_seq) return;
    const int nb = paged_blocks(a.seq_lens[s], a.max_blocks, a.page_size);
    if (b >= nb) return;
    const int page = a.table[s * a.table_stride + b];
    double best = -INFINITY;
    if ((unsigned)page >= (unsigned)a.n_pages) {
        if (lane == 0) record_status(B200_DEVSTATUS_BOUNDS);
        best = NAN;
    } else {
        float lo[E], hi[E];
        const uint32_t* pl = reinterpret_cast<const uint32_t*>(a.lo + ((int64_t)page * a.n_head_kv + h) * D) + lane * (E / 2);
        const uint32_t* ph = reinterpret_cast<const uint32_t*>(a.hi + ((int64_t)page * a.n_head_kv + h) * D) + lane * (E / 2);
#pragma unroll
        for (int e = 0; e < E / 2; ++e) {
            const float2 l = unpack16<BF16>(pl[e]), u = unpack16<BF16>(ph[e]);
            lo[2 * e] = l.x, lo[2 * e + 1] = l.y, hi[2 * e] = u.x, hi[2 * e + 1] = u.y;
        }
        const int G = a.n_head / a.n_head_kv;
        for (int j = 0; j < G; ++j) {
            const float* q = a.q + s * a.q_stride + (int64_t)(h * G + j) * D + lane * E;
            double x = 0.0;
#pragma unroll
            for (int e = 0; e < E; ++e) x += fmax((double)q[e] * lo[e], (double)q[e] * hi[e]);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
            best = (x != x || best != best) ? NAN : fmax(best, x);
        }
    }
    if (lane == 0) a.keys[(s * a.n_head_kv + h) * (int64_t)a.max_blocks + b] = order_key(best);
}

// One CTA per (sequence, KV head): the threshold key by a radix search from
// the top byte down, then one ordered pass that writes the chosen blocks.
__global__ void __launch_bounds__(kSelectThreads) paged_topk_kernel(PagedSelectArgs a) {
    __shared__ int hist[256];
    __shared__ int s_digit, s_left;
    __shared__ int wsum[2][kSelectThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int64_t sh = blockIdx.x;
    const int64_t s = sh / a.n_head_kv;
    const int len = a.seq_lens[s];
    const int nb = paged_blocks(len, a.max_blocks, a.page_size);
    if (tid == 0 && sh % a.n_head_kv == 0 && (len < 0 || len > (int64_t)a.max_blocks * a.page_size))
        record_status(B200_DEVSTATUS_BOUNDS);
    int32_t* out = a.sel + sh * a.n_sel;
    const unsigned long long* keys = a.keys + sh * (int64_t)a.max_blocks;
    if (nb <= a.n_sel) {
        for (int i = tid; i < a.n_sel; i += kSelectThreads) out[i] = i < nb ? i : -1;
        return;
    }
    // n_sel - 1 of the nb - 1 older blocks
    const int m = nb - 1;
    int left = a.n_sel - 1;
    unsigned long long prefix = 0, mask = 0;
    if (left > 0) {
        for (int shift = 56; shift >= 0; shift -= 8) {
            for (int i = tid; i < 256; i += kSelectThreads) hist[i] = 0;
            __syncthreads();
            for (int i = tid; i < m; i += kSelectThreads)
                if ((keys[i] & mask) == prefix) atomicAdd(&hist[(keys[i] >> shift) & 255], 1);
            __syncthreads();
            if (tid == 0) {
                int c = 255, need = left;
                while (c > 0 && hist[c] < need) need -= hist[c--];
                s_digit = c, s_left = need;
            }
            __syncthreads();
            prefix |= (unsigned long long)s_digit << shift;
            mask |= 255ull << shift;
            left = s_left;
            __syncthreads();
        }
    }
    // blocks above the threshold, and the first `left` at it
    int done = 0, ties = 0;
    for (int base = 0; base < m; base += kSelectThreads) {
        const int i = base + tid;
        const unsigned long long key = i < m ? keys[i] : 0ull;
        const bool above = i < m && a.n_sel > 1 && key > prefix;
        const bool at = i < m && a.n_sel > 1 && key == prefix;
        const unsigned tm = __ballot_sync(0xffffffffu, at);
        if (lane == 0) wsum[0][warp] = __popc(tm);
        __syncthreads();
        int tie = ties + __popc(tm & ((1u << lane) - 1u)), tie_all = 0;
        for (int w = 0; w < kSelectThreads / 32; ++w) {
            if (w < warp) tie += wsum[0][w];
            tie_all += wsum[0][w];
        }
        const bool take = above || (at && tie < left);
        const unsigned km = __ballot_sync(0xffffffffu, take);
        if (lane == 0) wsum[1][warp] = __popc(km);
        __syncthreads();
        int at_out = done + __popc(km & ((1u << lane) - 1u)), all = 0;
        for (int w = 0; w < kSelectThreads / 32; ++w) {
            if (w < warp) at_out += wsum[1][w];
            all += wsum[1][w];
        }
        if (take) out[at_out] = i;
        done += all;
        ties += tie_all;
        __syncthreads();
    }
    if (tid == 0) out[a.n_sel - 1] = m;
}

}  // namespace b200
