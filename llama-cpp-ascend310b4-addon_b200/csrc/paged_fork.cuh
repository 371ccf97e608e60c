// paged_fork.cuh -- rows of a block table become prefixes of other rows, pages
// shared between them, and copies of pages.
//
// Which pages go back and which rows need a page of their own follows from who
// holds each page before and after the call, so every entry leaves marks on its
// page in one pass and everything else is read from the marks.
//   mark   (a warp per row and 256 entries): old entries set was[p], new
//          ones full[p], or tails[p]
//          (the largest n_seq - s, so the lowest row) where the row's last block
//          is not full.  Only tails needs an atomic, and a maximum does not
//          depend on order.
//   count  (a CTA per 16384 pages): pages held before and by nobody after; one
//          more CTA numbers the rows that need a page.
//   write  table rows, lists and the stack.  The r-th row in need gets the r-th
//          page from the top of the stack; where that is a page which this call
//          frees, the thread that pushes it writes the row's entry, so nothing is
//          read that the launch has written.
// Latency bounds it: three launches of a few dependent reads each, after a memset of
// the marks.  The marks are scattered, so the phases are launches of the whole GPU
// rather than steps of one cluster.  64 rows of beams 17 to 19 us, 1024 rows with
// 350,000 entries 27 to 29 us.
#pragma once

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"

namespace b200 {

struct PagedForkArgs {
    const int32_t *src, *keep, *seq_lens;
    const int32_t* table;
    int64_t table_stride;
    int32_t* out;
    int64_t out_stride;
    int32_t *free_pages, *seq_lens_out, *n_free_out, *copy_src, *copy_dst, *copy_rows;
    const int32_t* n_free;
    int n_seq, max_blocks, page_size, n_pages;
    // workspace: was, full, tails start at zero
    uint8_t *was, *full;   // [n_pages] held before, held in full after
    unsigned int* tails;   // [n_pages] n_seq - (the lowest row that ends in the page), 0: none
    int32_t* staged;       // [n_seq][max_blocks] the old table, where out replaces it
    int32_t* len;          // [n_seq] tokens kept
    int32_t* rank;         // [n_seq] number among the rows that need a page, -1: needs none
    int32_t* need;         // [n_seq] the rows that need one, in order
    int32_t* total;        // [2] how many, and the stack's pages (n_free_out may replace them)
    int32_t* freed;        // [ctas] freed pages of every 16384
    int page_ctas;
    int cols;  // entries of a row that one warp takes
};

constexpr int kForkRowThreads = 256;
constexpr int kForkCols = 256;    // entries of a row that one warp takes, at least
constexpr int kForkAtOnce = 4;    // entries a lane has in flight
constexpr int kForkThreads = 1024;
constexpr int kForkPer = 16;      // pages per thread
constexpr int kForkPages = kForkThreads * kForkPer;

struct ForkRow {
    int src, old_b, len, blocks, tail;  // source row, old blocks; tokens, blocks and tokens of a last block not full
};
// Row s before and after, from the lengths (valid until seq_lens_out is written).
__device__ __forceinline__ ForkRow fork_row(const PagedForkArgs& a, int s, bool record) {
    const int64_t cap = min((int64_t)a.max_blocks * a.page_size, (int64_t)INT32_MAX);
    auto length = [&](int i) {
        const int n = a.seq_lens[i];
        if (n >= 0 && n <= cap) return n;
        if (record) record_status(B200_DEVSTATUS_BOUNDS);
        return n < 0 ? 0 : (int)cap;
    };
    const unsigned ps = a.page_size;
    ForkRow r;
    r.src = a.src[s];
    r.old_b = (int)(((unsigned)length(s) + ps - 1) / ps);
    if (r.src >= a.n_seq) {
        if (record) record_status(B200_DEVSTATUS_BOUNDS);
        r.src = -1;
    }
    r.len = r.src < 0 ? 0 : max(0, min(a.keep[s], length(r.src)));
    r.blocks = (int)(((unsigned)r.len + ps - 1) / ps);
    r.tail = (int)((unsigned)r.len % ps);
    return r;
}

__global__ void __launch_bounds__(kForkRowThreads) paged_fork_mark_kernel(PagedForkArgs a) {
    const int s = blockIdx.x * (kForkRowThreads / 32) + (threadIdx.x >> 5), lane = threadIdx.x & 31;
    if (s >= a.n_seq) return;
    const int b0 = blockIdx.y * a.cols, b1 = (int)min((int64_t)a.max_blocks, (int64_t)b0 + a.cols);
    const ForkRow r = fork_row(a, s, lane == 0 && b0 == 0);
    if (lane == 0 && b0 == 0) a.len[s] = r.len;
    const int32_t* mine = a.table + s * a.table_stride;
    const int32_t* from = a.table + max(r.src, 0) * a.table_stride;
    bool bad = false;
    const int end = min(b1, max(r.old_b, r.blocks));
    for (int b = b0 + lane; b < end; b += 32 * kForkAtOnce) {
        int p[kForkAtOnce], q[kForkAtOnce];
#pragma unroll
        for (int e = 0; e < kForkAtOnce; ++e) {
            p[e] = b + 32 * e < min(end, r.old_b) ? mine[b + 32 * e] : -1;
            q[e] = b + 32 * e < min(end, r.blocks) ? from[b + 32 * e] : -1;
        }
#pragma unroll
        for (int e = 0; e < kForkAtOnce; ++e) {
            const int at = b + 32 * e;
            if (at < min(end, r.old_b)) {
                if (a.staged) a.staged[(int64_t)s * a.max_blocks + at] = p[e];
                if ((unsigned)p[e] < (unsigned)a.n_pages) a.was[p[e]] = 1;
                else bad = true;
            }
            if ((unsigned)q[e] < (unsigned)a.n_pages) {
                if (at + 1 == r.blocks && r.tail) atomicMax(a.tails + q[e], (unsigned)(a.n_seq - s));
                else a.full[q[e]] = 1;
            }
        }
    }
    if (bad) record_status(B200_DEVSTATUS_BOUNDS);
}

// Exclusive sum of v over the CTA's kForkThreads threads; the total in *total.
// `part` has 33 entries; two calls in a row need no barrier between them.
__device__ __forceinline__ int fork_scan(int v, int* part, int* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = x;
    __syncthreads();
    const int w = part[lane];
    int sum = w, before = lane < warp ? w : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    *total = sum;
    return before + x - v;
}

// Which of the kForkPer pages from p0 on this call frees, a bit each.
__device__ __forceinline__ unsigned fork_freed(const PagedForkArgs& a, int64_t p0) {
    if (p0 >= a.n_pages) return 0;
    // (the workspace rounds every array up to 256 bytes)
    const uint4 was = *reinterpret_cast<const uint4*>(a.was + p0), full = *reinterpret_cast<const uint4*>(a.full + p0);
    const uint32_t gone[4] = {was.x & ~full.x, was.y & ~full.y, was.z & ~full.z, was.w & ~full.w};
    unsigned bits = 0;
#pragma unroll
    for (int i = 0; i < kForkPer; ++i)
        if ((gone[i >> 2] >> (8 * (i & 3)) & 1u) && a.tails[p0 + i] == 0) bits |= 1u << i;
    return bits;
}

__global__ void __launch_bounds__(kForkThreads) paged_fork_count_kernel(PagedForkArgs a) {
    __shared__ int part[33];
    griddep_wait();
    const int tid = threadIdx.x;
    int total;
    if ((int)blockIdx.x < a.page_ctas) {
        const unsigned bits = fork_freed(a, ((int64_t)blockIdx.x * kForkThreads + tid) * kForkPer);
        fork_scan(__popc(bits), part, &total);
        if (tid == 0) a.freed[blockIdx.x] = total;
        return;
    }
    int before = 0;
    for (int base = 0; base < a.n_seq; base += kForkThreads) {
        const int s = base + tid;
        int need = 0;
        if (s < a.n_seq) {
            const ForkRow r = fork_row(a, s, false);
            if (r.tail) {
                const int p = a.table[r.src * a.table_stride + r.blocks - 1];
                if ((unsigned)p < (unsigned)a.n_pages) need = a.full[p] || a.tails[p] != (unsigned)(a.n_seq - s);
            }
        }
        const int at = before + fork_scan(need, part, &total);
        if (s < a.n_seq) a.rank[s] = need ? at : -1;
        if (need) a.need[at] = s;
        before += total;
    }
    if (tid == 0) a.total[0] = before, a.total[1] = a.n_free[0];
}

__global__ void __launch_bounds__(kForkThreads) paged_fork_write_kernel(PagedForkArgs a) {
    __shared__ int part[33];
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31;
    const int32_t* old = a.staged ? a.staged : a.table;
    const int64_t old_stride = a.staged ? a.max_blocks : a.table_stride;
    // pages freed by the CTAs before this one, and by all
    int mine = 0, all = 0, before, sum;
    for (int c = tid; c < a.page_ctas; c += kForkThreads) {
        const int n = a.freed[c];
        all += n;
        if (c < (int)blockIdx.x) mine += n;
    }
    fork_scan(mine, part, &before);
    fork_scan(all, part, &sum);
    int n0 = a.total[1];
    if (n0 < 0 || n0 > a.n_pages) {
        if (tid == 0 && blockIdx.x == 0) record_status(B200_DEVSTATUS_BOUNDS);
        n0 = n0 < 0 ? 0 : a.n_pages;
    }
    if ((int64_t)n0 + sum > a.n_pages) {  // more pages than exist: the surplus is dropped
        if (tid == 0 && blockIdx.x == 0) record_status(B200_DEVSTATUS_BOUNDS);
        sum = a.n_pages - n0;
    }
    const int pool = n0 + sum, got = min(a.total[0], pool);
    const unsigned ps = a.page_size;
    if ((int)blockIdx.x < a.page_ctas) {
        const int64_t p0 = ((int64_t)blockIdx.x * kForkThreads + tid) * kForkPer;
        unsigned bits = fork_freed(a, p0);
        int total, at = before + fork_scan(__popc(bits), part, &total);
        for (; bits && at < sum; bits &= bits - 1, ++at) {
            const int p = (int)p0 + __ffs(bits) - 1, r = sum - 1 - at;
            a.free_pages[n0 + at] = p;
            if (r < got) {  // the r-th row in need takes it
                const int s = a.need[r];
                a.out[s * a.out_stride + ((unsigned)a.len[s] + ps - 1) / ps - 1] = p;
                a.copy_dst[s] = p;
            }
        }
        return;
    }
    // a warp per row and a.cols entries
    const int cols = (int)(((int64_t)a.max_blocks + a.cols - 1) / a.cols);
    const int64_t task = (int64_t)(blockIdx.x - a.page_ctas) * (kForkThreads / 32) + (tid >> 5);
    if (task == 0 && lane == 0) a.n_free_out[0] = pool - got;
    if (task >= (int64_t)a.n_seq * cols) return;
    const int s = (int)(task / cols), b0 = (int)(task % cols) * a.cols;
    const int b1 = (int)min((int64_t)a.max_blocks, (int64_t)b0 + a.cols);
    const int len = a.len[s], src = max(0, a.src[s]), rank = a.rank[s];
    const int blocks = (int)(((unsigned)len + ps - 1) / ps), tail = (int)((unsigned)len % ps);
    const int32_t* from = old + src * old_stride;
    int32_t* to = a.out + s * a.out_stride;
    const int whole = rank >= 0 ? blocks - 1 : blocks;  // entries taken as they are
    for (int b = b0 + lane; b < b1; b += 32 * kForkAtOnce) {
        int p[kForkAtOnce];
#pragma unroll
        for (int e = 0; e < kForkAtOnce; ++e) p[e] = b + 32 * e < min(b1, whole) ? from[b + 32 * e] : -1;
#pragma unroll
        for (int e = 0; e < kForkAtOnce; ++e) {
            const int at = b + 32 * e;
            if (at < b1 && (at < whole || at >= blocks)) to[at] = p[e];
        }
    }
    if (b0 != 0 || lane != 0) return;
    const bool served = rank >= 0 && rank < got;
    a.seq_lens_out[s] = rank >= 0 && !served ? len - tail : len;
    a.copy_src[s] = served ? from[blocks - 1] : -1;
    a.copy_rows[s] = served ? tail : 0;
    if (!served) {
        a.copy_dst[s] = -1;
        if (rank >= 0) to[blocks - 1] = -1;
    } else if (rank >= sum) {  // from the stack as it was; above that lie the freed pages
        const int p = a.free_pages[pool - 1 - rank];
        to[blocks - 1] = p;
        a.copy_dst[s] = p;
    }
}

// ------------------------------------------------------------------- copies

struct PagedCopyArgs {
    b200_paged_kv kv;
    const int32_t *src, *dst, *rows;
    int64_t n;
    int part;  // rows of a page that one CTA copies
};

constexpr int kCopyThreads = 256;

// CTA (entry, part of the page's rows): 16-byte pieces of K and of V, four of
// each in flight per thread.  Bound by memory: two bytes moved per byte copied.
// 4096 pages of 64 KB 88 us, 6.1 TB/s; 48 partial pages 6.3 us, latency.
__global__ void __launch_bounds__(kCopyThreads) paged_copy_kernel(PagedCopyArgs a) {
    const int64_t i = blockIdx.x;
    const int src = a.src[i], dst = a.dst[i];
    if (src < 0 || dst < 0 || src == dst) return;
    int rows = a.rows ? a.rows[i] : a.kv.page_size;
    const bool first = blockIdx.y == 0 && threadIdx.x == 0;
    if (src >= a.kv.n_pages || dst >= a.kv.n_pages || rows > a.kv.page_size) {
        if (first) record_status(B200_DEVSTATUS_BOUNDS);
        if (src >= a.kv.n_pages || dst >= a.kv.n_pages) return;
        rows = a.kv.page_size;
    }
    if (rows <= 0) return;
    const int per_head = a.kv.head_dim / 8, per_row = a.kv.n_head_kv * per_head;
    const int r0 = blockIdx.y * a.part, r1 = min(rows, r0 + a.part);
    const uint8_t* ks = static_cast<const uint8_t*>(a.kv.k) + src * a.kv.k_page;
    const uint8_t* vs = static_cast<const uint8_t*>(a.kv.v) + src * a.kv.v_page;
    uint8_t* kd = static_cast<uint8_t*>(a.kv.k) + dst * a.kv.k_page;
    uint8_t* vd = static_cast<uint8_t*>(a.kv.v) + dst * a.kv.v_page;
    // pieces of r0 .. r1 - 1 in order; below 2^31: a page has at most 2^36 / 16 bytes
    const int64_t end = (int64_t)(r1 - r0) * per_row;
    for (int64_t u = threadIdx.x; u < end; u += kCopyThreads * 4) {
        uint4 x[4], y[4];
        int64_t ko[4], vo[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t w = u + j * kCopyThreads;
            if (w >= end) continue;
            const int row = (int)((unsigned)w / (unsigned)per_row), c = (int)w - row * per_row;
            const int head = (int)((unsigned)c / (unsigned)per_head), d = c - head * per_head;
            ko[j] = (int64_t)(r0 + row) * a.kv.k_row + head * a.kv.k_head + d * 16;
            vo[j] = (int64_t)(r0 + row) * a.kv.v_row + head * a.kv.v_head + d * 16;
            x[j] = __ldcs(reinterpret_cast<const uint4*>(ks + ko[j]));
            y[j] = __ldcs(reinterpret_cast<const uint4*>(vs + vo[j]));
        }
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (u + j * kCopyThreads < end) {
                *reinterpret_cast<uint4*>(kd + ko[j]) = x[j];
                *reinterpret_cast<uint4*>(vd + vo[j]) = y[j];
            }
    }
    if (a.kv.k_lo && blockIdx.y == 0) {
        const uint4* lo = static_cast<const uint4*>(a.kv.k_lo);
        const uint4* hi = static_cast<const uint4*>(a.kv.k_hi);
        for (int c = threadIdx.x; c < per_row; c += kCopyThreads) {
            static_cast<uint4*>(a.kv.k_lo)[(int64_t)dst * per_row + c] = lo[(int64_t)src * per_row + c];
            static_cast<uint4*>(a.kv.k_hi)[(int64_t)dst * per_row + c] = hi[(int64_t)src * per_row + c];
        }
    }
}

}  // namespace b200
