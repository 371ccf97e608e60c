// paged_prefill.cuh -- attention of a chunk of new tokens per sequence over the
// paged cache, on the 5th-generation tensor cores.
//
// Rows are (token, query head of the KV head) pairs, flat within a sequence and
// a KV head: every one of them reads the same keys, so a tile of 128 rows is full
// whatever the number of heads to a KV head.  A unit is one or two such tiles of
// one (sequence, KV head) with the tiles of keys that any of its rows sees; a
// launch lays all units end to end (plan kernel), cuts the line of key tiles into
// equal ranges, one per SM, whatever lengths and heads are (main kernel), and
// joins the units that a cut went through (finish kernel).  Three launches, 40 bytes of
// schedule a unit and 11 KB, results that do not depend on timing.
//
// 8192 tokens, 64/8 heads x 128: 1010 to 1066 us, 1.03 to 1.09 PFLOP/s, in short runs,
// 1180 us in long ones (power limit, 1.67 GHz); the products and their barriers bound
// it.  2048 tokens at 129024: 8.4 to 8.9 ms, the power limit.  8 sequences of 5 tokens
// at up to 4160: 26 us, all of it latency.
//
// The weights are rounded once to 16 bits for their product with V: the tensor core
// takes them in V's type, and sums of two or three 16-bit parts, as paged_attn has them,
// would take as many products.  Against 64 bits f16 outputs are 2.6e-4 and bf16 2.3e-3 off
// (RMS), 1.3 to 1.45 times an output that is only rounded.
//
// The main kernel spills: the compiler counts 112 to 124 bytes of stores and 160 to 200 of
// loads at head dim 256, 256 to 268 and 316 to 328 at 128, 116 to 192 and 216 to 292 at 64.
// A row's 128 scores leave 72 of the 200 registers to the rest.
#pragma once

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"
#include "f32_pairs.cuh"
#include "paged_ring.h"
#include "paged_store.cuh"
#include "tcgen05.cuh"

namespace b200 {

struct PagedPrefillArgs {
    // [page][head][row][channel] views of K and V for boxes of box rows of a page by
    // 64 channels, and [KV head][token][head][channel] of q for boxes of 128 rows
    CUtensorMap map_k, map_v, map_q;
    int box;    // 0: a page has no eight rows in a row that start at a multiple of eight
    int q_box;  // tokens of 128 rows; 0: the heads of a KV head do not divide 128
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
    // workspace
    int64_t max_units;  // there is room for, and for n_tokens * n_head rows in bad
    struct PfHeader* header;
    int4* desc;         // two per unit: {sequence, first flat row, first key tile, key tiles}, {first, n, len, -}
    int64_t* prefix;    // [units + 1] steps of the units before
    int2* start;        // [CTAs] {unit, KV head} that a CTA's range starts in
    int4* cut;          // [CTAs] two for the unit that begins in a CTA's range and goes on past it:
                        // {sequence, KV head, first flat row, pieces (0: no such unit)}, {first, n, len, -}
    int2* bad;          // rows to compute again: {flat (token, head), unit}
    unsigned* claim;    // [CTAs][8] those of the unit that begins in a CTA's range and goes on past it: bits of its rows
    float4* piece_ml;   // [2 * CTAs][tiles][128] {reference, sum, mask reference, -} of cut units
    float4* piece_o;    // [2 * CTAs][tiles][D / 4][128] their sums of weighted values
};

struct PfHeader {
    int64_t total;    // steps of all units of one KV head
    int64_t per_cta;  // of all KV heads' units, to a CTA
    int units, n_bad;
    int whole;  // CTA c has unit c and nothing else
};

constexpr int kPfCtas = 148;   // one per SM
constexpr int kPfRows = 128;   // rows of a tile: the lanes of tensor memory
// A unit counts as many steps as it has key tiles and these: its queries, the first
// scores and the outputs, which nothing overlaps.  (8192 tokens, at a step where they
// took 1077 us with 3: 1105 with 2, 1094 with 4; 33 ragged sequences 76, 76, 79.)
constexpr int kPfUnitSteps = 3;
// A unit stays whole on a CTA of its own where all find one and the largest has at most
// this many steps more than an equal range: a second unit's start and the pieces'
// join would cost as much.  (us, always cut / 2 / 6 / 12: 512 tokens of 64/8 heads x 128
// 30.8 / 26.7 / 26.7 / 26.7; 384 at 700 40.9 / 40.9 / 37.0 / 36.9; 256 at 1000 36.9 / 36.9 /
// 36.9 / 39.0; 2 x 300 at 100, 32/8 29.3 / 29.3 / 26.7 / 26.7; 3 x 300 at 300, 16/4 x 256 36.9 /
// 37.0 / 30.8 / 30.8; 16 x 5 at 600, 12/2 22.6 / 22.6 / 26.5 / 26.3; five others alike.)
constexpr int kPfWholeSteps = 6;
// Key tiles and row tiles of a unit by head dim: two row tiles take turns between
// the tensor core and the exponentials; at head dim 256 the outputs of one fill
// half of tensor memory, and two score buffers of 64 keys take its place.
B200_HD constexpr int pf_tiles(int d) { return d == 256 ? 1 : 2; }
B200_HD constexpr int pf_keys(int d) { return d == 256 ? 64 : 128; }
B200_HD constexpr int pf_stages(int d) { return d == 64 ? 8 : 5; }

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

// ------------------------------------------------- rows computed once more

constexpr int kPfFinishThreads = 256;
constexpr int kPfAgainWarps = kPfFinishThreads / 32;

template <int D>
struct PfAgain {
    double m[kPfAgainWarps], sum[kPfAgainWarps], o[kPfAgainWarps][D];
};

// D / 32 channels of a row from their address on, as f32.
template <bool BF16, int E>
__device__ __forceinline__ void pf_channels(const void* at, float (&x)[E]) {
    uint32_t w[E / 2];
    if constexpr (E == 2) w[0] = __ldg(static_cast<const uint32_t*>(at));
    else if constexpr (E == 4) {
        const uint2 v = __ldg(static_cast<const uint2*>(at));
        w[0] = v.x, w[1] = v.y;
    } else {
        const uint4 v = __ldg(static_cast<const uint4*>(at));
        w[0] = v.x, w[1] = v.y, w[2] = v.z, w[3] = v.w;
    }
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const float2 f = unpack16<BF16>(w[e / 2]);
        x[e] = f.x, x[e + 1] = f.y;
    }
}

// One row of one head by a CTA, in f32 products of whole values: what the formula says
// whatever infinities and NaN meet.  Values near bf16's largest add up past the f32
// range though their mean is in it: sums are kept in 64 bits.  Every warp takes every
// eighth run of 32 positions, looked up by a lane each and read four at a time; lane l
// owns channels l * D / 32 on.  The warps' sums are joined in order.
// Bound by 64-bit arithmetic and conversions: 7 x 10^9 positions of a row a second with
// every SM at it.  5 rows of 12 heads over 131072 positions 5.3 to 6.3 ms (452 ms with a
// warp to a row and a position at a time); 512 rows of 64 heads over 16384 73 ms (167).
template <bool BF16, int D>
__device__ __noinline__ void pf_row(const PagedPrefillArgs& a, PfAgain<D>& sh, int s, int n, int len, int64_t t, int i,
                                    int head) {
    constexpr int E = D / 32, AT_ONCE = 4;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, h = head / a.group, ps = a.kv.page_size;
    float q[E];
    pf_channels<BF16, E>(a.q + t * a.q_stride + head * D + lane * E, q);
    double o[E], m = -INFINITY, sum = 0.;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.;
    const int at = len - n + i;  // may be negative: sees nothing
    const int p0 = a.window > 0 ? max(0, at - a.window + 1) : 0;
    const uint8_t* kb = static_cast<const uint8_t*>(a.kv.k) + h * a.kv.k_head + lane * E * 2;
    const uint8_t* vb = static_cast<const uint8_t*>(a.kv.v) + h * a.kv.v_head + lane * E * 2;
    for (int64_t first = (int64_t)p0 + 32 * warp; first <= at; first += 32 * kPfAgainWarps) {
        const int64_t p = first + lane;
        float bias = 0.f;
        int64_t ko = 0, vo = 0;
        bool seen = p <= at;
        if (seen && a.mask) {
            bias = h2f(a.mask[s * a.mask_stride + p]);
            seen = bias != -INFINITY;
        }
        if (seen) {
            const int page = a.table[s * a.table_stride + p / ps], r = (int)(p % ps);
            seen = (unsigned)page < (unsigned)a.kv.n_pages;
            if (!seen) record_status(B200_DEVSTATUS_BOUNDS);
            ko = seen ? page * a.kv.k_page + r * a.kv.k_row : 0;
            vo = seen ? page * a.kv.v_page + r * a.kv.v_row : 0;
        }
        for (unsigned left = __ballot_sync(0xffffffffu, seen); left;) {
            float k[AT_ONCE][E], v[AT_ONCE][E], x[AT_ONCE], b[AT_ONCE];
            int count = 0;
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {  // (past the last one: what lane 0 names, not counted)
                const int from = __ffs(left) - 1;
                if (from >= 0) count = j + 1, left &= left - 1;
                const int l = from >= 0 ? from : 0;
                pf_channels<BF16, E>(kb + __shfl_sync(0xffffffffu, ko, l), k[j]);
                pf_channels<BF16, E>(vb + __shfl_sync(0xffffffffu, vo, l), v[j]);
                b[j] = __shfl_sync(0xffffffffu, bias, l);
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                x[j] = 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) x[j] = fmaf(q[e], k[j][e], x[j]);
                x[j] = warp_sum(x[j]);
            }
            double y[AT_ONCE], top = m;  // a mask of the lowest value keeps the score's bits
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                y[j] = (double)(x[j] * a.scale) + (double)b[j];
                if (j < count && y[j] > top) top = y[j];
            }
            if (top > m) {
                if (m != -INFINITY) {
                    const double f = exp2f((float)((m - top) * 1.4426950408889634));
                    sum *= f;
#pragma unroll
                    for (int e = 0; e < E; ++e) o[e] *= f;
                }
                m = top;
            }
#pragma unroll
            for (int j = 0; j < AT_ONCE; ++j) {
                if (j >= count) break;
                const double w = y[j] == -INFINITY ? 0.f : exp2f((float)((y[j] - m) * 1.4426950408889634));
                sum += w;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] = fma(w, (double)v[j][e], o[e]);
            }
        }
    }
    __syncthreads();  // the row before has been read
    if (lane == 0) sh.m[warp] = m, sh.sum[warp] = sum;
#pragma unroll
    for (int e = 0; e < E; ++e) sh.o[warp][lane * E + e] = o[e];
    __syncthreads();
    const int c = 2 * threadIdx.x;
    if (c >= D) return;
    double most = -INFINITY, all = 0., y0 = 0., y1 = 0.;
    for (int w = 0; w < kPfAgainWarps; ++w) most = fmax(most, sh.m[w]);
    for (int w = 0; w < kPfAgainWarps; ++w) {
        const double f = sh.m[w] == -INFINITY ? 0.f : exp2f((float)((sh.m[w] - most) * 1.4426950408889634));
        all += f * sh.sum[w];
        y0 += f * sh.o[w][c], y1 += f * sh.o[w][c + 1];
    }
    const double inv = all == 0. ? 0. : 1. / all;
    *reinterpret_cast<uint32_t*>(a.out + (t * a.n_head + head) * D + c) =
        all == 0. ? 0u : pack16<BF16>((float)(y0 * inv), (float)(y1 * inv));
}

// ------------------------------------------------------------------- plan

// Exclusive sum of v over the CTA's 1024 threads; the total in *total.
__device__ __forceinline__ int64_t pf_scan(int64_t v, int64_t* part, int64_t* total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int64_t x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();
    if (lane == 31) part[warp] = x;
    __syncthreads();
    const int64_t w = part[lane];
    int64_t sum = w, before = lane < warp ? w : 0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        sum += __shfl_xor_sync(0xffffffffu, sum, o);
        before += __shfl_xor_sync(0xffffffffu, before, o);
    }
    *total = sum;
    return before + x - v;
}

constexpr int kPfPlanThreads = 1024;

// The units of one KV head in order of sequences and rows.  One CTA: latency only.
__global__ void __launch_bounds__(kPfPlanThreads) paged_prefill_plan_kernel(const __grid_constant__ PagedPrefillArgs a,
                                                                            int rows, int keys) {
    __shared__ int64_t part[32], s_base[kPfPlanThreads + 1];
    __shared__ PfSeq s_seq[kPfPlanThreads];
    __shared__ int64_t s_prefix[kPfPlanThreads + 1];
    const int tid = threadIdx.x;
    griddep_launch_dependents();
    int64_t units = 0, tiles = 0, sum;
    int largest = 0;
    for (int base = 0; base < a.n_seq; base += kPfPlanThreads) {
        const int s = base + tid, count = min(kPfPlanThreads, a.n_seq - base);
        PfSeq q = {0, 0, 0};
        if (s < a.n_seq) q = pf_seq(a, s, true);
        const int64_t at = pf_scan(((int64_t)q.n * a.group + rows - 1) / rows, part, &sum);
        s_base[tid] = at;
        s_seq[tid] = q;
        if (tid == 0) s_base[count] = sum;
        __syncthreads();
        if (units + sum > a.max_units) {  // starts that go back name rows more than once: what passes the room is left out
            if (tid == 0) record_status(B200_DEVSTATUS_BOUNDS);
            sum = a.max_units - units;
        }
        for (int64_t u0 = 0; u0 < sum; u0 += kPfPlanThreads) {
            const int64_t u = u0 + tid;
            int64_t steps = 0;
            int4 d0, d1;
            if (u < sum) {
                int lo = 0, hi = count;  // s_base[lo] <= u < s_base[hi]
                while (hi - lo > 1) {
                    const int mid = (lo + hi) >> 1;
                    if (s_base[mid] <= u) lo = mid;
                    else hi = mid;
                }
                const PfSeq t = s_seq[lo];
                const int row0 = (int)(u - s_base[lo]) * rows;
                const int row1 = (int)min((int64_t)row0 + rows, (int64_t)t.n * a.group) - 1;
                const int at0 = t.len - t.n + row0 / a.group, at1 = t.len - t.n + row1 / a.group;
                const int first = a.window > 0 ? max(0, max(-1, at0) - a.window + 1) / keys : 0;
                const int cost = at1 < 0 ? 1 : at1 / keys - first + 1;
                steps = cost + kPfUnitSteps;
                d0 = make_int4(base + lo, row0, first, cost);
                d1 = make_int4(t.first, t.n, t.len, 0);
            }
            int64_t more;
            const int64_t before = tiles + pf_scan(steps, part, &more);
            if (u < sum) {
                a.desc[2 * (units + u)] = d0;
                a.desc[2 * (units + u) + 1] = d1;
                a.prefix[units + u] = before;
                if (units + u < kPfPlanThreads) s_prefix[units + u] = before;
            }
            tiles += more;
            largest = max(largest, (int)min(steps, (int64_t)INT32_MAX));
        }
        units += sum;
        __syncthreads();  // s_base and s_seq are read no more
    }
    const int64_t all = tiles * a.kv.n_head_kv, per = max((int64_t)1, (all + kPfCtas - 1) / kPfCtas);
    const bool whole = __syncthreads_or(largest > per + kPfWholeSteps) == 0 && units * a.kv.n_head_kv <= kPfCtas;
    if (tid == 0) {
        a.prefix[units] = tiles;
        a.header->whole = whole;
        a.header->total = tiles;
        a.header->per_cta = per;
        a.header->units = (int)units;
        a.header->n_bad = 0;
    }
    // where every CTA starts (the loops above end with a barrier behind the last prefix),
    // and beside it no row is listed yet
    if (tid >= kPfPlanThreads / 2) {
        for (int i = tid - kPfPlanThreads / 2; i < kPfCtas * 8; i += kPfPlanThreads / 2) a.claim[i] = 0;
    } else if (whole) {
        if (tid < units * a.kv.n_head_kv) a.start[tid] = make_int2((int)(tid % units), (int)(tid / units));
    } else if (tid < kPfCtas && tid * per < all) {
        const int64_t h = tid * per / tiles, x = tid * per - h * tiles;
        const int64_t* prefix = units <= kPfPlanThreads ? s_prefix : a.prefix;
        int lo = 0, hi = (int)units;  // prefix[lo] <= x < prefix[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (prefix[mid] <= x) lo = mid;
            else hi = mid;
        }
        a.start[tid] = make_int2(lo, (int)h);
    }
}

// A unit, or the part of one that lies in a CTA's range.
struct PfUnit {
    int u, s, h, row0, first, n, len, tile0;  // tile0: the unit's first key tile
    int tb, te, cost;                      // key tiles tb .. te - 1 of cost
    int shift;                             // the first of them to be done, from tb
    // key tile of step t: all in turn, from `shift` on
    __device__ __forceinline__ int tile(int t) const {
        const int n = te - tb, i = t + shift;
        return tile0 + tb + (i < n ? i : i - n);
    }
};
// Walks over a range of the line of key tiles of all KV heads' units.
struct PfWalk {
    int64_t w, w1;
    int u, h;
    int steps;  // done by this CTA
    __device__ __forceinline__ bool next(const PagedPrefillArgs& a, int units, int64_t total, PfUnit& x) {
        while (w < w1) {
            const int4 d0 = __ldg(a.desc + 2 * (int64_t)u), d1 = __ldg(a.desc + 2 * (int64_t)u + 1);
            // the unit's first key tile, and where the range starts and ends from there
            const int64_t start = h * total + __ldg(reinterpret_cast<const long long*>(a.prefix) + u) + kPfUnitSteps;
            x.u = u, x.s = d0.x, x.row0 = d0.y, x.tile0 = d0.z, x.cost = d0.w;
            x.first = d1.x, x.n = d1.y, x.len = d1.z;
            x.h = h;
            x.tb = (int)max((int64_t)0, w - start);
            x.te = (int)min((int64_t)x.cost, w1 - start);
            w = start + x.cost;
            if (++u == units) u = 0, ++h;
            if (x.tb < x.te) {
                // units of one long sequence are done in step: CTAs that are at the same
                // step read the same keys, from the L2 cache all but one of them
                const int at = steps % x.cost;
                x.shift = at >= x.tb && at < x.te ? at - x.tb : 0;
                steps += x.te - x.tb + kPfUnitSteps;
                return true;
            }
        }
        return false;
    }
};

// ------------------------------------------------------------------- main

template <int D>
struct PfShared {
    static constexpr int ST = pf_stages(D);
    uint64_t q_full, q_empty, full[ST], empty[ST], s_full[2], p_ready[2], o_done[2], fix, done;
    uint32_t tmem;
    int aborted;                         // a wait ran out
    uint32_t filled[2], asked[2], fixed[2];  // phases of full, q_full and fix that each copying warp entered
    float tmax[4][2];  // the largest of each copying warp's rows
    // mask entries of the last tiles.  Those of V's tile i are written when its stage is
    // free: then the tile before i - 2 (i - 3 with 8 stages) has been through the softmax
    static constexpr int NB = ST == 8 ? 4 : 3;
    alignas(16) float bias[NB][pf_keys(D)];
};
template <int D>
B200_HD constexpr int pf_stage_bytes() { return pf_keys(D) * D * 2; }
template <int D>
B200_HD constexpr int pf_q_bytes() { return pf_tiles(D) * kPfRows * D * 2; }
template <int D>
B200_HD constexpr int pf_smem() { return pf_q_bytes<D>() + pf_stages(D) * pf_stage_bytes<D>() + 1024; }

// Place of key tile t's K and V in the order of loads K0 K1 V0 K2 V1 .. of n tiles.
__device__ __forceinline__ int pf_k_place(int t) { return t == 0 ? 0 : 2 * t - 1; }
__device__ __forceinline__ int pf_v_place(int t, int n) { return t == n - 1 ? 2 * n - 1 : 2 * t + 2; }

__device__ __forceinline__ void pf_arrive(uint64_t* bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
__device__ __forceinline__ void pf_tma(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w, uint64_t* bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
        "[%6];" ::"r"(dst),
        "l"(map), "r"(x), "r"(y), "r"(z), "r"(w), "r"(smem_u32(bar))
        : "memory");
}
// Bits lo .. hi of a word (none for hi < lo, hi < 0 or lo > 31).
__device__ __forceinline__ uint32_t pf_bits(int lo, int hi) {
    const int l = max(lo, 0), h = min(hi, 31);
    return h < l ? 0u : (0xffffffffu >> (31 - h + l)) << l;
}
// Waits of this kernel: the clock and the limit are read once in 256 tries that found
// nothing (a wait may last that much longer than the limit), by as few instructions as
// can be: there are twenty such places, and what they take of the instruction cache
// costs the others (8192 tokens 1231 -> 1115 us).
__device__ __forceinline__ bool pf_wait_one(uint64_t* bar, uint32_t parity) {
    unsigned long long began = 0;
#pragma unroll 1
    for (uint32_t i = 1; !mbar_try_wait(bar, parity); ++i)
        if ((i & 255u) == 0) {
            const unsigned long long now = globaltimer();
            if (began == 0) began = now;
            if (now - began > g_wait_timeout_ns) {
                record_status(B200_DEVSTATUS_TIMEOUT);
                return false;
            }
        }
    return true;
}
// A warp's wait: the same answer for every lane.
__device__ __forceinline__ bool pf_wait(uint64_t* bar, uint32_t parity) {
    return __all_sync(0xffffffffu, pf_wait_one(bar, parity));
}
// pf_land_phases on the barriers from bars on; a warp has `share` arrivals in a phase.
__device__ __forceinline__ void pf_land(uint64_t* bars, PfPhases p, uint32_t share) {
    pf_land_phases(
        p,
        [&](uint32_t stage) {
            asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bars + stage)), "r"(share)
                         : "memory");
        },
        [&](uint32_t stage, uint32_t parity) { mbar_wait_drain(bars + stage, parity); });
}
__device__ __forceinline__ void pf_cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
__device__ __forceinline__ void pf_cp16(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ float pf_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ const uint4 kPfNan = {0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};  // of f16 and of bf16

constexpr int kPfThreads = 384;     // two softmax warpgroups; two warps of copies, tensor-core issue
constexpr int kPfCopyThreads = 64;
constexpr int kPfIssueWarp = 10;
constexpr float kPfLazy = 8.f;      // the reference stays until the maximum passes it by 2^8
// f16 weights are taken times 2^7: 2^15 at most with the lazy reference, and 2^-31 of
// the reference is still a value
template <bool BF16>
constexpr float kPfShift = BF16 ? 0.f : 7.f;

template <bool BF16, int D, bool MASK>
__global__ void __launch_bounds__(kPfThreads, 1) paged_prefill_kernel(const __grid_constant__ PagedPrefillArgs a) {
    constexpr int NT = pf_tiles(D), KT = pf_keys(D), ST = pf_stages(D), STAGE = pf_stage_bytes<D>();
    constexpr int QTILE = kPfRows * D * 2, QHALF = kPfRows * 128, KHALF = KT * 128;
    constexpr uint32_t O_COL = NT == 2 ? 2 * KT : 256;  // scores from column 0, outputs from here
    constexpr uint32_t S_STEP = NT == 2 ? KT : 128;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ PfShared<D> sh;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, role = warp >> 2;
    const uint32_t q_smem = (smem_u32(smem_raw) + 1023u) & ~1023u, ring = q_smem + pf_q_bytes<D>();

    if (warp == kPfIssueWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&sh.tmem)),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (tid == 0) {
        mbar_init(&sh.q_full, kPfCopyThreads);
        mbar_init(&sh.q_empty, 1);
        for (int i = 0; i < ST; ++i) mbar_init(&sh.full[i], kPfCopyThreads + (MASK ? 2 : 0)), mbar_init(&sh.empty[i], 1);
        for (int j = 0; j < 2; ++j) mbar_init(&sh.s_full[j], 1), mbar_init(&sh.p_ready[j], 4), mbar_init(&sh.o_done[j], 1);
        mbar_init(&sh.fix, 2);
        mbar_init(&sh.done, 1);
        sh.aborted = 0;
        mbar_fence_init();
    }
    griddep_wait();  // the schedule
    griddep_launch_dependents();
    const int units = a.header->units;
    const int64_t total = a.header->total, per_cta = a.header->per_cta;
    PfWalk walk;
    walk.w = min(total * a.kv.n_head_kv, per_cta * blockIdx.x);
    walk.w1 = min(total * a.kv.n_head_kv, walk.w + per_cta);
    const int2 start = a.start[blockIdx.x];  // (not used by a CTA without work)
    if (a.header->whole) {
        walk.w = walk.w1 = 0;
        if ((int64_t)blockIdx.x < (int64_t)units * a.kv.n_head_kv) {
            walk.w = start.y * total + a.prefix[start.x];
            walk.w1 = start.y * total + a.prefix[start.x + 1];
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    walk.u = start.x, walk.h = start.y, walk.steps = 0;
    const uint32_t tmem = sh.tmem;
    PfUnit x;

    if (role == 2) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 104;");
        if (tid < 256 + kPfCopyThreads) {
            // ---- copies: keys and values by pages into 128-byte swizzled rows.  The
            // barrier of a tile counts its copies' ends; the thread that issues the
            // products puts the fence between the copies' writes and the tensor core
            const int pw = warp - 8;
            constexpr int CH = D / 8;            // 16-byte pieces of a row
            constexpr int RPI = 32 / CH;         // rows a warp copies at once
            constexpr int RPW = KT / 2, RPL = RPW / 32;  // rows of a tile to a warp, to a lane
            auto issued = [&](uint64_t* bar) {
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
            };
            // a warp's share of a barrier where TMA copies `bytes` for it
            auto expects = [&](uint64_t* bar, uint32_t bytes, uint32_t arrivals) {
                if (lane == 0) {
                    if (bytes) mbar_arrive_expect_tx(bar, bytes), --arrivals;
                    if (arrivals)
                        asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0], %1;" ::"r"(smem_u32(bar)), "r"(arrivals)
                                     : "memory");
                }
                __syncwarp();
            };
            constexpr int HALVES = D / 64, MINE = HALVES / 2;  // blocks of 64 channels; of each warp
            int stage = 0, unit = 0, tiles = 0;
            uint32_t lap = 0, fix = 0;  // laps of the ring, phases of sh.fix
            bool ok = true;
            const int ps = a.kv.page_size, box_log = __ffs(a.box) - 1;
            const uint64_t krow = a.kv.k_row >> 4, vrow = a.kv.v_row >> 4, kpage = a.kv.k_page >> 4, vpage = a.kv.v_page >> 4;
            int4 cut = make_int4(0, 0, 0, 0), cut_seq = cut;
            while (ok && walk.next(a, units, total, x)) {
                if (x.tb == 0 && x.te < x.cost) {
                    // its last key tile's CTA; walk.w is one past that tile
                    cut = make_int4(x.s, x.h, x.row0, (int)((walk.w - 1) / per_cta) - (int)blockIdx.x + 1);
                    cut_seq = make_int4(x.first, x.n, x.len, 0);
                }
                const int n = x.te - x.tb, rows = min(NT * kPfRows, x.n * a.group - x.row0);
                const int at1 = x.len - x.n + (x.row0 + rows - 1) / a.group;  // the last position that a row sees
                const int at0 = a.window > 0 ? x.len - x.n + x.row0 / a.group - a.window + 1 : 0;  // and the first
                if (unit && !(ok = pf_wait(&sh.q_empty, (unit - 1) & 1))) break;
                ++unit;
                if (a.q_box) {
                    // 128 rows of 64 channels to a copy; rows past the sequence's are not used
                    const int tiles = (rows + kPfRows - 1) / kPfRows;
                    const int mine = tiles * (HALVES == 1 ? 1 - pw : MINE);
                    expects(&sh.q_full, (uint32_t)(mine * QHALF), 32);
                    if (lane < mine) {
                        const int j = HALVES == 1 ? lane : lane / MINE, hf = HALVES == 1 ? 0 : 2 * (lane % MINE) + pw;
                        pf_tma(q_smem + j * QTILE + hf * QHALF, &a.map_q, hf * 64, 0, x.first + x.row0 / a.group + j * a.q_box,
                               x.h, &sh.q_full);
                    }
                } else {
                    // (token, head) of the lane's row, one step of 2 RPI rows after the other
                    int r = pw * RPI + lane / CH, i = (x.row0 + r) / a.group, g = x.row0 + r - i * a.group;
                    const int c = lane % CH, di = 2 * RPI / a.group, dg = 2 * RPI - di * a.group;
#pragma unroll 4
                    for (; r < rows; r += 2 * RPI) {
                        const uint16_t* src = a.q + (int64_t)(x.first + i) * a.q_stride + (x.h * a.group + g) * D + c * 8;
                        const int rr = r & (kPfRows - 1);
                        pf_cp16(q_smem + (r / kPfRows) * QTILE + (c >> 3) * QHALF + rr * 128 + (((c & 7) ^ (rr & 7)) << 4), src);
                        i += di, g += dg;
                        if (g >= a.group) g -= a.group, ++i;
                    }
                    issued(&sh.q_full);
                }
                const uint8_t* kb = static_cast<const uint8_t*>(a.kv.k) + x.h * a.kv.k_head;
                const uint8_t* vb = static_cast<const uint8_t*>(a.kv.v) + x.h * a.kv.v_head;
                const int32_t* table = a.table + x.s * a.table_stride;
                const uint16_t* mask = MASK ? a.mask + x.s * a.mask_stride : nullptr;
                // by TMA, a box of a page to a lane: its page and row
                struct Boxes {
                    int page, row, rows;  // rows: of the tile, that any query sees
                    bool on;              // this way, not the other
                };
                auto find_boxes = [&](int t) {
                    const int p0 = x.tile(t) * KT;
                    Boxes b;
                    b.page = b.row = 0;
                    b.rows = min(KT, max(0, at1 + 1 - p0));
                    b.on = a.box > 0;
                    if (b.on && lane * a.box < b.rows) {
                        const unsigned at = (unsigned)p0 + (unsigned)(lane * a.box), blk = at / (unsigned)ps;
                        b.page = __ldg(table + blk);
                        b.row = (int)(at - blk * (unsigned)ps);
                    }
                    return b;
                };
                auto send_boxes = [&](const CUtensorMap* map, const Boxes& b, uint64_t* bar, uint32_t arrivals) {
                    const int boxes = (b.rows + a.box - 1) >> box_log;
                    expects(bar, (uint32_t)(boxes * a.box * 128 * (HALVES == 1 ? 1 - pw : MINE)), arrivals);
                    if (lane < boxes)
#pragma unroll
                        for (int hf = pw; hf < HALVES; hf += 2)
                            pf_tma(ring + stage * STAGE + hf * KHALF + lane * a.box * 128, map, hf * 64, b.row, x.h, b.page,
                                   bar);
                };
                auto advance = [&] {
                    if (MASK) {
                        __syncwarp();
                        if (lane == 0) pf_arrive(&sh.full[stage]);  // the mask entries are written
                    }
                    if (++stage == ST) stage = 0, ++lap;
                };
                auto copy_boxes = [&](const Boxes& b, bool value) {
                    const bool part = value && b.rows < KT;
                    // (rows of K that no query sees: what was there)
                    send_boxes(value ? &a.map_v : &a.map_k, b, part ? &sh.fix : &sh.full[stage], part ? 1 : 32);
                    if (part) {
                        // a weight of 0 meets every value: rows that no query sees become 0
                        if (!(ok = pf_wait(&sh.fix, fix++ & 1u))) return;
                        const int per = (KT - b.rows) * 8;  // 16-byte pieces of a block of 64 channels
#pragma unroll 1
                        for (int hf = 0; hf < HALVES; ++hf)
#pragma unroll 1
                            for (int e = pw * 32 + lane; e < per; e += kPfCopyThreads)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                                                 ring + stage * STAGE + hf * KHALF + b.rows * 128 + e * 16),
                                             "r"(0)
                                             : "memory");
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                        expects(&sh.full[stage], 0, 32);
                    }
                };
                // by cp.async, a lane's rows of a tile: their places in 16-byte steps, or ~0 for
                // none; a bit each for those on a page out of range
                uint32_t k_off[RPL], v_off[RPL], v_next[RPL], v_lost = 0, lost_next = 0;
                auto find_rows = [&](int t) {
                    lost_next = 0;
#pragma unroll
                    for (int e = 0; e < RPL; ++e) {
                        const int p = x.tile(t) * KT + pw * RPW + 32 * e + lane;
                        k_off[e] = v_next[e] = ~0u;
                        if (p > at1) continue;
                        const int b = (int)((unsigned)p / (unsigned)ps), page = __ldg(table + b);
                        if ((unsigned)page < (unsigned)a.kv.n_pages) {
                            const unsigned r = (unsigned)p - (unsigned)b * (unsigned)ps;
                            k_off[e] = (uint32_t)((unsigned)page * kpage + r * krow);
                            v_next[e] = (uint32_t)((unsigned)page * vpage + r * vrow);
                        } else {
                            // (behind every row's window or masked, it has no part in any sum)
                            if (p >= at0 && !(MASK && __ldg(mask + p) == 0xfc00)) lost_next |= 1u << e;
                            record_status(B200_DEVSTATUS_BOUNDS);
                        }
                    }
                };
                auto copy_rows = [&](const uint8_t* base, const uint32_t (&off)[RPL]) {
                    const uint32_t dst = ring + stage * STAGE;
#pragma unroll
                    for (int e = 0; e < RPL; ++e)
#pragma unroll (D == 256 ? 8 : 16)
                        for (int j = 0; j < 32; j += RPI) {
                            const int rl = j + lane / CH, c = lane % CH, r = pw * RPW + 32 * e + rl;
                            const uint32_t o = __shfl_sync(0xffffffffu, off[e], rl);
                            pf_cp16(dst + (c >> 3) * KHALF + r * 128 + (((c & 7) ^ (r & 7)) << 4),
                                    o == ~0u ? base : base + ((uint64_t)o << 4) + c * 16, o != ~0u);
                        }
                };
                // Values on a page out of range are NaN, which no weight hides: every row of
                // the unit is computed again, and that leaves such positions out
                auto lose_rows = [&] {
                    if (!__any_sync(0xffffffffu, v_lost != 0)) return;
                    asm volatile("cp.async.wait_all;" ::: "memory");  // the zeros are written
                    __syncwarp();
#pragma unroll 1
                    for (int e = 0; e < RPL; ++e)
                        if (v_lost >> e & 1u) {
                            const uint32_t dst = ring + stage * STAGE + (pw * RPW + 32 * e + lane) * 128;
#pragma unroll 1
                            for (int c = 0; c < CH; ++c) pf_cp16(dst + (c >> 3) * KHALF + (c & 7) * 16, &kPfNan);
                        }
                };
                // the mask entries of a lane's rows
                uint16_t bias[RPL], bias_next[RPL];
                auto find_mask = [&](int t) {
                    if (MASK)
#pragma unroll
                        for (int e = 0; e < RPL; ++e) {
                            const int p = x.tile(t) * KT + pw * RPW + 32 * e + lane;
                            bias_next[e] = p <= at1 ? __ldg(mask + p) : (uint16_t)0xfc00;  // -inf
                        }
                };
                auto put_mask = [&] {
                    float m = -INFINITY;
                    const int at = tiles++ % PfShared<D>::NB;
#pragma unroll
                    for (int e = 0; e < RPL; ++e) {
                        sh.bias[at][pw * RPW + 32 * e + lane] = h2f(bias[e]);
                        m = fmaxf(m, h2f(bias[e]));
                    }
                    m = warp_max(m);
                    if (lane == 0) sh.tmax[at][pw] = m;
                };
                // (pages are looked up two tiles ahead: a look-up takes as long as a tile)
                Boxes now = find_boxes(0), next = n > 1 ? find_boxes(1) : now, before = now;
#pragma unroll 1
                for (int t = 0; t <= n && ok; ++t) {
                    if (t < n) {
                        now.on = now.on && __all_sync(0xffffffffu, (unsigned)now.page < (unsigned)a.kv.n_pages);
                        if (!now.on) find_rows(t);
                        find_mask(t);
                    }
                    if (t < n) {
                        if (!(ok = pf_wait(&sh.empty[stage], ~lap & 1u))) break;
                        if (now.on) copy_boxes(now, false);
                        else copy_rows(kb, k_off), issued(&sh.full[stage]);
                        advance();
                    }
                    const Boxes later = t + 2 < n ? find_boxes(t + 2) : next;
                    if (t > 0) {
                        if (!(ok = pf_wait(&sh.empty[stage], ~lap & 1u))) break;
                        if (MASK) put_mask();
                        if (before.on) copy_boxes(before, true);
                        else copy_rows(vb, v_off), lose_rows(), issued(&sh.full[stage]);
                        if (!ok) break;
                        advance();
                    }
                    before = now, now = next, next = later, v_lost = lost_next;
#pragma unroll
                    for (int e = 0; e < RPL; ++e) v_off[e] = v_next[e], bias[e] = bias_next[e];
                }
            }
            if (tid == 256) a.cut[2 * blockIdx.x] = cut, a.cut[2 * blockIdx.x + 1] = cut_seq;
            asm volatile("cp.async.wait_all;" ::: "memory");
            if (lane == 0) sh.filled[pw] = lap * ST + stage, sh.asked[pw] = unit, sh.fixed[pw] = fix;
            if (!ok) sh.aborted = 1;
        } else if (warp == kPfIssueWarp && lane == 0) {
            // ---- tensor-core issue
            constexpr uint32_t type = BF16 ? (1u << 7) | (1u << 10) : 0u;
            const uint32_t negate = a.scale < 0.f ? 1u << 13 : 0u;  // of q
            const uint32_t idesc_s = (1u << 4) | type | negate | ((uint32_t)(KT >> 3) << 17) | ((uint32_t)(kPfRows >> 4) << 24);
            const uint32_t idesc_o = (1u << 4) | type | (1u << 16) | ((uint32_t)(D >> 3) << 17) | ((uint32_t)(kPfRows >> 4) << 24);
            int base = 0, unit = 0;            // ring places before this unit
            uint32_t ready[2] = {0, 0};        // parities of p_ready
            bool ok = true;
            auto landed = [&](uint64_t* bar, uint32_t parity) {
                const bool there = pf_wait_one(bar, parity);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                return there;
            };
            auto stage_of = [&](int place) { return place % ST; };
            auto parity_of = [&](int place) { return (uint32_t)(place / ST) & 1u; };
            auto scores = [&](int j, uint32_t d, int stage) {
                const uint64_t da = tc_desc_sw128(q_smem + j * QTILE), db = tc_desc_sw128(ring + stage * STAGE);
#pragma unroll
                for (int k = 0; k < D / 16; ++k)
                    tc_mma_f16(d, da + (uint64_t)(((k >> 2) * QHALF + (k & 3) * 32) >> 4),
                               db + (uint64_t)(((k >> 2) * KHALF + (k & 3) * 32) >> 4), idesc_s, k > 0);
            };
            auto values = [&](uint32_t d, uint32_t p, int stage, bool add) {
                const uint64_t db = tc_desc_sw128_mn(ring + stage * STAGE, KHALF);
#pragma unroll
                for (int k = 0; k < KT / 16; ++k)
                    tc_mma_f16_ts(d, p + k * 8, db + (uint64_t)((k * 2048) >> 4), idesc_o, add || k > 0);
            };
            bool have = walk.next(a, units, total, x);
            while (ok && have) {
                const int n = x.te - x.tb;
                const bool two = NT == 2 && x.n * a.group - x.row0 > kPfRows;
                if (!(ok = landed(&sh.q_full, unit & 1))) break;
                int k_at = base;
                if (!(ok = landed(&sh.full[stage_of(k_at)], parity_of(k_at)))) break;
                tc_fence_after();
                scores(0, tmem, stage_of(k_at));
                tc_commit(&sh.s_full[0]);
                if (two) {
                    scores(1, tmem + S_STEP, stage_of(k_at));
                    tc_commit(&sh.s_full[1]);
                }
                tc_commit(&sh.empty[stage_of(k_at)]);
                if (n == 1) tc_commit(&sh.q_empty);
                have = walk.next(a, units, total, x);  // read while the scores are on their way
                for (int t = 0; t < n && ok; ++t) {
                    const bool more = t + 1 < n;
                    k_at = base + pf_k_place(t + 1);
                    const int v_at = base + pf_v_place(t, n);
                    if (more && !(ok = landed(&sh.full[stage_of(k_at)], parity_of(k_at)))) break;
                    if (NT == 1 && more) {
                        // the other score buffer: its weights went into the product before
                        tc_fence_after();
                        scores(0, tmem + ((t + 1) & 1) * S_STEP, stage_of(k_at));
                        tc_commit(&sh.s_full[(t + 1) & 1]);
                        tc_commit(&sh.empty[stage_of(k_at)]);
                        if (t + 2 == n) tc_commit(&sh.q_empty);
                    }
                    if (!(ok = landed(&sh.full[stage_of(v_at)], parity_of(v_at)))) break;
                    if (NT == 1) {
                        if (!(ok = pf_wait_one(&sh.p_ready[t & 1], ready[t & 1]))) break;
                        ready[t & 1] ^= 1u;
                        tc_fence_after();
                        values(tmem + O_COL, tmem + (t & 1) * S_STEP, stage_of(v_at), t > 0);
                        tc_commit(&sh.o_done[0]);
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            if (j == 1 && !two) break;
                            if (!(ok = pf_wait_one(&sh.p_ready[j], ready[j]))) break;
                            ready[j] ^= 1u;
                            tc_fence_after();
                            values(tmem + O_COL + j * D, tmem + j * S_STEP, stage_of(v_at), t > 0);
                            tc_commit(&sh.o_done[j]);
                            if (more) {
                                scores(j, tmem + j * S_STEP, stage_of(k_at));
                                tc_commit(&sh.s_full[j]);
                            }
                        }
                        if (!ok) break;
                        if (more) tc_commit(&sh.empty[stage_of(k_at)]);
                        if (t + 2 == n) tc_commit(&sh.q_empty);
                    }
                    tc_commit(&sh.empty[stage_of(v_at)]);
                }
                base += 2 * n;
                ++unit;
            }
            if (!ok) sh.aborted = 1;
        }
        __syncwarp();
    } else {
        // ---- softmax: a row to a thread
        asm volatile("setmaxnreg.inc.sync.aligned.u32 200;");
        const int j = role;
        const uint32_t lanes = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t o_addr = tmem + lanes + O_COL + (NT == 2 ? j * D : 0);
        const int row = (warp & 3) * 32 + lane;
        const float scale2 = fmaxf(fabsf(a.scale) * 1.4426950408889634f, 1.17549435e-38f);
        int base = 0;  // places before the unit
        uint32_t s_par[2] = {0, 0}, o_par = 0;  // o_par: products into this tile's outputs so far
        bool ok = j < NT;
        while (ok && walk.next(a, units, total, x)) {
            const int n = x.te - x.tb, count = x.n * a.group;
            if (j * kPfRows >= count - x.row0) {  // no rows for this tile
                base += 2 * n;
                continue;
            }
            const int flat = x.row0 + j * kPfRows + row;
            const bool real = flat < count, any = x.row0 + j * kPfRows + (warp & 3) * 32 < count;
            const int i = flat / a.group;
            const int at = real ? max(-1, x.len - x.n + i) : -1;
            float ref = -INFINITY, l = 0.f, c_ref = -INFINITY;
            for (int t = 0; t < n; ++t) {
                const int sb = NT == 2 ? j : (t & 1);
                const uint32_t s_addr = tmem + lanes + sb * S_STEP;
                if (!(ok = pf_wait(&sh.s_full[sb], s_par[sb]))) break;
                s_par[sb] ^= 1u;
                const int v_at = base + pf_v_place(t, n), v_stage = v_at % ST;
                if (MASK && !(ok = pf_wait(&sh.full[v_stage], (uint32_t)(v_at / ST) & 1u))) break;
                tc_fence_after();
                if (any) {
                    // columns lo .. hi are seen
                    const int p0 = x.tile(t) * KT;
                    const int hi = at - p0, lo = a.window > 0 ? max(0, at - a.window + 1) - p0 : 0;
                    const bool edge = __any_sync(0xffffffffu, hi < KT - 1 || lo > 0);
                    const int v_bias = (base / 2 + t) % PfShared<D>::NB;
                    const float4* entries = reinterpret_cast<const float4*>(sh.bias[v_bias]);
                    float c0 = 0.f;
                    if (MASK) {
                        float cm;
                        if (edge) {
                            cm = -INFINITY;
#pragma unroll 2
                            for (int c = 0; c < KT; c += 32) {
                                const uint32_t seen = pf_bits(lo - c, hi - c);
#pragma unroll
                                for (int e = 0; e < 32; e += 4) {
                                    const float4 w = entries[(c + e) / 4];
                                    cm = fmaxf(cm, seen & (1u << e) ? w.x : -INFINITY);
                                    cm = fmaxf(cm, seen & (2u << e) ? w.y : -INFINITY);
                                    cm = fmaxf(cm, seen & (4u << e) ? w.z : -INFINITY);
                                    cm = fmaxf(cm, seen & (8u << e) ? w.w : -INFINITY);
                                }
                            }
                        } else {
                            cm = fmaxf(sh.tmax[v_bias][0], sh.tmax[v_bias][1]);
                        }
                        // the mask relative to the largest entry that the row has seen:
                        // a row of lowest values keeps its scores' bits
                        if (cm > c_ref) {
                            ref += (c_ref - cm) * 1.4426950408889634f;
                            c_ref = cm;
                        }
                        c0 = c_ref == -INFINITY ? 0.f : c_ref;
                    }
                    const uint64_t scale22 = f2_pair(scale2, scale2), minus = f2_pair(-c0, -c0);
                    const uint64_t log2e2 = f2_pair(1.4426950408889634f, 1.4426950408889634f);
                    // 32 scores as loaded: with a mask times scale2 and the entries added,
                    // -inf where the row does not see
                    auto ready = [&](uint32_t (&s)[32], int c) {
                        if (MASK) {
#pragma unroll
                            for (int k = 0; k < 32; k += 4) {
                                const float4 w = entries[(c + k) / 4];
                                const uint64_t w0 = f2_mul(f2_add(f2_pair(w.x, w.y), minus), log2e2);
                                const uint64_t w1 = f2_mul(f2_add(f2_pair(w.z, w.w), minus), log2e2);
                                const float2 y0 = f2_unpair(f2_fma(
                                    f2_pair(__uint_as_float(s[k]), __uint_as_float(s[k + 1])), scale22, w0));
                                const float2 y1 = f2_unpair(f2_fma(
                                    f2_pair(__uint_as_float(s[k + 2]), __uint_as_float(s[k + 3])), scale22, w1));
                                s[k] = __float_as_uint(y0.x), s[k + 1] = __float_as_uint(y0.y);
                                s[k + 2] = __float_as_uint(y1.x), s[k + 3] = __float_as_uint(y1.y);
                            }
                        }
                        if (edge) {
                            const uint32_t seen = pf_bits(lo - c, hi - c);
#pragma unroll
                            for (int e = 0; e < 32; ++e) s[e] = seen & (1u << e) ? s[e] : 0xff800000u;
                        }
                    };
                    // the row's scores in registers: a load of tensor memory takes longer
                    // than all that is done with 32 of them
                    uint32_t s[KT / 32][32];
                    float m[2] = {-INFINITY, -INFINITY};
#pragma unroll
                    for (int c = 0; c < KT / 32; ++c) tc_ld_x32(s[c], s_addr + 32 * c);
                    tc_wait_ld();
#pragma unroll
                    for (int c = 0; c < KT / 32; ++c) {
                        tc_loaded(s[c]);
                        ready(s[c], 32 * c);
#pragma unroll
                        for (int e = 0; e < 32; e += 4) {
                            m[0] = f_max3(m[0], __uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
                            m[1] = f_max3(m[1], __uint_as_float(s[c][e + 2]), __uint_as_float(s[c][e + 3]));
                        }
                    }
                    float top = fmaxf(m[0], m[1]);
                    if (!MASK) top *= scale2;
                    const bool moves = top > ref + kPfLazy;
                    if (__any_sync(0xffffffffu, moves)) {
                        const float f = moves ? pf_exp2(ref - top) : 1.f;
                        l *= f;
                        if (moves) ref = top;
                        if (t > 0) {
                            if (!(ok = pf_wait(&sh.o_done[j], (o_par + 1u) & 1u))) break;
                            tc_fence_after();
#pragma unroll 1
                            for (int c = 0; c < D; c += 32) {
                                uint32_t o[32];
                                tc_ld_x32(o, o_addr + c);
                                tc_wait_ld();
                                tc_loaded(o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
                                tc_st_x32(o_addr + c, o);
                            }
                        }
                    }
                    const float off = (ref == -INFINITY ? 0.f : -ref) + kPfShift<BF16>;
                    const uint64_t off2 = f2_pair(off, off);
                    uint64_t sum = f2_pair(0.f, 0.f);
#pragma unroll
                    for (int c = 0; c < KT / 32; ++c) {
                        uint32_t p[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            const uint64_t y = f2_pair(__uint_as_float(s[c][e]), __uint_as_float(s[c][e + 1]));
                            const float2 z = f2_unpair(MASK ? f2_add(y, off2) : f2_fma(y, scale22, off2));
                            const float e0 = pf_exp2(z.x), e1 = pf_exp2(z.y);
                            sum = f2_add(sum, f2_pair(e0, e1));
                            p[e / 2] = pack16<BF16>(e0, e1);
                        }
                        // (over the scores, which are all in registers)
                        tc_st_x16(s_addr + 16 * c, p);
                    }
                    const float2 both = f2_unpair(sum);
                    l += both.x + both.y;
                    tc_wait_st();
                }
                // (one score buffer: the scores came after the product before.  Two: the parity
                // of o_done says which product ended only if none is passed over)
                if (NT == 1 && t > 0 && !(ok = pf_wait(&sh.o_done[0], (o_par + 1u) & 1u))) break;
                ++o_par;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) pf_arrive(&sh.p_ready[sb]);
            }
            if (!ok) break;
            base += 2 * n;
            // ---- the unit's outputs, or this CTA's piece of them
            if (!(ok = pf_wait(&sh.o_done[j], (o_par + 1u) & 1u))) break;
            tc_fence_after();
            if (!any) continue;
            const int64_t out_row = (int64_t)(x.first + i) * a.n_head + x.h * a.group + (flat - i * a.group);
            bool again;
            if (n == x.cost) {
                float odd = l * 0.f;  // NaN where anything is not finite
                const float inv = l == 0.f ? 0.f : 1.f / l;
                uint4* to = reinterpret_cast<uint4*>(a.out + out_row * D);
#pragma unroll 1
                for (int c = 0; c < D; c += 64) {
                    uint32_t o[2][32];
                    tc_ld_x32(o[0], o_addr + c);
                    tc_ld_x32(o[1], o_addr + c + 32);
                    tc_wait_ld();
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        tc_loaded(o[b]);
                        uint32_t w[16];
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float y0 = __uint_as_float(o[b][2 * e]), y1 = __uint_as_float(o[b][2 * e + 1]);
                            odd = fmaf(y0, 0.f, fmaf(y1, 0.f, odd));
                            w[e] = l == 0.f ? 0u : pack16<BF16>(y0 * inv, y1 * inv);
                        }
                        if (real)
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                to[c / 8 + 4 * b + e] = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
                    }
                }
                again = real && l != 0.f && odd != 0.f;
            } else {
                // at most one unit goes on from the CTA before, and one goes on in the next
                const int slot = 2 * blockIdx.x + (x.tb > 0 ? 0 : 1);
                float4* ml = a.piece_ml + ((int64_t)slot * NT + j) * kPfRows + row;
                float4* po = a.piece_o + ((int64_t)slot * NT + j) * (D / 4) * kPfRows + row;
                if (real) *ml = make_float4(ref, l, c_ref, 0.f);
                const uint64_t none = f2_pair(0.f, 0.f);
                uint64_t zero = none;  // NaN where anything is not finite
#pragma unroll 1
                for (int c = 0; c < D; c += 64) {
                    uint32_t o[2][32];
                    tc_ld_x32(o[0], o_addr + c);
                    tc_ld_x32(o[1], o_addr + c + 32);
                    tc_wait_ld();
#pragma unroll
                    for (int b = 0; b < 2; ++b) {
                        tc_loaded(o[b]);
#pragma unroll
                        for (int e = 0; e < 32; e += 2)
                            zero = f2_fma(f2_pair(__uint_as_float(o[b][e]), __uint_as_float(o[b][e + 1])), none, zero);
                        if (real)
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                po[(c / 4 + 8 * b + e) * kPfRows] =
                                    make_float4(__uint_as_float(o[b][4 * e]), __uint_as_float(o[b][4 * e + 1]),
                                                __uint_as_float(o[b][4 * e + 2]), __uint_as_float(o[b][4 * e + 3]));
                    }
                }
                const float2 odd = f2_unpair(zero);
                again = real && l * 0.f + odd.x + odd.y != 0.f;
            }
            unsigned votes = __ballot_sync(0xffffffffu, again);
            if (votes) {
                int at_list = 0;
                if (lane == 0) {
                    // (the CTA where the unit's first key tile is: one of its pieces lists the row)
                    if (n != x.cost)
                        votes &= ~atomicOr(a.claim + (walk.w - x.cost) / per_cta * 8 + j * 4 + (warp & 3), votes);
                    at_list = atomicAdd(&a.header->n_bad, __popc(votes));
                }
                votes = __shfl_sync(0xffffffffu, votes, 0);
                at_list = __shfl_sync(0xffffffffu, at_list, 0) + __popc(votes & ((1u << lane) - 1u));
                if ((votes >> lane & 1u) && at_list < a.n_tokens * a.n_head) a.bad[at_list] = make_int2((int)out_row, x.u);
            }
            tc_fence_before();
        }
        if (!ok && j < NT) sh.aborted = 1;
    }
    tc_fence_before();
    __syncthreads();  // every loop is over
    if (tid == 256 && sh.aborted) {
        // A wait ran out (recorded; the outputs are not what they should be): TMA copies
        // that nobody waited for must land before the CTA's shared memory is another's.
        pf_land(sh.full, {{sh.filled[0], sh.filled[1]}, (uint32_t)ST}, 32 + (MASK ? 1 : 0));
        pf_land(&sh.q_full, {{sh.asked[0], sh.asked[1]}, 1u}, 32);
        pf_land(&sh.fix, {{sh.fixed[0], sh.fixed[1]}, 1u}, 1);
    }
    if (tid == kPfIssueWarp * 32) tc_commit(&sh.done);  // every product issued has ended
    if (warp == kPfIssueWarp) {
        mbar_wait_drain(&sh.done, 0);
        tc_fence_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
    }
}

// ----------------------------------------------------------------- finish

// CTA (CTA of the main kernel, 32 rows): the pieces of the unit that begins in that
// one's range and goes on past it, joined in order.  Then the rows that infinities or NaN
// met, and which no product of whole tiles can tell apart from positions they do not see:
// a CTA to a row.
template <bool BF16, int D>
__global__ void __launch_bounds__(kPfFinishThreads) paged_prefill_finish_kernel(const __grid_constant__ PagedPrefillArgs a) {
    constexpr int NT = pf_tiles(D), W = kPfFinishThreads / 32, CPW = D / 4 / W;  // float4 columns to a warp
    __shared__ int s_odd[W][32];
    __shared__ PfAgain<D> s_again;
    griddep_wait();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int4 cut = a.cut[2 * blockIdx.y], d1 = a.cut[2 * blockIdx.y + 1];
    const int n_bad = min(a.header->n_bad, a.n_tokens * a.n_head);
    if (cut.w > 0) {
        const int h = cut.y, c0 = blockIdx.y, pieces = cut.w;
        const int r0 = blockIdx.x * 32, j = r0 / kPfRows, row = (r0 & (kPfRows - 1)) + lane;
        const int flat = cut.z + r0 + lane;
        const bool real = flat < d1.y * a.group;
        const unsigned listed = a.claim[c0 * 8 + r0 / 32];  // rows that a piece has listed are not joined
        if (cut.z + r0 < d1.y * a.group) {
            // piece k: the last of CTA c0's range, then the first of each one's
            auto slot = [&](int k) { return (int64_t)(2 * (c0 + k) + (k == 0 ? 1 : 0)) * NT + j; };
            float cm = -INFINITY, top = -INFINITY, l = 0.f;
            float4 o[CPW];
#pragma unroll
            for (int e = 0; e < CPW; ++e) o[e] = make_float4(0.f, 0.f, 0.f, 0.f);
            constexpr int AT_ONCE = D == 256 ? 2 : 4;
            for (int k0 = 0; k0 < pieces && real; k0 += AT_ONCE) {
                float4 ml[AT_ONCE], y[AT_ONCE][CPW];
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) {
                    if (k0 + k >= pieces) continue;
                    const int64_t at = slot(k0 + k);
                    ml[k] = a.piece_ml[at * kPfRows + row];
                    const float4* po = a.piece_o + (at * (D / 4) + warp * CPW) * kPfRows + row;
#pragma unroll
                    for (int e = 0; e < CPW; ++e) y[k][e] = po[e * kPfRows];
                }
#pragma unroll
                for (int k = 0; k < AT_ONCE; ++k) {
                    if (k0 + k >= pieces) continue;
                    float ref = ml[k].x;
                    if (a.mask) {  // relative to the largest mask entry so far
                        if (ml[k].z > cm) {
                            top += (cm - ml[k].z) * 1.4426950408889634f;
                            cm = ml[k].z;
                        } else if (ml[k].z < cm) {
                            ref += (ml[k].z - cm) * 1.4426950408889634f;
                        }
                    }
                    const float now = fmaxf(top, ref), base = now == -INFINITY ? 0.f : now;
                    const float fo = pf_exp2(top - base), f = pf_exp2(ref - base);
                    l = fo * l + f * ml[k].y;
                    top = now;
#pragma unroll
                    for (int e = 0; e < CPW; ++e) {
                        o[e].x = fo * o[e].x + f * y[k][e].x, o[e].y = fo * o[e].y + f * y[k][e].y;
                        o[e].z = fo * o[e].z + f * y[k][e].z, o[e].w = fo * o[e].w + f * y[k][e].w;
                    }
                }
            }
            const float inv = l == 0.f ? 0.f : 1.f / l;
            const int i = flat / a.group, g = flat - i * a.group;
            const int64_t out_row = (int64_t)(d1.x + i) * a.n_head + h * a.group + g;
            float odd = l * 0.f;
            uint32_t w[2 * CPW];
#pragma unroll
            for (int e = 0; e < CPW; ++e) {
                odd += o[e].x * 0.f + o[e].y * 0.f + o[e].z * 0.f + o[e].w * 0.f;
                w[2 * e] = l == 0.f ? 0u : pack16<BF16>(o[e].x * inv, o[e].y * inv);
                w[2 * e + 1] = l == 0.f ? 0u : pack16<BF16>(o[e].z * inv, o[e].w * inv);
            }
            const bool mine = real && !(listed >> lane & 1u);
            if (mine) {
                uint2* to = reinterpret_cast<uint2*>(a.out + out_row * D) + warp * CPW;
#pragma unroll
                for (int e = 0; e < CPW; ++e) to[e] = make_uint2(w[2 * e], w[2 * e + 1]);
            }
            s_odd[warp][lane] = mine && l != 0.f && odd != 0.f;
            __syncthreads();
            bool again = false;
#pragma unroll
            for (int v = 0; v < W; ++v) again |= s_odd[v][lane] != 0;
            unsigned votes = __ballot_sync(0xffffffffu, again);
            for (; votes; votes &= votes - 1) {  // finite pieces whose sum is not
                const int r = cut.z + r0 + __ffs(votes) - 1, i1 = r / a.group;
                pf_row<BF16, D>(a, s_again, cut.x, d1.y, d1.z, d1.x + i1, i1, h * a.group + r - i1 * a.group);
            }
        }
    }
    const int cta = blockIdx.y * gridDim.x + blockIdx.x, ctas = gridDim.x * gridDim.y;
    for (int64_t b = cta; b < n_bad; b += ctas) {
        const int2 e = a.bad[b];
        const int4 d0 = a.desc[2 * (int64_t)e.y], d1 = a.desc[2 * (int64_t)e.y + 1];
        const int t = e.x / a.n_head;
        pf_row<BF16, D>(a, s_again, d0.x, d1.y, d1.z, t, t - d1.x, e.x - t * a.n_head);
    }
}

}  // namespace b200
