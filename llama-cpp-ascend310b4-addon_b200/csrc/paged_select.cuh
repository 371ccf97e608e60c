// paged_select.cuh -- block selection for sparse attention: an upper bound of
// q . k per block from the page's key bounds, and the n_sel best blocks.
//
// The order of the scores is decided in 64 bits: f32 sums of 64 to 256
// products are off by some 1e-6 of a score, and with thousands of blocks per
// head the scores around the last place of the selection lie that close
// together, so 32 bits would pick blocks by rounding.  But only the few
// blocks around that place need 64 bits.  The first kernel reads all bounds
// once and finds every score to within a proven eps on the tensor cores; the
// second finds the need-th largest of those, tau.  The exact need-th largest
// score is within eps of tau, so a block above tau + 2 eps is chosen and one
// below tau - 2 eps is not, whatever the rounding; the blocks in between
// (three or so of 2048) are scored again in 64 bits and ranked.
//
// max(q lo, q hi) summed over d is  q+ . hi + q- . lo  with q+ = max(q, 0),
// q- = min(q, 0): two matrix products per block, with the operands of the
// attention kernel (heads x dims against rows of pages), reading 4 D bytes
// per block and KV head: bound by memory.  All in 64 bits it would be bound by
// the f64 pipe and the selects that feed it.
#pragma once

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"
#include "paged_attn.cuh"
#include "paged_work.cuh"

namespace b200 {

struct PagedSelectArgs {
    const uint16_t *lo, *hi;
    const float* q;
    int64_t q_stride;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_lens;
    int32_t* sel;
    unsigned long long* exact;  // [n_seq][n_head_kv][max_blocks] ordered 64-bit scores, where needed
    float* approx;              // [n_seq][n_head_kv][max_blocks] scores of q 2^-ex
    unsigned int* unit_max;     // [n_seq][n_head_kv][ceil(max_blocks / 16)] largest |bound|, as 16-bit patterns
    int n_seq, n_head, n_head_kv, max_blocks, page_size, n_pages, n_sel;
};

B200_HD constexpr int paged_units(int blocks) { return (blocks + kPaTok - 1) / kPaTok; }

// Exponent of the largest |q| of a KV head's query heads (n contiguous values,
// a multiple of 32), clamped as in the attention kernel; one warp.
__device__ __forceinline__ int group_exponent(const float* q, int n) {
    float m = 0.f;
    for (int i = threadIdx.x & 31; i < n; i += 32) m = fmaxf(m, fabsf(q[i]));
    m = pa_warp_max(m);
    return min(max((int)(__float_as_uint(m) >> 23) - 127, -120), 120);
}

template <int W, int S>
struct ScoreShared {
    PaRangeShared<W> range;
    unsigned valid[W][S];
};
template <int D>
constexpr int score_smem() {
    return pa_warps(D) * pa_stages(D) * 2 * pa_tile(D) + (int)sizeof(ScoreShared<pa_warps(D), pa_stages(D)>);
}

// Units of 16 blocks of one (sequence, KV head), streamed as in the attention
// kernel: equal ranges per warp, private cp.async rings.
template <bool BF16, int D>
__global__ void __launch_bounds__(32 * pa_warps(D), 1) paged_score_kernel(PagedSelectArgs a) {
    constexpr int W = pa_warps(D), S = pa_stages(D);
    constexpr int KT = D / 16, LPR = D / 8, RPI = 32 / LPR, TILE = pa_tile(D), RB = 2 * D;
    extern __shared__ __align__(128) uint8_t pa_sm[];
    ScoreShared<W, S>& sh = *reinterpret_cast<ScoreShared<W, S>*>(pa_sm + W * S * 2 * TILE);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t4 = lane & 3;
    const int G = a.n_head / a.n_head_kv, H = a.n_head_kv;
    const int max_units = paged_units(a.max_blocks);

    // blocks to score: none where every block is taken, or only the newest
    auto blocks = [&](int s) {
        const int nb = paged_blocks(a.seq_lens[s], a.max_blocks, a.page_size);
        return nb <= a.n_sel || a.n_sel == 1 ? 0 : nb;
    };
    const PaRange<W> range(sh.range, a.n_seq, H, [&](int s) { return paged_units(blocks(s)); });
    if (range.fb >= range.fe) return;

    const uint32_t ring = smem_u32(pa_sm) + warp * (S * 2 * TILE);
    struct Cursor {
        int s, head, u, nu, nb;
    } in, cur;
    in.s = range.seq0;
    in.nb = blocks(in.s);
    in.nu = paged_units(in.nb);
    in.head = (range.fb - range.base0) / in.nu;
    in.u = (range.fb - range.base0) - in.head * in.nu;
    cur = in;
    auto advance = [&](Cursor& c) -> bool {
        if (++c.u < c.nu) return true;
        c.u = 0;
        if (++c.head < H) return true;
        c.head = 0;
        do {
            if (++c.s >= a.n_seq) return false;
            c.nb = blocks(c.s);
            c.nu = paged_units(c.nb);
        } while (c.nu == 0);
        return true;
    };
    int to_issue = range.fe - range.fb, to_do = to_issue;

    // producer: lane & 15 looks after one block of the unit; the pages of the
    // unit after it are on their way
    auto page_of = [&](const Cursor& c) -> int {
        const int b = kPaTok * c.u + (lane & 15);
        return b < c.nb ? a.table[c.s * a.table_stride + b] : -1;
    };
    int page_next = page_of(in);
    auto issue = [&](int stage) {
        if (to_issue > 0) {
            const int page = page_next, head = in.head;
            const bool ok = (unsigned)page < (unsigned)a.n_pages;
            if (!ok && kPaTok * in.u + (lane & 15) < in.nb) record_status(B200_DEVSTATUS_BOUNDS);
            --to_issue;
            if (to_issue > 0) {
                if (advance(in)) page_next = page_of(in);
                else to_issue = 0;
            }
            const unsigned valid = __ballot_sync(0xffffffffu, ok) & 0xffffu;
            if (lane == 0) sh.valid[warp][stage] = valid;
            const uint32_t st = ring + stage * (2 * TILE), c = lane % LPR;
#pragma unroll
            for (int i = 0; i < kPaTok / RPI; ++i) {
                const int r = i * RPI + lane / LPR;
                const bool on = (valid >> r) & 1;
                const int p = __shfl_sync(0xffffffffu, page, r);
                const int64_t at = on ? ((int64_t)p * H + head) * D + 8 * c : 0;
                const uint32_t d = st + r * RB + ((c ^ (r & 7)) << 4);
                pa_cp16(d, a.hi + at, on);
                pa_cp16(d + TILE, a.lo + at, on);
            }
        }
        pa_commit();
    };

    // consumer
    uint32_t qf[KT][4], q3[BF16 ? KT : 1][2], plus[KT][2];  // plus: all ones where q > 0
    bool new_q = true;
    int stage = 0, ahead = 0;
    float up = 1.f;
    const int mi = lane >> 3, ri = lane & 7;
#pragma unroll 1
    for (int turn = 1 - S; to_do > 0; ++turn) {
        if (turn >= 0) {
            pa_wait<S - 2>();
            __syncwarp();
        }
        issue(ahead);
        ahead = ahead + 1 == S ? 0 : ahead + 1;
        if (turn < 0) continue;
        const float* qg = a.q + cur.s * a.q_stride + (int64_t)cur.head * G * D;
        if (new_q) up = __uint_as_float((unsigned)(127 - group_exponent(qg, G * D)) << 23);
        const uint32_t hst = ring + stage * (2 * TILE), lst = hst + TILE;
        float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        unsigned top = 0;
#pragma unroll 1
        for (int j0 = 0; j0 < G; j0 += kPaHeads) {
            if (new_q || G > kPaHeads) {
                const int j = min(j0 + g, G - 1);  // rows past the group repeat its last head
                const float* qr = qg + j * D + 2 * t4;
#pragma unroll
                for (int i = 0; i < 2 * KT; ++i) {
                    const float2 v = *reinterpret_cast<const float2*>(qr + 8 * i);
                    float x = v.x * up, y = v.y * up;
                    plus[i >> 1][i & 1] = (x > 0.f ? 0xffffu : 0u) | (y > 0.f ? 0xffff0000u : 0u);
                    qf[i >> 1][2 * (i & 1)] = pa_split<BF16>(x, y);
                    qf[i >> 1][2 * (i & 1) + 1] = pa_split<BF16>(x, y);
                    if (BF16) q3[i >> 1][i & 1] = pa_split<BF16>(x, y);
                }
            }
            float sc[2][4] = {};
#pragma unroll
            for (int half = 0; half < 2; ++half) {  // q+ with hi, then q- with lo
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    uint32_t b[4];
                    const int r = 8 * (mi >> 1) + ri, c = 2 * kt + (mi & 1);
                    pa_ldsm(b, (half ? lst : hst) + r * RB + ((c ^ ri) << 4));
#pragma unroll
                    for (int i = 0; i < 4; ++i) top = __vmaxu2(top, b[i] & 0x7fff7fffu);
                    const uint32_t m0 = half ? ~plus[kt][0] : plus[kt][0], m1 = half ? ~plus[kt][1] : plus[kt][1];
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        pa_mma<BF16>(sc[n], qf[kt][0] & m0, qf[kt][1] & m0, qf[kt][2] & m1, qf[kt][3] & m1, b[2 * n],
                                     b[2 * n + 1]);
                        if (BF16) pa_mma<BF16>(sc[n], q3[kt][0] & m0, 0u, q3[kt][1] & m1, 0u, b[2 * n], b[2 * n + 1]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) best[i] = fmaxf(best[i], sc[i >> 1][i & 1] + sc[i >> 1][2 + (i & 1)]);
        }
        const unsigned valid = sh.valid[warp][stage];
        // the largest over the heads, which are 8 lanes; then lanes 0-3 hold the unit
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], o));
        top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
        const int64_t sh_ = (int64_t)cur.s * H + cur.head;
        if (lane < 4) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int r = 8 * (i >> 1) + 2 * t4 + (i & 1), b = kPaTok * cur.u + r;
                if (b < cur.nb) a.approx[sh_ * a.max_blocks + b] = (valid >> r) & 1 ? best[i] : -INFINITY;
            }
        }
        if (lane == 0) a.unit_max[sh_ * max_units + cur.u] = top;
        stage = stage + 1 == S ? 0 : stage + 1;
        if (--to_do > 0) {
            new_q = cur.u + 1 == cur.nu;
            if (!advance(cur)) break;
        }
    }
    pa_wait<0>();
}

// Order-preserving keys; NaN below everything.
__device__ __forceinline__ unsigned long long order_key(double x) {
    if (x != x) return 0ull;
    const long long b = __double_as_longlong(x + 0.0);  // -0 -> +0
    return b < 0 ? ~(unsigned long long)b : (unsigned long long)b | 0x8000000000000000ull;
}
__device__ __forceinline__ unsigned order_key(float x) {
    const unsigned b = __float_as_uint(x);
    return b >> 31 ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float from_order_key(unsigned k) {
    return __uint_as_float(k >> 31 ? k & 0x7fffffffu : ~k);
}

// One warp: the 64-bit score of block b, every lane.
template <bool BF16, int D>
__device__ __forceinline__ unsigned long long exact_score(const PagedSelectArgs& a, int s, int h, int b) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31, G = a.n_head / a.n_head_kv;
    const int page = a.table[s * a.table_stride + b];
    if ((unsigned)page >= (unsigned)a.n_pages) return 0ull;
    const int64_t at = ((int64_t)page * a.n_head_kv + h) * D + lane * E;
    float lo[E], hi[E];
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const float2 l = unpack16<BF16>(*reinterpret_cast<const uint32_t*>(a.lo + at + e));
        const float2 u = unpack16<BF16>(*reinterpret_cast<const uint32_t*>(a.hi + at + e));
        lo[e] = l.x, lo[e + 1] = l.y, hi[e] = u.x, hi[e + 1] = u.y;
    }
    double best = -INFINITY;
    bool nan = false;
    for (int j = 0; j < G; ++j) {
        const float* q = a.q + s * a.q_stride + (int64_t)(h * G + j) * D + lane * E;
        double x = 0.0;
#pragma unroll
        for (int e = 0; e < E; ++e) x += fmax((double)q[e] * lo[e], (double)q[e] * hi[e]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
        nan |= x != x;
        best = fmax(best, x);
    }
    return nan ? 0ull : order_key(best);
}

constexpr int kTopkThreads = 512;
constexpr int kTopkKeys = 24576;  // scores kept in shared memory
constexpr int kTopkBand = 256;    // undecided blocks ranked in shared memory

// One CTA per (sequence, KV head).
template <bool BF16, int D>
__global__ void __launch_bounds__(kTopkThreads) paged_topk_kernel(PagedSelectArgs a) {
    constexpr int T = kTopkThreads, W = T / 32;
    extern __shared__ __align__(16) float topk_keys[];
    __shared__ int count[64];
    __shared__ int band[kTopkBand], chosen[kTopkBand];
    __shared__ unsigned long long band_key[kTopkBand];
    __shared__ int n_band, s_ties;
    __shared__ unsigned s_max;
    __shared__ float s_sum[W];
    __shared__ int wsum[2][W];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int sh_ = blockIdx.x, s = sh_ / a.n_head_kv, h = sh_ - s * a.n_head_kv;
    const int G = a.n_head / a.n_head_kv;
    griddep_wait();  // the scores
    const int len = a.seq_lens[s];
    const int nb = paged_blocks(len, a.max_blocks, a.page_size);
    if (tid == 0 && h == 0 && (len < 0 || len > (int64_t)a.max_blocks * a.page_size)) record_status(B200_DEVSTATUS_BOUNDS);
    int32_t* out = a.sel + (int64_t)sh_ * a.n_sel;
    if (nb <= a.n_sel) {
        for (int i = tid; i < a.n_sel; i += T) out[i] = i < nb ? i : -1;
        return;
    }
    const int m = nb - 1, need = a.n_sel - 1;  // `need` of the m older blocks
    if (need == 0) {
        if (tid == 0) out[0] = m;
        return;
    }
    const float* score = a.approx + (int64_t)sh_ * a.max_blocks;
    if (m <= kTopkKeys) {
        for (int i = tid; i < m; i += T) topk_keys[i] = score[i];
        score = topk_keys;
    }
    if (tid < 64) count[tid] = 0;
    if (tid == 0) n_band = 0, s_ties = 0, s_max = 0;
    // eps, with S = max_j sum |q'_jd| * max |bound| and q' = q 2^-ex, whose
    // largest entry is in [1, 2): the parts of q' leave out at most 2^-23 each, in
    // all D 2^-23 S; D / 8 instructions (bf16: D / 4) each truncate 17 terms
    // below 2^-24 S, in all 17 D 2^-27 S (bf16: twice that).  D 2^-21 S (bf16:
    // twice that) covers both, 1e-30 what underflows.
    const float* qg = a.q + s * a.q_stride + (int64_t)h * G * D;
    const float up = __uint_as_float((unsigned)(127 - group_exponent(qg, G * D)) << 23);
    float qs = 0.f;
    for (int j = warp; j < G; j += W) {
        float x = 0.f;
        for (int d = lane; d < D; d += 32) x += fabsf(qg[j * D + d] * up);
        x = warp_sum(x);
        qs = x > qs || x != x ? x : qs;  // NaN stays
    }
    __syncthreads();
    if (lane == 0) s_sum[warp] = qs;
    {
        const int nu = paged_units(nb);
        unsigned top = 0;
        for (int i = tid; i < nu; i += T) top = max(top, a.unit_max[(int64_t)sh_ * paged_units(a.max_blocks) + i]);
        top = __reduce_max_sync(0xffffffffu, top);
        if (lane == 0) atomicMax(&s_max, top);
    }
    __syncthreads();
#pragma unroll
    for (int w = 0; w < W; ++w) qs = s_sum[w] > qs || s_sum[w] != s_sum[w] ? s_sum[w] : qs;
    const float biggest = BF16 ? __uint_as_float(s_max << 16) : h2f((uint16_t)s_max);
    const float eps = qs * biggest * ((BF16 ? 2.f : 1.f) * D * 4.76837158e-7f) * 1.001f + 1e-30f;

    // tau: the need-th largest score, bit by bit from the top; with exactly
    // `need` scores at or above the trial it is the smallest of those
    unsigned tau_key = 0;
    bool sure = eps < 1e30f;  // false: bounds or queries that are not finite, nothing is decided by the scores
    if (sure) {
        int bit = 31;
        for (; bit >= 0; --bit) {
            const unsigned trial = tau_key | 1u << bit;
            int c = 0;
            for (int i = tid; i < m; i += T) c += order_key(score[i]) >= trial;
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0 && c) atomicAdd(&count[bit], c);
            __syncthreads();
            c = count[bit];
            if (c >= need) tau_key = trial;
            if (c == need) break;
        }
        if (bit >= 0) {
            unsigned low = 0xffffffffu;
            for (int i = tid; i < m; i += T) {
                const unsigned k = order_key(score[i]);
                if (k >= tau_key) low = min(low, k);
            }
            low = __reduce_min_sync(0xffffffffu, low);
            if (tid == 0) s_max = 0xffffffffu;
            __syncthreads();
            if (lane == 0) atomicMin(&s_max, low);
            __syncthreads();
            tau_key = s_max;
        }
    }
    const float tau = sure ? from_order_key(tau_key) : 0.f;
    const float above = sure ? tau + 2.01f * eps : INFINITY, below = sure ? tau - 2.01f * eps : -INFINITY;
    // in: score > above; undecided: [below, above]
    auto undecided = [&](float x) { return !sure || (x >= below && x <= above); };
    int n_in = 0;
    for (int i = tid; i < m; i += T) {
        const float x = score[i];
        if (undecided(x)) {
            const int k = atomicAdd(&n_band, 1);
            if (k < kTopkBand) band[k] = i;
        } else if (x > above) {
            ++n_in;
        }
    }
    n_in = __reduce_add_sync(0xffffffffu, n_in);
    if (lane == 0 && n_in) atomicAdd(&count[32], n_in);
    __syncthreads();
    const int nbnd = n_band, left = need - count[32];  // `left` of the nbnd undecided blocks
    const bool small = nbnd <= kTopkBand;
    unsigned long long cut = 0;  // large bands: the smallest 64-bit key chosen, `ties` of its equals
    int ties = 0;
    if (left == nbnd) {
        // all of them
    } else if (small) {
        for (int k = warp; k < nbnd; k += W) {
            const unsigned long long key = exact_score<BF16, D>(a, s, h, band[k]);
            if (lane == 0) band_key[k] = key;
        }
        __syncthreads();
        for (int k = tid; k < nbnd; k += T) {
            int rank = 0;
            for (int x = 0; x < nbnd; ++x)
                rank += band_key[x] > band_key[k] || (band_key[x] == band_key[k] && band[x] < band[k]);
            chosen[k] = rank < left;
        }
        __syncthreads();
    } else {
        unsigned long long* exact = a.exact + (int64_t)sh_ * a.max_blocks;
        for (int i = warp; i < m; i += W) {
            if (!undecided(score[i])) continue;
            const unsigned long long key = exact_score<BF16, D>(a, s, h, i);
            if (lane == 0) exact[i] = key;
        }
        __syncthreads();
        if (tid < 64) count[tid] = 0;
        __syncthreads();
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long trial = cut | 1ull << bit;
            int c = 0;
            for (int i = tid; i < m; i += T) c += undecided(score[i]) && exact[i] >= trial;
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0 && c) atomicAdd(&count[bit], c);
            __syncthreads();
            if (count[bit] >= left) cut = trial;
        }
        int c = 0;
        for (int i = tid; i < m; i += T) c += undecided(score[i]) && exact[i] > cut;
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0 && c) atomicAdd(&s_ties, c);
        __syncthreads();
        ties = left - s_ties;
    }

    // the chosen blocks in ascending order
    int done = 0, tied = 0;
    for (int base = 0; base < m; base += T) {
        const int i = base + tid;
        bool take = false, tie = false;
        if (i < m) {
            const float x = score[i];
            if (undecided(x)) {
                if (left == nbnd) {
                    take = true;
                } else if (small) {
                    for (int k = 0; k < nbnd; ++k)
                        if (band[k] == i) take = chosen[k];
                } else {
                    const unsigned long long key = a.exact[(int64_t)sh_ * a.max_blocks + i];
                    take = key > cut;
                    tie = key == cut;
                }
            } else {
                take = x > above;
            }
        }
        if (!small && left != nbnd) {  // equals of the cut: the first `ties` of them
            const unsigned tm = __ballot_sync(0xffffffffu, tie);
            if (lane == 0) wsum[0][warp] = __popc(tm);
            __syncthreads();
            int at = tied + __popc(tm & ((1u << lane) - 1u)), all = 0;
            for (int w = 0; w < W; ++w) {
                if (w < warp) at += wsum[0][w];
                all += wsum[0][w];
            }
            take |= tie && at < ties;
            tied += all;
        }
        const unsigned km = __ballot_sync(0xffffffffu, take);
        if (lane == 0) wsum[1][warp] = __popc(km);
        __syncthreads();
        int at = done + __popc(km & ((1u << lane) - 1u)), all = 0;
#pragma unroll
        for (int w = 0; w < W; ++w) {
            if (w < warp) at += wsum[1][w];
            all += wsum[1][w];
        }
        if (take) out[at] = i;
        done += all;
        __syncthreads();
    }
    if (tid == 0) out[need] = m;
}

}  // namespace b200
