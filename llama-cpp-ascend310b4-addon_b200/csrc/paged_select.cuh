// paged_select.cuh -- block selection for sparse attention: an upper bound of
// q . k per block from the page's key bounds, and the n_sel best blocks.
//
// The order of the scores is decided in 64 bits: f32 sums of 64 to 256
// products are off by some 1e-6 of a score, and with thousands of blocks per
// head the scores around the last place of the selection lie that close
// together, so 32 bits would pick blocks by rounding.  But only the few
// blocks around that place need 64 bits.  The first kernel reads all bounds
// once and finds every score to within a bound eps on the tensor cores; the
// second finds the need-th largest of those, tau.  The exact need-th largest
// score is within eps of tau, so a block above tau + 2 eps is chosen and one
// below tau - 2 eps is not, whatever the rounding; the blocks in between
// (mostly the one at tau) are scored again in 64 bits and ranked.
//
// max(q lo, q hi) summed over d is  q+ . hi + q- . lo  with q+ = max(q, 0),
// q- = min(q, 0): two matrix products per block, with the operands of the
// attention kernel (heads x dims against rows of pages), reading 4 D bytes
// per block and KV head: bound by memory.  All in 64 bits it would be bound by
// the f64 pipe and the selects that feed it.
//
// Measured: 26300 blocks x 8 KV heads x 128 dims (108 MB of bounds), 128 chosen
// per head, 35.5 us: 17 us of stream at the copy rate and 8 us of start and
// drain in the first kernel, 8 us in the second; all in 64 bits 292 us as a
// plain kernel.  eps assumes how the tensor core truncates (below, where it is
// computed); the error of the first kernel's scores was below 2% of eps over 72
// shapes and distributions.
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
    float2* group;              // [n_seq][n_head_kv] 2^-ex and max_j sum |q_jd| 2^-ex
    unsigned int* unit_max;     // [n_seq][n_head_kv][ceil(max_blocks / 16)] largest |bound|, as 16-bit patterns
    int n_seq, n_head, n_head_kv, max_blocks, page_size, n_pages, n_sel;
};

B200_HD constexpr int paged_units(int blocks) { return (blocks + kPaTok - 1) / kPaTok; }

// Larger magnitudes of two pairs of 16-bit values; NaN where either is NaN.
template <bool BF16>
__device__ __forceinline__ uint32_t max16_abs(uint32_t x, uint32_t y) {
    if (BF16) {
        const __nv_bfloat162 r = __hmax2_nan(*reinterpret_cast<const __nv_bfloat162*>(&x),
                                             __habs2(*reinterpret_cast<const __nv_bfloat162*>(&y)));
        return *reinterpret_cast<const uint32_t*>(&r);
    }
    const __half2 r =
        __hmax2_nan(*reinterpret_cast<const __half2*>(&x), __habs2(*reinterpret_cast<const __half2*>(&y)));
    return *reinterpret_cast<const uint32_t*>(&r);
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
    in.head = in.nu > 0 ? (range.fb - range.base0) / in.nu : H;
    if ((unsigned)in.head >= (unsigned)H) return;  // the lengths changed while the kernel runs
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
    // unit after it are on their way.  Offsets in 16-byte steps, in 32 bits.
    const uint32_t lc = lane % LPR, lr = lane / LPR;
    constexpr int SW = 8 / RPI;  // the swizzle repeats after 8 rows
    uint32_t dst_of[SW];
#pragma unroll
    for (int i = 0; i < SW; ++i) dst_of[i] = ring + lr * RB + ((lc ^ ((i * RPI + lr) & 7)) << 4);
    const uint8_t *hi = reinterpret_cast<const uint8_t*>(a.hi + 8 * lc), *lo = reinterpret_cast<const uint8_t*>(a.lo + 8 * lc);
    auto page_of = [&](const Cursor& c) -> int {
        const int b = kPaTok * c.u + (lane & 15);
        return b < c.nb ? a.table[c.s * a.table_stride + b] : -1;
    };
    int page_next = page_of(in);
    auto issue = [&](int stage) {
        if (to_issue > 0) {
            const int page = page_next;
            const bool ok = (unsigned)page < (unsigned)a.n_pages;
            if (!ok && kPaTok * in.u + (lane & 15) < in.nb) record_status(B200_DEVSTATUS_BOUNDS);
            const uint32_t row = ok ? ((uint32_t)page * H + in.head) * LPR : 0u;
            --to_issue;
            if (to_issue > 0) {
                if (advance(in)) page_next = page_of(in);
                else to_issue = 0;
            }
            const unsigned valid = __ballot_sync(0xffffffffu, ok) & 0xffffu;
            if (lane == 0) sh.valid[warp][stage] = valid;
            const uint32_t at = stage * (2 * TILE);
            unrolled(std::make_index_sequence<kPaTok / RPI>{}, [&](auto ic) {
                constexpr int I = decltype(ic)::value, OFF = I / SW * (SW * RPI * RB) + I % SW * (RPI * RB);
                const uint32_t x = __shfl_sync(0xffffffffu, row, I * RPI + lr);
                if (valid == 0xffffu) {
                    pa_cp16_at<OFF>(dst_of[I % SW] + at, pa_step<16>(hi, x));
                    pa_cp16_at<OFF + TILE>(dst_of[I % SW] + at, pa_step<16>(lo, x));
                } else {
                    const bool on = (valid >> (I * RPI + lr)) & 1;
                    pa_cp16(dst_of[I % SW] + at + OFF, pa_step<16>(hi, x), on);
                    pa_cp16(dst_of[I % SW] + at + OFF + TILE, pa_step<16>(lo, x), on);
                }
            });
        }
        pa_commit();
    };

    // consumer
    // q+ and q- apart where registers allow, else q and the mask of its positive
    // entries
    constexpr bool APART = D <= 128;
    uint32_t qf[APART ? 2 : 1][KT][4], q3[APART ? 2 : 1][BF16 ? KT : 1][2], plus[APART ? 1 : KT][2];
    bool new_q = true;
    int stage = 0, ahead = 0;
    float up = 1.f;
    const int mi = lane >> 3, ri = lane & 7;
    uint32_t b_at[4];  // this lane's ldmatrix rows, as K's in the attention kernel
#pragma unroll
    for (int i = 0; i < 4; ++i) b_at[i] = ring + (8 * (mi >> 1) + ri) * RB + (((2 * i + (mi & 1)) ^ ri) << 4);
#pragma unroll 1
    for (int turn = 1 - S; to_do > 0; ++turn) {
        if (turn >= 0) {
            pa_wait<S - 2>();
            __syncwarp();
        }
        issue(ahead);
        ahead = ahead + 1 == S ? 0 : ahead + 1;
        if (turn < 0) continue;
        const int64_t sh_ = (int64_t)cur.s * H + cur.head;
        const float* qg = a.q + cur.s * a.q_stride + (int64_t)cur.head * G * D + 2 * t4;
        // this thread's values of head j0 + g; rows past the group repeat its last head
        auto fetch_q = [&](int j0, float2 (&x)[2 * KT]) {
            const float* qr = qg + min(j0 + g, G - 1) * D;
#pragma unroll
            for (int i = 0; i < 2 * KT; ++i) x[i] = *reinterpret_cast<const float2*>(qr + 8 * i);
        };
        if (new_q) {  // one power of two for the whole group: the scores are compared across its heads
            float big = 0.f, sum = 0.f;
#pragma unroll 1
            for (int j0 = 0; j0 < G; j0 += kPaHeads) {
                float2 x[2 * KT];
                fetch_q(j0, x);
                float one = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * KT; ++i) {
                    big = fmaxf(big, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
                    one += fabsf(x[i].x) + fabsf(x[i].y);
                }
                one += __shfl_xor_sync(0xffffffffu, one, 1);
                one += __shfl_xor_sync(0xffffffffu, one, 2);
                sum = one > sum || one != one ? one : sum;  // NaN stays
            }
            big = pa_warp_max(big);
            asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(sum) : "f"(sum));
            const int ex = min(max((int)(__float_as_uint(big) >> 23) - 127, -120), 120);
            up = __uint_as_float((unsigned)(127 - ex) << 23);
            if (lane == 0 && cur.u == 0) a.group[sh_] = make_float2(up, sum * up);
        }
        const uint32_t st = stage * (2 * TILE);
        float best[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        unsigned top = 0;
#pragma unroll 1
        for (int j0 = 0; j0 < G; j0 += kPaHeads) {
            if (new_q || G > kPaHeads) {
                float2 v[2 * KT];
                fetch_q(j0, v);
#pragma unroll
                for (int i = 0; i < 2 * KT; ++i) {
                    float x = v[i].x * up, y = v[i].y * up;
                    const uint32_t pos = (x > 0.f ? 0xffffu : 0u) | (y > 0.f ? 0xffff0000u : 0u);
                    const int kt = i >> 1, e = i & 1;
                    const uint32_t p0 = pa_split<BF16>(x, y), p1 = pa_split<BF16>(x, y);
                    const uint32_t p2 = BF16 ? pa_split<BF16>(x, y) : 0u;
                    if (APART) {
#pragma unroll
                        for (int half = 0; half < (APART ? 2 : 1); ++half) {
                            const uint32_t m = half ? ~pos : pos;
                            qf[half][kt][2 * e] = p0 & m;
                            qf[half][kt][2 * e + 1] = p1 & m;
                            if (BF16) q3[half][BF16 ? kt : 0][e] = p2 & m;
                        }
                    } else {
                        plus[APART ? 0 : kt][e] = pos;
                        qf[0][kt][2 * e] = p0;
                        qf[0][kt][2 * e + 1] = p1;
                        if (BF16) q3[0][BF16 ? kt : 0][e] = p2;
                    }
                }
            }
            // four k steps at a time from zero, added up outside the tensor core,
            // which truncates: the bound on the sum is what keeps the undecided few
            float sc[4] = {}, d[2][4];
            unrolled(std::make_index_sequence<2 * KT>{}, [&](auto ic) {
                constexpr int half = decltype(ic)::value / KT, kt = decltype(ic)::value % KT, k3 = BF16 ? kt : 0;
                constexpr int from = APART ? half : 0, km = APART ? 0 : kt;
                uint32_t b[4];
                pa_ldsm_at<half * TILE + kt / 4 * 128>(b, b_at[kt % 4] + st);
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max16_abs<BF16>(top, b[i]);
                // q+ with hi, then q- with lo
                const uint32_t m0 = APART ? 0xffffffffu : half ? ~plus[km][0] : plus[km][0];
                const uint32_t m1 = APART ? 0xffffffffu : half ? ~plus[km][1] : plus[km][1];
                const uint32_t(&q)[4] = qf[from][kt];
                const uint32_t a0 = q[0] & m0, a1 = q[1] & m0, a2 = q[2] & m1, a3 = q[3] & m1;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    if (kt % 4 == 0) pa_mma0<BF16>(d[n], a0, a1, a2, a3, b[2 * n], b[2 * n + 1]);
                    else pa_mma<BF16>(d[n], a0, a1, a2, a3, b[2 * n], b[2 * n + 1]);
                    if (BF16)
                        pa_mma<BF16>(d[n], q3[from][k3][0] & m0, 0u, q3[from][k3][1] & m1, 0u, b[2 * n], b[2 * n + 1]);
                }
                if (kt % 4 == 3)
#pragma unroll
                    for (int i = 0; i < 4; ++i) sc[i] += d[i >> 1][i & 1] + d[i >> 1][2 + (i & 1)];
            });
#pragma unroll
            for (int i = 0; i < 4; ++i) best[i] = fmaxf(best[i], sc[i]);
        }
        const unsigned valid = sh.valid[warp][stage];
        // the largest over the heads, which are 8 lanes; then lanes 0-3 hold the unit
#pragma unroll
        for (int o = 4; o < 32; o <<= 1)
#pragma unroll
            for (int i = 0; i < 4; ++i) best[i] = fmaxf(best[i], __shfl_xor_sync(0xffffffffu, best[i], o));
        top = __reduce_max_sync(0xffffffffu, max(top & 0xffffu, top >> 16));
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

// The larger of two products; NaN where either is (fmax would drop it).
__device__ __forceinline__ double larger_or_nan(double x, double y) { return x > y || x != x ? x : y; }

// One warp: the 64-bit score of block b for query head j of KV head h, every
// lane.
template <bool BF16, int D>
__device__ __forceinline__ double exact_score(const PagedSelectArgs& a, int s, int h, int j, int page) {
    constexpr int E = D / 32;
    const int lane = threadIdx.x & 31;
    const int64_t at = ((int64_t)page * a.n_head_kv + h) * D + lane * E;
    const float* q = a.q + s * a.q_stride + (int64_t)(h * (a.n_head / a.n_head_kv) + j) * D + lane * E;
    double x = 0.0;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const float2 lo = unpack16<BF16>(*reinterpret_cast<const uint32_t*>(a.lo + at + e));
        const float2 hi = unpack16<BF16>(*reinterpret_cast<const uint32_t*>(a.hi + at + e));
        const float2 v = *reinterpret_cast<const float2*>(q + e);
        x += larger_or_nan((double)v.x * lo.x, (double)v.x * hi.x);
        x += larger_or_nan((double)v.y * lo.y, (double)v.y * hi.y);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
    return x;
}

constexpr int kTopkThreads = 1024;
constexpr int kTopkKeys = 8;      // consecutive scores a thread holds, at most
constexpr int kTopkBins = 2048;
constexpr int kTopkList = 256;    // scores of one bin, or undecided blocks, ranked in shared memory

// Exclusive prefix of v over the CTA's threads, and the total; part: 32 ints.
__device__ __forceinline__ int block_prefix(int v, int* part, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int incl = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    __syncthreads();  // the previous call's readers are done with part
    if (lane == 31) part[warp] = incl;
    __syncthreads();
    const int mine = lane < (int)blockDim.x / 32 ? part[lane] : 0;
    total = __reduce_add_sync(0xffffffffu, mine);
    return incl - v + __reduce_add_sync(0xffffffffu, lane < warp ? mine : 0);
}

// One CTA per (sequence, KV head).  A thread holds up to 8 consecutive scores
// (more than 8192 blocks: tile by tile, read again in every pass).
//   1. tau by a histogram of 2048 equal bins between the smallest and largest
//      score (x -> bin is monotone, so the bins are in order), then by rank in
//      the one bin that holds it; by bisection of the bits where that bin is
//      crowded, as with many equal scores.
//   2. the undecided blocks in 64 bits, one warp per block and query head, and
//      their ranks; by bisection where there are more than 256.
//   3. the chosen blocks in order, one prefix sum per tile.
template <bool BF16, int D>
__global__ void __launch_bounds__(kTopkThreads) paged_topk_kernel(PagedSelectArgs a) {
    constexpr int T = kTopkThreads, E = kTopkKeys, W = T / 32, L = kTopkList;
    __shared__ int hist[kTopkBins];
    __shared__ int count[64];
    __shared__ float list[L];
    __shared__ int band[L], band_nan[L], chosen[L];
    __shared__ unsigned long long band_key[L];
    __shared__ int part[32];
    __shared__ int n_list, n_band, n_in, s_bin, s_rank;
    __shared__ unsigned s_top, s_low, s_high, s_tau;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int sh_ = blockIdx.x, s = sh_ / a.n_head_kv, h = sh_ - s * a.n_head_kv;
    const int G = a.n_head / a.n_head_kv;
    for (int i = tid; i < kTopkBins; i += T) hist[i] = 0;
    if (tid < 64) count[tid] = 0;
    if (tid == 0) n_list = n_band = n_in = 0, s_top = s_high = 0, s_low = 0xffffffffu;
    const int len = a.seq_lens[s];
    griddep_wait();  // the scores
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
    float x[E];
    int tile = -1;
    const int per = min(E, (m + T - 1) / T), tiles = (m + T * per - 1) / (T * per);
    auto each = [&](auto f) {  // f(i, score) over this thread's scores
        for (int t = 0; t < tiles; ++t) {
            if (t != tile) {
                tile = t;
#pragma unroll
                for (int e = 0; e < E; ++e) {
                    const int i = (t * T + tid) * per + e;
                    x[e] = e < per && i < m ? score[i] : -INFINITY;
                }
            }
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const int i = (t * T + tid) * per + e;
                if (e < per && i < m) f(i, x[e]);
            }
        }
    };
    {
        unsigned top = 0, low = 0xffffffffu, high = 0;
        const int nu = paged_units(nb);
        for (int i = tid; i < nu; i += T) top = max(top, a.unit_max[(int64_t)sh_ * paged_units(a.max_blocks) + i]);
        each([&](int, float v) {
            const unsigned k = order_key(v);
            high = max(high, k);
            if (v != -INFINITY) low = min(low, k);
        });
        top = __reduce_max_sync(0xffffffffu, top);
        low = __reduce_min_sync(0xffffffffu, low);
        high = __reduce_max_sync(0xffffffffu, high);
        __syncthreads();  // the counters are cleared
        if (lane == 0) {
            atomicMax(&s_top, top);
            atomicMin(&s_low, low);
            atomicMax(&s_high, high);
        }
    }
    const float2 group = a.group[sh_];
    __syncthreads();
    // eps, with q' = q 2^-ex, whose largest entry is in [1, 2), M = max |bound| and
    // S = M max_j sum |q'_jd|: the parts of q' leave out at most 2^-23 of each
    // entry, in all D 2^-23 M; a chain of four instructions (bf16: eight) is assumed
    // to truncate its 67 (135) terms below 2^-24 of the largest (no document says
    // how the tensor core rounds), in all 135 2^-24 S; adding high
    // and low halves and the D / 32 chains rounds D / 32 + 1 times by 2^-24 S at
    // most.  1e-30 covers what underflows.
    const float biggest = BF16 ? __uint_as_float(s_top << 16) : h2f((uint16_t)s_top);
    const float eps = biggest * (D * 0x1p-23f + group.y * (140 + D / 32) * 0x1p-24f) * 1.01f + 1e-30f;
    const bool sure = eps < 1e30f;  // not: bounds or queries that are not finite, nothing is decided by the scores
    float tau = 0.f;
    if (sure) {
        const float low = from_order_key(s_low), high = from_order_key(s_high);
        const float per_bin = high > low ? (kTopkBins - 1) / (high - low) : 0.f;  // (0 where high - low overflows)
        auto bin = [&](float v) {
            return v == -INFINITY ? 0 : min(kTopkBins - 1, max(0, (int)((v - low) * per_bin)));
        };
        each([&](int, float v) { atomicAdd(&hist[bin(v)], 1); });
        __syncthreads();
        // from the top bin down: the one where the need-th score is
        static_assert(kTopkBins == 2 * T, "two bins a thread");
        const int b0 = kTopkBins - 1 - 2 * tid, h0 = hist[b0], h1 = hist[b0 - 1];
        int total;
        const int above = block_prefix(h0 + h1, part, total);
        if (above < need && need <= above + h0) s_bin = b0, s_rank = need - above;
        else if (above + h0 < need && need <= above + h0 + h1) s_bin = b0 - 1, s_rank = need - above - h0;
        __syncthreads();
        const int where = s_bin, rank = s_rank;  // the rank-th largest of this bin
        if (hist[where] <= L) {
            each([&](int, float v) {
                if (bin(v) == where) list[atomicAdd(&n_list, 1)] = v;
            });
            __syncthreads();
            const int n = n_list;
            for (int k = tid; k < n; k += T) {
                int more = 0, same = 0;
                for (int y = 0; y < n; ++y) more += list[y] > list[k], same += list[y] == list[k];
                if (more < rank && rank <= more + same) s_tau = order_key(list[k]);  // equal scores, equal keys
            }
        } else {
            unsigned key = 0;
            for (int bit = 31; bit >= 0; --bit) {
                const unsigned trial = key | 1u << bit;
                int c = 0;
                each([&](int, float v) { c += bin(v) == where && order_key(v) >= trial; });
                c = __reduce_add_sync(0xffffffffu, c);
                if (lane == 0 && c) atomicAdd(&count[bit], c);
                __syncthreads();
                if (count[bit] >= rank) key = trial;
            }
            if (tid == 0) s_tau = key;
        }
        __syncthreads();
        tau = from_order_key(s_tau);
    }
    // chosen: score > over; undecided: [under, over]
    const float over = sure ? tau + 2.01f * eps : INFINITY, under = sure ? tau - 2.01f * eps : -INFINITY;
    auto undecided = [&](float v) { return !sure || (v >= under && v <= over); };
    {
        int c = 0;
        each([&](int i, float v) {
            if (undecided(v)) {
                const int k = atomicAdd(&n_band, 1);
                if (k < L) band[k] = i;
            } else if (v > over) {
                ++c;
            }
        });
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0 && c) atomicAdd(&n_in, c);
    }
    __syncthreads();
    const int nbnd = n_band, left = need - n_in;  // `left` of the nbnd undecided blocks
    const bool all_in = left == nbnd, small = nbnd <= L;
    unsigned long long* exact = a.exact + (int64_t)sh_ * a.max_blocks;
    unsigned long long cut = 0;  // many undecided: the smallest 64-bit key chosen, and `ties` of its equals
    int ties = 0;
    if (!all_in && small) {
        for (int k = tid; k < nbnd; k += T) band_key[k] = 0, band_nan[k] = 0;
        __syncthreads();
        for (int y = warp; y < nbnd * G; y += W) {
            const int k = y / G, page = a.table[s * a.table_stride + band[k]];
            if ((unsigned)page >= (unsigned)a.n_pages) continue;  // stays below everything
            const double v = exact_score<BF16, D>(a, s, h, y - k * G, page);
            if (lane == 0) {
                if (v != v) band_nan[k] = 1;
                else atomicMax(&band_key[k], order_key(v));
            }
        }
        __syncthreads();
        for (int k = tid; k < nbnd; k += T) {
            const unsigned long long mine = band_nan[k] ? 0 : band_key[k];
            int rank = 0;
            for (int y = 0; y < nbnd; ++y) {
                const unsigned long long other = band_nan[y] ? 0 : band_key[y];
                rank += other > mine || (other == mine && band[y] < band[k]);
            }
            chosen[k] = rank < left;
        }
        __syncthreads();
    } else if (!all_in) {
        for (int i = warp; i < m; i += W) {
            if (!undecided(score[i])) continue;
            const int page = a.table[s * a.table_stride + i];
            unsigned long long key = 0;
            if ((unsigned)page < (unsigned)a.n_pages) {
                bool nan = false;
                for (int j = 0; j < G; ++j) {
                    const double v = exact_score<BF16, D>(a, s, h, j, page);
                    nan |= v != v;
                    if (v == v) key = max(key, order_key(v));
                }
                if (nan) key = 0;
            }
            if (lane == 0) exact[i] = key;
        }
        __syncthreads();
        if (tid < 64) count[tid] = 0;
        if (tid == 0) n_list = 0;
        __syncthreads();
        for (int bit = 63; bit >= 0; --bit) {
            const unsigned long long trial = cut | 1ull << bit;
            int c = 0;
            each([&](int i, float v) { c += undecided(v) && exact[i] >= trial; });
            c = __reduce_add_sync(0xffffffffu, c);
            if (lane == 0 && c) atomicAdd(&count[bit], c);
            __syncthreads();
            if (count[bit] >= left) cut = trial;
        }
        int c = 0;
        each([&](int i, float v) { c += undecided(v) && exact[i] > cut; });
        c = __reduce_add_sync(0xffffffffu, c);
        if (lane == 0 && c) atomicAdd(&n_list, c);
        __syncthreads();
        ties = left - n_list;
    }

    // the chosen blocks in ascending order
    int done = 0, tied = 0;
    for (int t = 0; t < tiles; ++t) {
        unsigned take = 0, tie = 0;  // bit e: this thread's e-th score of the tile
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int i = (t * T + tid) * per + e;
            if (e >= per || i >= m) break;
            const float v = tiles == 1 ? x[e] : score[i];
            if (!undecided(v)) {
                take |= (v > over ? 1u : 0u) << e;
            } else if (all_in) {
                take |= 1u << e;
            } else if (small) {
                for (int k = 0; k < nbnd; ++k)
                    if (band[k] == i && chosen[k]) take |= 1u << e;
            } else {
                take |= (exact[i] > cut ? 1u : 0u) << e;
                tie |= (exact[i] == cut ? 1u : 0u) << e;
            }
        }
        int total;
        if (!all_in && !small) {  // of the cut's equals the first `ties`
            int at = tied + block_prefix(__popc(tie), part, total);
            for (; tie != 0; tie &= tie - 1)
                if (at++ < ties) take |= tie & (0u - tie);
            tied += total;
        }
        int at = done + block_prefix(__popc(take), part, total);
        for (; take != 0; take &= take - 1, ++at)
            if (at < need) out[at] = (t * T + tid) * per + __ffs(take) - 1;  // (more only if lengths changed meanwhile)
        done += total;
    }
    if (tid == 0) out[need] = m;
}

}  // namespace b200
