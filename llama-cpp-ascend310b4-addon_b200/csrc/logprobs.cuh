// logprobs.cuh -- log probabilities of rows of logits with their entropy and
// the k largest alternatives, in one pass over the row.
//
// With M the row's largest logit, n1 the number of logits equal to it and
// t_i = x_i - M:
//   lse' = log(n1) + log1p(sum_{t_i < 0} e^{t_i} / n1)
//   log p_i = t_i - lse',  entropy = lse' + sum_i e^{t_i} (-t_i) / sum_i e^{t_i},
// sums of terms of one sign, so a distribution that one token holds almost alone
// keeps its digits.  A thread carries its own M, n1, sum and weighted sum and
// scales them when a larger logit comes (once per four vectors at most); threads,
// warps and CTAs are joined in a fixed order.
//
// The k largest: the k-th largest of the threads' largest logits is a lower bound
// of the k-th largest of all, and of the thread with the r-th largest only its
// k - r largest can be among them.  So a thread keeps its largest vector alone
// in the pass.  The k-th largest of 64 groups of threads bounds from below which
// threads can matter (a few more than k, as a rule); their winners are sorted by
// one warp, and the owners of the first k are read again for what else they hold
// above the k-th: their best vector, or all vectors of the few whose largest logit
// outside it (kept in the pass as well) is no smaller.  (All vectors of all owners:
// 156 instead of 125 us with k 20, 122 instead of 121 with k 5; 1024 rows.)  Keys are (order-preserving bits, inverted
// id): all differ, ties go to the lower id, NaN is smallest.
//
// 1024 rows of 151936 f32 logits: 103 us with k 0 (6.0 TB/s, the stream), 111 with k
// 5, 117 with k 20; one row of 128256 with k 20 11 to 12.5 us, with k 0 8.5.  16-bit
// logits are bound by the instructions instead: 1024 rows of f16 82 us with k 0 (3.8
// TB/s), 91 with k 5.
//
// A row is read once by a cluster of up to 8 CTAs, whose lists and sums meet in
// the first one's shared memory.
#pragma once

#include <cooperative_groups.h>
#include <cuda_bf16.h>

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"

namespace b200 {

struct LogprobsArgs {
    const uint8_t* logits;
    int64_t ld;  // bytes
    int64_t n_rows;
    int n_vocab, k, ctas;
    const int32_t* tokens;
    float *logprob, *entropy, *top_logprobs;
    int32_t* top_ids;
};

constexpr int kLpThreads = 256;
constexpr int kLpWarps = kLpThreads / 32;
constexpr int kLpBatch = 4;       // vectors of 16 bytes in flight per thread
constexpr int kLpMaxCtas = 8;
// CTAs on an SM at once.  f32 takes 40 registers where nothing is asked (0); asked for
// six CTAs it spills (1% slower), for one it takes 56 (6% slower).  16-bit types are
// held to 48 instead of 56, with 12 bytes spilled (1024 rows of bf16 97 -> 94 us).
constexpr int kLpPerSmF32 = 6, kLpPerSm16 = 5;
// kept by the thread of rank r: k - r at most or a vector's eight, besides the row's
// unaligned ends
constexpr int kLpFound = B200_LOGPROBS_MAX_K * (B200_LOGPROBS_MAX_K + 1) / 2 + B200_LOGPROBS_MAX_K * 8 + 16;

using LpKey = unsigned long long;

__device__ __forceinline__ LpKey lp_key(float x, unsigned id) {
    const unsigned b = __float_as_uint(x + 0.f);  // -0 counts as 0
    const unsigned v = x != x ? 0u : (b & 0x80000000u) ? ~b : (b | 0x80000000u);
    return ((LpKey)v << 32) | ~id;
}
__device__ __forceinline__ float lp_value(LpKey key) {
    const unsigned v = (unsigned)(key >> 32);
    if (v == 0) return __uint_as_float(0x7fc00000u);
    return __uint_as_float((v & 0x80000000u) ? v & 0x7fffffffu : ~v);
}
__device__ __forceinline__ unsigned lp_id(LpKey key) { return ~(unsigned)key; }

// A warp's keys into descending order (lane 0 the largest).
__device__ __forceinline__ LpKey lp_sort(LpKey x) {
    const int lane = threadIdx.x & 31;
#pragma unroll
    for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
        for (int o = size >> 1; o > 0; o >>= 1) {
            const LpKey y = __shfl_xor_sync(0xffffffffu, x, o);
            const bool larger = ((lane & o) == 0) == ((lane & size) == 0 || size == 32);
            x = (larger == (x > y)) ? x : y;
        }
    return x;
}
// The 32 largest of two descending lists, descending.
__device__ __forceinline__ LpKey lp_merge(LpKey x, LpKey y) {
    const int lane = threadIdx.x & 31;
    y = __shfl_sync(0xffffffffu, y, 31 - lane);
    x = x > y ? x : y;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const LpKey z = __shfl_xor_sync(0xffffffffu, x, o);
        x = (((lane & o) == 0) == (x > z)) ? x : z;
    }
    return x;
}

// What is known of some of the logits: the largest, how many equal it, the sum
// of the others' e^{x - m}, the sum of e^t t with t = (x - m) log2(e).
struct LpSums {
    float m, n1, s, a;
};
constexpr float kLog2e = 1.4426950408889634f;
__device__ __forceinline__ float lp_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// The same logits relative to m >= x.m.
__device__ __forceinline__ void lp_rescale(LpSums& x, float m) {
    if (x.m == m || x.m == -INFINITY) {
        // nothing but -inf so far holds no sums; infinities and NaN end up in s below
        x.m = m;
        return;
    }
    const float t = (x.m - m) * kLog2e, f = lp_exp2(t), all = x.s + x.n1;
    x.a = f * (x.a + (f > 0.f ? t * all : 0.f));
    x.s = f * all;
    x.n1 = 0.f;
    x.m = m;
}
__device__ __forceinline__ LpSums lp_join(LpSums x, LpSums y) {
    const float m = fmaxf(x.m, y.m);
    lp_rescale(x, m);
    lp_rescale(y, m);
    return {m, x.n1 + y.n1, x.s + y.s, x.a + y.a};
}
__device__ __forceinline__ void lp_add(LpSums& c, float x) {
    // (a reference of -inf: x is -inf or NaN)
    const float t = (x - (c.m == -INFINITY ? 0.f : c.m)) * kLog2e;
    const float e = lp_exp2(t);
    const bool top = t == 0.f;
    c.n1 += top ? 1.f : 0.f;
    c.s += top ? 0.f : e;
    c.a = fmaf(e, fmaxf(t, -1000.f), c.a);
}
__device__ __forceinline__ LpSums lp_shfl(const LpSums& x, int o) {
    return {__shfl_xor_sync(0xffffffffu, x.m, o), __shfl_xor_sync(0xffffffffu, x.n1, o),
            __shfl_xor_sync(0xffffffffu, x.s, o), __shfl_xor_sync(0xffffffffu, x.a, o)};
}

template <int TYPE>
struct LpType {
    static constexpr int kSize = TYPE == B200_TYPE_F32 ? 4 : 2;
    static constexpr int kVec = 16 / kSize;
    static __device__ __forceinline__ float one(const uint8_t* p) {
        if (TYPE == B200_TYPE_F32) return __ldg(reinterpret_cast<const float*>(p));
        const uint16_t h = __ldg(reinterpret_cast<const uint16_t*>(p));
        return TYPE == B200_TYPE_F16 ? h2f(h) : __uint_as_float((uint32_t)h << 16);
    }
    static __device__ __forceinline__ void split(const uint4& w, float (&x)[kVec]) {
        const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (TYPE == B200_TYPE_F32) {
                x[i] = __uint_as_float(u[i]);
            } else if (TYPE == B200_TYPE_F16) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
                x[(2 * i) % kVec] = f.x, x[(2 * i + 1) % kVec] = f.y;
            } else {
                x[(2 * i) % kVec] = __uint_as_float(u[i] << 16);
                x[(2 * i + 1) % kVec] = __uint_as_float(u[i] & 0xffff0000u);
            }
        }
    }
};

constexpr int kLpGroups = 64;                     // groups of neighbouring threads
constexpr int kLpGroup = kLpThreads / kLpGroups;  // threads in each
static_assert(kLpGroups >= B200_LOGPROBS_MAX_K, "k of the groups bound the k-th largest");

struct LpShared {
    LpSums sums[kLpWarps];
    alignas(16) float group[kLpGroups];  // largest logit of a group
    float second[kLpThreads];  // largest logit of a thread outside its best vector
    float bound;               // the k-th largest of them
    LpKey winner[kLpThreads];  // largest keys of the threads above the bound
    LpKey first[32];           // the first of them, descending
    int n_winners;
    LpKey found[kLpFound];
    int n_found;
    // the first CTA's: what the cluster's CTAs found
    LpSums cta_sums[kLpMaxCtas];
    LpKey cta_list[kLpMaxCtas][32];
};

template <int TYPE>
__global__ void __launch_bounds__(kLpThreads, TYPE == B200_TYPE_F32 ? 0 : kLpPerSm16)
logprobs_kernel(const __grid_constant__ LogprobsArgs a) {
    using T = LpType<TYPE>;
    constexpr int VEC = T::kVec;
    __shared__ LpShared sh;
    namespace cg = cooperative_groups;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ctas = a.ctas;  // of the row's cluster
    const int64_t r = blockIdx.x / (unsigned)ctas;
    const int cta = (int)(blockIdx.x - r * ctas);
    const uint8_t* row = a.logits + r * a.ld;
    if (ctas > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    // whole vectors between the row's unaligned ends; this CTA's are v0 .. v1 - 1
    const int head = min(a.n_vocab, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / T::kSize);
    const int n_vec = (a.n_vocab - head) / VEC, tail = head + n_vec * VEC;
    const uint4* vecs = reinterpret_cast<const uint4*>(row + (int64_t)head * T::kSize);
    const int per = (n_vec + ctas - 1) / ctas;
    const int v0 = min(n_vec, cta * per), v1 = min(n_vec, v0 + per);
    if (tid == 0) sh.n_found = sh.n_winners = 0;
    __syncthreads();

    LpSums c = {-INFINITY, 0.f, 0.f, 0.f};
    float best = -INFINITY;      // this thread's largest logit ..
    int best_v = v0 + tid;       // .. its vector ..
    float second = -INFINITY;    // .. and the largest outside that
    auto batch = [&](const uint4 (&w)[kLpBatch], int v, bool whole) {
        float top = -INFINITY;
        float x[kLpBatch][VEC];
#pragma unroll
        for (int j = 0; j < kLpBatch; ++j) {
            T::split(w[j], x[j]);
            float m = x[j][0];
#pragma unroll
            for (int e = 1; e < VEC; ++e) m = fmaxf(m, x[j][e]);
            if (!whole && v + j * kLpThreads >= v1) m = -INFINITY;
            second = fmaxf(second, fminf(m, best));
            if (m > best) best = m, best_v = v + j * kLpThreads;
            top = fmaxf(top, m);
        }
        if (top > c.m) lp_rescale(c, top);
#pragma unroll
        for (int j = 0; j < kLpBatch; ++j)
            if (whole || v + j * kLpThreads < v1)
#pragma unroll
                for (int e = 0; e < VEC; ++e) lp_add(c, x[j][e]);
    };
    int v = v0 + tid;
    for (; v + (kLpBatch - 1) * kLpThreads < v1; v += kLpBatch * kLpThreads) {
        uint4 w[kLpBatch];
#pragma unroll
        for (int j = 0; j < kLpBatch; ++j) w[j] = __ldcs(vecs + v + j * kLpThreads);
        batch(w, v, true);
    }
    if (v < v1) {
        uint4 w[kLpBatch];
#pragma unroll
        for (int j = 0; j < kLpBatch; ++j) w[j] = __ldg(vecs + min(v + j * kLpThreads, v1 - 1));
        batch(w, v, false);
    }
    const bool odd = c.s != c.s;  // a NaN or +inf among them: best may not be the largest
    // the row's ends: a logit to a thread of the first CTA, candidates all of them
    if (cta == 0) {
        const int n_ends = head + a.n_vocab - tail;
        if (tid < n_ends) {
            const int id = tid < head ? tid : tail + tid - head;
            const float x = T::one(row + (int64_t)id * T::kSize);
            if (x > c.m) lp_rescale(c, x);
            lp_add(c, x);
            if (a.k) sh.found[atomicAdd(&sh.n_found, 1)] = lp_key(x, id);
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) c = lp_join(c, lp_shfl(c, o));
    if (lane == 0) sh.sums[warp] = c;

    LpKey mine = 0;  // (warp 0) this CTA's largest, descending
    if (a.k) {
        auto vector_best = [&](int at, LpKey below, LpKey best_key) {
            float x[VEC];
            T::split(__ldg(vecs + at), x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const LpKey y = lp_key(x[e], head + at * VEC + e);
                if (y < below && y > best_key) best_key = y;
            }
            return best_key;
        };
        const bool some = v0 + tid < v1;
        float group = some ? best : -INFINITY;
#pragma unroll
        for (int o = 1; o < kLpGroup; o <<= 1) group = fmaxf(group, __shfl_xor_sync(0xffffffffu, group, o));
        if (tid % kLpGroup == 0) sh.group[tid / kLpGroup] = group;
        sh.second[tid] = odd ? INFINITY : second;
        __syncthreads();
        // How many groups exceed one: the k-th largest (ties by any order).  A group's
        // threads compare it with a quarter of all each (every warp ranking all groups: 121
        // instead of 111 us, 1024 rows).
        {
            const float mine_g = sh.group[tid / kLpGroup];
            int above = 0;  // and those equal to it, times 2^16
#pragma unroll
            for (int g = 4 * (tid % kLpGroup); g < kLpGroups; g += 4 * kLpGroup) {
                const float4 w = *reinterpret_cast<const float4*>(sh.group + g);
                above += (w.x > mine_g) + (w.y > mine_g) + (w.z > mine_g) + (w.w > mine_g);
                above += ((w.x == mine_g) + (w.y == mine_g) + (w.z == mine_g) + (w.w == mine_g)) << 16;
            }
#pragma unroll
            for (int o = 1; o < kLpGroup; o <<= 1) above += __shfl_xor_sync(0xffffffffu, above, o);
            const int larger = above & 0xffff;
            if (larger < a.k && larger + (above >> 16) >= a.k) sh.bound = mine_g;  // one value, whoever writes it
        }
        __syncthreads();
        const float bound = sh.bound;
        if (odd || (some && best >= bound)) {
            LpKey key = 0;
            if (odd)
                for (int u = v0 + tid; u < v1; u += kLpThreads) key = vector_best(u, ~0ull, key);
            else
                key = vector_best(best_v, ~0ull, 0);
            sh.winner[atomicAdd(&sh.n_winners, 1)] = key;
        }
        __syncthreads();
        if (warp == 0) {
            LpKey top = 0;
            for (int f = 0; f < sh.n_winners; f += 32) {
                const LpKey other = lp_sort(f + lane < sh.n_winners ? sh.winner[f + lane] : 0);
                top = f ? lp_merge(top, other) : other;
            }
            sh.first[lane] = top;
        }
        __syncthreads();
        const LpKey key = sh.first[lane];
        const LpKey least = __shfl_sync(0xffffffffu, key, a.k - 1);
        // A thread whose second is below the k-th winner has nothing to give outside its
        // best vector: a lane looks through that.  (A least of 0, fewer than k winners,
        // reads as NaN: no thread is.)
        const int at = (int)(lp_id(key) - head) / VEC;
        const int owned_by = key ? (int)((unsigned)(at - v0) % (unsigned)kLpThreads) : 0;
        const bool ranked = lane < a.k && key != 0, narrow = ranked && sh.second[owned_by] < lp_value(least);
        if (warp == kLpWarps - 1 && narrow) {
            float x[VEC];
            T::split(__ldg(vecs + at), x);
#pragma unroll
            for (int e = 0; e < VEC; ++e) {
                const LpKey y = lp_key(x[e], head + at * VEC + e);
                if (y >= least) sh.found[atomicAdd(&sh.n_found, 1)] = y;
            }
        }
        unsigned wide = __ballot_sync(0xffffffffu, ranked && !narrow);
        for (int n = 0; wide; wide &= wide - 1, ++n) {
            if (n % kLpWarps != warp) continue;
            const int i = __ffs(wide) - 1, owner = __shfl_sync(0xffffffffu, owned_by, i);
            LpKey last = __shfl_sync(0xffffffffu, key, i);
            for (int more = a.k - i; more > 0; --more) {  // last is among the k largest so far: what comes next?
                if (lane == 0) sh.found[atomicAdd(&sh.n_found, 1)] = last;
                if (more == 1) break;
                LpKey next = 0;
                for (int u = v0 + owner + lane * kLpThreads; u < v1; u += 32 * kLpThreads) next = vector_best(u, last, next);
                const unsigned hi = __reduce_max_sync(0xffffffffu, (unsigned)(next >> 32));
                const unsigned lo = __reduce_max_sync(0xffffffffu, (unsigned)(next >> 32) == hi ? (unsigned)next : 0u);
                last = ((LpKey)hi << 32) | lo;
                if (last == 0 || last < least) break;
            }
        }
        __syncthreads();
        if (warp == 0) {
            for (int f = 0; f < sh.n_found; f += 32) {
                const LpKey other = lp_sort(f + lane < sh.n_found ? sh.found[f + lane] : 0);
                mine = f ? lp_merge(mine, other) : other;
            }
        }
    } else {
        __syncthreads();
    }
    if (warp == 0) {
        c = sh.sums[lane < kLpWarps ? lane : 0];
        if (lane >= kLpWarps) c = {-INFINITY, 0.f, 0.f, 0.f};
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) c = lp_join(c, lp_shfl(c, o));
    }
    if (ctas > 1) {
        cg::cluster_group cluster = cg::this_cluster();
        LpShared* first = cluster.map_shared_rank(&sh, 0);
        asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the first CTA has started
        if (warp == 0) {
            if (lane == 0) first->cta_sums[cta] = c;
            if (a.k) first->cta_list[cta][lane] = mine;
        }
        cluster.sync();
        if (cta != 0 || warp != 0) return;
        for (int i = 1; i < ctas; ++i) {
            c = lp_join(c, sh.cta_sums[i]);
            if (a.k) mine = lp_merge(mine, sh.cta_list[i][lane]);
        }
    }
    if (warp != 0) return;
    // every lane holds the row's sums
    const float all = c.n1 + c.s;
    const float lse = logf(c.n1) + log1pf(c.s / c.n1);
    if (lane == 0) {
        if (a.entropy) a.entropy[r] = lse - c.a / all * 0.6931471805599453f;
        if (a.tokens) {
            const int t = a.tokens[r];
            if (t >= a.n_vocab) record_status(B200_DEVSTATUS_BOUNDS);
            a.logprob[r] = t < 0 || t >= a.n_vocab ? 0.f : (T::one(row + (int64_t)t * T::kSize) - c.m) - lse;
        }
    }
    if (lane < a.k) {
        a.top_ids[r * a.k + lane] = (int)lp_id(mine);
        a.top_logprobs[r * a.k + lane] = (lp_value(mine) - c.m) - lse;
    }
}

}  // namespace b200
