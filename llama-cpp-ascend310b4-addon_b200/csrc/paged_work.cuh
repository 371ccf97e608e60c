// paged_work.cuh -- what the kernels that stream pages share: equal ranges of
// units over sequences of any lengths, copies, tensor-core products of 16-bit
// pages with f32 operands.
#pragma once

#include <utility>

#include "common.cuh"
#include "paged_store.cuh"

namespace b200 {

constexpr int kPaTok = 16;    // rows (positions, blocks) per unit
constexpr int kPaCtas = 148;  // CTAs of a full grid: one per SM

// Blocks of a sequence; a length outside the table is clamped.
__device__ __forceinline__ int paged_blocks(int len, int max_blocks, int page_size) {
    const unsigned b = len <= 0 ? 0u : ((unsigned)len + (unsigned)page_size - 1u) / (unsigned)page_size;
    return (int)min(b, (unsigned)max_blocks);
}

__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
}
// 16 bytes to dst + OFF.
template <int OFF>
__device__ __forceinline__ void pa_cp16_at(uint32_t dst, const void* src) {
    asm volatile("cp.async.cg.shared.global [%0 + %2], [%1], 16;" ::"r"(dst), "l"(src), "n"(OFF) : "memory");
}
__device__ __forceinline__ void pa_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void pa_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void pa_ldsm(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
// The same at addr + OFF, and transposed.
template <int OFF>
__device__ __forceinline__ void pa_ldsm_at(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(OFF)
                 : "memory");
}
template <int OFF>
__device__ __forceinline__ void pa_ldsm_t_at(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4 + %5];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr), "n"(OFF)
                 : "memory");
}
template <bool BF16>
__device__ __forceinline__ void pa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    if (BF16)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// The same from a zero accumulator.
template <bool BF16>
__device__ __forceinline__ void pa_mma0(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                        uint32_t b1) {
    if (BF16)
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
    else
        asm(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ float pa_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// High 16-bit part of two values packed in a word; x, y become the remainders.
template <bool BF16>
__device__ __forceinline__ uint32_t pa_split(float& x, float& y) {
    const uint32_t w = pack16<BF16>(x, y);
    const float2 f = unpack16<BF16>(w);
    x -= f.x;
    y -= f.y;
    return w;
}

__device__ __forceinline__ float pa_warp_max(float v) {
    float r;
    asm("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
    return r;
}
// f(integral_constant<I>) for I of the sequence.
template <size_t... I, class F>
__device__ __forceinline__ void unrolled(std::index_sequence<I...>, F f) {
    (f(std::integral_constant<int, (int)I>{}), ...);
}

// p + I * step in one instruction.
template <int I>
__device__ __forceinline__ const uint8_t* pa_step(const uint8_t* p, uint32_t step) {
    if (I == 0) return p;
    uint64_t r;
    asm("mad.wide.u32 %0, %1, %2, %3;" : "=l"(r) : "r"(step), "n"(I), "l"(p));
    return reinterpret_cast<const uint8_t*>(r);
}

template <int W>
struct PaRangeShared {
    int part[W];           // prefix-sum partials
    int seq[W], base[W];   // the sequence a warp starts in and that one's first unit
};

// The units of all sequences (units(s) for each of `segs` segments of sequence
// s), in order, cut into equal ranges: [cb, ce) for this CTA, and that one
// into [fb, fe) for this warp, which starts in sequence seq0, whose first unit
// is base0.  Every CTA sums up the lengths for itself: up to 128 in each warp
// without a barrier, more across the CTA.  All threads call it; it ends with a
// CTA barrier.
template <int W>
struct PaRange {
    int per_cta, cb, ce, fb, fe, seq0, base0;

    template <class U>
    __device__ __forceinline__ PaRange(PaRangeShared<W>& sh, int n_seq, int segs, U units) {
        const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
        const bool few = n_seq <= 128;
        const int at = few ? lane : tid;
        const int per = few ? (n_seq + 31) >> 5 : (n_seq + 32 * W - 1) / (32 * W);
        const int s_lo = min(n_seq, at * per), s_hi = min(n_seq, s_lo + per);
        int mine = 0;
        for (int s = s_lo; s < s_hi; ++s) mine += units(s);
        int incl = mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        int total;
        if (few) {
            total = __shfl_sync(0xffffffffu, incl, 31);
        } else {
            if (lane == 31) sh.part[warp] = incl;
            __syncthreads();
            total = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) {
                if (w < warp) incl += sh.part[w];
                total += sh.part[w];
            }
        }
        int before = (incl - mine) * segs;
        total *= segs;
        per_cta = max((int)((total + gridDim.x - 1u) / gridDim.x), W);
        cb = (int)min((unsigned)total, (unsigned)per_cta * blockIdx.x);
        ce = (int)min((unsigned)total, (unsigned)cb + (unsigned)per_cta);
        const int per_warp = (ce - cb + W - 1) / W;
        fb = min(ce, cb + per_warp * warp);
        fe = min(ce, fb + per_warp);
        if (few) {
            const unsigned owner = __ballot_sync(0xffffffffu, fb >= before && fb < before + mine * segs);
            seq0 = s_lo;
            for (int s = s_lo; s < s_hi; ++s) {  // (no more than one owner, whose answer counts)
                const int end = before + units(s) * segs;
                if (fb < end) {
                    seq0 = s;
                    break;
                }
                before = end;
            }
            const int src = owner ? __ffs(owner) - 1 : 0;
            seq0 = __shfl_sync(0xffffffffu, seq0, src);
            base0 = __shfl_sync(0xffffffffu, before, src);
            __syncthreads();
        } else {
            for (int s = s_lo; s < s_hi; ++s) {
                const int end = before + units(s) * segs;
                if (end > cb && before < ce)
                    for (int w = 0; w < W; ++w) {
                        const int b = cb + per_warp * w;
                        if (b >= before && b < end) sh.seq[w] = s, sh.base[w] = before;
                    }
                before = end;
            }
            __syncthreads();
            seq0 = sh.seq[warp];
            base0 = sh.base[warp];
        }
    }
};

}  // namespace b200
