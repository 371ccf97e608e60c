// paged_range.cuh -- equal ranges of units over sequences of any lengths.
// Includes nothing and uses only the warp functions below, so that a host test
// can run it with functions of its own.
#pragma once

namespace b200 {

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
            if (lane == 0) sh.seq[warp] = 0, sh.base[warp] = 0;  // (stays where lengths change meanwhile)
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

// CTAs that hold units from, from + 1, .. from + nu - 1, at most to the grid's
// last (which only lengths that change while a kernel runs could pass).
__device__ __forceinline__ int pa_pieces(int from, int nu, int per_cta, int grid) {
    return (int)min((unsigned)grid, ((unsigned)from + (unsigned)nu - 1u) / (unsigned)per_cta + 1u) - from / per_cta;
}

}  // namespace b200
