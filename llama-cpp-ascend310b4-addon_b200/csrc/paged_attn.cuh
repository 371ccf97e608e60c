// paged_attn.cuh -- attention of one new token per sequence over a paged
// key-value cache, split over the cache's length and joined.
//
//   out_j = sum_p w_p v_p / sum_p w_p,  w_p = 2^(f q_j . k_p + bias_p - m)
//
// with f = scale log2(e) and m the running maximum.  Per cached token and KV
// head K and V are 4 D bytes for 4 D G flops (G <= 8 query heads a pass), so
// the kernel is bound by reading the cache; the arithmetic only has to keep
// up, and the split only has to keep every SM reading until the end.
//
// Work.  A unit is 16 positions of one (sequence, KV head, chunk of 8 query
// heads) segment.  The units of all segments, in order, are cut into equal
// ranges, one per CTA, and each CTA's range into equal ranges, one per warp,
// whatever the lengths are: the cut points follow from the lengths, which
// every CTA sums up for itself.  A warp streams its range through a private
// ring of cp.async stages (each row of K and V found through the block table,
// so any page size and layout works), never waiting for another warp; the
// ring runs ahead across segment borders.
//
// Join.  A segment inside one warp's range is written straight to the output.
// The pieces of a cut segment meet in shared memory once per CTA, and those
// cut by CTA borders in the workspace, where the CTA that finds the segment's
// ticket complete adds them up in CTA order: the result does not depend on
// which CTA that is.
//
// Arithmetic: mma.sync m16n8k16.  The 8 query heads take rows 0-7 with the
// high parts of q (and of the weights w) and rows 8-15 with the low parts, so
// one instruction gives both products and f16 keeps 22 bits of q and w: their
// own rounding stays below that of the f32 sums.  q is scaled by a power of
// two into f16's range, w by 2^12 out of f16's subnormals.  bf16 takes a third
// part in a second instruction.  Sums over positions are f32 additions
// outside the tensor core, which truncates its own.
#pragma once

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"
#include "paged_select.cuh"

namespace b200 {

constexpr int kPaHeads = 8;   // query heads of one KV head handled together
constexpr int kPaTok = 16;    // positions per unit
constexpr int kPaCtas = 148;  // CTAs of a full grid: one per SM

// Warps per CTA and ring stages per warp: 192 KB of ring in every case.
B200_HD constexpr int pa_warps(int D) { return D == 64 ? 12 : D == 128 ? 8 : 4; }
B200_HD constexpr int pa_stages(int D) { return D == 64 ? 4 : 3; }
// Floats of one piece: o [8][D], m [8], l [8], mask reference.
B200_HD constexpr int pa_piece(int D) { return kPaHeads * D + 2 * kPaHeads + 4; }
B200_HD constexpr int pa_tile(int D) { return kPaTok * D * 2; }

// Bookkeeping beside the ring and the pieces in shared memory.
template <int W, int S>
struct PaShared {
    int part[W], base[W];       // prefix-sum partials; first unit of the sequence a warp starts in
    int seq[W];                 // the sequence a warp starts in
    int from[2 * W];            // first unit of a piece's segment
    int seg[2 * W], nu[2 * W];  // a piece's segment (-1: no piece) and its units
    unsigned valid[W][S], live[W][S];  // positions of a stage that exist; that the mask leaves in
    float mask[W][S][kPaTok];
    float joint[3][kPaHeads];   // a joined segment's maxima, sums, mask reference
    int last;
};
template <int D>
constexpr int pa_smem() {
    return pa_warps(D) * (pa_stages(D) * 2 * pa_tile(D) + pa_piece(D) * 4) +
           (int)sizeof(PaShared<pa_warps(D), pa_stages(D)>);
}

struct PagedAttnArgs {
    b200_paged_kv kv;
    const float* q;
    int64_t q_stride;
    const int32_t* table;
    int64_t table_stride;
    const int32_t* seq_lens;
    const uint16_t* mask;
    int64_t mask_stride;
    const int32_t* sel;
    float* out;
    float* pieces;          // [kPaCtas][2][pa_piece]
    unsigned int* tickets;  // [n_seq * n_head_kv * chunks], zero between calls
    float scale;
    int n_seq, n_head, n_sel, max_blocks, chunks;
};

__device__ __forceinline__ void pa_cp16(uint32_t dst, const void* src, bool on) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(on ? 16 : 0) : "memory");
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
__device__ __forceinline__ void pa_ldsm_t(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr)
                 : "memory");
}
template <bool BF16>
__device__ __forceinline__ void pa_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                       uint32_t b1) {
    if (BF16)
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile(
            "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
            "{%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
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

// Where a warp is in its range: unit u of nu of the segment (s, hh).
struct PaCursor {
    int s, hh, u, nu, len;
};

__device__ __forceinline__ int pa_len(const PagedAttnArgs& a, int s) {
    const int len = a.seq_lens[s];
    const int cap = a.max_blocks * a.kv.page_size;
    return len < 0 ? 0 : (len > cap ? cap : len);
}
__device__ __forceinline__ int pa_units(const PagedAttnArgs& a, int len) {
    if (a.sel != nullptr && len > 0) len = a.n_sel * a.kv.page_size;
    return (int)(((unsigned)len + kPaTok - 1) / kPaTok);
}
// To the next unit; false past the last sequence.
__device__ __forceinline__ bool pa_advance(const PagedAttnArgs& a, PaCursor& c, int hh_n) {
    if (++c.u < c.nu) return true;
    c.u = 0;
    if (++c.hh < hh_n) return true;
    c.hh = 0;
    do {
        if (++c.s >= a.n_seq) return false;
        c.len = pa_len(a, c.s);
        c.nu = pa_units(a, c.len);
    } while (c.nu == 0);
    return true;
}

// Weight of a piece with maximum m and mask reference mk against the joint
// references.
__device__ __forceinline__ float pa_rel(float m, float mk, float mk_all) {
    return m == -INFINITY ? -INFINITY : m + (mk - mk_all) * 1.44269504f;
}

// Joins n pieces of a segment (piece(i) -> address, in shared memory or,
// written by other CTAs, in global memory): put(e, v) receives the
// unnormalised values of outputs e .. e + 3, with the references and sums of
// the 8 heads in `joint`.  wgt: n x 8 floats of shared memory.  A warp per
// head finds the pieces' weights, a lane per piece; the values are then summed
// four columns a thread, in order of the pieces, eight loads in flight.
template <int D, int T, bool GLOBAL, class F, class G>
__device__ __forceinline__ void pa_join(int n, F piece, float* wgt, float (&joint)[3][kPaHeads], G put) {
    constexpr int W = T / 32, AT_M = kPaHeads * D, AT_L = AT_M + kPaHeads, AT_MK = AT_L + kPaHeads;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto ld = [](const float* p) { return GLOBAL ? __ldcg(p) : *p; };
    for (int j = warp; j < kPaHeads; j += W) {
        float mk = -INFINITY;
        for (int k = lane; k < n; k += 32) mk = fmaxf(mk, ld(piece(k) + AT_MK));
        mk = warp_max(mk);
        float m = -INFINITY;
        for (int k = lane; k < n; k += 32) m = fmaxf(m, pa_rel(ld(piece(k) + AT_M + j), ld(piece(k) + AT_MK), mk));
        m = warp_max(m);
        float l = 0.f;
        for (int k = lane; k < n; k += 32) {
            const float r = pa_rel(ld(piece(k) + AT_M + j), ld(piece(k) + AT_MK), mk);
            const float w = r == -INFINITY ? 0.f : pa_exp2(r - m);
            wgt[k * kPaHeads + j] = w;
            l += w * ld(piece(k) + AT_L + j);
        }
        l = warp_sum(l);
        if (lane == 0) joint[0][j] = m, joint[1][j] = l, joint[2][j] = mk;
    }
    __syncthreads();
    for (int e = 4 * (int)threadIdx.x; e < kPaHeads * D; e += 4 * T) {
        float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
        int k = 0;
        for (; k + 8 <= n; k += 8) {
            float4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float4* p = reinterpret_cast<const float4*>(piece(k + i) + e);
                v[i] = GLOBAL ? __ldcg(p) : *p;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float w = wgt[(k + i) * kPaHeads + e / D];
                o.x += w * v[i].x, o.y += w * v[i].y, o.z += w * v[i].z, o.w += w * v[i].w;
            }
        }
        for (; k < n; ++k) {
            const float4* p = reinterpret_cast<const float4*>(piece(k) + e);
            const float4 v = GLOBAL ? __ldcg(p) : *p;
            const float w = wgt[k * kPaHeads + e / D];
            o.x += w * v.x, o.y += w * v.y, o.z += w * v.z, o.w += w * v.w;
        }
        put(e, o);
    }
}

template <bool BF16, int D>
__global__ void __launch_bounds__(32 * pa_warps(D), 1) paged_attn_kernel(PagedAttnArgs a) {
    constexpr int W = pa_warps(D), S = pa_stages(D), T = 32 * W;
    constexpr int KT = D / 16;             // k steps of q . k, pairs of output tiles
    constexpr int LPR = D / 8;             // 16-byte lanes per row
    constexpr int RPI = 32 / LPR;          // rows per copy instruction
    constexpr int TILE = pa_tile(D), RB = 2 * D, PIECE = pa_piece(D);
    extern __shared__ __align__(128) uint8_t pa_sm[];
    PaShared<W, S>& sh = *reinterpret_cast<PaShared<W, S>*>(pa_sm + W * (S * 2 * TILE + PIECE * 4));

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    const int ps = a.kv.page_size, G = a.n_head / a.kv.n_head_kv;
    const int hh_n = a.kv.n_head_kv * a.chunks;

    // ---- the lengths' prefix sums: this CTA's range and its warps' starts ----
    const int per = (a.n_seq + T - 1) / T;
    const int s_lo = min(a.n_seq, tid * per), s_hi = min(a.n_seq, s_lo + per);
    int mine = 0;
    for (int s = s_lo; s < s_hi; ++s) {
        const int len = a.seq_lens[s];
        if (blockIdx.x == 0 && (len < 0 || len > a.max_blocks * ps)) record_status(B200_DEVSTATUS_BOUNDS);
        mine += pa_units(a, pa_len(a, s));
    }
    int incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += x;
    }
    if (lane == 31) sh.part[warp] = incl;
    if (tid < 2 * W) sh.seg[tid] = -1;
    __syncthreads();
    int total = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
        if (w < warp) incl += sh.part[w];
        total += sh.part[w];
    }
    total *= hh_n;
    const int per_cta = max((int)((total + gridDim.x - 1u) / gridDim.x), W);
    const int cb = (int)min((unsigned)total, (unsigned)per_cta * blockIdx.x);
    const int ce = (int)min((unsigned)total, (unsigned)cb + (unsigned)per_cta);
    {
        int at = (incl - mine) * hh_n;
        for (int s = s_lo; s < s_hi; ++s) {
            const int end = at + pa_units(a, pa_len(a, s)) * hh_n;
            if (end > cb && at < ce)
                for (int w = 0; w < W; ++w) {
                    const int b = cb + (ce - cb) * w / W;
                    if (b >= at && b < end) sh.seq[w] = s, sh.base[w] = at;
                }
            at = end;
        }
    }
    // sequences without a unit
    for (int s = blockIdx.x; s < a.n_seq; s += gridDim.x)
        if (pa_len(a, s) == 0)
            for (int e = tid; e < a.n_head * D; e += T) a.out[(int64_t)s * a.n_head * D + e] = 0.f;
    __syncthreads();
    if (cb >= ce) return;

    const uint32_t ring = smem_u32(pa_sm) + warp * (S * 2 * TILE);
    float* const heads = reinterpret_cast<float*>(pa_sm + W * S * 2 * TILE);
    float* const head_piece = heads + warp * PIECE;  // a segment begun by an earlier warp
    float* const tail_piece = reinterpret_cast<float*>(pa_sm + warp * (S * 2 * TILE));  // one left to a later warp
    const int fb = cb + (ce - cb) * warp / W, fe = cb + (ce - cb) * (warp + 1) / W;

    if (fb < fe) {
        PaCursor in, cur;
        in.s = sh.seq[warp];
        in.len = pa_len(a, in.s);
        in.nu = pa_units(a, in.len);
        in.hh = (fb - sh.base[warp]) / in.nu;
        in.u = (fb - sh.base[warp]) - in.hh * in.nu;
        cur = in;
        int seg_from = fb - in.u;  // first unit of the current segment
        int to_issue = fe - fb, to_do = to_issue;

        // ---- producer: this lane looks after token lane & 15 of a unit ----
        const int q16 = kPaTok / ps, r16 = kPaTok % ps;
        int bi = 0, row = 0, w0 = 0;     // its block (list entry) and row; first entry of the page window
        int p0 = -1, p1 = -1, b0 = -1, b1 = -1;  // pages and blocks of entries w0 + lane, w0 + 32 + lane
        bool fresh = true;
        float mask_pending = 0.f;
        int mask_stage = -1;
        unsigned valid_pending = 0;
        auto entry = [&](int e, int& page, int& blk) {
            blk = e, page = -1;
            const int nb = (int)(((unsigned)in.len + (unsigned)ps - 1u) / (unsigned)ps);
            if (a.sel != nullptr) {
                const int64_t hk = (int64_t)in.s * a.kv.n_head_kv + in.hh / a.chunks;
                blk = e < a.n_sel ? a.sel[hk * a.n_sel + e] : -1;
            }
            if (blk >= 0 && blk < nb) {
                page = a.table[in.s * a.table_stride + blk];
                if ((unsigned)page >= (unsigned)a.kv.n_pages) {
                    record_status(B200_DEVSTATUS_BOUNDS);
                    page = -1;
                }
            }
        };
        auto flush_mask = [&]() {
            if (mask_stage >= 0) {
                const unsigned live = __ballot_sync(0xffffffffu, mask_pending != -INFINITY) & valid_pending;
                if (lane < kPaTok) sh.mask[warp][mask_stage][lane] = mask_pending;
                if (lane == 0) sh.live[warp][mask_stage] = live;
                mask_stage = -1;
            }
        };
        auto issue = [&](int stage) {
            if (a.mask != nullptr) flush_mask();
            if (to_issue > 0) {
                if (fresh) {
                    const unsigned vt = (unsigned)in.u * kPaTok + (lane & 15);
                    bi = (int)(vt / (unsigned)ps);
                    row = (int)(vt % (unsigned)ps);
                    w0 = (int)((unsigned)in.u * kPaTok / (unsigned)ps);
                    entry(w0 + lane, p0, b0);
                    entry(w0 + 32 + lane, p1, b1);
                    fresh = false;
                } else {
                    bi += q16;
                    row += r16;
                    if (row >= ps) row -= ps, ++bi;
                    if (__shfl_sync(0xffffffffu, bi, 0) >= w0 + 32) {
                        w0 += 32;
                        p0 = p1, b0 = b1;
                        entry(w0 + 32 + lane, p1, b1);
                    }
                }
                const int x = bi - w0;  // 0 .. 47
                const int pa = __shfl_sync(0xffffffffu, p0, x & 31), pb = __shfl_sync(0xffffffffu, p1, x & 31);
                const int page = x < 32 ? pa : pb;
                int blk = bi;
                if (a.sel != nullptr) {
                    const int ba = __shfl_sync(0xffffffffu, b0, x & 31), bb = __shfl_sync(0xffffffffu, b1, x & 31);
                    blk = x < 32 ? ba : bb;
                }
                const bool ok = page >= 0 && row < in.len - blk * ps;
                const unsigned valid = __ballot_sync(0xffffffffu, ok) & 0xffffu;
                const int head = in.hh / a.chunks;
                const long long ko = ok ? page * a.kv.k_page + row * a.kv.k_row + head * a.kv.k_head : 0;
                const long long vo = ok ? page * a.kv.v_page + row * a.kv.v_row + head * a.kv.v_head : 0;
                if (lane == 0) sh.valid[warp][stage] = valid;
                if (a.mask != nullptr) {
                    mask_pending = ok ? h2f(a.mask[in.s * a.mask_stride + (int64_t)blk * ps + row]) : -INFINITY;
                    mask_stage = stage;
                    valid_pending = valid;
                }
                const uint32_t kst = ring + stage * (2 * TILE), c = lane % LPR;
                const uint8_t* kp = static_cast<const uint8_t*>(a.kv.k) + 16 * c;
                const uint8_t* vp = static_cast<const uint8_t*>(a.kv.v) + 16 * c;
#pragma unroll
                for (int i = 0; i < kPaTok / RPI; ++i) {
                    const int r = i * RPI + lane / LPR;
                    const long long kr = __shfl_sync(0xffffffffu, ko, r), vr = __shfl_sync(0xffffffffu, vo, r);
                    const uint32_t d = kst + r * RB + ((c ^ (r & 7)) << 4);
                    const bool on = (valid >> r) & 1;
                    pa_cp16(d, kp + kr, on);
                    pa_cp16(d + TILE, vp + vr, on);
                }
                --to_issue;
                const int s_was = in.s, hh_was = in.hh;
                if (to_issue > 0 && !pa_advance(a, in, hh_n)) to_issue = 0;
                fresh = in.s != s_was || in.hh != hh_was;
            }
            pa_commit();
        };
#pragma unroll
        for (int st = 0; st < S - 1; ++st) issue(st);

        // ---- consumer: this thread holds head g, positions 2 t4, 2 t4 + 1 (+ 8) ----
        uint32_t qf[KT][4], q3[BF16 ? KT : 1][2];
        float o[2 * KT][2], m = -INFINITY, l = 0.f, mk = -INFINITY, f = 0.f;
        auto load_q = [&]() {
            const int chunk = cur.hh % a.chunks, head = cur.hh / a.chunks;
            const int j = chunk * kPaHeads + g;
            const float* qr = a.q + cur.s * a.q_stride + (int64_t)(head * G + (j < G ? j : 0)) * D + 2 * t4;
            float2 x[2 * KT];
            float amax = 0.f;
#pragma unroll
            for (int i = 0; i < 2 * KT; ++i) {
                x[i] = *reinterpret_cast<const float2*>(qr + 8 * i);
                if (j >= G) x[i] = make_float2(0.f, 0.f);
                amax = fmaxf(amax, fmaxf(fabsf(x[i].x), fabsf(x[i].y)));
            }
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
            // q 2^-ex has its largest entry in [1, 2)
            const int ex = min(max((int)(__float_as_uint(amax) >> 23) - 127, -120), 120);
            const float up = __uint_as_float((unsigned)(127 - ex) << 23);
            f = a.scale * 1.44269504f * __uint_as_float((unsigned)(127 + ex) << 23);
#pragma unroll
            for (int i = 0; i < 2 * KT; ++i) {
                x[i].x *= up, x[i].y *= up;
                qf[i >> 1][2 * (i & 1)] = pa_split<BF16>(x[i].x, x[i].y);
                qf[i >> 1][2 * (i & 1) + 1] = pa_split<BF16>(x[i].x, x[i].y);
                if (BF16) q3[i >> 1][i & 1] = pa_split<BF16>(x[i].x, x[i].y);
            }
#pragma unroll
            for (int i = 0; i < 2 * KT; ++i) o[i][0] = o[i][1] = 0.f;
            m = -INFINITY, l = 0.f, mk = a.mask != nullptr ? -INFINITY : 0.f;
        };
        load_q();
        int stage = 0;
        const int mi = lane >> 3, ri = lane & 7;
        for (; to_do > 0; --to_do) {
            pa_wait<S - 2>();
            __syncwarp();
            issue(stage == 0 ? S - 1 : stage - 1);
            const unsigned valid = sh.valid[warp][stage];
            const unsigned live = a.mask != nullptr ? sh.live[warp][stage] : valid;
            const uint32_t kst = ring + stage * (2 * TILE), vst = kst + TILE;
            if (live) {
                if (live != valid) {  // masked positions: their values may be anything
                    for (int r = 0; r < kPaTok; ++r)
                        if (((valid & ~live) >> r) & 1)
                            for (int c = lane; c < RB / 16; c += 32)
                                asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(vst + r * RB + 16 * c),
                                             "r"(0u)
                                             : "memory");
                    __syncwarp();
                }
                // S = q K^T: 8 heads (high parts, low parts) x 16 positions
                float sc[2][4] = {};
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    uint32_t b[4];  // positions 0-7: dims 0-7, 8-15; positions 8-15: the same
                    const int r = 8 * (mi >> 1) + ri, c = 2 * kt + (mi & 1);
                    pa_ldsm(b, kst + r * RB + ((c ^ ri) << 4));
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        pa_mma<BF16>(sc[n], qf[kt][0], qf[kt][1], qf[kt][2], qf[kt][3], b[2 * n], b[2 * n + 1]);
                        if (BF16) pa_mma<BF16>(sc[n], q3[kt][0], 0u, q3[kt][1], 0u, b[2 * n], b[2 * n + 1]);
                    }
                }
                float x[4], bias[4] = {};
#pragma unroll
                for (int i = 0; i < 4; ++i) x[i] = sc[i >> 1][i & 1] + sc[i >> 1][2 + (i & 1)];
                if (a.mask != nullptr) {
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        bias[i] = sh.mask[warp][stage][8 * (i >> 1) + 2 * t4 + (i & 1)];
                        top = fmaxf(top, bias[i]);
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (top > mk) {
                        m = pa_rel(m, mk, top);
                        mk = top;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) bias[i] = (bias[i] - mk) * 1.44269504f;
                }
                float top = -INFINITY;
                bool on[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    on[i] = (live >> (8 * (i >> 1) + 2 * t4 + (i & 1))) & 1;
                    if (on[i]) top = fmaxf(top, fmaf(x[i], f, bias[i]));
                }
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                const float mn = fmaxf(m, top);
                const float corr = pa_exp2(m - mn);  // 0 at the first unit: m is -inf, mn is not
                m = mn;
                float w[4], sum = 0.f;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    w[i] = on[i] ? pa_exp2(fmaf(x[i], f, bias[i] - mn)) * 4096.f : 0.f;
                    sum += w[i];
                }
                l = l * corr + sum;
                // O += w V: the pieces of w as they stand are the A operand
                uint32_t wa[4], w3[2];
                wa[0] = pa_split<BF16>(w[0], w[1]);
                wa[1] = pa_split<BF16>(w[0], w[1]);
                wa[2] = pa_split<BF16>(w[2], w[3]);
                wa[3] = pa_split<BF16>(w[2], w[3]);
                if (BF16) w3[0] = pa_split<BF16>(w[0], w[1]), w3[1] = pa_split<BF16>(w[2], w[3]);
#pragma unroll
                for (int kt = 0; kt < KT; ++kt) {
                    uint32_t b[4];  // dims 16 kt .. + 7: positions 0-7, 8-15; the next 8 dims
                    const int r = 8 * (mi & 1) + ri, c = 2 * kt + (mi >> 1);
                    pa_ldsm_t(b, vst + r * RB + ((c ^ ri) << 4));
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        float d[4] = {};
                        pa_mma<BF16>(d, wa[0], wa[1], wa[2], wa[3], b[2 * n], b[2 * n + 1]);
                        if (BF16) pa_mma<BF16>(d, w3[0], 0u, w3[1], 0u, b[2 * n], b[2 * n + 1]);
                        o[2 * kt + n][0] = fmaf(o[2 * kt + n][0], corr, d[0] + d[2]);
                        o[2 * kt + n][1] = fmaf(o[2 * kt + n][1], corr, d[1] + d[3]);
                    }
                }
            }
            stage = stage + 1 == S ? 0 : stage + 1;

            const bool seg_end = cur.u + 1 == cur.nu;
            if (seg_end || to_do == 1) {
                l += __shfl_xor_sync(0xffffffffu, l, 1);
                l += __shfl_xor_sync(0xffffffffu, l, 2);
                if (seg_end && seg_from >= fb) {  // the whole segment
                    const int chunk = cur.hh % a.chunks, head = cur.hh / a.chunks;
                    const int j = chunk * kPaHeads + g;
                    const float inv = l > 0.f ? 1.f / l : 0.f;
                    if (j < G) {
                        float* dst = a.out + ((int64_t)cur.s * a.n_head + head * G + j) * D + 2 * t4;
#pragma unroll
                        for (int i = 0; i < 2 * KT; ++i)
                            *reinterpret_cast<float2*>(dst + 8 * i) = make_float2(o[i][0] * inv, o[i][1] * inv);
                    }
                } else {
                    const bool tail = !seg_end;
                    if (tail) {  // the last piece of this warp: its ring is free
                        pa_wait<0>();
                        __syncwarp();
                    }
                    float* p = tail ? tail_piece : head_piece;
#pragma unroll
                    for (int i = 0; i < 2 * KT; ++i)
                        *reinterpret_cast<float2*>(p + g * D + 8 * i + 2 * t4) = make_float2(o[i][0], o[i][1]);
                    if (t4 == 0) p[kPaHeads * D + g] = m, p[kPaHeads * D + kPaHeads + g] = l;
                    if (lane == 0) {
                        p[kPaHeads * D + 2 * kPaHeads] = mk;
                        sh.seg[2 * warp + tail] = cur.s * hh_n + cur.hh;
                        sh.from[2 * warp + tail] = seg_from;
                        sh.nu[2 * warp + tail] = cur.nu;
                    }
                }
            }
            if (to_do > 1) {
                if (seg_end) seg_from += cur.nu;
                if (!pa_advance(a, cur, hh_n)) break;
                if (seg_end) load_q();
            }
        }
        pa_wait<0>();
    }
    __syncthreads();

    // ---- join the pieces of cut segments ----
    auto piece_at = [&](int i) -> float* {
        return (i & 1) ? reinterpret_cast<float*>(pa_sm + (i >> 1) * (S * 2 * TILE)) : heads + (i >> 1) * PIECE;
    };
    // weights of the pieces being joined: in warp 0's ring, behind its tail piece
    float* const wgt = reinterpret_cast<float*>(pa_sm + align256(PIECE * 4));
    static_assert(kPaCtas * kPaHeads * 4 + PIECE * 4 + 256 <= S * 2 * TILE, "weights beside the tail piece");
    for (int i = 0; i < 2 * W;) {
        const int seg = sh.seg[i];
        if (seg < 0) {
            ++i;
            continue;
        }
        int list[2 * W], n = 0;
        for (; i < 2 * W && (sh.seg[i] == seg || sh.seg[i] < 0); ++i)
            if (sh.seg[i] == seg) list[n++] = i;
        const int from = sh.from[list[0]], end = from + sh.nu[list[0]];
        const bool whole = from >= cb && end <= ce;
        const int s = seg / hh_n, hh = seg % hh_n, head = hh / a.chunks, j0 = (hh % a.chunks) * kPaHeads;
        float* out = a.out + ((int64_t)s * a.n_head + head * G + j0) * D;
        float* mine_g = a.pieces + (int64_t)(2 * blockIdx.x + (from >= cb ? 1 : 0)) * PIECE;
        auto finish = [&](int e, float4 o) {
            const float l = sh.joint[1][e / D], inv = l > 0.f ? 1.f / l : 0.f;
            if (j0 + e / D < G)
                *reinterpret_cast<float4*>(out + e) = make_float4(o.x * inv, o.y * inv, o.z * inv, o.w * inv);
        };
        pa_join<D, T, false>(n, [&](int k) -> const float* { return piece_at(list[k]); }, wgt, sh.joint,
                             [&](int e, float4 o) {
                                 if (whole) finish(e, o);
                                 else __stcg(reinterpret_cast<float4*>(mine_g + e), o);
                             });
        if (!whole) {
            if (tid < 2 * kPaHeads) __stcg(mine_g + kPaHeads * D + tid, sh.joint[tid / kPaHeads][tid % kPaHeads]);
            if (tid == 0) __stcg(mine_g + kPaHeads * D + 2 * kPaHeads, sh.joint[2][0]);
            const int c0 = from / per_cta, c1 = (end - 1) / per_cta;
            __threadfence();
            __syncthreads();
            if (tid == 0) sh.last = atomicAdd(a.tickets + seg, 1u) == (unsigned)(c1 - c0);
            __syncthreads();
            if (sh.last) {
                __threadfence();
                pa_join<D, T, true>(
                    c1 - c0 + 1,
                    [&](int k) -> const float* { return a.pieces + (int64_t)(2 * (c0 + k) + (k == 0 ? 1 : 0)) * PIECE; },
                    wgt, sh.joint, finish);
                if (tid == 0) a.tickets[seg] = 0u;
            }
        }
        __syncthreads();  // wgt and joint are free again
    }
}

}  // namespace b200
