// paged_attn.cuh -- attention of one new token per sequence over a paged
// key-value cache, split over the cache's length and joined.
//
//   out_j = sum_p w_p v_p / sum_p w_p,  w_p = 2^(f q_j . k_p + bias_p - m)
//
// with f = scale log2(e) and m the running maximum.  Per cached token and KV
// head K and V are 4 D bytes for 4 D G flops (G <= 16 query heads a pass), so
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
// ring runs ahead across segment borders.  What decides the rate at the power
// cap, where the SM clock is 1.5 GHz, is the instructions per unit (about 375
// with 16-row pages; with 539 the same stream was 17% slower), hence the fixed
// copy steps and offsets and the single counter per side below.
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
// two into f16's range, w (f16 pages) by 2^12 out of f16's subnormals.  bf16 takes a third
// part in a second instruction.  Sums over positions are f32 additions
// outside the tensor core, which truncates its own.  (tcgen05 has no use for 8
// rows of heads; mma.sync keeps the tensor pipe 19% busy.)
//
// Measured on a B200 whose copy runs at 6458 GB/s, 64/8 heads x 128, f16: 8
// sequences of 32768 to 131072 tokens 505 us, 6.76 TB/s; 48 of 0 to 8192 123 us,
// 5.83 TB/s; one of 4160 14.9 us, of which the start takes 3 us, two units per
// warp 3 us and joining the pieces 5 us.
#pragma once

#include "../../include/b200_paged.h"
#include "args.h"
#include "common.cuh"
#include "paged_work.cuh"

namespace b200 {

constexpr int kPaHeads = 8;   // query heads of one KV head handled together

// Groups of 8 query heads a pass takes (NC): one up to 8 query heads per KV
// head, else two, so that 9 to 16 read the cache once (head dim 256 lacks the
// registers).
B200_HD constexpr int pa_groups(int D, int G) { return G > kPaHeads && D < 256 ? 2 : 1; }
// Warps per CTA and ring stages per warp: up to 192 KB of ring.
B200_HD constexpr int pa_warps(int D, int NC = 1) {
    return NC == 2 ? (D == 64 ? 8 : 6) : D == 64 ? 12 : D == 128 ? 8 : 4;
}
B200_HD constexpr int pa_stages(int D, int NC = 1) { return NC == 2 ? (D == 64 ? 5 : 3) : D == 64 ? 4 : 3; }
// Floats of one piece: o [8 NC][D], m [8 NC], l [8 NC], mask reference.
B200_HD constexpr int pa_piece(int D, int NC = 1) { return kPaHeads * NC * (D + 2) + 4; }
// Bytes of the workspace's piece area, the same for every shape: the tickets
// behind it are zero whatever shapes used the workspace before.
B200_HD constexpr size_t pa_piece_area() {
    int most = pa_piece(256);
    for (int D = 64; D <= 128; D *= 2)
        if (pa_piece(D, 2) > most) most = pa_piece(D, 2);
    return ((size_t)kPaCtas * 2 * most * sizeof(float) + 255) & ~(size_t)255;
}
B200_HD constexpr int pa_tile(int D) { return kPaTok * D * 2; }

// Bookkeeping beside the ring and the pieces in shared memory.
template <int W, int S>
struct PaShared {
    PaRangeShared<W> range;
    // pieces of a warp, [0] of a segment begun by an earlier warp, [1] of one left
    // to a later warp: segment (-1: none), its first unit and length, its first
    // row of the output and rows
    int seg[2][W], from[2][W], nu[2][W], row[2][W], rows[2][W];
    unsigned valid[W][S], live[W][S];  // positions of a stage that exist; that the mask leaves in
    float mask[W][S][kPaTok];
};
template <int D, int NC>
constexpr int pa_smem() {
    return pa_warps(D, NC) * (pa_stages(D, NC) * 2 * pa_tile(D) + pa_piece(D, NC) * 4) +
           (int)sizeof(PaShared<pa_warps(D, NC), pa_stages(D, NC)>);
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
    unsigned int* tickets;  // [n_seq * n_head_kv * chunks][8 NC], zero between calls
    float scale;
    int n_seq, n_head, n_sel, max_blocks, chunks;
    int group;              // query heads per KV head
    int unit_blocks, unit_rows, aligned;  // 16 / page_size, 16 % page_size, page_size % 16 == 0
    int near_rows;          // 16 rows of a page span less than 2^31 bytes
    int same_rows;          // K and V have the same page and row strides
};

// Where a warp is in its range: unit u of nu of the segment (s, head, chunk).
struct PaCursor {
    int s, head, chunk, u, nu, len;
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
// To the first unit of the next segment; false past the last sequence.
__device__ __forceinline__ bool pa_next(const PagedAttnArgs& a, PaCursor& c) {
    c.u = 0;
    if (++c.chunk < a.chunks) return true;
    c.chunk = 0;
    if (++c.head < a.kv.n_head_kv) return true;
    c.head = 0;
    do {
        if (++c.s >= a.n_seq) return false;
        c.len = pa_len(a, c.s);
        c.nu = pa_units(a, c.len);
    } while (c.nu == 0);
    return true;
}

// Maximum m of a piece with mask reference mk, against the reference mk_all.
__device__ __forceinline__ float pa_rel(float m, float mk, float mk_all) {
    return m == -INFINITY ? -INFINITY : m + (mk - mk_all) * 1.44269504f;
}

__device__ __forceinline__ float4 pa_lds4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
                 : "r"(addr)
                 : "memory");
    return v;
}

// One head of a segment being joined by one warp: the unnormalised values of
// columns 4 (lane + 32 i) .. + 3 (D = 64: lanes 16-31 idle), their maximum,
// sum and mask reference.
template <int D>
struct PaJoint {
    static constexpr int NV = (D + 127) / 128;
    float4 v[NV];
    float m = -INFINITY, l = 0.f, mk = -INFINITY;

    // Adds n <= 32 pieces in order: lane k brings piece k's maximum, sum and
    // mask reference; its row of values is in shared memory at row + k * stride
    // (piece `odd` at odd_row).
    __device__ __forceinline__ void add(int n, float pm, float pl, float pk, bool masked, uint32_t row,
                                        uint32_t stride, int odd, uint32_t odd_row) {
        const int lane = threadIdx.x & 31;
        const float nk = masked ? fmaxf(mk, pa_warp_max(pk)) : 0.f;
        if (masked) pm = pa_rel(pm, pk, nk), m = pa_rel(m, mk, nk);
        mk = nk;
        const float nm = fmaxf(m, pa_warp_max(pm));
        const float old = m == -INFINITY ? 0.f : pa_exp2(m - nm);
        const float w = pm == -INFINITY ? 0.f : pa_exp2(pm - nm);
        m = nm;
        l = l * old + warp_sum(w * pl);
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i].x *= old, v[i].y *= old, v[i].z *= old, v[i].w *= old;
        const uint32_t col = 16 * (lane % (D / 4 < 32 ? D / 4 : 32));
#pragma unroll 4
        for (int k = 0; k < n; ++k) {
            const float wk = __shfl_sync(0xffffffffu, w, k);
            const uint32_t at = (k == odd ? odd_row : row + k * stride) + col;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                const float4 x = pa_lds4(at + 512 * i);
                v[i].x += wk * x.x, v[i].y += wk * x.y, v[i].z += wk * x.z, v[i].w += wk * x.w;
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < NV; ++i) v[i] = make_float4(0.f, 0.f, 0.f, 0.f);
    }
};

// Sequence s, KV head `head`, chunk `chunk` of its query heads, positions (of
// the sequence or of the listed blocks) first .. first + n - 1, again in f32
// products of whole values: for the segments in which the split products met
// an infinity or a NaN.  inf * high + inf * low is NaN where the low part is
// zero or of the other sign, and a unit whose scores are all -inf has no
// reference for its weights.  One warp, a head at a time; a lane has a position
// for its score and D / 32 columns for the values.  `out`: the output rows where
// `whole`, else the piece.  Nothing here is tuned: 48 ragged sequences with an
// infinite key in every page take 6.8 ms instead of 121 us.  In the loop, not
// behind it, since that is where the finite case pays least (one sequence of
// 4160 14.5 -> 14.9 us; behind the loop 48 ragged 120.5 -> 124 us, here 121).
template <bool BF16, int D, int NC>
__device__ __forceinline__ void pa_plain(const PagedAttnArgs& a, int s, int head, int chunk, int len, int first,
                                         int n, bool whole, float* out, float w_up) {
    constexpr int NH = kPaHeads * NC, E = D / 32;
    const int lane = threadIdx.x & 31, ps = a.kv.page_size, G = a.group;
    const int nb = (int)(((unsigned)len + (unsigned)ps - 1u) / (unsigned)ps);
    const uint8_t* kh = static_cast<const uint8_t*>(a.kv.k) + head * a.kv.k_head;
    const uint8_t* vh = static_cast<const uint8_t*>(a.kv.v) + head * a.kv.v_head + 2 * E * lane;
    const int32_t* table = a.table + s * a.table_stride;
    // position first + i: false where there is none or the mask leaves it out
    auto find = [&](int i, int& page, int& row, float& bias) -> bool {
        if (i >= n) return false;
        const unsigned p = (unsigned)first + (unsigned)i;
        int b = (int)(p / (unsigned)ps);
        row = (int)(p - (unsigned)b * (unsigned)ps);
        if (a.sel != nullptr) b = b < a.n_sel ? a.sel[((int64_t)s * a.kv.n_head_kv + head) * a.n_sel + b] : -1;
        if ((unsigned)b >= (unsigned)nb || row >= len - b * ps) return false;
        page = table[b];
        if ((unsigned)page >= (unsigned)a.kv.n_pages) return false;
        if (a.mask != nullptr) bias = h2f(a.mask[s * a.mask_stride + (int64_t)b * ps + row]);
        return bias != -INFINITY;
    };
    float mk = a.mask != nullptr ? -INFINITY : 0.f;
    if (a.mask != nullptr)
        for (int i = 0; i < n; i += 32) {
            int page = 0, row = 0;
            float bias = 0.f;
            mk = fmaxf(mk, pa_warp_max(find(i + lane, page, row, bias) ? bias : -INFINITY));
        }
#pragma unroll 1
    for (int r = 0; r < NH && chunk * NH + r < G; ++r) {
        const int64_t j = (int64_t)head * G + chunk * NH + r;
        const float* q = a.q + s * a.q_stride + j * D;
        float big = 0.f;
        for (int d = lane; d < D; d += 32) big = fmaxf(big, fabsf(q[d]));
        const int ex = min(max((int)(__float_as_uint(pa_warp_max(big)) >> 23) - 127, -120), 120);
        const float up = __uint_as_float((unsigned)(127 - ex) << 23);
        const float f = a.scale * 1.44269504f * __uint_as_float((unsigned)(127 + ex) << 23);
        float m = -INFINITY, l = 0.f, acc[E] = {};
#pragma unroll 1
        for (int i = 0; i < n; i += 32) {
            int page = 0, row = 0;
            float x = 0.f, bias = 0.f;
            const bool on = find(i + lane, page, row, bias);
            if (on) {
                const uint4* k = reinterpret_cast<const uint4*>(kh + page * a.kv.k_page + row * a.kv.k_row);
                float part[8] = {};
#pragma unroll 1
                for (int d = 0; d < D / 8; ++d) {
                    const uint4 w = k[d];
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float2 y = unpack16<BF16>(ws[e]);
                        part[2 * e] += q[8 * d + 2 * e] * up * y.x;
                        part[2 * e + 1] += q[8 * d + 2 * e + 1] * up * y.y;
                    }
                }
                x = ((part[0] + part[1]) + (part[2] + part[3])) + ((part[4] + part[5]) + (part[6] + part[7]));
                x = fmaf(x, f, (bias - mk) * 1.44269504f);
            }
            const float nm = fmaxf(m, pa_warp_max(on ? x : -INFINITY));
            const float old = m == -INFINITY ? 0.f : pa_exp2(m - nm);
            const float w = !on || x == -INFINITY ? 0.f : pa_exp2(x - nm) * w_up;
            m = nm;
            l = l * old + warp_sum(w);
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] *= old;
            for (unsigned todo = __ballot_sync(0xffffffffu, on); todo != 0; todo &= todo - 1) {
                const int y = __ffs(todo) - 1;
                const float wy = __shfl_sync(0xffffffffu, w, y);
                const int64_t at = __shfl_sync(0xffffffffu, page, y) * a.kv.v_page + __shfl_sync(0xffffffffu, row, y) * a.kv.v_row;
                const uint32_t* v = reinterpret_cast<const uint32_t*>(vh + at);
#pragma unroll
                for (int e = 0; e < E; e += 2) {
                    const float2 t = unpack16<BF16>(v[e / 2]);
                    acc[e] += wy * t.x, acc[e + 1] += wy * t.y;
                }
            }
        }
        const float scale = !whole ? 1.f : l > 0.f ? 1.f / l : 0.f;
        float* o = out + r * D + E * lane;
#pragma unroll
        for (int e = 0; e < E; ++e) o[e] = acc[e] * scale;
        if (!whole && lane == 0) out[NH * D + r] = m, out[NH * D + NH + r] = l;
    }
    if (!whole && lane == 0) out[NH * D + 2 * NH] = mk;
    __syncwarp();
}

template <bool BF16, int D, int NC, bool MASK>
__global__ void __launch_bounds__(32 * pa_warps(D, NC), 1) paged_attn_kernel(const __grid_constant__ PagedAttnArgs a) {
    constexpr int W = pa_warps(D, NC), S = pa_stages(D, NC), T = 32 * W;
    constexpr int NH = kPaHeads * NC;      // query heads of a pass
    constexpr int KT = D / 16;             // k steps of q . k, pairs of output tiles
    constexpr int LPR = D / 8;             // 16-byte lanes per row
    constexpr int RPI = 32 / LPR;          // rows per copy instruction
    constexpr int TILE = pa_tile(D), RB = 2 * D, PIECE = pa_piece(D, NC);
    constexpr bool EARLY_Q = NC == 1 && D <= 128;  // queries fetched before a unit is issued, if registers allow
    extern __shared__ __align__(128) uint8_t pa_sm[];
    PaShared<W, S>& sh = *reinterpret_cast<PaShared<W, S>*>(pa_sm + W * (S * 2 * TILE + PIECE * 4));

    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int g = lane >> 2, t4 = lane & 3;
    const int ps = a.kv.page_size, G = a.group;
    const int hh_n = a.kv.n_head_kv * a.chunks;

    if (tid < W) sh.seg[0][tid] = -1, sh.seg[1][tid] = -1;
    if (blockIdx.x == 0)
        for (int s = tid; s < a.n_seq; s += T)
            if (a.seq_lens[s] < 0 || a.seq_lens[s] > a.max_blocks * ps) record_status(B200_DEVSTATUS_BOUNDS);
    const PaRange<W> range(sh.range, a.n_seq, hh_n, [&](int s) { return pa_units(a, pa_len(a, s)); });
    const int cb = range.cb, ce = range.ce, per_cta = range.per_cta, fb = range.fb, fe = range.fe;
    // sequences without a unit
    for (int s = blockIdx.x; s < a.n_seq; s += gridDim.x)
        if (pa_len(a, s) == 0)
            for (int e = tid; e < a.n_head * D; e += T) a.out[(int64_t)s * a.n_head * D + e] = 0.f;
    if (cb >= ce) return;

    const uint32_t ring = smem_u32(pa_sm) + warp * (S * 2 * TILE);
    // Pieces: of a segment begun by an earlier warp, of one left to a later warp
    // (that one in the ring, which is free by then).
    auto head_piece = [&](int w) -> float* {
        return reinterpret_cast<float*>(pa_sm + W * S * 2 * TILE + w * PIECE * 4);
    };
    auto tail_piece = [&](int w) -> float* { return reinterpret_cast<float*>(pa_sm + w * (S * 2 * TILE)); };

    PaCursor in;
    in.s = range.seq0;
    in.len = fb < fe ? pa_len(a, in.s) : 0;
    in.nu = pa_units(a, in.len);
    // (lengths that change while the kernel runs give wrong results and tickets
    // that do not end at zero, but no address outside the tensors: a position that
    // does not fit ends the warp, and no piece is looked for past the grid)
    const int hh0 = in.nu > 0 ? (fb - range.base0) / in.nu : hh_n;
    if ((unsigned)hh0 < (unsigned)hh_n) {
        in.u = (fb - range.base0) - hh0 * in.nu;
        in.head = a.chunks == 1 ? hh0 : hh0 / a.chunks;
        in.chunk = hh0 - in.head * a.chunks;
        PaCursor cur = in;
        int seg_from = fb - in.u;  // first unit of the current segment
        int to_issue = fe - fb, to_do = to_issue;

        // the first segment's queries, on their way while the page table is read
        float2 qx[NC][2 * KT];
        auto fetch_q = [&]() {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const int j = cur.chunk * NH + kPaHeads * c + g;
                const float* qr = a.q + cur.s * a.q_stride + (int64_t)(cur.head * G + (j < G ? j : 0)) * D + 2 * t4;
#pragma unroll
                for (int i = 0; i < 2 * KT; ++i) qx[c][i] = *reinterpret_cast<const float2*>(qr + 8 * i);
            }
        };

        // ---- producer: this lane looks after token lane & 15 of a unit ----
        const int q16 = a.unit_blocks, r16 = a.unit_rows;  // 16 = q16 ps + r16
        const bool aligned = a.aligned != 0;               // a unit lies in one page
        const uint32_t lc = lane % LPR, lr = lane / LPR;  // this lane's 16 bytes of a row, its row of a copy
        // Offsets of pages and rows in 16-byte steps, in 32 bits: K and V span less
        // than 64 GiB each.  A unit of one page is copied at fixed steps from its
        // first row (near_rows), any other row by row.
        const bool near_rows = aligned && a.near_rows;
        constexpr int SW = 8 / RPI;  // the swizzle repeats after 8 rows
        uint32_t dst_of[SW];
#pragma unroll
        for (int i = 0; i < SW; ++i) dst_of[i] = ring + lr * RB + ((lc ^ ((i * RPI + lr) & 7)) << 4);
        const uint32_t kp16 = (uint32_t)(a.kv.k_page >> 4), kr16 = (uint32_t)(a.kv.k_row >> 4);
        const uint32_t vp16 = (uint32_t)(a.kv.v_page >> 4), vr16 = (uint32_t)(a.kv.v_row >> 4);
        const uint32_t k_step = (uint32_t)(RPI * a.kv.k_row), v_step = (uint32_t)(RPI * a.kv.v_row);
        const uint32_t k_lane = (uint32_t)(lr * a.kv.k_row) + 16 * lc, v_lane = (uint32_t)(lr * a.kv.v_row) + 16 * lc;
        int bi = 0, row = 0, w0 = 0;     // its block (list entry) and row; first entry of the page window
        int p0 = -1, p1 = -1, b0 = -1, b1 = -1;  // pages and blocks of entries w0 + lane, w0 + 32 + lane
        int run = 0;                     // units to go in this segment and this window
        bool fresh = true;
        const uint8_t *k_head = nullptr, *v_head = nullptr;
        uint16_t mask_pending = 0;  // as loaded: converting it here would wait for it
        int mask_stage = -1;
        unsigned valid_pending = 0;
        // entries e and e + 32 of the block list (only_second: the second alone);
        // the loads of both go out before either is looked at
        auto window = [&](int e, bool only_second) {
            const int nb = (int)(((unsigned)in.len + (unsigned)ps - 1u) / (unsigned)ps);
            int x0 = e, x1 = e + 32;
            if (a.sel != nullptr) {
                const int32_t* list = a.sel + ((int64_t)in.s * a.kv.n_head_kv + in.head) * a.n_sel;
                x0 = !only_second && e < a.n_sel ? list[e] : -1;
                x1 = e + 32 < a.n_sel ? list[e + 32] : -1;
            }
            const int32_t* row_of = a.table + in.s * a.table_stride;
            const bool on0 = !only_second && (unsigned)x0 < (unsigned)nb, on1 = (unsigned)x1 < (unsigned)nb;
            int y0 = -1, y1 = -1;
            if (on0) y0 = row_of[x0];
            if (on1) y1 = row_of[x1];
            const bool bad0 = on0 && (unsigned)y0 >= (unsigned)a.kv.n_pages;
            const bool bad1 = on1 && (unsigned)y1 >= (unsigned)a.kv.n_pages;
            if (bad0 || bad1) record_status(B200_DEVSTATUS_BOUNDS);
            if (!only_second) p0 = bad0 ? -1 : y0, b0 = x0;
            p1 = bad1 ? -1 : y1, b1 = x1;
        };
        auto flush_mask = [&]() {
            if (mask_stage >= 0) {
                const float v = (valid_pending >> (lane & 15)) & 1 ? h2f(mask_pending) : -INFINITY;
                const unsigned live = __ballot_sync(0xffffffffu, v != -INFINITY) & 0xffffu;
                if (lane < kPaTok) sh.mask[warp][mask_stage][lane] = v;
                if (lane == 0) sh.live[warp][mask_stage] = live;
                mask_stage = -1;
            }
        };
        // another segment, or the next 32 entries of this one's list
        auto refill = [&]() -> bool {
            if (in.u == in.nu) {
                if (!pa_next(a, in)) return false;
                fresh = true;
            }
            const unsigned vt = (unsigned)in.u * kPaTok + (lane & 15);
            bi = (int)(vt / (unsigned)ps);
            row = (int)(vt - (unsigned)bi * (unsigned)ps);
            if (fresh) {
                w0 = (int)((unsigned)in.u * kPaTok / (unsigned)ps);
                window(w0 + lane, false);
                k_head = static_cast<const uint8_t*>(a.kv.k) + in.head * a.kv.k_head;
                v_head = static_cast<const uint8_t*>(a.kv.v) + in.head * a.kv.v_head;
                fresh = false;
            } else {
                w0 += 32;
                p0 = p1, b0 = b1;
                window(w0 + lane, true);
            }
            // units that begin before entry w0 + 32
            const long long here = ((long long)(w0 + 32) * ps - (long long)in.u * kPaTok + kPaTok - 1) / kPaTok;
            run = (int)min((long long)(in.nu - in.u), here);
            return true;
        };
        auto issue = [&](int stage) {
            if (MASK) flush_mask();
            if (to_issue > 0) {
                if (run != 0) {
                    bi += q16;
                    row += r16;
                    if (row >= ps) row -= ps, ++bi;
                } else if (!refill()) {
                    to_issue = 0;
                }
            }
            if (to_issue > 0) {
                const int x = bi - w0;  // 0 .. 31, 46 where a unit spans pages
                int page = __shfl_sync(0xffffffffu, p0, x & 31), blk = bi;
                if (a.sel != nullptr) blk = __shfl_sync(0xffffffffu, b0, x & 31);
                if (!aligned) {
                    const int pb = __shfl_sync(0xffffffffu, p1, x & 31);
                    const int bb = __shfl_sync(0xffffffffu, b1, x & 31);
                    if (x >= 32) page = pb, blk = a.sel != nullptr ? bb : bi;
                }
                const bool ok = page >= 0 && row < in.len - blk * ps;
                const unsigned valid = __ballot_sync(0xffffffffu, ok) & 0xffffu;
                if (lane == 0) sh.valid[warp][stage] = valid;
                if (MASK) {
                    if (ok) mask_pending = a.mask[in.s * a.mask_stride + (int64_t)blk * ps + row];
                    mask_stage = stage;
                    valid_pending = valid;
                }
                const uint32_t at = stage * (2 * TILE);
                if (near_rows && valid == 0xffffu) {  // 16 rows of one page: a base and steps
                    const uint32_t row0 = row - (lane & 15);
                    const uint8_t* kb = pa_step<16>(k_head + k_lane, page * kp16 + row0 * kr16);
                    const uint8_t* vb = pa_step<16>(v_head + v_lane, page * vp16 + row0 * vr16);
                    unrolled(std::make_index_sequence<kPaTok / RPI>{}, [&](auto ic) {
                        constexpr int I = decltype(ic)::value, OFF = I / SW * (SW * RPI * RB) + I % SW * (RPI * RB);
                        pa_cp16_at<OFF>(dst_of[I % SW] + at, pa_step<I>(kb, k_step));
                        pa_cp16_at<OFF + TILE>(dst_of[I % SW] + at, pa_step<I>(vb, v_step));
                    });
                } else {  // row by row from the lane that looks after it; zeros for those that do not exist
                    const uint32_t ko = ok ? page * kp16 + row * kr16 : 0u, vo = ok ? page * vp16 + row * vr16 : 0u;
#pragma unroll
                    for (int i = 0; i < kPaTok / RPI; ++i) {
                        const int r = i * RPI + lr;
                        const uint32_t d = dst_of[i % SW] + at + i * RPI * RB;
                        const uint32_t kr = __shfl_sync(0xffffffffu, ko, r);
                        const uint32_t vr = a.same_rows ? kr : __shfl_sync(0xffffffffu, vo, r);
                        const bool on = (valid >> r) & 1;
                        pa_cp16(d, pa_step<16>(k_head, kr + lc), on);
                        pa_cp16(d + TILE, pa_step<16>(v_head, vr + lc), on);
                    }
                }
                --to_issue;
                --run;
                ++in.u;
            }
            pa_commit();
        };
        // ---- consumer: this thread holds head g, positions 2 t4, 2 t4 + 1 (+ 8) ----
        uint32_t qf[NC][KT][4], q3[NC][BF16 ? KT : 1][2];
        // Outputs: acc is what the tensor core adds up itself (high and low parts of
        // w apart), emptied into o every FLUSH units: it truncates, and 4 of its
        // additions stay below the rounding of one f32.  m is the weights'
        // reference: it follows the running maximum only when that has grown by
        // 2^3, which w has room for (w <= 2^15 in f16), so o is rarely rescaled.
        // bf16's third parts take rows 0-7 of an instruction; two groups share one
        constexpr bool PAIR = BF16 && NC == 2;
        constexpr int THIRDS = PAIR ? 1 : NC;
        constexpr float W_UP = BF16 ? 1.f : 4096.f;  // bf16 has no subnormals to keep out of
        constexpr int FLUSH = D * NC <= 128 ? 4 : 1;  // (the others lack the registers)
        float o[NC][2 * KT][2], acc[NC][FLUSH > 1 ? 2 * KT : 1][4];
        float m[NC], l[NC], f[NC], mk = -INFINITY;
        int pending = 0;  // units in acc
        auto flush = [&]() {
            if (FLUSH == 1) return;
#pragma unroll
            for (int c = 0; c < NC; ++c)
#pragma unroll
                for (int i = 0; i < (FLUSH > 1 ? 2 * KT : 0); ++i) {
                    float(&d)[4] = acc[c][i];
                    o[c][i][0] += d[0] + d[2];
                    o[c][i][1] += d[1] + d[3];
                    d[0] = d[1] = d[2] = d[3] = 0.f;
                }
            pending = 0;
        };
        auto take_q = [&]() {
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                const bool mine_q = cur.chunk * NH + kPaHeads * c + g < G;
                float amax = 0.f;
#pragma unroll
                for (int i = 0; i < 2 * KT; ++i) {
                    if (!mine_q) qx[c][i] = make_float2(0.f, 0.f);
                    amax = fmaxf(amax, fmaxf(fabsf(qx[c][i].x), fabsf(qx[c][i].y)));
                }
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
                amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
                // q 2^-ex has its largest entry in [1, 2)
                const int ex = min(max((int)(__float_as_uint(amax) >> 23) - 127, -120), 120);
                const float up = __uint_as_float((unsigned)(127 - ex) << 23);
                f[c] = a.scale * 1.44269504f * __uint_as_float((unsigned)(127 + ex) << 23);
#pragma unroll
                for (int i = 0; i < 2 * KT; ++i) {
                    float x = qx[c][i].x * up, y = qx[c][i].y * up;
                    qf[c][i >> 1][2 * (i & 1)] = pa_split<BF16>(x, y);
                    qf[c][i >> 1][2 * (i & 1) + 1] = pa_split<BF16>(x, y);
                    if (BF16) q3[c][i >> 1][i & 1] = pa_split<BF16>(x, y);
                }
#pragma unroll
                for (int i = 0; i < 2 * KT; ++i) o[c][i][0] = o[c][i][1] = 0.f;
#pragma unroll
                for (int i = 0; i < (FLUSH > 1 ? 2 * KT : 0); ++i)
                    acc[c][i][0] = acc[c][i][1] = acc[c][i][2] = acc[c][i][3] = 0.f;
                m[c] = -INFINITY, l[c] = 0.f;
            }
            pending = 0;
            mk = MASK ? -INFINITY : 0.f;
        };
        // The loop runs S - 1 units ahead with the copies: its first S - 1 turns
        // only issue.
        int stage = 0, ahead = 0, lead = S - 1;
        int part = min(cur.nu - cur.u, to_do), turns = part;  // units of this segment in this range, and to go
        bool special = true, fetch = true;  // the first turns, or a new segment: queries to fetch
        // this lane's ldmatrix rows: 16 dims of a k step are 32 bytes, which the
        // swizzle moves within 128; K: positions 0-7 dims 0-7, 8-15, positions
        // 8-15 the same; V: dims 0-7 positions 0-7, 8-15, the next 8 dims the same
        const int mi = lane >> 3, ri = lane & 7;
        uint32_t k_at[4], v_at[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            k_at[i] = ring + (8 * (mi >> 1) + ri) * RB + (((2 * i + (mi & 1)) ^ ri) << 4);
            v_at[i] = ring + TILE + (8 * (mi & 1) + ri) * RB + (((2 * i + (mi >> 1)) ^ ri) << 4);
        }
#pragma unroll 1
        for (;;) {
            if (special && EARLY_Q && fetch) {
                fetch_q();
                fetch = false;
            }
            pa_wait<S - 2>();
            __syncwarp();
            issue(ahead);
            ahead = ahead + 1 == S ? 0 : ahead + 1;
            if (special) {
                if (lead > 0) {
                    --lead;
                    continue;
                }
                if (!EARLY_Q) fetch_q();
                take_q();
                special = false;
            }
            const unsigned valid = sh.valid[warp][stage];
            const unsigned live = MASK ? sh.live[warp][stage] : valid;
            const uint32_t st = stage * (2 * TILE);
            if (live) {
                if (live != valid) {  // masked positions: their values may be anything
#pragma unroll
                    for (int i = 0; i < kPaTok / RPI; ++i)
                        if (((valid & ~live) >> (i * RPI + lr)) & 1)
                            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(
                                             ring + st + TILE + (i * RPI + lr) * RB + 16 * lc),
                                         "r"(0u)
                                         : "memory");
                    __syncwarp();
                }
                // S = q K^T: 8 heads (high parts, low parts) x 16 positions
                // Chains of at most 4 k steps, added up outside the tensor core, which
                // truncates every addition; bf16's third parts in a chain of their
                // own, where what is truncated is 2^-16 as large.
                constexpr int CHAINS = (KT + 3) / 4;
                float sc[NC][2][CHAINS][4], s3[THIRDS][2][4];
                unrolled(std::make_index_sequence<KT>{}, [&](auto ic) {
                    constexpr int kt = decltype(ic)::value, k3 = BF16 ? kt : 0;
                    uint32_t b[4];
                    pa_ldsm_at<kt / 4 * 128>(b, k_at[kt % 4] + st);
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            const uint32_t(&q)[4] = qf[c][kt];
                            float(&d)[4] = sc[c][n][kt / 4];
                            if (kt % 4 == 0) pa_mma0<BF16>(d, q[0], q[1], q[2], q[3], b[2 * n], b[2 * n + 1]);
                            else pa_mma<BF16>(d, q[0], q[1], q[2], q[3], b[2 * n], b[2 * n + 1]);
                            if (BF16 && c < THIRDS) {
                                const uint32_t(&r)[2] = q3[c][k3];
                                const uint32_t r1 = PAIR ? q3[NC - 1][k3][0] : 0u, r3 = PAIR ? q3[NC - 1][k3][1] : 0u;
                                if (kt == 0) pa_mma0<BF16>(s3[c][n], r[0], r1, r[1], r3, b[2 * n], b[2 * n + 1]);
                                else pa_mma<BF16>(s3[c][n], r[0], r1, r[1], r3, b[2 * n], b[2 * n + 1]);
                            }
                        }
                });
                float bias[4] = {};
                if (MASK) {
                    float top = -INFINITY;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        bias[i] = sh.mask[warp][stage][8 * (i >> 1) + 2 * t4 + (i & 1)];
                        top = fmaxf(top, bias[i]);
                    }
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
                    top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
                    if (top > mk) {
#pragma unroll
                        for (int c = 0; c < NC; ++c) m[c] = pa_rel(m[c], mk, top);
                        mk = top;
                    }
#pragma unroll
                    for (int i = 0; i < 4; ++i) bias[i] = (bias[i] - mk) * 1.44269504f;
                }
                float x[NC][4], top[NC];
                bool grown = false;
#pragma unroll
                for (int c = 0; c < NC; ++c) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float lows = !BF16 ? 0.f : PAIR ? s3[0][i >> 1][2 * c + (i & 1)] : s3[PAIR ? 0 : c][i >> 1][i & 1];
                        float highs = 0.f;
#pragma unroll
                        for (int y = 0; y < CHAINS; ++y) {
                            highs += sc[c][i >> 1][y][i & 1];
                            lows += sc[c][i >> 1][y][2 + (i & 1)];
                        }
                        x[c][i] = highs + lows;
                    }
                    if (live == 0xffffu) {
                        top[c] = fmaxf(fmaxf(fmaf(x[c][0], f[c], bias[0]), fmaf(x[c][1], f[c], bias[1])),
                                       fmaxf(fmaf(x[c][2], f[c], bias[2]), fmaf(x[c][3], f[c], bias[3])));
                    } else {
                        top[c] = -INFINITY;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if ((live >> (8 * (i >> 1) + 2 * t4 + (i & 1))) & 1)
                                top[c] = fmaxf(top[c], fmaf(x[c][i], f[c], bias[i]));
                    }
                    top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 1));
                    top[c] = fmaxf(top[c], __shfl_xor_sync(0xffffffffu, top[c], 2));
                    grown |= top[c] > m[c] + 3.f;  // (at the first unit m is -inf)
                }
                if (__any_sync(0xffffffffu, grown)) {
                    flush();
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const float mn = top[c] > m[c] + 3.f ? top[c] : m[c];
                        const float corr = m[c] == -INFINITY ? 0.f : pa_exp2(m[c] - mn);
                        l[c] *= corr;
#pragma unroll
                        for (int i = 0; i < 2 * KT; ++i) o[c][i][0] *= corr, o[c][i][1] *= corr;
                        m[c] = mn;
                    }
                }
                // O += w V: the pieces of w as they stand are the A operand
                uint32_t wa[NC][4], w3[NC][2];
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    float w[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) w[i] = pa_exp2(fmaf(x[c][i], f[c], bias[i] - m[c])) * W_UP;
                    if (live != 0xffffu) {
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!((live >> (8 * (i >> 1) + 2 * t4 + (i & 1))) & 1)) w[i] = 0.f;
                    }
                    l[c] += (w[0] + w[1]) + (w[2] + w[3]);
                    wa[c][0] = pa_split<BF16>(w[0], w[1]);
                    wa[c][1] = pa_split<BF16>(w[0], w[1]);
                    wa[c][2] = pa_split<BF16>(w[2], w[3]);
                    wa[c][3] = pa_split<BF16>(w[2], w[3]);
                    if (BF16) w3[c][0] = pa_split<BF16>(w[0], w[1]), w3[c][1] = pa_split<BF16>(w[2], w[3]);
                }
                unrolled(std::make_index_sequence<KT>{}, [&](auto ic) {
                    constexpr int kt = decltype(ic)::value;
                    uint32_t b[4];
                    pa_ldsm_t_at<kt / 4 * 128>(b, v_at[kt % 4] + st);
                    if (PAIR) {
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            float d[4];
                            pa_mma0<BF16>(d, w3[0][0], w3[NC - 1][0], w3[0][1], w3[NC - 1][1], b[2 * n], b[2 * n + 1]);
                            o[0][2 * kt + n][0] += d[0], o[0][2 * kt + n][1] += d[1];
                            o[NC - 1][2 * kt + n][0] += d[2], o[NC - 1][2 * kt + n][1] += d[3];
                        }
                    }
#pragma unroll
                    for (int c = 0; c < NC; ++c)
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            if (FLUSH > 1) {
                                float(&d)[4] = acc[c][FLUSH > 1 ? 2 * kt + n : 0];
                                pa_mma<BF16>(d, wa[c][0], wa[c][1], wa[c][2], wa[c][3], b[2 * n], b[2 * n + 1]);
                                if (BF16 && !PAIR) pa_mma<BF16>(d, w3[c][0], 0u, w3[c][1], 0u, b[2 * n], b[2 * n + 1]);
                            } else {
                                float d[4];
                                pa_mma0<BF16>(d, wa[c][0], wa[c][1], wa[c][2], wa[c][3], b[2 * n], b[2 * n + 1]);
                                if (BF16 && !PAIR) pa_mma<BF16>(d, w3[c][0], 0u, w3[c][1], 0u, b[2 * n], b[2 * n + 1]);
                                o[c][2 * kt + n][0] += d[0] + d[2];
                                o[c][2 * kt + n][1] += d[1] + d[3];
                            }
                        }
                });
                if (FLUSH > 1 && ++pending == FLUSH) flush();
            }
            stage = stage + 1 == S ? 0 : stage + 1;

            if (--turns == 0) {
                const bool seg_end = cur.u + part == cur.nu;
                flush();
                const bool whole = seg_end && seg_from >= fb;
                float* p = seg_end ? head_piece(warp) : tail_piece(warp);
                if (!seg_end) {  // the last piece of this warp: its ring is free
                    pa_wait<0>();
                    __syncwarp();
                }
                float rest = 0.f;  // stays 0 unless something is infinite or NaN
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    l[c] += __shfl_xor_sync(0xffffffffu, l[c], 1);
                    l[c] += __shfl_xor_sync(0xffffffffu, l[c], 2);
                    rest = fmaf(l[c], 0.f, rest);
#pragma unroll
                    for (int i = 0; i < 2 * KT; ++i) rest = fmaf(o[c][i][0], 0.f, fmaf(o[c][i][1], 0.f, rest));
                }
                if (__builtin_expect(__any_sync(0xffffffffu, rest != 0.f), 0)) {
                    const int64_t row0 = (int64_t)cur.s * a.n_head + cur.head * G + cur.chunk * NH;
                    pa_plain<BF16, D, NC>(a, cur.s, cur.head, cur.chunk, cur.len, kPaTok * cur.u, kPaTok * part, whole,
                                          whole ? a.out + row0 * D : p, W_UP);
                } else {
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const int r = kPaHeads * c + g, j = cur.chunk * NH + r;
                        float scale = 1.f;
                        float* dst = p + r * D;
                        if (whole) {
                            scale = l[c] > 0.f ? 1.f / l[c] : 0.f;
                            dst = a.out + ((int64_t)cur.s * a.n_head + cur.head * G + j) * D;
                        } else if (t4 == 0) {
                            p[NH * D + r] = m[c], p[NH * D + NH + r] = l[c];
                        }
                        if (!whole || j < G)
#pragma unroll
                            for (int i = 0; i < 2 * KT; ++i)
                                *reinterpret_cast<float2*>(dst + 8 * i + 2 * t4) =
                                    make_float2(o[c][i][0] * scale, o[c][i][1] * scale);
                    }
                    if (!whole && lane == 0) p[NH * D + 2 * NH] = mk;
                }
                if (!whole && lane == 0) {
                    const int x = seg_end ? 0 : 1;
                    sh.seg[x][warp] = (cur.s * a.kv.n_head_kv + cur.head) * a.chunks + cur.chunk;
                    sh.from[x][warp] = seg_from;
                    sh.nu[x][warp] = cur.nu;
                    sh.row[x][warp] = cur.s * a.n_head + cur.head * G + cur.chunk * NH;
                    sh.rows[x][warp] = min(NH, G - cur.chunk * NH);
                }
                to_do -= part;
                if (to_do == 0) break;
                seg_from += cur.nu;  // the range goes on, so the segment has ended
                if (!pa_next(a, cur)) break;
                part = turns = min(cur.nu, to_do);
                special = fetch = true;
            }
        }
        pa_wait<0>();
    }
    __syncthreads();

    // ---- join the pieces of cut segments: a warp per head ----
    // A segment's pieces lie in consecutive warps: tail pieces, and the last one
    // a head piece where the segment ends inside this CTA.  Masks over warps:
    const int tl = lane < W ? sh.seg[1][lane] : -1, hd = lane < W ? sh.seg[0][lane] : -1;
    int prev = __shfl_up_sync(0xffffffffu, tl, 1);
    if (lane == 0) prev = -1;
    const unsigned goes_on = __ballot_sync(0xffffffffu, tl >= 0 && tl == prev);  // tail of the same segment as before
    const unsigned starts = __ballot_sync(0xffffffffu, tl >= 0 && tl != prev);
    const unsigned ends = __ballot_sync(0xffffffffu, hd >= 0 && hd == prev);     // head of the tail before
    const unsigned alone = __ballot_sync(0xffffffffu, hd >= 0 && hd != prev);
    constexpr int AT_M = NH * D, AT_L = AT_M + NH, AT_MK = AT_L + NH, NV = PaJoint<D>::NV;
    const bool masked = MASK, has_col = 4 * lane < D;
    auto put = [&](float* row, const PaJoint<D>& t, float scale) {
        float4* out = reinterpret_cast<float4*>(row) + lane;
        if (has_col)
#pragma unroll
            for (int i = 0; i < NV; ++i)
                out[32 * i] = make_float4(t.v[i].x * scale, t.v[i].y * scale, t.v[i].z * scale, t.v[i].w * scale);
    };
    int open0 = -1, open1 = -1;  // segments cut by the CTA's borders: where to find them in sh (2 * warp + slot)
#pragma unroll 1
    for (unsigned todo = starts | alone << 16; todo != 0; todo &= todo - 1) {
        const int bit = __ffs(todo) - 1, w0 = bit & 15, slot = bit >= 16 ? 0 : 1;
        const int run = slot == 0 ? 0 : __ffs(~(goes_on >> (w0 + 1))) - 1;  // further tail pieces
        const bool closed = slot == 0 || ((ends >> (w0 + run + 1)) & 1);
        const int n = slot == 0 ? 1 : 1 + run + (closed ? 1 : 0);
        const int from = sh.from[slot][w0], end = from + sh.nu[slot][w0], rows = sh.rows[slot][w0];
        const bool whole = from >= cb && end <= ce;
        if (!whole) {
            if (open0 < 0) open0 = 2 * w0 + slot;
            else open1 = 2 * w0 + slot;
        }
#pragma unroll 1
        for (int j = warp; j < rows; j += W) {
            PaJoint<D> t;
            t.clear();
            float pm = -INFINITY, pl = 0.f, pk = -INFINITY;
            if (lane < n) {
                const float* p = closed && lane == n - 1 ? head_piece(w0 + lane) : tail_piece(w0 + lane);
                pm = p[AT_M + j], pl = p[AT_L + j], pk = p[AT_MK];
            }
            t.add(n, pm, pl, pk, masked, smem_u32(tail_piece(w0) + j * D), S * 2 * TILE, closed ? n - 1 : -1,
                  smem_u32(head_piece(w0 + n - 1) + j * D));
            // the output, or this CTA's piece of the segment (one path: most of what
            // this costs is fetching its instructions)
            float* p = a.pieces + (int64_t)(2 * blockIdx.x + (from >= cb ? 1 : 0)) * PIECE;
            const float inv = t.l > 0.f ? 1.f / t.l : 0.f;
            put(whole ? a.out + (int64_t)(sh.row[slot][w0] + j) * D : p + j * D, t, whole ? inv : 1.f);
            if (!whole && lane == 0) p[AT_M + j] = t.m, p[AT_L + j] = t.l, p[AT_MK] = t.mk;
        }
    }
    if (open0 < 0) return;
    // The CTA whose ticket completes a head's segment joins that head.  Lane i
    // draws the tickets of this warp's i-th head.
    __threadfence();
    __syncwarp();
    unsigned got0 = 0, got1 = 0;
    const int my_j = warp + lane * W;
    if (my_j < sh.rows[open0 & 1][open0 >> 1])
        got0 = atomicAdd(a.tickets + (int64_t)sh.seg[open0 & 1][open0 >> 1] * NH + my_j, 1u);
    if (open1 >= 0 && my_j < sh.rows[open1 & 1][open1 >> 1])
        got1 = atomicAdd(a.tickets + (int64_t)sh.seg[open1 & 1][open1 >> 1] * NH + my_j, 1u);
    __threadfence();
#pragma unroll 1
    for (int i = 0; i < 2; ++i) {
        const int at = i ? open1 : open0;
        if (at < 0) break;
        const int from = sh.from[at & 1][at >> 1], rows = sh.rows[at & 1][at >> 1];
        const int c0 = from / per_cta, n = pa_pieces(from, sh.nu[at & 1][at >> 1], per_cta, (int)gridDim.x);
        // piece k: slot 1 of CTA c0, where the segment starts, then slot 0 of the next CTAs
        auto piece = [&](int k) -> const float* { return a.pieces + (int64_t)(2 * (c0 + k) + (k == 0 ? 1 : 0)) * PIECE; };
#pragma unroll 1
        for (int j = warp, x = 0; j < rows; j += W, ++x) {
            if (__shfl_sync(0xffffffffu, i ? got1 : got0, x) != (unsigned)(n - 1)) continue;
            // up to 32 pieces at a time into this warp's ring, behind its tail piece
            // (which other warps may still be reading)
            const uint32_t buf = smem_u32(tail_piece(warp)) + (uint32_t)align256(PIECE * 4);
            constexpr int ROOM = (S * 2 * TILE - PIECE * 4 - 256) / (4 * D), BATCH = ROOM < 32 ? ROOM : 32;
            PaJoint<D> t;
            t.clear();
#pragma unroll 1
            for (int c = 0; c < n; c += BATCH) {
                const int here = min(BATCH, n - c);
                float pm = -INFINITY, pl = 0.f, pk = -INFINITY;
#pragma unroll 4
                for (int k = 0; k < here; ++k)
#pragma unroll
                    for (int y = 0; y < NV; ++y)
                        if (has_col) pa_cp16(buf + k * (4 * D) + 16 * lane + 512 * y, piece(c + k) + j * D + 4 * lane + 128 * y, true);
                pa_commit();
                if (lane < here) {
                    const float* p = piece(c + lane);
                    pm = __ldcg(p + AT_M + j), pl = __ldcg(p + AT_L + j), pk = __ldcg(p + AT_MK);
                }
                pa_wait<0>();
                __syncwarp();
                t.add(here, pm, pl, pk, masked, buf, 4 * D, -1, 0u);
                __syncwarp();
            }
            put(a.out + (int64_t)(sh.row[at & 1][at >> 1] + j) * D, t, t.l > 0.f ? 1.f / t.l : 0.f);
            if (lane == 0) a.tickets[(int64_t)sh.seg[at & 1][at >> 1] * NH + j] = 0u;
        }
    }
}

}  // namespace b200
