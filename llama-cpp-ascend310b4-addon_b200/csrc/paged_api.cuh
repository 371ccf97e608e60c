// paged_api.cuh -- the C ABI of include/b200_paged.h: argument checks and
// launches.  Included by kernels.cu, whose helpers it uses.
#pragma once

#include "paged_attn.cuh"
#include "paged_plan.cuh"
#include "paged_select.cuh"
#include "paged_store.cuh"
#include "paged_work.cuh"

namespace {

int check_paged_kv(const b200_paged_kv* kv) {
    if (!kv || !kv->k || !kv->v || kv->n_head_kv <= 0 || kv->page_size <= 0 || kv->n_pages <= 0 ||
        kv->n_pages >= INT32_MAX / kv->page_size)
        return B200_EINVAL;
    if (kv->type != B200_TYPE_F16 && kv->type != B200_TYPE_BF16) return B200_EUNSUPPORTED;
    if (kv->head_dim != 64 && kv->head_dim != 128 && kv->head_dim != 256) return B200_EUNSUPPORTED;
    const int64_t strides = kv->k_page | kv->k_row | kv->k_head | kv->v_page | kv->v_row | kv->v_head;
    if (!aligned16(kv->k) || !aligned16(kv->v) || (strides & 15) || strides < 0) return B200_EINVAL;
    // the last byte of K and of V: offsets are counted in 16-byte steps in 32 bits.
    // Each term is compared by division first, so the sums cannot wrap around
    const int64_t span = (int64_t)1 << 36;
    const int64_t last[3] = {kv->n_pages - 1, kv->page_size - 1, kv->n_head_kv - 1};
    const int64_t steps[2][3] = {{kv->k_page, kv->k_row, kv->k_head}, {kv->v_page, kv->v_row, kv->v_head}};
    for (const auto& step : steps) {
        int64_t end = 0;
        for (int i = 0; i < 3; ++i) {
            if (step[i] >= span || (step[i] > 0 && last[i] > span / step[i])) return B200_EUNSUPPORTED;
            end += last[i] * step[i];
        }
        if (end >= span) return B200_EUNSUPPORTED;
    }
    if ((kv->k_lo == nullptr) != (kv->k_hi == nullptr) || !aligned16(kv->k_lo) || !aligned16(kv->k_hi))
        return B200_EINVAL;
    return B200_OK;
}

// What the queries, the block table and the lengths of a batch must satisfy.
int check_paged_batch(const b200_paged_kv* kv, const float* q, int64_t q_stride, int n_seq, int n_head,
                      const int32_t* block_table, int64_t table_stride, int max_blocks, const int32_t* seq_lens) {
    if (!q || !block_table || !seq_lens || n_seq < 0 || n_seq > 65535 || n_head <= 0 || n_head % kv->n_head_kv ||
        n_head > 65535)
        return B200_EINVAL;
    if (!aligned16(q) || (q_stride & 3) || (n_seq > 1 && q_stride < (int64_t)n_head * kv->head_dim)) return B200_EINVAL;
    // (a row stride of 0: one row for every sequence)
    if (max_blocks <= 0 || (n_seq > 1 && table_stride != 0 && table_stride < max_blocks) ||
        max_blocks > INT32_MAX / kv->page_size)
        return B200_EINVAL;
    return B200_OK;
}

// Whether `size` bytes at out meet one of n rows of `row` bytes, `stride` bytes
// apart from q on.
bool meets_rows(const void* out, int64_t size, const void* q, int64_t stride, int64_t row, int64_t n) {
    const int64_t ahead = reinterpret_cast<intptr_t>(out) - reinterpret_cast<intptr_t>(q);
    // the first row that ends behind out's first byte
    const int64_t s = ahead < row ? 0 : n == 1 || stride == 0 ? n : (ahead - row) / stride + 1;
    return s < n && s * stride < ahead + size;
}

bool g_paged_plan_attr[kMaxDevices];

int launch_paged_plan(const PagedPlanArgs& a, cudaStream_t st) {
    const int dev = current_device();
    if (dev < 0 || dev >= kMaxDevices) return B200_EINVAL;
    {
        std::lock_guard<std::mutex> lk(g_attr_mu);
        if (!g_paged_plan_attr[dev]) {
            CR_(cuda_status(cudaFuncSetAttribute(paged_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                 (int)plan_smem_bytes(B200_PAGED_PLAN_MAX_SEQS))));
            g_paged_plan_attr[dev] = true;
        }
    }
    // one cluster: every CTA scans the sequences, and each takes its share of
    // the token rows.  One CTA alone, launched without a cluster, up to a token
    // row per thread: 64 sequences with one token each 3.4 us against 4.0 on
    // two CTAs, 1024 sequences 6.5 against 7.1; twice the rows 7.6 against 6.9
    const int64_t tokens = a.max_tokens, rows = std::max<int64_t>(tokens, a.n_seq);
    const int64_t ctas = tokens <= kPlanThreads ? 1 : (tokens + 2 * kPlanThreads - 1) / (2 * kPlanThreads) + 1;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3((unsigned)std::min<int64_t>(kPlanThreads, (rows + 63) / 64 * 64), 1, 1);
    cfg.gridDim = dim3((unsigned)std::min<int64_t>(kPlanCtas, ctas), 1, 1);
    cfg.dynamicSmemBytes = plan_smem_bytes(a.n_seq);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = cfg.gridDim.x;
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = cfg.gridDim.x > 1 ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, paged_plan_kernel, a));
}

template <bool BF16>
int launch_paged_store(const PagedStoreArgs& a, cudaStream_t st) {
    // two tiles for every place a CTA of this size has on the GPU: decode steps,
    // whose tokens are runs of their own, get one CTA each, prompts few that
    // find no run
    const int64_t want = (a.n_tokens * a.kv.n_head_kv + 2367) / 2368;
    const int tile = (int)std::max<int64_t>(1, std::min<int64_t>(want, std::min(kStoreTile, a.kv.page_size)));
    const dim3 grid((unsigned)((a.n_tokens + tile - 1) / tile), (unsigned)a.kv.n_head_kv);
    switch (a.kv.head_dim) {
        case 64: paged_store_kernel<BF16, 64><<<grid, kStoreThreads, 0, st>>>(a, tile); break;
        case 128: paged_store_kernel<BF16, 128><<<grid, kStoreThreads, 0, st>>>(a, tile); break;
        default: paged_store_kernel<BF16, 256><<<grid, kStoreThreads, 0, st>>>(a, tile); break;
    }
    return cuda_status(cudaGetLastError());
}

bool g_paged_select_attr[kMaxDevices][2][3];

template <bool BF16, int D>
int launch_paged_select_d(const PagedSelectArgs& a, cudaStream_t st) {
    const int dev = current_device();
    if (dev < 0 || dev >= kMaxDevices) return B200_EINVAL;
    {
        bool& done = g_paged_select_attr[dev][BF16][D == 64 ? 0 : D == 128 ? 1 : 2];
        std::lock_guard<std::mutex> lk(g_attr_mu);
        if (!done) {
            CR_(cuda_status(cudaFuncSetAttribute(paged_score_kernel<BF16, D>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, score_smem<D>())));
            done = true;
        }
    }
    const int64_t units = (int64_t)a.n_seq * a.n_head_kv * paged_units(a.max_blocks);
    const int64_t grid = std::min<int64_t>(kPaCtas, (units + pa_warps(D) - 1) / pa_warps(D));
    paged_score_kernel<BF16, D><<<(unsigned)grid, 32 * pa_warps(D), score_smem<D>(), st>>>(a);
    CR_(cuda_status(cudaGetLastError()));
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n_seq * a.n_head_kv), 1, 1);
    cfg.blockDim = dim3(kTopkThreads, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute at = pdl_attr();
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, paged_topk_kernel<BF16, D>, a));
}

template <bool BF16>
int launch_paged_select(const PagedSelectArgs& a, int head_dim, cudaStream_t st) {
    switch (head_dim) {
        case 64: return launch_paged_select_d<BF16, 64>(a, st);
        case 128: return launch_paged_select_d<BF16, 128>(a, st);
        default: return launch_paged_select_d<BF16, 256>(a, st);
    }
}

bool g_paged_attn_attr[kMaxDevices][2][3][2][2];

template <bool BF16, int D, int NC, bool MASK>
int launch_paged_attn_dm(const PagedAttnArgs& a, cudaStream_t st) {
    const int dev = current_device();
    if (dev < 0 || dev >= kMaxDevices) return B200_EINVAL;
    {
        bool& done = g_paged_attn_attr[dev][BF16][D == 64 ? 0 : D == 128 ? 1 : 2][NC - 1][MASK];
        std::lock_guard<std::mutex> lk(g_attr_mu);
        if (!done) {
            CR_(cuda_status(cudaFuncSetAttribute(paged_attn_kernel<BF16, D, NC, MASK>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, pa_smem<D, NC>())));
            done = true;
        }
    }
    // the lengths are on the device: at most this many units
    const int64_t width = (int64_t)(a.sel ? a.n_sel : a.max_blocks) * a.kv.page_size;
    const int64_t units = (int64_t)a.n_seq * a.kv.n_head_kv * a.chunks * ((width + kPaTok - 1) / kPaTok);
    const int64_t grid = std::min<int64_t>(kPaCtas, (units + pa_warps(D, NC) - 1) / pa_warps(D, NC));
    paged_attn_kernel<BF16, D, NC, MASK><<<(unsigned)grid, 32 * pa_warps(D, NC), pa_smem<D, NC>(), st>>>(a);
    return cuda_status(cudaGetLastError());
}

template <bool BF16, int D, int NC>
int launch_paged_attn_d(const PagedAttnArgs& a, cudaStream_t st) {
    return a.mask ? launch_paged_attn_dm<BF16, D, NC, true>(a, st) : launch_paged_attn_dm<BF16, D, NC, false>(a, st);
}

template <bool BF16>
int launch_paged_attn(const PagedAttnArgs& a, cudaStream_t st) {
    const bool two = pa_groups(a.kv.head_dim, a.n_head / a.kv.n_head_kv) == 2;
    switch (a.kv.head_dim) {
        case 64: return two ? launch_paged_attn_d<BF16, 64, 2>(a, st) : launch_paged_attn_d<BF16, 64, 1>(a, st);
        case 128: return two ? launch_paged_attn_d<BF16, 128, 2>(a, st) : launch_paged_attn_d<BF16, 128, 1>(a, st);
        default: return launch_paged_attn_d<BF16, 256, 1>(a, st);
    }
}

// Passes over a KV head's query heads, and heads of one.
int paged_heads(int head_dim, int n_head, int n_head_kv) { return kPaHeads * pa_groups(head_dim, n_head / n_head_kv); }
int paged_chunks(int head_dim, int n_head, int n_head_kv) {
    const int heads = paged_heads(head_dim, n_head, n_head_kv);
    return (n_head / n_head_kv + heads - 1) / heads;
}
}  // namespace

extern "C" {

int b200_paged_plan(const int32_t* new_lens, const int32_t* seq_lens, int n_seq, int32_t* block_table,
                    int64_t table_stride, int max_blocks, int page_size, int32_t* free_pages, int64_t n_pages,
                    const int32_t* n_free, int64_t max_tokens, int64_t* slots, int32_t* positions, int32_t* cu,
                    int32_t* seq_lens_out, int32_t* n_free_out, b200_stream_t stream) {
    if (!new_lens || !seq_lens || !block_table || !free_pages || !n_free || !cu || !seq_lens_out || !n_free_out)
        return B200_EINVAL;
    if (n_seq <= 0 || max_blocks <= 0 || page_size <= 0 || n_pages <= 0 || max_tokens < 0 || max_tokens >= INT32_MAX ||
        (max_tokens > 0 && (!slots || !positions)) || (n_seq > 1 && table_stride < max_blocks) ||
        max_blocks > INT32_MAX / page_size || n_pages >= INT32_MAX / page_size)
        return B200_EINVAL;
    if (n_seq > B200_PAGED_PLAN_MAX_SEQS) return B200_EUNSUPPORTED;
    PagedPlanArgs a;
    a.new_lens = new_lens;
    a.seq_lens = seq_lens;
    a.table = block_table;
    a.table_stride = table_stride;
    a.free_pages = free_pages;
    a.n_free = n_free;
    a.slots = slots;
    a.positions = positions;
    a.cu = cu;
    a.seq_lens_out = seq_lens_out;
    a.n_free_out = n_free_out;
    a.n_seq = n_seq;
    a.max_blocks = max_blocks;
    a.page_size = page_size;
    a.n_pages = (int)n_pages;
    a.max_tokens = (int)max_tokens;
    return launch_paged_plan(a, (cudaStream_t)stream);
}

int b200_paged_store(const b200_paged_kv* kv, const float* k, int64_t k_ld, const float* v, int64_t v_ld,
                     const int64_t* slots, int64_t n_tokens, b200_stream_t stream) {
    CR_(check_paged_kv(kv));
    if (n_tokens == 0) return B200_OK;
    const int64_t row = (int64_t)kv->n_head_kv * kv->head_dim;
    if (!k || !v || !slots || n_tokens < 0 || n_tokens > INT32_MAX || kv->n_head_kv > 65535 || !aligned16(k) ||
        !aligned16(v) || (k_ld & 3) || (v_ld & 3) || (n_tokens > 1 && (k_ld < row || v_ld < row)))
        return B200_EINVAL;
    PagedStoreArgs a;
    a.kv = *kv;
    a.k = k;
    a.v = v;
    a.k_ld = k_ld;
    a.v_ld = v_ld;
    a.slots = slots;
    a.n_tokens = n_tokens;
    return kv->type == B200_TYPE_BF16 ? launch_paged_store<true>(a, (cudaStream_t)stream)
                                      : launch_paged_store<false>(a, (cudaStream_t)stream);
}

size_t b200_paged_select_workspace_size(int n_seq, int n_head_kv, int max_blocks) {
    if (n_seq < 0 || n_seq > 65535 || n_head_kv <= 0 || n_head_kv > 65535 || max_blocks <= 0 ||
        max_blocks > B200_PAGED_SELECT_MAX_BLOCKS)
        return 0;
    const size_t rows = (size_t)n_seq * n_head_kv;
    return std::max((size_t)256, align256(rows * max_blocks * sizeof(unsigned long long)) +
                                     align256(rows * max_blocks * sizeof(float)) + align256(rows * sizeof(float2)) +
                                     align256(rows * paged_units(max_blocks) * sizeof(unsigned int)));
}

int b200_paged_select(const b200_paged_kv* kv, const float* q, int64_t q_stride, int n_seq, int n_head,
                      const int32_t* block_table, int64_t table_stride, int max_blocks, const int32_t* seq_lens,
                      int n_sel, int32_t* sel, void* workspace, size_t workspace_size, b200_stream_t stream) {
    CR_(check_paged_kv(kv));
    if (n_seq == 0) return B200_OK;
    CR_(check_paged_batch(kv, q, q_stride, n_seq, n_head, block_table, table_stride, max_blocks, seq_lens));
    if (!kv->k_lo || !sel || n_sel <= 0 || !workspace || !aligned16(workspace)) return B200_EINVAL;
    if (max_blocks > B200_PAGED_SELECT_MAX_BLOCKS) return B200_EUNSUPPORTED;
    if ((int64_t)n_seq * kv->n_head_kv * paged_units(max_blocks) > INT32_MAX / 2) return B200_EUNSUPPORTED;
    if (kv->n_pages > ((int64_t)1 << 35) / kv->n_head_kv / kv->head_dim) return B200_EUNSUPPORTED;  // bounds below 64 GiB
    if (workspace_size < b200_paged_select_workspace_size(n_seq, kv->n_head_kv, max_blocks)) return B200_EINVAL;
    PagedSelectArgs a;
    a.lo = static_cast<const uint16_t*>(kv->k_lo);
    a.hi = static_cast<const uint16_t*>(kv->k_hi);
    a.q = q;
    a.q_stride = q_stride;
    a.table = block_table;
    a.table_stride = table_stride;
    a.seq_lens = seq_lens;
    a.sel = sel;
    const size_t rows = (size_t)n_seq * kv->n_head_kv;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.exact = reinterpret_cast<unsigned long long*>(ws);
    ws += align256(rows * max_blocks * sizeof(unsigned long long));
    a.approx = reinterpret_cast<float*>(ws);
    ws += align256(rows * max_blocks * sizeof(float));
    a.group = reinterpret_cast<float2*>(ws);
    ws += align256(rows * sizeof(float2));
    a.unit_max = reinterpret_cast<unsigned int*>(ws);
    a.n_seq = n_seq;
    a.n_head = n_head;
    a.n_head_kv = kv->n_head_kv;
    a.max_blocks = max_blocks;
    a.page_size = kv->page_size;
    a.n_pages = (int)kv->n_pages;
    a.n_sel = n_sel;
    return kv->type == B200_TYPE_BF16 ? launch_paged_select<true>(a, kv->head_dim, (cudaStream_t)stream)
                                      : launch_paged_select<false>(a, kv->head_dim, (cudaStream_t)stream);
}

size_t b200_paged_attn_workspace_size(int head_dim, int n_seq, int n_head, int n_head_kv) {
    if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || n_seq < 0 || n_seq > 65535 || n_head <= 0 ||
        n_head > 65535 || n_head_kv <= 0 || n_head % n_head_kv)
        return 0;
    return pa_piece_area() +
           align256((size_t)n_seq * n_head_kv * paged_chunks(head_dim, n_head, n_head_kv) *
                    paged_heads(head_dim, n_head, n_head_kv) * sizeof(unsigned int));
}

int b200_paged_attn(const b200_paged_kv* kv, const float* q, int64_t q_stride, int n_seq, int n_head,
                    const int32_t* block_table, int64_t table_stride, int max_blocks, const int32_t* seq_lens,
                    const void* mask, int64_t mask_stride, const int32_t* sel, int n_sel, float scale, float* out,
                    void* workspace, size_t workspace_size, b200_stream_t stream) {
    CR_(check_paged_kv(kv));
    if (n_seq == 0) return B200_OK;
    CR_(check_paged_batch(kv, q, q_stride, n_seq, n_head, block_table, table_stride, max_blocks, seq_lens));
    if (!out || !aligned16(out) || !workspace || !aligned16(workspace) || (sel && n_sel <= 0) ||
        (reinterpret_cast<uintptr_t>(mask) & 1) ||
        (mask && n_seq > 1 && mask_stride != 0 && mask_stride < (int64_t)max_blocks * kv->page_size) ||
        (sel && n_sel > (INT32_MAX - 4096) / kv->page_size) ||
        workspace_size < b200_paged_attn_workspace_size(kv->head_dim, n_seq, n_head, kv->n_head_kv))
        return B200_EINVAL;
    const int64_t row = (int64_t)n_head * kv->head_dim * (int64_t)sizeof(float);
    if (meets_rows(out, n_seq * row, q, q_stride * (int64_t)sizeof(float), row, n_seq)) return B200_EINVAL;
    const int64_t width = (int64_t)(sel ? n_sel : max_blocks) * kv->page_size;
    const int64_t segments = (int64_t)n_seq * kv->n_head_kv * paged_chunks(kv->head_dim, n_head, kv->n_head_kv);
    if (segments * ((width + kPaTok - 1) / kPaTok) > INT32_MAX / 2) return B200_EUNSUPPORTED;  // units are counted in int
    PagedAttnArgs a;
    a.kv = *kv;
    a.q = q;
    a.q_stride = q_stride;
    a.table = block_table;
    a.table_stride = table_stride;
    a.seq_lens = seq_lens;
    a.mask = static_cast<const uint16_t*>(mask);
    a.mask_stride = mask_stride;
    a.sel = sel;
    a.out = out;
    a.chunks = paged_chunks(kv->head_dim, n_head, kv->n_head_kv);
    a.pieces = static_cast<float*>(workspace);
    a.tickets = reinterpret_cast<unsigned int*>(static_cast<uint8_t*>(workspace) + pa_piece_area());
    a.scale = scale;
    a.n_seq = n_seq;
    a.n_head = n_head;
    a.n_sel = n_sel;
    a.max_blocks = max_blocks;
    a.group = n_head / kv->n_head_kv;
    a.unit_blocks = kPaTok / kv->page_size;
    a.unit_rows = kPaTok % kv->page_size;
    a.aligned = kv->page_size % kPaTok == 0;
    a.same_rows = kv->k_page == kv->v_page && kv->k_row == kv->v_row;
    a.near_rows = std::max(kv->k_row, kv->v_row) < ((int64_t)1 << 31) / kPaTok;
    return kv->type == B200_TYPE_BF16 ? launch_paged_attn<true>(a, (cudaStream_t)stream)
                                      : launch_paged_attn<false>(a, (cudaStream_t)stream);
}

}  // extern "C"
