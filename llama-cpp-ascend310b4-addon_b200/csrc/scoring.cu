// scoring.cu -- the second device translation unit: chunks of tokens over the
// paged cache, sequences that share its pages, and log probabilities.
//
// Built apart from kernels.cu to halve the time of a build; it has a status word
// and a wait limit of its own, which b200_device_status and
// b200_set_wait_timeout read and set with the others.
#include <cuda_runtime.h>

#include <algorithm>
#include <mutex>

#include "common.cuh"
#include "host_util.h"
#include "internal.h"
#include "logprobs.cuh"
#include "paged_check.h"
#include "paged_fork.cuh"
#include "paged_prefill.cuh"

using namespace b200;

int b200i_scoring_status(unsigned int* status, int reset) {
    unsigned int word = 0;
    CR_(cuda_status(cudaMemcpyFromSymbol(&word, g_status, sizeof(word))));
    *status |= word;
    const unsigned int z = 0;
    return reset ? cuda_status(cudaMemcpyToSymbol(g_status, &z, sizeof(z))) : B200_OK;
}

int b200i_scoring_timeout(unsigned long long ns) {
    return cuda_status(cudaMemcpyToSymbol(g_wait_timeout_ns, &ns, sizeof(ns)));
}

namespace {

// kernel<<<grid, threads, smem, st>>>(a), programmatically dependent on the launch before.
template <class A>
int launch_after(void (*kernel)(A), dim3 grid, int threads, cudaStream_t st, const A& a, int smem = 0) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3((unsigned)threads, 1, 1);
    cfg.dynamicSmemBytes = (size_t)smem;
    cfg.stream = st;
    cudaLaunchAttribute at = pdl_attr();
    cfg.attrs = &at;
    cfg.numAttrs = 1;
    return cuda_status(cudaLaunchKernelEx(&cfg, kernel, a));
}

// ------------------------------------------------------------------ prefill

bool g_prefill_attr[kMaxDevices][2][3][2];
std::mutex g_attr_mu;

template <bool BF16, int D, bool MASK>
int launch_prefill_main(const PagedPrefillArgs& a, cudaStream_t st) {
    const int dev = current_device();
    if (dev < 0 || dev >= kMaxDevices) return B200_EINVAL;
    {
        bool& done = g_prefill_attr[dev][BF16][D == 64 ? 0 : D == 128 ? 1 : 2][MASK];
        std::lock_guard<std::mutex> lk(g_attr_mu);
        if (!done) {
            CR_(cuda_status(cudaFuncSetAttribute(paged_prefill_kernel<BF16, D, MASK>,
                                                 cudaFuncAttributeMaxDynamicSharedMemorySize, pf_smem<D>())));
            done = true;
        }
    }
    return launch_after(paged_prefill_kernel<BF16, D, MASK>, dim3(kPfCtas), kPfThreads, st, a, pf_smem<D>());
}

template <bool BF16, int D>
int launch_prefill_d(const PagedPrefillArgs& a, cudaStream_t st) {
    paged_prefill_plan_kernel<<<1, kPfPlanThreads, 0, st>>>(a, pf_tiles(D) * kPfRows, pf_keys(D));
    CR_(cuda_status(cudaGetLastError()));
    CR_(a.mask ? (launch_prefill_main<BF16, D, true>(a, st)) : (launch_prefill_main<BF16, D, false>(a, st)));
    return launch_after(paged_prefill_finish_kernel<BF16, D>, dim3(pf_tiles(D) * kPfRows / 32, kPfCtas),
                        kPfFinishThreads, st, a);
}

template <bool BF16>
int launch_prefill(const PagedPrefillArgs& a, cudaStream_t st) {
    switch (a.kv.head_dim) {
        case 64: return launch_prefill_d<BF16, 64>(a, st);
        case 128: return launch_prefill_d<BF16, 128>(a, st);
        default: return launch_prefill_d<BF16, 256>(a, st);
    }
}

// A 16-bit view of four dimensions, the first contiguous, for boxes of 64 values by
// b1 by b2; false where TMA has no such view.
bool encode_view(CUtensorMap* m, const void* base, const int64_t (&dims)[4], const int64_t (&strides)[3], int b1, int b2) {
    PFN_cuTensorMapEncodeTiled_v12000 enc = tensor_map_encoder();
    if (!enc) return false;
    cuuint64_t d[4], st[3];
    for (int i = 0; i < 4; ++i) d[i] = (cuuint64_t)dims[i];
    for (int i = 0; i < 3; ++i) {
        const bool single = dims[i + 1] == 1;
        if (!single && (strides[i] <= 0 || strides[i] >= (int64_t)1 << 40)) return false;
        st[i] = single ? 16 : (cuuint64_t)strides[i];
    }
    const cuuint32_t box[4] = {64, (cuuint32_t)b1, (cuuint32_t)b2, 1}, step[4] = {1, 1, 1, 1};
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<void*>(base), d, st, box, step,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct PrefillLayout {
    int64_t units;  // at most
    size_t start, cut, claim, desc, prefix, bad, ml, o, total;
};

PrefillLayout prefill_layout(int head_dim, int64_t n_tokens, int64_t n_seq, int64_t n_head, int64_t n_head_kv) {
    const int64_t rows = pf_tiles(head_dim) * kPfRows;
    PrefillLayout l;
    l.units = n_tokens * (n_head / n_head_kv) / rows + n_seq;
    l.start = 256;
    l.cut = l.start + align256(kPfCtas * sizeof(int2));
    l.claim = l.cut + align256(2 * kPfCtas * sizeof(int4));
    l.desc = l.claim + align256(8 * kPfCtas * sizeof(unsigned));
    l.prefix = l.desc + align256((size_t)l.units * 2 * sizeof(int4));
    l.bad = l.prefix + align256((size_t)(l.units + 1) * sizeof(int64_t));
    l.ml = l.bad + align256((size_t)(n_tokens * n_head) * sizeof(int2));
    l.o = l.ml + (size_t)2 * kPfCtas * rows * sizeof(float4);
    l.total = l.o + (size_t)2 * kPfCtas * rows * head_dim * sizeof(float);
    return l;
}

// --------------------------------------------------------------------- fork

struct ForkLayout {
    size_t zeroed, total;  // the arrays that start at zero come first
    size_t full, tails, staged, len, rank, need, count, freed;
};

ForkLayout fork_layout(int64_t n_seq, int64_t max_blocks, int64_t n_pages) {
    ForkLayout l;
    l.full = align256((size_t)n_pages);
    l.tails = l.full + align256((size_t)n_pages);
    l.zeroed = l.tails + align256((size_t)n_pages * 4);
    l.staged = l.zeroed;
    l.len = l.staged + align256((size_t)n_seq * max_blocks * 4);
    l.rank = l.len + align256((size_t)n_seq * 4);
    l.need = l.rank + align256((size_t)n_seq * 4);
    l.count = l.need + align256((size_t)n_seq * 4);
    l.freed = l.count + 256;
    l.total = l.freed + align256((size_t)((n_pages + kForkPages - 1) / kForkPages) * 4);
    return l;
}

// ----------------------------------------------------------------- logprobs

template <int TYPE>
int launch_logprobs(const LogprobsArgs& a, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(a.n_rows * a.ctas), 1, 1);
    cfg.blockDim = dim3(kLpThreads, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute at;
    at.id = cudaLaunchAttributeClusterDimension;
    at.val.clusterDim.x = (unsigned)a.ctas;
    at.val.clusterDim.y = 1;
    at.val.clusterDim.z = 1;
    cfg.attrs = &at;
    cfg.numAttrs = a.ctas > 1 ? 1 : 0;
    return cuda_status(cudaLaunchKernelEx(&cfg, logprobs_kernel<TYPE>, a));
}

}  // namespace

extern "C" {

size_t b200_paged_prefill_workspace_size(int head_dim, int64_t n_tokens, int n_seq, int n_head, int n_head_kv) {
    if ((head_dim != 64 && head_dim != 128 && head_dim != 256) || n_tokens < 0 || n_tokens > INT32_MAX || n_seq < 0 ||
        n_seq > 65535 || n_head <= 0 || n_head > 65535 || n_head_kv <= 0 || n_head % n_head_kv)
        return 0;
    return prefill_layout(head_dim, n_tokens, n_seq, n_head, n_head_kv).total;
}

int b200_paged_prefill(const b200_paged_kv* kv, const void* q, int64_t q_stride, int64_t n_tokens, int n_head,
                       const int32_t* block_table, int64_t table_stride, int n_seq, int max_blocks,
                       const int32_t* seq_lens, const int32_t* cu, const void* mask, int64_t mask_stride, int window,
                       float scale, void* out, void* workspace, size_t workspace_size, b200_stream_t stream) {
    CR_(check_paged_kv(kv));
    if (n_seq == 0 || n_tokens == 0) return B200_OK;
    const int64_t row = (int64_t)n_head * kv->head_dim;
    if (!q || !block_table || !seq_lens || !cu || !out || !workspace || n_seq < 0 || n_seq > 65535 || n_tokens < 0 ||
        n_head <= 0 || n_head % kv->n_head_kv || n_head > 65535 || window < 0 || scale != scale)
        return B200_EINVAL;
    if (!aligned16(q) || !aligned16(out) || !aligned16(workspace) || (q_stride & 7) || (n_tokens > 1 && q_stride < row))
        return B200_EINVAL;
    // (a row stride of 0: one row for every sequence)
    if (max_blocks <= 0 || (n_seq > 1 && table_stride != 0 && table_stride < max_blocks) ||
        max_blocks > INT32_MAX / kv->page_size)
        return B200_EINVAL;
    if ((reinterpret_cast<uintptr_t>(mask) & 1) ||
        (mask && n_seq > 1 && mask_stride != 0 && mask_stride < (int64_t)max_blocks * kv->page_size))
        return B200_EINVAL;
    // rows and positions are counted in int: a unit's two tiles of rows from the last row
    // on, and a tile of positions past the last
    if (n_tokens > (INT32_MAX - 2 * kPfRows) / n_head || (int64_t)max_blocks * kv->page_size > INT32_MAX - kPfRows)
        return B200_EUNSUPPORTED;
    if (workspace_size < b200_paged_prefill_workspace_size(kv->head_dim, n_tokens, n_seq, n_head, kv->n_head_kv))
        return B200_EINVAL;
    if (q_stride > INT64_MAX / 4 / n_tokens) return B200_EINVAL;
    if (meets_rows(out, n_tokens * row * 2, q, q_stride * 2, row * 2, n_tokens)) return B200_EINVAL;
    PagedPrefillArgs a = {};
    a.kv = *kv;
    // Rows of a page to a box: the largest power of two that divides the page, a tile
    // of keys at most, eight (a group of the swizzle) at least; other pages go row by
    // row.  8192 tokens, 64/8 heads x 128: pages of 64 1010 to 1066 us, of 5 by rows 1455
    // to 1480; at a step where these took 1090 and 1476, pages of 24 1095 and of 100 in
    // boxes of four rows 1594.
    a.box = std::min(kv->page_size & -kv->page_size, pf_keys(kv->head_dim));
    const int64_t d = kv->head_dim, group = n_head / kv->n_head_kv;
    const int64_t page_dims[4] = {d, kv->page_size, kv->n_head_kv, kv->n_pages};
    if (a.box < 8 || !encode_view(&a.map_k, kv->k, page_dims, {kv->k_row, kv->k_head, kv->k_page}, a.box, 1) ||
        !encode_view(&a.map_v, kv->v, page_dims, {kv->v_row, kv->v_head, kv->v_page}, a.box, 1))
        a.box = 0;
    a.q_box = kPfRows % group == 0 ? (int)(kPfRows / group) : 0;
    if (a.q_box && !encode_view(&a.map_q, q, {d, group, n_tokens, kv->n_head_kv}, {d * 2, q_stride * 2, group * d * 2},
                                (int)group, a.q_box))
        a.q_box = 0;
    a.q = static_cast<const uint16_t*>(q);
    a.q_stride = q_stride;
    a.table = block_table;
    a.table_stride = table_stride;
    a.seq_lens = seq_lens;
    a.cu = cu;
    a.mask = static_cast<const uint16_t*>(mask);
    a.mask_stride = mask_stride;
    a.out = static_cast<uint16_t*>(out);
    a.n_tokens = (int)n_tokens;
    a.n_head = n_head;
    a.group = n_head / kv->n_head_kv;
    a.n_seq = n_seq;
    a.max_blocks = max_blocks;
    // (a window of every position is none)
    a.window = window >= (int64_t)max_blocks * kv->page_size ? 0 : window;
    a.scale = scale;
    const PrefillLayout l = prefill_layout(kv->head_dim, n_tokens, n_seq, n_head, kv->n_head_kv);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    a.max_units = l.units;
    a.header = reinterpret_cast<PfHeader*>(ws);
    a.start = reinterpret_cast<int2*>(ws + l.start);
    a.cut = reinterpret_cast<int4*>(ws + l.cut);
    a.claim = reinterpret_cast<unsigned*>(ws + l.claim);
    a.desc = reinterpret_cast<int4*>(ws + l.desc);
    a.prefix = reinterpret_cast<int64_t*>(ws + l.prefix);
    a.bad = reinterpret_cast<int2*>(ws + l.bad);
    a.piece_ml = reinterpret_cast<float4*>(ws + l.ml);
    a.piece_o = reinterpret_cast<float4*>(ws + l.o);
    return kv->type == B200_TYPE_BF16 ? launch_prefill<true>(a, (cudaStream_t)stream)
                                      : launch_prefill<false>(a, (cudaStream_t)stream);
}

size_t b200_paged_fork_workspace_size(int n_seq, int max_blocks, int64_t n_pages) {
    if (n_seq <= 0 || max_blocks <= 0 || n_pages <= 0 || n_pages >= INT32_MAX ||
        (int64_t)n_seq * max_blocks > INT32_MAX)
        return 0;
    return fork_layout(n_seq, max_blocks, n_pages).total;
}

int b200_paged_fork(const int32_t* src, const int32_t* keep, const int32_t* seq_lens, int n_seq,
                    const int32_t* block_table, int64_t table_stride, int max_blocks, int page_size,
                    int32_t* free_pages, int64_t n_pages, const int32_t* n_free, int32_t* table_out,
                    int64_t table_out_stride, int32_t* seq_lens_out, int32_t* n_free_out, int32_t* copy_src,
                    int32_t* copy_dst, int32_t* copy_rows, void* workspace, size_t workspace_size,
                    b200_stream_t stream) {
    if (!src || !keep || !seq_lens || !block_table || !free_pages || !n_free || !table_out || !seq_lens_out ||
        !n_free_out || !copy_src || !copy_dst || !copy_rows || !workspace || !aligned16(workspace))
        return B200_EINVAL;
    if (n_seq <= 0 || max_blocks <= 0 || page_size <= 0 || n_pages <= 0 || n_pages >= INT32_MAX / page_size ||
        max_blocks > INT32_MAX / page_size ||
        (n_seq > 1 && (table_stride < max_blocks || table_out_stride < max_blocks)))
        return B200_EINVAL;
    if ((int64_t)n_seq * max_blocks > INT32_MAX) return B200_EUNSUPPORTED;
    if (workspace_size < b200_paged_fork_workspace_size(n_seq, max_blocks, n_pages)) return B200_EINVAL;
    // the new table replaces the old one or stands apart from it
    const bool in_place = table_out == block_table && (n_seq == 1 || table_out_stride == table_stride);
    if (n_seq > 1 && (table_stride > INT64_MAX / 8 / n_seq || table_out_stride > INT64_MAX / 8 / n_seq))
        return B200_EINVAL;
    // (rows of one stride may stand between each other's, as two halves of one tensor do)
    const int64_t ahead = (reinterpret_cast<intptr_t>(table_out) - reinterpret_cast<intptr_t>(block_table)) / 4;
    const int64_t place = table_stride > 0 ? (ahead % table_stride + table_stride) % table_stride : 0;
    const bool between = n_seq > 1 && table_out_stride == table_stride && place >= max_blocks &&
                         place <= table_stride - max_blocks;
    if (!in_place && !between &&
        meets_rows(table_out, ((n_seq - 1) * (n_seq > 1 ? table_out_stride : 0) + max_blocks) * 4, block_table,
                   (n_seq > 1 ? table_stride : 0) * 4, (int64_t)max_blocks * 4, n_seq))
        return B200_EINVAL;
    const ForkLayout l = fork_layout(n_seq, max_blocks, n_pages);
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    PagedForkArgs a;
    a.src = src;
    a.keep = keep;
    a.seq_lens = seq_lens;
    a.table = block_table;
    a.table_stride = table_stride;
    a.out = table_out;
    a.out_stride = table_out_stride;
    a.free_pages = free_pages;
    a.n_free = n_free;
    a.seq_lens_out = seq_lens_out;
    a.n_free_out = n_free_out;
    a.copy_src = copy_src;
    a.copy_dst = copy_dst;
    a.copy_rows = copy_rows;
    a.n_seq = n_seq;
    a.max_blocks = max_blocks;
    a.page_size = page_size;
    a.n_pages = (int)n_pages;
    a.was = ws;
    a.full = ws + l.full;
    a.tails = reinterpret_cast<unsigned int*>(ws + l.tails);
    a.staged = in_place ? reinterpret_cast<int32_t*>(ws + l.staged) : nullptr;
    a.len = reinterpret_cast<int32_t*>(ws + l.len);
    a.rank = reinterpret_cast<int32_t*>(ws + l.rank);
    a.need = reinterpret_cast<int32_t*>(ws + l.need);
    a.total = reinterpret_cast<int32_t*>(ws + l.count);
    a.freed = reinterpret_cast<int32_t*>(ws + l.freed);
    a.page_ctas = (int)((n_pages + kForkPages - 1) / kForkPages);
    a.cols = std::max(kForkCols, (max_blocks + 65534) / 65535);
    const unsigned cols = (unsigned)(((int64_t)max_blocks + a.cols - 1) / a.cols);
    const cudaStream_t st = (cudaStream_t)stream;
    CR_(cuda_status(cudaMemsetAsync(ws, 0, l.zeroed, st)));
    const unsigned rows = kForkRowThreads / 32;
    paged_fork_mark_kernel<<<dim3((unsigned)(n_seq + rows - 1) / rows, cols), kForkRowThreads, 0, st>>>(a);
    CR_(cuda_status(cudaGetLastError()));
    CR_(launch_after(paged_fork_count_kernel, dim3((unsigned)a.page_ctas + 1), kForkThreads, st, a));
    const int64_t tasks = (int64_t)n_seq * cols;
    return launch_after(paged_fork_write_kernel,
                        dim3((unsigned)(a.page_ctas + (tasks + kForkThreads / 32 - 1) / (kForkThreads / 32))),
                        kForkThreads, st, a);
}

int b200_paged_copy(const b200_paged_kv* kv, const int32_t* src, const int32_t* dst, const int32_t* rows, int64_t n,
                    b200_stream_t stream) {
    CR_(check_paged_kv(kv));
    if (n == 0) return B200_OK;
    if (!src || !dst || n < 0 || n > INT32_MAX || kv->n_head_kv > 65535) return B200_EINVAL;
    const int per_row = kv->n_head_kv * (kv->head_dim / 8);
    PagedCopyArgs a;
    a.kv = *kv;
    a.src = src;
    a.dst = dst;
    a.rows = rows;
    a.n = n;
    // 4096 pieces of 16 bytes to a CTA, or one row
    a.part = std::max({1, kCopyThreads * 16 / per_row, (kv->page_size + 65534) / 65535});
    a.part = std::min(a.part, kv->page_size);
    if ((int64_t)a.part * per_row > INT32_MAX / 2) return B200_EUNSUPPORTED;
    const dim3 grid((unsigned)n, (unsigned)((kv->page_size + a.part - 1) / a.part));
    paged_copy_kernel<<<grid, kCopyThreads, 0, (cudaStream_t)stream>>>(a);
    return cuda_status(cudaGetLastError());
}

int b200_token_logprobs(const void* logits, int type, int64_t ld, int64_t n_rows, int64_t n_vocab,
                        const int32_t* tokens, int k, float* logprob, float* entropy, int32_t* top_ids,
                        float* top_logprobs, b200_stream_t stream) {
    if (type != B200_TYPE_F32 && type != B200_TYPE_F16 && type != B200_TYPE_BF16) return B200_EUNSUPPORTED;
    if (n_rows == 0) return B200_OK;
    const int size = type == B200_TYPE_F32 ? 4 : 2;
    if (!logits || n_rows < 0 || n_vocab < 1 || n_vocab >= INT32_MAX || k < 0 ||
        k > std::min<int64_t>(B200_LOGPROBS_MAX_K, n_vocab) || (tokens == nullptr) != (logprob == nullptr) ||
        (k > 0) != (top_ids != nullptr) || (k > 0) != (top_logprobs != nullptr) ||
        (reinterpret_cast<uintptr_t>(logits) & (size - 1)) || (n_rows > 1 && ld < n_vocab) ||
        (n_rows > 1 && ld > INT64_MAX / 8 / n_rows))
        return B200_EINVAL;
    LogprobsArgs a;
    a.logits = static_cast<const uint8_t*>(logits);
    a.ld = n_rows > 1 ? ld * size : 0;
    a.n_rows = n_rows;
    a.n_vocab = (int)n_vocab;
    a.k = k;
    a.tokens = tokens;
    a.logprob = logprob;
    a.entropy = entropy;
    a.top_ids = top_ids;
    a.top_logprobs = top_logprobs;
    // CTAs to a row: as many as make waves of CTAs x (logits to a thread + what the
    // selection costs, about 100 logits) least, while every thread gets a vector.  Rows of
    // 151936 f32 logits: 200 take 31 us with four, 39 with eight; 600 70 with one, 73 with
    // two; 1024 124 with one, 111 with two, 123 with four; in bf16 89, 97, 124
    const int64_t places = 148 * (type == B200_TYPE_F32 ? kLpPerSmF32 : kLpPerSm16);
    int64_t least = INT64_MAX;
    for (int ctas = 1; ctas <= kLpMaxCtas; ctas *= 2) {
        if (ctas > 1 && n_vocab * size / 16 / ctas < kLpThreads) break;
        const int64_t cost = (n_rows * ctas + places - 1) / places * (n_vocab / (ctas * kLpThreads) + 100);
        if (cost < least) least = cost, a.ctas = ctas;
    }
    if (n_rows * a.ctas > INT32_MAX) return B200_EUNSUPPORTED;
    const cudaStream_t st = (cudaStream_t)stream;
    return type == B200_TYPE_F32   ? launch_logprobs<B200_TYPE_F32>(a, st)
           : type == B200_TYPE_F16 ? launch_logprobs<B200_TYPE_F16>(a, st)
                                   : launch_logprobs<B200_TYPE_BF16>(a, st);
}

}  // extern "C"
