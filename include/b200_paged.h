/*
 * b200_paged.h -- C ABI of batched single-token decode over a paged
 * key-value cache: page allocation and slot maps, the K/V store, block
 * selection for sparse attention, and attention of one new token per
 * sequence.
 *
 * The conventions are those of b200_decode.h: plain C, device pointers of the
 * device current on the calling thread, byte strides where stated, an int
 * status, every call asynchronous on its stream.  No call allocates device
 * memory, and every call may be captured into a CUDA graph: lengths, tables
 * and page counts are read on the device when the graph runs.
 *
 * The cache of one layer is n_pages pages of page_size tokens.  Sequence s
 * with seq_lens[s] cached tokens owns ceil(seq_lens[s] / page_size) pages;
 * its token at position p lives in page block_table[s][p / page_size] at row
 * p % page_size, that is in slot page * page_size + row.  Memory of the cache
 * that no cached token owns may hold anything, NaN included: it is never
 * used.  A page index outside [0, n_pages) or a length outside
 * [0, max_blocks * page_size] is never followed: the access is skipped (the
 * length clamped) and B200_DEVSTATUS_BOUNDS recorded (b200_device_status).
 * Lengths, tables, lists and masks must not change while a call that reads them
 * runs: it then still touches nothing outside its tensors, but its results are
 * wrong, and an attention workspace has to be zero-filled again.
 *
 * A batch has at most 65535 sequences and 65535 query heads (B200_EINVAL).
 *
 * The reference serves one sequence over one contiguous cache; these are the
 * counterparts of its attention step, its SET_ROWS and its kv_lengths input
 * (patch:1370-1432, patch:1179-1184, patch:2009-2023) for many sequences.
 */
#ifndef B200_PAGED_H
#define B200_PAGED_H

#include <stddef.h>
#include <stdint.h>

#include "b200_decode.h"

#ifdef __cplusplus
extern "C" {
#endif

#define B200_TYPE_BF16 30 /* the value of ggml's GGML_TYPE_BF16 */

/* Sequences one b200_paged_plan call handles. */
#define B200_PAGED_PLAN_MAX_SEQS 8192
/* Blocks of one sequence that b200_paged_select scores. */
#define B200_PAGED_SELECT_MAX_BLOCKS (1 << 20)

/* One layer's cache.  Element (page, row, head, d) of K is at byte
 * page * k_page + row * k_row + head * k_head + d * 2 of k, V likewise: any
 * order of rows and heads inside a page works.  k, v and every stride are
 * multiples of 16 bytes; K and V span less than 64 GiB each. */
typedef struct {
    int type;      /* B200_TYPE_F16 or B200_TYPE_BF16 */
    int head_dim;  /* 64, 128 or 256 */
    int n_head_kv;
    int page_size; /* tokens per page, >= 1; n_pages * page_size < 2^31 */
    int64_t n_pages;
    void *k, *v;
    int64_t k_page, k_row, k_head;
    int64_t v_page, v_row, v_head;
    /* Key bounds of every page, or NULL both: contiguous
     * [n_pages][n_head_kv][head_dim] elements of `type`, 16-byte aligned.
     * k_lo / k_hi hold the smallest / largest key value per channel over the
     * rows stored in the page since its row 0 was last stored. */
    void *k_lo, *k_hi;
} b200_paged_kv;

/* ------------------------------------------------------------------------
 * One scheduler step: pages, lengths and slots from request lengths.
 *   new_lens[s]  > 0: sequence s appends that many tokens; 0: nothing; < 0:
 *                it ends and its pages are given back
 *   seq_lens[s]  cached tokens before the step
 *   free_pages, n_free: a stack of free pages (n_free[0] entries; room for
 *                n_pages)
 * Ending sequences push their pages (in order of s, then of block).  Then
 * sequence s needs ceil((len + new) / page_size) - ceil(len / page_size)
 * pages; it is served when its tokens fit both the table (max_blocks) and
 * the token rows (max_tokens) and, if it needs pages, when the needs of all
 * fitting sequences up to and including s do not exceed the pages on the
 * stack.  Pages are popped from the top in order of s, then of block, into
 * block_table[s] (row stride table_stride elements).
 * Outputs:
 *   cu[s]         first token row of sequence s, cu[n_seq] the number of
 *                 rows (both at most max_tokens): rows [cu[s], cu[s + 1])
 *   slots[t], positions[t]  t < max_tokens: slot and position of the token
 *                 row; -1 for the rows of a sequence that was not served and
 *                 for rows at or past cu[n_seq]
 *   seq_lens_out  len + new where served, 0 where ended, else len
 *   n_free_out    entries left on the stack
 * seq_lens_out may be seq_lens and n_free_out n_free (in place); with
 * separate ones the call can be repeated.  Rows of block_table that gain no
 * page and stack entries below n_free[0] are left as they are. */
int b200_paged_plan(const int32_t *new_lens, const int32_t *seq_lens, int n_seq, int32_t *block_table,
                    int64_t table_stride, int max_blocks, int page_size, int32_t *free_pages, int64_t n_pages,
                    const int32_t *n_free, int64_t max_tokens, int64_t *slots, int32_t *positions, int32_t *cu,
                    int32_t *seq_lens_out, int32_t *n_free_out, b200_stream_t stream);

/* ------------------------------------------------------------------------
 * K and V rows of new tokens into their slots: row t of k and v (f32
 * [n_tokens][n_head_kv * head_dim], row strides k_ld and v_ld floats,
 * multiples of 4; 16-byte aligned) is rounded to the cache type (nearest,
 * ties to even) and stored at slots[t]; negative slots are skipped.  With
 * k_lo / k_hi set, the bounds of every page that receives a row are widened
 * by the new keys, or started afresh where its row 0 is among them (NaN keys
 * leave them alone).  The slots of one call differ, and those of one page
 * are consecutive in it, as b200_paged_plan makes them. */
int b200_paged_store(const b200_paged_kv *kv, const float *k, int64_t k_ld, const float *v, int64_t v_ld,
                     const int64_t *slots, int64_t n_tokens, b200_stream_t stream);

/* ------------------------------------------------------------------------
 * Which blocks of its sequence each KV head should attend to.  With the key
 * bounds lo, hi of block b's page,
 *   score(s, h, b) = max over the query heads j of KV head h of
 *                    sum_d max(q[s][j][d] * lo[d], q[s][j][d] * hi[d]),
 * an upper bound of q . k over the block's keys, summed in 64 bits.  sel[s][h]
 * (int32 [n_seq][n_head_kv][n_sel]) receives the sequence's newest block and
 * the n_sel - 1 blocks of largest score among the others (ties: the lower
 * block; NaN scores come last), in ascending order, then -1 where the
 * sequence has fewer blocks.  A block whose page index is out of range is
 * scored as NaN.  A product that is NaN (a NaN bound, 0 times an infinite one)
 * makes the score NaN.  (b200_paged_store leaves lo = +inf and hi = -inf in a
 * channel whose every key is NaN.)  q as in b200_paged_attn; workspace: 16-byte
 * aligned, no initial contents needed, not shared by calls that overlap on the
 * GPU. */
size_t b200_paged_select_workspace_size(int n_seq, int n_head_kv, int max_blocks);
int b200_paged_select(const b200_paged_kv *kv, const float *q, int64_t q_stride, int n_seq, int n_head,
                      const int32_t *block_table, int64_t table_stride, int max_blocks, const int32_t *seq_lens,
                      int n_sel, int32_t *sel, void *workspace, size_t workspace_size, b200_stream_t stream);

/* ------------------------------------------------------------------------
 * Attention of one new token per sequence (GQA, online softmax, split over
 * the cache's length and joined in a fixed order):
 *   out[s][j] = sum_p w_p v_p / sum_p w_p,
 *   w_p = exp(scale * q[s][j] . k_p + mask[s][p])
 * over the positions p < seq_lens[s], or with sel set over the positions of
 * the blocks sel[s][h] lists (int32 [n_seq][n_head_kv][n_sel]; negative
 * entries are skipped, a block listed twice counts twice; entries past the
 * sequence's blocks hold no position).
 *   q     f32, row s at q + s * q_stride (floats, a multiple of 4), heads
 *         [n_head][head_dim] contiguous, 16-byte aligned
 *   mask  f16, additive, row s at mask + s * mask_stride (elements), at least
 *         max_blocks * page_size entries, or NULL; finite or -inf.  Positions
 *         at -inf are left out whatever their key and value hold.  A stride of
 *         0 gives every sequence the same row, as table_stride 0 does (here
 *         and in b200_paged_select).
 *   out   f32 [n_seq][n_head][head_dim], 16-byte aligned, apart from q's rows
 *         (B200_EINVAL); a sequence with no position gets zeros
 * Keys, values and queries may be infinite or NaN (b200_paged_store makes
 * infinities of values past the f16 range): a score of -inf has weight 0, and
 * zeros come out where every weight is 0; a score that is +inf or NaN makes its
 * head's output NaN; infinite values make their columns infinite, or NaN where
 * both signs or a weight of 0 (below 2^-126 of the largest) meet them.  A
 * sequence whose every page holds such values takes up to 60 times as long.
 * At most 2^30 units of 16 positions of a (sequence, KV head, 8 or 16 query
 * heads) a call, counted at the table's width (B200_EUNSUPPORTED).
 * Products of K and V with q and w run on tensor cores; q and w enter as sums
 * of 16-bit parts (two of f16, three of bf16) that keep 22 bits of each.
 * The workspace must be zero-filled before its first use; every call leaves
 * it ready for the next, of any shape.  Calls that share one must not overlap
 * on the GPU, and nothing else (b200_paged_select among it) may write to it. */
size_t b200_paged_attn_workspace_size(int head_dim, int n_seq, int n_head, int n_head_kv);
int b200_paged_attn(const b200_paged_kv *kv, const float *q, int64_t q_stride, int n_seq, int n_head,
                    const int32_t *block_table, int64_t table_stride, int max_blocks, const int32_t *seq_lens,
                    const void *mask, int64_t mask_stride, const int32_t *sel, int n_sel, float scale, float *out,
                    void *workspace, size_t workspace_size, b200_stream_t stream);

#ifdef __cplusplus
}
#endif
#endif /* B200_PAGED_H */
