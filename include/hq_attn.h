/*
 * hq_attn.h — C ABI of the attention operators and their paged key/value cache (gfx950).
 *
 * What stands between a decoder layer's q | k | v projections and its output projection
 * (include/hq_qgemm.h): causal attention of packed prompts, of new tokens over a paged cache and
 * of a batch whose sequences share a long prefix, and the cache's page keeping. Types, status
 * codes, hq_last_error, streams and workspaces are those of hq_qgemm.h: every pointer is a device
 * pointer unless it says otherwise, the caller owns every buffer, a call returns after enqueueing
 * its kernels on `stream`, on error nothing is enqueued, and results are deterministic.
 *
 * Definition. Row (t, h) is query head h of token t; sequence b has n_q new tokens (rows
 * [q0, q0 + n_q) of Q) and n_k keys, its new tokens' own among them; query head h reads
 * key/value head h / (heads / kv_heads).
 *   s_j = scale * sum_d q[t, h, d] k[j, d]    over the keys that t may see: j <= t + n_k - n_q
 *                                             (the new tokens are the last ones; causal), or all
 *   O[t, h, d] = sum_j exp(s_j - m) v[j, d] / sum_j exp(s_j - m),   m = max_j s_j
 *   lse[t, h] = m + log(sum_j exp(s_j - m))
 * A row that may see no key (n_k < n_q, an empty sequence) gets O = 0 and lse = -infinity. Keys a
 * row may not see take no part in it, whatever their K and V hold (infinities and NaN too).
 * Scores, the running maximum and sum and the products are kept in fp32; the weights exp(s - m)
 * are rounded to the activation type for the second product, O once at the end.
 */
#ifndef HQ_ATTN_H
#define HQ_ATTN_H

#include "hq_qgemm.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Queries and outputs of a call: element (t, h, d) of Q at t * q_row + h * q_head + d, of O
 * likewise, no two of O in one place. Strides are in elements and multiples of 8, Q and O 16-byte aligned. lse: NULL, or
 * fp32 [rows][heads]. head_dim: 64, 128 or 256. scale: positive and finite. */
typedef struct hq_attn_io {
    const void* Q;
    void* O;
    float* lse;
    int64_t q_row, q_head;
    int64_t o_row, o_head;
    uint32_t rows;      /* tokens of the call, all sequences */
    uint32_t heads;     /* query heads, a multiple of the key/value heads */
    uint32_t head_dim;
    hq_dtype dtype;
    float scale;
} hq_attn_io;

/* A paged cache. K and V of layer l, page p: element (head, token, d) at
 * l * layer_stride + p * page_stride + head * head_stride + token * token_stride + d (elements, the
 * same for K and V, multiples of 8; K and V 16-byte aligned). A page is dense: heads before tokens
 * (token_stride = head_dim, head_stride = page_tokens * head_dim) or tokens before heads
 * (head_stride = head_dim, token_stride = kv_heads * head_dim). A pool may be larger than 4 GiB.
 * Sequence r holds lens[r] tokens, token j of it at slot j % page_tokens of page
 * table[r * table_stride + j / page_tokens]; entries past them are -1. refs[p] counts the sequences
 * that hold page p; 0: free. A part-filled page has one holder. status: one word, to which calls
 * OR the HQ_CACHE_* faults that they meet on the device (the caller clears it). refused[r]: zero at
 * first; not zero from an hq_cache_reserve that was refused room for row r to the next one that was
 * not: hq_cache_append writes nothing to such a row (both calls need it, the others do not read it). */
typedef struct hq_kv_cache {
    void* K;
    void* V;
    int64_t layer_stride, page_stride, head_stride, token_stride;
    uint32_t layers, pages, kv_heads, page_tokens /* a power of two, 16 to 65536 */, head_dim;
    hq_dtype dtype;
    int32_t* table;
    int64_t table_stride;
    uint32_t rows, max_pages; /* max_pages: table entries of a row */
    int32_t* lens;
    int32_t* refs;
    uint32_t* status;
    int32_t* refused;
} hq_kv_cache;

#define HQ_CACHE_BAD_ROW 1u      /* a row number out of range, repeated, or not as the call needs it */
#define HQ_CACHE_NO_PAGES 2u     /* too few free pages: the call changed nothing */
#define HQ_CACHE_ROW_FULL 4u     /* a sequence would pass max_pages: the call changed nothing */
#define HQ_CACHE_BAD_PAGE 8u     /* a page number out of range, a count below zero, an append to a page of several rows; it was not followed */
#define HQ_CACHE_MAX_BATCH 1024u /* sequences of one hq_cache_* call */

/* ---- attention ---- */
typedef HQ_ENUM(hq_attn_kind) { HQ_ATTN_PROMPT = 1, HQ_ATTN_PAGED = 2, HQ_ATTN_SHARED = 3 } hq_attn_kind;

/* Workspace of one attention call on the current device (0: none), as hq_workspace_bytes: seqs
 * sequences (groups of them for HQ_ATTN_SHARED), rows tokens, max_keys the call's max_k or max_len, or
 * where that is 0 what it stands for (0 is refused here), max_prefix as in the call. The size does not fall as
 * max_keys and max_prefix grow: one taken at the largest serves every call of as many rows and
 * sequences on fewer keys, which may use less of it. The buffer obeys the rules there and can be the same one. */
hq_status hq_attn_workspace_bytes(hq_attn_kind kind, uint32_t rows, uint32_t seqs, uint32_t groups,
                                  uint32_t heads, uint32_t kv_heads, uint32_t head_dim, uint32_t max_keys,
                                  uint32_t max_prefix, size_t* bytes);
/* The kernels and the splits such a call runs and the workspace that it uses, as text. */
hq_status hq_describe_attn(hq_attn_kind kind, uint32_t rows, uint32_t seqs, uint32_t groups, uint32_t heads,
                           uint32_t kv_heads, uint32_t head_dim, uint32_t max_keys, uint32_t max_prefix,
                           char* buf, size_t buf_len);

/* Packed prompts. Sequence b's new tokens are rows [cu_q[b], cu_q[b + 1]) of Q, its keys rows
 * [cu_k[b], cu_k[b + 1]) of K and V (cu_k NULL: cu_q, the whole prompt). cu_*: int32 [seqs + 1],
 * not falling, cu_q[seqs] <= rows, cu_k[seqs] <= total_k (values outside are clamped). K: element (j, head, d)
 * at j * k_row + head * k_head + d, V likewise; strides multiples of 8 (k_row, v_row at most 2^23), 16-byte aligned. max_k: no
 * sequence has more keys (0: total_k); it only chooses how the work is split. */
hq_status hq_attn_prompt(const hq_attn_io* io, const void* K, int64_t k_row, int64_t k_head, const void* V,
                         int64_t v_row, int64_t v_head, uint32_t kv_heads, uint32_t total_k, const int32_t* cu_q,
                         const int32_t* cu_k, uint32_t seqs, int causal, uint32_t max_k, void* workspace,
                         size_t workspace_bytes, hq_stream stream);

/* New tokens over a layer of the cache, causal. Sequence b is row rows[b] of the cache (rows NULL:
 * row b); its lens tokens are the keys, and the last cu_q[b + 1] - cu_q[b] of them (cu_q NULL: the
 * last one; then io->rows = seqs) are those of Q. max_len as max_k above (0: what a row can hold). The kernel
 * is chosen by the mean number of new tokens: single tokens and a long chunk are faster as two calls. */
hq_status hq_attn_paged(const hq_attn_io* io, const hq_kv_cache* cache, uint32_t layer, const int32_t* rows,
                        const int32_t* cu_q, uint32_t seqs, uint32_t max_len, void* workspace,
                        size_t workspace_bytes, hq_stream stream);

/* One new token of each sequence, where the sequences [starts[g], starts[g + 1]) of the batch share
 * their first prefix_lens[g] tokens (starts: int32 [groups + 1], from 0 to seqs, not falling; where they are
 * not that, HQ_CACHE_BAD_ROW is reported and every sequence reads all its keys from its own pages). The
 * whole pages among those tokens are read once for the group, from its first sequence's table (after
 * hq_cache_fork every table of the group names the same ones); all later tokens from each sequence's
 * own pages. max_prefix: no prefix_lens is larger (0: not known), as max_len only a bound for the split. */
hq_status hq_attn_shared_prefix(const hq_attn_io* io, const hq_kv_cache* cache, uint32_t layer,
                                const int32_t* rows, uint32_t seqs, const int32_t* starts,
                                const int32_t* prefix_lens, uint32_t groups, uint32_t max_prefix, uint32_t max_len,
                                void* workspace, size_t workspace_bytes, hq_stream stream);

/* ---- the cache's pages ----
 * n is at most HQ_CACHE_MAX_BATCH; the rows, counts and lists are device int32 arrays. New pages are
 * the lowest free numbers, in the order of the list. */

/* Workspace of hq_cache_fork and hq_cache_compact on this cache, by the same rules (zero before its first use). */
hq_status hq_cache_workspace_bytes(const hq_kv_cache* cache, size_t* bytes);
/* Room for counts[i] (>= 0) more tokens of row rows[i]: pages for them, lens[rows[i]] += counts[i].
 * All rows or, with a fault in `status`, none; the appends of a refused call's rows then write nothing, so
 * a step can be enqueued whole and its fault be met at the end. */
hq_status hq_cache_reserve(const hq_kv_cache* cache, const int32_t* rows, const int32_t* counts, uint32_t n,
                           hq_stream stream);
/* Writes the keys and values of the last cu[i + 1] - cu[i] tokens of each row (cu NULL: of the last
 * one; then tokens = n) into one layer: source row cu[i] + t; a row appears once. Strides as in
 * hq_attn_prompt. Call it after hq_cache_reserve has made room. Rows that it was refused for (BAD_ROW), and
 * tokens on a page that several rows hold (BAD_PAGE), are skipped and reported. */
hq_status hq_cache_append(const hq_kv_cache* cache, uint32_t layer, const void* K, int64_t k_row, int64_t k_head,
                          const void* V, int64_t v_row, int64_t v_head, uint32_t tokens, const int32_t* rows,
                          const int32_t* cu, uint32_t n, hq_stream stream);
/* children[i] (an empty row, each once) becomes a copy of parents[i]: the parent's full pages are
 * shared, the tokens of a part-filled last page copied to a page of its own, in every layer. All
 * children or, with a fault in `status`, none. */
hq_status hq_cache_fork(const hq_kv_cache* cache, const int32_t* parents, const int32_t* children, uint32_t n,
                        void* workspace, size_t workspace_bytes, hq_stream stream);
/* Empties rows; pages that no row holds any more are free. A repeated or out-of-range row is skipped
 * and reported. */
hq_status hq_cache_free(const hq_kv_cache* cache, const int32_t* rows, uint32_t n, hq_stream stream);
/* Copies whole pages in every layer, dst[i] from src[i]; no dst is a src or a dst twice. */
hq_status hq_cache_copy_pages(const hq_kv_cache* cache, const int32_t* src, const int32_t* dst, uint32_t n,
                              hq_stream stream);
/* Moves the live pages to the front of the pool: of n_live live pages, the k-th at or past n_live
 * goes to the k-th free one below it, in every layer. The table and the counts after the move go to
 * out_table (out_stride entries a row) and out_refs, which may be the cache's own or tensors apart:
 * only pages that were free are written, so the old table stays good until one of them is reused. */
hq_status hq_cache_compact(const hq_kv_cache* cache, int32_t* out_table, int64_t out_stride, int32_t* out_refs,
                           void* workspace, size_t workspace_bytes, hq_stream stream);

#ifdef __cplusplus
}
#endif
#endif /* HQ_ATTN_H */
