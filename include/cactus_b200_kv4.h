/*
 * cactus_b200_kv4.h — C ABI of the 4-bit paged KV cache: append, read, attention, page copies and
 * compaction as kernel entry points, and a cache handle that keeps the pages of many sequences
 * (grow, fork, truncate, compact, free).
 *
 * Conventions are those of cactus_b200.h: DEVICE pointers unless a comment says host, fp16 as
 * uint16_t bits, asynchronous calls on `stream`, 0 or a negative code with a message in
 * cactus_cuda_last_error(). The kernel entry points allocate nothing and can be captured in a
 * CUDA graph (after a first call of the same kind outside of it, which sets kernel attributes).
 * Lengths, offsets, tables and row lists are read on the device; what they name outside the
 * arguments (a page id that is not in [0, num_pages), a position past the end of a table row,
 * token rows past num_tokens) is skipped and raises the device error word
 * (cactus_cuda_device_error() == 3).
 *
 * Format. A pool holds pages of page_size rows (16, 32, 64, 128 or 256); page p's bytes for one
 * layer start at pool + p * page_stride and are, for each kv head,
 *
 *   key codes [page_size][head_dim / 2] | key parameters [page_size][head_dim / group_size]
 *   | value codes | value parameters
 *
 * Byte i of a row holds element 2i in its low and 2i + 1 in its high half. The parameters of a
 * group of group_size consecutive elements are two fp16 numbers, (step, low); code c stands for
 * fp16(c * step + low) with one rounding. The append takes low = the group's smallest element,
 * step = (largest - smallest) / 15 rounded towards zero, c = round-half-even((x - low) / step) in
 * 0..15, all of the exact differences. A constant group has step 0 and codes 0. A group that holds
 * an infinity or a NaN reads as NaN throughout, so that it shows in every output that sees it.
 *
 * Row r of sequence b is row r % page_size of page block_table[b * table_stride + r / page_size].
 * table_stride * page_size is below 2^31 - 1024. head_dim is 64, 128 or 256; group_size 32, 64 or
 * 128 and a divisor of head_dim. Pool and strides are 16-byte aligned.
 *
 * Batches are ragged: sequence b has the token rows token_offsets[b] .. token_offsets[b + 1] - 1
 * (token_offsets: [num_seqs + 1], rising from 0; token_offsets[num_seqs] <= num_tokens, and rows
 * past it are ignored) and context_lens[b] rows in the cache, its new ones included. So token i of
 * S has position context_lens[b] - S + i. Positions below 0 are ignored by the append, and such
 * queries see nothing but what the rule of the attention below gives them.
 */
#ifndef CACTUS_B200_KV4_H
#define CACTUS_B200_KV4_H

#include "cactus_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one page of one layer (the least page_stride); 0 where the geometry is not supported. */
CB_API size_t cactus_cuda_kv4_page_bytes(size_t page_size, size_t num_kv_heads, size_t head_dim, size_t group_size);

/* Quantises keys and values [num_tokens][num_kv_heads][head_dim], whose rows are row_stride fp16
 * elements apart (a multiple of 8; keys and values 16-byte aligned), into the pages. */
CB_API int cactus_cuda_kv4_append(const uint16_t* keys, const uint16_t* values, size_t row_stride,
                                  const int32_t* token_offsets, const int32_t* context_lens,
                                  const int32_t* block_table, size_t table_stride, void* pool, size_t num_pages,
                                  size_t page_stride, size_t num_seqs, size_t num_tokens, size_t page_size,
                                  size_t num_kv_heads, size_t head_dim, size_t group_size, void* stream);

/* Reads rows back as fp16: row j of sequence b's row_offsets[b + 1] - row_offsets[b] rows is its
 * position first_rows[b] + j (first_rows NULL: 0 for all) and goes to row row_offsets[b] + j of
 * keys and values [num_rows][num_kv_heads][head_dim] (16-byte aligned; either may be NULL). */
CB_API int cactus_cuda_kv4_read(const void* pool, size_t num_pages, size_t page_stride, const int32_t* block_table,
                                size_t table_stride, const int32_t* row_offsets, const int32_t* first_rows,
                                uint16_t* keys, uint16_t* values, size_t num_seqs, size_t num_rows, size_t page_size,
                                size_t num_kv_heads, size_t head_dim, size_t group_size, void* stream);

/* Softmax attention of queries [num_tokens][num_q_heads][head_dim] (rows query_stride elements
 * apart, a multiple of 8, 16-byte aligned) over the cached rows; q head h reads kv head
 * h / (num_q_heads / num_kv_heads). The query at position p sees position k of its sequence's
 * context_lens[b] rows where k <= p (if is_causal) and k > p - window_size (if window_size > 0).
 * output [num_tokens][num_q_heads][head_dim] fp16 (16-byte aligned), lse
 * [num_tokens][num_q_heads] fp32, natural log-sum-exp of the scaled scores (may be NULL). A query
 * that sees no row gives zeros and -inf. Pages that hold no visible row are not read (their table
 * entries may be anything); rows past context_lens[b] on a page that holds one may be loaded, and
 * whatever they hold does not reach a result. Scores, weights, their sums and the sums of weighted
 * values are fp32 (weights enter the products as two fp16 numbers, 22 bits); results are rounded once.
 * max_query_len bounds every sequence's token count; a longer one is cut there and raises the
 * device error word. workspace: cactus_cuda_kv4_attention_workspace() bytes, 16-byte aligned, zeroed
 * once before its first use; every call leaves it ready for the next, also of other shapes that
 * need no more bytes. Calls that may overlap in time need a workspace each. */
CB_API size_t cactus_cuda_kv4_attention_workspace(size_t num_seqs, size_t num_tokens, size_t num_q_heads,
                                                  size_t num_kv_heads, size_t head_dim);
CB_API int cactus_cuda_kv4_attention(const uint16_t* queries, size_t query_stride, const int32_t* token_offsets,
                                     const int32_t* context_lens, const int32_t* block_table, size_t table_stride,
                                     const void* pool, size_t num_pages, size_t page_stride, uint16_t* output,
                                     float* lse, size_t num_seqs, size_t num_tokens, size_t max_query_len,
                                     size_t num_q_heads, size_t page_size, size_t num_kv_heads, size_t head_dim,
                                     size_t group_size, float scale, size_t window_size, int is_causal,
                                     void* workspace, size_t workspace_bytes, void* stream);

/* Copies page src_pages[i] to page dst_pages[i] in each of num_planes planes (layers) that lie
 * plane_stride bytes apart: page_bytes bytes each, all sizes multiples of 16. Pages of any format.
 * A page may be the source of many copies; a destination is neither a source nor named twice. */
CB_API int cactus_cuda_kv_copy_pages(void* pool, size_t num_pages, size_t page_bytes, size_t page_stride,
                                     size_t num_planes, size_t plane_stride, const int32_t* src_pages,
                                     const int32_t* dst_pages, size_t num_copies, void* stream);

/* Moves the rows that sequences keep into other pages: row j of dst_table's sequence b becomes row
 * kept_rows[kept_offsets[b] + j] of src_table's (both [num_seqs][table_stride]), in every plane;
 * kept_offsets [num_seqs + 1] rises from 0 to num_kept. Destination pages are not source pages. */
CB_API int cactus_cuda_kv4_compact(void* pool, size_t num_pages, size_t page_stride, size_t num_planes,
                                   size_t plane_stride, const int32_t* src_table, const int32_t* dst_table,
                                   size_t table_stride, const int32_t* kept_rows, const int32_t* kept_offsets,
                                   size_t num_seqs, size_t num_kept, size_t page_size, size_t num_kv_heads,
                                   size_t head_dim, size_t group_size, void* stream);

/* ---- The cache as a handle: one pool for all layers of a model, and the pages of many sequences,
 * shared between forked ones until they are written. Lists of sequences, row counts and kept rows
 * are HOST arrays; keys, values, queries and results are device pointers. Sequences are numbered 0
 * to max_seqs - 1 and empty at first. The calls of one cache are made in order, on one stream or on
 * streams that the caller orders (a page that is freed is given out again); not from two threads at
 * once. They cannot be captured in a CUDA graph (a batch's counts are the host's; a call on a capturing
 * stream fails), the kernel entry points above can. A call that fails for its arguments or for lack of
 * pages changes nothing. */
typedef void* cactus_kv4_t;

/* num_pages pages of page_size rows for every layer, block tables for max_context rows, batches of up
 * to max_tokens new rows. NULL on failure. */
CB_API cactus_kv4_t cactus_kv4_create(size_t num_layers, size_t num_q_heads, size_t num_kv_heads, size_t head_dim,
                                      size_t group_size, size_t page_size, size_t num_pages, size_t max_seqs,
                                      size_t max_context, size_t max_tokens, int device);
/* Waits for nothing: no work of the cache may be in flight. */
CB_API void cactus_kv4_destroy(cactus_kv4_t cache);
/* Makes room for new_rows[i] rows at the end of sequence seqs[i] (none of them twice; a shared page
 * that these rows would be written into is copied first, in every layer) and makes these sequences the
 * batch that the next appends, for each layer, and attention calls are about: token rows of seqs[0],
 * seqs[1], ... one after another. The rows count as cached from here on. */
CB_API int cactus_kv4_begin(cactus_kv4_t cache, const int32_t* seqs, const int32_t* new_rows, size_t num_seqs,
                            void* stream);
/* cactus_cuda_kv4_append / _attention for the batch. */
CB_API int cactus_kv4_append(cactus_kv4_t cache, size_t layer, const uint16_t* keys, const uint16_t* values,
                             size_t row_stride, void* stream);
CB_API int cactus_kv4_attention(cactus_kv4_t cache, size_t layer, const uint16_t* queries, size_t query_stride,
                                uint16_t* output, float* lse, float scale, size_t window_size, int is_causal,
                                void* stream);
/* Rows first .. first + count - 1 of a sequence as fp16 [count][num_kv_heads][head_dim]. */
CB_API int cactus_kv4_read(cactus_kv4_t cache, size_t layer, int32_t seq, size_t first, size_t count, uint16_t* keys,
                           uint16_t* values, void* stream);
/* Sequence dst[i] becomes a copy of what src[i] was before the call (its pages are shared, nothing is
 * moved); what dst[i] held is freed. Beams are reordered in one call. Ends the batch, as do the next
 * three. */
CB_API int cactus_kv4_fork(cactus_kv4_t cache, const int32_t* src, const int32_t* dst, size_t n);
/* Keeps a sequence's first `length` rows (drafted tokens that were refused, for instance). */
CB_API int cactus_kv4_truncate(cactus_kv4_t cache, int32_t seq, size_t length);
CB_API int cactus_kv4_free(cactus_kv4_t cache, const int32_t* seqs, size_t n);
/* Keeps the rows kept_rows[kept_offsets[i]] .. of sequence seqs[i], in that order, in new pages; there
 * have to be enough free ones for them before the old ones are freed. */
CB_API int cactus_kv4_compact(cactus_kv4_t cache, const int32_t* seqs, const int32_t* kept_rows,
                              const int32_t* kept_offsets, size_t num_seqs, void* stream);
/* Rows of a sequence, or a negative error code. */
CB_API int cactus_kv4_length(cactus_kv4_t cache, int32_t seq);
/* out4 (host): pages, free pages, bytes of a page in one layer, bytes of the pool. */
CB_API int cactus_kv4_info(cactus_kv4_t cache, size_t* out4);

#ifdef __cplusplus
}
#endif
#endif
