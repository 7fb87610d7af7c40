/*
 * ltx25_attention.h -- C ABI of attention on MI355X (gfx950): packed prompts,
 * and a paged cache of 8-bit keys and values with the attention that reads it.
 *
 * These ops stand between the block's projections and the per-head gate
 * (ltx25_linear_q ... ltx25_gate_heads in ltx25_qlinear.h) and keep that
 * header's conventions: caller-owned device tensors, asynchronous on the
 * caller's stream, LTX25_OK or an LTX25_E_* code with the message in
 * ltx25_last_error(), arguments checked before any device work. Unlike the
 * linears they keep no scratch of the library's own: what a call needs beyond
 * its tensors is the caller's `workspace`, so calls on different streams may
 * overlap and a call may be captured into a HIP graph.
 *
 * A call takes at most 2^27 packed tokens (queries, keys or new cache tokens), and
 * sequences of a cache at most 2^30.
 *
 * Lengths, cumulative lengths and page tables are device memory, so that a
 * serving loop can keep them on the GPU; they are read when the kernels run.
 * The kernels keep every access inside the sizes given by the host whatever
 * they hold: a length past its bound is cut to it, a page id outside the cache
 * is a page that no query sees.
 */
#ifndef LTX25_ATTENTION_H
#define LTX25_ATTENTION_H

#include "ltx25_qlinear.h"

#ifdef __cplusplus
extern "C" {
#endif

/* How a call's heads lie in its tensors. A token's query heads are
 * [heads][head_dim] bf16, its keys and values [kv_heads][head_dim], side by
 * side; the strides are the elements from one token to the next, so q, k and v
 * may be parts of one fused projection's output. Query head h reads kv head
 * h / (heads / kv_heads).
 *   head_dim 64 or 128; heads a multiple of kv_heads; strides multiples of 8,
 *   at least the token's own width and below 2^23; tensors 16-byte aligned.
 * scale: the logits' factor, positive and finite (0: 1 / sqrt(head_dim)).
 * causal: the last query of a sequence sees its last key, the one before it
 * one key less, and so on; else every query sees every key. */
typedef struct ltx25_attn {
  int heads;
  int kv_heads;
  int head_dim;
  int causal;
  float scale;
  int64_t q_stride;
  int64_t k_stride;     /* ltx25_attention alone */
  int64_t v_stride;     /* ltx25_attention alone */
  int64_t out_stride;
} ltx25_attn;

/* Attention of `batch` sequences packed one after another.
 *   q [total_q], k and v [total_k], out [total_q] tokens (ltx25_attn).
 *   cu_q, cu_k: int32 [batch + 1], sequence b's queries are tokens
 *   cu_q[b] .. cu_q[b + 1] - 1 and its keys cu_k[b] .. cu_k[b + 1] - 1; the
 *   numbers of queries and keys may differ, either may be zero. Both may be
 *   NULL with batch 1: one sequence of total_q queries and total_k keys.
 *   lse: float [total_q][heads] or NULL: the natural logarithm of the sum of
 *   the exponentials, to merge with attention over other keys.
 * out may not overlap q, k or v.
 * A query that sees no key gives zeros and an lse of -infinity. A key or value
 * that a query does not see adds nothing to it, be it infinite or NaN; an infinite
 * value that it does see shows in its channel, however small its weight. (Rows side
 * by side take their maxima together: what one of them sees may change the last bits
 * of another's rounding, within the errors below. A call with the same tensors gives
 * the same bits.) Values count over f32's whole range of normal numbers.
 * Products of bf16, sums and softmax statistics in f32; the weights are rounded
 * to bf16 for the second product; one rounding to bf16 at the end. */
int ltx25_attention(void* stream, const ltx25_attn* a, const void* q, const void* k, const void* v,
                    void* out, float* lse, const int* cu_q, const int* cu_k, int batch,
                    int total_q, int total_k);

/* The same where few rows see many keys (a few queries behind a long prefix, few
 * heads): the keys are split over more workgroups and the parts joined in one fixed
 * order, in a workspace as ltx25_attention_cached's: device memory of at least
 * ltx25_attention_workspace() bytes, 16-byte aligned, any contents, in use until the
 * call has run. Where that is 0 there is nothing to split, no workspace is needed and
 * the call is ltx25_attention's. */
int ltx25_attention_split(void* stream, const ltx25_attn* a, const void* q, const void* k,
                          const void* v, void* out, float* lse, const int* cu_q, const int* cu_k,
                          int batch, int total_q, int total_k, void* workspace,
                          size_t workspace_bytes);

/* Bytes of workspace that ltx25_attention_split needs; 0 for sizes it refuses and where
 * it splits nothing. Not monotone in the sizes. */
size_t ltx25_attention_workspace(const ltx25_attn* a, int batch, int total_q, int total_k);

/* A cache of keys and values in pages of page_tokens tokens, held as signed
 * bytes with one scale for each page and kv head: value = code * scale.
 *   k        int8 [pages][kv_heads][page_tokens][head_dim]
 *   v        int8 [pages][kv_heads][head_dim][page_tokens]: a channel's tokens
 *            side by side, as the product with the weights reads them
 *   k_scale, v_scale   float [pages][kv_heads]
 * page_tokens 16, 32, 64 or 128; head_dim 64 or 128; k and v 16-byte aligned.
 * Any contents are valid, and a page needs no clearing before its first use.
 *
 * Tables: int32 [batch][table_stride]; token t of sequence b lies in page
 * table[b][t / page_tokens]. */
typedef struct ltx25_kv_cache {
  void* k;
  void* v;
  float* k_scale;
  float* v_scale;
  int pages;
  int page_tokens;
  int kv_heads;
  int head_dim;
} ltx25_kv_cache;

/* Quantizes new keys and values into the cache.
 *   k, v: bf16 [total] tokens of [kv_heads][head_dim] at k_stride / v_stride
 *   (as in ltx25_attn); cu int32 [batch + 1] as cu_k above.
 *   start int32 [batch]: the tokens that sequence b's cache holds already; its
 *   new ones become tokens start[b], start[b] + 1, ...
 * A page's scale is absmax / 127 over the finite values written to it, and only
 * grows while tokens before the new ones stay in the page; those are then
 * requantized from their codes: rint(code * old scale / new scale). Codes are
 * rint(x / scale), ties to even, within +-127; infinities give +-127, NaN 0.
 * Contents of a written page past the last new token are undefined, and no page
 * may be written by two sequences of one call. The table must hold pages for
 * the new tokens; tokens past table_stride pages are dropped. */
int ltx25_kv_append(void* stream, const ltx25_kv_cache* cache, const int* table, int table_stride,
                    const void* k, const void* v, int64_t k_stride, int64_t v_stride,
                    const int* cu, const int* start, int batch, int total);

/* Reads tokens back as bf16 (code * scale, rounded once): sequence b's tokens
 * start[b], start[b] + 1, ... become tokens cu[b] .. cu[b + 1] - 1 of k and v
 * [total], the packed layout of ltx25_attention's keys: a resumed prompt
 * attends to its prefix that way. Tokens without a page give zeros. */
int ltx25_kv_read(void* stream, const ltx25_kv_cache* cache, const int* table, int table_stride,
                  void* k, void* v, int64_t k_stride, int64_t v_stride, const int* cu,
                  const int* start, int batch, int total);

/* Attention over the cache: q_len queries of each of `batch` sequences (1 when
 * decoding, a few when a draft is checked; any number is taken), q and out
 * [batch * q_len] tokens, sequence by sequence, lse [batch * q_len][heads] or
 * NULL as in ltx25_attention.
 *   lens int32 [batch]: the tokens of each sequence's cache, the queries' own
 *   among them (ltx25_kv_append comes first). max_len: at least the largest; a
 *   longer one is cut to it.
 *   workspace: device memory of at least ltx25_attention_cached_workspace()
 *   bytes, 16-byte aligned, any contents, in use until the call has run (NULL
 *   where that is 0).
 * Keys and values enter both products as their exact codes; a page's scales
 * multiply the logits and the weights in f32, and these are rounded to f16 (under
 * a power of two of the row's) for the second product: a weight times its scale that
 * is 2^26 times smaller than the row's largest has fewer than 11 bits, and one 2^37
 * times smaller counts as zero. The tokens are split over
 * workgroups and the parts joined in one fixed order: the same call gives the
 * same bits. */
int ltx25_attention_cached(void* stream, const ltx25_attn* a, const ltx25_kv_cache* cache,
                           const int* table, int table_stride, const int* lens, const void* q,
                           void* out, float* lse, int batch, int q_len, int max_len,
                           void* workspace, size_t workspace_bytes);

/* Bytes of workspace that ltx25_attention_cached needs; 0 for sizes it refuses
 * and where it needs none. Not monotone: a smaller batch or fewer queries may be
 * split into more parts and need more. A program that makes calls of several sizes
 * with one workspace takes the largest of theirs. */
size_t ltx25_attention_cached_workspace(int batch, int q_len, int heads, int kv_heads, int head_dim,
                                        int max_len);

#ifdef __cplusplus
}
#endif

#endif /* LTX25_ATTENTION_H */
