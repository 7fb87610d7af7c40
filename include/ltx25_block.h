/*
 * ltx25_block.h -- C ABI of what a block does around its linears and its attention
 * on MI355X (gfx950): norms fused with the gate, the residual and the modulation,
 * positions rotated into queries and keys, and keys rotated on their way into the
 * paged cache.
 *
 * Conventions as in ltx25_qlinear.h and ltx25_attention.h: caller-owned device
 * tensors, asynchronous on the caller's stream, LTX25_OK or an LTX25_E_* code with
 * the message in ltx25_last_error(), arguments checked before any device work; no
 * scratch, so calls on different streams may overlap and a call may be captured
 * into a HIP graph.
 *
 * A call takes at most 2^27 tokens. Indices, positions and tables are device memory,
 * read when the kernels run; whatever they hold, every access stays inside the sizes
 * given by the host.
 */
#ifndef LTX25_BLOCK_H
#define LTX25_BLOCK_H

#include "ltx25_attention.h"
#include "ltx25_mx4.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LTX25_DT_I32 3   /* positions alone */

/* ---- norms ------------------------------------------------------------------ */

/* Sizes and types of a norm's tensors. Strides: elements from a token (a modulation
 * row) to the next, multiples of 8, at least the width; every tensor 16-byte
 * aligned.
 *   width      1 .. 16384 values a token, a multiple of 8 (32 with 4-bit output)
 *   layer      0: x / sqrt(mean(x^2) + eps); 1: the same of x - mean(x)
 *   eps        2^-80 or more
 *   residual_scale  alpha below; finite
 *   x_dtype    LTX25_DT_BF16 or LTX25_DT_F32: x and x_out
 *   mod_dtype, weight_dtype   the same choice for gate, scale and shift, and for the
 *              two weights
 *   mod_rows   rows of gate, scale and shift (1 or more where one of them is given) */
typedef struct ltx25_norm {
  int width;
  int layer;
  float eps;
  float residual_scale;
  int x_dtype;
  int mod_dtype;
  int weight_dtype;
  int mod_rows;
  int64_t x_stride;
  int64_t x_out_stride;
  int64_t y_stride;
  int64_t mod_stride;
  int64_t out_stride;
} ltx25_norm;

/* The end of one block and the start of the next, for each token:
 *   u     = y, or norm(y) post_weight where post_weight is given   (y bf16 or NULL)
 *   x_out = alpha x + gate u                                       (where y is given)
 *   out   = norm(x_out) weight (1 + scale) + shift                 (bf16, one rounding)
 * Without y, out is of x, and post_weight, gate and x_out must be NULL. gate, weight,
 * scale and shift may each be NULL (1, 1, 0, 0), and out may where y is given.
 * weight, post_weight [width]; gate, scale and shift [mod_rows][width].
 *   rows: int32 [tokens], the modulation row of each token (cut to the rows there
 *   are), or NULL: the rows belong to equal runs of tokens one after another (tokens
 *   a multiple of mod_rows).
 * out is of x_out before that is rounded. Sums and statistics in f32, for values over
 * f32's whole range. x_out may be x, and out may be x (bf16, of one stride) where y is
 * not given, or y; else outputs overlap nothing. */
int ltx25_block_norm(void* stream, const ltx25_norm* n, const void* x, const void* y, void* x_out,
                     const void* post_weight, const void* gate, const void* weight,
                     const void* scale, const void* shift, const int* rows, void* out, int tokens);

/* The same with out in 4 bits (q->rows tokens of width q->K), coded from the values
 * before any rounding to bf16: the activations of ltx25_mx4_gemm. out_stride is not
 * used; the outputs overlap nothing but x_out, which may be x. */
int ltx25_block_norm_mx4(void* stream, const ltx25_norm* n, const void* x, const void* y,
                         void* x_out, const void* post_weight, const void* gate,
                         const void* weight, const void* scale, const void* shift,
                         const int* rows, const ltx25_mx4* q, int tokens);

/* ---- positions -------------------------------------------------------------- */

/* Rotated positions of one to four axes. Pair p of a head is turned by the angle
 * position[token][axis[p]] * freq[p] (radians): (a, b) becomes
 * (a cos - b sin, a sin + b cos).
 *   head_dim  16 .. 256, a multiple of 16
 *   rot_dim   the channels that are rotated, the head's first ones: a multiple of 16,
 *             at most head_dim (0: head_dim); rot_dim / 2 pairs
 *   interleaved  pair p is channels 2 p and 2 p + 1; else p and p + rot_dim / 2
 *   freqs     float [freq_heads][rot_dim / 2], 16-byte aligned
 *   axes      int32 [freq_heads][rot_dim / 2], 16-byte aligned (cut to the axes there
 *             are), or NULL: the first axis
 *   freq_heads  1, or the number of heads (of the queries and of the keys): a head's
 *             own frequencies
 *   positions [tokens][n_axes], LTX25_DT_F32 or LTX25_DT_I32 (pos_dtype)
 * Whole turns are taken off the product in 64 bits before it is rounded: angles lose
 * nothing that counts below 2^52 radians (every int32 position at a frequency up to 2^21;
 * larger ones turn by no particular angle). Sines and cosines are good to 2^-20. Negated
 * frequencies turn back. */
typedef struct ltx25_rotation {
  int head_dim;
  int rot_dim;
  int interleaved;
  int n_axes;
  int freq_heads;
  int pos_dtype;
  const float* freqs;
  const int* axes;
  const void* positions;
} ltx25_rotation;

/* Rotates queries and keys, bf16 [tokens] of [heads][head_dim] at their strides (as in
 * ltx25_attn), into q_out and k_out, which may be q and k (q_out q, k_out k, at the same
 * strides); else the outputs overlap nothing. q or k may be NULL with 0 heads. One
 * rounding to bf16. */
int ltx25_rope(void* stream, const ltx25_rotation* r, const void* q, void* q_out, int heads,
               int64_t q_stride, int64_t q_out_stride, const void* k, void* k_out, int kv_heads,
               int64_t k_stride, int64_t k_out_stride, int tokens);

/* ltx25_kv_append with the keys rotated on the way: the bits of ltx25_rope on k (one
 * rounding to bf16, the type that a prompt's attention reads) and ltx25_kv_append,
 * without writing the rotated keys. head_dim is the cache's.
 *   r->positions [total][n_axes] of the new tokens, or NULL: every axis of a token is
 *   its place in its sequence, start[b] + i. */
int ltx25_kv_append_rope(void* stream, const ltx25_kv_cache* cache, const int* table,
                         int table_stride, const void* k, const void* v, int64_t k_stride,
                         int64_t v_stride, const int* cu, const int* start,
                         const ltx25_rotation* r, int batch, int total);

#ifdef __cplusplus
}
#endif

#endif /* LTX25_BLOCK_H */
