/*
 * ltx25_mx4.h -- C ABI of the microscaled 4-bit tier on MI355X (gfx950): rows
 * coded in 4 bits with an exponent for each block of 32, and the product of two
 * such operands on the matrix cores, at twice the int8 tier's rate and half its
 * bytes.
 *
 * Conventions as in ltx25_qlinear.h: caller-owned device tensors, asynchronous on
 * the caller's stream, LTX25_OK or an LTX25_E_* code with the message in
 * ltx25_last_error(), arguments checked before any device work. These calls keep
 * no scratch of the library's own: what a call needs beyond its tensors is the
 * caller's `workspace` (device memory, 16-byte aligned, any contents, in use until
 * the call has run), so calls on different streams may overlap and a call may be
 * captured into a HIP graph. Outputs and the workspace overlap nothing else of the call.
 */
#ifndef LTX25_MX4_H
#define LTX25_MX4_H

#include "ltx25_qlinear.h"

#ifdef __cplusplus
extern "C" {
#endif

/* `rows` rows of K values in blocks of 32 along K; K a multiple of 32. A value is a
 * code, a sign and one of the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6 (E2M1), times its
 * block's 2^exponent (E8M0: a byte, the exponent plus 127; 255 stands for a block of
 * NaN). Both lie in the order in which a wave of the matrix cores takes them, so that
 * its loads are whole lines (ltx25_mx4_pack lays out what a checkpoint holds):
 *   codes   ltx25_mx4_code_bytes(rows, K) bytes, 16-byte aligned, two values a byte with
 *           the earlier one in the low half; tiles of 16 rows by 128 values, the 16
 *           bytes of block b of row r at
 *             ((r / 16) * ceil(K / 128) + b / 4) * 1024 + ((b % 4) * 16 + r % 16) * 16
 *   scales  ltx25_mx4_scale_bytes(rows, K) bytes, 4-byte aligned; tiles of 16 rows by 16
 *           blocks, the byte of block b of row r at
 *             ((r / 16) * ceil(K / 512) + b / 16) * 256
 *               + ((b % 4) * 16 + r % 16) * 4 + (b / 4) % 4
 * The bytes of blocks past K in a row's last tile are 0; every call here that writes a
 * row writes them so. Those of rows past the last may hold anything. */
typedef struct ltx25_mx4 {
  void* codes;
  void* scales;
  int rows;
  int K;
} ltx25_mx4;

/* Bytes of `rows` rows of K values; 0 for sizes below 1 and a K that is no multiple
 * of 32. */
size_t ltx25_mx4_code_bytes(int rows, int K);
size_t ltx25_mx4_scale_bytes(int rows, int K);

/* Codes of q->rows rows of x, bf16 or f32 (x_dtype), x_stride elements from a row
 * to the next (at least K, rows 16-byte aligned). A block's exponent is
 * floor(log2(its largest magnitude)) - 2 within -127 .. 127, its codes are the
 * values divided by 2^exponent, rounded to the nearest code, ties to the even one,
 * magnitudes above 6 to 6. A block of zeros has exponent -127; a block that holds
 * an infinity or a NaN becomes a block of NaN. */
int ltx25_mx4_quantize_rows(void* stream, const void* x, int x_dtype, int64_t x_stride,
                            const ltx25_mx4* q);

/* The values as bf16, out_stride elements from a row to the next (a multiple of 8,
 * at least K; out 16-byte aligned). Exact, but for values above bf16's largest, which
 * are infinite. */
int ltx25_mx4_dequant(void* stream, const ltx25_mx4* q, void* out, int64_t out_stride);

/* From u8 codes [rows][K / 2] and scales [rows][K / 32], as checkpoints hold them, to
 * q's order, and back. Both 16-byte aligned. */
int ltx25_mx4_pack(void* stream, const void* codes, const void* scales, const ltx25_mx4* q);
int ltx25_mx4_unpack(void* stream, const ltx25_mx4* q, void* codes, void* scales);

/* y[M][N] = epilogue(x . w^T + bias): M = x->rows, N = w->rows, both of one K. Both
 * operands are exact in the products, which are added in f32; bias (LTX25_DT_*) and
 * epilogue (LTX25_EPI_*) in f32 as in ltx25_linear_q_ex, one rounding to bf16.
 * y 16-byte aligned and dense. Codes of w below 2 GiB (LTX25_E_UNSUPPORTED).
 * workspace: at least ltx25_mx4_gemm_workspace(M, K, N) bytes. */
int ltx25_mx4_gemm(void* stream, const ltx25_mx4* x, const ltx25_mx4* w, const void* bias,
                   int bias_dtype, void* y, int epilogue, void* workspace, size_t workspace_bytes);
/* 0: no size needs any at present, and none is looked at. */
size_t ltx25_mx4_gemm_workspace(int M, int K, int N);

/* The same with M rows of bf16 activations (x_stride elements from a row to the next,
 * a multiple of 8; x 16-byte aligned), which are coded as ltx25_mx4_quantize_rows
 * codes them on the way: the bits of the two calls.
 * workspace: at least ltx25_linear_mx4_workspace(M, K, N) bytes, the coded rows' (0 where
 * up to 16 rows are coded in the product's own kernel, and for sizes that the call
 * refuses); what the largest sizes of several calls need is enough for all. */
int ltx25_linear_mx4(void* stream, const void* x, int64_t x_stride, int M, const ltx25_mx4* w,
                     const void* bias, int bias_dtype, void* y, int epilogue, void* workspace,
                     size_t workspace_bytes);
size_t ltx25_linear_mx4_workspace(int M, int K, int N);

#ifdef __cplusplus
}
#endif

#endif /* LTX25_MX4_H */
