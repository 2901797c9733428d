/*
 * aih_mx4.h -- C ABI of the operators on microscaled 4-bit rows.
 *
 *   aih_mx4_quant    rows of a storage type to 4 bits
 *   aih_mx4_dequant  the values that 4-bit rows stand for
 *   aih_mx4_pw       the pointwise conv (1x1) of 4-bit rows and 4-bit weights, with
 *                    bias, activation and residual
 *   aih_kv4_append   position rotation of queries and keys (after a norm of every
 *                    head, if wanted) and the new keys and values into the pages of
 *                    a 4-bit cache
 *   aih_kv4_attn     softmax attention over such a cache, prompts and single tokens
 *
 * The format (the OCP microscaling one with E2M1 elements): a row's elements in
 * blocks of 32, each with a scale byte s that stands for 2^(s - 127); an element is
 * a sign and one of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (codes 0 to 7, the sign is bit 3)
 * times the scale. Elements 2i and 2i + 1 are the low and the high half of a
 * block's byte i. Of a block with the largest magnitude m
 *   s = max(floor(log2 m) - 2, -127) + 127,
 * and an element becomes the nearest value, of two as near that of the even code,
 * above 6 scales 6. A block with a NaN or an infinity has s = 255 and codes 0 and
 * reads as NaN. The scale bytes 253 and 254 are never written; what they stand for
 * leaves fp32's range.
 *
 * The reference has no counterpart (its tensors are fp32 and f16); the conventions
 * are those of aih_conv.h: AIH_OK / AIH_ERR with the calling thread's message in
 * aih_last_error(), no exception across the boundary, caller-owned device buffers
 * on the current device, asynchronous on the caller's stream, nothing allocated by a
 * call, safe to call on several streams at once (each with a workspace of its own).
 * Rows of a storage type are `stride` elements apart (0 = dense); every tensor is
 * aligned to 16 bytes.
 */
#ifndef AIH_MX4_H
#define AIH_MX4_H

#include <stddef.h>
#include <stdint.h>

#include "aih_conv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Rows in 4 bits, as aih_mx4_quant writes and aih_mx4_pw reads them, one after
 * another: AIH_MX4_CODE_BYTES(k) bytes of codes, whole 128s of elements with 0 past
 * k, and AIH_MX4_SCALE_BYTES(k) bytes of scales, whole 512s; those of no element
 * are not written and may hold anything. */
#define AIH_MX4_CODE_BYTES(k) (((k) + 127) / 128 * 64)
#define AIH_MX4_SCALE_BYTES(k) (((k) + 511) / 512 * 16)

typedef struct {
  uint32_t rows;
  uint32_t k;        /* elements of a row: a multiple of 4, at most 2^20 */
  int32_t dt;        /* enum aih_dtype of x */
  uint64_t x_stride; /* elements, a multiple of 4, at most 2^22; 0 = k */
} aih_mx4_quant_desc;

/* x [rows][x_stride] -> codes and scales as above. */
int aih_mx4_quant(const aih_mx4_quant_desc *d, const void *x, void *codes, void *scales, aih_stream stream);

typedef struct {
  uint32_t rows;
  uint32_t k;            /* as above */
  int32_t dt;            /* enum aih_dtype of y */
  uint32_t code_stride;  /* bytes between rows of codes, a multiple of 16; 0 = AIH_MX4_CODE_BYTES(k) */
  uint32_t scale_stride; /* bytes between rows of scales; 0 = AIH_MX4_SCALE_BYTES(k) */
  uint64_t y_stride;     /* elements, a multiple of 4, at most 2^22; 0 = k */
} aih_mx4_dequant_desc;

/* codes, scales -> y [rows][y_stride], rounded once where y's type has not the
 * value (f16 alone). A 4-bit cache reads back with code_stride d / 2 and
 * scale_stride d / 32, its rows those of the pages. */
int aih_mx4_dequant(const aih_mx4_dequant_desc *d, const void *codes, const void *scales, void *y, aih_stream stream);

/* y[i][n] = act(sum_k x[i][k] w[n][k] + bias[n]) + res[i][n]; sums in fp32, one
 * rounding at the store. */
typedef struct {
  uint32_t m;       /* pixels (rows) of x and y */
  uint32_t k;       /* input channels: a multiple of 4, at most 2^20 */
  uint32_t cout;    /* output channels: a multiple of 4, at most 2^20 */
  int32_t act;      /* enum aih_act */
  int32_t residual; /* 0 or 1 */
  int32_t dt;       /* enum aih_dtype of bias, res and y */
} aih_mx4_pw_desc;

/* x_codes, x_scales [m] and w_codes, w_scales [cout]: rows as aih_mx4_quant makes
 * them (the weights of [cout][k]); bias [cout] or NULL; res (when d->residual) and
 * y [m][cout]. y may be res. */
int aih_mx4_pw(const aih_mx4_pw_desc *d, const void *x_codes, const void *x_scales, const void *w_codes,
               const void *w_scales, const void *bias, const void *res, void *y, aih_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* AIH_MX4_H */
