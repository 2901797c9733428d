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
 * another: AIH_MX4_CODE_BYTES(k) bytes of codes, whole 128s of elements, and
 * AIH_MX4_SCALE_BYTES(k) bytes of scales, room for whole 512s. Codes and scales of a
 * row's last 128 that are past k are 0; scales behind those are not written and may
 * hold anything. */
#define AIH_MX4_CODE_BYTES(k) (((k) + 127) / 128 * 64)
#define AIH_MX4_SCALE_BYTES(k) (((k) + 511) / 512 * 16)

typedef struct {
  uint32_t rows;     /* rows of k rounded up to 128 hold at most 2^35 - 2048 elements */
  uint32_t k;        /* elements of a row: a multiple of 4, at most 2^20 */
  int32_t dt;        /* enum aih_dtype of x */
  uint64_t x_stride; /* elements, a multiple of 4, at most 2^22; 0 = k */
} aih_mx4_quant_desc;

/* x [rows][x_stride] -> codes and scales as above. */
int aih_mx4_quant(const aih_mx4_quant_desc *d, const void *x, void *codes, void *scales, aih_stream stream);

typedef struct {
  uint32_t rows;         /* rows of k rounded up to 8 hold at most 2^35 - 2048 elements */
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
  uint32_t m;       /* pixels (rows) of x and y, at most 2^31 - 256 */
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

/* A 4-bit cache. It holds rows of `hkv` heads of d elements in pages of `page` rows:
 * codes [pages][hkv][page][d / 2] and scales [pages][hkv][page][d / 32] bytes, each
 * for the keys and for the values. Row r of the cache is row r % page of page r / page.
 *
 * Row t of x holds hq query, hkv key and hkv value heads. Of each query and key head
 *   y = x * rsqrt(mean(x^2) + eps) * w   when `norm` (w: wq or wk, d elements; NULL =
 * 1), else y = x, and, for i < rot / 2 with (a, b) = (y[i], y[i + rot/2]), or (y[2i],
 * y[2i+1]) when `pairs`, c and s = row pos[t] of the tables,
 *   a' = a c - b s,  b' = a s + b c
 * in fp32, every product and sum rounded by itself; dims from `rot` on are not
 * rotated. Queries are rounded to q; keys and values (as they are in x) become row
 * slots[t] of the cache. */
typedef struct {
  uint32_t tokens;    /* rows of x and q; tokens * (hq + 2 hkv) at most (2^24 - 1) * 4 * (512 / d) */
  uint32_t hq, hkv;   /* heads; hq may be 0, hkv not */
  uint32_t d;         /* elements of a head: a multiple of 32, at most 256 */
  uint32_t rot;       /* rotated dims: a multiple of 16, at most d; 0 = none */
  int32_t pairs;      /* 1 = adjacent pairs, 0 = halves */
  int32_t norm;       /* 0 or 1 */
  float eps;          /* >= 0, finite; with 0 a head of zeros has no norm (NaN) */
  int32_t dt;         /* enum aih_dtype: x, wq, wk, q */
  uint32_t positions; /* rows of the tables (used when rot > 0) */
  uint32_t page;      /* rows of a page: a power of two, 16 to 4096 */
  uint32_t pages;     /* pages of the cache; pages * page below 2^31 */
  uint64_t x_stride, q_stride; /* elements, whole 16-byte units; 0 = dense */
} aih_kv4_append_desc;

/* cosines, sines [positions][rot/2] fp32; pos [tokens] int32, NULL = the token's own
 * index (positions outside the tables use the nearest row); slots [tokens] int32,
 * outside [0, pages * page) = the key and value are dropped; tokens of one call with the
 * same slot leave a row that mixes theirs. q may be x's own query heads (same pointer and
 * row stride). */
int aih_kv4_append(const aih_kv4_append_desc *d, const void *x, const void *wq, const void *wk, const float *cosines,
                   const float *sines, const int32_t *pos, const int32_t *slots, void *q, void *k_codes, void *k_scales,
                   void *v_codes, void *v_scales, aih_stream stream);

/* Attention over a 4-bit cache. Sequence b has the query rows [q_start[b],
 * q_start[b+1]); its key and value j are row j % page of page table[b][j / page], j <
 * k_len[b]. Query head h reads key head h / (hq / hkv). With Lq queries and Lk keys,
 * query i sees the keys j < Lk, of those only j <= i + Lk - Lq when `causal` (the
 * queries are the last Lq positions), and none in a page outside [0, pages):
 *   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * q_i . k_j)
 * A query that sees no key gives 0. What a query does not see never reaches its
 * output. Keys and values are exact in the products, statistics and sums fp32; fp32
 * queries and probabilities enter as three bf16 terms (all their bits), f16 ones as
 * two (16 bits of a probability), bf16 probabilities are rounded to bf16 and their sum is
 * of the rounded ones. Values of any size are averaged without leaving fp32's range, but
 * those below 6 * 2^-122 * Lk (Lk rounded up to a power of two, 32 at least) may read as
 * zero; what fp32 queries have below 2^-133 is lost. */
typedef struct {
  uint32_t nseq;        /* sequences; 0 is allowed */
  uint32_t tokens;      /* rows of q and o; tokens * hq below 2^31 */
  uint32_t hq, hkv;     /* hq a multiple of hkv */
  uint32_t d;           /* elements of a head: a multiple of 32, at most 256 */
  uint32_t page, pages; /* as above */
  uint32_t table_width; /* entries of a sequence in the table; table_width * page below 2^31 */
  int32_t causal;       /* 0 or 1 */
  float scale;          /* finite, 1e-20 to 1e20; 0 = 1 / sqrt(d) */
  int32_t dt;           /* enum aih_dtype: q, o */
  uint32_t max_len;     /* the longest k_len, as far as known (0: all that a table row holds); steers
                           how the keys are split, results hold for any lengths. A call is planned
                           by its average sequence: where that has more than 32 (query, head of a
                           group) rows and the tiles fill the chip, no keys are split, so single
                           tokens over long caches beside prompts belong in a call of their own */
  uint64_t q_stride, o_stride; /* elements, whole 16-byte units; 0 = dense */
} aih_kv4_attn_desc;

typedef struct {
  uint32_t bm;     /* (query, head of a group) rows of a workgroup's tile */
  uint32_t parts;  /* most parts a sequence's keys are cut into */
  uint32_t chunk;  /* keys of a part, unless more parts would be needed; 0 = not cut */
  uint32_t grid;   /* workgroups, at most */
  size_t ws_bytes; /* workspace: (d + 2) fp32 values for each of tokens * hq rows and each
                      part; 0 when no row's keys are cut */
} aih_kv4_attn_plan_info;

int aih_kv4_attn_plan(const aih_kv4_attn_desc *d, aih_kv4_attn_plan_info *out);

/* q_start [nseq + 1] (not descending), table [nseq][table_width], k_len [nseq]: int32
 * device arrays; lengths past the table and starts past the tensors are cut there, and a
 * row of o that no sequence covers is not written. ws: plan.ws_bytes of device
 * memory (may be NULL when 0). */
int aih_kv4_attn(const aih_kv4_attn_desc *d, const void *q, const void *k_codes, const void *k_scales,
                 const void *v_codes, const void *v_scales, const int32_t *q_start, const int32_t *table,
                 const int32_t *k_len, void *o, void *ws, size_t ws_bytes, aih_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* AIH_MX4_H */
