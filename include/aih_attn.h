/*
 * aih_attn.h -- C ABI of the attention operators that run between the two
 * pointwise convs of an attention block (aih_conv_pw makes the rows of
 * queries, keys and values and projects the result back).
 *
 *   aih_qk_norm_rope  norm of every query and key head and the position
 *                     rotation in one pass over the projection's rows; keys
 *                     and values go to their cache rows
 *   aih_attn          softmax attention of packed sequences of different
 *                     lengths with grouped heads: whole prompts, one or a few
 *                     tokens over a long cache, and either behind a prefix
 *                     that all sequences share
 *
 * The reference has no counterpart (its graphs are convolutional); the
 * conventions are those of aih_conv.h: AIH_OK / AIH_ERR with the calling
 * thread's message in aih_last_error(), no exception across the boundary,
 * caller-owned device buffers, asynchronous on the caller's stream, nothing
 * allocated by a call, safe to call on several streams at once (each with a
 * workspace of its own). Statistics, sums and partial results are fp32 in every
 * storage type; probabilities are rounded to it for their product with the
 * values, and their sum is of the rounded ones.
 *
 * A row of a tensor holds its heads one after another, d elements each; rows
 * are `stride` elements apart (0 = dense), so keys and values may stay inside
 * the projection's rows (a pointer to their first head and the row's stride).
 * Tensors are aligned to 16 bytes and row strides are whole 16-byte units of at
 * most 2^22 elements.
 */
#ifndef AIH_ATTN_H
#define AIH_ATTN_H

#include <stddef.h>
#include <stdint.h>

#include "aih_conv.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Head norms and rotation. Row t of x holds hq query, hkv key and hkv value
 * heads. Of each query and key head
 *   y = x * rsqrt(mean(x^2) + eps) * w          (w: wq or wk, d elements; NULL = 1)
 * and, for i < rot / 2 with (a, b) = (y[i], y[i + rot/2]), or (y[2i], y[2i+1])
 * when `pairs`, c and s = row pos[t] of the tables,
 *   a' = a c - b s,  b' = a s + b c;
 * dims from `rot` on are not rotated; one rounding, at the store. */
typedef struct {
  uint32_t tokens;    /* rows of x and q */
  uint32_t hq, hkv;   /* heads; hkv 0: no keys and values */
  uint32_t d;         /* elements of a head: a multiple of 8, at most 256 */
  uint32_t rot;       /* rotated dims: a multiple of 4, at most d; 0 = none */
  int32_t pairs;      /* 1 = adjacent pairs, 0 = halves */
  float eps;          /* >= 0, finite; with 0 a head of zeros has no norm (NaN) */
  int32_t dt;         /* enum aih_dtype: x, wq, wk, q, k, v */
  uint32_t positions; /* rows of the tables (used when rot > 0) */
  uint32_t rows;      /* rows of k and v */
  uint64_t x_stride, q_stride, k_stride, v_stride; /* elements; 0 = dense */
} aih_qk_norm_rope_desc;

/* cosines, sines [positions][rot/2] fp32; pos [tokens] int32, NULL = the
 * token's own index (positions outside the tables use the nearest row); slots
 * [tokens] int32, NULL = row t: the row of k and v that token t's key and
 * value go to, outside [0, rows) = they are dropped. Two tokens with the same
 * slot leave either's key and value. v NULL leaves the values in x. q may be
 * x's own query heads (same pointer and row stride), and so may k with slots
 * NULL be its key heads. */
int aih_qk_norm_rope(const aih_qk_norm_rope_desc *d, const void *x, const void *wq, const void *wk,
                     const float *cosines, const float *sines, const int32_t *pos, const int32_t *slots, void *q,
                     void *k, void *v, aih_stream stream);

/* Attention. Sequence b has the query rows [q_start[b], q_start[b+1]) and the
 * key and value rows [k_start[b], k_start[b] + k_len[b]); query head h reads
 * key head h / (hq / hkv). With Lq queries and Lk keys, query i sees the
 * prefix and the keys j < Lk, of those only j <= i + Lk - Lq when `causal` (the
 * queries are the last Lq positions):
 *   o_i = sum_j p_ij v_j / sum_j p_ij,   p_ij = exp(scale * q_i . k_j)
 * A query that sees no key gives 0. What a query does not see never reaches
 * its output, NaN and infinity included. */
typedef struct {
  uint32_t nseq;    /* sequences; 0 is allowed */
  uint32_t tokens;  /* rows of q and o: all sequences together */
  uint32_t rows;    /* rows of k and v */
  uint32_t hq, hkv; /* hq a multiple of hkv */
  uint32_t d;       /* elements of a head: a multiple of 8, at most 256 */
  int32_t causal;   /* 0 or 1 */
  float scale;      /* finite, 1e-20 to 1e20; 0 = 1 / sqrt(d) */
  int32_t dt;       /* enum aih_dtype: q, k, v, prefix, o */
  uint32_t max_len; /* the longest k_len, as far as known (0: rows / nseq); steers how
                       the keys are split, results hold for any lengths */
  uint32_t prefix;  /* rows of the shared prefix, 0 = none */
  uint64_t q_stride, k_stride, v_stride, o_stride; /* elements; 0 = dense */
  uint64_t pk_stride, pv_stride;                   /* of the prefix */
} aih_attn_desc;

enum aih_attn_kernel {
  AIH_ATTN_ROWS = 1, /* a tile's query rows spread over the wavefronts, keys shared */
  AIH_ATTN_KEYS = 2  /* 32 query rows, the keys spread over the wavefronts */
};

typedef struct {
  int32_t kernel;        /* enum aih_attn_kernel of the sequences' own keys */
  uint32_t bm;           /* (query, head of a group) rows of a workgroup's tile */
  uint32_t parts;        /* most parts a sequence's keys are cut into */
  uint32_t chunk;        /* keys of a part, unless more parts would be needed */
  int32_t prefix_kernel; /* the same for the prefix, 0 = no prefix */
  uint32_t prefix_bm, prefix_parts, prefix_chunk;
  uint32_t grid;         /* workgroups of the first launch, which a prefix leads or has to
                            itself; at most: where keys are cut, no more than run at once
                            are launched and share the work */
  size_t ws_bytes;       /* workspace: (d + 2) fp32 values for each of tokens * hq rows and
                            each part, the prefix's and the own keys' together; 0 when no
                            row's keys are cut. A prefix always leaves two parts or more */
} aih_attn_plan_info;

int aih_attn_plan(const aih_attn_desc *d, aih_attn_plan_info *out);

/* q_start [nseq + 1] (not descending), k_start and k_len [nseq]: int32 device
 * arrays; starts and lengths that reach past the tensors are cut there, and a
 * row of o that no sequence covers is not written. prefix_k / prefix_v are read when
 * d->prefix > 0. ws: plan.ws_bytes of device memory, aligned to 16 bytes (may
 * be NULL when 0). */
int aih_attn(const aih_attn_desc *d, const void *q, const void *k, const void *v, const int32_t *q_start,
             const int32_t *k_start, const int32_t *k_len, const void *prefix_k, const void *prefix_v, void *o,
             void *ws, size_t ws_bytes, aih_stream stream);

#ifdef __cplusplus
}
#endif

#endif /* AIH_ATTN_H */
