// attn.h -- kernel arguments and launchers of the attention operators
// (include/aih_attn.h). Everything here is checked by attn_capi.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/aih_attn.h"
#include "aih_device.h"

namespace aih {

struct QkRopeArgs {
  const void *x, *wq, *wk;
  const float *cs, *sn;
  const int32_t *pos, *slots;
  void *q, *k, *v;
  uint64_t xs, qs, ks, vs;  // row strides, elements
  uint32_t hq, hkv, ht;     // ht: heads handled per token (without the values when v is NULL)
  uint32_t d, rot, pairs;
  uint32_t units, ru;       // vectors per head; of them in the first rotated half (halves only)
  uint32_t nl;              // lanes a head needs: ceil(units / 2)
  uint32_t positions, rows;
  uint64_t items;           // tokens * ht
  float eps, inv_d;
};

hipError_t launch_qk_norm_rope(const QkRopeArgs &a, int dt, hipStream_t st);

// One launch: the sequences against their own keys, with the prefix's work in
// front (pre_tiles > 0, AIH_ATTN_KEYS only); or, with k_start NULL
// (AIH_ATTN_ROWS only), all rows against k and v as one sequence.
struct AttnArgs {
  const void *q, *k, *v, *pk, *pv;
  void *o;
  float *ws;  // partial results; NULL: no row's keys are cut, o is written
  const int32_t *q_start, *k_start, *k_len;
  uint64_t qs, ks, vs, os, pks, pvs;  // row strides, elements
  uint32_t nseq, tokens, rows, prefix;
  uint32_t hq, hkv, g, d;
  uint32_t causal;
  float scale_log2;  // scale * log2(e)
  uint32_t tiles;    // row tiles of a key head, at most
  uint32_t parts, shift, part0;             // parts of a sequence at most, log2 keys of a part, first part's index in ws
  uint32_t pre_tiles, pre_parts, pre_shift;  // the prefix's
  FastDiv by_g, by_hkv, by_pre_tiles;
  uint32_t all_parts;
  uint32_t span;  // keys of the longest part, as far as known
  uint32_t sort;  // 1: the sequences with the most keys go first
};

// The workspace: O of every part [all_parts][tokens * hq][d] fp32, not yet
// divided by the sum, then (maximum, sum) pairs [all_parts][tokens * hq][2]; a
// sum of -1 in part 0: the row's o is written already.
__host__ __device__ inline uint64_t attn_ws_ml(const AttnArgs &a) {
  return (uint64_t)a.all_parts * a.tokens * a.hq * a.d;
}

// Rows of a tile (enum aih_attn_kernel).
uint32_t attn_bm(int kernel);

hipError_t launch_attn(const AttnArgs &a, int kernel, int dt, hipStream_t st);
hipError_t launch_attn_f32(const AttnArgs &a, int kernel, hipStream_t st);
hipError_t launch_attn_f16(const AttnArgs &a, int kernel, hipStream_t st);
hipError_t launch_attn_bf16(const AttnArgs &a, int kernel, hipStream_t st);
hipError_t launch_attn_join(const AttnArgs &a, int dt, hipStream_t st);

}  // namespace aih
