// attn.h -- kernel arguments and launchers of the attention operators
// (include/aih_attn.h). Everything here is checked by attn_capi.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/aih_attn.h"

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

struct AttnArgs {
  const void *q, *k, *v, *pk, *pv;
  void *o;
  float *ws;
  const int32_t *q_start, *k_start, *k_len;
  uint64_t qs, ks, vs, os, pks, pvs;  // row strides, elements
  uint32_t nseq, tokens, rows, prefix;
  uint32_t hq, hkv, g, d;
  uint32_t causal;
  float scale_log2;  // scale * log2(e)
};

hipError_t launch_attn_simple(const AttnArgs &a, int dt, hipStream_t st);

}  // namespace aih
