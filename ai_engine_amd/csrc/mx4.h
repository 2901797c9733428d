// mx4.h -- kernel arguments, launchers and device helpers of the operators on
// microscaled 4-bit rows (include/aih_mx4.h). Everything here is checked by
// mx4_capi.hip.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/aih_mx4.h"
#include "aih_device.h"
#include "attn.h"

namespace aih {

struct Mx4RowsArgs {
  const void *src;     // quant: values; dequant: codes
  const uint8_t *src_scales;
  void *dst;           // quant: codes; dequant: values
  uint8_t *dst_scales;
  uint64_t stride;     // of the values' rows, elements
  uint32_t k;          // elements of a row
  uint32_t upr;        // units of 8 elements of a row: with quant of the padded row
  uint64_t units;      // of all rows, below 2^32 - 255
  uint32_t code_stride, scale_stride;  // bytes
  FastDiv by_upr;
};

hipError_t launch_mx4_quant(const Mx4RowsArgs &a, int dt, hipStream_t st);
hipError_t launch_mx4_dequant(const Mx4RowsArgs &a, int dt, hipStream_t st);

struct Mx4PwArgs {
  const uint8_t *xc, *xs, *wc, *ws;
  const void *bias, *res;  // or null
  void *y;
  uint32_t m, cout;
  uint32_t nst;       // stages of 128 elements
  uint32_t cb, sb;    // bytes of a row's codes and scales
  int32_t act;
  uint32_t mtiles, ntiles, nxcd;
};

hipError_t launch_mx4_pw(const Mx4PwArgs &a, int dt, hipStream_t st);

struct Kv4AppendArgs {
  const void *x, *wq, *wk;
  const float *cs, *sn;
  const int32_t *pos, *slots;
  void *q;
  uint8_t *kc, *ks, *vc, *vs;
  uint64_t xs, qs;          // row strides, elements
  uint32_t hq, hkv;
  uint32_t d, rot, pairs, norm;
  uint32_t positions, rows; // rows: pages * page
  uint32_t pshift;          // log2 of the rows of a page
  uint32_t items;           // tokens * (hq + 2 hkv)
  uint32_t nl, per;         // lanes of a head, heads of a wavefront
  float eps, inv_d;
  FastDiv by_ht, by_nl;
};

hipError_t launch_kv4_append(const Kv4AppendArgs &a, int dt, hipStream_t st);

// The rows, sequences and parts are those of AttnArgs (its key fields are not
// used), so the parts join as there.
struct Kv4AttnArgs {
  AttnArgs at;
  const uint8_t *kc, *ks, *vc, *vs;
  const int32_t *table;
  uint32_t width, pages, pshift;
  uint32_t rb;  // a tile's rows: 16 rb
};

hipError_t launch_kv4_attn(const Kv4AttnArgs &a, int dt, hipStream_t st);
hipError_t launch_kv4_attn_f32(const Kv4AttnArgs &a, hipStream_t st);
hipError_t launch_kv4_attn_f16(const Kv4AttnArgs &a, hipStream_t st);
hipError_t launch_kv4_attn_bf16(const Kv4AttnArgs &a, hipStream_t st);

// A scale byte as the conversion instructions take it: a float of which they read
// the exponent alone (0 is 2^-127, 255 makes NaN of whatever is converted).
__device__ __forceinline__ float mx4_scale(uint32_t byte) { return __uint_as_float(byte << 23); }

// The scale byte of a block whose largest magnitude has these bits.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t top) {
  return top >= 0x7f800000u ? 255u : (uint32_t)max((int)(top >> 23) - 2, 0);
}

// Eight values as codes, element 0 in the low bits. The conversions round to the
// nearest, ties to the even code, and stop at 6 (checked against the definition for every
// scale, at the borders and in between).
__device__ __forceinline__ uint32_t mx4_encode8(const float (&f)[8], uint32_t byte) {
  const float s = mx4_scale(byte);
  uint32_t c = 0;
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[0], f[1], s, 0);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[2], f[3], s, 1);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[4], f[5], s, 2);
  c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, f[6], f[7], s, 3);
  return byte == 255 ? 0u : c;
}

// The maximum over the four lanes of a quad, in all of them.
__device__ __forceinline__ uint32_t mx4_quad_max(uint32_t v) {
  v = max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0xb1, 0xf, 0xf, true));  // quad_perm 1 0 3 2
  return max(v, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)v, 0x4e, 0xf, 0xf, true));  // quad_perm 2 3 0 1
}

// Eight values of a storage type, as loaded and as fp32.
template <int DT>
struct Mx4Unit {
  static constexpr int W = DT == DT_F32 ? 2 : 1;
  u32x4 r[W];
  // the first `n` (0, 4 or 8) of them; WIDE: at a 16-byte boundary
  template <bool WIDE>
  __device__ __forceinline__ void load(const void *p, uint32_t n) {
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = u32x4{};
    if constexpr (DT == DT_F32) {
      if (n >= 4) r[0] = *reinterpret_cast<const u32x4 *>(p);
      if (n == 8) r[1] = *(reinterpret_cast<const u32x4 *>(p) + 1);
    } else if (WIDE && n == 8) {
      r[0] = *reinterpret_cast<const u32x4 *>(p);
    } else {
      if (n >= 4) {
        const u32x2 a = *reinterpret_cast<const u32x2 *>(p);
        r[0].x = a.x, r[0].y = a.y;
      }
      if (!WIDE && n == 8) {
        const u32x2 b = *(reinterpret_cast<const u32x2 *>(p) + 1);
        r[0].z = b.x, r[0].w = b.y;
      }
    }
  }
  template <bool WIDE>
  __device__ __forceinline__ void store(void *p, uint32_t n) const {
    if constexpr (DT == DT_F32) {
      if (n >= 4) *reinterpret_cast<u32x4 *>(p) = r[0];
      if (n == 8) *(reinterpret_cast<u32x4 *>(p) + 1) = r[1];
    } else if (WIDE && n == 8) {
      *reinterpret_cast<u32x4 *>(p) = r[0];
    } else {
      if (n >= 4) *reinterpret_cast<u32x2 *>(p) = u32x2{r[0].x, r[0].y};
      if (!WIDE && n == 8) *(reinterpret_cast<u32x2 *>(p) + 1) = u32x2{r[0].z, r[0].w};
    }
  }
  __device__ __forceinline__ void get(float (&f)[8]) const {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      if constexpr (DT == DT_F32) f[i] = __uint_as_float(r[i / 4][i % 4]);
      else if constexpr (DT == DT_F16) f[i] = f16_to_f32((r[0][i / 2] >> (16 * (i & 1))) & 0xffffu);
      else f[i] = bf16_to_f32((r[0][i / 2] >> (16 * (i & 1))) & 0xffffu);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[8]) {
#pragma unroll
    for (int i = 0; i < 4 * W; ++i) {
      if constexpr (DT == DT_F32) r[i / 4][i % 4] = __float_as_uint(f[i]);
      else r[0][i] = pack2<DT>(f[2 * i], f[2 * i + 1]);
    }
  }
};

}  // namespace aih
