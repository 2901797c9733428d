// qk_norm_rope.hip -- norms of query and key heads with the position rotation,
// in one pass over the projection's rows (aih_qk_norm_rope).
//
// y = x * rsqrt(mean(x^2) + eps) * w per head, then a' = a c - b s, b' = a s + b c
// for the rotated pairs. Everything is fp32 between the load and the store,
// which rounds once.
//
// An item is one head of one token; P lanes (a power of two, or the exact number
// where that would leave more than a quarter of them idle: 30000 tokens of 24 f16
// heads of 80 61 -> 52 us, of 72 85 -> 60) take it, each two vectors of VW elements. With halves the two are partners (unit j and unit
// j + rot/2), so a rotation needs no exchange between lanes; the only exchange
// is the sum of squares over the P lanes. VW is 16 bytes unless the rotated
// half is no whole number of such units, then 8 or 4 bytes. Items follow the
// memory order of the rows, so a wavefront reads one contiguous run.
//
// Bound by memory: each element is read and written once, the table rows come
// from the caches (all heads of a token use the same one). 46080 tokens of 8 + 2 + 2
// f16 heads of 64 take 33.1 us, 4.6 TB/s, where a large copy reaches 4.76. Few
// tokens (8: 3.3 us on the device, 5.7 from call to call) are bound by the
// host's call.
#include <hip/hip_runtime.h>

#include "aih_device.h"
#include "attn.h"

namespace aih {
namespace {

constexpr int kThreads = 256;
constexpr uint32_t kAnyLanes = 31;  // for pshift: the lanes of an item are no power of two

// VW elements as stored, and as fp32.
template <int DT, int VW>
struct Vec {
  static constexpr int BYTES = VW * Storage<DT>::bytes;
  static constexpr int W = BYTES / 4;
  uint32_t r[W];
  __device__ __forceinline__ void load(const void *p) {
    if constexpr (W == 4) {
      const u32x4 t = *reinterpret_cast<const u32x4 *>(p);
      r[0] = t.x, r[1] = t.y, r[2] = t.z, r[3] = t.w;
    } else if constexpr (W == 2) {
      const u32x2 t = *reinterpret_cast<const u32x2 *>(p);
      r[0] = t.x, r[1] = t.y;
    } else {
      r[0] = *reinterpret_cast<const uint32_t *>(p);
    }
  }
  __device__ __forceinline__ void store(void *p) const {
    if constexpr (W == 4) *reinterpret_cast<u32x4 *>(p) = u32x4{r[0], r[1], r[2], r[3]};
    else if constexpr (W == 2) *reinterpret_cast<u32x2 *>(p) = u32x2{r[0], r[1]};
    else *reinterpret_cast<uint32_t *>(p) = r[0];
  }
  __device__ __forceinline__ void get(float (&f)[VW]) const {
#pragma unroll
    for (int i = 0; i < VW; ++i) {
      if constexpr (DT == DT_F32) f[i] = __uint_as_float(r[i]);
      else if constexpr (DT == DT_F16) f[i] = f16_to_f32((r[i / 2] >> (16 * (i & 1))) & 0xffffu);
      else f[i] = bf16_to_f32((r[i / 2] >> (16 * (i & 1))) & 0xffffu);
    }
  }
  __device__ __forceinline__ void set(const float (&f)[VW]) {
#pragma unroll
    for (int i = 0; i < W; ++i) {
      if constexpr (DT == DT_F32) r[i] = __float_as_uint(f[i]);
      else r[i] = pack2<DT>(f[2 * i], f[2 * i + 1]);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < W; ++i) r[i] = 0;
  }
};

template <int DT, int VW>
__global__ __launch_bounds__(kThreads) void qk_norm_rope_kernel(QkRopeArgs a, uint32_t pshift) {
  constexpr int EB = Storage<DT>::bytes;
  const uint32_t lane = threadIdx.x & 63;
  uint32_t j = lane & ((1u << pshift) - 1);
  uint64_t item = ((uint64_t)blockIdx.x * kThreads + threadIdx.x) >> pshift;
  if (pshift == kAnyLanes) {  // groups of nl lanes; the last ones of a wavefront have none
    const uint32_t per = 64 / a.nl, g = lane / a.nl;
    j = lane - g * a.nl;
    item = g < per ? ((uint64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * per + g : a.items;
  }
  // a group past the end keeps to the last item, and stores nothing: the lanes
  // of a wavefront stay together for the exchange
  const bool live = item < a.items;
  const uint64_t it = live ? item : a.items - 1;
  const uint64_t t = it / a.ht;
  const uint32_t h = (uint32_t)(it - t * a.ht);
  const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;

  // the lane's two units; rotated ones are partners with halves
  const bool halves = a.rot != 0 && !a.pairs;
  uint32_t u0 = j, u1 = j + a.nl;
  if (halves) {
    u1 = j + a.ru;
    if (j >= a.ru) u0 = 2 * a.ru + 2 * (j - a.ru), u1 = u0 + 1;
  }
  const bool on0 = j < a.nl && u0 < a.units, on1 = j < a.nl && u1 < a.units;

  const char *src = (const char *)a.x + (t * a.xs + (uint64_t)h * a.d) * EB;
  Vec<DT, VW> v0, v1;
  v0.zero(), v1.zero();
  if (on0) v0.load(src + u0 * VW * EB);
  if (on1) v1.load(src + u1 * VW * EB);

  char *dst;
  bool store = live;
  if (is_q) {
    dst = (char *)a.q + (t * a.qs + (uint64_t)h * a.d) * EB;
  } else {
    uint64_t row = t;
    if (a.slots) {
      const int32_t s = a.slots[t];
      store &= s >= 0;
      row = (uint32_t)s;
    }
    store &= row < a.rows;
    dst = is_v ? (char *)a.v + (row * a.vs + (uint64_t)(h - a.hq - a.hkv) * a.d) * EB
               : (char *)a.k + (row * a.ks + (uint64_t)(h - a.hq) * a.d) * EB;
  }

  float f0[VW], f1[VW];
  v0.get(f0), v1.get(f1);
  auto squares = [&]() {  // of the whole head
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < VW; ++i) ss += f0[i] * f0[i] + f1[i] * f1[i];
    if (pshift == kAnyLanes) {  // to the group's first lane, and from there to all
      for (uint32_t m = 1; m < a.nl; m <<= 1) {
        const float up = __shfl(ss, lane + m);
        if (j % (2 * m) == 0 && j + m < a.nl) ss += up;
      }
      return __shfl(ss, lane - j);
    }
    for (uint32_t m = 1; m < (1u << pshift); m <<= 1) ss += __shfl_xor(ss, m);
    return ss;
  };
  float mean = squares() * a.inv_d + a.eps;
  // Squares leave fp32's range, and the root's that of normal numbers, long before
  // the values do: such heads (below 1e-15 or above 1e15 or so) are taken times a
  // power of two, which rounds nothing.
  const bool out = !is_v && !(mean >= 0x1p-100f && mean <= 0x1p100f);
  if (__any(out)) {
    const float up = !out ? 1.0f : mean < 0x1p-100f ? 0x1p100f : 0x1p-70f;
#pragma unroll
    for (int i = 0; i < VW; ++i) f0[i] *= up, f1[i] *= up;
    mean = squares() * a.inv_d + a.eps * up * up;
  }

  if (!is_v) {  // a value head keeps the bits it was loaded with
    const float r = __builtin_amdgcn_rsqf(mean);
    const char *w = (const char *)(is_q ? a.wq : a.wk);
#pragma unroll
    for (int i = 0; i < VW; ++i) f0[i] *= r, f1[i] *= r;
    if (w) {
      Vec<DT, VW> w0, w1;
      w0.zero(), w1.zero();
      if (on0) w0.load(w + u0 * VW * EB);
      if (on1) w1.load(w + u1 * VW * EB);
      float g0[VW], g1[VW];
      w0.get(g0), w1.get(g1);
#pragma unroll
      for (int i = 0; i < VW; ++i) f0[i] *= g0[i], f1[i] *= g1[i];
    }
    if (a.rot) {
      uint64_t p = t;
      if (a.pos) {
        const int32_t pi = a.pos[t];
        p = pi < 0 ? 0 : (uint32_t)pi;
      }
      if (p >= a.positions) p = a.positions - 1;
      const uint64_t row = p * (a.rot / 2);
      if (halves) {
        if (j < a.ru) {
          const float *c = a.cs + row + j * VW, *s = a.sn + row + j * VW;
#pragma unroll
          for (int i = 0; i < VW; i += 2) {  // rows are whole 8-byte units
            const f32x2 ci = *reinterpret_cast<const f32x2 *>(c + i), si = *reinterpret_cast<const f32x2 *>(s + i);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float x = f0[i + e], y = f1[i + e];
              f0[i + e] = x * ci[e] - y * si[e];
              f1[i + e] = x * si[e] + y * ci[e];
            }
          }
        }
      } else {
        auto turn = [&](float(&f)[VW], uint32_t e0) {
#pragma unroll
          for (int i = 0; i < VW; i += 4) {  // rot is a multiple of 4
            if (e0 + i < a.rot) {
              const f32x2 ci = *reinterpret_cast<const f32x2 *>(a.cs + row + (e0 + i) / 2);
              const f32x2 si = *reinterpret_cast<const f32x2 *>(a.sn + row + (e0 + i) / 2);
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const float x = f[i + 2 * e], y = f[i + 2 * e + 1];
                f[i + 2 * e] = x * ci[e] - y * si[e];
                f[i + 2 * e + 1] = x * si[e] + y * ci[e];
              }
            }
          }
        };
        if constexpr (VW >= 4) {
          if (on0) turn(f0, u0 * VW);
          if (on1) turn(f1, u1 * VW);
        }
      }
    }
    v0.set(f0), v1.set(f1);
  }
  if (store && on0) v0.store(dst + u0 * VW * EB);
  if (store && on1) v1.store(dst + u1 * VW * EB);
}

template <int DT, int VW>
hipError_t launch_vw(const QkRopeArgs &a, hipStream_t st) {
  // Lanes of an item: a power of two, or, where that left more than a quarter of
  // them idle, exactly those it needs.
  uint32_t ps = 0;
  while ((1u << ps) < a.nl) ++ps;
  uint64_t blocks = ((a.items << ps) + kThreads - 1) / kThreads;
  if (4 * a.nl < 3u << ps) {
    const uint32_t per = kThreads / 64 * (64 / a.nl);
    ps = kAnyLanes;
    blocks = (a.items + per - 1) / per;
  }
  if ((ps > 6 && ps != kAnyLanes) || blocks > 0x7fffffffu) return hipErrorInvalidValue;
  hipLaunchKernelGGL((qk_norm_rope_kernel<DT, VW>), dim3((uint32_t)blocks), dim3(kThreads), 0, st, a, ps);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_qk_norm_rope(const QkRopeArgs &a0, int dt, hipStream_t st) {
  QkRopeArgs a = a0;
  if (a.items == 0) return hipSuccess;
  // the widest vector that the rotated half is a whole number of
  uint32_t vw = dt == DT_F32 ? 4 : 8;
  if (a.rot && !a.pairs)
    while ((a.rot / 2) % vw) vw /= 2;
  a.units = a.d / vw;
  a.ru = a.rot && !a.pairs ? a.rot / 2 / vw : 0;
  a.nl = (a.units + 1) / 2;
#define AIH_QR_CASE(DT, VW) \
  if (dt == DT && vw == VW) return launch_vw<DT, VW>(a, st);
  AIH_QR_CASE(DT_F32, 4)
  AIH_QR_CASE(DT_F32, 2)
  AIH_QR_CASE(DT_F16, 8)
  AIH_QR_CASE(DT_F16, 4)
  AIH_QR_CASE(DT_F16, 2)
  AIH_QR_CASE(DT_BF16, 8)
  AIH_QR_CASE(DT_BF16, 4)
  AIH_QR_CASE(DT_BF16, 2)
#undef AIH_QR_CASE
  return hipErrorInvalidValue;
}

}  // namespace aih
