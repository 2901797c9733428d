// kv4_append.hip -- the way of new tokens into a 4-bit cache (aih_kv4_append):
// head norms, position rotation, quantisation and the pages in one pass over
// the projection's rows.
//
// A lane takes 8 elements of a head, the d / 8 lanes of a head are neighbours, and
// so are the four lanes of a block (see mx4_quant.hip). A rotation's partner is
// loaded as well where it is another lane's (halves): from the cache, since the
// head's row has just been read. Products and sums are rounded one by one, so that
// a key's codes follow from its row and the tables by plain fp32 arithmetic.
#include <hip/hip_runtime.h>

#include "aih_device.h"
#include "mx4.h"

namespace aih {
namespace {

constexpr int kThreads = 256;

// a c -+ b s of eight elements
__device__ __forceinline__ void turn(float (&f)[8], const float (&other)[8], const float *c, const float *s, float sign) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = f[e] * c[e], y = other[e] * s[e];
    f[e] = x + sign * y;
  }
}
// adjacent pairs: (a, b) -> (a c - b s, a s + b c)
__device__ __forceinline__ void turn_pairs(float (&f)[8], const float *c, const float *s) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const float a = f[2 * e], b = f[2 * e + 1];
    const float ac = a * c[e], bs = b * s[e], as = a * s[e], bc = b * c[e];
    f[2 * e] = ac - bs;
    f[2 * e + 1] = as + bc;
  }
}

// All of a lane's loads go out before anything is computed, the tables' as soon as the
// position is there. 46080 tokens of 8 + 2 + 2 f16 heads of 64, adjacent pairs, take 32 us
// (3.9 TB/s), without rotation 27, where a large copy would take 24; with the tables' loads
// behind the elements' it took 38, with two to four items a lane 38 to 44.
// NORM apart, so that plain appends do not carry its exchange.
template <int DT, bool NORM>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(Kv4AppendArgs a) {
  constexpr int EB = Storage<DT>::bytes;
  const uint32_t lane = threadIdx.x & 63, nl = a.d / 8, per = 64 / nl, g = lane / nl, j = lane - g * nl;
  const uint64_t at = ((uint64_t)blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * per + g;
  // lanes without an item keep to the last one, and store nothing: the lanes of a
  // wavefront stay together for the exchanges
  const bool live = g < per && at < a.items;
  const uint32_t item = live ? (uint32_t)at : a.items - 1;
  const uint32_t t = fdiv(item, a.by_ht), h = item - t * (a.hq + 2 * a.hkv);
  const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
  const uint32_t jj = g < per ? j : 0;  // the lanes left over read what is there
  const uint32_t half = a.rot / 16;     // lanes of a rotated half
  const bool turns = !is_v && jj * 8 < a.rot, halves = turns && !a.pairs;
  const uint32_t pj = halves ? (jj < half ? jj + half : jj - half) : jj;

  const int32_t pos = a.pos && turns ? a.pos[t] : (int32_t)t;
  const uint32_t slot = is_q ? 0u : (uint32_t)a.slots[t];
  const char *src = (const char *)a.x + ((uint64_t)t * a.xs + (uint64_t)h * a.d) * EB;
  Mx4Unit<DT> v, p;  // the elements, and a rotation's partners where they are another lane's
  v.template load<true>(src + jj * 8 * EB, 8);
  p.template load<true>(src + pj * 8 * EB, halves ? 8 : 0);
  float c[8], s[8];
  if (turns) {
    const uint64_t row = (uint64_t)min((uint32_t)max(pos, 0), a.positions - 1) * (a.rot / 2) + (a.pairs ? jj * 4 : min(jj, pj) * 8);
    auto take = [&](float(&to)[8], const float *from) {
      const f32x4 lo = *reinterpret_cast<const f32x4 *>(from);
#pragma unroll
      for (int e = 0; e < 4; ++e) to[e] = lo[e];
      if (!a.pairs) {
        const f32x4 hi = *reinterpret_cast<const f32x4 *>(from + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) to[4 + e] = hi[e];
      }
    };
    take(c, a.cs + row), take(s, a.sn + row);
  }

  float f[8], o[8];
  v.get(f), p.get(o);
  if constexpr (NORM) {
    auto squares = [&]() {  // of the whole head: to its first lane, and from there to all
      float ss = 0.0f;
#pragma unroll
      for (int e = 0; e < 8; ++e) ss += f[e] * f[e];
      for (uint32_t m = 1; m < nl; m <<= 1) {
        const float up = __shfl(ss, lane + m);
        if (j % (2 * m) == 0 && j + m < nl) ss += up;
      }
      return __shfl(ss, lane - j);
    };
    float mean = squares() * a.inv_d + a.eps;
    // squares leave fp32's range long before the values do: such heads are taken
    // times a power of two, which rounds nothing
    const bool out = !is_v && !(mean >= 0x1p-100f && mean <= 0x1p100f);
    if (__any(out)) {
      const float up = !out ? 1.0f : mean < 0x1p-100f ? 0x1p100f : 0x1p-70f;
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= up, o[e] *= up;
      mean = squares() * a.inv_d + a.eps * up * up;
    }
    if (!is_v) {
      const float r = __builtin_amdgcn_rsqf(mean);
      const char *w = (const char *)(is_q ? a.wq : a.wk);
#pragma unroll
      for (int e = 0; e < 8; ++e) f[e] *= r, o[e] *= r;
      if (w) {
        Mx4Unit<DT> wv;
        float wf[8];
        wv.template load<true>(w + jj * 8 * EB, 8);
        wv.get(wf);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= wf[e];
        if (halves) {
          wv.template load<true>(w + pj * 8 * EB, 8);
          wv.get(wf);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] *= wf[e];
        }
      }
    }
  }
  if (turns) {
    if (a.pairs) turn_pairs(f, c, s);
    else turn(f, o, c, s, jj < half ? -1.0f : 1.0f);
  }
  if (is_q && live) {
    v.set(f);
    v.template store<true>((char *)a.q + ((uint64_t)t * a.qs + (uint64_t)h * a.d + jj * 8) * EB, 8);
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
  const uint32_t byte = mx4_scale_byte(mx4_quad_max(top));
  if (!is_q && live && slot < a.rows) {  // negative slots are not, either
    const uint32_t hk = h - a.hq - (is_v ? a.hkv : 0);
    const uint64_t row = (((uint64_t)(slot >> a.pshift) * a.hkv + hk) << a.pshift) | (slot & ((1u << a.pshift) - 1));
    *reinterpret_cast<uint32_t *>((is_v ? a.vc : a.kc) + row * (a.d / 2) + j * 4) = mx4_encode8(f, byte);
    if (j % 4 == 0) (is_v ? a.vs : a.ks)[row * (a.d / 32) + j / 4] = (uint8_t)byte;
  }
}

template <int DT>
hipError_t append_dt(const Kv4AppendArgs &a, hipStream_t st) {
  const uint32_t per = kThreads / 64 * (64 / (a.d / 8));
  const dim3 grid((a.items + per - 1) / per);
  if (a.norm) hipLaunchKernelGGL((kv4_append_kernel<DT, true>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((kv4_append_kernel<DT, false>), grid, dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv4_append(const Kv4AppendArgs &a, int dt, hipStream_t st) {
  return dt == DT_F32 ? append_dt<DT_F32>(a, st) : dt == DT_F16 ? append_dt<DT_F16>(a, st) : append_dt<DT_BF16>(a, st);
}

}  // namespace aih
