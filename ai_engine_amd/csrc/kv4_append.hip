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
__device__ __forceinline__ void turn(float (&f)[8], const float (&other)[8], const f32x4 (&c)[2], const f32x4 (&s)[2], float sign) {
#pragma clang fp contract(off)
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const float x = f[e] * c[e / 4][e % 4], y = other[e] * s[e / 4][e % 4];
    f[e] = x + sign * y;
  }
}
// adjacent pairs: (a, b) -> (a c - b s, a s + b c)
__device__ __forceinline__ void turn_pairs(float (&f)[8], f32x4 c, f32x4 s) {
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
// position is there, none of them behind a branch that a wait would follow: the
// rotation is computed by all lanes and taken by those it is for. 46080 tokens of 8 + 2 + 2
// f16 heads of 64 take 32 us with adjacent pairs (3.9 TB/s), 36 with halves, 26.5 without
// rotation, where a large copy would take 24; 16384 of 32 + 8 + 8 bf16 heads of 128 70 and 78.
// With the loads behind branches it was 38, 41 and, with halves, 95. Head norms, whose sums
// cross the lanes of a head: 34 and 41, 81 and 99. NORM and MODE apart, so that an
// append carries what it needs.
enum : int { MODE_NONE = 0, MODE_HALVES = 1, MODE_PAIRS = 2 };
template <int DT, bool NORM, int MODE>
__global__ __launch_bounds__(kThreads) void kv4_append_kernel(Kv4AppendArgs a) {
  constexpr int EB = Storage<DT>::bytes;
  const uint32_t lane = threadIdx.x & 63, nl = a.nl, per = a.per, g = fdiv(lane, a.by_nl), j = lane - g * nl;
  const uint32_t at = (blockIdx.x * (kThreads / 64) + (threadIdx.x >> 6)) * per + g;  // below items + 256
  // lanes without an item keep to the last one, and store nothing: the lanes of a
  // wavefront stay together for the exchanges
  const bool live = g < per && at < a.items;
  const uint32_t item = live ? at : a.items - 1;
  const uint32_t t = fdiv(item, a.by_ht), h = item - t * (a.hq + 2 * a.hkv);
  const bool is_q = h < a.hq, is_v = h >= a.hq + a.hkv;
  const uint32_t jj = g < per ? j : 0;  // the lanes left over read what is there
  const uint32_t half = a.rot / 16;     // lanes of a rotated half
  const bool turns = MODE != MODE_NONE && !is_v && jj * 8 < a.rot;
  const uint32_t pj = MODE == MODE_HALVES && turns ? (jj < half ? jj + half : jj - half) : jj;

  const int32_t given = (a.pos ? a.pos : a.slots)[t], pos = a.pos ? given : (int32_t)t;
  const uint32_t slot = (uint32_t)a.slots[t];
  const char *src = (const char *)a.x + ((uint64_t)t * a.xs + (uint64_t)h * a.d) * EB;
  Mx4Unit<DT> v, p;  // the elements, and a rotation's partners where they are another lane's
  v.template load<true>(src + jj * 8 * EB, 8);
  if constexpr (MODE == MODE_HALVES) p.template load<true>(src + pj * 8 * EB, 8);
  f32x4 c[2], s[2];
  if constexpr (MODE != MODE_NONE) {
    const uint64_t row = (uint64_t)min((uint32_t)max(pos, 0), a.positions - 1) * (a.rot / 2) +
                         (!turns ? 0 : MODE == MODE_PAIRS ? jj * 4 : min(jj, pj) * 8);
    const f32x4 *cr = reinterpret_cast<const f32x4 *>(a.cs + row), *sr = reinterpret_cast<const f32x4 *>(a.sn + row);
    c[0] = cr[0], s[0] = sr[0];
    if constexpr (MODE == MODE_HALVES) c[1] = cr[1], s[1] = sr[1];
  }

  float f[8], o[8];
  v.get(f);
  if constexpr (MODE == MODE_HALVES) p.get(o);
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
      for (int e = 0; e < 8; ++e) {
        f[e] *= up;
        if constexpr (MODE == MODE_HALVES) o[e] *= up;
      }
      mean = squares() * a.inv_d + a.eps * up * up;
    }
    if (!is_v) {
      const float r = __builtin_amdgcn_rsqf(mean);
      const char *w = (const char *)(is_q ? a.wq : a.wk);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        f[e] *= r;
        if constexpr (MODE == MODE_HALVES) o[e] *= r;
      }
      if (w) {
        Mx4Unit<DT> wv;
        float wf[8];
        wv.template load<true>(w + jj * 8 * EB, 8);
        wv.get(wf);
#pragma unroll
        for (int e = 0; e < 8; ++e) f[e] *= wf[e];
        if constexpr (MODE == MODE_HALVES) {
          wv.template load<true>(w + pj * 8 * EB, 8);
          wv.get(wf);
#pragma unroll
          for (int e = 0; e < 8; ++e) o[e] *= wf[e];
        }
      }
    }
  }
  if constexpr (MODE != MODE_NONE) {  // for all lanes: the loads would move behind a branch
    float y[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e] = f[e];
    if constexpr (MODE == MODE_PAIRS) turn_pairs(y, c[0], s[0]);
    else turn(y, o, c, s, jj < half ? -1.0f : 1.0f);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[e] = turns ? y[e] : f[e];
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
  const uint32_t per = kThreads / 64 * a.per;
  const dim3 grid((a.items + per - 1) / per);
  const int mode = a.rot == 0 ? MODE_NONE : a.pairs ? MODE_PAIRS : MODE_HALVES;
#define AIH_APPEND_CASE(MODE)                                                                                          \
  if (mode == MODE) {                                                                                                  \
    if (a.norm) hipLaunchKernelGGL((kv4_append_kernel<DT, true, MODE>), grid, dim3(kThreads), 0, st, a);               \
    else hipLaunchKernelGGL((kv4_append_kernel<DT, false, MODE>), grid, dim3(kThreads), 0, st, a);                     \
  }
  AIH_APPEND_CASE(MODE_NONE)
  AIH_APPEND_CASE(MODE_HALVES)
  AIH_APPEND_CASE(MODE_PAIRS)
#undef AIH_APPEND_CASE
  return hipGetLastError();
}

}  // namespace

hipError_t launch_kv4_append(const Kv4AppendArgs &a, int dt, hipStream_t st) {
  return dt == DT_F32 ? append_dt<DT_F32>(a, st) : dt == DT_F16 ? append_dt<DT_F16>(a, st) : append_dt<DT_BF16>(a, st);
}

}  // namespace aih
