// attn_simple.hip -- attention of one query row per wavefront: 64 keys at a
// time, a key per lane for the scores, a dim per lane for the values, with the
// running maximum and sum of the softmax (aih_attn).
#include <hip/hip_runtime.h>

#include "aih_device.h"
#include "attn.h"

namespace aih {
namespace {

template <int DT>
__device__ __forceinline__ float at1(const void *p, uint64_t i) {
  if constexpr (DT == DT_F32) return reinterpret_cast<const float *>(p)[i];
  else if constexpr (DT == DT_F16) return f16_to_f32(reinterpret_cast<const uint16_t *>(p)[i]);
  else return bf16_to_f32(reinterpret_cast<const uint16_t *>(p)[i]);
}

template <int DT>
__global__ __launch_bounds__(64) void attn_simple_kernel(AttnArgs a) {
  __shared__ float qs[256], ps[64];
  const uint32_t lane = threadIdx.x;
  const uint32_t t = blockIdx.x / a.hq, h = blockIdx.x % a.hq, hk = h / a.g;
  // the sequence whose query rows hold t
  uint32_t b = 0, q0 = 0, q1 = 0;
  for (; b < a.nseq; ++b) {
    q0 = min((uint32_t)max(a.q_start[b], 0), a.tokens);
    q1 = min((uint32_t)max(a.q_start[b + 1], 0), a.tokens);
    if (t >= q0 && t < q1) break;
  }
  if (b == a.nseq) return;
  const uint32_t k0 = min((uint32_t)max(a.k_start[b], 0), a.rows);
  const uint32_t len = min((uint32_t)max(a.k_len[b], 0), a.rows - k0);
  int64_t seen = len;
  if (a.causal) seen = min(seen, max((int64_t)(t - q0) + 1 + (int64_t)len - (int64_t)(q1 - q0), (int64_t)0));

  for (uint32_t i = lane; i < a.d; i += 64) qs[i] = at1<DT>(a.q, t * a.qs + h * a.d + i);
  float m = -3.402823466e38f, l = 0.0f, acc[4] = {};
  for (int part = 0; part < 2; ++part) {
    const void *k = part ? a.k : a.pk, *v = part ? a.v : a.pv;
    const uint64_t kst = part ? a.ks : a.pks, vst = part ? a.vs : a.pvs, r0 = part ? k0 : 0;
    const uint32_t n = part ? (uint32_t)seen : a.prefix;
    for (uint32_t j0 = 0; j0 < n; j0 += 64) {
      const uint32_t j = j0 + lane;
      float s = -__builtin_huge_valf();
      __syncthreads();
      if (j < n) {
        s = 0.0f;
        for (uint32_t i = 0; i < a.d; ++i) s += qs[i] * at1<DT>(k, (r0 + j) * kst + hk * a.d + i);
        s *= a.scale_log2;
      }
      float mx = s;
      for (int w = 1; w < 64; w <<= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
      const float mn = fmaxf(m, mx), al = exp2f(m - mn), p = exp2f(s - mn);
      m = mn;
      float sum = p;
      for (int w = 1; w < 64; w <<= 1) sum += __shfl_xor(sum, w);
      l = l * al + sum;
      ps[lane] = p;
      __syncthreads();
      const uint32_t nk = min(64u, n - j0);
      for (int c = 0; c < 4; ++c) {
        const uint32_t i = lane + 64 * c;
        if (i >= a.d) break;
        acc[c] *= al;
        for (uint32_t e = 0; e < nk; ++e) acc[c] += ps[e] * at1<DT>(v, (r0 + j0 + e) * vst + hk * a.d + i);
      }
    }
  }
  for (int c = 0; c < 4; ++c) {
    const uint32_t i = lane + 64 * c;
    if (i >= a.d) break;
    const float y = l == 0.0f ? 0.0f : acc[c] / l;
    const uint64_t o = t * a.os + h * a.d + i;
    if constexpr (DT == DT_F32) reinterpret_cast<float *>(a.o)[o] = y;
    else if constexpr (DT == DT_F16) reinterpret_cast<uint16_t *>(a.o)[o] = (uint16_t)f32_to_f16(y);
    else reinterpret_cast<uint16_t *>(a.o)[o] = (uint16_t)f32_to_bf16(y);
  }
}

}  // namespace

hipError_t launch_attn_simple(const AttnArgs &a, int dt, hipStream_t st) {
  const dim3 grid(a.tokens * a.hq);
  if (dt == DT_F32) hipLaunchKernelGGL(attn_simple_kernel<DT_F32>, grid, dim3(64), 0, st, a);
  else if (dt == DT_F16) hipLaunchKernelGGL(attn_simple_kernel<DT_F16>, grid, dim3(64), 0, st, a);
  else hipLaunchKernelGGL(attn_simple_kernel<DT_BF16>, grid, dim3(64), 0, st, a);
  return hipGetLastError();
}

}  // namespace aih
