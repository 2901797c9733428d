// attn_join.hip -- joins the parts that a row's keys were cut into (aih_attn):
// o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p with M the largest m_p.
//
// A workgroup of 4 wavefronts takes a row; its lanes hold 4 dims each, and the
// lanes that d leaves over, like the wavefronts, take other parts. Parts are
// summed in an order that depends on their number alone. Bound by memory: a
// part's 4 d + 8 bytes a row are read once.
#include <hip/hip_runtime.h>

#include "aih_device.h"
#include "attn.h"

namespace aih {
namespace {

template <int DT>
__global__ __launch_bounds__(256) void attn_join_kernel(AttnArgs a, uint32_t ldim) {
  __shared__ float red[3][256];
  const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  const uint64_t row = blockIdx.x;
  const uint64_t rows_all = (uint64_t)a.tokens * a.hq;
  const float *ml = a.ws + attn_ws_ml(a) + 2 * row;

  float mx = -3.402823466e38f;
  for (uint32_t p = lane; p < a.all_parts; p += 64) mx = fmaxf(mx, ml[2 * p * rows_all]);
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) mx = fmaxf(mx, __shfl_xor(mx, w));
  float sum = 0.0f;
  for (uint32_t p = lane; p < a.all_parts; p += 64)
    sum += ml[2 * p * rows_all + 1] * __builtin_amdgcn_exp2f(ml[2 * p * rows_all] - mx);
#pragma unroll
  for (int w = 1; w < 64; w <<= 1) sum += __shfl_xor(sum, w);

  const uint32_t dim = 4 * (lane & ((1u << ldim) - 1));
  const uint32_t subs = 4u * (64u >> ldim), sub = wave * (64u >> ldim) + (lane >> ldim);
  f32x4 x{};
  if (dim < a.d) {
    const float *o = a.ws + row * a.d + dim;
#pragma unroll 4
    for (uint32_t p = sub; p < a.all_parts; p += subs) {
      const float l = ml[2 * p * rows_all + 1], f = __builtin_amdgcn_exp2f(ml[2 * p * rows_all] - mx);
      const f32x4 y = *reinterpret_cast<const f32x4 *>(o + p * rows_all * a.d);
      if (l != 0.0f) x += y * f;  // a part without keys left nothing to read
    }
  }
#pragma unroll
  for (uint32_t w = 32; w >= 1; w >>= 1) {
    if (w < (1u << ldim)) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], w);
  }
  if (wave > 0)
    *reinterpret_cast<f32x4 *>(&red[wave - 1][4 * lane]) = x;
  __syncthreads();
  if (wave == 0 && lane < (1u << ldim) && dim < a.d) {
#pragma unroll
    for (int w = 0; w < 3; ++w) x += *reinterpret_cast<const f32x4 *>(&red[w][4 * lane]);
    x *= sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint64_t t = row / a.hq, h = row - t * a.hq;
    const uint64_t e = t * a.os + h * a.d + dim;
    if constexpr (DT == DT_F32) *reinterpret_cast<f32x4 *>((float *)a.o + e) = x;
    else *reinterpret_cast<u32x2 *>((uint16_t *)a.o + e) = pack4<DT>(x);
  }
}

}  // namespace

hipError_t launch_attn_join(const AttnArgs &a, int dt, hipStream_t st) {
  uint32_t ldim = 0;  // lanes of a row's dims, as a power of two
  while ((4u << ldim) < a.d) ++ldim;
  const dim3 grid(a.tokens * a.hq);
  if (dt == DT_F32) hipLaunchKernelGGL(attn_join_kernel<DT_F32>, grid, dim3(256), 0, st, a, ldim);
  else if (dt == DT_F16) hipLaunchKernelGGL(attn_join_kernel<DT_F16>, grid, dim3(256), 0, st, a, ldim);
  else hipLaunchKernelGGL(attn_join_kernel<DT_BF16>, grid, dim3(256), 0, st, a, ldim);
  return hipGetLastError();
}

uint32_t attn_bm(int kernel, int, uint32_t) { return kernel == AIH_ATTN_ROWS ? 128 : 32; }

hipError_t launch_attn(const AttnArgs &a, int kernel, int dt, hipStream_t st) {
  return dt == DT_F32 ? launch_attn_f32(a, kernel, st)
                      : dt == DT_F16 ? launch_attn_f16(a, kernel, st) : launch_attn_bf16(a, kernel, st);
}

}  // namespace aih
