// attn_join.hip -- joins the parts that a row's keys were cut into (aih_attn):
// o = sum_p 2^(m_p - M) O_p / sum_p 2^(m_p - M) l_p with M the largest m_p.
//
// NW wavefronts take a row; a wavefront's lanes hold 4 dims each, and the
// lanes that d leaves over, like the wavefronts, take other parts. Parts are
// summed in an order that depends on their number alone. The loads of the
// parts do not wait for the maximum, so a row costs little more than one trip
// to memory: with few rows that is all of the time, with many the 4 d + 8 bytes
// of each row and part. 2048 rows of 5 or 8 parts of 128 take 4.2 to 4.8 us, 32 rows
// of 128 parts 5.4, 48 rows of 2 parts of 64 3.6.
#include <hip/hip_runtime.h>

#include "aih_device.h"
#include "attn.h"

namespace aih {
namespace {

constexpr int kWaves = 4;  // of a workgroup with NW = 1: four rows

template <int DT, int NW>
__global__ __launch_bounds__(64 * (NW == 1 ? kWaves : NW)) void attn_join_kernel(AttnArgs a, uint32_t ldim) {
  __shared__ float red[NW][256];
  const uint32_t lane = threadIdx.x & 63, w = threadIdx.x >> 6, wave = NW == 1 ? 0 : w;
  const uint64_t rows_all = (uint64_t)a.tokens * a.hq;
  const uint64_t row = NW == 1 ? (uint64_t)blockIdx.x * kWaves + w : blockIdx.x;
  if (row >= rows_all) return;
  const f32x2 *ml = reinterpret_cast<const f32x2 *>(a.ws + attn_ws_ml(a)) + row;
  const int q0 = a.q_start[0], q1 = a.q_start[a.nseq];

  // (maximum, sum) of the part that this lane's next vector belongs to
  const uint32_t subs = NW * (64u >> ldim), sub = wave * (64u >> ldim) + (lane >> ldim);
  const uint32_t dim = 4 * (lane & ((1u << ldim) - 1));
  const float *o = a.ws + row * a.d + dim;
  constexpr int PRE = 4;
  f32x4 y[PRE];
  f32x2 z[PRE];
#pragma unroll
  for (int i = 0; i < PRE; ++i) {
    const uint32_t p = sub + i * subs;
    y[i] = f32x4{};
    z[i] = f32x2{-3.402823466e38f, 0.0f};
    if (p < a.all_parts) {
      z[i] = ml[p * rows_all];
      if (dim < a.d) y[i] = *reinterpret_cast<const f32x4 *>(o + p * rows_all * a.d);
    }
  }
  float mx = -3.402823466e38f, sum = 0.0f;
  bool done = false;
  for (uint32_t p = lane; p < a.all_parts; p += 64) {
    const f32x2 t = ml[p * rows_all];
    done |= p == 0 && t.y == -1.0f;
    const float mn = fmaxf(mx, t.x);
    sum = sum * __builtin_amdgcn_exp2f(mx - mn) + t.y * __builtin_amdgcn_exp2f(t.x - mn);
    mx = mn;
  }
  const uint64_t t = row / a.hq, h = row - t * a.hq;
  done |= (int64_t)t < q0 || (int64_t)t >= q1;  // of no sequence: no part holds anything
  if (__any(done)) return;  // the whole row's wavefronts find the same
  float all = mx;
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) all = fmaxf(all, __shfl_xor(all, s));
  sum *= __builtin_amdgcn_exp2f(mx - all);
#pragma unroll
  for (int s = 1; s < 64; s <<= 1) sum += __shfl_xor(sum, s);

  f32x4 x{};
#pragma unroll
  for (int i = 0; i < PRE; ++i)
    if (z[i].y != 0.0f) x += y[i] * __builtin_amdgcn_exp2f(z[i].x - all);  // a part without keys left nothing to read
  for (uint32_t p = sub + PRE * subs; p < a.all_parts; p += subs) {
    const f32x2 t = ml[p * rows_all];
    if (t.y != 0.0f && dim < a.d)
      x += *reinterpret_cast<const f32x4 *>(o + p * rows_all * a.d) * __builtin_amdgcn_exp2f(t.x - all);
  }
#pragma unroll
  for (uint32_t s = 32; s >= 1; s >>= 1) {
    if (s < (1u << ldim)) break;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] += __shfl_xor(x[e], s);
  }
  if constexpr (NW > 1) {
    *reinterpret_cast<f32x4 *>(&red[wave][4 * lane]) = x;
    __syncthreads();
    if (wave > 0) return;
#pragma unroll
    for (int i = 1; i < NW; ++i) x += *reinterpret_cast<const f32x4 *>(&red[i][4 * lane]);
  }
  if (lane < (1u << ldim) && dim < a.d) {
    x *= sum == 0.0f ? 0.0f : 1.0f / sum;
    const uint64_t e = t * a.os + h * a.d + dim;
    if constexpr (DT == DT_F32) *reinterpret_cast<f32x4 *>((float *)a.o + e) = x;
    else *reinterpret_cast<u32x2 *>((uint16_t *)a.o + e) = pack4<DT>(x);
  }
}

template <int DT>
hipError_t join_dt(const AttnArgs &a, uint32_t ldim, hipStream_t st) {
  const uint32_t rows = a.tokens * a.hq;  // below 2^31
  // a wavefront holds 4 parts of each of its lane groups in flight; more parts
  // than that take more wavefronts
  if (a.all_parts <= 4u * (64u >> ldim))
    hipLaunchKernelGGL((attn_join_kernel<DT, 1>), dim3((rows + kWaves - 1) / kWaves), dim3(64 * kWaves), 0, st, a, ldim);
  else if (a.all_parts <= 16u * (64u >> ldim))
    hipLaunchKernelGGL((attn_join_kernel<DT, 4>), dim3(rows), dim3(256), 0, st, a, ldim);
  else
    hipLaunchKernelGGL((attn_join_kernel<DT, 16>), dim3(rows), dim3(1024), 0, st, a, ldim);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_attn_join(const AttnArgs &a, int dt, hipStream_t st) {
  uint32_t ldim = 0;  // lanes of a row's dims, as a power of two
  while ((4u << ldim) < a.d) ++ldim;
  return dt == DT_F32 ? join_dt<DT_F32>(a, ldim, st)
                      : dt == DT_F16 ? join_dt<DT_F16>(a, ldim, st) : join_dt<DT_BF16>(a, ldim, st);
}

uint32_t attn_bm(int kernel) { return kernel == AIH_ATTN_ROWS ? 128 : 32; }

hipError_t launch_attn(const AttnArgs &a, int kernel, int dt, hipStream_t st) {
  return dt == DT_F32 ? launch_attn_f32(a, kernel, st)
                      : dt == DT_F16 ? launch_attn_f16(a, kernel, st) : launch_attn_bf16(a, kernel, st);
}

}  // namespace aih
