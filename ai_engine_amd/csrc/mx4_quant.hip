// mx4_quant.hip -- rows to microscaled 4-bit floating point and back
// (aih_mx4_quant, aih_mx4_dequant).
//
// A lane takes a unit of 8 elements, four neighbouring lanes a block: the block's
// largest magnitude is one exchange within the four (on the bits, whose order is
// the magnitudes'), its exponent less 2 the scale byte, and the conversion
// instructions do the rest. All of it is exact: the scales are powers of two.
//
// Bound by memory: 46080 rows of 960 f16 elements to 4 bits 20.6 us (5.4 TB/s of what
// has to be read and written, where a large copy reaches 5.1) and back 18.2. A few rows are
// bound by the host's call (9 x 4096: 2.5 us on the device, 4.6 from call to call).
#include <hip/hip_runtime.h>

#include "aih_device.h"
#include "mx4.h"

namespace aih {
namespace {

constexpr int kThreads = 256;

// Units are numbered over the padded rows, which are whole 128s of elements, so a
// block's four never part and a unit's codes are at its own number.
template <int DT, bool WIDE>
__global__ __launch_bounds__(kThreads) void mx4_quant_kernel(Mx4RowsArgs a) {
  constexpr int EB = Storage<DT>::bytes;
  const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.units) return;  // whole quads
  const uint32_t unit = (uint32_t)i, row = fdiv(unit, a.by_upr), u = unit - row * a.upr;
  const uint32_t left = u * 8 < a.k ? min(a.k - u * 8, 8u) : 0;
  Mx4Unit<DT> v;
  v.template load<WIDE>((const char *)a.src + ((uint64_t)row * a.stride + (uint64_t)u * 8) * EB, left);
  float f[8];
  v.get(f);
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, __float_as_uint(f[e]) & 0x7fffffffu);
  const uint32_t byte = mx4_scale_byte(mx4_quad_max(top));
  ((uint32_t *)a.dst)[i] = mx4_encode8(f, byte);
  if ((threadIdx.x & 3) == 0) a.dst_scales[(uint64_t)row * a.scale_stride + u / 4] = (uint8_t)byte;
}

template <int DT, bool WIDE>
__global__ __launch_bounds__(kThreads) void mx4_dequant_kernel(Mx4RowsArgs a) {
  constexpr int EB = Storage<DT>::bytes;
  const uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x;
  if (i >= a.units) return;
  const uint32_t unit = (uint32_t)i, row = fdiv(unit, a.by_upr), u = unit - row * a.upr;
  const uint32_t c = *reinterpret_cast<const uint32_t *>((const char *)a.src + (uint64_t)row * a.code_stride + u * 4);
  const float s = mx4_scale(a.src_scales[(uint64_t)row * a.scale_stride + u / 4]);
  float f[8];
  const f32x2 f0 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0), f1 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
  const f32x2 f2 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2), f3 = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
  f[0] = f0.x, f[1] = f0.y, f[2] = f1.x, f[3] = f1.y, f[4] = f2.x, f[5] = f2.y, f[6] = f3.x, f[7] = f3.y;
  Mx4Unit<DT> v;
  v.set(f);
  v.template store<WIDE>((char *)a.dst + ((uint64_t)row * a.stride + (uint64_t)u * 8) * EB, min(a.k - u * 8, 8u));
}

// 16-byte accesses need rows that start at such boundaries
template <int DT>
bool wide(const Mx4RowsArgs &a) {
  return a.stride * Storage<DT>::bytes % 16 == 0;
}

template <int DT>
hipError_t quant_dt(const Mx4RowsArgs &a, hipStream_t st) {
  const dim3 grid((uint32_t)((a.units + kThreads - 1) / kThreads));
  if (wide<DT>(a)) hipLaunchKernelGGL((mx4_quant_kernel<DT, true>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((mx4_quant_kernel<DT, false>), grid, dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

template <int DT>
hipError_t dequant_dt(const Mx4RowsArgs &a, hipStream_t st) {
  const dim3 grid((uint32_t)((a.units + kThreads - 1) / kThreads));
  if (wide<DT>(a)) hipLaunchKernelGGL((mx4_dequant_kernel<DT, true>), grid, dim3(kThreads), 0, st, a);
  else hipLaunchKernelGGL((mx4_dequant_kernel<DT, false>), grid, dim3(kThreads), 0, st, a);
  return hipGetLastError();
}

}  // namespace

hipError_t launch_mx4_quant(const Mx4RowsArgs &a, int dt, hipStream_t st) {
  return dt == DT_F32 ? quant_dt<DT_F32>(a, st) : dt == DT_F16 ? quant_dt<DT_F16>(a, st) : quant_dt<DT_BF16>(a, st);
}

hipError_t launch_mx4_dequant(const Mx4RowsArgs &a, int dt, hipStream_t st) {
  return dt == DT_F32 ? dequant_dt<DT_F32>(a, st)
                      : dt == DT_F16 ? dequant_dt<DT_F16>(a, st) : dequant_dt<DT_BF16>(a, st);
}

}  // namespace aih
