// mx4_capi.hip -- the extern "C" boundary of include/aih_mx4.h: checks of every
// argument that the host knows, the plan, the launches. What only the device knows
// (slots, page tables, lengths, positions) the kernels bound themselves.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <string>

#include "aih_device.h"
#include "capi_util.h"
#include "mx4.h"

namespace aih {
namespace {

constexpr uint32_t kMaxK = 1u << 20;
constexpr uint64_t kMaxStride = 1u << 22;

bool dt_ok(int32_t dt) { return dt == AIH_F32 || dt == AIH_F16 || dt == AIH_BF16; }
std::string num(uint64_t v) { return std::to_string(v); }

bool aligned16(std::initializer_list<const void *> ps) {
  for (const void *p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}
bool none_null(std::initializer_list<const void *> ps) {
  for (const void *p : ps)
    if (!p) return false;
  return true;
}

hipStream_t stream_of(aih_stream s) { return static_cast<hipStream_t>(s); }

int launched(const char *fn, hipError_t e) {
  if (e == hipSuccess) return AIH_OK;
  return api_fail(std::string(fn) + ": launch failed: " + hipGetErrorString(e));
}

int k_ok(const char *fn, uint32_t k) {
  if (k == 0 || k % 4 || k > kMaxK)
    return api_fail(std::string(fn) + ": k must be a multiple of 4, 4 to " + num(kMaxK) + ", not " + num(k));
  return AIH_OK;
}

int rows_stride(const char *fn, const char *what, uint64_t given, uint32_t k, uint64_t *out) {
  *out = given ? given : k;
  if (*out < k || *out % 4 || *out > kMaxStride)
    return api_fail(std::string(fn) + ": " + what + " must be 0 or a multiple of 4 from k to " + num(kMaxStride) + ", not " + num(given));
  return AIH_OK;
}

}  // namespace
}  // namespace aih

using namespace aih;

extern "C" int aih_mx4_quant(const aih_mx4_quant_desc *d, const void *x, void *codes, void *scales, aih_stream stream) {
  return api_guarded([&]() -> int {
    const char *fn = "aih_mx4_quant";
    if (!d) return api_fail("aih_mx4_quant: NULL descriptor");
    if (!dt_ok(d->dt)) return api_fail("aih_mx4_quant: unknown dtype " + std::to_string(d->dt));
    if (int rc = k_ok(fn, d->k)) return rc;
    Mx4RowsArgs a{};
    if (int rc = rows_stride(fn, "x_stride", d->x_stride, d->k, &a.stride)) return rc;
    a.k = d->k, a.upr = AIH_MX4_CODE_BYTES(d->k) / 4, a.units = (uint64_t)d->rows * a.upr;
    if (a.units > 0xffffffffu) return api_fail("aih_mx4_quant: rows of k rounded to 128 must hold less than 2^35 elements");
    if (d->rows == 0) return AIH_OK;
    if (!none_null({x, codes, scales})) return api_fail("aih_mx4_quant: NULL tensor");
    if (!aligned16({x, codes, scales})) return api_fail("aih_mx4_quant: tensors must be aligned to 16 bytes");
    a.src = x, a.dst = codes, a.dst_scales = static_cast<uint8_t *>(scales);
    a.scale_stride = AIH_MX4_SCALE_BYTES(d->k);
    a.by_upr = make_fastdiv(a.upr);
    return launched(fn, launch_mx4_quant(a, d->dt, stream_of(stream)));
  });
}

extern "C" int aih_mx4_dequant(const aih_mx4_dequant_desc *d, const void *codes, const void *scales, void *y,
                               aih_stream stream) {
  return api_guarded([&]() -> int {
    const char *fn = "aih_mx4_dequant";
    if (!d) return api_fail("aih_mx4_dequant: NULL descriptor");
    if (!dt_ok(d->dt)) return api_fail("aih_mx4_dequant: unknown dtype " + std::to_string(d->dt));
    if (int rc = k_ok(fn, d->k)) return rc;
    Mx4RowsArgs a{};
    if (int rc = rows_stride(fn, "y_stride", d->y_stride, d->k, &a.stride)) return rc;
    const uint32_t blocks = (d->k + 31) / 32;
    a.code_stride = d->code_stride ? d->code_stride : AIH_MX4_CODE_BYTES(d->k);
    a.scale_stride = d->scale_stride ? d->scale_stride : AIH_MX4_SCALE_BYTES(d->k);
    if (a.code_stride % 16 || a.code_stride < blocks * 16)
      return api_fail("aih_mx4_dequant: code_stride must be a multiple of 16 that holds " + num(blocks) + " blocks, not " + num(d->code_stride));
    if (a.scale_stride < blocks)
      return api_fail("aih_mx4_dequant: scale_stride must hold " + num(blocks) + " blocks, not " + num(d->scale_stride));
    a.k = d->k, a.upr = (d->k + 7) / 8, a.units = (uint64_t)d->rows * a.upr;
    if (a.units > 0xffffffffu) return api_fail("aih_mx4_dequant: rows must hold less than 2^35 elements");
    if (d->rows == 0) return AIH_OK;
    if (!none_null({codes, scales, y})) return api_fail("aih_mx4_dequant: NULL tensor");
    if (!aligned16({codes, y})) return api_fail("aih_mx4_dequant: tensors must be aligned to 16 bytes");
    a.src = codes, a.src_scales = static_cast<const uint8_t *>(scales), a.dst = y;
    a.by_upr = make_fastdiv(a.upr);
    return launched(fn, launch_mx4_dequant(a, d->dt, stream_of(stream)));
  });
}

extern "C" int aih_mx4_pw(const aih_mx4_pw_desc *d, const void *x_codes, const void *x_scales, const void *w_codes,
                          const void *w_scales, const void *bias, const void *res, void *y, aih_stream stream) {
  return api_guarded([&]() -> int {
    const char *fn = "aih_mx4_pw";
    if (!d) return api_fail("aih_mx4_pw: NULL descriptor");
    if (!dt_ok(d->dt)) return api_fail("aih_mx4_pw: unknown dtype " + std::to_string(d->dt));
    if (int rc = k_ok(fn, d->k)) return rc;
    if (d->cout == 0 || d->cout % 4 || d->cout > kMaxK)
      return api_fail("aih_mx4_pw: cout must be a multiple of 4, 4 to " + num(kMaxK) + ", not " + num(d->cout));
    if (d->m > 0x7fffffffu) return api_fail("aih_mx4_pw: m must be below 2^31");
    if (d->act < AIH_ACT_NONE || d->act > AIH_ACT_RECIP) return api_fail("aih_mx4_pw: unknown activation " + std::to_string(d->act));
    if (d->residual != 0 && d->residual != 1) return api_fail("aih_mx4_pw: residual must be 0 or 1");
    if (d->m == 0) return AIH_OK;
    if (!none_null({x_codes, x_scales, w_codes, w_scales, y})) return api_fail("aih_mx4_pw: NULL tensor");
    if (d->residual && !res) return api_fail("aih_mx4_pw: residual needs res");
    if (!aligned16({x_codes, x_scales, w_codes, w_scales, bias, res, y}))
      return api_fail("aih_mx4_pw: tensors must be aligned to 16 bytes");
    Mx4PwArgs a{};
    a.xc = static_cast<const uint8_t *>(x_codes), a.xs = static_cast<const uint8_t *>(x_scales);
    a.wc = static_cast<const uint8_t *>(w_codes), a.ws = static_cast<const uint8_t *>(w_scales);
    a.bias = bias, a.res = d->residual ? res : nullptr, a.y = y;
    a.m = d->m, a.cout = d->cout, a.act = d->act;
    a.cb = AIH_MX4_CODE_BYTES(d->k), a.sb = AIH_MX4_SCALE_BYTES(d->k), a.nst = a.cb / 64;
    a.nxcd = device_xcds();
    return launched(fn, launch_mx4_pw(a, d->dt, stream_of(stream)));
  });
}
