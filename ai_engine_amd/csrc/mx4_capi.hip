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
// Workgroups of 256 threads: a launch takes less than 2^32 threads, and one of more may run a
// few of them and report nothing.
constexpr uint32_t kMaxGroups = 0xffffff;

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

// A row stride in elements of `row`-long rows: whole 16-byte units.
int heads_stride(const char *fn, const char *what, uint64_t given, uint64_t row, int32_t dt, uint64_t *out) {
  *out = given ? given : row;
  if (*out < row || *out * (dt == AIH_F32 ? 4 : 2) % 16 || *out > kMaxStride)
    return api_fail(std::string(fn) + ": " + what + " must be 0 or whole 16-byte units from " + num(row) + " to " +
                    num(kMaxStride) + ", not " + num(given));
  return AIH_OK;
}

int cache_ok(const char *fn, uint32_t hkv, uint32_t d, uint32_t page, uint32_t pages, int32_t dt) {
  if (!dt_ok(dt)) return api_fail(std::string(fn) + ": unknown dtype " + std::to_string(dt));
  if (d == 0 || d % 32 || d > 256) return api_fail(std::string(fn) + ": d must be a multiple of 32, 32 to 256, not " + num(d));
  if (hkv == 0 || hkv > 4096) return api_fail(std::string(fn) + ": hkv must be 1 to 4096");
  if (page < 16 || page > 4096 || (page & (page - 1)))
    return api_fail(std::string(fn) + ": page must be a power of two, 16 to 4096, not " + num(page));
  if ((uint64_t)pages * page > 0x7fffffffu) return api_fail(std::string(fn) + ": pages * page must be below 2^31");
  return AIH_OK;
}

uint32_t log2_of(uint32_t pow2) {
  uint32_t s = 0;
  while ((1u << s) < pow2) ++s;
  return s;
}

struct Kv4Plan {
  uint32_t rb;     // a tile's rows: 16 rb
  uint64_t tiles;  // of a key head, at most
  uint32_t parts, shift;
  uint64_t ws_floats;
};

// How the keys are cut. A workgroup's rows against all keys are a chain, about 0.8 us
// for each 128; cutting it costs partial results and a launch that joins them, 4 us.
// Measured, whole | cut to 256, 512, 1024, 2048 (32/8 heads of 128 bf16): 32 x 700 keys,
// 8/2 heads of 64 9.0 | 11.7, 11.7 us; 1 x 4000 33 | 11.7, 12.4, 15.4, 22; 16 x 2000 22 |
// 16.7, 15.6, 17.4; 64 of 0 to 8192 82 | 46, 38, 31.4, 37.7; 1 x 131071, 16/4 heads f16
// 902 | 40, 28.5, 23.3, 25.2. Prompts are cut where their tiles leave CUs without one: 1024
// tokens, 8/2 heads of 64 (256) 11.1 | 19, 16.3; 2000 tokens, 8/4 heads of 128 f16 (500) 31 to
// 1024 45; 2 x 300 behind 4000 keys, 8/2 heads (154) 43 | 51, 43, 35.2, 35.8. Heads of more than
// 128 take longer for a key: from 512 on whole | 512 | 256, 4 x 600 keys, 16/4 heads of 256 14.7 |
// 16.1 | 13.5, 4 x 1000 19.4 | 16.2 | 13.6, 64 x 900, 8/2 heads of 192 18.0 | 16.0 | 15.6, unless
// every CU has one anyway: 64 x 600, 16/4 heads of 256 16.5 | 22.9 | 23.5, 64 x 900 21.8 | 22.8 | 29.1.
//
// Prompts whose tiles fill the CUs are never cut, as the host does not know which of them
// are long: cut to 16384 keys, 4 x 500 tokens behind 20000, 32/8 heads of 128, take 952 for 733,
// 4 x 2000 behind 30000 4683 for 4227. Single tokens among them pay for it: 7 of 131072 keys
// beside a prompt of 2000 2016 (cut 431), in calls of their own 228 and 67.
int check_kv4_attn(const aih_kv4_attn_desc *d, AttnArgs *a, Kv4Plan *p) {
  const char *fn = "aih_kv4_attn";
  if (!d) return api_fail("aih_kv4_attn: NULL descriptor");
  if (int rc = cache_ok(fn, d->hkv, d->d, d->page, d->pages, d->dt)) return rc;
  if (d->hq == 0 || d->hq > 4096 || d->hq % d->hkv) return api_fail("aih_kv4_attn: hq must be a multiple of hkv, at most 4096");
  if (d->causal != 0 && d->causal != 1) return api_fail("aih_kv4_attn: causal must be 0 or 1");
  if (d->nseq > 0x7fffffffu || d->tokens > 0x7fffffffu) return api_fail("aih_kv4_attn: counts must be below 2^31");
  if ((uint64_t)d->tokens * d->hq > 0x7fffffffu) return api_fail("aih_kv4_attn: tokens * hq must be below 2^31");
  if ((uint64_t)d->table_width * d->page > 0x7fffffffu) return api_fail("aih_kv4_attn: table_width * page must be below 2^31");
  if (d->scale != 0.0f && !(d->scale >= 1e-20f && d->scale <= 1e20f))
    return api_fail("aih_kv4_attn: scale must be 0 or 1e-20 to 1e20");
  *a = AttnArgs{};
  *p = Kv4Plan{1, 0, 1, 31, 0};
  a->nseq = d->nseq, a->tokens = d->tokens;
  a->rows = d->pages ? d->table_width * d->page : 0;  // keys of a sequence at most
  a->hq = d->hq, a->hkv = d->hkv, a->g = d->hq / d->hkv, a->d = d->d;
  a->causal = (uint32_t)d->causal;
  const double scale = d->scale != 0.0f ? (double)d->scale : 1.0 / std::sqrt((double)d->d);
  a->scale_log2 = (float)(scale * 1.4426950408889634);
  if (int rc = heads_stride(fn, "q_stride", d->q_stride, (uint64_t)d->hq * d->d, d->dt, &a->qs)) return rc;
  if (int rc = heads_stride(fn, "o_stride", d->o_stride, (uint64_t)d->hq * d->d, d->dt, &a->os)) return rc;
  if (d->nseq == 0 || d->tokens == 0) return AIH_OK;
  const uint64_t rows = (uint64_t)d->tokens * a->g;
  const uint32_t cus = device_cus();
  const bool few = rows <= 32ull * d->nseq;
  // 64 rows convert the keys half as often as 32, where sequences have more than 32 of them
  // and there are two such tiles a CU.
  // 32 | 64, bf16: four prompts of 100 to 1024 behind 2000 keys, 32/8 heads of 128
  // (1112 tiles of 64) 148 | 137 us, 4096 tokens (2048) 218 | 177, 4 x 500 behind 100, 16/4
  // heads of 96 (516) 24.5 | 21.8; f16, 8 x 720, 8/2 heads of 64 (368) 31.8 | 33.9; 4096
  // tokens, 32/8 heads, f16 of 32 111 | 118, of 64 156 | 158, of 96 266 | 213, fp32 of 96 325 |
  // 271, of 128 552 | 472. Above 128 the registers do not hold 64 rows' results. Of 32 rows a
  // sequence at most half of a tile of 64 is empty: 128 x 5 tokens over 500 keys, 32/8 heads of
  // 128 bf16 27.3 | 41.1, fp32 62 | 88; 1024 tokens over 400, 32/1 heads of 128 bf16 46.3 | 53.3
  const bool wide = !few && d->d >= 64 && d->d <= 128 && (rows / 64 + d->nseq / 2) * d->hkv >= 2ull * cus;
  p->rb = rows <= 16ull * d->nseq ? 1 : wide ? 4 : 2;
  const uint32_t bm = 16 * p->rb;
  p->tiles = d->nseq == 1 ? (rows + bm - 1) / bm : rows / bm + d->nseq;
  const uint32_t len = d->max_len ? std::min(d->max_len, a->rows) : a->rows;
  auto parts = [&](uint32_t x) { return (uint32_t)std::max<uint64_t>(1, ((uint64_t)len + (1ull << x) - 1) >> x); };
  const uint64_t base = p->tiles * d->hkv;
  // the join's launch takes 1024 threads a row at the most; the chip is full without
  const bool joins = (uint64_t)d->tokens * d->hq < 1u << 22;
  if (joins && few && len > (d->d > 128 && base < cus ? 512u : 1024u)) {
    p->shift = 10;
    while (p->shift > 8 && base * parts(p->shift) < 2ull * cus) --p->shift;
  } else if (!few && base < cus) {
    while (p->shift > 10 && base * parts(p->shift) < 2ull * cus) --p->shift;
  }
  p->parts = parts(p->shift);
  if (p->parts == 1) p->shift = 31;
  if (base * p->parts > 0x7fffffffu) return api_fail("aih_kv4_attn: more than 2^31 - 1 tiles");
  if (p->parts > 1) p->ws_floats = (uint64_t)p->parts * d->tokens * d->hq * (d->d + 2);
  return AIH_OK;
}

}  // namespace

hipError_t launch_kv4_attn(const Kv4AttnArgs &a, int dt, hipStream_t st) {
  return dt == DT_F32 ? launch_kv4_attn_f32(a, st) : dt == DT_F16 ? launch_kv4_attn_f16(a, st) : launch_kv4_attn_bf16(a, st);
}

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
    if (a.units > 256ull * kMaxGroups)
      return api_fail("aih_mx4_quant: rows of k rounded to 128 must hold at most 2^35 - 2048 elements");
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
    if (a.units > 256ull * kMaxGroups) return api_fail("aih_mx4_dequant: rows must hold at most 2^35 - 2048 elements");
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
    if (d->m > 0x7fffff00u) return api_fail("aih_mx4_pw: m must be at most 2^31 - 256");
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

extern "C" int aih_kv4_append(const aih_kv4_append_desc *d, const void *x, const void *wq, const void *wk,
                              const float *cosines, const float *sines, const int32_t *pos, const int32_t *slots,
                              void *q, void *k_codes, void *k_scales, void *v_codes, void *v_scales, aih_stream stream) {
  return api_guarded([&]() -> int {
    const char *fn = "aih_kv4_append";
    if (!d) return api_fail("aih_kv4_append: NULL descriptor");
    if (int rc = cache_ok(fn, d->hkv, d->d, d->page, d->pages, d->dt)) return rc;
    if (d->hq > 4096) return api_fail("aih_kv4_append: hq must be at most 4096");
    if (d->rot % 16 || d->rot > d->d)
      return api_fail("aih_kv4_append: rot must be a multiple of 16, at most d, not " + num(d->rot));
    if (d->pairs != 0 && d->pairs != 1) return api_fail("aih_kv4_append: pairs must be 0 or 1");
    if (d->norm != 0 && d->norm != 1) return api_fail("aih_kv4_append: norm must be 0 or 1");
    if (!(d->eps >= 0.0f) || !std::isfinite(d->eps)) return api_fail("aih_kv4_append: eps must be >= 0 and finite");
    if (d->rot && (d->positions == 0 || d->positions > 0x7fffffffu))
      return api_fail("aih_kv4_append: the tables need 1 to 2^31 - 1 rows");
    const uint64_t heads = (uint64_t)d->hq + 2 * (uint64_t)d->hkv;
    if (d->tokens * heads > 0x7fffffffu) return api_fail("aih_kv4_append: tokens * (hq + 2 hkv) must be below 2^31");
    // a workgroup takes four wavefronts of 64 / (d / 8) heads
    if ((d->tokens * heads + 4 * (512 / d->d) - 1) / (4 * (512 / d->d)) > kMaxGroups)
      return api_fail("aih_kv4_append: tokens * (hq + 2 hkv) must be at most (2^24 - 1) * 4 * (512 / d)");
    Kv4AppendArgs a{};
    if (int rc = heads_stride(fn, "x_stride", d->x_stride, heads * d->d, d->dt, &a.xs)) return rc;
    if (int rc = heads_stride(fn, "q_stride", d->q_stride, (uint64_t)d->hq * d->d, d->dt, &a.qs)) return rc;
    if (d->tokens == 0) return AIH_OK;
    if (!none_null({x, slots, k_codes, k_scales, v_codes, v_scales}) || (d->hq && !q))
      return api_fail("aih_kv4_append: NULL tensor");
    if (d->rot && (!cosines || !sines)) return api_fail("aih_kv4_append: rot > 0 needs cosines and sines");
    if (!aligned16({x, wq, wk, cosines, sines, q, k_codes, k_scales, v_codes, v_scales}))
      return api_fail("aih_kv4_append: tensors must be aligned to 16 bytes");
    a.x = x, a.wq = wq, a.wk = wk, a.cs = cosines, a.sn = sines, a.pos = pos, a.slots = slots, a.q = q;
    a.kc = static_cast<uint8_t *>(k_codes), a.ks = static_cast<uint8_t *>(k_scales);
    a.vc = static_cast<uint8_t *>(v_codes), a.vs = static_cast<uint8_t *>(v_scales);
    a.hq = d->hq, a.hkv = d->hkv, a.d = d->d, a.rot = d->rot, a.pairs = (uint32_t)d->pairs, a.norm = (uint32_t)d->norm;
    a.positions = d->positions, a.rows = d->pages * d->page, a.pshift = log2_of(d->page);
    a.items = (uint32_t)(d->tokens * heads);
    a.eps = d->eps, a.inv_d = 1.0f / (float)d->d;
    a.nl = d->d / 8, a.per = 64 / a.nl;
    a.by_ht = make_fastdiv((uint32_t)heads), a.by_nl = make_fastdiv(a.nl);
    return launched(fn, launch_kv4_append(a, d->dt, stream_of(stream)));
  });
}

extern "C" int aih_kv4_attn_plan(const aih_kv4_attn_desc *d, aih_kv4_attn_plan_info *out) {
  return api_guarded([&]() -> int {
    AttnArgs a;
    Kv4Plan p;
    if (int rc = check_kv4_attn(d, &a, &p)) return rc;
    if (!out) return api_fail("aih_kv4_attn_plan: NULL output");
    *out = aih_kv4_attn_plan_info{};
    out->bm = 16 * p.rb, out->parts = p.parts, out->chunk = p.parts > 1 ? 1u << p.shift : 0;
    out->grid = (uint32_t)(p.tiles * d->hkv * p.parts);
    out->ws_bytes = p.ws_floats * 4;
    return AIH_OK;
  });
}

extern "C" int aih_kv4_attn(const aih_kv4_attn_desc *d, const void *q, const void *k_codes, const void *k_scales,
                            const void *v_codes, const void *v_scales, const int32_t *q_start, const int32_t *table,
                            const int32_t *k_len, void *o, void *ws, size_t ws_bytes, aih_stream stream) {
  return api_guarded([&]() -> int {
    const char *fn = "aih_kv4_attn";
    Kv4AttnArgs a{};
    Kv4Plan p;
    if (int rc = check_kv4_attn(d, &a.at, &p)) return rc;
    if (d->nseq == 0 || d->tokens == 0) return AIH_OK;
    if (!none_null({q, q_start, k_len, o})) return api_fail("aih_kv4_attn: NULL tensor");
    if (a.at.rows && !none_null({k_codes, k_scales, v_codes, v_scales, table}))
      return api_fail("aih_kv4_attn: a cache with pages must not be NULL");
    if (!aligned16({q, k_codes, k_scales, v_codes, v_scales, o, ws}))
      return api_fail("aih_kv4_attn: tensors must be aligned to 16 bytes");
    if (p.ws_floats && (!ws || ws_bytes < p.ws_floats * 4))
      return api_fail("aih_kv4_attn: the workspace needs " + num(p.ws_floats * 4) + " bytes, not " + num(ws ? ws_bytes : 0));
    AttnArgs &t = a.at;
    t.q = q, t.o = o, t.ws = p.ws_floats ? static_cast<float *>(ws) : nullptr;
    t.q_start = q_start, t.k_len = k_len;
    t.by_g = make_fastdiv(t.g), t.by_hkv = make_fastdiv(t.hkv);
    t.tiles = (uint32_t)p.tiles, t.parts = p.parts, t.shift = p.shift, t.all_parts = p.parts;
    // prompts of different lengths start with the longest
    t.sort = d->nseq > 1 && d->nseq <= 32 && (uint64_t)d->tokens * t.g > 16ull * p.rb * d->nseq;
    a.kc = static_cast<const uint8_t *>(k_codes), a.ks = static_cast<const uint8_t *>(k_scales);
    a.vc = static_cast<const uint8_t *>(v_codes), a.vs = static_cast<const uint8_t *>(v_scales);
    a.rb = p.rb;
    a.table = table, a.width = d->table_width, a.pages = d->pages, a.pshift = log2_of(d->page);
    const hipStream_t st = stream_of(stream);
    if (int rc = launched(fn, launch_kv4_attn(a, d->dt, st))) return rc;
    if (!t.ws) return AIH_OK;
    return launched(fn, launch_attn_join(t, d->dt, st));
  });
}
