// attn_capi.hip -- the extern "C" boundary of include/aih_attn.h: checks of
// every argument that the host knows, the plan, the launches. What only the
// device knows (lengths, positions, slots) the kernels bound themselves.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <initializer_list>
#include <string>

#include "aih_device.h"
#include "attn.h"
#include "capi_util.h"

namespace aih {
namespace {

constexpr uint64_t kMaxRow = 1u << 22;  // elements of a row stride: 128 rows stay within 32-bit byte offsets

bool dt_ok(int32_t dt) { return dt == AIH_F32 || dt == AIH_F16 || dt == AIH_BF16; }
uint32_t dt_bytes(int32_t dt) { return dt == AIH_F32 ? 4 : 2; }

bool aligned16(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

std::string num(uint64_t v) { return std::to_string(v); }

// A row stride in elements: 0 becomes `row`, anything else must hold a row in
// whole 16-byte units.
int take_stride(const char *what, uint64_t given, uint64_t row, int32_t dt, uint64_t *out) {
  *out = given ? given : row;
  if (*out < row) return api_fail(std::string(what) + " " + num(given) + " is shorter than a row of " + num(row));
  if (*out * dt_bytes(dt) % 16) return api_fail(std::string(what) + " " + num(given) + " is not a whole number of 16-byte units");
  if (*out > kMaxRow) return api_fail(std::string(what) + " " + num(*out) + " is above " + num(kMaxRow));
  return AIH_OK;
}

int heads_ok(const char *fn, uint32_t hq, uint32_t hkv, uint32_t d, int32_t dt) {
  if (!dt_ok(dt)) return api_fail(std::string(fn) + ": unknown dtype " + std::to_string(dt));
  if (d == 0 || d % 8 || d > 256) return api_fail(std::string(fn) + ": d must be a multiple of 8, 8 to 256, not " + num(d));
  if (hq == 0 || hq > 4096 || hkv > 4096) return api_fail(std::string(fn) + ": heads must be 1 to 4096");
  return AIH_OK;
}

hipStream_t stream_of(aih_stream s) { return static_cast<hipStream_t>(s); }

int launched(const char *fn, hipError_t e) {
  if (e == hipSuccess) return AIH_OK;
  return api_fail(std::string(fn) + ": launch failed: " + hipGetErrorString(e));
}

// How a launch covers its rows and keys.
struct Cover {
  int32_t kernel;
  uint32_t bm, tiles, parts, shift, span;
};

uint32_t div_up(uint64_t a, uint64_t b) { return (uint32_t)((a + b - 1) / b); }

enum class Use { OWN, PREFIX };

// `nseq` sequences of `rows` (query, head of the group) rows altogether, each
// against about `len` keys. What cutting the keys gains in spread it pays for
// with partial results and a launch that joins them, which the prefix needs
// anyway. Measured with AIH_ATTN_KEYS (16 bit; heads, keys: whole | cut):
//   1 stream, 32/8 heads of 128: 512 8.0 | 9.3 us, 1024 11.7 | 9.6, 4096 24 | 10.5
//   16 streams: 1024 14.5 | 18.9 us, 2048 in 2 parts 34.6, in 8 36.9
//   a prompt of 1500, 4/4 heads of 64 (188 items) 11.8 | 16.9 us
// fp32, 1 stream, 8/2 heads of 64: 384 10.9 | 11.5 us, 512 13.1 | 11.6; a prompt of
// 1024, 4/4 heads (128 items) 22.7 | 18.8. Few rows are cut at 1024 anyway, since
// the sequences' lengths may differ a lot. 64 streams behind a prefix of 4096,
// 32/8 heads of 128: 8 parts 29.2 us, 4 parts 25.1; but 64 of 4 tokens, heads of 64
// (512 items) 1 part 34.9, 2 parts 26.9: more than 2048 of a prefix's 16-bit keys
// are too long a chain.
//
// A stage of 128 fp32 keys takes 1 us per 32 elements, a chain that shorter parts
// make the shorter the larger the heads (`heavy`; 1 stream of 271 keys, 16/4 heads of
// 256: 33.0 | 18.2 us; 5 behind a prefix of 651: 2 parts 47.3, 6 parts 19.8), as
// long as the parts still run at once: a first cut that does not fit the CUs loses
// (40 x 600 keys, 4/4 heads of 32, 160 items 11.7 | 18.9; a prompt of 300, 16/4 heads
// of 256, 152 items 37.7 | 44.3), another one where it leaves a few over (8 x 2000,
// 18/3 heads of 256, 8 parts 39.1, 16 parts, 432 items, 49.2). Few rows of at most 128
// elements run twice a CU: 16 x 2000 keys, 32/8 heads of 64, 2 parts 34.6, 4 parts 33.4, of
// lengths from 0 to 2000 28.5 | 19.3; in 16 bit that is a tenth slower.
// One of 256 16-bit elements takes 2 us: with few rows shorter parts pay, too (4 x 600
// keys, 16/4 heads 14.6 | 11.8; 16 x 600, 72 items 15.5 | 18.6).
Cover cover(int32_t kernel, uint32_t nseq, uint64_t rows, uint32_t len, uint32_t hkv, int32_t dt, uint32_t d, Use use) {
  const uint32_t cus = device_cus();
  Cover c{};
  c.kernel = kernel;
  c.bm = attn_bm(c.kernel);
  c.tiles = nseq == 1 ? div_up(rows, c.bm) : (uint32_t)(rows / c.bm) + nseq;
  const uint64_t base = (uint64_t)c.tiles * hkv;
  auto parts = [&](uint32_t x) { return std::max(1u, div_up(len, 1ull << x)); };
  const bool few = rows <= 32ull * nseq;
  const uint32_t heavy = dt != AIH_F32 ? d > 128 && 4 * base < cus : d > 128 ? 2 : d > 64 ? 1 : 0;
  const uint32_t whole = use == Use::PREFIX ? 0 : kernel == AIH_ATTN_ROWS ? len : (dt == AIH_F32 ? 384 : 768) >> heavy;
  // what the chip runs at once: two workgroups a CU, but one of large or many rows
  const uint32_t slots = few && use == Use::OWN && heavy < 2 ? 2 * cus : cus;
  const uint32_t items = dt == AIH_F32 ? slots : use == Use::PREFIX ? cus : cus / 2;
  const uint32_t least = std::max(7u, (few && use == Use::OWN ? 8 : 9) - heavy);
  c.shift = 31;
  if (len > whole) {
    if (use == Use::PREFIX && dt != AIH_F32)
      while (c.shift > 11 && base * parts(c.shift) < 2 * cus) --c.shift;
    if (few && use == Use::OWN) c.shift = dt == AIH_F32 && len > 2u << (10 - heavy) ? 10 - heavy : 10;
    while (c.shift > least && base * parts(c.shift) < items &&
           (dt != AIH_F32 || use == Use::PREFIX ||
            base * parts(c.shift - 1) <= (parts(c.shift) > 1 ? slots + cus / 4 : cus)))
      --c.shift;
  }
  c.parts = parts(c.shift);
  if (c.parts == 1) c.shift = 31;
  c.span = (uint32_t)std::min<uint64_t>(len, 1ull << c.shift);
  return c;
}

struct AttnPlan {
  Cover own, pre;
  bool together;  // the prefix in the same launch
  uint32_t all_parts;
  uint64_t ws_floats;
};

int check_attn(const aih_attn_desc *d, AttnArgs *a, AttnPlan *p) {
  if (!d) return api_fail("aih_attn: NULL descriptor");
  if (int rc = heads_ok("aih_attn", d->hq, d->hkv, d->d, d->dt)) return rc;
  if (d->hkv == 0 || d->hq % d->hkv) return api_fail("aih_attn: hq must be a multiple of hkv");
  if (d->causal != 0 && d->causal != 1) return api_fail("aih_attn: causal must be 0 or 1");
  if (d->nseq > 0x7fffffffu || d->tokens > 0x7fffffffu || d->rows > 0x7fffffffu || d->prefix > 0x7fffffffu)
    return api_fail("aih_attn: counts must be below 2^31");
  if ((uint64_t)d->tokens * d->hq > 0x7fffffffu) return api_fail("aih_attn: tokens * hq must be below 2^31");
  if (d->scale != 0.0f && !(d->scale >= 1e-20f && d->scale <= 1e20f))
    return api_fail("aih_attn: scale must be 0 or 1e-20 to 1e20");
  *a = AttnArgs{};
  *p = AttnPlan{};
  a->nseq = d->nseq, a->tokens = d->tokens, a->rows = d->rows;
  a->hq = d->hq, a->hkv = d->hkv, a->g = d->hq / d->hkv, a->d = d->d;
  a->causal = (uint32_t)d->causal;
  const double scale = d->scale != 0.0f ? (double)d->scale : 1.0 / std::sqrt((double)d->d);
  a->scale_log2 = (float)(scale * 1.4426950408889634);
  if (int rc = take_stride("aih_attn: q_stride", d->q_stride, (uint64_t)d->hq * d->d, d->dt, &a->qs)) return rc;
  if (int rc = take_stride("aih_attn: o_stride", d->o_stride, (uint64_t)d->hq * d->d, d->dt, &a->os)) return rc;
  if (int rc = take_stride("aih_attn: k_stride", d->k_stride, (uint64_t)d->hkv * d->d, d->dt, &a->ks)) return rc;
  if (int rc = take_stride("aih_attn: v_stride", d->v_stride, (uint64_t)d->hkv * d->d, d->dt, &a->vs)) return rc;
  if (int rc = take_stride("aih_attn: pk_stride", d->pk_stride, (uint64_t)d->hkv * d->d, d->dt, &a->pks)) return rc;
  if (int rc = take_stride("aih_attn: pv_stride", d->pv_stride, (uint64_t)d->hkv * d->d, d->dt, &a->pvs)) return rc;
  if (d->nseq == 0 || d->tokens == 0) return AIH_OK;
  const uint64_t rows = (uint64_t)d->tokens * a->g;
  const uint32_t len = d->max_len ? std::min(d->max_len, d->rows) : div_up(d->rows, d->nseq);
  const bool rows_fit = d->d * dt_bytes(d->dt) <= 512;  // else the registers do not hold a wavefront's queries
  // Prompts of few tiles: a wavefront's 32 rows against all keys are a chain
  // that sets the time while others have nothing to do, so the keys go over
  // the wavefronts. Measured, rows | keys over the wavefronts: fp32 causal, 4096
  // tokens, 16/4 heads of 96 (512 tiles) 564 | 436 us, 4 x 2048 tokens (1040) 573 |
  // 487, 16 x 720 (1504) 293 | 321; 16 bit, 2880 tokens, 8/2 heads of 64 (180) 41 |
  // 25, 16/4 heads (360) 44.6 | 43.6, of 128 63 | 70; 40 x 100 tokens, 8/2 heads of
  // 128 (330) 14 | 19: too short to share. So are fp32 heads above 64 elements, the
  // longer the more there are: 16/4 heads of 128, 4 x 100 tokens (60 tiles) 21 | 11.5,
  // 40 x 64 (400) 30 | 41, 8 x 260 (276) 76 | 50, 20 x 300 (792) 125 | 137, 3 x 700
  // (268) 105 | 80. Above 128 16-bit elements a wavefront's chain is written out: 8/4
  // heads of 256, 520 tokens (36) 26 | 15, 2 x 900 (120) 38 | 30, 8 x 260 (148) 20 | 28,
  // 6 x 520 (208) 28 | 42, 3000 (188) 100 | 92, not causal 105 | 149.
  const uint64_t tiles = (uint64_t)d->hkv * (div_up(rows, attn_bm(AIH_ATTN_ROWS)) + d->nseq / 2);
  const uint64_t cus = device_cus();
  const bool chain = d->dt == AIH_F32 ? tiles < 5 * cus && (d->d <= 64 || 180 * tiles < cus * len)
                                      : tiles < (d->d > 128 ? cus / 2 : cus) && len >= 256;
  const int32_t kernel = rows <= 32ull * d->nseq || !rows_fit || chain ? AIH_ATTN_KEYS : AIH_ATTN_ROWS;
  p->own = cover(kernel, d->nseq, rows, len, d->hkv, d->dt, d->d, Use::OWN);
  p->all_parts = p->own.parts;
  if (d->prefix) {
    // The prefix's keys over the wavefronts re-read them for every 32 rows, but
    // share a launch and leave few partial results: the faster as long as that is not
    // much to read. 1 to 134 own keys, bf16, together | apart: 64 streams of 4 tokens,
    // 12/2 heads of 128, behind 4096 keys 24 | 30 us, behind 8000 34 | 39; 128 of 1
    // token behind 24000 49 | 49; 64 x 4, 8/2 heads of 64, behind 8000 20 | 23, behind
    // 24000 37 | 35; 64 x 1, 32/8 heads of 128, behind 24000 74 | 58; 16 x 4, 16/4 heads
    // of 256, behind 24000 86 | 84, behind 60000 147 | 127. fp32 is bound by its
    // products: 64 x 4, 32/8 heads of 64 behind 1500 to 24000 keys 43 | 55, 89 | 92, 161
    // | 160, 481 | 526, of 128 76 | 99, 172 | 168, 341 | 296, 996 | 1011.
    const bool little = rows * d->hkv * d->prefix <= (1ull << 32) / std::max(d->d, 128u);
    p->together = kernel == AIH_ATTN_KEYS && (little || d->dt == AIH_F32);
    p->pre = cover(p->together ? AIH_ATTN_KEYS : AIH_ATTN_ROWS, 1, rows, d->prefix, d->hkv, d->dt, d->d, Use::PREFIX);
    p->all_parts += p->pre.parts;
  }
  if ((uint64_t)p->own.tiles * d->hkv * p->own.parts + (uint64_t)p->pre.tiles * d->hkv * p->pre.parts > 0x7fffffffu)
    return api_fail("aih_attn: more than 2^31 - 1 tiles");
  if (p->all_parts > 1) p->ws_floats = (uint64_t)p->all_parts * d->tokens * d->hq * (d->d + 2);
  return AIH_OK;
}

}  // namespace
}  // namespace aih

using namespace aih;

extern "C" int aih_qk_norm_rope(const aih_qk_norm_rope_desc *d, const void *x, const void *wq, const void *wk,
                                const float *cosines, const float *sines, const int32_t *pos, const int32_t *slots,
                                void *q, void *k, void *v, aih_stream stream) {
  return api_guarded([&]() -> int {
    if (!d) return api_fail("aih_qk_norm_rope: NULL descriptor");
    if (int rc = heads_ok("aih_qk_norm_rope", d->hq, d->hkv, d->d, d->dt)) return rc;
    if (d->rot % 4 || d->rot > d->d)
      return api_fail("aih_qk_norm_rope: rot must be a multiple of 4, at most d, not " + num(d->rot));
    if (d->pairs != 0 && d->pairs != 1) return api_fail("aih_qk_norm_rope: pairs must be 0 or 1");
    if (!(d->eps >= 0.0f) || !std::isfinite(d->eps)) return api_fail("aih_qk_norm_rope: eps must be >= 0 and finite");
    if (d->rot && d->positions == 0) return api_fail("aih_qk_norm_rope: the tables need at least one row");
    if (d->tokens > 0x7fffffffu || d->rows > 0x7fffffffu)
      return api_fail("aih_qk_norm_rope: counts must be below 2^31");
    QkRopeArgs a{};
    const uint64_t heads = (uint64_t)d->hq + 2 * (uint64_t)d->hkv;
    if (int rc = take_stride("aih_qk_norm_rope: x_stride", d->x_stride, heads * d->d, d->dt, &a.xs)) return rc;
    if (int rc = take_stride("aih_qk_norm_rope: q_stride", d->q_stride, (uint64_t)d->hq * d->d, d->dt, &a.qs)) return rc;
    if (int rc = take_stride("aih_qk_norm_rope: k_stride", d->k_stride, (uint64_t)d->hkv * d->d, d->dt, &a.ks)) return rc;
    if (int rc = take_stride("aih_qk_norm_rope: v_stride", d->v_stride, (uint64_t)d->hkv * d->d, d->dt, &a.vs)) return rc;
    if (d->tokens == 0) return AIH_OK;
    if (!x || !q || (d->hkv && !k)) return api_fail("aih_qk_norm_rope: x, q and k must not be NULL");
    if (d->rot && (!cosines || !sines)) return api_fail("aih_qk_norm_rope: rot > 0 needs cosines and sines");
    if (!aligned16(x) || !aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(wq) || !aligned16(wk) ||
        !aligned16(cosines) || !aligned16(sines))
      return api_fail("aih_qk_norm_rope: tensors must be aligned to 16 bytes");
    a.x = x, a.wq = wq, a.wk = wk, a.cs = cosines, a.sn = sines, a.pos = pos, a.slots = slots;
    a.q = q, a.k = k, a.v = v;
    a.hq = d->hq, a.hkv = d->hkv, a.ht = d->hq + d->hkv + (v ? d->hkv : 0);
    a.d = d->d, a.rot = d->rot, a.pairs = (uint32_t)d->pairs;
    a.positions = d->positions, a.rows = d->rows;
    a.items = (uint64_t)d->tokens * a.ht;
    a.eps = d->eps, a.inv_d = 1.0f / (float)d->d;
    return launched("aih_qk_norm_rope", launch_qk_norm_rope(a, d->dt, stream_of(stream)));
  });
}

extern "C" int aih_attn_plan(const aih_attn_desc *d, aih_attn_plan_info *out) {
  return api_guarded([&]() -> int {
    AttnArgs a;
    AttnPlan p;
    if (int rc = check_attn(d, &a, &p)) return rc;
    if (!out) return api_fail("aih_attn_plan: NULL output");
    *out = aih_attn_plan_info{};
    out->kernel = p.own.kernel, out->bm = p.own.bm, out->parts = p.own.parts;
    out->chunk = p.own.parts > 1 ? 1u << p.own.shift : 0;
    out->prefix_kernel = p.pre.kernel, out->prefix_bm = p.pre.bm, out->prefix_parts = p.pre.parts;
    out->prefix_chunk = p.pre.parts > 1 ? 1u << p.pre.shift : 0;
    const uint32_t own = p.own.tiles * d->hkv * p.own.parts, pre = p.pre.tiles * d->hkv * p.pre.parts;
    out->grid = p.pre.parts && !p.together ? pre : own + pre;
    out->ws_bytes = p.ws_floats * 4;
    return AIH_OK;
  });
}

extern "C" int aih_attn(const aih_attn_desc *d, const void *q, const void *k, const void *v, const int32_t *q_start,
                        const int32_t *k_start, const int32_t *k_len, const void *prefix_k, const void *prefix_v,
                        void *o, void *ws, size_t ws_bytes, aih_stream stream) {
  return api_guarded([&]() -> int {
    AttnArgs a;
    AttnPlan p;
    if (int rc = check_attn(d, &a, &p)) return rc;
    if (d->nseq == 0 || d->tokens == 0) return AIH_OK;
    if (!q || !o || !q_start || !k_start || !k_len) return api_fail("aih_attn: NULL tensor");
    if (d->rows && (!k || !v)) return api_fail("aih_attn: k and v must not be NULL");
    if (d->prefix && (!prefix_k || !prefix_v)) return api_fail("aih_attn: prefix > 0 needs prefix_k and prefix_v");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(prefix_k) || !aligned16(prefix_v) ||
        !aligned16(o) || !aligned16(ws))
      return api_fail("aih_attn: tensors must be aligned to 16 bytes");
    if (p.ws_floats && (!ws || ws_bytes < p.ws_floats * 4))
      return api_fail("aih_attn: the workspace needs " + num(p.ws_floats * 4) + " bytes, not " + num(ws ? ws_bytes : 0));
    const hipStream_t st = stream_of(stream);
    a.q = q, a.k = k, a.v = v, a.o = o, a.ws = p.ws_floats ? static_cast<float *>(ws) : nullptr;
    a.q_start = q_start, a.k_start = k_start, a.k_len = k_len;
    a.all_parts = p.all_parts;
    a.by_g = make_fastdiv(a.g), a.by_hkv = make_fastdiv(a.hkv);
    a.by_pre_tiles = make_fastdiv(std::max(1u, p.pre.tiles));
    a.pk = prefix_k, a.pv = prefix_v, a.prefix = d->prefix;
    a.tiles = p.own.tiles, a.parts = p.own.parts, a.shift = p.own.shift, a.part0 = p.pre.parts;
    // Prompts of different lengths: the longest first leave short ones for the end. As
    // given | sorted, 16 of 20 to 500 tokens, 8/4 heads of 96 fp32 45 | 36 us, 32/8 heads of
    // 128 bf16 30 | 26, 7 of 181 to 1441 56 | 48, 24 of 60 to 2500, 8/2 heads of 64 59 | 49;
    // of 128, with more tiles than the order matters for, 277 | 280. Each workgroup sorts
    // for itself: 60 sequences cost more (89 | 95).
    a.sort = d->nseq > 1 && d->nseq <= 32 && (uint64_t)d->tokens * a.g > 32ull * d->nseq;
    a.span = std::max(p.own.span, p.together ? p.pre.span : 0);
    if (d->prefix && !p.together) {
      AttnArgs b = a;
      b.k = prefix_k, b.v = prefix_v, b.ks = a.pks, b.vs = a.pvs, b.k_start = nullptr;
      b.rows = d->prefix, b.causal = 0, b.sort = 0;
      b.tiles = p.pre.tiles, b.parts = p.pre.parts, b.shift = p.pre.shift, b.part0 = 0;
      if (int rc = launched("aih_attn", launch_attn(b, AIH_ATTN_ROWS, d->dt, st))) return rc;
    } else {
      a.pre_tiles = p.pre.tiles, a.pre_parts = p.pre.parts, a.pre_shift = p.pre.shift;
    }
    if (int rc = launched("aih_attn", launch_attn(a, p.own.kernel, d->dt, st))) return rc;
    if (!a.ws) return AIH_OK;
    return launched("aih_attn", launch_attn_join(a, d->dt, st));
  });
}
