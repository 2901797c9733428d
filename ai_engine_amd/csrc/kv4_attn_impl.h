// kv4_attn_impl.h -- attention over a 4-bit paged cache (aih_kv4_attn).
//
// The products, softmax and order of a tile are attn_impl.h's: S^T = K Q^T with 32
// keys and 32 (query, head of the group) rows, O^T += V^T P^T. A code times its
// scale has two significant bits, so it is exact in bf16, and the matrix
// instructions run in bf16 for every type: fp32 queries and probabilities are
// taken as three bf16 terms, which hold all their 24 bits, f16 ones as two
// (all 11 bits of a query, 16 of a probability), whose products are summed in fp32.
//
// A lane holds a key's codes as they lie in the cache: 16 bytes are one block,
// whose elements are the operands of four products after conversion, so K goes
// from memory to the matrix unit without LDS. V has to be transposed: its blocks
// are converted into a bf16 tile in LDS that transposing reads take. The keys are
// spread over the wavefronts, which run without barriers until their results are
// joined; the next keys' codes are on their way meanwhile.
#pragma once

#include "attn_impl.h"
#include "mx4.h"

namespace aih {
namespace {

// x as N bf16 terms that add up to it (three hold fp32's 24 bits): each takes the
// leading bits of what is left.
template <int N>
__device__ __forceinline__ void kv_terms(float x, float (&t)[N]) {
  float rest = x;
#pragma unroll
  for (int i = 0; i < N; ++i) {
    t[i] = __uint_as_float(__float_as_uint(rest) & 0xffff0000u);
    rest -= t[i];
  }
}
// two bf16 of floats whose low halves do not count
__device__ __forceinline__ uint32_t kv_pack(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// Four dwords of bf16: eight codes times their scale.
__device__ __forceinline__ u32x4 kv_decode8(uint32_t c, float s) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
}

__device__ __forceinline__ f32x16 kv_mfma(u32x4 a, u32x4 b, f32x16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

template <int DT_, int DP_, int WK_>
struct KvCfg {
  static constexpr int DT = DT_, DP = DP_, WK = WK_;
  static constexpr int NT = DT == DT_F32 ? 3 : DT == DT_F16 ? 2 : 1;  // terms
  using TQ = AtTile<DT, DP>;                                          // of the queries as stored
  using TV = AtTile<DT_BF16, DP>;                                     // of V in LDS
  using TS = AtTile<NT == 1 ? DT_BF16 : DT_F32, DP>;                  // of the softmax
  static constexpr int NB = DP / 32, DB = DP / 32;                    // blocks of a head
  static constexpr int NP = NB / 2;                                   // whole blocks of a lane (half h: 2 p + h)
  static constexpr bool ODD = NB % 2;                                 // the last one shared by the halves
  static constexpr int NS = 2 * NB;                                   // products of 16 elements
  static constexpr int KEYS = 32 * WK;
  static constexpr uint32_t VT = 32 * TV::RB;                         // V of a wavefront
  // queries that the registers do not hold go to LDS
  static constexpr bool QL = NT * DP > 384;
  static constexpr uint32_t QB = QL ? NT * NS * 1024 : 0;
  static constexpr int JD = DP < 64 ? DP : 64, JP = JD + 4;           // dims of a pass of the join
  static constexpr uint32_t JOIN = WK * 32u * JP * 4;
  static constexpr uint32_t ML = WK * 64u * 4;
  static constexpr uint32_t BUF = WK * VT + QB > JOIN ? WK * VT + QB : JOIN;
  static constexpr uint32_t LDS = BUF + ML;
  static constexpr int WPE = DP <= 128 && NT < 3 ? 2 : 1;             // wavefronts of a SIMD
  static_assert(LDS <= 160 * 1024, "LDS");
};

// The unit of 8 elements of a row that a lane half takes in product s.
template <class C>
__device__ __forceinline__ uint32_t kv_unit(int s, uint32_t lh) {
  return C::ODD && s >= 4 * C::NP ? 4 * (C::NB - 1) + 2 * lh + (s - 4 * C::NP) : 4 * (2 * (s / 4) + lh) + s % 4;
}

// The codes and scales of 32 keys on their way: of K a lane's part of key
// lane % 32, of V block i % NB of a key for every i = lane + 64 n.
template <class C>
struct KvLoad {
  static constexpr int NV = (32 * C::NB + 63) / 64;  // V blocks of a lane
  u32x4 k[C::NP > 0 ? C::NP : 1], v[NV];
  u32x2 ko;
  uint32_t ks[C::NP + 1], vs[NV];
  uint32_t seen;  // bit j: key j is there
};

// The key and block of V that lane's n-th load is, and the LDS row and first unit
// they go to. The lanes of a group of 16, whose stores share a cycle, take rows
// whose swizzles differ (for 4 blocks a row).
template <class C>
__device__ __forceinline__ void kv_v_place(int n, uint32_t lane, uint32_t &key, uint32_t &block) {
  const uint32_t i = lane + 64 * n;
  block = i % C::NB;
  key = i / C::NB;
}
// LDS slot of unit u of row r; as at_vswz in its high bits, which the transposing
// reads need
template <class C>
__device__ __forceinline__ uint32_t kv_swz(uint32_t r) {
  return at_vswz<typename C::TV>(r);
}

// Sequence b's rows and keys, cut to the tensors and the table.
__device__ __forceinline__ AtSeq kv_load_seq(const Kv4AttnArgs &a, uint32_t b) {
  AtSeq s{0, 0, 0, 0};
  if (b < a.at.nseq) {
    s.q0 = min((uint32_t)max(a.at.q_start[b], 0), a.at.tokens);
    const uint32_t q1 = min((uint32_t)max(a.at.q_start[b + 1], 0), a.at.tokens);
    s.lq = q1 > s.q0 ? q1 - s.q0 : 0;
    s.k0 = b;  // its row of the table
    s.len = min((uint32_t)max(a.at.k_len[b], 0), a.at.rows);
  }
  return s;
}

template <class C, bool MANY>
__global__ __launch_bounds__(64 * C::WK, C::WPE) void kv4_attn_kernel(Kv4AttnArgs ka) {
  using TV = typename C::TV;
  using TS = typename C::TS;
  using TQ = typename C::TQ;
  constexpr int WK = C::WK, DB = C::DB, NB = C::NB, NP = C::NP, NS = C::NS, NT = C::NT, DP = C::DP, EB = TQ::EB;
  constexpr int NV = KvLoad<C>::NV;
  const AttnArgs &a = ka.at;
  extern __shared__ __align__(16) char lds[];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char *vt = lds + wave * C::VT, *ql = lds + WK * C::VT;
  float *jml = reinterpret_cast<float *>(lds + C::BUF);

  // 64 sequences at a time, one a lane: items up to and including each
  AtSeq mine{};
  uint32_t b0 = 0, base = 0, n = 0, sum = 0, tiles = 0, parts = 0;
  auto count = [&]() {
    mine = kv_load_seq(ka, b0 + (threadIdx.x & 63));
    if (a.sort) mine = at_sort(a, mine, threadIdx.x & 63, true);
    tiles = (mine.lq * a.g + 31) / 32;
    const uint32_t x = at_shift(a, mine.len);
    parts = max(1u, (uint32_t)(((uint64_t)mine.len + (1ull << x) - 1) >> x));
    n = tiles * parts * a.hkv;
    sum = at_scan(n);
  };
  count();

  for (uint32_t item = blockIdx.x;; item += gridDim.x) {
    int tid = threadIdx.x;
    if constexpr (MANY) __asm__ volatile("" : "+v"(tid));  // offsets are worked out again for every item
    const int lane = tid & 63, l32 = lane & 31, lh = lane >> 5;
    for (;;) {
      const uint32_t here = __builtin_amdgcn_readlane(sum, 63);
      if (item < base + here) break;
      if (b0 + 64 >= a.nseq) return;  // the same for the whole workgroup
      base += here;
      b0 += 64;
      count();
    }
    const int sl = __ffsll((unsigned long long)__ballot(base + sum > item)) - 1;
    const AtSeq s = at_seq_of(mine, sl);
    const uint32_t nt = __builtin_amdgcn_readlane(tiles, sl), nparts = __builtin_amdgcn_readlane(parts, sl);
    const uint32_t at = item - base - (__builtin_amdgcn_readlane(sum, sl) - __builtin_amdgcn_readlane(n, sl));
    const uint32_t rest = fdiv(at, a.by_hkv), hk = at - rest * a.hkv;
    const uint32_t part = nt == 1 ? rest : rest / nt;
    const uint32_t tile = nt - 1 - (rest - part * nt);  // the last rows see the most keys: they go first
    const uint32_t shift = at_shift(a, s.len);
    const uint32_t nrows = s.lq * a.g, row0 = tile * 32;
    const uint32_t kbeg = part << shift;  // below len, or 0
    const uint32_t smax = at_limit(a, a.causal, s, min(row0 + 32, nrows) - 1);
    const uint32_t kend = (uint32_t)min((uint64_t)smax, (uint64_t)kbeg + (1ull << shift));

    const uint32_t nb = a.d / 32, pmask = (1u << ka.pshift) - 1;
    const int32_t *table = ka.table + (uint64_t)s.k0 * ka.width;
    // the page of the lane's key; -1: no such key
    auto page_of = [&](uint32_t key) {
      const uint32_t kk = key + l32;
      const uint32_t p = (uint32_t)table[min(kk, max(kend, 1u) - 1) >> ka.pshift];
      return kk < kend && p < ka.pages ? (int32_t)p : -1;
    };
    // every lane loads, those without a key from the cache's first row
    auto load = [&](KvLoad<C> &x, uint32_t key, int32_t page) {
      x.seen = (uint32_t)__ballot(page >= 0);
      const uint64_t row = page < 0 ? 0 : (((uint64_t)(uint32_t)page * a.hkv + hk) << ka.pshift) | ((key + l32) & pmask);
      const uint8_t *c = ka.kc + row * (a.d / 2), *sc = ka.ks + row * nb;
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const uint32_t b = 2 * p + lh, bb = DP > 128 && b >= nb ? 0 : b;
        x.k[p] = *reinterpret_cast<const u32x4 *>(c + bb * 16);
        x.ks[p] = sc[bb];
      }
      if constexpr (C::ODD) {
        x.ko = *reinterpret_cast<const u32x2 *>(c + (NB - 1) * 16 + lh * 8);
        x.ks[NP] = sc[NB - 1];
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        uint32_t j, b;
        kv_v_place<C>(i, lane, j, b);
        const bool on = (NB % 2 == 0 || j < 32) && (DP <= 128 || b < nb);
        const int32_t vp = __shfl(page, j & 31);
        const uint64_t vrow = vp < 0 || !on ? 0 : (((uint64_t)(uint32_t)vp * a.hkv + hk) << ka.pshift) | ((key + j) & pmask);
        const uint32_t vb = on ? b : 0;
        x.v[i] = *reinterpret_cast<const u32x4 *>(ka.vc + vrow * (a.d / 2) + vb * 16);
        x.vs[i] = ka.vs[vrow * nb + vb];
      }
    };

    uint32_t key = kbeg + wave * 32;
    KvLoad<C> cur, nxt;
    int32_t page1 = -1;
    if (kend > 0) {  // else there may be no cache
      const int32_t page = page_of(key);
      page1 = page_of(key + C::KEYS);
      load(cur, key, page);
    }

    // the queries as bf16 terms
    u32x4 q[C::QL ? 1 : NT][C::QL ? 1 : NS];
    const AtQuery<TQ> src(a, s, hk, row0, l32);
#pragma unroll
    for (int st = 0; st < NS; ++st) {
      if (C::QL && st % WK != wave) continue;
      const uint32_t u = kv_unit<C>(st, lh);
      u32x4 out[NT];
      if constexpr (NT == 1) {
        out[0] = src.unit(a, u);
      } else {
        float f[8];
        if constexpr (TQ::F32) {
          const u32x4 x0 = src.unit(a, 2 * u), x1 = src.unit(a, 2 * u + 1);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = __uint_as_float(e < 4 ? x0[e] : x1[e % 4]);
        } else {
          const u32x4 x0 = src.unit(a, u);
#pragma unroll
          for (int e = 0; e < 8; ++e) f[e] = f16_to_f32((x0[e / 2] >> (16 * (e & 1))) & 0xffffu);
        }
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
          float t0[NT], t1[NT];
          kv_terms(f[e], t0), kv_terms(f[e + 1], t1);
          // of infinity and NaN the first term is the value and the others nothing
          const bool n0 = !(__builtin_fabsf(f[e]) < __builtin_huge_valf()), n1 = !(__builtin_fabsf(f[e + 1]) < __builtin_huge_valf());
          if (n0) t0[0] = f[e] == f[e] ? f[e] : __uint_as_float(0x7fc00000u);
          if (n1) t1[0] = f[e + 1] == f[e + 1] ? f[e + 1] : __uint_as_float(0x7fc00000u);
#pragma unroll
          for (int t = 0; t < NT; ++t) out[t][e / 2] = kv_pack(t > 0 && n0 ? 0.0f : t0[t], t > 0 && n1 ? 0.0f : t1[t]);
        }
      }
#pragma unroll
      for (int t = 0; t < NT; ++t) {
        if constexpr (C::QL) *reinterpret_cast<u32x4 *>(ql + (t * NS + st) * 1024 + lane * 16) = out[t];
        else q[t][st] = out[t];
      }
    }
    if constexpr (C::QL) __syncthreads();
    const uint32_t lim = at_limit(a, a.causal, s, row0 + l32);

    f32x16 o[DB];
    float m = kAtLowest, l = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};

    for (; key < kend; key += C::KEYS) {
      const int32_t page2 = page_of(key + 2 * C::KEYS);
      load(nxt, key + C::KEYS, page1);

      // scores
      f32x16 sc[1];
      sc[0] = f32x16{};
      auto product = [&](int st, uint32_t codes, float scale) __attribute__((always_inline)) {
        const u32x4 k = kv_decode8(codes, scale);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          u32x4 qt;
          if constexpr (C::QL) qt = *reinterpret_cast<const u32x4 *>(ql + (t * NS + st) * 1024 + lane * 16);
          else qt = q[t][st];
          sc[0] = kv_mfma(k, qt, sc[0]);
        }
      };
#pragma unroll
      for (int p = 0; p < NP; ++p) {
        const bool on = DP <= 128 || 2 * p + lh < nb;
        const float scale = mx4_scale(on ? cur.ks[p] : 127u);
#pragma unroll
        for (int e = 0; e < 4; ++e) product(4 * p + e, on ? cur.k[p][e] : 0u, scale);
      }
      if constexpr (C::ODD) {
        const float scale = mx4_scale(cur.ks[NP]);
        product(4 * NP, cur.ko.x, scale), product(4 * NP + 1, cur.ko.y, scale);
      }

      // V into LDS; blocks that are NaN as zeros, to be added to the rows that see them
      uint64_t bad[NV];
      bool any_bad = false;
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        uint32_t j, b;
        kv_v_place<C>(i, lane, j, b);
        const bool in = NB % 2 == 0 || j < 32;
        const bool there = in && (DP <= 128 || b < nb) && (cur.seen >> (j & 31) & 1);
        const bool nan = there && cur.vs[i] > 252;
        bad[i] = __ballot(nan);
        any_bad |= bad[i] != 0;
        const bool on = there && !nan;
        const float scale = mx4_scale(on ? cur.vs[i] : 127u);
        if (in) {
          char *to = vt + j * TV::RB;
          const uint32_t sw = kv_swz<C>(j);
#pragma unroll
          for (int e = 0; e < 4; ++e)
            *reinterpret_cast<u32x4 *>(to + ((4 * b + e) ^ sw) * 16) = kv_decode8(on ? cur.v[i][e] : 0u, scale);
        }
      }

      // the keys that this lane's row sees
      const uint32_t to = max(min(kend, lim), key) - key;
      const uint32_t vis = cur.seen & (to >= 32 ? 0xffffffffu : (1u << to) - 1);
      if (__any(vis != 0xffffffffu)) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (!(vis >> (8 * (r / 4) + r % 4 + 4 * lh) & 1)) sc[0][r] = -__builtin_huge_valf();
      }
      typename TS::Probs p[1];
      at_softmax<TS>(sc, p, m, l, o, a.scale_log2);

      if (any_bad) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
          for (uint64_t left = bad[i]; left; left &= left - 1) {
            uint32_t j, b;
            kv_v_place<C>(i, __builtin_ctzll(left), j, b);
            const float x = vis >> j & 1 ? __uint_as_float(0x7fc00000u) : 0.0f;
#pragma unroll
            for (int db = 0; db < DB; ++db)
              if (db == (int)b) {
#pragma unroll
                for (int r = 0; r < 16; ++r) o[db][r] += x;
              }
          }
      }

      // probabilities as bf16 terms of 16 keys each
      u32x4 pt[NT][2];
      if constexpr (NT == 1) {
        pt[0][0] = p[0].h[0], pt[0][1] = p[0].h[1];
      } else {
#pragma unroll
        for (int w = 0; w < 8; ++w) {
          float t0[NT], t1[NT];
          kv_terms(p[0][2 * w], t0), kv_terms(p[0][2 * w + 1], t1);
#pragma unroll
          for (int t = 0; t < NT; ++t) pt[t][w / 4][w % 4] = kv_pack(t0[t], t1[t]);
        }
      }
      // O^T += V^T P^T: a transposing read has 16 lanes read 4 rows x 16 columns, 8 bytes each
      // (row lane / 4, columns 4 (lane % 4) ..), and lane i gets column i
      const uint32_t vr = 4 * lh + ((lane & 15) >> 2), vsw = kv_swz<C>(vr);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int db = 0; db < DB; ++db) {
          const uint32_t unit = (4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vsw;
          const char *pv = vt + (16 * h + vr) * TV::RB + unit * 16 + (lane & 1) * 8;
          const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)pv);
          const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)(pv + 8 * TV::RB));
          const u32x4 v = __builtin_bit_cast(u32x4, s16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
#pragma unroll
          for (int t = 0; t < NT; ++t) o[db] = kv_mfma(v, pt[t][h], o[db]);
        }
      cur = nxt;
      page1 = page2;
    }
    l = at_pair_sum(l);

    // join the wavefronts' keys: a common maximum, scaled sums through LDS, JD dims at a time
    if (lh == 0) {
      jml[wave * 64 + l32] = m;
      jml[wave * 64 + 32 + l32] = l;
    }
    __syncthreads();  // and all are done with V and the queries
    float mm = jml[l32];
#pragma unroll
    for (int w = 1; w < WK; ++w) mm = fmaxf(mm, jml[w * 64 + l32]);
    const float f = __builtin_amdgcn_exp2f(m - mm);
    float *jo = reinterpret_cast<float *>(lds);
    const uint64_t rows_all = (uint64_t)a.tokens * a.hq, ml0 = attn_ws_ml(a);
    const bool direct = !a.ws || nparts == 1;
#pragma unroll
    for (int d0 = 0; d0 < DP; d0 += C::JD) {
      if (d0) __syncthreads();
#pragma unroll
      for (int db = d0 / 32; db < (d0 + C::JD) / 32 && db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          *reinterpret_cast<f32x4 *>(jo + (wave * 32 + l32) * C::JP + 32 * db - d0 + 8 * r4 + 4 * lh) =
              f32x4{o[db][4 * r4], o[db][4 * r4 + 1], o[db][4 * r4 + 2], o[db][4 * r4 + 3]} * f;
      __syncthreads();
      constexpr int UR = C::JD / 8;
      for (uint32_t i = tid; i < 32 * UR; i += 64 * WK) {
        const uint32_t rr = i / UR, dj = (i - rr * UR) * 8, dim = d0 + dj, row = row0 + rr;
        if (row >= nrows || dim >= a.d) continue;
        f32x4 x0{}, x1{};
        float mr = jml[rr], lr = 0.0f;
#pragma unroll
        for (int w = 1; w < WK; ++w) mr = fmaxf(mr, jml[w * 64 + rr]);
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float *jp = jo + (w * 32 + rr) * C::JP + dj;
          x0 += *reinterpret_cast<const f32x4 *>(jp);
          x1 += *reinterpret_cast<const f32x4 *>(jp + 4);
          lr += jml[w * 64 + 32 + rr] * __builtin_amdgcn_exp2f(jml[w * 64 + rr] - mr);
        }
        const uint32_t tok = fdiv(row, a.by_g), hd = hk * a.g + (row - tok * a.g);
        const uint64_t r0 = (uint64_t)(s.q0 + tok) * a.hq + hd;
        if (!direct) {
          const uint64_t r = (uint64_t)part * rows_all + r0;
          *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim) = x0;
          *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim + 4) = x1;
          if (dim == 0) {
            a.ws[ml0 + 2 * r] = mr;
            a.ws[ml0 + 2 * r + 1] = lr;
            if (part == 0)  // parts that this sequence does not have
              for (uint32_t pp = nparts; pp < a.parts; ++pp) {
                a.ws[ml0 + 2 * ((uint64_t)pp * rows_all + r0)] = kAtLowest;
                a.ws[ml0 + 2 * ((uint64_t)pp * rows_all + r0) + 1] = 0.0f;
              }
          }
        } else {
          if (a.ws && dim == 0) a.ws[ml0 + 2 * r0 + 1] = -1.0f;  // nothing to join
          const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
          x0 *= inv, x1 *= inv;
          const uint64_t e = (uint64_t)(s.q0 + tok) * a.os + (uint64_t)hd * a.d + dim;
          if constexpr (TQ::F32) {
            *reinterpret_cast<f32x4 *>((float *)a.o + e) = x0;
            *reinterpret_cast<f32x4 *>((float *)a.o + e + 4) = x1;
          } else {
            const u32x2 p0 = pack4<C::DT>(x0), p1 = pack4<C::DT>(x1);
            *reinterpret_cast<u32x4 *>((uint16_t *)a.o + e) = u32x4{p0.x, p0.y, p1.x, p1.y};
          }
        }
      }
    }
    if constexpr (!MANY) return;
    __syncthreads();  // the next item's tiles go where the results were read
  }
}

template <class C, bool MANY>
hipError_t kv_launch_items(const Kv4AttnArgs &a, uint64_t items, uint32_t cus, hipStream_t st) {
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(kv4_attn_kernel<C, MANY>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (attr != hipSuccess) return attr;
  if constexpr (MANY) {
    // workgroups of a CU that run at once
    static const int occ = [] {
      int v = 0;
      if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, reinterpret_cast<const void *>(kv4_attn_kernel<C, MANY>),
                                                       64 * C::WK, C::LDS) != hipSuccess || v < 1)
        v = 1;
      return v;
    }();
    if (items > (uint64_t)cus * occ) items = (uint64_t)cus * occ;
  }
  hipLaunchKernelGGL((kv4_attn_kernel<C, MANY>), dim3((uint32_t)items), dim3(64 * C::WK), C::LDS, st, a);
  return hipGetLastError();
}

// Uncut keys: one item a workgroup, handed out as others end. Cut ones: of the items
// that the host counts (the longest length for all) few may exist, so the
// workgroups that run at once share them.
template <int DT, int DP>
hipError_t kv_launch(const Kv4AttnArgs &a, hipStream_t st) {
  using C = KvCfg<DT, DP, 4>;
  const uint32_t cus = device_cus();
  const uint64_t items = (uint64_t)a.at.hkv * a.at.parts * a.at.tiles;
  if (items == 0 || items > 0x7fffffffu) return hipErrorInvalidValue;
  if (a.at.parts > 1 && items > cus) return kv_launch_items<C, true>(a, items, cus, st);
  return kv_launch_items<C, false>(a, items, cus, st);
}

template <int DT>
hipError_t kv_launch_dt(const Kv4AttnArgs &a, hipStream_t st) {
  if (a.at.d == 32) return kv_launch<DT, 32>(a, st);
  if (a.at.d == 64) return kv_launch<DT, 64>(a, st);
  if (a.at.d == 96) return kv_launch<DT, 96>(a, st);
  if (a.at.d == 128) return kv_launch<DT, 128>(a, st);
  return kv_launch<DT, 256>(a, st);
}

}  // namespace
}  // namespace aih
