// attn_keys.h -- attention of 32 query rows with the keys spread over the
// wavefronts: one or a few tokens per sequence over a long cache, a prefix under
// few rows, prompts of few tiles.
//
// A single token's g rows fill g of a tile's 32 columns; the products are cheap
// beside the keys and values that are read once for them, so that serving is bound
// by memory: 64 sequences of up to 8192 keys, 32/8 bf16 heads of 128, 82 us at 4.3
// TB/s, one of 131071 keys 58 us at 4.6 (a large copy reaches 4.76, a large sum
// 4.0). Short calls are a chain of launch, first keys, softmax and join (180 fp32
// keys: 8.8 us, 3 of them launch to launch), a short prefix that of its stages, 64 KB
// that a CU takes 1 us to bring from L2 into LDS, by one workgroup or two (64 tokens
// behind 4096 keys, 32/8 heads of 128: 22.4 us). fp32 prompts run at 80
// TFLOP/s where a matrix product reaches 154 (7 of 181 to 1441 tokens, 8/4 heads of
// 96: 117 us; matrix instructions 62 % of the time).
#pragma once

#include "attn_impl.h"

namespace aih {
namespace {

// WK wavefronts, each with its own 32 keys of a stage in LDS. One buffer for
// K and one for V: K's is free again after the scores, V's after the product,
// so the next stage's K arrives during the softmax and the product, its V
// during the next scores. ONE: the two take turns in one buffer, where LDS would
// otherwise hold one wavefront a SIMD: fp32 heads above 64 elements, whose long
// products of one wavefront cover the waits and the softmax of another.
template <int DT, int DP, int WK_>
struct AtKeysCfg {
  using T = AtTile<DT, DP>;
  static constexpr int WK = WK_;
  static constexpr int KEYS = 32 * WK;
  static constexpr bool ONE = T::RB >= 512 && T::F32;
  static constexpr uint32_t HALF = 32 * T::RB;   // K or V of a wavefront
  static constexpr uint32_t MINE = ONE ? HALF : 2 * HALF;
  static constexpr int NI = 32 / T::RPI;         // DMA instructions of a half
  static constexpr int OPITCH = DP + 4;
  // the join of the wavefronts' results reuses the buffers
  static constexpr uint32_t JOIN = WK * 32u * OPITCH * 4 + WK * 64u * 4;
  static constexpr uint32_t BUF = WK * MINE;
  // then also the queries are in LDS: the registers hold the results
  static constexpr bool QL = ONE;
  static constexpr uint32_t LDS = BUF + (QL ? HALF : 0) > JOIN ? BUF + (QL ? HALF : 0) : JOIN;
  // wavefronts of a SIMD that LDS has room for
  static constexpr int WPE = WK == 8 || 2 * LDS <= 160 * 1024 ? 2 : 1;
  static_assert(NI >= 1 && NI < 64, "DMA instructions in flight");
};

// Work items: first the prefix's (part, row tile, key head), then sequence by
// sequence (part, row tile, key head): neighbours stream neighbouring heads of
// the same rows. A workgroup takes one, or (MANY) every gridDim.x-th.
template <class C, bool MANY>
__global__ __launch_bounds__(64 * C::WK, C::WPE) void attn_keys_kernel(AttnArgs a) {
  using T = typename C::T;
  constexpr int WK = C::WK, DB = T::DB, EB = T::EB, DP = T::DP;
  extern __shared__ __align__(16) char lds[];

  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  char *kt = lds + wave * C::MINE, *vt = C::ONE ? kt : kt + C::HALF;

  // 64 sequences at a time, one a lane: items up to and including each
  const uint32_t pre_items = a.pre_tiles * a.pre_parts * a.hkv;
  AtSeq mine{};
  uint32_t b0 = 0, base = pre_items, n = 0, sum = 0, tiles = 0, parts = 0;
  auto count = [&]() {
    mine = at_load_seq(a, b0 + (threadIdx.x & 63));
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
    // the lane's offsets are worked out again for every item: kept over the
    // loop they would not fit the registers
    if constexpr (MANY) __asm__ volatile("" : "+v"(tid));
    const int lane = tid & 63, l32 = lane & 31, lh = lane >> 5;
    AtSeq s;
    const char *kp, *vp;
    uint64_t ks, vs;
    uint32_t hk, part, tile, shift, causal, nparts, gpart;
    if (item < pre_items) {  // all rows against the prefix
      s = AtSeq{0, a.tokens, 0, a.prefix};
      const uint32_t rest = fdiv(item, a.by_hkv);
      hk = item - rest * a.hkv;
      part = fdiv(rest, a.by_pre_tiles), tile = rest - part * a.pre_tiles;
      shift = a.pre_shift, causal = 0, nparts = a.pre_parts, gpart = part;
      kp = (const char *)a.pk, vp = (const char *)a.pv, ks = a.pks, vs = a.pvs;
    } else {
      for (;;) {
        const uint32_t here = __builtin_amdgcn_readlane(sum, 63);
        if (item < base + here) break;
        if (b0 + 64 >= a.nseq) return;  // the same for the whole workgroup
        base += here;
        b0 += 64;
        count();
      }
      const int l = __ffsll((unsigned long long)__ballot(base + sum > item)) - 1;
      s = at_seq_of(mine, l);
      const uint32_t nt = __builtin_amdgcn_readlane(tiles, l);
      nparts = __builtin_amdgcn_readlane(parts, l);
      const uint32_t at = item - base - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l));
      const uint32_t rest = fdiv(at, a.by_hkv);
      hk = at - rest * a.hkv;
      part = nt == 1 ? rest : rest / nt;
      tile = nt - 1 - (rest - part * nt);  // the last rows see the most keys: they go first
      shift = at_shift(a, s.len);
      causal = a.causal, gpart = a.part0 + part;
      kp = (const char *)a.k, vp = (const char *)a.v, ks = a.ks, vs = a.vs;
    }
    const uint32_t nrows = s.lq * a.g, row0 = tile * 32;
    const uint32_t rlast = min(row0 + 32, nrows) - 1;
    const uint32_t kbeg = part << shift;  // below len, or 0
    const uint32_t smax = at_limit(a, causal, s, rlast), smin = at_limit(a, causal, s, row0);
    const uint32_t kend = (uint32_t)min((uint64_t)smax, (uint64_t)kbeg + (1ull << shift));

    const uint32_t kstr = (uint32_t)ks * EB, vstr = (uint32_t)vs * EB, du = a.d / T::UE;
    const char *kbase = kp + ((uint64_t)s.k0 * ks + (uint64_t)hk * a.d) * EB;
    const char *vbase = vp + ((uint64_t)s.k0 * vs + (uint64_t)hk * a.d) * EB;
    auto rows_of = [&](uint32_t key) { return key < kend ? min(kend - key, 32u) : 0; };
    auto issue_k = [&](uint32_t key) {
      const uint32_t rem = rows_of(key);
      at_dma<T, C::NI, false>(kbase + (rem ? (uint64_t)key * kstr : 0), kstr, rem, du, 0, lane, kt);
    };
    auto issue_v = [&](uint32_t key) {
      const uint32_t rem = rows_of(key);
      at_dma<T, C::NI, true>(vbase + (rem ? (uint64_t)key * vstr : 0), vstr, rem, du, 0, lane, vt);
    };

    uint32_t key = kbeg + wave * 32;
    issue_k(key);
    if constexpr (!C::ONE) issue_v(key);
    u32x4 q[C::QL ? 1 : T::NC];
    char *ql = lds + C::BUF + l32 * T::RB;
    const AtQuery<T> src(a, s, hk, row0, l32);
    if constexpr (C::QL) {  // row l32 in LDS as a row of K, the wavefronts sharing the units
#pragma unroll 4
      for (int c = wave; c < T::NC; c += WK)
        *reinterpret_cast<u32x4 *>(ql + (((2 * c + lh) ^ at_kswz<T>(l32)) * 16)) = src.unit(a, 2 * c + lh);
      __syncthreads();
    } else {
      // The compiler waits for these in the loop, in the scores, and with that for
      // V. A wait of its own in front of the loop makes prompts 3 % and a prefix 2 %
      // faster and decode steps 2 to 5 % slower (16 x 1024 keys 13.9 -> 14.6 us).
#pragma unroll
      for (int c = 0; c < T::NC; ++c) q[c] = src.unit(a, 2 * c + lh);
    }
    auto query = [&](int c) -> u32x4 {
      if constexpr (C::QL) return *reinterpret_cast<const u32x4 *>(ql + (((2 * c + lh) ^ at_kswz<T>(l32)) * 16));
      else return q[c];
    };
    const uint32_t lim = at_limit(a, causal, s, row0 + l32);

    f32x16 o[DB];
    float m = kAtLowest, l = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db] = f32x16{};

    for (; key < kend; key += C::KEYS) {
      at_wait_vm<C::ONE ? 0 : C::NI>();  // K is there, V may still be on its way
      __asm__ volatile("" ::: "memory");
      f32x16 sc[1];
      typename T::Probs p[1];
      at_qk<T>(kt, query, sc, lane);
      // K's buffer is requested again: its reads are behind this wavefront
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if constexpr (C::ONE) issue_v(key);
      else issue_k(key + C::KEYS);
      const uint32_t to = max(min(kend, lim), key) - key;
      if (key + 32 > min(kend, smin)) at_mask(sc[0], to, lane);
      at_softmax<T>(sc, p, m, l, o, a.scale_log2);
      at_wait_vm<C::ONE ? 0 : C::NI>();  // V is there, the next K on its way
      __asm__ volatile("" ::: "memory");
      const uint32_t end = min(kend, key + 32);
      if (smin < end && at_spread_nonfinite<T>(vt, max(smin, key) - key, end - key, to, o, lane))
        at_pv<T, true>(vt, p[0], o, lane);
      else
        at_pv<T, false>(vt, p[0], o, lane);
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      if constexpr (C::ONE) issue_k(key + C::KEYS);
      else issue_v(key + C::KEYS);
    }
    at_wait_vm<0>();  // nothing is on its way into LDS any more
    l = at_pair_sum(l);

    // join the wavefronts' keys: a common maximum, scaled sums through LDS
    float *jo = reinterpret_cast<float *>(lds);
    float *jml = jo + WK * 32 * C::OPITCH;
    __syncthreads();
    if (lh == 0) {
      jml[wave * 64 + l32] = m;
      jml[wave * 64 + 32 + l32] = l;
    }
    __syncthreads();
    float mm = jml[l32];
#pragma unroll
    for (int w = 1; w < WK; ++w) mm = fmaxf(mm, jml[w * 64 + l32]);
    const float f = __builtin_amdgcn_exp2f(m - mm);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        *reinterpret_cast<f32x4 *>(jo + (wave * 32 + l32) * C::OPITCH + 32 * db + 8 * r4 + 4 * lh) =
            f32x4{o[db][4 * r4], o[db][4 * r4 + 1], o[db][4 * r4 + 2], o[db][4 * r4 + 3]} * f;
    __syncthreads();
    const uint64_t rows_all = (uint64_t)a.tokens * a.hq;
    const uint64_t ml0 = attn_ws_ml(a);
    // rows whose keys are all in this part need no join with others
    const bool direct = !a.ws || (nparts == 1 && a.part0 == 0);
    for (uint32_t i = tid; i < 32 * (DP / 8); i += 64 * WK) {
      const uint32_t rr = i / (DP / 8), dim = (i - rr * (DP / 8)) * 8;
      const uint32_t row = row0 + rr;
      if (row >= nrows || dim >= a.d) continue;
      f32x4 x0{}, x1{};
      float mr = jml[rr], lr = 0.0f;
#pragma unroll
      for (int w = 1; w < WK; ++w) mr = fmaxf(mr, jml[w * 64 + rr]);
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float *p = jo + (w * 32 + rr) * C::OPITCH + dim;
        x0 += *reinterpret_cast<const f32x4 *>(p);
        x1 += *reinterpret_cast<const f32x4 *>(p + 4);
        lr += jml[w * 64 + 32 + rr] * __builtin_amdgcn_exp2f(jml[w * 64 + rr] - mr);
      }
      const uint32_t tok = fdiv(row, a.by_g), hd = hk * a.g + (row - tok * a.g);
      const uint64_t r0 = (uint64_t)(s.q0 + tok) * a.hq + hd;
      if (!direct) {
        const uint64_t r = (uint64_t)gpart * rows_all + r0;
        *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim) = x0;
        *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim + 4) = x1;
        if (dim == 0) {
          a.ws[ml0 + 2 * r] = mr;
          a.ws[ml0 + 2 * r + 1] = lr;
          if (item >= pre_items && part == 0)  // parts that this sequence does not have
            for (uint32_t p = nparts; p < a.parts; ++p) {
              a.ws[ml0 + 2 * ((uint64_t)(a.part0 + p) * rows_all + r0)] = kAtLowest;
              a.ws[ml0 + 2 * ((uint64_t)(a.part0 + p) * rows_all + r0) + 1] = 0.0f;
            }
        }
      } else {
        if (a.ws && dim == 0) a.ws[ml0 + 2 * r0 + 1] = -1.0f;  // nothing to join
        const float inv = lr == 0.0f ? 0.0f : 1.0f / lr;
        x0 *= inv, x1 *= inv;
        const uint64_t e = (uint64_t)(s.q0 + tok) * a.os + (uint64_t)hd * a.d + dim;
        if constexpr (T::F32) {
          *reinterpret_cast<f32x4 *>((float *)a.o + e) = x0;
          *reinterpret_cast<f32x4 *>((float *)a.o + e + 4) = x1;
        } else {
          const u32x2 p0 = pack4<T::DT>(x0), p1 = pack4<T::DT>(x1);
          *reinterpret_cast<u32x4 *>((uint16_t *)a.o + e) = u32x4{p0.x, p0.y, p1.x, p1.y};
        }
      }
    }
    if constexpr (!MANY) return;
    __syncthreads();  // the next item's copies go where the results were read
  }
}

template <class C, bool MANY>
hipError_t at_launch_items(const AttnArgs &a, uint64_t items, uint32_t cus, hipStream_t st) {
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(attn_keys_kernel<C, MANY>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (attr != hipSuccess) return attr;
  if constexpr (MANY) {
    // workgroups of a CU that run at once
    static const int occ = [] {
      int v = 0;
      if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, reinterpret_cast<const void *>(attn_keys_kernel<C, MANY>),
                                                       64 * C::WK, C::LDS) != hipSuccess || v < 1)
        v = 1;
      return v;
    }();
    if (items > (uint64_t)cus * occ) items = (uint64_t)cus * occ;
  }
  hipLaunchKernelGGL((attn_keys_kernel<C, MANY>), dim3((uint32_t)items), dim3(64 * C::WK), C::LDS, st, a);
  return hipGetLastError();
}

// Uncut keys: one item a workgroup, handed out as others end. Cut ones: the
// items are many, and of those that the host counts (the longest length for
// all) few may exist, so the workgroups that run at once share them. fp32 heads above
// 64 elements whose items leave every CU at most one take eight wavefronts, if the
// keys are more than four take at once: long products of two wavefronts a SIMD fill
// each other's waits (24 x 130 keys, 32/8 heads of 128 17.4 -> 15.7 us, 24 x 750 46 -> 39;
// others are too short for the larger join: 180 keys, heads of 64 8.9 -> 9.8).
template <int DT, int DP>
hipError_t at_launch_keys(const AttnArgs &a, uint32_t cus, hipStream_t st) {
  using C = AtKeysCfg<DT, DP, 4>;
  static_assert(C::LDS <= 160 * 1024, "LDS");
  const uint64_t items = (uint64_t)a.hkv * a.parts * a.tiles + (uint64_t)a.hkv * a.pre_parts * a.pre_tiles;
  if (items == 0 || items > 0x7fffffffu) return hipErrorInvalidValue;
  if (a.parts > 1 && items > cus) return at_launch_items<C, true>(a, items, cus, st);
  if constexpr (C::ONE) {
    using C8 = AtKeysCfg<DT, DP, 8>;
    if constexpr (C8::LDS <= 160 * 1024)
      if (items <= cus && a.span > C::KEYS) return at_launch_items<C8, false>(a, items, cus, st);
  }
  return at_launch_items<C, false>(a, items, cus, st);
}

}  // namespace
}  // namespace aih
