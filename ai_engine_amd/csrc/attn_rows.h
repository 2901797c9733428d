// attn_rows.h -- attention with a tile's query rows spread over the
// wavefronts and its keys shared (whole prompts, a prefix under many rows).
//
// 128 rows a workgroup: a key row is then read from L2 once per 128 products, and
// a wavefront's 32 x 32 tile of scores leaves the registers for two to four
// wavefronts a SIMD. What bounds it, bf16 or f16: heads of 128 and more the matrix
// instructions (16384 tokens causal, 32/8 heads of 128: 2.0 ms, 1.09 PFLOP/s, where
// a large matrix product reaches 1.12; the clock is down to 1.8 GHz for the power);
// heads of 64 those and the exponentials together (64 x 720 tokens, 8/2 heads: 93
// us, 730 TFLOP/s; vector instructions 66 %, matrix instructions 40 % of the time,
// and hardly any of it at once: taking half of either out saves what they cost).
// fp32 is the matrix instructions (16 x 720 causal, 16/4 heads of 128: 375 us).
#pragma once

#include "attn_impl.h"

namespace aih {
namespace {

// WR wavefronts of 32 rows; stages of SB blocks of 32 keys, two of them in LDS.
//
// JOINT: one softmax for a stage, else one for each block: that leaves the
// registers for four wavefronts a SIMD at 64 16-bit elements (64 x 720 tokens, 8/2
// heads 101 -> 94 us; with 512 workgroups, two a CU anyway, 60 -> 62).
//
// AHEAD: a wavefront's step takes the scores of a block, the softmax of the one
// before and the product of the one before that side by side (at_step). With one
// wavefront a SIMD, at 256 16-bit elements, nothing else runs beside them (4096
// tokens causal, 16/4 heads 202 -> 163 us, 16 x 720 255 -> 214). Smaller heads have
// other wavefronts for that: 128 elements 0 to 8 % slower, 64 0 to 7 %. A stage then
// holds K of blocks SB st + 1 .. SB st + SB and V of blocks SB st - 1 .. SB st + SB
// - 2; a stage of K stands in front, and block -1 of V is zeros.
template <int DT, int DP, int WR_, int SB_, bool AHEAD_, bool JOINT_>
struct AtRowsCfg {
  using T = AtTile<DT, DP>;
  static constexpr bool AHEAD = AHEAD_, JOINT = JOINT_;
  static constexpr int WR = WR_, SB = SB_;
  static constexpr int BM = 32 * WR, KEYS = 32 * SB;
  static constexpr uint32_t HALF = KEYS * T::RB, STAGE = 2 * HALF;
  static constexpr uint32_t LDS = 2 * STAGE;
  static constexpr int NI = KEYS / T::RPI / WR;  // K instructions of a wavefront per stage, and as many of V
  // wavefronts a SIMD that the registers have to leave room for
  static constexpr int WPE = DP <= 64 ? (DT == DT_F32 ? 3 : 4) : DP <= 128 ? 2 : 1;
  static_assert(NI >= 1 && 32 % (NI * T::RPI) == 0, "a wavefront's DMA instructions are of one block");
  static_assert(LDS <= 160 * 1024, "LDS");
};

template <class C>
__global__ __launch_bounds__(64 * C::WR, C::WPE) void attn_rows_kernel(AttnArgs a) {
  using T = typename C::T;
  constexpr int SB = C::SB, DB = T::DB, EB = T::EB;
  extern __shared__ __align__(16) char lds[];

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // The sequences' tiles are counted off 64 sequences at a time, one a lane. The
  // last tiles, which see the most keys under the causal mask, come first.
  // Workgroups go to the XCDs in turn, so eight neighbouring ones take a tile
  // of eight key heads each: an XCD stays with a head, whose keys its L2 keeps,
  // and all XCDs get the same share of long and short tiles (with heads in
  // contiguous ranges of workgroups four heads of a causal prompt, on two XCDs
  // each, took 1.3 times as long: the later half has three times the keys).
  AtSeq s{0, a.tokens, 0, a.rows};  // all rows against the prefix
  uint32_t total = a.tiles, row0 = 0, hk, part;
  AtSeq mine{};
  uint32_t n = 0, sum = 0, base = 0;
  auto count = [&](uint32_t b0) {
    mine = at_load_seq(a, b0 + lane);
    if (a.sort) mine = at_sort(a, mine, lane, false);  // the last come first
    n = (mine.lq * a.g + C::BM - 1) / C::BM;  // tokens * hq is below 2^31
    sum = at_scan(n);
  };
  if (a.k_start) {
    total = 0;
    for (uint32_t b0 = 0; b0 < a.nseq; b0 += 64) {
      count(b0);
      base = total;
      total += __builtin_amdgcn_readlane(sum, 63);
    }
  }
  const uint32_t all = total * a.hkv * a.parts;  // at most the grid
  if (blockIdx.x >= all) return;
  const uint32_t octet = blockIdx.x / (8 * total * a.parts);
  const uint32_t id = blockIdx.x - octet * (8 * total * a.parts), heads = min(8u, a.hkv - 8 * octet);
  const uint32_t rest = id / heads;
  hk = 8 * octet + (id - rest * heads);
  part = rest / total;
  const uint32_t t = total - 1 - (rest - part * total);
  if (a.k_start) {
    if (t < base) {  // not among the last 64 sequences
      base = 0;
      for (uint32_t b0 = 0;; b0 += 64) {
        count(b0);
        const uint32_t here = __builtin_amdgcn_readlane(sum, 63);
        if (t < base + here) break;
        base += here;
      }
    }
    const int l = __ffsll((unsigned long long)__ballot(base + sum > t)) - 1;
    s = at_seq_of(mine, l);
    row0 = (t - base - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l))) * C::BM;
  } else {
    row0 = t * C::BM;
  }
  const uint32_t nrows = s.lq * a.g;

  const uint32_t shift = at_shift(a, s.len);
  const uint64_t kbeg64 = (uint64_t)part << shift;
  const uint32_t kbeg = (uint32_t)min(kbeg64, (uint64_t)s.len);
  const uint32_t kend = (uint32_t)min((uint64_t)at_limit(a, a.causal, s, min(row0 + C::BM, nrows) - 1),
                                      kbeg64 + (1ull << shift));

  const uint32_t kstr = (uint32_t)a.ks * EB, vstr = (uint32_t)a.vs * EB, du = a.d / T::UE;
  const char *kbase = (const char *)a.k + ((uint64_t)s.k0 * a.ks + (uint64_t)hk * a.d) * EB;
  const char *vbase = (const char *)a.v + ((uint64_t)s.k0 * a.vs + (uint64_t)hk * a.d) * EB;
  // From block `at` of the keys on; what is in front of kbeg and behind kend comes
  // as zeros. Keys count from one block before the first (AHEAD: at may be -1).
  constexpr uint32_t F = C::AHEAD ? 32 : 0;
  auto issue = [&](auto v, int32_t at, uint32_t stage) {
    constexpr bool V = decltype(v)::value;
    const uint32_t key = kbeg + 32 * at + F, str = V ? vstr : kstr;
    const bool front = C::AHEAD && 32 * at + (int32_t)(wave * C::NI * T::RPI) < 0;
    const uint32_t rem = !front && key < kend + F ? min(kend + F - key, (uint32_t)C::KEYS) : 0;
    at_dma<T, C::NI, V>((V ? vbase : kbase) - (uint64_t)F * str + (rem ? (uint64_t)key * str : (uint64_t)F * str), str,
                        rem, du, wave * C::NI, lane, lds + (stage & 1) * C::STAGE + (V ? C::HALF : 0));
  };
  constexpr int A = C::AHEAD ? 1 : 0;
  auto issue_k = [&](int32_t st) { issue(std::false_type{}, SB * st + A, st); };
  auto issue_v = [&](int32_t st) { issue(std::true_type{}, SB * st - A, st); };

  issue_k(-A);  // on their way while the rest is set up
  if constexpr (!C::AHEAD) issue_v(0);

  const uint32_t wrow = row0 + wave * 32;
  const uint32_t lim = at_limit(a, a.causal, s, wrow + l32);
  u32x4 q[T::NC];
  const AtQuery<T> src(a, s, hk, wrow, l32);
#pragma unroll
  for (int c = 0; c < T::NC; ++c) q[c] = src.unit(a, 2 * c + lh);
  auto query = [&](int c) __attribute__((always_inline)) { return q[c]; };
  // the first row of a wavefront sees the fewest keys, its last one the most
  const uint32_t wmin = wrow < nrows ? at_limit(a, a.causal, s, wrow) : 0;
  const uint32_t wmax = wrow < nrows ? at_limit(a, a.causal, s, min(wrow + 32, nrows) - 1) : 0;

  f32x16 o[DB];
  float m = kAtLowest, l = 0.0f;
#pragma unroll
  for (int db = 0; db < DB; ++db) o[db] = f32x16{};

  // the product of the block from `key` on, V at vt, where rows may differ in what they see
  auto product = [&](uint32_t key, const char *vt, const typename T::Probs &p) __attribute__((always_inline)) {
    if (key >= min(kend, wmax)) return;  // none of them sees it
    const uint32_t end = min(kend, key + 32);
    if (wmin < end &&
        at_spread_nonfinite<T>(vt, max(wmin, key) - key, end - key, max(min(kend, lim), key) - key, o, lane))
      at_pv<T, true>(vt, p, o, lane);
    else
      at_pv<T, false>(vt, p, o, lane);
  };

  const uint32_t nst = kend > kbeg ? (kend - kbeg + C::KEYS - 1) / C::KEYS : 0;
  const uint32_t whole = min(kend, wmin);  // keys that every row of the wavefront sees
  const uint32_t nfull = whole > kbeg ? (whole - kbeg) / C::KEYS : 0;
  // every wavefront's copies of a stage are in LDS, and every wavefront is done
  // reading the buffers that are requested next. A bare barrier:
  // __syncthreads() would also wait for the copies still in flight.
  auto sync = [&]() { __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };
  f32x16 sc[1];  // AHEAD: the scores of the next block, and the probabilities of the last
  typename T::Probs p[1] = {};
  if constexpr (C::AHEAD) {
    issue_k(0);
    issue_v(0);
    at_wait_vm<2 * C::NI>();
    sync();
    at_qk<T>(lds + C::STAGE + (SB - 1) * 32 * T::RB, query, sc, lane);
  }

  // EDGE: a stage that some of the wavefront's rows see in part, or not at all
  auto turn = [&](uint32_t st, auto edge) __attribute__((always_inline)) {
    constexpr bool EDGE = decltype(edge)::value;
    at_wait_vm<0>();
    sync();
    issue_k(st + 1);
    issue_v(st + 1);
    const char *kt = lds + (st & 1) * C::STAGE, *vt = kt + C::HALF;
    const uint32_t key0 = kbeg + 32 * SB * st;
    if constexpr (!EDGE && C::AHEAD) {
#pragma unroll
      for (int i = 0; i < SB; ++i)
        at_step<T>(kt + i * 32 * T::RB, vt + i * 32 * T::RB, query, sc, p, m, l, o, a.scale_log2, lane);
    } else if constexpr (C::AHEAD) {
#pragma unroll 1
      for (int i = 0; i < SB; ++i, kt += 32 * T::RB, vt += 32 * T::RB) {
        const uint32_t key = key0 + 32 * i;
        if (key > kbeg) {
          if (key - 32 >= min(kend, wmax)) break;  // neither this block nor the one before is seen
          product(key - 32, vt, p[0]);
        }
        at_mask(sc[0], max(min(kend, lim), key) - key, lane);
        f32x16 next[1];
        at_qk<T>(kt, query, next, lane);
        at_softmax<T>(sc, p, m, l, o, a.scale_log2);
        sc[0] = next[0];
      }
    } else if constexpr (EDGE && !C::JOINT) {
#pragma unroll 1
      for (int i = 0; i < SB; ++i, kt += 32 * T::RB, vt += 32 * T::RB) {
        const uint32_t key = key0 + 32 * i;
        if (key >= min(kend, wmax)) break;
        f32x16 s[1];
        typename T::Probs pi[1];
        at_qk<T>(kt, query, s, lane);
        at_mask(s[0], max(min(kend, lim), key) - key, lane);
        at_softmax<T>(s, pi, m, l, o, a.scale_log2);
        product(key, vt, pi[0]);
      }
    } else {
      if (EDGE && key0 >= min(kend, wmax)) return;
      constexpr int N = C::JOINT ? SB : 1;  // blocks of a softmax
      f32x16 s[SB / N][N];
      if constexpr (N == SB) {
        at_qk<T>(kt, query, s[0], lane);
      } else {
#pragma unroll
        for (int i = 0; i < SB; ++i) at_qk<T>(kt + i * 32 * T::RB, query, s[i], lane);
      }
#pragma unroll
      for (int i = 0; i < SB / N; ++i) {
        typename T::Probs pi[N];
        if constexpr (EDGE) {
#pragma unroll
          for (int j = 0; j < N; ++j) {
            const uint32_t key = key0 + 32 * (i * N + j);
            at_mask(s[i][j], max(min(kend, lim), key) - key, lane);
          }
        }
        at_softmax<T>(s[i], pi, m, l, o, a.scale_log2);
#pragma unroll
        for (int j = 0; j < N; ++j) {
          const char *t = vt + (i * N + j) * 32 * T::RB;
          if constexpr (EDGE) product(key0 + 32 * (i * N + j), t, pi[j]);
          else at_pv<T, false>(t, pi[j], o, lane);
        }
      }
    }
  };
  // Every wavefront takes nst turns, some of them with other rows' stages whole
  // and its own at the edge: the loop is cut in two per wavefront, the barriers
  // are the same.
  uint32_t st = 0;
  for (; st < nfull; ++st) turn(st, std::false_type{});
  for (; st < nst; ++st) turn(st, std::true_type{});
  at_wait_vm<0>();  // nothing may still be on its way into LDS at the end
  if constexpr (C::AHEAD) {
    sync();
    const uint32_t last = kbeg + 32 * (SB * nst - 1);
    if (nst) product(last, lds + (nst & 1) * C::STAGE + C::HALF, p[0]);
  }

  const uint64_t rows_all = (uint64_t)a.tokens * a.hq;
  const uint64_t ml0 = attn_ws_ml(a);
  const float lsum = at_pair_sum(l);
  const uint32_t row = wrow + l32;
  const bool on = row < nrows;
  const uint32_t tok = fdiv(row, a.by_g), hd = hk * a.g + (row - tok * a.g);
  if (a.ws) {
    if (!on) return;
    const uint64_t r = (uint64_t)(a.part0 + part) * rows_all + (uint64_t)(s.q0 + tok) * a.hq + hd;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const uint32_t dim = 32 * db + 8 * r4 + 4 * lh;
        if (dim < a.d)
          *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim) =
              f32x4{o[db][4 * r4], o[db][4 * r4 + 1], o[db][4 * r4 + 2], o[db][4 * r4 + 3]};
      }
    if (lh == 0) {
      a.ws[ml0 + 2 * r] = m;
      a.ws[ml0 + 2 * r + 1] = lsum;
    }
    return;
  }
  const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
  const uint64_t e = (uint64_t)(s.q0 + tok) * a.os + (uint64_t)hd * a.d;
#pragma unroll
  for (int db = 0; db < DB; ++db) {
    f32x4 x[4];
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4)
      x[r4] = f32x4{o[db][4 * r4], o[db][4 * r4 + 1], o[db][4 * r4 + 2], o[db][4 * r4 + 3]} * inv;
    if constexpr (T::F32) {
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const uint32_t dim = 32 * db + 8 * r4 + 4 * lh;
        if (on && dim < a.d) *reinterpret_cast<f32x4 *>((float *)a.o + e + dim) = x[r4];
      }
    } else {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        // two runs of 4 dims in either half -> one run of 8 a lane
        const u32x2 x0 = pack4<T::DT>(x[2 * k]), x1 = pack4<T::DT>(x[2 * k + 1]);
        const auto sx = __builtin_amdgcn_permlane32_swap(x0.x, x1.x, false, false);
        const auto sy = __builtin_amdgcn_permlane32_swap(x0.y, x1.y, false, false);
        const uint32_t dim = 32 * db + 8 * (2 * k + lh);
        if (on && dim < a.d)
          *reinterpret_cast<u32x4 *>((uint16_t *)a.o + e + dim) = u32x4{sx[0], sy[0], sx[1], sy[1]};
      }
    }
  }
}

template <class C>
hipError_t at_launch_rows(const AttnArgs &a, hipStream_t st) {
  const uint64_t grid = (uint64_t)a.hkv * a.parts * a.tiles;
  if (grid == 0 || grid > 0x7fffffffu) return hipErrorInvalidValue;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(attn_rows_kernel<C>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL((attn_rows_kernel<C>), dim3((uint32_t)grid), dim3(64 * C::WR), C::LDS, st, a);
  return hipGetLastError();
}

// The heads of more than 128 fp32 elements leave no registers for this kernel.
template <int DT, int DP>
constexpr bool kAtRowsFit = DP * Storage<DT>::bytes <= 512;
// Stages of 64 keys, or of 32 where two of 64 leave no room: fp32 heads above 64
// elements (at 256 16-bit elements 64 keys beat 32 by 2 to 7 %, one workgroup a
// CU either way).
template <int DT, int DP>
using AtRows = AtRowsCfg<DT, DP, 4, (DT == DT_F32 && DP > 64) ? 1 : 2, DT != DT_F32 && (DP > 128), DT != DT_F32 && DP != 64>;

}  // namespace
}  // namespace aih
