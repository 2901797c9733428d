// attn_rows.h -- attention with a tile's query rows spread over the
// wavefronts and its keys shared (whole prompts, a prefix under many rows).
#pragma once

#include "attn_impl.h"

namespace aih {
namespace {

// WR wavefronts of 32 NQ rows; stages of 32 KB keys, two of them in LDS.
template <int DT, int DP, int WR_, int NQ, int KB>
struct AtRowsCfg {
  using T = AtTile<DT, DP, NQ, KB>;
  static constexpr int WR = WR_;
  static constexpr int BM = 32 * NQ * WR;
  static constexpr uint32_t HALF = T::KEYS * T::RB, STAGE = 2 * HALF;
  static constexpr uint32_t LDS = 2 * STAGE;
  static constexpr int NI = T::KEYS / T::RPI / WR;  // K instructions of a wavefront per stage, and as many of V
  // wavefronts a SIMD that the registers have to leave room for
  static constexpr int WPE = DP <= 64 ? 3 : DP <= 128 ? 2 : 1;
  static_assert(NI >= 1, "DMA instructions");
  static_assert(LDS <= 160 * 1024, "LDS");
};

template <class C>
__global__ __launch_bounds__(64 * C::WR, C::WPE) void attn_rows_kernel(AttnArgs a) {
  using T = typename C::T;
  constexpr int NQ = T::NQ, DB = T::DB, EB = T::EB;
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
  auto issue = [&](uint32_t st, uint32_t b) {
    const uint32_t key = kbeg + st * T::KEYS;
    const uint32_t rem = key < kend ? min(kend - key, (uint32_t)T::KEYS) : 0;
    char *dst = lds + b * C::STAGE;
    at_dma<T, C::NI, false>(kbase + (rem ? (uint64_t)key * kstr : 0), kstr, rem, du, wave * C::NI, lane, dst);
    at_dma<T, C::NI, true>(vbase + (rem ? (uint64_t)key * vstr : 0), vstr, rem, du, wave * C::NI, lane, dst + C::HALF);
  };

  issue(0, 0);  // on its way while the rest is set up

  const uint32_t wrow = row0 + wave * 32 * NQ;
  uint32_t lim[NQ];
  u32x4 q[NQ][T::NC];
  const AtQuery<T> src(a, s, hk, wrow, l32);
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    lim[i] = at_limit(a, a.causal, s, wrow + 32 * i + l32);
#pragma unroll
    for (int c = 0; c < T::NC; ++c) q[i][c] = src.unit(a, i, 2 * c + lh);
  }
  // the first row of a wavefront sees the fewest keys, its last one the most
  const uint32_t wmin = wrow < nrows ? at_limit(a, a.causal, s, wrow) : 0;
  const uint32_t wmax = wrow < nrows ? at_limit(a, a.causal, s, min(wrow + 32 * NQ, nrows) - 1) : 0;

  f32x16 o[DB][NQ];
  float m[NQ], l[NQ];
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    m[i] = kAtLowest;
    l[i] = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db][i] = f32x16{};
  }

  // EDGE: a stage that some of the wavefront's rows see in part, or not at all
  auto compute = [&](uint32_t st, uint32_t b, auto edge) {
    constexpr bool EDGE = decltype(edge)::value;
    const uint32_t key = kbeg + st * T::KEYS;
    if (EDGE && key >= min(kend, wmax)) return;
    const char *kt = lds + b * C::STAGE, *vt = kt + C::HALF;
    f32x16 sc[T::KB][NQ];
    u32x4 pb[T::KB][2][NQ];
    at_qk<T>(kt, [&](int i, int c) { return q[i][c]; }, sc, lane);
    if constexpr (EDGE) {
      uint32_t to[NQ];
#pragma unroll
      for (int i = 0; i < NQ; ++i) to[i] = max(min(kend, lim[i]), key) - key;
      at_mask<T>(sc, to, lane);
      at_softmax<T>(sc, pb, m, l, o, a.scale_log2);
      const uint32_t end = min(kend, key + T::KEYS);
      if (wmin < end && at_spread_nonfinite<T>(vt, max(wmin, key) - key, end - key, to, o, lane)) {
        at_pv<T, true>(vt, sc, pb, o, lane);
        return;
      }
    } else {
      at_softmax<T>(sc, pb, m, l, o, a.scale_log2);
    }
    at_pv<T, false>(vt, sc, pb, o, lane);
  };

  const uint32_t nst = kend > kbeg ? (kend - kbeg + T::KEYS - 1) / T::KEYS : 0;
  const uint32_t whole = min(kend, wmin);  // keys that every row of the wavefront sees
  const uint32_t nfull = whole > kbeg ? (whole - kbeg) / T::KEYS : 0;
  // Every wavefront takes nst turns, some of them with other rows' stages whole
  // and its own at the edge: the loop is cut in two per wavefront, the barriers
  // are the same.
  uint32_t st = 0;
  auto turn = [&](auto edge) {
    // every wavefront's copies of the stage are in LDS, and every wavefront is
    // done reading the buffer that is requested next. A bare barrier:
    // __syncthreads() would also wait for the copies still in flight.
    at_wait_vm<0>();
    __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    issue(st + 1, (st + 1) & 1);
    compute(st, st & 1, edge);
  };
  for (; st < nfull; ++st) turn(std::false_type{});
  for (; st < nst; ++st) turn(std::true_type{});
  at_wait_vm<0>();  // nothing may still be on its way into LDS at the end

  const uint64_t rows_all = (uint64_t)a.tokens * a.hq;
  const uint64_t ml0 = attn_ws_ml(a);
#pragma unroll
  for (int i = 0; i < NQ; ++i) {
    const float lsum = at_pair_sum(l[i]);
    const uint32_t row = wrow + 32 * i + l32;
    const bool on = row < nrows;
    const uint32_t tok = fdiv(row, a.by_g), hd = hk * a.g + (row - tok * a.g);
    if (a.ws) {
      if (!on) continue;
      const uint64_t r = (uint64_t)(a.part0 + part) * rows_all + (uint64_t)(s.q0 + tok) * a.hq + hd;
#pragma unroll
      for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const uint32_t dim = 32 * db + 8 * r4 + 4 * lh;
          if (dim < a.d)
            *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim) =
                f32x4{o[db][i][4 * r4], o[db][i][4 * r4 + 1], o[db][i][4 * r4 + 2], o[db][i][4 * r4 + 3]};
        }
      if (lh == 0) {
        a.ws[ml0 + 2 * r] = m[i];
        a.ws[ml0 + 2 * r + 1] = lsum;
      }
      continue;
    }
    const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
    const uint64_t e = (uint64_t)(s.q0 + tok) * a.os + (uint64_t)hd * a.d;
#pragma unroll
    for (int db = 0; db < DB; ++db) {
      f32x4 x[4];
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        x[r4] = f32x4{o[db][i][4 * r4], o[db][i][4 * r4 + 1], o[db][i][4 * r4 + 2], o[db][i][4 * r4 + 3]} * inv;
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
using AtRows = AtRowsCfg<DT, DP, 4, 1, (DT == DT_F32 && DP > 64) ? 1 : 2>;

}  // namespace
}  // namespace aih
