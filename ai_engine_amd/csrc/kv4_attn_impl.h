// kv4_attn_impl.h -- attention over a 4-bit paged cache (aih_kv4_attn).
//
// A code times its scale has two significant bits, so keys and values are exact in
// bf16, and the matrix instructions run in bf16 for every type: fp32 queries and
// probabilities are taken as three bf16 terms, which hold all their 24 bits, f16
// ones as two (all 11 bits of a query, 16 of a probability), whose products are
// summed in fp32. bf16 probabilities are rounded to bf16, and their sum is of the rounded
// ones, so that the roundings cancel where one key has most of it: results are off by 2.3e-3
// (four prompts behind 2000 keys) and 1.4e-3 (64 tokens over 0 to 8192), by 1.7e-3 and
// 1.3e-3, which is their own rounding, with a second term, for 160 us instead of 136 and 36.8
// instead of 31.3.
//
// As in attn_impl.h the scores are S^T = K Q^T and the result O^T += V^T P^T, here
// with 16x16x32 instructions and 16 RB (query, head of the group) rows a
// workgroup: a single token's g rows fill most of 16, and a lane's share of the
// softmax, which vector instructions do, is half of a 32-row tile's. A lane of a
// score block holds keys 4 g + 0..3 (g = lane / 16) of one row, of the two blocks
// of a step together what the second product takes as its operand.
//
// 16 keys are always in one page. Of them lane l holds key l % 16, and its quarter
// g of every block's codes (or block 4 i + g of four): the order of the elements inside
// a product is free, and the queries follow it. K goes from memory to the matrix
// unit without LDS; V is converted into a bf16 tile in LDS that transposing reads
// take. The keys are spread over the wavefronts, 32 a step, which run without
// barriers until their results are joined. A step's registers are requested again
// as soon as they are converted, so the next codes are on their way during the rest
// of it.
//
// Single tokens are bound by memory between a start and an end: 64 sequences of 0 to 8192
// keys, 32/8 bf16 heads of 128, 23.7 us and 4.2 to join their parts (94 MB: 18.4 us at a
// large copy's 5.1 TB/s), one of 131071 keys, 16/4 f16 heads of 128, 19.8 and 4.7 (71 MB:
// 14). The first loads (lengths, table, codes) follow each other, 3 us. With 32x32x16
// products, whose tile a token's rows fill an eighth of, and addresses of each lane's own
// it was 38 and 28. Prompts are bound by vector instructions (conversions, softmax) and
// matrix instructions in turn: four behind 2000 keys, 87 GFLOP, 136 us, 640 TFLOP/s,
// where a large matrix product reaches 1220.
#pragma once

#include "attn_impl.h"
#include "mx4.h"

namespace aih {
namespace {

// x as N bf16 terms that add up to it (three hold fp32's 24 bits): each takes the
// leading bits of what is left. The last one is cut by kv_pack.
template <int N>
__device__ __forceinline__ void kv_terms(float x, float (&t)[N]) {
#pragma unroll
  for (int i = 0; i < N - 1; ++i) {
    t[i] = __uint_as_float(__float_as_uint(x) & 0xffff0000u);
    x -= t[i];
  }
  t[N - 1] = x;
}
// two bf16 of floats, cut
__device__ __forceinline__ uint32_t kv_pack(float lo, float hi) {
  return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
}

// Eight codes times their scale.
__device__ __forceinline__ u32x4 kv_decode8(uint32_t c, float s) {
  return u32x4{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 0)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 1)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 2)),
               __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, s, 3))};
}

__device__ __forceinline__ f32x4 kv_mfma(u32x4 a, u32x4 b, f32x4 c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// over the four lanes that hold a row (l % 16)
__device__ __forceinline__ float kv_row_max(float x) {
  x = at_pair_max(x);
  const uint32_t u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float kv_row_sum(float x) {
  x = at_pair_sum(x);
  const uint32_t u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Heads of at most 32 NB elements, 16 RB rows, WK wavefronts.
template <int DT_, int NB_, int RB_, int WK_>
struct KvCfg {
  static constexpr int DT = DT_, NB = NB_, RB = RB_, WK = WK_;
  static constexpr int NT = DT == DT_F32 ? 3 : DT == DT_F16 ? 2 : 1;  // terms
  static constexpr int DP = 32 * NB, TR = 16 * RB;
  static constexpr bool EXACT = NB <= 4;                              // d is 32 NB, else it may be less
  static constexpr int SETS = NB / 4, REST = NB % 4;                  // blocks in fours, and the others
  static constexpr int KEYS = 32 * WK;
  static constexpr int PU = NB == 1 ? 4 : NB == 2 ? 8 : NB <= 4 ? 16 : 32;  // 16-byte units of an LDS row
  static constexpr uint32_t VT = 32 * PU * 16;                        // V of a wavefront
  static constexpr int JD = DP < 64 || RB > 2 ? 32 : 64, JP = JD + 4;  // dims of a pass of the join
  static constexpr uint32_t JOIN = WK * TR * JP * 4u;
  static constexpr uint32_t ML = WK * 2u * TR * 4u;
  // queries that the registers do not hold go to LDS
  static constexpr bool QL = NT * NB * RB > (RB > 2 ? 8 : 24);
  static constexpr uint32_t QB = QL ? NT * NB * RB * 1024u : 0;
  static constexpr uint32_t BUF = WK * VT + QB > JOIN ? WK * VT + QB : JOIN;
  static constexpr uint32_t LDS = BUF + ML;
  static_assert(LDS <= 160 * 1024, "LDS");
  // registers that a wavefront cannot do without: queries, results, scores, probabilities, codes
  static constexpr int NEED = (QL ? 0 : 4 * NT * NB * RB) + 8 * NB * RB + 8 * RB + 4 * NT * RB + 5 * NB;
  // wavefronts of a SIMD: a few registers that spill cost less than one of them. One | two, where the
  // limits decide (us; 64 rows: 4 x 1000 tokens behind 500 keys, 32/8 heads; 32 rows: 8 x 500 behind 500,
  // 8/2 heads; 16 rows: 64 tokens over 1000, 16/4 heads): 64 rows of 128 bf16 177 | 112, f16 229 | 163,
  // fp32 285 | 373, of 96 fp32 245 | 168; 32 rows of 256 bf16 88 | 118, f16 111 | 133, of 128 fp32 75.6 | 56.1
  // (which the limits miss); 16 rows of 256 fp32 28.5 | 37.7. Two | four, 16 rows: one workgroup a CU, 128 bf16 12.2
  // | 14.3; several, 64 tokens over 0 to 8192 keys, 32.8 | 32.4; one of 131071 keys, 128 f16, 23.5 | 32.5
  static constexpr int WPE = NEED <= 80 && 4 * LDS <= 160 * 1024 ? 4 : NEED <= (NT == 3 ? 195 : 215) && 2 * LDS <= 160 * 1024 ? 2 : 1;
};

// Product s of a head's: where a lane group's eight elements are. Sets of four
// blocks: block 4 i + g, dword s % 4 of it; of two blocks left over, block g / 2;
// of one, dword g.
template <class C>
struct KvPlace {
  // 16-byte unit of the values (8 elements)
  static __device__ __forceinline__ uint32_t unit(int s, uint32_t g) {
    if (s < 4 * C::SETS) return 4 * (4 * (s / 4) + g) + s % 4;
    const int r = s - 4 * C::SETS;
    if (C::REST >= 2 && r < 2) return 4 * (4 * C::SETS + (g >> 1)) + 2 * (g & 1) + r;
    return 4 * (C::NB - 1) + g;
  }
};

// The codes and scales of 16 keys, as a lane holds them.
template <class C>
struct KvCodes {
  u32x4 w[C::SETS > 0 ? C::SETS : 1];
  u32x2 two;
  uint32_t one;
  uint32_t sw[C::SETS > 0 ? C::SETS : 1], s2, s1;
  // codes: the first of the 16 keys' rows of d / 2 bytes, scales theirs of nb bytes
  __device__ __forceinline__ void load(const uint8_t *codes, const uint8_t *scales, uint32_t row, uint32_t g, uint32_t nb) {
    const uint32_t cb = C::EXACT ? C::NB * 16 : nb * 16, sb = C::EXACT ? C::NB : nb;
    const uint32_t co = row * cb, so = row * sb;
    auto at = [&](uint32_t b) { return C::EXACT || b < nb ? b : 0u; };  // blocks past the head: read something
#pragma unroll
    for (int i = 0; i < C::SETS; ++i) {
      const uint32_t b = at(4 * i + g);
      w[i] = *reinterpret_cast<const u32x4 *>(codes + (co + b * 16));
      sw[i] = scales[so + b];
    }
    if constexpr (C::REST >= 2) {
      const uint32_t b = at(4 * C::SETS + (g >> 1));
      two = *reinterpret_cast<const u32x2 *>(codes + (co + b * 16 + (g & 1) * 8));
      s2 = scales[so + b];
    }
    if constexpr (C::REST & 1) {
      one = *reinterpret_cast<const uint32_t *>(codes + (co + (C::NB - 1) * 16 + g * 4));
      s1 = scales[so + C::NB - 1];
    }
  }
  // the eight codes of product s
  __device__ __forceinline__ uint32_t code(int s) const {
    if (s < 4 * C::SETS) return w[s / 4][s % 4];
    const int r = s - 4 * C::SETS;
    if (C::REST >= 2 && r < 2) return two[r];
    return one;
  }
  __device__ __forceinline__ uint32_t scale(int s) const {
    if (s < 4 * C::SETS) return sw[s / 4];
    return C::REST >= 2 && s - 4 * C::SETS < 2 ? s2 : s1;
  }
  // the block of product s
  static __device__ __forceinline__ uint32_t block(int s, uint32_t g) { return KvPlace<C>::unit(s, g) / 4; }
  // nothing, where the key is not to count or the head has no such block
  __device__ __forceinline__ void clear(bool all, uint32_t g, uint32_t nb) {
#pragma unroll
    for (int i = 0; i < C::SETS; ++i)
      if (all || (!C::EXACT && 4 * i + g >= nb)) w[i] = u32x4{}, sw[i] = 127;
    if constexpr (C::REST >= 2)
      if (all || (!C::EXACT && 4 * C::SETS + (g >> 1) >= nb)) two = u32x2{}, s2 = 127;
    if constexpr (C::REST & 1)
      if (all) one = 0, s1 = 127;
  }
  // scale bytes that the product does not take: of NaN, and those below `less`
  static __device__ __forceinline__ bool odd(uint32_t byte, uint32_t less) { return byte - less > 252 - less; }
  __device__ __forceinline__ void clear_odd(uint32_t less) {
#pragma unroll
    for (int i = 0; i < C::SETS; ++i)
      if (odd(sw[i], less)) w[i] = u32x4{}, sw[i] = 127;
    if constexpr (C::REST >= 2)
      if (odd(s2, less)) two = u32x2{}, s2 = 127;
    if constexpr (C::REST & 1)
      if (odd(s1, less)) one = 0, s1 = 127;
  }
  // whether one of the blocks has such a scale
  __device__ __forceinline__ bool odd(uint32_t less) const {
    bool x = false;
#pragma unroll
    for (int i = 0; i < C::SETS; ++i) x |= odd(sw[i], less);
    if constexpr (C::REST >= 2) x |= odd(s2, less);
    if constexpr (C::REST & 1) x |= odd(s1, less);
    return x;
  }
  // whether one of the blocks is NaN
  __device__ __forceinline__ bool nan() const {
    bool x = false;
#pragma unroll
    for (int i = 0; i < C::SETS; ++i) x |= sw[i] > 252;
    if constexpr (C::REST >= 2) x |= s2 > 252;
    if constexpr (C::REST & 1) x |= s1 > 252;
    return x;
  }
};

// LDS slot of unit u of row r: u ^ kv_swz(r). A cycle serves 256 bytes. 16 lanes store one unit of
// 16 rows each, which land in 16 different groups of 4 banks; 32 lanes of a
// transposing read take two units of 8 rows (r / 4 even and odd).
template <class C>
__device__ __forceinline__ uint32_t kv_swz(uint32_t r) {
  if constexpr (C::PU >= 16) return (r & 3) << 2 | (r >> 1 & 2) | (r >> 3 & 1);
  else if constexpr (C::PU == 8) return (r >> 1 & 3) << 1 | (r >> 3 & 1);
  else return (r >> 1 & 2) | (r >> 3 & 1);
}

// Scores of 8 keys -> probabilities as the product's operands; returns their sum.
template <int NT>
__device__ __forceinline__ float kv_probs(const float (&s)[8], u32x4 (&pt)[NT], float off, float scale) {
  float sum = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * w], scale, off));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[2 * w + 1], scale, off));
    if constexpr (NT == 1) {
      const uint32_t x = pack2<DT_BF16>(p0, p1);
      pt[0][w] = x;
      sum = at_dot_ones<DT_BF16>(x, sum);
    } else {
      float t0[NT], t1[NT];
      kv_terms(p0, t0), kv_terms(p1, t1);
#pragma unroll
      for (int t = 0; t < NT; ++t) pt[t][w] = kv_pack(t0[t], t1[t]);
      sum += p0 + p1;
    }
  }
  return sum;
}

// The probabilities of a lane and step, 8 keys, from which a row's maximum is found anew.
constexpr float kKvMost = 256.0f;

// Values reach 6 * 2^125, a third below fp32's largest number, and sums of them times
// probabilities must not leave its range where the mean does not. A row's probabilities add
// up to at most kKvMost / 8 for each key (in whole steps of 32): values are taken 2^-kv_less
// times as large, which costs nothing (their scales are made with one add), and the sum of the
// probabilities too, at the end. What becomes less than the format's smallest scale is read as
// zero: values below 6 * 2^(kv_less - 127), 2^-102 with 131072 keys.
__device__ __forceinline__ uint32_t kv_less(uint32_t keys) { return 32 - __builtin_clz(max(keys, 32u) - 1) + 5; }

// The softmax of a step: as at_settle, the maximum of a row is left as it is until
// its probabilities add up to kKvMost, and found then.
template <class C>
__device__ __forceinline__ void kv_softmax(float (&s)[8], u32x4 (&pt)[C::NT], float &m, float &l, f32x4 (&o)[2 * C::NB],
                                           float scale) {
#pragma clang fp contract(off)
  float sum = kv_probs<C::NT>(s, pt, -m, scale);
  const bool far0 = __builtin_fabsf(m) >= kAtFar, big = !(sum < kKvMost) || far0;
  if (__any(big)) {
    const bool row = kv_row_max(big ? 1.0f : 0.0f) != 0.0f;
    float mx = s[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) mx = fmaxf(mx, s[i]);
    mx = kv_row_max(mx) * scale;
    const float mn = row ? fmaxf(m, mx) : m, al = __builtin_amdgcn_exp2f(m - mn);
    m = mn;
    l *= al;
#pragma unroll
    for (int i = 0; i < 2 * C::NB; ++i) o[i] *= al;
    float off = -m;
    const bool far = __builtin_fabsf(m) >= kAtFar;  // see at_far
    if (__any(far)) {
      off = far ? 0.0f : off;
      const float inv = __builtin_amdgcn_rcpf(scale);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float at = s[i] * scale;
        s[i] = far ? (at - m) * inv : s[i];
      }
    }
    sum = kv_probs<C::NT>(s, pt, off, scale);
  }
  l += sum;
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

// 8 elements of a query row, unit u, as the terms of an operand.
template <class C>
__device__ __forceinline__ void kv_query(const AttnArgs &a, const AtQuery<AtTile<C::DT, 32>> &src, uint32_t u, u32x4 (&out)[C::NT]) {
  constexpr int NT = C::NT;
  if constexpr (NT == 1) {
    out[0] = src.unit(a, u);
  } else {
    float f[8];
    if constexpr (C::DT == DT_F32) {
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
      float t[2][NT];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float x = f[e + i];
        kv_terms(x, t[i]);
        // of infinity and NaN the first term is the value and the others nothing
        if (!(__builtin_fabsf(x) < __builtin_huge_valf())) {
          t[i][0] = x == x ? x : __uint_as_float(0x7fc00000u);
#pragma unroll
          for (int k = 1; k < NT; ++k) t[i][k] = 0.0f;
        }
      }
#pragma unroll
      for (int k = 0; k < NT; ++k) out[k][e / 2] = kv_pack(t[0][k], t[1][k]);
    }
  }
}

// Work items: sequence by sequence (part, row tile, key head). A workgroup takes
// every gridDim.x-th.
template <class C>
__global__ __launch_bounds__(64 * C::WK, C::WPE) void kv4_attn_kernel(Kv4AttnArgs ka) {
  constexpr int WK = C::WK, NB = C::NB, NT = C::NT, RB = C::RB, DP = C::DP, TR = C::TR;
  constexpr uint32_t RW = C::PU * 16;  // bytes of an LDS row
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
    tiles = (mine.lq * a.g + TR - 1) / TR;
    const uint32_t x = at_shift(a, mine.len);
    parts = max(1u, (uint32_t)(((uint64_t)mine.len + (1ull << x) - 1) >> x));
    n = tiles * parts * a.hkv;
    sum = at_scan(n);
  };
  count();

  for (uint32_t item = blockIdx.x;; item += gridDim.x) {
    int tid = threadIdx.x;
    __asm__ volatile("" : "+v"(tid));  // offsets are worked out again for every item: they would fill the registers
    const int lane = tid & 63, l16 = lane & 15, g = lane >> 4;
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
    const uint32_t rest = __builtin_amdgcn_readfirstlane(fdiv(at, a.by_hkv)), hk = at - rest * a.hkv;
    const uint32_t part = nt == 1 ? rest : rest / nt;
    const uint32_t tile = nt - 1 - (rest - part * nt);  // the last rows see the most keys: they go first
    const uint32_t shift = at_shift(a, s.len);
    const uint32_t nrows = s.lq * a.g, row0 = tile * TR;
    const uint32_t kbeg = part << shift;  // below len, or 0
    const uint32_t smax = at_limit(a, a.causal, s, min(row0 + TR, nrows) - 1);
    const uint32_t kend = __builtin_amdgcn_readfirstlane((uint32_t)min((uint64_t)smax, (uint64_t)kbeg + (1ull << shift)));

    const uint32_t less = kv_less(s.len);
    const uint32_t nb = a.d / 32, pmask = (1u << ka.pshift) - 1;
    const int32_t *table = ka.table + (uint64_t)s.k0 * ka.width;
    // the pages of keys key .. key + 15 and the next 16, in lanes 0 and 1
    auto pages_of = [&](uint32_t key) { return (uint32_t)table[min(key + 16 * (lane & 1), kend - 1) >> ka.pshift]; };
    // Which of a step's keys are there: bit j for key j.
    auto there = [&](uint32_t key, uint32_t p0, uint32_t p1) {
      const uint32_t left = key < kend ? min(kend - key, 32u) : 0;
      uint32_t x = left == 32 ? 0xffffffffu : (1u << left) - 1;
      if (p0 >= ka.pages) x &= 0xffff0000u;
      if (p1 >= ka.pages) x &= 0x0000ffffu;
      return x;
    };
    // the first of 16 keys' rows in the cache; where there are none, the cache's own first
    auto row_of = [&](uint32_t key, uint32_t page) -> uint64_t {
      if (key >= kend || page >= ka.pages) return 0;
      return (((uint64_t)page * a.hkv + hk) << ka.pshift) + (key & pmask);
    };
    KvCodes<C> kx[2], vx[2];
    auto load = [&](KvCodes<C> &x, const uint8_t *codes, const uint8_t *scales, uint64_t row) {
      x.load(codes + row * (C::EXACT ? NB * 16 : nb * 16), scales + row * (C::EXACT ? NB : nb), l16, g, nb);
    };

    uint32_t key = kbeg + wave * 32, p0 = 0xffffffffu, p1 = 0xffffffffu, pn = 0;
    if (kend > 0) {  // else there may be no cache
      const uint32_t pv = pages_of(key);
      pn = pages_of(key + C::KEYS);
      p0 = __builtin_amdgcn_readlane(pv, 0), p1 = __builtin_amdgcn_readlane(pv, 1);
      const uint64_t r0 = row_of(key, p0), r1 = row_of(key + 16, p1);
      load(kx[0], ka.kc, ka.ks, r0), load(kx[1], ka.kc, ka.ks, r1);
      load(vx[0], ka.vc, ka.vs, r0), load(vx[1], ka.vc, ka.vs, r1);
    }

    // the queries
    u32x4 q[C::QL ? 1 : RB][C::QL ? 1 : NB][C::QL ? 1 : NT];
    uint32_t lim[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      const AtQuery<AtTile<C::DT, 32>> src(a, s, hk, row0, 16 * rb + l16);
      lim[rb] = at_limit(a, a.causal, s, row0 + 16 * rb + l16);
#pragma unroll
      for (int st = 0; st < NB; ++st) {
        if (C::QL && (rb * NB + st) % WK != wave) continue;
        u32x4 out[NT];
        kv_query<C>(a, src, KvPlace<C>::unit(st, g), out);
#pragma unroll
        for (int t = 0; t < NT; ++t) {
          if constexpr (C::QL) *reinterpret_cast<u32x4 *>(ql + ((rb * NB + st) * NT + t) * 1024 + lane * 16) = out[t];
          else q[rb][st][t] = out[t];
        }
      }
    }
    if constexpr (C::QL) __syncthreads();

    f32x4 o[RB][2 * NB];
    float m[RB], l[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      m[rb] = kAtLowest, l[rb] = 0.0f;
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) o[rb][i] = f32x4{};
    }

    for (; key < kend; key += C::KEYS) {
      const uint32_t seen = there(key, p0, p1);
      const uint32_t n0 = __builtin_amdgcn_readlane(pn, 0), n1 = __builtin_amdgcn_readlane(pn, 1);
      const uint64_t r0 = row_of(key + C::KEYS, n0), r1 = row_of(key + C::KEYS + 16, n1);
      pn = pages_of(key + 2 * C::KEYS);

      // scores
      f32x4 sc[RB][2];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) sc[rb][0] = sc[rb][1] = f32x4{};
      if constexpr (!C::EXACT) kx[0].clear(false, g, nb), kx[1].clear(false, g, nb);
#pragma unroll
      for (int st = 0; st < NB; ++st)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const u32x4 k = kv_decode8(kx[h].code(st), mx4_scale(kx[h].scale(st)));
#pragma unroll
          for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int t = 0; t < NT; ++t) {
              u32x4 qt;
              if constexpr (C::QL) qt = *reinterpret_cast<const u32x4 *>(ql + ((rb * NB + st) * NT + t) * 1024 + lane * 16);
              else qt = q[rb][st][t];
              sc[rb][h] = kv_mfma(k, qt, sc[rb][h]);
            }
        }
      load(kx[0], ka.kc, ka.ks, r0), load(kx[1], ka.kc, ka.ks, r1);

      // the keys that this lane's rows see
      uint32_t vis[RB];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        const uint32_t to = max(min(kend, lim[rb]), key) - key;
        vis[rb] = seen & (to >= 32 ? 0xffffffffu : (1u << to) - 1);
      }

      // V into LDS. Keys that are not there as zeros, and so are blocks of scales that are too small
      // (see kv_less) and blocks that are NaN, which are added to the rows that see them here
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (!C::EXACT || seen != 0xffffffffu) vx[h].clear(!(seen >> (16 * h + l16) & 1), g, nb);
      if (__any(vx[0].odd(less) || vx[1].odd(less))) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          for (uint64_t left = __ballot(vx[h].nan()); left; left &= left - 1) {
            const int from = __builtin_ctzll(left);
            const uint32_t kb = 1u << (16 * h + (from & 15));
#pragma unroll
            for (int st = 0; st < NB; ++st) {
              if ((uint32_t)__builtin_amdgcn_readlane(vx[h].scale(st), from) <= 252) continue;
              const int blk = KvCodes<C>::block(st, from >> 4);
#pragma unroll
              for (int b = 0; b < NB; ++b)
                if (b == blk) {
#pragma unroll
                  for (int rb = 0; rb < RB; ++rb) {
                    const float x = vis[rb] & kb ? __uint_as_float(0x7fc00000u) : 0.0f;
                    o[rb][2 * b] += x, o[rb][2 * b + 1] += x;
                  }
                }
            }
          }
          vx[h].clear_odd(less);
        }
      }
      const uint32_t vsw = kv_swz<C>(l16);
#pragma unroll
      for (int st = 0; st < NB; ++st)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          *reinterpret_cast<u32x4 *>(vt + (16 * h + l16) * RW + ((KvPlace<C>::unit(st, g) ^ vsw) * 16)) =
              kv_decode8(vx[h].code(st), mx4_scale(vx[h].scale(st) - less));
      load(vx[0], ka.vc, ka.vs, r0), load(vx[1], ka.vc, ka.vs, r1);

      // the softmax; of block h this lane has keys 16 h + 4 g + 0..3
      u32x4 pt[RB][NT];
#pragma unroll
      for (int rb = 0; rb < RB; ++rb) {
        float x[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = sc[rb][i / 4][i % 4];
        if (__any(vis[rb] != 0xffffffffu)) {
          const uint32_t mine_of = vis[rb] >> (4 * g);
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (!(mine_of >> (16 * (i / 4) + i % 4) & 1)) x[i] = -__builtin_huge_valf();
        }
        kv_softmax<C>(x, pt[rb], m[rb], l[rb], o[rb], a.scale_log2);
      }

      // O^T += V^T P^T: in a transposing read 16 lanes read 4 rows x 16 columns, 8 bytes each
      // (row lane / 4, columns 4 (lane % 4) ..), and lane i gets column i
      const uint32_t vr = 4 * g + (l16 >> 2), rsw = kv_swz<C>(vr);
#pragma unroll
      for (int i = 0; i < 2 * NB; ++i) {
        const uint32_t unit = (2 * i + ((lane & 3) >> 1)) ^ rsw;
        const char *pv = vt + vr * RW + unit * 16 + (lane & 1) * 8;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)pv);
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)(pv + 16 * RW));
        const u32x4 v = __builtin_bit_cast(u32x4, s16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
          for (int t = 0; t < NT; ++t) o[rb][i] = kv_mfma(v, pt[rb][t], o[rb][i]);
      }
      p0 = n0, p1 = n1;
    }

    // join the wavefronts' keys: a common maximum, scaled sums through LDS, JD dims at a time
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      l[rb] = kv_row_sum(l[rb]) * __uint_as_float((127 - less) << 23);  // as the values are
      if (g == 0) {
        jml[(2 * wave) * TR + 16 * rb + l16] = m[rb];
        jml[(2 * wave + 1) * TR + 16 * rb + l16] = l[rb];
      }
    }
    __syncthreads();  // and all are done with V and the queries
    float f[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
      float mm = jml[16 * rb + l16];
#pragma unroll
      for (int w = 1; w < WK; ++w) mm = fmaxf(mm, jml[2 * w * TR + 16 * rb + l16]);
      f[rb] = __builtin_amdgcn_exp2f(m[rb] - mm);
    }
    float *jo = reinterpret_cast<float *>(lds);
    const uint64_t rows_all = (uint64_t)a.tokens * a.hq, ml0 = attn_ws_ml(a);
    const bool direct = !a.ws || nparts == 1;
#pragma unroll
    for (int d0 = 0; d0 < DP; d0 += C::JD) {
      if (d0) __syncthreads();
#pragma unroll
      for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int i = d0 / 16; i < (d0 + C::JD) / 16 && i < 2 * NB; ++i)
          *reinterpret_cast<f32x4 *>(jo + (wave * TR + 16 * rb + l16) * C::JP + 16 * i - d0 + 4 * g) = o[rb][i] * f[rb];
      __syncthreads();
      constexpr int UR = C::JD / 8;
      for (uint32_t i = tid; i < TR * UR; i += 64 * WK) {
        const uint32_t rr = i / UR, dj = (i - rr * UR) * 8, dim = d0 + dj, row = row0 + rr;
        if (row >= nrows || dim >= a.d) continue;
        f32x4 x0{}, x1{};
        float mr = jml[rr], lr = 0.0f;
#pragma unroll
        for (int w = 1; w < WK; ++w) mr = fmaxf(mr, jml[2 * w * TR + rr]);
#pragma unroll
        for (int w = 0; w < WK; ++w) {
          const float *jp = jo + (w * TR + rr) * C::JP + dj;
          x0 += *reinterpret_cast<const f32x4 *>(jp);
          x1 += *reinterpret_cast<const f32x4 *>(jp + 4);
          lr += jml[(2 * w + 1) * TR + rr] * __builtin_amdgcn_exp2f(jml[2 * w * TR + rr] - mr);
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
          if constexpr (C::DT == DT_F32) {
            *reinterpret_cast<f32x4 *>((float *)a.o + e) = x0;
            *reinterpret_cast<f32x4 *>((float *)a.o + e + 4) = x1;
          } else {
            const u32x2 y0 = pack4<C::DT>(x0), y1 = pack4<C::DT>(x1);
            *reinterpret_cast<u32x4 *>((uint16_t *)a.o + e) = u32x4{y0.x, y0.y, y1.x, y1.y};
          }
        }
      }
    }
    __syncthreads();  // the next item's tiles go where the results were read
  }
}

// Items beyond the workgroups that run at once are shared by those: where keys are
// cut, of the items that the host counts (the longest length for all) few may exist; and
// where there are many sequences, which every workgroup counts up to its first item (single
// tokens over 40 keys, 32/8 heads of 64, a workgroup for each item | shared: 256 sequences
// 13.8 | 11.6 us, 1024 84 | 38, 65536 214000 | 2318). Fewer ones of different lengths are better
// off without (100 prompts of 16 to 1024 472 | 478, of 512 behind 512 207 | 225). A launch takes
// less than 2^32 threads.
template <class C>
hipError_t kv_launch_items(const Kv4AttnArgs &a, hipStream_t st) {
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(kv4_attn_kernel<C>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (attr != hipSuccess) return attr;
  static const int occ = [] {
    int v = 0;
    if (hipOccupancyMaxActiveBlocksPerMultiprocessor(&v, reinterpret_cast<const void *>(kv4_attn_kernel<C>), 64 * C::WK,
                                                     C::LDS) != hipSuccess || v < 1)
      v = 1;
    return v;
  }();
  uint64_t items = (uint64_t)a.at.hkv * a.at.parts * a.at.tiles;
  if (items == 0 || items > 0x7fffffffu) return hipErrorInvalidValue;
  const bool shared = a.at.parts > 1 || a.at.nseq > 256;
  const uint64_t most = shared ? (uint64_t)device_cus() * occ : 0xffffffffu / (64 * C::WK);
  items = items < most ? items : most;
  hipLaunchKernelGGL((kv4_attn_kernel<C>), dim3((uint32_t)items), dim3(64 * C::WK), C::LDS, st, a);
  return hipGetLastError();
}

template <int DT, int RB>
hipError_t kv_launch_rows(const Kv4AttnArgs &a, hipStream_t st) {
  switch (a.at.d / 32) {
    case 1: return kv_launch_items<KvCfg<DT, 1, RB, 4>>(a, st);
    case 2: return kv_launch_items<KvCfg<DT, 2, RB, 4>>(a, st);
    case 3: return kv_launch_items<KvCfg<DT, 3, RB, 4>>(a, st);
    case 4: return kv_launch_items<KvCfg<DT, 4, RB, 4>>(a, st);
    case 5:
    case 6: return kv_launch_items<KvCfg<DT, 6, RB, 4>>(a, st);
    default: return kv_launch_items<KvCfg<DT, 8, RB, 4>>(a, st);
  }
}

template <int DT>
hipError_t kv_launch_dt(const Kv4AttnArgs &a, hipStream_t st) {
  if (a.rb == 1) return kv_launch_rows<DT, 1>(a, st);
  if (a.rb == 2) return kv_launch_rows<DT, 2>(a, st);
  switch (a.at.d / 32) {
    case 2: return kv_launch_items<KvCfg<DT, 2, 4, 4>>(a, st);
    case 3: return kv_launch_items<KvCfg<DT, 3, 4, 4>>(a, st);
    case 4: return kv_launch_items<KvCfg<DT, 4, 4, 4>>(a, st);
    default: return hipErrorInvalidValue;
  }
}

}  // namespace
}  // namespace aih
