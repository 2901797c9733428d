// attn_impl.h -- what the two MFMA attention kernels (attn_rows.h, attn_keys.h)
// share: the products of a wavefront with one tile of keys, the running
// softmax between them, and where a tile's rows and keys are.
//
// With the scores as S^T = K Q^T a lane of the 32x32 result holds 16 keys of
// one query (lanes l and l + 32 the two halves): the row maximum and sum are
// in-lane but for one exchange, a row's rescale is one factor per lane, and
// the probabilities are already the B operand of O^T = V^T P^T -- the order of
// the keys inside a product is free, so V is read in the order the scores
// came out (lane half h: keys 8 i + 4 h + 0..3). V^T itself comes from the
// row-major tile by transposing LDS reads.
#pragma once

#include <hip/hip_runtime.h>

#include <type_traits>

#include "aih_device.h"
#include "attn.h"

namespace aih {
namespace {

typedef __attribute__((address_space(3))) void at_lds_void;
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef __attribute__((address_space(3))) s16x4 at_lds_s16x4;

constexpr uint32_t kAtOob = 0x80000000u;  // a byte offset past every buffer
constexpr float kAtLowest = -3.402823466e38f;
// A row's maximum is left stale until a score exceeds it by 2^8, so that the
// accumulators are rescaled a few times per row instead of once per stage; p
// stays below 2^8, exact enough in every type. LAZY tiles do not even look for
// the maximum before a block's probabilities, whose sum is at hand before they
// are used, add up to 2^15: 16-bit heads of at most 64 elements, whose vector
// instructions set the time (4096 tokens, 16/4 heads causal: of 32 elements
// 50.0 -> 43.4 us, of 64 62.0 -> 58.9), and of more than 128, whose steps are
// written out (at_step) and have nothing to wait for. At 96 and 128 elements the
// exponentials then wait for the check instead of running beside the next
// product (2 to 3 % lost), fp32's few long ones lose it (3 to 5 % of a short
// call: a row's first block is always taken twice). A row goes by its own values
// alone: what others in the wavefront hold does not change its rounding.
constexpr float kAtSlack = 8.0f;
constexpr float kAtMost = 32768.0f;
// The exponent's argument is one fma: the exact product of score and scale less the
// maximum, which is rounded. The two are up to half a unit of the maximum's last
// place apart, a common factor of a row's probabilities while its maximum stays, but
// from 2^24 on it counts, later it leaves the range. Rows whose maximum is that far
// out take the product rounded as well (at_far), which fp32 scores are precise to.
constexpr float kAtFar = 16777216.0f;
// f16 probabilities are held 2^7 times larger (below 2^15): those of 2^-22 and
// more keep all their bits, where without it they would be subnormal from 2^-15
// on. The sum carries the same factor. fp32 and bf16 have the range.
template <int DT> constexpr float kAtBias = DT == DT_F16 ? 7.0f : 0.0f;

__device__ __forceinline__ __amdgpu_buffer_rsrc_t at_rsrc(const void *base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)bytes, 0x00020000);
}

template <int N>
__device__ __forceinline__ void at_wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
}

// max / sum over the two lanes that hold a row (l and l ^ 32)
__device__ __forceinline__ float at_pair_max(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float at_pair_sum(float x) {
  const uint32_t u = __float_as_uint(x);
  const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Nonzero where one of the values in r is infinite or NaN: an exponent of
// ones carries into the sign's bit.
template <int DT>
__device__ __forceinline__ uint32_t at_nonfinite(uint32_t r) {
  if constexpr (DT == DT_F32) return ((r & 0x7f800000u) + 0x00800000u) & 0x80000000u;
  else if constexpr (DT == DT_F16) return ((r & 0x7c007c00u) + 0x04000400u) & 0x80008000u;
  else return ((r & 0x7f807f80u) + 0x00800080u) & 0x80008000u;
}

// r with its infinite and NaN values as zeros
template <int DT>
__device__ __forceinline__ uint32_t at_finite_only(uint32_t r) {
  const uint32_t b = at_nonfinite<DT>(r);
  if constexpr (DT == DT_F32) return b ? 0u : r;
  else return r & ~((b >> 15) * 0xffffu);
}

// c + the two values in p: one instruction, subnormal f16 included. The sums are
// of the probabilities as rounded for the product, so that the roundings cancel
// in their quotient.
template <int DT>
__device__ __forceinline__ float at_dot_ones(uint32_t p, float c) {
  if constexpr (DT == DT_F16)
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, p), f16x2{(_Float16)1.0f, (_Float16)1.0f}, c, false);
  else
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, p), bf16x2{(__bf16)1.0f, (__bf16)1.0f}, c, false);
}

// A wavefront's tile: 32 query rows, 32 keys, heads of at most DP elements.
template <int DT_, int DP_>
struct AtTile {
  static constexpr int DT = DT_, DP = DP_;
  static constexpr bool F32 = DT == DT_F32;
  static constexpr bool LAZY = !F32 && (DP <= 64 || DP > 128);  // see kAtMost
  static constexpr int EB = Storage<DT>::bytes, UE = 16 / EB;
  static constexpr int U = DP / UE;                   // 16-byte units of a head
  static constexpr int PU = DP == 96 ? 128 / UE : U;  // units of an LDS row: a power of two
  static constexpr int RB = PU * 16;
  static constexpr int NC = U / 2, DB = DP / 32;
  static constexpr int RPI = 64 / PU;                 // rows of a DMA instruction (1 KB)
  // probabilities of 32 keys: as they are, or packed, 16 keys an operand
  struct Packed { u32x4 h[2]; };
  using Probs = std::conditional_t<F32, f32x16, Packed>;
};

// LDS layout of a tile of rows: unit u of row r at slot u ^ swz(r) of its PU
// slots. A cycle serves 256 bytes, all 64 banks: 16 lanes of a read of K (16
// consecutive rows, one unit each) or 32 of a transposing read of 16-bit V (4
// rows, 4 units each), which the slots spread over the 16 groups of 4 banks. With
// swizzles for 8 groups every read of 128 elements took twice the cycles. fp32 V
// is read along its rows and has none.
template <class T>
__device__ __forceinline__ uint32_t at_kswz(uint32_t r) {
  return T::PU >= 16 ? r & 15 : T::PU == 8 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <class T>
__device__ __forceinline__ uint32_t at_vswz(uint32_t r) {
  return T::F32 ? 0 : T::PU >= 16 ? (r & 3) << 2 : T::PU == 8 ? (r & 3) << 1 : 0;
}

// DMA of instructions i0 .. i0 + NI - 1 of a tile (1 KB, RPI rows each): lane ->
// row i RPI + lane / PU, slot lane % PU. Rows past `rows` and units past the
// head land as zeros.
//
// Written out, because the compiler makes every transposing LDS read wait for
// all copies it knows of, those of the next stage too (it cannot tell their
// places apart). The kernels wait for a stage's copies themselves
// (at_wait_vm); no register is written, and a count that the compiler waits for
// on behalf of its own loads only gets stricter by copies it does not know of.
template <class T, int NI, bool V>
__device__ __forceinline__ void at_dma(const char *base, uint32_t stride, uint32_t rows, uint32_t du, int i0, int lane,
                                       char *dst) {
  const uint64_t at = reinterpret_cast<uint64_t>(base);
  const u32x4 rs = {(uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)at),
                    (uint32_t)__builtin_amdgcn_readfirstlane((uint32_t)(at >> 32) & 0xffffu),
                    (uint32_t)__builtin_amdgcn_readfirstlane(rows ? (rows - 1) * stride + du * 16 : 0), 0x00020000u};
  const uint32_t lr = lane / T::PU, ls = lane % T::PU;
  const uint32_t lu = ls ^ (V ? at_vswz<T>(lr) : at_kswz<T>(lr));
  const uint32_t to = (uint32_t)(uintptr_t)(at_lds_void *)dst;
  constexpr int G = NI < 4 ? NI : 4;  // copies written out together
  static_assert(NI % G == 0, "DMA instructions");
#pragma unroll
  for (int k = 0; k < NI; k += G) {
    uint32_t off[G];
#pragma unroll
    for (int e = 0; e < G; ++e) {
      const uint32_t i = i0 + k + e;
      // rows i RPI and lr share no bit, so the XORs add up
      const uint32_t u = lu ^ (T::PU < 8 ? 0 : V ? at_vswz<T>(i * T::RPI) : at_kswz<T>(i * T::RPI));
      off[e] = u < du ? u * 16 + (i * T::RPI + lr) * stride : kAtOob;
    }
    const uint32_t m0 = __builtin_amdgcn_readfirstlane(to + (i0 + k) * 1024);
    // One wait state after m0; five after a vector instruction that may have
    // written the descriptor, which any piece of text has to hold for itself:
    // scalar registers that the compiler spills come back through v_readlane, and
    // it does not know what the text reads.
#define AIH_AT_COPY(OFF) "buffer_load_dwordx4 " OFF ", %1, 0 offen lds\n\t"
#define AIH_AT_NEXT(AT) "s_add_u32 m0, %0, " AT "\n\ts_nop 0\n\t"
    if constexpr (G == 1)
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\t" AIH_AT_COPY("%2")
                       :
                       : "s"(m0), "s"(rs), "v"(off[0])
                       : "memory", "m0");
    else if constexpr (G == 2)
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\t" AIH_AT_COPY("%2") AIH_AT_NEXT("0x400") AIH_AT_COPY("%3")
                       :
                       : "s"(m0), "s"(rs), "v"(off[0]), "v"(off[1])
                       : "memory", "m0", "scc");
    else
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\t" AIH_AT_COPY("%2") AIH_AT_NEXT("0x400") AIH_AT_COPY("%3")
                           AIH_AT_NEXT("0x800") AIH_AT_COPY("%4") AIH_AT_NEXT("0xc00") AIH_AT_COPY("%5")
                       :
                       : "s"(m0), "s"(rs), "v"(off[0]), "v"(off[1]), "v"(off[G > 2 ? 2 : 0]), "v"(off[G > 2 ? 3 : 0])
                       : "memory", "m0", "scc");
#undef AIH_AT_COPY
#undef AIH_AT_NEXT
  }
}

// c + A B of 16-bit operands
template <class T>
__device__ __forceinline__ f32x16 at_mfma(u32x4 a, u32x4 b, f32x16 c) {
  if constexpr (T::DT == DT_F16)
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// S^T = K Q^T of N tiles; q(c): units 2c + h (lane half h) of this lane's row.
template <class T, int N, class Q>
__device__ __forceinline__ void at_qk(const char *kt, Q q, f32x16 (&sc)[N], int lane) {
  const uint32_t l32 = lane & 31, lh = lane >> 5, sw = at_kswz<T>(l32);
#pragma unroll
  for (int i = 0; i < N; ++i) sc[i] = f32x16{};
#pragma unroll
  for (int c = 0; c < T::NC; ++c)
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const u32x4 k = *reinterpret_cast<const u32x4 *>(kt + (32 * i + l32) * T::RB + (((2 * c + lh) ^ sw) * 16)), qc = q(c);
      if constexpr (T::F32) {
        const f32x4 k4 = __builtin_bit_cast(f32x4, k), q4 = __builtin_bit_cast(f32x4, qc);
#pragma unroll
        for (int e = 0; e < 4; ++e) sc[i] = __builtin_amdgcn_mfma_f32_32x32x2f32(k4[e], q4[e], sc[i], 0, 0, 0);
      } else {
        sc[i] = at_mfma<T>(k, qc, sc[i]);
      }
    }
}

// Keys from `to` on (relative to the tile) do not count: result register r is key
// 8 (r / 4) + r % 4 + 4 h.
__device__ __forceinline__ void at_mask(f32x16 &sc, uint32_t to, int lane) {
  const int mine = (int)min(to, 32u) - 4 * (lane >> 5);
#pragma unroll
  for (int r = 0; r < 16; ++r)
    if (8 * (r / 4) + r % 4 >= mine) sc[r] = -__builtin_huge_valf();
}

// Scores -> probabilities 2^(scale s + off), off the bias less the running maximum
// (in the exponent's units); returns `sum` plus this lane's. Words w0 .. w1 - 1, two
// keys each.
template <class T>
__device__ __forceinline__ float at_probs(const f32x16 &sc, typename T::Probs &p, float off, float scale, int w0 = 0,
                                          int w1 = 8, float sum = 0.0f) {
#pragma unroll
  for (int w = w0; w < w1; ++w) {
    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * w], scale, off));
    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[2 * w + 1], scale, off));
    if constexpr (T::F32) {
      p[2 * w] = p0, p[2 * w + 1] = p1;
      sum += p0 + p1;
    } else {
      const uint32_t x = pack2<T::DT>(p0, p1);
      p.h[w / 4][w % 4] = x;
      sum = at_dot_ones<T::DT>(x, sum);
    }
  }
  return sum;
}
// at_probs' `off` for the maximum m. The scores of rows that are far out become
// differences to the maximum, whose off is the bias alone.
template <class T, int N>
__device__ __forceinline__ float at_far(f32x16 (&sc)[N], float m, float scale) {
#pragma clang fp contract(off)
  const bool far = __builtin_fabsf(m) >= kAtFar;
  float off = kAtBias<T::DT> - m;
  if (__builtin_expect(__any(far), 0)) {
    off = far ? kAtBias<T::DT> : off;
    const float inv = __builtin_amdgcn_rcpf(scale);
#pragma unroll
    for (int i = 0; i < N; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float at = sc[i][r] * scale;
        sc[i][r] = far ? (at - m) * inv : sc[i][r];
      }
  }
  return off;
}
// The rows' maximum over N blocks, in the exponent's units.
template <class T, int N>
__device__ __forceinline__ float at_top(const f32x16 (&sc)[N], float scale) {
  float mx = sc[0][0];
#pragma unroll
  for (int i = 0; i < N; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[i][r]);
  return at_pair_max(mx) * scale;
}
// The rows that need it (`row`) get the larger maximum.
template <class T>
__device__ __forceinline__ void at_raise(float mx, bool row, float &m, float &l, f32x16 (&o)[T::DB]) {
  const float mn = row ? fmaxf(m, mx) : m, al = __builtin_amdgcn_exp2f(m - mn);
  m = mn;
  l *= al;
#pragma unroll
  for (int db = 0; db < T::DB; ++db)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[db][r] *= al;
}
// `sum` is at_probs' of N blocks: the rows that it is too large for get their
// maximum found and their probabilities again, and those far out always do.
template <class T, int N>
__device__ __forceinline__ void at_settle(f32x16 (&sc)[N], typename T::Probs (&p)[N], float sum, float &m, float &l,
                                          f32x16 (&o)[T::DB], float scale) {
  const bool big = !(sum < kAtMost) || __builtin_fabsf(m) >= kAtFar;
  if (__any(big)) {
    at_raise<T>(at_top<T>(sc, scale), at_pair_max(big ? 1.0f : 0.0f) != 0.0f, m, l, o);
    const float off = at_far<T>(sc, m, scale);
    sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) sum = at_probs<T>(sc[i], p[i], off, scale, 0, 8, sum);
  }
  l += sum;
}
// The softmax of N blocks: p, the maximum m and this lane's share of the sum l. The
// scores are used up.
template <class T, int N>
__device__ __forceinline__ void at_softmax(f32x16 (&sc)[N], typename T::Probs (&p)[N], float &m, float &l,
                                           f32x16 (&o)[T::DB], float scale) {
  float off = kAtBias<T::DT> - m;
  if constexpr (!T::LAZY) {
    const float mx = at_top<T>(sc, scale);
    const bool row = mx > m + kAtSlack;
    if (__any(row || __builtin_fabsf(m) >= kAtFar)) {
      at_raise<T>(mx, row, m, l, o);
      off = at_far<T>(sc, m, scale);
    }
  }
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < N; ++i) sum = at_probs<T>(sc[i], p[i], off, scale, 0, 8, sum);
  if constexpr (T::LAZY) at_settle<T>(sc, p, sum, m, l, o, scale);
  else l += sum;
}

// O^T += V^T P^T; CLEAN: infinite and NaN values of V count as zero.
template <class T, bool CLEAN>
__device__ __forceinline__ void at_pv(const char *vt, const typename T::Probs &pb, f32x16 (&o)[T::DB], int lane) {
  const uint32_t l32 = lane & 31, lh = lane >> 5;
  if constexpr (T::F32) {
    const char *p = vt + 4 * lh * T::RB + l32 * 4;
#pragma unroll
    for (int r = 0; r < 16; ++r)
#pragma unroll
      for (int db = 0; db < T::DB; ++db) {
        uint32_t v = *reinterpret_cast<const uint32_t *>(p + (8 * (r / 4) + r % 4) * T::RB + 128 * db);
        if constexpr (CLEAN) v = at_finite_only<T::DT>(v);
        o[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v), pb[r], o[db], 0, 0, 0);
      }
  } else {
    // a transposing read: 16 lanes read 4 rows x 16 columns, 8 bytes each
    // (row lane / 4, columns 4 (lane % 4) ..), and lane i gets column i
    const uint32_t row = 4 * lh + ((lane & 15) >> 2), sw = at_vswz<T>(row);
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int db = 0; db < T::DB; ++db) {
        const uint32_t unit = (4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ sw;
        const char *p = vt + (16 * h + row) * T::RB + unit * 16 + (lane & 1) * 8;
        const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)p);
        const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)(p + 8 * T::RB));
        u32x4 v = __builtin_bit_cast(u32x4, s16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
        if constexpr (CLEAN) {
#pragma unroll
          for (int e = 0; e < 4; ++e) v[e] = at_finite_only<T::DT>(v[e]);
        }
        o[db] = at_mfma<T>(v, pb.h[h], o[db]);
      }
  }
}

// A step of 16-bit heads: the scores of the next block (K at kt; they replace
// sc), the product of the last block's probabilities (V at vt; p) and the
// probabilities of the block in between (sc; they replace p). None waits for
// another: a product of each kind and a share of the exponentials at a time, the
// operands of the next two on their way. The compiler on its own puts each
// product behind the wait for its operand, and the exponentials after them.
template <class T, class Q>
__device__ __forceinline__ void at_step(const char *kt, const char *vt, Q q, f32x16 (&sc)[1], typename T::Probs (&p)[1],
                                        float &m, float &l, f32x16 (&o)[T::DB], float scale, int lane) {
  constexpr int N = T::NC, FIRST = 2;  // products of each kind; operands on their way
  const uint32_t l32 = lane & 31, lh = lane >> 5, sw = at_kswz<T>(l32);
  const uint32_t row = 4 * lh + ((lane & 15) >> 2), vsw = at_vswz<T>(row);
  u32x4 kk[N], vv[N];
  auto load = [&](int i) __attribute__((always_inline)) {
    kk[i] = *reinterpret_cast<const u32x4 *>(kt + l32 * T::RB + (((2 * i + lh) ^ sw) * 16));
    const int h = i / T::DB, db = i % T::DB;
    const uint32_t unit = (4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vsw;
    const char *at = vt + (16 * h + row) * T::RB + unit * 16 + (lane & 1) * 8;
    const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)at);
    const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)(at + 8 * T::RB));
    vv[i] = __builtin_bit_cast(u32x4, s16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
  };
  f32x16 next{};
  typename T::Probs pn[1];
  const float off = kAtBias<T::DT> - m;
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < FIRST; ++i) load(i);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    __builtin_amdgcn_sched_barrier(0);
    if (i + FIRST < N) load(i + FIRST);
    sum = at_probs<T>(sc[0], pn[0], off, scale, 8 * i / N, 8 * (i + 1) / N, sum);
    next = at_mfma<T>(kk[i], q(i), next);
    o[i % T::DB] = at_mfma<T>(vv[i], p[0].h[i / T::DB], o[i % T::DB]);
  }
  __builtin_amdgcn_sched_barrier(0);
  p[0] = pn[0];
  at_settle<T>(sc, p, sum, m, l, o, scale);
  sc[0] = next;
}

// The larger magnitude, per value, of a running maximum and of four words of V.
template <int DT>
__device__ __forceinline__ uint32_t at_max_abs(uint32_t m, u32x4 v) {
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    if constexpr (DT == DT_F32) {
      m = max(m, v[e] & 0x7fffffffu);
    } else {
      const u16x2 x = __builtin_bit_cast(u16x2, v[e] & 0x7fff7fffu), y = __builtin_bit_cast(u16x2, m);
      m = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(x, y));
    }
  }
  return m;
}

// Keys that some rows of a tile see and others do not: 0 * NaN or 0 * inf of an
// unseen value must not reach a row. If keys `from` .. `end` - 1 of the tile,
// which hold all of those, have such values, the tile's are added to the rows
// that see them (keys below `to`) one by one, and the product runs without
// them. True: it has some.
template <class T>
__device__ __forceinline__ bool at_spread_nonfinite(const char *vt, uint32_t from, uint32_t end,
                                                    uint32_t to, f32x16 (&o)[T::DB], int lane) {
  uint32_t big = 0;
  end = min(end, 32u);
  for (uint32_t i = from * T::PU + lane; i < end * T::PU; i += 64)
    big = at_max_abs<T::DT>(big, *reinterpret_cast<const u32x4 *>(vt + i * 16));
  if (!__any(at_nonfinite<T::DT>(big) != 0)) return false;
  const uint32_t lh = lane >> 5;
  for (uint32_t j = 0; j < 32; ++j) {
#pragma unroll
    for (int db = 0; db < T::DB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const uint32_t dim = 32 * db + 8 * r4 + 4 * lh;  // four dims of this lane
        const char *p = vt + j * T::RB + ((dim / T::UE) ^ at_vswz<T>(j)) * 16 + (dim % T::UE) * T::EB;
        f32x4 v;
        if constexpr (T::F32) v = *reinterpret_cast<const f32x4 *>(p);
        else v = unpack4<T::DT>(*reinterpret_cast<const u32x2 *>(p));
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (at_nonfinite<DT_F32>(__float_as_uint(v[e])) && j < to) o[db][4 * r4 + e] += v[e];
      }
  }
  return true;
}

// One lane's sequence, cut to the tensors: nothing behind this reads or writes
// outside them, whatever the arrays hold.
struct AtSeq {
  uint32_t q0, lq, k0, len;
};
__device__ __forceinline__ AtSeq at_load_seq(const AttnArgs &a, uint32_t b) {
  AtSeq s{0, 0, 0, 0};
  if (b < a.nseq) {
    s.q0 = min((uint32_t)max(a.q_start[b], 0), a.tokens);
    const uint32_t q1 = min((uint32_t)max(a.q_start[b + 1], 0), a.tokens);
    s.lq = q1 > s.q0 ? q1 - s.q0 : 0;
    s.k0 = min((uint32_t)max(a.k_start[b], 0), a.rows);
    s.len = min((uint32_t)max(a.k_len[b], 0), a.rows - s.k0);
  }
  return s;
}
// The sequences of a wavefront's lanes (a.nseq of them, at most 64) by the number
// of their keys: the most first, or last.
__device__ __forceinline__ AtSeq at_sort(const AttnArgs &a, const AtSeq &s, uint32_t lane, bool most_first) {
  if (!__any(lane < a.nseq && s.len != (uint32_t)__builtin_amdgcn_readfirstlane(s.len))) return s;
  uint32_t rank = 0;
  for (uint32_t i = 0; i < a.nseq; ++i) {
    const uint32_t other = __builtin_amdgcn_readlane(s.len, i);
    rank += other > s.len || (other == s.len && i < lane);
  }
  const int to = 4 * (lane >= a.nseq ? lane : most_first ? rank : a.nseq - 1 - rank);
  return AtSeq{(uint32_t)__builtin_amdgcn_ds_permute(to, s.q0), (uint32_t)__builtin_amdgcn_ds_permute(to, s.lq),
               (uint32_t)__builtin_amdgcn_ds_permute(to, s.k0), (uint32_t)__builtin_amdgcn_ds_permute(to, s.len)};
}
__device__ __forceinline__ AtSeq at_seq_of(const AtSeq &s, int l) {
  return AtSeq{(uint32_t)__builtin_amdgcn_readlane(s.q0, l), (uint32_t)__builtin_amdgcn_readlane(s.lq, l),
               (uint32_t)__builtin_amdgcn_readlane(s.k0, l), (uint32_t)__builtin_amdgcn_readlane(s.len, l)};
}
// Inclusive prefix sum over a wavefront: within rows of 16 lanes by shifts, then
// a row's total into the next row and the first half's into the second.
__device__ __forceinline__ uint32_t at_scan(uint32_t v) {
  int x = (int)v;
  x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xf, 0xf, true);   // row_shr:1
  x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xf, 0xf, true);   // row_shr:2
  x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xf, 0xf, true);   // row_shr:4
  x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xf, 0xf, true);   // row_shr:8
  x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xa, 0xf, false);  // row_bcast:15 into rows 1 and 3
  x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xc, 0xf, false);  // row_bcast:31 into rows 2 and 3
  return (uint32_t)x;
}

// Keys that (query, head of the group) row `row` of a sequence sees.
__device__ __forceinline__ uint32_t at_limit(const AttnArgs &a, uint32_t causal, const AtSeq &s, uint32_t row) {
  if (!causal) return s.len;
  const int64_t n = (int64_t)fdiv(row, a.by_g) + 1 + (int64_t)s.len - (int64_t)s.lq;
  return (uint32_t)max((int64_t)0, min(n, (int64_t)s.len));
}

// log2 of the keys of a part: the plan's, unless it foresaw fewer keys.
__device__ __forceinline__ uint32_t at_shift(const AttnArgs &a, uint32_t len) {
  uint32_t x = a.shift;
  while (((uint64_t)a.parts << x) < len) ++x;
  return x;
}

// The query rows of a wavefront from row0 on: unit u of row l32, zero where there
// is none. Offsets from the first row's token fit 32 bits.
template <class T>
struct AtQuery {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t off;
  __device__ __forceinline__ AtQuery(const AttnArgs &a, const AtSeq &s, uint32_t hk, uint32_t row0, uint32_t l32) {
    const uint32_t nrows = s.lq * a.g, tok0 = fdiv(min(row0, nrows - 1), a.by_g);
    rs = at_rsrc((const char *)a.q + ((uint64_t)(s.q0 + tok0) * a.qs + (uint64_t)hk * a.g * a.d) * T::EB, 0x7fffffffu);
    const uint32_t row = row0 + l32, tok = fdiv(row, a.by_g);
    off = row < nrows ? ((tok - tok0) * (uint32_t)a.qs + (row - tok * a.g) * a.d) * T::EB : kAtOob;
  }
  __device__ __forceinline__ u32x4 unit(const AttnArgs &a, uint32_t u) const {
    const uint32_t o = u * T::UE < a.d ? off + u * 16 : kAtOob;
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0));
  }
};

}  // namespace
}  // namespace aih
