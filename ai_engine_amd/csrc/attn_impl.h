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
// stays below 2^8, exact enough in every type. For 16-bit heads of at most 64
// elements, where the vector instructions and not the products set the time,
// the maximum is not even looked for until a tile's probabilities, whose sum
// is at hand before they are used, add up to 2^15 (AtTile::LAZY; 4096 tokens,
// 16/4 heads causal: of 32 elements 50.0 -> 43.4 us, of 64 62.0 -> 58.9, of 96
// and 256 nothing gained, of 128 2 % lost: the exponentials then wait for the check
// instead of running beside the next product). A row goes by its own values
// alone: what others in the wavefront hold does not change its rounding.
constexpr float kAtSlack = 8.0f;
constexpr float kAtMost = 32768.0f;
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

// A wavefront's tile: NQ blocks of 32 query rows, KB blocks of 32 keys, heads of
// at most DP elements.
template <int DT_, int DP_, int NQ_, int KB_>
struct AtTile {
  static constexpr int DT = DT_, DP = DP_, NQ = NQ_, KB = KB_;
  static constexpr bool F32 = DT == DT_F32;
  static constexpr bool LAZY = !F32 && DP <= 64;
  static constexpr int EB = Storage<DT>::bytes, UE = 16 / EB;
  static constexpr int U = DP / UE;                   // 16-byte units of a head
  static constexpr int PU = DP == 96 ? 128 / UE : U;  // units of an LDS row: a power of two
  static constexpr int RB = PU * 16;
  static constexpr int NC = U / 2, DB = DP / 32;
  static constexpr int RPI = 64 / PU;                 // rows of a DMA instruction (1 KB)
  static constexpr int KEYS = 32 * KB;
};

// LDS layout of a tile of rows: unit u of row r at slot u ^ swz(r) of its PU
// slots, so that the operand reads (8 consecutive rows, one unit each, of K; 4
// rows, 2 units each, of 16-bit V) touch 8 distinct bank groups. fp32 V is read
// along its rows and needs none.
template <class T>
__device__ __forceinline__ uint32_t at_kswz(uint32_t r) { return T::PU >= 8 ? r & 7 : (r >> 1) & 3; }
template <class T>
__device__ __forceinline__ uint32_t at_vswz(uint32_t r) {
  return T::F32 ? 0 : T::PU >= 8 ? (r & 3) << 1 : ((r >> 1) & 1) << 1;
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
#pragma unroll
  for (int k = 0; k < NI; ++k) {
    const uint32_t i = i0 + k;
    // rows i RPI and lr share no bit, so the XORs add up
    const uint32_t u = lu ^ (T::PU < 8 ? 0 : V ? at_vswz<T>(i * T::RPI) : at_kswz<T>(i * T::RPI));
    const uint32_t off = u < du ? u * 16 + (i * T::RPI + lr) * stride : kAtOob;
    const uint32_t m0 = __builtin_amdgcn_readfirstlane(to + i * 1024);
    // one wait state after m0; five after a vector instruction that may have
    // written the descriptor
    if (k == 0)
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                       :
                       : "s"(m0), "v"(off), "s"(rs)
                       : "memory", "m0");
    else
      __asm__ volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                       :
                       : "s"(m0), "v"(off), "s"(rs)
                       : "memory", "m0");
  }
}

// S^T = K Q^T of a tile; q(n, c): units 2c + h (lane half h) of this lane's row of
// block n.
template <class T, class Q>
__device__ __forceinline__ void at_qk(const char *kt, Q q, f32x16 (&sc)[T::KB][T::NQ], int lane) {
  const uint32_t l32 = lane & 31, lh = lane >> 5, sw = at_kswz<T>(l32);
#pragma unroll
  for (int kb = 0; kb < T::KB; ++kb) {
#pragma unroll
    for (int n = 0; n < T::NQ; ++n) sc[kb][n] = f32x16{};
#pragma unroll
    for (int c = 0; c < T::NC; ++c) {
      const u32x4 k = *reinterpret_cast<const u32x4 *>(kt + (32 * kb + l32) * T::RB + (((2 * c + lh) ^ sw) * 16));
#pragma unroll
      for (int n = 0; n < T::NQ; ++n) {
        const u32x4 qn = q(n, c);
        if constexpr (T::F32) {
          const f32x4 k4 = __builtin_bit_cast(f32x4, k), q4 = __builtin_bit_cast(f32x4, qn);
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[kb][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(k4[e], q4[e], sc[kb][n], 0, 0, 0);
        } else if constexpr (T::DT == DT_F16) {
          sc[kb][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, k),
                                                             __builtin_bit_cast(f16x8, qn), sc[kb][n], 0, 0, 0);
        } else {
          sc[kb][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, k),
                                                              __builtin_bit_cast(bf16x8, qn), sc[kb][n], 0, 0, 0);
        }
      }
    }
  }
}

// Key of result register r in block kb, relative to the tile.
__device__ __forceinline__ uint32_t at_key(int kb, int r, uint32_t lh) { return 32 * kb + 8 * (r / 4) + 4 * lh + r % 4; }

// Keys from to[n] on (relative to the tile) do not count.
template <class T>
__device__ __forceinline__ void at_mask(f32x16 (&sc)[T::KB][T::NQ], const uint32_t (&to)[T::NQ], int lane) {
  const uint32_t lh = lane >> 5;
#pragma unroll
  for (int n = 0; n < T::NQ; ++n)
#pragma unroll
    for (int kb = 0; kb < T::KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        if (at_key(kb, r, lh) >= to[n]) sc[kb][n][r] = -__builtin_huge_valf();
}

// Scores -> probabilities 2^(scale s - m + bias) with the running maximum m (in
// the exponent's units) and this lane's share of the sum l. 16-bit types get
// them packed for the product, 16 keys an operand.
template <class T>
__device__ __forceinline__ void at_softmax(f32x16 (&sc)[T::KB][T::NQ], u32x4 (&pb)[T::KB][2][T::NQ], float (&m)[T::NQ],
                                           float (&l)[T::NQ], f32x16 (&o)[T::DB][T::NQ], float scale) {
#pragma unroll
  for (int n = 0; n < T::NQ; ++n) {
    // the row's maximum over this tile, in the exponent's units
    auto top = [&]() {
      float mx = sc[0][n][0];
#pragma unroll
      for (int kb = 0; kb < T::KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[kb][n][r]);
      return at_pair_max(mx) * scale;
    };
    auto raise = [&](float mx, bool need) {
      const float mn = need ? fmaxf(m[n], mx) : m[n], al = __builtin_amdgcn_exp2f(m[n] - mn);
      m[n] = mn;
      l[n] *= al;
#pragma unroll
      for (int db = 0; db < T::DB; ++db)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[db][n][r] *= al;
    };
    // p of all keys; their sum
    auto probs = [&]() -> float {
      const float off = kAtBias<T::DT> - m[n];
      float sum = 0.0f;
#pragma unroll
      for (int kb = 0; kb < T::KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; r += 2) {
          const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][n][r], scale, off));
          const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][n][r + 1], scale, off));
          if constexpr (T::F32) {
            sc[kb][n][r] = p0, sc[kb][n][r + 1] = p1;
            sum += p0 + p1;
          } else {
            const uint32_t p = pack2<T::DT>(p0, p1);
            pb[kb][r / 8][n][r % 8 / 2] = p;
            sum = at_dot_ones<T::DT>(p, sum);
          }
        }
      return sum;
    };
    float sum;
    if constexpr (T::LAZY) {
      sum = probs();
      const bool big = !(sum < kAtMost);
      if (__any(big)) {
        raise(top(), at_pair_max(big ? 1.0f : 0.0f) != 0.0f);
        sum = probs();
      }
    } else {
      const float mx = top();
      const bool need = mx > m[n] + kAtSlack;
      if (__any(need)) raise(mx, need);
      sum = probs();
    }
    l[n] += sum;
  }
}

// O^T += V^T P^T; CLEAN: infinite and NaN values of V count as zero.
template <class T, bool CLEAN>
__device__ __forceinline__ void at_pv(const char *vt, const f32x16 (&sc)[T::KB][T::NQ],
                                      const u32x4 (&pb)[T::KB][2][T::NQ], f32x16 (&o)[T::DB][T::NQ], int lane) {
  const uint32_t l32 = lane & 31, lh = lane >> 5;
  if constexpr (T::F32) {
    const char *p = vt + 4 * lh * T::RB + l32 * 4;
#pragma unroll
    for (int kb = 0; kb < T::KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r)
#pragma unroll
        for (int db = 0; db < T::DB; ++db) {
          uint32_t v = *reinterpret_cast<const uint32_t *>(p + (32 * kb + 8 * (r / 4) + r % 4) * T::RB + 128 * db);
          if constexpr (CLEAN) v = at_finite_only<T::DT>(v);
#pragma unroll
          for (int n = 0; n < T::NQ; ++n)
            o[db][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v), sc[kb][n][r], o[db][n], 0, 0, 0);
        }
  } else {
    // a transposing read: 16 lanes read 4 rows x 16 columns, 8 bytes each
    // (row lane / 4, columns 4 (lane % 4) ..), and lane i gets column i
    const uint32_t row = 4 * lh + ((lane & 15) >> 2), sw = at_vswz<T>(row);
#pragma unroll
    for (int kb = 0; kb < T::KB; ++kb)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int db = 0; db < T::DB; ++db) {
          const uint32_t unit = (4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ sw;
          const char *p = vt + (32 * kb + 16 * h + row) * T::RB + unit * 16 + (lane & 1) * 8;
          const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)p);
          const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)(p + 8 * T::RB));
          u32x4 v = __builtin_bit_cast(u32x4, s16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
          if constexpr (CLEAN) {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] = at_finite_only<T::DT>(v[e]);
          }
#pragma unroll
          for (int n = 0; n < T::NQ; ++n) {
            if constexpr (T::DT == DT_F16)
              o[db][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                  __builtin_bit_cast(f16x8, v), __builtin_bit_cast(f16x8, pb[kb][h][n]), o[db][n], 0, 0, 0);
            else
              o[db][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(
                  __builtin_bit_cast(bf16x8, v), __builtin_bit_cast(bf16x8, pb[kb][h][n]), o[db][n], 0, 0, 0);
          }
        }
  }
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
// that see them (keys below to[n]) one by one, and the product runs without
// them. True: it has some.
template <class T>
__device__ __forceinline__ bool at_spread_nonfinite(const char *vt, uint32_t from, uint32_t end,
                                                    const uint32_t (&to)[T::NQ], f32x16 (&o)[T::DB][T::NQ], int lane) {
  uint32_t big = 0;
  for (uint32_t i = from * T::PU + lane; i < end * T::PU; i += 64)
    big = at_max_abs<T::DT>(big, *reinterpret_cast<const u32x4 *>(vt + i * 16));
  if (!__any(at_nonfinite<T::DT>(big) != 0)) return false;
  const uint32_t lh = lane >> 5;
  for (uint32_t j = 0; j < T::KEYS; ++j) {
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
#pragma unroll
          for (int n = 0; n < T::NQ; ++n)
            if (at_nonfinite<DT_F32>(__float_as_uint(v[e])) && j < to[n]) o[db][n][4 * r4 + e] += v[e];
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

// The query rows of a wavefront from row0 on: unit u of block n's row l32, zero
// where there is none. Offsets from the first row's token fit 32 bits.
template <class T>
struct AtQuery {
  __amdgpu_buffer_rsrc_t rs;
  uint32_t off[T::NQ];
  __device__ __forceinline__ AtQuery(const AttnArgs &a, const AtSeq &s, uint32_t hk, uint32_t row0, uint32_t l32) {
    const uint32_t nrows = s.lq * a.g, tok0 = fdiv(min(row0, nrows - 1), a.by_g);
    rs = at_rsrc((const char *)a.q + ((uint64_t)(s.q0 + tok0) * a.qs + (uint64_t)hk * a.g * a.d) * T::EB, 0x7fffffffu);
#pragma unroll
    for (int n = 0; n < T::NQ; ++n) {
      const uint32_t row = row0 + 32 * n + l32, tok = fdiv(row, a.by_g);
      off[n] = row < nrows ? ((tok - tok0) * (uint32_t)a.qs + (row - tok * a.g) * a.d) * T::EB : kAtOob;
    }
  }
  __device__ __forceinline__ u32x4 unit(const AttnArgs &a, int n, uint32_t u) const {
    const uint32_t o = u * T::UE < a.d ? off[n] + u * 16 : kAtOob;
    return __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rs, o, 0, 0));
  }
};

}  // namespace
}  // namespace aih
