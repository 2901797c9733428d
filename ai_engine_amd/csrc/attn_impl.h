// attn_impl.h -- the MFMA attention kernel (aih_attn), one template for whole
// prompts and for few rows over many keys.
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
typedef __attribute__((address_space(3))) s16x4 at_lds_s16x4;

constexpr uint32_t kAtOob = 0x80000000u;   // a byte offset past every buffer
constexpr float kAtLowest = -3.402823466e38f;
// A row's maximum is left stale until a score exceeds it by 2^8: p then stays
// below 2^8, exact enough in every type, and the accumulators are rescaled a
// few times per row instead of once per stage.
constexpr float kAtSlack = 8.0f;
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

template <int DT, int DP_, int WR_, int WK_, int NQ_, int KB_, int NST_>
struct AtCfg {
  static constexpr int DP = DP_, WR = WR_, WK = WK_, NQ = NQ_, KB = KB_, NST = NST_;
  static constexpr int NW = WR * WK;
  static constexpr int EB = Storage<DT>::bytes, UE = 16 / EB;
  static constexpr int U = DP / UE;                    // 16-byte units of a head
  static constexpr int PU = DP == 96 ? 128 / UE : U;   // units of an LDS row: a power of two
  static constexpr int RB = PU * 16;
  static constexpr int NC = U / 2, DB = DP / 32;
  static constexpr int BM = 32 * NQ * WR;
  static constexpr int KEYS = 32 * KB * WK;
  static constexpr uint32_t STAGE = 2u * KEYS * RB;
  static constexpr int OPITCH = DP + 4;
  // the join of WK wavefronts' results reuses the stages
  static constexpr uint32_t JOIN = WK > 1 ? WK * 32u * OPITCH * 4 + WK * 64u * 4 : 0;
  static constexpr uint32_t LDS = NST * STAGE > JOIN ? NST * STAGE : JOIN;
  static_assert(WR == 1 || WK == 1, "rows or keys over the wavefronts");
  static_assert(WK == 1 || NQ == 1, "the join holds 32 rows");
  static_assert(LDS <= 160 * 1024, "LDS");
};

// Where a tile's rows and keys are.
struct AtTile {
  uint32_t q0, lq;    // query rows of the sequence
  uint32_t k0, len;   // its keys
  uint32_t row0;      // the tile's first (query, head of the group) row
  bool any;
};

// The sequence that row tile `t` belongs to: the sequences' tiles are counted
// off 64 sequences at a time, one a lane. Starts and lengths are cut to the
// tensors here, so nothing behind this reads or writes outside them.
template <int BM>
__device__ __forceinline__ AtTile at_find(const AttnArgs &a, uint32_t t, uint32_t lane) {
  AtTile r{0, 0, 0, 0, 0, false};
  if (!a.k_start) {  // all rows against the prefix
    r.lq = a.tokens;
    r.len = a.rows;
    r.row0 = t * BM;
    r.any = (uint64_t)r.row0 < (uint64_t)r.lq * a.g;
    return r;
  }
  uint32_t before = 0;
  for (uint32_t b0 = 0; b0 < a.nseq; b0 += 64) {
    const uint32_t b = b0 + lane;
    uint32_t q0 = 0, q1 = 0, k0 = 0, len = 0;
    if (b < a.nseq) {
      q0 = min((uint32_t)max(a.q_start[b], 0), a.tokens);
      q1 = min((uint32_t)max(a.q_start[b + 1], 0), a.tokens);
      k0 = min((uint32_t)max(a.k_start[b], 0), a.rows);
      len = min((uint32_t)max(a.k_len[b], 0), a.rows - k0);
    }
    const uint32_t lq = q1 > q0 ? q1 - q0 : 0;
    const uint32_t n = (lq * a.g + BM - 1) / BM;  // tokens * hq is below 2^31
    uint32_t sum = n;
#pragma unroll
    for (uint32_t w = 1; w < 64; w <<= 1) {
      const uint32_t o = __shfl_up(sum, w);
      if (lane >= w) sum += o;
    }
    const uint64_t hit = __ballot(before + sum > t);
    if (hit) {
      const int l = __ffsll((unsigned long long)hit) - 1;
      r.q0 = __builtin_amdgcn_readlane(q0, l);
      r.lq = __builtin_amdgcn_readlane(lq, l);
      r.k0 = __builtin_amdgcn_readlane(k0, l);
      r.len = __builtin_amdgcn_readlane(len, l);
      r.row0 = (t - before - (__builtin_amdgcn_readlane(sum, l) - __builtin_amdgcn_readlane(n, l))) * BM;
      r.any = true;
      return r;
    }
    before += __builtin_amdgcn_readlane(sum, 63);
  }
  return r;
}

template <int DT, class C>
__global__ __launch_bounds__(64 * C::NW) void attn_kernel(AttnArgs a) {
  constexpr int NQ = C::NQ, KB = C::KB, NST = C::NST, NC = C::NC, DB = C::DB, PU = C::PU, RB = C::RB;
  constexpr int EB = C::EB, UE = C::UE, WR = C::WR, WK = C::WK;
  constexpr bool F32 = DT == DT_F32;
  constexpr int RPI = 64 / PU;                                   // rows of a DMA instruction (1 KB)
  constexpr int NI = KB * 32 / RPI / (WK > 1 ? 1 : WR);          // K instructions of a wavefront per stage, and V
  static_assert(NI >= 1 && 2 * NI * (NST - (WK > 1 ? 1 : 2)) < 64, "DMA instructions in flight");
  extern __shared__ __align__(16) char lds[];

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);

  // key head, part, row tile: a head's tiles stay on one XCD, which keeps the
  // head's keys in its L2; the last tiles, which see the most keys under the
  // causal mask, come first
  const uint32_t id = xcd_remap(blockIdx.x, gridDim.x, a.nxcd);
  const uint32_t hk = id / (a.tiles * a.parts), rest = id - hk * (a.tiles * a.parts);
  const uint32_t part = rest / a.tiles;
  const AtTile t = at_find<C::BM>(a, a.tiles - 1 - (rest - part * a.tiles), lane);
  if (!t.any) return;
  const uint32_t nrows = t.lq * a.g;

  // keys that a row sees: all, or up to its own position
  const int64_t shift = (int64_t)t.len - (int64_t)t.lq + 1;
  auto limit = [&](uint32_t row) -> uint32_t {
    if (!a.causal) return t.len;
    const int64_t n = (int64_t)(row / a.g) + shift;
    return (uint32_t)max((int64_t)0, min(n, (int64_t)t.len));
  };
  const uint32_t last = min(t.row0 + C::BM, nrows) - 1;
  const uint32_t per = (t.len + a.parts - 1) / a.parts;
  const uint32_t chunk = max(a.chunk, (per + 31) & ~31u);
  const uint64_t kbeg64 = (uint64_t)part * chunk;
  const uint32_t kbeg = (uint32_t)min(kbeg64, (uint64_t)t.len);
  const uint32_t kend = (uint32_t)min((uint64_t)limit(last), kbeg64 + chunk);

  // this lane's query rows: row base of the wavefront + 32 nq + l32
  const uint32_t wrow = t.row0 + (WK > 1 ? 0 : wave * 32 * NQ);
  uint32_t lim[NQ];
  u32x4 q[NQ][NC];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    const uint32_t row = wrow + 32 * n + l32;
    const bool on = row < nrows;
    const uint32_t tok = row / a.g, hd = hk * a.g + (row - tok * a.g);
    lim[n] = on ? limit(row) : 0;
    const char *src = (const char *)a.q + ((uint64_t)(t.q0 + (on ? tok : 0)) * a.qs + (uint64_t)(on ? hd : 0) * a.d) * EB;
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const uint32_t u = 2 * c + lh;
      q[n][c] = u32x4{0, 0, 0, 0};
      if (on && u * UE < a.d) q[n][c] = *reinterpret_cast<const u32x4 *>(src + u * 16);
    }
  }
  // the first row of a wavefront sees the fewest keys, its last one the most
  const uint32_t wmin = wrow < nrows ? limit(wrow) : 0;
  const uint32_t wmax = wrow < nrows ? limit(min(wrow + 32 * NQ, nrows) - 1) : 0;

  // ---- DMA: LDS slot n of a stage's rows holds unit (n % PU) ^ swz(row) of row n / PU
  const uint32_t lr = lane / PU, ls = lane % PU;
  const uint32_t ku = ls ^ (PU >= 8 ? lr & 7 : (lr >> 1) & 3);
  const uint32_t vu = F32 ? ls : ls ^ (PU >= 8 ? (lr & 3) << 1 : ((lr >> 1) & 1) << 1);
  const uint32_t kstr = (uint32_t)a.ks * EB, vstr = (uint32_t)a.vs * EB;
  const uint32_t du = a.d / UE;  // units of a head in memory
  const int i0 = WK > 1 ? 0 : wave * NI;
  const char *kbase = (const char *)a.k + ((uint64_t)t.k0 * a.ks + (uint64_t)hk * a.d) * EB;
  const char *vbase = (const char *)a.v + ((uint64_t)t.k0 * a.vs + (uint64_t)hk * a.d) * EB;
  auto issue = [&](uint32_t s, uint32_t b) {
    // first key of the wavefront's rows in this stage; rows from kend on are
    // past the buffer and land as zeros
    const uint32_t key = kbeg + s * C::KEYS + (WK > 1 ? wave * 32 * KB : 0);
    const uint32_t rem = key < kend ? min(kend - key, 32u * KB) : 0;
    const uint32_t klen = rem ? (rem - 1) * kstr + a.d * EB : 0, vlen = rem ? (rem - 1) * vstr + a.d * EB : 0;
    const __amdgpu_buffer_rsrc_t rk = at_rsrc(kbase + (rem ? (uint64_t)key * kstr : 0), klen);
    const __amdgpu_buffer_rsrc_t rv = at_rsrc(vbase + (rem ? (uint64_t)key * vstr : 0), vlen);
    char *base = lds + b * C::STAGE + (WK > 1 ? wave * (C::STAGE / WK) : 0);
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      const uint32_t i = i0 + k, u = ku ^ (PU >= 8 ? (i * RPI) & 7 : 0);
      const uint32_t off = u < du ? u * 16 + (i * RPI + lr) * kstr : kAtOob;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (at_lds_void *)(base + i * 1024), 16, off, 0, 0, 0);
    }
    char *vb = base + C::STAGE / 2 / WK;
#pragma unroll
    for (int k = 0; k < NI; ++k) {
      const uint32_t i = i0 + k, u = vu ^ (F32 || PU < 8 ? 0 : ((i * RPI) & 3) << 1);
      const uint32_t off = u < du ? u * 16 + (i * RPI + lr) * vstr : kAtOob;
      __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (at_lds_void *)(vb + i * 1024), 16, off, 0, 0, 0);
    }
  };

  // LDS byte offsets of this lane's operands: K row l32, unit 2c + lh; V by
  // transposing reads (16 bit: 4 rows x 16 columns per 16 lanes) or one
  // element (fp32)
  const uint32_t ksw = PU >= 8 ? l32 & 7 : (l32 >> 1) & 3;
  const uint32_t vrow = F32 ? 4 * lh : 4 * lh + ((lane & 15) >> 2);
  const uint32_t vsw = PU >= 8 ? (vrow & 3) << 1 : ((vrow >> 1) & 1) << 1;

  f32x16 o[DB][NQ];
  float m[NQ], l[NQ];
#pragma unroll
  for (int n = 0; n < NQ; ++n) {
    m[n] = kAtLowest;
    l[n] = 0.0f;
#pragma unroll
    for (int db = 0; db < DB; ++db) o[db][n] = f32x16{};
  }

  auto compute = [&](uint32_t s, uint32_t b) {
    const uint32_t key = kbeg + s * C::KEYS + (WK > 1 ? wave * 32 * KB : 0);
    if (key >= min(kend, wmax)) return;
    const char *kt = lds + b * C::STAGE + (WK > 1 ? wave * (C::STAGE / WK) : 0);
    const char *vt = kt + C::STAGE / 2 / WK;
    f32x16 sc[KB][NQ];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) sc[kb][n] = f32x16{};
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        const u32x4 kv = *reinterpret_cast<const u32x4 *>(kt + (32 * kb + l32) * RB + (((2 * c + lh) ^ ksw) * 16));
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          if constexpr (F32) {
            const f32x4 k4 = __builtin_bit_cast(f32x4, kv), q4 = __builtin_bit_cast(f32x4, q[n][c]);
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[kb][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(k4[e], q4[e], sc[kb][n], 0, 0, 0);
          } else if constexpr (DT == DT_F16) {
            sc[kb][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, kv),
                                                               __builtin_bit_cast(f16x8, q[n][c]), sc[kb][n], 0, 0, 0);
          } else {
            sc[kb][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, kv),
                                                                __builtin_bit_cast(bf16x8, q[n][c]), sc[kb][n], 0, 0, 0);
          }
        }
      }
    }
    // lane l of a result holds query l32 and keys 8 (r / 4) + 4 lh + r % 4
    const bool masked = key + 32 * KB > min(kend, wmin);
    if (masked) {
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const uint32_t to = min(kend, lim[n]);
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int r = 0; r < 16; ++r)
            if (key + 32 * kb + 8 * (r / 4) + 4 * lh + r % 4 >= to) sc[kb][n][r] = -__builtin_huge_valf();
      }
    }
    u32x4 pb[KB][2][NQ];  // 16 bit: the packed probabilities of 16 keys
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      float mx = sc[0][n][0];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) mx = fmaxf(mx, sc[kb][n][r]);
      mx = at_pair_max(mx) * a.scale_log2;
      if (__any(mx > m[n] + kAtSlack)) {
        const float mn = fmaxf(m[n], mx), al = __builtin_amdgcn_exp2f(m[n] - mn);
        m[n] = mn;
        l[n] *= al;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r = 0; r < 16; ++r) o[db][n][r] *= al;
      }
      float sum = 0.0f;
      const float off = kAtBias<DT> - m[n];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[kb][n][r], a.scale_log2, off));
          sc[kb][n][r] = p;
          sum += p;
        }
        if constexpr (!F32) {
#pragma unroll
          for (int h = 0; h < 2; ++h)
            pb[kb][h][n] = u32x4{pack2<DT>(sc[kb][n][8 * h], sc[kb][n][8 * h + 1]),
                                 pack2<DT>(sc[kb][n][8 * h + 2], sc[kb][n][8 * h + 3]),
                                 pack2<DT>(sc[kb][n][8 * h + 4], sc[kb][n][8 * h + 5]),
                                 pack2<DT>(sc[kb][n][8 * h + 6], sc[kb][n][8 * h + 7])};
        }
      }
      l[n] += sum;
    }
    // O^T += V^T P^T; `clean`: infinite and NaN values of V count as zero
    auto pv = [&](auto clean) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        if constexpr (F32) {
#pragma unroll
          for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              uint32_t v = *reinterpret_cast<const uint32_t *>(vt + (32 * kb + 8 * (r / 4) + r % 4 + vrow) * RB +
                                                               (32 * db + l32) * 4);
              if constexpr (decltype(clean)::value) v = at_finite_only<DT>(v);
#pragma unroll
              for (int n = 0; n < NQ; ++n)
                o[db][n] = __builtin_amdgcn_mfma_f32_32x32x2f32(__uint_as_float(v), sc[kb][n][r], o[db][n], 0, 0, 0);
            }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int db = 0; db < DB; ++db) {
              const uint32_t unit = (4 * db + 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ vsw;
              const char *p = vt + (32 * kb + 16 * h + vrow) * RB + unit * 16 + (lane & 1) * 8;
              const s16x4 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)p);
              const s16x4 v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((at_lds_s16x4 *)(p + 8 * RB));
              u32x4 v = __builtin_bit_cast(u32x4, s16x8{v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]});
              if constexpr (decltype(clean)::value) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[e] = at_finite_only<DT>(v[e]);
              }
#pragma unroll
              for (int n = 0; n < NQ; ++n) {
                if constexpr (DT == DT_F16)
                  o[db][n] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, v),
                                                                    __builtin_bit_cast(f16x8, pb[kb][h][n]), o[db][n],
                                                                    0, 0, 0);
                else
                  o[db][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v),
                                                                     __builtin_bit_cast(bf16x8, pb[kb][h][n]), o[db][n],
                                                                     0, 0, 0);
              }
            }
        }
      }
    };
    // Keys that some rows see and others do not: 0 * NaN or 0 * inf of an
    // unseen value must not reach a row. If the tile holds such values, they
    // are added to the rows that see them one by one, and the product runs
    // without them.
    if (min(wmin, kend) < min(kend, key + 32 * KB)) {
      uint32_t bad = 0;
      for (int i = lane; i < 32 * KB * PU; i += 64) {
        const u32x4 v = *reinterpret_cast<const u32x4 *>(vt + i * 16);
#pragma unroll
        for (int e = 0; e < 4; ++e) bad |= at_nonfinite<DT>(v[e]);
      }
      if (__any(bad != 0)) {
        for (uint32_t j = 0; j < 32 * KB; ++j) {
#pragma unroll
          for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
              const uint32_t dim = 32 * db + 8 * r4 + 4 * lh;  // four dims of this lane
              const uint32_t sw = F32 ? 0 : PU >= 8 ? (j & 3) << 1 : ((j >> 1) & 1) << 1;
              const char *p = vt + j * RB + ((dim / UE) ^ sw) * 16 + (dim % UE) * EB;
              float v[4];
              if constexpr (F32) {
                const f32x4 x = *reinterpret_cast<const f32x4 *>(p);
                v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
              } else {
                const f32x4 x = unpack4<DT>(*reinterpret_cast<const u32x2 *>(p));
                v[0] = x.x, v[1] = x.y, v[2] = x.z, v[3] = x.w;
              }
#pragma unroll
              for (int e = 0; e < 4; ++e)
#pragma unroll
                for (int n = 0; n < NQ; ++n)
                  if (at_nonfinite<DT_F32>(__float_as_uint(v[e])) && key + j < min(kend, lim[n]))
                    o[db][n][4 * r4 + e] += v[e];
            }
        }
        pv(std::true_type{});
        return;
      }
    }
    pv(std::false_type{});
  };

  const uint32_t nst = kend > kbeg ? (kend - kbeg + C::KEYS - 1) / C::KEYS : 0;
#pragma unroll
  for (int s = 0; s < NST - 1; ++s) issue(s, s);
  uint32_t bc = 0, bi = NST - 1;
  for (uint32_t s = 0; s < nst; ++s) {
    if constexpr (WK > 1) {
      // the wavefront's own rows: its reads of the buffer that is requested
      // again are behind it
      __asm__ volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
      issue(s + NST - 1, bi);
      at_wait_vm<2 * NI * (NST - 1)>();
      __asm__ volatile("" ::: "memory");
    } else {
      at_wait_vm<2 * NI * (NST - 2)>();
      __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
      issue(s + NST - 1, bi);
    }
    compute(s, bc);
    bc = bc + 1 == NST ? 0 : bc + 1;
    bi = bi + 1 == NST ? 0 : bi + 1;
  }
  // nothing may still be on its way into LDS when it is reused or given back
  at_wait_vm<0>();

#pragma unroll
  for (int n = 0; n < NQ; ++n) l[n] = at_pair_sum(l[n]);

  const uint64_t rows_all = (uint64_t)a.tokens * a.hq;
  const uint64_t ml0 = attn_ws_ml(a);
  const uint32_t gpart = a.part0 + part;

  if constexpr (WK > 1) {
    // join the wavefronts' keys: a common maximum, scaled sums through LDS
    float *jo = reinterpret_cast<float *>(lds);
    float *jml = jo + WK * 32 * C::OPITCH;
    __syncthreads();
    if (lh == 0) {
      jml[wave * 64 + l32] = m[0];
      jml[wave * 64 + 32 + l32] = l[0];
    }
    __syncthreads();
    float mm = jml[l32];
#pragma unroll
    for (int w = 1; w < WK; ++w) mm = fmaxf(mm, jml[w * 64 + l32]);
    float ll = 0.0f;
#pragma unroll
    for (int w = 0; w < WK; ++w) ll += jml[w * 64 + 32 + l32] * __builtin_amdgcn_exp2f(jml[w * 64 + l32] - mm);
    const float f = __builtin_amdgcn_exp2f(m[0] - mm);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4)
        *reinterpret_cast<f32x4 *>(jo + (wave * 32 + l32) * C::OPITCH + 32 * db + 8 * r4 + 4 * lh) =
            f32x4{o[db][0][4 * r4], o[db][0][4 * r4 + 1], o[db][0][4 * r4 + 2], o[db][0][4 * r4 + 3]} * f;
    __syncthreads();
    // the row sums go where every thread finds them
    if (wave == 0 && lh == 0) {
      jml[l32] = mm;
      jml[32 + l32] = ll;
    }
    __syncthreads();
    for (uint32_t i = tid; i < 32 * (C::DP / 8); i += 64 * C::NW) {
      const uint32_t rr = i / (C::DP / 8), dim = (i - rr * (C::DP / 8)) * 8;
      const uint32_t row = t.row0 + rr;
      if (row >= nrows || dim >= a.d) continue;
      f32x4 x0{}, x1{};
#pragma unroll
      for (int w = 0; w < WK; ++w) {
        const float *p = jo + (w * 32 + rr) * C::OPITCH + dim;
        x0 += *reinterpret_cast<const f32x4 *>(p);
        x1 += *reinterpret_cast<const f32x4 *>(p + 4);
      }
      const uint32_t tok = row / a.g, hd = hk * a.g + (row - tok * a.g);
      const float lsum = jml[32 + rr];
      if (a.ws) {
        const uint64_t r = (uint64_t)gpart * rows_all + (uint64_t)(t.q0 + tok) * a.hq + hd;
        *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim) = x0;
        *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim + 4) = x1;
        if (dim == 0) {
          a.ws[ml0 + 2 * r] = jml[rr];
          a.ws[ml0 + 2 * r + 1] = lsum;
        }
      } else {
        const float inv = lsum == 0.0f ? 0.0f : 1.0f / lsum;
        x0 *= inv, x1 *= inv;
        const uint64_t e = (uint64_t)(t.q0 + tok) * a.os + (uint64_t)hd * a.d + dim;
        if constexpr (F32) {
          *reinterpret_cast<f32x4 *>((float *)a.o + e) = x0;
          *reinterpret_cast<f32x4 *>((float *)a.o + e + 4) = x1;
        } else {
          const u32x2 p0 = pack4<DT>(x0), p1 = pack4<DT>(x1);
          *reinterpret_cast<u32x4 *>((uint16_t *)a.o + e) = u32x4{p0.x, p0.y, p1.x, p1.y};
        }
      }
    }
  } else {
#pragma unroll
    for (int n = 0; n < NQ; ++n) {
      const uint32_t row = wrow + 32 * n + l32;
      const bool on = row < nrows;
      const uint32_t tok = row / a.g, hd = hk * a.g + (row - tok * a.g);
      if (a.ws) {
        if (!on) continue;
        const uint64_t r = (uint64_t)gpart * rows_all + (uint64_t)(t.q0 + tok) * a.hq + hd;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const uint32_t dim = 32 * db + 8 * r4 + 4 * lh;
            if (dim < a.d)
              *reinterpret_cast<f32x4 *>(a.ws + r * a.d + dim) = f32x4{o[db][n][4 * r4], o[db][n][4 * r4 + 1],
                                                                       o[db][n][4 * r4 + 2], o[db][n][4 * r4 + 3]};
          }
        if (lh == 0) {
          a.ws[ml0 + 2 * r] = m[n];
          a.ws[ml0 + 2 * r + 1] = l[n];
        }
        continue;
      }
      const float inv = l[n] == 0.0f ? 0.0f : 1.0f / l[n];
      const uint64_t e = (uint64_t)(t.q0 + tok) * a.os + (uint64_t)hd * a.d;
#pragma unroll
      for (int db = 0; db < DB; ++db) {
        if constexpr (F32) {
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const uint32_t dim = 32 * db + 8 * r4 + 4 * lh;
            if (on && dim < a.d)
              *reinterpret_cast<f32x4 *>((float *)a.o + e + dim) =
                  f32x4{o[db][n][4 * r4], o[db][n][4 * r4 + 1], o[db][n][4 * r4 + 2], o[db][n][4 * r4 + 3]} * inv;
          }
        } else {
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            // two runs of 4 dims in either half -> one run of 8 a lane
            u32x2 x[2];
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int r4 = 2 * k + y;
              x[y] = pack4<DT>(f32x4{o[db][n][4 * r4], o[db][n][4 * r4 + 1], o[db][n][4 * r4 + 2],
                                     o[db][n][4 * r4 + 3]} * inv);
            }
            const auto sx = __builtin_amdgcn_permlane32_swap(x[0].x, x[1].x, false, false);
            const auto sy = __builtin_amdgcn_permlane32_swap(x[0].y, x[1].y, false, false);
            const uint32_t dim = 32 * db + 8 * (2 * k + lh);
            if (on && dim < a.d)
              *reinterpret_cast<u32x4 *>((uint16_t *)a.o + e + dim) = u32x4{sx[0], sy[0], sx[1], sy[1]};
          }
        }
      }
    }
  }
}

template <int DT, class C>
hipError_t at_launch(const AttnArgs &a, hipStream_t st) {
  const uint64_t grid = (uint64_t)a.hkv * a.parts * a.tiles;
  if (grid == 0 || grid > 0x7fffffffu) return hipErrorInvalidValue;
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(attn_kernel<DT, C>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (attr != hipSuccess) return attr;
  hipLaunchKernelGGL((attn_kernel<DT, C>), dim3((uint32_t)grid), dim3(64 * C::NW), C::LDS, st, a);
  return hipGetLastError();
}

// The kernels of a head size: rows over 4 wavefronts, 64 or 32 keys a stage;
// or 32 rows, the keys over as many wavefronts as two stages leave room for.
template <int DT, int DP>
struct AtKernels {
  static constexpr int RB = (DP == 96 ? 128 : DP) * Storage<DT>::bytes;
  using Rows = AtCfg<DT, DP, 4, 1, 1, RB >= 512 ? 1 : 2, 2>;
  using Keys = AtCfg<DT, DP, 1, RB >= 512 ? 2 : 4, 1, 1, RB <= 128 ? 4 : 2>;
};
template <int DT>
struct AtKernels<DT, 256> {
  static constexpr int RB = 256 * Storage<DT>::bytes;
  using Rows = AtCfg<DT, 256, 4, 1, 1, 1, 2>;
  // fp32: one wavefront of keys, the rows of a stage are 64 KB
  using Keys = AtCfg<DT, 256, 1, RB >= 1024 ? 1 : 2, 1, 1, 2>;
};

template <int DT>
hipError_t at_launch_dt(const AttnArgs &a, int kernel, hipStream_t st) {
#define AIH_AT_CASE(DP)                                                                    \
  if (a.d <= DP)                                                                           \
    return kernel == AIH_ATTN_ROWS ? at_launch<DT, typename AtKernels<DT, DP>::Rows>(a, st) \
                                   : at_launch<DT, typename AtKernels<DT, DP>::Keys>(a, st);
  AIH_AT_CASE(32)
  AIH_AT_CASE(64)
  AIH_AT_CASE(96)
  AIH_AT_CASE(128)
  AIH_AT_CASE(256)
#undef AIH_AT_CASE
  return hipErrorInvalidValue;
}

}  // namespace
}  // namespace aih
