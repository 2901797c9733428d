// mx4_pw.hip -- the pointwise conv of microscaled 4-bit rows (aih_mx4_pw).
//
// y[i][n] = act(sum_b 2^(sx[i][b] + sw[n][b]) sum_{k in b} x w + bias[n]) + res[i][n].
// The scaled matrix instructions take the codes and the scale bytes as they are
// stored: a lane holds one row's block of 32 codes (16 bytes) and its scale.
// Weights are the A operand and pixels the B operand, so that a lane ends up with
// one pixel's channels.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <type_traits>

#include "aih_device.h"
#include "mx4.h"

namespace aih {
namespace {

typedef __attribute__((address_space(3))) void mx_lds_void;
typedef int i32x8 __attribute__((ext_vector_type(8)));

constexpr uint32_t kOob = 0x80000000u;  // a byte offset past every buffer

__device__ __forceinline__ __amdgpu_buffer_rsrc_t mx_rsrc(const void *base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void *>(base), 0, (int)bytes, 0x00020000);
}

// 16 bytes a lane from rs to LDS, lane after lane
__device__ __forceinline__ void mx_dma(__amdgpu_buffer_rsrc_t rs, char *to, uint32_t off, uint32_t soff) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(rs, (mx_lds_void *)to, 16, off, soff, 0, 0);
}

template <int N>
__device__ __forceinline__ void mx_wait_vm() {
  static_assert(N >= 0 && N < 64, "vmcnt");
  __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | 0x0F70);
}
// vmcnt(n) for a wavefront-uniform n in [0, MAXN]
template <int MAXN>
__device__ __forceinline__ void mx_wait_vm_n(uint32_t n) {
  if constexpr (MAXN > 0) {
    if (n >= (uint32_t)MAXN) {
      mx_wait_vm<MAXN>();
      return;
    }
    mx_wait_vm_n<MAXN - 1>(n);
  } else {
    mx_wait_vm<0>();
  }
}

// c + A B, both 4-bit; byte T of each lane's scale word is its block's scale.
template <int T>
__device__ __forceinline__ f32x16 mx_mfma32(u32x4 a, u32x4 b, f32x16 c, uint32_t sa, uint32_t sb) {
  const i32x8 a8 = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8 b8 = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(a8, b8, c, 4, 4, T, (int)sa, T, (int)sb);
}
__device__ __forceinline__ f32x4 mx_mfma16(u32x4 a, u32x4 b, f32x4 c, uint32_t sa, uint32_t sb) {
  const i32x8 a8 = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
  const i32x8 b8 = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a8, b8, c, 4, 4, 0, (int)sa, 0, (int)sb);
}

// act(v + bias) + res of four channels of a pixel
template <int DT>
__device__ __forceinline__ void mx_store4(const Mx4PwArgs &a, const Act &act, uint32_t i, uint32_t n, f32x4 v) {
  if (i >= a.m || n >= a.cout) return;
  if (a.bias) v += Vec4IO<DT>::load(a.bias, n / 4);
  v = act4(act, v);
  const size_t at = (size_t)i * (a.cout / 4) + n / 4;
  if (a.res) v += Vec4IO<DT>::load(a.res, at);
  Vec4IO<DT>::store(a.y, at, v);
}

// ---------------------------------------------------------------- few pixels
//
// Up to 32 pixels: the weights' bytes are the floor, but what bounds it is waiting for them:
// 16 x 8192 x 8192 takes 17 us, 2.1 TB/s where a large copy reaches 5.1, 8 x 4096 x 4096 5.7
// with wavefronts waiting for 69 % of their time (half a cache line a row and stage, two stages
// on their way, a load for every byte of scales). A workgroup owns 16 channels, its W
// wavefronts take turns at the stages of 128 elements, operands straight into registers
// (a lane: channel lane % 16, block lane / 16 of the stage, 64 contiguous bytes a row),
// and the partial sums are joined in LDS in the wavefronts' order.
template <int DT, int TM, int W>
__global__ __launch_bounds__(64 * W) void mx4_pw_few_kernel(Mx4PwArgs a) {
  __shared__ f32x4 part[W][TM][64];
  const uint32_t lane = threadIdx.x & 63, r = lane & 15, b = lane >> 4;
  const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const uint32_t n0 = blockIdx.x * 16, nw = min(16u, a.cout - n0);
  const __amdgpu_buffer_rsrc_t rwc = mx_rsrc(a.wc + (uint64_t)n0 * a.cb, nw * a.cb);
  const __amdgpu_buffer_rsrc_t rws = mx_rsrc(a.ws + (uint64_t)n0 * a.sb, nw * a.sb);
  const __amdgpu_buffer_rsrc_t rxc = mx_rsrc(a.xc, a.m * a.cb), rxs = mx_rsrc(a.xs, a.m * a.sb);
  f32x4 acc[TM];
#pragma unroll
  for (int t = 0; t < TM; ++t) acc[t] = f32x4{};
  constexpr int U = 2;  // stages on their way
  for (uint32_t s0 = wave; s0 < a.nst; s0 += U * W) {
    u32x4 wc[U], xc[U][TM];
    uint32_t ws[U], xs[U][TM];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint32_t s = s0 + u * W;
      const bool on = s < a.nst;
      wc[u] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rwc, on ? r * a.cb + s * 64 + b * 16 : kOob, 0, 0));
      ws[u] = __builtin_amdgcn_raw_buffer_load_b8(rws, on ? r * a.sb + s * 4 + b : kOob, 0, 0);
#pragma unroll
      for (int t = 0; t < TM; ++t) {
        xc[u][t] = __builtin_bit_cast(u32x4, __builtin_amdgcn_raw_buffer_load_b128(rxc, on ? (16 * t + r) * a.cb + s * 64 + b * 16 : kOob, 0, 0));
        xs[u][t] = __builtin_amdgcn_raw_buffer_load_b8(rxs, on ? (16 * t + r) * a.sb + s * 4 + b : kOob, 0, 0);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int t = 0; t < TM; ++t) acc[t] = mx_mfma16(wc[u], xc[u][t], acc[t], ws[u], xs[u][t]);
  }
#pragma unroll
  for (int t = 0; t < TM; ++t) part[wave][t][lane] = acc[t];
  __syncthreads();
  const Act act = act_params(a.act);
  for (uint32_t t = wave; t < TM; t += W) {
    f32x4 v = part[0][t][lane];
#pragma unroll
    for (int w = 1; w < W; ++w) v += part[w][t][lane];
    mx_store4<DT>(a, act, 16 * t + r, n0 + 4 * b, v);
  }
}

// ---------------------------------------------------------------- tiles
//
// WM x WN wavefronts of TM x TN blocks of 32 pixels x 32 channels. Stages of U
// blocks of 32 elements (16 U bytes a row; 8 are a whole cache line) come into LDS by
// DMA: while a stage is worked on the next NST - 1 are in LDS or on their way; the scales
// of 16 blocks a row come with every 16 / U-th one. Unit u of tile row r is at slot
// u ^ mx_swz(r), which spreads 16 rows' units over the banks.
//
// A stage is U / 2 products of 64 elements. The operands of each are read while the
// one before it runs, those of the next stage's first too, so that the matrix unit has a
// product's work in registers when the wavefronts meet. 8192 cubed takes 285 us, 3.85
// PFLOP/s, where the matrix unit alone reaches 7.1; without the copies it took 230, without
// the products 236: neither alone is the bound, and the reads from LDS (six operands for eight
// products of a wavefront) keep the matrix unit from its rate even without copies. With the products of a stage
// behind its barrier, and half a cache line a row, it took 353.
template <int WM_, int WN_, int TM_, int TN_, int NST_, int U_>
struct MxTile {
  static constexpr int WM = WM_, WN = WN_, TM = TM_, TN = TN_, NST = NST_, U = U_;
  static constexpr int NW = WM * WN, BM = 32 * WM * TM, BN = 32 * WN * TN;
  static constexpr int RB = 16 * U, RPI = 64 / U;                 // bytes of a row, rows of a DMA instruction
  static constexpr uint32_t STAGE = (BM + BN) * RB;
  static constexpr int CX = BM / RPI, CI = CX + BN / RPI;         // DMA instructions of a stage
  static constexpr int G = 16 / U;                                // stages of a group of scales
  static constexpr int SX = (BM + 63) / 64, SI = SX + (BN + 63) / 64;
  static constexpr uint32_t SCALES = SI * 1024;
  static constexpr int CW = TN % 2 == 0 ? 64 : 32, PITCH = CW + 4;  // channels of a staged pixel, its floats
  static constexpr uint32_t OUT = NW * 32u * PITCH * 4u, IN = NST * STAGE + 2 * SCALES;
  static constexpr uint32_t LDS = IN > OUT ? IN : OUT;
  // two groups of scales at a time
  static_assert((U == 4 || U == 8) && NST >= 2 && NST <= G && LDS <= 160 * 1024, "LDS");
};
template <class C>
__device__ __forceinline__ uint32_t mx_swz(uint32_t r) {
  return C::U == 4 ? (r >> 2) & 3 : (r >> 1) & 7;
}

// The operands of 64 elements.
template <class C>
struct MxOperands {
  u32x4 x[C::TM], w[C::TN];
  // `at`: where the lane's unit is in its rows
  __device__ __forceinline__ void read(const char *px, const char *pw, uint32_t at) {
#pragma unroll
    for (int j = 0; j < C::TN; ++j) w[j] = *reinterpret_cast<const u32x4 *>(pw + j * 32 * C::RB + at);
#pragma unroll
    for (int i = 0; i < C::TM; ++i) x[i] = *reinterpret_cast<const u32x4 *>(px + i * 32 * C::RB + at);
  }
};
// The scales of a stage: byte T of a word is that of product T.
template <class C>
struct MxScales {
  uint32_t x[C::TM], w[C::TN];
  using Word = std::conditional_t<C::U == 4, uint16_t, uint32_t>;
  __device__ __forceinline__ void read(const char *px, const char *pw) {
#pragma unroll
    for (int j = 0; j < C::TN; ++j) w[j] = *reinterpret_cast<const Word *>(pw + j * 512);
#pragma unroll
    for (int i = 0; i < C::TM; ++i) x[i] = *reinterpret_cast<const Word *>(px + i * 512);
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int j = 0; j < C::TN; ++j) w[j] = 0;
#pragma unroll
    for (int i = 0; i < C::TM; ++i) x[i] = 0;
  }
};
template <class C, int T>
__device__ __forceinline__ void mx_product(const MxOperands<C> &p, const MxScales<C> &s, f32x16 (&acc)[C::TM][C::TN]) {
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j) acc[i][j] = mx_mfma32<T>(p.w[j], p.x[i], acc[i][j], s.w[j], s.x[i]);
}
// Products are no memory accesses, and the compiler moves them down, past the barrier
// and the next reads; an empty text that takes the sums keeps them here.
template <class C>
__device__ __forceinline__ void mx_pin(f32x16 (&acc)[C::TM][C::TN]) {
#pragma unroll
  for (int i = 0; i < C::TM; ++i)
#pragma unroll
    for (int j = 0; j < C::TN; ++j) __asm__ volatile("" : "+v"(acc[i][j])::"memory");
}

template <int DT, class C>
__global__ __launch_bounds__(64 * C::NW, 2) void mx4_pw_kernel(Mx4PwArgs a) {
  constexpr int TM = C::TM, TN = C::TN, NW = C::NW, NST = C::NST;
  constexpr int CK = (C::CI + NW - 1) / NW, SK = (C::SI + NW - 1) / NW;
  extern __shared__ __align__(16) char lds[];
  const int lane = threadIdx.x & 63, l32 = lane & 31, lh = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave % C::WM, wn = wave / C::WM;

  // tiles in groups of 8 rows of them: those that run at once share operands
  const uint32_t t = xcd_remap(blockIdx.x, gridDim.x, a.nxcd);
  const uint32_t group = t / (8 * a.ntiles), first = group * 8, rows = min(a.mtiles - first, 8u);
  const uint32_t rest = t - group * 8 * a.ntiles, nt = rest / rows, mt = first + (rest - nt * rows);
  const uint32_t m0 = mt * C::BM, n0 = nt * C::BN;
  const uint32_t mr = min(a.m - m0, (uint32_t)C::BM), nr = min(a.cout - n0, (uint32_t)C::BN);

  const __amdgpu_buffer_rsrc_t rxc = mx_rsrc(a.xc + (uint64_t)m0 * a.cb, mr * a.cb);
  const __amdgpu_buffer_rsrc_t rwc = mx_rsrc(a.wc + (uint64_t)n0 * a.cb, nr * a.cb);
  const __amdgpu_buffer_rsrc_t rxs = mx_rsrc(a.xs + (uint64_t)m0 * a.sb, mr * a.sb);
  const __amdgpu_buffer_rsrc_t rws = mx_rsrc(a.ws + (uint64_t)n0 * a.sb, nr * a.sb);

  // Instruction i of a stage: tile rows RPI i + lane / U (pixels, then channels).
  // The last stage may be half a one.
  uint32_t coff[CK];
  bool past[CK];  // the unit is in the second half
#pragma unroll
  for (int k = 0; k < CK; ++k) {
    const int i = wave + k * NW;
    const uint32_t r = (i < C::CX ? C::RPI * i : C::RPI * (i - C::CX)) + lane / C::U;
    const uint32_t u = (uint32_t)(lane % C::U) ^ mx_swz<C>(r);
    coff[k] = r < (i < C::CX ? mr : nr) ? r * a.cb + u * 16 : kOob;
    past[k] = u >= 4;
  }
  const uint32_t nst = C::U == 4 ? a.nst : (a.nst + 1) / 2;
  const bool odd = C::U == 8 && (a.nst & 1);
  uint32_t soff[SK];
#pragma unroll
  for (int k = 0; k < SK; ++k) {
    const int i = wave + k * NW;
    const uint32_t r = (i < C::SX ? 64 * i : 64 * (i - C::SX)) + lane;
    soff[k] = r < (i < C::SX ? mr : nr) ? r * a.sb : kOob;
  }
  const uint32_t nc = C::CI % NW == 0 ? CK : (C::CI - wave + NW - 1) / NW;  // this wavefront's
  const uint32_t ns = C::SI % NW == 0 ? SK : C::SI > wave ? (C::SI - wave + NW - 1) / NW : 0;

  // requests stage s; stages are requested in order
  auto issue = [&](uint32_t s, uint32_t buf) {
    if (s % C::G == 0) {
      char *to = lds + NST * C::STAGE + (s / C::G & 1) * C::SCALES;
#pragma unroll
      for (int k = 0; k < SK; ++k) {
        const int i = wave + k * NW;
        if (C::SI % NW != 0 && i >= C::SI) break;
        if (i < C::SX) mx_dma(rxs, to + i * 1024, soff[k], s * C::U);
        else mx_dma(rws, to + i * 1024, soff[k], s * C::U);
      }
    }
    char *to = lds + buf * C::STAGE;
#pragma unroll
    for (int k = 0; k < CK; ++k) {
      const int i = wave + k * NW;
      if (C::CI % NW != 0 && i >= C::CI) break;
      const uint32_t off = odd && s == nst - 1 && past[k] ? kOob : coff[k];
      if (i < C::CX) mx_dma(rxc, to + i * 1024, off, s * C::RB);
      else mx_dma(rwc, to + i * 1024, off, s * C::RB);
    }
  };
  // waits for stage s, of the stages up to `last` that are requested
  auto arrived = [&](uint32_t s, uint32_t last) {
    const uint32_t later = last > s ? last - s : 0;
    const uint32_t scales = later && last / C::G != s / C::G ? ns : 0;
    mx_wait_vm_n<CK * (NST - 1) + SK>(later * nc + scales);
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = f32x16{};

  const uint32_t pr = 32 * TM * wm + l32, cr = 32 * TN * wn + l32;  // the lane's first rows
  // half h takes blocks h U / 2 .. of a stage, one a product
  constexpr int NP = C::U / 2;
  uint32_t at[NP];
#pragma unroll
  for (int T = 0; T < NP; ++T) at[T] = ((NP * lh + T) ^ mx_swz<C>(l32)) * 16;
  const char *px = lds + pr * C::RB, *pw = lds + (C::BM + cr) * C::RB;
  const char *sx = lds + NST * C::STAGE + pr * 16 + NP * lh;
  const char *sn = lds + NST * C::STAGE + C::SX * 1024 + cr * 16 + NP * lh;
  auto scale_at = [&](uint32_t s) { return (s / C::G & 1) * C::SCALES + (s % C::G) * C::U; };

#pragma unroll
  for (int s = 0; s < NST; ++s)
    if ((uint32_t)s < nst) issue(s, s);
  arrived(0, min(nst, (uint32_t)NST) - 1);
  // A bare barrier: a workgroup fence would wait for the copies on their way.
  __asm__ volatile("s_barrier" ::: "memory");
  MxOperands<C> p[2];
  MxScales<C> sc, sc_next;
  sc.read(sx, sn);
  if (odd && nst == 1 && lh) sc.clear();  // no scales: whatever is behind the row's
  p[0].read(px, pw, at[0]);
  uint32_t buf = 0;  // stage s's
  for (uint32_t s = 0; s < nst; ++s) {
    const uint32_t cur = buf * C::STAGE, next_buf = buf + 1 == NST ? 0 : buf + 1, next = next_buf * C::STAGE;
    p[1].read(px + cur, pw + cur, at[1]);
    mx_product<C, 0>(p[0], sc, acc);
    mx_pin<C>(acc);
    if constexpr (C::U == 8) {
      p[0].read(px + cur, pw + cur, at[NP - 2]);
      mx_product<C, 1>(p[1], sc, acc);
      mx_pin<C>(acc);
      p[1].read(px + cur, pw + cur, at[NP - 1]);
      mx_product<C, NP - 2>(p[0], sc, acc);
      mx_pin<C>(acc);
    }
    // the next stage is there for every wavefront, and all have read this one
    arrived(s + 1, min(nst - 1, s + NST - 1));
    __asm__ volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    if (s + NST < nst) issue(s + NST, buf);
    sc_next.read(sx + scale_at(s + 1), sn + scale_at(s + 1));  // behind the last stage: something, and not used
    p[0].read(px + next, pw + next, at[0]);
    mx_product<C, NP - 1>(p[1], sc, acc);
    mx_pin<C>(acc);
    sc = sc_next;
    if (odd && s + 2 == nst && lh) sc.clear();
    buf = next_buf;
  }
  __syncthreads();  // the buffers become the wavefronts' staging rows

  // act(acc + bias) + res, whole runs of a pixel's channels
  const Act act = act_params(a.act);
  constexpr bool F32 = DT == DT_F32;
  constexpr int CW = C::CW, PITCH = C::PITCH, CB = CW / 32;
  constexpr int CPL = F32 ? 4 : 8, LPR = CW / CPL, PPI = 64 / LPR;  // channels of a lane, lanes of a pixel, pixels at once
  float *st = reinterpret_cast<float *>(lds) + wave * 32 * PITCH;
  const bool row16 = F32 || a.cout % 8 == 0;  // 16-byte runs stay aligned from pixel to pixel
  const uint32_t rl = lane / LPR, cl = (lane % LPR) * CPL;
#pragma unroll
  for (int j0 = 0; j0 < TN; j0 += CB) {
    const uint32_t n = n0 + 32 * (TN * wn + j0) + cl;
    const bool n_ok = n < a.cout, two = !F32 && n + 8 <= a.cout;
    const f32x4 b0 = a.bias && n_ok ? Vec4IO<DT>::load(a.bias, n / 4) : f32x4{};
    const f32x4 b1 = a.bias && two ? Vec4IO<DT>::load(a.bias, n / 4 + 1) : f32x4{};
#pragma unroll
    for (int i = 0; i < TM; ++i) {
#pragma unroll
      for (int j = 0; j < CB; ++j)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4)
          *reinterpret_cast<f32x4 *>(st + l32 * PITCH + 32 * j + 8 * r4 + 4 * lh) =
              f32x4{acc[i][j0 + j][4 * r4], acc[i][j0 + j][4 * r4 + 1], acc[i][j0 + j][4 * r4 + 2], acc[i][j0 + j][4 * r4 + 3]};
      __builtin_amdgcn_wave_barrier();
#pragma unroll 2
      for (int g = 0; g < 32 / PPI; ++g) {
        const uint32_t r = g * PPI + rl, m = m0 + 32 * (TM * wm + i) + r;
        if (m >= a.m || !n_ok) continue;
        const size_t vi = (size_t)m * (a.cout / 4) + n / 4;
        f32x4 v0 = *reinterpret_cast<const f32x4 *>(st + r * PITCH + cl) + b0;
        if constexpr (F32) {
          v0 = act4(act, v0);
          if (a.res) v0 += reinterpret_cast<const f32x4 *>(a.res)[vi];
          reinterpret_cast<f32x4 *>(a.y)[vi] = v0;
        } else {
          f32x4 v1 = *reinterpret_cast<const f32x4 *>(st + r * PITCH + cl + 4) + b1;
          float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
          act_array<8>(act, v);
          v0 = f32x4{v[0], v[1], v[2], v[3]}, v1 = f32x4{v[4], v[5], v[6], v[7]};
          if (a.res) {
            if (row16) {
              const u32x4 x = reinterpret_cast<const u32x4 *>(a.res)[vi / 2];
              v0 += unpack4<DT>(u32x2{x.x, x.y}), v1 += unpack4<DT>(u32x2{x.z, x.w});
            } else {
              v0 += Vec4IO<DT>::load(a.res, vi);
              if (two) v1 += Vec4IO<DT>::load(a.res, vi + 1);
            }
          }
          const u32x2 lo = pack4<DT>(v0), hi = pack4<DT>(v1);
          if (row16) {
            reinterpret_cast<u32x4 *>(a.y)[vi / 2] = u32x4{lo.x, lo.y, hi.x, hi.y};
          } else {
            reinterpret_cast<u32x2 *>(a.y)[vi] = lo;
            if (two) reinterpret_cast<u32x2 *>(a.y)[vi + 1] = hi;
          }
        }
      }
      __builtin_amdgcn_wave_barrier();
    }
  }
}

template <int DT, class C>
hipError_t launch_tile(Mx4PwArgs a, hipStream_t st) {
  static const hipError_t attr = hipFuncSetAttribute(reinterpret_cast<const void *>(mx4_pw_kernel<DT, C>),
                                                     hipFuncAttributeMaxDynamicSharedMemorySize, C::LDS);
  if (attr != hipSuccess) return attr;
  a.mtiles = (a.m + C::BM - 1) / C::BM, a.ntiles = (a.cout + C::BN - 1) / C::BN;
  if ((uint64_t)a.mtiles * a.ntiles * (64 * C::NW) > 0xffffffffu) return hipErrorInvalidValue;
  hipLaunchKernelGGL((mx4_pw_kernel<DT, C>), dim3(a.mtiles * a.ntiles), dim3(64 * C::NW), C::LDS, st, a);
  return hipGetLastError();
}

template <int DT, int TM>
hipError_t launch_few(const Mx4PwArgs &a, hipStream_t st) {
  const dim3 grid((a.cout + 15) / 16);
  if (a.nst >= 32) hipLaunchKernelGGL((mx4_pw_few_kernel<DT, TM, 16>), grid, dim3(1024), 0, st, a);
  else hipLaunchKernelGGL((mx4_pw_few_kernel<DT, TM, 4>), grid, dim3(256), 0, st, a);
  return hipGetLastError();
}

// Measured, bf16, us, calls in a row: 8192 cubed with tiles of 256 x 256 289, 128 x 128 356, 64 x 128 483;
// 4096 cubed 40.6 | 48 | 63; 2048 cubed 20 | 12.0 | 11.0, 64 x 64 12.0; 1024 x 4096 x 4096 32 |
// 17.9 | 17.7 | 20.1; 3000 x 4096 x 4096 34.8 | 39 | 48; 5000 x 8192 x 1000 54 | 39 | 48; 300 x
// 4096 x 4096 31 | 15.5 | 13.0 | 11.6. A short sum gives little
// to overlap within a workgroup, so stages are half as long and more workgroups
// share a CU: 46080 x 960 x 160 with a residual, 128 x 128, long and short stages 23.0
// | 17.4, 46080 x 192 x 768 28.4 | 21.4, 184320 x 64 x 64, 64 x 64, 12.8 | 9.8. Few pixels,
// split over wavefronts | tiles of 64 x 64: 8 x 4096 x 4096 6.3 | 7.9, 20 6.5 | 8.2, 48 10.0 | 8.6.
template <int DT>
hipError_t launch_dt(const Mx4PwArgs &a, hipStream_t st) {
  if (a.m <= 16) return launch_few<DT, 1>(a, st);
  if (a.m <= 32) return launch_few<DT, 2>(a, st);
  auto tiles = [&](uint32_t bm, uint32_t bn) { return (uint64_t)((a.m + bm - 1) / bm) * ((a.cout + bn - 1) / bn); };
  const uint64_t cus = device_cus(), big = tiles(256, 256), mid = tiles(128, 128);
  if (a.nst < 16) {
    // a launch takes less than 2^24 workgroups of 256 threads
    if ((a.cout > 64 && mid >= cus) || tiles(64, 64) >> 24) return launch_tile<DT, MxTile<2, 2, 2, 2, 2, 4>>(a, st);
    return launch_tile<DT, MxTile<2, 2, 1, 1, 2, 4>>(a, st);
  }
  // rounds of tiles; one of 128 x 128, two a CU, takes 0.6 of one of 256 x 256
  const uint64_t big_rounds = (big + cus - 1) / cus, mid_rounds = (mid + 2 * cus - 1) / (2 * cus);
  if (10 * big_rounds <= 6 * mid_rounds) return launch_tile<DT, MxTile<2, 4, 4, 2, 2, 8>>(a, st);
  if (mid > cus) return launch_tile<DT, MxTile<2, 2, 2, 2, 2, 8>>(a, st);
  if (tiles(64, 128) >= cus) return launch_tile<DT, MxTile<2, 2, 1, 2, 2, 8>>(a, st);
  return launch_tile<DT, MxTile<2, 2, 1, 1, 2, 8>>(a, st);
}

}  // namespace

hipError_t launch_mx4_pw(const Mx4PwArgs &a, int dt, hipStream_t st) {
  return dt == DT_F32 ? launch_dt<DT_F32>(a, st) : dt == DT_F16 ? launch_dt<DT_F16>(a, st) : launch_dt<DT_BF16>(a, st);
}

}  // namespace aih
