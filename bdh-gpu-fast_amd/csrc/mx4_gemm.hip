// Products with 4-bit weights for gfx950 (bdh_mx4_gemm):
//
//   out[h, m, n] = [mul[h, m, n] *] [relu] sum_k a[h, m, k] wt[h, n, k]
//
// a in bf16: the weights become bf16 in registers (exact: two significant bits
// and a power of two) and meet a on the bf16 matrix instructions.  a in mx4: the
// scaled 4-bit instructions take codes and scale bytes as they lie in memory, at
// four times that rate.
//
// Two kernels.  Few rows (a generate step) are bound by the weights' bytes:
// k_mx4_few streams them from memory into registers.  Many rows
// are bound by the matrix cores: k_mx4_tile stages both operands through an LDS
// ring.  Where either has too few workgroups for the chip, K goes in splits, whose
// fp32 partials k_mx4_sum adds up in their order before the epilogue.
#include <algorithm>
#include <utility>

#include "few.h"
#include "lds_dma.h"
#include "mx4.h"

namespace bdh {
namespace {

struct MxGemmArgs {
  View a;    // bf16 (1, H, M, K), or
  View4 a4;  // mx4
  View4 w;   // (1, H, N, K)
  View mul;  // (1, H, M, N), p null: none
  View o;
  int64_t M, N, K, kb;
  int64_t Np;   // columns of a partial's row (N to a multiple of 8)
  float* part;  // [split][H][M][Np]; null: one split, which writes o
  int relu, mul_bf16;
  int vec_a;  // rows of a in 16-byte pieces
  int vec_o;  // rows of out (and of mul) in pieces of eight
  int vec4;   // and of four
  int splits, steps;  // steps of K in all
  int H, mt, nt;
};

__device__ __forceinline__ bf16x8 as_bf8(u32x4 w) { return __builtin_bit_cast(bf16x8, w); }

template <typename F, int... I>
__device__ __forceinline__ void static_for_impl(F&& f, std::integer_sequence<int, I...>) {
  (f(std::integral_constant<int, I>()), ...);
}
template <int N, typename F>
__device__ __forceinline__ void static_for(F&& f) {
  static_for_impl(f, std::make_integer_sequence<int, N>());
}

typedef int i32x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ i32x8 as_i8(u32x4 w) {  // (a 4-bit operand is the first four)
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  const i32x4 x = __builtin_bit_cast(i32x4, w);
  return __builtin_shufflevector(x, x, 0, 1, 2, 3, -1, -1, -1, -1);
}

// ---------------------------------------------------------------- epilogue
__device__ __forceinline__ float gemm_act(const MxGemmArgs& g, float v) {
  return g.relu ? (v != v ? v : fmaxf(v, 0.f)) : v;
}
__device__ __forceinline__ float gemm_mul(const MxGemmArgs& g, int64_t at) {
  return g.mul_bf16 ? to_f(static_cast<const bf16_t*>(g.mul.p)[at]) : static_cast<const float*>(g.mul.p)[at];
}

// Eight sums of columns n .. n + 7 of row (h, m) to out.
template <typename TO>
__device__ __forceinline__ void gemm_out8(const MxGemmArgs& g, int h, int64_t m, int64_t n, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = gemm_act(g, v[e]);
  TO* op = static_cast<TO*>(const_cast<void*>(g.o.p)) + h * g.o.s1 + m * g.o.s2 + n;
  const int64_t at = h * g.mul.s1 + m * g.mul.s2 + n;
  if (g.vec_o) {
    if (g.mul.p != nullptr) {
      if (g.mul_bf16) {
        const u32x4 x = *reinterpret_cast<const u32x4*>(static_cast<const bf16_t*>(g.mul.p) + at);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint32_t xe = x[e];
          v[2 * e] *= __uint_as_float(xe << 16);
          v[2 * e + 1] *= __uint_as_float(xe & 0xffff0000u);
        }
      } else {
        const float* x = static_cast<const float*>(g.mul.p) + at;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] *= x[e];
      }
    }
    if constexpr (sizeof(TO) == 2) {
      *reinterpret_cast<u32x4*>(op) =
          u32x4{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7])};
    } else {
      reinterpret_cast<f32x4*>(op)[0] = f32x4{v[0], v[1], v[2], v[3]};
      reinterpret_cast<f32x4*>(op)[1] = f32x4{v[4], v[5], v[6], v[7]};
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (n + e < g.N) {
        if (g.mul.p != nullptr) v[e] *= gemm_mul(g, at + e);
        op[e] = from_f<TO>(v[e]);
      }
  }
}

// out from the splits' partials, eight columns a thread; with few outputs G threads of
// each take every G-th split (a chain of loads otherwise: 8 rows of 256, 32 splits
// 8.7 -> 4.8 us) and their sums are added in order through LDS.
template <typename TO, int G>
__global__ __launch_bounds__(256) void k_mx4_sum(const MxGemmArgs g) {
  __shared__ f32x4 sums[G > 1 ? G : 1][G > 1 ? 256 / G : 1][2];
  const int l = threadIdx.x % (256 / G), grp = threadIdx.x / (256 / G);
  const int64_t each = g.Np / 8, rows = g.H * g.M, i = int64_t(blockIdx.x) * (256 / G) + l;
  const bool in = i < rows * each;
  const int64_t row = in ? i / each : 0, n = in ? (i - row * each) * 8 : 0;
  const float* p = g.part + row * g.Np + n;
  f32x4 lo{0, 0, 0, 0}, hi{0, 0, 0, 0};
#pragma unroll 4
  for (int s = grp; s < g.splits; s += G) {
    lo += reinterpret_cast<const f32x4*>(p + s * rows * g.Np)[0];
    hi += reinterpret_cast<const f32x4*>(p + s * rows * g.Np)[1];
  }
  if constexpr (G > 1) {
    sums[grp][l][0] = lo;
    sums[grp][l][1] = hi;
    __syncthreads();
    if (grp != 0) return;
#pragma unroll
    for (int u = 1; u < G; ++u) {
      lo += sums[u][l][0];
      hi += sums[u][l][1];
    }
  }
  if (!in) return;
  float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
  const int64_t h = row / g.M;
  gemm_out8<TO>(g, int(h), row - h * g.M, n, v);
}

// --------------------------------------------------------------- few rows
// A wave 32 rows of wt and 32 of a, a step two blocks (64 of K): lane l holds
// row l % 32 and block 2 s + l / 32 of each.  kFewSteps steps' loads are in flight
// together: the codes in 128-byte pieces of rows, which LDS turns to the lanes of their blocks
// (loaded there by the lanes themselves, 32 bytes of a row at a time and past the L2, 3 rows
// of 4 x 8192 x 13504 took 174 us, 8 of 28672 x 4096 44; so 87 and 24).  WK of a workgroup's
// waves take one tile's K in turn ranges and add up through LDS; the others take further tiles.
constexpr int kFewSteps = 4;  // (eight blocks, as the pieces and an 8-byte load of their scales have)
constexpr int64_t kFewRows = 65535 * 32;  // (its grid's second dimension)

template <bool A4, typename TO, int WK>
__global__ __launch_bounds__(256) void k_mx4_few(const MxGemmArgs g) {
  __shared__ float red[WK > 1 ? 4 : 1][WK > 1 ? 16 * 64 : 1];
  __shared__ u32x4 turn[4][256];
  const int lane = threadIdx.x & 63, l32 = lane & 31, hl = lane >> 5, wave = threadIdx.x >> 6;
  const int h = blockIdx.z / g.splits, split = blockIdx.z - h * g.splits;
  const int64_t n0 = (int64_t(blockIdx.x) * (4 / WK) + wave / WK) * 32, m0 = int64_t(blockIdx.y) * 32;
  const int64_t nr = min(n0 + l32, g.N - 1), mr = min(m0 + l32, g.M - 1);
  // this wave's steps
  const int per = g.splits * WK, part = split * WK + wave % WK;
  const int64_t c0 = 2 * (int64_t(g.steps) * part / per), c1 = min(2 * (int64_t(g.steps) * (part + 1) / per), g.kb);
  const uint8_t* wq = g.w.q + h * g.w.q1 + nr * g.w.q2;
  const uint8_t* wp[4];  // piece lane % 8 of rows 8 u + lane / 8
#pragma unroll
  for (int u = 0; u < 4; ++u)
    wp[u] = g.w.q + h * g.w.q1 + min(n0 + 8 * u + lane / 8, g.N - 1) * g.w.q2 + 16 * (lane & 7);
  const uint8_t* ws = g.w.s + h * g.w.s1 + nr * g.w.s2;
  const bf16_t* ap = static_cast<const bf16_t*>(g.a.p) + h * g.a.s1 + mr * g.a.s2;
  const uint8_t* aq = g.a4.q + h * g.a4.q1 + mr * g.a4.q2;
  const uint8_t* as = g.a4.s + h * g.a4.s1 + mr * g.a4.s2;
  // the factors, loaded beside the operands
  const int64_t mat = h * g.mul.s1 + mr * g.mul.s2;
  float mulv[16];
  if (g.vec4 && g.mul.p != nullptr && g.part == nullptr) {
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int64_t n = min(n0 + 8 * q + 4 * hl, g.N - 4);
      if (g.mul_bf16) {
        const u32x2 w = *reinterpret_cast<const u32x2*>(static_cast<const bf16_t*>(g.mul.p) + mat + n);
        const uint32_t w0 = w.x, w1 = w.y;
        mulv[4 * q] = __uint_as_float(w0 << 16);
        mulv[4 * q + 1] = __uint_as_float(w0 & 0xffff0000u);
        mulv[4 * q + 2] = __uint_as_float(w1 << 16);
        mulv[4 * q + 3] = __uint_as_float(w1 & 0xffff0000u);
      } else {
        const f32x4 w = *reinterpret_cast<const f32x4*>(static_cast<const float*>(g.mul.p) + mat + n);
#pragma unroll
        for (int e = 0; e < 4; ++e) mulv[4 * q + e] = w[e];
      }
    }
  }
  f32x16 acc;
#pragma unroll
  for (int r = 0; r < 16; ++r) acc[r] = 0.f;
  for (int64_t c = c0 + hl; c - hl < c1 && n0 < g.N; c += 2 * kFewSteps) {
    u32x4 w[kFewSteps], x[kFewSteps][A4 ? 1 : 4];
    uint32_t sw[kFewSteps], sa[kFewSteps];
    const int64_t c8 = c - hl;
    const bool whole = c8 + 2 * kFewSteps <= c1;  // eight blocks (the same for a wave's lanes)
    uint64_t sw8 = 0;
    u32x4 wt[4];
    if (whole) {
      __builtin_memcpy(&sw8, ws + c8, 8);
#pragma unroll
      for (int u = 0; u < 4; ++u) wt[u] = *reinterpret_cast<const u32x4*>(wp[u] + 16 * c8);
    }
#pragma unroll
    for (int s = 0; s < kFewSteps; ++s) {
      const int64_t cs = c + 2 * s;
      w[s] = u32x4{0, 0, 0, 0};
      sw[s] = sa[s] = 127u;  // behind the end: zeros
      if (!whole && cs < c1) {
        w[s] = *reinterpret_cast<const u32x4*>(wq + 16 * cs);
        sw[s] = ws[cs];
      }
      if constexpr (A4) {
        x[s][0] = u32x4{0, 0, 0, 0};
        if (cs < c1) {
          x[s][0] = *reinterpret_cast<const u32x4*>(aq + 16 * cs);
          sa[s] = as[cs];
        }
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const int64_t k = 32 * cs + 8 * j;
          x[s][j] = u32x4{0, 0, 0, 0};
          if (g.vec_a) {
            if (cs < c1 && k < g.K) x[s][j] = *reinterpret_cast<const u32x4*>(ap + k);
          } else if (cs < c1) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
              if (k + e < g.K) x[s][j][e / 2] |= uint32_t(ap[k + e]) << (16 * (e % 2));
          }
        }
      }
    }
    if (whole) {
#pragma unroll
      for (int u = 0; u < 4; ++u) turn[wave][(8 * u + lane / 8) * 8 + ((lane & 7) ^ (lane / 8))] = wt[u];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
#pragma unroll
      for (int s = 0; s < kFewSteps; ++s) {
        w[s] = turn[wave][l32 * 8 + ((2 * s + hl) ^ (l32 & 7))];
        sw[s] = uint32_t(sw8 >> (16 * s + 8 * hl)) & 255u;
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
#pragma unroll
    for (int s = 0; s < kFewSteps; ++s) {
      if constexpr (A4) {
        acc = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(as_i8(w[s]), as_i8(x[s][0]), acc, 4, 4, 0, int(sw[s]), 0,
                                                              int(sa[s]));
      } else {
        const float f = mx4_scale_f(sw[s]);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const uint32_t wj = w[s][j];
          acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(mx4_bf8(wj, f)), as_bf8(x[s][j]), acc, 0, 0, 0);
        }
      }
    }
  }
  if constexpr (WK > 1) {
    if (wave % WK != 0)
#pragma unroll
      for (int r = 0; r < 16; ++r) red[wave][64 * r + lane] = acc[r];
    __syncthreads();
    if (wave % WK != 0) return;
#pragma unroll
    for (int u = 1; u < WK; ++u)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[r] += red[wave + u][64 * r + lane];
  }
  // lane: row m0 + l32 of out, columns n0 + 8 q + 4 hl + 0 .. 3
  const int64_t m = m0 + l32;
  if (m >= g.M) return;
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int64_t n = n0 + 8 * q + 4 * hl;
    if (g.part != nullptr) {
      if (n < g.Np)
        *reinterpret_cast<f32x4*>(g.part + ((int64_t(split) * g.H + h) * g.M + m) * g.Np + n) =
            f32x4{acc[4 * q], acc[4 * q + 1], acc[4 * q + 2], acc[4 * q + 3]};
      continue;
    }
    TO* op = static_cast<TO*>(const_cast<void*>(g.o.p)) + h * g.o.s1 + m * g.o.s2 + n;
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = gemm_act(g, acc[4 * q + e]);
    if (g.vec4) {
      if (n >= g.N) continue;
      if (g.mul.p != nullptr) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] *= mulv[4 * q + e];
      }
      if constexpr (sizeof(TO) == 2)
        *reinterpret_cast<u32x2*>(op) = u32x2{pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3])};
      else
        *reinterpret_cast<f32x4*>(op) = f32x4{v[0], v[1], v[2], v[3]};
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (n + e < g.N) op[e] = from_f<TO>(g.mul.p != nullptr ? v[e] * gemm_mul(g, mat + n + e) : v[e]);
    }
  }
}

View strides_of(const bdh_tensor4* t) {
  View v;
  v.p = t != nullptr ? t->data : nullptr;
  v.s0 = t != nullptr ? t->stride[0] : 0;
  v.s1 = t != nullptr ? t->stride[1] : 0;
  v.s2 = t != nullptr ? t->stride[2] : 0;
  return v;
}

// -------------------------------------------------------------- many rows
// Operands as the tile kernel streams them: scale bytes gathered by stage (the
// bytes of a stage of 256 rows lie together), padded with 2^-127; and rows of a
// whose pieces are not 16-byte aligned, or end inside a stage, copied with zeros
// behind them.
struct PackArgs {
  View4 m[2];  // wt, a in mx4
  View a;      // a in bf16 (copied where ap is not null)
  uint8_t* sp[2];
  bf16_t* ap;
  int64_t rows[2], rp[2];  // rows, padded rows
  int64_t kb, K, Kp, wgs[2];
  int H, aH, nst, sb, nch, vec[2];  // nch pieces of 16 scales a row; vec: 16-byte loads of them
};

__global__ __launch_bounds__(256) void k_mx4_pack(const PackArgs p) {
  int64_t wg = blockIdx.x;
  for (int j = 0; j < 2; ++j) {
    if (wg >= p.wgs[j]) {
      wg -= p.wgs[j];
      continue;
    }
    const int64_t i = wg * 256 + threadIdx.x, hc = i / p.rp[j], r = i - hc * p.rp[j], h = hc / p.nch, c = hc - h * p.nch;
    if (h >= p.H) return;
    const uint8_t* src = p.m[j].s + h * p.m[j].s1 + min(r, p.rows[j] - 1) * p.m[j].s2 + 16 * c;
    const int n = int(min(int64_t(16), p.kb - 16 * c));
    uint32_t v[4] = {0, 0, 0, 0};
    if (p.vec[j] && n == 16) {
      const u32x4 w = *reinterpret_cast<const u32x4*>(src);
#pragma unroll
      for (int b = 0; b < 4; ++b) v[b] = w[b];
    } else {
#pragma unroll
      for (int b = 0; b < 16; ++b)
        if (b < n) v[b / 4] |= uint32_t(src[b]) << (8 * (b % 4));
    }
    const int64_t st = c * (16 / p.sb), at = (h * p.nst + st) * p.rp[j] + r;
    if (p.sb == 4) {
#pragma unroll
      for (int b = 0; b < 4; ++b)
        if (st + b < p.nst) reinterpret_cast<uint32_t*>(p.sp[j])[at + b * p.rp[j]] = v[b];
    } else {
#pragma unroll
      for (int b = 0; b < 8; ++b)
        if (st + b < p.nst) reinterpret_cast<uint16_t*>(p.sp[j])[at + b * p.rp[j]] = uint16_t(v[b / 2] >> (16 * (b % 2)));
    }
    return;
  }
  const int64_t each = p.Kp / 8, i = wg * 256 + threadIdx.x, row = i / each, k = (i - row * each) * 8;
  const int64_t h = row / p.rows[1], m = row - h * p.rows[1];
  if (h >= p.aH) return;
  const bf16_t* src = static_cast<const bf16_t*>(p.a.p) + h * p.a.s1 + m * p.a.s2 + k;
  u32x4 w{0, 0, 0, 0};
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (k + e < p.K) w[e / 2] |= uint32_t(src[e]) << (16 * (e % 2));
  *reinterpret_cast<u32x4*>(p.ap + row * p.Kp + k) = w;
}

// dma16 by the lanes of a mask (all are active before and after), skipped where it is
// empty: an instruction costs its time whatever its lanes, so each wave's share of the
// scales in one of its own made a stage 15 % slower.  No branch that the compiler sees:
// that would end the basic block in which the loop's instructions are scheduled.
template <int IMM>
__device__ __forceinline__ void dma16_mask(uint32_t mask_lo, uint32_t mask_hi, uint32_t m0base, const void* gbase,
                                           uint32_t voff) {
  asm volatile(
      "s_cmp_eq_u32 %4, 0\n\ts_cbranch_scc1 .Lmask%=\n\ts_add_u32 m0, %0, %3\n\ts_mov_b32 exec_lo, %4\n\t"
      "s_mov_b32 exec_hi, %5\n\tglobal_load_lds_dwordx4 %1, %2\n\ts_mov_b64 exec, -1\n.Lmask%=:"
      :
      : "s"(m0base), "v"(voff), "s"(gbase), "i"(IMM), "s"(mask_lo), "s"(mask_hi)
      : "memory", "m0", "scc");
}

// A workgroup of eight waves (two a SIMD) makes 64 MI rows x 256 columns; wave (wm,
// wn) 32 MI x 64 of them, MI x 2 blocks of 32 x 32.  K goes in stages of KB blocks of 32
// through a ring of LDS slots filled by LDS DMA; a stage has two
// halves, and the fragments of a half are read while the other's MFMAs run, so the
// barrier sits between two halves whose operands are in registers.  16-byte pieces
// are swizzled by row so that a fragment's 16 rows fall on all banks.
// KB is 4, and 2 where four blocks of bf16 do not fit the ring (MI 4) or do not divide K:
// a's rows then come in pieces of 128 bytes instead of 256, and the stream of 6216 x 256 x
// 32768 alone takes 96 us instead of 78.
constexpr int kTileWaves = 8;
template <bool A4, int MI_, int KB_>
struct TileShape {
  static constexpr int MI = MI_, NI = 2, BM = 64 * MI, BN = 256, KB = KB_;  // KB: also scale bytes a row
  static_assert(KB == 4 || (KB == 2 && !A4), "stages");
  static constexpr bool WH = KB == 4;                          // a block of wt is of one half (else of both)
  static constexpr int RA = A4 ? 64 : 64 * KB, RW = 16 * KB;   // bytes of a row of each a stage
  static constexpr int OW = BM * RA, OSW = OW + BN * RW, OSA = OSW + BN * KB, SLOT = OSA + (A4 ? BM * KB : 0);
  static constexpr int DA = BM * RA / 8192, DW = BN * RW / 8192;  // DMA instructions a wave
  // What a wave has in flight a stage at least: waves 0 and 1 issue one more, the scales
  // (first of its stage, so that waiting by this count waits for no later stage's rows).
  static constexpr int C = DA + DW;
  static constexpr int RING = 163840 / SLOT < 6 ? 163840 / SLOT : 6;
  static constexpr int PITCH = 32 * NI + 8;  // floats of a row in the output piece of a wave
  static_assert(RING >= 3 && kTileWaves * 32 * PITCH * 4 <= RING * SLOT && (RING - 1) * C < 64, "LDS ring");
};

struct TileArgs {
  MxGemmArgs g;
  const uint8_t *a, *w;            // rows of a (codes or bf16) and of wt, in bytes
  const uint8_t *sa, *sw;          // gathered scales [h][stage][padded rows]
  int64_t a1, a2, w1, w2;          // byte strides
  int64_t sa_rows, sw_rows;        // padded rows
  int64_t items, per_xcd;
};

// ONCE: one column of tiles, so that no other workgroup reads a's rows (6216 x 256 x 32768 in
// stages of two blocks: 117 -> 113 us).  A slot is filled again as soon as both halves of its stage
// are in registers, RING stages ahead: with RING - 1 the three slots of KB 4 took 114 us, not 105.
template <bool A4, int MI, int KB, bool ONCE, typename TO>
__global__ __launch_bounds__(64 * kTileWaves, 1) void k_mx4_tile(const TileArgs t) {
  using S = TileShape<A4, MI, KB>;
  constexpr int NI = S::NI, RING = S::RING;
  __shared__ __attribute__((aligned(1024))) uint8_t lds[RING * S::SLOT];
  const MxGemmArgs& g = t.g;
  const int64_t item = int64_t(blockIdx.x & 7) * t.per_xcd + (blockIdx.x >> 3);
  if ((blockIdx.x >> 3) >= t.per_xcd || item >= t.items) return;
  // (h, split), then tiles: groups of eight columns of tiles, rows within, so that the
  // tiles an XCD runs at a time share both operands in its L2
  const int tiles = g.mt * g.nt, hs = int(item / tiles), ti = int(item - int64_t(hs) * tiles);
  const int h = hs / g.splits, split = hs - h * g.splits;
  const int grp = ti / (8 * g.mt), rem = ti - grp * 8 * g.mt, gw = min(8, g.nt - 8 * grp);
  const int64_t m0 = int64_t(rem / gw) * S::BM, n0 = int64_t(8 * grp + rem % gw) * S::BN;
  const int st0 = __builtin_amdgcn_readfirstlane(int(int64_t(g.steps) * split / g.splits));
  const int st1 = __builtin_amdgcn_readfirstlane(int(int64_t(g.steps) * (split + 1) / g.splits));

  const int tid = threadIdx.x, lane = tid & 63, l32 = lane & 31, hl = lane >> 5;
  const int wv = __builtin_amdgcn_readfirstlane(tid >> 6), wm = wv >> 2, wn = wv & 3;
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_u8*)lds);

  // ---- DMA: instruction i = 8 u + wave fills KB i of an operand's part of the slot
  constexpr int PA = S::RA / 16, PW = S::RW / 16;  // pieces a row
  const int ca = A4        ? (lane & 3) ^ ((lane >> 4) & 3)
                 : KB == 4 ? (lane & 15) ^ (4 * (wv & 3) + (lane >> 4))
                           : (lane & 7) ^ ((4 * (wv & 1) + (lane >> 4)) & 7);
  const int cw = KB == 4 ? (lane & 3) ^ ((lane >> 4) & 3) : (lane & 1) ^ ((lane >> 4) & 1);
  uint32_t goa[S::DA], gow[S::DW];
#pragma unroll
  for (int u = 0; u < S::DA; ++u) {
    const int64_t r = min(int64_t((8 * u + wv) * (64 / PA) + lane / PA), g.M - 1 - m0);
    goa[u] = uint32_t(r * t.a2 + 16 * ca);
  }
#pragma unroll
  for (int u = 0; u < S::DW; ++u) {
    const int64_t r = min(int64_t((8 * u + wv) * (64 / PW) + lane / PW), g.N - 1 - n0);
    gow[u] = uint32_t(r * t.w2 + 16 * cw);
  }
  // blocks behind the row's end in the last stage: its last block again (a's scale and
  // wt's are 2^-127 there, or a is zero)
  const int left = int(g.kb - int64_t(g.steps - 1) * S::KB);
  const uint32_t enda = A4 ? 16u * uint32_t(max(0, ca - (left - 1))) : 0u, endw = 16u * uint32_t(max(0, cw - (left - 1)));
  // scales: wt's by wave 0, a's by wave 1
  const bool sca = A4 && wv == 1;
  constexpr int BW = S::BN * S::KB / 16, BA = S::BM * S::KB / 16;  // 16-byte pieces
  const uint32_t smask = __builtin_amdgcn_readfirstlane(wv == 0 || sca ? ~0u : 0u);  // (32 pieces or 64)
  const uint32_t smask_hi = __builtin_amdgcn_readfirstlane((sca ? BA : BW) == 64 ? smask : 0u);
  static_assert((BW == 32 || BW == 64) && (!A4 || BA == 32 || BA == 64), "whole halves of a wave");
  const uint32_t sat = sca ? S::OSA : S::OSW;
  const int sd = int(sca ? t.sa_rows : t.sw_rows) * S::KB;
  // the next stage to issue: its operands, and where it goes
  struct Issue {
    const uint8_t *pa, *pw, *ps;
    uint32_t b;  // LDS address of the slot
    uint32_t ea, ew;
    int st, slot;
  } x;
  x.st = st0;
  x.slot = 0;
  x.b = lds0;
  x.pa = static_cast<const uint8_t*>(sgpr_ptr(t.a + h * t.a1 + m0 * t.a2 + int64_t(st0) * S::RA));
  x.pw = static_cast<const uint8_t*>(sgpr_ptr(t.w + h * t.w1 + n0 * t.w2 + int64_t(st0) * S::RW));
  x.ps = static_cast<const uint8_t*>(
      sgpr_ptr(sca ? t.sa + ((int64_t(h) * g.steps + st0) * t.sa_rows + m0) * S::KB
                   : t.sw + ((int64_t(h) * g.steps + st0) * t.sw_rows + n0) * S::KB));
  auto issue_ends = [&]() __attribute__((always_inline)) {
    x.ea = x.st == g.steps - 1 ? enda : 0u;
    x.ew = x.st == g.steps - 1 ? endw : 0u;
  };
  issue_ends();
  auto issue_next = [&]() __attribute__((always_inline)) {
    x.slot = x.slot == RING - 1 ? 0 : x.slot + 1;
    x.b = lds0 + uint32_t(x.slot * S::SLOT);
    const int step = x.st + 1 < st1 ? 1 : 0;  // (past the end: the last stage again, not read)
    x.st += step;
    x.pa += step * S::RA;
    x.pw += step * S::RW;
    x.ps += step * sd;
    issue_ends();
  };
  // instruction j of a stage's S::C + 1: scales, rows of a, of wt
  auto issue = [&](auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value - 1;
    const uint32_t bw = x.b + uint32_t(wv) * 1024u;
    if constexpr (j < 0)
      dma16_mask<0>(smask, smask_hi, x.b + sat, x.ps, uint32_t(16 * lane));
    else if constexpr (j < S::DA && ONCE)
      dma16_once<j * 8192>(bw, x.pa, goa[j] - x.ea);
    else if constexpr (j < S::DA)
      dma16<j * 8192>(bw, x.pa, goa[j] - x.ea);
    else
      dma16<S::OW + (j - S::DA) * 8192>(bw, x.pw, gow[j - S::DA] - x.ew);
  };

  // ---- fragments
  struct Half {
    u32x4 a[A4 ? 1 : KB][MI];
    u32x4 w[S::WH ? NI : 1];
  };
  struct Stage {  // what both halves use
    uint32_t sa[A4 ? MI : 1], sw[NI];
    u32x4 w[S::WH ? 1 : NI];
  };
  const uint32_t ra = uint32_t((32 * MI * wm + l32) * S::RA), rw = uint32_t(S::OW + (32 * NI * wn + l32) * S::RW);
  // Reads as items of the loop below: of a stage (SR of them), of a half (HR).
  constexpr int SR = A4 ? NI + MI : S::WH ? NI : 2 * NI, RF = A4 ? MI : KB * MI, HR = RF + (S::WH ? NI : 0);
  auto read_stage = [&](Stage& s, const uint8_t* b, auto jc) __attribute__((always_inline)) {
    constexpr int j = decltype(jc)::value, i = j < NI ? j : j - NI;
    const uint8_t* p = b + S::OSW + (32 * NI * wn + 32 * i + l32) * S::KB;
    if constexpr (S::WH && j < NI)
      s.sw[i] = *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (A4)
      s.sa[i] = *reinterpret_cast<const uint32_t*>(b + S::OSA + (32 * MI * wm + 32 * i + l32) * 4);
    else if constexpr (j < NI)
      s.sw[i] = p[hl];
    else
      s.w[i] = *reinterpret_cast<const u32x4*>(b + rw + 32 * S::RW * i + 16 * (hl ^ ((l32 >> 3) & 1)));
  };
  // the lane's bytes of a stage's scales (block 2 q + hl of half q) to bytes 0 and 2
  auto turn = [&](Stage& s) __attribute__((always_inline)) {
    if constexpr (S::WH)
#pragma unroll
      for (int i = 0; i < NI; ++i) s.sw[i] >>= 8 * hl;
    if constexpr (A4)
#pragma unroll
      for (int i = 0; i < MI; ++i) s.sa[i] >>= 8 * hl;
  };
  auto read_half = [&](Half& f, const uint8_t* b, auto qc, auto jc) __attribute__((always_inline)) {
    constexpr int q = decltype(qc)::value, j = decltype(jc)::value;
    const int at = 16 * ((2 * q + hl) ^ ((l32 >> 2) & 3));  // of rows of 64 bytes
    if constexpr (j >= RF) {
      f.w[j - RF] = *reinterpret_cast<const u32x4*>(b + rw + 32 * S::RW * (j - RF) + at);
    } else if constexpr (A4) {
      f.a[0][j] = *reinterpret_cast<const u32x4*>(b + ra + 32 * S::RA * j + at);
    } else {
      constexpr int k = j / MI, i = j % MI;
      const int piece = KB == 4 ? (8 * q + 4 * hl + k) ^ (l32 & 15) : (4 * hl + 2 * q + k) ^ ((l32 >> 1) & 7);
      f.a[k][i] = *reinterpret_cast<const u32x4*>(b + ra + 32 * S::RA * i + 16 * piece);
    }
  };
  f32x16 acc[MI][NI];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int n = 0; n < NI; ++n)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][n][r] = 0.f;
  // A half's MFMAs, and after each its share of ITEMS other instructions, which issue
  // while the matrix core is busy.
  auto mma = [&](const Half& f, const Stage& s, auto qc, auto itemsc, auto&& item) __attribute__((always_inline)) {
    constexpr int q = decltype(qc)::value, NM = (A4 ? 1 : KB) * MI * NI, ITEMS = decltype(itemsc)::value;
    bf16x8 wf{};
    static_for<NM>([&](auto kc) __attribute__((always_inline)) {
      constexpr int k = decltype(kc)::value, i = k % MI;
      if constexpr (A4) {
        constexpr int n = k / MI;
        acc[i][n] = __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(as_i8(f.a[0][i]), as_i8(f.w[n]), acc[i][n], 4, 4, 2 * q,
                                                                    int(s.sa[i]), 2 * q, int(s.sw[n]));
      } else {
        constexpr int n = k / MI / KB, j = k / MI % KB;
        if constexpr (i == 0 && S::WH) {
          const uint32_t w = f.w[n][j];
          wf = as_bf8(mx4_bf8(w, mx4_scale_f((s.sw[n] >> (16 * q)) & 255u)));
        } else if constexpr (i == 0) {
          const uint32_t w = s.w[n][2 * q + j];
          wf = as_bf8(mx4_bf8(w, mx4_scale_f(s.sw[n])));
        }
        acc[i][n] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(as_bf8(f.a[j][i]), wf, acc[i][n], 0, 0, 0);
      }
      constexpr int from = k * ITEMS / NM, to = (k + 1) * ITEMS / NM;
      static_for<to - from>([&](auto uc) __attribute__((always_inline)) {
        item(std::integral_constant<int, from + decltype(uc)::value>());
      });
      __builtin_amdgcn_sched_barrier(0);
    });
  };
  auto barrier = [] __device__ { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); };

  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  static_for<RING>([&](auto) {
    static_for<S::C + 1>([&](auto jc) { issue(jc); });
    issue_next();
  });
  sy_wait<(RING - 1) * S::C>();
  barrier();
  Half f0, f1;
  Stage sx, sy;
  const uint8_t* b = lds;  // the slot of the stage at hand
  static_for<SR>([&](auto jc) { read_stage(sx, b, jc); });
  turn(sx);
  static_for<HR>([&](auto jc) { read_half(f0, b, I0(), jc); });
  auto stage = [&](const Stage& cur, Stage& nxt) __attribute__((always_inline)) {
    mma(f0, cur, I0(), std::integral_constant<int, HR>(), [&](auto jc) { read_half(f1, b, I1(), jc); });
    sy_wait<(RING - 2) * S::C>();  // this wave's part of the next stage landed
    barrier();                     // every wave's; this stage's other half is in registers, its slot x.slot free
    b = b == lds + (RING - 1) * S::SLOT ? lds : b + S::SLOT;
    mma(f1, cur, I1(), std::integral_constant<int, SR + HR + S::C + 3>(), [&](auto jc) __attribute__((always_inline)) {
      constexpr int j = decltype(jc)::value;
      if constexpr (j < SR)
        read_stage(nxt, b, jc);
      else if constexpr (j < SR + HR)
        read_half(f0, b, I0(), std::integral_constant<int, j - SR>());
      else if constexpr (j <= SR + HR + S::C)
        issue(std::integral_constant<int, j - SR - HR>());
      else if constexpr (j == SR + HR + S::C + 1)
        issue_next();
      else
        turn(nxt);
    });
  };
  int st = st0;
  for (; st + 2 <= st1; st += 2) {
    stage(sx, sy);
    stage(sy, sx);
  }
  if (st < st1) stage(sx, sy);
  sy_wait<0>();
  barrier();

  // ---- out: 32 rows of a wave at a time through LDS, then eight columns a lane
  float* piece = reinterpret_cast<float*>(lds) + wv * 32 * S::PITCH;
  const int rr = lane / (4 * NI), cc = 8 * (lane % (4 * NI));  // its row of 16 / NI at a time, its columns
  const int64_t n = n0 + 32 * NI * wn + cc;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
#pragma unroll
    for (int k = 0; k < NI; ++k)
#pragma unroll
      for (int r = 0; r < 16; ++r) piece[(8 * (r >> 2) + 4 * hl + (r & 3)) * S::PITCH + 32 * k + l32] = acc[i][k][r];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    f32x4 v[2 * NI][2];
#pragma unroll
    for (int it = 0; it < 2 * NI; ++it) {
      const float* p = piece + (16 / NI * it + rr) * S::PITCH + cc;
      v[it][0] = reinterpret_cast<const f32x4*>(p)[0];
      v[it][1] = reinterpret_cast<const f32x4*>(p)[1];
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (n >= g.N) continue;
    const int64_t m = m0 + 32 * (MI * wm + i) + rr;
    if (g.part != nullptr) {
      float* p = g.part + ((int64_t(split) * g.H + h) * g.M + m) * g.Np + n;
#pragma unroll
      for (int it = 0; it < 2 * NI; ++it) {
        if (m + 16 / NI * it >= g.M) break;
        reinterpret_cast<f32x4*>(p + 16 / NI * it * g.Np)[0] = v[it][0];
        reinterpret_cast<f32x4*>(p + 16 / NI * it * g.Np)[1] = v[it][1];
      }
    } else {
#pragma unroll
      for (int it = 0; it < 2 * NI; ++it) {
        if (m + 16 / NI * it >= g.M) break;
        float e[8] = {v[it][0][0], v[it][0][1], v[it][0][2], v[it][0][3], v[it][1][0], v[it][1][1], v[it][1][2], v[it][1][3]};
        gemm_out8<TO>(g, h, m + 16 / NI * it, n, e);
      }
    }
  }
}

// ------------------------------------------------------------------- plans
struct GemmPlan {
  bool tile, a4, copy;
  int mi, kb, steps, splits, wk;
  int64_t mt, nt, Kp;
  size_t sw, sa, ap, part, end;  // workspace: gathered scales, copied rows, partials
};

// Few rows: splits of K and waves a tile, four waves a CU where K has a wave's four
// steps for each of them; up to four waves a tile of long rows to make sixteen a CU (3 rows of
// 4 x 8192 x 13504 116 -> 88 us, 8 of 4 x 8192 x 8192 71 -> 55, but of 4 x 8192 x 1024 10.7 -> 13.1).
void few_plan(int64_t H, int64_t M, int64_t N, int64_t K, GemmPlan& p) {
  p.steps = int((mx4_blocks(K) + 1) / 2);
  const int64_t tiles = H * ((M + 31) / 32) * ((N + 31) / 32);
  int64_t want = (1024 + tiles - 1) / tiles;
  if (p.steps >= 128) want = std::max(want, std::min<int64_t>(4, (4096 + tiles - 1) / tiles));
  want = std::max<int64_t>(1, std::min<int64_t>(want, p.steps / kFewSteps));
  p.wk = want >= 4 ? 4 : want >= 2 ? 2 : 1;
  p.splits = int(std::min<int64_t>((want + p.wk - 1) / p.wk, 1024));
}

// Many rows: the tile's height and the splits of the least time, which is returned: 6 us
// for gathering the scales, a round's stages and its way in and out, and what the sum of the
// splits costs at 5 TB/s and one more launch.  A stage slows with the CUs at work (by two
// fifths and more; the matrix cores' power, and the streams).  Modelled and measured: bf16
// 6216 x 256 x 32768 in five splits of MI 2 97 us and 107, in ten of MI 4 104 and 119, 4096 x
// 4096 x 4096 of MI 4 106 and 107, of MI 2 112 and 113; mx4 4096 x 8192 x 8192 149 and 146, 500 x
// 300 x 16384 in ten splits of MI 2 21 and 27.
double tile_plan(int64_t H, int64_t M, int64_t N, int64_t K, GemmPlan& p) {
  double best = 1e30;
  for (int mi = 2; mi <= 4; mi += 2) {
    const int kb = p.a4 || (mi == 2 && (p.copy || K % 128 == 0)) ? 4 : 2;
    const int steps = int((mx4_blocks(K) + kb - 1) / kb);
    const double idle = p.a4 ? (mi == 4 ? 0.63 : 0.37) : mi == 4 ? 1.05 : kb == 4 ? 1.08 : 0.66;  // us a stage, few CUs
    const double full = p.a4 ? (mi == 4 ? 1.0 : 0.67) : mi == 4 ? 1.45 : kb == 4 ? 1.5 : 0.88;    // and all
    const int64_t mt = (M + 64 * mi - 1) / (64 * mi), nt = (N + 255) / 256, tiles = H * mt * nt;
    for (int s = 1; s <= 16 && s <= steps; ++s) {
      const double us = idle + (full - idle) * std::min(1.0, double(tiles * s) / 256);
      const double t = 6 + double((tiles * s + 255) / 256) * (double((steps + s - 1) / s) * us + (mi == 4 ? 7.5 : 5)) +
                       (s > 1 ? 3 + 4e-6 / 5 * double(s) * double(H) * double(M) * double(N) : 0);
      if (t < best) {
        best = t;
        p.mi = mi;
        p.kb = kb;
        p.steps = steps;
        p.splits = s;
        p.mt = mt;
        p.nt = nt;
      }
    }
  }
  return best;
}

// The few-row kernel's: 7 us and 240 TFLOP/s in bf16, 500 in mx4, half where rows are long, of
// whole tiles, and a's bytes at 3 TB/s.  Measured against the tile kernel: bf16 256 x 4096 x 1024
// 14 us and 25, 1000 x 512 x 2048 15 and 31, 1500 x 256 x 8192 41 and 35, 2048 x 2048 x 2048 71 and
// 31, 6216 x 32 x 32768 122 and 97 (though it computes 256 columns); mx4 80 x 100 x 256 7 and 19,
// 64 x 8192 x 4096 13 and 27, 128 x 4096 x 16384 44 and 30, 813 x 8192 x 512 20 and 21.  It leaves out
// the weights' bytes, which bound few rows: up to 32 this kernel is taken unasked.
double few_us(int64_t H, int64_t M, int64_t N, int64_t K, bool a4) {
  const double hmk = double(H) * double(M) * double(K);
  return 7 + std::max(2e-6 * hmk * double(align_up(N, 32)) / ((a4 ? 500 : 240) * (K < 8192 ? 1 : 0.5)),
                      hmk * (a4 ? 17.0 / 32 : 2) / 3e6);
}

GemmPlan gemm_plan(const bdh_tensor4* a, const bdh_mx4* a4, const bdh_mx4* wt) {
  GemmPlan p{};
  const int64_t* as = a != nullptr ? a->size : a4->size;
  const int64_t H = as[1], M = as[2], K = as[3], N = wt->size[2];
  p.a4 = a4 != nullptr;
  // DMA offsets inside a tile are 32-bit: rows (copied ones, too) at most 8 MB apart.  The
  // gathered scales of a stage are stepped over by 32 bits: at most 4 bytes of 2^28 rows.
  const int64_t apart = a != nullptr ? 2 * a->stride[2] : a4->code_stride[2];
  p.copy = a != nullptr && (K % 64 != 0 || !vec16_ok(a));
  p.tile = M > 32 && K > 0 && apart <= (1 << 23) && wt->code_stride[2] <= (1 << 23) && K <= (a != nullptr ? 1 << 22 : 1 << 24) &&
           M <= (1 << 28) && N <= (1 << 28) &&
           (tile_plan(H, M, N, K, p) < few_us(H, M, N, K, p.a4) || M > kFewRows);
  if (!p.tile) {
    few_plan(H, M, N, K, p);
  } else {
    p.Kp = (K + 32 * p.kb - 1) / (32 * p.kb) * (32 * p.kb);
  }
  auto take = [&](size_t bytes) {
    const size_t at = p.end;
    p.end = align_up(p.end + bytes, 256);
    return at;
  };
  if (p.tile) {
    const size_t hs = size_t(H) * size_t(p.steps) * size_t(p.kb);
    p.sw = take(hs * size_t(p.nt) * 256);
    p.sa = take(p.a4 ? hs * size_t(p.mt) * size_t(64 * p.mi) : 0);
    p.ap = take(p.copy ? size_t(a->stride[1] == 0 ? 1 : H) * size_t(M) * size_t(p.Kp) * 2 : 0);
  }
  p.part = take(p.splits > 1 ? size_t(p.splits) * size_t(H) * size_t(M) * size_t((N + 7) / 8 * 8) * sizeof(float) : 0);
  return p;
}

template <typename TO>
int launch_sum(const MxGemmArgs& g, hipStream_t s) {
  const int64_t n = int64_t(g.H) * g.M * (g.Np / 8);
  const bool few = n < 16384;  // 64 workgroups of single threads
  const int64_t wgs = few ? (n + 31) / 32 : (n + 255) / 256;
  if (wgs >= (int64_t(1) << 31)) return BDH_ERR_SHAPE;
  if (few)
    BDH_LAUNCH("k_mx4_sum", (k_mx4_sum<TO, 8>), dim3(unsigned(wgs)), dim3(256), 0, s, g);
  else
    BDH_LAUNCH("k_mx4_sum", (k_mx4_sum<TO, 1>), dim3(unsigned(wgs)), dim3(256), 0, s, g);
  return BDH_OK;
}

template <bool A4, typename TO>
int launch_few(const MxGemmArgs& g, const GemmPlan& p, hipStream_t s) {
  const int64_t nx = (g.N + 32 * (4 / p.wk) - 1) / (32 * (4 / p.wk)), mx = (g.M + 31) / 32;
  if (nx >= (int64_t(1) << 31) || g.M > kFewRows || int64_t(g.H) * p.splits > 65535) return BDH_ERR_SHAPE;
  const dim3 grid(unsigned(nx), unsigned(mx), unsigned(g.H * p.splits));
  if (p.wk == 4)
    BDH_LAUNCH("k_mx4_few", (k_mx4_few<A4, TO, 4>), grid, dim3(256), 0, s, g);
  else if (p.wk == 2)
    BDH_LAUNCH("k_mx4_few", (k_mx4_few<A4, TO, 2>), grid, dim3(256), 0, s, g);
  else
    BDH_LAUNCH("k_mx4_few", (k_mx4_few<A4, TO, 1>), grid, dim3(256), 0, s, g);
  return BDH_OK;
}

template <bool A4, typename TO>
int launch_tile(const MxGemmArgs& g, const GemmPlan& p, const bdh_tensor4* a, const bdh_mx4* a4, const bdh_mx4* wt,
                uint8_t* ws, hipStream_t s) {
  PackArgs k{};
  k.m[0] = g.w;
  k.m[1] = g.a4;
  k.a = g.a;
  k.sp[0] = ws + p.sw;
  k.sp[1] = ws + p.sa;
  k.ap = reinterpret_cast<bf16_t*>(ws + p.ap);
  k.rows[0] = g.N;
  k.rows[1] = g.M;
  k.rp[0] = p.nt * 256;
  k.rp[1] = p.mt * 64 * p.mi;
  k.kb = g.kb;
  k.K = g.K;
  k.Kp = p.Kp;
  k.H = g.H;
  k.aH = p.copy ? (a->stride[1] == 0 ? 1 : g.H) : 0;
  k.nst = p.steps;
  k.sb = p.kb;
  auto groups = [](int64_t n) { return (n + 255) / 256; };
  k.nch = int((g.kb + 15) / 16);
  for (int j = 0; j < 2; ++j)
    k.vec[j] = (reinterpret_cast<uintptr_t>(k.m[j].s) & 15) == 0 && (g.H == 1 || k.m[j].s1 % 16 == 0) && k.m[j].s2 % 16 == 0;
  k.wgs[0] = groups(int64_t(g.H) * k.nch * k.rp[0]);
  k.wgs[1] = A4 ? groups(int64_t(g.H) * k.nch * k.rp[1]) : 0;
  const int64_t wgs = k.wgs[0] + k.wgs[1] + (p.copy ? groups(int64_t(k.aH) * g.M * (p.Kp / 8)) : 0);
  TileArgs t{};
  t.g = g;
  t.items = int64_t(g.H) * p.splits * p.mt * p.nt;
  t.per_xcd = (t.items + 7) / 8;
  if (wgs >= (int64_t(1) << 31) || t.items >= (int64_t(1) << 31) - 8 || p.mt * p.nt >= (int64_t(1) << 31)) return BDH_ERR_SHAPE;
  BDH_LAUNCH("k_mx4_pack", k_mx4_pack, dim3(unsigned(wgs)), dim3(256), 0, s, k);
  t.w = g.w.q;
  t.w1 = g.w.q1;
  t.w2 = g.w.q2;
  t.sw = k.sp[0];
  t.sa = k.sp[1];
  t.sw_rows = k.rp[0];
  t.sa_rows = k.rp[1];
  if (A4) {
    t.a = g.a4.q;
    t.a1 = g.a4.q1;
    t.a2 = g.a4.q2;
  } else if (p.copy) {
    t.a = reinterpret_cast<const uint8_t*>(k.ap);
    t.a2 = 2 * p.Kp;
    t.a1 = k.aH == 1 ? 0 : g.M * t.a2;
  } else {
    t.a = static_cast<const uint8_t*>(g.a.p);
    t.a1 = 2 * g.a.s1;
    t.a2 = 2 * g.a.s2;
  }
  const dim3 grid(unsigned(8 * t.per_xcd));
  auto go = [&](auto mi, auto kb, auto once) {
    BDH_LAUNCH("k_mx4_tile", (k_mx4_tile<A4, mi(), kb(), once(), TO>), grid, dim3(64 * kTileWaves), 0, s, t);
    return BDH_OK;
  };
  using std::integral_constant;
  constexpr integral_constant<int, 2> i2;
  constexpr integral_constant<int, 4> i4;
  if constexpr (A4) {
    return p.mi == 4 ? go(i4, i4, std::false_type()) : go(i2, i4, std::false_type());
  } else {
    auto one = [&](auto once) { return p.mi == 4 ? go(i4, i2, once) : p.kb == 4 ? go(i2, i4, once) : go(i2, i2, once); };
    return p.nt == 1 ? one(std::true_type()) : one(std::false_type());
  }
}

template <bool A4, typename TO>
int launch_gemm(const MxGemmArgs& g, const GemmPlan& p, const bdh_tensor4* a, const bdh_mx4* a4, const bdh_mx4* wt,
                uint8_t* ws, hipStream_t s) {
  if (p.tile)
    BDH_TRY(launch_tile<A4, TO>(g, p, a, a4, wt, ws, s));
  else
    BDH_TRY(launch_few<A4, TO>(g, p, s));
  return p.splits > 1 ? launch_sum<TO>(g, s) : BDH_OK;
}

// The operands' types and sizes.
int gemm_operands(const bdh_tensor4* a, const bdh_mx4* a4, const bdh_mx4* wt) {
  if ((a == nullptr) == (a4 == nullptr)) return BDH_ERR_ARG;
  if (a != nullptr) BDH_TRY(check_view(a));
  if (a4 != nullptr) BDH_TRY(check_mx4(a4));
  BDH_TRY(check_mx4(wt));
  if (a != nullptr && a->dtype != BDH_BF16) return BDH_ERR_DTYPE;
  const int64_t* as = a != nullptr ? a->size : a4->size;
  if (as[0] != 1 || wt->size[0] != 1 || wt->size[1] != as[1] || wt->size[3] != as[3]) return BDH_ERR_SHAPE;
  if (as[1] > 65535 || std::max({as[2], as[3], wt->size[2]}) > (int64_t(1) << 30)) return BDH_ERR_SHAPE;
  return BDH_OK;
}

void gemm_args(const bdh_tensor4* a, const bdh_mx4* a4, const bdh_mx4* wt, const GemmPlan& p, MxGemmArgs& g) {
  const int64_t* as = a != nullptr ? a->size : a4->size;
  g.a = strides_of(a);
  g.a4 = a4 != nullptr ? view_of(a4) : View4{};
  g.w = view_of(wt);
  g.H = int(as[1]);
  g.M = as[2];
  g.N = wt->size[2];
  g.K = as[3];
  g.kb = mx4_blocks(g.K);
  g.Np = (g.N + 7) / 8 * 8;
  g.vec_a = a != nullptr && vec16_ok(a);
  g.steps = p.steps;
  g.splits = p.splits;
  g.mt = int(p.mt);
  g.nt = int(p.nt);
}

}  // namespace

int mx4_few_splits(int64_t M, int64_t N, int64_t K) {
  GemmPlan p{};
  few_plan(1, M, N, K, p);
  return p.splits;
}

int mx4_few_parts(const bdh_tensor4* a, const bdh_mx4* wt, float* part, hipStream_t s) {
  BDH_TRY(gemm_operands(a, nullptr, wt));
  if (wt->size[2] % 8 != 0) return BDH_ERR_SHAPE;
  GemmPlan p{};
  few_plan(a->size[1], a->size[2], wt->size[2], a->size[3], p);
  MxGemmArgs g{};
  gemm_args(a, nullptr, wt, p, g);
  g.part = part;
  return launch_few<false, float>(g, p, s);
}

}  // namespace bdh

using namespace bdh;

extern "C" size_t bdh_mx4_gemm_workspace(const bdh_tensor4* a, const bdh_mx4* a4, const bdh_mx4* wt) {
  if (gemm_operands(a, a4, wt) != BDH_OK) return 0;
  const int64_t* as = a != nullptr ? a->size : a4->size;
  return as[1] * as[2] * wt->size[2] == 0 ? 0 : gemm_plan(a, a4, wt).end;
}

extern "C" int bdh_mx4_gemm(const bdh_tensor4* a, const bdh_mx4* a4, const bdh_mx4* wt, const bdh_tensor4* mul,
                            int32_t relu, const bdh_tensor4* out, void* workspace, size_t workspace_bytes,
                            bdh_stream stream) {
  BDH_TRY(gemm_operands(a, a4, wt));
  if (mul != nullptr) BDH_TRY(check_view(mul));
  BDH_TRY(check_view(out));
  const int64_t* as = a != nullptr ? a->size : a4->size;
  const int64_t H = as[1], M = as[2], K = as[3], N = wt->size[2];
  for (const bdh_tensor4* t : {mul, out})
    if (t != nullptr && (t->size[0] != 1 || t->size[1] != H || t->size[2] != M || t->size[3] != N)) return BDH_ERR_SHAPE;
  if ((a != nullptr && views_overlap(out, a)) || (a4 != nullptr && overlap(a4, out)) || overlap(wt, out) ||
      (mul != nullptr && views_overlap(out, mul)) || repeats(out->size, out->stride))
    return BDH_ERR_ALIAS;
  if (numel4(out) == 0) return BDH_OK;
  const GemmPlan p = gemm_plan(a, a4, wt);
  if (p.end > 0 &&
      (workspace == nullptr || workspace_bytes < p.end || (reinterpret_cast<uintptr_t>(workspace) & 15) != 0))
    return BDH_ERR_WORKSPACE;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  MxGemmArgs g{};
  gemm_args(a, a4, wt, p, g);
  g.mul = strides_of(mul);
  g.mul_bf16 = mul != nullptr && mul->dtype == BDH_BF16;
  g.o = strides_of(out);
  g.relu = relu != 0;
  g.vec_o = N % 8 == 0 && vec16_ok(out) && (mul == nullptr || vec16_ok(mul));
  auto four = [](const bdh_tensor4* t) {  // rows in pieces of four elements
    return reinterpret_cast<uintptr_t>(t->data) % size_t(4 * esize(t->dtype)) == 0 &&
           (t->size[1] <= 1 || t->stride[1] % 4 == 0) && (t->size[2] <= 1 || t->stride[2] % 4 == 0);
  };
  g.vec4 = N % 4 == 0 && four(out) && (mul == nullptr || four(mul));
  g.part = p.splits > 1 ? reinterpret_cast<float*>(ws + p.part) : nullptr;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const bool bf = out->dtype == BDH_BF16;
  if (a4 != nullptr)
    return bf ? launch_gemm<true, bf16_t>(g, p, a, a4, wt, ws, s) : launch_gemm<true, float>(g, p, a, a4, wt, ws, s);
  return bf ? launch_gemm<false, bf16_t>(g, p, a, a4, wt, ws, s) : launch_gemm<false, float>(g, p, a, a4, wt, ws, s);
}
