// Gated feed-forward block and its gradients:
//   g = x Wg^T, u = x Wu^T, h = act(g) u, y = h Wd^T       (act: silu, or gelu by erf)
//   dh = dy Wd, dg = dh u act'(g), du = dh act(g)
//   dx = dg Wg + du Wu, dWg = dg^T x, dWu = du^T x, dWd = dy^T h
//
// All products run on mm_kernel (mm_sm100.cuh). The first one takes rows of both
// Wg and Wu into a tile (kSecondHalves), so that a thread of its epilogue
// holds g[n, j] and u[n, j] and writes h alone. The backward's first product
// recomputes h from what was kept and turns dh into dg and du in its epilogue: dh
// is never in memory either. dx is one product over both halves of the inner
// width (kSecondTerms), dWg and dWu are one product.
//
// Roundings, bf16: h, dg and du are rounded to bf16 to be operands, and the
// result once more, which is sqrt(2) of the result's own rounding. g and u
// are kept in fp16 with a power of two for every 16 of them (11 bits relative
// to their largest, 4 bytes an inner column and token as bf16 would take): in bf16 they
// would add another rounding to dg and du each (dx 1.75 times its own). Up
// to kFine tokens keep h, dg and du in two bf16 planes, as little averages
// their errors.
// fp32: all operands in three bf16 planes and six products (24 bits), g and u
// in fp32.
//
// Bound by the tensor cores, and by the epilogues with the activation where a tile's products are short:
// 32768 tokens of 1536 x 4096, bf16: g and u's product 589 us (824 GF: 1.40 PFLOP/s), y 264 + 12 us of joining split
// tiles (412 GF), dh's 393, dx 514 + 16, dWd 295 + 16, [dWg; dWu] 487 + 18; the training step 3.0 to 3.15 ms, under the
// power cap. 4095 tokens of 1408 x 3749: 73, 44 + 9, 63, 72 + 8, 51 + 9, 77 + 8. fp32, 1000 of 512 x 1365: 31, 20 + 6,
// 37, 28 + 9, 21 + 6, 26 + 7 and 7 + 7 of packing.
//
// Few tokens without gradients take gated_few.cu's kernel instead (few_tokens).
#include <math.h>

#include <algorithm>

#include "gated.cuh"
#include "gated_act.cuh"
#include "mm_rows.cuh"

namespace llattn {
namespace gated {
namespace {

using namespace mm;

constexpr int kFine = 64;
// K = 64 steps a tensor-core sum takes (MmArgs::chain) in fp32: as the loss's products (xent.cu)
constexpr int kFineF32Chain = 1, kF32Chain = 4;
// and in bf16 of sums of more than kLongSum products: what the additions drop makes K products of one sign up to
// K 2^-27 short (2^20 of them: 0.6 %), from 2^18 on as much as bf16's own rounding. Shorter ones stay whole, as chains
// leave shape 3 out (step of 140000 tokens of 1536 x 4096: 13.7 ms for 12.9).
constexpr int kLongSum = 1 << 17, kLongChain = 1024;
constexpr int kBlock = 16;  // inner columns of a kept block

// act(g) and act'(g) for h in P planes. 3: to fp32's last bits. Otherwise ex2's and rcp's 2^-22, and phi(-|g|) =
// exp(-g^2 / 2) t P(t) with t = 1 / (1 + p |g|), which shares its exponential with the density: P fitted to 1.2e-7 of the
// value over all of [0, 19], as the tail's values are rounded relative to themselves (an approximation of erf to 1.5e-7
// was off by 1 % at -8): 2^-20 with all roundings. ex2's rounded argument costs 3e-6 at -8, 8e-6 at -13, which h in two
// planes would show: what it lost comes back there.
// (8 and 22 instructions: the epilogues that use them are as long as their tile's products. For 48 tokens of 1536 x 4096
// erfc and exp take 99 us a step for 89.)
__device__ __forceinline__ float fast_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <int ACT, int P>
__device__ __forceinline__ void activation(float g, float& a, float& slope) {
  if (ACT == LLATTN_ACT_SILU) {
    const float s = P == 3 ? 1.f / (1.f + expf(-g)) : fast_rcp(1.f + fast_exp2(g * -1.44269504f));
    a = g * s;
    slope = fmaf(a, 1.f - s, s);
  } else {
    float phi, e;
    if (P == 3) {
      gaussian(g, phi, e);
    } else {
      if (P == 1) {
        e = fast_exp2(g * g * -0.72134752f);
      } else {
        const float b = fminf(fabsf(g), 40.f), h = b * b, y = h * -0.72134752f;
        const float lost = fmaf(fmaf(b, b, -h), -0.72134752f, fmaf(h, -0.72134752f, -y)) + h * -9.6298e-9f;
        e = fast_exp2(y);
        e = fmaf(e, lost * 0.69314718f, e);
      }
      const float t = fast_rcp(fmaf(fabsf(g), 0.23663878f, 1.f));
      float q = fmaf(t, -0.06061577f, 0.19103926f);
      q = fmaf(q, t, -0.11808938f);
      q = fmaf(q, t, 0.15785509f);
      q = fmaf(q, t, 0.045865543f);
      q = fmaf(q, t, 0.09585728f);
      q = fmaf(q, t, 0.093646936f);
      q = fmaf(q, t, 0.09444093f);
      q *= t * e;
      phi = g > 0.f ? 1.f - q : q;
    }
    a = g * phi;
    slope = phi + g * (0.39894228f * e);
  }
}

// Kept g and u: for every 32 tokens and 16 inner columns a block of 16-byte chunks, lane by
// lane (token by token), so that the warp that wrote it and the one that reads it
// each move whole lines without going through shared memory: a token's 16 values of g,
// then of u. bf16 inputs: fp16 times 2^(s - 127), s a byte for g and for u each,
// chosen so that the largest of the 16 lies in [2^14, 2^15); fp32 inputs: as they are.
struct Kept {
  uint8_t* gu;      // [token groups][blocks][4 or 8 chunks][32][16]
  uint16_t* scale;  // [token groups][blocks][32] (bf16)
  int blocks;
};
__device__ __forceinline__ uint32_t block_scale(const float (&v)[16]) {
  float m = 0.f;
#pragma unroll
  for (int q = 0; q < 16; ++q) m = fmaxf(m, fabsf(v[q]));
  if (m == INFINITY) {  // (a weight's row that overflows leaves its neighbours as they are)
    m = 0.f;
#pragma unroll
    for (int q = 0; q < 16; ++q) m = fabsf(v[q]) < INFINITY ? fmaxf(m, fabsf(v[q])) : m;
  }
  const int e = __float_as_uint(m) >> 23;  // 2^(e - 127) <= m
  return (uint32_t)min(253, 127 + 14 + 127 - e);
}
__device__ __forceinline__ float scale_of(uint32_t s) { return __uint_as_float(s << 23); }
__device__ __forceinline__ float unscale_of(uint32_t s) { return __uint_as_float((254u - s) << 23); }

// 8 and 16 columns of this thread's row
__device__ __forceinline__ void load8(uint32_t taddr, bool zero, float (&v)[8]) {
  uint32_t r[8];
  if (!zero) {
    tmem_ld8(taddr, r);
    tmem_ld_wait();
  }
#pragma unroll
  for (int q = 0; q < 8; ++q) v[q] = zero ? 0.f : __uint_as_float(r[q]);
}
__device__ __forceinline__ void load16(uint32_t taddr, bool zero, float (&v)[16]) {
  uint32_t r[16];
  if (!zero) {
    tmem_ld16(taddr, r);
    tmem_ld_wait();
  }
#pragma unroll
  for (int q = 0; q < 16; ++q) v[q] = zero ? 0.f : __uint_as_float(r[q]);
}
// A block's 16 columns of this thread's row in P bf16 planes, 32 bytes a store: a whole sector, so that nothing is
// gained by bringing rows together in shared memory first (bulk stores of 64-byte rows from there: 145 and 122 us for
// 142 and 105 at the same point, 8192 x 1536 x 4096).
__device__ __forceinline__ void store16(const uint32_t (&w)[8], bf16* p) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
               "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
               : "memory");
}
__device__ __forceinline__ void pack8(const float* v, uint32_t* w) {
#pragma unroll
  for (int q = 0; q < 4; ++q) w[q] = pack_bf16(v[2 * q], v[2 * q + 1]);
}
template <int P>
__device__ __forceinline__ void store_planes(float (&v)[16], bf16* p, int64_t plane) {
#pragma unroll
  for (int k = 0; k < P; ++k) {
    uint32_t w[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      w[q] = pack_bf16(v[2 * q], v[2 * q + 1]);
      v[2 * q] -= __uint_as_float(w[q] << 16);
      v[2 * q + 1] -= __uint_as_float(w[q] & 0xffff0000u);
    }
    store16(w, p + k * plane);
  }
}

// ---- g, u -> h ------------------------------------------------------------------

// P: planes of h (3: fp32 inputs)
template <int ACT, int P>
struct EpiGated {
  static constexpr bool kNarrow = true, kWide = false, kChain = P == 3, kBegin = false;
  static constexpr int kSecond = kSecondHalves;
  static constexpr bool F32 = P == 3;
  struct Pre {};
  __device__ __forceinline__ void fetch(Pre&, const MmArgs&, MmTile, int, int, int) const {}
  bf16* h;  // [P][tokens][ld]
  int64_t ld, plane;
  Kept kept;  // gu null: nothing is kept
  int ff;

  __device__ __forceinline__ void keep(const float (&g)[16], const float (&u)[16], int row0, int col, int lane) const {
    const int64_t at = (int64_t)(row0 / 32) * kept.blocks + col / 16;
    if constexpr (F32) {
      uint4* dst = reinterpret_cast<uint4*>(kept.gu + at * 4096) + lane;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        dst[32 * c] = make_uint4(__float_as_uint(g[4 * c]), __float_as_uint(g[4 * c + 1]), __float_as_uint(g[4 * c + 2]),
                                 __float_as_uint(g[4 * c + 3]));
        dst[32 * c + 128] = make_uint4(__float_as_uint(u[4 * c]), __float_as_uint(u[4 * c + 1]), __float_as_uint(u[4 * c + 2]),
                                       __float_as_uint(u[4 * c + 3]));
      }
    } else {
      uint4* dst = reinterpret_cast<uint4*>(kept.gu + at * 2048) + lane;
      const uint32_t sg = block_scale(g), su = block_scale(u);
      const float fg = scale_of(sg), fu = scale_of(su);
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const float *x = g + 8 * c, *y = u + 8 * c;
        dst[32 * c] = make_uint4(pack_half(x[0] * fg, x[1] * fg), pack_half(x[2] * fg, x[3] * fg),
                                 pack_half(x[4] * fg, x[5] * fg), pack_half(x[6] * fg, x[7] * fg));
        dst[32 * c + 64] = make_uint4(pack_half(y[0] * fu, y[1] * fu), pack_half(y[2] * fu, y[3] * fu),
                                      pack_half(y[4] * fu, y[5] * fu), pack_half(y[6] * fu, y[7] * fu));
      }
      kept.scale[at * 32 + lane] = (uint16_t)(sg | su << 8);
    }
  }

  template <int CW, int BR>
  __device__ __forceinline__ void tile(const MmArgs&, MmTile, int row, int col0, int M, uint32_t taddr, bool zero, uint8_t*,
                                       Pre&) const {
    constexpr int W = CW / 2;  // of the BR columns: BR / 2 of g, BR / 2 of u; this warp's: W of each
    static_assert(W % kBlock == 0, "whole blocks");
    const int lane = threadIdx.x % 32, row0 = row - lane, o = col0 % BR, f0 = (col0 - o) / 2 + o / 2;
    if (row0 >= M) return;  // warp-uniform
    const uint32_t gt = taddr - o + o / 2, ut = gt + BR / 2;
#pragma unroll 1
    for (int cc = 0; cc < W; cc += 16) {
      const int col = f0 + cc;
      if (col >= ff) break;  // warp-uniform
      float g[16], u[16];
      load16(gt + cc, zero, g);
      load16(ut + cc, zero, u);
      if (kept.gu) keep(g, u, row0, col, lane);
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        float a, slope;
        activation<ACT, P>(g[q], a, slope);
        g[q] = a * u[q];
      }
      bf16* dst = h + row * ld + col;
      if (row < M) store_planes<P>(g, dst, plane);
    }
  }
};

// ---- dh -> dg, du and h again ----------------------------------------------------

template <int ACT, int P>
struct EpiGrad {
  static constexpr bool kNarrow = true, kWide = false, kChain = P == 3, kBegin = false;
  static constexpr bool F32 = P == 3;
  struct Pre {
    uint4 x[F32 ? 8 : 4];
    uint32_t scale;
  };
  bf16* dgu;  // [tokens][P][2][ld] (dg, du), or null
  bf16* h;    // [P][tokens][ld], or null
  int64_t ld, plane;
  Kept kept;

  __device__ __forceinline__ void ask(Pre& pre, int row0, int col, int lane) const {
    const int64_t at = (int64_t)(row0 / 32) * kept.blocks + col / 16;
    const uint4* src = reinterpret_cast<const uint4*>(kept.gu + at * (F32 ? 4096 : 2048)) + lane;
#pragma unroll
    for (int c = 0; c < (F32 ? 8 : 4); ++c) pre.x[c] = src[32 * c];
    if (!F32) pre.scale = kept.scale[at * 32 + lane];
  }
  __device__ __forceinline__ void fetch(Pre& pre, const MmArgs& a, MmTile, int row, int col0, int M) const {
    const int lane = threadIdx.x % 32;
    if (row - lane < M && col0 < a.N) ask(pre, row - lane, col0, lane);
  }
  // columns [8 e, 8 e + 8) of the block
  static __device__ __forceinline__ void values(const Pre& pre, int e, float (&g)[8], float (&u)[8]) {
    if constexpr (F32) {
#pragma unroll
      for (int q = 0; q < 8; ++q) {
        g[q] = __uint_as_float(word(pre.x, 8 * e + q));
        u[q] = __uint_as_float(word(pre.x, 16 + 8 * e + q));
      }
    } else {
      const float fg = unscale_of(pre.scale & 255u), fu = unscale_of(pre.scale >> 8);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const uint32_t wg = word(pre.x, 4 * e + q), wu = word(pre.x, 8 + 4 * e + q);
        const float2 pg = __half22float2(*reinterpret_cast<const __half2*>(&wg));
        const float2 pu = __half22float2(*reinterpret_cast<const __half2*>(&wu));
        g[2 * q] = pg.x * fg;
        g[2 * q + 1] = pg.y * fg;
        u[2 * q] = pu.x * fu;
        u[2 * q + 1] = pu.y * fu;
      }
    }
  }

  // One block of 16 columns after another, in halves: what a warp holds of it has to fit beside the block
  // that it has asked for in 96 registers (whole blocks spill 112 bytes, two at a time 208: 8192 x
  // 1536 x 4096, 122 us).
  template <int CW>
  __device__ __forceinline__ void tile(const MmArgs& a, MmTile, int row, int col0, int M, uint32_t taddr, bool zero, uint8_t*,
                                       Pre& pre) const {
    const int lane = threadIdx.x % 32, row0 = row - lane;
    if (row0 >= M) return;  // warp-uniform
#pragma unroll 1
    for (int cc = 0; cc < CW; cc += 16) {
      const int col = col0 + cc;
      if (col >= a.N) break;  // warp-uniform
      bf16 *hd = h + row * ld + col, *gd = dgu + 2 * P * (row * ld) + col;
      uint32_t wh[8], wg[8], wu[8];  // (P = 1)
      float vh[16], vg[16], vu[16];  // (otherwise)
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float g[8], u[8], dh[8];
        values(pre, e, g, u);
        if (e == 1 && cc + 16 < CW && col + 16 < a.N) ask(pre, row0, col + 16, lane);  // while this block is worked on
        load8(taddr + cc + 8 * e, zero, dh);
#pragma unroll
        for (int q = 0; q < 8; ++q) {
          float act, slope;
          activation<ACT, P>(g[q], act, slope);
          g[q] = act * u[q];
          u[q] = dh[q] * u[q] * slope;
          dh[q] *= act;
        }
        if constexpr (P == 1) {
          pack8(g, wh + 4 * e);
          pack8(u, wg + 4 * e);
          pack8(dh, wu + 4 * e);
        } else {
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            vh[8 * e + q] = g[q];
            vg[8 * e + q] = u[q];
            vu[8 * e + q] = dh[q];
          }
        }
      }
      if (row >= M) continue;
      if constexpr (P == 1) {
        if (h) store16(wh, hd);
        if (dgu) {
          store16(wg, gd);
          store16(wu, gd + ld);
        }
      } else {
        if (h) store_planes<P>(vh, hd, plane);
        if (dgu) {
          store_planes<P>(vg, gd, 2 * ld);
          store_planes<P>(vu, gd + ld, 2 * ld);
        }
      }
    }
  }
};

// ---- dWg and dWu ------------------------------------------------------------------

// Row m of the product is row m of dWg (m < ff) or m - half of dWu.
struct EpiTwo {
  static constexpr bool kNarrow = true, kWide = true, kChain = true, kBegin = false;
  struct Pre {};
  __device__ __forceinline__ void fetch(Pre&, const MmArgs&, MmTile, int, int, int) const {}
  void *first, *second;  // each may be null
  int64_t ldo;
  int half, ff, out_bf16, vec;

  __device__ __forceinline__ uint8_t* at(int row, int col) const {
    const int t = row >= half, r = row - t * half;
    uint8_t* base = static_cast<uint8_t*>(t ? second : first);
    return base && r < ff ? base + (r * ldo + col) * (out_bf16 ? 2 : 4) : nullptr;
  }
  __device__ __forceinline__ void quad(int row, int col, int n, float4 v) const {
    uint8_t* dst = at(row, col);
    if (!dst) return;
    const float x[4] = {v.x, v.y, v.z, v.w};
    if (out_bf16) {
      if (vec) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
      } else {
        for (int q = 0; q < n; ++q) reinterpret_cast<bf16*>(dst)[q] = __float2bfloat16_rn(x[q]);
      }
    } else if (vec) {
      *reinterpret_cast<float4*>(dst) = v;
    } else {
      for (int q = 0; q < n; ++q) reinterpret_cast<float*>(dst)[q] = x[q];
    }
  }
  template <int CW>
  __device__ __forceinline__ void tile(const MmArgs& a, MmTile, int row, int col0, int M, uint32_t taddr, bool zero,
                                       uint8_t* buf, Pre&) const {
    const int lane = threadIdx.x % 32;
    const MappedRows dst{row < M ? at(row, col0) : nullptr};
    if (CW == 128 && out_bf16 && vec) {  // whole 128-byte lines
#pragma unroll 1
      for (int cc = 0; cc < CW; cc += 64) {
        const int n = a.N - col0 - cc;
        if (n <= 0) break;
        uint4 u[8];
        row64_bf16(taddr + cc, zero, 1.f, u);
        block_store(buf, lane, u, dst.at(cc * 2), n * 2);
      }
      return;
    }
#pragma unroll 1
    for (int cc = 0; cc < CW; cc += 32) {
      const int n = a.N - col0 - cc;
      if (n <= 0) break;  // warp-uniform
      float v[32];
      load32(taddr + cc, zero, v);
      if (out_bf16) {
        uint4 u[4];
        bf16_row(v, u);
        if (vec)
          block_store(buf, lane, u, dst.at(cc * 2), n * 2);
        else
          block_store_odd<bf16>(buf, lane, u, dst.at(cc * 2), n);
      } else {
        uint4 u[8];
        f32_row(v, u);
        if (vec)
          block_store(buf, lane, u, dst.at(cc * 4), n * 4);
        else
          block_store_odd<float>(buf, lane, u, dst.at(cc * 4), n);
      }
    }
  }
};

// dx: term t of the inner width's halves takes Wg or Wu
struct EpiDx : EpiOut {
  static constexpr int kSecond = kSecondTerms;
};

// ---- host side ------------------------------------------------------------------

struct Plan {
  bool f32, fine;
  int elt, planes, hplanes;
  bool pack_x, pack_g, pack_u, pack_d, pack_dy;
  int64_t ldx, ldg, ldu, ldd, ldy, ldf;
  int blocks;
  size_t x, g, u, d, dy, h, dgu, part, total;
};

MmArgs product(const Plan& q, int M, int N, int K, volatile unsigned* fault) {
  MmArgs p = {};
  p.M = M;
  p.N = N;
  p.K = K;
  p.nz = 1;
  p.n_terms = q.f32 ? 6 : 1;
  p.pa = q.f32 ? kTermsA : 0;
  p.pb = q.f32 ? kTermsB : 0;
  p.chain = q.f32 ? (q.fine ? kFineF32Chain : kF32Chain) : K > kLongSum ? kLongChain : 0;
  p.fault_host = fault;
  return p;
}
// y = h Wd^T
MmArgs y_args(const Plan& q, const llattn_gated_args& a, volatile unsigned* fault) {
  MmArgs p = product(q, a.tokens, a.d_out, a.ff, fault);
  if (q.hplanes == 2) {
    p.n_terms = 2;
    p.pa = 0x01u;
  }
  p.split = 2;
  return p;
}
// dx = dg Wg + du Wu: for each term of fp32's planes (or of G's two), smallest first, a
// pass over each half. dgu's z is 2 plane + half.
MmArgs dx_args(const Plan& q, const llattn_gated_args& a, volatile unsigned* fault) {
  MmArgs p = product(q, a.tokens, a.d, a.ff, fault);
  const int n = q.f32 ? 6 : q.hplanes;
  const uint64_t ta = q.f32 ? kTermsA : q.hplanes == 2 ? 0x01u : 0u, tb = q.f32 ? kTermsB : 0u;
  p.pa = p.pb = 0;
  for (int t = 0; t < n; ++t)
    for (int half = 0; half < 2; ++half) {
      p.pa |= (2 * ((ta >> (4 * t)) & 15u) + half) << (4 * (2 * t + half));
      p.pb |= ((tb >> (4 * t)) & 15u) << (4 * (2 * t + half));
      p.b2 |= (uint32_t)half << (2 * t + half);
    }
  p.n_terms = 2 * n;
  p.majors = 2;
  p.split = 2;
  return p;
}
// dWd = dy^T h
MmArgs dwd_args(const Plan& q, const llattn_gated_args& a, volatile unsigned* fault) {
  MmArgs p = product(q, a.d_out, a.ff, a.tokens, fault);
  if (q.hplanes == 2) {
    p.n_terms = 2;
    p.pb = 0x01u;
  }
  p.split = 2;
  return p;
}
// [dWg; dWu] = [dg, du]^T x
MmArgs dwgu_args(const Plan& q, const llattn_gated_args& a, volatile unsigned* fault) {
  MmArgs p = product(q, (int)(2 * q.ldf), a.d, a.tokens, fault);
  if (q.hplanes == 2) {
    p.n_terms = 2;
    p.pa = 0x01u;
  }
  p.split = 2;
  return p;
}

Plan make_plan(const llattn_gated_args& a, bool backward) {
  Plan q;
  q.f32 = a.dtype == LLATTN_F32;
  q.fine = a.tokens <= kFine;
  q.elt = q.f32 ? 4 : 2;
  q.planes = q.f32 ? 3 : 1;
  q.hplanes = q.f32 ? 3 : q.fine ? 2 : 1;
  const int64_t n = a.tokens;
  auto pack = [&](const void* p, int64_t ld, int64_t rows) { return q.f32 || !aligned_rows(p, ld, rows, 2); };
  auto stride = [&](bool packed, int64_t ld, int64_t rows, int cols) { return packed || rows == 1 ? up8(cols) : ld; };
  q.pack_x = pack(a.x, a.ldx, n);
  q.pack_g = pack(a.w_gate, a.ldg, a.ff);
  q.pack_u = pack(a.w_up, a.ldu, a.ff);
  q.pack_d = pack(a.w_down, a.ldd, a.d_out);
  q.pack_dy = backward && pack(a.dy, a.lddy, n);
  q.ldx = stride(q.pack_x, a.ldx, n, a.d);
  q.ldg = stride(q.pack_g, a.ldg, a.ff, a.d);
  q.ldu = stride(q.pack_u, a.ldu, a.ff, a.d);
  q.ldd = stride(q.pack_d, a.ldd, a.d_out, a.ff);
  q.ldy = stride(q.pack_dy, a.lddy, n, a.d_out);
  q.ldf = cdiv(a.ff, kBlock) * kBlock;
  q.blocks = cdiv(a.ff, kBlock);
  const bool need_x = !backward || a.dw_gate || a.dw_up, need_gu = !backward || a.dx, inner = a.dx || a.dw_gate || a.dw_up;
  size_t off = 0;
  auto take = [&](size_t b) { size_t o = off; off += up256(b); return o; };
  const size_t pl = 2 * (size_t)q.planes;
  q.x = take(q.pack_x && need_x ? pl * n * q.ldx : 0);
  q.g = take(q.pack_g && need_gu ? pl * a.ff * q.ldg : 0);
  q.u = take(q.pack_u && need_gu ? pl * a.ff * q.ldu : 0);
  q.d = take(q.pack_d ? pl * a.d_out * q.ldd : 0);
  q.dy = take(q.pack_dy ? pl * n * q.ldy : 0);
  q.h = take(!backward || a.dw_down ? 2 * (size_t)q.hplanes * n * q.ldf : 0);
  q.dgu = take(backward && inner ? 4 * (size_t)q.hplanes * n * q.ldf : 0);
  int64_t part = 0;
  if (!backward) {
    part = mm_part_floats(y_args(q, a, nullptr));
  } else {
    if (a.dx) part = mm_part_floats(dx_args(q, a, nullptr));
    if (a.dw_down) part = std::max(part, mm_part_floats(dwd_args(q, a, nullptr)));
    if (a.dw_gate || a.dw_up) part = std::max(part, mm_part_floats(dwgu_args(q, a, nullptr)));
  }
  q.part = take(4 * (size_t)part);
  q.total = off;
  return q;
}

Kept kept_at(const Plan& q, const llattn_gated_args& a) {
  Kept k;
  k.gu = static_cast<uint8_t*>(a.kept);
  k.blocks = q.blocks;
  k.scale = reinterpret_cast<uint16_t*>(k.gu + (size_t)cdiv(a.tokens, 32) * q.blocks * 2048);
  return k;
}

EpiOut rows_out(const Plan& q, void* out, int cols) {
  EpiOut o{};
  o.out = out;
  o.ldo = cols;
  o.out_bf16 = !q.f32;
  o.vec = aligned_rows(out, cols, 2, q.elt);
  return o;
}

// The tiles of the two products with the activation in their epilogues: shape 5
// instead of 2 for bf16 (fp32's values spill in 96 registers: steps of 2048 x 1024 x 2816 774 us for 710, of 8192 x
// 1536 x 4096 5600 for 5250; 620 and 4650 since with stores of whole sectors), and for g and u at least 32 columns of each to a warp (shape 0 holds 16).
template <typename Epi>
cudaError_t launch_active(MmArgs p, const Operand& a, const Operand& b, const Epi& e, cudaStream_t s,
                          const Operand* b2 = nullptr) {
  p.a_mn = a.mn;
  p.b_mn = b.mn;
  if constexpr (!Epi::F32) {  // (d or d_out: one shape will do)
    if (p.chain) return launch_mm_sh<1, true>(p, a, b, e, s, b2);
  }
  const double t2 = mm_time<2>(p), t1 = mm_time<1>(p), t4 = mm_time<4>(p);
  if constexpr (SecondB<Epi>::value != kSecondHalves) {
    const double t0 = mm_time<0>(p);
    if (t0 <= t4 && t0 < std::min(t1, t2)) return launch_mm_sh<0>(p, a, b, e, s, b2);
  }
  if (t4 < std::min(t1, t2)) return launch_mm_sh<4>(p, a, b, e, s, b2);
  if (t2 <= t1) return launch_mm_sh<Epi::F32 ? 2 : 5>(p, a, b, e, s, b2);
  return launch_mm_sh<1>(p, a, b, e, s, b2);
}

template <typename T, int ACT, int P>
cudaError_t run_fwd(const llattn_gated_args& a, const Plan& q, volatile unsigned* fault, cudaStream_t s) {
  char* ws = static_cast<char*>(a.workspace);
  const int n = a.tokens;
  Packs packs = {};
  if (q.pack_x) packs.add(a.x, a.ldx, n, a.d, ws + q.x, q.ldx);
  if (q.pack_g) packs.add(a.w_gate, a.ldg, a.ff, a.d, ws + q.g, q.ldg);
  if (q.pack_u) packs.add(a.w_up, a.ldu, a.ff, a.d, ws + q.u, q.ldu);
  if (q.pack_d) packs.add(a.w_down, a.ldd, a.d_out, a.ff, ws + q.d, q.ldd);
  TRY(launch_packs<T>(packs, s));
  const Operand x{q.pack_x ? ws + q.x : a.x, n, a.d, q.ldx, q.planes, n * q.ldx, 0};
  const Operand g{q.pack_g ? ws + q.g : a.w_gate, a.ff, a.d, q.ldg, q.planes, a.ff * q.ldg, 0};
  const Operand u{q.pack_u ? ws + q.u : a.w_up, a.ff, a.d, q.ldu, q.planes, a.ff * q.ldu, 0};
  const Operand d{q.pack_d ? ws + q.d : a.w_down, a.d_out, a.ff, q.ldd, q.planes, a.d_out * q.ldd, 0};
  bf16* h = reinterpret_cast<bf16*>(ws + q.h);
  const int64_t hplane = n * q.ldf;
  EpiGated<ACT, P> e{};
  e.ff = a.ff;
  e.h = h;
  e.ld = q.ldf;
  e.plane = hplane;
  if (a.kept) e.kept = kept_at(q, a);
  TRY(launch_active(product(q, n, 2 * a.ff, a.d, fault), x, g, e, s, &u));
  MmArgs p = y_args(q, a, fault);
  p.part = reinterpret_cast<float*>(ws + q.part);
  return launch_mm(p, Operand{h, n, a.ff, q.ldf, P, hplane, 0}, d, rows_out(q, a.y, a.d_out), s);
}

template <typename T, int ACT, int P>
cudaError_t run_bwd(const llattn_gated_args& a, const Plan& q, volatile unsigned* fault, cudaStream_t s) {
  char* ws = static_cast<char*>(a.workspace);
  const int n = a.tokens;
  const bool weights = a.dw_gate || a.dw_up;
  Packs packs = {};
  if (q.pack_dy) packs.add(a.dy, a.lddy, n, a.d_out, ws + q.dy, q.ldy);
  if (q.pack_d) packs.add(a.w_down, a.ldd, a.d_out, a.ff, ws + q.d, q.ldd);
  if (q.pack_g && a.dx) packs.add(a.w_gate, a.ldg, a.ff, a.d, ws + q.g, q.ldg);
  if (q.pack_u && a.dx) packs.add(a.w_up, a.ldu, a.ff, a.d, ws + q.u, q.ldu);
  if (q.pack_x && weights) packs.add(a.x, a.ldx, n, a.d, ws + q.x, q.ldx);
  TRY(launch_packs<T>(packs, s));
  const void* dy = q.pack_dy ? ws + q.dy : a.dy;
  const int64_t dyplane = n * q.ldy, hplane = n * q.ldf;
  bf16 *h = reinterpret_cast<bf16*>(ws + q.h), *dgu = reinterpret_cast<bf16*>(ws + q.dgu);
  float* part = reinterpret_cast<float*>(ws + q.part);
  EpiGrad<ACT, P> e{};
  e.kept = kept_at(q, a);
  e.dgu = a.dx || weights ? dgu : nullptr;
  e.h = a.dw_down ? h : nullptr;
  e.ld = q.ldf;
  e.plane = hplane;
  TRY(launch_active(product(q, n, a.ff, a.d_out, fault), Operand{dy, n, a.d_out, q.ldy, q.planes, dyplane, 0},
                Operand{q.pack_d ? ws + q.d : a.w_down, a.d_out, a.ff, q.ldd, q.planes, a.d_out * q.ldd, 1}, e, s));
  if (a.dx) {
    MmArgs p = dx_args(q, a, fault);
    p.part = part;
    const Operand g{q.pack_g ? ws + q.g : a.w_gate, a.ff, a.d, q.ldg, q.planes, a.ff * q.ldg, 1};
    const Operand u{q.pack_u ? ws + q.u : a.w_up, a.ff, a.d, q.ldu, q.planes, a.ff * q.ldu, 1};
    EpiDx o{rows_out(q, a.dx, a.d)};
    TRY(launch_mm(p, Operand{dgu, n, a.ff, 2 * P * q.ldf, 2 * P, q.ldf, 0}, g, o, s, &u));
  }
  if (a.dw_down) {
    MmArgs p = dwd_args(q, a, fault);
    p.part = part;
    TRY(launch_mm(p, Operand{dy, n, a.d_out, q.ldy, q.planes, dyplane, 1}, Operand{h, n, a.ff, q.ldf, P, hplane, 1},
                  rows_out(q, a.dw_down, a.ff), s));
  }
  if (weights) {
    MmArgs p = dwgu_args(q, a, fault);
    p.part = part;
    EpiTwo o{};
    o.first = a.dw_gate;
    o.second = a.dw_up;
    o.ldo = a.d;
    o.half = (int)q.ldf;
    o.ff = a.ff;
    o.out_bf16 = !q.f32;
    o.vec = (!a.dw_gate || aligned_rows(a.dw_gate, a.d, 2, q.elt)) && (!a.dw_up || aligned_rows(a.dw_up, a.d, 2, q.elt));
    TRY(launch_mm(p, Operand{dgu, n, 2 * q.ldf, 2 * P * q.ldf, P, 2 * q.ldf, 1},
                  Operand{q.pack_x ? ws + q.x : a.x, n, a.d, q.ldx, q.planes, n * q.ldx, 1}, o, s));
  }
  return cudaSuccess;
}

template <int ACT>
cudaError_t run(const llattn_gated_args& a, bool backward, volatile unsigned* fault, cudaStream_t s) {
  const Plan q = make_plan(a, backward);
  if (q.f32) return backward ? run_bwd<float, ACT, 3>(a, q, fault, s) : run_fwd<float, ACT, 3>(a, q, fault, s);
  if (q.hplanes == 2) return backward ? run_bwd<bf16, ACT, 2>(a, q, fault, s) : run_fwd<bf16, ACT, 2>(a, q, fault, s);
  return backward ? run_bwd<bf16, ACT, 1>(a, q, fault, s) : run_fwd<bf16, ACT, 1>(a, q, fault, s);
}

}  // namespace

size_t kept_bytes(const llattn_gated_args& a) {
  return (size_t)cdiv(a.tokens, 32) * cdiv(a.ff, kBlock) * (a.dtype == LLATTN_F32 ? 4096 : 2048 + 64);
}

static bool few(const llattn_gated_args& a, bool backward) { return !backward && !a.kept && a.tokens <= few_tokens(a); }

size_t workspace_bytes(const llattn_gated_args& a, bool backward) {
  if (few(a, backward)) return up256(few_workspace_bytes(a));
  return std::max<size_t>(256, make_plan(a, backward).total);
}

int launches(const llattn_gated_args& a, bool backward) {
  if (few(a, backward)) return 2;
  const Plan q = make_plan(a, backward);
  const bool weights = a.dw_gate || a.dw_up;
  if (!backward) return (q.pack_x || q.pack_g || q.pack_u || q.pack_d) + 1 + mm_launches<EpiOut>(y_args(q, a, nullptr), 0, 0);
  int n = (q.pack_dy || q.pack_d || (a.dx && (q.pack_g || q.pack_u)) || (weights && q.pack_x)) + 1;
  if (a.dx) n += mm_launches<EpiDx>(dx_args(q, a, nullptr), 0, 1);
  if (a.dw_down) n += mm_launches<EpiOut>(dwd_args(q, a, nullptr), 1, 1);
  if (weights) n += mm_launches<EpiTwo>(dwgu_args(q, a, nullptr), 1, 1);
  return n;
}

cudaError_t launch(const llattn_gated_args& a, bool backward, volatile unsigned* fault, cudaStream_t s) {
  if (few(a, backward)) return launch_few(a, s);
  return a.activation == LLATTN_ACT_SILU ? run<LLATTN_ACT_SILU>(a, backward, fault, s)
                                         : run<LLATTN_ACT_GELU>(a, backward, fault, s);
}

unsigned read_fault_word(bool reset) { return read_fault(reset); }

}  // namespace gated
}  // namespace llattn
