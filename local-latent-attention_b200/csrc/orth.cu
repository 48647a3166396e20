// Orthogonalised updates by Newton-Schulz products: for each matrix G of a
// batch (short side q = min(m, n); written for the short side first)
//   X0 = G / (|G|_F + eps),  S = X X^T,  B = b S + c S^2,  X <- a X + B X
// repeated `steps` times, which drives every singular value of X towards 1.
// (No counterpart in the reference, whose training uses AdamW.)
//
// Three products per step on mm_kernel (mm_sm100.cuh) with 16-bit operands
// and fp32 accumulation. A tall matrix keeps its orientation: S = X^T X reads
// X with the columns as rows (MN-major), and the update is X B. S and B are
// symmetric: only tiles on and below the diagonal are computed, the epilogue
// writes each one's mirror image as well.
//
// 16 bits: fp16, whose 11 bits cost the same as bf16's 8; values are kept in
// its range by powers of two: X * 2^6, S * 2^8 and B * 2^8 (entries of X and S
// are at most about 1.2, those of B at most |b| + |c| times that). The
// starting X is G times a power of two near 2^6 / |G| (exact for bf16 G), the
// rest of the normalisation is a factor s0 in the first step's epilogues.
//
// Two roundings matter and are compensated:
//  * a X: early steps multiply the smallest singular values by a = 3.4 each
//    time, and the rounding of X with them. The update's linear term reads X
//    as hi + lo (fp16 and the remainder in bf16); only the products use hi,
//    where small singular values enter cubed.
//  * B near the end is close to (b + c) I, and a X + B X cancels to about
//    (a + b + c) X: rounding B would cost 4 times its 2^-12. The last two
//    steps therefore hold B + a I, about (a + b + c) I, and update by the
//    product alone, which also saves their epilogues the reading of X.
// Measured on the CPU in the same arithmetic: 0.5 to 1.6e-3 (2-norm) from the
// exact iteration over spectra from flat to 1 / k, where plain bf16 products
// give 1 to 4e-2.
#include <cooperative_groups.h>
#include <math.h>

#include <algorithm>
#include <array>
#include <map>
#include <mutex>

#include "mm_sm100.cuh"
#include "xent.cuh"

namespace llattn {
namespace orth {
namespace {

using namespace mm;

constexpr float kX = 64.f, kS = 256.f;  // scales of X and of S, B
constexpr int kFolded = 2;              // last steps that hold B + a I
constexpr int kParts = 64;              // partial sums of squares per matrix
constexpr int kPtrs = 64;               // matrices per conversion launch
// Gram sums of more than kLong K = 64 steps run in chains of kGramChain (MmArgs::chain).
// In one sum they come out up to 3 x 2^-26 per 16 products short, 5e-5 at the
// limit and 6e-4 of all of S at 200000, which five steps' polynomials make
// several times that (a flat 1 x 200000: 4.1e-3 of the result, 2.2e-3 in chains;
// 5 x 300000 3.6e-3 and 2.8e-3, in the same time).
constexpr int kLong = 256, kGramChain = 64;

struct Ptrs {
  const void* p[kPtrs];
};

// Stores 32 columns of a symmetric matrix's tile, and off the diagonal (of the
// square tile shapes, which skip those above it) their mirror image: column nc + lane of the block becomes that row, from row0 on.
__device__ __forceinline__ void store_symmetric(__half* base, int64_t ld, bool mirror, int row, int nc, int M, int N,
                                                const float (&v)[32], uint8_t* buf) {
  const int lane = threadIdx.x % 32, row0 = row - lane;
  uint4 u[4];
  half_row(v, u);
  block_store(buf, lane, u, Rows{base + row0 * ld + nc, ld * 2, M - row0}, (N - nc) * 2);
  if (mirror) block_mirror(buf, lane, Rows{base + nc * ld + row0, ld * 2, N - nc}, (M - row0) * 2);
}

// S = X X^T (scaled by kS), from hi * 2^6 (or the first step's G * 2^e)
struct EpiGram {
  static constexpr bool kNarrow = true, kWide = false, kChain = true, kBegin = false;
  struct Pre {};
  __device__ __forceinline__ void fetch(Pre&, const MmArgs&, MmTile, int, int, int) const {}
  __half* s;
  int64_t ld, zs;
  const float* s0;  // first step: X = s0[z] * stored, else null (2^-6)
  template <int CW>
  __device__ __forceinline__ void tile(const MmArgs& a, MmTile w, int row, int col0, int M, uint32_t taddr,
                                       bool zero, uint8_t* buf, Pre&) const {
    const float x = s0 ? s0[w.z] : 1.f / kX;
    const float f = x * x * kS;
    __half* base = s + w.z * zs;
#pragma unroll 1
    for (int cc = 0; cc < CW; cc += 32) {
      const int nc = col0 + cc;
      if (nc >= a.N) break;
      float v[32];
      load32(taddr + cc, zero, v);
#pragma unroll
      for (int q = 0; q < 32; ++q) v[q] *= f;
      store_symmetric(base, ld, a.sym && w.m0 != w.n0, row, nc, M, a.N, v, buf);
    }
  }
};

// B = b S + c S^2 + k I (scaled by kS)
struct EpiPoly {
  static constexpr bool kNarrow = true, kWide = false, kChain = false, kBegin = false;
  const __half* s;
  __half* b;
  int64_t ld, zs;
  float cb, cc2, k;  // b, c / kS, k * kS
  struct Pre {
    uint4 u[4];
  };
  __device__ __forceinline__ Rows src(const MmTile& w, int row0, int col0, int M) const {
    return Rows{s + w.z * zs + row0 * ld + col0, ld * 2, M - row0};
  }
  __device__ __forceinline__ void fetch(Pre& pre, const MmArgs& a, MmTile w, int row, int col0, int M) const {
    const int lane = threadIdx.x % 32;
    if (col0 < a.N) block_fetch(lane, pre.u, src(w, row - lane, col0, M), (a.N - col0) * 2);
  }
  template <int CW>
  __device__ __forceinline__ void tile(const MmArgs& a, MmTile w, int row, int col0, int M, uint32_t taddr,
                                       bool zero, uint8_t* buf, Pre& pre) const {
    const int lane = threadIdx.x % 32;
    __half* base = b + w.z * zs;
    const Rows from = src(w, row - lane, col0, M);
    uint4(&u)[4] = pre.u;  // fetched a block ahead: its latency passes during the stores
#pragma unroll 1
    for (int cc = 0; cc < CW; cc += 32) {
      const int nc = col0 + cc, n = a.N - nc;
      if (n <= 0) break;
      float v[32];
      load32(taddr + cc, zero, v);
      block_spread(buf, lane, u);
#pragma unroll
      for (int q = 0; q < 16; ++q) {
        const float2 x = half_pair(u, q);
        v[2 * q] = fmaf(cb, x.x, cc2 * v[2 * q]) + (row == nc + 2 * q ? k : 0.f);
        v[2 * q + 1] = fmaf(cb, x.y, cc2 * v[2 * q + 1]) + (row == nc + 2 * q + 1 ? k : 0.f);
      }
      if (cc + 32 < CW && n > 32) block_fetch(lane, u, from.at((cc + 32) * 2), (n - 32) * 2);
      store_symmetric(base, ld, a.sym && w.m0 != w.n0, row, nc, M, a.N, v, buf);
    }
  }
};

// X <- a X + B X, or (B + a I) X
struct EpiUpdate {
  static constexpr bool kNarrow = true, kWide = false, kChain = false, kBegin = false;
  const __half* hi;
  bf16* lo;          // remainder of X, read where rd_lo, written (in place) where wr_lo
  __half* next;      // next X (hi), or null in the last step
  bf16* out;         // last step: [count, rows, cols]
  int64_t ld, zs, ldo, zso;
  const float* s0;
  float ca;          // a
  int rd_hi, rd_lo, wr_lo, vec_out;
  struct Pre {
    uint4 h[4], l[4];
  };
  // 32 columns of hi and lo, n of them valid
  __device__ __forceinline__ void block(Pre& pre, int64_t at, int rows, int n) const {
    const int lane = threadIdx.x % 32;
    if (rd_hi) block_fetch(lane, pre.h, Rows{hi + at, ld * 2, rows}, n * 2);
    if (rd_lo) block_fetch(lane, pre.l, Rows{lo + at, ld * 2, rows}, n * 2);
  }
  __device__ __forceinline__ void fetch(Pre& pre, const MmArgs& a, MmTile w, int row, int col0, int M) const {
    const int row0 = row - (int)(threadIdx.x % 32);
    if (col0 < a.N) block(pre, w.z * zs + row0 * ld + col0, M - row0, a.N - col0);
  }
  template <int CW>
  __device__ __forceinline__ void tile(const MmArgs& a, MmTile w, int row, int col0, int M, uint32_t taddr,
                                       bool zero, uint8_t* buf, Pre& pre) const {
    const int lane = threadIdx.x % 32;
    const int row0 = row - lane, rows = M - row0;
    const float x = s0 ? s0[w.z] : 1.f / kX;
    const float fl = ca * x, fp = x / kS;
    uint4(&h)[4] = pre.h, (&l)[4] = pre.l;  // fetched a block ahead, as in EpiPoly
#pragma unroll 1
    for (int cc = 0; cc < CW; cc += 32) {
      const int nc = col0 + cc, n = a.N - nc;
      if (n <= 0) break;
      const int64_t at = w.z * zs + row0 * ld + nc;
      float v[32];
      load32(taddr + cc, zero, v);
#pragma unroll
      for (int q = 0; q < 32; ++q) v[q] *= fp;
      if (rd_hi) {
        block_spread(buf, lane, h);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float2 y = half_pair(h, q);
          v[2 * q] = fmaf(fl, y.x, v[2 * q]);
          v[2 * q + 1] = fmaf(fl, y.y, v[2 * q + 1]);
        }
      }
      if (rd_lo) {
        block_spread(buf, lane, l);
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float2 y = bf16_pair(l, q);
          v[2 * q] = fmaf(fl, y.x, v[2 * q]);
          v[2 * q + 1] = fmaf(fl, y.y, v[2 * q + 1]);
        }
      }
      if (cc + 32 < CW && n > 32) block(pre, at + 32, rows, n - 32);
      uint4 u[4];
      if (out) {
        const Rows dst{out + w.z * zso + row0 * ldo + nc, ldo * 2, rows};
        bf16_row(v, u);
        if (vec_out)
          block_store(buf, lane, u, dst, n * 2);
        else
          block_store_odd<bf16>(buf, lane, u, dst, n);
        continue;
      }
#pragma unroll
      for (int q = 0; q < 32; ++q) v[q] *= kX;
      half_row(v, u);
      block_store(buf, lane, u, Rows{next + at, ld * 2, rows}, n * 2);
      if (wr_lo) {
#pragma unroll
        for (int q = 0; q < 16; ++q) {
          const float2 y = half_pair(u, q);
          v[2 * q] -= y.x;
          v[2 * q + 1] -= y.y;
        }
        bf16_row(v, u);
        block_store(buf, lane, u, Rows{lo + at, ld * 2, rows}, n * 2);
      }
    }
  }
};

// partial sums of squares of matrix blockIdx.y, fixed order
template <typename T>
__global__ void __launch_bounds__(256) orth_square(const __grid_constant__ Ptrs g, int64_t n, float* part) {
  __shared__ float red[8];
  pdl_next();
  pdl_wait();
  const T* src = static_cast<const T*>(g.p[blockIdx.y]);
  float s = 0.f;
  constexpr int VN = 16 / sizeof(T);
  if ((reinterpret_cast<uintptr_t>(src) & 15) == 0) {
    const int64_t nv = n / VN;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < nv; i += (int64_t)gridDim.x * 256) {
      const uint4 u = reinterpret_cast<const uint4*>(src)[i];
      if (sizeof(T) == 2) {
        float f[8];
        unpack8(u, f);
#pragma unroll
        for (int q = 0; q < 8; ++q) s = fmaf(f[q], f[q], s);
      } else {
        const float x = __uint_as_float(u.x), y = __uint_as_float(u.y), z = __uint_as_float(u.z),
                    t = __uint_as_float(u.w);
        s = fmaf(x, x, fmaf(y, y, fmaf(z, z, fmaf(t, t, s))));
      }
    }
    if (blockIdx.x == 0 && threadIdx.x < n - nv * VN) {
      const float x = to_f<T>(src[nv * VN + threadIdx.x]);
      s = fmaf(x, x, s);
    }
  } else {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
      const float x = to_f<T>(src[i]);
      s = fmaf(x, x, s);
    }
  }
  s = warp_sum(s);
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = s;
  __syncthreads();
  if (threadIdx.x == 0) {
    float r = 0.f;
    for (int i = 0; i < 8; ++i) r += red[i];
    part[blockIdx.y * kParts + blockIdx.x] = r;
  }
}

// hi = fp16(G 2^e), lo = bf16(G 2^e - hi) (optional), s0 = 2^-e / (|G| + eps)
template <typename T>
__global__ void __launch_bounds__(256) orth_convert(const __grid_constant__ Ptrs g, int rows, int cols,
                                                    const float* part, int n_parts, float eps,
                                                    __half* hi, bf16* lo, int64_t ld, int64_t zs,
                                                    float* s0) {
  __shared__ float sh[2];
  pdl_next();
  pdl_wait();
  const int z = blockIdx.y;
  if (threadIdx.x == 0) {
    float sum = 0.f;
    for (int i = 0; i < n_parts; ++i) sum += part[z * kParts + i];
    const float inv = 1.f / (sqrtf(sum) + eps);
    // inv = 0 (the sum overflowed) or NaN: straight through, X = G * inv
    const bool fine = inv > 0.f && inv < INFINITY;
    const int e = fine ? min(120, max(-120, ilogbf(inv * kX))) : 0;
    sh[0] = fine ? ldexpf(1.f, e) : inv;
    sh[1] = fine ? inv * ldexpf(1.f, -e) : 1.f;
    if (blockIdx.x == 0) s0[z] = sh[1];
  }
  __syncthreads();
  const float f = sh[0];
  const T* src = static_cast<const T*>(g.p[z]);
  __half* h = hi + z * zs;
  bf16* l = lo ? lo + z * zs : nullptr;
  if (cols % 8 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0) {  // ld == cols: one run of 8-element chunks
    const int64_t n8 = (int64_t)rows * cols / 8;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n8; i += (int64_t)gridDim.x * 256) {
      float v[8];
      if (sizeof(T) == 2) {
        unpack8(reinterpret_cast<const uint4*>(src)[i], v);
      } else {
        const float4 x = reinterpret_cast<const float4*>(src)[2 * i], y = reinterpret_cast<const float4*>(src)[2 * i + 1];
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
      }
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] *= f;
      const uint4 u = make_uint4(pack_half(v[0], v[1]), pack_half(v[2], v[3]), pack_half(v[4], v[5]), pack_half(v[6], v[7]));
      reinterpret_cast<uint4*>(h)[i] = u;
      if (l) {
        const __half2* k = reinterpret_cast<const __half2*>(&u);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const float2 y = __half22float2(k[q]);
          v[2 * q] -= y.x;
          v[2 * q + 1] -= y.y;
        }
        reinterpret_cast<uint4*>(l)[i] =
            make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
      }
    }
    return;
  }
  for (int row = blockIdx.x; row < rows; row += gridDim.x) {
    const T* r = src + (int64_t)row * cols;
    for (int c = threadIdx.x; c < cols; c += 256) {
      const float v = to_f<T>(r[c]) * f;
      const __half q = __float2half_rn(v);
      h[row * ld + c] = q;
      if (l) l[row * ld + c] = __float2bfloat16_rn(v - __half2float(q));
    }
  }
}

// ---- small matrices ---------------------------------------------------------
// Short side q <= 64: the whole iteration in one launch. A cluster of CL CTAs
// holds one matrix, each CTA a slice of its long side in shared memory; per
// step each CTA forms its slice's part of S, the parts are summed over the
// cluster's shared memory (fixed order, every CTA a share of the elements
// handed to all), every CTA forms B for itself and updates its slice. What
// bounds it is the length of that chain (two cluster barriers a step), not
// bytes or flops: a few 10 MFLOP, so the products run on mma.sync from
// shared memory, which needs no descriptors, TMEM or copies in between.
//
// X, S and B are fp16 pairs hi + lo (22 bits), scaled by 2^8, and each product
// sums hi hi + hi lo + lo hi in fp32: the result is exact to about 1e-6
// before its rounding. Rows are padded by 16 bytes, an odd number of 16-byte
// slots, so ldmatrix meets all banks.
constexpr int kSmallQ = 64, kSmallT = 512, kSmallW = kSmallT / 32;
constexpr float kSm = 256.f;

struct SmallShape {
  int q, L, w, wp, qp, fp;  // padded short side, slice, row strides of X, of S / B (halves) and of the parts (floats)
  int mt, units, groups;
  __host__ __device__ SmallShape(int q_, int L_, int CL) {
    q = cdiv(q_, 16) * 16;
    L = L_;
    w = cdiv(cdiv(L, CL), 16) * 16;
    wp = w + 8;
    qp = q + 8;
    fp = q + 4;
    mt = q / 16;
    units = mt * mt;           // 16 x 16 blocks of S: at most a warp's each
    groups = kSmallW / units;  // ranges of K side by side
  }
  // X hi, lo; S (then B) hi, lo; parts of S
  __host__ __device__ int bytes() const { return 2 * (2 * q * wp + 2 * q * qp) + 4 * groups * q * fp; }
};

__device__ __forceinline__ void ldm4(uint32_t (&r)[4], const __half* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(smem_u32(p))
               : "memory");
}
__device__ __forceinline__ void ldm2t(uint32_t (&r)[2], const __half* p) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x2.trans.shared.b16 {%0, %1}, [%2];"
               : "=r"(r[0]), "=r"(r[1])
               : "r"(smem_u32(p))
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void split2(float v, __half& h, __half& l) {
  h = __float2half_rn(v);
  l = __float2half_rn(v - __half2float(h));
}
__device__ __forceinline__ void split2x2(float a, float b, __half2& h, __half2& l) {
  h = __floats2half2_rn(a, b);
  const float2 f = __half22float2(h);
  l = __floats2half2_rn(a - f.x, b - f.y);
}

// A 16 x 16 block of a symmetric product Y Y^T, Y = hi + lo [.., ld] halves:
// rows 16 m.., columns 16 n.., K steps of 16 from k0 by dk
__device__ __forceinline__ void small_product(const __half* hi, const __half* lo, int ld, int m, int n, int k0, int k1,
                                              int dk, float (&acc)[2][4]) {
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int t = 0; t < 2; ++t)
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[t][i] = 0.f;
  // A: lane -> row lane % 16, K half lane / 16; B (both column tiles of 8 in a
  // load): lane -> row lane % 8 of tile lane / 16, K half (lane / 8) % 2
  const int ao = (16 * m + lane % 16) * ld + lane / 16 * 8;
  const int bo = (16 * n + lane / 16 * 8 + lane % 8) * ld + lane / 8 % 2 * 8;
#pragma unroll 4
  for (int k = k0; k < k1; k += dk) {
    uint32_t ah[4], al[4], bh[4], bl[4];
    ldm4(ah, hi + ao + k);
    ldm4(al, lo + ao + k);
    ldm4(bh, hi + bo + k);
    ldm4(bl, lo + bo + k);
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      mma16816(acc[j], al, bh[2 * j], bh[2 * j + 1]);
      mma16816(acc[j], ah, bl[2 * j], bl[2 * j + 1]);
      mma16816(acc[j], ah, bh[2 * j], bh[2 * j + 1]);
    }
  }
}

// the slice's elements of the matrix in memory order of the slice, 8 at a
// time where aligned: f(i, j, value) with i along the short side
template <typename T, typename F>
__device__ __forceinline__ void small_read(const T* src, bool tall, int q, int L, int j0, int jn, F f) {
  // wide: q runs of jn; tall: one run of jn q
  const int runs = tall ? 1 : q, len = tall ? jn * q : jn;
  const int64_t start = tall ? (int64_t)j0 * q : j0, step = tall ? 0 : L;
  const bool vec = len % 8 == 0 && start % 8 == 0 && step % 8 == 0 && (reinterpret_cast<uintptr_t>(src) & 15) == 0;
  if (vec) {
    const int per = len / 8, n = runs * per;
#pragma unroll 4
    for (int e = threadIdx.x; e < n; e += kSmallT) {
      const int r = e / per, c = (e - r * per) * 8;
      const T* p = src + start + r * step + c;
      float v[8];
      if (sizeof(T) == 2) {
        unpack8(*reinterpret_cast<const uint4*>(p), v);
      } else {
        const float4 x = reinterpret_cast<const float4*>(p)[0], y = reinterpret_cast<const float4*>(p)[1];
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
        v[4] = y.x; v[5] = y.y; v[6] = y.z; v[7] = y.w;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (tall) {
          const int j = (c + k) / q;
          f(c + k - j * q, j, v[k]);
        } else {
          f(r, c + k, v[k]);
        }
      }
    }
    return;
  }
  const int n = runs * len;
#pragma unroll 4
  for (int e = threadIdx.x; e < n; e += kSmallT) {
    const int r = e / max(len, 1), c = e - r * len;
    const float v = to_f<T>(src[start + r * step + c]);
    if (tall) {
      const int j = c / q;
      f(c - j * q, j, v);
    } else {
      f(r, c, v);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kSmallT) orth_small(const __grid_constant__ Ptrs g, int rows, int cols, int steps,
                                                      float ca, float cb, float cc, float eps, bf16* out) {
  namespace cg = cooperative_groups;
  cg::cluster_group cluster = cg::this_cluster();
  const int CL = cluster.num_blocks(), rank = cluster.block_rank();
  const int z = blockIdx.x / CL;
  const bool tall = rows > cols;
  const int q = tall ? cols : rows, L = tall ? rows : cols;
  const SmallShape h(q, L, CL);
  extern __shared__ uint4 orth_smem[];
  __half* xh = reinterpret_cast<__half*>(orth_smem);
  __half* xl = xh + h.q * h.wp;
  __half* sh = xl + h.q * h.wp;
  __half* sl = sh + h.q * h.qp;
  float* P = reinterpret_cast<float*>(sl + h.q * h.qp);
  __shared__ float red[kSmallW], total;
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  const int j0 = rank * h.w, jn = max(0, min(h.w, L - j0));
  const T* src = static_cast<const T*>(g.p[z]);

  pdl_next();
  pdl_wait();
  float s = 0.f;
  small_read(src, tall, q, L, j0, jn, [&](int, int, float v) { s = fmaf(v, v, s); });
  s = warp_sum(s);
  if (lane == 0) red[warp] = s;
  for (int i = tid; i < 2 * h.q * h.wp / 8; i += kSmallT) orth_smem[i] = make_uint4(0, 0, 0, 0);
  __syncthreads();
  if (tid == 0) {
    float r = 0.f;
    for (int i = 0; i < kSmallW; ++i) r += red[i];
    total = r;
  }
  cluster.sync();
  float sum = 0.f;
  for (int r = 0; r < CL; ++r) sum += *cluster.map_shared_rank(&total, r);
  const float inv = 1.f / (sqrtf(sum) + eps);
  small_read(src, tall, q, L, j0, jn,
             [&](int i, int j, float v) { split2(v * inv * kSm, xh[i * h.wp + j], xl[i * h.wp + j]); });
  __syncthreads();

  const int fr = lane / 4, fc = lane % 4 * 2;  // an accumulator's first row and column
  for (int step = 0; step < steps; ++step) {
    // this slice's part of S, the K ranges' one after another in P
    const int gr = warp / h.units, u = warp - gr * h.units, um = u / h.mt, un = u - um * h.mt;
    float acc[2][4];
    if (gr < h.groups) {
      small_product(xh, xl, h.wp, um, un, 16 * gr, h.w, 16 * h.groups, acc);
      float* dst = P + gr * h.q * h.fp + (16 * um + fr) * h.fp + 16 * un + fc;
#pragma unroll
      for (int t = 0; t < 2; ++t) {
        *reinterpret_cast<float2*>(dst + 8 * t) = make_float2(acc[t][0], acc[t][1]);
        *reinterpret_cast<float2*>(dst + 8 * h.fp + 8 * t) = make_float2(acc[t][2], acc[t][3]);
      }
    }
    if (h.groups > 1) {
      __syncthreads();
      for (int e = tid; e < h.q * h.q; e += kSmallT) {
        const int at = e / h.q * h.fp + e % h.q;
        float v = P[at];
        for (int r = 1; r < h.groups; ++r) v += P[r * h.q * h.fp + at];
        P[at] = v;
      }
    }
    cluster.sync();
    // every CTA sums its share of the quads over the cluster, up to 8 threads
    // a quad, and gives the result to all: the next step's parts are written
    // after the second barrier, the next S after that step's first one
    const int tq = min(CL, 8), per = h.q * h.q / 4 / CL;
    for (int e0 = 32 * warp; e0 < per * tq; e0 += kSmallT) {
      const int e = e0 + lane, sub = e % tq, quad = min(rank * per + e / tq, h.q * h.q / 4 - 1);
      const int i = quad / (h.q / 4), j = (quad - i * (h.q / 4)) * 4;
      float4 t = *reinterpret_cast<const float4*>(cluster.map_shared_rank(P, sub) + i * h.fp + j);
      if (CL > 8) {
        const float4 v = *reinterpret_cast<const float4*>(cluster.map_shared_rank(P, sub + 8) + i * h.fp + j);
        t = make_float4(t.x + v.x, t.y + v.y, t.z + v.z, t.w + v.w);
      }
      for (int o = 1; o < tq; o *= 2) {  // a + b = b + a: every thread gets the same bits
        t.x += __shfl_xor_sync(0xffffffffu, t.x, o);
        t.y += __shfl_xor_sync(0xffffffffu, t.y, o);
        t.z += __shfl_xor_sync(0xffffffffu, t.z, o);
        t.w += __shfl_xor_sync(0xffffffffu, t.w, o);
      }
      if (e >= per * tq) continue;
      // products of 2^8 X: S 2^16 -> S 2^8
      __half2 hi[2], lo[2];
      split2x2(t.x / kSm, t.y / kSm, hi[0], lo[0]);
      split2x2(t.z / kSm, t.w / kSm, hi[1], lo[1]);
      const int at = i * h.qp + j;
      for (int r = sub; r < CL; r += 8) {
        *reinterpret_cast<uint2*>(cluster.map_shared_rank(sh, r) + at) = *reinterpret_cast<const uint2*>(hi);
        *reinterpret_cast<uint2*>(cluster.map_shared_rank(sl, r) + at) = *reinterpret_cast<const uint2*>(lo);
      }
    }
    cluster.sync();
    // B = b S + c S^2 over S, once every warp has read what it needs
    if (warp < h.units) small_product(sh, sl, h.qp, um, un, 0, h.q, 16, acc);
    __syncthreads();
    if (warp < h.units) {
      const int at = (16 * um + fr) * h.qp + 16 * un + fc;
#pragma unroll
      for (int t = 0; t < 2; ++t)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          __half2* ph = reinterpret_cast<__half2*>(sh + at + 8 * t + 8 * k * h.qp);
          __half2* pl = reinterpret_cast<__half2*>(sl + at + 8 * t + 8 * k * h.qp);
          const float2 x = __half22float2(*ph), y = __half22float2(*pl);
          split2x2(fmaf(cb, x.x + y.x, cc / kSm * acc[t][2 * k]), fmaf(cb, x.y + y.y, cc / kSm * acc[t][2 * k + 1]), *ph,
                   *pl);
        }
    }
    __syncthreads();
    // X = a X + B X: a warp owns column tiles of 8 (it reads no others, so it
    // overwrites them in place) and holds all their row tiles' sums
    for (int c0 = 8 * warp; c0 < h.w; c0 += 8 * kSmallW) {
      float d[4][4];
#pragma unroll
      for (int m = 0; m < 4; ++m)
#pragma unroll
        for (int i = 0; i < 4; ++i) d[m][i] = 0.f;
#pragma unroll
      for (int k = 0; k < kSmallQ; k += 16) {
        if (k >= h.q) break;
        uint32_t bh[2], bl[2];
        ldm2t(bh, xh + (k + lane % 16) * h.wp + c0);
        ldm2t(bl, xl + (k + lane % 16) * h.wp + c0);
#pragma unroll
        for (int m = 0; m < 4; ++m) {
          if (m >= h.mt) break;
          uint32_t ah[4], al[4];
          const int ao = (16 * m + lane % 16) * h.qp + lane / 16 * 8 + k;
          ldm4(ah, sh + ao);
          ldm4(al, sl + ao);
          mma16816(d[m], al, bh[0], bh[1]);
          mma16816(d[m], ah, bl[0], bl[1]);
          mma16816(d[m], ah, bh[0], bh[1]);
        }
      }
      __syncwarp();
#pragma unroll
      for (int m = 0; m < 4; ++m) {
        if (m >= h.mt) break;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
          const int at = (16 * m + fr + 8 * k) * h.wp + c0 + fc;
          __half2* ph = reinterpret_cast<__half2*>(xh + at);
          __half2* pl = reinterpret_cast<__half2*>(xl + at);
          const float2 x = __half22float2(*ph), y = __half22float2(*pl);
          split2x2(fmaf(ca, x.x + y.x, d[m][2 * k] / kSm), fmaf(ca, x.y + y.y, d[m][2 * k + 1] / kSm), *ph, *pl);
        }
      }
      __syncwarp();
    }
    __syncthreads();
  }
  bf16* dst = out + (int64_t)z * rows * cols;
  auto value = [&](int i, int j) {
    return __float2bfloat16_rn((__half2float(xh[i * h.wp + j]) + __half2float(xl[i * h.wp + j])) / kSm);
  };
  if (tall) {
#pragma unroll 4
    for (int e = tid; e < jn * q; e += kSmallT) {
      const int j = e / q;
      dst[(int64_t)j0 * q + e] = value(e - j * q, j);
    }
  } else {
#pragma unroll 4
    for (int e = tid; e < jn * q; e += kSmallT) {
      const int i = e / jn, j = e - i * jn;
      dst[(int64_t)i * cols + j0 + j] = value(i, j);
    }
  }
  cluster.sync();  // the others have read this CTA's parts
}

template <typename T>
cudaError_t small_attributes(int smem, int cl) {
  cudaError_t e = set_smem_once(orth_small<T>, smem);
  if (e == cudaSuccess && cl > 8) e = cudaFuncSetAttribute(orth_small<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  return e;
}

// Whether the current device can hold a cluster of cl CTAs with that much
// shared memory (a partition of a GPU may not). Asked once per device and form.
template <typename T>
bool cluster_fits(int cl, int smem) {
  static std::mutex mu;
  static std::map<std::array<int, 3>, bool> known;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  const std::array<int, 3> key{dev, cl, smem};
  std::lock_guard<std::mutex> lock(mu);
  const auto it = known.find(key);
  if (it != known.end()) return it->second;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(cl);
  cfg.blockDim = dim3(kSmallT);
  cfg.dynamicSmemBytes = smem;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim = {(unsigned)cl, 1, 1};
  cfg.attrs = &at;
  cfg.numAttrs = 1;
  int n = 0;
  if (small_attributes<T>(smem, cl) != cudaSuccess || cudaOccupancyMaxActiveClusters(&n, orth_small<T>, &cfg) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  return known[key] = n > 0;
}

// CTAs per matrix of the one-launch form (more than 8 need an opt-in), 0 where
// it does not apply: as many as give slices of 128 columns, one column tile per
// warp, or the most that fit the device, 16 at most, with wider slices.
int small_cluster(const llattn_orth_args& a) {
  const int q = std::min(a.rows, a.cols), L = std::max(a.rows, a.cols);
  if (q > kSmallQ) return 0;
  int cl = 1;
  while (cl < 16 && L > 128 * cl) cl *= 2;
  for (; cl >= 1; cl /= 2) {
    const int smem = SmallShape(q, L, cl).bytes();
    if (smem > 220 * 1024) return 0;
    if (a.dtype == LLATTN_F32 ? cluster_fits<float>(cl, smem) : cluster_fits<bf16>(cl, smem)) return cl;
  }
  return 0;
}

template <typename T>
cudaError_t run_small(const llattn_orth_args& a, int cl, cudaStream_t st) {
  const int smem = SmallShape(std::min(a.rows, a.cols), std::max(a.rows, a.cols), cl).bytes();
  cudaError_t e = small_attributes<T>(smem, cl);
  if (e != cudaSuccess) return e;
  for (int i0 = 0; i0 < a.count; i0 += kPtrs) {
    const int cnt = std::min(kPtrs, a.count - i0);
    Ptrs g;
    for (int i = 0; i < cnt; ++i) g.p[i] = a.g[i0 + i];
    e = launch_pdl(orth_small<T>, dim3((unsigned)(cnt * cl)), kSmallT, smem, cl, st, g, (int)a.rows, (int)a.cols, (int)a.steps,
                   a.a, a.b, a.c, a.eps, static_cast<bf16*>(a.out) + (int64_t)i0 * a.rows * a.cols);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

// ---- host side ------------------------------------------------------------------

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
int64_t up8(int64_t v) { return (v + 7) & ~(int64_t)7; }

struct Plan {
  bool tall;
  int q, slice, n_slices;  // short side; matrices in flight
  int64_t ldx, xz, ldb, bz;
  size_t x0, x1, lo, s, b, part, s0, total;
};

Plan make_plan(const llattn_orth_args& a) {
  Plan p;
  p.tall = a.rows > a.cols;
  p.q = std::min(a.rows, a.cols);
  p.ldx = up8(a.cols);
  p.xz = p.ldx * a.rows;
  p.ldb = up8(p.q);
  p.bz = p.ldb * p.q;
  // a GiB of X, its remainder, S and B at a time (at least one matrix)
  const int64_t each = 6 * p.xz + 4 * p.bz;
  p.slice = (int)std::max<int64_t>(1, std::min<int64_t>(std::min(a.count, kPtrs), ((int64_t)1 << 30) / each));
  p.n_slices = cdiv(a.count, p.slice);
  p.slice = cdiv(a.count, p.n_slices);
  size_t off = 0;
  auto take = [&](size_t b) { size_t o = off; off += up256(b); return o; };
  p.x0 = take(2 * (size_t)p.slice * p.xz);
  p.x1 = take(2 * (size_t)p.slice * p.xz);
  p.lo = take(2 * (size_t)p.slice * p.xz);
  p.s = take(2 * (size_t)p.slice * p.bz);
  p.b = take(2 * (size_t)p.slice * p.bz);
  p.part = take(sizeof(float) * (size_t)p.slice * kParts);
  p.s0 = take(sizeof(float) * p.slice);
  p.total = off;
  return p;
}

#define TRY(x)                        \
  do {                                \
    cudaError_t e_ = (x);             \
    if (e_ != cudaSuccess) return e_; \
  } while (0)

template <typename T>
cudaError_t run(const llattn_orth_args& a, const Plan& p, volatile unsigned* fault, cudaStream_t st) {
  char* ws = static_cast<char*>(a.workspace);
  __half* x[2] = {reinterpret_cast<__half*>(ws + p.x0), reinterpret_cast<__half*>(ws + p.x1)};
  bf16* lo = reinterpret_cast<bf16*>(ws + p.lo);
  __half* S = reinterpret_cast<__half*>(ws + p.s);
  __half* B = reinterpret_cast<__half*>(ws + p.b);
  float* part = reinterpret_cast<float*>(ws + p.part);
  float* s0 = reinterpret_cast<float*>(ws + p.s0);
  const int m = a.rows, n = a.cols;
  for (int i0 = 0; i0 < a.count; i0 += p.slice) {
    const int cnt = std::min(p.slice, a.count - i0);
    Ptrs g;
    for (int i = 0; i < cnt; ++i) g.p[i] = a.g[i0 + i];
    const int n_parts = (int)std::max<int64_t>(1, std::min<int64_t>(kParts, (int64_t)m * n / 4096));
    TRY(launch_pdl(orth_square<T>, dim3(n_parts, cnt), 256, 0, 1, st, g, (int64_t)m * n, part));
    // steps before the folded ones read X as hi + lo
    const int comp0 = a.steps - kFolded;
    bf16* lo0 = sizeof(T) == 4 && comp0 > 0 ? lo : nullptr;
    TRY(launch_pdl(orth_convert<T>, dim3((unsigned)std::min<int64_t>(((int64_t)m * n + 2047) / 2048, cdiv(8 * sm_count(), cnt)), cnt), 256, 0, 1, st, g, m, n, part, n_parts, a.eps, x[0], lo0,
                                                                            p.ldx, p.xz, s0));
    for (int i = 0; i < a.steps; ++i) {
      const float* sc = i ? nullptr : s0;
      const bool folded = i >= comp0;
      const bool last = i + 1 == a.steps;
      const __half* X = x[i & 1];
      MmArgs ma = {};
      ma.fp16 = 1;
      ma.nz = cnt;
      ma.fault_host = fault;
      const Operand ok{X, m, n, p.ldx, cnt, p.xz, 0}, on{X, m, n, p.ldx, cnt, p.xz, 1};
      MmArgs gm = ma;
      gm.M = gm.N = p.q;
      gm.K = p.tall ? m : n;
      gm.sym = 1;
      gm.chain = cdiv(gm.K, 64) > kLong ? kGramChain : 0;
      const Operand& og = p.tall ? on : ok;
      TRY(launch_mm(gm, og, og, EpiGram{S, p.ldb, p.bz, sc}, st));
      gm.K = p.q;
      gm.chain = 0;
      const Operand os{S, p.q, p.q, p.ldb, cnt, p.bz, 0}, ob{B, p.q, p.q, p.ldb, cnt, p.bz, 0};
      TRY(launch_mm(gm, os, os, EpiPoly{S, B, p.ldb, p.bz, a.b, a.c / kS, folded ? a.a * kS : 0.f}, st));
      MmArgs um = ma;
      um.M = m;
      um.N = n;
      um.K = p.q;
      EpiUpdate eu{};
      eu.hi = X;
      eu.lo = lo;
      eu.next = x[(i + 1) & 1];
      eu.out = last ? static_cast<bf16*>(a.out) + (int64_t)i0 * m * n : nullptr;
      eu.ld = p.ldx;
      eu.zs = p.xz;
      eu.ldo = n;
      eu.zso = (int64_t)m * n;
      eu.s0 = sc;
      eu.ca = a.a;
      eu.rd_hi = !folded;
      eu.rd_lo = !folded && (i > 0 || lo0);
      eu.wr_lo = i + 1 < comp0;
      eu.vec_out = n % 8 == 0 && ((uintptr_t)a.out & 15) == 0;
      TRY(p.tall ? launch_mm(um, ok, ob, eu, st) : launch_mm(um, ob, on, eu, st));
    }
  }
  return cudaSuccess;
}

}  // namespace

size_t workspace_bytes(const llattn_orth_args& a) { return small_cluster(a) ? 256 : make_plan(a).total; }

int launches(const llattn_orth_args& a) {
  return small_cluster(a) ? cdiv(a.count, kPtrs) : make_plan(a).n_slices * (2 + 3 * a.steps);
}

cudaError_t launch(const llattn_orth_args& a, volatile unsigned* fault, cudaStream_t s) {
  if (const int cl = small_cluster(a)) return a.dtype == LLATTN_F32 ? run_small<float>(a, cl, s) : run_small<bf16>(a, cl, s);
  const Plan p = make_plan(a);
  return a.dtype == LLATTN_F32 ? run<float>(a, p, fault, s) : run<bf16>(a, p, fault, s);
}

unsigned read_fault_word(bool reset) { return read_fault(reset); }

}  // namespace orth
}  // namespace llattn
