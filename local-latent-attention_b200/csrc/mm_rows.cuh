// What the training operators put around mm_kernel: operands packed into aligned
// rows and bf16 planes, the epilogue that writes rows out, and host helpers
// (included by xent.cu and gated.cu).
#pragma once

#include <algorithm>

#include "mm_sm100.cuh"

namespace llattn {
namespace mm {
namespace {

// fp32's plane products, smallest first: (0,2) (2,0) (1,1) (0,1) (1,0) (0,0)
constexpr uint32_t kTermsA = 0x010120u, kTermsB = 0x001102u;

// ---- packing ------------------------------------------------------------------

// whether rows can be read in 16-byte chunks (and need no padding columns)
template <typename T>
__device__ __forceinline__ bool vec_rows(const T* p, int64_t ld, int d) {
  return ld % 8 == 0 && d % 8 == 0 && (reinterpret_cast<uintptr_t>(p) & 15) == 0;
}

// fp32 pair -> three bf16 planes, whose sum is the value to 2^-24
__device__ __forceinline__ void split3(float a, float b, uint32_t (&o)[3]) {
#pragma unroll
  for (int k = 0; k < 3; ++k) {
    o[k] = pack_bf16(a, b);
    a -= __uint_as_float(o[k] << 16);
    b -= __uint_as_float(o[k] & 0xffff0000u);
  }
}

// A warp's row: dst = src (bf16, or three planes of fp32), zeros from column d
// to lds, or everywhere where src is null.
template <typename T>
__device__ __forceinline__ void pack_row(const T* src, int d, bf16* dst, int64_t lds, int64_t plane, bool vec) {
  const int lane = threadIdx.x % 32;
  if (sizeof(T) == 2 && (vec || !src)) {  // d a multiple of 8, 16-byte aligned rows
#pragma unroll 8
    for (int c = lane; c < lds / 8; c += 32)
      reinterpret_cast<uint4*>(dst)[c] = src ? reinterpret_cast<const uint4*>(src)[c] : make_uint4(0, 0, 0, 0);
    return;
  }
  if (sizeof(T) == 4 && vec && src) {  // lds == d
#pragma unroll 8
    for (int c = lane; c < d / 4; c += 32) {
      const float4 v = reinterpret_cast<const float4*>(src)[c];
      uint32_t a[3], b[3];
      split3(v.x, v.y, a);
      split3(v.z, v.w, b);
#pragma unroll
      for (int k = 0; k < 3; ++k) reinterpret_cast<uint2*>(dst + k * plane)[c] = make_uint2(a[k], b[k]);
    }
    return;
  }
#pragma unroll 4
  for (int c = lane; c < lds; c += 32) {
    const float v = src && c < d ? to_f<T>(src[c]) : 0.f;
    if (sizeof(T) == 2) {
      dst[c] = __float2bfloat16_rn(v);
    } else {
      uint32_t o[3];
      split3(v, 0.f, o);
#pragma unroll
      for (int k = 0; k < 3; ++k) reinterpret_cast<uint16_t*>(dst)[k * plane + c] = (uint16_t)o[k];
    }
  }
}

// Rows of up to 5 matrices, packed in one launch: a thread for 8 columns, whole 16-byte
// chunks out. (A warp a row, lane by lane, took 51 us for 1408 unaligned rows of 3749, this 6.)
struct Packed {
  const void* x;
  int64_t ldx;
  bf16* xs;
  int64_t lds;
  int n, d;
  unsigned block;  // its first
};
struct Packs {
  int count;
  unsigned blocks;
  Packed m[5];
  // rows of cols from src to dst, planes `rows` apart
  void add(const void* src, int64_t ld, int rows, int cols, void* dst, int64_t lds) {
    m[count++] = {src, ld, static_cast<bf16*>(dst), lds, rows, cols, blocks};
    blocks += (unsigned)((rows * (lds / 8) + 255) / 256);
  }
};
template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const __grid_constant__ Packs p) {
  pdl_next();
  pdl_wait();
  int k = 0;
  while (k + 1 < p.count && blockIdx.x >= p.m[k + 1].block) ++k;
  const T* x = static_cast<const T*>(p.m[k].x);
  const int64_t ldx = p.m[k].ldx, lds = p.m[k].lds, plane = p.m[k].n * lds;
  bf16* xs = p.m[k].xs;
  const int n = p.m[k].n, d = p.m[k].d;
  const int64_t i = (int64_t)(blockIdx.x - p.m[k].block) * 256 + threadIdx.x, per = lds / 8, total = n * per;
  if (i >= total) return;
  const int64_t r = total <= INT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)per) : i / per;
  const int c = (int)(i - r * per) * 8;
  const T* src = x + r * ldx + c;
  bf16* dst = xs + r * lds + c;
  if constexpr (sizeof(T) == 2) {
    uint4 u;
    if (vec_rows(x, ldx, d)) {
      u = *reinterpret_cast<const uint4*>(src);
    } else {
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int q = 0; q < 8; ++q) e[q] = c + q < d ? src[q] : from_f<T>(0.f);
    }
    *reinterpret_cast<uint4*>(dst) = u;
  } else {
    float v[8];
    if (vec_rows(x, ldx, d)) {
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const float4 f = reinterpret_cast<const float4*>(src)[q];
        v[4 * q] = f.x;
        v[4 * q + 1] = f.y;
        v[4 * q + 2] = f.z;
        v[4 * q + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int q = 0; q < 8; ++q) v[q] = c + q < d ? src[q] : 0.f;
    }
    uint32_t o[4][3];
#pragma unroll
    for (int q = 0; q < 4; ++q) split3(v[2 * q], v[2 * q + 1], o[q]);
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(dst + k * plane) = make_uint4(o[0][k], o[1][k], o[2][k], o[3][k]);
  }
}

template <typename T>
cudaError_t launch_packs(const Packs& p, cudaStream_t s) {
  return p.count ? launch_pdl(pack_kernel<T>, dim3(p.blocks), 256, 0, 1, s, p) : cudaSuccess;
}
template <typename T>
cudaError_t launch_pack(const void* src, int64_t ld, int rows, int cols, void* dst, int64_t lds, cudaStream_t s) {
  Packs p = {};
  p.add(src, ld, rows, cols, dst, lds);
  return launch_packs<T>(p, s);
}

// ---- rows out -----------------------------------------------------------------

struct EpiOut {
  static constexpr bool kNarrow = true, kWide = true, kChain = true, kBegin = true;
  struct Pre {};
  __device__ __forceinline__ void fetch(Pre&, const MmArgs&, MmTile, int, int, int) const {}
  void* out;
  int64_t ldo;
  int out_bf16;
  int vec;              // base and row stride 16-byte aligned (whole rows may be padded to 16 bytes)
  int add;              // fp32, vec: added to what out holds (one writer per element and launch: in order)
  const float* acc;     // added first (fp32, row stride ldacc), or null
  int64_t ldacc;
  const int* idx;       // output row of row m, or null
  const int* count;     // the result is divided by max(1, *count), or null
  const float* factor;  // and multiplied by *factor, or null
  const int64_t* zero;  // rows of out whose target, of zero_n, is `ignore` become zeros; or null
  int zero_n;
  int64_t ignore;

  __device__ __forceinline__ float scale() const {
    return (count ? 1.f / (float)max(1, *count) : 1.f) * (factor ? *factor : 1.f);
  }
  __device__ __forceinline__ void begin(int warp, int warps) const {
    if (!zero) return;
    for (int64_t r = warp; r < zero_n; r += warps) {
      if (zero[r] != ignore) continue;
      for (int64_t c = r * ldo + threadIdx.x % 32; c < (r + 1) * ldo; c += 32) {
        if (out_bf16)
          static_cast<bf16*>(out)[c] = __float2bfloat16_rn(0.f);
        else
          static_cast<float*>(out)[c] = 0.f;
      }
    }
  }

  // 4 columns of a row of a split tile, joined
  __device__ __forceinline__ void quad(int row, int col, int n, float4 v) const {
    if (acc) {
      const float4 c = *reinterpret_cast<const float4*>(acc + (int64_t)row * ldacc + col);
      v = make_float4(v.x + c.x, v.y + c.y, v.z + c.z, v.w + c.w);
    }
    const float f = scale();
    v = make_float4(v.x * f, v.y * f, v.z * f, v.w * f);
    const int64_t at = (int64_t)(idx ? idx[row] : row) * ldo + col;
    const float x[4] = {v.x, v.y, v.z, v.w};
    if (out_bf16) {
      bf16* dst = static_cast<bf16*>(out) + at;
      if (vec) {
        *reinterpret_cast<uint2*>(dst) = make_uint2(pack_bf16(v.x, v.y), pack_bf16(v.z, v.w));
      } else {
        for (int q = 0; q < n; ++q) dst[q] = __float2bfloat16_rn(x[q]);
      }
    } else {
      float* dst = static_cast<float*>(out) + at;
      if (vec) {
        if (add) {
          const float4 c = *reinterpret_cast<const float4*>(dst);
          v = make_float4(v.x + c.x, v.y + c.y, v.z + c.z, v.w + c.w);
        }
        *reinterpret_cast<float4*>(dst) = v;
      } else {
        for (int q = 0; q < n; ++q) dst[q] = x[q];
      }
    }
  }

  template <int CW>
  __device__ __forceinline__ void tile(const MmArgs& a, MmTile w, int row, int col0, int M, uint32_t taddr,
                                       bool zero, uint8_t* buf, Pre&) const {
    const int lane = threadIdx.x % 32, row0 = row - lane, rows = M - row0;
    const int64_t at = row < M ? (idx ? (int64_t)idx[row] : row) * ldo + col0 : -1;
    const float f = scale();
    const MappedRows dst{at < 0 ? nullptr : static_cast<uint8_t*>(out) + at * (out_bf16 ? 2 : 4)};
    if (CW == 128 && out_bf16 && vec && !acc) {  // 64 columns, whole 128-byte lines, at a time
#pragma unroll 1
      for (int cc = 0; cc < CW; cc += 64) {
        const int n = a.N - col0 - cc;
        if (n <= 0) break;
        uint4 u[8];
        row64_bf16(taddr + cc, zero, f, u);
        block_store(buf, lane, u, dst.at(cc * 2), n * 2);
      }
      return;
    }
    // what was summed before is fetched one block ahead: its latency passes
    // during the previous block's stores
    const Rows src{acc + (int64_t)row0 * ldacc + col0, ldacc * 4, rows};  // ldacc is a multiple of 8
    uint4 x[8];
    if (acc && col0 < a.N) block_fetch(lane, x, src, (a.N - col0) * 4);
#pragma unroll 1
    for (int cc = 0; cc < CW; cc += 32) {
      const int n = a.N - col0 - cc;
      if (n <= 0) break;  // warp-uniform
      float v[32];
      load32(taddr + cc, zero, v);
      if (acc) {
        block_spread(buf, lane, x);
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] += __uint_as_float(word(x, q));
        if (cc + 32 < CW && n > 32) block_fetch(lane, x, src.at((cc + 32) * 4), (n - 32) * 4);
      }
#pragma unroll
      for (int q = 0; q < 32; ++q) v[q] *= f;
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
        if (add)
          block_store<true>(buf, lane, u, dst.at(cc * 4), n * 4);
        else if (vec)
          block_store(buf, lane, u, dst.at(cc * 4), n * 4);
        else
          block_store_odd<float>(buf, lane, u, dst.at(cc * 4), n);
      }
    }
  }
};

// ---- host side ------------------------------------------------------------------

inline size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
inline int64_t up8(int64_t v) { return (v + 7) & ~(int64_t)7; }

inline bool aligned_rows(const void* p, int64_t ld, int64_t rows, int elt) {
  return ((uintptr_t)p & 15) == 0 && (rows == 1 || ld % (16 / elt) == 0);
}

#define TRY(x)                          \
  do {                                  \
    cudaError_t e_ = (x);               \
    if (e_ != cudaSuccess) return e_;   \
  } while (0)

}  // namespace
}  // namespace mm
}  // namespace llattn
