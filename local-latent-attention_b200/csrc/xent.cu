// Softmax cross-entropy of an output projection without its [tokens,
// vocabulary] logits, and its gradients:
//   l[n, v] = x[n] . w[v],  loss[n] = log sum_v exp(l[n, v]) - l[n, t(n)]
//   G[n, v] = g(n) (exp(l[n, v]) / sum_v' exp(l[n, v']) - [v == t(n)])
//   dx = G w,  dw = G^T x
// (the head and loss of models.py:505-518 and train.py's F.cross_entropy;
// the reference materialises the fp32 logits).
//
// All three products run on mm_kernel (mm_sm100.cuh). The logits never leave
// the chip: the first product's epilogue turns each row's 128-column tile
// into exponentials against the tile's own maximum m, keeps (m, sum) per
// (row, tile), and, when gradients are wanted, stores the exponentials of a
// bounded piece of the tokens as fp16 scaled by 2^15: relative to the tile's
// maximum every stored value above 2^-29 keeps 11 bits, and one above 2^-32
// bf16's 8 (none below 2^-40: such a word of such a token gets no gradient), so
// the later normalisation is the only 8-bit rounding G goes through. xent_rows then
// joins the tiles' (m, sum) to the row's logsumexp and rewrites the
// piece in place as bf16 G, which the other two products read. One pass over
// the exponentials (4 bytes per element) replaces a second 2 N V d product.
// The mean's 1 / count stays out of G (a common factor rounded to 8 bits would
// be a common error of all rows, and p - 1 would not be exact near -1); the
// gradients' epilogues apply it in fp32.
//
// Gradients run over the tokens that count only: xent_prep lists them (in
// order), the sizes of the products follow the device-side count, and rows
// of ignored tokens are never read, so their values cannot reach dw.
//
// fp32: x, w and G are split into three bf16 planes each (24 bits, and fp32's
// range), and every product sums the six plane products above 2^-24, smallest
// first. Two fp16 planes and three products take two thirds of the time (step
// of 2048 x 1024 x 8192: 345 us, these 538), but their 22 bits need a common
// scale and end 2^-17 below the largest value of the matrix: entries of dw for
// improbable words, small columns and rows of small upstream gradients lost
// their bits.
#include <math.h>

#include <algorithm>
#include <utility>

#include "mm_sm100.cuh"
#include "xent.cuh"

namespace llattn {
namespace xent {
namespace {

using namespace mm;

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr int kTile = 128;  // columns per (max, sum) statistic

// fp32's plane products, smallest first: (0,2) (2,0) (1,1) (0,1) (1,0) (0,0); (1,.) (0,.) of G's two in bf16
constexpr uint32_t kTermsA = 0x010120u, kTermsB = 0x001102u, kFineA = 0x01u;

// Calls of few tokens have little to average an error over and time to spare: up
// to kFine tokens keep G in two bf16 planes (one plane's rounding of p - 1 is an
// error of the whole row, up to 1.5 times the output's own rounding for a
// single token, 1.2 times over some tens; 20 tokens of V = 32000: 155 us in two
// planes, 127 in one), and their tensor-core sums are short chains
// (MmArgs::chain): of 4 K = 64 steps for bf16 logits (the loss of 1 token at d = 2048: 2e-6 off
// without chains, 4e-7 with; one token's time is the same, 129 tokens of V = 32000
// would take 150 instead of 143 us), of 1 for fp32's. fp32's sums
// always run in chains (d = 2048, 300 tokens: gradients 1.4e-6 off at 1024
// products a sum, 7e-7 at 512, in the same time), bf16 logits where they are longer than kChain
// steps (losses of 1024 tokens, d = 2048: 1.0e-6 off in one sum, 5e-7 in two;
// d = 1536: 7.7e-7 in one, and two would take 148 instead of 142 us for 2048
// tokens).
constexpr int kFine = 64, kFineChain = 4, kFineF32Chain = 1, kF32Chain = 8, kChain = 24;

// ---- first product: statistics and exponentials ----------------------------

struct EpiStats {
  static constexpr bool kNarrow = false, kWide = false, kChain = true, kBegin = false;
  struct Pre {};
  __device__ __forceinline__ void fetch(Pre&, const MmArgs&, MmTile, int, int, int) const {}
  // not wide: sums over d are short, its long epilogue shows (757 us for 620)
  float2* stats;       // [rows][n_tiles]: (max, sum of exp(l - max))
  int n_tiles;
  const int* tgt;      // [rows] target of row (dev_base already added); < 0: none
  const int64_t* tgt64;
  float* lt;           // [rows] target logit
  void* p;             // exponentials of the rows, or null
  int64_t ldp;
  int p_f32;           // fp32 instead of fp16 * 2^15

  template <int CW>
  __device__ __forceinline__ void tile(const MmArgs& a, MmTile w, int row, int col0, int M, uint32_t taddr,
                                       bool zero, uint8_t* buf, Pre&) const {
    const int nv = min(kTile, a.N - col0);  // columns of this tile
    if (nv <= 0) return;                    // warp-uniform
    const int lane = threadIdx.x % 32;
    const bool row_ok = row < M;
    int t = -1;
    if (row_ok) t = tgt ? tgt[row] : (int)max((int64_t)-1, min(tgt64[row], (int64_t)a.N));
    t -= col0;
    float m = -INFINITY;
    float tv = 0.f;
#pragma unroll 1
    for (int cc = 0; cc < nv; cc += 32) {
      float v[32];
      load32(taddr + cc, zero, v);
      if (cc + 32 <= nv) {
#pragma unroll
        for (int q = 0; q < 32; ++q) m = fmaxf(m, v[q]);
      } else {
#pragma unroll
        for (int q = 0; q < 32; ++q) m = cc + q < nv ? fmaxf(m, v[q]) : m;
      }
      if ((unsigned)(t - cc) < 32u) {
#pragma unroll
        for (int q = 0; q < 32; ++q) tv = q == t - cc ? v[q] : tv;
      }
    }
    // fmaxf drops NaN: a row of NaN leaves m at -inf, and the sums below carry it
    // (the maximum itself gives exactly 1: a difference, not a fused product)
    const float mm = m == -INFINITY ? 0.f : m;
    float s0 = 0.f, s1 = 0.f;
    const int row0 = row - lane;
    const int64_t at = (int64_t)row0 * ldp + col0;
#pragma unroll 1
    for (int cc = 0; cc < nv; cc += 32) {
      float v[32];
      load32(taddr + cc, zero, v);
#pragma unroll
      for (int q = 0; q < 32; ++q) v[q] = cc + q < nv ? fast_exp2((v[q] - mm) * kLog2e) : 0.f;
#pragma unroll
      for (int q = 0; q < 32; q += 2) {
        s0 += v[q];
        s1 += v[q + 1];
      }
      if (!p) continue;
      if (p_f32) {
        uint4 u[8];
        f32_row(v, u);
        block_store(buf, lane, u, Rows{static_cast<float*>(p) + at + cc, ldp * 4, M - row0}, (nv - cc) * 4);
      } else {
        uint4 u[4];
#pragma unroll
        for (int q = 0; q < 32; ++q) v[q] *= 32768.f;
        half_row(v, u);
        block_store(buf, lane, u, Rows{static_cast<__half*>(p) + at + cc, ldp * 2, M - row0}, (nv - cc) * 2);
      }
    }
    if (row_ok) {
      // every column -inf: nothing to add
      const float sum = s0 + s1;
      stats[(int64_t)row * n_tiles + col0 / kTile] = make_float2(m == -INFINITY && sum == 0.f ? -INFINITY : mm, sum);
      if ((unsigned)t < (unsigned)nv) lt[row] = tv;
    }
  }
};

// Few tokens, no gradients: the vocabulary on the tile's long side (A = w), up
// to 32 tokens on its short one, so that w's rows are all that is copied.
// Statistics per token and 32 rows of w (a warp's).
constexpr int kFew = 32;

// lane q's result: op over the warp's lanes of their v[q] (v is used up; each of the
// five exchanges halves the values a lane still holds: 31 shuffles, not 160)
template <typename Op>
__device__ __forceinline__ float warp_transposed(float (&v)[32], int lane, Op op) {
#pragma unroll
  for (int s = 16; s >= 1; s >>= 1) {
    const bool up = lane & s;
#pragma unroll
    for (int i = 0; i < s; ++i) {
      const float away = up ? v[i] : v[i + s], mine = up ? v[i + s] : v[i];
      v[i] = op(mine, __shfl_xor_sync(0xffffffffu, away, s));
    }
  }
  return v[0];
}

struct EpiScore {
  static constexpr bool kNarrow = true, kWide = false, kChain = true, kBegin = false;
  struct Pre {};
  __device__ __forceinline__ void fetch(Pre&, const MmArgs&, MmTile, int, int, int) const {}
  float2* stats;  // [tokens][n_tiles]
  int n_tiles;
  const int64_t* targets;
  float* lt;

  template <int CW>
  __device__ __forceinline__ void tile(const MmArgs& a, MmTile w, int row, int col0, int M, uint32_t taddr,
                                       bool zero, uint8_t* buf, Pre&) const {
    const int lane = threadIdx.x % 32, n = min(CW, a.N - col0);
    if (row - lane >= M) return;  // warp-uniform
    float v[32];
    load32(taddr, zero, v);
    const int64_t t = lane < n ? targets[col0 + lane] : -1;
    float2 mine = make_float2(0.f, 0.f);
    // (32000 rows of w, 32 tokens: 47 us one token at a time, 39 transposed; 1 token: 34)
    if (n <= 4) {
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (q >= n) break;
        const float x = row < M ? v[q] : -INFINITY;
        const float m = warp_max(x), mm = m == -INFINITY ? 0.f : m;
        const float s = warp_sum(row < M ? fast_exp2((x - mm) * kLog2e) : 0.f);
        if (lane == q) mine = make_float2(m, s);
      }
    } else {
      float x[32];
#pragma unroll
      for (int q = 0; q < 32; ++q) x[q] = row < M ? v[q] : -INFINITY;
      mine.x = warp_transposed(x, lane, [](float a, float b) { return fmaxf(a, b); });
      const float mm = mine.x == -INFINITY ? 0.f : mine.x;
#pragma unroll
      for (int q = 0; q < 32; ++q) {
        const float mq = __shfl_sync(0xffffffffu, mm, q);  // (every lane takes part)
        x[q] = row < M ? fast_exp2((v[q] - mq) * kLog2e) : 0.f;
      }
      mine.y = warp_transposed(x, lane, [](float a, float b) { return a + b; });
    }
    mine.x = mine.x == -INFINITY && mine.y != 0.f ? 0.f : mine.x;
#pragma unroll
    for (int q = 0; q < 32; ++q) {
      if (q >= n) break;
      if (__shfl_sync(0xffffffffu, t, q) == row) lt[col0 + q] = v[q];
    }
    if (lane < n) stats[(int64_t)(col0 + lane) * n_tiles + row / 32] = mine;
  }
};

// ---- second and third product: rows out --------------------------------------

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

// ---- small kernels ------------------------------------------------------------

template <int NT>
__device__ __forceinline__ float block_max(float v, float* red) {
  v = warp_max(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float r = red[0];
#pragma unroll
  for (int i = 1; i < NT / 32; ++i) r = fmaxf(r, red[i]);
  return r;
}
template <int NT>
__device__ __forceinline__ float block_sum(float v, float* red) {
  v = warp_sum(v);
  __syncthreads();
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = v;
  __syncthreads();
  float r = 0.f;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) r += red[i];
  return r;
}

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

// rows of a matrix, packed; one warp per row
template <typename T>
__global__ void __launch_bounds__(256) xent_pack(const T* __restrict__ x, int64_t ldx, int n, int d, bf16* __restrict__ xs,
                                                 int64_t lds, int64_t plane) {
  pdl_next();
  pdl_wait();
  const int64_t r = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  if (r < n) pack_row<T>(x + r * ldx, d, xs + r * lds, lds, plane, vec_rows(x, ldx, d));
}

// Before the products of a training call. Lists the tokens that count, in
// order: idx[j] = row of the j-th, tgt[j] = its target (-1: out of range, which
// makes the row's loss and gradients NaN; lt[j] starts at NaN for the same
// reason), *count; packs their rows of x, xs[j] = x[idx[j]], and zeros the rows
// past the count. Each CTA takes `per` rows
// (a multiple of 8) and counts the targets before them for itself: reading a
// few hundred KB from L2 again costs less than a second launch or a wait
// (32768 targets: one CTA's scan alone took 56 us, this launch takes 55 with its
// 200 MB of packed rows, read and written). The first n_w CTAs pack w instead, 16 rows each.
template <typename T>
__global__ void __launch_bounds__(256) xent_prep(const T* __restrict__ x, int64_t ldx, int d,
                                                 const int64_t* __restrict__ targets, int n, int64_t ignore, int vocab,
                                                 int per, int* __restrict__ idx, int* __restrict__ tgt,
                                                 float* __restrict__ lt, int* __restrict__ count, bf16* __restrict__ xs,
                                                 int64_t lds, int64_t plane, const T* __restrict__ w, int64_t ldw,
                                                 bf16* __restrict__ wp, int64_t ldwp, int64_t wplane, int n_w) {
  pdl_next();
  pdl_wait();
  const int tid = threadIdx.x, lane = tid % 32, warp = tid / 32;
  if ((int)blockIdx.x < n_w) {
    const bool v = vec_rows(w, ldw, d);
    for (int64_t r = (int64_t)blockIdx.x * 16 + warp; r < min(vocab, ((int)blockIdx.x + 1) * 16); r += 8)
      pack_row<T>(w + r * ldw, d, wp + r * ldwp, ldwp, wplane, v);
    return;
  }
  __shared__ int red[2][8], pos[256];
  const int r0 = (blockIdx.x - n_w) * per, r1 = min(n, r0 + per);
  int before = 0, all = 0;
#pragma unroll 8
  for (int i = tid; i < n; i += 256) {
    const int k = targets[i] != ignore;
    all += k;
    before += i < r0 ? k : 0;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  all = __reduce_add_sync(0xffffffffu, all);
  if (lane == 0) {
    red[0][warp] = before;
    red[1][warp] = all;
  }
  __syncthreads();
  before = all = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    before += red[0][i];
    all += red[1][i];
  }
  if (blockIdx.x == n_w && tid == 0) {
    count[0] = all;
    count[1] = 0;  // rows done (xent_rows)
  }
  const bool vec = vec_rows(x, ldx, d);
  for (int c0 = r0; c0 < r1; c0 += 256) {
    const int i = c0 + tid;
    const int64_t t = i < r1 ? targets[i] : ignore;
    const bool keep = t != ignore;
    const unsigned b = __ballot_sync(0xffffffffu, keep);
    __syncthreads();
    if (lane == 0) red[0][warp] = __popc(b);
    __syncthreads();
    int j = before + __popc(b & ((1u << lane) - 1u));
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      j += k < warp ? red[0][k] : 0;
      before += red[0][k];
    }
    pos[tid] = keep ? j : -1;
    if (keep) {
      idx[j] = i;
      tgt[j] = t >= 0 && t < vocab ? (int)t : -1;
      lt[j] = __int_as_float(0x7fc00000);
    }
    __syncthreads();
    for (int k = warp; k < min(256, r1 - c0); k += 8) {
      const int64_t row = c0 + k;
      if (pos[k] >= 0) pack_row<T>(x + row * ldx, d, xs + pos[k] * lds, lds, plane, vec);
      if (row >= all) pack_row<T>(nullptr, d, xs + row * lds, lds, plane, vec);
    }
  }
}

// logsumexp of a row from its tiles, as (max, log2 of the sum relative to it)
template <int NT>
__device__ __forceinline__ float2 join_tiles(const float2* __restrict__ st, int n_tiles, float* red) {
  // the first 8 NT tiles (all of them up to V = 32 K a tile of 32 columns) are
  // read once, together
  constexpr int KEEP = 8;
  float2 c[KEEP];
  float m = -INFINITY;
#pragma unroll
  for (int r = 0; r < KEEP; ++r) {
    const int i = threadIdx.x + r * NT;
    c[r] = i < n_tiles ? st[i] : make_float2(-INFINITY, 0.f);
  }
#pragma unroll
  for (int r = 0; r < KEEP; ++r) m = fmaxf(m, c[r].x);
#pragma unroll 4
  for (int i = threadIdx.x + KEEP * NT; i < n_tiles; i += NT) m = fmaxf(m, st[i].x);
  m = block_max<NT>(m, red);
  float s = 0.f;
  auto add = [&](float2 v) { s += v.x == -INFINITY ? 0.f : v.y * exp2f((v.x - m) * kLog2e); };
#pragma unroll
  for (int r = 0; r < KEEP; ++r)
    if (r * NT < n_tiles) add(c[r]);
#pragma unroll 4
  for (int i = threadIdx.x + KEEP * NT; i < n_tiles; i += NT) add(st[i]);
  s = block_sum<NT>(s, red);
  return make_float2(m, log2f(s));
}

__device__ __forceinline__ float row_loss(float2 lse, float lt) { return (lse.x - lt) + lse.y * kLn2; }

// Losses without gradients: one CTA per row.
__global__ void __launch_bounds__(128) xent_losses(const float2* __restrict__ stats, int n_tiles,
                                                   const float* __restrict__ lt, const int64_t* __restrict__ targets,
                                                   int64_t ignore, int vocab, float* __restrict__ losses) {
  __shared__ float red[4];
  pdl_next();
  pdl_wait();
  const int64_t row = blockIdx.x, t = targets[row];
  const float at = lt[row];
  const float2 lse = join_tiles<128>(stats + row * n_tiles, n_tiles, red);
  if (threadIdx.x == 0) {
    const float l = t >= 0 && t < vocab ? row_loss(lse, at) : __int_as_float(0x7fc00000);
    losses[row] = t == ignore ? 0.f : l;
  }
}

// The last of the grid's CTAs to come here sums losses[0, n) into *loss.
__device__ __forceinline__ void sum_losses(int* count, const float* losses, int n, int mean, float* loss, float* red,
                                           int* last) {
  __syncthreads();
  if (threadIdx.x == 0) {
    __threadfence();
    *last = atomicAdd(count + 1, 1) == (int)(gridDim.x * gridDim.y) - 1;
  }
  __syncthreads();
  if (!*last) return;
  __threadfence();
  float s = 0.f;
#pragma unroll 32
  for (int i = threadIdx.x; i < n; i += 256) s += __ldcg(losses + i);
  s = block_sum<256>(s, red);
  if (threadIdx.x == 0) *loss = mean ? s / (float)max(n, 1) : s;
}

// One CTA per row of a piece (few rows: SHARES of them, along y, each a share
// of the columns): joins the tiles, writes the row's loss and rewrites the
// exponentials as G = g (p - onehot), g = 1 or grad_rows: in place, or, from fp32
// exponentials, in two or three bf16 planes apart. Rows between the count and the next multiple
// of 64 become zeros: the third product reads them. The last CTA of the last
// piece to finish sums the losses (thread t those of index t mod 256, then
// in thread order: the same bits whichever CTA it is).
template <int PLANES, int SHARES>
__global__ void __launch_bounds__(256) xent_rows(const float2* __restrict__ stats, int n_tiles, int rows, int vocab,
                                                 int* __restrict__ count, int base, const int* __restrict__ idx,
                                                 const int* __restrict__ tgt, const float* __restrict__ lt,
                                                 const float* __restrict__ grad_rows, int mean, float* losses,
                                                 void* __restrict__ p, int64_t ldp, bf16* __restrict__ planes,
                                                 int64_t plane, float* __restrict__ loss) {
  constexpr bool SPLIT = PLANES > 1;
  extern __shared__ float xent_f[];  // [n_tiles]
  __shared__ float red[8];
  __shared__ int last;
  pdl_next();
  pdl_wait();
  const int n_all = *count;
  const int n = cut_rows(rows, count, base);
  const int64_t row = blockIdx.x;
  if (row >= n) {
    if (row < cdiv(n, 64) * 64) {
      const uint4 z = make_uint4(0, 0, 0, 0);
      for (int64_t c = blockIdx.y * 256 + threadIdx.x; c < ldp / 8; c += 256 * SHARES) {
        if (SPLIT) {
          for (int k = 0; k < PLANES; ++k) reinterpret_cast<uint4*>(planes + k * plane + row * ldp)[c] = z;
        } else {
          reinterpret_cast<uint4*>(static_cast<bf16*>(p) + row * ldp)[c] = z;
        }
      }
    }
    if (loss) sum_losses(count, losses, n_all, mean, loss, red, &last);
    return;
  }
  const float2* st = stats + row * n_tiles;
  const float2 lse = join_tiles<256>(st, n_tiles, red);
  const int t = tgt[row];
  if (threadIdx.x == 0 && blockIdx.y == 0) losses[base + row] = row_loss(lse, lt[row]);
  float g = grad_rows ? grad_rows[idx[row]] : 1.f;
  if (t < 0) g = __int_as_float(0x7fc00000);
  // tile factors: g 2^(m_tile - lse)
  for (int i = threadIdx.x; i < n_tiles; i += 256) {
    const float m = st[i].x;
    xent_f[i] = m == -INFINITY ? 0.f : g * exp2f((m - lse.x) * kLog2e - lse.y) * (SPLIT ? 1.f : 0x1p-15f);
  }
  __syncthreads();
  for (int c = (blockIdx.y * 256 + threadIdx.x) * 8; c < vocab; c += 256 * 8 * SHARES) {
    const float f = xent_f[c / kTile];
    float v[8];
    if (SPLIT) {
      const float4* src = reinterpret_cast<const float4*>(static_cast<const float*>(p) + row * ldp + c);
      const float4 a = src[0], b = src[1];
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
      v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
      const uint4 u = *reinterpret_cast<const uint4*>(static_cast<const __half*>(p) + row * ldp + c);
      const __half2* h = reinterpret_cast<const __half2*>(&u);
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float2 x = __half22float2(h[q]);
        v[2 * q] = x.x;
        v[2 * q + 1] = x.y;
      }
    }
#pragma unroll
    for (int q = 0; q < 8; ++q) v[q] = v[q] * f - (c + q == t ? g : 0.f);
    if (SPLIT) {
      uint32_t o[4][3];
#pragma unroll
      for (int q = 0; q < 4; ++q) split3(v[2 * q], v[2 * q + 1], o[q]);
#pragma unroll
      for (int k = 0; k < PLANES; ++k)
        *reinterpret_cast<uint4*>(planes + k * plane + row * ldp + c) = make_uint4(o[0][k], o[1][k], o[2][k], o[3][k]);
    } else {
      *reinterpret_cast<uint4*>(static_cast<bf16*>(p) + row * ldp + c) =
          make_uint4(pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[4], v[5]), pack_bf16(v[6], v[7]));
    }
  }
  if (loss) sum_losses(count, losses, n_all, mean, loss, red, &last);
}

// loss = sum of the losses (ignored tokens' are 0), over the number that count
// when mean. One CTA, fixed order.
__global__ void __launch_bounds__(1024) xent_reduce(const float* __restrict__ losses, int n,
                                                    const int64_t* __restrict__ targets, int64_t ignore, int mean,
                                                    float* __restrict__ loss) {
  pdl_next();
  pdl_wait();
  __shared__ float red[32];
  float s = 0.f, c = 0.f;
  for (int i = threadIdx.x; i < n; i += 1024) {
    s += losses[i];
    c += targets[i] != ignore ? 1.f : 0.f;  // per thread: exact up to 2^24
  }
  s = block_sum<1024>(s, red);
  c = block_sum<1024>(c, red);
  if (threadIdx.x == 0) *loss = mean ? s / fmaxf(c, 1.f) : s;
}

// a *= *s, b *= *s, unless *s is 1; whole 16-byte chunks where aligned
template <typename T>
__device__ __forceinline__ void scale_run(T* p, int64_t n, float f) {
  constexpr int PER = 16 / sizeof(T);
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  const int64_t nv = (reinterpret_cast<uintptr_t>(p) & 15) ? 0 : n / PER;
  for (int64_t i = i0; i < nv; i += step) {
    uint4 u = reinterpret_cast<uint4*>(p)[i];
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int q = 0; q < PER; ++q) e[q] = from_f<T>(to_f<T>(e[q]) * f);
    reinterpret_cast<uint4*>(p)[i] = u;
  }
  for (int64_t i = nv * PER + i0; i < n; i += step) p[i] = from_f<T>(to_f<T>(p[i]) * f);
}
template <typename T>
__global__ void __launch_bounds__(256) scale_kernel(T* __restrict__ a, int64_t na, T* __restrict__ b, int64_t nb,
                                                    const float* __restrict__ s) {
  pdl_next();
  pdl_wait();
  const float f = *s;
  if (f == 1.f) return;
  scale_run(a, na, f);
  scale_run(b, nb, f);
}

// ---- host side ------------------------------------------------------------------

size_t up256(size_t v) { return (v + 255) & ~(size_t)255; }
int64_t up8(int64_t v) { return (v + 7) & ~(int64_t)7; }

bool aligned_rows(const void* p, int64_t ld, int64_t rows, int elt) {
  return ((uintptr_t)p & 15) == 0 && (rows == 1 || ld % (16 / elt) == 0);
}

struct Plan {
  bool f32, train, few, pack_x, pack_w;
  int elt, planes, gplanes, n_tiles, piece, n_pieces;
  int64_t ldx, ldw, ldp, ldd;
  size_t part_bytes;
  size_t xs, ws, stats, lt, idx, tgt, count, losses, p, g, acc, part, total;
};

MmArgs base_args(const Plan& q, volatile unsigned* fault) {
  MmArgs p = {};
  p.n_terms = q.f32 ? 6 : 1;
  p.pa = q.f32 ? kTermsA : 0;
  p.pb = q.f32 ? kTermsB : 0;
  p.nz = 1;
  p.fault_host = fault;
  return p;
}

// dx = G w and dw = G^T x of a piece
MmArgs grad_args(const Plan& q, const llattn_xent_args& a, volatile unsigned* fault) {
  MmArgs m = base_args(q, fault);
  if (q.f32) {
    m.chain = a.tokens <= kFine ? kFineF32Chain : kF32Chain;
  } else if (q.gplanes == 2) {
    m.n_terms = 2;
    m.pa = kFineA;
  }
  return m;
}
MmArgs dx_args(const Plan& q, const llattn_xent_args& a, int rows, volatile unsigned* fault) {
  MmArgs m = grad_args(q, a, fault);
  m.M = rows;
  m.N = a.d;
  m.K = a.vocab;
  m.split = 1;
  return m;
}
MmArgs dw_args(const Plan& q, const llattn_xent_args& a, int rows, volatile unsigned* fault) {
  MmArgs m = grad_args(q, a, fault);
  m.M = a.vocab;
  m.N = a.d;
  m.K = rows;
  m.split = 1;
  return m;
}

int logits_chain(const Plan& q, const llattn_xent_args& a) {
  const int steps = cdiv(a.d, 64);
  if (q.f32) return a.tokens <= kFine ? kFineF32Chain : kF32Chain;
  return a.tokens <= kFine ? kFineChain : steps > kChain ? cdiv(steps, cdiv(steps, kChain)) : 0;
}

Plan make_plan(const llattn_xent_args& a) {
  Plan q;
  q.f32 = a.dtype == LLATTN_F32;
  q.elt = q.f32 ? 4 : 2;
  q.planes = q.f32 ? 3 : 1;
  q.train = a.dx || a.dw || a.stage != LLATTN_XENT_ALL;
  q.gplanes = q.f32 ? 3 : a.tokens <= kFine ? 2 : 1;
  q.pack_x = q.f32 || q.train || !aligned_rows(a.x, a.ldx, a.tokens, 2);
  q.pack_w = q.f32 || !aligned_rows(a.w, a.ldw, a.vocab, 2);
  q.ldx = q.pack_x ? up8(a.d) : (a.tokens == 1 ? up8(a.d) : a.ldx);
  q.ldw = q.pack_w ? up8(a.d) : (a.vocab == 1 ? up8(a.d) : a.ldw);
  q.ldp = up8(a.vocab);
  q.ldd = up8(a.d);
  q.few = !q.train && a.tokens <= kFew;
  q.n_tiles = cdiv(a.vocab, q.few ? 32 : kTile);
  // rows of exponentials held at a time: half a GiB of them (V = 32000 in
  // bf16: 8192 rows), whole row tiles
  const int p_bytes = q.gplanes > 1 ? 4 : 2;  // an exponential's
  const int64_t row_bytes = q.ldp * (q.gplanes > 1 ? p_bytes + 2 * q.gplanes : p_bytes);
  const int64_t piece = std::max<int64_t>(256, (int64_t)(512u << 20) / row_bytes / 256 * 256);
  q.piece = (int)std::min<int64_t>(piece, a.tokens);
  if (!q.train) q.piece = a.tokens;
  q.n_pieces = cdiv(a.tokens, q.piece);
  size_t off = 0;
  auto take = [&](size_t b) { size_t o = off; off += up256(b); return o; };
  const size_t n = a.tokens;
  q.xs = take(q.pack_x ? 2 * (size_t)q.planes * n * q.ldx : 0);
  q.ws = take(q.pack_w ? 2 * (size_t)q.planes * a.vocab * q.ldw : 0);
  q.stats = take(sizeof(float2) * (size_t)q.piece * q.n_tiles);
  q.lt = take(4 * n);
  q.idx = take(q.train ? 4 * n : 0);
  q.tgt = take(q.train ? 4 * n : 0);
  q.count = take(8);
  q.losses = take(4 * n);
  q.p = take(q.train ? (size_t)q.piece * q.ldp * p_bytes : 0);
  q.g = take(q.train && q.gplanes > 1 ? 2 * (size_t)q.gplanes * q.piece * q.ldp : 0);
  q.acc = take(q.train && a.dw && q.n_pieces > 1 ? 4 * (size_t)a.vocab * q.ldd : 0);
  int64_t part = 0;
  if (a.dx) part = mm_part_floats(dx_args(q, a, q.piece, nullptr));
  if (a.dw) part = std::max(part, mm_part_floats(dw_args(q, a, q.piece, nullptr)));
  q.part_bytes = 4 * (size_t)part;
  q.part = take(a.stage == LLATTN_XENT_ALL ? q.part_bytes : 0);
  q.total = off;
  return q;
}

#define TRY(x)                          \
  do {                                  \
    cudaError_t e_ = (x);               \
    if (e_ != cudaSuccess) return e_;   \
  } while (0)

template <typename T>
cudaError_t run(const llattn_xent_args& a, const Plan& q, volatile unsigned* fault, cudaStream_t s) {
  const bool grads = a.stage == LLATTN_XENT_GRADS;  // on what a call of stage LOSS left in its workspace
  char* ws = static_cast<char*>(grads ? a.kept : a.workspace);
  bf16* xs = reinterpret_cast<bf16*>(ws + q.xs);
  bf16* wp = reinterpret_cast<bf16*>(ws + q.ws);
  float2* stats = reinterpret_cast<float2*>(ws + q.stats);
  float* lt = reinterpret_cast<float*>(ws + q.lt);
  int* idx = reinterpret_cast<int*>(ws + q.idx);
  int* tgt = reinterpret_cast<int*>(ws + q.tgt);
  int* count = reinterpret_cast<int*>(ws + q.count);
  const int n = a.tokens, d = a.d, V = a.vocab;
  const bool mean = a.reduction == LLATTN_XENT_MEAN;
  const int64_t xplane = (int64_t)n * q.ldx, wplane = (int64_t)V * q.ldw;
  const void* wv = q.pack_w ? wp : a.w;
  if (!q.train) {
    if (q.pack_w) {
      TRY(launch_pdl(xent_pack<T>, dim3(cdiv(V, 8)), 256, 0, 1, s, static_cast<const T*>(a.w), a.ldw, V, d, wp, q.ldw, wplane));
    }
    if (q.pack_x) {
      TRY(launch_pdl(xent_pack<T>, dim3(cdiv(n, 8)), 256, 0, 1, s, static_cast<const T*>(a.x), a.ldx, n, d, xs, q.ldx, xplane));
    }
    MmArgs p = base_args(q, fault);
    const Operand ox{q.pack_x ? xs : a.x, n, d, q.ldx, q.planes, xplane, 0}, ow{wv, V, d, q.ldw, q.planes, wplane, 0};
    p.K = d;
    p.chain = logits_chain(q, a);
    if (q.few) {
      p.M = V;
      p.N = n;
      std::swap(p.pa, p.pb);
      TRY(launch_mm_sh<0>(p, ow, ox, EpiScore{stats, q.n_tiles, a.targets, lt}, s));
    } else {
      p.M = n;
      p.N = V;
      TRY(launch_mm(p, ox, ow, EpiStats{stats, q.n_tiles, nullptr, a.targets, lt, nullptr, 0, 0}, s));
    }
    float* losses = a.losses ? a.losses : reinterpret_cast<float*>(ws + q.losses);
    TRY(launch_pdl(xent_losses, dim3(n), 128, 0, 1, s, stats, q.n_tiles, lt, a.targets, a.ignore_index, V, losses));
    if (a.loss) {
      TRY(launch_pdl(xent_reduce, dim3(1), 1024, 0, 1, s, losses, n, a.targets, a.ignore_index, mean, a.loss));
    }
    return cudaSuccess;
  }
  const int per = std::max(8, cdiv(cdiv(n, 512), 8) * 8), n_w = q.pack_w ? cdiv(V, 16) : 0;
  if (!grads)
    TRY(launch_pdl(xent_prep<T>, dim3(n_w + cdiv(n, per)), 256, 0, 1, s, static_cast<const T*>(a.x), a.ldx, d, a.targets, n,
                   a.ignore_index, V, per, idx, tgt, lt, count, xs, q.ldx, xplane, static_cast<const T*>(a.w), a.ldw, wp,
                   q.ldw, wplane, n_w));
  float* losses = reinterpret_cast<float*>(ws + q.losses);
  void* pbuf = ws + q.p;
  bf16* gpl = reinterpret_cast<bf16*>(ws + q.g);
  float* acc = reinterpret_cast<float*>(ws + q.acc);
  float* part = reinterpret_cast<float*>(grads ? static_cast<char*>(a.workspace) : ws + q.part);  // split tiles of one product at a time
  const int64_t gplane = (int64_t)q.piece * q.ldp;
  for (int c = 0; c < q.n_pieces; ++c) {
    const int base = c * q.piece, rows = std::min(q.piece, n - base);
    const Operand ox{xs + (int64_t)base * q.ldx, rows, d, q.ldx, q.planes, xplane, 0};
    MmArgs p = base_args(q, fault);
    p.m_dev = count;
    p.dev_base = base;
    p.M = rows;
    p.N = V;
    p.K = d;
    p.chain = logits_chain(q, a);
    EpiStats ep{stats, q.n_tiles, tgt + base, nullptr, lt + base, pbuf, q.ldp, q.gplanes > 1};
    if (!grads) TRY(launch_mm(p, ox, Operand{wv, V, d, q.ldw, q.planes, wplane, 0}, ep, s));
    const size_t sm = sizeof(float) * q.n_tiles;
    auto rows_pass = [&](auto kernel, int shares) {
      if (sm > 48 * 1024) {  // V past 1.5 M, of at most 2 M
        const cudaError_t e = set_smem_once(kernel, 64 * 1024);
        if (e != cudaSuccess) return e;
      }
      return launch_pdl(kernel, dim3(rows, shares), 256, sm, 1, s, stats, q.n_tiles, rows, V, count, base, idx + base, tgt + base,
                        lt + base, a.grad_rows, mean, losses, pbuf, q.ldp, gpl, gplane, c + 1 == q.n_pieces ? a.loss : nullptr);
    };
    const bool share = rows <= 2 * sm_count() && V >= 4096;  // (129 rows of 32000: 12.7 -> 9.1 us)
    auto rows_as = [&](auto planes) {
      constexpr int P = decltype(planes)::value;
      return share ? rows_pass(xent_rows<P, 4>, 4) : rows_pass(xent_rows<P, 1>, 1);
    };
    using std::integral_constant;
    if (grads) {
    } else if constexpr (sizeof(T) == 4) {
      TRY(rows_as(integral_constant<int, 3>{}));
    } else if (q.gplanes == 2) {
      TRY(rows_as(integral_constant<int, 2>{}));
    } else {
      TRY(rows_as(integral_constant<int, 1>{}));
    }
    const void* g = q.gplanes > 1 ? gpl : pbuf;
    if (a.dx) {
      MmArgs m = dx_args(q, a, rows, fault);
      m.m_dev = count;
      m.dev_base = base;
      m.part = part;
      EpiOut eo{};
      eo.out = a.dx;
      eo.ldo = d;
      eo.out_bf16 = !q.f32;
      eo.vec = aligned_rows(a.dx, d, 2, q.elt);
      eo.factor = a.factor;
      eo.zero = c ? nullptr : a.targets;
      eo.zero_n = n;
      eo.ignore = a.ignore_index;
      eo.idx = idx + base;
      eo.count = mean ? count : nullptr;
      TRY(launch_mm(m, Operand{g, rows, V, q.ldp, q.gplanes, gplane, 0}, Operand{wv, V, d, q.ldw, q.planes, wplane, 1}, eo,
                    s));
    }
    if (a.dw) {
      MmArgs m = dw_args(q, a, rows, fault);
      m.k_dev = count;
      m.dev_base = base;
      m.part = part;
      EpiOut eo{};
      const bool last = c + 1 == q.n_pieces;
      eo.out = last ? a.dw : acc;
      eo.ldo = last ? d : q.ldd;
      eo.out_bf16 = last && !q.f32;
      eo.vec = last ? aligned_rows(a.dw, d, 2, q.elt) : 1;
      eo.add = c && !last;
      eo.acc = c && last ? acc : nullptr;
      eo.ldacc = q.ldd;
      eo.count = last && mean ? count : nullptr;
      eo.factor = a.factor;
      TRY(launch_mm(m, Operand{g, rows, V, q.ldp, q.gplanes, gplane, 1}, Operand{ox.p, rows, d, q.ldx, q.planes, xplane, 1},
                    eo, s));
    }
  }
  return cudaSuccess;
}

}  // namespace

size_t workspace_bytes(const llattn_xent_args& a) {
  const Plan q = make_plan(a);
  if (a.stage != LLATTN_XENT_ALL && q.n_pieces > 1) return 0;
  return a.stage == LLATTN_XENT_GRADS ? std::max<size_t>(256, up256(q.part_bytes)) : q.total;
}

int launches(const llattn_xent_args& a) {
  const Plan q = make_plan(a);
  if (!q.train) return q.pack_w + q.pack_x + 2 + (a.loss ? 1 : 0);
  const int loss = a.stage == LLATTN_XENT_GRADS ? 0 : 1;
  return loss + q.n_pieces * (2 * loss + (a.dx ? 1 + joins(dx_args(q, a, q.piece, nullptr)) : 0) +
                           (a.dw ? 1 + joins(dw_args(q, a, q.piece, nullptr)) : 0));
}

cudaError_t launch(const llattn_xent_args& a, volatile unsigned* fault, cudaStream_t s) {
  const Plan q = make_plan(a);
  return q.f32 ? run<float>(a, q, fault, s) : run<bf16>(a, q, fault, s);
}

cudaError_t launch_scale(void* a, int64_t na, void* b, int64_t nb, int dtype, const float* f, cudaStream_t s) {
  const int64_t blocks = std::max<int64_t>(1, std::min<int64_t>((std::max(na, nb) + 2047) / 2048, 8 * sm_count()));
  const dim3 grid((unsigned)blocks);
  if (dtype == LLATTN_BF16)
    return launch_pdl(scale_kernel<bf16>, grid, 256, 0, 1, s, static_cast<bf16*>(a), na, static_cast<bf16*>(b), nb, f);
  return launch_pdl(scale_kernel<float>, grid, 256, 0, 1, s, static_cast<float*>(a), na, static_cast<float*>(b), nb, f);
}

unsigned read_fault_word(bool reset) { return read_fault(reset); }

}  // namespace xent
}  // namespace llattn
