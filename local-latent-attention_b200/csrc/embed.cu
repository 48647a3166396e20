// Token embedding with its positions, and its gradients:
//   out[b, t] = scale W[ids[b, t]] + P[t]
//   dW[v] = scale sum_{(b, t): ids[b, t] = v} dout[b, t],  dP[t] = sum_b dout[b, t]
//
// dW goes by the tokens sorted by word. The sort is one launch: each CTA
// owns a range of words and reads all ids (from the L2) for itself, so that no CTA
// waits for another: it counts its words' tokens and the tokens of smaller words,
// then writes its tokens, word by word and in their order, to where these
// start. Rows are then summed in that order, whatever the launch: a warp per word and
// 2 KB of columns, zeros for a word without tokens. A word of more than kHot tokens
// is cut at the multiples of kHot of the sorted order; the pieces' sums go
// through the workspace and are added in order. No atomics on values: the same bits
// every run.
#include <math.h>

#include <algorithm>

#include "embed.cuh"
#include "pdl.cuh"

namespace llattn {
namespace embed {
namespace {

constexpr int kHot = 64;
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kMostWords = 1280;  // of a sorting CTA: 32 counters each, 160 KB
constexpr int kSlice = 4;         // 16-byte vectors a lane takes of a row at a time

struct Ids {
  const void* p;
  int wide;  // int64, else int32
  int64_t vocab, padding;
  __device__ __forceinline__ int64_t at(int64_t i) const {
    return wide ? static_cast<const int64_t*>(p)[i] : (int64_t) static_cast<const int*>(p)[i];
  }
};

// V consecutive elements of a row: 16 bytes, or one element
template <typename T, bool VEC>
struct Pack {
  static constexpr int N = VEC ? 16 / sizeof(T) : 1;
  float v[N];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC) {
      const uint4 u = *reinterpret_cast<const uint4*>(p);
      const T* e = reinterpret_cast<const T*>(&u);
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = to_f<T>(e[i]);
    } else {
      v[0] = to_f<T>(*p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (VEC) {
      uint4 u;
      T* e = reinterpret_cast<T*>(&u);
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = from_f<T>(v[i]);
      *reinterpret_cast<uint4*>(p) = u;
    } else {
      *p = from_f<T>(v[0]);
    }
  }
  __device__ __forceinline__ void fill(float x) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = x;
  }
  __device__ __forceinline__ void add(const Pack& o) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += o.v[i];
  }
  __device__ __forceinline__ void times(float f) {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] *= f;
  }
};

// ---- forward ----------------------------------------------------------------------

// A thread per pack of columns. per_row: packs of a row.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) embed_rows(Ids ids, const T* __restrict__ w, int64_t ldw, const T* __restrict__ pos,
                                                  int64_t ldp, int length, int64_t total, int per_row, int d, float scale,
                                                  T* __restrict__ out) {
  pdl_next();
  pdl_wait();
  using P = Pack<T, VEC>;
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= total) return;
  const int64_t n = total <= INT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)per_row) : i / per_row;
  const int c = (int)(i - n * per_row) * P::N;
  const int64_t id = ids.at(n);
  P r, q;
  if (id >= 0 && id < ids.vocab) {
    r.load(w + id * ldw + c);
    if (pos) {
      const int t = (int)(n % length);
      q.load(pos + t * ldp + c);
#pragma unroll
      for (int k = 0; k < P::N; ++k) r.v[k] = fmaf(r.v[k], scale, q.v[k]);
    } else {
      r.times(scale);
    }
  } else {
    r.fill(__int_as_float(0x7fc00000));  // no such word
  }
  r.store(out + n * d + c);
}

// ---- the sort -----------------------------------------------------------------------

// order: the counted tokens by word, then by index; words: their words; start[v]: a
// word's first place, start[vocab]: their number.
__global__ void __launch_bounds__(kSortThreads) embed_sort(Ids ids, int n, int span, int* __restrict__ order,
                                                           int* __restrict__ words, int* __restrict__ start) {
  extern __shared__ int counts[];  // [kSortWarps][span]
  __shared__ int sums[kSortWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int64_t lo = (int64_t)blockIdx.x * span;
  const int mine = (int)min((int64_t)span, ids.vocab - lo);
  int* my = counts + warp * span;
  for (int i = threadIdx.x; i < kSortWarps * span; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  pdl_next();
  pdl_wait();
  const int per = cdiv(cdiv(n, kSortWarps), 32) * 32, i0 = min(n, warp * per), i1 = min(n, i0 + per);
  int below = 0;
  auto each = [&](auto body) {  // groups of 32 ids in order, several loads in flight
#pragma unroll 1
    for (int i = i0; i < i1; i += 256) {
      int64_t id[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int j = i + 32 * k + lane;
        id[k] = j < i1 ? ids.at(j) : -1;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (id[k] == ids.padding || id[k] >= ids.vocab) id[k] = -1;
        body(id[k], i + 32 * k + lane);
      }
    }
  };
  each([&](int64_t id, int) {
    below += id >= 0 && id < lo;
    if (id >= lo && id < lo + mine) atomicAdd(my + (int)(id - lo), 1);
  });
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) sums[warp] = below;
  __syncthreads();
  // counters -> places: over the warps of a word, then over the words
  int base = 0;
#pragma unroll
  for (int i = 0; i < kSortWarps; ++i) base += sums[i];
  __syncthreads();
  for (int r0 = 0; r0 < mine; r0 += kSortThreads) {
    const int r = r0 + threadIdx.x;
    int all = 0;
    if (r < mine)
      for (int k = 0; k < kSortWarps; ++k) all += counts[k * span + r];
    int scan = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += v;
    }
    if (lane == 31) sums[warp] = scan;
    __syncthreads();
    int at = base + scan - all;
#pragma unroll
    for (int k = 0; k < kSortWarps; ++k) {
      at += k < warp ? sums[k] : 0;
      base += sums[k];
    }
    __syncthreads();
    if (r < mine) {
      start[lo + r] = at;
      for (int k = 0; k < kSortWarps; ++k) {
        const int c = counts[k * span + r];
        counts[k * span + r] = at;
        at += c;
      }
    }
  }
  if (threadIdx.x == 0 && lo + mine == ids.vocab) start[ids.vocab] = base;
  __syncthreads();
  each([&](int64_t id, int i) {
    const bool in = id >= lo && id < lo + mine;
    const unsigned some = __ballot_sync(0xffffffffu, in);
    if (!some) return;
    if (in) {
      const int r = (int)(id - lo);
      const unsigned same = __match_any_sync(some, r);
      const int at = my[r] + __popc(same & ((1u << lane) - 1u));
      __syncwarp(some);
      order[at] = i;
      words[at] = (int)id;
      if ((same >> lane) == 1u) my[r] = at + 1;  // the last of them
    }
    __syncwarp();
  });
}

// ---- gradients ------------------------------------------------------------------------

// Columns [c0, c0 + kSlice 32 packs) of the sum of rows order[s, e) of dout, one warp.
template <typename T, bool VEC>
__device__ __forceinline__ void sum_rows(Pack<T, VEC> (&a)[kSlice], const T* __restrict__ dout, const int* __restrict__ order,
                                         int s, int e, int d, int c0) {
  using P = Pack<T, VEC>;
  const int lane = threadIdx.x % 32;
#pragma unroll
  for (int k = 0; k < kSlice; ++k) a[k].fill(0.f);
  for (int b = s; b < e; b += 32) {
    const int mine = b + lane < e ? order[b + lane] : 0, m = min(32, e - b);
#pragma unroll 2
    for (int j = 0; j < m; ++j) {
      const T* row = dout + (int64_t)__shfl_sync(0xffffffffu, mine, j) * d;
      P r[kSlice];
#pragma unroll
      for (int k = 0; k < kSlice; ++k) {
        const int c = c0 + (k * 32 + lane) * P::N;
        r[k].fill(0.f);
        if (c < d) r[k].load(row + c);
      }
#pragma unroll
      for (int k = 0; k < kSlice; ++k) a[k].add(r[k]);
    }
  }
}

// Warps [0, vocab slices) write the words of up to kHot tokens, the next ones the sums
// of the pieces of the others: slot 2 p holds what interval p of the sorted order has
// of its first word, slot 2 p + 1 what it has of its last one, where that is another.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) embed_sums(const T* __restrict__ dout, const int* __restrict__ order,
                                                  const int* __restrict__ words, const int* __restrict__ start, int64_t vocab,
                                                  int d, int slices, int pieces, float scale, float* __restrict__ part,
                                                  T* __restrict__ dw) {
  pdl_next();
  pdl_wait();
  using P = Pack<T, VEC>;
  const int lane = threadIdx.x % 32;
  const int64_t w = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t v = w / slices;
  const int c0 = (int)(w - v * slices) * (kSlice * 32 * P::N);
  P a[kSlice];
  if (v < vocab) {
    const int s = start[v], e = start[v + 1];
    if (e - s > kHot) return;
    sum_rows<T, VEC>(a, dout, order, s, e, d, c0);
#pragma unroll
    for (int k = 0; k < kSlice; ++k) {
      const int c = c0 + (k * 32 + lane) * P::N;
      a[k].times(scale);
      if (c < d) a[k].store(dw + v * d + c);
    }
    return;
  }
  const int64_t p = v - vocab;
  const int total = start[vocab];
  if (p >= pieces || p * kHot >= total) return;
  const int lo = (int)p * kHot, hi = min(lo + kHot, total);
  for (int last = 0; last < 2; ++last) {
    const int word = words[last ? hi - 1 : lo];
    if (last && word == words[lo]) break;
    const int s = start[word], e = start[word + 1];
    if (e - s <= kHot) continue;
    sum_rows<T, VEC>(a, dout, order, max(s, lo), min(e, hi), d, c0);
#pragma unroll
    for (int k = 0; k < kSlice; ++k) {
      const int c = c0 + (k * 32 + lane) * P::N;
      if (c < d)
#pragma unroll
        for (int i = 0; i < P::N; ++i) part[(2 * p + last) * d + c + i] = a[k].v[i];
    }
  }
}

// The words of more than kHot tokens: a warp for each that starts in interval p (there
// is one at most: the interval's last word), 32 columns.
template <typename T>
__global__ void __launch_bounds__(256) embed_join(const int* __restrict__ words, const int* __restrict__ start, int64_t vocab,
                                                  int d, int slices, int pieces, float scale, const float* __restrict__ part,
                                                  T* __restrict__ dw) {
  pdl_next();
  pdl_wait();
  const int64_t w = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t p = w / slices;
  const int c = (int)(w - p * slices) * 32 + threadIdx.x % 32;
  const int total = start[vocab];
  if (p >= pieces || p * kHot >= total) return;
  const int word = words[min((int)p * kHot + kHot, total) - 1];
  const int s = start[word], e = start[word + 1];
  if (e - s <= kHot || s / kHot != p || c >= d) return;
  const int q1 = (e - 1) / kHot;
  float a = part[(2 * p + (s % kHot != 0)) * d + c];
#pragma unroll 8
  for (int q = (int)p + 1; q <= q1; ++q) a += part[(int64_t)2 * q * d + c];
  dw[(int64_t)word * d + c] = from_f<T>(a * scale);
}

// dP: sums over the batch of a piece of its rows (all of them where `part` is null);
// rows of P past the length become zeros.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) embed_positions(const T* __restrict__ dout, int batch, int per, int64_t cols,
                                                       int64_t all, float* __restrict__ part, T* __restrict__ dp) {
  pdl_next();
  pdl_wait();
  using P = Pack<T, VEC>;
  const int64_t c = ((int64_t)blockIdx.x * 256 + threadIdx.x) * P::N;
  if (c >= all) return;
  P a;
  a.fill(0.f);
  if (c < cols) {
    const int b1 = min(batch, ((int)blockIdx.y + 1) * per);
#pragma unroll 8
    for (int b = blockIdx.y * per; b < b1; ++b) {
      P r;
      r.load(dout + b * cols + c);
      a.add(r);
    }
  }
  if (part) {
    if (c < cols)
#pragma unroll
      for (int i = 0; i < P::N; ++i) part[blockIdx.y * cols + c + i] = a.v[i];
    if (c >= cols && blockIdx.y == 0) a.store(dp + c);
  } else {
    a.store(dp + c);
  }
}
template <typename T>
__global__ void __launch_bounds__(256) embed_positions_join(const float* __restrict__ part, int parts, int64_t cols,
                                                            T* __restrict__ dp) {
  pdl_next();
  pdl_wait();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float a = 0.f;
#pragma unroll 8
  for (int k = 0; k < parts; ++k) a += part[k * cols + c];
  dp[c] = from_f<T>(a);
}

// ---- host side ------------------------------------------------------------------------

struct Plan {
  int n, elt, span, ctas, slices, pieces, splits, per;
  bool vec;
  int64_t cols;
  size_t order, words, start, part, pos, total;
};

bool vectors(const void* p, int64_t ld, int elt) { return ((uintptr_t)p & 15) == 0 && ld * elt % 16 == 0; }
int64_t cdiv64(int64_t a, int64_t b) { return (a + b - 1) / b; }

Plan make_plan(const llattn_embed_args& a) {
  Plan q;
  q.n = a.batch * a.length;
  q.elt = a.dtype == LLATTN_F32 ? 4 : 2;
  q.vec = vectors(a.dout, a.d, q.elt) && vectors(a.dw, a.d, q.elt) && vectors(a.dpositions, a.d, q.elt);
  const int pack = q.vec ? 16 / q.elt : 1;
  // a range of words for every SM, at least 32 of them
  q.span = (int)std::min<int64_t>(kMostWords, std::max<int64_t>(32, cdiv64(a.vocab, sm_count())));
  q.ctas = (int)cdiv64(a.vocab, q.span);
  q.slices = cdiv(a.d, kSlice * 32 * pack);
  q.pieces = q.n > kHot ? cdiv(q.n, kHot) : 0;
  q.cols = (int64_t)a.length * a.d;
  // positions: the batch in as many pieces as fill the GPU twice, of at least 16 rows
  const int64_t ctas = cdiv64(q.cols, 256 * pack);
  q.splits = (int)std::max<int64_t>(1, std::min<int64_t>(a.batch / 16, cdiv64(16 * sm_count(), ctas)));
  q.per = cdiv(a.batch, q.splits);
  q.splits = cdiv(a.batch, q.per);
  size_t off = 0;
  auto take = [&](size_t b) { size_t o = off; off += (b + 255) & ~(size_t)255; return o; };
  q.order = take(a.dw ? 4 * (size_t)q.n : 0);
  q.words = take(a.dw ? 4 * (size_t)q.n : 0);
  q.start = take(a.dw ? 4 * (size_t)(a.vocab + 1) : 0);
  q.part = take(a.dw ? 8 * (size_t)q.pieces * a.d : 0);
  q.pos = take(a.dpositions && q.splits > 1 ? 4 * (size_t)q.splits * q.cols : 0);
  q.total = off;
  return q;
}

Ids ids_of(const llattn_embed_args& a) { return Ids{a.ids, a.ids_wide, a.vocab, a.padding}; }

#define TRY(x)                          \
  do {                                  \
    cudaError_t e_ = (x);               \
    if (e_ != cudaSuccess) return e_;   \
  } while (0)

template <typename T, bool VEC>
cudaError_t fwd(const llattn_embed_args& a, cudaStream_t s) {
  const int per_row = a.d / Pack<T, VEC>::N;
  const int64_t total = (int64_t)a.batch * a.length * per_row, grid = cdiv64(total, 256);
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  return launch_pdl(embed_rows<T, VEC>, dim3((unsigned)grid), 256, 0, 1, s, ids_of(a), static_cast<const T*>(a.w), a.ldw,
                    static_cast<const T*>(a.positions), a.ldp, a.length, total, per_row, a.d, a.scale, static_cast<T*>(a.out));
}

template <typename T, bool VEC>
cudaError_t bwd(const llattn_embed_args& a, const Plan& q, cudaStream_t s) {
  char* ws = static_cast<char*>(a.workspace);
  int *order = reinterpret_cast<int*>(ws + q.order), *words = reinterpret_cast<int*>(ws + q.words);
  int* start = reinterpret_cast<int*>(ws + q.start);
  float* part = reinterpret_cast<float*>(ws + q.part);
  const T* dout = static_cast<const T*>(a.dout);
  if (a.dw) {
    const int smem = 4 * kSortWarps * q.span;
    TRY(set_smem_once(embed_sort, smem));
    TRY(launch_pdl(embed_sort, dim3(q.ctas), kSortThreads, smem, 1, s, ids_of(a), q.n, q.span, order, words, start));
    T* dw = static_cast<T*>(a.dw);
    const int64_t grid = cdiv64((a.vocab + q.pieces) * q.slices, 8);
    if (grid > INT32_MAX) return cudaErrorInvalidValue;
    TRY(launch_pdl(embed_sums<T, VEC>, dim3((unsigned)grid), 256, 0, 1, s, dout, order, words, start, a.vocab, a.d, q.slices,
                   q.pieces, a.scale, part, dw));
    if (q.pieces) {
      const int slices = cdiv(a.d, 32);
      TRY(launch_pdl(embed_join<T>, dim3((unsigned)cdiv64((int64_t)q.pieces * slices, 8)), 256, 0, 1, s, words, start, a.vocab,
                     a.d, slices, q.pieces, a.scale, part, dw));
    }
  }
  if (a.dpositions) {
    const int64_t all = (int64_t)a.position_rows * a.d;
    float* pos = q.splits > 1 ? reinterpret_cast<float*>(ws + q.pos) : nullptr;
    const int64_t grid = cdiv64(all, 256 * Pack<T, VEC>::N);
    TRY(launch_pdl(embed_positions<T, VEC>, dim3((unsigned)grid, q.splits), 256, 0, 1, s, dout, a.batch, q.per, q.cols, all,
                   pos, static_cast<T*>(a.dpositions)));
    if (pos)
      TRY(launch_pdl(embed_positions_join<T>, dim3((unsigned)cdiv64(q.cols, 256)), 256, 0, 1, s, pos, q.splits, q.cols,
                     static_cast<T*>(a.dpositions)));
  }
  return cudaSuccess;
}

}  // namespace

size_t workspace_bytes(const llattn_embed_args& a) { return std::max<size_t>(256, make_plan(a).total); }

int launches(const llattn_embed_args& a, bool backward) {
  if (!backward) return 1;
  const Plan q = make_plan(a);
  return (a.dw ? 2 + (q.pieces > 0) : 0) + (a.dpositions ? 1 + (q.splits > 1) : 0);
}

cudaError_t launch_fwd(const llattn_embed_args& a, cudaStream_t s) {
  const int elt = a.dtype == LLATTN_F32 ? 4 : 2;
  const bool vec = vectors(a.w, a.ldw, elt) && vectors(a.out, a.d, elt) && (!a.positions || vectors(a.positions, a.ldp, elt));
  if (elt == 4) return vec ? fwd<float, true>(a, s) : fwd<float, false>(a, s);
  return vec ? fwd<bf16, true>(a, s) : fwd<bf16, false>(a, s);
}

cudaError_t launch_bwd(const llattn_embed_args& a, cudaStream_t s) {
  const Plan q = make_plan(a);
  if (q.elt == 4) return q.vec ? bwd<float, true>(a, q, s) : bwd<float, false>(a, q, s);
  return q.vec ? bwd<bf16, true>(a, q, s) : bwd<bf16, false>(a, q, s);
}

}  // namespace embed
}  // namespace llattn
