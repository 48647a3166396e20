// Token embedding with its positions, and its gradients:
//   out[b, t] = scale W[ids[b, t]] + P[t]
//   dW[v] = scale sum_{(b, t): ids[b, t] = v} dout[b, t],  dP[t] = sum_b dout[b, t]
//
// dW goes by the tokens sorted by word. The sort runs beside dP's sums, in one
// launch with them: each of 128 CTAs owns every 128th word (neighbours in a
// vocabulary are of like frequency) and reads all ids for itself, from the L2, so
// that no CTA waits for another: it counts its words' tokens and those of the CTAs
// before it, then writes its tokens, word by word and in their order, to where these
// start. Rows are then summed in that order, whatever the launch: a warp per word and
// 1 KB of columns, zeros for a word without tokens. A word of more than kHot tokens
// is cut at the multiples of kHot of the sorted order; these pieces go first, their sums
// through the workspace, and are added in order, 32 and 32: no sum is one long chain. No atomics on values: the same bits
// every run. Where words and tokens are few (`small`), a CTA a word picks its
// tokens out of the ids itself, and one launch does it all.
//
// Bound by memory: dout is read twice with positions (once in each order), W's rows once.
// 16 x 2048 ids of 32000 words of 1536 fp32: rows out 50 us (237 MB moved), sort and dP 39 us (202 MB of dout
// at 5.2 TB/s), sums 65 (399 MB moved at 6.1), all 172 with the join of the frequent words beside the sums' end; a
// sort by another launch and a dP after it: 235. 8197 tokens of 1408 bf16, a fifth of them
// padding: 14, 13, 30 and 7 us.
#include <math.h>

#include <algorithm>
#include <type_traits>

#include "embed.cuh"
#include "pdl.cuh"

namespace llattn {
namespace embed {
namespace {

// (with pieces of 64 tokens, 2 KB of columns and two rows at a time, 8197 tokens of 1408 bf16 took 84 us
// for their sums, the longest words' 25 us a warp among them)
constexpr int kHot = 32;
constexpr int kSortThreads = 1024, kSortWarps = kSortThreads / 32;
constexpr int kSorters = 128, kSortBits = 7;  // sorting CTAs a round: word v is the (v >> 7)-th of CTA v % 128
constexpr int kMostBits = 10;                 // at most 1024 words a sorting CTA and round: 32 counters each, 128 KB
constexpr int kSlice = 2, kRows = 4;          // 16-byte vectors a lane takes of a row, and rows, at a time
constexpr int kWords = 4;                     // words of a summing warp
constexpr int kHeld = 40960;                  // tokens whose places the sort keeps, 80 KB

struct Ids {
  const void* p;
  int wide;  // int64, else int32
  int vocab, padding;
  // the i-th id, -1 where there is no such word
  __device__ __forceinline__ int at(int64_t i) const {
    int id, high = 0;
    if (wide) {
      const int2 v = static_cast<const int2*>(p)[i];
      id = v.x;
      high = v.y;
    } else {
      id = static_cast<const int*>(p)[i];
    }
    return high == 0 && (unsigned)id < (unsigned)vocab ? id : -1;
  }
  __device__ __forceinline__ int counted(int64_t i) const {  // -1 for the padding too
    const int id = at(i);
    return id == padding ? -1 : id;
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
  using Raw = std::conditional_t<VEC, uint4, T>;  // as it is in memory
  __device__ __forceinline__ void add(const Raw& p, const Raw& q, const Raw& r, const Raw& s) {
    const T *a = reinterpret_cast<const T*>(&p), *b = reinterpret_cast<const T*>(&q), *c = reinterpret_cast<const T*>(&r),
            *d = reinterpret_cast<const T*>(&s);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] += (to_f<T>(a[i]) + to_f<T>(b[i])) + (to_f<T>(c[i]) + to_f<T>(d[i]));
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

// A warp per token and 4 packs a lane of its columns.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) embed_rows(Ids ids, const T* w, int64_t ldw, const T* pos,
                                                  int64_t ldp, int length, int64_t tokens, int slices, int d, float scale,
                                                  T* out) {
  pdl_next();
  pdl_wait();
  using P = Pack<T, VEC>;
  constexpr int U = 4;
  const int lane = threadIdx.x % 32;
  const int64_t i = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t n = i <= INT32_MAX ? (int64_t)((uint32_t)i / (uint32_t)slices) : i / slices;
  if (n >= tokens) return;
  const int c0 = ((int)(i - n * slices) * U * 32 + lane) * P::N;
  const int id = ids.at(n);
  const T* src = w + (int64_t)max(id, 0) * ldw;
  P r[U], q[U];
#pragma unroll
  for (int k = 0; k < U; ++k)
    if (c0 + k * 32 * P::N < d) r[k].load(src + c0 + k * 32 * P::N);
  if (pos) {
    const T* at = pos + (int64_t)(n <= INT32_MAX ? (uint32_t)n % (uint32_t)length : n % length) * ldp;
#pragma unroll
    for (int k = 0; k < U; ++k)
      if (c0 + k * 32 * P::N < d) q[k].load(at + c0 + k * 32 * P::N);
  }
#pragma unroll
  for (int k = 0; k < U; ++k) {
    if (c0 + k * 32 * P::N >= d) break;
#pragma unroll
    for (int e = 0; e < P::N; ++e) {
      const float v = pos ? fmaf(r[k].v[e], scale, q[k].v[e]) : r[k].v[e] * scale;
      r[k].v[e] = id < 0 ? __int_as_float(0x7fc00000) : v;  // no such word
    }
    r[k].store(out + n * d + c0 + k * 32 * P::N);
  }
}

// ---- dP, beside the sort -------------------------------------------------------------

// Sums over a piece of the batch (all of it where `part` is null); rows of P past the
// length become zeros.
template <typename T>
struct Positions {
  const T* dout;
  int batch, per;
  int64_t cols, all;  // length d, position_rows d
  float* part;
  T* dp;
};
template <typename T, bool VEC>
__device__ __forceinline__ void position_sums(const Positions<T>& q, int64_t thread, int split) {
  using P = Pack<T, VEC>;
  const int64_t c = thread * P::N;
  if (c >= q.all) return;
  P a;
  a.fill(0.f);
  if (c < q.cols) {
    const int b1 = min(q.batch, (split + 1) * q.per);
#pragma unroll 4
    for (int b = split * q.per; b < b1; ++b) {
      P r;
      r.load(q.dout + b * q.cols + c);
      a.add(r);
    }
  }
  if (!q.part || c >= q.cols) {
    if (split == 0 || !q.part) a.store(q.dp + c);
  } else {
#pragma unroll
    for (int i = 0; i < P::N; ++i) q.part[split * q.cols + c + i] = a.v[i];
  }
}
template <typename T>
__global__ void __launch_bounds__(256) embed_positions_join(const float* part, int parts, int64_t cols,
                                                            T* dp) {
  pdl_next();
  pdl_wait();
  const int64_t c = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (c >= cols) return;
  float a = 0.f;
#pragma unroll 8
  for (int k = 0; k < parts; ++k) a += part[k * cols + c];
  dp[c] = from_f<T>(a);
}

// ---- the sort -----------------------------------------------------------------------

// A word's slot: those of a sorting CTA and round in a row, so that its tokens are
// consecutive. start[slot]: its tokens' first place in the sorted order, start[slot + 1]:
// the place behind them.
__device__ __forceinline__ int slot_of(int v, int bits) {  // span = 1 << bits
  const int k = v >> kSortBits;
  return ((((k >> bits) << kSortBits) + (v & (kSorters - 1))) << bits) + (k & ((1 << bits) - 1));
}

// CTA: words v with v % 128 = CTA % 128 and (v >> 7) / span = its round. order: the counted
// tokens by slot, then by index; words: their words; start [rounds 128 span + 1].
// held: the tokens' places stay in shared memory for the second pass, n of them; otherwise each
// pass reads the ids. (Places in registers took a loop unrolled 32 times: 11 us of fetching it.)
__device__ __forceinline__ void sort_tokens(const Ids& ids, int n, int bits, bool held, int cta, int ctas,
                                            int* order, int* words, int* start) {
  extern __shared__ int counts[];  // [kSortWarps][span], then the places
  __shared__ int sums[kSortWarps];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int span = 1 << bits, round = cta >> kSortBits, low = cta & (kSorters - 1);
  const int per = cdiv(cdiv(n, kSortWarps), 256) * 256, i0 = min(n, warp * per), i1 = min(n, i0 + per);
  int* my = counts + warp * span;
  int16_t* places = reinterpret_cast<int16_t*>(counts + kSortWarps * span) + warp * (held ? per : 256);
  for (int i = threadIdx.x; i < kSortWarps * span; i += kSortThreads) counts[i] = 0;
  __syncthreads();
  // 256 ids from i on -> their places: r of this CTA's words, -1: another's, -2: of a CTA before this one
  auto place = [&](int i, auto body) {
    int id[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) id[k] = i + 32 * k + lane < i1 ? ids.counted(i + 32 * k + lane) : -1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const int q = (id[k] >> kSortBits) - round * span, other = id[k] & (kSorters - 1);
      const bool here = (unsigned)q < (unsigned)span;
      const int r = id[k] < 0 ? -1 : q < 0 || (here && other < low) ? -2 : here && other == low ? q : -1;
      places[(held ? i - i0 : 0) + 32 * k + lane] = (int16_t)r;
      body(r);
    }
  };
  int below = 0;
  for (int i = i0; i < i1; i += 256)
    place(i, [&](int r) {
      below += r == -2;
      if (r >= 0) atomicAdd(my + r, 1);
    });
  below = __reduce_add_sync(0xffffffffu, below);
  if (lane == 0) sums[warp] = below;
  __syncthreads();
  // counters -> places in the order: over the warps of a word, then over the words
  int base = 0;
#pragma unroll
  for (int i = 0; i < kSortWarps; ++i) base += sums[i];
  __syncthreads();
  int* first = start + (int64_t)cta * span;
  const int r = threadIdx.x;  // (span <= kSortThreads)
  int all = 0;
  if (r < span) {
#pragma unroll 8
    for (int k = 0; k < kSortWarps; ++k) all += counts[k * span + r];
  }
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
  if (r < span) {
    first[r] = at;
#pragma unroll 8
    for (int k = 0; k < kSortWarps; ++k) {
      const int c = counts[k * span + r];
      counts[k * span + r] = at;
      at += c;
    }
  }
  if (threadIdx.x == 0 && cta == ctas - 1) first[span] = base;
  __syncthreads();
  for (int i = i0; i < i1; i += 256) {
    if (!held) {
      __syncwarp();
      place(i, [](int) {});
    }
    __syncwarp();
#pragma unroll 1
    for (int k = 0; k < 8; ++k) {
      const int r = places[(held ? i - i0 : 0) + 32 * k + lane];
      const unsigned some = __ballot_sync(0xffffffffu, r >= 0);
      if (r >= 0) {
        const unsigned same = __match_any_sync(some, r);
        const int at = my[r] + __popc(same & ((1u << lane) - 1u));
        __syncwarp(some);
        order[at] = i + 32 * k + lane;
        words[at] = ((round * span + r) << kSortBits) + low;
        if ((same >> lane) == 1u) my[r] = at + 1;  // the last of them
      }
      __syncwarp();
    }
  }
}

// The first `sorters` CTAs sort, the others sum dP.
template <typename T, bool VEC>
__global__ void __launch_bounds__(kSortThreads, 2) embed_sort(Ids ids, int n, int bits, int held, int sorters,
                                                           int* order, int* words,
                                                           int* start, Positions<T> q, int per_split) {
  pdl_next();
  pdl_wait();
  if ((int)blockIdx.x < sorters) {
    sort_tokens(ids, n, bits, held, blockIdx.x, sorters, order, words, start);
    return;
  }
  const int b = blockIdx.x - sorters, split = b / per_split;
  position_sums<T, VEC>(q, (int64_t)(b - split * per_split) * kSortThreads + threadIdx.x, split);
}

// ---- dW -----------------------------------------------------------------------------

// Columns [c0, c0 + 32 kSlice packs) of rows added to a, the j-th of up to 32 being row index(j) of dout.
template <typename T, bool VEC, typename Index>
__device__ __forceinline__ void add_rows(Pack<T, VEC> (&a)[kSlice], const T* dout, int d, int c0, int m, Index index) {
  using P = Pack<T, VEC>;
  const int lane = threadIdx.x % 32;
#pragma unroll 1
  for (int j0 = 0; j0 < m; j0 += kRows) {
    typename P::Raw r[kRows][kSlice];
#pragma unroll
    for (int j = 0; j < kRows; ++j) {
      const T* row = dout + (int64_t)index(min(j0 + j, m - 1)) * d;
#pragma unroll
      for (int k = 0; k < kSlice; ++k) {
        const int c = c0 + (k * 32 + lane) * P::N;
        r[j][k] = typename P::Raw{};
        if (j0 + j < m && c < d) r[j][k] = *reinterpret_cast<const typename P::Raw*>(row + c);
      }
    }
    static_assert(kRows == 4, "rows in pairs, so that m of them are m / 4 additions in a row");
#pragma unroll
    for (int k = 0; k < kSlice; ++k) a[k].add(r[0][k], r[1][k], r[2][k], r[3][k]);
  }
}

// Warps [0, pieces slices): the pieces of words of more than kHot tokens: slot 2 p of `part` holds what
// interval p of the sorted order has of its first word, slot 2 p + 1 what it has of its last
// one, where that is another. The warps after write the other words, kWords each, a quarter of
// the vocabulary apart: most words have no token and cost little but the wait for their count.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) embed_sums(const T* dout, const int* order,
                                                  const int* words, const int* start, int vocab,
                                                  int bits, int total_at, int d, int slices, int pieces, float scale,
                                                  float* part, T* dw) {
  pdl_next();
  pdl_wait();
  using P = Pack<T, VEC>;
  const int lane = threadIdx.x % 32;
  const int64_t w = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int u = w <= INT32_MAX ? (int)((uint32_t)w / (uint32_t)slices) : (int)(w / slices);
  const int c0 = (int)(w - (int64_t)u * slices) * (kSlice * 32 * P::N);
  P a[kSlice];
  if (u >= pieces) {
    const int apart = cdiv(vocab, kWords), first = u - pieces;
    if (first >= apart) return;
    // lane 2 k: where word k's tokens start, lane 2 k + 1: where they end
    const int mine = first + lane / 2 * apart;
    const int bound = lane < 2 * kWords && mine < vocab ? start[slot_of(mine, bits) + lane % 2] : 0;
    int s[kWords], n[kWords], row[kWords];
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      s[k] = __shfl_sync(0xffffffffu, bound, 2 * k);
      n[k] = __shfl_sync(0xffffffffu, bound, 2 * k + 1) - s[k];
      row[k] = lane < n[k] && n[k] <= kHot ? order[s[k] + lane] : 0;
    }
#pragma unroll
    for (int k = 0; k < kWords; ++k) {
      const int v = first + k * apart;
      if (v >= vocab || n[k] > kHot) continue;  // (warp-uniform)
#pragma unroll
      for (int i = 0; i < kSlice; ++i) a[i].fill(0.f);
      add_rows<T, VEC>(a, dout, d, c0, n[k], [&](int j) { return __shfl_sync(0xffffffffu, row[k], j); });
#pragma unroll
      for (int i = 0; i < kSlice; ++i) {
        const int c = c0 + (i * 32 + lane) * P::N;
        a[i].times(scale);
        if (c < d) a[i].store(dw + (int64_t)v * d + c);
      }
    }
    return;
  }
  const int64_t p = u;
  const int total = start[total_at];
  if (p * kHot >= total) return;
  const int lo = (int)p * kHot, hi = min(lo + kHot, total);
  for (int last = 0; last < 2; ++last) {
    const int word = words[last ? hi - 1 : lo];
    if (last && word == words[lo]) break;
    const int* at = start + slot_of(word, bits);
    const int s = max(at[0], lo), e = min(at[1], hi);
    if (at[1] - at[0] <= kHot) continue;
    const int row = s + lane < e ? order[s + lane] : 0;
#pragma unroll
    for (int i = 0; i < kSlice; ++i) a[i].fill(0.f);
    add_rows<T, VEC>(a, dout, d, c0, e - s, [&](int j) { return __shfl_sync(0xffffffffu, row, j); });
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
__global__ void __launch_bounds__(256) embed_join(const int* words, const int* start, int bits,
                                                  int total_at, int d, int slices, int pieces, float scale,
                                                  const float* part, T* dw) {
  pdl_next();
  pdl_wait();
  const int64_t w = (int64_t)blockIdx.x * 8 + threadIdx.x / 32;
  const int64_t p = w / slices;
  const int c = (int)(w - p * slices) * 32 + threadIdx.x % 32;
  const int total = start[total_at];
  if (p >= pieces || p * kHot >= total) return;
  const int word = words[min((int)p * kHot + kHot, total) - 1];
  const int* at = start + slot_of(word, bits);
  const int s = at[0], e = at[1];
  if (e - s <= kHot || s / kHot != p || c >= d) return;
  const int q1 = (e - 1) / kHot;
  float a = part[(2 * p + (s % kHot != 0)) * d + c];
  for (int q = (int)p + 1; q <= q1; q += 32) {  // 32 loads at a time: their latency is all there is
    float x[32];
#pragma unroll
    for (int k = 0; k < 32; ++k) x[k] = q + k <= q1 ? part[(int64_t)2 * (q + k) * d + c] : 0.f;
#pragma unroll
    for (int k = 1; k < 32; ++k) x[0] += x[k];
    a += x[0];  // (c tokens are 10, 31 and c / 1024 additions in a row)
  }
  dw[(int64_t)word * d + c] = from_f<T>(a * scale);
}

// Few words and tokens: a CTA per word and 1 KB of columns, whose warps each pick the word's tokens out of
// an eighth of the ids; then the CTAs of dP.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) embed_small(Ids ids, int n, const T* dout, int d, int slices, float scale,
                                                   T* dw, int word_ctas, Positions<T> q, int per_split) {
  pdl_next();
  pdl_wait();
  if ((int)blockIdx.x >= word_ctas) {
    const int b = blockIdx.x - word_ctas, split = b / per_split;
    position_sums<T, VEC>(q, (int64_t)(b - split * per_split) * 256 + threadIdx.x, split);
    return;
  }
  using P = Pack<T, VEC>;
  __shared__ float red[8][32][kSlice * P::N];
  __shared__ int hit[8][32];
  const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
  const int v = blockIdx.x / slices, c0 = (blockIdx.x - v * slices) * (kSlice * 32 * P::N);
  const int per = cdiv(cdiv(n, 8), 32) * 32, i0 = min(n, warp * per), i1 = min(n, i0 + per);
  P a[kSlice];
#pragma unroll
  for (int k = 0; k < kSlice; ++k) a[k].fill(0.f);
  for (int i = i0; i < i1; i += 256) {
    int id[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) id[k] = i + 32 * k + lane < i1 ? ids.counted(i + 32 * k + lane) : -1;
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned some = __ballot_sync(0xffffffffu, id[k] == v);
      if (!some) continue;
      if (id[k] == v) hit[warp][__popc(some & ((1u << lane) - 1u))] = i + 32 * k + lane;
      __syncwarp();
      add_rows<T, VEC>(a, dout, d, c0, __popc(some), [&](int j) { return hit[warp][j]; });
      __syncwarp();
    }
  }
#pragma unroll
  for (int k = 0; k < kSlice; ++k)
#pragma unroll
    for (int e = 0; e < P::N; ++e) red[warp][lane][k * P::N + e] = a[k].v[e];
  __syncthreads();
  if (warp) return;
#pragma unroll
  for (int k = 0; k < kSlice; ++k) {
#pragma unroll
    for (int e = 0; e < P::N; ++e) {
      float x = red[0][lane][k * P::N + e];
#pragma unroll
      for (int o = 1; o < 8; ++o) x += red[o][lane][k * P::N + e];
      a[k].v[e] = x * scale;
    }
    const int c = c0 + (k * 32 + lane) * P::N;
    if (c < d) a[k].store(dw + (int64_t)v * d + c);
  }
}

// ---- host side ------------------------------------------------------------------------

struct Plan {
  int n, elt, bits, sorters, total_at, slices, pieces, splits, per;
  bool vec, small, held;
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
  q.held = q.n <= kHeld;
  const int share = (int)cdiv64(a.vocab, kSorters);  // words of a sorting CTA, in rounds
  q.bits = 0;
  while (q.bits < kMostBits && 1 << q.bits < share) ++q.bits;
  q.sorters = cdiv(share, 1 << q.bits) * kSorters;
  q.total_at = q.sorters << q.bits;
  q.slices = cdiv(a.d, kSlice * 32 * pack);
  q.pieces = q.n > kHot ? cdiv(q.n, kHot) : 0;
  // One launch while its CTAs, 1 KB of a word's columns each, take less time than the launches of the sort (2048 tokens
  // of 128 fp32: 9.8 us for 18.8 with 2048 CTAs, 15.1 for 19.0 with 4096, 25.9 for 18.9 with 8192; 256 tokens 8.9 for
  // 13.7, 14.2 for 14.1, 24.9 for 14.0). A CTA of bf16 adds twice the columns (2048 tokens: 12.0 for 19.4 with 1024, 15.2
  // for 19.2 with 2048, 25.4 for 19.5 with 4096; 256: 10.1 for 14.7, 14.5 for 14.2, 24.8 for 15.0). Past 2048 tokens
  // each CTA's reading of all ids tells (4096 of 512 columns, 64 words: 26.6 for 26.7).
  q.small = q.n <= 2048 && a.vocab * q.slices <= (q.elt == 4 ? 4096 : 2048);
  q.cols = (int64_t)a.length * a.d;
  // positions: the batch in as many pieces as fill the GPU, of at least 16 rows
  const int64_t ctas = cdiv64(q.cols, 1024 * pack);
  q.splits = (int)std::max<int64_t>(1, std::min<int64_t>(a.batch / 16, cdiv64(4 * sm_count(), ctas)));
  q.per = cdiv(a.batch, q.splits);
  q.splits = cdiv(a.batch, q.per);
  size_t off = 0;
  auto take = [&](size_t b) { size_t o = off; off += (b + 255) & ~(size_t)255; return o; };
  const bool sorted = a.dw && !q.small;
  q.order = take(sorted ? 4 * (size_t)q.n : 0);
  q.words = take(sorted ? 4 * (size_t)q.n : 0);
  q.start = take(sorted ? 4 * (size_t)(q.total_at + 1) : 0);
  q.part = take(sorted ? 8 * (size_t)q.pieces * a.d : 0);
  q.pos = take(a.dpositions && q.splits > 1 ? 4 * (size_t)q.splits * q.cols : 0);
  q.total = off;
  return q;
}

Ids ids_of(const llattn_embed_args& a) { return Ids{a.ids, a.ids_wide, (int)a.vocab, (int)std::max<int64_t>(a.padding, -1)}; }

#define TRY(x)                          \
  do {                                  \
    cudaError_t e_ = (x);               \
    if (e_ != cudaSuccess) return e_;   \
  } while (0)

template <typename T, bool VEC>
cudaError_t fwd(const llattn_embed_args& a, cudaStream_t s) {
  const int slices = cdiv(a.d, 4 * 32 * Pack<T, VEC>::N);
  const int64_t tokens = (int64_t)a.batch * a.length, grid = cdiv64(tokens * slices, 8);
  if (grid > INT32_MAX) return cudaErrorInvalidValue;
  return launch_pdl(embed_rows<T, VEC>, dim3((unsigned)grid), 256, 0, 1, s, ids_of(a), static_cast<const T*>(a.w), a.ldw,
                    static_cast<const T*>(a.positions), a.ldp, a.length, tokens, slices, a.d, a.scale, static_cast<T*>(a.out));
}

template <typename T, bool VEC>
cudaError_t bwd(const llattn_embed_args& a, const Plan& q, cudaStream_t s) {
  char* ws = static_cast<char*>(a.workspace);
  int *order = reinterpret_cast<int*>(ws + q.order), *words = reinterpret_cast<int*>(ws + q.words);
  int* start = reinterpret_cast<int*>(ws + q.start);
  float* part = reinterpret_cast<float*>(ws + q.part);
  const T* dout = static_cast<const T*>(a.dout);
  T* dw = static_cast<T*>(a.dw);
  const int64_t all = a.dpositions ? (int64_t)a.position_rows * a.d : 0;
  float* pos = q.splits > 1 ? reinterpret_cast<float*>(ws + q.pos) : nullptr;
  const Positions<T> pq{dout, a.batch, q.per, q.cols, all, pos, static_cast<T*>(a.dpositions)};
  const bool small = !dw || q.small;
  const int threads = small ? 256 : kSortThreads;
  const int64_t per_split = cdiv64(all, (int64_t)threads * Pack<T, VEC>::N), pos_ctas = per_split * q.splits;
  const int64_t word_ctas = !dw ? 0 : small ? a.vocab * q.slices : q.sorters;
  if (pos_ctas + word_ctas > INT32_MAX) return cudaErrorInvalidValue;
  const dim3 grid((unsigned)(word_ctas + pos_ctas));
  if (small) {
    TRY(launch_pdl(embed_small<T, VEC>, grid, threads, 0, 1, s, ids_of(a), q.n, dout, a.d, q.slices, a.scale, dw, (int)word_ctas, pq,
                   (int)per_split));
  } else {
    const int smem = (4 * kSortWarps << q.bits) + 2 * kSortWarps * (q.held ? cdiv(cdiv(q.n, kSortWarps), 256) * 256 : 256);
    TRY(set_smem_once(embed_sort<T, VEC>, smem));
    TRY(launch_pdl(embed_sort<T, VEC>, grid, threads, smem, 1, s, ids_of(a), q.n, q.bits, q.held, q.sorters, order, words, start, pq,
                   (int)per_split));
    const int64_t sums = cdiv64((cdiv64(a.vocab, kWords) + q.pieces) * q.slices, 8);
    if (sums > INT32_MAX) return cudaErrorInvalidValue;
    TRY(launch_pdl(embed_sums<T, VEC>, dim3((unsigned)sums), 256, 0, 1, s, dout, order, words, start, (int)a.vocab, q.bits,
                   q.total_at, a.d, q.slices, q.pieces, a.scale, part, dw));
    if (q.pieces) {
      const int slices = cdiv(a.d, 32);
      TRY(launch_pdl(embed_join<T>, dim3((unsigned)cdiv64((int64_t)q.pieces * slices, 8)), 256, 0, 1, s, words, start, q.bits,
                     q.total_at, a.d, slices, q.pieces, a.scale, part, dw));
    }
  }
  if (a.dpositions && pos)
    TRY(launch_pdl(embed_positions_join<T>, dim3((unsigned)cdiv64(q.cols, 256)), 256, 0, 1, s, pos, q.splits, q.cols,
                   static_cast<T*>(a.dpositions)));
  return cudaSuccess;
}

}  // namespace

size_t workspace_bytes(const llattn_embed_args& a) { return std::max<size_t>(256, make_plan(a).total); }

int launches(const llattn_embed_args& a, bool backward) {
  if (!backward) return 1;
  const Plan q = make_plan(a);
  return (!a.dw || q.small ? 1 : 2 + (q.pieces > 0)) + (a.dpositions && q.splits > 1);
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
