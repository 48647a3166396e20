// Norm over a list of tensors, and their scaling to at most a given norm:
//   norm = sqrt(sum_i |t_i|^2) or max_i |t_i|,  t_i *= min(1, max_norm / (norm + 1e-6))
//
// Two launches whatever the number of tensors (up to kTensors; that many more per
// pair after): the list travels in the kernel's parameters, every tensor is cut
// into chunks of 16 KB at 16-byte boundaries, and each CTA takes a run of consecutive
// chunks, so that finding the first one's tensor is all the searching there is. The
// first kernel leaves a sum per CTA; every CTA of the second one adds those up in the
// same order, which costs less than a counter and a wait, and scales its run from
// the back: what the first kernel read last is still in the L2. Nothing is
// written where the factor is 1.
//
// Bound by memory: 434 tensors of 590 M fp32 elements (2.36 GB): the norm 364 us (6.5 TB/s), norm and scaling 1165
// (7.1 GB at 6.1 TB/s). 200 of 31 M: 33 and 77 us; 39 of 0.36 M: 6 us on the GPU, 15 on the host, where 0.5 us
// a tensor go.
//
// Squares are summed in fp32 over a 16-byte vector and in fp64 from there on; a
// vector whose sum leaves fp32's comfortable range is squared in fp64.
#include <math.h>

#include <algorithm>

#include "clip.cuh"
#include "pdl.cuh"

namespace llattn {
namespace clip {
namespace {

// entries of 24 bytes in the parameters, which hold 32 KB; a short list takes the short form (the
// parameters are copied with every launch)
constexpr int kTensors = 1300, kShort = 96;
constexpr int kThreads = 256, kUnroll = 4, kChunk = kThreads * kUnroll * 16;
constexpr int kMaxGrid = 1184;

struct Entry {
  char* p;
  int64_t bytes;
  int chunk;  // its first chunk
  int bf16;
};
template <int CAP>
struct Table {
  int n, chunks;
  Entry e[CAP];
};
static_assert(sizeof(Table<kTensors>) <= 32000, "kernel parameters");

__device__ __forceinline__ float element(const char* p, int bf) {
  return bf ? __bfloat162float(*reinterpret_cast<const bf16*>(p)) : *reinterpret_cast<const float*>(p);
}
__device__ __forceinline__ void unpack(const uint4& u, int bf, float (&v)[8], int& n) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
  n = bf ? 8 : 4;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (bf) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    } else {
      v[i] = __uint_as_float(w[i]);
    }
  }
}

// A CTA's run of chunks [first, last), and the table's entry of a chunk.
template <int CAP>
__device__ __forceinline__ int2 run_of(const Table<CAP>& t) {
  return make_int2((int)((int64_t)t.chunks * blockIdx.x / gridDim.x), (int)((int64_t)t.chunks * (blockIdx.x + 1) / gridDim.x));
}
template <int CAP>
__device__ __forceinline__ int entry_of(const Table<CAP>& t, int chunk) {
  int lo = 0, hi = t.n - 1;  // the last entry that starts at or before chunk
  while (lo < hi) {
    const int mid = (lo + hi + 1) / 2;
    if (t.e[mid].chunk <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

// A thread's 16-byte vectors of a chunk: whole(v, inside) for all of them, `inside` a
// bit for each that lies in the tensor; part(address) for each element of those that
// lie in it partly (a tensor's first and last at most).
template <typename Whole, typename Part>
__device__ __forceinline__ void walk(const Entry& e, int k, Whole whole, Part part) {
  char* base = reinterpret_cast<char*>(reinterpret_cast<uintptr_t>(e.p) & ~uintptr_t(15)) + (int64_t)k * kChunk;
  char* end = e.p + e.bytes;
  char* v = base + threadIdx.x * 16;
  if (base >= e.p && base + kChunk <= end) {
    whole(v, (1u << kUnroll) - 1u);
    return;
  }
  uint32_t inside = 0;
#pragma unroll
  for (int i = 0; i < kUnroll; ++i) {
    const char* q = v + i * kThreads * 16;
    inside |= (q >= e.p && q + 16 <= end ? 1u : 0u) << i;
  }
  whole(v, inside);
#pragma unroll 1
  for (int i = 0; i < kUnroll; ++i) {
    char* w = v + i * kThreads * 16;
    if ((inside >> i & 1u) || w + 16 <= e.p || w >= end) continue;
    for (char* q = w; q < w + 16; q += e.bf16 ? 2 : 4)
      if (q >= e.p && q < end) part(q);
  }
}
__device__ __forceinline__ void read(uint4 (&u)[kUnroll], const char* v, uint32_t inside) {
#pragma unroll
  for (int i = 0; i < kUnroll; ++i)
    u[i] = inside >> i & 1u ? *reinterpret_cast<const uint4*>(v + i * kThreads * 16) : make_uint4(0, 0, 0, 0);
}

struct Squares {
  using Acc = double;
  static __device__ __forceinline__ Acc zero() { return 0.0; }
  static __device__ __forceinline__ void add(Acc& a, float v) { a += (double)v * (double)v; }
  static __device__ __forceinline__ void add(Acc& a, const uint4& u, int bf) {
    float v[8], s = 0.f;
    int n;
    unpack(u, bf, v, n);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) s = fmaf(v[i], v[i], s);
    if (s > 0x1p-90f && s < 0x1p120f) {
      a += (double)s;
    } else if ((u.x | u.y | u.z | u.w) & (bf ? 0x7fff7fffu : 0x7fffffffu)) {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (i < n) add(a, v[i]);
    }
  }
  static __device__ __forceinline__ Acc join(Acc a, Acc b) { return a + b; }
  static __device__ __forceinline__ double norm(Acc a) { return sqrt(a); }
};
// magnitudes as integers: a NaN's is above infinity's
struct Largest {
  using Acc = double;  // (as Squares's; the low word's bits are the magnitude)
  static __device__ __forceinline__ Acc zero() { return __longlong_as_double(0); }
  static __device__ __forceinline__ void add(Acc& a, float v) {
    a = join(a, __longlong_as_double((long long)(__float_as_uint(v) & 0x7fffffffu)));
  }
  static __device__ __forceinline__ void add(Acc& a, const uint4& u, int bf) {
    float v[8];
    int n;
    unpack(u, bf, v, n);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (i < n) add(a, v[i]);
  }
  static __device__ __forceinline__ Acc join(Acc a, Acc b) {
    return __longlong_as_double(max(__double_as_longlong(a), __double_as_longlong(b)));
  }
  static __device__ __forceinline__ double norm(Acc a) {
    return (double)__uint_as_float((unsigned)__double_as_longlong(a));
  }
};

template <typename Op>
__device__ __forceinline__ double block_join(double a, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) a = Op::join(a, __shfl_xor_sync(0xffffffffu, a, o));
  if (threadIdx.x % 32 == 0) red[threadIdx.x / 32] = a;
  __syncthreads();
  a = red[0];
#pragma unroll
  for (int i = 1; i < kThreads / 32; ++i) a = Op::join(a, red[i]);
  return a;
}

template <typename Op, int CAP>
__global__ void __launch_bounds__(kThreads) norm_kernel(const __grid_constant__ Table<CAP> t, double* part) {
  __shared__ double red[kThreads / 32];
  const int2 run = run_of(t);
  int e = entry_of(t, run.x);
  pdl_next();
  pdl_wait();
  double a = Op::zero();
  for (int c = run.x; c < run.y; ++c) {
    while (e + 1 < t.n && t.e[e + 1].chunk <= c) ++e;
    const int bf = t.e[e].bf16;
    walk(
        t.e[e], c - t.e[e].chunk,
        [&](const char* v, uint32_t inside) {
          uint4 u[kUnroll];
          read(u, v, inside);
#pragma unroll
          for (int i = 0; i < kUnroll; ++i) Op::add(a, u[i], bf);
        },
        [&](const char* q) { Op::add(a, element(q, bf)); });
  }
  a = block_join<Op>(a, red);
  if (threadIdx.x == 0) part[blockIdx.x] = a;
}

// n_part: all batches' sums. scale: 0 writes the norm alone.
template <typename Op, int CAP>
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ Table<CAP> t, const double* part,
                                                        int n_part, double max_norm, int scale, float* norm) {
  __shared__ double red[kThreads / 32];
  const int2 run = run_of(t);
  int e = scale && run.y > run.x ? entry_of(t, run.y - 1) : 0;
  pdl_next();
  pdl_wait();
  double a = Op::zero();
  for (int i = threadIdx.x; i < n_part; i += kThreads) a = Op::join(a, part[i]);
  const double total = Op::norm(block_join<Op>(a, red));
  if (norm && blockIdx.x == 0 && threadIdx.x == 0) *norm = (float)total;
  if (!scale) return;
  // by the norm that the call returns where that is infinite: a finite one above fp32's range counts as infinity
  const double c = max_norm / ((isinf((float)total) ? (double)INFINITY : total) + 1e-6);
  const float f = c > 1.0 ? 1.f : (float)c;  // (a NaN stays one)
  if (f == 1.f) return;
  for (int k = run.y - 1; k >= run.x; --k) {
    while (t.e[e].chunk > k) --e;
    const int bf = t.e[e].bf16;
    walk(
        t.e[e], k - t.e[e].chunk,
        [&](char* v, uint32_t inside) {
          uint4 u[kUnroll];
          read(u, v, inside);
#pragma unroll
          for (int i = 0; i < kUnroll; ++i) {
            uint32_t* w = reinterpret_cast<uint32_t*>(&u[i]);
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              if (bf) {
                __nv_bfloat162 h = __floats2bfloat162_rn(__uint_as_float(w[q] << 16) * f, __uint_as_float(w[q] & 0xffff0000u) * f);
                w[q] = *reinterpret_cast<uint32_t*>(&h);
              } else {
                w[q] = __float_as_uint(__uint_as_float(w[q]) * f);
              }
            }
            if (inside >> i & 1u) *reinterpret_cast<uint4*>(v + i * kThreads * 16) = u[i];
          }
        },
        [&](char* q) {
          if (bf)
            *reinterpret_cast<bf16*>(q) = __float2bfloat16_rn(element(q, 1) * f);
          else
            *reinterpret_cast<float*>(q) *= f;
        });
  }
}

int chunks_of(const llattn_clip_args& a, int i) {
  const int64_t bytes = a.sizes[i] * (a.dtypes[i] == LLATTN_BF16 ? 2 : 4);
  return (int)(((int64_t)((uintptr_t)a.tensors[i] & 15) + bytes + kChunk - 1) / kChunk);
}

// One batch of the list: take(tensor, its first chunk, chunks) for those from i on that hold something, up to
// `most`. Returns where the next batch starts: behind the empty tensors that follow, so that every batch but an
// empty list's holds something, and all that walk the list count the same ones.
template <typename Take>
int batch(const llattn_clip_args& a, int i, int most, Take take) {
  for (int n = 0, chunks = 0; i < a.count; ++i) {
    if (!a.sizes[i]) continue;
    const int c = chunks_of(a, i);
    if (n == most || (n && chunks > (1 << 30) - c)) break;
    take(i, chunks, c);
    ++n;
    chunks += c;
  }
  return i;
}
template <int CAP>
void fill(const llattn_clip_args& a, int* i, Table<CAP>* t) {
  t->n = t->chunks = 0;
  *i = batch(a, *i, CAP, [&](int k, int chunk, int chunks) {
    const int bf = a.dtypes[k] == LLATTN_BF16;
    t->e[t->n++] = {static_cast<char*>(a.tensors[k]), a.sizes[k] * (bf ? 2 : 4), chunk, bf};
    t->chunks = chunk + chunks;
  });
}
template <int CAP>
int grid_of(const Table<CAP>& t) { return std::max(1, std::min(t.chunks, std::min(kMaxGrid, 8 * sm_count()))); }

int batches(const llattn_clip_args& a) {  // (the same with the short table, which holds all of a list that takes it)
  int n = 0, i = 0;
  do {
    i = batch(a, i, kTensors, [](int, int, int) {});
    ++n;
  } while (i < a.count);
  return n;
}

template <typename Op, int CAP>
cudaError_t run(const llattn_clip_args& a, cudaStream_t s) {
  double* part = static_cast<double*>(a.workspace);
  Table<CAP> t;
  int n_part = 0, i = 0, n = 0;
  do {
    fill(a, &i, &t);
    const int grid = grid_of(t);
    const cudaError_t e = launch_pdl(norm_kernel<Op, CAP>, dim3(grid), kThreads, 0, 1, s, t, part + n_part);
    if (e != cudaSuccess) return e;
    n_part += grid;
    ++n;
  } while (i < a.count);
  const bool again = a.scale && n > 1;  // (otherwise t is the only batch, or its tensors are not touched)
  if (again) i = 0;
  float* norm = a.norm;
  do {
    if (again) fill(a, &i, &t);
    const cudaError_t e = launch_pdl(clip_kernel<Op, CAP>, dim3(a.scale ? grid_of(t) : 1), kThreads, 0, 1, s, t, part, n_part,
                                     a.max_norm, a.scale, norm);
    if (e != cudaSuccess) return e;
    norm = nullptr;
  } while (i < a.count);
  return cudaSuccess;
}

}  // namespace

size_t workspace_bytes(const llattn_clip_args& a) { return (size_t)batches(a) * kMaxGrid * sizeof(double); }
int launches(const llattn_clip_args& a) { return batches(a) * (a.scale ? 2 : 1) + !a.scale; }

cudaError_t launch(const llattn_clip_args& a, cudaStream_t s) {
  if (a.count <= kShort) return a.norm_type == LLATTN_NORM_INF ? run<Largest, kShort>(a, s) : run<Squares, kShort>(a, s);
  return a.norm_type == LLATTN_NORM_INF ? run<Largest, kTensors>(a, s) : run<Squares, kTensors>(a, s);
}

}  // namespace clip
}  // namespace llattn
