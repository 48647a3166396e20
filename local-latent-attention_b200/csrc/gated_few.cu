// Gated feed-forward block of few tokens without gradients (decoding): two launches, the
// first g, u -> h, the second h -> y. What they cost is reading the weights, once each: 6 d ff
// bytes in bf16 (1536 x 4096: 38 MB, 5.8 us at 6.55 TB/s), and the latency of two launches.
//
// A CTA owns 16 rows of a weight matrix (of both, in the first launch) and a range of K; its 8
// warps take 64 bytes each of every 512 of a row. A lane reads 16 bytes of row lane / 4 and of the row
// 8 further straight to registers, several steps ahead, across row blocks where a CTA has several: in
// bf16 they are, in an order of K that x is read in as well, its part of two m16n8k16 fragments (mma.sync:
// 8 tokens fill its columns, the loads bound the kernel, not the products), and its 16 bytes of token
// lane / 4 the other operand. No operand is read twice by a CTA, so none goes through shared memory: no
// barrier before the sums. Rows off a 16-byte boundary: bf16 reads the two chunks that hold the 16 bytes and shifts
// them. fp32 takes rows 4 apart, which are all off it by as much, reads whole chunks that begin before
// the rows, and shifts x, by elements (1 token of 1411 x 3749: 37 -> 21 us; in bf16 x is in fragments, and
// two chunks of it for one of the weights cost more than they save: 24 tokens 37 us for 30). Rings of
// asynchronous copies in shared memory with one CTA per SM were slower (1 token: 27 us for 17): what a launch
// this short waits for is its first loads, its barriers and its last sums, and those pass beside another CTA's
// loads only where an SM holds several.
//
// The ranges of K of a row block are a cluster: their sums meet in the shared memory of its
// first CTA, which adds them in order. The second launch reads its weights before the first one is
// done (these do not depend on it: the first launch lets it start only after everything before is
// complete), and only then waits for h; the first one asks the L2 for its weights before it waits. (Asking for
// the second one's too won nothing: 15.4 us for 15.2.)
//
// bf16: h is stored in two bf16 parts and multiplied in both. fp32: products on the SIMT cores, 8 tokens at a time.
//
// Measured (us, by CUDA graph over weights that come from memory; floor = the weights at 6.55 TB/s; 33: mm_kernel's
// way): 1536 x 4096 (5.8): 14.2 for 1 token, 17.9 for 16, 21.7 for 24, 25.3 for 33; 2048 x 8192 (15.4): 28, 4096 x
// 14336 (53.8): 86; 1411 x 3749 (4.8): 22, 24 tokens 31, 33: 38; fp32 1536 x 4096 (11.5): 27, 8 tokens
// 40, 1411 x 3749 (9.7): 21. The
// large ones are bound by how evenly the row blocks fill the SMs and by the pauses between CTAs, the small ones by two
// launches of some 4 us.
#include <algorithm>

#include "gated.cuh"
#include "gated_act.cuh"
#include "pdl.cuh"
#include "sm100_ptx.cuh"

namespace llattn {
namespace gated {
namespace {

using namespace ptx;

constexpr int kWarps = 8, kThreads = 32 * kWarps;

struct FewArgs {
  const void* x;  // [tokens][ldx]; the second launch's in bf16: [2][tokens][ldx], 16-byte aligned rows
  int64_t ldx;
  int tokens, K, rows;
  const void* w[2];
  int64_t ldw[2];
  void* out;  // h (fp32, or bf16 [2][tokens][ldo]), or y
  int64_t ldo;
  int act, ranges, per;  // ranges of K, columns of one
};

// C: tokens of a CTA
template <typename T, int C, int NW, bool SHIFT>
struct FewShape {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int NT = F32 ? 1 : C / 8;                             // token groups: columns of a fragment
  static constexpr int VALUES = NW * NT * 128;                           // sums of a CTA: 16 rows of 8 tokens each
  static constexpr int LANE = 16 / sizeof(T), STEP = 4 * LANE * kWarps;  // columns of 16 bytes, of the CTA's step
  // steps of loads under way: what 128 registers hold (two CTAs to an SM), less where more were slower (bf16, 1
  // token of 1536 x 4096: 15.1 us with 3 and 4 steps, 16.0 with 4 and 6, 16.8 with 2 and 4 and three CTAs)
  static constexpr int AHEAD = F32       ? (C > 4 ? 2 : SHIFT ? 3 : NW == 2 ? 4 : 6)
                               : NT > 1  ? (SHIFT && NW == 2 ? 1 : 2)
                               : SHIFT   ? (NW == 2 ? 2 : 3)
                                         : (NW == 2 ? 3 : 4);
  static constexpr int GAP = SHIFT && F32 ? LANE : 1;  // rows between those of a CTA
};

// Columns [k, k + 16 bytes) of a row as the aligned chunks that hold them (the second one where the row is off).
struct Raw {
  uint4 c[2];
};
// kConst: by the read-only path, for what was complete before this kernel started: w_down, in the second launch. x
// and the first launch's weights may come from the kernel ahead, which that path does not allow for. kOnce: past the
// L1, where the weights leave x its place.
enum Load { kPlain, kConst, kOnce };
template <Load L>
__device__ __forceinline__ uint4 load16(uintptr_t q) {
  const uint4* p = reinterpret_cast<const uint4*>(q);
  if (L == kConst) return __ldg(p);
  if (L == kPlain) return *p;
  uint4 v;
  asm volatile("ld.global.L1::no_allocate.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "l"(p));
  return v;
}
// [lo, hi): the matrix's bytes.
// GAP: k may lie before the row, by less than a chunk.
template <typename T, bool SHIFT, Load L, bool GAP>
__device__ __forceinline__ void raw_load(Raw& r, const T* row, int k, int K, bool ok, uintptr_t lo, uintptr_t hi) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(row + k), q = SHIFT ? a & ~uintptr_t(15) : a;
  const uintptr_t b = a + min(16, (K - k) * (int)sizeof(T));  // the end of what is there
  ok = ok && k < K;
  const uint4 z = make_uint4(0, 0, 0, 0);
  const bool first = ok && (!(SHIFT || GAP) || q >= lo) && q + 16 <= hi, second = SHIFT && ok && q + 16 < b && q + 32 <= hi;
  r.c[0] = first ? load16<L>(q) : z;
  if (SHIFT) r.c[1] = second ? load16<L>(q + 16) : z;
  // the matrix's first and last bytes, where a chunk reaches past them
  const bool edge0 = ok && !first, edge1 = SHIFT && ok && !second && q + 16 < b;
  if (edge0 || edge1) {
#pragma unroll
    for (int c = 0; c < (SHIFT ? 2 : 1); ++c) {
      if (!(c ? edge1 : edge0)) continue;
      uint32_t v[4] = {0, 0, 0, 0};
#pragma unroll
      for (int i = 0; i < 16 / (int)sizeof(T); ++i) {
        const uintptr_t e = q + 16 * c + i * sizeof(T);
        if (e < (GAP ? lo : a) || e >= b) continue;
        if constexpr (sizeof(T) == 2)
          v[i / 2] |= (uint32_t) * reinterpret_cast<const uint16_t*>(e) << (i % 2 * 16);
        else
          v[i] = *reinterpret_cast<const uint32_t*>(e);
      }
      r.c[c] = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}
// The four words of it, `off` bytes into the chunks, zeros outside the columns [head, n) that are there.
template <typename T, bool SHIFT>
__device__ __forceinline__ void words(const Raw& r, int off, int head, int n, uint32_t (&w)[4]) {
  if constexpr (SHIFT) {
    uint32_t v[8] = {r.c[0].x, r.c[0].y, r.c[0].z, r.c[0].w, r.c[1].x, r.c[1].y, r.c[1].z, r.c[1].w};
    if (off & 8) {
#pragma unroll
      for (int i = 0; i < 6; ++i) v[i] = v[i + 2];
    }
    if (off & 4) {
#pragma unroll
      for (int i = 0; i < 5; ++i) v[i] = v[i + 1];
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = off & 2 ? __funnelshift_r(v[i], v[i + 1], 16) : v[i];
  } else {
    w[0] = r.c[0].x;
    w[1] = r.c[0].y;
    w[2] = r.c[0].z;
    w[3] = r.c[0].w;
  }
  if (n < 16 / (int)sizeof(T) || (sizeof(T) == 4 && head > 0)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = i >= head && i < n ? w[i] : 0u;
      else
        w[i] = 2 * i + 1 < n ? w[i] : 2 * i < n ? w[i] & 0xffffu : 0u;
    }
  }
}

__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[2][4], int half, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0][2 * half]), "r"(a[1][2 * half]), "r"(a[0][2 * half + 1]), "r"(a[1][2 * half + 1]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float gate(float g, int act) {
  if (act == LLATTN_ACT_SILU) return g / (1.f + expf(-g));
  float phi, e;
  gaussian(g, phi, e);
  return g * phi;
}

// SHIFT: rows (of x too) may be off a 16-byte boundary. WHOLE: a row block takes whole turns of the load
// buffers, the steps past its columns on zeros, so that no branch stands between loads and products and
// another row block's loads follow; otherwise a CTA has one row block, whose steps stop where it ends.
template <typename T, int C, int NW, bool SHIFT, bool WHOLE>
__global__ void __launch_bounds__(kThreads, 2) few_kernel(const __grid_constant__ FewArgs p) {
  using S = FewShape<T, C, NW, SHIFT>;
  constexpr bool F32 = S::F32;
  constexpr int PLANES = !F32 && NW == 1 ? 2 : 1, GAP = S::GAP;
  constexpr bool OFF = SHIFT && GAP == 1;  // rows each off by their own
  constexpr int NT = S::NT, XN = F32 ? 1 : NT * PLANES;
  constexpr bool XSHIFT = OFF && NW == 2;
  extern __shared__ float few_smem[];  // [2][kWarps][VALUES], [ranges][VALUES]
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int rank = (int)blockIdx.x % p.ranges, first = (int)blockIdx.x / p.ranges, stride = (int)gridDim.x / p.ranges;
  const int blocks = cdiv(p.rows, 16 * GAP) * GAP;
  const int tok0 = blockIdx.y * C, tokens = min(C, p.tokens - tok0);
  // columns of a row, with GAP from the chunk on that its first one lies in, the o-th of it: [o, K + o)
  const int kb = rank * p.per, most = min(p.K + GAP - 1, kb + p.per);
  constexpr int TURN = WHOLE ? S::AHEAD : 1;
  const int steps = kb < most ? cdiv(most - kb, S::STEP * TURN) * TURN : 0;
  const int kl = kb + (warp * 4 + t) * S::LANE;  // this lane's first column
  if (p.ranges > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  uintptr_t lo[NW], hi[NW];
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const T* base = static_cast<const T*>(p.w[w]);
    lo[w] = reinterpret_cast<uintptr_t>(base);
    hi[w] = reinterpret_cast<uintptr_t>(base + (p.rows - 1) * p.ldw[w] + p.K);
  }
  auto row_of = [&](int block, int i) { return block / GAP * (16 * GAP) + block % GAP + GAP * i; };  // the i-th of 16
  auto o_of = [&](int block) { return GAP > 1 ? (int)((lo[0] / sizeof(T) + row_of(block, 0) * p.ldw[0]) % S::LANE) : 0; };
  auto end_of = [&](int o) { return min(p.K + o, kb + p.per); };
  auto start_of = [&](int block, int w, int h) {  // of this lane's rows
    const int r = row_of(block, g + 8 * h);
    return static_cast<const T*>(p.w[w]) + (int64_t)(r < p.rows ? r : 0) * p.ldw[w];
  };
  // x's rows of this lane (bf16): the second launch's has two planes of aligned rows
  const T* xr[NT];
  int xoff[NT];
  const uintptr_t xlo = reinterpret_cast<uintptr_t>(p.x),
                  xhi = reinterpret_cast<uintptr_t>(static_cast<const T*>(p.x) + (p.tokens - 1) * p.ldx + p.K);
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    xr[i] = static_cast<const T*>(p.x) + (tok0 + (8 * i + g < tokens ? 8 * i + g : 0)) * p.ldx;
    xoff[i] = XSHIFT ? (int)(reinterpret_cast<uintptr_t>(xr[i] + kl) & 15) : 0;
  }

  // loads run AHEAD steps before the products, into the next row block where this one's are done
  Raw buf[S::AHEAD][NW][2], xbuf[S::AHEAD][XN];
  const T* row[NW][2];
  int next = first, nj = 0, xj = 0, no = 0;
  auto set_rows = [&]() {
    no = o_of(next);
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) row[w][h] = start_of(next, w, h);
  };
  set_rows();
  auto issue = [&](Raw (&b)[NW][2]) {
    const int k = kl + nj * S::STEP;
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h)
        raw_load<T, OFF, NW == 1 ? kConst : kOnce, (GAP > 1)>(b[w][h], row[w][h], k - no, end_of(no) - no, row_of(next, g + 8 * h) < p.rows, lo[w], hi[w]);
    if (++nj == steps && WHOLE) {
      nj = 0;
      next += stride;
      set_rows();
    }
  };
  auto issue_x = [&](Raw (&b)[XN]) {
    if constexpr (!F32) {
      const int k = kl + xj * S::STEP;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        const bool x_ok = 8 * i + g < tokens;
        if constexpr (NW == 2) {
          raw_load<T, XSHIFT, kPlain, false>(b[i], xr[i], k, end_of(0), x_ok, xlo, xhi);
        } else {
#pragma unroll
          for (int pl = 0; pl < PLANES; ++pl)
            b[i * PLANES + pl].c[0] =
                x_ok && k < end_of(0) ? *reinterpret_cast<const uint4*>(xr[i] + pl * p.tokens * p.ldx + k) : make_uint4(0, 0, 0, 0);
        }
      }
      if (++xj == steps && WHOLE) xj = 0;
    }
  };
  if (NW == 2) {
#pragma unroll
    for (int j = 0; j < S::AHEAD; ++j)
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (row_of(first, g + 8 * h) < p.rows && kl + j * S::STEP < p.K)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(row[w][h] + kl + j * S::STEP));
    pdl_wait();
    pdl_next();  // not before: the second launch's loads rest on it
  }
#pragma unroll
  for (int u = 0; u < S::AHEAD; ++u) {
    issue(buf[u]);
    if (NW == 2) issue_x(xbuf[u]);
  }
  if (NW == 1) {
    pdl_wait();
    pdl_next();
#pragma unroll
    for (int u = 0; u < S::AHEAD; ++u) issue_x(xbuf[u]);
  }

  constexpr int ACC = F32 ? 2 * C : 4 * NT;  // fp32: [row half][token]; else the fragments
  float acc[NW][ACC];
  int off[NW][2], o = 0, ke = 0;  // of this row block
  auto compute = [&](const Raw (&b)[NW][2], const Raw (&xb)[XN], int k) {
    const int head = GAP > 1 ? o - k : 0;
    uint32_t a[NW][2][4];
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) words<T, OFF>(b[w][h], off[w][h], head, ke - k, a[w][h]);
    if constexpr (F32) {
#pragma unroll
      for (int i0 = 0; i0 < C; i0 += 4) {  // loads of up to 4 tokens together
        constexpr int G = C < 4 ? C : 4;
        float xv[G][4];
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const float* src = static_cast<const float*>(p.x) + (int64_t)(tok0 + min(i0 + i, tokens - 1)) * p.ldx + (k - o);
          if (!SHIFT) {  // (a row's last columns are masked in the weights; what lies behind them may not be there)
            const float4 v = k + 4 <= ke ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            xv[i][0] = v.x; xv[i][1] = v.y; xv[i][2] = v.z; xv[i][3] = v.w;
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) xv[i][q] = q >= head && k + q < ke ? src[q] : 0.f;
          }
        }
        if (!SHIFT && k < ke && k + 4 > ke) {
#pragma unroll
          for (int i = 0; i < G; ++i)
#pragma unroll
            for (int q = 0; q < 4; ++q)
              if (k + q < ke) xv[i][q] = static_cast<const float*>(p.x)[(int64_t)(tok0 + min(i0 + i, tokens - 1)) * p.ldx + k + q];
        }
#pragma unroll
        for (int i = 0; i < G; ++i)
#pragma unroll
          for (int w = 0; w < NW; ++w)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int q = 0; q < 4; ++q)
                acc[w][h * C + i0 + i] = fmaf(__uint_as_float(a[w][h][q]), xv[i][q], acc[w][h * C + i0 + i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < XN; ++i) {
        uint32_t x[4];
        words<T, XSHIFT>(xb[i], xoff[i / PLANES], 0, ke - k, x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          float(&c)[4] = *reinterpret_cast<float(*)[4]>(&acc[w][i / PLANES * 4]);
          mma16816(c, a[w], 0, x[0], x[1]);
          mma16816(c, a[w], 1, x[2], x[3]);
        }
      }
    }
  };
#pragma unroll 1
  for (int block = first, turn = 0; block < blocks; block += stride, turn ^= 1) {
    o = o_of(block);
    ke = end_of(o);
#pragma unroll
    for (int w = 0; w < NW; ++w) {
#pragma unroll
      for (int i = 0; i < ACC; ++i) acc[w][i] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) off[w][h] = OFF ? (int)(reinterpret_cast<uintptr_t>(start_of(block, w, h) + kl) & 15) : 0;
    }
#pragma unroll 1
    for (int j0 = 0; j0 < steps; j0 += S::AHEAD) {
#pragma unroll
      for (int u = 0; u < S::AHEAD; ++u) {
        if (WHOLE || j0 + u < steps) {
          compute(buf[u], xbuf[u], kl + (j0 + u) * S::STEP);
          issue(buf[u]);
          issue_x(xbuf[u]);
        }
      }
    }

    // sums of the warps, then of the ranges; a value's place: product, fragment register, lane
    float* red = few_smem + turn * kWarps * S::VALUES;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      if constexpr (F32) {
#pragma unroll
        for (int i = 0; i < ACC; ++i) {
          acc[w][i] += __shfl_xor_sync(0xffffffffu, acc[w][i], 1);
          acc[w][i] += __shfl_xor_sync(0xffffffffu, acc[w][i], 2);
        }
      }
#pragma unroll
      for (int r = 0; r < 4 * NT; ++r) {
        float v;
        if constexpr (F32) {
          v = 0.f;  // (of no token)
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (2 * q + (r & 1) < C) v = t == q ? acc[w][(r >> 1) * C + 2 * q + (r & 1)] : v;
        } else {
          v = acc[w][r];
        }
        red[warp * S::VALUES + (w * NT * 4 + r) * 32 + lane] = v;
      }
    }
    __syncthreads();
    const float* sums = red;
    int n_sums = kWarps;
    if (p.ranges > 1) {  // (one row block to a cluster)
      asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the first CTA is there
      float* slots = few_smem + 2 * kWarps * S::VALUES;
      for (int i = tid; i < S::VALUES; i += kThreads) {
        float s = red[i];
#pragma unroll
        for (int k = 1; k < kWarps; ++k) s += red[k * S::VALUES + i];
        asm volatile(
            "{\n\t.reg .b32 ra;\n\t"
            "mapa.shared::cluster.u32 ra, %0, 0;\n\t"
            "st.shared::cluster.f32 [ra], %1;\n\t}" ::"r"(smem_u32(slots + rank * S::VALUES + i)),
            "f"(s)
            : "memory");
      }
      asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
      if (rank) return;
      sums = slots;
      n_sums = p.ranges;
    }
    for (int i = tid; i < 128 * NT; i += kThreads) {
      float v[NW];
#pragma unroll
      for (int w = 0; w < NW; ++w) {
        v[w] = sums[w * NT * 128 + i];
#pragma unroll 8
        for (int k = 1; k < n_sums; ++k) v[w] += sums[k * S::VALUES + w * NT * 128 + i];
      }
      const int l = i % 32, r = i / 32 % 4, tok = i / 128 * 8 + 2 * (l % 4) + (r & 1), f = row_of(block, l / 4 + 8 * (r >> 1));
      if (tok >= tokens || f >= p.rows) continue;
      const int64_t at = (tok0 + tok) * p.ldo + f;
      if constexpr (NW == 2) {
        const float h = gate(v[0], p.act) * v[1];
        if constexpr (F32) {
          static_cast<float*>(p.out)[at] = h;
        } else {
          const bf16 hi16 = __float2bfloat16_rn(h);
          static_cast<bf16*>(p.out)[at] = hi16;
          static_cast<bf16*>(p.out)[p.tokens * p.ldo + at] = __float2bfloat16_rn(h - __bfloat162float(hi16));
        }
      } else {
        static_cast<T*>(p.out)[at] = from_f<T>(v[0]);
      }
    }
  }
}

template <typename T, int C, int NW, bool SHIFT, bool WHOLE>
cudaError_t launch(const FewArgs& p, int grid, cudaStream_t s) {
  const int smem = (2 * kWarps + p.ranges) * FewShape<T, C, NW, SHIFT>::VALUES * 4;
  const cudaError_t e = set_smem_once(few_kernel<T, C, NW, SHIFT, WHOLE>, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(few_kernel<T, C, NW, SHIFT, WHOLE>, dim3(grid, cdiv(p.tokens, C)), kThreads, smem, p.ranges, s, p);
}
template <typename T, int C, int NW, bool SHIFT>
cudaError_t launch(FewArgs p, cudaStream_t s) {
  using S = FewShape<T, C, NW, SHIFT>;
  // ranges of K while the CTAs do not fill the SMs once, each of at least two steps
  const int tiles = cdiv(p.rows, 16 * S::GAP) * S::GAP, K = p.K + S::GAP - 1;
  p.ranges = 1;
  while (p.ranges < 8 && p.ranges * tiles < sm_count() && K >= 4 * p.ranges * S::STEP) p.ranges *= 2;
  p.per = cdiv(cdiv(K, p.ranges), S::STEP) * S::STEP;
  const int grid = p.ranges > 1 ? tiles * p.ranges : std::min(tiles, 2 * sm_count());
  // whole turns (1 token of 2048 x 8192: 26.8 us for 29.8, of 1536 x 4096: 14.0 for 14.6), but not where a single
  // row block would pay for empty steps (1024 x 2816: 11.8 us for 9.8) or shifted rows spill (1411 x 3749: 22.1 for 20.7)
  const bool whole = grid < tiles || ((!SHIFT || S::F32) && p.per / S::STEP % S::AHEAD == 0);
  return whole ? launch<T, C, NW, SHIFT, true>(p, grid, s) : launch<T, C, NW, SHIFT, false>(p, grid, s);
}

template <typename T, int NW>
cudaError_t launch_as(const FewArgs& p, bool shift, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    if (p.tokens == 1) return shift ? launch<T, 1, NW, true>(p, s) : launch<T, 1, NW, false>(p, s);
    if (p.tokens <= 4) return shift ? launch<T, 4, NW, true>(p, s) : launch<T, 4, NW, false>(p, s);
  } else {
    if (p.tokens > 16) return shift ? launch<T, 24, NW, true>(p, s) : launch<T, 24, NW, false>(p, s);
    if (p.tokens > 8) return shift ? launch<T, 16, NW, true>(p, s) : launch<T, 16, NW, false>(p, s);
  }
  return shift ? launch<T, 8, NW, true>(p, s) : launch<T, 8, NW, false>(p, s);
}

bool whole(const void* p, int64_t ld, int64_t rows, int elt) { return ((uintptr_t)p & 15) == 0 && (rows == 1 || ld * elt % 16 == 0); }
bool all_whole(const llattn_gated_args& a) {
  const int elt = a.dtype == LLATTN_F32 ? 4 : 2;
  return whole(a.w_gate, a.ldg, a.ff, elt) && whole(a.w_up, a.ldu, a.ff, elt) && whole(a.x, a.ldx, a.tokens, elt);
}
int64_t padded(int ff) { return (ff + 7) / 8 * 8; }

template <typename T>
cudaError_t run(const llattn_gated_args& a, cudaStream_t s) {
  FewArgs p = {};
  p.x = a.x;
  p.ldx = a.ldx;
  p.tokens = a.tokens;
  p.K = a.d;
  p.rows = a.ff;
  p.w[0] = a.w_gate;
  p.w[1] = a.w_up;
  p.ldw[0] = a.ldg;
  p.ldw[1] = a.ldu;
  p.out = a.workspace;
  p.ldo = padded(a.ff);
  p.act = a.activation;
  constexpr int elt = sizeof(T);
  const cudaError_t e = launch_as<T, 2>(p, !all_whole(a), s);
  if (e != cudaSuccess) return e;
  FewArgs q = {};
  q.x = a.workspace;
  q.ldx = padded(a.ff);
  q.tokens = a.tokens;
  q.K = a.ff;
  q.rows = a.d_out;
  q.w[0] = a.w_down;
  q.ldw[0] = a.ldd;
  q.out = a.y;
  q.ldo = a.d_out;
  return launch_as<T, 1>(q, !whole(a.w_down, a.ldd, a.d_out, elt), s);
}

}  // namespace

// As many tokens as this form is faster for (us here, and by mm_kernel). bf16: beyond 8 it reads x more often than the
// weights' rows come in, and only small weights, for which mm_kernel's launches are long, make up for that: 24 tokens of
// 1024 x 2816 14.3 for 17.3, 1536 x 4096 21.7 for 25.3, 1800 x 4800 33.5 for 33.1, 2048 x 5461 (2^25 weights) 40.7 for
// 41.1, 2304 x 6144 41.7 for 35.6, 2048 x 8192 42.3 for 37.8; 25, another group, 36.7 for 24.3 at 1536 x 4096. Past 2^25
// weights 8 tokens are 26.6 for 36.8 and 28.5 for 38.1, 16 34.1 for 35.5 and 34.7 for 37.8: near enough for one limit.
// fp32: 8 at a time, each reading the weights again: 16 tokens 40 for 67 (1024 x 2816), 71 for 101, 158 for 204 (2048 x
// 8192), 17 46 for 67, 86 for 101, 215 for 204; where w_gate's and w_up's rows are off a 16-byte boundary by
// different shifts it has none, as a CTA's rows have to be off by the same.
int few_tokens(const llattn_gated_args& a) {
  if (a.dtype == LLATTN_F32) {
    const bool alike = (((uintptr_t)a.w_gate ^ (uintptr_t)a.w_up) & 15) == 0 && (a.ldg - a.ldu) % 4 == 0;
    return alike || all_whole(a) ? 16 : 0;
  }
  return (2 * (int64_t)a.d + a.d_out) * a.ff <= 1 << 25 ? 24 : 8;
}
size_t few_workspace_bytes(const llattn_gated_args& a) { return 4 * (size_t)a.tokens * padded(a.ff); }
cudaError_t launch_few(const llattn_gated_args& a, cudaStream_t s) {
  return a.dtype == LLATTN_F32 ? run<float>(a, s) : run<bf16>(a, s);
}

}  // namespace gated
}  // namespace llattn
