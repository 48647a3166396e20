// Gated feed-forward block of few tokens without gradients (decoding): two launches, the
// first g, u -> h, the second h -> y. What they cost is reading the weights, once each: 6 d ff
// bytes in bf16 (1536 x 4096: 38 MB, 5.8 us at 6.55 TB/s), and the latency of two launches.
//
// A CTA owns 16 rows of a weight matrix (of both, in the first launch) and a range of K; its 8
// warps take 64 bytes each of every 512 of a row. A lane reads 16 bytes of row lane / 4 and of the row
// 8 further straight to registers, several steps ahead: in bf16 they are, in an order of K that
// x is read in as well, its part of two m16n8k16 fragments (mma.sync: 8 tokens fill its columns, the
// loads bound the kernel, not the products), and its 16 bytes of token lane / 4 the other operand. No
// operand is read twice by a CTA, so none goes through shared memory: no barrier before the
// sums. Rows off a 16-byte boundary are read as the two chunks that hold them and shifted. Rings of
// asynchronous copies in shared memory with one CTA per SM were slower (1 token: 27 us for 17): what a
// launch this short waits for is its first loads, its barriers and its last sums, and those pass beside
// another CTA's loads only where an SM holds several.
//
// The ranges of K of a row block are a cluster: their sums meet in the shared memory of its
// first CTA, which adds them in order. The second launch reads its weights before the first one is
// done (these do not depend on it: the first launch lets it start only after everything before is
// complete), and only then waits for h; the first one asks the L2 for its weights before it waits.
//
// bf16: h is stored in two bf16 parts and multiplied in both. fp32: products on the SIMT cores, 8 tokens at a time.
#include <algorithm>

#include "gated.cuh"
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

// C: tokens that fp32 products are made for (bf16: 8)
template <typename T, int C, int NW, bool SHIFT>
struct FewShape {
  static constexpr bool F32 = sizeof(T) == 4;
  static constexpr int VALUES = NW * 128;                                // sums of a CTA: 16 rows of 8 tokens
  static constexpr int LANE = 16 / sizeof(T), STEP = 4 * LANE * kWarps;  // columns of 16 bytes, of the CTA's step
  // steps of loads under way: what 128 registers hold (two CTAs to an SM), less where more were slower (bf16, 1
  // token of 1536 x 4096: 15.1 us with 3 and 4 steps, 16.0 with 4 and 6, 16.8 with 2 and 4 and three CTAs)
  static constexpr int AHEAD = F32 ? (SHIFT || C > 4 ? 2 : NW == 2 ? 4 : 6) : SHIFT ? (NW == 2 ? 2 : 3) : NW == 2 ? 3 : 4;
};

// Columns [k, k + 16 bytes) of a row as the aligned chunks that hold them (the second one where the row is off).
struct Raw {
  uint4 c[2];
};
// [lo, hi): the matrix's bytes. W: a weight, by the read-only path; otherwise what the kernel before
// may have written while this one was already there, which the read-only path does not allow for.
template <bool W>
__device__ __forceinline__ uint4 load16(uintptr_t q) {
  const uint4* p = reinterpret_cast<const uint4*>(q);
  return W ? __ldg(p) : *p;
}
template <typename T, bool SHIFT, bool W>
__device__ __forceinline__ void raw_load(Raw& r, const T* row, int k, int K, bool ok, uintptr_t lo, uintptr_t hi) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(row + k), q = SHIFT ? a & ~uintptr_t(15) : a;
  const uintptr_t b = a + min(16, (K - k) * (int)sizeof(T));  // the end of what is there
  ok = ok && k < K;
  const uint4 z = make_uint4(0, 0, 0, 0);
  const bool first = ok && (!SHIFT || q >= lo) && q + 16 <= hi, second = SHIFT && ok && q + 16 < b && q + 32 <= hi;
  r.c[0] = first ? load16<W>(q) : z;
  if (SHIFT) r.c[1] = second ? load16<W>(q + 16) : z;
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
        if (e < a || e >= b) continue;
        if constexpr (sizeof(T) == 2)
          v[i / 2] |= (uint32_t) * reinterpret_cast<const uint16_t*>(e) << (i % 2 * 16);
        else
          v[i] = *reinterpret_cast<const uint32_t*>(e);
      }
      r.c[c] = make_uint4(v[0], v[1], v[2], v[3]);
    }
  }
}
// The four words of it, `off` bytes into the chunks, zeros past the n columns that are there.
template <typename T, bool SHIFT>
__device__ __forceinline__ void words(const Raw& r, int off, int n, uint32_t (&w)[4]) {
  if (SHIFT) {
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
  if (n < 16 / (int)sizeof(T)) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (sizeof(T) == 4)
        w[i] = i < n ? w[i] : 0u;
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
  return 0.5f * g * erfcf(g * -0.70710678f);
}

// SHIFT: rows (of x too) may be off a 16-byte boundary
template <typename T, int C, int NW, bool SHIFT>
__global__ void __launch_bounds__(kThreads, 2) few_kernel(const __grid_constant__ FewArgs p) {
  using S = FewShape<T, C, NW, SHIFT>;
  constexpr bool F32 = S::F32;
  constexpr int PLANES = !F32 && NW == 1 ? 2 : 1;
  __shared__ float red[kWarps * S::VALUES];
  extern __shared__ float slots[];  // [ranges][VALUES]
  const int tid = threadIdx.x, warp = tid / 32, lane = tid % 32, g = lane / 4, t = lane % 4;
  const int rank = (int)blockIdx.x % p.ranges, row0 = (int)blockIdx.x / p.ranges * 16;
  const int tok0 = blockIdx.y * C, tokens = min(C, p.tokens - tok0);
  const int kb = rank * p.per, ke = min(p.K, kb + p.per), steps = kb < ke ? cdiv(ke - kb, S::STEP) : 0;
  const int kl = kb + (warp * 4 + t) * S::LANE;  // this lane's first column
  if (p.ranges > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");

  const T* row[NW][2];
  uintptr_t lo[NW], hi[NW];
  int off[NW][2];
  bool ok[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) ok[h] = row0 + g + 8 * h < p.rows;
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    const T* base = static_cast<const T*>(p.w[w]);
    lo[w] = reinterpret_cast<uintptr_t>(base);
    hi[w] = reinterpret_cast<uintptr_t>(base + (p.rows - 1) * p.ldw[w] + p.K);
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      row[w][h] = base + (int64_t)(ok[h] ? row0 + g + 8 * h : 0) * p.ldw[w];
      off[w][h] = SHIFT ? (int)(reinterpret_cast<uintptr_t>(row[w][h] + kl) & 15) : 0;
    }
  }
  // x's row of this lane (bf16): the second launch's has two planes of aligned rows
  const T* xr = static_cast<const T*>(p.x) + (tok0 + (g < tokens ? g : 0)) * p.ldx;
  const bool x_ok = g < tokens;
  constexpr bool XSHIFT = SHIFT && NW == 2;
  const uintptr_t xlo = reinterpret_cast<uintptr_t>(p.x),
                  xhi = reinterpret_cast<uintptr_t>(static_cast<const T*>(p.x) + (p.tokens - 1) * p.ldx + p.K);
  const int xoff = XSHIFT ? (int)(reinterpret_cast<uintptr_t>(xr + kl) & 15) : 0;

  Raw buf[S::AHEAD][NW][2], xbuf[S::AHEAD][F32 ? 1 : PLANES];
  auto issue = [&](int j, Raw (&b)[NW][2]) {
    const int k = kl + j * S::STEP;
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) raw_load<T, SHIFT, true>(b[w][h], row[w][h], k, ke, ok[h], lo[w], hi[w]);
  };
  auto issue_x = [&](int j, Raw (&b)[F32 ? 1 : PLANES]) {
    if constexpr (!F32) {
      const int k = kl + j * S::STEP;
      if constexpr (NW == 2) {
        raw_load<T, XSHIFT, false>(b[0], xr, k, ke, x_ok, xlo, xhi);
      } else {
#pragma unroll
        for (int pl = 0; pl < PLANES; ++pl)
          b[pl].c[0] = x_ok && k < ke ? *reinterpret_cast<const uint4*>(xr + pl * p.tokens * p.ldx + k) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  if (NW == 2) {
#pragma unroll
    for (int j = 0; j < S::AHEAD; ++j)
#pragma unroll
      for (int w = 0; w < NW; ++w)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          if (ok[h] && kl + j * S::STEP < ke) asm volatile("prefetch.global.L2 [%0];" ::"l"(row[w][h] + kl + j * S::STEP));
    pdl_wait();
    pdl_next();  // not before: the second launch's loads rest on it
  }
#pragma unroll
  for (int u = 0; u < S::AHEAD; ++u) {
    issue(u, buf[u]);
    if (NW == 2) issue_x(u, xbuf[u]);
  }
  if (NW == 1) {
    pdl_wait();
    pdl_next();
#pragma unroll
    for (int u = 0; u < S::AHEAD; ++u) issue_x(u, xbuf[u]);
  }

  constexpr int ACC = F32 ? 2 * C : 4;  // fp32: [row half][token]; else the fragments
  float acc[NW][ACC];
#pragma unroll
  for (int w = 0; w < NW; ++w)
#pragma unroll
    for (int i = 0; i < ACC; ++i) acc[w][i] = 0.f;
  auto compute = [&](const Raw (&b)[NW][2], const Raw (&xb)[F32 ? 1 : PLANES], int k) {
    uint32_t a[NW][2][4];
#pragma unroll
    for (int w = 0; w < NW; ++w)
#pragma unroll
      for (int h = 0; h < 2; ++h) words<T, SHIFT>(b[w][h], off[w][h], ke - k, a[w][h]);
    if constexpr (F32) {
#pragma unroll
      for (int i0 = 0; i0 < C; i0 += 4) {  // loads of up to 4 tokens together
        constexpr int G = C < 4 ? C : 4;
        float xv[G][4];
#pragma unroll
        for (int i = 0; i < G; ++i) {
          const float* src = static_cast<const float*>(p.x) + (int64_t)(tok0 + min(i0 + i, tokens - 1)) * p.ldx + k;
          if (!SHIFT) {  // (a row's last columns are masked in the weights; what lies behind them may not be there)
            const float4 v = k + 4 <= ke ? *reinterpret_cast<const float4*>(src) : make_float4(0.f, 0.f, 0.f, 0.f);
            xv[i][0] = v.x; xv[i][1] = v.y; xv[i][2] = v.z; xv[i][3] = v.w;
          } else {
#pragma unroll
            for (int q = 0; q < 4; ++q) xv[i][q] = k + q < ke ? src[q] : 0.f;
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
      for (int pl = 0; pl < PLANES; ++pl) {
        uint32_t x[4];
        words<T, XSHIFT>(xb[pl], xoff, ke - k, x);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          float(&c)[4] = *reinterpret_cast<float(*)[4]>(&acc[w][0]);
          mma16816(c, a[w], 0, x[0], x[1]);
          mma16816(c, a[w], 1, x[2], x[3]);
        }
      }
    }
  };
#pragma unroll 1
  for (int j0 = 0; j0 < steps; j0 += S::AHEAD) {
#pragma unroll
    for (int u = 0; u < S::AHEAD; ++u) {
      const int j = j0 + u;
      if (j < steps) {
        compute(buf[u], xbuf[u], kl + j * S::STEP);
        issue(j + S::AHEAD, buf[u]);
        issue_x(j + S::AHEAD, xbuf[u]);
      }
    }
  }

  // sums of the warps, then of the ranges; a value's place: product, fragment register, lane
#pragma unroll
  for (int w = 0; w < NW; ++w) {
    if constexpr (F32) {
#pragma unroll
      for (int i = 0; i < ACC; ++i) {
        acc[w][i] += __shfl_xor_sync(0xffffffffu, acc[w][i], 1);
        acc[w][i] += __shfl_xor_sync(0xffffffffu, acc[w][i], 2);
      }
    }
    for (int r = 0; r < 4; ++r) {
      float v;
      if constexpr (F32) {
        v = 0.f;  // (of no token)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (2 * q + (r & 1) < C) v = t == q ? acc[w][(r >> 1) * C + 2 * q + (r & 1)] : v;
      } else {
        v = acc[w][r];
      }
      red[warp * S::VALUES + (w * 4 + r) * 32 + lane] = v;
    }
  }
  __syncthreads();
  if (p.ranges > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the first CTA is there
  for (int i = tid; i < S::VALUES; i += kThreads) {
    float s = red[i];
#pragma unroll
    for (int k = 1; k < kWarps; ++k) s += red[k * S::VALUES + i];
    float* dst = slots + rank * S::VALUES + i;
    if (p.ranges > 1)
      asm volatile(
          "{\n\t.reg .b32 ra;\n\t"
          "mapa.shared::cluster.u32 ra, %0, 0;\n\t"
          "st.shared::cluster.f32 [ra], %1;\n\t}" ::"r"(smem_u32(dst)),
          "f"(s)
          : "memory");
    else
      *dst = s;
  }
  if (p.ranges > 1) {
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank) return;
  } else {
    __syncthreads();
  }
  for (int i = tid; i < 128; i += kThreads) {
    float v[NW];
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      v[w] = slots[w * 128 + i];
      for (int k = 1; k < p.ranges; ++k) v[w] += slots[k * S::VALUES + w * 128 + i];
    }
    const int l = i % 32, r = i / 32, tok = 2 * (l % 4) + (r & 1), f = row0 + l / 4 + 8 * (r >> 1);
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

template <typename T, int C, int NW, bool SHIFT>
cudaError_t launch(FewArgs p, cudaStream_t s) {
  using S = FewShape<T, C, NW, SHIFT>;
  // ranges of K while the CTAs do not fill the SMs once, each of at least two steps
  const int tiles = cdiv(p.rows, 16);
  p.ranges = 1;
  while (p.ranges < 8 && p.ranges * tiles < sm_count() && p.K >= 4 * p.ranges * S::STEP) p.ranges *= 2;
  p.per = cdiv(cdiv(p.K, p.ranges), S::STEP) * S::STEP;
  const int smem = p.ranges * S::VALUES * 4;
  const cudaError_t e = set_smem_once(few_kernel<T, C, NW, SHIFT>, smem);
  if (e != cudaSuccess) return e;
  return launch_pdl(few_kernel<T, C, NW, SHIFT>, dim3(tiles * p.ranges, cdiv(p.tokens, C)), kThreads, smem, p.ranges, s, p);
}

template <typename T, int NW>
cudaError_t launch_as(const FewArgs& p, bool shift, cudaStream_t s) {
  if constexpr (sizeof(T) == 4) {
    if (p.tokens == 1) return shift ? launch<T, 1, NW, true>(p, s) : launch<T, 1, NW, false>(p, s);
    if (p.tokens <= 4) return shift ? launch<T, 4, NW, true>(p, s) : launch<T, 4, NW, false>(p, s);
  }
  return shift ? launch<T, 8, NW, true>(p, s) : launch<T, 8, NW, false>(p, s);
}

bool whole(const void* p, int64_t ld, int64_t rows, int elt) { return ((uintptr_t)p & 15) == 0 && (rows == 1 || ld * elt % 16 == 0); }
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
  const bool all = whole(a.w_gate, a.ldg, a.ff, elt) && whole(a.w_up, a.ldu, a.ff, elt) && whole(a.x, a.ldx, a.tokens, elt);
  const cudaError_t e = launch_as<T, 2>(p, !all, s);
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

int few_tokens(int dtype) { return dtype == LLATTN_F32 ? 16 : 8; }
size_t few_workspace_bytes(const llattn_gated_args& a) { return 4 * (size_t)a.tokens * padded(a.ff); }
cudaError_t launch_few(const llattn_gated_args& a, cudaStream_t s) {
  return a.dtype == LLATTN_F32 ? run<float>(a, s) : run<bf16>(a, s);
}

}  // namespace gated
}  // namespace llattn
