// Persistent tensor-core product of the training operators (included by
// xent.cu and orth.cu): C[M, N] = A[M, K] B[N, K]^T per batch element z, 16-bit
// operands (both bf16 or both fp16), fp32 accumulation in TMEM, and an
// epilogue functor that consumes the accumulator rows in registers.
//
// Each operand is K-major (stored [MN, K], K contiguous) or MN-major (stored
// [K, MN]); tensor maps are 3-D (contiguous, rows, z) with 128-byte-swizzled
// boxes of 64 x 128 (K-major) or 64 x 64 (MN-major, two panels per 128
// rows); out-of-range rows, columns and K are zero-filled by the copies.
//
// The large tile is 256 x 256 on a pair of CTAs (a cluster of two SMs, CG = 2):
// each CTA copies its own 128 rows of A and 128 of the tile's 256
// rows of B, the leader (cluster rank 0) issues cta_group::2 MMAs for both,
// and each CTA ends up with its 128 rows x 256 columns of the accumulator.
// Per K = 64 step a CTA copies 32 KB for 128 x 256 x 64 products, half the L2
// traffic per flop of a 128 x 128 tile on one CTA, which smaller products use
// because it spreads over more SMs. All keep a ring of stages (6 to 8) that
// runs on across tiles and two accumulators in TMEM, so one tile's epilogue
// overlaps the next tile's MMAs; the 256 x 512 tile of long sums has 4 stages
// and one accumulator, in two halves.
//
// Warps: 0 copies, 1 issues MMAs, the others (one per 32 rows x 128 columns of
// the CTA's accumulator) run the epilogue: thread = row, 128 columns.
// Every wait is bounded (mbar_wait); a CTA whose wait runs out raises the
// fault word, which ends every other wait, and all warps still meet at the
// final barriers.
#pragma once

#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"
#include "pdl.cuh"
#include "sm100.cuh"
#include "sm100_ptx.cuh"

namespace llattn {
namespace mm {
namespace {

using namespace ptx;

// as local_sm100.cu's fault word, for the kernels of this translation unit
__device__ unsigned int g_mm_fault = 0;

unsigned read_fault(bool reset) {
  unsigned v = 0;
  cudaMemcpyFromSymbol(&v, g_mm_fault, sizeof(v));
  if (reset) {
    const unsigned z = 0;
    cudaMemcpyToSymbol(g_mm_fault, &z, sizeof(z));
  }
  return v;
}

// The schedule: total tiles, of which the first `full` run whole, one after
// another on each CTA (pair), and the rest in s ranges of K each.
struct MmPlan {
  int total, full, s, items;
};

// One product. M, N, K are the host's sizes; m_dev / k_dev (optional) hold a
// device-side row count from which M / K are cut: max(0, min(M, *m_dev -
// dev_base)) (the rows past it are not computed, the K past it not read
// beyond the next multiple of 64, whose rows the caller keeps at zero).
struct MmArgs {
  int M, N, K;
  int a_mn, b_mn;
  int nz;                   // batch elements (tensor-map z)
  // Split K of the tiles that do not fill a wave: each range's sums go to part
  // (fp32, one BM x BN block per range) and mm_join adds them up. 0: no split; 1: ranges of at
  // least 8 steps of K; 2: of 8 steps counting every term's.
  int split;
  float* part;
  // The tensor cores' additions drop what lies below the running sum's last
  // bits: a sum that grows evenly comes out 2^-30 (a few thousand products) to
  // 2^-27 (2^19) per product short (measured for bf16 operands, three times
  // that for fp16), always towards zero. chain > 0 bounds each such sum to that many K = 64 steps (of
  // the last term's, or the last `majors`'; the terms before, smaller by 2^-8 and less, make one
  // more): the epilogue warps add it to the tile's fp32 sum in TMEM, rounded to
  // nearest, while the next one is under way (Epi::kChain; not shape 3).
  int chain;
  int sym;                  // C symmetric: tiles with n <= m only (square tiles)
  int fp16;                 // operands fp16 instead of bf16
  // products over planes: operand z coordinates (pa, pb) of n_terms passes
  // over K, 4 bits each (fp32 operands in three bf16 planes, G in two)
  int n_terms;
  int majors;               // how many of them, the last ones, are the large ones (0: 1)
  uint64_t pa, pb;
  uint32_t b2;              // kSecondTerms: bit t set, term t takes B from its second map
  const int* m_dev;
  const int* k_dev;
  int dev_base;
  MmPlan plan;              // set by the launch where there is no device-side count
  volatile unsigned* fault_host;
};

__device__ __forceinline__ void mm_raise(const MmArgs& p, unsigned bit, volatile int* abort) {
  atomicOr(&g_mm_fault, bit);
  if (p.fault_host) {
    *p.fault_host |= bit;
    __threadfence_system();
  }
  *abort = 1;
}

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// Arrive on the barrier at the same shared-memory offset in the cluster's CTA 0.
// Release at CTA scope: what the leader's MMAs touch after it is this CTA's
// TMEM, whose order the tcgen05 fence before it sees to; a cluster-scope
// release waits some 1500 cycles for unrelated writes.
__device__ __forceinline__ void mbar_arrive_leader(uint64_t* bar) {
  asm volatile(
      "{\n\t.reg .b32 ra;\n\t"
      "mapa.shared::cluster.u32 ra, %0, 0;\n\t"
      "mbarrier.arrive.shared::cluster.b64 _, [ra];\n\t}" ::"r"(smem_u32(bar))
      : "memory");
}
// tile copy whose bytes count on the leader's barrier (clearing the CTA-rank
// bit of a shared::cluster address of a pair gives CTA 0's); no multicast
__device__ __forceinline__ void tma_load_3d_pair(const CUtensorMap* map, uint64_t* bar, void* dst, int c0, int c1,
                                                 int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_u32(bar) & 0xFEFFFFFFu), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// true in one lane of a converged warp
__device__ __forceinline__ bool elect_one() {
  uint32_t e;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(e));
  return e != 0;
}

template <int CG>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  if (CG == 1) {
    mma_bf16(d, a, b, idesc, acc);  // kind::f16; the descriptor names the type
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc)
        : "memory");
  }
}
// the barrier (in both CTAs of a pair) arrives when the MMAs issued so far are done
template <int CG>
__device__ __forceinline__ void commit(uint64_t* bar) {
  if (CG == 1) {
    mma_commit(bar);
  } else {
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
  }
}
template <int CG>
__device__ __forceinline__ void mm_tmem_alloc(uint32_t* dst, uint32_t ncols) {
  if (CG == 1) {
    tmem_alloc(dst, ncols);
    tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG>
__device__ __forceinline__ void mm_tmem_dealloc(uint32_t t, uint32_t ncols) {
  if (CG == 1)
    tmem_dealloc(t, ncols);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(t), "r"(ncols) : "memory");
}

// Tile shapes:
//  3 = 256 x 512 on a pair, for long sums: one accumulator fills the TMEM, as two
//      halves of 256 columns that the epilogue frees one after the other. An
//      SM takes in about 64 bytes a cycle, which the 32 KB a step of shape 2
//      need as long as their products take; 48 KB for twice the products do
//      not hold the tensor cores up.
//  2 = 256 x 256 on a pair, two accumulators
//  5 = the same with 16 epilogue warps instead of 8, at 96 registers a thread, for
//      epilogues that work on every value for long: they have no staging blocks
//      (and one stage less: a sixth made dh's product of 8192 x 1536 x 4096 110 us instead of 105)
//  1 = 128 x 128 on a CTA, two accumulators
//  4 = 128 x 64 on a CTA, between 1 and 0
//  0 = 128 x 32 on a CTA, for products too small to occupy the SMs otherwise:
//      its epilogue is one block of 32 columns per warp instead of four (4.2 ->
//      1.1 us at the end of a kernel), and a step copies 20 KB instead of 32.
template <int SH>
struct MmShape {
  static constexpr int CG = SH == 2 || SH == 3 || SH == 5 ? 2 : 1;
  static constexpr int NH = SH == 3 ? 2 : 1;  // column halves of the accumulator, an MMA each
  static constexpr int BM = 128 * CG, BN = SH == 3 ? 512 : SH == 2 || SH == 5 ? 256 : SH == 1 ? 128 : SH == 4 ? 64 : 32;  // tile of the CTA (pair)
  static constexpr int HN = BN / NH;              // columns of an MMA
  static constexpr int CW = SH == 5 ? 64 : HN < 128 ? HN : 128;  // columns of an epilogue warp (32 rows) in a half
  static constexpr int EW = 4 * (HN / CW);        // epilogue warps
  static constexpr int THREADS = 64 + 32 * EW;
  static constexpr int ST = SH == 3 ? 4 : SH == 5 ? 5 : BN < 128 ? 8 : 6;
  static constexpr int BR = HN / CG;        // rows of B that a CTA copies per half
  static constexpr int AB = 128 * 64 * 2;   // one CTA's A tile: 128 rows x 64 K, 16 KB
  static constexpr int BB = (BR < 64 ? 64 : BR) * 64 * 2;  // B tile of a half (a whole panel of 64 if MN-major)
  static constexpr int STG = SH == 5 ? 0 : 4096;  // an epilogue warp's staging block: 32 rows of 128 bytes
  static constexpr int A = 0, B = A + ST * AB, STAGE = B + ST * NH * BB, BAR = STAGE + EW * STG;
  static constexpr int ACC = NH == 2 ? 1 : 2;      // accumulators in TMEM
  static constexpr int BLOCK = 205 * (BM * BN / 1024) / 64;  // mm_plan's `block`
  static constexpr int TCOLS = BN < 256 ? 4 * BN : 512;  // (and with chains a sum, after the accumulators)
  static constexpr int BYTES = BAR + 256;
  static constexpr int SMEM = BYTES + 1024;  // + alignment
  static_assert(SMEM <= 227 * 1024, "shared memory");
};

struct MmTile {
  int z, m0, n0;
};

// s splits the last, partial wave of `units`, each range at least 8 steps of K
// (`terms` of them a step of the sum, for split = 2), by the time of its ceil(tail s / units) rounds in steps: the range's own,
// 6 for its epilogue, and the partial sums' way through memory (a 256 x 256
// block written and read takes the memory 0.2 of a step: `block`, in 1/1024).
__host__ __device__ inline MmPlan mm_plan(int total, int units, int ksteps, int split, int terms, int block) {
  MmPlan r{total, total, 1, total};
  if (!split || total == 0) return r;
  if (split == 1) terms = 1;
  const int full = total / units * units, tail = total - full;
  if (tail == 0) return r;
  int best = 1;
  int64_t cost = INT64_MAX;  // (integers: the product's and the join's kernel have to agree)
  for (int s = 1; s <= 32; ++s) {
    if (s > 1 && (ksteps < s || ksteps * terms < 8 * s || (int64_t)tail * s > 4 * (int64_t)units)) break;
    const int64_t c = 1024 * (int64_t)cdiv(tail * s, units) * (cdiv(ksteps, s) * terms + 6) + (s > 1 ? (int64_t)block * tail * s : 0);
    if (c < cost) {
      cost = c;
      best = s;
    }
  }
  if (best == 1) return r;
  return MmPlan{total, full, best, full + tail * best};
}

template <int SH>
struct MmGrid {
  int n_mt, n_nt, per_z;
  __host__ __device__ __forceinline__ MmGrid(const MmArgs& p, int M) {
    n_mt = cdiv(M, MmShape<SH>::BM);
    n_nt = cdiv(p.N, MmShape<SH>::BN);
    per_z = p.sym ? n_mt * (n_mt + 1) / 2 : n_mt * n_nt;
  }
  __device__ __forceinline__ MmTile at(const MmArgs& p, int t) const {
    MmTile r;
    r.z = p.nz > 1 ? t / per_z : 0;
    int u = t - r.z * per_z, i, j;
    if (p.sym) {  // row i of the lower triangle holds i + 1 tiles
      i = (int)((sqrtf(8.f * u + 1.f) - 1.f) * 0.5f);
      while (i * (i + 1) / 2 > u) --i;
      while ((i + 1) * (i + 2) / 2 <= u) ++i;
      j = u - i * (i + 1) / 2;
    } else {
      // bands of 8 row tiles, walked column by column: the tiles in flight
      // share about 8 row and 9 column strips of the operands in L2
      const int band = 8 * n_nt, bi = u / band, v = u - bi * band;
      const int h = n_mt - bi * 8 < 8 ? n_mt - bi * 8 : 8;
      j = v / h;
      i = bi * 8 + (v - j * h);
    }
    r.m0 = i * MmShape<SH>::BM;
    r.n0 = j * MmShape<SH>::BN;
    return r;
  }
};

// item -> tile index, range of K [k0, k1), partial block (-1: whole)
struct MmItem {
  int tile, k0, k1, block;
};
__device__ __forceinline__ MmItem mm_item(const MmPlan& pl, int t, int K) {
  if (t < pl.full) return {t, 0, K, -1};
  const int u = t - pl.full, tile = u / pl.s, j = u - tile * pl.s;
  const int per = cdiv(cdiv(K, 64), pl.s) * 64;
  const int k0 = j * per;
  return {pl.full + tile, k0, min(K, k0 + per), u};
}

__device__ __forceinline__ int cut_rows(int n, const int* dev, int base) {
  if (!dev) return n;
  const int v = *dev - base;
  return v < 0 ? 0 : (v < n ? v : n);
}

// 32 accumulator columns of this thread's row
__device__ __forceinline__ void load32(uint32_t taddr, bool zero, float (&v)[32]) {
  uint32_t r[32];
  if (!zero) {
    tmem_ld32(taddr, r);
    tmem_ld_wait();
  }
#pragma unroll
  for (int q = 0; q < 32; ++q) v[q] = zero ? 0.f : __uint_as_float(r[q]);
}

// Block transfers of an epilogue warp: thread = row holds CH 16-byte chunks of
// its row (32 columns of 16 or 32 bits: 4 or 8 chunks); global memory is
// accessed with CH lanes per row, whole 64- or 128-byte segments, through the
// staging block (chunks rotated by the row, so both sides meet every bank). A
// thread-per-row access would touch 32 lines per instruction and half of
// each 32-byte sector.
template <int CH>
__device__ __forceinline__ int stage_at(int r, int c) {
  return CH == 8 ? r * 128 + ((c ^ (r & 7)) * 16) : r * 64 + ((c ^ ((r >> 1) & 3)) * 16);
}
// The 32 rows of a block in memory (16-byte aligned where not said otherwise):
// row r at p + r stride (bytes), `rows` of them exist; or each lane's own row.
// row(r) is null for one that does not exist; at(b): the same rows b bytes on.
struct Rows {
  uint8_t* p;
  int64_t stride;
  int rows;
  __device__ __forceinline__ Rows(const void* p_, int64_t stride_, int rows_)
      : p(static_cast<uint8_t*>(const_cast<void*>(p_))), stride(stride_), rows(rows_) {}
  __device__ __forceinline__ uint8_t* row(int r) const { return r < rows ? p + r * stride : nullptr; }
  __device__ __forceinline__ Rows at(int bytes) const { return Rows(p + bytes, stride, rows); }
};
struct MappedRows {
  uint8_t* p;  // this lane's row, or null
  __device__ __forceinline__ uint8_t* row(int r) const {
    return reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<uint64_t>(p), r));
  }
  __device__ __forceinline__ MappedRows at(int bytes) const { return MappedRows{p ? p + bytes : nullptr}; }
};

template <bool ADD, int CH, typename R>
__device__ __forceinline__ void block_write_out(const uint8_t* buf, int lane, const R& dst, int bytes) {
  const int c = lane % CH;
  // all reads before the first write: the compiler may not move them across it
  uint4 u[CH];
#pragma unroll
  for (int i = 0; i < CH; ++i) u[i] = *reinterpret_cast<const uint4*>(buf + stage_at<CH>(32 / CH * i + lane / CH, c));
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    uint8_t* q = dst.row(32 / CH * i + lane / CH);
    if (q && 16 * c < bytes) {
      if (ADD)  // fp32: added in the L2, nothing waits for the old value
        asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(q + 16 * c), "f"(__uint_as_float(u[i].x)),
                     "f"(__uint_as_float(u[i].y)), "f"(__uint_as_float(u[i].z)), "f"(__uint_as_float(u[i].w)));
      else
        asm volatile("st.global.v4.b32 [%0], {%1, %2, %3, %4};" ::"l"(q + 16 * c), "r"(u[i].x), "r"(u[i].y), "r"(u[i].z),
                     "r"(u[i].w));
    }
  }
  __syncwarp();
}
// bytes: valid bytes of the rows (rounded up to 16 in memory)
template <bool ADD = false, int CH, typename R>
__device__ __forceinline__ void block_store(uint8_t* buf, int lane, const uint4 (&v)[CH], const R& dst, int bytes) {
#pragma unroll
  for (int i = 0; i < CH; ++i) *reinterpret_cast<uint4*>(buf + stage_at<CH>(lane, i)) = v[i];
  __syncwarp();
  block_write_out<ADD, CH>(buf, lane, dst, bytes);
}
// After a block_store of 32 x 32 16-bit values: the block's transpose, column c
// of it as row c of dst. 8 x 8 matrices go through registers (transposed on
// the load) into the second half of the staging block.
__device__ __forceinline__ void block_mirror(uint8_t* buf, int lane, const Rows& dst, int bytes) {
  uint8_t* tb = buf + 2048;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    uint32_t a, b, c, d;
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d)
                 : "r"(smem_u32(buf + stage_at<4>(lane, j)))
                 : "memory");
    asm volatile("stmatrix.sync.aligned.m8n8.x4.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(
                     smem_u32(tb + stage_at<4>(8 * j + lane % 8, lane / 8))),
                 "r"(a), "r"(b), "r"(c), "r"(d)
                 : "memory");
  }
  __syncwarp();
  block_write_out<false, 4>(tb, lane, dst, bytes);
}
// The reverse, in two halves so that the caller may have several in flight:
// fetch reads global memory, spread hands each thread its row (zeros where
// nothing was read).
template <int CH>
__device__ __forceinline__ void block_fetch(int lane, uint4 (&v)[CH], const Rows& src, int bytes) {
  const int c = lane % CH;
#pragma unroll
  for (int i = 0; i < CH; ++i) {
    const uint8_t* q = src.row(32 / CH * i + lane / CH);
    v[i] = q && 16 * c < bytes ? *reinterpret_cast<const uint4*>(q + 16 * c) : make_uint4(0, 0, 0, 0);
  }
}
template <int CH>
__device__ __forceinline__ void block_spread(uint8_t* buf, int lane, uint4 (&v)[CH]) {
  const int c = lane % CH;
#pragma unroll
  for (int i = 0; i < CH; ++i) *reinterpret_cast<uint4*>(buf + stage_at<CH>(32 / CH * i + lane / CH, c)) = v[i];
  __syncwarp();
#pragma unroll
  for (int i = 0; i < CH; ++i) v[i] = *reinterpret_cast<const uint4*>(buf + stage_at<CH>(lane, i));
  __syncwarp();
}
// Rows without 16-byte alignment: the staged block written element by
// element, lanes along the 32 columns (n of them valid).
template <typename E, int CH, typename R>
__device__ __forceinline__ void block_store_odd(uint8_t* buf, int lane, const uint4 (&v)[CH], const R& dst, int n) {
#pragma unroll
  for (int i = 0; i < CH; ++i) *reinterpret_cast<uint4*>(buf + stage_at<CH>(lane, i)) = v[i];
  __syncwarp();
  constexpr int PER = 16 / sizeof(E);
#pragma unroll 4
  for (int r = 0; r < 32; ++r) {
    E* q = reinterpret_cast<E*>(dst.row(r));
    const E e = *reinterpret_cast<const E*>(buf + stage_at<CH>(r, lane / PER) + (lane % PER) * sizeof(E));
    if (q && lane < n) q[lane] = e;
  }
  __syncwarp();
}

__device__ __forceinline__ uint32_t pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&h);
}

__device__ __forceinline__ void half_row(const float (&v)[32], uint4 (&u)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    u[q] = make_uint4(pack_half(v[8 * q], v[8 * q + 1]), pack_half(v[8 * q + 2], v[8 * q + 3]),
                      pack_half(v[8 * q + 4], v[8 * q + 5]), pack_half(v[8 * q + 6], v[8 * q + 7]));
}
__device__ __forceinline__ void bf16_row(const float (&v)[32], uint4 (&u)[4]) {
#pragma unroll
  for (int q = 0; q < 4; ++q)
    u[q] = make_uint4(pack_bf16(v[8 * q], v[8 * q + 1]), pack_bf16(v[8 * q + 2], v[8 * q + 3]),
                      pack_bf16(v[8 * q + 4], v[8 * q + 5]), pack_bf16(v[8 * q + 6], v[8 * q + 7]));
}
__device__ __forceinline__ void f32_row(const float (&v)[32], uint4 (&u)[8]) {
#pragma unroll
  for (int q = 0; q < 8; ++q)
    u[q] = make_uint4(__float_as_uint(v[4 * q]), __float_as_uint(v[4 * q + 1]), __float_as_uint(v[4 * q + 2]),
                      __float_as_uint(v[4 * q + 3]));
}
// 64 accumulator columns of this thread's row, times f, as bf16
__device__ __forceinline__ void row64_bf16(uint32_t taddr, bool zero, float f, uint4 (&u)[8]) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    float v[32];
    load32(taddr + 32 * h, zero, v);
#pragma unroll
    for (int q = 0; q < 32; ++q) v[q] *= f;
#pragma unroll
    for (int q = 0; q < 4; ++q)
      u[4 * h + q] = make_uint4(pack_bf16(v[8 * q], v[8 * q + 1]), pack_bf16(v[8 * q + 2], v[8 * q + 3]),
                                pack_bf16(v[8 * q + 4], v[8 * q + 5]), pack_bf16(v[8 * q + 6], v[8 * q + 7]));
  }
}
template <int CH>
__device__ __forceinline__ uint32_t word(const uint4 (&u)[CH], int i) {
  return i % 4 == 0 ? u[i / 4].x : i % 4 == 1 ? u[i / 4].y : i % 4 == 2 ? u[i / 4].z : u[i / 4].w;
}
__device__ __forceinline__ float2 half_pair(const uint4 (&u)[4], int i) {  // values 2i, 2i + 1
  const uint32_t w = word(u, i);
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 bf16_pair(const uint4 (&u)[4], int i) {
  const uint32_t w = word(u, i);
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}

// sum (+)= an accumulator's CW columns of this thread's row
template <int CW>
__device__ __forceinline__ void drain(uint32_t acc, uint32_t sum, bool add) {
#pragma unroll 1
  for (int cc = 0; cc < CW; cc += 32) {
    uint32_t a[32], b[32];
    tmem_ld32(acc + cc, a);
    if (add) tmem_ld32(sum + cc, b);
    tmem_ld_wait();
    if (add) {
#pragma unroll
      for (int q = 0; q < 32; ++q) a[q] = __float_as_uint(__uint_as_float(a[q]) + __uint_as_float(b[q]));
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      uint32_t c[16];
#pragma unroll
      for (int q = 0; q < 16; ++q) c[q] = a[16 * h + q];
      tmem_st16(sum + cc + 16 * h, c);
    }
  }
  tmem_st_wait();
}

// The tensor-core sums of a tile of `steps` K = 64 steps over n_terms terms:
// the one that starts at step i ends before step chain_end.
__device__ __forceinline__ int chain_end(const MmArgs& p, int i, int steps) {
  const int minor = p.n_terms > 1 ? steps / p.n_terms * (p.n_terms - max(p.majors, 1)) : 0;
  return i < minor ? minor : min(steps, i + p.chain);
}

// one range's sums of a tile: its fp32 block of part, [BM][BN]
template <int SH>
__device__ __forceinline__ void store_part(const MmArgs& p, const MmItem& x, const MmTile& w, int row, int col, int M,
                                           uint32_t taddr, uint8_t* buf) {
  using S = MmShape<SH>;
  const int lane = threadIdx.x % 32, row0 = row - lane;
  const Rows dst{p.part + ((int64_t)x.block * S::BM + row0) * S::BN + col, S::BN * 4, M - w.m0 - row0};
#pragma unroll 1
  for (int cc = 0; cc < S::CW; cc += 32) {
    const int n = p.N - (w.n0 + col + cc);
    if (n <= 0) break;  // warp-uniform
    float v[32];
    load32(taddr + cc, x.k1 <= x.k0, v);
    uint4 u[8];
    f32_row(v, u);
    block_store(buf, lane, u, dst.at(cc * 4), n * 4);
  }
}

// A second map for B, asked for by Epi::kSecond:
//   kSecondHalves: both maps' rows in one tile: of every BR columns of C (a CTA's share
//     of a tile, an epilogue warp's columns) the first half are rows of the first map and
//     the other half the same rows of the second one, so that a thread holds column
//     j of both products. C's columns count both: N = 2 x rows, rounded up to
//     whole BR. K-major only.
//   kSecondTerms: MmArgs::b2 says which terms take the second map.
// tile has a second template argument then, BR.
enum { kSecondNone = 0, kSecondHalves = 1, kSecondTerms = 2 };
template <typename Epi, typename = void>
struct SecondB : std::integral_constant<int, kSecondNone> {};
template <typename Epi>
struct SecondB<Epi, std::void_t<decltype(Epi::kSecond)>> : std::integral_constant<int, Epi::kSecond> {};
struct NoMap {};
template <typename Epi>
using SecondMap = std::conditional_t<SecondB<Epi>::value == kSecondNone, NoMap, CUtensorMap>;

// Epi: struct with
//   template <int CW> __device__ void tile(const MmArgs&, MmTile, int row, int col0, int M, uint32_t taddr,
//                                          bool zero, uint8_t* buf, Pre& pre) const
//   struct Pre; void fetch(Pre&, const MmArgs&, MmTile, int row, int col0, int M) const: what tile reads from memory
//     first, asked for while the tile's products are under way (4 x 256^2 update 81 -> 77 us)
//   static constexpr bool kNarrow, kWide: shapes 0 and 4 (CW = 32 and 64, else 128), and 3, may be used
//   static constexpr bool kChain: MmArgs::chain may be set
//   static constexpr bool kBegin: __device__ void begin(int warp, int warps) const is called once, by every warp
//     of the grid's epilogue warps, while the first tile's products are under way
// tile is called by every thread of an epilogue warp (all 32 lanes,
// converged) for its row and CW columns [col0, col0 + CW); taddr: TMEM address of the warp's
// lanes and columns; zero: the K range is empty, the accumulator holds
// nothing; buf: the warp's staging block.
// CHAIN: sums are bounded by MmArgs::chain.
template <int SH, bool CHAIN, typename Epi>
__global__ void __launch_bounds__(MmShape<SH>::THREADS, 1)
    mm_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b,
              const __grid_constant__ SecondMap<Epi> tm_b2, const __grid_constant__ MmArgs p,
              const __grid_constant__ Epi epi) {
  using S = MmShape<SH>;
  constexpr int SECOND = SecondB<Epi>::value;
  constexpr int ST = S::ST, CG = S::CG;
  extern __shared__ uint8_t mm_smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(mm_smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* bars = reinterpret_cast<uint64_t*>(smem + S::BAR);
  uint64_t *full = bars, *empty = bars + ST, *acc_full = bars + 2 * ST, *acc_empty = acc_full + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  volatile int* abort = reinterpret_cast<volatile int*>(tmem_slot + 1);
  MmPlan* plan = reinterpret_cast<MmPlan*>(tmem_slot + 2);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x / 32, 0), lane = threadIdx.x % 32;  // (uniform)
  const int rank = CG == 2 ? (int)cluster_rank() : 0;
  const int unit = blockIdx.x / CG, n_units = gridDim.x / CG;

  if (threadIdx.x == 0) {
    for (int s = 0; s < ST; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int b = 0; b < 2; ++b) {
      mbar_init(&acc_full[b], 1);
      mbar_init(&acc_empty[b], CG * S::EW);
    }
    *abort = 0;
    fence_barrier_init();
    prefetch_tmap(&tm_a);
    prefetch_tmap(&tm_b);
    if constexpr (SECOND != kSecondNone) prefetch_tmap(&tm_b2);
  }
  if (warp == 1) {
    __syncwarp();
    mm_tmem_alloc<CG>(tmem_slot, S::TCOLS);
  }
  pdl_next();
  // Without device-side counts the schedule is known before the kernels ahead are
  // done, and only the warps that touch global memory wait for them, as late as
  // they can: what an SM does for the first time, from reading the parameters on,
  // takes it long (4 x 256^2 update: 88 us with the wait here, 66 so).
  const bool counted = p.m_dev || p.k_dev;
  if (counted) pdl_wait();
  if (counted && threadIdx.x == 0) {
    const MmGrid<SH> g0(p, cut_rows(p.M, p.m_dev, p.dev_base));
    *plan = mm_plan(g0.per_z * p.nz, n_units, cdiv(cut_rows(p.K, p.k_dev, p.dev_base), 64), p.split, p.n_terms, S::BLOCK);
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // the peer's barriers are initialised
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;  // accumulator (or half) b at columns [b * HN, (b + 1) * HN)

  const int M = cut_rows(p.M, p.m_dev, p.dev_base);
  const int K = cut_rows(p.K, p.k_dev, p.dev_base);
  const MmGrid<SH> grid(p, M);
  const MmPlan pl = counted ? *plan : p.plan;
  // one accumulator at a time: both halves of shape 3, or, with chains, where
  // the sum takes the place of the second
  constexpr bool one = S::ACC == 1 || (CHAIN && S::BN == 256);

  if (warp == 0) {
    if (lane == 0) {
      int it = 0;
      bool ok = true;
      // the copies of a K = 64 step into stage s
      const CUtensorMap* mb = &tm_b;
      auto copy = [&](int s, int ma, int nb, int k, int za, int zb, bool first) {
        if (rank == 0) mbar_expect_tx(&full[s], CG * (S::AB + S::NH * (S::BR < 64 && !p.b_mn ? S::BR * 128 : S::BB)));
        uint8_t* sa = smem + S::A + s * S::AB;
        uint8_t* sb = smem + S::B + s * S::NH * S::BB;
        auto load = [&](const CUtensorMap* map, void* dst, int c0, int c1, int c2) {
          if (CG == 1)
            tma_load_3d(map, &full[s], dst, c0, c1, c2);
          else
            tma_load_3d_pair(map, &full[s], dst, c0, c1, c2);
        };
        if (first) pdl_wait();
        if (p.a_mn) {
          load(&tm_a, sa, ma, k, za);
          load(&tm_a, sa + S::AB / 2, ma + 64, k, za);
        } else {
          load(&tm_a, sa, k, ma, za);
        }
#pragma unroll
        for (int h = 0; h < S::NH; ++h) {
          uint8_t* dst = sb + h * S::BB;
          const int n = nb + h * S::HN;
          if constexpr (SECOND == kSecondHalves) {
            load(&tm_b, dst, k, n / 2, zb);
            load(&tm_b2, dst + S::BR * 64, k, n / 2, zb);
          } else if (p.b_mn) {
            load(mb, dst, n, k, zb);
            if (S::BR > 64) load(mb, dst + S::BB / 2, n + 64, k, zb);
          } else {
            load(mb, dst, k, n, zb);
          }
        }
      };
      for (int t = unit; ok && t < pl.items; t += n_units) {
        const MmItem x = mm_item(pl, t, K);
        const MmTile w = grid.at(p, x.tile);
        const int ma = w.m0 + rank * 128, nb = w.n0 + rank * S::BR;
        for (int term = 0; ok && term < p.n_terms; ++term) {
          const int za = w.z + (int)((p.pa >> (4 * term)) & 15u), zb = w.z + (int)((p.pb >> (4 * term)) & 15u);
          if constexpr (SECOND == kSecondTerms) mb = (p.b2 >> term) & 1 ? &tm_b2 : &tm_b;
          int k = x.k0;
          if (!counted && it == 0 && k < x.k1) {  // (apart: a test in the loop costs a long product 3 %)
            copy(0, ma, nb, k, za, zb, true);
            k += 64;
            ++it;
          }
          for (; k < x.k1; k += 64, ++it) {
            const int s = it % ST;
            if (it >= ST && !(ok = mbar_wait(&empty[s], ((it / ST) - 1) & 1, abort, &g_mm_fault))) break;
            copy(s, ma, nb, k, za, zb, false);
          }
        }
      }
      // every stage's last commit has arrived (in a pair, on this CTA's
      // barrier too): none is in flight when the CTA exits
      for (int i = it - ST < 0 ? 0 : it - ST; ok && i < it; ++i)
        ok = mbar_wait(&empty[i % ST], (i / ST) & 1, abort, &g_mm_fault);
      if (!ok) mm_raise(p, 1u, abort);
      if (*abort && rank == 0) {  // let the copies already issued land before the CTA (pair) can exit
        volatile int none = 0;
        volatile unsigned gnone = 0;
        for (int i = it - ST < 0 ? 0 : it - ST; i < it; ++i)
          mbar_wait(&full[i % ST], (i / ST) & 1, &none, &gnone, 100000000ull);
      }
    }
  } else if (warp == 1) {
    if (rank == 0) {
      // The whole warp walks the loop and one elected lane issues: the
      // descriptors stay in uniform registers, where the instruction reads
      // them. Issued from a branch of lane 0, every descriptor moves there
      // first, which left the tensor cores waiting (160 instead of 130 cycles
      // per MMA).
      const uint32_t fmt = p.fp16 ? 0u : 1u;
      const uint32_t id = (1u << 4) | (fmt << 7) | (fmt << 10) | ((p.a_mn ? 1u : 0u) << 15) |
                          ((p.b_mn ? 1u : 0u) << 16) | ((uint32_t)(S::HN >> 3) << 17) | ((uint32_t)(S::BM >> 4) << 24);
      // K-major: a K step of 16 is 32 bytes of the 128-byte rows; MN-major: 16
      // rows of 128 bytes, panels of 64 rows (MN) 8 KB apart
      const uint32_t a_step = (p.a_mn ? 2048 : 32) >> 4, b_step = (p.b_mn ? 2048 : 32) >> 4;
      const uint32_t a_lbo = p.a_mn ? S::AB / 2 : 16, b_lbo = p.b_mn ? S::BB / 2 : 16;
      const uint64_t da0 = desc_sw128(smem_u32(smem + S::A), a_lbo, 1024), db0 = desc_sw128(smem_u32(smem + S::B), b_lbo, 1024);
      const uint32_t td = __shfl_sync(0xffffffffu, tmem, 0);
      int k = 0, stage = 0, phase = 0;  // k: accumulators filled so far
      bool ok = true;
      for (int t = unit; ok && t < pl.items; t += n_units) {
        const MmItem x = mm_item(pl, t, K);
        const int steps = x.k1 > x.k0 ? cdiv(x.k1 - x.k0, 64) * p.n_terms : 0;
        auto wait = [&](uint64_t* bar, int parity) {
          return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort, &g_mm_fault));
        };
        // 4 MMAs of a stage's K = 64 into accumulator (half) h
        auto issue = [&](int st, int b, int h, int first) {
          const uint32_t d = td + S::HN * b;
          const uint64_t da = da0 + st * (S::AB >> 4), db = db0 + (st * S::NH + h) * (S::BB >> 4);
          mma_f16<CG>(d, da, db, id, first ? 0u : 1u);
          mma_f16<CG>(d, da + a_step, db + b_step, id, 1u);
          mma_f16<CG>(d, da + 2 * a_step, db + 2 * b_step, id, 1u);
          mma_f16<CG>(d, da + 3 * a_step, db + 3 * b_step, id, 1u);
        };
        auto advance = [&] {
          stage = stage + 1 == ST ? 0 : stage + 1;
          phase ^= stage == 0;
        };
        int i = 0;
        if (S::NH == 2) {
          // the first half may start while the epilogue reads the second:
          // as many stages as the ring holds, whose second halves follow
          if (k >= 1 && !(ok = wait(&acc_empty[0], (k - 1) & 1))) break;
          tc_fence_after();
          const int ahead = min(steps, ST), stage0 = stage;
          for (; i < ahead; ++i) {
            if (!(ok = wait(&full[stage], phase))) break;
            if (elect_one()) issue(stage, 0, 0, i == 0);
            __syncwarp();
            advance();
          }
          if (!ok || (k >= 1 && !(ok = wait(&acc_empty[1], (k - 1) & 1)))) break;
          tc_fence_after();
          for (int j = 0, st = stage0; j < ahead; ++j) {
            if (elect_one()) {
              issue(st, 1, 1, j == 0);
              commit<CG>(&empty[st]);
            }
            __syncwarp();
            st = st + 1 == ST ? 0 : st + 1;
          }
        }
        do {
          const int end = CHAIN ? chain_end(p, i, steps) : steps, begin = i;
          const int buf = one ? 0 : k & 1, use = one ? k : k >> 1;
          if (S::NH == 1) {
            // the epilogue has read what this accumulator held before
            if (use && !(ok = wait(&acc_empty[buf], (use - 1) & 1))) break;
            tc_fence_after();
          }
          for (; i < end; ++i) {
            if (!(ok = wait(&full[stage], phase))) break;
            if (elect_one()) {
              issue(stage, S::NH == 1 ? buf : 0, 0, S::NH == 1 && i == begin);
              if (S::NH == 2) issue(stage, 1, 1, 0);
              commit<CG>(&empty[stage]);
            }
            __syncwarp();
            advance();
          }
          if (!ok) break;
          if (elect_one()) commit<CG>(&acc_full[buf]);
          __syncwarp();
          ++k;
        } while (CHAIN && i < steps);
      }
      if (!ok && lane == 0) mm_raise(p, 2u, abort);
    }
  } else {
    const int quad = warp & 3, half = (warp - 2) / 4;  // TMEM lanes 32 quad.., columns CW half..
    int k = 0;
    bool ok = true;
    if (!counted && (Epi::kBegin || unit >= pl.items)) pdl_wait();
    if constexpr (Epi::kBegin) epi.begin(blockIdx.x * S::EW + warp - 2, gridDim.x * S::EW);
    auto release = [&](int b) {  // accumulator (half) b may be filled again
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CG == 1)
          mbar_arrive(&acc_empty[b]);
        else
          mbar_arrive_leader(&acc_empty[b]);
      }
    };
    for (int t = unit; ok && t < pl.items; t += n_units) {
      const MmItem x = mm_item(pl, t, K);
      const MmTile w = grid.at(p, x.tile);
      uint8_t* stage = smem + S::STAGE + (warp - 2) * S::STG;
      const int row = rank * 128 + 32 * quad + lane;
      const uint32_t t0 = tmem + S::CW * half + ((uint32_t)(32 * quad) << 16);
      if (!counted && t == unit) pdl_wait();
      typename Epi::Pre pre;
      if (x.block < 0) epi.fetch(pre, p, w, w.m0 + row, w.n0 + S::CW * half, M);
      auto out = [&](int col, uint32_t ta) {
        if constexpr (SECOND == kSecondHalves)
          epi.template tile<S::CW, S::BR>(p, w, w.m0 + row, w.n0 + col, M, ta, x.k1 <= x.k0, stage, pre);
        else if (x.block < 0)
          epi.template tile<S::CW>(p, w, w.m0 + row, w.n0 + col, M, ta, x.k1 <= x.k0, stage, pre);
        else
          store_part<SH>(p, x, w, row, col, M, ta, stage);
      };
      auto wait = [&] {
        const int buf = one ? 0 : k & 1, use = one ? k : k >> 1;
        ok = __all_sync(0xffffffffu, mbar_wait(&acc_full[buf], use & 1, abort, &g_mm_fault));
        tc_fence_after();
        ++k;
        return buf;
      };
      if constexpr (CHAIN) {
        const int steps = x.k1 > x.k0 ? cdiv(x.k1 - x.k0, 64) * p.n_terms : 0;
        const uint32_t sum = t0 + (S::BN == 256 ? 1 : 2) * S::HN;
        int i = 0;
        do {
          const int buf = wait();
          if (!ok) break;
          if (steps) drain<S::CW>(t0 + S::HN * buf, sum, i > 0);
          release(buf);
          i = chain_end(p, i, steps);
        } while (i < steps);
        if (ok) out(S::CW * half, sum);
      } else {
        const int buf = wait();
        if (!ok) break;
#pragma unroll
        for (int h = 0; h < S::NH; ++h) {
          const int b = S::NH == 2 ? h : buf;
          out(S::HN * h + S::CW * half, t0 + S::HN * b);
          release(b);
        }
      }
    }
    if (!ok) mm_raise(p, 8u, abort);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();  // the peer reads this CTA's shared memory and arrives on its barriers until here
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    mm_tmem_dealloc<CG>(tmem, S::TCOLS);
  }
}

// Adds up the ranges of the split tiles in order, and hands 4 columns of a row
// at a time to Epi::quad(row, col, n valid, values). grid (split tiles at
// most, BM / 8), one warp per row.
template <int SH, typename Epi>
__global__ void __launch_bounds__(256) mm_join(const __grid_constant__ MmArgs p, const __grid_constant__ Epi epi, int units) {
  using S = MmShape<SH>;
  __shared__ MmPlan plan;
  pdl_next();
  pdl_wait();
  const int M = cut_rows(p.M, p.m_dev, p.dev_base);
  const MmGrid<SH> grid(p, M);
  const bool counted = p.m_dev || p.k_dev;
  if (counted) {
    if (threadIdx.x == 0)
      plan = mm_plan(grid.per_z * p.nz, units, cdiv(cut_rows(p.K, p.k_dev, p.dev_base), 64), p.split, p.n_terms, S::BLOCK);
    __syncthreads();
  }
  const MmPlan pl = counted ? plan : p.plan;
  const int tile = pl.full + blockIdx.x;
  if (tile >= pl.total) return;
  const MmTile w = grid.at(p, tile);
  const int r = blockIdx.y * 8 + threadIdx.x / 32, row = w.m0 + r;
  if (row >= M) return;
  const float* src = p.part + ((int64_t)blockIdx.x * pl.s * S::BM + r) * S::BN;
  for (int c = threadIdx.x % 32 * 4; c < S::BN; c += 128) {
    const int n = p.N - (w.n0 + c);
    if (n <= 0) break;
    float4 v = *reinterpret_cast<const float4*>(src + c);
#pragma unroll 4
    for (int s = 1; s < pl.s; ++s) {
      const float4 x = *reinterpret_cast<const float4*>(src + (int64_t)s * S::BM * S::BN + c);
      v = make_float4(v.x + x.x, v.y + x.y, v.z + x.z, v.w + x.w);
    }
    epi.quad(row, w.n0 + c, min(4, n), v);
  }
}

// ---- host side --------------------------------------------------------------

// 3-D operand view: rows x cols with cols contiguous, row stride ld and z
// stride zs (elements, multiples of 8; 16-byte aligned base)
struct Operand {
  const void* p;
  int64_t rows, cols, ld, nz, zs;
  int mn;  // stored MN-major (rows = K, cols = MN) instead of K-major (rows = MN, cols = K)
};

inline int mm_units(int sh) { return sh == 2 || sh == 3 || sh == 5 ? sm_count() / 2 : sm_count(); }

// Estimated time (us) of a product in a shape: waves of tiles (the last one
// split where allowed), each K / 64 steps and a gap, and the last tile's
// epilogue. The constants are measured on a B200: a step of the pair's tile
// takes 0.385 us, of its 512-wide one 0.70, of the others 0.28, 0.22 and 0.18.
template <int SH>
double mm_time(const MmArgs& p) {
  constexpr double step = SH == 3 ? 0.70 : SH == 2 ? 0.385 : SH == 1 ? 0.28 : SH == 4 ? 0.22 : 0.18;
  constexpr double gap = SH == 3 ? 3.0 : 0.5, tail = SH == 3 ? 8.0 : SH == 2 ? 5.5 : SH == 1 ? 4.3 : SH == 4 ? 2.3 : 1.2;
  const MmGrid<SH> g(p, p.M);
  const int units = mm_units(SH), ks = cdiv(p.K, 64);
  const MmPlan pl = mm_plan(g.per_z * p.nz, units, ks, p.split, p.n_terms, MmShape<SH>::BLOCK);
  double t = (pl.full / units + (pl.full % units ? 1 : 0)) * (ks * p.n_terms * step + gap);
  const int split = pl.items - pl.full;
  if (split) t += cdiv(split, units) * (cdiv(ks, pl.s) * p.n_terms * step + gap) + split * step * MmShape<SH>::BLOCK / 1024;
  return t + tail;
}

// whether mm_plan may split anything, whatever the device-side counts
inline int mm_ranges(const MmArgs& p) {
  const int ks = cdiv(p.K, 64);
  return !p.split ? 1 : std::min(32, p.split == 2 ? std::min(ks, ks * p.n_terms / 8) : ks / 8);
}
inline bool joins(const MmArgs& p) { return mm_ranges(p) > 1; }

// fp32 elements of MmArgs::part for a product of at most these sizes: mm_plan
// splits fewer tiles than units, each into as many ranges as K's steps allow
// (32 at most), 4 waves of ranges at most
template <int SH>
int64_t mm_part_blocks(const MmArgs& p) {
  const int64_t tiles = (int64_t)cdiv(p.M, MmShape<SH>::BM) * cdiv(p.N, MmShape<SH>::BN) * std::max(p.nz, 1);
  const int64_t units = mm_units(SH), ranges = mm_ranges(p);
  return std::min(4 * units, std::min(tiles, units - 1) * ranges) * MmShape<SH>::BM * MmShape<SH>::BN;
}
inline int64_t mm_part_floats(const MmArgs& p) {
  if (!joins(p)) return 0;
  return std::max({mm_part_blocks<0>(p), mm_part_blocks<1>(p), mm_part_blocks<2>(p), mm_part_blocks<3>(p), mm_part_blocks<4>(p)});
}

template <int SH, typename Epi>
cudaError_t launch_join(const MmArgs& p, const Epi& epi, int units, cudaStream_t s, decltype(&Epi::quad)) {
  using S = MmShape<SH>;
  const MmGrid<SH> g(p, p.M);
  // with counts the device may have fewer tiles than the host's sizes say, never more
  const int tail = p.m_dev || p.k_dev ? std::min(g.per_z * p.nz, units - 1) : p.plan.s > 1 ? p.plan.total - p.plan.full : 0;
  if (tail < 1) return cudaSuccess;
  return launch_pdl(mm_join<SH, Epi>, dim3(tail, S::BM / 8), 256, 0, 1, s, p, epi, units);
}
template <int SH, typename Epi>
cudaError_t launch_join(const MmArgs&, const Epi&, int, cudaStream_t, ...) {
  return cudaErrorInvalidValue;  // an epilogue without quad() cannot be split
}

// b2: the second map's operand (Epi::kSecond; kSecondHalves: N is set here).
template <int SH, bool CHAIN = false, typename Epi>
cudaError_t launch_mm_sh(MmArgs p, const Operand& a, const Operand& b, const Epi& epi, cudaStream_t s,
                         const Operand* b2 = nullptr) {
  if constexpr (Epi::kChain && !CHAIN && SH != 3) {
    if (p.chain) return launch_mm_sh<SH, true>(p, a, b, epi, s, b2);
  }
  using S = MmShape<SH>;
  constexpr int SECOND = SecondB<Epi>::value;
  const int br = SECOND == kSecondHalves ? S::BR / 2 : S::BR;
  CUtensorMap ta, tb;
  SecondMap<Epi> tb2;
  if (!sm100::make_operand_map(&ta, a.p, a.rows, a.cols, a.ld, a.nz, a.zs, a.mn ? 64 : 128) ||
      !sm100::make_operand_map(&tb, b.p, b.rows, b.cols, b.ld, b.nz, b.zs, b.mn ? 64 : br))
    return cudaErrorInvalidValue;
  if constexpr (SECOND != kSecondNone) {
    if (!b2 || b2->mn != b.mn ||
        !sm100::make_operand_map(&tb2, b2->p, b2->rows, b2->cols, b2->ld, b2->nz, b2->zs, b2->mn ? 64 : br))
      return cudaErrorInvalidValue;
  }
  if (SECOND == kSecondHalves) {
    if (b.mn || p.split) return cudaErrorInvalidValue;
    p.N = cdiv((int)b.rows, br) * S::BR;
  }
  cudaError_t e = set_smem_once(mm_kernel<SH, CHAIN, Epi>, S::SMEM);
  if (e != cudaSuccess) return e;
  const int64_t m = cdiv(p.M, S::BM), n = cdiv(p.N, S::BN);
  const int64_t tiles = (p.sym ? m * (m + 1) / 2 : m * n) * p.nz;
  if (tiles > 0x1ffffff) return cudaErrorInvalidValue;
  const int units = p.split ? mm_units(SH) : (int)std::min<int64_t>(tiles, mm_units(SH));
  // (on the device the schedule of a split product takes some 2 us, of every CTA of the join as well)
  if (!p.m_dev && !p.k_dev) p.plan = mm_plan((int)tiles, units, cdiv(p.K, 64), p.split, p.n_terms, S::BLOCK);
  e = launch_pdl(mm_kernel<SH, CHAIN, Epi>, dim3((unsigned)(units * S::CG)), S::THREADS, S::SMEM, S::CG, s, ta, tb, tb2, p, epi);
  if (e != cudaSuccess || !joins(p)) return e;
  return launch_join<SH, Epi>(p, epi, units, s, nullptr);
}

// the shape that launch_mm takes
template <typename Epi>
int mm_choose(const MmArgs& p) {
  const double t2 = mm_time<2>(p), t1 = mm_time<1>(p);
  if (Epi::kNarrow) {
    MmArgs q = p;
    q.sym = 0;
    const double t4 = mm_time<4>(q), t0 = mm_time<0>(q);
    if (std::min(t0, t4) < std::min(t1, t2)) return t0 <= t4 ? 0 : 4;
  }
  if (Epi::kWide && !p.chain && mm_time<3>(p) < std::min(t1, t2)) return 3;
  return t2 <= t1 ? 2 : 1;
}

template <typename Epi>
cudaError_t launch_mm(MmArgs p, const Operand& a, const Operand& b, const Epi& epi, cudaStream_t s,
                      const Operand* b2 = nullptr) {
  p.a_mn = a.mn;
  p.b_mn = b.mn;
  if (p.nz < 1) p.nz = 1;
  if (p.n_terms < 1) p.n_terms = 1;
  if (p.M < 1 || p.N < 1 || p.K < 1 || (joins(p) && !p.part)) return cudaErrorInvalidValue;
  const int shape = mm_choose<Epi>(p);
  if constexpr (Epi::kNarrow) {
    if (shape == 0 || shape == 4) p.sym = 0;  // not square: every tile is computed
    if (shape == 0) return launch_mm_sh<0>(p, a, b, epi, s, b2);
    if (shape == 4) return launch_mm_sh<4>(p, a, b, epi, s, b2);
  }
  if constexpr (Epi::kWide) {
    if (shape == 3) return launch_mm_sh<3>(p, a, b, epi, s, b2);
  }
  return shape == 2 ? launch_mm_sh<2>(p, a, b, epi, s, b2) : launch_mm_sh<1>(p, a, b, epi, s, b2);
}

// Kernels of launch_mm without device-side counts: the product's, and the join's where tiles are split.
template <typename Epi>
int mm_launches(MmArgs p, bool a_mn, bool b_mn) {
  p.a_mn = a_mn;
  p.b_mn = b_mn;
  auto split = [&](auto shape) {
    constexpr int SH = decltype(shape)::value;
    const MmGrid<SH> g(p, p.M);
    return mm_plan(g.per_z * p.nz, mm_units(SH), cdiv(p.K, 64), p.split, p.n_terms, MmShape<SH>::BLOCK).s > 1;
  };
  switch (mm_choose<Epi>(p)) {
    case 0: return 1 + split(std::integral_constant<int, 0>());
    case 1: return 1 + split(std::integral_constant<int, 1>());
    case 2: return 1 + split(std::integral_constant<int, 2>());
    case 3: return 1 + split(std::integral_constant<int, 3>());
    default: return 1 + split(std::integral_constant<int, 4>());
  }
}

}  // namespace
}  // namespace mm
}  // namespace llattn
