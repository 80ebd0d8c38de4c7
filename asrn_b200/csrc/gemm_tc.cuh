// The matrix product under the fine-tuning operators: D = A B^T in bf16 with fp32 accumulators in TMEM, persistent and
// warp-specialised, with the operator's own work as its epilogue.
//
//   warp 0        streams both operands through a ring of 64-deep K blocks by TMA (128-byte swizzle)
//   warp 1        issues tcgen05.mma into one of two 256-column TMEM accumulators
//   warps 2-9     drain the other accumulator: thread = row, two warps per 32-lane quadrant, each half of the columns,
//   (or 2-17)     32 at a time (an epilogue that computes much: four warps, each a quarter); bf16 results leave by TMA
//                 through 2 KB pieces of shared memory (direct stores, a row's 16 bytes per lane, touch 32 half-written
//                 sectors each)
//
// Either operand may lie in memory with its K dimension innermost (K-major) or with its M / N dimension innermost
// (MN-major), so the products of a backward pass read the forward pass's tensors as they are. Pairs of blocks
// (CG = 2) work on one 256 x 256 tile: each block stages its 128 rows of A and its 128 of B's 256 rows, half of what a
// block working alone has to stage per multiplication, and the pair's first block issues the MMAs for both.
// Rows (M) and depth (K) may be cut by counts that only the device knows.
//
// Products with few tiles or a last round that leaves many SMs idle are walked in equal shares instead (`shares`): the
// clusters stand side by side in groups, one for each tile of N, and each group takes the same number of K blocks of the
// M tiles laid end to end, so that the blocks that read the same part of A do so together. A share's pieces of tiles go
// to fp32 slots that k_join adds up in order.
//
// Measured: the four products of the head at 16384 x 50304 x 768 take 0.81 to 0.92 ms each, 1.38 to 1.56 PFLOP/s, 0.82 to
// 0.93 of cuBLAS's measured burst; the whole operator 5.48 ms with blocks working alone, 5.06 in pairs. dh's product there:
// 1.26 ms by whole tiles (1.3 rounds), 0.91 in shares. Stage counts: what shared memory holds beside the results' pieces.
//
// An operand that was rounded to bf16 can be given as two, the rounded values and what the rounding took, stacked in one
// tensor: the product then runs over K twice (`second_pass`), the second time on the remainders. Operators do so for few rows,
// where it is cheap: a weight's gradient, a sum over these rows, would hold one rounding error for nearly all of its own,
// where many rows average them. Results by row (the sums run over a width or the vocabulary) gain a factor of 1.4 in the
// 2-norm at any number of rows; they come along.
//
// Every wait is bounded; after a timeout the kernel records it in the status word, waits (bounded, too) for the copies and
// the multiplications that it has under way, frees its TMEM and ends. What the word holds from earlier calls stops no later one.
#pragma once
#include <algorithm>
#include <atomic>
#include "layout.h"
#include "umma.cuh"

namespace asrn {
namespace gemm {

constexpr int kBM = 128, kBN = 256, kBK = 64;
template <class Epi> constexpr int threads_of() { return (2 + Epi::kWarps) * 32; }
constexpr int kBytesA = kBM * 128;                       // one block's share of a stage
template <int CG> constexpr int bytes_b() { return kBN / CG * 128; }
template <int CG> constexpr int stage_bytes() { return kBytesA + bytes_b<CG>(); }
// Pieces of shared memory for results: two per warp of eight; sixteen warps share as many unless the epilogue has two
// results (kOwn = 2), which costs a stage.
template <int CG, class Epi> constexpr int stages() {
  return (CG == 1 ? 4 : 6) - (Epi::kWarps * Epi::kOwn > 16) - (Epi::kTable > 0);
}
constexpr int kPiece = 32 * 64;                          // 32 rows x 32 bf16 columns, 64-byte swizzle
template <int CG, class Epi> constexpr size_t smem_bytes() {
  return 1024 + (size_t)stages<CG, Epi>() * stage_bytes<CG>() + Epi::kWarps * Epi::kOwn * kPiece + Epi::kTable + 256;
}

struct Shape {
  int M, N, K;             // bounds known to the host
  const int* m_dev;        // rows that count: min(M, *m_dev - m_off), or null
  int m_off;
  const int* k_dev;        // the same for K
  int k_off;
  int shares;              // groups of clusters that walk equal shares, or 0: whole tiles
  int group;               // whole tiles: M tiles walked before the next N tile
  int* status;
  int second_pass;         // 1: K is walked again with the operands' outer coordinates moved by these
  int a_step, b_step;
};

struct Tile {
  int m, n, k0, k1;        // K blocks [k0, k1)
  int slot;                // of the fp32 pieces
};

ASRN_DEV int cut(int most, const int* dev, int off) {
  if (!dev) return most;
  const int n = *dev - off;
  return n < 0 ? 0 : n < most ? n : most;
}

// Shares of a walk over mt x kblocks blocks where `most` groups stand: 8 blocks each at least, but one per M tile. From
// the counts that the device knows: rows left out change no sum's order.
__host__ ASRN_DEV int shares_of(int64_t mt, int64_t kblocks, int most) {
  const int64_t n = mt * kblocks / 8 > mt ? mt * kblocks / 8 : mt;
  return n < 1 ? 1 : n < most ? (int)n : most;
}
// The first of `shares` shares of mt x kblocks K blocks that holds block u, and a share's first block.
__host__ ASRN_DEV int64_t share_of(int64_t u, int64_t all, int64_t shares) { return ((u + 1) * shares - 1) / all; }
__host__ ASRN_DEV int64_t share_begin(int64_t g, int64_t all, int64_t shares) { return all * g / shares; }

// A cluster's tiles, the same sequence for each of its warps.
struct Walk {
  int mt, nt, kblocks, group, at, step, share;
  int64_t u, end;
  ASRN_DEV Walk(const Shape& s, int M, int K, int cg, int cluster, int clusters)
      : mt((M + kBM * cg - 1) / (kBM * cg)), nt((s.N + kBN - 1) / kBN), kblocks((K + kBK - 1) / kBK), group(s.group),
        at(cluster), step(clusters), share(-1), u(0), end(0) {
    kblocks *= 1 + s.second_pass;
    if (s.shares) {
      share = cluster / nt;
      at = cluster % nt;
      const int64_t all = (int64_t)mt * kblocks;
      const int shares = shares_of(mt, kblocks, s.shares);
      if (share < shares) {
        u = share_begin(share, all, shares);
        end = share_begin(share + 1, all, shares);
      }
    }
  }
  ASRN_DEV bool next(Tile& t) {
    if (share >= 0) {
      if (u >= end) return false;
      t.m = (int)(u / kblocks);
      t.n = at;
      t.k0 = (int)(u - (int64_t)t.m * kblocks);
      t.k1 = (int)min((int64_t)kblocks, t.k0 + (end - u));
      t.slot = (share + t.m) * nt + at;
      u += t.k1 - t.k0;
      return true;
    }
    if (at >= mt * nt) return false;
    const int first = at / (group * nt) * group;
    const int rows = min(group, mt - first), v = at - first * nt;
    t.m = first + v % rows;
    t.n = v / rows;
    t.k0 = 0;
    t.k1 = kblocks;
    t.slot = 0;
    at += step;
    return true;
  }
};

ASRN_DEV uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
ASRN_DEV void cluster_sync() {
  asm volatile("barrier.cluster.arrive.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
}
// The shared::cluster address of `p`'s counterpart in block `rank` of the cluster.
ASRN_DEV uint32_t peer_u32(const void* p, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(umma::smem_u32(p)), "r"(rank));
  return r;
}

// umma::mbar_wait, but for the status word, which is only written: each role of a block ends with the first of its waits
// that runs out, so a block ends after a few limits whatever the word held before. It may lie in the host's memory.
ASRN_DEV bool wait(uint64_t* bar, uint32_t parity, int* status) {
  if (umma::mbar_wait_limit(bar, parity, nullptr, umma::kWaitLimitNs)) return true;
  if (status) {
    *reinterpret_cast<volatile int*>(status) = ASRN_ERR_TIMEOUT;
    __threadfence_system();
  }
  return false;
}

template <int CG> ASRN_DEV void load_box(void* dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  if (CG == 1)
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
        ::"r"(umma::smem_u32(dst)), "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 "
        "[%0], [%1, {%2, %3}], [%4];" ::"r"(umma::smem_u32(dst)),
        "l"(map), "r"(x), "r"(y), "r"(bar)
        : "memory");
}
template <int CG> ASRN_DEV void mma(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  if (CG == 1)
    umma::mma_bf16(d, a, b, idesc, accumulate);
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
        : "memory");
}
// Arrive on `bar` of every block of the pair once the MMAs issued so far have completed.
template <int CG> ASRN_DEV void commit(uint64_t* bar) {
  if (CG == 1)
    umma::mma_commit(bar);
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            umma::smem_u32(bar)),
        "h"((uint16_t)3)
        : "memory");
}
template <int CG> ASRN_DEV void alloc(uint32_t* dst) {
  if (CG == 1) {
    umma::tmem_alloc(dst, 2 * kBN);
    umma::tmem_relinquish();
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(umma::smem_u32(dst)),
                 "r"(2 * kBN)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
}
template <int CG> ASRN_DEV void dealloc(uint32_t taddr) {
  if (CG == 1)
    umma::tmem_dealloc(taddr, 2 * kBN);
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(2 * kBN) : "memory");
}

// Two fp32 values in one register pair: one instruction for both.
struct F2 {
  uint64_t v;
  ASRN_DEV F2() {}
  ASRN_DEV F2(float a, float b) { asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b)); }
  ASRN_DEV explicit F2(float a) : F2(a, a) {}
  ASRN_DEV void get(float& a, float& b) const { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
};
ASRN_DEV F2 fma2(F2 a, F2 b, F2 c) {
  F2 r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}
ASRN_DEV F2 mul2(F2 a, F2 b) {
  F2 r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
ASRN_DEV F2 add2(F2 a, F2 b) {
  F2 r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
// v less what rounding it to bf16 leaves.
ASRN_DEV void remainder(float* v) {
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] -= round_bf16(v[i]);
}
ASRN_DEV float exp2_fast(float x) {                      // 2^x, 2 units in the last place
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

ASRN_DEV uint4 pack8(const float* v) {
  return make_uint4(umma::pack_bf16x2(v[0], v[1]), umma::pack_bf16x2(v[2], v[3]), umma::pack_bf16x2(v[4], v[5]),
                    umma::pack_bf16x2(v[6], v[7]));
}

// A warp's way out for 32 rows x 32 columns of bf16: written to a piece of shared memory, from there by TMA. A piece is
// written again once the copy that read it last is done.
template <int Pieces> struct Out {
  const uint32_t* table;                                 // the epilogue's
  uint8_t* piece;                                        // the warp's own
  int lane, turn;
  ASRN_DEV void put(const CUtensorMap* map, const float* v, int column, int first_row) {
    uint4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = pack8(v + 8 * i);
    put(map, w, column, first_row);
  }
  ASRN_DEV void put(const CUtensorMap* map, const uint4* w, int column, int first_row) {
    uint8_t* at = piece + turn * kPiece;
    turn = (turn + 1) % Pieces;
    if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(Pieces - 1) : "memory");
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i)
      *reinterpret_cast<uint4*>(at + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4)) = w[i];
    umma::fence_proxy_async();
    __syncwarp();
    if (lane == 0) {
      asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.tile.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map),
                   "r"(column), "r"(first_row), "r"(umma::smem_u32(at))
                   : "memory");
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
  }
  ASRN_DEV void drain() {
    if (lane == 0) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
  }
};

// Epi: struct with a Params type, kWarps (8 or 16), kOwn (pieces per warp), kTable (bytes of a table that its fill() makes
// once per block; costs a stage), a constructor (Params, row, rows, shape, tile, the warp's part of the columns) and chunk(v[32],
// column, Out, map_o, map_p), called by whole warps for the tile's chunks of 32 columns, then finish().
template <int CG, bool AMn, bool BMn, class Epi>
__global__ void __launch_bounds__(threads_of<Epi>(), 1)
k_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
       const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_p, const Shape s,
       const typename Epi::Params p) {
  using namespace umma;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sm = smem_raw + (((raw + 1023) & ~1023u) - raw);
  constexpr int kS = stages<CG, Epi>(), kStageB = bytes_b<CG>();
  uint8_t* sA = sm;
  uint8_t* sB = sm + kS * kBytesA;
  uint8_t* sO = sB + kS * kStageB;
  uint32_t* table = reinterpret_cast<uint32_t*>(sO + Epi::kWarps * Epi::kOwn * kPiece);
  uint64_t* full = reinterpret_cast<uint64_t*>(sO + Epi::kWarps * Epi::kOwn * kPiece + Epi::kTable);
  uint64_t* empty = full + kS;
  uint64_t* tfull = empty + kS;
  uint64_t* tempty = tfull + 2;
  uint32_t* tmem_s = reinterpret_cast<uint32_t*>(tempty + 2);

  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const uint32_t rank = CG == 1 ? 0u : cluster_rank();
  if (tid == 0) {
    for (int i = 0; i < kS; ++i) {
      mbar_init(full + i, 1);
      mbar_init(empty + i, 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(tfull + i, 1);
      mbar_init(tempty + i, CG * Epi::kWarps);
    }
    fence_mbar_init();
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_b);
  }
  if (wid == 1) alloc<CG>(tmem_s);
  if constexpr (Epi::kTable > 0) Epi::fill(table, tid, threads_of<Epi>());
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_s;
  wait_previous();                                      // the setup above overlaps the end of the kernel before
  let_next();

  const int M = cut(s.M, s.m_dev, s.m_off), K = cut(s.K, s.k_dev, s.k_off);
  Walk walk(s, M, K, CG, blockIdx.x / CG, gridDim.x / CG);
  Tile u;

  if (wid == 0) {
    if (lane == 0) {                                    // operand producer
      const int kblocks = (K + kBK - 1) / kBK;          // of one pass
      int it = 0;
      bool ok = true;
      while (ok && walk.next(u)) {
        const int m0 = (u.m * CG + (int)rank) * kBM, n0 = u.n * kBN + (int)rank * (kBN / CG);
        for (int kt = u.k0; kt < u.k1; ++kt, ++it) {
          const int again = kt >= kblocks, kb = kt - again * kblocks;
          const int a_at = again * s.a_step, b_at = again * s.b_step;
          const int st = it % kS;
          if (it >= kS && !(ok = wait(empty + st, ((it / kS) - 1) & 1, s.status))) break;
          if (rank == 0) mbar_expect_tx(full + st, (uint32_t)(CG * stage_bytes<CG>()));
          const uint32_t bar = CG == 1 ? smem_u32(full + st) : peer_u32(full + st, 0);
          if (AMn) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i)
              load_box<CG>(sA + st * kBytesA + i * 8192, &map_a, m0 + i * 64, kb * kBK + a_at, bar);
          } else {
            load_box<CG>(sA + st * kBytesA, &map_a, kb * kBK, m0 + a_at, bar);
          }
          if (BMn) {
#pragma unroll
            for (int i = 0; i < kBN / CG / 64; ++i)
              load_box<CG>(sB + st * kStageB + i * 8192, &map_b, n0 + i * 64, kb * kBK + b_at, bar);
          } else {
            load_box<CG>(sB + st * kStageB, &map_b, kb * kBK, n0 + b_at, bar);
          }
        }
      }
      // No block may end with copies under way into its shared memory. The first block's barriers count the pair's; the other
      // one waits for it at the end.
      if (rank == 0)
        for (int i = max(0, it - kS); i < it; ++i)
          if (!mbar_wait_limit(full + i % kS, (i / kS) & 1, nullptr, kWaitLimitNs)) break;
    }
  } else if (wid == 1) {
    if (lane == 0 && rank == 0) {                       // MMA issuer, for both blocks of a pair
      constexpr uint32_t idesc = idesc_bf16(kBM * CG, kBN) | (AMn ? 1u << 15 : 0u) | (BMn ? 1u << 16 : 0u);
      int it = 0, jt = 0;
      bool ok = true;
      for (; ok && walk.next(u); ++jt) {
        const int b = jt & 1;
        if (jt >= 2 && !(ok = wait(tempty + b, ((jt >> 1) - 1) & 1, s.status))) break;
        tc_fence_after();
        for (int kb = u.k0; kb < u.k1; ++kb, ++it) {
          const int st = it % kS;
          if (!(ok = wait(full + st, (it / kS) & 1, s.status))) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + st * kBytesA), b0 = smem_u32(sB + st * kStageB);
#pragma unroll
          for (int q = 0; q < kBK / 16; ++q)
            mma<CG>(tmem + (uint32_t)(b * kBN), AMn ? desc_mn_sw128(a0 + q * 2048, 8192) : desc_sw128(a0 + q * 32),
                    BMn ? desc_mn_sw128(b0 + q * 2048, 8192) : desc_sw128(b0 + q * 32), idesc,
                    (kb > u.k0 || q > 0) ? 1u : 0u);
          commit<CG>(empty + st);
        }
        commit<CG>(tfull + b);
      }
      // Nor with multiplications under way: the last of these barriers follows all of them.
      if (jt > 0) mbar_wait_limit(tfull + ((jt - 1) & 1), ((jt - 1) >> 1) & 1, nullptr, kWaitLimitNs);
    }
  } else {                                              // epilogue
    constexpr int kCols = kBN * 4 / Epi::kWarps, kOwn = Epi::kOwn;
    const int q4 = wid & 3, part = (wid - 2) >> 2;
    Out<kOwn> out{table, sO + (wid - 2) * kOwn * kPiece, lane, 0};
    const uint32_t trow = tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(part * kCols);
    int jt = 0;
    for (; walk.next(u); ++jt) {
      const int b = jt & 1;
      if (!wait(tfull + b, (jt >> 1) & 1, s.status)) break;
      tc_fence_after();
      const int c0 = u.n * kBN + part * kCols;
      Epi e(p, (u.m * CG + (int)rank) * kBM + q4 * 32 + lane, M, s, u, part);
#pragma unroll 1
      for (int ch = 0; ch < kCols / 32; ++ch) {
        float v[32];
        tmem_ld32(trow + (uint32_t)(b * kBN + ch * 32), v);
        if (ch == kCols / 32 - 1) {                       // the accumulator is read: the next product may have it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 1)
              mbar_arrive(tempty + b);
            else
              asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(peer_u32(tempty + b, 0)) : "memory");
          }
        }
        if (u.k0 == u.k1) {                             // no depth at all
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }
        e.chunk(v, c0 + ch * 32, out, &map_o, &map_p);
      }
      e.finish();
    }
    out.drain();
  }
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  if (wid == 1) {
    tc_fence_after();
    dealloc<CG>(tmem);
  }
}

// ---- epilogues that only store -----------------------------------------------------------------------------------------

// v += bias[0 .. min(32, n)), n a multiple of 8.
ASRN_DEV void add_bias(float* v, const __nv_bfloat16* bias, int n) {
#pragma unroll
  for (int i = 0; i < 32; i += 8)
    if (i < n) {
      const uint4 b = __ldg(reinterpret_cast<const uint4*>(bias + i));
      const uint32_t w[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i + 2 * j] += __uint_as_float(w[j] << 16);
        v[i + 2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
      }
    }
}

// The fp32 sums of a piece of a tile, whole, to its slot: by blocks of 32 rows x 32 columns, each as the warp holds it
// (four columns of all 32 rows are 512 neighbouring bytes).
struct StorePiece {
  static constexpr int kWarps = 8, kOwn = 2, kTable = 0;
  struct Params {
    float* slots;
    int tile_rows;
  };
  float* at;
  ASRN_DEV StorePiece(const Params& p, int row, int, const Shape&, const Tile& u, int)
      : at(p.slots + ((int64_t)u.slot * p.tile_rows + (row % p.tile_rows & ~31)) * kBN + (row & 31) * 4 -
           (int64_t)u.n * kBN * 32) {}
  template <class O> ASRN_DEV void chunk(const float* v, int c, O&, const CUtensorMap*, const CUtensorMap*) {
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      *reinterpret_cast<float4*>(at + (int64_t)c * 32 + i * 32) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
  }
  ASRN_DEV void finish() {}
};

// bf16(sum + bias + before): out[row][column] through map_o (N a multiple of 8). before: fp32 (M, N), the sum of what
// came earlier; or, when `after` is given, the sum goes there in fp32 instead.
struct StoreBf16 {
  static constexpr int kWarps = 8, kOwn = 2, kTable = 0;
  struct Params {
    const __nv_bfloat16* bias;
    const float* before;
    float* after;
  };
  const Params& p;
  int64_t at;
  int N, first;
  bool on;
  ASRN_DEV StoreBf16(const Params& pp, int row, int rows, const Shape& s, const Tile&, int)
      : p(pp), at((int64_t)row * s.N), N(s.N), first(row & ~31), on(row < rows) {}
  template <class O> ASRN_DEV void chunk(float* v, int c, O& out, const CUtensorMap* map_o, const CUtensorMap*) {
    if (c >= N) return;
    if (p.bias) add_bias(v, p.bias + c, N - c);
    if (p.before && on) {
#pragma unroll
      for (int i = 0; i < 32; i += 4)
        if (c + i < N) {
          const float4 y = *reinterpret_cast<const float4*>(p.before + at + c + i);
          v[i] += y.x; v[i + 1] += y.y; v[i + 2] += y.z; v[i + 3] += y.w;
        }
    }
    if (p.after) {
      if (on)
#pragma unroll
        for (int i = 0; i < 32; i += 4)
          if (c + i < N) *reinterpret_cast<float4*>(p.after + at + c + i) = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
    } else {
      out.put(map_o, v, c, first);
    }
  }
  ASRN_DEV void finish() {}
};

// The pieces of each tile added up in order and rounded: out[row_of ? row_of[r] : r][c], a warp per 32 rows x 32 columns.
// Positions i < zero_n with pos[i] < 0 get zero rows (whole grid).
struct JoinArgs {
  const float* slots;
  __nv_bfloat16* out;
  int tile_rows;
  const int* row_of;
  const int* pos;
  int64_t zero_n;
};
static __global__ void __launch_bounds__(256) k_join(const Shape s, const JoinArgs a) {
  wait_previous();
  let_next();
  const int M = cut(s.M, s.m_dev, s.m_off), K = cut(s.K, s.k_dev, s.k_off);
  const int mt = (M + a.tile_rows - 1) / a.tile_rows, nt = (s.N + kBN - 1) / kBN;
  const int kblocks = (K + kBK - 1) / kBK * (1 + s.second_pass);
  const int per = a.tile_rows / 32, lane = threadIdx.x & 31;              // blocks of 32 rows of a tile
  const int64_t all = (int64_t)mt * kblocks;
  const int tile = blockIdx.x / per, m = tile / nt, n = tile % nt, part = blockIdx.x % per;
  const int c = n * kBN + (threadIdx.x >> 5) * 32, r = m * a.tile_rows + part * 32 + lane;
  if (m < mt && c < s.N) {
    int g0 = 0, g1 = -1;
    if (kblocks) {
      const int shares = shares_of(mt, kblocks, s.shares);
      g0 = (int)share_of((int64_t)m * kblocks, all, shares);
      g1 = (int)share_of((int64_t)(m + 1) * kblocks - 1, all, shares);
    }
    float v[32] = {};
    for (int g = g0; g <= g1; ++g) {
      const float4* q = reinterpret_cast<const float4*>(a.slots + ((int64_t)((g + m) * nt + n) * a.tile_rows + part * 32) * kBN +
                                                        (threadIdx.x >> 5) * 1024) + lane;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 x = q[i * 32];
        v[4 * i] += x.x; v[4 * i + 1] += x.y; v[4 * i + 2] += x.z; v[4 * i + 3] += x.w;
      }
    }
    if (r < M) {
      __nv_bfloat16* out = a.out + (int64_t)(a.row_of ? a.row_of[r] : r) * s.N + c;
#pragma unroll
      for (int i = 0; i < 32; i += 8)
        if (c + i < s.N) *reinterpret_cast<uint4*>(out + i) = pack8(v + i);
    }
  }
  for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < a.zero_n; i += (int64_t)gridDim.x * 8)
    if (a.pos[i] < 0)
      for (int x = lane * 8; x < s.N; x += 256)
        *reinterpret_cast<uint4*>(a.out + i * s.N + x) = make_uint4(0, 0, 0, 0);
}

// ---- host ---------------------------------------------------------------------------------------------------------------

inline int sm_count() {
  static int n = 0;
  if (n == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) n = 148;
  }
  return n;
}

inline int64_t tiles_m(int64_t M, int cg) { return (M + kBM * cg - 1) / (kBM * cg); }
inline int64_t tiles_n(int64_t N) { return (N + kBN - 1) / kBN; }

// A K-major operand (rows, depth) or an MN-major one (depth, rows), rows of `pitch` elements.
inline bool operand_map(CUtensorMap* map, const void* base, bool mn, int64_t rows, int64_t depth, int64_t pitch,
                        int box_rows) {
  return mn ? make_tmap_bf16(map, base, (uint64_t)rows, (uint64_t)depth, (uint64_t)pitch * 2, 64, kBK)
            : make_tmap_bf16(map, base, (uint64_t)depth, (uint64_t)rows, (uint64_t)pitch * 2, kBK, (uint32_t)box_rows);
}

// The tensor map call needs a current context: a thread gets its device's with its first call here.
inline bool bind_context() {
  static thread_local bool bound = false;
  int dev = 0;
  if (!bound) bound = cudaGetDevice(&dev) == cudaSuccess && cudaSetDevice(dev) == cudaSuccess;
  return bound;
}

// Where an epilogue's bf16 rows go: (rows, columns) of `pitch` elements.
struct Dest {
  void* base;
  int64_t rows, columns, pitch;
};

template <int CG, bool AMn, bool BMn, class Epi>
int launch_cg(const void* A, int64_t pitch_a, const void* B, int64_t pitch_b, const Shape& s,
              const typename Epi::Params& p, const Dest& o, const Dest& q, cudaStream_t stream) {
  CUtensorMap ma, mb, mo, mq;
  if (!bind_context()) return ASRN_ERR_CUDA;
  const int again = s.second_pass;                     // the stacked operand is longer in its outer dimension
  if (!operand_map(&ma, A, AMn, AMn ? s.M : s.M + again * s.a_step, AMn ? s.K + again * s.a_step : s.K, pitch_a, kBM) ||
      !operand_map(&mb, B, BMn, BMn ? s.N : s.N + again * s.b_step, BMn ? s.K + again * s.b_step : s.K, pitch_b, kBN / CG))
    return ASRN_ERR_CUDA;
  mo = mq = ma;                                            // not read where there is no destination
  if ((o.base && !make_tmap_bf16_sw64(&mo, o.base, (uint64_t)o.columns, (uint64_t)o.rows, (uint64_t)o.pitch * 2, 32, 32)) ||
      (q.base && !make_tmap_bf16_sw64(&mq, q.base, (uint64_t)q.columns, (uint64_t)q.rows, (uint64_t)q.pitch * 2, 32, 32)))
    return ASRN_ERR_CUDA;
  auto kernel = k_gemm<CG, AMn, BMn, Epi>;
  constexpr size_t smem = smem_bytes<CG, Epi>();
  static std::atomic<uint64_t> ready{0};                  // devices that know the kernel's shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ASRN_ERR_CUDA;
  if (dev > 63 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return ASRN_ERR_CUDA;
    if (dev <= 63) ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  const int64_t tiles = s.shares ? s.shares * tiles_n(s.N) : tiles_m(s.M, CG) * tiles_n(s.N);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(tiles, sm_count() / CG) * CG));
  cfg.blockDim = dim3(threads_of<Epi>());
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = CG;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG;
  return cudaLaunchKernelEx(&cfg, kernel, ma, mb, mo, mq, s, p) == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
}

// Blocks in pairs unless one block's 128 rows hold all of M.
inline int pair_for(int64_t M) { return M > kBM ? 2 : 1; }

template <bool AMn, bool BMn, class Epi>
int launch(const void* A, int64_t pitch_a, const void* B, int64_t pitch_b, const Shape& s,
           const typename Epi::Params& p, cudaStream_t stream, const Dest& o = {}, const Dest& q = {}) {
  return pair_for(s.M) == 2 ? launch_cg<2, AMn, BMn, Epi>(A, pitch_a, B, pitch_b, s, p, o, q, stream)
                            : launch_cg<1, AMn, BMn, Epi>(A, pitch_a, B, pitch_b, s, p, o, q, stream);
}

// Groups for a walk in shares: as many as the SMs hold and the work fills. shares_for: 0 (whole tiles) unless shares save 40
// K blocks in a row, about 11 us: what the pieces and their joining cost on the device (6 to 8 us) and the host (3 us).
inline int groups_for(int64_t M, int64_t N, int64_t K) {
  return shares_of(tiles_m(M, pair_for(M)), (K + kBK - 1) / kBK,
                   (int)std::max<int64_t>(1, sm_count() / pair_for(M) / tiles_n(N)));
}
inline int shares_for(int64_t M, int64_t N, int64_t K) {
  const int cg = pair_for(M);
  const int64_t slots = sm_count() / cg, nt = tiles_n(N), mt = tiles_m(M, cg), groups = groups_for(M, N, K);
  const int64_t rounds = (mt * nt + slots - 1) / slots, kb = (K + kBK - 1) / kBK;
  return groups * nt <= slots && rounds * kb - mt * kb / groups > 40 ? (int)groups : 0;
}
// The slots' sums to out (contiguous rows of N).
inline int join(const Shape& s, const float* slots, void* out, const int* row_of, const int* pos, int64_t zero_n,
                cudaStream_t stream) {
  const int rows = kBM * pair_for(s.M);
  const int64_t blocks = tiles_m(s.M, pair_for(s.M)) * tiles_n(s.N) * (rows / 32);
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)blocks);
  cfg.blockDim = dim3(256);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const JoinArgs a{slots, reinterpret_cast<__nv_bfloat16*>(out), rows, row_of, pos, zero_n};
  return cudaLaunchKernelEx(&cfg, k_join, s, a) == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
}
// Bytes of a share walk's slots.
inline size_t slot_bytes(int64_t M, int64_t N, int shares) {
  const int cg = pair_for(M);
  return (size_t)(shares + tiles_m(M, cg)) * tiles_n(N) * kBM * cg * kBN * 4;
}

}  // namespace gemm
}  // namespace asrn
