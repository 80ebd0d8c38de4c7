// The matrix product under the fine-tuning operators: D = A B^T in bf16 with fp32 accumulators in TMEM, persistent and
// warp-specialised, with the operator's own work as its epilogue.
//
//   warp 0        streams both operands through a ring of 64-deep K blocks by TMA (128-byte swizzle)
//   warp 1        issues tcgen05.mma into one of two 256-column TMEM accumulators
//   warps 2-9     drain the other accumulator: thread = row, two warps per 32-lane quadrant, each half of the columns
//
// Either operand may lie in memory with its K dimension innermost (K-major) or with its M / N dimension innermost
// (MN-major), so the products of a backward pass read the forward pass's tensors as they are. Pairs of blocks
// (CG = 2) work on one 256 x 256 tile: each block stages its 128 rows of A and its 128 of B's 256 rows, half of what a
// block working alone has to stage per multiplication, and the pair's first block issues the MMAs for both.
// Rows (M) and depth (K) may be cut by counts that only the device knows.
//
// Every wait is bounded (umma::mbar_wait); after a timeout the kernel records it in the status word, frees its TMEM and
// ends.
#pragma once
#include <algorithm>
#include <atomic>
#include "layout.h"
#include "umma.cuh"

namespace asrn {
namespace gemm {

constexpr int kBM = 128, kBN = 256, kBK = 64;
constexpr int kEpiWarps = 8;
constexpr int kThreads = (2 + kEpiWarps) * 32;
constexpr int kBytesA = kBM * 128;                       // one block's share of a stage
template <int CG> constexpr int bytes_b() { return kBN / CG * 128; }
template <int CG> constexpr int stage_bytes() { return kBytesA + bytes_b<CG>(); }
template <int CG> constexpr int stages() { return CG == 1 ? 4 : 6; }
template <int CG> constexpr size_t smem_bytes() { return 1024 + (size_t)stages<CG>() * stage_bytes<CG>() + 256; }

struct Shape {
  int M, N, K;             // bounds known to the host
  const int* m_dev;        // rows that count: min(M, *m_dev - m_off), or null
  int m_off;
  const int* k_dev;        // the same for K
  int k_off;
  int splits;              // parts of K, each with an output of its own
  int group;               // M tiles walked before the next N tile
  int* status;
};

struct Tile {
  int m, n, sp;
};

ASRN_DEV int cut(int most, const int* dev, int off) {
  if (!dev) return most;
  const int n = *dev - off;
  return n < 0 ? 0 : n < most ? n : most;
}

ASRN_DEV Tile tile_at(int t, int mt, int nt, int group) {
  Tile r;
  r.sp = t / (mt * nt);
  const int u = t - r.sp * mt * nt;
  const int first = u / (group * nt) * group;
  const int rows = min(group, mt - first);
  const int v = u - first * nt;
  r.m = first + v % rows;
  r.n = v / rows;
  return r;
}

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

// Epi: struct with a Params type, a constructor (Params, row, rows, column, tile's n index, split, warp half) and
// chunk(float v[32], column) for four chunks of 32 columns, then finish().
template <int CG, bool AMn, bool BMn, class Epi>
__global__ void __launch_bounds__(kThreads, 1)
k_gemm(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, const Shape s,
       const typename Epi::Params p) {
  using namespace umma;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  uint8_t* sm = smem_raw + (((raw + 1023) & ~1023u) - raw);
  constexpr int kS = stages<CG>(), kStageB = bytes_b<CG>();
  uint8_t* sA = sm;
  uint8_t* sB = sm + kS * kBytesA;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + kS * kStageB);
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
      mbar_init(tempty + i, CG * kEpiWarps);
    }
    fence_mbar_init();
    prefetch_tensormap(&map_a);
    prefetch_tensormap(&map_b);
  }
  if (wid == 1) alloc<CG>(tmem_s);
  tc_fence_before();
  __syncthreads();
  if (CG == 2) cluster_sync();
  tc_fence_after();
  const uint32_t tmem = *tmem_s;

  const int M = cut(s.M, s.m_dev, s.m_off), K = cut(s.K, s.k_dev, s.k_off);
  const int mt = (M + kBM * CG - 1) / (kBM * CG), nt = (s.N + kBN - 1) / kBN;
  const int kblocks = (K + kBK - 1) / kBK;
  const int tiles = mt * nt * s.splits;
  const int first = blockIdx.x / CG, step = gridDim.x / CG;

  if (wid == 0) {
    if (lane == 0) {                                    // operand producer
      int it = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step) {
        const Tile u = tile_at(t, mt, nt, s.group);
        const int m0 = (u.m * CG + (int)rank) * kBM, n0 = u.n * kBN + (int)rank * (kBN / CG);
        const int k0 = (int)((int64_t)kblocks * u.sp / s.splits), k1 = (int)((int64_t)kblocks * (u.sp + 1) / s.splits);
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int st = it % kS;
          if (it >= kS && !(ok = mbar_wait(empty + st, ((it / kS) - 1) & 1, s.status))) break;
          if (rank == 0) mbar_expect_tx(full + st, (uint32_t)(CG * stage_bytes<CG>()));
          const uint32_t bar = CG == 1 ? smem_u32(full + st) : peer_u32(full + st, 0);
          if (AMn) {
#pragma unroll
            for (int i = 0; i < kBM / 64; ++i)
              load_box<CG>(sA + st * kBytesA + i * 8192, &map_a, m0 + i * 64, kb * kBK, bar);
          } else {
            load_box<CG>(sA + st * kBytesA, &map_a, kb * kBK, m0, bar);
          }
          if (BMn) {
#pragma unroll
            for (int i = 0; i < kBN / CG / 64; ++i)
              load_box<CG>(sB + st * kStageB + i * 8192, &map_b, n0 + i * 64, kb * kBK, bar);
          } else {
            load_box<CG>(sB + st * kStageB, &map_b, kb * kBK, n0, bar);
          }
        }
      }
    }
  } else if (wid == 1) {
    if (lane == 0 && rank == 0) {                       // MMA issuer, for both blocks of a pair
      constexpr uint32_t idesc = idesc_bf16(kBM * CG, kBN) | (AMn ? 1u << 15 : 0u) | (BMn ? 1u << 16 : 0u);
      int it = 0, jt = 0;
      bool ok = true;
      for (int t = first; t < tiles && ok; t += step, ++jt) {
        const Tile u = tile_at(t, mt, nt, s.group);
        const int k0 = (int)((int64_t)kblocks * u.sp / s.splits), k1 = (int)((int64_t)kblocks * (u.sp + 1) / s.splits);
        const int b = jt & 1;
        if (jt >= 2 && !(ok = mbar_wait(tempty + b, ((jt >> 1) - 1) & 1, s.status))) break;
        tc_fence_after();
        for (int kb = k0; kb < k1; ++kb, ++it) {
          const int st = it % kS;
          if (!(ok = mbar_wait(full + st, (it / kS) & 1, s.status))) break;
          tc_fence_after();
          const uint32_t a0 = smem_u32(sA + st * kBytesA), b0 = smem_u32(sB + st * kStageB);
#pragma unroll
          for (int q = 0; q < kBK / 16; ++q)
            mma<CG>(tmem + (uint32_t)(b * kBN), AMn ? desc_mn_sw128(a0 + q * 2048, 8192) : desc_sw128(a0 + q * 32),
                    BMn ? desc_mn_sw128(b0 + q * 2048, 8192) : desc_sw128(b0 + q * 32), idesc,
                    (kb > k0 || q > 0) ? 1u : 0u);
          commit<CG>(empty + st);
        }
        commit<CG>(tfull + b);
      }
    }
  } else {                                              // epilogue
    const int q4 = wid & 3, half = (wid - 2) >> 2;
    const uint32_t trow = tmem + ((uint32_t)(q4 * 32) << 16) + (uint32_t)(half * (kBN / 2));
    int jt = 0;
    for (int t = first; t < tiles; t += step, ++jt) {
      const Tile u = tile_at(t, mt, nt, s.group);
      const bool none = (int64_t)kblocks * u.sp / s.splits == (int64_t)kblocks * (u.sp + 1) / s.splits;
      const int b = jt & 1;
      if (!mbar_wait(tfull + b, (jt >> 1) & 1, s.status)) break;
      tc_fence_after();
      const int c0 = u.n * kBN + half * (kBN / 2);
      Epi e(p, (u.m * CG + (int)rank) * kBM + q4 * 32 + lane, M, c0, s, u, half);
#pragma unroll 1
      for (int ch = 0; ch < kBN / 64; ++ch) {
        float v[32];
        tmem_ld32(trow + (uint32_t)(b * kBN + ch * 32), v);
        if (ch == kBN / 64 - 1) {                       // the accumulator is read: the next product may have it
          tc_fence_before();
          __syncwarp();
          if (lane == 0) {
            if (CG == 1)
              mbar_arrive(tempty + b);
            else
              asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(peer_u32(tempty + b, 0)) : "memory");
          }
        }
        if (none) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = 0.f;
        }
        e.chunk(v, c0 + ch * 32);
      }
      e.finish();
    }
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

ASRN_DEV uint4 pack8(const float* v) {
  return make_uint4(umma::pack_bf16x2(v[0], v[1]), umma::pack_bf16x2(v[2], v[3]), umma::pack_bf16x2(v[4], v[5]),
                    umma::pack_bf16x2(v[6], v[7]));
}

// fp32 sums of one part of K: out[split][row][column] (N a multiple of 8), stored or added to what is there.
struct StoreF32 {
  struct Params {
    float* out;
    int add;
  };
  float* at;
  int N;
  bool on, add;
  ASRN_DEV StoreF32(const Params& p, int row, int rows, int, const Shape& s, const Tile& u, int)
      : at(p.out + ((int64_t)u.sp * s.M + row) * s.N), N(s.N), on(row < rows), add(p.add != 0) {}
  ASRN_DEV void chunk(const float* v, int c) {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < 32; i += 4)
      if (c + i < N) {
        float4* o = reinterpret_cast<float4*>(at + c + i);
        float4 x = make_float4(v[i], v[i + 1], v[i + 2], v[i + 3]);
        if (add) {
          const float4 y = *o;
          x = make_float4(x.x + y.x, x.y + y.y, x.z + y.z, x.w + y.w);
        }
        *o = x;
      }
  }
  ASRN_DEV void finish() {}
};

// bf16(sum + bias): out[row][column] (N a multiple of 8).
struct StoreBf16 {
  struct Params {
    __nv_bfloat16* out;
    const __nv_bfloat16* bias;
  };
  const Params& p;
  __nv_bfloat16* at;
  int N;
  bool on;
  ASRN_DEV StoreBf16(const Params& pp, int row, int rows, int, const Shape& s, const Tile&, int)
      : p(pp), at(pp.out + (int64_t)row * s.N), N(s.N), on(row < rows) {}
  ASRN_DEV void chunk(float* v, int c) {
    if (!on) return;
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      if (c + i < N) {
        if (p.bias) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[i + j] += __bfloat162float(p.bias[c + i + j]);
        }
        *reinterpret_cast<uint4*>(at + c + i) = pack8(v + i);
      }
  }
  ASRN_DEV void finish() {}
};

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

inline int tiles_of(int64_t M, int64_t N, int cg) {
  return (int)(((M + kBM * cg - 1) / (kBM * cg)) * ((N + kBN - 1) / kBN));
}

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

template <int CG, bool AMn, bool BMn, class Epi>
int launch_cg(const void* A, int64_t pitch_a, const void* B, int64_t pitch_b, const Shape& s,
              const typename Epi::Params& p, cudaStream_t stream) {
  CUtensorMap ma, mb;
  if (!bind_context()) return ASRN_ERR_CUDA;
  if (!operand_map(&ma, A, AMn, s.M, s.K, pitch_a, kBM) || !operand_map(&mb, B, BMn, s.N, s.K, pitch_b, kBN / CG))
    return ASRN_ERR_CUDA;
  auto kernel = k_gemm<CG, AMn, BMn, Epi>;
  constexpr size_t smem = smem_bytes<CG>();
  static std::atomic<uint64_t> ready{0};                  // devices that know the kernel's shared memory
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return ASRN_ERR_CUDA;
  if (dev > 63 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem) != cudaSuccess)
      return ASRN_ERR_CUDA;
    if (dev <= 63) ready.fetch_or(1ull << dev, std::memory_order_release);
  }
  const int64_t tiles = (int64_t)tiles_of(s.M, s.N, CG) * s.splits;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(std::min<int64_t>(tiles, sm_count() / CG) * CG));
  cfg.blockDim = dim3(kThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = CG;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = CG == 1 ? 0 : 1;
  return cudaLaunchKernelEx(&cfg, kernel, ma, mb, s, p) == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
}

// Blocks in pairs unless one block's 128 rows hold all of M.
inline int pair_for(int64_t M) { return M > kBM ? 2 : 1; }

template <bool AMn, bool BMn, class Epi>
int launch(const void* A, int64_t pitch_a, const void* B, int64_t pitch_b, const Shape& s,
           const typename Epi::Params& p, cudaStream_t stream) {
  return pair_for(s.M) == 2 ? launch_cg<2, AMn, BMn, Epi>(A, pitch_a, B, pitch_b, s, p, stream)
                            : launch_cg<1, AMn, BMn, Epi>(A, pitch_a, B, pitch_b, s, p, stream);
}

// Parts of K that give every SM a tile, each of 8 K blocks at least.
inline int splits_for(int64_t M, int64_t N, int64_t K) {
  const int cg = pair_for(M);
  const int tiles = std::max(1, tiles_of(M, N, cg)), slots = sm_count() / cg;
  const int64_t most = std::max<int64_t>(1, (K + kBK - 1) / kBK / 8);
  return (int)std::max<int64_t>(1, std::min<int64_t>(slots / tiles, most));
}

}  // namespace gemm
}  // namespace asrn
