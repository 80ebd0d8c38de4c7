// The matrix product with bias, activation and residual in its epilogue, forward and backward:
//   a = x W^T + b,  y = act(a) + r;  kept: act'(a) in fp16
//   dA = dY act'(a),  dX = dA W,  dW = dA^T x,  db = sum of dA,  dr = dY
// x, W, b bf16; r bf16 or fp32, y of r's type (bf16 without); act: none, gelu (erf), silu, relu.
//
// act'(a) is kept rather than a: it lies in [-0.13, 1.13], where fp16 is off by 2^-11 of it at the most, an eighth of what dA's
// rounding to bf16 takes (a in bf16 would move act'(a) by as much as that), and the backward pass has nothing left to compute.
// dA is rounded once, as operand of both products; up to kTwiceRows rows they take what the rounding took, too.
//
//   k_linear_few   few results: too few tiles of 128 x 256 for the SMs, and with few rows memory bound (the weight is read once,
//                  2 operations a byte and row), so the rows of W are spread over all SMs, sixteen a block with up to 64 rows of
//                  x, K over its warps; mma.sync, whose 16 x 8 tiles fit such rows
//   k_gemm<Fused>  more: tcgen05 products, the rest in the epilogue
//   k_linear_slope backward: dA in bf16 and its columns' sums by 64 rows; memory bound: 32768 x 1536 from bf16 dY 47 us (302 MB,
//                  6.3 TB/s), 32768 x 768 from fp32 dY without a slope 24.5
//   k_gemm x 2     dX, dW (dW in shares of the rows where its tiles are few)
//   k_colsum       db
#include <cuda_fp16.h>
#include "common.cuh"
#include "gemm_tc.cuh"
#include "products.cuh"

namespace asrn {

namespace {

constexpr int kF32 = 0, kBf16 = 1, kNone = 2;            // types of the C interface
constexpr int kGelu = 1, kSilu = 2, kRelu = 3;
constexpr int64_t kTwiceRows = 512;
// Graph replays, us, few | by 128 x 256 tiles: 768 -> 1536, 64 rows 6.8 | 11.0, 213 rows 10.2 | 11.5, 341 rows 11.9 | 11.5;
// 1536 -> 768, 256 rows 9.4 | 15.1, 682 rows 17 | 15; 128 -> 128, 2048 rows 4.2 | 7.3, 8192 rows 14 | 7.5; 4096 -> 512, 384 rows
// 17 | 29, 1024 rows 32 | 29; 768 -> 8192, 32 rows 7.3 | 11, 64 rows 12 | 11. Up to 16 rows the weight's bytes count, which it loads
// faster: 768 -> 50304, 8 rows 15 | 22, 16 rows 21 | 23, 24 rows 33 | 23.
bool few_rows(int64_t N, int64_t n) { return N * n <= 3 << 17 || (N <= 16 && N * n <= 1 << 20); }

ASRN_DEV uint32_t half2_of(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// Of two values: act(a) in place, the slopes as fp16. Large: infinite a give the limits (products with what vanishes take |a| held
// to kLarge), NaN stays; else |a| <= kLarge or NaN.
constexpr float kLarge = 200.f;
template <int Act, bool Large> ASRN_DEV uint32_t activate(float& a0, float& a1) {
  using namespace gemm;
  if constexpr (Act == kGelu) {
    F2 e, q;
    tails(a0, a1, e, q);
    const float m0 = Large ? fminf(fabsf(a0), kLarge) : fabsf(a0), m1 = Large ? fminf(fabsf(a1), kLarge) : fabsf(a1);
    const F2 held = Large ? F2(copysignf(m0, a0), copysignf(m1, a1)) : F2(a0, a1);
    float h0, h1, s0, s1;
    fma2(q, F2(-1.f), F2(0.5f)).get(h0, h1);                                     // 1/2 - q
    const F2 cdf = add2(F2(copysignf(h0, a0), copysignf(h1, a1)), F2(0.5f));
    fma2(mul2(held, F2(0.39894228040143268f)), e, cdf).get(s0, s1);
    fma2(F2(-m0, -m1), q, F2(fmaxf(a0, 0.f), fmaxf(a1, 0.f))).get(a0, a1);
    return half2_of(s0, s1);
  } else if constexpr (Act == kSilu) {
    float* a[2] = {&a0, &a1};
    float s[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float low = Large ? fmaxf(*a[i], -kLarge) : *a[i];
      float p = 1.f + exp2_fast(*a[i] * -1.4426950408889634f);
      asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(p));
      s[i] = p * fmaf(Large ? fminf(low, kLarge) : low, 1.f - p, 1.f);
      *a[i] = low * p;
    }
    return half2_of(s[0], s[1]);
  } else {
    const uint32_t s = half2_of(a0 > 0.f ? 1.f : 0.f, a1 > 0.f ? 1.f : 0.f);
    a0 = a0 < 0.f ? 0.f : a0;
    a1 = a1 < 0.f ? 0.f : a1;
    return s;
  }
}
template <int Act, bool Large, int N> ASRN_DEV void activate_all(float* v, uint32_t* s) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = activate<Act, Large>(v[2 * i], v[2 * i + 1]);
}
// The same for 2 N values.
template <int N> ASRN_DEV void activate(int act, float* v, uint32_t* s) {
  float most = 0.f;
#pragma unroll
  for (int i = 0; i < 2 * N; ++i) most = fmaxf(most, fabsf(v[i]));
  if (act == kRelu)
    activate_all<kRelu, true, N>(v, s);
  else if (most > kLarge)
    act == kGelu ? activate_all<kGelu, true, N>(v, s) : activate_all<kSilu, true, N>(v, s);
  else
    act == kGelu ? activate_all<kGelu, false, N>(v, s) : activate_all<kSilu, false, N>(v, s);
}

// What follows the product.
struct Rest {
  const __nv_bfloat16* bias;                 // or null
  const void* res;
  int act, res_type;
  int keep;                                  // the slopes are wanted
};

// 16 warps: with 8 the epilogue, not the products, sets the pace. 32768 x 768 x 1536 (77 GFLOP; 46 us at the measured burst, a library
// product alone 61.5 us): without anything 65 us, gelu 77, with the slopes kept 85, bf16 residual 80, fp32 106; 32768 x 1536 x 768: 63,
// 70, 76, fp32 residual 82.
struct Fused {
  static constexpr int kWarps = 16, kOwn = 2, kTable = 0;
  using Params = Rest;
  const Params& p;
  int N, first, rows;
  ASRN_DEV Fused(const Params& pp, int r, int m, const gemm::Shape& s, const gemm::Tile&, int)
      : p(pp), N(s.N), first(r & ~31), rows(m) {}

  // v += the residual's 32 x 32 values, brought through the warp's pieces: whole rows of them are read side by side, where each
  // lane's own row would touch 32 half-used sectors at a time.
  template <class O> ASRN_DEV void add_residual(float* v, int c, O& out) {
    const int lane = threadIdx.x & 31;
    if (p.res_type == kF32) {
      const float* res = reinterpret_cast<const float*>(p.res);
      float4 q[8];
      const int col = c + (lane & 7) * 4;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = first + i * 4 + (lane >> 3);
        q[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < rows && col < N) q[i] = __ldg(reinterpret_cast<const float4*>(res + (int64_t)r * N + col));
      }
      uint8_t* room = out.room();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + (lane >> 3);
        *reinterpret_cast<float4*>(room + r * 128 + (((lane & 7) ^ (r & 7)) << 4)) = q[i];
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(room + lane * 128 + ((i ^ (lane & 7)) << 4));
        v[4 * i] += x.x; v[4 * i + 1] += x.y; v[4 * i + 2] += x.z; v[4 * i + 3] += x.w;
      }
    } else {
      const __nv_bfloat16* res = reinterpret_cast<const __nv_bfloat16*>(p.res);
      uint4 q[4];
      const int col = c + (lane & 3) * 8;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = first + i * 8 + (lane >> 2);
        q[i] = make_uint4(0, 0, 0, 0);
        if (r < rows && col < N) q[i] = __ldg(reinterpret_cast<const uint4*>(res + (int64_t)r * N + col));
      }
      uint8_t* room = out.room();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = i * 8 + (lane >> 2);
        *reinterpret_cast<uint4*>(room + r * 64 + (((lane & 3) ^ (r >> 1 & 3)) << 4)) = q[i];
      }
      __syncwarp();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const uint4 x = *reinterpret_cast<const uint4*>(room + lane * 64 + ((i ^ (lane >> 1 & 3)) << 4));
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          v[8 * i + 2 * j] += __uint_as_float(w[j] << 16);
          v[8 * i + 2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
        }
      }
    }
    __syncwarp();                            // the pieces are written again by what follows
  }

  template <class O> ASRN_DEV void chunk(float* v, int c, O& out, const CUtensorMap* map_o, const CUtensorMap* map_p) {
    if (c >= N || first >= rows) return;     // the same for the whole warp
    if (p.bias) gemm::add_bias(v, p.bias + c, N - c);
    if (p.act) {
      uint32_t s[16];
      activate<16>(p.act, v, s);
      if (p.keep) {
        uint4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) w[i] = make_uint4(s[4 * i], s[4 * i + 1], s[4 * i + 2], s[4 * i + 3]);
        out.put(map_p, w, c, first);
      }
    }
    if (p.res_type != kNone) add_residual(v, c, out);
    if (p.res_type == kF32) {
#pragma unroll
      for (int half = 0; half < 32; half += 16) {
        if (c + half >= N) break;
        uint4 w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          w[i] = make_uint4(__float_as_uint(v[half + 4 * i]), __float_as_uint(v[half + 4 * i + 1]),
                            __float_as_uint(v[half + 4 * i + 2]), __float_as_uint(v[half + 4 * i + 3]));
        out.put(map_o, w, c + half, first);
      }
    } else {
      out.put(map_o, v, c, first);
    }
  }
  ASRN_DEV void finish() {}
};

// 16 columns of y for 8 NT rows of x: A = 16 rows of W, B = the rows of x. The order of K inside a tile is free as long as
// A and B agree, so a lane takes 8 neighbouring values (16 bytes) of each operand's row for two multiplications: no shared
// memory, and four lanes read 64 neighbouring bytes. A block's warps take every eighth 32 of K; the blocks of a cluster share K
// where the columns alone leave SMs idle; the sums meet in shared memory, the blocks' through the cluster's. Graph replays at 768 ->
// 1536: 1, 8, 16, 32, 64 rows 3.3, 3.4, 3.9, 4.9, 6.8 us, launch and one round trip to memory (2.4 MB take 0.4).
constexpr int kFewWarps = 8;
ASRN_DEV float2 residual_of(const Rest& p, int64_t at) {
  if (p.res_type == kF32) return __ldg(reinterpret_cast<const float2*>(reinterpret_cast<const float*>(p.res) + at));
  if (p.res_type == kNone) return make_float2(0.f, 0.f);
  const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(reinterpret_cast<const __nv_bfloat16*>(p.res) + at));
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
ASRN_DEV float2 bias_of(const Rest& p, int c) {
  return p.bias ? __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p.bias + c)) : make_float2(0.f, 0.f);
}
// U: steps of K whose loads are under way together, no more than a warp has. Many: more rows than 8 NT, by chunks (blockIdx.y).
template <int NT, int U, bool Many>
__global__ void __launch_bounds__(kFewWarps * 32, 2)
k_linear_few(int all, int n, int d, int split, const __nv_bfloat16* __restrict__ x, const __nv_bfloat16* __restrict__ w,
             const Rest p, void* __restrict__ y, __half* __restrict__ slope) {
  __shared__ float sh[kFewWarps][8 * NT][17];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int first = Many ? blockIdx.y * 8 * NT : 0, rows = Many ? min(all - first, 8 * NT) : all;
  const int rank = split > 1 ? (int)gemm::cluster_rank() : 0, o0 = blockIdx.x / split * 16, step = split * kFewWarps * 32;
  // Rows past the last are the last one's again (their sums go nowhere), and what is past K is read from its end, and then zero: loads
  // without a condition are all under way at once.
  const __nv_bfloat16 *wp = w + (int64_t)o0 * d + 8 * t, *xp = x + (int64_t)first * d + 8 * t;
  int wr[2], xr[NT];                                     // to the rows
#pragma unroll
  for (int i = 0; i < 2; ++i) wr[i] = min(g + i * 8, n - 1 - o0) * d;
#pragma unroll
  for (int i = 0; i < NT; ++i) xr[i] = min(g + i * 8, rows - 1) * d;
  wait_previous();
  let_next();
  // Up to 8 rows a thread writes two values at most: their bias and residual are on their way while the products run. (1536 -> 768:
  // 8 rows 3.8 us with, 4.1 without, before the launches overlapped; with more rows the registers cost more, 64 rows 9.4 and 8.1.)
  const int mine = threadIdx.x * split + rank;
  float2 early = make_float2(0.f, 0.f), shift = early;
  if (NT == 1 && mine / 8 < rows && o0 + mine % 8 * 2 < n) {
    early = residual_of(p, (int64_t)(first + mine / 8) * n + o0 + mine % 8 * 2);
    shift = bias_of(p, o0 + mine % 8 * 2);
  }
  float acc[NT][4] = {};
  for (int k0 = (rank * kFewWarps + wid) * 32; k0 < d; k0 += U * step) {
    uint4 a[U][2], b[U][NT];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u * step >= d) break;                     // the same for the whole warp
      const int k = min(k0 + u * step, d - 8 - 8 * t);
#pragma unroll
      for (int i = 0; i < 2; ++i) a[u][i] = __ldg(reinterpret_cast<const uint4*>(wp + (wr[i] + k)));
#pragma unroll
      for (int i = 0; i < NT; ++i) b[u][i] = __ldg(reinterpret_cast<const uint4*>(xp + (xr[i] + k)));
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      if (k0 + u * step >= d) break;                     // the same for the whole warp
      if (k0 + u * step + 8 * t >= d) {
        a[u][0] = a[u][1] = make_uint4(0, 0, 0, 0);
#pragma unroll
        for (int i = 0; i < NT; ++i) b[u][i] = make_uint4(0, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < NT; ++i) {
        mma16x8(acc[i], a[u][0].x, a[u][1].x, a[u][0].y, a[u][1].y, b[u][i].x, b[u][i].y);
        mma16x8(acc[i], a[u][0].z, a[u][1].z, a[u][0].w, a[u][1].w, b[u][i].z, b[u][i].w);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sh[wid][i * 8 + 2 * t + (j & 1)][g + (j >> 1) * 8] = acc[i][j];
  __syncthreads();
  if (split > 1) {                                       // the warps' sums to the first one's place, for the other blocks
    for (int e = threadIdx.x; e < 8 * NT * 16; e += kFewWarps * 32) {
      float v = sh[0][e / 16][e % 16];
#pragma unroll
      for (int k = 1; k < kFewWarps; ++k) v += sh[k][e / 16][e % 16];
      sh[0][e / 16][e % 16] = v;
    }
    gemm::cluster_sync();
  }
  // Two columns each; a cluster's blocks take the pairs in turn.
  for (int e = mine; e < 8 * NT * 8; e += kFewWarps * 32 * split) {
    const int r = e / 8, c = e % 8 * 2;
    if (r >= rows || o0 + c >= n) continue;
    float v[2] = {};
    if (split > 1) {
      for (int k = 0; k < split; ++k) {
        const uint32_t at = gemm::peer_u32(&sh[0][r][c], k);
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          float q;
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(q) : "r"(at + 4 * j));
          v[j] += q;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kFewWarps; ++k) {
        v[0] += sh[k][r][c];
        v[1] += sh[k][r][c + 1];
      }
    }
    const int64_t at = (int64_t)(first + r) * n + o0 + c;
    if (NT > 1) shift = bias_of(p, o0 + c);
    v[0] += shift.x;
    v[1] += shift.y;
    if (p.act) {
      uint32_t s;
      activate<1>(p.act, v, &s);
      if (p.keep) *reinterpret_cast<uint32_t*>(slope + at) = s;
    }
    if (p.res_type != kNone) {
      if (NT > 1) early = residual_of(p, at);
      v[0] += early.x;
      v[1] += early.y;
    }
    if (p.res_type == kF32)
      *reinterpret_cast<float2*>(reinterpret_cast<float*>(y) + at) = make_float2(v[0], v[1]);
    else
      *reinterpret_cast<uint32_t*>(reinterpret_cast<__nv_bfloat16*>(y) + at) = pack2_bf16(v[0], v[1]);
  }
  if (split > 1) gemm::cluster_sync();                   // no block ends while another reads its sums
}

// dA = dY slope in bf16 (da null: not wanted; slope null: 1; relu: what it left out takes no part, whatever dY holds there), its
// remainder `below` rows further on unless that is 0 (then rows from `rows` to `below` are zeros in both; an infinity leaves no
// remainder), and its columns' sums over 64 rows. Block = 64 rows x 256 columns, a lane 8 columns,
// a warp every eighth row.
constexpr int kSlopeRows = 64;
template <bool F32>
__global__ void __launch_bounds__(256)
k_linear_slope(int64_t rows, int n, int below, bool relu, const void* __restrict__ dy, const __half* __restrict__ slope,
               __nv_bfloat16* __restrict__ da, float* __restrict__ sums) {
  __shared__ float sh[8][256];
  const int wide = (n + 255) / 256, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c0 = blockIdx.x % wide * 256, c = c0 + lane * 8;
  const int64_t r0 = (int64_t)(blockIdx.x / wide) * kSlopeRows;
  float s[8] = {};
  constexpr int kEach = kSlopeRows / 8, kHalf = kEach / 2;
#pragma unroll
  for (int h = 0; h < kEach; h += kHalf) {
    uint4 q[kHalf][2], f[kHalf];
#pragma unroll
    for (int k = 0; k < kHalf; ++k) {
      const int64_t r = r0 + (h + k) * 8 + wid, at = r * n + c;
      q[k][0] = q[k][1] = make_uint4(0, 0, 0, 0);
      if (r < rows && c < n) {
        const uint4* src = reinterpret_cast<const uint4*>(reinterpret_cast<const char*>(dy) + at * (F32 ? 4 : 2));
        q[k][0] = __ldg(src);
        if (F32) q[k][1] = __ldg(src + 1);
        if (slope) f[k] = __ldg(reinterpret_cast<const uint4*>(slope + at));
      }
    }
#pragma unroll
    for (int k = 0; k < kHalf; ++k) {
      const int64_t r = r0 + (h + k) * 8 + wid;
      if (c >= n || r >= (rows > below ? rows : below)) continue;
      float v[8];
      const uint32_t w[8] = {q[k][0].x, q[k][0].y, q[k][0].z, q[k][0].w, q[k][1].x, q[k][1].y, q[k][1].z, q[k][1].w};
#pragma unroll
      for (int j = 0; j < 8; ++j)
        v[j] = __uint_as_float(F32 ? w[j] : j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
      if (slope && r < rows) {
        const uint32_t z[4] = {f[k].x, f[k].y, f[k].z, f[k].w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float2 x = __half22float2(*reinterpret_cast<const __half2*>(&z[j]));
          v[2 * j] = !relu ? v[2 * j] * x.x : x.x == 0.f ? 0.f : v[2 * j];
          v[2 * j + 1] = !relu ? v[2 * j + 1] * x.y : x.y == 0.f ? 0.f : v[2 * j + 1];
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s[j] += v[j];
      if (da) {
        *reinterpret_cast<uint4*>(da + r * n + c) = gemm::pack8(v);
        if (below) {
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const float r = round_bf16(v[j]);
            v[j] = fabsf(r) < INFINITY ? v[j] - r : 0.f;
          }
          *reinterpret_cast<uint4*>(da + (r + below) * n + c) = gemm::pack8(v);
        }
      }
    }
  }
  if (!sums || r0 >= rows) return;
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[wid][lane + 32 * j] = s[j];
  __syncthreads();
  const int own = c0 + lane * 8 + wid;                   // this thread's column: its lane's wid-th
  float v = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) v += sh[k][threadIdx.x];
  if (own < n) sums[(int64_t)(blockIdx.x / wide) * n + own] = v;
}

struct LinearWs {
  int below, shares;                           // below: rows to dA's remainder (a multiple of 32), 0: none
  int64_t rows;                                // of dA, its remainder among them
  size_t da, sums, slots, total;
};

// own: dA is dY itself.
LinearWs linear_ws(int64_t N, int64_t d, int64_t n, bool own) {
  LinearWs w{};
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes); return at; };
  w.below = N <= kTwiceRows && !own ? (int)((N + 31) / 32 * 32) : 0;
  w.rows = w.below ? 2 * w.below : N;
  w.shares = gemm::shares_for(n, d, w.rows);
  w.da = take(own ? 0 : (size_t)w.rows * n * 2);
  w.sums = take((size_t)((N + kSlopeRows - 1) / kSlopeRows) * n * 4);
  w.slots = take(w.shares ? gemm::slot_bytes(n, d, w.shares) : 0);
  w.total = o;
  return w;
}

int check_linear(int64_t N, int32_t d, int32_t n) {
  if (N < 0 || d < 1 || n < 1) return ASRN_ERR_ARG;
  if (d % 8 || n % 8 || d > 65536 || n > (1 << 20) || N > (1 << 26)) return ASRN_ERR_UNSUPPORTED;
  if ((int64_t)((N + 127) / 128) * ((std::max(d, n) + 255) / 256) >= ((int64_t)1 << 30)) return ASRN_ERR_UNSUPPORTED;
  return ASRN_OK;
}

int launched() { return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA; }

template <int NT, bool Many = false>
int few(int64_t N, int d, int n, const void* x, const void* w, const Rest& p, void* y, void* slope, cudaStream_t s) {
  const int blocks = (n + 15) / 16, chunks = (int)((N + 8 * NT - 1) / (8 * NT));
  int split = 1;                                         // blocks of a cluster: until the SMs are full or K is
  while (split < 8 && blocks * chunks * split < gemm::sm_count() && d > split * kFewWarps * 32) split *= 2;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)(blocks * split), (unsigned)chunks);
  cfg.blockDim = dim3(kFewWarps * 32);
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = split > 1 ? 2 : 1;
  const int steps = (d + split * kFewWarps * 32 - 1) / (split * kFewWarps * 32);
  // Blocks enough to keep the memory busy: more of them on an SM (8 rows x 768 -> 50304: 15 us, with four steps under way 21).
  const bool many = blocks > 4 * gemm::sm_count();
  auto kernel = steps == 1                     ? k_linear_few<NT, 1, Many>
                : steps == 2 || NT > 2 || many ? k_linear_few<NT, 2, Many>
                                               : k_linear_few<NT, (NT > 2 ? 2 : 4), Many>;
  return cudaLaunchKernelEx(&cfg, kernel, (int)N, n, d, split, reinterpret_cast<const __nv_bfloat16*>(x),
                            reinterpret_cast<const __nv_bfloat16*>(w), p, y, reinterpret_cast<__half*>(slope)) == cudaSuccess
             ? ASRN_OK
             : ASRN_ERR_CUDA;
}

}  // namespace
}  // namespace asrn

extern "C" {

int asrn_linear_forward(int64_t N, int32_t d, int32_t n, const void* x, const void* weight, const void* bias, int32_t act,
                        const void* residual, int32_t res_type, void* y, void* slope, int* status, void* stream) {
  using namespace asrn;
  int st = check_linear(N, d, n);
  if (st) return st;
  if (act < 0 || act > kRelu || (residual && res_type != kF32 && res_type != kBf16)) return ASRN_ERR_ARG;
  if (N == 0) return ASRN_OK;
  if (!x || !weight || !y || ((uintptr_t)x | (uintptr_t)weight | (uintptr_t)bias | (uintptr_t)residual | (uintptr_t)y |
                              (uintptr_t)slope) % 16)
    return ASRN_ERR_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Rest p{reinterpret_cast<const __nv_bfloat16*>(bias), residual, act, residual ? res_type : kNone, act && slope};
  if (few_rows(N, n))
    return N <= 8    ? few<1>(N, d, n, x, weight, p, y, slope, s)
           : N <= 16 ? few<2>(N, d, n, x, weight, p, y, slope, s)
           : N <= 32 ? few<4>(N, d, n, x, weight, p, y, slope, s)
           : N <= 64 ? few<8>(N, d, n, x, weight, p, y, slope, s)
                     : few<8, true>(N, d, n, x, weight, p, y, slope, s);
  gemm::Shape a{};
  a.M = (int)N; a.N = n; a.K = d; a.group = 16; a.status = status;
  return gemm::launch<false, false, Fused>(x, d, weight, d, a, p, s, {y, N, n, n, p.res_type == kF32},
                                           {p.keep ? slope : nullptr, N, n, n});
}

size_t asrn_linear_workspace_bytes(int64_t N, int32_t d, int32_t n, int32_t act, int32_t y_type) {
  if (asrn::check_linear(N, d, n) || N == 0) return 0;
  return asrn::linear_ws(N, d, n, !act && y_type == asrn::kBf16).total;
}

int asrn_linear_backward(int64_t N, int32_t d, int32_t n, const void* dy, int32_t y_type, const void* x, const void* weight,
                         int32_t act, const void* slope, void* dx, void* dw, void* db, void* workspace,
                         size_t workspace_bytes, int* status, void* stream) {
  using namespace asrn;
  int st = check_linear(N, d, n);
  if (st) return st;
  if (act < 0 || act > kRelu || (y_type != kF32 && y_type != kBf16)) return ASRN_ERR_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (N == 0) {
    if ((dw && cudaMemsetAsync(dw, 0, (size_t)n * d * 2, s) != cudaSuccess) ||
        (db && cudaMemsetAsync(db, 0, (size_t)n * 2, s) != cudaSuccess))
      return ASRN_ERR_CUDA;
    return ASRN_OK;
  }
  if (!dy || !x || !weight || (act && !slope) || ((uintptr_t)dy | (uintptr_t)x | (uintptr_t)weight | (uintptr_t)slope |
                                                  (uintptr_t)dx | (uintptr_t)dw) % 16 || (uintptr_t)db % 2)
    return ASRN_ERR_ARG;
  const bool own = !act && y_type == kBf16;
  const LinearWs ws = linear_ws(N, d, n, own);
  if (!workspace || workspace_bytes < ws.total || (uintptr_t)workspace % 256) return ASRN_ERR_WORKSPACE;
  char* W = reinterpret_cast<char*>(workspace);
  float* sums = reinterpret_cast<float*>(W + ws.sums);
  __nv_bfloat16* made = reinterpret_cast<__nv_bfloat16*>(W + ws.da);
  if (db || (!own && (dx || dw))) {
    const int64_t all = std::max<int64_t>(N, ws.below), blocks = (all + kSlopeRows - 1) / kSlopeRows * ((n + 255) / 256);
    __nv_bfloat16* to = own || !(dx || dw) ? nullptr : made;
    const __half* f = act ? reinterpret_cast<const __half*>(slope) : nullptr;
    if (y_type == kF32)
      k_linear_slope<true><<<(unsigned)blocks, 256, 0, s>>>(N, n, ws.below, act == kRelu, dy, f, to, db ? sums : nullptr);
    else
      k_linear_slope<false><<<(unsigned)blocks, 256, 0, s>>>(N, n, ws.below, act == kRelu, dy, f, to, db ? sums : nullptr);
    if ((st = launched())) return st;
  }
  const void* da = own ? dy : made;
  if (dx) {
    gemm::Shape a{};
    a.M = (int)N; a.N = d; a.K = n; a.group = 16; a.status = status;
    a.second_pass = ws.below > 0; a.a_step = ws.below;
    if ((st = gemm::launch<false, true, gemm::StoreBf16>(da, n, weight, d, a, {}, s, {dx, N, d, d}))) return st;
  }
  if (dw && (st = weight_grad(N, n, d, da, ws.below, x, 0, ws.shares, reinterpret_cast<float*>(W + ws.slots), dw, status, s)))
    return st;
  if (db) {
    const ColSum q{(N + kSlopeRows - 1) / kSlopeRows, n, sums, reinterpret_cast<__nv_bfloat16*>(db)};
    k_colsum<<<(unsigned)((n + 31) / 32), 1024, 0, s>>>(q, ColSum{}, (n + 31) / 32);
    return launched();
  }
  return ASRN_OK;
}

}  // extern "C"
