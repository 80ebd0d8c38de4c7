// What the operators around the products share: gelu and its slope in an epilogue, column sums, the product that makes a
// weight's gradient, and the multiplication of products with few rows.
#pragma once
#include "gemm_tc.cuh"

namespace asrn {

// Of two values a: e = exp(-a^2 / 2) and q = Q(|a|), the normal distribution's tail, by Abramowitz and Stegun's 7.1.26,
// erfc(x) = (a1 t + .. + a5 t^5) exp(-x^2), t = 1 / (1 + p x), with x = |a| / sqrt 2. The formula's own error is 1.5e-7 of
// erfc, 7.5e-8 of q; with the arithmetic's q is off by up to 3.2e-7 for |a| below 1, 1.2e-7 below 2 and less from there on,
// gelu by 2e-7 max(1, |a|), gelu' by 3.6e-7 (against erfc and exp in 64 bits at 2^24 points of each range). Then
// gelu(a) = max(a, 0) - |a| q and gelu'(a) = 1/2 + sign(a) (1/2 - q) + a e / sqrt(2 pi).
ASRN_DEV void tails(float a0, float a1, gemm::F2& e, gemm::F2& q) {
  using namespace gemm;
  const F2 a(a0, a1), m(fabsf(a0), fabsf(a1));
  float x, y;
  mul2(mul2(a, a), F2(-0.72134752044448170f)).get(x, y);
  e = F2(exp2_fast(x), exp2_fast(y));
  fma2(m, F2(0.3275911f * 0.70710678118654752f), F2(1.f)).get(x, y);
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(x));
  asm("rcp.approx.ftz.f32 %0, %0;" : "+f"(y));
  const F2 t(x, y);
  F2 r = fma2(t, F2(0.5f * 1.061405429f), F2(0.5f * -1.453152027f));
  r = fma2(r, t, F2(0.5f * 1.421413741f));
  r = fma2(r, t, F2(0.5f * -0.284496736f));
  r = fma2(r, t, F2(0.5f * 0.254829592f));
  q = mul2(mul2(r, t), e);
}

// gelu(a) and gelu'(a) for the pair's cdf and density.
ASRN_DEV void gelu_both(float a0, float a1, gemm::F2& g, gemm::F2& slope) {
  using namespace gemm;
  F2 e, q;
  tails(a0, a1, e, q);
  float h0, h1;
  fma2(q, F2(-1.f), F2(0.5f)).get(h0, h1);                                       // 1/2 - q
  const F2 a(a0, a1), cdf = add2(F2(copysignf(h0, a0), copysignf(h1, a1)), F2(0.5f));
  g = mul2(a, cdf);
  slope = fma2(mul2(a, F2(0.39894228040143268f)), e, cdf);
}

// Column sums over a warp's 32 rows: lane i gets the sum of v[i].
ASRN_DEV float column_sum(float* v, int lane) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const bool up = lane & o;
#pragma unroll
    for (int i = 0; i < o; ++i) {
      const float keep = up ? v[i + o] : v[i], send = up ? v[i] : v[i + o];
      v[i] = keep + __shfl_xor_sync(0xffffffffu, send, o);
    }
  }
  return v[0];
}

// out[c] = bf16(sum of the parts' [..][c]) in order, for two sets: block = 32 columns x 32 warps.
struct ColSum {
  int64_t parts;
  int n;
  const float* sums;
  __nv_bfloat16* out;
};
static __global__ void __launch_bounds__(1024) k_colsum(const ColSum a, const ColSum b, int blocks_a) {
  __shared__ float sh[32][33];
  const bool second = (int)blockIdx.x >= blocks_a;
  const ColSum& q = second ? b : a;
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c = ((int)blockIdx.x - (second ? blocks_a : 0)) * 32 + lane;
  float s = 0.f;
  if (c < q.n)
#pragma unroll 4
    for (int64_t k = wid; k < q.parts; k += 32) s += q.sums[k * q.n + c];
  sh[wid][lane] = s;
  __syncthreads();
  if (wid) return;
  s = 0.f;
  for (int w = 0; w < 32; ++w) s += sh[w][lane];
  if (c < q.n) q.out[c] = __float2bfloat16_rn(s);
}

// out (M, n) = A^T B over the rows they share, both as they lie in memory.
inline int weight_grad(int64_t rows, int M, int n, const void* A, int below_a, const void* B, int below_b, int shares,
                float* slots, void* out, int* status, cudaStream_t s) {
  gemm::Shape a{};
  a.M = M; a.N = n; a.K = (int)rows; a.shares = shares; a.group = 16; a.status = status;
  a.second_pass = below_a || below_b; a.a_step = below_a; a.b_step = below_b;
  if (!shares) return gemm::launch<true, true, gemm::StoreBf16>(A, M, B, n, a, {}, s, {out, M, n, n});
  const gemm::StorePiece::Params q{slots, gemm::kBM * gemm::pair_for(M)};
  const int st = gemm::launch<true, true, gemm::StorePiece>(A, M, B, n, a, q, s);
  return st ? st : gemm::join(a, slots, out, nullptr, nullptr, 0, s);
}

// D (16 x 8) += A (16 x 16) B (16 x 8).
ASRN_DEV void mma16x8(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

}  // namespace asrn
