// Log probabilities of given tokens through the tied head, forward and backward, without the (rows, V) logits in memory:
//   s_iv = h_i . w_v / tau,  lse_i = log sum_v exp s_iv,  logp_i = s_{i,y_i} - lse_i
//   dS_iv = (g_i / tau) (delta_{v,y_i} - exp(s_iv - lse_i)),  dh = dS W,  dW = dS^T h
// 2 N V d operations forward and 6 N V d backward (the scores are formed again), against 2 N d + 2 V d elements read:
// bound by the tensor cores at any training size.
//
// Positions without a target (token < 0: prompts, padding) are left out before the products: their rows are never
// gathered, so a batch whose half is prompt costs half. How many rows are left stays on the device.
//   k_head_count   (many rows) targets per block of 1024 tokens
//   k_head_gather  the rows with a target, in order, with their tokens and the maps both ways
//   k_gemm<Lse>    scores by tiles of 256 tokens; each thread keeps the running maximum and sum of exponentials of its
//                  row over its 128 columns and writes that pair; the target's score goes into none of the sums, it is
//                  written by itself: with x = s_y - m and S the sum of the others' exp(s - m), logp = -log1p(S exp(-x))
//                  and 1 - p_y = -expm1(logp) keep their leading digits where p_y is all but 1
//   k_head_join    the pairs of a row joined: logp, and lse and 1 - p_y for the backward pass
//   k_gemm<Slope>  backward, by chunks of rows: the scores again, dS in bf16
//   k_gemm         dh = dS W (parts of V where rows are few) and dW = dS^T h, sums in fp32
// dS is rounded to bf16 once, as the operand of both products: their results are off by 2.3e-3 of themselves in the 2-norm,
// 1.7e-3 with an unrounded dS. For few rows (kTwiceRows, left-out ones counted) the products take its remainder too: where
// few rows add up in dW, the target's rounding error would be nearly all of its. dh, whose sums run over V, gains the same
// at any number of rows and comes along.
#include "head.cuh"

namespace asrn {

namespace {

using gemm::exp2_fast;

struct HeadForwardWs {
  size_t counts, top, part, total;
};

HeadForwardWs head_forward_ws(int64_t N, int64_t V) {
  HeadForwardWs w{};
  const size_t P = (size_t)pad256(N), halves = (size_t)((V + gemm::kBN - 1) / gemm::kBN) * 2;
  w.counts = 0;
  w.top = align_up((size_t)((N + kCountRows - 1) / kCountRows) * 4);
  w.part = align_up(w.top + P * 4);
  w.total = align_up(w.part + halves * P * 8);
  return w;
}

// 855 us at 16384 x 50304 x 768, 1.48 PFLOP/s; one ex2 for a score takes a third of the tensor cores' time there.
// Running maximum (of the unscaled scores) and sum of exponentials over the thread's columns.
struct Lse {
  static constexpr int kWarps = 8, kOwn = 1, kTable = 0;
  struct Params {
    const int* tok;
    float k;                               // log2(e) / tau
    float* top;                            // the targets' unscaled scores
    float2* part;                          // [2 n-tiles][pad]
    int64_t pad;
  };
  const Params& p;
  int row, V, y, at;
  bool on;
  float m = -INFINITY, s = 0.f;
  ASRN_DEV Lse(const Params& pp, int r, int rows, const gemm::Shape& sh, const gemm::Tile& u, int half)
      : p(pp), row(r), V(sh.N), y(-1), at(u.n * 2 + half), on(r < rows) {
    if (on) y = p.tok[r];
  }
  template <class O> ASRN_DEV void chunk(float* v, int c, O&, const CUtensorMap*, const CUtensorMap*) {
    if (c >= V) return;
    const int n = V - c, j = y - c;        // n: valid columns, 32 or more but in the last tile
    if (j >= 0 && j < 32) {
      float own = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        own = i == j ? v[i] : own;
        v[i] = i == j ? -INFINITY : v[i];
      }
      p.top[row] = own;
    }
    float t = m;
    if (n < 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = i < n ? v[i] : -INFINITY;
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) t = fmaxf(t, v[i]);
    const float off = t == -INFINITY ? 0.f : t * p.k;
    const gemm::F2 k2(p.k), off2(-off);
    gemm::F2 add(0.f);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float a, b;
      gemm::fma2(gemm::F2(v[i], v[i + 1]), k2, off2).get(a, b);
      add = gemm::add2(add, gemm::F2(exp2_fast(a), exp2_fast(b)));
    }
    float a, b;
    add.get(a, b);
    s = s * exp2_fast(fmaf(m, p.k, -off)) + (a + b);
    m = t;
  }
  ASRN_DEV void finish() {
    if (on) p.part[at * p.pad + row] = make_float2(m, s);
  }
};

// 17 us at 16384 rows x 394 halves (52 MB, 3.0 TB/s; 39 us with 8 warps and a rescaling for every pair).
// Block = 32 positions x 16 warps over the halves of the vocabulary's tiles, 8 at a time.
constexpr int kJoinWarps = 16;
__global__ void __launch_bounds__(kJoinWarps * 32)
k_head_join(int64_t N, int halves, int64_t pad, float k, float inv_tau, const int* __restrict__ pos,
            const int* __restrict__ tok, const float* __restrict__ top, const float2* __restrict__ part,
            float* __restrict__ lse2, float* __restrict__ rest, float* __restrict__ logp) {
  __shared__ float2 sh[kJoinWarps][32];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;
  const int r = i < N ? pos[i] : -1;
  float m = -INFINITY, s = 0.f;
  auto join = [&](const float2* q, int n) {    // n of at most 8 pairs
    float t = m;
#pragma unroll
    for (int j = 0; j < 8; ++j) t = j < n ? fmaxf(t, q[j].x) : t;
    if (t == -INFINITY) {                      // no score yet but NaNs, which the maxima pass over: the sums hold them
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j < n) s += q[j].y;
      return;
    }
    s *= exp2_fast((m - t) * k);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < n) s = fmaf(q[j].y, exp2_fast((q[j].x - t) * k), s);
    m = t;
  };
  if (r >= 0)
    for (int j0 = wid; j0 < halves; j0 += 8 * kJoinWarps) {
      float2 q[8];
      int n = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (j0 + j * kJoinWarps < halves) {
          q[j] = __ldg(part + (j0 + j * kJoinWarps) * pad + r);
          n = j + 1;
        }
      join(q, n);
    }
  sh[wid][lane] = make_float2(m, s);
  __syncthreads();
  if (wid || i >= N) return;
  m = -INFINITY;
  s = 0.f;
  for (int w = 0; w < kJoinWarps; w += 8) {
    float2 q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) q[j] = sh[w + j][lane];
    join(q, 8);
  }
  if (r < 0) {
    logp[i] = 0.f;
    return;
  }
  if (tok[r] < 0) {
    logp[i] = NAN;
    return;
  }
  const float own = top[r], x = (own - m) * inv_tau;
  const float lp = s == 0.f ? own * 0.f : x > 0.f ? -log1pf(s * expf(-x)) : x - logf(s + expf(x));
  logp[i] = lp;
  lse2[r] = own * k - lp * kLog2e;
  rest[r] = -expm1f(lp);
}

// 917 us at 16384 x 50304 x 768, 1.38 PFLOP/s (947 with sixteen warps and a piece each; direct stores: 1250).
// dS of one chunk in bf16; the rows that pad the last tile get zeros.
struct Slope {
  static constexpr int kWarps = 8, kOwn = 2, kTable = 0;
  struct Params {
    const int *tok, *row;                  // of the chunk's rows
    const float *lse2, *rest, *g;
    float k, inv_tau;
    int below;                             // rows from dS to its remainder, 0: none
  };
  const Params& p;
  int V, y, first;
  bool on;
  float off, g, own;                       // lse, -dL/dlogp / tau, the target's dS
  ASRN_DEV Slope(const Params& pp, int r, int rows, const gemm::Shape& sh, const gemm::Tile&, int)
      : p(pp), V(sh.N), y(-1), first(r & ~31), on(r < rows), off(0.f), g(0.f), own(0.f) {
    if (on) {
      y = p.tok[r];
      off = p.lse2[r];
      g = y < 0 ? NAN : -p.g[p.row[r]] * p.inv_tau;
      own = -g * p.rest[r];
    }
  }
  template <class O> ASRN_DEV void chunk(float* v, int c, O& out, const CUtensorMap* map_o, const CUtensorMap*) {
    if (c >= V) return;
    const gemm::F2 k2(p.k), off2(-off), g2(g);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float a, b;
      gemm::fma2(gemm::F2(v[i], v[i + 1]), k2, off2).get(a, b);
      gemm::mul2(g2, gemm::F2(exp2_fast(a), exp2_fast(b))).get(v[i], v[i + 1]);
    }
    const int j = y - c;
    if (j >= 0 && j < 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = i == j ? own : v[i];
    }
    if (!on) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = 0.f;
    }
    out.put(map_o, v, c, first);
    if (p.below) {
      gemm::remainder(v);
      out.put(map_o, v, c, first + p.below);
    }
  }
  ASRN_DEV void finish() {}
};

}  // namespace

}  // namespace asrn

extern "C" {

size_t asrn_head_saved_bytes(int64_t N, int32_t d) {
  if (asrn::check_head(N, 1, d)) return 0;
  return asrn::head_saved(N, d).total;
}

size_t asrn_head_workspace_bytes(int64_t N, int64_t V, int32_t d, int32_t backward) {
  if (asrn::check_head(N, V, d)) return 0;
  return backward ? asrn::head_backward_ws(N, V, d).total : asrn::head_forward_ws(N, V).total;
}

int asrn_head_forward(int64_t N, int64_t V, int32_t d, const void* h, const void* weight, const int64_t* tokens,
                      float tau, float* logp, void* saved, size_t saved_bytes, void* workspace,
                      size_t workspace_bytes, int* status, void* stream) {
  using namespace asrn;
  int st = check_head(N, V, d);
  if (st) return st;
  if (!(tau > 0.f) || tau > 1e30f) return ASRN_ERR_ARG;
  if (N == 0) return ASRN_OK;
  if (!h || !weight || !tokens || !logp || (uintptr_t)h % 16 || (uintptr_t)weight % 16) return ASRN_ERR_ARG;
  const HeadSaved sv = head_saved(N, d);
  const HeadForwardWs ws = head_forward_ws(N, V);
  if (!saved || saved_bytes < sv.total || (uintptr_t)saved % 256 || !workspace || workspace_bytes < ws.total ||
      (uintptr_t)workspace % 256)
    return ASRN_ERR_WORKSPACE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* S = reinterpret_cast<char*>(saved);
  char* W = reinterpret_cast<char*>(workspace);
  int* count = reinterpret_cast<int*>(S + sv.count);
  int* tok = reinterpret_cast<int*>(S + sv.tok);
  int* pos = reinterpret_cast<int*>(S + sv.pos);
  __nv_bfloat16* hc = reinterpret_cast<__nv_bfloat16*>(S + sv.hc);
  if ((st = head_gather(N, V, d, h, tokens, reinterpret_cast<int*>(W + ws.counts), S, sv, s))) return st;
  gemm::Shape sh{};
  sh.M = (int)N; sh.N = (int)V; sh.K = d; sh.m_dev = count; sh.group = 16; sh.status = status;
  const float inv_tau = 1.f / tau;
  Lse::Params p{tok, kLog2e * inv_tau, reinterpret_cast<float*>(W + ws.top), reinterpret_cast<float2*>(W + ws.part),
                pad256(N)};
  if ((st = gemm::launch<false, false, Lse>(hc, d, weight, d, sh, p, s))) return st;
  k_head_join<<<(unsigned)((N + 31) / 32), kJoinWarps * 32, 0, s>>>(N, (int)((V + gemm::kBN - 1) / gemm::kBN) * 2, p.pad, p.k,
                                                        inv_tau, pos, tok, p.top, p.part,
                                                        reinterpret_cast<float*>(S + sv.lse2),
                                                        reinterpret_cast<float*>(S + sv.rest), logp);
  return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
}

int asrn_head_backward(int64_t N, int64_t V, int32_t d, const void* weight, const void* saved, size_t saved_bytes,
                       float tau, const float* g, void* dh, void* dw, void* workspace, size_t workspace_bytes,
                       int* status, void* stream) {
  using namespace asrn;
  int st = check_head(N, V, d);
  if (st) return st;
  if (!(tau > 0.f) || tau > 1e30f) return ASRN_ERR_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (N == 0) {
    if (dw && cudaMemsetAsync(dw, 0, (size_t)V * d * 2, s) != cudaSuccess) return ASRN_ERR_CUDA;
    return ASRN_OK;
  }
  if (!weight || !g || (uintptr_t)weight % 16 || (uintptr_t)dh % 16 || (uintptr_t)dw % 16) return ASRN_ERR_ARG;
  const HeadSaved sv = head_saved(N, d);
  const HeadBackwardWs ws = head_backward_ws(N, V, d);
  if (!saved || saved_bytes < sv.total || (uintptr_t)saved % 256 || !workspace || workspace_bytes < ws.total ||
      (uintptr_t)workspace % 256)
    return ASRN_ERR_WORKSPACE;
  const char* S = reinterpret_cast<const char*>(saved);
  return head_backward<Slope>(N, V, d, weight, S, sv, ws, reinterpret_cast<char*>(workspace), dh, dw, status, s,
                              [&](int64_t first, int below) {
                         return Slope::Params{reinterpret_cast<const int*>(S + sv.tok) + first,
                                              reinterpret_cast<const int*>(S + sv.row) + first,
                                              reinterpret_cast<const float*>(S + sv.lse2) + first,
                                              reinterpret_cast<const float*>(S + sv.rest) + first, g, kLog2e / tau,
                                              1.f / tau, below};
                       });
}

}  // extern "C"
