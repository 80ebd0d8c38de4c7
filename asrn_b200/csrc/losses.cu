// Losses of fine-tuning on per-token log probabilities, each with its gradient in the same call: the preference loss of
// answer pairs and the clipped policy loss with a KL term. Both read each token once (13 and 17 to 21 bytes with the
// gradient written) and compute next to nothing, so they are bound by HBM when large and by the launches when small.
//
// Every sum is formed in a fixed order in fp64 (per thread, then by warp shuffles, then over the blocks' partials in
// index order): the results do not depend on the blocks' timing. Positions outside the mask are read but selected away,
// never multiplied, so a NaN or infinity there reaches nothing.
#include "common.cuh"
#include "layout.h"

namespace asrn {

namespace {

constexpr int kLossThreads = 256;
constexpr int kLossChunk = 2048;         // tokens of one row that a block takes at a time: 8 per thread
constexpr int kLossPer = kLossChunk / kLossThreads;
constexpr int kSmallRows = 1024;         // rows a single block keeps in shared memory

struct RowSum {                          // of one chunk of one row
  double sum;
  int64_t n;
};

__device__ __forceinline__ int warp_sum_i(int v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

// Sum over the block, in every thread; `slots` holds one value per warp.
template <class T> __device__ __forceinline__ T block_sum(T v, T* slots) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) slots[threadIdx.x >> 5] = v;
  __syncthreads();
  T s = 0;
  for (int i = 0; i < (int)(blockDim.x >> 5); ++i) s += slots[i];
  return s;
}

// ---- preference loss -----------------------------------------------------------------------------------------------

struct PrefArgs {
  int64_t P, L;
  const float *logp, *ref;               // (2, P, L): the chosen answers, then the rejected ones
  const uint8_t* mask;
  int32_t kind;                          // 0: logistic, 1: squared distance of the mean log ratios (IPO)
  double beta, smoothing;
  float *loss, *grad, *rewards;          // scalar, (2, P, L) or null, (2, P)
};

struct Pair {
  double loss, slope0, slope1;           // l_p, dl/dlogp of a chosen / a rejected token (before the mean over pairs)
  bool on;
};

// l and its slopes from the two rows' sums of log ratios and token counts.
__device__ __forceinline__ Pair pair_of(const PrefArgs& a, double r0, double r1, int64_t n0, int64_t n1) {
  Pair p{0., 0., 0., n0 > 0 && n1 > 0};
  if (!p.on) return p;
  if (a.kind == 1) {
    const double gap = r0 / (double)n0 - r1 / (double)n1 - 0.5 / a.beta;
    p.loss = gap * gap;
    p.slope0 = 2. * gap / (double)n0;
    p.slope1 = -2. * gap / (double)n1;
  } else {
    const double x = a.beta * (r0 - r1);
    const double soft = log1p(exp(-fabs(x)));                    // -log sigma(|x|)
    const double e = exp(-fabs(x));
    const double up = x >= 0. ? e / (1. + e) : 1. / (1. + e);     // sigma(-x)
    p.loss = (1. - a.smoothing) * (soft - fmin(x, 0.)) + a.smoothing * (soft + fmax(x, 0.));
    if (x != x) p.loss = x;
    p.slope0 = a.beta * (a.smoothing - up);
    p.slope1 = -p.slope0;
  }
  return p;
}

__device__ __forceinline__ double log_ratio(const PrefArgs& a, int64_t at) {
  return a.mask[at] ? (double)a.logp[at] - (double)a.ref[at] : 0.;
}

// All of it in one block: a warp per row for the sums, then the pairs, then the gradient.
__global__ void __launch_bounds__(1024) k_pref_small(PrefArgs a) {
  __shared__ double tot[kSmallRows];
  __shared__ int64_t cnt[kSmallRows];
  __shared__ double slots[32];
  const int rows = (int)(2 * a.P), P = (int)a.P, lane = threadIdx.x & 31;
  for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5) {
    double s = 0.;
    int n = 0;
#pragma unroll 4
    for (int64_t t = lane; t < a.L; t += 32) {
      const int64_t at = (int64_t)r * a.L + t;
      s += log_ratio(a, at);
      n += a.mask[at] != 0;
    }
    s = warp_sum_d(s);
    n = warp_sum_i(n);
    if (lane == 0) {
      tot[r] = s;
      cnt[r] = n;
      a.rewards[r] = (float)(a.beta * s);
    }
  }
  __syncthreads();
  Pair p{0., 0., 0., false};
  if (threadIdx.x < P) p = pair_of(a, tot[threadIdx.x], tot[P + threadIdx.x], cnt[threadIdx.x], cnt[P + threadIdx.x]);
  const double pairs = fmax(1., block_sum(p.on ? 1. : 0., slots));
  const double loss = block_sum(p.loss, slots);
  if (threadIdx.x == 0) a.loss[0] = (float)(loss / pairs);
  if (!a.grad) return;
  if (threadIdx.x < P) {
    tot[threadIdx.x] = p.slope0 / pairs;
    tot[P + threadIdx.x] = p.slope1 / pairs;
  }
  __syncthreads();
  for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5) {
    const float g = (float)tot[r];
    for (int64_t t = lane; t < a.L; t += 32) {
      const int64_t at = (int64_t)r * a.L + t;
      a.grad[at] = a.mask[at] ? g : 0.f;
    }
  }
}

// Row sums by chunks: block (chunk, row).
__global__ void __launch_bounds__(kLossThreads) k_pref_sums(PrefArgs a, int64_t items, int64_t chunks,
                                                            RowSum* __restrict__ part) {
  __shared__ double slots[8];
  __shared__ int islots[8];
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t row = it / chunks, t0 = (it % chunks) * kLossChunk;
    const int64_t base = row * a.L + t0, left = a.L - t0;
    float lp[kLossPer], rf[kLossPer];
    uint8_t m[kLossPer];
#pragma unroll
    for (int j = 0; j < kLossPer; ++j) {
      const int64_t t = j * kLossThreads + threadIdx.x;
      const bool in = t < left;
      m[j] = in ? a.mask[base + t] : 0;
      lp[j] = in ? __ldg(a.logp + base + t) : 0.f;
      rf[j] = in ? __ldg(a.ref + base + t) : 0.f;
    }
    double s = 0.;
    int n = 0;
#pragma unroll
    for (int j = 0; j < kLossPer; ++j) {
      s += m[j] ? (double)lp[j] - (double)rf[j] : 0.;
      n += m[j] != 0;
    }
    s = block_sum(s, slots);
    n = block_sum(n, islots);
    if (threadIdx.x == 0) part[it] = RowSum{s, n};
  }
}

__device__ __forceinline__ RowSum row_total(const RowSum* part, int64_t row, int64_t chunks) {
  RowSum t{0., 0};
  for (int64_t c = 0; c < chunks; ++c) {
    t.sum += part[row * chunks + c].sum;
    t.n += part[row * chunks + c].n;
  }
  return t;
}

// The pairs that count, the loss (block 0) and the gradient.
__global__ void __launch_bounds__(kLossThreads) k_pref_finish(PrefArgs a, int64_t items, int64_t chunks,
                                                              const RowSum* __restrict__ part) {
  __shared__ double slots[8];
  __shared__ float slope_s;
  double on = 0., loss = 0.;
  for (int64_t p = threadIdx.x; p < a.P; p += kLossThreads) {
    const RowSum r0 = row_total(part, p, chunks), r1 = row_total(part, a.P + p, chunks);
    on += r0.n > 0 && r1.n > 0 ? 1. : 0.;
    if (blockIdx.x == 0) {
      loss += pair_of(a, r0.sum, r1.sum, r0.n, r1.n).loss;
      a.rewards[p] = (float)(a.beta * r0.sum);
      a.rewards[a.P + p] = (float)(a.beta * r1.sum);
    }
  }
  const double pairs = fmax(1., block_sum(on, slots));
  if (blockIdx.x == 0) {
    loss = block_sum(loss, slots);
    if (threadIdx.x == 0) a.loss[0] = (float)(loss / pairs);
  }
  if (!a.grad) return;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t row = it / chunks, t0 = (it % chunks) * kLossChunk;
    const int64_t base = row * a.L + t0, left = a.L - t0;
    uint8_t m[kLossPer];
#pragma unroll
    for (int j = 0; j < kLossPer; ++j) {
      const int64_t t = j * kLossThreads + threadIdx.x;
      m[j] = t < left ? a.mask[base + t] : 0;
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      const int64_t p = row % a.P;
      const RowSum r0 = row_total(part, p, chunks), r1 = row_total(part, a.P + p, chunks);
      const Pair q = pair_of(a, r0.sum, r1.sum, r0.n, r1.n);
      slope_s = (float)((row < a.P ? q.slope0 : q.slope1) / pairs);
    }
    __syncthreads();
    const float g = slope_s;
#pragma unroll
    for (int j = 0; j < kLossPer; ++j) {
      const int64_t t = j * kLossThreads + threadIdx.x;
      if (t < left) a.grad[base + t] = m[j] ? g : 0.f;
    }
  }
}

// ---- clipped policy loss -------------------------------------------------------------------------------------------

struct PolicyArgs {
  int64_t B, L;
  const float *logp, *old, *ref, *adv;   // (B, L); ref may be null; adv (B, L) or (B)
  const uint8_t* mask;
  int32_t adv_per_token, per_sequence;
  double log_low, log_high;              // log(1 - clip_low), log(1 + clip_high)
  float low, high, kl;                   // 1 - clip_low, 1 + clip_high, KL coefficient
  float *loss, *grad, *stats;            // scalar, (B, L) or null, (2): mean KL estimate, share of clipped tokens
};

struct TokenSum {
  double loss, kl;
  int64_t n, cut;
};

struct Token {
  float loss, slope, kl;
  bool cut;
};

// exp(q) - 1 - q without the cancellation near 0 (Taylor's series below 1/4: its next term is under 4e-7 of the sum).
__device__ __forceinline__ float expm1_minus(float q) {
  if (fabsf(q) < 0.25f)
    return q * q * (0.5f + q * (1.f / 6 + q * (1.f / 24 + q * (1.f / 120 + q * (1.f / 720)))));
  return expm1f(q) - q;
}

// One token of the loss: the ratio's bounds are compared in the log domain, where the log ratio is exact or nearly so,
// against fp64 bounds: which side a token falls on does not hang on expf's last bit.
__device__ __forceinline__ Token token_of(const PolicyArgs& a, float lp, float old, float rf, float adv) {
  Token t{0.f, 0.f, 0.f, false};
  const float d = lp - old;
  const bool held = d > 20.f || d < -20.f;
  const float lr = d > 20.f ? 20.f : d < -20.f ? -20.f : d;
  t.cut = (adv > 0.f && (double)lr > a.log_high) || (adv < 0.f && (double)lr < a.log_low);
  const float r = expf(lr);
  t.loss = t.cut ? -(adv > 0.f ? a.high : a.low) * adv : -r * adv;
  t.slope = t.cut || held ? 0.f : -r * adv;
  if (a.ref) {
    const float dq = rf - lp;
    const bool qheld = dq > 20.f || dq < -20.f;
    const float q = dq > 20.f ? 20.f : dq < -20.f ? -20.f : dq;
    t.kl = expm1_minus(q);
    t.loss += a.kl * t.kl;
    if (!qheld) t.slope -= a.kl * expm1f(q);
  }
  return t;
}

__device__ __forceinline__ void policy_results(const PolicyArgs& a, double loss, double kl, double n, double cut,
                                               double rows) {
  const double total = fmax(1., n);
  a.loss[0] = (float)(loss / (a.per_sequence ? fmax(1., rows) : total));
  a.stats[0] = (float)(kl / total);
  a.stats[1] = (float)(cut / total);
}

__global__ void __launch_bounds__(1024) k_policy_small(PolicyArgs a) {
  __shared__ int cnt[kSmallRows];
  __shared__ double slots[32];
  const int rows = (int)a.B, L = (int)a.L, lane = threadIdx.x & 31;
  double n = 0., full = 0.;
  for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5) {
    int c = 0;
#pragma unroll 4
    for (int t = lane; t < L; t += 32) c += a.mask[(int64_t)r * L + t] != 0;
    c = warp_sum_i(c);
    if (lane == 0) {
      cnt[r] = c;
      n += c;
      full += c > 0 ? 1. : 0.;
    }
  }
  n = block_sum(n, slots);
  full = block_sum(full, slots);
  const double total = fmax(1., n), seqs = fmax(1., full);
  double loss = 0., kl = 0., cut = 0.;
  const int all = rows * L;
  for (int i = threadIdx.x; i < all; i += blockDim.x) {
    const int row = i / L;
    float g = 0.f;
    if (a.mask[i]) {
      const Token t = token_of(a, a.logp[i], a.old[i], a.ref ? a.ref[i] : 0.f, a.adv[a.adv_per_token ? i : row]);
      const double w = a.per_sequence ? 1. / cnt[row] : 1.;
      loss += w * (double)t.loss;
      kl += (double)t.kl;
      cut += t.cut ? 1. : 0.;
      g = (float)((double)t.slope * w / (a.per_sequence ? seqs : total));
    }
    if (a.grad) a.grad[i] = g;
  }
  loss = block_sum(loss, slots);
  kl = block_sum(kl, slots);
  cut = block_sum(cut, slots);
  if (threadIdx.x == 0) policy_results(a, loss, kl, n, cut, full);
}

// Tokens of each chunk of each row; block 0 clears the ticket that the next launch's blocks take.
__global__ void __launch_bounds__(kLossThreads) k_policy_counts(PolicyArgs a, int64_t items, int64_t chunks,
                                                                int* __restrict__ counts, unsigned* ticket) {
  __shared__ int slots[8];
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0u;
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t row = it / chunks, t0 = (it % chunks) * kLossChunk;
    const int64_t base = row * a.L + t0, left = a.L - t0;
    int n = 0;
#pragma unroll
    for (int j = 0; j < kLossPer; ++j) {
      const int64_t t = j * kLossThreads + threadIdx.x;
      n += t < left ? a.mask[base + t] != 0 : 0;
    }
    n = block_sum(n, slots);
    if (threadIdx.x == 0) counts[it] = n;
  }
}

// The tokens, the gradient and each item's sums; the block that finishes last adds the sums up in index order.
__global__ void __launch_bounds__(kLossThreads) k_policy_main(PolicyArgs a, int64_t items, int64_t chunks,
                                                              const int* __restrict__ counts, TokenSum* part,
                                                              unsigned* ticket) {
  __shared__ double slots[8];
  __shared__ bool last;
  double n = 0., full = 0.;
  for (int64_t b = threadIdx.x; b < a.B; b += kLossThreads) {
    int64_t c = 0;
    for (int64_t k = 0; k < chunks; ++k) c += counts[b * chunks + k];
    n += (double)c;
    full += c > 0 ? 1. : 0.;
  }
  n = block_sum(n, slots);
  full = block_sum(full, slots);
  for (int64_t it = blockIdx.x; it < items; it += gridDim.x) {
    const int64_t row = it / chunks, t0 = (it % chunks) * kLossChunk;
    const int64_t base = row * a.L + t0, left = a.L - t0;
    double w = 1. / fmax(1., n);
    if (a.per_sequence) {
      int64_t c = 0;
      for (int64_t k = 0; k < chunks; ++k) c += counts[row * chunks + k];
      w = 1. / (fmax(1., (double)c) * fmax(1., full));
    }
    const float gw = (float)w;
    const float row_adv = a.adv_per_token ? 0.f : a.adv[row];
    float lp[kLossPer], old[kLossPer], rf[kLossPer], adv[kLossPer];
    uint8_t m[kLossPer];
#pragma unroll
    for (int j = 0; j < kLossPer; ++j) {
      const int64_t t = j * kLossThreads + threadIdx.x;
      const bool in = t < left;
      m[j] = in ? a.mask[base + t] : 0;
      lp[j] = in ? __ldg(a.logp + base + t) : 0.f;
      old[j] = in ? __ldg(a.old + base + t) : 0.f;
      rf[j] = in && a.ref ? __ldg(a.ref + base + t) : 0.f;
      adv[j] = in && a.adv_per_token ? __ldg(a.adv + base + t) : row_adv;
    }
    double loss = 0., kl = 0.;
    int cut = 0, cn = 0;
#pragma unroll
    for (int j = 0; j < kLossPer; ++j) {
      const int64_t t = j * kLossThreads + threadIdx.x;
      float g = 0.f;
      if (m[j]) {
        const Token k = token_of(a, lp[j], old[j], rf[j], adv[j]);
        loss += (double)k.loss;
        kl += (double)k.kl;
        cut += k.cut;
        ++cn;
        g = k.slope * gw;
      }
      if (a.grad && t < left) a.grad[base + t] = g;
    }
    loss = block_sum(loss, slots);
    kl = block_sum(kl, slots);
    const double tc = block_sum((double)cut, slots);
    const double tn = block_sum((double)cn, slots);
    if (threadIdx.x == 0) part[it] = TokenSum{a.per_sequence ? loss * w * fmax(1., full) : loss, kl, (int64_t)tn, (int64_t)tc};
  }
  if (threadIdx.x == 0) {
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  double loss = 0., kl = 0., cut = 0.;
  for (int64_t it = threadIdx.x; it < items; it += kLossThreads) {
    const TokenSum t = part[it];
    loss += t.loss;
    kl += t.kl;
    cut += (double)t.cut;
  }
  loss = block_sum(loss, slots);
  kl = block_sum(kl, slots);
  cut = block_sum(cut, slots);
  if (threadIdx.x == 0) policy_results(a, loss, kl, n, cut, full);
}

int64_t loss_chunks(int64_t L) { return (L + kLossChunk - 1) / kLossChunk; }

int loss_grid(int64_t items) {
  return (int)(items < 148 * 8 ? items : 148 * 8);
}

bool small_loss(int64_t rows, int64_t L) { return rows <= kSmallRows && rows * L <= 16384; }

}  // namespace
}  // namespace asrn

extern "C" {

size_t asrn_preference_workspace_bytes(int64_t P, int64_t L) {
  if (P < 0 || L < 0 || asrn::small_loss(2 * P, L)) return 0;
  return asrn::align_up((size_t)(2 * P * asrn::loss_chunks(L)) * sizeof(asrn::RowSum) + 1);
}

int asrn_preference_loss(int64_t P, int64_t L, const float* logp, const float* ref_logp, const uint8_t* mask,
                         int32_t kind, double beta, double smoothing, float* loss, float* grad, float* rewards,
                         void* workspace, size_t workspace_bytes, void* stream) {
  using namespace asrn;
  if (P < 0 || L < 0 || kind < 0 || kind > 1 || !(beta > 0.) || !(smoothing >= 0. && smoothing < 0.5) || !loss)
    return ASRN_ERR_ARG;
  if (kind == 1 && smoothing != 0.) return ASRN_ERR_ARG;
  if (P > ((int64_t)1 << 30) || L > ((int64_t)1 << 30)) return ASRN_ERR_UNSUPPORTED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const PrefArgs a{P, L, logp, ref_logp, mask, kind, beta, smoothing, loss, grad, rewards};
  if (P * L > 0 && (!logp || !ref_logp || !mask)) return ASRN_ERR_ARG;
  if (P > 0 && !rewards) return ASRN_ERR_ARG;
  if (small_loss(2 * P, L)) {
    k_pref_small<<<1, 1024, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
  }
  if (!workspace || workspace_bytes < asrn_preference_workspace_bytes(P, L) || (uintptr_t)workspace % 16)
    return ASRN_ERR_WORKSPACE;
  const int64_t chunks = loss_chunks(L), items = 2 * P * chunks;
  RowSum* part = reinterpret_cast<RowSum*>(workspace);
  const int grid = items > 0 ? loss_grid(items) : 1;
  k_pref_sums<<<grid, kLossThreads, 0, s>>>(a, items, chunks, part);
  k_pref_finish<<<grid, kLossThreads, 0, s>>>(a, items, chunks, part);
  return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
}

size_t asrn_policy_workspace_bytes(int64_t B, int64_t L) {
  if (B < 0 || L < 0 || asrn::small_loss(B, L)) return 0;
  const size_t items = (size_t)(B * asrn::loss_chunks(L));
  return 256 + asrn::align_up(items * sizeof(asrn::TokenSum)) + asrn::align_up(items * sizeof(int));
}

int asrn_policy_loss(int64_t B, int64_t L, const float* logp, const float* old_logp, const float* ref_logp,
                     const float* advantages, int32_t adv_per_token, const uint8_t* mask, double clip_low,
                     double clip_high, double kl, int32_t per_sequence, float* loss, float* grad, float* stats,
                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace asrn;
  if (B < 0 || L < 0 || !(clip_low >= 0. && clip_low < 1.) || !(clip_high >= 0.) || !(kl >= 0.) || !loss || !stats)
    return ASRN_ERR_ARG;
  if (kl > 0. && !ref_logp) return ASRN_ERR_ARG;
  if (B > ((int64_t)1 << 30) || L > ((int64_t)1 << 30)) return ASRN_ERR_UNSUPPORTED;
  if (B * L > 0 && (!logp || !old_logp || !advantages || !mask)) return ASRN_ERR_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const PolicyArgs a{B, L, logp, old_logp, ref_logp, advantages, mask, adv_per_token != 0, per_sequence != 0,
                     log1p(-clip_low), log1p(clip_high), (float)(1. - clip_low), (float)(1. + clip_high), (float)kl,
                     loss, grad, stats};
  if (small_loss(B, L)) {
    k_policy_small<<<1, 1024, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
  }
  if (!workspace || workspace_bytes < asrn_policy_workspace_bytes(B, L) || (uintptr_t)workspace % 16)
    return ASRN_ERR_WORKSPACE;
  const int64_t chunks = loss_chunks(L), items = B * chunks;
  char* base = reinterpret_cast<char*>(workspace);
  unsigned* ticket = reinterpret_cast<unsigned*>(base);
  TokenSum* part = reinterpret_cast<TokenSum*>(base + 256);
  int* counts = reinterpret_cast<int*>(base + 256 + align_up((size_t)items * sizeof(TokenSum)));
  const int grid = items > 0 ? loss_grid(items) : 1;
  k_policy_counts<<<grid, kLossThreads, 0, s>>>(a, items, chunks, counts, ticket);
  k_policy_main<<<grid, kLossThreads, 0, s>>>(a, items, chunks, counts, part, ticket);
  return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
}

}  // extern "C"
