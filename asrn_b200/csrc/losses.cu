// Losses of fine-tuning on per-token log probabilities, each with its gradient in the same call: the preference loss of
// answer pairs and the clipped policy loss with a KL term. Both read each token once (13 and 17 to 21 bytes with the
// gradient written; the policy loss reads only the mask where a warp's tokens are all outside it) and compute next to
// nothing, so HBM bounds what they could do when large, and the launches when small.
//
// Every sum is formed in a fixed order in fp64 (per thread, then by warp shuffles, then over the blocks' partials in
// index order; in policy_main four neighbouring tokens are added in fp32 first): the results do not depend on the blocks'
// timing. On the device: preference 512 pairs x 4096 19 us (54.5 MB),
// policy 512 x 8192 26 us (88 MB, a third of the tokens counted): dependent rounds of loads, and about 100 instructions
// for a counted token; small calls 5.5 to 8 us, half of what the host needs to issue them. What is read outside the mask is
// selected away, never multiplied, so a NaN or infinity there reaches nothing.
#include <algorithm>
#include <initializer_list>
#include <cooperative_groups.h>
#include "common.cuh"
#include "layout.h"

namespace asrn {

namespace {

constexpr int kLossThreads = 256;
constexpr int kLossChunk = 4 * kLossThreads;   // tokens of one row that a block takes at a time, 4 a thread
constexpr int kLossBlocks = 5;           // that an SM holds at a time, by the kernels' launch bounds
constexpr int kLossGrid = 148 * 8;
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

// Sums over the block, in every thread; `slots` holds N values per warp. By shuffles within a warp, then each warp adds
// up the warps' sums, in the same order.
template <int N> __device__ __forceinline__ void block_sum(double (&v)[N], double* slots) {
  const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum_d(v[i]);
  __syncthreads();
  if (lane == 0)
#pragma unroll
    for (int i = 0; i < N; ++i) slots[(threadIdx.x >> 5) * N + i] = v[i];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < N; ++i) v[i] = warp_sum_d(lane < warps ? slots[lane * N + i] : 0.);
}

// A thread's four values of a chunk of a row: neighbours (Vec: rows and pointers allow 16-byte loads) or a block's width
// apart. place(j) is the j-th one's place in the chunk.
template <bool Vec> __device__ __forceinline__ int place(int j) {
  return Vec ? 4 * (int)threadIdx.x + j : j * kLossThreads + (int)threadIdx.x;
}
template <bool Vec> __device__ __forceinline__ void load4(float* v, const float* p, int left) {
  if (Vec) {
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (place<Vec>(0) < left) x = __ldg(reinterpret_cast<const float4*>(p + place<Vec>(0)));
    v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = place<Vec>(j) < left ? __ldg(p + place<Vec>(j)) : 0.f;
  }
}
template <bool Vec> __device__ __forceinline__ uint32_t load_mask(const uint8_t* p, int left) {   // bit j
  uint32_t m = 0;
  if (Vec) {
    if (place<Vec>(0) < left) {
      const uchar4 x = __ldg(reinterpret_cast<const uchar4*>(p + place<Vec>(0)));
      m = (uint32_t)((x.x != 0) | (x.y != 0) << 1 | (x.z != 0) << 2 | (x.w != 0) << 3);
    }
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (place<Vec>(j) < left) m |= (uint32_t)(__ldg(p + place<Vec>(j)) != 0) << j;
  }
  return m;
}
template <bool Vec> __device__ __forceinline__ void store4(float* p, const float* v, int left) {
  if (Vec) {
    if (place<Vec>(0) < left)
      *reinterpret_cast<float4*>(p + place<Vec>(0)) = make_float4(v[0], v[1], v[2], v[3]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (place<Vec>(j) < left) p[place<Vec>(j)] = v[j];
  }
}

__device__ __forceinline__ int chunk_left(int64_t L, int64_t t) { return (int)min(L - t, (int64_t)kLossChunk); }

// Rows in parts that blocks take: items = rows x parts, each of `width` tokens, a multiple of the chunk.
struct Split {
  int64_t items, parts, width;
};

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
    p.loss = (1. - a.smoothing) * (soft - fmin(x, 0.));
    if (a.smoothing > 0.) p.loss += a.smoothing * (soft + fmax(x, 0.));      // infinite where x is
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
  __shared__ double slots[64];
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
  double sums[2] = {p.on ? 1. : 0., p.loss};
  block_sum(sums, slots);
  const double pairs = fmax(1., sums[0]);
  if (threadIdx.x == 0) a.loss[0] = (float)(sums[1] / pairs);
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

__device__ __forceinline__ RowSum row_total(const RowSum* part, int64_t row, int64_t parts) {
  RowSum t{0., 0};
  for (int64_t c = 0; c < parts; ++c) {
    t.sum += part[row * parts + c].sum;
    t.n += part[row * parts + c].n;
  }
  return t;
}

// First the rows' sums by parts: item = (row, part of `width` tokens, a multiple of the chunk). Returns the masks of the
// first 16 chunks of the block's first item.
template <bool Vec> __device__ __forceinline__ uint64_t pref_sums(const PrefArgs& a, const Split& w, RowSum* part) {
  __shared__ double slots[16];
  uint64_t bits = 0;
  for (int64_t it = blockIdx.x; it < w.items; it += gridDim.x) {
    const int64_t begin = it % w.parts * w.width, base = it / w.parts * a.L + begin;
    const int64_t len = min(a.L - begin, w.width);         // none in the last parts of a short row
    double v[2] = {0., 0.};
    int n = 0;
#pragma unroll 4
    for (int64_t t = 0; t < len; t += kLossChunk) {
      float lp[4], rf[4];
      const int left = chunk_left(len, t);
      const uint32_t m = load_mask<Vec>(a.mask + base + t, left);
      load4<Vec>(lp, a.logp + base + t, left);
      load4<Vec>(rf, a.ref + base + t, left);
      if (it == blockIdx.x && t < 16 * kLossChunk) bits |= (uint64_t)m << (t / kLossChunk * 4);
      n += __popc(m);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[0] += m >> j & 1 ? (double)lp[j] - (double)rf[j] : 0.;
    }
    v[1] = (double)n;
    block_sum(v, slots);
    if (threadIdx.x == 0) part[it] = RowSum{v[0], (int64_t)v[1]};
  }
  return bits;
}

// Then, with every part there, the pairs that count, the loss (block 0) and the gradient. A block's first threads find the
// slopes of its items, one each, all at once.
template <bool Vec>
__device__ __forceinline__ void pref_finish(const PrefArgs& a, const Split& w, const RowSum* part, uint64_t bits) {
  __shared__ double slots[16];
  __shared__ float slope[kLossThreads];
  double v[2] = {0., 0.};
  for (int64_t p = threadIdx.x; p < a.P; p += kLossThreads) {
    const RowSum r0 = row_total(part, p, w.parts), r1 = row_total(part, a.P + p, w.parts);
    v[0] += r0.n > 0 && r1.n > 0 ? 1. : 0.;
    if (blockIdx.x == 0) {
      v[1] += pair_of(a, r0.sum, r1.sum, r0.n, r1.n).loss;
      a.rewards[p] = (float)(a.beta * r0.sum);
      a.rewards[a.P + p] = (float)(a.beta * r1.sum);
    }
  }
  block_sum(v, slots);
  const double pairs = fmax(1., v[0]);
  if (blockIdx.x == 0 && threadIdx.x == 0) a.loss[0] = (float)(v[1] / pairs);
  if (!a.grad) return;
  for (int64_t it0 = blockIdx.x; it0 < w.items; it0 += (int64_t)gridDim.x * kLossThreads) {
    const int64_t mine = it0 + (int64_t)threadIdx.x * gridDim.x;
    __syncthreads();
    if (mine < w.items) {
      const int64_t row = mine / w.parts, p = row % a.P;
      const RowSum r0 = row_total(part, p, w.parts), r1 = row_total(part, a.P + p, w.parts);
      const Pair q = pair_of(a, r0.sum, r1.sum, r0.n, r1.n);
      slope[threadIdx.x] = (float)((row < a.P ? q.slope0 : q.slope1) / pairs);
    }
    __syncthreads();
    for (int k = 0; k < kLossThreads; ++k) {
      const int64_t it = it0 + (int64_t)k * gridDim.x;
      if (it >= w.items) break;
      const int64_t begin = it % w.parts * w.width, base = it / w.parts * a.L + begin;
      const int64_t len = min(a.L - begin, w.width);
      const float s = slope[k];
#pragma unroll 4
      for (int64_t t = 0; t < len; t += kLossChunk) {
        const int left = chunk_left(len, t);
        const uint32_t m = it == blockIdx.x && t < 16 * kLossChunk ? (uint32_t)(bits >> (t / kLossChunk * 4)) & 15u
                                                                   : load_mask<Vec>(a.mask + base + t, left);
        const float d[4] = {m & 1 ? s : 0.f, m & 2 ? s : 0.f, m & 4 ? s : 0.f, m & 8 ? s : 0.f};
        store4<Vec>(a.grad + base + t, d, left);
      }
    }
  }
}

// Both in one cooperative launch, or in two that overlap.
template <bool Vec> __global__ void __launch_bounds__(kLossThreads, kLossBlocks) k_pref(PrefArgs a, Split w, RowSum* part) {
  const uint64_t bits = pref_sums<Vec>(a, w, part);
  cooperative_groups::this_grid().sync();
  pref_finish<Vec>(a, w, part, bits);
}
template <bool Vec> __global__ void __launch_bounds__(kLossThreads) k_pref_sums(PrefArgs a, Split w, RowSum* part) {
  let_next();
  pref_sums<Vec>(a, w, part);
}
template <bool Vec> __global__ void __launch_bounds__(kLossThreads) k_pref_finish(PrefArgs a, Split w, const RowSum* part) {
  uint64_t bits = 0;                             // the masks of the first item come while the sums are still being made
  if (blockIdx.x < w.items) {
    const int64_t begin = blockIdx.x % w.parts * w.width, base = blockIdx.x / w.parts * a.L + begin;
    const int64_t len = min(a.L - begin, w.width);
#pragma unroll 4
    for (int64_t t = 0; t < min(len, (int64_t)16 * kLossChunk); t += kLossChunk)
      bits |= (uint64_t)load_mask<Vec>(a.mask + base + t, chunk_left(len, t)) << (t / kLossChunk * 4);
  }
  wait_previous();
  pref_finish<Vec>(a, w, part, bits);
}

// ---- clipped policy loss -------------------------------------------------------------------------------------------

struct PolicyArgs {
  int64_t B, L;
  const float *logp, *old, *ref, *adv;   // (B, L); ref may be null; adv (B, L) or (B)
  const uint8_t* mask;
  int32_t adv_per_token, per_sequence;
  float log_low, log_high;               // log(1 - clip_low) rounded up, log(1 + clip_high) rounded down: a float
                                         // is beyond the rounded bound exactly when it is beyond the bound
  float low, high, kl;                   // 1 - clip_low, 1 + clip_high, KL coefficient
  float *loss, *grad, *stats;            // scalar, (B, L) or null, (2): mean KL estimate, share of clipped tokens
};

struct BlockSum {                        // of one block's tokens
  double loss, kl, cut;
};

struct Token {
  float loss, slope, kl;
  bool cut;
};

// x held to [-20, 20], a NaN staying one.
__device__ __forceinline__ float held20(float x) {
  float y;
  asm("{\n\t.reg .f32 t;\n\tmin.NaN.f32 t, %1, 0f41A00000;\n\tmax.NaN.f32 %0, t, 0fC1A00000;\n\t}" : "=f"(y) : "f"(x));
  return y;
}

// e^x for |x| <= 20 as 2^t, t = x log2 e rounded. What the rounding took (the product's by fma, and the part of log2 e that
// its float leaves out) is x log2 e - t = `lost`, below 2^-19; 2^lost = 1 + lost ln 2 to the first order, whose error is below
// 2^-40: within ex2.approx's 2^-22 and one rounding of e^x.
__device__ __forceinline__ float exp_held(float x) {
  const float t = x * 1.4426950408889634f;
  const float lost = fmaf(x, 1.4426950408889634f, -t) + x * 1.9259629911e-8f;
  float e;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(t));
  return fmaf(e * 0.6931471805599453f, lost, e);
}

// One token of the loss. The ratio's bounds are compared in the log domain, where the log ratio is exact or nearly so:
// which side a token falls on does not hang on an exponential's last bit. exp(q) - 1 - q and exp(q) - 1 come from Taylor's series
// below 1/4 (its next term is under 4e-7 of the sum), where the differences would cancel.
template <bool Ref>
__device__ __forceinline__ Token token_of(const PolicyArgs& a, float lp, float old, float rf, float adv) {
  Token t;
  const float d = lp - old, lr = held20(d);
  t.cut = adv > 0.f ? lr > a.log_high : adv < 0.f && lr < a.log_low;
  const float r = t.cut ? (adv > 0.f ? a.high : a.low) : exp_held(lr);
  t.loss = -r * adv;
  t.slope = t.cut || fabsf(d) > 20.f ? 0.f : t.loss;
  t.kl = 0.f;
  if (Ref) {
    const float dq = rf - lp, q = held20(dq);
    const bool near = fabsf(q) < 0.25f;
    const float e = exp_held(q) - 1.f;
    t.kl = near ? q * q * (0.5f + q * (1.f / 6 + q * (1.f / 24 + q * (1.f / 120 + q * (1.f / 720))))) : e - q;
    t.loss = fmaf(a.kl, t.kl, t.loss);
    t.slope = fabsf(dq) > 20.f ? t.slope : fmaf(-a.kl, near ? q + t.kl : e, t.slope);
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

template <bool Ref> __global__ void __launch_bounds__(1024) k_policy_small(PolicyArgs a) {
  __shared__ int cnt[kSmallRows];
  __shared__ double slots[96];
  const int rows = (int)a.B, L = (int)a.L, lane = threadIdx.x & 31;
  double n[2] = {0., 0.};
  for (int r = threadIdx.x >> 5; r < rows; r += blockDim.x >> 5) {
    int c = 0;
#pragma unroll 4
    for (int t = lane; t < L; t += 32) c += a.mask[(int64_t)r * L + t] != 0;
    c = warp_sum_i(c);
    if (lane == 0) {
      cnt[r] = c;
      n[0] += c;
      n[1] += c > 0 ? 1. : 0.;
    }
  }
  block_sum(n, slots);
  const double total = fmax(1., n[0]), seqs = fmax(1., n[1]);
  double v[3] = {0., 0., 0.};
  const int all = rows * L;
#pragma unroll 2
  for (int i = threadIdx.x; i < all; i += blockDim.x) {
    const int row = i / L;
    const bool on = a.mask[i];
    const float lp = a.logp[i], old = a.old[i], rf = Ref ? a.ref[i] : 0.f, adv = a.adv[a.adv_per_token ? i : row];
    float g = 0.f;
    if (on) {
      const Token t = token_of<Ref>(a, lp, old, rf, adv);
      const double w = a.per_sequence ? 1. / cnt[row] : 1.;
      v[0] += w * (double)t.loss;
      v[1] += (double)t.kl;
      v[2] += t.cut ? 1. : 0.;
      g = (float)((double)t.slope * w / (a.per_sequence ? seqs : total));
    }
    if (a.grad) a.grad[i] = g;
  }
  block_sum(v, slots);
  if (threadIdx.x == 0) policy_results(a, v[0], v[1], n[0], v[2], n[1]);
}

__device__ __forceinline__ int row_count(const int* counts, int64_t row, int64_t parts) {
  int c = 0;
  for (int64_t k = 0; k < parts; ++k) c += counts[row * parts + k];
  return c;
}

// First the tokens of each part of each row (and block 0 clears the ticket).
template <bool Vec>
__device__ __forceinline__ void policy_counts(const PolicyArgs& a, const Split& w, int* counts, unsigned* ticket) {
  __shared__ double slots[8];
  if (blockIdx.x == 0 && threadIdx.x == 0) *ticket = 0u;
  for (int64_t it = blockIdx.x; it < w.items; it += gridDim.x) {
    const int64_t begin = it % w.parts * w.width, base = it / w.parts * a.L + begin;
    const int64_t len = min(a.L - begin, w.width);
    int c = 0;
#pragma unroll 4
    for (int64_t t = 0; t < len; t += kLossChunk) c += __popc(load_mask<Vec>(a.mask + base + t, chunk_left(len, t)));
    double v[1] = {(double)c};
    block_sum(v, slots);
    if (threadIdx.x == 0) counts[it] = (int)v[0];
  }
}

// Then, once `ready` has every count there, the tokens' losses, the gradient and each block's sums, chunks dealt out in
// turn (a row's prompt and padding cost little); the block that finishes last adds the sums up in index order.
template <bool Vec, bool Ref, class Ready>
__device__ __forceinline__ void policy_main(const PolicyArgs& a, int64_t chunks, int64_t parts, const int* counts,
                                            BlockSum* part, unsigned* ticket, Ready ready) {
  __shared__ double slots[24];
  __shared__ bool last;
  const int64_t step_r = gridDim.x / chunks, step_c = gridDim.x % chunks, stride_c = step_c * kLossChunk;
  int64_t row = blockIdx.x / chunks, t = blockIdx.x % chunks * kLossChunk;
  // the mask comes an item ahead: a warp whose tokens are all outside it reads nothing else
  uint32_t next = row < a.B ? load_mask<Vec>(a.mask + row * a.L + t, chunk_left(a.L, t)) : 0;
  // and so do its row's count and advantage
  const auto row_share = [&](int64_t r) {
    return a.per_sequence && r < a.B ? 1.f / (float)max(1, row_count(counts, r, parts)) : 1.f;
  };
  const auto row_advantage = [&](int64_t r) { return a.adv_per_token || r >= a.B ? 0.f : __ldg(a.adv + r); };
  float next_adv = row_advantage(row);
  ready();
  float next_share = row_share(row);
  double n[2] = {0., 0.};
  for (int64_t b = threadIdx.x; b < a.B; b += kLossThreads) {
    const int c = row_count(counts, b, parts);
    n[0] += (double)c;
    n[1] += c > 0 ? 1. : 0.;
  }
  block_sum(n, slots);
  const float over = (float)(1. / (a.per_sequence ? fmax(1., n[1]) : fmax(1., n[0])));
  double v[3] = {0., 0., 0.};
  int cut = 0;
  while (row < a.B) {
    const float share = next_share, row_adv = next_adv;
    const float w = share * over;
    const int64_t at = row * a.L + t;
    const int left = chunk_left(a.L, t);
    const uint32_t m = next;
    t += stride_c;
    row += step_r;
    if (t >= chunks * kLossChunk) {
      t -= chunks * kLossChunk;
      ++row;
    }
    float lp[4], old[4], rf[4] = {0.f, 0.f, 0.f, 0.f}, adv[4] = {row_adv, row_adv, row_adv, row_adv};
    float d[4] = {0.f, 0.f, 0.f, 0.f};
    const bool any = __any_sync(0xffffffffu, m);
    if (any) {
      load4<Vec>(lp, a.logp + at, left);
      load4<Vec>(old, a.old + at, left);
      if (Ref) load4<Vec>(rf, a.ref + at, left);
      if (a.adv_per_token) load4<Vec>(adv, a.adv + at, left);
    }
    if (row < a.B) next = load_mask<Vec>(a.mask + row * a.L + t, chunk_left(a.L, t));
    next_share = row_share(row);
    next_adv = row_advantage(row);
    if (any) {
      float loss = 0.f, kl = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {                // a token outside the mask: all zeros, whose loss and slope are zero
        const bool on = m >> j & 1;
        const Token k = token_of<Ref>(a, on ? lp[j] : 0.f, on ? old[j] : 0.f, on ? rf[j] : 0.f, on ? adv[j] : 0.f);
        loss += k.loss;
        kl += k.kl;
        cut += k.cut;
        d[j] = k.slope * w;
      }
      v[0] += (double)(share * loss);              // 4 terms in fp32, then fp64
      v[1] += (double)kl;
    }
    if (a.grad) store4<Vec>(a.grad + at, d, left);
  }
  v[2] = (double)cut;
  block_sum(v, slots);
  if (threadIdx.x == 0) {
    part[blockIdx.x] = BlockSum{v[0], v[1], v[2]};
    __threadfence();
    last = atomicAdd(ticket, 1u) == gridDim.x - 1;
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  v[0] = v[1] = v[2] = 0.;
  for (int b = threadIdx.x; b < (int)gridDim.x; b += kLossThreads) {
    const volatile BlockSum* t = part + b;
    v[0] += t->loss;
    v[1] += t->kl;
    v[2] += t->cut;
  }
  block_sum(v, slots);
  if (threadIdx.x == 0) policy_results(a, v[0], v[1], n[0], v[2], n[1]);
}

// Both in one cooperative launch, or in two that overlap.
template <bool Vec, bool Ref>
__global__ void __launch_bounds__(kLossThreads, kLossBlocks)
k_policy(PolicyArgs a, int64_t chunks, Split w, int* counts, BlockSum* part, unsigned* ticket) {
  policy_counts<Vec>(a, w, counts, ticket);
  policy_main<Vec, Ref>(a, chunks, w.parts, counts, part, ticket, [] { cooperative_groups::this_grid().sync(); });
}
template <bool Vec>
__global__ void __launch_bounds__(kLossThreads) k_policy_counts(PolicyArgs a, Split w, int* counts, unsigned* ticket) {
  let_next();
  policy_counts<Vec>(a, w, counts, ticket);
}
template <bool Vec, bool Ref>
__global__ void __launch_bounds__(kLossThreads, kLossBlocks)
k_policy_main(PolicyArgs a, int64_t chunks, Split w, const int* counts, BlockSum* part, unsigned* ticket) {
  policy_main<Vec, Ref>(a, chunks, w.parts, counts, part, ticket, [] { wait_previous(); });
}

int64_t loss_chunks(int64_t L) { return (L + kLossChunk - 1) / kLossChunk; }

// Tokens up to which one cooperative launch does it all, and above which two overlapping launches do. The second launch
// costs the host about 2.5 us; the cooperative one costs the GPU about 4: it starts on an idle GPU, holds fewer blocks, and
// waits at its barrier. Us a call, two launches / one: preference 16.1 / 13.3 at 2^18 tokens, 16.4 / 14.4 at 512 x 2048, 16.4 /
// 16.4 at 2^21, 22.5 / 25.7 at 2^22; policy 11.0 / 10.3 at 2^18, 12.3 / 13.5 at 2^19, 14.4 / 18.4 at 2^20.
constexpr int64_t kPrefTogether = 1 << 21, kPolicyTogether = 1 << 18;

int loss_grid(int64_t items, int per_sm) {
  static int sms = 0;
  int dev = 0;
  if (sms == 0 && (cudaGetDevice(&dev) != cudaSuccess ||
                   cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0))
    sms = 148;
  return (int)std::max<int64_t>(1, std::min<int64_t>(items, std::min(kLossGrid, sms * per_sm)));
}

// Cooperatively, or behind the kernel before it on the stream, which it waits for itself (wait_previous).
template <class... P, class... A>
int launch_with(cudaLaunchAttributeID how, void (*kernel)(P...), int grid, cudaStream_t s, const A&... args) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(kLossThreads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = how;
  if (how == cudaLaunchAttributeCooperative) attr[0].val.cooperative = 1;
  else attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, (P)args...) == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
}

// Rows of a multiple of 4 tokens on 16-byte boundaries (the mask's on 4) are read four tokens at a time.
bool vec_ok(int64_t L, std::initializer_list<const void*> fs, const void* mask) {
  if (L % 4 || (uintptr_t)mask % 4) return false;
  for (const void* f : fs)
    if ((uintptr_t)f % 16) return false;
  return true;
}

float rounded(double x, bool up) {
  const float f = (float)x;
  return up ? ((double)f < x ? nextafterf(f, INFINITY) : f) : ((double)f > x ? nextafterf(f, -INFINITY) : f);
}

// Rows in parts: as many as a full grid has blocks for, each of a chunk at least (every block adds all parts up again).
Split split_rows(int64_t rows, int64_t L) {
  const int64_t chunks = loss_chunks(L);
  const int64_t parts = std::max<int64_t>(1, std::min<int64_t>(kLossGrid / std::max<int64_t>(1, rows), chunks));
  return Split{rows * parts, parts, (chunks + parts - 1) / parts * kLossChunk};
}

// Tokens up to which one block does it by itself, without a workspace. Us a call, one block / the cooperative launch:
// preference 11.9 / 13.3 at 2^14 tokens, 15.0 / 13.7 at 2^15; policy, with more to compute for a token, 8.8 / 10.2 at 2^12,
// 12.1 / 10.2 at 2^13.
constexpr int64_t kPrefSmall = 1 << 14, kPolicySmall = 1 << 12;
bool small_loss(int64_t rows, int64_t L, int64_t most) { return rows <= kSmallRows && rows * L <= most; }

}  // namespace
}  // namespace asrn

extern "C" {

size_t asrn_preference_workspace_bytes(int64_t P, int64_t L) {
  if (P < 0 || L < 0 || asrn::small_loss(2 * P, L, asrn::kPrefSmall)) return 0;
  return asrn::align_up((size_t)asrn::split_rows(2 * P, L).items * sizeof(asrn::RowSum) + 1);
}

int asrn_preference_loss(int64_t P, int64_t L, const float* logp, const float* ref_logp, const uint8_t* mask,
                         int32_t kind, double beta, double smoothing, float* loss, float* grad, float* rewards,
                         void* workspace, size_t workspace_bytes, void* stream) {
  using namespace asrn;
  if (P < 0 || L < 0 || kind < 0 || kind > 1 || !(beta > 0.) || !(smoothing >= 0. && smoothing < 0.5) || !loss)
    return ASRN_ERR_ARG;
  if (P > ((int64_t)1 << 30) || L > ((int64_t)1 << 30)) return ASRN_ERR_UNSUPPORTED;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const PrefArgs a{P, L, logp, ref_logp, mask, kind, beta, smoothing, loss, grad, rewards};
  if (P * L > 0 && (!logp || !ref_logp || !mask)) return ASRN_ERR_ARG;
  if (P > 0 && !rewards) return ASRN_ERR_ARG;
  if (small_loss(2 * P, L, kPrefSmall)) {
    k_pref_small<<<1, 1024, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
  }
  if (!workspace || workspace_bytes < asrn_preference_workspace_bytes(P, L) || (uintptr_t)workspace % 16)
    return ASRN_ERR_WORKSPACE;
  const Split w = split_rows(2 * P, L);
  RowSum* part = reinterpret_cast<RowSum*>(workspace);
  const bool vec = vec_ok(L, {logp, ref_logp, grad}, mask);
  if (2 * P * L <= kPrefTogether)
    return launch_with(cudaLaunchAttributeCooperative, vec ? k_pref<true> : k_pref<false>, loss_grid(w.items, kLossBlocks), s,
                       a, w, part);
  const int grid = loss_grid(w.items, 8);
  if (vec) k_pref_sums<true><<<grid, kLossThreads, 0, s>>>(a, w, part);
  else k_pref_sums<false><<<grid, kLossThreads, 0, s>>>(a, w, part);
  if (cudaGetLastError() != cudaSuccess) return ASRN_ERR_CUDA;
  return launch_with(cudaLaunchAttributeProgrammaticStreamSerialization, vec ? k_pref_finish<true> : k_pref_finish<false>,
                     grid, s, a, w, part);
}

size_t asrn_policy_workspace_bytes(int64_t B, int64_t L) {
  if (B < 0 || L < 0 || asrn::small_loss(B, L, asrn::kPolicySmall)) return 0;
  return 256 + asrn::align_up(asrn::kLossGrid * sizeof(asrn::BlockSum)) +
         asrn::align_up((size_t)asrn::split_rows(B, L).items * sizeof(int) + 1);
}

int asrn_policy_loss(int64_t B, int64_t L, const float* logp, const float* old_logp, const float* ref_logp,
                     const float* advantages, int32_t adv_per_token, const uint8_t* mask, double clip_low,
                     double clip_high, double kl, int32_t per_sequence, float* loss, float* grad, float* stats,
                     void* workspace, size_t workspace_bytes, void* stream) {
  using namespace asrn;
  if (B < 0 || L < 0 || !(clip_low >= 0. && clip_low < 1.) || !(clip_high >= 0.) || !(kl >= 0.) || !loss || !stats)
    return ASRN_ERR_ARG;
  if (B > ((int64_t)1 << 30) || L > ((int64_t)1 << 30)) return ASRN_ERR_UNSUPPORTED;
  if (B * L > 0 && (!logp || !old_logp || !advantages || !mask || (kl > 0. && !ref_logp))) return ASRN_ERR_ARG;
  if (L == 0) B = 0;                     // sequences without positions: nothing to count, read or write but the results
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const PolicyArgs a{B, L, logp, old_logp, ref_logp, advantages, mask, adv_per_token != 0, per_sequence != 0,
                     rounded(log1p(-clip_low), true), rounded(log1p(clip_high), false), (float)(1. - clip_low), (float)(1. + clip_high), (float)kl,
                     loss, grad, stats};
  if (small_loss(B, L, kPolicySmall)) {
    if (ref_logp) k_policy_small<true><<<1, 1024, 0, s>>>(a);
    else k_policy_small<false><<<1, 1024, 0, s>>>(a);
    return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
  }
  if (!workspace || workspace_bytes < asrn_policy_workspace_bytes(B, L) || (uintptr_t)workspace % 16)
    return ASRN_ERR_WORKSPACE;
  char* base = reinterpret_cast<char*>(workspace);
  unsigned* ticket = reinterpret_cast<unsigned*>(base);
  BlockSum* part = reinterpret_cast<BlockSum*>(base + 256);
  int* counts = reinterpret_cast<int*>(base + 256 + align_up(kLossGrid * sizeof(BlockSum)));
  const Split w = split_rows(B, L);
  const int64_t chunks = loss_chunks(L);
  const bool vec = vec_ok(L, {logp, old_logp, ref_logp, adv_per_token ? advantages : nullptr, grad}, mask);
  const int grid = loss_grid(B * chunks, kLossBlocks);
  if (B * L <= kPolicyTogether) {
    const auto kernel = vec ? (ref_logp ? k_policy<true, true> : k_policy<true, false>)
                            : (ref_logp ? k_policy<false, true> : k_policy<false, false>);
    return launch_with(cudaLaunchAttributeCooperative, kernel, grid, s, a, chunks, w, counts, part, ticket);
  }
  const int cgrid = loss_grid(w.items, 8);
  if (vec) k_policy_counts<true><<<cgrid, kLossThreads, 0, s>>>(a, w, counts, ticket);
  else k_policy_counts<false><<<cgrid, kLossThreads, 0, s>>>(a, w, counts, ticket);
  if (cudaGetLastError() != cudaSuccess) return ASRN_ERR_CUDA;
  const auto kernel = vec ? (ref_logp ? k_policy_main<true, true> : k_policy_main<true, false>)
                          : (ref_logp ? k_policy_main<false, true> : k_policy_main<false, false>);
  return launch_with(cudaLaunchAttributeProgrammaticStreamSerialization, kernel, grid, s, a, chunks, w, counts, part, ticket);
}

}  // extern "C"
