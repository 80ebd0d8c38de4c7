// Log probabilities through the tied head with the distribution's entropy and its likeliest tokens, forward and backward:
//   s_iv = h_i . w_v / tau,  lse = log sum_v exp s_v,  logp = s_y - lse,  H = lse - sum_v p_v s_v,  the `top` largest s_v - lse
//   dS_v = (1 / tau) [g (delta_{v,y} - p_v) - gH p_v (log p_v + H)],  dh = dS W,  dW = dS^T h
// The products are those of the log probabilities alone (head.cu): 2 N V d operations forward and 6 N V d backward, bound by the
// tensor cores at any training size, and by the weight's bytes where rows are few.
//
//   k_gemm<Scan>   scores by tiles; each thread keeps of its row's 64 columns the maximum m, S = sum exp(s - m), T = sum
//                  exp(s - m) (s - m); the target is in none of the sums. Where the likeliest tokens are wanted, it notes of each
//                  group of 32 or 64 columns the largest score, and the second largest with the largest one's column in its low
//                  6 bits (small vocabularies: all scores)
//   k_stats_few    the same for few rows
//   k_stats_sizes  the largest |w|^2 of W's rows, beside or behind the scan (k_stats_few's blocks find it themselves)
//   k_stats_rows   a warp per row: its sums joined, logp, H; then the groups with the largest scores, which in most rows are the
//                  likeliest tokens'. Where a second score of a group may count, scores are formed again from h and W by sums
//                  in fp32, and where these or the products' leave the order open by sums in 64 bits. So the order of the tokens
//                  is that of their exact scores, equal ones by their numbers. What a sum in fp32 may be off by is taken from
//                  |h| |w| >= sum |h w|, with the largest |w| of the vocabulary
//   k_gemm<Slope>  backward: the scores again, dS in bf16; then the two products
#include <algorithm>
#include "head.cuh"
#include "products.cuh"

namespace asrn {

namespace {

using gemm::exp2_fast;

constexpr float kLn2 = 0.69314718055994531f;
constexpr float kNothing = -3.3e38f;       // of columns that do not count: its exponential is 0, and its bits can be marked
constexpr float kLeast = -200.f;           // log2 of what is as good as 0: keeps 0 x infinity out of the sums of p log p
constexpr int kMaxTop = 32;

struct StatsSaved {                        // HeadSaved with logp in the place of `rest`, and
  HeadSaved head;
  size_t ent, total;
};

StatsSaved stats_saved(int64_t N, int64_t d) {
  StatsSaved w{};
  w.head = head_saved(N, d);
  w.ent = w.head.total;
  w.total = align_up(w.ent + (size_t)pad256(N) * 4);
  return w;
}

// A row's sums are kept by 64 columns, what one thread of the products' epilogue holds of it.
constexpr int kPart = 64;
__host__ ASRN_DEV int parts_of(int64_t V) { return (int)((V + gemm::kBN - 1) / gemm::kBN) * (gemm::kBN / kPart); }

// Columns of a group: of a group that holds two of the likeliest tokens all have to be looked at, so 32 as long as a row's groups
// stay few enough for a warp to hold in registers. Where looking at them (top^2 / V groups, 32 scores of d products) costs more than
// reading a score of each column, groups of 1: all scores are kept.
// All scores | groups of 32, us: 10816 x 1265 x 608, 8 tokens 122 | 104, 12 tokens 142 | 157, 32 tokens 283 | 722;
// 4096 x 2000 x 256, 20 tokens 95 | 73, 32 tokens 151 | 181; 8192 x 256 x 64, 3 tokens 28 | 29, 8 tokens 37 | 47.
int span_of(int64_t V, int d, int top) { return V <= 2048 && V * V <= 24 * top * top * (int64_t)d ? 1 : V <= 32768 ? 32 : 64; }
int64_t notes_of(int64_t V, int d, int top) { return (V + span_of(V, d, top) - 1) / span_of(V, d, top); }
// Bytes of a row's notes: two numbers a group, or one a column (whole chunks of 32).
int64_t note_bytes(int64_t V, int d, int top) { return span_of(V, d, top) == 1 ? (V + 31) / 32 * 128 : notes_of(V, d, top) * 8; }

// Numbers that say how large W's rows are, one of each block of k_stats_few or of k_stats_sizes (no more than stay on the SMs at once).
constexpr int kSizeWarps = 8, kSizeRows = 4;             // k_stats_sizes: a block's warps, a warp's rows at a time
int size_blocks(int64_t V) { return (int)std::min<int64_t>(3 * gemm::sm_count(), (V + kSizeWarps * kSizeRows - 1) / (kSizeWarps * kSizeRows)); }

struct StatsWs {
  size_t counts, top, part, notes, sizes, total;
};

StatsWs stats_ws(int64_t N, int64_t V, int d, int top) {
  StatsWs w{};
  const size_t P = (size_t)pad256(N), parts = (size_t)parts_of(V);
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes); return at; };
  w.counts = take((size_t)((N + kCountRows - 1) / kCountRows) * 4);
  w.top = take(P * 4);
  w.part = take(parts * P * 16);
  w.notes = take(top ? (size_t)note_bytes(V, d, top) * P : 0);
  w.sizes = take(top ? (size_t)std::max(size_blocks(V), parts_of(V) / 2) * 4 : 0);
  w.total = o;
  return w;
}

ASRN_DEV float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// What is noted of a group: its largest score, and its second largest with the largest one's column in the low 6 bits.
ASRN_DEV float2 note_of(float most, float first, float second) {
  return make_float2(most, __uint_as_float((__float_as_uint(second) & ~63u) | (__float_as_uint(first) & 63u)));
}

// Bound by the tensor cores and, where the two largest of each group are tracked, by the epilogue's instructions beside them (16 warps;
// with 8 the epilogue waits for itself): 16384 x 50304 x 768 (1.27 TFLOP) 870 us without, 1000 us with, 1.27 PFLOP/s; a look at
// 2048 rows: tensor pipe 62 % active, L2 hits 84 %.
template <bool Top> struct Scan {
  static constexpr int kWarps = 16, kOwn = 1, kTable = 0;
  struct Params {
    const int* tok;                        // null: no targets
    float k;                               // log2(e) / tau
    float* top;                            // the targets' unscaled scores
    float4* part;                          // m, S, T log2(e): [rows][parts]
    float2* notes;                         // of each group: [rows][groups]; span 1: the scores, floats [rows][whole chunks]
    int span, groups;
    float* sizes;                          // k_stats_few: the largest |w|^2 of each block's columns
  };
  const Params& p;
  int row, V, y, at, parts;
  bool on;
  float m = -INFINITY, s = 0.f, t = 0.f, most = kNothing, first = kNothing, second = kNothing;
  ASRN_DEV Scan(const Params& pp, int r, int rows, const gemm::Shape& sh, const gemm::Tile& u, int quarter)
      : p(pp), row(r), V(sh.N), y(-1), at(u.n * (gemm::kBN / kPart) + quarter), parts(parts_of(sh.N)), on(r < rows) {
    if (on && p.tok) y = p.tok[r];
  }
  template <class O> ASRN_DEV void chunk(float* v, int c, O&, const CUtensorMap*, const CUtensorMap*) {
    if (c >= V) return;
    const int n = V - c, j = y - c;        // n: valid columns, 32 or more but in the last tile
    if (j >= 0 && j < 32) {
      float own = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        own = i == j ? v[i] : own;
        v[i] = i == j ? kNothing : v[i];
      }
      p.top[row] = own;
    }
    if (n < 32) {
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = i < n ? v[i] : kNothing;
    }
    float here = v[0];
#pragma unroll
    for (int i = 1; i < 31; i += 2) here = max3(here, v[i], v[i + 1]);
    here = fmaxf(here, v[31]);
    const float now = fmaxf(m, here);
    const float off = now <= kNothing ? 0.f : now * p.k;
    const gemm::F2 k2(p.k), off2(-off);
    gemm::F2 add(0.f), sum(0.f);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float a, b;
      const gemm::F2 x = gemm::fma2(gemm::F2(v[i], v[i + 1]), k2, off2);
      x.get(a, b);
      const gemm::F2 e(exp2_fast(a), exp2_fast(b));
      add = gemm::add2(add, e);
      sum = gemm::fma2(e, x, sum);
    }
    float a, b, c0, c1;
    sum.get(a, b);
    add.get(c0, c1);
    float part = a + b;
    if (!(fabsf(part) < INFINITY)) {       // 0 x infinity, of a column that does not count: again without it
      part = 0.f;
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        const float x = fmaf(v[i], p.k, -off);
        part = fmaf(exp2_fast(x), fmaxf(x, kLeast), part);
      }
    }
    const float step = fmaxf(fmaf(m, p.k, -off), kLeast), f = exp2_fast(fmaf(m, p.k, -off));
    t = fmaf(f, fmaf(step, s, t), part);
    s = fmaf(s, f, c0 + c1);
    m = now;
    if constexpr (Top) {
      if (p.span == 1) {
        if (on) {
          float4* to = reinterpret_cast<float4*>(reinterpret_cast<float*>(p.notes) + (int64_t)row * ((V + 31) / 32 * 32) + c);
#pragma unroll
          for (int i = 0; i < 8; ++i) to[i] = make_float4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3]);
        }
        return;
      }
      // Two chains of pairs, then one; the chunk's place in the group in the low bits, too.
      float m1[2] = {kNothing, kNothing}, m2[2] = {kNothing, kNothing};
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const float u0 = __uint_as_float((__float_as_uint(v[i]) & ~63u) | (uint32_t)i);
        const float u1 = __uint_as_float((__float_as_uint(v[i + 1]) & ~63u) | (uint32_t)(i + 1));
        const float hi = fmaxf(u0, u1), lo = fminf(u0, u1);
        float &q1 = m1[i >> 1 & 1], &q2 = m2[i >> 1 & 1];
        q2 = max3(q2, lo, fminf(q1, hi));
        q1 = fmaxf(q1, hi);
      }
      const float lo = fminf(m1[0], m1[1]);
      const float hi = __uint_as_float(__float_as_uint(fmaxf(m1[0], m1[1])) | (uint32_t)(c & (p.span - 1)));
      second = fmaxf(max3(second, lo, fminf(first, hi)), fmaxf(m2[0], m2[1]));
      first = fmaxf(first, hi);
      most = fmaxf(most, here);
      if (((c + 32) & (p.span - 1)) == 0 || c + 32 >= V) {
        if (on) p.notes[(int64_t)row * p.groups + c / p.span] = note_of(most, first, second);
        most = first = second = kNothing;
      }
    }
  }
  ASRN_DEV void finish() {
    if (!on) return;
    p.part[(int64_t)row * parts + at] = make_float4(m <= kNothing ? -INFINITY : m, s, t, 0.f);
  }
};

// Squares of sums |w|^2 whose terms leave fp32's range: below, twice this stands for them.
constexpr float kSmallSquare = 0x1p-100f;
ASRN_DEV bool plain_square(float q) { return q >= kSmallSquare && q < INFINITY; }
// The squares of eight values added up in bf16, by twos (a quarter of fp32's instructions: 8 x 50304 x 768 12.5 us, with mma.sync of the
// rows by themselves 13.7, with fp32 16.6): half a step is 2^-8, so 16 of them are off by up to 2^-4 of the sum, a norm by 2^-5.
using Two = __nv_bfloat162;
ASRN_DEV Two no_squares() { return __floats2bfloat162_rn(0.f, 0.f); }
ASRN_DEV void add_squares(Two& q, const uint4& a) {
  const uint32_t x[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const Two v = *reinterpret_cast<const Two*>(&x[i]);
    q = __hfma2(v, v, q);
  }
}
ASRN_DEV float sum_of(const Two& q) { return __low2float(q) + __high2float(q); }

// A row's |w|^2 but for that, for the whole warp: 0 for a row of zeros, and for one with an infinity or a NaN, whose scores are not
// finite whatever the sums round; infinity where it is out of range.
ASRN_DEV float row_square(const uint4* row, int vecs) {
  float q = 0.f;
  uint32_t any = 0;
  bool bad = false;
#pragma unroll 4
  for (int c = threadIdx.x & 31; c < vecs; c += 32) {
    const uint4 a = __ldcg(row + c);                     // from L2, as k_stats_sizes reads
    const uint32_t x[4] = {a.x, a.y, a.z, a.w};
    Two sum = no_squares();
    add_squares(sum, a);
    q += sum_of(sum);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      any |= x[k] & 0x7fff7fffu;
      bad |= (x[k] & 0x7f80u) == 0x7f80u || (x[k] >> 16 & 0x7f80u) == 0x7f80u;
    }
  }
  q = warp_sum(q);
  if (plain_square(q)) return q;
  if (__any_sync(0xffffffffu, bad) || !__any_sync(0xffffffffu, any != 0)) return 0.f;
  return fmaxf(q, 2.f * kSmallSquare);
}

// The largest |w|^2 of each block's rows of W. Launched behind k_gemm<Scan>, whose blocks let it start once all that was before them is
// complete: it needs nothing of the scan's, and runs beside it on SMs that the scan leaves idle, else behind it. (Loads past L1, which
// no wait of its own has made sure of.) Then it waits for the scan, so that the kernel behind waits for both. Bound by memory, once
// over W: 50304 x 768 16.5 us (77 MB, 4.7 TB/s), 9 from L2 behind a scan of few rows; a block for each SM 33 and 22.
__global__ void __launch_bounds__(kSizeWarps * 32, 3)
k_stats_sizes(int64_t V, int vecs, const uint4* __restrict__ W, float* __restrict__ sizes) {
  constexpr int kU = 3;                                  // loads of a row under way together
  __shared__ float most[kSizeWarps];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  let_next();
  float best = 0.f;
  for (int64_t v0 = ((int64_t)blockIdx.x * kSizeWarps + wid) * kSizeRows; v0 < V; v0 += (int64_t)gridDim.x * kSizeWarps * kSizeRows) {
    const uint4* row[kSizeRows];
    float sum[kSizeRows] = {};
#pragma unroll
    for (int i = 0; i < kSizeRows; ++i) row[i] = W + (v0 + i < V ? v0 + i : V - 1) * vecs;   // past the last one: that one again
    for (int c = lane; c - lane < vecs; c += 32 * kU) {
      uint4 a[kU][kSizeRows];
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int i = 0; i < kSizeRows; ++i) a[u][i] = __ldcg(row[i] + min(c + 32 * u, vecs - 1));
#pragma unroll
      for (int i = 0; i < kSizeRows; ++i) {
        Two q = no_squares();
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (c + 32 * u < vecs) add_squares(q, a[u][i]);
        sum[i] += sum_of(q);
      }
    }
#pragma unroll
    for (int i = 0; i < kSizeRows; ++i) {
      float q = warp_sum(sum[i]);
      if (!plain_square(q)) q = row_square(row[i], vecs);
      best = fmaxf(best, q);
    }
  }
  if (lane == 0) most[wid] = best;
  __syncthreads();
  if (threadIdx.x == 0) {
#pragma unroll
    for (int k = 1; k < kSizeWarps; ++k) best = fmaxf(best, most[k]);
    sizes[blockIdx.x] = best;
  }
  wait_previous();
}

// The same for few rows, bound by the weight's bytes: block = 128 columns, a warp 16 of them and all of K; mma.sync from
// registers (A = 16 rows of W, B = the rows of h; the order of K inside a tile is free as long as both agree, so a lane takes 8
// neighbouring values of each), whose loads keep the memory busier than two rounds of 128 x 256 tiles do. Then a warp per row
// of h over the 128 scores. 8 x 50304 x 768: 12.5 us with 77 MB partly from L2, 6.2 TB/s (11.8 without the squares of W's rows).
// The whole call as a graph replay, so | by tiles, us, 5 tokens: 50304 x 768, 1 row 19 | 36, 8 rows 24 | 39, 16 rows 33 | 41, 20 rows 42 | 40;
// 16384 x 768, 8 rows 16 | 23, 16 rows 20 | 25, 32 rows 24 | 25; 5003 x 200, 32 rows 17 | 18; without tokens: 50304 x 768, 8 rows
// 13 | 21, 16 rows 20 | 21, 20 rows 27 | 21; 16384 x 768, 16 rows 10 | 12, 32 rows 12 | 11.
bool few_rows(int64_t N, int64_t V) { return N <= 16 || (N <= 32 && N * V < (1 << 18)); }
template <int NT, bool Top>
__global__ void __launch_bounds__(256)
k_stats_few(int N, int V, int d, const __nv_bfloat16* __restrict__ h, const __nv_bfloat16* __restrict__ w,
            const int* __restrict__ count, const typename Scan<Top>::Params p) {
  constexpr int kU = NT <= 2 ? 4 : 2;                    // steps of K whose loads are under way together
  __shared__ __align__(16) float sh[8 * NT][132];
  __shared__ float sizes[8];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
  const int v0 = blockIdx.x * 128 + wid * 16;
  wait_previous();
  let_next();
  const int rows = count ? *count : N;
  if (rows <= 0) return;
  // Rows past the last are the last one's again (their scores go nowhere), and what is past K is read from its end, and then zero: loads
  // without a condition are all under way at once.
  const __nv_bfloat16 *wp[2], *hp[NT];
#pragma unroll
  for (int i = 0; i < 2; ++i) wp[i] = w + (int64_t)min(v0 + g + i * 8, V - 1) * d + 8 * t;
#pragma unroll
  for (int i = 0; i < NT; ++i) hp[i] = h + (int64_t)min(g + i * 8, rows - 1) * d + 8 * t;
  float acc[NT][4] = {};
  float squares[2] = {};                                 // of W's two rows
  for (int k0 = 0; k0 < d; k0 += kU * 32) {
    uint4 a[kU][2], b[kU][NT];
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (k0 + u * 32 >= d) break;                       // the same for the whole warp
      const int k = min(k0 + u * 32, d - 8 - 8 * t);
#pragma unroll
      for (int i = 0; i < 2; ++i) a[u][i] = __ldg(reinterpret_cast<const uint4*>(wp[i] + k));
#pragma unroll
      for (int i = 0; i < NT; ++i) b[u][i] = __ldg(reinterpret_cast<const uint4*>(hp[i] + k));
    }
#pragma unroll
    for (int u = 0; u < kU; ++u) {
      if (k0 + u * 32 >= d) break;
      if (k0 + u * 32 + 8 * t >= d) {
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
    if (Top) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        Two q = no_squares();
#pragma unroll
        for (int u = 0; u < kU; ++u)
          if (k0 + u * 32 < d) add_squares(q, a[u][i]);
        squares[i] += sum_of(q);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < NT; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sh[i * 8 + 2 * t + (j & 1)][wid * 16 + g + (j >> 1) * 8] = acc[i][j];
  if (Top) {
    float q = 0.f;
    bool plain = true;
#pragma unroll
    for (int i = 0; i < 2; ++i) {                        // four lanes hold a row's
      float one = squares[i];
      one += __shfl_xor_sync(0xffffffffu, one, 1);
      one += __shfl_xor_sync(0xffffffffu, one, 2);
      plain &= plain_square(one);
      q = fmaxf(q, one);
    }
    q = warp_max(q);
    if (!__all_sync(0xffffffffu, plain)) {
      q = 0.f;
      for (int i = 0; i < 16; ++i) q = fmaxf(q, row_square(reinterpret_cast<const uint4*>(w) + (int64_t)min(v0 + i, V - 1) * (d / 8), d / 8));
    }
    if (lane == 0) sizes[wid] = q;
  }
  __syncthreads();
  if (Top && threadIdx.x == 0) {
    float q = sizes[0];
#pragma unroll
    for (int k = 1; k < 8; ++k) q = fmaxf(q, sizes[k]);
    p.sizes[blockIdx.x] = q;
  }
  const int parts = parts_of(V);
  for (int r = wid; r < rows && r < 8 * NT; r += 8) {
    const int y = p.tok ? p.tok[r] : kNoTarget, c0 = blockIdx.x * 128 + lane * 4;
    const float4 q = *reinterpret_cast<const float4*>(&sh[r][lane * 4]);
    float v[4] = {q.x, q.y, q.z, q.w};
    float m = -INFINITY, first = kNothing, second = kNothing;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (c0 + j == y) p.top[r] = v[j];
      if (c0 + j == y || c0 + j >= V) v[j] = kNothing;
      m = fmaxf(m, v[j]);
      if (Top) {
        const float u = __uint_as_float((__float_as_uint(v[j]) & ~63u) | (uint32_t)((lane * 4 + j) & (p.span - 1)));
        second = fmaxf(second, fminf(first, u));
        first = fmaxf(first, u);
      }
    }
    if (Top && p.span == 1) {
      const int wide = (V + 31) / 32 * 32;
      if (c0 < wide)
        *reinterpret_cast<float4*>(reinterpret_cast<float*>(p.notes) + (int64_t)r * wide + c0) = make_float4(v[0], v[1], v[2], v[3]);
    } else if (Top) {
      float most = fmaxf(m, kNothing);
      for (int o = 1; o < p.span / 4; o <<= 1) {         // over the lanes of a group
        const float f2 = __shfl_xor_sync(0xffffffffu, first, o), s2 = __shfl_xor_sync(0xffffffffu, second, o);
        second = fmaxf(fmaxf(second, s2), fminf(first, f2));
        first = fmaxf(first, f2);
        most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, o));
      }
      if (lane % (p.span / 4) == 0 && c0 < V) p.notes[(int64_t)r * p.groups + c0 / p.span] = note_of(most, first, second);
    }
    // The two parts' sums, each over half of the warp.
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    const float off = m <= kNothing ? 0.f : m * p.k;
    float s = 0.f, e = 0.f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float x = fmaf(v[j], p.k, -off), f = exp2_fast(x);
      s += f;
      e = fmaf(f, fmaxf(x, kLeast), e);
    }
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      e += __shfl_xor_sync(0xffffffffu, e, o);
    }
    if (lane % 16 == 0)
      p.part[(int64_t)r * parts + blockIdx.x * 2 + lane / 16] = make_float4(m <= kNothing ? -INFINITY : m, s, e, 0.f);
  }
}

// Sums relative to a maximum: S = sum exp(s - m), T = log2(e) sum exp(s - m) (s - m).
struct Sums {
  float m, s, t;
};

// What a row's sums (without the target's score) give. A row is void when its target is outside the vocabulary or its scores have no
// finite log of their sum of exponentials (an infinity or a NaN among them): NaN in all its results.
struct Row {
  float lp, H, l2;                                 // logp, entropy, log2 of the sum of exponentials
  double base;                                     // log of it
  ASRN_DEV Row(int y, float own, const Sums& q, float k, float inv_tau) : lp(0.f) {
    const float t = q.t * kLn2;
    float from = q.m, off;                         // base = from / tau + off
    if (y < 0) {
      off = logf(q.s);
      H = off - t / q.s;
      l2 = q.m * k + log2f(q.s);
    } else if (q.s == 0.f) {
      lp = H = own * 0.f;
      off = 0.f;
      from = own;
      l2 = own * k;
    } else {
      const float x = (own - q.m) * inv_tau;
      if (x > 0.f) {
        const float f = expf(-x), a = q.s * f;
        lp = -log1pf(a);
        H = -lp - f * (t - fminf(x, -kLeast) * q.s) / (1.f + a);
        off = -lp;
        from = own;
        l2 = own * k - lp * kLog2e;
      } else {
        const float e = expf(x), all = q.s + e;
        off = logf(all);
        lp = x - off;
        H = off - (t + e * fmaxf(x, kLeast)) / all;
        l2 = q.m * k + log2f(all);
      }
    }
    if (y == -1 || !(fabsf(l2) < INFINITY)) lp = H = l2 = NAN;
    H = H < 0.f ? 0.f : H;                         // what the rounding of two equal terms leaves
    base = (double)from * inv_tau + off;
  }
};

// A noted score as a number that orders as it does, its low 7 bits 0; 0: none.
ASRN_DEV uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v);
  return v <= -3e38f ? 0u : (u >> 31 ? ~u : u | 0x80000000u) & ~127u;
}

// A row's notes; Whole: its scores, groups of one column.
template <bool Whole> struct Notes {
  const float* at;
  ASRN_DEV float largest(int g) const { return __ldg(at + (Whole ? g : 2 * g)); }
  ASRN_DEV float2 operator()(int g) const {
    return Whole ? make_float2(__ldg(at + g), kNothing) : __ldg(reinterpret_cast<const float2*>(at) + g);
  }
};
// A row's groups in the order of their largest scores, equal ones by their numbers. Each lane holds the next of its own; up to
// 32 Each groups all of them, in registers.
template <int Each, class Notes> struct Groups {
  Notes notes;
  uint32_t key[Each], best;                      // a group's order, its place among the lane's in the low bits, the first's larger
  ASRN_DEV Groups(const Notes& p, int groups) : notes(p), best(0) {
    const int lane = threadIdx.x & 31;
    float v[Each];
#pragma unroll
    for (int j = 0; j < Each; ++j) v[j] = notes.largest(min(lane + 32 * j, groups - 1));  // no condition: all under way at once
#pragma unroll
    for (int j = 0; j < Each; ++j) {
      const uint32_t o = lane + 32 * j < groups ? order_of(v[j]) : 0u;
      key[j] = o ? o | (uint32_t)(Each - 1 - j) : 0u;
      best = max(best, key[j]);
    }
  }
  ASRN_DEV int next() {                          // the next group, -1: none left
    const int lane = threadIdx.x & 31;
    const uint32_t most = __reduce_max_sync(0xffffffffu, best & ~127u);
    if (most == 0) return -1;
    const int j = Each - 1 - (int)(best & 127u);
    const int mine = (best & ~127u) == most ? lane + 32 * j : 0x7fffffff;
    const int g = (int)__reduce_min_sync(0xffffffffu, (unsigned)mine);
    if (mine == g) {
      best = 0;
#pragma unroll
      for (int i = 0; i < Each; ++i) {
        if (i == j) key[i] = 0;
        best = max(best, key[i]);
      }
    }
    __syncwarp();
    return g;
  }
};
// Any number of groups: read again after each.
template <class Notes> struct Groups<0, Notes> {
  Notes notes;
  int groups, group, last_group;
  uint32_t key, last;
  ASRN_DEV Groups(const Notes& p, int n, uint32_t after = 0xffffffffu, int after_group = -1)
      : notes(p), groups(n), last_group(after_group), last(after) {
    find();
  }
  ASRN_DEV void find() {
    key = 0;
    group = 0x7fffffff;
#pragma unroll 8
    for (int g = threadIdx.x & 31; g < groups; g += 32) {
      const uint32_t o = order_of(notes.largest(g));
      if ((o < last || (o == last && g > last_group)) && o > key) {
        key = o;
        group = g;
      }
    }
  }
  ASRN_DEV int next() {
    const uint32_t most = __reduce_max_sync(0xffffffffu, key);
    if (most == 0) return -1;
    const int g = (int)__reduce_min_sync(0xffffffffu, key == most ? (unsigned)group : 0x7fffffffu);
    last = most;
    last_group = g;
    if (group == g && key == most) find();
    __syncwarp();
    return g;
  }
};

// h . w for four rows of W, products of bf16 exact in fp32, summed in 64 bits.
ASRN_DEV void dots(const uint4* h, const uint4* W, int vecs, const int (&token)[4], double (&out)[4]) {
  const int lane = threadIdx.x & 31;
  double acc[4] = {};
#pragma unroll 2
  for (int c = lane; c < vecs; c += 32) {
    const uint4 a = __ldg(h + c);
    uint4 b[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) b[j] = __ldg(W + (int64_t)token[j] * vecs + c);
    const uint32_t x[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const uint32_t y[4] = {b[j].x, b[j].y, b[j].z, b[j].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        acc[j] += (double)(__uint_as_float(x[i] << 16) * __uint_as_float(y[i] << 16));
        acc[j] += (double)(__uint_as_float(x[i] & 0xffff0000u) * __uint_as_float(y[i] & 0xffff0000u));
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) out[j] = warp_sum_d(acc[j]);
}
// The same for sixteen rows of W by mma.sync, in two chains of fp32 sums: lane 4 j gets the rows j (first) and j + 8 (second)
// that its lanes 4 j to 4 j + 3 name. Loads as in k_stats_few.
struct Pair {
  float a, b;
};
template <int U> ASRN_DEV Pair dots16(const uint4* h, const uint4* W, int vecs, int row_a, int row_b) {
  const int lane = threadIdx.x & 31, t = lane & 3;
  const uint4 *wa = W + (int64_t)row_a * vecs, *wb = W + (int64_t)row_b * vecs;
  float acc[2][4] = {};
  for (int k = t; k - t < vecs; k += 4 * U) {
    uint4 a[U], b[U], x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int at = min(k + 4 * u, vecs - 1);   // what is past the end meets zeros of h
      a[u] = __ldg(wa + at);
      b[u] = __ldg(wb + at);
      x[u] = __ldg(h + at);                      // the first of eight columns; the others are not looked at
      if (k + 4 * u >= vecs) x[u] = make_uint4(0, 0, 0, 0);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      mma16x8(acc[u & 1], a[u].x, b[u].x, a[u].y, b[u].y, x[u].x, x[u].y);
      mma16x8(acc[u & 1], a[u].z, b[u].z, a[u].w, b[u].w, x[u].z, x[u].w);
    }
  }
  return Pair{acc[0][0] + acc[1][0], acc[0][2] + acc[1][2]};
}

// The best so far, lane l the l-th, larger scores first, then smaller numbers; and the largest that was not kept.
template <class T> struct Best {
  T score = -INFINITY, lost = -INFINITY;
  int token = 0x7fffffff;
  ASRN_DEV void put(T s, int t) {                // minus infinity is not put in
    if (s == -INFINITY) return;
    const int lane = threadIdx.x & 31;
    const unsigned behind = __ballot_sync(0xffffffffu, s > score || (s == score && t < token));
    const T out = behind ? __shfl_sync(0xffffffffu, score, 31) : s;
    lost = lost < out ? out : lost;
    if (!behind) return;
    const T up = __shfl_up_sync(0xffffffffu, score, 1);
    const int ut = __shfl_up_sync(0xffffffffu, token, 1);
    const int at = __ffs(behind) - 1;
    if (lane > at) {
      score = up;
      token = ut;
    } else if (lane == at) {
      score = s;
      token = t;
    }
  }
};

constexpr int kRowWarps = 4;
// What a product's sum loses by a step, of the magnitudes: a step adds 16 products to the sum so far, each of which loses up to 2^-25 of
// the largest of them, their sum up to 2^-23: 2.6 2^-22 (one large value and small ones lose 2.05 2^-22 by tcgen05, 1.05 by mma.sync).
// With what both norms are off by (2^-4) 2.8; the rest is room.
constexpr float kOff = 3 * 0x1p-22f;
struct RowArgs {
  int64_t N;
  int V, d, top, parts, span, groups, sizes_n;
  float k, inv_tau;
  const uint4 *hc, *W;
  const int *pos, *tok;                          // null: every position is a row, without a target
  const float4* part;
  const float *notes, *own, *sizes;
  float *lse2, *kept_logp, *kept_ent;            // by rows, for the backward pass; or null
  float *logp, *entropy, *top_logp;              // by positions; logp may be null
  int64_t* top_tokens;
};

// U: steps of K whose loads are under way together: 8 where a slow row's latency is what counts, 2 where rows are many and short, so that
// more share an SM (8 tokens, us, 8 | 2, before rows kept the products' sums: 50304 x 768, 2048 rows 54 | 105, 4096 78 | 108,
// 8192 125 | 150; 5003 x 200, 2048 rows 22 | 30, 8192 59 | 50). Now 45 us at 2048 x 50304 x 768, 22 at 2048 x 5003 x 200.
template <int Each, int U, bool Whole>
__global__ void __launch_bounds__(kRowWarps * 32, U > 2 ? 2 : Each > 32 ? 4 : 6) k_stats_rows(const RowArgs f) {
  const int lane = threadIdx.x & 31, top = f.top, vecs = f.d / 8;
  const int64_t i = (int64_t)blockIdx.x * kRowWarps + (threadIdx.x >> 5);
  wait_previous();
  let_next();
  if (i >= f.N) return;
  const int r = f.pos ? f.pos[i] : (int)i, y = r < 0 ? -1 : f.tok ? f.tok[r] : kNoTarget;
  float lp = 0.f, H = 0.f, l2 = 0.f, own = 0.f;
  double base = 0.0;
  // How large the row and W's are, of which more below. Where latency counts: loads that are under way while the sums are joined.
  constexpr int kEarly = U > 2 ? 16 : 1, kOwn = U > 2 ? 4 : 1;
  const uint4* h = f.hc + (int64_t)(r < 0 ? 0 : r) * vecs;
  float early[kEarly];
  uint4 row[kOwn];
  if (U > 2 && top && r >= 0) {
#pragma unroll
    for (int j = 0; j < kEarly; ++j) early[j] = __ldg(f.sizes + min(lane + 32 * j, f.sizes_n - 1));
#pragma unroll
    for (int j = 0; j < kOwn; ++j) row[j] = __ldg(h + min(lane + 32 * j, vecs - 1));
  }
  if (r >= 0) {                                  // the row's sums: by lanes, then the lanes'
    own = y >= 0 ? f.own[r] : 0.f;
    const float4* part = f.part + (int64_t)r * f.parts;
    Sums q{-INFINITY, 0.f, 0.f};
    constexpr int kAt = 8;                       // loads under way at once
    for (int g0 = lane; g0 - lane < f.parts; g0 += 32 * kAt) {
      float v[kAt];
#pragma unroll
      for (int j = 0; j < kAt; ++j) v[j] = __ldg(&part[min(g0 + 32 * j, f.parts - 1)].x);
#pragma unroll
      for (int j = 0; j < kAt; ++j) q.m = fmaxf(q.m, v[j]);
    }
    q.m = warp_max(q.m);
    const float from = q.m == -INFINITY ? 0.f : q.m;   // no score but NaNs, which the maxima pass over: the sums hold them
    for (int g0 = lane; g0 - lane < f.parts; g0 += 32 * kAt) {
      float4 p[kAt];
#pragma unroll
      for (int j = 0; j < kAt; ++j) p[j] = __ldg(part + min(g0 + 32 * j, f.parts - 1));
#pragma unroll
      for (int j = 0; j < kAt; ++j)
        if (g0 + 32 * j < f.parts) {
          const float x = (p[j].x - from) * f.k, e = exp2_fast(x);
          q.t = fmaf(e, fmaf(fmaxf(x, kLeast), p[j].y, p[j].z), q.t);
          q.s = fmaf(e, p[j].y, q.s);
        }
    }
    q.s = warp_sum(q.s);
    q.t = warp_sum(q.t);
    const Row row(y, own, q, f.k, f.inv_tau);
    lp = row.lp;
    H = row.H;
    l2 = row.l2;
    base = row.base;
    if (lane == 0 && f.lse2) {
      f.lse2[r] = l2;
      f.kept_logp[r] = lp;
      f.kept_ent[r] = H;
    }
  }
  if (lane == 0) {
    if (f.logp) f.logp[i] = lp;
    f.entropy[i] = H;
  }
  if (top == 0) return;
  auto write = [&](float logp, int token) {
    if (lane < top) {
      f.top_logp[i * top + lane] = logp;
      f.top_tokens[i * top + lane] = token;
    }
  };
  if (r < 0 || !(fabsf(l2) < INFINITY)) {
    write(r < 0 ? 0.f : NAN, -1);
    return;
  }
  // What a sum of the products may be off by, for any token: kOff a step of |h| |w|, which is no less than sum |h w|.
  float own_square = 0.f, square = 0.f;
  if (U > 2) {
#pragma unroll
    for (int j = 0; j < kEarly; ++j) square = fmaxf(square, early[j]);
    Two q = no_squares();
#pragma unroll
    for (int j = 0; j < kOwn; ++j)
      if (lane + 32 * j < vecs) add_squares(q, row[j]);
    own_square = sum_of(q);
  }
#pragma unroll 8
  for (int g = lane + (U > 2 ? 32 * kEarly : 0); g < f.sizes_n; g += 32) square = fmaxf(square, __ldg(f.sizes + g));
  if (U > 2) own_square = warp_sum(own_square);
  if (U == 2 || vecs > 32 * kOwn || !plain_square(own_square)) own_square = row_square(h, vecs);
  square = warp_max(square);
  const float slack = square == 0.f ? 0.f : (float)(f.d / 16 + 2) * kOff * sqrtf(own_square) * sqrtf(square);
  if (own_square == 0.f) {                       // a row of zeros: all scores are 0
    write((float)-base, lane);
    return;
  }
  const Notes<Whole> notes{f.notes + (int64_t)r * (Whole ? (f.V + 31) / 32 * 32 : 2 * f.groups)};
  auto column_of = [&](int g, float2 note) { return Whole ? g : g * f.span + (int)(__float_as_uint(note.y) & 63u); };

  // The first groups by lane, `top` and some more, so that the one after them hardly ever counts (where each costs reading the notes
  // again, without these); and the one after them.
  const int limit = Each ? min(32, top + 4) : top;
  float2 pair = make_float2(kNothing, kNothing), held = pair;
  int held_group = 0, have = 0, after = -1;
  {
    Groups<Each, Notes<Whole>> groups(notes, f.groups);
    while (true) {
      after = groups.next();
      if (after < 0 || have == limit) break;
      if (lane == have) held_group = after;
      ++have;
    }
    if (lane < have) held = notes(held_group);
    if (after >= 0) pair = notes(after);
  }
  const int column = column_of(held_group, held);

  // Their largest, and the target: in most rows these are the answer, as the products summed them. For the row's scores may be off by
  // `slack`, notes by their low bits more.
  Best<float> best;
  for (int q = 0; q < have; ++q) best.put(__shfl_sync(0xffffffffu, held.x, q), __shfl_sync(0xffffffffu, column, q));
  if (y >= 0) best.put(own, y);
  auto low = [&]() { return __shfl_sync(0xffffffffu, best.score, top - 1); };
  float off = 0.f;
  auto above = [&](float v) { return v + (fabsf(v) * 0x1p-15f + slack + off); };
  // Those that stand within `width` of their neighbours, down to that far below the last one that counts, by sums in 64 bits; others
  // keep their places among them.
  double score;
  auto settle = [&](float width) {
    const float then = __shfl_down_sync(0xffffffffu, best.score, 1);
    const float least = low() - width;
    unsigned near = __ballot_sync(0xffffffffu, lane < 31 && then > -INFINITY && then >= least && best.score - then <= width);
    score = best.score;
    if (!near) return;
    near |= near << 1;
    const int n = 32 - __clz(near);              // those behind keep their places
    while (near) {                               // four at a time
      int t[4], from[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        from[j] = near ? __ffs(near) - 1 : from[max(j - 1, 0)];
        t[j] = __shfl_sync(0xffffffffu, best.token, from[j]);
        near &= near - 1;
      }
      double sums[4];
      dots(h, f.W, vecs, t, sums);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (lane == from[j]) score = sums[j];
    }
    // Each lane's place among the n, and whose place is its number. As whole numbers that order as the scores do: without branches.
    const long long bits = __double_as_longlong(score + 0.0), key = bits ^ (bits >> 63 & 0x7fffffffffffffffll);
    int place = lane < n ? 0 : lane, whose = lane;
    for (int q = 0; q < n; ++q) {
      const long long other = __shfl_sync(0xffffffffu, key, q);
      const int t = __shfl_sync(0xffffffffu, best.token, q);
      place += (lane < n) & ((other > key) | ((other == key) & (t < best.token)));
    }
    for (int q = 0; q < n; ++q) whose = __shfl_sync(0xffffffffu, place, q) == lane ? q : whose;
    best.token = __shfl_sync(0xffffffffu, best.token, whose);
    score = __shfl_sync(0xffffffffu, score, whose);
  };
  {
    const float lowest = low() - slack;
    const bool open = (lane < top && best.token >= f.V) || (lane < have && held.y > -3e38f && above(held.y) >= lowest) ||
                      (after >= 0 && above(pair.x) >= lowest) || best.lost >= lowest - slack;
    if (!__any_sync(0xffffffffu, open)) {
      settle(2 * slack);
      write((float)(score * f.inv_tau - base), best.token);
      return;
    }
  }

  // Else all that may count, by the products' sums or by sums here (two chains, off by less).
  off = slack;
  float bar = low();                             // no more than the last score that counts
  bar -= fabsf(bar) * 0x1p-15f;
  unsigned hidden = __ballot_sync(0xffffffffu, lane < have && held.y > -3e38f && above(held.y) >= bar);
  // Of two that the notes cannot tell apart the noted column may be either's: left to `expand`.
  const unsigned either = hidden & __ballot_sync(0xffffffffu, held.y >= held.x - fabsf(held.x) * 0x1p-15f);
  if (either) {
    best = Best<float>{};
    for (int q = 0; q < have; ++q) {
      const float v = __shfl_sync(0xffffffffu, held.x, q);
      const int t = __shfl_sync(0xffffffffu, column, q);
      if (!(either >> q & 1u)) best.put(v, t);
    }
    if (y >= 0) best.put(own, y);
  }
  // The columns of a group that may count, but for one and the target's.
  auto expand = [&](int g, int except, auto&& take) {
    const int begin = g * f.span, end = min(f.V, begin + f.span);
    for (int c = begin; c < end; c += 16) {
      const int ra = c + (lane >> 2), rb = ra + 8;
      const Pair about = dots16<U>(h, f.W, vecs, min(ra, end - 1), min(rb, end - 1));
      const float least = fmaxf(low(), bar) - 2 * off;
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const int own = j ? rb : ra;
        const float v = j ? about.b : about.a;
        unsigned set = __ballot_sync(0xffffffffu, !(lane & 3) && own < end && own != y && own != except && v >= least);
        for (; set; set &= set - 1) {
          const int from = __ffs(set) - 1;
          take(__shfl_sync(0xffffffffu, v, from), __shfl_sync(0xffffffffu, own, from));
        }
      }
    }
  };
  auto about_put = [&](float about, int token) { best.put(about, token); };
  for (; hidden; hidden &= hidden - 1) {
    const int q = __ffs(hidden) - 1, g = __shfl_sync(0xffffffffu, held_group, q), c = __shfl_sync(0xffffffffu, column, q);
    if (either >> q & 1u)
      expand(g, -1, about_put);
    else if (above(__shfl_sync(0xffffffffu, held.y, q)) >= low())
      expand(g, c, about_put);
  }
  if (after >= 0 && above(pair.x) >= low()) {
    Groups<0, Notes<Whole>> rest(notes, f.groups, order_of(pair.x), after);
    for (; after >= 0; after = rest.next()) {
      pair = notes(after);
      if (above(pair.x) < low()) break;
      const int c = column_of(after, pair);
      const bool unsure = pair.y > -3e38f && pair.y >= pair.x - fabsf(pair.x) * 0x1p-15f;
      if (!unsure) best.put(pair.x, c);
      if (unsure || (pair.y > -3e38f && above(pair.y) >= low())) expand(after, unsure ? -1 : c, about_put);
    }
  }

  // Scores that stand as near one another as the sums may be off: by sums in 64 bits.
  const float least = low() - 2 * off;
  if (best.lost < least) {                       // the few that were kept hold all that may count
    settle(2 * off);
  } else {
    // Many that are equal or all but that: all of them, four at a time.
    int t[4] = {}, waiting = 0;
    Best<double> exact;
    auto settle_waiting = [&]() {
      double s[4];
      dots(h, f.W, vecs, t, s);
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (j < waiting) exact.put(s[j], t[j]);
      waiting = 0;
    };
    auto exact_put = [&](float, int token) {
#pragma unroll
      for (int j = 0; j < 4; ++j) t[j] = j == waiting ? token : t[j];
      if (++waiting == 4) settle_waiting();
    };
    if (y >= 0) exact_put(0.f, y);
    for (int g0 = 0; g0 < f.groups; g0 += 32) {
      const float largest = notes.largest(min(g0 + lane, f.groups - 1)), lowest = low();   // a shuffle: not behind a condition
      unsigned set = __ballot_sync(0xffffffffu, g0 + lane < f.groups && largest > -3e38f && above(largest) >= lowest);
      for (; set; set &= set - 1) {
        const int g = g0 + __ffs(set) - 1;
        const float most = above(__shfl_sync(0xffffffffu, largest, g - g0));
        // nothing of it comes before the last one that counts so far, not as its equal either
        const double last = __shfl_sync(0xffffffffu, exact.score, top - 1);
        const int number = __shfl_sync(0xffffffffu, exact.token, top - 1);
        if ((double)most < last || ((double)most == last && number < g * f.span)) continue;
        if constexpr (Whole) {
          if (g != y) exact_put(0.f, g);
        } else {
          expand(g, -1, exact_put);
        }
      }
    }
    if (waiting) settle_waiting();
    best.token = exact.token;
    score = exact.score;
  }
  // Scores of minus infinity are in no group: the smallest numbers that are left.
  int l = __popc(__ballot_sync(0xffffffffu, lane < top && best.token < f.V));
  for (int c = 0; l < top && c < f.V; ++c) {
    if (__any_sync(0xffffffffu, lane < l && best.token == c)) continue;
    if (lane == l) best.token = c;
    ++l;
  }
  write((float)(score * f.inv_tau - base), best.token);
}

// dS of one chunk in bf16; the rows that pad the last tile get zeros. With x = log2 p: dS = p (a + b x). 2048 x 50304 x 768: 126 us, tensor
// pipe 74 % active, 1.25 PFLOP/s.
struct Slope {
  static constexpr int kWarps = 8, kOwn = 2, kTable = 0;
  struct Params {
    const int *tok, *row;                  // of the chunk's rows
    const float *lse2, *logp, *ent;
    const float *g, *gh;                   // by position; either may be null
    float k, inv_tau;
    int below;                             // rows from dS to its remainder, 0: none
  };
  const Params& p;
  int V, y, first;
  bool on;
  float off, a, b, own;                    // own: the target's dS
  ASRN_DEV Slope(const Params& pp, int r, int rows, const gemm::Shape& sh, const gemm::Tile&, int)
      : p(pp), V(sh.N), y(-1), first(r & ~31), on(r < rows), off(0.f), a(0.f), b(0.f), own(0.f) {
    if (!on) return;
    y = p.tok[r];
    off = p.lse2[r];
    const int at = p.row[r];
    const float g = p.g && y >= 0 ? p.g[at] * p.inv_tau : 0.f, gh = p.gh ? p.gh[at] * p.inv_tau : 0.f;
    const float H = p.ent[r], lp = p.logp[r];
    a = -g - gh * H;
    b = -gh * kLn2;
    const float slow = lp < kLeast * kLn2 ? 0.f : expf(lp) * (lp + H);    // p (log p + H)
    own = -g * expm1f(lp) - gh * slow;
    if (y == -1) a = NAN;
  }
  template <class O> ASRN_DEV void chunk(float* v, int c, O& out, const CUtensorMap* map_o, const CUtensorMap*) {
    if (c >= V) return;
    const gemm::F2 k2(p.k), off2(-off), a2(a), b2(b);
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      float x0, x1;
      gemm::fma2(gemm::F2(v[i], v[i + 1]), k2, off2).get(x0, x1);
      const gemm::F2 e(exp2_fast(x0), exp2_fast(x1));
      gemm::mul2(e, gemm::fma2(b2, gemm::F2(fmaxf(x0, kLeast), fmaxf(x1, kLeast)), a2)).get(v[i], v[i + 1]);
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

template <int NT, bool Top>
int few(int64_t N, int64_t V, int d, const void* hc, const void* weight, const int* count, const typename Scan<Top>::Params& p,
        cudaStream_t s) {
  return launch_next(k_stats_few<NT, Top>, parts_of(V) / 2, 256, 0, s, (int)N, (int)V, d, reinterpret_cast<const __nv_bfloat16*>(hc),
                     reinterpret_cast<const __nv_bfloat16*>(weight), count, p);
}
template <bool Top>
int scan(int64_t N, int64_t V, int d, const void* hc, const void* weight, const gemm::Shape& sh,
         const typename Scan<Top>::Params& p, cudaStream_t s) {
  if (!few_rows(N, V)) return gemm::launch<false, false, Scan<Top>>(hc, d, weight, d, sh, p, s);
  return N <= 8    ? few<1, Top>(N, V, d, hc, weight, sh.m_dev, p, s)
         : N <= 16 ? few<2, Top>(N, V, d, hc, weight, sh.m_dev, p, s)
                   : few<4, Top>(N, V, d, hc, weight, sh.m_dev, p, s);
}

}  // namespace

}  // namespace asrn

extern "C" {

size_t asrn_head_stats_saved_bytes(int64_t N, int32_t d) {
  if (asrn::check_head(N, 1, d)) return 0;
  return asrn::stats_saved(N, d).total;
}

size_t asrn_head_stats_workspace_bytes(int64_t N, int64_t V, int32_t d, int32_t top, int32_t backward) {
  if (asrn::check_head(N, V, d)) return 0;
  return backward ? asrn::head_backward_ws(N, V, d).total : asrn::stats_ws(N, V, d, top).total;
}

int asrn_head_stats_forward(int64_t N, int64_t V, int32_t d, const void* h, const void* weight, const int64_t* tokens,
                            float tau, int32_t top, float* logp, float* entropy, float* top_logp, int64_t* top_tokens,
                            void* saved, size_t saved_bytes, void* workspace, size_t workspace_bytes, int* status,
                            void* stream) {
  using namespace asrn;
  int st = check_head(N, V, d);
  if (st) return st;
  if (!(tau > 0.f) || tau > 1e30f || top < 0 || top > V) return ASRN_ERR_ARG;
  if (top > kMaxTop) return ASRN_ERR_UNSUPPORTED;
  if (N == 0) return ASRN_OK;
  if (!h || !weight || !entropy || (tokens && !logp) || (top && (!top_logp || !top_tokens)) || (uintptr_t)h % 16 ||
      (uintptr_t)weight % 16)
    return ASRN_ERR_ARG;
  const StatsSaved sv = stats_saved(N, d);
  const StatsWs ws = stats_ws(N, V, d, top);
  if (!saved && tokens) return ASRN_ERR_WORKSPACE;
  if ((saved && (saved_bytes < sv.total || (uintptr_t)saved % 256)) || !workspace || workspace_bytes < ws.total ||
      (uintptr_t)workspace % 256)
    return ASRN_ERR_WORKSPACE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* S = reinterpret_cast<char*>(saved);
  char* W = reinterpret_cast<char*>(workspace);
  // Nothing kept and every position counted: h's rows as they lie.
  if (S && (st = head_gather(N, V, d, h, tokens, reinterpret_cast<int*>(W + ws.counts), S, sv.head, s))) return st;
  auto kept = [&](size_t at) { return S ? S + at : nullptr; };
  const int *tok = reinterpret_cast<int*>(kept(sv.head.tok)), *pos = reinterpret_cast<int*>(kept(sv.head.pos));
  const void* hc = S ? kept(sv.head.hc) : h;
  const int parts = parts_of(V);
  gemm::Shape sh{};
  sh.M = (int)N; sh.N = (int)V; sh.K = d; sh.m_dev = reinterpret_cast<int*>(kept(sv.head.count)); sh.group = 16;
  sh.status = status;
  const float inv_tau = 1.f / tau, k = kLog2e * inv_tau;
  float* own = reinterpret_cast<float*>(W + ws.top);
  float4* part = reinterpret_cast<float4*>(W + ws.part);
  float2* notes = reinterpret_cast<float2*>(W + ws.notes);
  float* sizes = reinterpret_cast<float*>(W + ws.sizes);
  const int span = span_of(V, d, top), groups = (int)notes_of(V, d, top);
  if (top)
    st = scan<true>(N, V, d, hc, weight, sh, {tok, k, own, part, notes, span, groups, sizes}, s);
  else
    st = scan<false>(N, V, d, hc, weight, sh, {tok, k, own, part, notes, span, groups, nullptr}, s);
  if (st) return st;
  const bool own_sizes = few_rows(N, V);
  if (top && !own_sizes &&
      (st = launch_next(k_stats_sizes, size_blocks(V), kSizeWarps * 32, 0, s, V, d / 8, reinterpret_cast<const uint4*>(weight), sizes)))
    return st;
  const RowArgs f{N, (int)V, d, top, parts, span, groups, own_sizes ? parts / 2 : size_blocks(V), k, inv_tau, reinterpret_cast<const uint4*>(hc),
                  reinterpret_cast<const uint4*>(weight), pos, tok, part, reinterpret_cast<const float*>(notes), own, sizes,
                  reinterpret_cast<float*>(kept(sv.head.lse2)), reinterpret_cast<float*>(kept(sv.head.rest)),
                  reinterpret_cast<float*>(kept(sv.ent)), tokens ? logp : nullptr, entropy, top_logp, top_tokens};
  const bool few = N <= (int64_t)gemm::sm_count() * kRowWarps * std::max(4, d / 48);
  auto rows = span == 1       ? V <= 512 ? (few ? k_stats_rows<16, 8, true> : k_stats_rows<16, 2, true>)
                                         : (few ? k_stats_rows<64, 8, true> : k_stats_rows<64, 2, true>)
              : groups <= 512  ? (few ? k_stats_rows<16, 8, false> : k_stats_rows<16, 2, false>)
              : groups <= 1024 ? (few ? k_stats_rows<32, 8, false> : k_stats_rows<32, 2, false>)
                               : (few ? k_stats_rows<0, 8, false> : k_stats_rows<0, 2, false>);
  return launch_next(rows, (N + kRowWarps - 1) / kRowWarps, kRowWarps * 32, 0, s, f);
}

int asrn_head_stats_backward(int64_t N, int64_t V, int32_t d, const void* weight, const void* saved, size_t saved_bytes,
                             float tau, const float* g, const float* g_entropy, void* dh, void* dw, void* workspace,
                             size_t workspace_bytes, int* status, void* stream) {
  using namespace asrn;
  int st = check_head(N, V, d);
  if (st) return st;
  if (!(tau > 0.f) || tau > 1e30f) return ASRN_ERR_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (N == 0) {
    if (dw && cudaMemsetAsync(dw, 0, (size_t)V * d * 2, s) != cudaSuccess) return ASRN_ERR_CUDA;
    return ASRN_OK;
  }
  if (!weight || (uintptr_t)weight % 16 || (uintptr_t)dh % 16 || (uintptr_t)dw % 16) return ASRN_ERR_ARG;
  const StatsSaved sv = stats_saved(N, d);
  const HeadBackwardWs ws = head_backward_ws(N, V, d);
  if (!saved || saved_bytes < sv.total || (uintptr_t)saved % 256 || !workspace || workspace_bytes < ws.total ||
      (uintptr_t)workspace % 256)
    return ASRN_ERR_WORKSPACE;
  const char* S = reinterpret_cast<const char*>(saved);
  auto floats = [&](size_t at, int64_t first) { return reinterpret_cast<const float*>(S + at) + first; };
  auto ints = [&](size_t at, int64_t first) { return reinterpret_cast<const int*>(S + at) + first; };
  return head_backward<Slope>(N, V, d, weight, S, sv.head, ws, reinterpret_cast<char*>(workspace), dh, dw, status, s,
                              [&](int64_t first, int below) {
                                return Slope::Params{ints(sv.head.tok, first), ints(sv.head.row, first),
                                                     floats(sv.head.lse2, first), floats(sv.head.rest, first),
                                                     floats(sv.ent, first), g, g_entropy, kLog2e / tau, 1.f / tau, below};
                              });
}

}  // extern "C"
