// What the operators on the head's scores share: the positions that count, gathered; what is kept for the backward pass and its
// plan; the backward pass over dS, which each operator's epilogue makes from the scores.
#pragma once
#include "common.cuh"
#include "gemm_tc.cuh"

namespace asrn {

constexpr int kGatherRows = 16, kGatherThreads = 256;
constexpr int kCountRows = 1024;
constexpr int64_t kDirectRows = 4096;    // up to here each block counts the targets before it by itself: a launch less
// Rows, and rows x V x d, up to which dS's remainder is multiplied too. At the limit that is 4 2^34 = 69 Gflop more, 41 us at
// the measured burst rate; forward and backward of 512 x 43688 x 768 take 194 us on the device, of 513 rows without it 181.
constexpr int64_t kTwiceRows = 512, kTwiceWork = (int64_t)1 << 34;
constexpr int kNoTarget = -2;             // -1: a target outside the vocabulary
constexpr float kLog2e = 1.4426950408889634f;

inline int64_t pad256(int64_t n) { return (n + 255) / 256 * 256; }

struct HeadSaved {                       // what the forward pass keeps
  size_t count, tok, row, pos, lse2, rest, hc, total;
};

inline HeadSaved head_saved(int64_t N, int64_t d) {
  HeadSaved w{};
  const size_t P = (size_t)pad256(N);
  size_t o = 256;                        // count
  auto take = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes); return at; };
  w.tok = take(P * 4);
  w.row = take(P * 4);
  w.pos = take(P * 4);
  w.lse2 = take(P * 4);
  w.rest = take(P * 4);
  w.hc = take(P * d * 2);
  w.total = o;
  return w;
}

// The backward pass's plan: chunks of rows (256 at least) whose dS stays within two gigabytes. dh's sums run over V: always in shares.
// dW's over the rows: shares, or whole tiles when there are enough of them or when the sum runs over several chunks (their
// sum so far then waits in fp32).
struct HeadBackwardWs {
  int64_t rows, pitch;
  int twice, chunks, shares_h, shares_w;
  size_t ds, dh, dw, total;
};

inline HeadBackwardWs head_backward_ws(int64_t N, int64_t V, int64_t d) {
  HeadBackwardWs w{};
  w.pitch = (V + 63) / 64 * 64;
  const int64_t most = std::max<int64_t>(256, ((int64_t)1 << 31) / (2 * w.pitch) / 256 * 256);
  w.chunks = (int)((pad256(N) + most - 1) / most);
  w.rows = std::max<int64_t>(256, pad256((N + w.chunks - 1) / std::max(1, w.chunks)));
  w.chunks = (int)((pad256(N) + w.rows - 1) / w.rows);
  w.twice = N <= kTwiceRows && N * V * d <= kTwiceWork && w.chunks == 1;
  w.shares_h = gemm::groups_for(w.rows, d, V * (1 + w.twice));
  w.shares_w = w.chunks > 1 ? 0 : gemm::shares_for(V, d, w.rows * (1 + w.twice));
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes); return at; };
  w.ds = take((size_t)(1 + w.twice) * w.rows * w.pitch * 2);
  w.dh = take(gemm::slot_bytes(w.rows, d, w.shares_h));
  w.dw = take(w.shares_w ? gemm::slot_bytes(V, d, w.shares_w) : w.chunks > 1 ? (size_t)V * d * 4 : 0);
  w.total = o;
  return w;
}

static __global__ void __launch_bounds__(kCountRows) k_head_count(int64_t N, const int64_t* __restrict__ tokens,
                                                           int* __restrict__ counts) {
  const int64_t i = (int64_t)blockIdx.x * kCountRows + threadIdx.x;
  const int n = __syncthreads_count(i < N && tokens[i] >= 0);
  if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// Block b takes positions [16 b, 16 b + 16) (64 at a time left SMs idle: 18 us against 8.5 at 4096 x 768; 11.6 us at 16384
// x 768, 50 MB, 4.3 TB/s): the targets before them (from the tokens, or from the counts of the
// blocks of 1024), then its own, in order. The last block zeroes the rows up to the next multiple of 64: dW's sums run over
// whole K blocks (what the rows after those hold reaches nothing that is kept). tokens null: every position counts, with
// kNoTarget for its token.
static __global__ void __launch_bounds__(kGatherThreads)
k_head_gather(int64_t N, int64_t V, int d, const __nv_bfloat16* __restrict__ h, const int64_t* __restrict__ tokens,
              const int* __restrict__ counts, int* count, int* __restrict__ tok, int* __restrict__ row,
              int* __restrict__ pos, __nv_bfloat16* __restrict__ hc) {
  __shared__ int warps[kGatherThreads / 32];
  __shared__ int at[kGatherRows];
  const int tid = threadIdx.x, lane = tid & 31, wid = tid >> 5;
  const int64_t i0 = (int64_t)blockIdx.x * kGatherRows;
  let_next();                                            // launched after all that was before it: nothing else is waited for
  int before = tokens || tid ? 0 : (int)i0;
  const int64_t from = !tokens ? i0 : counts ? i0 / kCountRows * kCountRows : 0;
  if (counts)
    for (int64_t c = tid; c < i0 / kCountRows; c += kGatherThreads) before += counts[c];
#pragma unroll 8
  for (int64_t i = from + tid; i < i0; i += kGatherThreads) before += __ldg(tokens + i) >= 0;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
  if (lane == 0) warps[wid] = before;
  __syncthreads();
  before = 0;
  for (int w = 0; w < kGatherThreads / 32; ++w) before += warps[w];
  __syncthreads();
  const int64_t i = i0 + tid;
  const bool mine = tid < kGatherRows && i < N;
  const int64_t y = !mine ? -1 : tokens ? tokens[i] : 0;
  const unsigned set = __ballot_sync(0xffffffffu, y >= 0);          // the rows are the first warp's
  const int r = before + __popc(set & ((1u << lane) - 1u));
  if (tid < kGatherRows) at[tid] = y >= 0 ? r : -1;
  if (tid == 0) warps[0] = __popc(set);
  if (mine) pos[i] = y >= 0 ? r : -1;
  if (y >= 0) {
    tok[r] = !tokens ? kNoTarget : y < V ? (int)y : -1;    // outside the vocabulary: NaN from here on
    row[r] = (int)i;
  }
  __syncthreads();
  const unsigned nv = d / 8;
#pragma unroll 8
  for (unsigned x = tid; x < kGatherRows * nv; x += kGatherThreads) {
    const unsigned k = x / nv, c = x - k * nv;
    if (at[k] >= 0)
      reinterpret_cast<uint4*>(hc + (int64_t)at[k] * d)[c] = __ldg(reinterpret_cast<const uint4*>(h + (i0 + k) * d) + c);
  }
  if (i0 + kGatherRows >= N) {
    const int total = before + warps[0];
    if (tid == 0) *count = total;
    const int64_t end = ((int64_t)total + 63) / 64 * 64;
    uint4* dst = reinterpret_cast<uint4*>(hc);
    for (int64_t c = (int64_t)total * nv + tid; c < end * nv; c += kGatherThreads) dst[c] = make_uint4(0, 0, 0, 0);
  }
}

inline int check_head(int64_t N, int64_t V, int32_t d) {
  if (N < 0 || V < 1 || d < 1) return ASRN_ERR_ARG;
  if (d % 8 || d > 16384 || V > (1 << 24) || N > (1 << 24)) return ASRN_ERR_UNSUPPORTED;
  if (((N + 127) / 128) * ((V + 255) / 256) >= (1 << 30)) return ASRN_ERR_UNSUPPORTED;      // tiles are counted in 32 bits
  return ASRN_OK;
}

// The positions that count, in order, to `saved`. counts: room for the counts of blocks of kCountRows tokens.
inline int head_gather(int64_t N, int64_t V, int d, const void* h, const int64_t* tokens, int* counts, char* S,
                       const HeadSaved& sv, cudaStream_t s) {
  if (!tokens || N <= kDirectRows)
    counts = nullptr;
  else
    k_head_count<<<(unsigned)((N + kCountRows - 1) / kCountRows), kCountRows, 0, s>>>(N, tokens, counts);
  k_head_gather<<<(unsigned)((N + kGatherRows - 1) / kGatherRows), kGatherThreads, 0, s>>>(
      N, V, d, reinterpret_cast<const __nv_bfloat16*>(h), tokens, counts, reinterpret_cast<int*>(S + sv.count),
      reinterpret_cast<int*>(S + sv.tok), reinterpret_cast<int*>(S + sv.row), reinterpret_cast<int*>(S + sv.pos),
      reinterpret_cast<__nv_bfloat16*>(S + sv.hc));
  return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA;
}

// dh and dW (either may be null) by chunks of rows: dS from the scores by the epilogue Slope, whose parameters for the rows from
// `first` on `params(first, rows to the remainder or 0)` makes; then the two products.
template <class Slope, class Make>
int head_backward(int64_t N, int64_t V, int32_t d, const void* weight, const char* S, const HeadSaved& sv,
                  const HeadBackwardWs& ws, char* W, void* dh, void* dw, int* status, cudaStream_t s, const Make& params) {
  int st = ASRN_OK;
  const int* count = reinterpret_cast<const int*>(S + sv.count);
  __nv_bfloat16* ds = reinterpret_cast<__nv_bfloat16*>(W + ws.ds);
  float* dh_slots = reinterpret_cast<float*>(W + ws.dh);
  float* dw_sum = reinterpret_cast<float*>(W + ws.dw);
  for (int c = 0; c < ws.chunks; ++c) {
    const int64_t first = c * ws.rows;
    const int rows = (int)ws.rows;
    const __nv_bfloat16* hc = reinterpret_cast<const __nv_bfloat16*>(S + sv.hc) + first * d;
    const int64_t left = std::min<int64_t>(rows, pad256(N) - first);   // rows of hc from here on
    gemm::Shape sh{};
    sh.M = (int)left; sh.N = (int)V; sh.K = d; sh.m_dev = count; sh.m_off = (int)first; sh.group = 16;
    sh.status = status;
    const int* row = reinterpret_cast<const int*>(S + sv.row) + first;
    const typename Slope::Params p = params(first, ws.twice ? rows : 0);
    if ((st = gemm::launch<false, false, Slope>(hc, d, weight, d, sh, p, s, {ds, (1 + ws.twice) * rows, ws.pitch, ws.pitch})))
      return st;
    if (dh) {
      gemm::Shape a{};
      a.M = rows; a.N = d; a.K = (int)V; a.m_dev = count; a.m_off = (int)first; a.shares = ws.shares_h; a.status = status;
      a.second_pass = ws.twice; a.a_step = rows;
      const gemm::StorePiece::Params q{dh_slots, gemm::kBM * gemm::pair_for(rows)};
      if ((st = gemm::launch<false, true, gemm::StorePiece>(ds, ws.pitch, weight, d, a, q, s)) ||
          (st = gemm::join(a, dh_slots, dh, row, reinterpret_cast<const int*>(S + sv.pos), c ? 0 : N, s)))
        return st;
    }
    if (dw) {
      gemm::Shape a{};
      a.M = (int)V; a.N = d; a.K = (int)left; a.k_dev = count; a.k_off = (int)first; a.shares = ws.shares_w; a.group = 16;
      a.status = status; a.second_pass = ws.twice; a.a_step = rows;
      if (ws.shares_w) {
        const gemm::StorePiece::Params q{dw_sum, gemm::kBM * gemm::pair_for(V)};
        if ((st = gemm::launch<true, true, gemm::StorePiece>(ds, ws.pitch, hc, d, a, q, s)) ||
            (st = gemm::join(a, dw_sum, dw, nullptr, nullptr, 0, s)))
          return st;
      } else {
        const gemm::StoreBf16::Params q{nullptr, c ? dw_sum : nullptr, c + 1 < ws.chunks ? dw_sum : nullptr};
        if ((st = gemm::launch<true, true, gemm::StoreBf16>(ds, ws.pitch, hc, d, a, q, s, {dw, V, d, d}))) return st;
      }
    }
  }
  return ASRN_OK;
}

}  // namespace asrn
