// The MLP of a local block with its activations kept in 8 bits for the backward pass:
//   a = x W1^T + b1,  y = gelu(a) W2^T + b2;  kept: Q(x) and Q(a)
//   dA = (dY W2) gelu'(a'),  dX = dA W1,  dW1 = dA^T x',  dW2 = dY^T gelu(a'),  db1 = sum dA,  db2 = sum dY
// with x' = Q(x), a' = Q(a) read back. Q keeps blocks of 32 values along a row as int8 codes and one power-of-two scale
// 2^e, the least with max|v| <= 127 2^e (e >= -120): code = rint(v 2^-e), so the product back is exact in bf16, and 32
// columns are what one thread holds of a row in a product's epilogue: no exchange is needed to find the maximum.
// (d + ff) 33/32 bytes a row instead of bf16 x, a and gelu(a) and their fp32 neighbours.
//
// Bound by the tensor cores: 12 N d ff operations in six products; the elementwise work is their epilogue. gelu(a) and
// dA are rounded to bf16 once each, as operands; dY W2 stays in fp32 until it is multiplied by gelu'.
//   k_pack8        x -> Q(x)
//   k_gemm<Up>     a, Q(a), gelu(a)
//   k_gemm         y
//   k_colsum_rows  db2's partial sums
//   k_gemm<Down>   dY W2 -> dA, gelu(a'), db1's partial sums by 32 rows
//   k_unpack8      x'
//   k_gemm x 3     dX, dW1, dW2 (parts of N where there are few tiles)
//   k_colsum       db1, db2
#include "common.cuh"
#include "gemm_tc.cuh"

namespace asrn {

int sum_parts(int64_t n, int parts, const float* part, __nv_bfloat16* out, cudaStream_t s);

namespace {

constexpr int kBad = -128;                     // exponent byte of a block that holds an infinity or a NaN

// The exponent of a block whose largest magnitude is m.
ASRN_DEV int block_exp(float m) {
  const uint32_t u = __float_as_uint(m);
  if (u >= 0x7f800000u) return kBad;
  const int e = (int)(u >> 23) - 127 - 6 + ((u & 0x7fffffu) > 0x7e0000u);      // mantissa above 127 / 64
  return max(e, -120);
}
ASRN_DEV float pow2(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }   // -126 <= e <= 127
ASRN_DEV float scale_of(int e) { return e == kBad ? NAN : pow2(e); }
ASRN_DEV float inv_scale_of(int e) { return e == kBad ? 0.f : pow2(-e); }

ASRN_DEV uint32_t codes4(const float* v, float inv) {
  uint32_t r = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) r |= ((uint32_t)__float2int_rn(v[i] * inv) & 255u) << (8 * i);
  return r;
}
ASRN_DEV float value_of(uint32_t w, int i, float scale) { return (float)(int8_t)(w >> (8 * i)) * scale; }

ASRN_DEV float abs_max32(const float* v) {     // a NaN counts as the largest
  float m = 0.f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < 32; ++i) {
    m = fmaxf(m, fabsf(v[i]));
    bad |= v[i] != v[i];
  }
  return bad ? NAN : m;
}

// Phi(a) and a phi(a) of the standard normal: gelu = a Phi, gelu' = Phi + a phi.
struct Normal {
  float cdf, apdf;
};
ASRN_DEV Normal normal_of(float a) {
  return Normal{0.5f * (1.f + erff(a * 0.70710678118654752f)), a * expf(-0.5f * a * a) * 0.39894228040143268f};
}

// One thread per block of 32 of a row of bf16.
__global__ void __launch_bounds__(256) k_pack8(int64_t blocks, int f, int per_row, const __nv_bfloat16* __restrict__ x,
                                               uint8_t* __restrict__ codes, int8_t* __restrict__ exps) {
  for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < blocks; b += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = b / per_row;
    const int c = (int)(b % per_row) * 32;
    const int64_t at = row * f + c;
    float v[32];
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      uint4 q = make_uint4(0, 0, 0, 0);
      if (c + i < f) q = *reinterpret_cast<const uint4*>(x + at + i);
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[i + 2 * j] = __uint_as_float(w[j] << 16);
        v[i + 2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
    }
    const int e = block_exp(abs_max32(v));
    const float inv = inv_scale_of(e);
    exps[b] = (int8_t)e;
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      if (c + i < f)
        *reinterpret_cast<uint2*>(codes + at + i) = make_uint2(codes4(v + i, inv), codes4(v + i + 4, inv));
  }
}

// One thread per 8 values.
__global__ void __launch_bounds__(256) k_unpack8(int64_t eighths, int f, const uint8_t* __restrict__ codes,
                                                 const int8_t* __restrict__ exps, __nv_bfloat16* __restrict__ x) {
  const int per = f / 8, per_row = (f + 31) / 32;
  for (int64_t b = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; b < eighths; b += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = b / per;
    const int c = (int)(b % per) * 8;
    const uint2 w = *reinterpret_cast<const uint2*>(codes + row * f + c);
    const float scale = scale_of(exps[row * per_row + c / 32]);
    float v[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = value_of(w.x, i, scale);
      v[4 + i] = value_of(w.y, i, scale);
    }
    *reinterpret_cast<uint4*>(x + row * f + c) = gemm::pack8(v);
  }
}

// a = sum + b1 -> Q(a) (unless codes is null) and gelu(a) in bf16.
struct Up {
  struct Params {
    const __nv_bfloat16* bias;
    __nv_bfloat16* g;
    uint8_t* codes;
    int8_t* exps;
  };
  const Params& p;
  int64_t at, eat;
  int N;
  bool on;
  ASRN_DEV Up(const Params& pp, int row, int rows, int, const gemm::Shape& s, const gemm::Tile&, int)
      : p(pp), at((int64_t)row * s.N), eat((int64_t)row * ((s.N + 31) / 32)), N(s.N), on(row < rows) {}
  ASRN_DEV void chunk(float* v, int c) {
    if (!on || c >= N) return;
#pragma unroll
    for (int i = 0; i < 32; ++i)
      v[i] = c + i < N ? v[i] + __bfloat162float(p.bias[c + i]) : 0.f;
    if (p.codes) {
      const int e = block_exp(abs_max32(v));
      const float inv = inv_scale_of(e);
      p.exps[eat + c / 32] = (int8_t)e;
#pragma unroll
      for (int i = 0; i < 32; i += 8)
        if (c + i < N)
          *reinterpret_cast<uint2*>(p.codes + at + c + i) = make_uint2(codes4(v + i, inv), codes4(v + i + 4, inv));
    }
#pragma unroll
    for (int i = 0; i < 32; ++i) v[i] *= normal_of(v[i]).cdf;
#pragma unroll
    for (int i = 0; i < 32; i += 8)
      if (c + i < N) *reinterpret_cast<uint4*>(p.g + at + c + i) = gemm::pack8(v + i);
  }
  ASRN_DEV void finish() {}
};

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

// dG = sum -> dA = dG gelu'(a') and gelu(a') in bf16, and dA's column sums by 32 rows.
struct Down {
  struct Params {
    const uint8_t* codes;
    const int8_t* exps;
    __nv_bfloat16 *da, *g;
    float* sums;                               // [ceil(rows / 32)][N]
  };
  const Params& p;
  int64_t at, eat;
  int N, row, rows;
  bool on;
  ASRN_DEV Down(const Params& pp, int r, int m, int, const gemm::Shape& s, const gemm::Tile&, int)
      : p(pp), at((int64_t)r * s.N), eat((int64_t)r * ((s.N + 31) / 32)), N(s.N), row(r), rows(m), on(r < m) {}
  ASRN_DEV void chunk(float* v, int c) {
    if (c >= N) return;                        // the same for the whole warp
    const float scale = on ? scale_of(p.exps[eat + c / 32]) : 0.f;
#pragma unroll
    for (int i = 0; i < 32; i += 8) {
      const bool in = on && c + i < N;
      uint2 w = make_uint2(0, 0);
      if (in) w = *reinterpret_cast<const uint2*>(p.codes + at + c + i);
      float g[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float a = value_of(j < 4 ? w.x : w.y, j & 3, scale);
        const Normal n = normal_of(a);
        g[j] = a * n.cdf;
        v[i + j] = in ? v[i + j] * (n.cdf + n.apdf) : 0.f;
      }
      if (in) {
        *reinterpret_cast<uint4*>(p.g + at + c + i) = gemm::pack8(g);
        *reinterpret_cast<uint4*>(p.da + at + c + i) = gemm::pack8(v + i);
      }
    }
    const int lane = threadIdx.x & 31;
    const float s = column_sum(v, lane);
    const int first = row - lane;              // the warp's rows start on a multiple of 32
    if (p.sums && first < rows && c + lane < N) p.sums[(int64_t)(first / 32) * N + c + lane] = s;
  }
  ASRN_DEV void finish() {}
};

// Sums of bf16 columns over 64 rows: block (64 rows, 256 columns), thread = column.
constexpr int kColRows = 64;
__global__ void __launch_bounds__(256) k_colsum_rows(int64_t rows, int n, const __nv_bfloat16* __restrict__ x,
                                                     float* __restrict__ sums) {
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= n) return;
  const int64_t r0 = (int64_t)blockIdx.x * kColRows;
  const int64_t r1 = r0 + kColRows < rows ? r0 + kColRows : rows;
  float s = 0.f;
#pragma unroll 8
  for (int64_t r = r0; r < r1; ++r) s += __bfloat162float(x[r * n + c]);
  sums[(int64_t)blockIdx.x * n + c] = s;
}

// out[c] = bf16(sum of parts[..][c]) in order: block = 32 columns x 32 warps.
__global__ void __launch_bounds__(1024) k_colsum(int64_t parts, int n, const float* __restrict__ sums,
                                                 __nv_bfloat16* __restrict__ out) {
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float s = 0.f;
  if (c < n)
#pragma unroll 4
    for (int64_t k = wid; k < parts; k += 32) s += sums[k * n + c];
  sh[wid][lane] = s;
  __syncthreads();
  if (wid) return;
  s = 0.f;
  for (int w = 0; w < 32; ++w) s += sh[w][lane];
  if (c < n) out[c] = __float2bfloat16_rn(s);
}

struct Mlp8Saved {
  size_t xc, xe, ac, ae, total;
};

Mlp8Saved mlp8_saved(int64_t N, int64_t d, int64_t ff) {
  Mlp8Saved w{};
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes); return at; };
  w.xc = take((size_t)N * d);
  w.xe = take((size_t)N * ((d + 31) / 32));
  w.ac = take((size_t)N * ff);
  w.ae = take((size_t)N * ((ff + 31) / 32));
  w.total = o;
  return w;
}

struct Mlp8Ws {
  int split1, split2;
  size_t da, g, x, sum1, sum2, part, total;
};

Mlp8Ws mlp8_ws(int64_t N, int64_t d, int64_t ff, int64_t dout, bool backward) {
  Mlp8Ws w{};
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes); return at; };
  w.g = take((size_t)N * ff * 2);
  if (backward) {
    w.split1 = gemm::splits_for(ff, d, N);
    w.split2 = gemm::splits_for(dout, ff, N);
    w.da = take((size_t)N * ff * 2);
    w.x = take((size_t)N * d * 2);
    w.sum1 = take((size_t)((N + 31) / 32) * ff * 4);
    w.sum2 = take((size_t)((N + kColRows - 1) / kColRows) * dout * 4);
    w.part = take((size_t)std::max(w.split1 * d, w.split2 * dout) * ff * 4);
  }
  w.total = o;
  return w;
}

int check_mlp8(int64_t N, int32_t d, int32_t ff, int32_t dout) {
  if (N < 0 || d < 1 || ff < 1 || dout < 1) return ASRN_ERR_ARG;
  if (d % 8 || ff % 8 || dout % 8 || d > 65536 || ff > 65536 || dout > 65536 || N > (1 << 26)) return ASRN_ERR_UNSUPPORTED;
  if ((int64_t)((N + 127) / 128) * ((std::max(ff, std::max(d, dout)) + 255) / 256) >= ((int64_t)1 << 30))
    return ASRN_ERR_UNSUPPORTED;
  return ASRN_OK;
}

int launched() { return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA; }

unsigned grid_for(int64_t threads) { return (unsigned)std::min<int64_t>((threads + 255) / 256, 148 * 16); }

int pack8(int64_t rows, int f, const void* x, void* codes, void* exps, cudaStream_t s) {
  const int64_t blocks = rows * ((f + 31) / 32);
  k_pack8<<<grid_for(blocks), 256, 0, s>>>(blocks, f, (f + 31) / 32, reinterpret_cast<const __nv_bfloat16*>(x),
                                           reinterpret_cast<uint8_t*>(codes), reinterpret_cast<int8_t*>(exps));
  return launched();
}

int unpack8(int64_t rows, int f, const void* codes, const void* exps, void* x, cudaStream_t s) {
  k_unpack8<<<grid_for(rows * (f / 8)), 256, 0, s>>>(rows * (f / 8), f, reinterpret_cast<const uint8_t*>(codes),
                                                     reinterpret_cast<const int8_t*>(exps),
                                                     reinterpret_cast<__nv_bfloat16*>(x));
  return launched();
}

// out (M, n) = A^T B over the rows they share, both as they lie in memory: parts of the rows when there are few tiles.
int weight_grad(int64_t rows, int M, int n, const void* A, const void* B, int splits, float* part, void* out,
                int* status, cudaStream_t s) {
  gemm::Shape a{};
  a.M = M; a.N = n; a.K = (int)rows; a.splits = splits; a.group = 16; a.status = status;
  __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(out);
  if (splits == 1) return gemm::launch<true, true, gemm::StoreBf16>(A, M, B, n, a, {o, nullptr}, s);
  const int st = gemm::launch<true, true, gemm::StoreF32>(A, M, B, n, a, {part, 0}, s);
  return st ? st : sum_parts((int64_t)M * n, splits, part, o, s);
}

}  // namespace
}  // namespace asrn

extern "C" {

int asrn_pack8(int64_t rows, int32_t f, const void* x, void* codes, void* exps, void* stream) {
  using namespace asrn;
  if (rows < 0 || f < 1) return ASRN_ERR_ARG;
  if (f % 8) return ASRN_ERR_UNSUPPORTED;
  if (rows == 0) return ASRN_OK;
  if (!x || !codes || !exps || (uintptr_t)x % 16 || (uintptr_t)codes % 8) return ASRN_ERR_ARG;
  return pack8(rows, f, x, codes, exps, reinterpret_cast<cudaStream_t>(stream));
}

int asrn_unpack8(int64_t rows, int32_t f, const void* codes, const void* exps, void* x, void* stream) {
  using namespace asrn;
  if (rows < 0 || f < 1) return ASRN_ERR_ARG;
  if (f % 8) return ASRN_ERR_UNSUPPORTED;
  if (rows == 0) return ASRN_OK;
  if (!x || !codes || !exps || (uintptr_t)x % 16 || (uintptr_t)codes % 8) return ASRN_ERR_ARG;
  return unpack8(rows, f, codes, exps, x, reinterpret_cast<cudaStream_t>(stream));
}

size_t asrn_mlp8_saved_bytes(int64_t N, int32_t d, int32_t ff) {
  if (asrn::check_mlp8(N, d, ff, 8)) return 0;
  return asrn::mlp8_saved(N, d, ff).total;
}

size_t asrn_mlp8_workspace_bytes(int64_t N, int32_t d, int32_t ff, int32_t dout, int32_t backward) {
  if (asrn::check_mlp8(N, d, ff, dout)) return 0;
  return asrn::mlp8_ws(N, d, ff, dout, backward != 0).total;
}

int asrn_mlp8_forward(int64_t N, int32_t d, int32_t ff, int32_t dout, const void* x, const void* w1, const void* b1,
                      const void* w2, const void* b2, void* y, void* saved, size_t saved_bytes, void* workspace,
                      size_t workspace_bytes, int* status, void* stream) {
  using namespace asrn;
  int st = check_mlp8(N, d, ff, dout);
  if (st) return st;
  if (N == 0) return ASRN_OK;
  if (!x || !w1 || !b1 || !w2 || !b2 || !y || (uintptr_t)x % 16 || (uintptr_t)w1 % 16 || (uintptr_t)w2 % 16 ||
      (uintptr_t)y % 16)
    return ASRN_ERR_ARG;
  const Mlp8Saved sv = mlp8_saved(N, d, ff);
  const Mlp8Ws ws = mlp8_ws(N, d, ff, dout, false);
  if ((saved && (saved_bytes < sv.total || (uintptr_t)saved % 256)) || !workspace || workspace_bytes < ws.total ||
      (uintptr_t)workspace % 256)
    return ASRN_ERR_WORKSPACE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* S = reinterpret_cast<char*>(saved);
  __nv_bfloat16* g = reinterpret_cast<__nv_bfloat16*>(reinterpret_cast<char*>(workspace) + ws.g);
  if (S && (st = pack8(N, d, x, S + sv.xc, S + sv.xe, s))) return st;
  gemm::Shape a{};
  a.M = (int)N; a.N = ff; a.K = d; a.splits = 1; a.group = 16; a.status = status;
  Up::Params p{reinterpret_cast<const __nv_bfloat16*>(b1), g, S ? reinterpret_cast<uint8_t*>(S + sv.ac) : nullptr,
               S ? reinterpret_cast<int8_t*>(S + sv.ae) : nullptr};
  if ((st = gemm::launch<false, false, Up>(x, d, w1, d, a, p, s))) return st;
  a.N = dout; a.K = ff;
  return gemm::launch<false, false, gemm::StoreBf16>(
      g, ff, w2, ff, a, {reinterpret_cast<__nv_bfloat16*>(y), reinterpret_cast<const __nv_bfloat16*>(b2)}, s);
}

int asrn_mlp8_backward(int64_t N, int32_t d, int32_t ff, int32_t dout, const void* dy, const void* w1, const void* w2,
                       const void* saved, size_t saved_bytes, void* dx, void* dw1, void* db1, void* dw2, void* db2,
                       void* workspace, size_t workspace_bytes, int* status, void* stream) {
  using namespace asrn;
  int st = check_mlp8(N, d, ff, dout);
  if (st) return st;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (N == 0) {
    const struct { void* p; size_t n; } zero[] = {{dw1, (size_t)ff * d}, {db1, (size_t)ff}, {dw2, (size_t)dout * ff},
                                                  {db2, (size_t)dout}};
    for (const auto& z : zero)
      if (z.p && cudaMemsetAsync(z.p, 0, z.n * 2, s) != cudaSuccess) return ASRN_ERR_CUDA;
    return ASRN_OK;
  }
  if (!dy || !w1 || !w2 || (uintptr_t)dy % 16 || (uintptr_t)w1 % 16 || (uintptr_t)w2 % 16 || (uintptr_t)dx % 16 ||
      (uintptr_t)dw1 % 16 || (uintptr_t)dw2 % 16)
    return ASRN_ERR_ARG;
  const Mlp8Saved sv = mlp8_saved(N, d, ff);
  const Mlp8Ws ws = mlp8_ws(N, d, ff, dout, true);
  if (!saved || saved_bytes < sv.total || (uintptr_t)saved % 256 || !workspace || workspace_bytes < ws.total ||
      (uintptr_t)workspace % 256)
    return ASRN_ERR_WORKSPACE;
  const char* S = reinterpret_cast<const char*>(saved);
  char* W = reinterpret_cast<char*>(workspace);
  __nv_bfloat16* da = reinterpret_cast<__nv_bfloat16*>(W + ws.da);
  __nv_bfloat16* g = reinterpret_cast<__nv_bfloat16*>(W + ws.g);
  float* part = reinterpret_cast<float*>(W + ws.part);
  float* sum1 = reinterpret_cast<float*>(W + ws.sum1);
  float* sum2 = reinterpret_cast<float*>(W + ws.sum2);
  const int64_t groups = (N + 31) / 32, blocks = (N + kColRows - 1) / kColRows;
  gemm::Shape a{};
  a.M = (int)N; a.splits = 1; a.group = 16; a.status = status;
  if (dx || dw1 || db1 || dw2) {
    a.N = ff; a.K = dout;
    Down::Params p{reinterpret_cast<const uint8_t*>(S + sv.ac), reinterpret_cast<const int8_t*>(S + sv.ae), da, g,
                   db1 ? sum1 : nullptr};
    if ((st = gemm::launch<false, true, Down>(dy, dout, w2, ff, a, p, s))) return st;
  }
  if (dx) {
    a.N = d; a.K = ff;
    if ((st = gemm::launch<false, true, gemm::StoreBf16>(da, ff, w1, d, a,
                                                               {reinterpret_cast<__nv_bfloat16*>(dx), nullptr}, s)))
      return st;
  }
  if (dw1) {
    if ((st = unpack8(N, d, S + sv.xc, S + sv.xe, W + ws.x, s))) return st;
    if ((st = weight_grad(N, ff, d, da, W + ws.x, ws.split1, part, dw1, status, s))) return st;
  }
  if (dw2 && (st = weight_grad(N, dout, ff, dy, g, ws.split2, part, dw2, status, s))) return st;
  if (db1) {
    k_colsum<<<(unsigned)((ff + 31) / 32), 1024, 0, s>>>(groups, ff, sum1, reinterpret_cast<__nv_bfloat16*>(db1));
    if ((st = launched())) return st;
  }
  if (db2) {
    k_colsum_rows<<<dim3((unsigned)blocks, (unsigned)((dout + 255) / 256)), 256, 0, s>>>(
        N, dout, reinterpret_cast<const __nv_bfloat16*>(dy), sum2);
    k_colsum<<<(unsigned)((dout + 31) / 32), 1024, 0, s>>>(blocks, dout, sum2, reinterpret_cast<__nv_bfloat16*>(db2));
    if ((st = launched())) return st;
  }
  return ASRN_OK;
}

}  // extern "C"
