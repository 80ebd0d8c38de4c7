// The MLP of a local block with its activations kept in 8 bits for the backward pass:
//   a = x W1^T + b1,  y = gelu(a) W2^T + b2;  kept: Q(x) and Q(a)
//   dA = (dY W2) gelu'(a'),  dX = dA W1,  dW1 = dA^T x',  dW2 = dY^T gelu(a'),  db1 = sum dA,  db2 = sum dY
// with x' = Q(x), a' = Q(a) read back. Q keeps blocks of 32 values along a row as int8 codes and one power-of-two scale
// 2^e, the least with max|v| <= 127 2^e (e >= -120): code = rint(v 2^-e), so the product back is exact in bf16, and 32
// columns are what one thread holds of a row in a product's epilogue: no exchange is needed to find the maximum.
// (d + ff) 33/32 bytes a row instead of bf16 x, a and gelu(a) and their fp32 neighbours.
//
// Bound by the tensor cores: 12 N d ff operations in six products; the elementwise work is their epilogue. gelu(a) and
// dA are rounded to bf16 once each, as operands (up to kTwiceRows rows the products take what the rounding took, too); dY
// W2 stays in fp32 until it is multiplied by gelu', which comes from a table in fp16 (Down). 512 x 768 x 1536 takes 107 us
// on the device, forward and backward, 513 rows without the remainders 76.
//   k_pack8        x -> Q(x)
//   k_gemm<Up>     a, Q(a), gelu(a)
//   k_gemm         y
//   k_prepare      x', and db2's partial sums by 64 rows
//   k_gemm<Down>   dY W2 -> dA, gelu(a'), db1's partial sums by 32 rows
//   k_gemm x 3     dX, dW1, dW2 (the last two in shares of N: few tiles)
//   k_colsum       db1, db2
#include <cuda_fp16.h>
#include "common.cuh"
#include "gemm_tc.cuh"
#include "products.cuh"

namespace asrn {

namespace {

constexpr int64_t kTwiceRows = 512;
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

// Codes of four values: v inv + 1.5 2^23 holds the nearest integer, ties to even, in its low bits.
ASRN_DEV uint32_t codes4(const float* v, float inv) {
  const gemm::F2 k(inv), magic(12582912.f);
  float f[4];
  gemm::fma2(gemm::F2(v[0], v[1]), k, magic).get(f[0], f[1]);
  gemm::fma2(gemm::F2(v[2], v[3]), k, magic).get(f[2], f[3]);
  const uint32_t lo = __byte_perm(__float_as_uint(f[0]), __float_as_uint(f[1]), 0x0040);
  const uint32_t hi = __byte_perm(__float_as_uint(f[2]), __float_as_uint(f[3]), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// And back: byte + 128 as the low bits of 2^23, less 2^23 + 128, times the scale; each step is exact.
ASRN_DEV void values4(float* v, uint32_t w, float scale) {
  const uint32_t u = w ^ 0x80808080u;
  const gemm::F2 k(scale), off(-8388736.f);
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(__byte_perm(u, 0x4B000000u, 0x7650 + i));
  gemm::mul2(gemm::add2(gemm::F2(f[0], f[1]), off), k).get(v[0], v[1]);
  gemm::mul2(gemm::add2(gemm::F2(f[2], f[3]), off), k).get(v[2], v[3]);
}

// The larger magnitude, of either sign; a NaN is the largest.
ASRN_DEV float abs_max(float a, float b) {
  asm("max.NaN.xorsign.abs.f32 %0, %0, %1;" : "+f"(a) : "f"(b));
  return a;
}
ASRN_DEV float abs_max32(const float* v) {
  float m[4] = {v[0], v[1], v[2], v[3]};
#pragma unroll
  for (int i = 4; i < 32; ++i) m[i & 3] = abs_max(m[i & 3], v[i]);
  return fabsf(abs_max(abs_max(m[0], m[1]), abs_max(m[2], m[3])));
}

// mlp8 keeps a's codes by 32 rows x 32 columns, as a warp of the products' epilogues holds them: first 16 columns of the 32
// rows, then the other 16, so that its 16 bytes a lane are 512 neighbouring ones (rows as they lie would make 32 half-used
// accesses of each). The last rows may be fewer than 32. A lane's two places:
struct CodesAt {
  int64_t first;
  int other;                                             // from the first 16 columns to the others
  ASRN_DEV CodesAt(int row, int rows, int c, int f) {
    const int in = min(32, rows - (row & ~31));
    first = (int64_t)(row & ~31) * ((f + 31) / 32 * 32) + c * in + (row & 31) * 16;
    other = in * 16;
  }
};
// The codes of a lane's 32 columns; their exponent.
ASRN_DEV int store_codes(const float* v, uint8_t* codes, const CodesAt& at) {
  const int e = block_exp(abs_max32(v));
  const float inv = inv_scale_of(e);
#pragma unroll
  for (int i = 0; i < 32; i += 16) {
    uint4 w = make_uint4(codes4(v + i, inv), codes4(v + i + 4, inv), codes4(v + i + 8, inv), codes4(v + i + 12, inv));
    if (e == kBad) w = make_uint4(0, 0, 0, 0);
    *reinterpret_cast<uint4*>(codes + at.first + (i ? at.other : 0)) = w;
  }
  return e;
}

// Where the exponent of block b of a row stands: row * by_row + b * by_block. mlp8 keeps those of x W1^T + b1 with a
// block's rows side by side (32 rows at a time write and read them); x's and pack8's are kept by rows.
struct Exps {
  int8_t* at;
  int64_t by_row, by_block;
  ASRN_DEV int8_t& operator()(int64_t row, int64_t block) const { return at[row * by_row + block * by_block]; }
};

// t = row * wide + the rest, in 32 bits where `all` of them fit.
ASRN_DEV int64_t row_of(int64_t t, int64_t all, int wide) {
  return all < (1ll << 31) ? (int64_t)((uint32_t)t / (uint32_t)wide) : t / wide;
}

// 17.5 us at 32768 x 768, 76 MB, 4.4 TB/s (18.7 with the exponents kept by blocks): 0.67 of the measured copy rate; what
// holds it from the rest has not been found.
// Four threads per block of 32 of a row of bf16, 8 values each; each thread kEach of them, all loaded first.
constexpr int kEach = 4;
__global__ void __launch_bounds__(256) k_pack8(int64_t rows, int f, int wide, const __nv_bfloat16* __restrict__ x,
                                               uint8_t* __restrict__ codes, const Exps exps) {
  const int64_t total = rows * wide;                     // wide: threads per row, a multiple of 4
  for (int64_t t0 = (int64_t)blockIdx.x * 256 * kEach; t0 < total; t0 += (int64_t)gridDim.x * 256 * kEach) {
    uint4 q[kEach];
    int64_t row[kEach];
    int c[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int64_t t = t0 + k * 256 + threadIdx.x;
      row[k] = row_of(t, total, wide);
      c[k] = (int)(t - row[k] * wide) * 8;
      if (t >= total) c[k] = f;
      q[k] = make_uint4(0, 0, 0, 0);
      if (c[k] < f) q[k] = __ldg(reinterpret_cast<const uint4*>(x + row[k] * f + c[k]));
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const uint32_t w[4] = {q[k].x, q[k].y, q[k].z, q[k].w};
      float v[8], m = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = __uint_as_float(w[j] << 16);
        v[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) m = abs_max(m, v[i]);
      m = abs_max(m, __shfl_xor_sync(0xffffffffu, m, 1));
      m = fabsf(abs_max(m, __shfl_xor_sync(0xffffffffu, m, 2)));
      const int e = block_exp(m);
      const float inv = inv_scale_of(e);
      if (c[k] >= f) continue;
      uint2 o = make_uint2(codes4(v, inv), codes4(v + 4, inv));
      if (e == kBad) o = make_uint2(0, 0);
      *reinterpret_cast<uint2*>(codes + row[k] * f + c[k]) = o;
      if (c[k] % 32 == 0) exps(row[k], c[k] / 32) = (int8_t)e;
    }
  }
}

// 8 values per thread and turn, kEach turns loaded first; `blocks` blocks, this one the `block`-th.
ASRN_DEV void unpack(int64_t block, int64_t blocks, int64_t total, int f, const uint8_t* __restrict__ codes,
                     const Exps& exps, __nv_bfloat16* __restrict__ x) {
  const int per = f / 8;
  for (int64_t t0 = block * 256 * kEach; t0 < total; t0 += blocks * 256 * kEach) {
    uint2 w[kEach];
    int e[kEach];
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int64_t t = t0 + k * 256 + threadIdx.x;
      if (t >= total) break;
      const int64_t row = row_of(t, total, per);
      w[k] = __ldg(reinterpret_cast<const uint2*>(codes) + t);
      e[k] = exps(row, (t - row * per) / 4);
    }
#pragma unroll
    for (int k = 0; k < kEach; ++k) {
      const int64_t t = t0 + k * 256 + threadIdx.x;
      if (t >= total) break;
      const float scale = scale_of(e[k]);
      float v[8];
      values4(v, w[k].x, scale);
      values4(v + 4, w[k].y, scale);
      reinterpret_cast<uint4*>(x)[t] = gemm::pack8(v);
    }
  }
}
__global__ void __launch_bounds__(256) k_unpack8(int64_t total, int f, const uint8_t* __restrict__ codes, const Exps exps,
                                                 __nv_bfloat16* __restrict__ x) {
  unpack(blockIdx.x, gridDim.x, total, f, codes, exps, x);
}

// 73 us at 32768 x 1536 x 768 (a product that only stores: 60); 149 with libm's erf and direct stores, 102 with eight warps.
// a = sum + b1 -> Q(a) (unless codes is null) and gelu(a) in bf16.
struct Up {
  static constexpr int kWarps = 16, kOwn = 1, kTable = 0;
  struct Params {
    const __nv_bfloat16* bias;
    uint8_t* codes;
    Exps exps;
    int below;                                 // rows from gelu(a) to its remainder, 0: none
  };
  const Params& p;
  int N, row, first, rows;
  bool on;
  ASRN_DEV Up(const Params& pp, int r, int m, const gemm::Shape& s, const gemm::Tile&, int)
      : p(pp), N(s.N), row(r), first(r & ~31), rows(m), on(r < m) {}
  template <class O> ASRN_DEV void chunk(float* v, int c, O& out, const CUtensorMap* map_o, const CUtensorMap*) {
    if (c >= N || first >= rows) return;       // the same for the whole warp; columns past N of the last block are zeros
    gemm::add_bias(v, p.bias + c, N - c);
    if (p.codes && on) p.exps(row, c / 32) = (int8_t)store_codes(v, p.codes, CodesAt(row, rows, c, N));
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      gemm::F2 e, q;
      tails(v[i], v[i + 1], e, q);
      gemm::fma2(gemm::F2(-fabsf(v[i]), -fabsf(v[i + 1])), q, gemm::F2(fmaxf(v[i], 0.f), fmaxf(v[i + 1], 0.f)))
          .get(v[i], v[i + 1]);
    }
    out.put(map_o, v, c, first);
    if (p.below) {
      gemm::remainder(v);
      out.put(map_o, v, c, first + p.below);
    }
  }
  ASRN_DEV void finish() {}
};

// dG = sum -> dA = dG gelu'(a') and gelu(a') in bf16, and dA's column sums by 32 rows. 87 us at 32768 x 1536 x 768 (210 with
// libm's functions and direct stores; 100 computed, 92 with the table, 87 with the codes by blocks).
// a' = code 2^e takes 256 values for each e, so gelu and gelu' of the 16 exponents that matter lie in a table of shared
// memory (gelu in bf16, as it leaves; gelu' in fp16, so that both fit 32 bits: its 2^-11 adds 1 % to the bf16 rounding of
// dA, and where it is subnormal, for a < -4.6, it is off by up to 2^-25, less than gelu_both's own 3.6e-7): one 32-bit load
// for an element instead of about 20 instructions. Blocks with another exponent (all of a below 0.004, or some above 254)
// are computed.
struct Down {
  static constexpr int kWarps = 16, kOwn = 2, kLow = -14, kExps = 16, kTable = kExps * 1024;
  struct Params {
    const uint8_t* codes;
    Exps exps;
    float* sums;                               // [ceil(rows / 32)][N], or null
    int below;                                 // rows from dA and gelu(a') to their remainders, 0: none
  };
  const Params& p;
  int N, row, first, rows;
  bool on;
  ASRN_DEV Down(const Params& pp, int r, int m, const gemm::Shape& s, const gemm::Tile&, int)
      : p(pp), N(s.N), row(r), first(r & ~31), rows(m), on(r < m) {}
  static ASRN_DEV void fill(uint32_t* table, int tid, int threads) {
    for (int t = tid; t < kExps * 128; t += threads) {     // two codes each: code = place - 128
      const float scale = pow2(t / 128 + kLow), a0 = (float)(2 * (t % 128) - 128) * scale, a1 = a0 + scale;
      gemm::F2 g, slope;
      gelu_both(a0, a1, g, slope);
      float g0, g1, s0, s1;
      g.get(g0, g1);
      slope.get(s0, s1);
      const uint32_t w = umma::pack_bf16x2(g0, g1);
      table[2 * t] = w << 16 | __half_as_ushort(__float2half_rn(s0));
      table[2 * t + 1] = (w & 0xffff0000u) | __half_as_ushort(__float2half_rn(s1));
    }
  }
  template <class O> ASRN_DEV void chunk(float* v, int c, O& out, const CUtensorMap* map_o, const CUtensorMap* map_p) {
    if (c >= N || first >= rows) return;       // the same for the whole warp
    const int exp = on ? p.exps(row, c / 32) : kLow;
    uint4 codes[2] = {};
    if (on) {
      const CodesAt at(row, rows, c, N);
      codes[0] = __ldg(reinterpret_cast<const uint4*>(p.codes + at.first));
      codes[1] = __ldg(reinterpret_cast<const uint4*>(p.codes + at.first + at.other));
    }
    uint4 packed[4], rest[4];
    if (!p.below && __all_sync(0xffffffffu, exp >= kLow && exp < kLow + kExps)) {
      const uint32_t* row_of_e = out.table + (exp - kLow) * 256 + 128;
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        const uint4& k = codes[i / 16];
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          const uint32_t four = (j < 4) == (i % 16 == 0) ? (j < 4 ? k.x : k.w) : (j < 4 ? k.z : k.y);
          const uint32_t t0 = row_of_e[(int8_t)(four >> (8 * (j & 3)))], t1 = row_of_e[(int8_t)(four >> (8 * (j & 3) + 8))];
          v[i + j] *= __half2float(__ushort_as_half((unsigned short)t0));
          v[i + j + 1] *= __half2float(__ushort_as_half((unsigned short)t1));
          w[j / 2] = __byte_perm(t0, t1, 0x7632);
        }
        packed[i / 8] = make_uint4(w[0], w[1], w[2], w[3]);
      }
    } else {
      const float scale = scale_of(exp);
#pragma unroll
      for (int i = 0; i < 32; i += 8) {
        const uint4& k = codes[i / 16];
        float g[8];
        values4(g, i % 16 ? k.z : k.x, scale);
        values4(g + 4, i % 16 ? k.w : k.y, scale);
#pragma unroll
        for (int j = 0; j < 8; j += 2) {
          gemm::F2 f, slope;
          gelu_both(g[j], g[j + 1], f, slope);
          f.get(g[j], g[j + 1]);
          gemm::mul2(gemm::F2(v[i + j], v[i + j + 1]), slope).get(v[i + j], v[i + j + 1]);
        }
        packed[i / 8] = gemm::pack8(g);
        if (p.below) {
          float r[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) r[j] = g[j] - round_bf16(g[j]);
          rest[i / 8] = gemm::pack8(r);
        }
      }
      if (p.below) out.put(map_p, rest, c, first + p.below);
    }
    out.put(map_p, packed, c, first);
    out.put(map_o, v, c, first);
    if (p.below) {
      float r[32];
#pragma unroll
      for (int i = 0; i < 32; ++i) r[i] = v[i] - round_bf16(v[i]);
      out.put(map_o, r, c, first + p.below);
    }
    if (p.sums) {                              // rows past the end are zeros: the operand's rows were
      const int lane = threadIdx.x & 31;
      const float s = column_sum(v, lane);
      if (c + lane < N) p.sums[(int64_t)(first / 32) * N + c + lane] = s;
    }
  }
  ASRN_DEV void finish() {}
};

// 29 us at 32768 x 768 both, 126 MB, 4.3 TB/s, 0.66 of the measured copy rate.
// x' from its codes (the first `unpackers` blocks), and sums of dY's columns over 64 rows (the others: block = 64 rows x
// 256 columns, a lane 8 columns, a warp every eighth row).
constexpr int kColRows = 64;
__global__ void __launch_bounds__(256)
k_prepare(int unpackers, int64_t eighths, int d, const uint8_t* __restrict__ codes, const Exps exps,
          __nv_bfloat16* __restrict__ x, int64_t rows, int n, const __nv_bfloat16* __restrict__ dy,
          float* __restrict__ sums) {
  __shared__ float sh[8][256];
  if ((int)blockIdx.x < unpackers) {
    unpack(blockIdx.x, unpackers, eighths, d, codes, exps, x);
    return;
  }
  const int wide = (n + 255) / 256, block = blockIdx.x - unpackers, lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int c0 = block % wide * 256, c = c0 + lane * 8;
  const int64_t r0 = (int64_t)(block / wide) * kColRows;
  float s[8] = {};
#pragma unroll
  for (int k = 0; k < kColRows / 8; ++k) {
    const int64_t r = r0 + k * 8 + wid;
    if (r < rows && c < n) {
      const uint4 q = __ldg(reinterpret_cast<const uint4*>(dy + r * n + c));
      const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[2 * j] += __uint_as_float(w[j] << 16);
        s[2 * j + 1] += __uint_as_float(w[j] & 0xffff0000u);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[wid][lane + 32 * j] = s[j];
  __syncthreads();
  const int own = c0 + lane * 8 + wid;                   // this thread's column: its lane's wid-th
  float t = 0.f;
#pragma unroll
  for (int k = 0; k < 8; ++k) t += sh[k][threadIdx.x];
  if (own < n) sums[(int64_t)(block / wide) * n + own] = t;
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
  w.ac = take((size_t)N * ((ff + 31) / 32) * 32);
  w.ae = take((size_t)N * ((ff + 31) / 32));
  w.total = o;
  return w;
}

struct Mlp8Ws {
  int64_t rows;                                // of gelu(a) and dA, their remainders among them
  int below, shares1, shares2;                 // below: rows to the remainders (a multiple of 32), 0: none
  size_t da, g, x, sum1, sum2, slots, total;
};

Mlp8Ws mlp8_ws(int64_t N, int64_t d, int64_t ff, int64_t dout, bool backward) {
  Mlp8Ws w{};
  size_t o = 0;
  auto take = [&](size_t bytes) { const size_t at = o; o = align_up(o + bytes); return at; };
  w.below = N <= kTwiceRows ? (int)((N + 31) / 32 * 32) : 0;
  w.rows = w.below ? 2 * w.below : N;
  w.g = take((size_t)w.rows * ff * 2);
  if (backward) {
    w.shares1 = gemm::shares_for(ff, d, w.rows);
    w.shares2 = gemm::shares_for(dout, ff, w.rows);
    w.da = take((size_t)w.rows * ff * 2);
    w.x = take((size_t)N * d * 2);
    w.sum1 = take((size_t)((N + 31) / 32) * ff * 4);
    w.sum2 = take((size_t)((N + kColRows - 1) / kColRows) * dout * 4);
    w.slots = take(std::max(w.shares1 ? gemm::slot_bytes(ff, d, w.shares1) : 0,
                            w.shares2 ? gemm::slot_bytes(dout, ff, w.shares2) : 0));
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

unsigned grid_for(int64_t threads) {
  return (unsigned)std::min<int64_t>((threads + 256 * kEach - 1) / (256 * kEach), 148 * 16);
}

Exps by_rows(const void* p, int f) { return Exps{(int8_t*)p, (f + 31) / 32, 1}; }
Exps by_blocks(const void* p, int64_t rows) { return Exps{(int8_t*)p, 1, rows}; }

int pack8(int64_t rows, int f, const void* x, void* codes, const Exps& exps, cudaStream_t s) {
  const int wide = (f + 31) / 32 * 4;
  k_pack8<<<grid_for(rows * wide), 256, 0, s>>>(rows, f, wide, reinterpret_cast<const __nv_bfloat16*>(x),
                                                reinterpret_cast<uint8_t*>(codes), exps);
  return launched();
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
  return pack8(rows, f, x, codes, by_rows(exps, f), reinterpret_cast<cudaStream_t>(stream));
}

int asrn_unpack8(int64_t rows, int32_t f, const void* codes, const void* exps, void* x, void* stream) {
  using namespace asrn;
  if (rows < 0 || f < 1) return ASRN_ERR_ARG;
  if (f % 8) return ASRN_ERR_UNSUPPORTED;
  if (rows == 0) return ASRN_OK;
  if (!x || !codes || !exps || (uintptr_t)x % 16 || (uintptr_t)codes % 8) return ASRN_ERR_ARG;
  k_unpack8<<<grid_for(rows * (f / 8)), 256, 0, reinterpret_cast<cudaStream_t>(stream)>>>(
      rows * (f / 8), f, reinterpret_cast<const uint8_t*>(codes), by_rows(exps, f), reinterpret_cast<__nv_bfloat16*>(x));
  return launched();
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
      (uintptr_t)y % 16 || (uintptr_t)b1 % 16 || (uintptr_t)b2 % 16)
    return ASRN_ERR_ARG;
  const Mlp8Saved sv = mlp8_saved(N, d, ff);
  const Mlp8Ws ws = mlp8_ws(N, d, ff, dout, false);
  if ((saved && (saved_bytes < sv.total || (uintptr_t)saved % 256)) || !workspace || workspace_bytes < ws.total ||
      (uintptr_t)workspace % 256)
    return ASRN_ERR_WORKSPACE;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  char* S = reinterpret_cast<char*>(saved);
  __nv_bfloat16* g = reinterpret_cast<__nv_bfloat16*>(reinterpret_cast<char*>(workspace) + ws.g);
  if (S && (st = pack8(N, d, x, S + sv.xc, by_rows(S + sv.xe, d), s))) return st;
  gemm::Shape a{};
  a.M = (int)N; a.N = ff; a.K = d; a.group = 16; a.status = status;
  const Up::Params p{reinterpret_cast<const __nv_bfloat16*>(b1), S ? reinterpret_cast<uint8_t*>(S + sv.ac) : nullptr,
                     S ? by_blocks(S + sv.ae, N) : Exps{}, ws.below};
  if ((st = gemm::launch<false, false, Up>(x, d, w1, d, a, p, s, {g, ws.rows, ff, ff}))) return st;
  a.N = dout; a.K = ff; a.second_pass = ws.below > 0; a.a_step = ws.below;
  return gemm::launch<false, false, gemm::StoreBf16>(g, ff, w2, ff, a,
                                                     {reinterpret_cast<const __nv_bfloat16*>(b2), nullptr, nullptr}, s,
                                                     {y, N, dout, dout});
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
  float* slots = reinterpret_cast<float*>(W + ws.slots);
  float* sum1 = reinterpret_cast<float*>(W + ws.sum1);
  float* sum2 = reinterpret_cast<float*>(W + ws.sum2);
  const int64_t blocks = (N + kColRows - 1) / kColRows;
  gemm::Shape a{};
  a.M = (int)N; a.group = 16; a.status = status;
  if (dw1 || db2) {
    const int64_t eighths = dw1 ? N * (d / 8) : 0;
    const unsigned unpackers = dw1 ? grid_for(eighths) : 0;
    const unsigned summers = db2 ? (unsigned)(blocks * ((dout + 255) / 256)) : 0;
    k_prepare<<<unpackers + summers, 256, 0, s>>>(
        (int)unpackers, eighths, d, reinterpret_cast<const uint8_t*>(S + sv.xc),
        by_rows(S + sv.xe, d), reinterpret_cast<__nv_bfloat16*>(W + ws.x), N, dout,
        reinterpret_cast<const __nv_bfloat16*>(dy), sum2);
    if ((st = launched())) return st;
  }
  if (dx || dw1 || db1 || dw2) {
    a.N = ff; a.K = dout;
    const Down::Params p{reinterpret_cast<const uint8_t*>(S + sv.ac), by_blocks(S + sv.ae, N), db1 ? sum1 : nullptr,
                         ws.below};
    if ((st = gemm::launch<false, true, Down>(dy, dout, w2, ff, a, p, s, {da, ws.rows, ff, ff},
                                                    {g, ws.rows, ff, ff}))) return st;
  }
  if (dx) {
    a.N = d; a.K = ff; a.second_pass = ws.below > 0; a.a_step = ws.below;
    if ((st = gemm::launch<false, true, gemm::StoreBf16>(da, ff, w1, d, a, {}, s, {dx, N, d, d}))) return st;
  }
  if (dw1 && (st = weight_grad(N, ff, d, da, ws.below, W + ws.x, 0, ws.shares1, slots, dw1, status, s))) return st;
  if (dw2 && (st = weight_grad(N, dout, ff, dy, 0, g, ws.below, ws.shares2, slots, dw2, status, s))) return st;
  if (db1 || db2) {
    const ColSum q1{(N + 31) / 32, db1 ? ff : 0, sum1, reinterpret_cast<__nv_bfloat16*>(db1)};
    const ColSum q2{blocks, db2 ? dout : 0, sum2, reinterpret_cast<__nv_bfloat16*>(db2)};
    const int b1 = (q1.n + 31) / 32, b2 = (q2.n + 31) / 32;
    k_colsum<<<(unsigned)(b1 + b2), 1024, 0, s>>>(q1, q2, b1);
    return launched();
  }
  return ASRN_OK;
}

}  // extern "C"
