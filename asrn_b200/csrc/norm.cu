// Layer norm of rows of d values, with the residual sum before it, forward and backward:
//   s = x + r (rounded to r's type, handed on),  m = mean s,  v = mean (s - m)^2,  k = 1 / sqrt(v + eps)
//   h = (s - m) k,  y = h w + b
//   g = dy w,  ds' = k (g - mean g - h mean(g h)) + ds,  dx = dr = ds',  dw = sum over the rows of dy h,  db = sum of dy
// Sums in fp32, the variance from the differences (a second walk over registers, none over memory). Kept for the backward pass:
// s (or x) and each row's m and k in fp32.
//
// Bound by memory: each row is read once into registers and written once. A warp holds a row of up to 1024 values, a block
// of 256 or 512 threads a longer one, eight values (16 or 32 bytes) a load. Rows of a width that is no multiple of 8 start anywhere
// between two such loads: they are read from the last boundary before them on, their first value the `shift`-th of its eight; the
// rows' ends are written value by value (k_norm_shifted, and Shifted below). Tensors that are not 16-byte aligned go value by value.
// The backward pass's blocks stay for many rows with their columns' sums of dy h and dy in registers; a block's sums go to fp32
// parts that k_norm_sums adds up in order (4 us at 32768 x 768).
#include "common.cuh"
#include "layout.h"

#include <algorithm>
#include <atomic>
#include <type_traits>

namespace asrn {

namespace {

constexpr int kF32 = 0, kBf16 = 1, kNone = 2;            // types of the C interface
using F32 = std::integral_constant<int, kF32>;
using Bf16 = std::integral_constant<int, kBf16>;
using None = std::integral_constant<int, kNone>;
constexpr int kMaxD = 16384;

// V values of type t at an element offset, as they lie in memory; then as floats.
template <int V> struct Raw;
template <> struct Raw<8> { uint4 a, b; };
template <> struct Raw<1> { uint32_t a; };

ASRN_DEV Raw<8> load(Raw<8>*, const void* p, int64_t at, int t) {
  Raw<8> r;
  const char* q = reinterpret_cast<const char*>(p) + at * (t == kBf16 ? 2 : 4);
  r.a = __ldg(reinterpret_cast<const uint4*>(q));
  if (t == kF32) r.b = __ldg(reinterpret_cast<const uint4*>(q) + 1);
  return r;
}
ASRN_DEV Raw<1> load(Raw<1>*, const void* p, int64_t at, int t) {
  Raw<1> r;
  r.a = t == kBf16 ? (uint32_t)__ldg(reinterpret_cast<const unsigned short*>(p) + at)
                   : __ldg(reinterpret_cast<const uint32_t*>(p) + at);
  return r;
}
ASRN_DEV void floats(const Raw<8>& r, int t, float* v) {
  if (t == kBf16) {
    const uint32_t w[4] = {r.a.x, r.a.y, r.a.z, r.a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[2 * i] = __uint_as_float(w[i] << 16);
      v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
    }
  } else {
    const uint32_t w[8] = {r.a.x, r.a.y, r.a.z, r.a.w, r.b.x, r.b.y, r.b.z, r.b.w};
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = __uint_as_float(w[i]);
  }
}
ASRN_DEV void floats(const Raw<1>& r, int t, float* v) { v[0] = __uint_as_float(t == kBf16 ? r.a << 16 : r.a); }

template <int V> ASRN_DEV void store(void* p, int64_t at, int t, const float* v) {
  char* q = reinterpret_cast<char*>(p) + at * (t == kBf16 ? 2 : 4);
  if constexpr (V == 8) {
    if (t == kBf16) {
      *reinterpret_cast<uint4*>(q) = make_uint4(pack2_bf16(v[0], v[1]), pack2_bf16(v[2], v[3]), pack2_bf16(v[4], v[5]),
                                                pack2_bf16(v[6], v[7]));
    } else {
      reinterpret_cast<float4*>(q)[0] = make_float4(v[0], v[1], v[2], v[3]);
      reinterpret_cast<float4*>(q)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
  } else {
    if (t == kBf16)
      *reinterpret_cast<__nv_bfloat16*>(q) = __float2bfloat16_rn(v[0]);
    else
      *reinterpret_cast<float*>(q) = v[0];
  }
}

// The sum over a row's T threads: a warp's or half of one, or a whole block's (each sum with its own room, so one barrier serves).
template <int T> ASRN_DEV float row_sum(float v, float* room) {
#pragma unroll
  for (int o = (T < 32 ? T : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (T <= 32) return v;
  if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < T / 32; ++i) s += room[i];
  return s;
}

constexpr int threads_of(int T) { return T <= 32 ? 128 : T; }

// V values a load, C loads a thread, T threads a row; types XT, RT known at compile time unless they are -1.
// 32768 x 768, bf16 x, fp32 r and s, bf16 y: 302 MB in 51 us, 5.9 TB/s; 64 rows 2 us, latency (a row's load and two reductions).
// 65536 x 100 with 16 threads a row 25 us, with 32 threads 43.
struct Forward {
  int64_t rows;
  int d;
  const void *x, *res, *w, *b;
  int xt, rt, wt, yt;
  float eps;
  void *sum, *y;
  float2* stats;                                         // m and k of each row, or null
};
template <int V, int XT, int RT, int C, int T>
__global__ void __launch_bounds__(threads_of(T), 1) k_norm(const Forward f) {
  __shared__ float room[2][32];
  wait_previous();
  let_next();
  const int xt = XT < 0 ? f.xt : XT, rt = RT < 0 ? f.rt : RT;
  const int tid = T <= 32 ? threadIdx.x % T : threadIdx.x;
  const int64_t own = T <= 32 ? (int64_t)blockIdx.x * (blockDim.x / T) + threadIdx.x / T : blockIdx.x;
  const bool on = own < f.rows;                          // a warp's second row may be none: it goes along
  const int64_t row = T < 32 ? min(own, f.rows - 1) : own, at = row * f.d;
  if (T == 32 && !on) return;
  Raw<V> rx[C], rr[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {                          // without a condition: all under way at once
    const int64_t c = at + min((tid + i * T) * V, f.d - V);
    rx[i] = load((Raw<V>*)0, f.x, c, xt);
    if (rt != kNone) rr[i] = load((Raw<V>*)0, f.res, c, rt);
  }
  float v[C * V], s = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = (tid + i * T) * V;
    float* u = v + i * V;
    if (c >= f.d) {
#pragma unroll
      for (int j = 0; j < V; ++j) u[j] = 0.f;
      continue;
    }
    floats(rx[i], xt, u);
    if (rt != kNone) {
      float r[V];
      floats(rr[i], rt, r);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        u[j] += r[j];
        if (rt == kBf16) u[j] = round_bf16(u[j]);
      }
      if (T >= 32 || on) store<V>(f.sum, at + c, rt, u);
    }
#pragma unroll
    for (int j = 0; j < V; ++j) s += u[j];
  }
  const float m = row_sum<T>(s, room[0]) / (float)f.d;
  s = 0.f;
#pragma unroll
  for (int i = 0; i < C; ++i)
    if ((tid + i * T) * V < f.d)
#pragma unroll
      for (int j = 0; j < V; ++j) s = fmaf(v[i * V + j] - m, v[i * V + j] - m, s);
  const float k = 1.f / sqrtf(row_sum<T>(s, room[1]) / (float)f.d + f.eps);
  if (f.stats && tid == 0 && on) f.stats[row] = make_float2(m, k);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = (tid + i * T) * V;
    if (c >= f.d || !on) continue;
    float w[V], b[V], *u = v + i * V;
    floats(load((Raw<V>*)0, f.w, c, f.wt), f.wt, w);
#pragma unroll
    for (int j = 0; j < V; ++j) u[j] = (u[j] - m) * k * w[j];
    if (f.b) {
      floats(load((Raw<V>*)0, f.b, c, f.wt), f.wt, b);
#pragma unroll
      for (int j = 0; j < V; ++j) u[j] += b[j];
    }
    store<V>(f.y, at + c, f.yt, u);
  }
}

// ---- rows that start anywhere -------------------------------------------------------------------------------------------------
// Vector v of a row whose first value is the shift-th of its eight holds the columns 8 v - shift + j. The weights stand in shared memory
// by planes of every eighth column (so that neighbouring vectors read neighbouring words), fp32.
struct Planes {
  float* at;
  int pitch;
  ASRN_DEV Planes(float* p, int d) : at(p), pitch(d / 8 + 3) {}
  static __host__ ASRN_DEV int floats(int d) { return 8 * (d / 8 + 3); }
  ASRN_DEV void fill(const void* w, int t, int d) const {
    for (int c = threadIdx.x; c < d; c += blockDim.x) {
      float v;
      asrn::floats(load((Raw<1>*)0, w, c, t), t, &v);
      at[(c & 7) * pitch + (c >> 3) + 1] = v;
    }
  }
  ASRN_DEV float operator()(int v, int j, int shift) const {
    const int q = j - shift;
    return at[(q < 0 ? (q + 8) * pitch : q * pitch + 1) + v];
  }
};
// Eight values at a flat index that is a multiple of 8, those past the tensor's end as zeros.
ASRN_DEV Raw<8> load_to(const void* p, int64_t at, int64_t total, int t) {
  if (at + 8 <= total) return load((Raw<8>*)0, p, at, t);
  Raw<8> r;
  uint32_t w[8] = {};
  for (int j = 0; j < 8 && at + j < total; ++j) {
    const uint32_t u = load((Raw<1>*)0, p, at + j, t).a;
    if (t == kBf16)
      w[j / 2] |= u << (16 * (j & 1));
    else
      w[j] = u;
  }
  r.a = make_uint4(w[0], w[1], w[2], w[3]);
  r.b = make_uint4(w[4], w[5], w[6], w[7]);
  return r;
}
// Where the vectors of a row that starts anywhere stand: from `at` on, vector 0 to `last`, its first value the shift-th of vector 0.
// inside: all of them end within the tensor (a row of few values may be followed by others that do not reach a vector's end).
struct RowAt {
  int shift, last;
  int64_t at;
  bool inside;
  __host__ ASRN_DEV RowAt(int64_t row, int64_t rows, int d)
      : shift((int)(row * d & 7)), last((d + shift - 1) / 8), at(row * d - shift), inside(at + 8 * (int64_t)(last + 1) <= rows * d) {}
};
// Those of a vector's values that are the row's: j from `low` on, below `high`.
struct Span {
  int low, high;
  ASRN_DEV Span(int v, int shift, int d) : low(v == 0 ? shift : 0), high(min(8, d + shift - 8 * v)) {}
  ASRN_DEV bool whole() const { return low == 0 && high == 8; }
  ASRN_DEV bool none() const { return low >= high; }
};
ASRN_DEV void store_span(void* p, int64_t at, int t, const float* v, const Span& in) {
  if (in.whole()) {
    store<8>(p, at, t, v);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j >= in.low && j < in.high) store<1>(p, at + j, t, v + j);
  }
}

// Rows that start anywhere. Each vector is loaded whole, from the last 16-byte boundary before the row on, and its values outside the
// row count for nothing; the weights lie in shared memory, where any shift reads them without bank conflicts (Planes); blocks stay for
// many rows so that they are filled once. 33870 x 431 bf16 43 us, with gradients 128 (value by value
// 190); 2067 x 7159 46 us.

// Its blocks that stay on an SM at once.
constexpr int stay_shifted(int C, int T) {
  return T <= 32 ? (C == 1 ? 10 : C == 2 ? 7 : C == 3 ? 5 : 4) : T == 256 ? (C == 1 ? 5 : 4) : C == 2 ? 2 : 1;
}
template <int XT, int RT, int C, int T>
__global__ void __launch_bounds__(threads_of(T), stay_shifted(C, T)) k_norm_shifted(const Forward f) {
  extern __shared__ float planes[];
  __shared__ float room[2][2][32];
  constexpr int kRows = threads_of(T) / T;
  const Planes w(planes, f.d), b(planes + Planes::floats(f.d), f.d);
  wait_previous();
  let_next();
  w.fill(f.w, f.wt, f.d);
  if (f.b) b.fill(f.b, f.wt, f.d);
  __syncthreads();
  const int tid = T <= 32 ? threadIdx.x % T : threadIdx.x, sub = T <= 32 ? threadIdx.x / T : 0;
  int turn = 0;
  for (int64_t first = (int64_t)blockIdx.x * kRows; first < f.rows; first += (int64_t)gridDim.x * kRows, turn ^= 1) {
    const int64_t row = min(first + sub, f.rows - 1);
    const bool on = first + sub < f.rows;                // else the last row goes along, for its warp's other half
    const RowAt own(row, f.rows, f.d);
    const int shift = own.shift, last = own.last;
    const int64_t at = own.at;
    Raw<8> rx[C], rr[C];
    if (own.inside) {                                    // without a condition of each: all under way at once
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t to = at + 8 * min(tid + i * T, last);
        rx[i] = load((Raw<8>*)0, f.x, to, XT);
        if (RT != kNone) rr[i] = load((Raw<8>*)0, f.res, to, RT);
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t to = at + 8 * min(tid + i * T, last);
        rx[i] = load_to(f.x, to, f.rows * f.d, XT);
        if (RT != kNone) rr[i] = load_to(f.res, to, f.rows * f.d, RT);
      }
    }
    float u[C * 8], s = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int v = tid + i * T;
      const Span in(v, shift, f.d);
      float* e = u + i * 8;
      floats(rx[i], XT, e);
      if (RT != kNone) {
        float r[8];
        floats(rr[i], RT, r);
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          e[j] += r[j];
          if (RT == kBf16) e[j] = round_bf16(e[j]);
        }
        if (!in.none() && on) store_span(f.sum, at + 8 * v, RT, e, in);
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) s += j >= in.low && j < in.high ? e[j] : 0.f;
    }
    const float m = row_sum<T>(s, room[turn][0]) / (float)f.d;
    s = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const Span in(tid + i * T, shift, f.d);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float q = j >= in.low && j < in.high ? u[i * 8 + j] - m : 0.f;
        s = fmaf(q, q, s);
      }
    }
    const float k = 1.f / sqrtf(row_sum<T>(s, room[turn][1]) / (float)f.d + f.eps);
    if (f.stats && tid == 0 && on) f.stats[row] = make_float2(m, k);
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int v = tid + i * T;
      const Span in(v, shift, f.d);
      if (in.none() || !on) continue;
      float* e = u + i * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e[j] = (e[j] - m) * k * w(v, j, shift);
        if (f.b) e[j] += b(v, j, shift);
      }
      store_span(f.y, at + 8 * v, f.yt, e, in);
    }
  }
}

// s, ds and out of type ST, dy of type YT; `other`: the same gradient in the other type. parts: [blocks][2][d] sums of dy h
// and dy, or null.
struct Backward {
  int64_t rows;
  int d;
  const void *s, *dy, *ds, *w;
  int st, yt, wt;
  const float2* stats;
  void *out, *other;
  float* parts;
};
template <int V, int ST, int YT, int C, int T>
__global__ void __launch_bounds__(threads_of(T), T == 256 ? 2 : 1) k_norm_back(const Backward f) {
  constexpr int kRows = threads_of(T) / T;               // of a block at a time
  __shared__ float room[2][2][32];
  __shared__ float sums[T == 32 ? 2 * 32 * C * V : 1];
  wait_previous();
  let_next();
  const int st = ST < 0 ? f.st : ST, yt = YT < 0 ? f.yt : YT;
  const int tid = T == 32 ? threadIdx.x & 31 : threadIdx.x, wid = T == 32 ? threadIdx.x >> 5 : 0;
  float dw[C * V] = {}, db[C * V] = {};
  const float inv = 1.f / (float)f.d;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + wid; row < f.rows; row += (int64_t)gridDim.x * kRows, turn ^= 1) {
    const int64_t at = row * f.d;
    Raw<V> rs[C], ry[C], rd[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {                        // without a condition: all under way at once
      const int64_t c = at + min((tid + i * T) * V, f.d - V);
      rs[i] = load((Raw<V>*)0, f.s, c, st);
      ry[i] = load((Raw<V>*)0, f.dy, c, yt);
      if (f.ds) rd[i] = load((Raw<V>*)0, f.ds, c, st);
    }
    const float2 mk = __ldg(f.stats + row);
    float h[C * V], g[C * V], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = (tid + i * T) * V;
      float *u = h + i * V, *e = g + i * V;
      if (c >= f.d) {
#pragma unroll
        for (int j = 0; j < V; ++j) u[j] = e[j] = 0.f;
        continue;
      }
      float w[V];
      floats(load((Raw<V>*)0, f.w, c, f.wt), f.wt, w);
      floats(rs[i], st, u);
      floats(ry[i], yt, e);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        u[j] = (u[j] - mk.x) * mk.y;
        dw[i * V + j] = fmaf(e[j], u[j], dw[i * V + j]);
        db[i * V + j] += e[j];
        e[j] *= w[j];
        s1 += e[j];
        s2 = fmaf(e[j], u[j], s2);
      }
    }
    if (!f.out && !f.other) continue;
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if constexpr (T > 32) {                              // the rooms of two rows in turn: one barrier a row
      if ((tid & 31) == 0) {
        room[turn][0][tid >> 5] = s1;
        room[turn][1][tid >> 5] = s2;
      }
      __syncthreads();
      s1 = s2 = 0.f;
#pragma unroll
      for (int i = 0; i < T / 32; ++i) {
        s1 += room[turn][0][i];
        s2 += room[turn][1][i];
      }
    }
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = (tid + i * T) * V;
      if (c >= f.d) continue;
      float *u = h + i * V, *e = g + i * V;
#pragma unroll
      for (int j = 0; j < V; ++j) e[j] = mk.y * (e[j] - s1 - u[j] * s2);
      if (f.ds) {
        floats(rd[i], st, u);
#pragma unroll
        for (int j = 0; j < V; ++j) e[j] += u[j];
      }
      if (f.out) store<V>(f.out, at + c, st, e);
      if (f.other) store<V>(f.other, at + c, 1 - st, e);
    }
  }
  if (!f.parts) return;
  float* part = f.parts + (int64_t)blockIdx.x * 2 * f.d;
  if constexpr (T > 32) {
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = (tid + i * T) * V;
      if (c < f.d) {
        store<V>(part, c, kF32, dw + i * V);
        store<V>(part + f.d, c, kF32, db + i * V);
      }
    }
  } else {                                               // the block's warps, one after another
    for (int w = 0; w < kRows; ++w) {
      if (wid == w)
#pragma unroll
        for (int i = 0; i < C * V; ++i) {
          sums[i * 32 + tid] = w ? sums[i * 32 + tid] + dw[i] : dw[i];
          sums[(C * V + i) * 32 + tid] = w ? sums[(C * V + i) * 32 + tid] + db[i] : db[i];
        }
      __syncthreads();
    }
    for (int c = threadIdx.x; c < f.d; c += blockDim.x) {
      const int q = c / V, own = (q / 32 * V + c % V) * 32 + q % 32;     // where column c's thread put it
      part[c] = sums[own];
      part[f.d + c] = sums[C * V * 32 + own];
    }
  }
}

// The same for rows that start anywhere, by blocks. A block's rows are eight apart, so that they all start alike.
template <int ST, int YT, int C, int T>
__global__ void __launch_bounds__(T, T == 256 ? 2 : 1) k_norm_back_shifted(const Backward f) {
  extern __shared__ float planes[];
  __shared__ float room[2][2][32];
  const Planes w(planes, f.d);
  wait_previous();
  let_next();
  w.fill(f.w, f.wt, f.d);
  __syncthreads();
  const RowAt first(blockIdx.x, f.rows, f.d);
  const int tid = threadIdx.x, shift = first.shift, last = first.last;
  const int64_t total = f.rows * f.d;
  float dw[C * 8] = {}, db[C * 8] = {};
  const float inv = 1.f / (float)f.d;
  int turn = 0;
  for (int64_t row = blockIdx.x; row < f.rows; row += gridDim.x, turn ^= 1) {
    const RowAt own(row, f.rows, f.d);
    const int64_t at = own.at;
    Raw<8> rs[C], ry[C], rd[C];
    if (own.inside) {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t to = at + 8 * min(tid + i * T, last);
        rs[i] = load((Raw<8>*)0, f.s, to, ST);
        ry[i] = load((Raw<8>*)0, f.dy, to, YT);
        if (f.ds) rd[i] = load((Raw<8>*)0, f.ds, to, ST);
      }
    } else {
#pragma unroll
      for (int i = 0; i < C; ++i) {
        const int64_t to = at + 8 * min(tid + i * T, last);
        rs[i] = load_to(f.s, to, total, ST);
        ry[i] = load_to(f.dy, to, total, YT);
        if (f.ds) rd[i] = load_to(f.ds, to, total, ST);
      }
    }
    const float2 mk = __ldg(f.stats + row);
    float h[C * 8], g[C * 8], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int v = tid + i * T;
      const Span in(v, shift, f.d);
      float *u = h + i * 8, *e = g + i * 8;
      floats(rs[i], ST, u);
      floats(ry[i], YT, e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const bool on = j >= in.low && j < in.high;
        u[j] = on ? (u[j] - mk.x) * mk.y : 0.f;
        e[j] = on ? e[j] : 0.f;
        dw[i * 8 + j] = fmaf(e[j], u[j], dw[i * 8 + j]);
        db[i * 8 + j] += e[j];
        e[j] = on ? e[j] * w(v, j, shift) : 0.f;
        s1 += e[j];
        s2 = fmaf(e[j], u[j], s2);
      }
    }
    if (!f.out && !f.other) continue;
    s1 = warp_sum(s1);
    s2 = warp_sum(s2);
    if ((tid & 31) == 0) {                               // the rooms of two rows in turn: one barrier a row
      room[turn][0][tid >> 5] = s1;
      room[turn][1][tid >> 5] = s2;
    }
    __syncthreads();
    s1 = s2 = 0.f;
#pragma unroll
    for (int i = 0; i < T / 32; ++i) {
      s1 += room[turn][0][i];
      s2 += room[turn][1][i];
    }
    s1 *= inv;
    s2 *= inv;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int v = tid + i * T;
      const Span in(v, shift, f.d);
      if (in.none()) continue;
      float *u = h + i * 8, *e = g + i * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = mk.y * (e[j] - s1 - u[j] * s2);
      if (f.ds) {
        floats(rd[i], ST, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] += u[j];
      }
      if (f.out) store_span(f.out, at + 8 * v, ST, e, in);
      if (f.other) store_span(f.other, at + 8 * v, 1 - ST, e, in);
    }
  }
  if (!f.parts) return;
  float* part = f.parts + (int64_t)blockIdx.x * 2 * f.d;
#pragma unroll
  for (int i = 0; i < C; ++i)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int c = (tid + i * T) * 8 - shift + j;
      if (c >= 0 && c < f.d) {
        part[c] = dw[i * 8 + j];
        part[f.d + c] = db[i * 8 + j];
      }
    }
}

// The same for rows that a warp holds, eight values a load (d <= 1024; Shifted: 7 less): each warp's next row comes to shared memory
// by asynchronous copies while it works on the one before, which costs no registers beside the columns' sums. 72 us at 32768 x 768,
// fp32 s and ds, bf16 dy and dx, 403 MB, 5.6 TB/s; with three or four rows under way, and fewer warps, 77 and more.
constexpr int kWarps = 4, kStages = 2;
ASRN_DEV void copy_row(uint8_t* to, const void* from, int64_t at, int bytes, int64_t left, int lane) {
  const char* p = reinterpret_cast<const char*>(from) + at;
  for (int b = lane * 16; b < bytes; b += 512) {
    const int n = (int)max((int64_t)0, min((int64_t)16, left - b));        // the tensor's last bytes: the rest are zeros
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((uint32_t)__cvta_generic_to_shared(to + b)),
                 "l"(n ? p + b : p), "r"(n)
                 : "memory");
  }
}
ASRN_DEV Raw<8> staged(const uint8_t* p, int c, int t) {
  Raw<8> r;
  const uint4* q = reinterpret_cast<const uint4*>(p + c * (t == kBf16 ? 2 : 4));
  r.a = q[0];
  if (t == kF32) r.b = q[1];
  return r;
}
// Bytes of a row as it is staged: whole vectors, one more where rows start anywhere.
constexpr int row_bytes(int d, int t) { return ((d + 7) / 8 + (d % 8 != 0)) * (t == kBf16 ? 16 : 32); }
size_t staged_bytes(int d, int st, int yt, bool ds) {
  return (size_t)kWarps * kStages * (row_bytes(d, st) * (1 + ds) + row_bytes(d, yt));
}
template <int ST, int YT, int C, bool Shifted>
__global__ void __launch_bounds__(kWarps * 32, C == 1 ? 5 : C < 4 ? 3 : 2) k_norm_back_rows(const Backward f) {
  extern __shared__ __align__(16) uint8_t room[];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int sb = row_bytes(f.d, ST), yb = row_bytes(f.d, YT), stage = sb * (f.ds ? 2 : 1) + yb;
  constexpr int se = ST == kBf16 ? 2 : 4, ye = YT == kBf16 ? 2 : 4;
  uint8_t* mine = room + wid * kStages * stage;
  const int64_t step = (int64_t)gridDim.x * kWarps, row0 = (int64_t)blockIdx.x * kWarps + wid, total = f.rows * f.d;
  const int shift = Shifted ? (int)(row0 * f.d & 7) : 0;   // a warp's rows start alike: step is a multiple of 8
  const Planes w(reinterpret_cast<float*>(room + (size_t)kWarps * kStages * stage), f.d);
  auto fetch = [&](int64_t row, int turn) {
    if (row < f.rows) {
      uint8_t* to = mine + turn * stage;
      const int64_t at = row * f.d - shift, left = total - at;
      const int n = Shifted ? (f.d + shift + 7) / 8 * 8 : f.d;
      copy_row(to, f.s, at * se, n * se, left * se, lane);
      copy_row(to + sb, f.dy, at * ye, n * ye, left * ye, lane);
      if (f.ds) copy_row(to + sb + yb, f.ds, at * se, n * se, left * se, lane);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float dw[C * 8] = {}, db[C * 8] = {};
  const float inv = 1.f / (float)f.d;
  int turn = 0;
  wait_previous();
  let_next();
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) fetch(row0 + j * step, j);
  if (Shifted) {
    w.fill(f.w, f.wt, f.d);
    __syncthreads();
  }
  float2 next = row0 < f.rows ? __ldg(f.stats + row0) : make_float2(0.f, 0.f);
  for (int64_t row = row0; row < f.rows; row += step, turn = turn + 1 == kStages ? 0 : turn + 1) {
    __syncwarp();                                        // the room's last row has been read by every lane
    fetch(row + (kStages - 1) * step, turn == 0 ? kStages - 1 : turn - 1);
    const float2 mk = next;
    if (row + step < f.rows) next = __ldg(f.stats + row + step);
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
    __syncwarp();
    const uint8_t* at = mine + turn * stage;
    float h[C * 8], g[C * 8], s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int v = lane + i * 32;
      const Span in(v, shift, f.d);
      float *u = h + i * 8, *e = g + i * 8;
      if (in.none()) {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = e[j] = 0.f;
        continue;
      }
      float q[8];
      if (Shifted) {
#pragma unroll
        for (int j = 0; j < 8; ++j) q[j] = w(v, j, shift);
      } else {
        floats(load((Raw<8>*)0, f.w, v * 8, f.wt), f.wt, q);
      }
      floats(staged(at, v * 8, ST), ST, u);
      floats(staged(at + sb, v * 8, YT), YT, e);
      if (Shifted && !in.whole())
#pragma unroll
        for (int j = 0; j < 8; ++j)
          if (j < in.low || j >= in.high) {
            u[j] = mk.x;
            e[j] = q[j] = 0.f;
          }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[j] = (u[j] - mk.x) * mk.y;
        dw[i * 8 + j] = fmaf(e[j], u[j], dw[i * 8 + j]);
        db[i * 8 + j] += e[j];
        e[j] *= q[j];
        s1 += e[j];
        s2 = fmaf(e[j], u[j], s2);
      }
    }
    if (!f.out && !f.other) continue;
    s1 = warp_sum(s1) * inv;
    s2 = warp_sum(s2) * inv;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int v = lane + i * 32;
      const Span in(v, shift, f.d);
      if (in.none()) continue;
      float *u = h + i * 8, *e = g + i * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = mk.y * (e[j] - s1 - u[j] * s2);
      if (f.ds) {
        floats(staged(at + sb + yb, v * 8, ST), ST, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] += u[j];
      }
      const int64_t to = row * f.d - shift + v * 8;
      if (f.out) Shifted ? store_span(f.out, to, ST, e, in) : store<8>(f.out, to, ST, e);
      if (f.other) Shifted ? store_span(f.other, to, 1 - ST, e, in) : store<8>(f.other, to, 1 - ST, e);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (!f.parts) return;
  __syncthreads();
  // The columns' sums [2][8][32 C + 1], a vector's columns in planes; the block's warps add theirs one after another. Where rows start
  // anywhere, a warp's columns are not another's: by their own places [2][d] then.
  float* sums = reinterpret_cast<float*>(room);
  if (Shifted) {
    for (int c = threadIdx.x; c < 2 * f.d; c += blockDim.x) sums[c] = 0.f;
    __syncthreads();
  }
  for (int k = 0; k < kWarps; ++k) {
    if (wid == k)
#pragma unroll
      for (int i = 0; i < C * 8; ++i) {
        if (Shifted) {
          const int c = (lane + i / 8 * 32) * 8 - shift + i % 8;
          if (c >= 0 && c < f.d) {
            sums[c] += dw[i];
            sums[f.d + c] += db[i];
          }
        } else {
          sums[i * 32 + lane] = k ? sums[i * 32 + lane] + dw[i] : dw[i];
          sums[(C * 8 + i) * 32 + lane] = k ? sums[(C * 8 + i) * 32 + lane] + db[i] : db[i];
        }
      }
    __syncthreads();
  }
  float* part = f.parts + (int64_t)blockIdx.x * 2 * f.d;
  for (int c = threadIdx.x; c < f.d; c += blockDim.x) {
    const int q = c / 8, own = Shifted ? c : (q / 32 * 8 + c % 8) * 32 + q % 32;       // where column c's thread put it
    part[c] = sums[own];
    part[f.d + c] = sums[own + (Shifted ? f.d : C * 256)];
  }
}

// out[c] = the sum of the parts' [..][c] in order, c < n of 2 d: block = 32 columns x 32 warps.
__global__ void __launch_bounds__(1024) k_norm_sums(int parts, int d, const float* __restrict__ sums, void* dw, void* db,
                                                    int wt) {
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
  wait_previous();
  let_next();
  float s = 0.f;
  if (c < 2 * d)
#pragma unroll 8
    for (int k = wid; k < parts; k += 32) s += sums[(int64_t)k * 2 * d + c];
  sh[wid][lane] = s;
  __syncthreads();
  if (wid || c >= 2 * d) return;
  s = 0.f;
#pragma unroll
  for (int w = 0; w < 32; ++w) s += sh[w][lane];
  void* out = c < d ? dw : db;
  if (out) store<1>(out, c < d ? c : c - d, wt, &s);
}

int sms() {
  static std::atomic<int> n{0};
  int v = n.load(std::memory_order_relaxed);
  if (v == 0) {
    int dev = 0;
    cudaGetDevice(&dev);
    if (cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || v <= 0) v = 148;
    n.store(v, std::memory_order_relaxed);
  }
  return v;
}

// Blocks of the backward pass: as many as stay on the SMs at once, each with 2 d sums of its own; a multiple of 8 where rows start
// anywhere, so that a warp's or block's own rows start alike.
int64_t blocks_back(int64_t rows, int d) {
  const int per = d <= 1024 ? kWarps : 1, stay = d <= 256 ? 5 : d <= 768 ? 3 : d <= 4096 ? 2 : 1;
  const int64_t n = std::max<int64_t>(1, std::min<int64_t>((int64_t)sms() * stay, (rows + per - 1) / per));
  return d % 8 ? (n + 7) / 8 * 8 : n;
}

template <int V, int XT, int RT, int C, int T> int run(const Forward& f, cudaStream_t s) {
  // few rows: a warp for a block, so that they spread over the SMs
  const int threads = T > 32 ? T : f.rows <= 4 * sms() ? 32 : threads_of(T), per = T <= 32 ? threads / T : 1;
  return launch_next(k_norm<V, XT, RT, C, T>, (f.rows + per - 1) / per, threads, 0, s, f);
}
template <int XT, int RT> int widths(const Forward& f, cudaStream_t s) {
  if (f.d <= 128) return run<8, XT, RT, 1, 16>(f, s);
  if (f.d <= 256) return run<8, XT, RT, 1, 32>(f, s);
  if (f.d <= 512) return run<8, XT, RT, 2, 32>(f, s);
  if (f.d <= 768) return run<8, XT, RT, 3, 32>(f, s);
  if (f.d <= 1024) return run<8, XT, RT, 4, 32>(f, s);
  if (f.d <= 2048) return run<8, XT, RT, 1, 256>(f, s);
  if (f.d <= 4096) return run<8, XT, RT, 2, 256>(f, s);
  if (f.d <= 8192) return run<8, XT, RT, 2, 512>(f, s);
  return run<8, XT, RT, 4, 512>(f, s);
}
// Value by value, for tensors that are not 16-byte aligned, and the six odd widths below kMaxD.
template <class Args> int singles(const Args& f, cudaStream_t s) {
  if (f.d <= 256) return run<1, -1, -1, 8, 32>(f, s);
  if (f.d <= 1024) return run<1, -1, -1, 32, 32>(f, s);
  if (f.d <= 8192) return run<1, -1, -1, 32, 256>(f, s);
  return run<1, -1, -1, 32, 512>(f, s);
}

// A kernel whose dynamic shared memory may pass 48 KB: `most` is what any call asks for.
template <class Kernel, class Args>
int launch(Kernel kernel, std::atomic<uint64_t>& ready, size_t most, int64_t blocks, int threads, size_t bytes, const Args& f,
           cudaStream_t s) {
  if (most > 48 << 10) {                                 // `ready`: devices that know it
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return ASRN_ERR_CUDA;
    if (dev > 63 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess)
        return ASRN_ERR_CUDA;
      if (dev <= 63) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
  }
  return launch_next(kernel, blocks, threads, bytes, s, f);
}

template <int XT, int RT, int C, int T> int run_shifted(const Forward& f, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  constexpr int per = threads_of(T) / T;
  const int64_t most = (int64_t)sms() * stay_shifted(C, T);
  return launch(k_norm_shifted<XT, RT, C, T>, ready, (size_t)2 * Planes::floats(T * C * 8) * 4,
                std::min(most, (f.rows + per - 1) / per), threads_of(T), (size_t)2 * Planes::floats(f.d) * 4, f, s);
}
template <int XT, int RT> int shifted(const Forward& f, cudaStream_t s) {
  const int n = f.d + 7;                                 // values from the last boundary before the row to its end, at most
  if (n <= 128) return run_shifted<XT, RT, 1, 16>(f, s);
  if (n <= 256) return run_shifted<XT, RT, 1, 32>(f, s);
  if (n <= 512) return run_shifted<XT, RT, 2, 32>(f, s);
  if (n <= 768) return run_shifted<XT, RT, 3, 32>(f, s);
  if (n <= 1024) return run_shifted<XT, RT, 4, 32>(f, s);
  if (n <= 2048) return run_shifted<XT, RT, 1, 256>(f, s);
  if (n <= 4096) return run_shifted<XT, RT, 2, 256>(f, s);
  if (n <= 8192) return run_shifted<XT, RT, 2, 512>(f, s);
  return n <= kMaxD ? run_shifted<XT, RT, 4, 512>(f, s) : singles(f, s);
}

template <int V, int ST, int YT, int C, int T> int run(const Backward& f, cudaStream_t s) {
  return launch_next(k_norm_back<V, ST, YT, C, T>, blocks_back(f.rows, f.d), threads_of(T), 0, s, f);
}
template <int ST, int YT, int C, bool Shifted> int run_rows(const Backward& f, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  constexpr int d = C * 256 - Shifted;                   // the largest
  constexpr size_t sums = std::max<size_t>(C * 8 * 32 * 2 * 4, 2 * d * 4);
  constexpr size_t most = kWarps * kStages * (row_bytes(d, ST) * 2 + row_bytes(d, YT)) + 8 * (d / 8 + 3) * 4 + sums;
  const size_t bytes = staged_bytes(f.d, ST, YT, f.ds != nullptr) + (Shifted ? Planes::floats(f.d) * 4 : 0);
  return launch(k_norm_back_rows<ST, YT, C, Shifted>, ready, most, blocks_back(f.rows, f.d), kWarps * 32,
                std::max<size_t>(bytes, f.parts ? sums : 0), f, s);
}
template <int ST, int YT, int C, int T> int run_shifted(const Backward& f, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};
  return launch(k_norm_back_shifted<ST, YT, C, T>, ready, (size_t)Planes::floats(T * C * 8) * 4, blocks_back(f.rows, f.d), T,
                (size_t)Planes::floats(f.d) * 4, f, s);
}
template <int ST, int YT> int widths(const Backward& f, cudaStream_t s) {
  if (f.d <= 256) return run_rows<ST, YT, 1, false>(f, s);
  if (f.d <= 512) return run_rows<ST, YT, 2, false>(f, s);
  if (f.d <= 768) return run_rows<ST, YT, 3, false>(f, s);
  if (f.d <= 1024) return run_rows<ST, YT, 4, false>(f, s);
  if (f.d <= 2048) return run<8, ST, YT, 1, 256>(f, s);
  if (f.d <= 4096) return run<8, ST, YT, 2, 256>(f, s);
  if (f.d <= 8192) return run<8, ST, YT, 2, 512>(f, s);
  return run<8, ST, YT, 4, 512>(f, s);
}
template <int ST, int YT> int shifted(const Backward& f, cudaStream_t s) {
  const int n = f.d + 7;
  if (n <= 256) return run_rows<ST, YT, 1, true>(f, s);
  if (n <= 512) return run_rows<ST, YT, 2, true>(f, s);
  if (n <= 768) return run_rows<ST, YT, 3, true>(f, s);
  if (n <= 1024) return run_rows<ST, YT, 4, true>(f, s);
  if (n <= 2048) return run_shifted<ST, YT, 1, 256>(f, s);
  if (n <= 4096) return run_shifted<ST, YT, 2, 256>(f, s);
  if (n <= 8192) return run_shifted<ST, YT, 2, 512>(f, s);
  return n <= kMaxD ? run_shifted<ST, YT, 4, 512>(f, s) : singles(f, s);
}

int check_norm(int64_t rows, int32_t d) {
  if (rows < 0 || d < 1) return ASRN_ERR_ARG;
  if (d > kMaxD || rows > ((int64_t)1 << 31) - 1) return ASRN_ERR_UNSUPPORTED;
  return ASRN_OK;
}
bool type_ok(int t) { return t == kF32 || t == kBf16; }
bool aligned(std::initializer_list<const void*> ps) {
  uintptr_t all = 0;
  for (const void* p : ps) all |= (uintptr_t)p;
  return all % 16 == 0;
}
// And is a multiple of its type's size.
bool placed(const void* p, int t) { return (uintptr_t)p % (t == kBf16 ? 2 : 4) == 0; }

}  // namespace
}  // namespace asrn

extern "C" {

int asrn_test_norm_reads(int64_t rows, int32_t d, int64_t row, int64_t* from, int64_t* to) {
  if (!from || !to || d < 1 || row < 0 || row >= rows) return ASRN_ERR_ARG;
  const asrn::RowAt own(row, rows, d);
  const int64_t total = rows * d, end = own.at + 8 * (int64_t)(own.last + 1);
  *from = own.at;
  *to = own.inside ? end : std::min(end, total);         // load_to reads no value past the end
  return ASRN_OK;
}

int asrn_layer_norm(int64_t rows, int32_t d, const void* x, int32_t x_type, const void* residual, int32_t res_type,
                    const void* weight, const void* bias, int32_t w_type, float eps, void* sum, void* y, int32_t y_type,
                    float* stats, void* stream) {
  using namespace asrn;
  int st = check_norm(rows, d);
  if (st) return st;
  if (!type_ok(x_type) || !type_ok(w_type) || !type_ok(y_type) || (residual && !type_ok(res_type)) || !(eps >= 0.f))
    return ASRN_ERR_ARG;
  if (rows == 0) return ASRN_OK;
  if (!x || !weight || !y || (residual && !sum) || !placed(x, x_type) || !placed(y, y_type) || !placed(weight, w_type) ||
      !placed(bias, w_type) || (uintptr_t)stats % 8 || (residual && (!placed(residual, res_type) || !placed(sum, res_type))))
    return ASRN_ERR_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  const Forward f{rows, d, x, residual, weight, bias, x_type, residual ? res_type : kNone, w_type, y_type, eps, sum, y,
                  reinterpret_cast<float2*>(stats)};
  if (!aligned({x, residual, weight, bias, residual ? sum : nullptr, y})) return singles(f, s);
  auto with = [&](auto xt, auto rt) {
    constexpr int a = decltype(xt)::value, b = decltype(rt)::value;
    return d % 8 ? shifted<a, b>(f, s) : widths<a, b>(f, s);
  };
  if (x_type == kF32) return f.rt == kNone ? with(F32{}, None{}) : f.rt == kF32 ? with(F32{}, F32{}) : with(F32{}, Bf16{});
  return f.rt == kNone ? with(Bf16{}, None{}) : f.rt == kF32 ? with(Bf16{}, F32{}) : with(Bf16{}, Bf16{});
}

size_t asrn_layer_norm_workspace_bytes(int64_t rows, int32_t d) {
  if (asrn::check_norm(rows, d) || rows == 0) return 0;
  return (size_t)asrn::blocks_back(rows, d) * 2 * d * 4;
}

int asrn_layer_norm_backward(int64_t rows, int32_t d, const void* s_in, int32_t s_type, const float* stats, const void* dy,
                             int32_t y_type, const void* ds, const void* weight, int32_t w_type, void* out, void* other,
                             void* dw, void* db, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace asrn;
  int st = check_norm(rows, d);
  if (st) return st;
  if (!type_ok(s_type) || !type_ok(y_type) || !type_ok(w_type)) return ASRN_ERR_ARG;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows == 0) {
    const size_t bytes = (size_t)d * (w_type == kBf16 ? 2 : 4);
    if ((dw && cudaMemsetAsync(dw, 0, bytes, s) != cudaSuccess) || (db && cudaMemsetAsync(db, 0, bytes, s) != cudaSuccess))
      return ASRN_ERR_CUDA;
    return ASRN_OK;
  }
  if (!s_in || !stats || !dy || !weight || !placed(s_in, s_type) || !placed(dy, y_type) || !placed(ds, s_type) ||
      !placed(weight, w_type) || !placed(out, s_type) || !placed(other, 1 - s_type) || !placed(dw, w_type) ||
      !placed(db, w_type) || (uintptr_t)stats % 8)
    return ASRN_ERR_ARG;
  const bool sums = dw || db;
  if (sums && (!workspace || (uintptr_t)workspace % 256 || workspace_bytes < asrn_layer_norm_workspace_bytes(rows, d)))
    return ASRN_ERR_WORKSPACE;
  const Backward f{rows, d, s_in, dy, ds, weight, s_type, y_type, w_type, reinterpret_cast<const float2*>(stats), out, other,
                   sums ? reinterpret_cast<float*>(workspace) : nullptr};
  if (!sums && !out && !other) return ASRN_OK;
  auto with = [&](auto a, auto b) {
    constexpr int x = decltype(a)::value, y = decltype(b)::value;
    return d % 8 ? shifted<x, y>(f, s) : widths<x, y>(f, s);
  };
  if (!aligned({s_in, dy, ds, weight, out, other}))
    st = singles(f, s);
  else if (s_type == kF32)
    st = y_type == kF32 ? with(F32{}, F32{}) : with(F32{}, Bf16{});
  else
    st = y_type == kF32 ? with(Bf16{}, F32{}) : with(Bf16{}, Bf16{});
  if (st || !sums) return st;
  return launch_next(k_norm_sums, (2 * d + 31) / 32, 1024, 0, s, (int)blocks_back(rows, d), d, f.parts, dw, db, w_type);
}

}  // extern "C"
