// Layer norm of rows of d values, with the residual sum before it, forward and backward:
//   s = x + r (rounded to r's type, handed on),  m = mean s,  v = mean (s - m)^2,  k = 1 / sqrt(v + eps)
//   h = (s - m) k,  y = h w + b
//   g = dy w,  ds' = k (g - mean g - h mean(g h)) + ds,  dx = dr = ds',  dw = sum over the rows of dy h,  db = sum of dy
// Sums in fp32, the variance from the differences (a second walk over registers, none over memory). Kept for the backward pass:
// s (or x) and each row's m and k in fp32.
//
// Bound by memory: each row is read once into registers and written once. A warp holds a row of up to 1024 values, a block
// of 256 or 512 threads a longer one, eight values (16 or 32 bytes) a load; widths that are no multiple of 8, and rows that are not
// 16-byte aligned, go value by value. The backward pass's blocks stay for many rows with their columns' sums of dy h and dy
// in registers; a block's sums go to fp32 parts that k_norm_sums adds up in order.
#include "common.cuh"
#include "layout.h"

#include <algorithm>
#include <atomic>

namespace asrn {

namespace {

constexpr int kF32 = 0, kBf16 = 1, kNone = 2;            // types of the C interface
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

// The sum over a row's T threads: a warp's, or a whole block's (each sum with its own room, so one barrier serves).
template <int T> ASRN_DEV float row_sum(float v, float* room) {
  v = warp_sum(v);
  if constexpr (T == 32) return v;
  if ((threadIdx.x & 31) == 0) room[threadIdx.x >> 5] = v;
  __syncthreads();
  float s = 0.f;
#pragma unroll
  for (int i = 0; i < T / 32; ++i) s += room[i];
  return s;
}

constexpr int threads_of(int T) { return T == 32 ? 128 : T; }

// V values a load, C loads a thread, T threads a row; types XT, RT known at compile time unless they are -1.
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
  const int xt = XT < 0 ? f.xt : XT, rt = RT < 0 ? f.rt : RT;
  const int tid = T == 32 ? threadIdx.x & 31 : threadIdx.x;
  const int64_t row = T == 32 ? (int64_t)blockIdx.x * (blockDim.x / 32) + (threadIdx.x >> 5) : blockIdx.x;
  if (row >= f.rows) return;
  const int64_t at = row * f.d;
  Raw<V> rx[C], rr[C];
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = (tid + i * T) * V;
    if (c < f.d) {
      rx[i] = load((Raw<V>*)0, f.x, at + c, xt);
      if (rt != kNone) rr[i] = load((Raw<V>*)0, f.res, at + c, rt);
    }
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
      store<V>(f.sum, at + c, rt, u);
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
  if (f.stats && tid == 0) f.stats[row] = make_float2(m, k);
#pragma unroll
  for (int i = 0; i < C; ++i) {
    const int c = (tid + i * T) * V;
    if (c >= f.d) continue;
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
  const int st = ST < 0 ? f.st : ST, yt = YT < 0 ? f.yt : YT;
  const int tid = T == 32 ? threadIdx.x & 31 : threadIdx.x, wid = T == 32 ? threadIdx.x >> 5 : 0;
  float dw[C * V] = {}, db[C * V] = {};
  const float inv = 1.f / (float)f.d;
  int turn = 0;
  for (int64_t row = (int64_t)blockIdx.x * kRows + wid; row < f.rows; row += (int64_t)gridDim.x * kRows, turn ^= 1) {
    const int64_t at = row * f.d;
    Raw<V> rs[C], ry[C], rd[C];
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = (tid + i * T) * V;
      if (c < f.d) {
        rs[i] = load((Raw<V>*)0, f.s, at + c, st);
        ry[i] = load((Raw<V>*)0, f.dy, at + c, yt);
        if (f.ds) rd[i] = load((Raw<V>*)0, f.ds, at + c, st);
      }
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

// The same for rows that a warp holds, eight values a load (d <= 1024): each warp's next row comes to shared memory by
// asynchronous copies while it works on the one before, which costs no registers beside the columns' sums.
constexpr int kWarps = 4, kStages = 2;
ASRN_DEV void copy_row(uint8_t* to, const void* from, int64_t at, int bytes, int lane) {
  const char* p = reinterpret_cast<const char*>(from) + at;
  for (int b = lane * 16; b < bytes; b += 512)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"((uint32_t)__cvta_generic_to_shared(to + b)), "l"(p + b)
                 : "memory");
}
ASRN_DEV Raw<8> staged(const uint8_t* p, int c, int t) {
  Raw<8> r;
  const uint4* q = reinterpret_cast<const uint4*>(p + c * (t == kBf16 ? 2 : 4));
  r.a = q[0];
  if (t == kF32) r.b = q[1];
  return r;
}
constexpr int row_bytes(int d, int t) { return d * (t == kBf16 ? 2 : 4); }
size_t staged_bytes(int d, int st, int yt, bool ds) {
  return (size_t)kWarps * kStages * (row_bytes(d, st) * (1 + ds) + row_bytes(d, yt));
}
template <int ST, int YT, int C>
__global__ void __launch_bounds__(kWarps * 32, C == 1 ? 5 : C < 4 ? 3 : 2) k_norm_back_rows(const Backward f) {
  extern __shared__ __align__(16) uint8_t room[];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5;
  const int sb = row_bytes(f.d, ST), yb = row_bytes(f.d, YT), stage = sb * (f.ds ? 2 : 1) + yb;
  uint8_t* mine = room + wid * kStages * stage;
  auto fetch = [&](int64_t row, int turn) {
    if (row < f.rows) {
      uint8_t* to = mine + turn * stage;
      copy_row(to, f.s, row * sb, sb, lane);
      copy_row(to + sb, f.dy, row * yb, yb, lane);
      if (f.ds) copy_row(to + sb + yb, f.ds, row * sb, sb, lane);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  float dw[C * 8] = {}, db[C * 8] = {};
  const float inv = 1.f / (float)f.d;
  const int64_t step = (int64_t)gridDim.x * kWarps, row0 = (int64_t)blockIdx.x * kWarps + wid;
  int turn = 0;
#pragma unroll
  for (int j = 0; j < kStages - 1; ++j) fetch(row0 + j * step, j);
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
      const int c = (lane + i * 32) * 8;
      float *u = h + i * 8, *e = g + i * 8;
      if (c >= f.d) {
#pragma unroll
        for (int j = 0; j < 8; ++j) u[j] = e[j] = 0.f;
        continue;
      }
      float w[8];
      floats(load((Raw<8>*)0, f.w, c, f.wt), f.wt, w);
      floats(staged(at, c, ST), ST, u);
      floats(staged(at + sb, c, YT), YT, e);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        u[j] = (u[j] - mk.x) * mk.y;
        dw[i * 8 + j] = fmaf(e[j], u[j], dw[i * 8 + j]);
        db[i * 8 + j] += e[j];
        e[j] *= w[j];
        s1 += e[j];
        s2 = fmaf(e[j], u[j], s2);
      }
    }
    if (!f.out && !f.other) continue;
    s1 = warp_sum(s1) * inv;
    s2 = warp_sum(s2) * inv;
#pragma unroll
    for (int i = 0; i < C; ++i) {
      const int c = (lane + i * 32) * 8;
      if (c >= f.d) continue;
      float *u = h + i * 8, *e = g + i * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) e[j] = mk.y * (e[j] - s1 - u[j] * s2);
      if (f.ds) {
        floats(staged(at + sb + yb, c, ST), ST, u);
#pragma unroll
        for (int j = 0; j < 8; ++j) e[j] += u[j];
      }
      if (f.out) store<8>(f.out, row * f.d + c, ST, e);
      if (f.other) store<8>(f.other, row * f.d + c, 1 - ST, e);
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  if (!f.parts) return;
  __syncthreads();
  float* sums = reinterpret_cast<float*>(room);          // [2][C 8][32]
  for (int w = 0; w < kWarps; ++w) {                     // the block's warps, one after another
    if (wid == w)
#pragma unroll
      for (int i = 0; i < C * 8; ++i) {
        sums[i * 32 + lane] = w ? sums[i * 32 + lane] + dw[i] : dw[i];
        sums[(C * 8 + i) * 32 + lane] = w ? sums[(C * 8 + i) * 32 + lane] + db[i] : db[i];
      }
    __syncthreads();
  }
  float* part = f.parts + (int64_t)blockIdx.x * 2 * f.d;
  for (int c = threadIdx.x; c < f.d; c += blockDim.x) {
    const int q = c / 8, own = (q / 32 * 8 + c % 8) * 32 + q % 32;       // where column c's thread put it
    part[c] = sums[own];
    part[f.d + c] = sums[C * 256 + own];
  }
}

// out[c] = the sum of the parts' [..][c] in order, c < n of 2 d: block = 32 columns x 32 warps.
__global__ void __launch_bounds__(1024) k_norm_sums(int parts, int d, const float* __restrict__ sums, void* dw, void* db,
                                                    int wt) {
  __shared__ float sh[32][33];
  const int lane = threadIdx.x & 31, wid = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
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

// Blocks of the backward pass: as many as stay on the SMs at once, each with 2 d sums of its own.
int64_t blocks_back(int64_t rows, int d) {
  const int per = d <= 1024 ? kWarps : 1, stay = d <= 256 ? 5 : d <= 768 ? 3 : d <= 4096 ? 2 : 1;
  return std::max<int64_t>(1, std::min<int64_t>((int64_t)sms() * stay, (rows + per - 1) / per));
}

int launched() { return cudaGetLastError() == cudaSuccess ? ASRN_OK : ASRN_ERR_CUDA; }

template <int V, int XT, int RT, int C, int T> int run(const Forward& f, cudaStream_t s) {
  // few rows: a warp for a block, so that they spread over the SMs
  const int threads = T > 32 ? T : f.rows <= 4 * sms() ? 32 : threads_of(T), per = T == 32 ? threads / 32 : 1;
  k_norm<V, XT, RT, C, T><<<(unsigned)((f.rows + per - 1) / per), threads, 0, s>>>(f);
  return launched();
}
template <int XT, int RT> int widths(const Forward& f, cudaStream_t s) {
  if (f.d <= 256) return run<8, XT, RT, 1, 32>(f, s);
  if (f.d <= 512) return run<8, XT, RT, 2, 32>(f, s);
  if (f.d <= 768) return run<8, XT, RT, 3, 32>(f, s);
  if (f.d <= 1024) return run<8, XT, RT, 4, 32>(f, s);
  if (f.d <= 2048) return run<8, XT, RT, 1, 256>(f, s);
  if (f.d <= 4096) return run<8, XT, RT, 2, 256>(f, s);
  if (f.d <= 8192) return run<8, XT, RT, 2, 512>(f, s);
  return run<8, XT, RT, 4, 512>(f, s);
}
template <class Args> int singles(const Args& f, cudaStream_t s) {
  if (f.d <= 128) return run<1, -1, -1, 4, 32>(f, s);
  if (f.d <= 256) return run<1, -1, -1, 8, 32>(f, s);
  if (f.d <= 384) return run<1, -1, -1, 12, 32>(f, s);
  if (f.d <= 512) return run<1, -1, -1, 16, 32>(f, s);
  if (f.d <= 768) return run<1, -1, -1, 24, 32>(f, s);
  if (f.d <= 1024) return run<1, -1, -1, 32, 32>(f, s);
  if (f.d <= 2048) return run<1, -1, -1, 8, 256>(f, s);
  if (f.d <= 4096) return run<1, -1, -1, 16, 256>(f, s);
  if (f.d <= 8192) return run<1, -1, -1, 16, 512>(f, s);
  return run<1, -1, -1, 32, 512>(f, s);
}

template <int V, int ST, int YT, int C, int T> int run(const Backward& f, cudaStream_t s) {
  k_norm_back<V, ST, YT, C, T><<<(unsigned)blocks_back(f.rows, f.d), threads_of(T), 0, s>>>(f);
  return launched();
}
template <int ST, int YT, int C> int run_rows(const Backward& f, cudaStream_t s) {
  auto kernel = k_norm_back_rows<ST, YT, C>;
  constexpr size_t most = (size_t)kWarps * kStages * (row_bytes(C * 256, ST) * 2 + row_bytes(C * 256, YT));
  static std::atomic<uint64_t> ready{0};                 // devices that know the kernel's shared memory
  int dev = 0;
  if (most > 48 << 10) {
    if (cudaGetDevice(&dev) != cudaSuccess) return ASRN_ERR_CUDA;
    if (dev > 63 || !(ready.load(std::memory_order_acquire) >> dev & 1)) {
      if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)most) != cudaSuccess)
        return ASRN_ERR_CUDA;
      if (dev <= 63) ready.fetch_or(1ull << dev, std::memory_order_release);
    }
  }
  const size_t bytes = std::max<size_t>(staged_bytes(f.d, ST, YT, f.ds != nullptr), f.parts ? C * 8 * 32 * 2 * 4 : 0);
  kernel<<<(unsigned)blocks_back(f.rows, f.d), kWarps * 32, bytes, s>>>(f);
  return launched();
}
template <int ST, int YT> int widths(const Backward& f, cudaStream_t s) {
  if (f.d <= 256) return run_rows<ST, YT, 1>(f, s);
  if (f.d <= 512) return run_rows<ST, YT, 2>(f, s);
  if (f.d <= 768) return run_rows<ST, YT, 3>(f, s);
  if (f.d <= 1024) return run_rows<ST, YT, 4>(f, s);
  if (f.d <= 2048) return run<8, ST, YT, 1, 256>(f, s);
  if (f.d <= 4096) return run<8, ST, YT, 2, 256>(f, s);
  if (f.d <= 8192) return run<8, ST, YT, 2, 512>(f, s);
  return run<8, ST, YT, 4, 512>(f, s);
}

int check_norm(int64_t rows, int32_t d) {
  if (rows < 0 || d < 1) return ASRN_ERR_ARG;
  if (d > kMaxD || rows > ((int64_t)1 << 31) - 1) return ASRN_ERR_UNSUPPORTED;
  return ASRN_OK;
}
bool type_ok(int t) { return t == kF32 || t == kBf16; }
// Every tensor's address allows 16-byte loads of rows of d.
bool vectors(int d, std::initializer_list<const void*> ps) {
  uintptr_t all = 0;
  for (const void* p : ps) all |= (uintptr_t)p;
  return d % 8 == 0 && all % 16 == 0;
}
// And is a multiple of its type's size.
bool placed(const void* p, int t) { return (uintptr_t)p % (t == kBf16 ? 2 : 4) == 0; }

}  // namespace
}  // namespace asrn

extern "C" {

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
  if (!vectors(d, {x, residual, weight, bias, residual ? sum : nullptr, y})) return singles(f, s);
  if (x_type == kF32)
    return f.rt == kNone ? widths<kF32, kNone>(f, s) : f.rt == kF32 ? widths<kF32, kF32>(f, s) : widths<kF32, kBf16>(f, s);
  return f.rt == kNone ? widths<kBf16, kNone>(f, s) : f.rt == kF32 ? widths<kBf16, kF32>(f, s) : widths<kBf16, kBf16>(f, s);
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
  if (!vectors(d, {s_in, dy, ds, weight, out, other}))
    st = singles(f, s);
  else if (s_type == kF32)
    st = y_type == kF32 ? widths<kF32, kF32>(f, s) : widths<kF32, kBf16>(f, s);
  else
    st = y_type == kF32 ? widths<kBf16, kF32>(f, s) : widths<kBf16, kBf16>(f, s);
  if (st || !sums) return st;
  k_norm_sums<<<(unsigned)((2 * d + 31) / 32), 1024, 0, s>>>((int)blocks_back(rows, d), d, f.parts, dw, db, w_type);
  return launched();
}

}  // extern "C"
