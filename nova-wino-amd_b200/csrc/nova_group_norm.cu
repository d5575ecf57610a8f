// Group normalisation with its activation on channels-last activations.
//
//   u = x + shift[b][c]                       (shift optional)
//   m, v = mean and variance of u over the pixels and channels of (b, group)
//   n = (u - m) / sqrt(v + eps),  z = w n + beta,  y = act(z)
//
// and its gradient
//
//   dz = dy act'(z),  A = mean(w dz),  D = mean(w dz n)   over (b, group)
//   dx = (w dz - A - n D) / sqrt(v + eps)
//   dw = sum dz n,  dbeta = sum dz  (over b and pixels),  dshift = sum dx (over pixels)
//
// x is [B][HW][C] with a pixel stride and a batch stride of its own; y and dx
// are dense.  No reference counterpart: the reference's UNet callers leave the
// norm to the host framework (benchmarks/bench_sd_unet.py:38-109).
//
// Two forms.  Resident: one launch, x read once; a cluster of blocks keeps a sample's
// channel block in registers, of FP32 at least half of it and the rest in L2.
// Streaming: a pass that sums, one that joins, one that writes; for what does not fit
// the SMs at once.  make_slab has the rule.
//
// Statistics.  The resident form takes the mean of its registers, then the squared
// deviations from it; a streaming thread keeps sums relative to the first value it
// sees: a mean far from zero costs the statistics no digits.  (The passes fold it into an
// offset, rounded once at its own size: as a subtraction of the rounded mean would be.)
// Parts are joined as means and squared deviations, a group's and the samples' in 64
// bits.  Every sum has a fixed order: results repeat bit for bit.
//
// What bounds it.  8 x 960 x 128 x 128 FP16 forward, 504 MB at least: 156 us, 49 % of the
// measured copy bandwidth (the summing pass 53 us, 4.8 TB/s; the writing pass 101 us,
// which reads x again); the vector instructions of conversion and activation, 15 for an
// element, keep the issue slots half busy and do not all hide behind the loads.
// 1 x 1280 x 8 x 8: 5.2 us, the launch and three exchanges.
#include <algorithm>
#include <string>

#include "../../include/nova_winograd.h"
#include "nova_unet_ops.h"

namespace nova {
namespace gn {

using namespace unet;

enum Act : int { kNone = 0, kSilu = 1 };

struct Args {
  const void* x;
  const void* dy;
  const void* w;      // [C] or null
  const void* beta;   // [C] or null
  const void* shift;  // [B][C] or null
  void* y;            // y, or dx in the gradient
  long long xb, xp;   // batch and pixel stride of x, in elements
  long long yb, yp;   // of dy (the outputs are dense)
  int B, HW, C, G, cpg;
  int wtype, stype;
  float eps;
};

// How the grid walks one tensor: a block takes TX vector columns, TY pixels at a time;
// a tile is U times TY pixels, U vectors that every thread has on their way together,
// and block `chunk` of a sample has `per` pixels in a row, a multiple of TY.
struct Walk {
  int cv;      // vector columns of a pixel
  int ncb;     // column blocks
  int tx, ty;  // threads
  int tile;    // pixels of a tile
  int per, nchunk;
  int cell;    // channels that share a part of the statistics: a group's, or one
};

constexpr int kThreads = 256;
// Vectors that a streaming thread has on their way: with the blocks that fit an SM,
// the 60 to 90 KB in flight that its share of the bandwidth takes.
constexpr int kAhead = 8;
constexpr int kBlocksForward = 3, kBlocksGrad = 2;  // of a streaming kernel on an SM

// Channels are worked on in pairs (the paired 32-bit instructions halve the count),
// or singly where a thread holds one.
__device__ __forceinline__ float2 add(float2 x, float2 y) { return __fadd2_rn(x, y); }
__device__ __forceinline__ float2 mul(float2 x, float2 y) { return __fmul2_rn(x, y); }
__device__ __forceinline__ float2 fma(float2 x, float2 y, float2 z) { return __ffma2_rn(x, y, z); }
__device__ __forceinline__ float add(float x, float y) { return x + y; }
__device__ __forceinline__ float mul(float x, float y) { return x * y; }
__device__ __forceinline__ float fma(float x, float y, float z) { return fmaf(x, y, z); }
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename F>
__device__ __forceinline__ F splat(float x);
template <>
__device__ __forceinline__ float splat<float>(float x) { return x; }
template <>
__device__ __forceinline__ float2 splat<float2>(float x) { return make_float2(x, x); }

// 1 / (1 + e^-z).  A pair shares one reciprocal, 1 / (d e) = (1/d) (1/e): the special
// function unit, at 16 results a clock and SM, is the nearest bound of these passes
// after memory, and this takes a quarter of its work away.  The exponent stops at 2^63
// to keep the product finite: below z = -43 the sigmoid is 2^-63 instead of less.
__device__ __forceinline__ float sigmoid(float z) { return rcp(ex2(z * -1.4426950408889634f) + 1.f); }
__device__ __forceinline__ float2 sigmoid(float2 z) {
  const float2 t = mul(z, splat<float2>(-1.4426950408889634f));
  const float2 d = add(make_float2(ex2(fminf(t.x, 63.f)), ex2(fminf(t.y, 63.f))), splat<float2>(1.f));
  const float r = rcp(d.x * d.y);
  return mul(make_float2(r, r), make_float2(d.y, d.x));
}
template <int ACT, typename F>
__device__ __forceinline__ F act(F z) {
  return ACT == kSilu ? mul(z, sigmoid(z)) : z;
}
// dy act'(z); silu: s (1 + z (1 - s)) = s + (z s) (1 - s).
template <int ACT, typename F>
__device__ __forceinline__ F act_grad(F dy, F z) {
  if (ACT != kSilu) return dy;
  const F s = sigmoid(z), zs = mul(z, s);
  return mul(dy, fma(zs, fma(s, splat<F>(-1.f), splat<F>(1.f)), s));
}

// Channels j W .. j W + W - 1 of a vector, and of an array in shared memory or
// registers.
template <typename T, int V>
struct Lanes {
  static constexpr int W = 2;
  using F = float2;
  static __device__ __forceinline__ float2 get(const Pack<T, V>& p, int j) {
    return make_float2(to_f32(p.e[2 * j]), to_f32(p.e[2 * j + 1]));
  }
  static __device__ __forceinline__ void set(Pack<T, V>& p, int j, float2 f) {
    p.e[2 * j] = from_f32<T>(f.x);
    p.e[2 * j + 1] = from_f32<T>(f.y);
  }
  static __device__ __forceinline__ float2 at(const float* a, int j) {
    return make_float2(a[2 * j], a[2 * j + 1]);
  }
  static __device__ __forceinline__ void put(float* a, int j, float2 f) {
    a[2 * j] = f.x;
    a[2 * j + 1] = f.y;
  }
};
template <typename T>
struct Lanes<T, 1> {
  static constexpr int W = 1;
  using F = float;
  static __device__ __forceinline__ float get(const Pack<T, 1>& p, int) { return to_f32(p.e[0]); }
  static __device__ __forceinline__ void set(Pack<T, 1>& p, int, float f) {
    p.e[0] = from_f32<T>(f);
  }
  static __device__ __forceinline__ float at(const float* a, int) { return a[0]; }
  static __device__ __forceinline__ void put(float* a, int, float f) { a[0] = f; }
};

// Joins (nb, mb, qb) into (na, ma, qa): counts, means, squared deviations.
__device__ __forceinline__ void join(float& na, float& ma, float& qa, float nb, float mb,
                                     float qb) {
  if (nb == 0.f) return;
  const float n = na + nb, d = mb - ma, f = nb / n;
  ma = fmaf(d, f, ma);
  qa += qb + d * d * na * f;
  na = n;
}

struct Place {
  int b, chunk, tx, ty, col;
  bool active;
};
__device__ __forceinline__ Place place(const Args& a, const Walk& k) {
  Place q;
  unsigned id = blockIdx.x;
  const int cb = id % k.ncb;
  id /= k.ncb;
  q.chunk = id % k.nchunk;
  q.b = id / k.nchunk;
  q.tx = threadIdx.x % k.tx;
  q.ty = threadIdx.x / k.tx;
  q.col = cb * k.tx + q.tx;
  q.active = q.ty < k.ty && q.col < k.cv;
  return q;
}
// Pixels of a chunk, and of the chunk's thread row `r` (a row takes every TY-th).
__device__ __forceinline__ int chunk_pixels(const Args& a, const Walk& k, int chunk) {
  return min(a.HW - chunk * k.per, k.per);
}
// One past its last pixel.  The chunks may reach past 2^31, no pixel does.
__device__ __forceinline__ int chunk_end(const Args& a, const Walk& k, int chunk) {
  return chunk * k.per + chunk_pixels(a, k, chunk);
}
__device__ __forceinline__ int row_pixels(const Args& a, const Walk& k, int chunk, int r) {
  const int left = chunk_pixels(a, k, chunk) - r;
  return left > 0 ? (left + k.ty - 1) / k.ty : 0;
}

// Per-channel mean and squared deviations of x over one chunk of pixels.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads, kBlocksForward) partial_stats(Args a, Walk k, float2* part) {
  __shared__ float2 red[kThreads * V];
  pdl_wait();
  pdl_trigger();
  const Place q = place(a, k);
  using L = Lanes<T, V>;
  using F = typename L::F;
  float s1[V] = {}, s2[V] = {}, pivot[V] = {};
  const int n = q.active ? row_pixels(a, k, q.chunk, q.ty) : 0;
  if (n) {
    const T* x = static_cast<const T*>(a.x) + q.b * a.xb + q.col * V;
    bool fresh = true;
    const int end = chunk_end(a, k, q.chunk);
    for (int p = q.chunk * k.per + q.ty; p < end; p += k.tile) {
      Pack<T, V> v[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (p + u * k.ty < end) v[u] = load_pack<T, V>(x + (p + u * k.ty) * a.xp);
      if (fresh) {
#pragma unroll
        for (int e = 0; e < V; ++e) pivot[e] = to_f32(v[0].e[e]);
        fresh = false;
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u)
        if (p + u * k.ty < end) {
#pragma unroll
          for (int j = 0; j < V / L::W; ++j) {
            const F d = fma(L::at(pivot, j), splat<F>(-1.f), L::get(v[u], j));
            L::put(s1, j, add(L::at(s1, j), d));
            L::put(s2, j, fma(d, d, L::at(s2, j)));
          }
        }
    }
  }
  if (q.ty < k.ty) {
    const float inv = n ? 1.f / n : 0.f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float md = s1[e] * inv;
      red[(q.ty * k.tx + q.tx) * V + e] = make_float2(pivot[e] + md, fmaxf(s2[e] - s1[e] * md, 0.f));
    }
  }
  __syncthreads();
  const int c0 = (q.col - q.tx) * V, cols = min(k.tx * V, a.C - c0), width = k.tx * V;
  for (int j = threadIdx.x; j < cols; j += kThreads) {
    float cn = 0.f, cm = 0.f, cq = 0.f;
    for (int r = 0; r < k.ty; ++r) {
      const float2 v = red[r * width + j];
      join(cn, cm, cq, (float)row_pixels(a, k, q.chunk, r), v.x, v.y);
    }
    if (a.shift) cm += load_param(a.shift, a.stype, (long long)q.b * a.C + c0 + j);
    red[j] = make_float2(cm, cq);  // row 0 of this channel has been read
  }
  __syncthreads();
  const float pixels = (float)chunk_pixels(a, k, q.chunk);
  float2* out = part + ((long long)q.b * k.nchunk + q.chunk) * (a.C / k.cell) + c0 / k.cell;
  for (int j = threadIdx.x; j < cols / k.cell; j += kThreads) {
    float cn = 0.f, cm = 0.f, cq = 0.f;
    for (int c = 0; c < k.cell; ++c) {
      const float2 v = red[j * k.cell + c];
      join(cn, cm, cq, pixels, v.x, v.y);
    }
    out[j] = make_float2(cm, cq);
  }
}

__device__ __forceinline__ float warp_total(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// Mean and 1/sqrt(variance + eps) of (b, group) from the parts, by one warp.  A group
// of thousands of channels has a part for each: the sums are in 64 bits (in 32, 8192
// channels of FP16 had a mean off by 4e-6 of their spread).
__device__ __forceinline__ float2 join_parts(const Args& a, const Walk& k, const float2* part,
                                             int b, int g) {
  const int lane = threadIdx.x & 31, cells = a.cpg / k.cell, items = k.nchunk * cells;
  const double total = (double)a.HW * a.cpg;
  const auto each = [&](auto&& use) {
    for (int i = lane; i < items; i += 32) {
      const int ch = i / cells;
      use((float)chunk_pixels(a, k, ch) * k.cell,
          part[((long long)b * k.nchunk + ch) * (a.C / k.cell) + g * cells + (i - ch * cells)]);
    }
  };
  // The mean relative to the first part's, which keeps its digits.
  const float pivot = part[(long long)b * k.nchunk * (a.C / k.cell) + g * cells].x;
  double t = 0, s = 0;
  each([&](float n, float2 v) { t += (double)(n * (v.x - pivot)); });
  const float off = (float)(warp_total(t) / total);
  each([&](float n, float2 v) {
    const float d = v.x - pivot - off;
    s += (double)fmaf(n * d, d, v.y);
  });
  return make_float2(pivot + off, 1.f / sqrtf((float)(warp_total(s) / total) + a.eps));
}

__global__ void __launch_bounds__(128) finish_stats(Args a, Walk k, const float2* part,
                                                    float* stats) {
  pdl_wait();
  pdl_trigger();
  const int bg = blockIdx.x * 4 + (threadIdx.x >> 5);
  if (bg >= a.B * a.G) return;
  const float2 v = join_parts(a, k, part, bg / a.G, bg % a.G);
  if ((threadIdx.x & 31) == 0) {
    stats[bg] = v.x;
    stats[(long long)a.B * a.G + bg] = v.y;
  }
}

// A block's channel constants, in shared memory: n = (x + mu) r, z = n w + beta.
template <int V>
struct Chan {
  float mu[kThreads * V], r[kThreads * V], w[kThreads * V], beta[kThreads * V];
};
template <int V>
__device__ __forceinline__ void channels(Chan<V>& h, const Args& a, const Walk& k, const Place& q,
                                         const float* stats) {
  const int c0 = (q.col - q.tx) * V, cols = min(k.tx * V, a.C - c0);
  for (int j = threadIdx.x; j < cols; j += kThreads) {
    const int c = c0 + j;
    const long long bg = (long long)q.b * a.G + c / a.cpg;
    h.mu[j] = (a.shift ? load_param(a.shift, a.stype, (long long)q.b * a.C + c) : 0.f) - stats[bg];
    h.r[j] = stats[(long long)a.B * a.G + bg];
    h.w[j] = a.w ? load_param(a.w, a.wtype, c) : 1.f;
    h.beta[j] = a.beta ? load_param(a.beta, a.wtype, c) : 0.f;
  }
}

template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kBlocksForward) apply(Args a, Walk k, const float* stats) {
  using L = Lanes<T, V>;
  using F = typename L::F;
  constexpr int J = V / L::W;
  __shared__ Chan<V> h;
  pdl_trigger();
  const Place q = place(a, k);
  const int end = q.active ? chunk_end(a, k, q.chunk) : 0;
  int p = q.chunk * k.per + q.ty;
  const T* x = static_cast<const T*>(a.x) + q.b * a.xb + q.col * V;
  T* y = static_cast<T*>(a.y) + (long long)q.b * a.HW * a.C + q.col * V;
  Pack<T, V> v[kAhead];
  const auto load = [&] {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (p + u * k.ty < end) v[u] = load_pack<T, V>(x + (p + u * k.ty) * a.xp);
  };
  // x is older than the pass before, which lets this one start once it has seen it.
  load();
  pdl_wait();
  channels<V>(h, a, k, q, stats);
  __syncthreads();
  F w[J], beta[J];  // z = x w + beta
#pragma unroll
  for (int j = 0; j < J; ++j) {
    w[j] = mul(L::at(h.w + q.tx * V, j), L::at(h.r + q.tx * V, j));
    beta[j] = fma(L::at(h.mu + q.tx * V, j), w[j], L::at(h.beta + q.tx * V, j));
  }
  for (; p < end; p += k.tile, load()) {
#pragma unroll
    for (int u = 0; u < kAhead; ++u)
      if (p + u * k.ty < end) {
#pragma unroll
        for (int j = 0; j < J; ++j)
          L::set(v[u], j, act<ACT>(fma(L::get(v[u], j), w[j], beta[j])));
        store_pack<T, V>(y + (long long)(p + u * k.ty) * a.C, v[u]);
      }
  }
}

// Gradient, first pass: per channel of one chunk, sums of dz, dz n and n.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kBlocksGrad) partial_grad(Args a, Walk k, const float* stats,
                                                         float* part) {
  using L = Lanes<T, V>;
  using F = typename L::F;
  constexpr int J = V / L::W;
  __shared__ union {
    Chan<V> h;
    float red[3][kThreads * V];
  } sm;
  pdl_trigger();
  pdl_wait();
  const Place q = place(a, k);
  channels<V>(sm.h, a, k, q, stats);
  __syncthreads();
  F s1[J], s2[J], s3[J], mu[J], r[J], w[J], beta[J];  // t = x + mu, n = t r, z = t w + beta
#pragma unroll
  for (int j = 0; j < J; ++j) {
    s1[j] = s2[j] = s3[j] = splat<F>(0.f);
    mu[j] = L::at(sm.h.mu + q.tx * V, j), r[j] = L::at(sm.h.r + q.tx * V, j);
    w[j] = mul(L::at(sm.h.w + q.tx * V, j), r[j]), beta[j] = L::at(sm.h.beta + q.tx * V, j);
  }
  __syncthreads();
  if (q.active) {
    const T* x = static_cast<const T*>(a.x) + q.b * a.xb + q.col * V;
    const T* dy = static_cast<const T*>(a.dy) + q.b * a.yb + q.col * V;
    constexpr int U = kAhead / 2;
    const int end = chunk_end(a, k, q.chunk);
    for (int p = q.chunk * k.per + q.ty; p < end; p += k.tile) {
      Pack<T, V> v[U], d[U];
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p + u * k.ty < end) {
          v[u] = load_pack<T, V>(x + (p + u * k.ty) * a.xp);
          d[u] = load_pack<T, V>(dy + (p + u * k.ty) * a.yp);
        }
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (p + u * k.ty < end) {
#pragma unroll
          for (int j = 0; j < J; ++j) {
            const F t = add(L::get(v[u], j), mu[j]);
            const F dz = act_grad<ACT>(L::get(d[u], j), fma(t, w[j], beta[j]));
            s1[j] = add(s1[j], dz);
            s2[j] = fma(dz, t, s2[j]);
            s3[j] = add(s3[j], t);
          }
        }
    }
  }
#pragma unroll
  for (int j = 0; j < J; ++j) s2[j] = mul(s2[j], r[j]), s3[j] = mul(s3[j], r[j]);
  const int width = k.tx * V;
  if (q.ty < k.ty) {
    const int i = q.ty * width + q.tx * V;
#pragma unroll
    for (int j = 0; j < J; ++j) {
      L::put(sm.red[0] + i, j, s1[j]);
      L::put(sm.red[1] + i, j, s2[j]);
      L::put(sm.red[2] + i, j, s3[j]);
    }
  }
  __syncthreads();
  const int c0 = (q.col - q.tx) * V, cols = min(width, a.C - c0);
  const long long plane = (long long)a.B * k.nchunk * a.C;
  for (int j = threadIdx.x; j < 3 * cols; j += kThreads) {
    const int i = j / cols, c = j - i * cols;
    float t = 0.f;
    for (int r = 0; r < k.ty; ++r) t += sm.red[i][r * width + c];
    part[i * plane + ((long long)q.b * k.nchunk + q.chunk) * a.C + c0 + c] = t;
  }
}

// The chunks' sums of every (b, channel), in order: sums[3][B][C].
__global__ void __launch_bounds__(256) join_grad(Args a, Walk k, const float* part, float* sums) {
  __shared__ double buf[8][32];
  pdl_trigger();
  pdl_wait();
  const int cblocks = (a.C + 31) / 32, lane = threadIdx.x & 31, row = threadIdx.x >> 5;
  const int b = blockIdx.x / cblocks, c = blockIdx.x % cblocks * 32 + lane;
  double t = 0;
  if (c < a.C) {
    const float* from = part + ((long long)blockIdx.y * a.B + b) * k.nchunk * a.C + c;
    for (int ch = row; ch < k.nchunk; ch += 8) t += from[(long long)ch * a.C];
  }
  buf[row][lane] = t;
  __syncthreads();
  if (row == 0 && c < a.C) {
#pragma unroll
    for (int r = 1; r < 8; ++r) t += buf[r][lane];
    sums[((long long)blockIdx.y * a.B + b) * a.C + c] = (float)t;
  }
}

// dw and dbeta: the samples' sums, in order.
__global__ void __launch_bounds__(128) param_grad(Args a, const float* sums, void* dw,
                                                  void* dbeta) {
  pdl_trigger();
  pdl_wait();
  const int c = blockIdx.x * 128 + threadIdx.x;
  if (c >= a.C) return;
  const long long plane = (long long)a.B * a.C;
  double s = 0, t = 0;
  for (int b = 0; b < a.B; ++b) {
    s += sums[(long long)b * a.C + c];
    t += sums[plane + (long long)b * a.C + c];
  }
  if (dw) store_param(dw, a.wtype, c, (float)t);
  if (dbeta) store_param(dbeta, a.wtype, c, (float)s);
}

// Second pass: dx, and from a sample's first chunk the shift's gradient.
template <typename T, int V, int ACT>
__global__ void __launch_bounds__(kThreads, kBlocksGrad) apply_grad(Args a, Walk k, const float* stats,
                                                       const float* sums, void* dshift) {
  using L = Lanes<T, V>;
  using F = typename L::F;
  constexpr int J = V / L::W, U = kAhead / 2;
  __shared__ Chan<V> h;
  __shared__ float A[kThreads * V], D[kThreads * V];  // minus the means, by channel
  pdl_trigger();
  pdl_wait();
  const Place q = place(a, k);
  const int c0 = (q.col - q.tx) * V, cols = min(k.tx * V, a.C - c0);
  const long long plane = (long long)a.B * a.C, bc = (long long)q.b * a.C;
  const int end = q.active ? chunk_end(a, k, q.chunk) : 0;
  int p = q.chunk * k.per + q.ty;
  const T* x = static_cast<const T*>(a.x) + q.b * a.xb + q.col * V;
  const T* dy = static_cast<const T*>(a.dy) + q.b * a.yb + q.col * V;
  T* dx = static_cast<T*>(a.y) + (long long)q.b * a.HW * a.C + q.col * V;
  Pack<T, V> v[U], d[U];
  const auto load = [&] {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u * k.ty < end) {
        v[u] = load_pack<T, V>(x + (p + u * k.ty) * a.xp);
        d[u] = load_pack<T, V>(dy + (p + u * k.ty) * a.yp);
      }
  };
  load();  // needs no sums
  channels<V>(h, a, k, q, stats);
  __syncthreads();
  const float inv = 1.f / ((float)a.HW * a.cpg);
  for (int g = c0 / a.cpg + (threadIdx.x >> 5); g <= (c0 + cols - 1) / a.cpg; g += kThreads / 32) {
    // The whole group's, also where the block has a part of its channels.
    const int lane = threadIdx.x & 31;
    float wa = 0.f, wd = 0.f;
    for (int c = g * a.cpg + lane; c < (g + 1) * a.cpg; c += 32) {
      const float wc = a.w ? load_param(a.w, a.wtype, c) : 1.f;
      wa = fmaf(wc, sums[bc + c], wa);
      wd = fmaf(wc, sums[plane + bc + c], wd);
    }
    wa = warp_total(wa) * inv;
    wd = warp_total(wd) * inv;
    for (int c = max(c0, g * a.cpg) + lane; c < min(c0 + cols, (g + 1) * a.cpg); c += 32) {
      A[c - c0] = -wa;
      D[c - c0] = -wd;
      if (dshift && q.chunk == 0)
        store_param(dshift, a.stype, bc + c,
                    h.r[c - c0] * (h.w[c - c0] * sums[bc + c] - a.HW * wa -
                                   wd * sums[2 * plane + bc + c]));
    }
  }
  __syncthreads();
  // t = x + mu, z = t w + beta, dx = dz w - r A - t r^2 D (w holds r).
  F mu[J], w[J], beta[J], ca[J], cd[J];
#pragma unroll
  for (int j = 0; j < J; ++j) {
    const F r = L::at(h.r + q.tx * V, j);
    mu[j] = L::at(h.mu + q.tx * V, j);
    w[j] = mul(L::at(h.w + q.tx * V, j), r), beta[j] = L::at(h.beta + q.tx * V, j);
    ca[j] = mul(L::at(A + q.tx * V, j), r), cd[j] = mul(mul(L::at(D + q.tx * V, j), r), r);
  }
  for (; p < end; p += k.tile, load()) {
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (p + u * k.ty < end) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
          const F t = add(L::get(v[u], j), mu[j]);
          const F dz = act_grad<ACT>(L::get(d[u], j), fma(t, w[j], beta[j]));
          L::set(v[u], j, fma(t, cd[j], fma(dz, w[j], ca[j])));
        }
        store_pack<T, V>(dx + (long long)(p + u * k.ty) * a.C, v[u]);
      }
  }
}

// ---------------------------------------------------------------------------
// Resident form: a cluster of blocks keeps a sample's channel block in registers
// ---------------------------------------------------------------------------
//
// x is read once and y written once.  A cluster of `cs` blocks owns `gb` whole
// groups of one sample, each block a range of the pixels, every thread up to NV
// vectors of it.  The blocks form (mean, squared deviations) of their range in two
// passes over their registers and exchange them through distributed shared memory.

struct Slab {
  int gb, nblk;  // groups per channel block, channel blocks
  int cs;        // blocks of a cluster
  int ppc;       // pixels per block
  int tx, ty;    // threads: vector columns x pixels
  int nv;        // vectors that a thread holds; the forward pass reads the rest again
  int threads;
};

constexpr int kSlabThreads = 512;
constexpr int kMostForward = 16, kMostGrad = 8;  // vectors a thread can hold
constexpr int kAgain = 4;  // width of the vectors that the forward pass may read again: FP32's

__device__ __forceinline__ void cluster_arrive() {
  __syncwarp();
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
}
__device__ __forceinline__ void cluster_wait() {
  __syncwarp();
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// A float of the same shared variable in the cluster's block `rank`.
__device__ __forceinline__ float peer_float(const float* p, int rank) {
  uint32_t at;
  float v;
  asm("mapa.shared::cluster.u32 %0, %1, %2;"
      : "=r"(at)
      : "r"(static_cast<uint32_t>(__cvta_generic_to_shared(p))), "r"(rank));
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// Keeps a vector packed: without this the compiler holds the 32-bit forms of all
// vectors from one pass over them to the next, which spills.
template <typename T, int V, int NV>
__device__ __forceinline__ void stay_packed(Pack<T, V> (&d)[NV]) {
  if constexpr (V > 1) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      uint4& q = reinterpret_cast<uint4&>(d[v]);
      asm volatile("" : "+r"(q.x), "+r"(q.y), "+r"(q.z), "+r"(q.w));
    }
  }
}

struct Spot {
  int b, rank, c0, nch, ng, g0, p0, p1, tx, ty, nv;
  bool active;
};
__device__ __forceinline__ Spot spot(const Args& a, const Slab& k, int V) {
  Spot q;
  unsigned id = blockIdx.x;
  q.rank = id % k.cs;
  id /= k.cs;
  const int blk = id % k.nblk;
  q.b = id / k.nblk;
  q.g0 = blk * k.gb;
  q.ng = min(k.gb, a.G - q.g0);
  q.c0 = q.g0 * a.cpg;
  q.nch = q.ng * a.cpg;
  q.p0 = min(a.HW, q.rank * k.ppc);
  q.p1 = min(a.HW, q.p0 + k.ppc);
  q.tx = threadIdx.x % k.tx;
  q.ty = threadIdx.x / k.tx;
  q.active = q.ty < k.ty && q.tx * V < q.nch;
  const int left = q.p1 - q.p0 - q.ty;
  q.nv = q.active && left > 0 ? (left + k.ty - 1) / k.ty : 0;
  return q;
}

template <typename T, int V, int NV, int ACT>
__global__ void __launch_bounds__(kSlabThreads, 1)
    resident_forward(Args a, Slab k, float* stats) {
  using L = Lanes<T, V>;
  using F = typename L::F;
  constexpr int W = L::W;
  extern __shared__ float sm[];
  const int width = k.tx * V;  // channels of the block, padded to vectors
  float* red = sm;                      // [ty][width]
  float* mu = red + k.ty * width;       // [width] what is added to x: shift - mean
  float* sh = mu + width;               // [width] shift
  float* wt = sh + width;               // [width] weight, later weight / sigma
  float* bt = wt + width;               // [width] bias, later the whole offset
  float* part = bt + width;             // [2][gb] the block's mean and deviations
  pdl_trigger();
  pdl_wait();
  Spot q = spot(a, k, V);
  q.nv = min(q.nv, NV);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;

  Pack<T, V> d[NV];
  {
    const T* x = static_cast<const T*>(a.x) + q.b * a.xb + (q.p0 + q.ty) * a.xp + q.c0 + q.tx * V;
    const long long step = k.ty * a.xp;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v < q.nv) d[v] = load_pack<T, V>(x + v * step);
  }
  for (int c = threadIdx.x; c < q.nch; c += blockDim.x) {
    sh[c] = a.shift ? load_param(a.shift, a.stype, (long long)q.b * a.C + q.c0 + c) : 0.f;
    wt[c] = a.w ? load_param(a.w, a.wtype, q.c0 + c) : 1.f;
    bt[c] = a.beta ? load_param(a.beta, a.wtype, q.c0 + c) : 0.f;
  }
  float* mine = red + q.ty * width + q.tx * V;
  // Most threads hold NV vectors and need no test for each: every pass comes twice.
  const auto pass = [&](auto&& body) {
    if (!q.active) return;
    if (q.nv == NV) body([](int) { return true; });
    else body([&](int v) { return v < q.nv; });
  };
  // The vectors that the registers do not hold, out of L2, four on their way.
  const auto rest = [&](auto&& use) {
    if constexpr (NV < kMostForward || V != kAgain) return;
    if (!q.active) return;
    const T* x = static_cast<const T*>(a.x) + q.b * a.xb + q.c0 + q.tx * V;
    for (int p = q.p0 + q.ty + NV * k.ty; p < q.p1; p += 4 * k.ty) {
      Pack<T, V> v[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (p + u * k.ty < q.p1) v[u] = load_pack<T, V>(x + (p + u * k.ty) * a.xp);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (p + u * k.ty < q.p1) use(v[u], p + u * k.ty);
    }
  };
  pass([&](auto has) {
#pragma unroll
    for (int j = 0; j < V / W; ++j) {
      F t = splat<F>(0.f);
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (has(v)) t = add(t, L::get(d[v], j));
      L::put(mine, j, t);
    }
  });
  rest([&](const Pack<T, V>& v, int) {
#pragma unroll
    for (int j = 0; j < V / W; ++j) L::put(mine, j, add(L::at(mine, j), L::get(v, j)));
  });
  __syncthreads();
  stay_packed(d);
  // `segs` threads for every channel add up their rows; a warp then takes a group's
  // segs x cpg sums.
  const int segs = max(1, min(k.ty, (int)blockDim.x / width));
  auto fold_rows = [&] {
    for (int i = threadIdx.x; i < width * segs; i += blockDim.x) {
      const int sg = i / width, c = i - sg * width;
      float t = 0.f;
      for (int r = sg; r < k.ty; r += segs) t += red[r * width + c];
      red[sg * width + c] = t;  // no other thread reads this row's channel
    }
    __syncthreads();
  };
  auto group_sum = [&](int g) {
    float t = 0.f;
    for (int c = g * a.cpg + lane; c < (g + 1) * a.cpg; c += 32)
      for (int r = 0; r < segs; ++r) t += red[r * width + c];
    return t;
  };
  fold_rows();
  const float pixels = (float)(q.p1 - q.p0);
  for (int g = warp; g < q.ng; g += warps) {
    float t = group_sum(g);
    for (int c = lane; c < a.cpg; c += 32) t = fmaf(pixels, sh[g * a.cpg + c], t);
    const float m = pixels > 0.f ? warp_total(t) / (pixels * a.cpg) : 0.f;
    for (int c = lane; c < a.cpg; c += 32) mu[g * a.cpg + c] = sh[g * a.cpg + c] - m;
    if (lane == 0) part[g] = m;
  }
  __syncthreads();
  pass([&](auto has) {
#pragma unroll
    for (int j = 0; j < V / W; ++j) {
      const F m = L::at(mu + q.tx * V, j);
      F t = splat<F>(0.f);
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (has(v)) {
          const F u = add(L::get(d[v], j), m);
          t = fma(u, u, t);
        }
      L::put(mine, j, t);
    }
  });
  rest([&](const Pack<T, V>& v, int) {
#pragma unroll
    for (int j = 0; j < V / W; ++j) {
      const F u = add(L::get(v, j), L::at(mu + q.tx * V, j));
      L::put(mine, j, fma(u, u, L::at(mine, j)));
    }
  });
  __syncthreads();
  stay_packed(d);
  fold_rows();
  for (int g = warp; g < q.ng; g += warps) {
    const float t = warp_total(group_sum(g));
    if (lane == 0) part[k.gb + g] = t;
  }
  cluster_arrive();
  cluster_wait();
  for (int g = warp; g < q.ng; g += warps) {
    // Every block joins the cluster's parts in the same order.
    float pm = 0.f, pq = 0.f;
    if (lane < k.cs) {
      pm = peer_float(part + g, lane);
      pq = peer_float(part + k.gb + g, lane);
    }
    float n = 0.f, m = 0.f, s = 0.f;
    for (int r = 0; r < k.cs; ++r) {
      const float np = (float)max(0, min(k.ppc, a.HW - r * k.ppc)) * a.cpg;
      join(n, m, s, np, __shfl_sync(~0u, pm, r), __shfl_sync(~0u, pq, r));
    }
    const float rstd = 1.f / sqrtf(s / n + a.eps);
    if (stats && q.rank == 0 && lane == 0) {
      const long long bg = (long long)q.b * a.G + q.g0 + g;
      stats[bg] = m;
      stats[(long long)a.B * a.G + bg] = rstd;
    }
    for (int c = g * a.cpg + lane; c < (g + 1) * a.cpg; c += 32) {
      wt[c] *= rstd;
      bt[c] = fmaf(sh[c] - m, wt[c], bt[c]);
    }
  }
  cluster_arrive();  // this block has read its peers' parts
  __syncthreads();
  pass([&](auto has) {
#pragma unroll
    for (int j = 0; j < V / W; ++j) {
      const F w = L::at(wt + q.tx * V, j), b = L::at(bt + q.tx * V, j);
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (has(v)) L::set(d[v], j, act<ACT>(fma(L::get(d[v], j), w, b)));
    }
    T* y = static_cast<T*>(a.y) + ((long long)q.b * a.HW + q.p0 + q.ty) * a.C + q.c0 + q.tx * V;
    const long long step = (long long)k.ty * a.C;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (has(v)) store_pack<T, V>(y + v * step, d[v]);
  });
  rest([&](Pack<T, V> v, int p) {
#pragma unroll
    for (int j = 0; j < V / W; ++j)
      L::set(v, j, act<ACT>(fma(L::get(v, j), L::at(wt + q.tx * V, j), L::at(bt + q.tx * V, j))));
    store_pack<T, V>(static_cast<T*>(a.y) + ((long long)q.b * a.HW + p) * a.C + q.c0 + q.tx * V, v);
  });
  cluster_wait();
}

// The gradient of a slab: x and dy in registers, the channels' sums exchanged.
template <typename T, int V, int NV, int ACT>
__global__ void __launch_bounds__(kSlabThreads, 1)
    resident_grad(Args a, Slab k, const float* stats, float* sums, void* dshift) {
  using L = Lanes<T, V>;
  using F = typename L::F;
  constexpr int W = L::W;
  extern __shared__ float sm[];
  const int width = k.tx * V;
  const int rows = k.ty * width;
  float* red = sm;                 // [3][ty][width]
  float* mu = red + 3 * rows;      // [width] each
  float* rs = mu + width;
  float* wt = rs + width;
  float* bt = wt + width;
  float* own = bt + width;         // [3][width] the block's sums
  float* all = own + 3 * width;    // [3][width] the sample's sums
  float* ga = all + 3 * width;     // [width] -A
  float* gd = ga + width;          // [width] -D
  pdl_trigger();
  pdl_wait();
  const Spot q = spot(a, k, V);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;

  Pack<T, V> d[NV], e[NV];
  {
    const T* x = static_cast<const T*>(a.x) + q.b * a.xb + (q.p0 + q.ty) * a.xp + q.c0 + q.tx * V;
    const T* y = static_cast<const T*>(a.dy) + q.b * a.yb + (q.p0 + q.ty) * a.yp + q.c0 + q.tx * V;
    const long long sx = k.ty * a.xp, sy = k.ty * a.yp;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (v < q.nv) {
        d[v] = load_pack<T, V>(x + v * sx);
        e[v] = load_pack<T, V>(y + v * sy);
      }
  }
  for (int c = threadIdx.x; c < q.nch; c += blockDim.x) {
    const long long bg = (long long)q.b * a.G + q.g0 + c / a.cpg;
    mu[c] = (a.shift ? load_param(a.shift, a.stype, (long long)q.b * a.C + q.c0 + c) : 0.f) -
            stats[bg];
    rs[c] = stats[(long long)a.B * a.G + bg];
    wt[c] = a.w ? load_param(a.w, a.wtype, q.c0 + c) : 1.f;
    bt[c] = a.beta ? load_param(a.beta, a.wtype, q.c0 + c) : 0.f;
  }
  __syncthreads();
  const auto pass = [&](auto&& body) {
    if (!q.active) return;
    if (q.nv == NV) body([](int) { return true; });
    else body([&](int v) { return v < q.nv; });
  };
  pass([&](auto has) {
    float* mine = red + q.ty * width + q.tx * V;
#pragma unroll
    for (int j = 0; j < V / W; ++j) {
      // t = x + m, n = t r, z = t w + b
      const F m = L::at(mu + q.tx * V, j), r = L::at(rs + q.tx * V, j);
      const F w = mul(L::at(wt + q.tx * V, j), r), b = L::at(bt + q.tx * V, j);
      F s1 = splat<F>(0.f), s2 = s1, s3 = s1;
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (has(v)) {
          const F t = add(L::get(d[v], j), m);
          const F dz = act_grad<ACT>(L::get(e[v], j), fma(t, w, b));
          s1 = add(s1, dz);
          s2 = fma(dz, t, s2);
          s3 = add(s3, t);
        }
      L::put(mine, j, s1);
      L::put(mine + rows, j, mul(s2, r));
      L::put(mine + 2 * rows, j, mul(s3, r));
    }
  });
  __syncthreads();
  stay_packed(d);
  stay_packed(e);
  // A few threads for every channel, then one.
  const int segs = max(1, min(k.ty, (int)blockDim.x / (3 * width)));
  for (int i = threadIdx.x; i < 3 * width * segs; i += blockDim.x) {
    const int sg = i / (3 * width), s = i / width % 3, c = i % width;
    float t = 0.f;
    if (c < q.nch)
      for (int r = sg; r < k.ty; r += segs) t += red[s * rows + r * width + c];
    // The first row that this thread alone has read takes its sum.
    red[s * rows + sg * width + c] = t;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 3 * width; i += blockDim.x) {
    const int s = i / width, c = i % width;
    float t = 0.f;
    for (int r = 0; r < segs; ++r) t += red[s * rows + r * width + c];
    own[i] = t;
  }
  cluster_arrive();
  cluster_wait();
  for (int i = threadIdx.x; i < 3 * width; i += blockDim.x) {
    float t = 0.f;
    for (int r = 0; r < k.cs; ++r) t += peer_float(own + i, r);
    all[i] = t;
  }
  cluster_arrive();
  __syncthreads();
  const float inv = 1.f / ((float)a.HW * a.cpg);
  for (int g = warp; g < q.ng; g += warps) {
    float wa = 0.f, wd = 0.f;
    for (int c = g * a.cpg + lane; c < (g + 1) * a.cpg; c += 32) {
      wa = fmaf(wt[c], all[c], wa);
      wd = fmaf(wt[c], all[width + c], wd);
    }
    wa = warp_total(wa) * inv;
    wd = warp_total(wd) * inv;
    for (int c = g * a.cpg + lane; c < (g + 1) * a.cpg; c += 32) {
      ga[c] = -wa;
      gd[c] = -wd;
      if (q.rank == 0) {
        const long long bc = (long long)q.b * a.C + q.c0 + c;
        sums[bc] = all[c];
        sums[(long long)a.B * a.C + bc] = all[width + c];
        if (dshift)
          store_param(dshift, a.stype, bc,
                      rs[c] * (wt[c] * all[c] - a.HW * wa - wd * all[2 * width + c]));
      }
    }
  }
  __syncthreads();
  pass([&](auto has) {
#pragma unroll
    for (int j = 0; j < V / W; ++j) {
      const F m = L::at(mu + q.tx * V, j), r = L::at(rs + q.tx * V, j);
      const F w = mul(L::at(wt + q.tx * V, j), r), b = L::at(bt + q.tx * V, j);
      const F A = mul(L::at(ga + q.tx * V, j), r), D = mul(mul(L::at(gd + q.tx * V, j), r), r);
#pragma unroll
      for (int v = 0; v < NV; ++v)
        if (has(v)) {
          const F t = add(L::get(d[v], j), m);
          const F dz = act_grad<ACT>(L::get(e[v], j), fma(t, w, b));
          L::set(d[v], j, fma(t, D, fma(dz, w, A)));
        }
    }
    T* y = static_cast<T*>(a.y) + ((long long)q.b * a.HW + q.p0 + q.ty) * a.C + q.c0 + q.tx * V;
    const long long step = (long long)k.ty * a.C;
#pragma unroll
    for (int v = 0; v < NV; ++v)
      if (has(v)) store_pack<T, V>(y + v * step, d[v]);
  });
  cluster_wait();
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

Walk make_walk(int B, int HW, int C, int G, int V, bool grad) {
  Walk k;
  const int cpg = C / G;
  k.cv = C / V;
  k.ncb = (k.cv + kThreads - 1) / kThreads;
  k.tx = (k.cv + k.ncb - 1) / k.ncb;
  k.ty = kThreads / k.tx;
  k.cell = k.ncb == 1 || k.tx * V % cpg == 0 ? cpg : 1;
  const int U = grad ? kAhead / 2 : kAhead;
  k.tile = U * k.ty;
  // One wave of blocks, by their registers, of a tile at least.
  const int rows = (HW + k.ty - 1) / k.ty;
  long long chunks = (long long)(grad ? kBlocksGrad : kBlocksForward) * device_sms() / ((long long)B * k.ncb);
  if (chunks > (rows + U - 1) / U) chunks = (rows + U - 1) / U;
  if (chunks < 1) chunks = 1;
  k.per = (int)((rows + chunks - 1) / chunks) * k.ty;
  k.nchunk = (int)(((long long)HW + k.per - 1) / k.per);
  return k;
}

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

int gcd(int a, int b) { return b ? gcd(b, a % b) : a; }

constexpr int kSlabSmem = 220 * 1024;
size_t slab_smem(const Slab& k, int V, bool grad) {
  const size_t width = (size_t)k.tx * V;
  return 4 * (grad ? 3 * k.ty * width + 12 * width : k.ty * width + 4 * width + 2 * k.gb);
}


// The resident form of a call, where it fits and pays.
bool make_slab(int B, int HW, int C, int G, int V, bool grad, int sms, Slab* best) {
  const int most = grad ? kMostGrad : kMostForward;
  const int cpg = C / G;
  const int unit = V / gcd(cpg, V);  // groups whose channels fill whole vectors
  bool found = false;
  double best_cost = 0;
  for (int gb = unit;; gb *= 2) {
    if (gb > G) gb = G;
    const int tx = gb * cpg / V;
    if (tx > kSlabThreads) break;
    for (int cs = 1; cs <= 8; cs *= 2)
      for (int nv = 2; nv <= most; nv *= 2) {
        Slab k;
        k.gb = gb;
        k.nblk = (G + gb - 1) / gb;
        k.cs = cs;
        k.ppc = (HW + cs - 1) / cs;
        k.tx = tx;
        k.nv = nv;
        k.ty = (k.ppc + nv - 1) / nv;
        // The share of the vectors that is read again, three times over.  It pays for
        // FP32, whose vectors need no conversion, on most of the SMs and with rows of
        // whole lines: 4x320x61x67 15.0 us, streaming 18.6; 2x640x64x64 15.4, streaming
        // 21.1.  Not in FP16 (8x320x64x64 25.2 us, streaming 24.7; values one by one
        // 4x76x64x70 19.1, streaming 14.8), on 32 blocks (1x128x120x120 in 4 groups 16.7,
        // streaming 14.7) or in rows of 80 bytes (1x320x128x128 29.4, streaming 21.4).
        double again = 0;
        if (!grad && nv == most && (long long)tx * k.ty > kSlabThreads) {
          k.ty = kSlabThreads / tx;
          again = 1.0 - (double)nv * k.ty / k.ppc;
          if (again > 0.5 || V != kAgain || tx * 16 < 128 ||
              (long long)B * k.nblk * cs * 4 < 3 * sms)
            continue;
        }
        if ((long long)tx * k.ty > kSlabThreads || slab_smem(k, V, grad) > kSlabSmem) continue;
        k.threads = (tx * k.ty + 31) / 32 * 32;
        // The resident form pays while its blocks fit the SMs at once (twice at most in
        // the gradient, whose streaming form has four launches): its phases do not
        // overlap, so further waves cost it more than the second read it saves.
        // Measured, FP16: 8x640x32x32 forward 12.5 us (streaming 20), 8x320x64x64 in
        // two waves 27.7 us (streaming 24.7).
        const long long blocks = (long long)B * k.nblk * cs;
        const int per_sm = std::min(32, 65536 / ((nv * 4 * (grad ? 2 : 1) + 64) * k.threads));
        const long long room = (long long)sms * per_sm;
        if (blocks > room * (grad ? 2 : 1)) continue;
        // Bytes of the busiest SM, short rows counted with the sectors they touch, and
        // the cluster's exchange.
        const double cost = (double)((blocks + sms - 1) / sms) * k.ppc * (tx * 16 + 16) *
                                (1 + again) / 22.0 +
                            150.0 * cs;
        if (!found || cost < best_cost) {
          found = true;
          best_cost = cost;
          *best = k;
        }
      }
    if (gb >= G) break;
  }
  return found;
}

template <auto Kernel, typename... Args2>
cudaError_t slab_launch(const Slab& k, int B, size_t smem, cudaStream_t s, Args2&&... args) {
  static std::atomic<unsigned long long> allowed{0};
  const cudaError_t e = allow_smem(Kernel, &allowed, kSlabSmem);
  if (e != cudaSuccess) return e;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)((long long)B * k.nblk * k.cs));
  cfg.blockDim = dim3(k.threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = k.cs;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = pdl_enabled(kPdlInput) ? 1 : 0;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  return cudaLaunchKernelEx(&cfg, Kernel, std::forward<Args2>(args)...);
}

template <typename T, int V, int ACT>
cudaError_t forward_resident(const Args& a, const Slab& k, float* stats, cudaStream_t s) {
  const size_t smem = slab_smem(k, V, false);
#define NOVA_GN_SLAB(NV) \
  slab_launch<resident_forward<T, V, NV, ACT>>(k, a.B, smem, s, a, k, stats)
  if (k.nv <= 2) return NOVA_GN_SLAB(2);
  if (k.nv <= 4) return NOVA_GN_SLAB(4);
  if (k.nv <= 8) return NOVA_GN_SLAB(8);
  return NOVA_GN_SLAB(16);
#undef NOVA_GN_SLAB
}

template <typename T, int V, int ACT>
cudaError_t grad_resident(const Args& a, const Slab& k, const float* stats, float* sums,
                          void* dshift, cudaStream_t s) {
  const size_t smem = slab_smem(k, V, true);
#define NOVA_GN_SLAB(NV) \
  slab_launch<resident_grad<T, V, NV, ACT>>(k, a.B, smem, s, a, k, stats, sums, dshift)
  if (k.nv <= 2) return NOVA_GN_SLAB(2);
  if (k.nv <= 4) return NOVA_GN_SLAB(4);
  return NOVA_GN_SLAB(8);
#undef NOVA_GN_SLAB
}

// Workspace of a call with vectors of V elements.
long long workspace_bytes(int B, int HW, int C, int G, int V, bool grad) {
  Slab slab;
  if (make_slab(B, HW, C, G, V, grad, device_sms(), &slab))
    return grad ? (long long)align256((size_t)B * C * 12) : 0;
  const Walk k = make_walk(B, HW, C, G, V, grad);
  const size_t parts = (size_t)B * k.nchunk * C;
  return (long long)(grad ? align256(parts * 12) + align256((size_t)B * C * 12)
                          : align256(parts / k.cell * 8) + align256((size_t)B * G * 8));
}

template <typename T, int V>
cudaError_t forward(const Args& a, int act, float* stats, unsigned char* ws, cudaStream_t s) {
  Slab slab;
  if (make_slab(a.B, a.HW, a.C, a.G, V, false, device_sms(), &slab))
    return act == kSilu ? forward_resident<T, V, kSilu>(a, slab, stats, s)
                        : forward_resident<T, V, kNone>(a, slab, stats, s);
  const Walk k = make_walk(a.B, a.HW, a.C, a.G, V, false);
  if (!stats) {
    stats = reinterpret_cast<float*>(ws);
    ws += align256((size_t)a.B * a.G * 8);
  }
  float2* part = reinterpret_cast<float2*>(ws);
  const dim3 grid((unsigned)((long long)a.B * k.nchunk * k.ncb));
  cudaError_t e = launch_pdl(kPdlInput, partial_stats<T, V>, grid, dim3(kThreads), 0, s, a, k, part);
  // A kernel of its own: joined by every block of the next pass instead, 55 parts for each
  // of 32 groups cost that pass 5 us (8 x 320 x 64 x 64: 29.7 us, as it is 24.7).
  if (e == cudaSuccess)
    e = launch_pdl(kPdlInput, finish_stats, dim3((a.B * a.G + 3) / 4), dim3(128), 0, s, a, k,
                   (const float2*)part, stats);
  if (e != cudaSuccess) return e;
  return act == kSilu ? launch_pdl(kPdlInput, apply<T, V, kSilu>, grid, dim3(kThreads), 0, s, a, k,
                                   (const float*)stats)
                      : launch_pdl(kPdlInput, apply<T, V, kNone>, grid, dim3(kThreads), 0, s, a, k,
                                   (const float*)stats);
}

template <typename T, int V, int ACT>
cudaError_t backward(const Args& a, const float* stats, void* dw, void* dbeta, void* dshift,
                     unsigned char* ws, cudaStream_t s) {
  const Walk k = make_walk(a.B, a.HW, a.C, a.G, V, true);
  float* sums = reinterpret_cast<float*>(ws);  // [3][B][C]
  float* part = reinterpret_cast<float*>(ws + align256((size_t)a.B * a.C * 12));
  const dim3 grid((unsigned)((long long)a.B * k.nchunk * k.ncb));
  cudaError_t e;
  Slab slab;
  if (make_slab(a.B, a.HW, a.C, a.G, V, true, device_sms(), &slab)) {
    e = grad_resident<T, V, ACT>(a, slab, stats, sums, dshift, s);
    if (e == cudaSuccess && (dw || dbeta))
      e = launch_pdl(kPdlInput, param_grad, dim3((a.C + 127) / 128), dim3(128), 0, s, a,
                     (const float*)sums, dw, dbeta);
    return e;
  }
  e = launch_pdl(kPdlInput, partial_grad<T, V, ACT>, grid, dim3(kThreads), 0, s, a, k,
                             stats, part);
  if (e == cudaSuccess)
    e = launch_pdl(kPdlInput, join_grad, dim3(a.B * ((a.C + 31) / 32), 3), dim3(256), 0, s, a, k,
                   (const float*)part, sums);
  if (e == cudaSuccess)
    e = launch_pdl(kPdlInput, apply_grad<T, V, ACT>, grid, dim3(kThreads), 0, s, a, k, stats,
                   (const float*)sums, dshift);
  if (e == cudaSuccess && (dw || dbeta))
    e = launch_pdl(kPdlInput, param_grad, dim3((a.C + 127) / 128), dim3(128), 0, s, a,
                   (const float*)sums, dw, dbeta);
  return e;
}

// 16-byte accesses where every vector of every operand starts on 16 bytes.
bool wide(const Args& a, int dtype, bool grad) {
  const int V = 16 / dtype_bytes(dtype);
  return a.C % V == 0 && a.xp % V == 0 && a.xb % V == 0 && aligned16(a.x) && aligned16(a.y) &&
         (!grad || (a.yp % V == 0 && a.yb % V == 0 && aligned16(a.dy)));
}

// Pixels, and groups of all samples, are counted in 32 bits.
bool too_many(int B, int HW, int G) {
  constexpr long long kMost = (1ll << 31) - 4096;
  return (long long)B * HW > kMost || (long long)B * G > kMost;
}

int check(const char* what, const Args& a, int dtype, bool grad) {
  auto bad = [&](const char* why) {
    return record_error(NOVA_ERR_INVALID_ARGUMENT, std::string(what) + ": " + why);
  };
  if (a.B < 1 || a.HW < 1 || a.C < 1 || a.G < 1) return bad("bad sizes");
  if (a.C % a.G) return bad("channels must divide into the groups");
  if (a.cpg > 8192) return bad("more than 8192 channels per group");
  if (!dtype_ok(dtype) || !dtype_ok(a.wtype) || !dtype_ok(a.stype)) return bad("bad element type");
  if (!a.x || !a.y || (grad && !a.dy)) return bad("null pointer");
  if (a.xp < a.C || a.xb < 0 || (grad && (a.yp < a.C || a.yb < 0)))
    return bad("a pixel stride below the channels, or a negative batch stride");
  if (!(a.eps >= 0.f)) return bad("eps must not be negative");
  if (too_many(a.B, a.HW, a.G)) return bad("more than 2^31 - 4096 pixels or groups");
  return NOVA_OK;
}

// The workspace of checked arguments, by the current device: the operands' by then,
// whose SMs the launch plans for.
int check_workspace(const char* what, const Args& a, int dtype, const void* ws, long long ws_bytes,
                    bool grad) {
  const int V = wide(a, dtype, grad) ? 16 / dtype_bytes(dtype) : 1;
  const long long need = workspace_bytes(a.B, a.HW, a.C, a.G, V, grad);
  if (need > 0 && (!ws || reinterpret_cast<uintptr_t>(ws) % 256))
    return record_error(NOVA_ERR_INVALID_ARGUMENT,
                        std::string(what) + ": workspace missing or not 256-byte aligned");
  if (ws_bytes < need)
    return record_error(NOVA_ERR_WORKSPACE,
                        std::string(what) + ": workspace needs " + std::to_string(need) + " bytes");
  return NOVA_OK;
}

int done(const char* what, cudaError_t e) {
  if (e == cudaSuccess) return NOVA_OK;
  return record_error(NOVA_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
}

}  // namespace gn
}  // namespace nova

#define NOVA_EXPORT extern "C" __attribute__((visibility("default")))

NOVA_EXPORT long long nova_group_norm_workspace_bytes(int batch, int pixels, int C, int groups,
                                                      int dtype, int aligned, int grad) {
  if (batch < 1 || pixels < 1 || C < 1 || groups < 1 || C % groups ||
      !nova::unet::dtype_ok(dtype) || nova::gn::too_many(batch, pixels, groups))
    return -1;
  const int V = 16 / nova::unet::dtype_bytes(dtype);
  const bool wide = C % V == 0;
  // Where it is not known whether the operands are aligned: enough for both.
  return std::max(
      wide ? nova::gn::workspace_bytes(batch, pixels, C, groups, V, grad != 0) : 0,
      wide && aligned ? 0 : nova::gn::workspace_bytes(batch, pixels, C, groups, 1, grad != 0));
}

NOVA_EXPORT int nova_group_norm_v2(const void* d_input, const void* d_weight, const void* d_bias,
                                   const void* d_shift, void* d_output, void* d_stats,
                                   void* d_workspace, long long ws_bytes, int batch, int pixels,
                                   int C, int groups, long long batch_stride,
                                   long long pixel_stride, int dtype, int param_dtype,
                                   int shift_dtype, int activation, float eps, void* stream) try {
  using namespace nova;
  using namespace nova::gn;
  Args a{d_input, nullptr, d_weight, d_bias, d_shift, d_output, batch_stride, pixel_stride, 0, 0,
         batch, pixels, C, groups, groups > 0 ? C / groups : 0, param_dtype, shift_dtype, eps};
  if (const int rc = check("group_norm", a, dtype, false)) return rc;
  if (activation != kNone && activation != kSilu)
    return record_error(NOVA_ERR_INVALID_ARGUMENT, "group_norm: bad activation");
  const OnDeviceOf device(d_input);
  if (const int rc = check_workspace("group_norm", a, dtype, d_workspace, ws_bytes, false)) return rc;
  if (device.status() != cudaSuccess) return done("group_norm: input", device.status());
  unsigned char* ws = static_cast<unsigned char*>(d_workspace);
  float* stats = static_cast<float*>(d_stats);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool v = wide(a, dtype, false);
  cudaError_t e;
  if (dtype == kF16)
    e = v ? forward<__half, 8>(a, activation, stats, ws, s)
          : forward<__half, 1>(a, activation, stats, ws, s);
  else if (dtype == kBF16)
    e = v ? forward<__nv_bfloat16, 8>(a, activation, stats, ws, s)
          : forward<__nv_bfloat16, 1>(a, activation, stats, ws, s);
  else
    e = v ? forward<float, 4>(a, activation, stats, ws, s)
          : forward<float, 1>(a, activation, stats, ws, s);
  return done("group_norm", e);
} catch (...) {
  return NOVA_ERR_ALLOC;
}

namespace nova {
namespace gn {
template <typename T, int V>
cudaError_t backward_act(const Args& a, int act, const float* stats, void* dw, void* dbeta,
                         void* dshift, unsigned char* ws, cudaStream_t s) {
  return act == kSilu ? backward<T, V, kSilu>(a, stats, dw, dbeta, dshift, ws, s)
                      : backward<T, V, kNone>(a, stats, dw, dbeta, dshift, ws, s);
}
}  // namespace gn
}  // namespace nova

NOVA_EXPORT int nova_group_norm_grad_v2(
    const void* d_input, const void* d_grad_output, const void* d_weight, const void* d_bias,
    const void* d_shift, const void* d_stats, void* d_grad_input, void* d_grad_weight,
    void* d_grad_bias, void* d_grad_shift, void* d_workspace, long long ws_bytes, int batch,
    int pixels, int C, int groups, long long batch_stride, long long pixel_stride,
    long long grad_batch_stride, long long grad_pixel_stride, int dtype, int param_dtype,
    int shift_dtype, int activation, void* stream) try {
  using namespace nova;
  using namespace nova::gn;
  Args a{d_input, d_grad_output, d_weight, d_bias, d_shift, d_grad_input, batch_stride,
         pixel_stride, grad_batch_stride, grad_pixel_stride, batch, pixels, C, groups,
         groups > 0 ? C / groups : 0, param_dtype, shift_dtype, 0.f};
  if (const int rc = check("group_norm_grad", a, dtype, true)) return rc;
  if (!d_stats) return record_error(NOVA_ERR_INVALID_ARGUMENT, "group_norm_grad: null pointer");
  if (activation != kNone && activation != kSilu)
    return record_error(NOVA_ERR_INVALID_ARGUMENT, "group_norm_grad: bad activation");
  const OnDeviceOf device(d_input);
  if (const int rc = check_workspace("group_norm_grad", a, dtype, d_workspace, ws_bytes, true)) return rc;
  if (device.status() != cudaSuccess) return done("group_norm_grad: input", device.status());
  unsigned char* ws = static_cast<unsigned char*>(d_workspace);
  const float* stats = static_cast<const float*>(d_stats);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const bool v = wide(a, dtype, true);
  cudaError_t e;
#define NOVA_GN_BACKWARD(T, V) \
  backward_act<T, V>(a, activation, stats, d_grad_weight, d_grad_bias, d_grad_shift, ws, s)
  if (dtype == kF16)
    e = v ? NOVA_GN_BACKWARD(__half, 8) : NOVA_GN_BACKWARD(__half, 1);
  else if (dtype == kBF16)
    e = v ? NOVA_GN_BACKWARD(__nv_bfloat16, 8) : NOVA_GN_BACKWARD(__nv_bfloat16, 1);
  else
    e = v ? NOVA_GN_BACKWARD(float, 4) : NOVA_GN_BACKWARD(float, 1);
#undef NOVA_GN_BACKWARD
  return done("group_norm_grad", e);
} catch (...) {
  return NOVA_ERR_ALLOC;
}
