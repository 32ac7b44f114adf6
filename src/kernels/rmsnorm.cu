// Root-mean-square norm of a sum of partials and the residual, and its
// gradient (see rmsnorm.h).
//
//   h = x_0 + ... + x_{n-1} + residual        (fp32, in rank order)
//   rstd = 1 / sqrt(mean(h^2) + eps)
//   y = h * rstd * w                           (rounded once, from the fp32 h)
//
//   n = h * rstd,  g = dy * w
//   dx = rstd * (g - n * mean(g * n)) + dh,    dw = sum over rows of dy * n
//
// Both are bound by HBM: a row is read once into registers, as octets of
// eight neighbouring columns per thread, reduced over its threads (shuffles,
// then one shared-memory exchange) and written once. Sums, the mean and the
// scales are fp32; h is rounded to its type only for the copy that is stored.
#include <cuda_runtime.h>

#include <cmath>
#include <cstdio>

#include "kernels/octet.cuh"
#include "kernels/ophost.h"
#include "kernels/rmsnorm.h"

namespace nb {
namespace {

using namespace octet;

constexpr int kLongThreads = 1024;
constexpr int kRingThreads = 512;
// Threads of a norm's block at most: 64 registers do for one aligned sum and its residual.
__host__ __device__ constexpr int max_threads(bool vec, bool many) { return vec && !many ? 1024 : 512; }

struct Rows {
  const void* p;
  long long outer, inner;
};

// r / inner and r % inner for row numbers below 2^31 by a multiplication
// (Granlund and Montgomery, 1994): q = (mulhi(r, magic) + r) >> shift.
struct RowSplit {
  unsigned inner, magic, shift;
};

struct FwdArgs {
  Rows x[8];
  Rows residual;
  const void* weight;
  void* y;
  float* scale;
  void* h;
  float* rstd;
  long long rows;
  RowSplit split;
  int hidden, parts, group, tpr, groups;
  float eps, inv_hidden;
};

struct BwdArgs {
  Rows dy, h, dh;
  const void* weight;
  const float* rstd;
  void* dx;
  float* partial;  // [blocks][hidden]
  long long rows;
  RowSplit split;
  int hidden, tpr;
  float inv_hidden;
};

// A row's place in every tensor of a call.
struct Row {
  long long outer, inner;

  __device__ __forceinline__ Row(long long r, const RowSplit& s) {
    const unsigned n = unsigned(r), q = (__umulhi(n, s.magic) + n) >> s.shift;
    outer = q;
    inner = n - q * s.inner;
  }
  template <typename T>
  __device__ __forceinline__ const T* of(const Rows& t) const {
    return static_cast<const T*>(t.p) + outer * t.outer + inner * t.inner;
  }
};

// Sum over the threads of one row: `tpr` lanes of a warp (a power of two), or
// the whole block (tpr > 32), whose warps meet in `red`.
__device__ __forceinline__ float row_sum(float s, int tpr, float* red) {
  const int top = tpr < 32 ? tpr : 32;
  for (int o = top >> 1; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  if (tpr <= 32) return s;
  const int warps = tpr >> 5, lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = s;
  __syncthreads();
  s = lane < warps ? red[lane] : 0.0f;
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return s;
}

__device__ __forceinline__ uint32_t row_max(uint32_t m, int tpr, uint32_t* red) {
  const int top = tpr < 32 ? tpr : 32;
  for (int o = top >> 1; o; o >>= 1) m = max(m, __shfl_xor_sync(~0u, m, o));
  if (tpr <= 32) return m;
  const int warps = tpr >> 5, lane = threadIdx.x & 31;
  if (lane == 0) red[threadIdx.x >> 5] = m;
  __syncthreads();
  return __reduce_max_sync(~0u, lane < warps ? red[lane] : 0u);
}

// A thread's K times eight elements of a row: where the first of each eight
// is, how far apart they are, and how much of the row is left from there on.
// The k-th eight of a warp's 32 threads (of a row's `tpr`, if fewer) are 256
// (8 tpr) neighbours; each thread has eight of them in a row (VEC), or every
// 32nd (tpr-th). Without any (left <= 0) it reads the row's first ones and
// drops them.
template <int K, bool VEC>
struct Part {
  int lane, step, at[K], left[K];

  __device__ __forceinline__ Part(int lane_, int tpr, int hidden) : lane(lane_) {
    const int width = tpr < 32 ? tpr : 32, in = lane & (width - 1);
    step = VEC ? 1 : width;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      at[k] = (lane - in + k * tpr) * 8 + (VEC ? in * 8 : in);
      left[k] = hidden - at[k];
      if (left[k] <= 0) at[k] = 0;
    }
  }
};

// A thread's elements of one row of a tensor.
template <typename T, bool VEC, int K>
struct Load {
  Raw<T, VEC> raw[K];

  __device__ __forceinline__ void load(const T* row, const Part<K, VEC>& part) {
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k].load(row + part.at[k], part.step, part.left[k]);
  }
  __device__ __forceinline__ void get(int k, Pair (&f)[4]) const { raw[k].get(f); }
};

__device__ __forceinline__ void add(Pair (&h)[4], const Pair (&f)[4]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) h[j] = h[j] + f[j];
}

__device__ __forceinline__ float sum_of(Pair p) {
  float a, b;
  split(p, a, b);
  return a + b;
}

// Eight values times their scales' reciprocals to e4m3.
template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[8], const float (&inv)[8], int step, int left) {
  float z[8];
#pragma unroll
  for (int j = 0; j < 8; j += 2) split(pair(f[j], f[j + 1]) * pair(inv[j], inv[j + 1]), z[j], z[j + 1]);
  const uint2 q = to_e4m3(z);
  if constexpr (VEC) {
    if (left > 0) *reinterpret_cast<uint2*>(p) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * step < left) p[j * step] = uint8_t((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
  }
}

// 1 / scale, for a scale of at least 2^-126: off by an ulp at most, so that a
// value within that of the middle between two codes may take either.
__device__ __forceinline__ float reciprocal(float scale) { return __fdividef(1.0f, scale); }

// The reciprocals of the scales of groups of 32, 64 or 128 columns, one for each
// of a thread's eight values; the group's first thread stores its scale. `whole`: the
// largest magnitude of the row's part, where a group is wider than that.
template <bool VEC>
__device__ __forceinline__ void group_scales(const FwdArgs& a, const float (&y)[8], uint32_t whole, int tpr,
                                             long long row, int at, int left, float (&inv)[8]) {
  const int width = tpr < 32 ? tpr : 32;
  float* to = a.scale + row * a.groups;
  if constexpr (VEC) {  // a thread's values are in one group, with its neighbours
    uint32_t top = left > 0 ? top_of(y) : 0;
    int lanes = a.group >> 3;
    if (lanes > width) {
      lanes = width;
      top = whole;
    }
    for (int o = lanes >> 1; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
    const float s = scale_of(top), i = reciprocal(s);
    if (left > 0 && (at & (a.group - 1)) == 0) to[unsigned(at) / unsigned(a.group)] = s;
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = i;
  } else {  // a group is `per` neighbouring j of all the row's lanes
    const int per = a.group / width;
    uint32_t top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) top[j] = j * width < left ? magnitude(y[j]) : 0;
    if (per > 8) {
#pragma unroll
      for (int j = 0; j < 8; ++j) top[j] = whole;
    }
#pragma unroll
    for (int half = 1; half < 8; half *= 2)
      if (per > half) {
        uint32_t other[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) other[j] = top[j ^ half];
#pragma unroll
        for (int j = 0; j < 8; ++j) top[j] = max(top[j], other[j]);
      }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      for (int o = width >> 1; o; o >>= 1) top[j] = max(top[j], __shfl_xor_sync(~0u, top[j], o));
      const float s = scale_of(top[j]);
      inv[j] = reciprocal(s);
      const int col = at + j * width;
      if (j * width < left && (col & (a.group - 1)) == 0) to[unsigned(col) / unsigned(a.group)] = s;
    }
  }
}

// One row per tpr threads, in registers: every load is issued before the
// first value is used, and a row's threads meet once (twice with one e4m3
// scale per row). W: the weight's type; MANY: more than one partial sum.
template <typename T, typename W, bool F8, bool VEC, bool MANY, int K>
__global__ void __launch_bounds__(max_threads(VEC, MANY)) norm_kernel(const __grid_constant__ FwdArgs a) {
  __shared__ float red[32];
  __shared__ uint32_t top_red[32];
  const int tpr = a.tpr, hidden = a.hidden;
  const int lane = tpr > 32 ? threadIdx.x : threadIdx.x & (tpr - 1);
  const long long row = tpr > 32 ? (long long)blockIdx.x
                                 : (long long)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < a.rows;  // every thread stays for the shuffles
  const Row from(live ? row : 0, a.split);
  Part<K, VEC> part(lane, tpr, hidden);
  // Four partial sums at a time, with the first of them the residual too.
  constexpr int N = MANY ? 4 : 1;
  Load<T, VEC, K> xv[N], rv;
  Load<W, VEC, K> wv;
  Pair h[K][4], f[4];
#pragma unroll 1
  for (int s0 = 0; s0 < (MANY ? a.parts : 1); s0 += N) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (s0 + i < a.parts) xv[i].load(from.of<T>(a.x[s0 + i]), part);
    if (s0 == 0 && a.residual.p) rv.load(from.of<T>(a.residual), part);
    if (s0 == 0) wv.load(static_cast<const W*>(a.weight), part);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (s0 == 0) {
        xv[0].get(k, h[k]);
      } else {
        xv[0].get(k, f);
        add(h[k], f);
      }
#pragma unroll
      for (int i = 1; i < N; ++i)
        if (s0 + i < a.parts) {
          xv[i].get(k, f);
          add(h[k], f);
        }
    }
  }
  if (a.residual.p) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      rv.get(k, f);
      add(h[k], f);
    }
  }
  if (!live) {
#pragma unroll
    for (int k = 0; k < K; ++k) part.left[k] = 0;
  }
  Pair sum = pair(0.0f, 0.0f);
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (part.left[k] > 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fma(h[k][j], h[k][j], sum);
    }
  const long long out = row * a.hidden;
  if (a.h) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float e[8];
      split(h[k], e);
      store8<T, VEC>(static_cast<T*>(a.h) + out + part.at[k], e, part.step, part.left[k]);
    }
  }
  const float s = row_sum(sum_of(sum), tpr, red);
  const float rstd = rsqrtf(fmaf(s, a.inv_hidden, a.eps));
  if (live && lane == 0) a.rstd[row] = rstd;
  const Pair r2 = pair(rstd, rstd);
  float y[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    wv.get(k, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = h[k][j] * r2 * f[j];
    split(f, y[k]);
  }
  if constexpr (!F8) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      store8<T, VEC>(static_cast<T*>(a.y) + out + part.at[k], y[k], part.step, part.left[k]);
  } else {
    uint32_t most = 0;
    if (a.group == 0 || a.group > 8 * tpr) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (part.left[k] > 0) most = max(most, top_of<VEC>(y[k], part.step, part.left[k]));
    }
    float inv[8];
    if (a.group == 0) {
      const float scale = scale_of(row_max(most, tpr, top_red));
      if (live && lane == 0) a.scale[row] = scale;
#pragma unroll
      for (int j = 0; j < 8; ++j) inv[j] = reciprocal(scale);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (a.group) group_scales<VEC>(a, y[k], most, tpr, row, part.at[k], part.left[k], inv);
      store_e4m3<VEC>(static_cast<uint8_t*>(a.y) + out + part.at[k], y[k], inv, part.step, part.left[k]);
    }
  }
}

// The sum of every partial and the residual at eight elements.
template <typename T, bool VEC>
__device__ __forceinline__ void sum8(const FwdArgs& a, const Row& from, const Part<1, VEC>& part, Pair (&h)[4]) {
  Load<T, VEC, 1> v;
  Pair f[4];
  v.load(from.of<T>(a.x[0]), part);
  v.get(0, h);
#pragma unroll 1
  for (int s = 1; s < a.parts + (a.residual.p ? 1 : 0); ++s) {
    v.load(from.of<T>(s < a.parts ? a.x[s] : a.residual), part);
    v.get(0, f);
    add(h, f);
  }
}

// The turns that a block of kLongThreads takes over a long row: turn k is the
// k-th eight elements of its threads. Whole warps take every turn.
template <bool VEC, typename F>
__device__ __forceinline__ void each_turn(int hidden, F f) {
  const int turns = (hidden + 8 * kLongThreads - 1) / (8 * kLongThreads);
  Part<1, VEC> part(threadIdx.x, kLongThreads, hidden);
  const int first = part.at[0];  // 0 too for a thread without elements in a row below one turn
  for (int k = 0; k < turns; ++k) {
    part.at[0] = first + k * 8 * kLongThreads;
    part.left[0] = hidden - part.at[0];
    if (part.left[0] <= 0) part.at[0] = 0;
    f(part);
  }
}

// Rows that do not fit the registers of a block: the sum is formed again in
// each pass over the row (from L2), and h is written in the last one, so that
// it may still replace an input.
template <typename T, typename W, bool F8, bool VEC>
__global__ void __launch_bounds__(kLongThreads) norm_long_kernel(const __grid_constant__ FwdArgs a) {
  __shared__ float red[32];
  __shared__ uint32_t top_red[32];
  const long long row = blockIdx.x, out = row * a.hidden;
  const Row from(row, a.split);
  const auto normal = [&](const Part<1, VEC>& part, float rstd, const Pair (&h)[4], float (&y)[8]) {
    Load<W, VEC, 1> wv;
    Pair w[4];
    wv.load(static_cast<const W*>(a.weight), part);
    wv.get(0, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = h[j] * pair(rstd, rstd) * w[j];
    split(w, y);
  };
  Pair sum = pair(0.0f, 0.0f);
  each_turn<VEC>(a.hidden, [&](const Part<1, VEC>& part) {
    if (part.left[0] <= 0) return;
    Pair h[4];
    sum8<T, VEC>(a, from, part, h);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fma(h[j], h[j], sum);
  });
  const float s = row_sum(sum_of(sum), kLongThreads, red);
  const float rstd = rsqrtf(fmaf(s, a.inv_hidden, a.eps));
  if (threadIdx.x == 0) a.rstd[row] = rstd;
  float inv[8] = {};
  if (F8 && a.group == 0) {
    uint32_t top = 0;
    each_turn<VEC>(a.hidden, [&](const Part<1, VEC>& part) {
      if (part.left[0] <= 0) return;
      Pair h[4];
      float y[8];
      sum8<T, VEC>(a, from, part, h);
      normal(part, rstd, h, y);
      top = max(top, top_of<VEC>(y, part.step, part.left[0]));
    });
    const float scale = scale_of(row_max(top, kLongThreads, top_red));
    if (threadIdx.x == 0) a.scale[row] = scale;
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = reciprocal(scale);
  }
  each_turn<VEC>(a.hidden, [&](const Part<1, VEC>& part) {
    const int at = part.at[0], left = part.left[0];
    Pair h[4] = {};
    float y[8] = {}, e[8];
    if (left > 0) {
      sum8<T, VEC>(a, from, part, h);
      normal(part, rstd, h, y);
      split(h, e);
      if (a.h) store8<T, VEC>(static_cast<T*>(a.h) + out + at, e, part.step, left);
    }
    if constexpr (F8) {
      if (a.group) group_scales<VEC>(a, y, 0, kLongThreads, row, at, left, inv);
      store_e4m3<VEC>(static_cast<uint8_t*>(a.y) + out + at, y, inv, part.step, left);
    } else {
      store8<T, VEC>(static_cast<T*>(a.y) + out + at, y, part.step, left);
    }
  });
}

// A row of the gradient, from this thread's elements: adds to dw's part and
// stores dx.
template <typename T, typename W, bool VEC, int K, typename In>
__device__ __forceinline__ void finish_grad(const BwdArgs& a, long long row, bool live, const Part<K, VEC>& part,
                                            const In& dy, const In& h, const In& dh, float rstd,
                                            const Load<W, VEC, K>& wv, Pair (&acc)[K][4], float* red) {
  Pair g[K][4], n[K][4], sum = pair(0.0f, 0.0f);
  const Pair r2 = pair(rstd, rstd);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Pair w[4];
    dy.get(k, g[k]);
    h.get(k, n[k]);
    wv.get(k, w);
    if (part.left[k] > 0 && live) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        n[k][j] = n[k][j] * r2;
        acc[k][j] = fma(g[k][j], n[k][j], acc[k][j]);
        g[k][j] = g[k][j] * w[j];
        sum = fma(g[k][j], n[k][j], sum);
      }
    }
  }
  const float c = row_sum(sum_of(sum), a.tpr, red) * -a.inv_hidden;
  const Pair c2 = pair(c, c);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Pair e[4];
    if (a.dh.p) dh.get(k, e);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const Pair t = fma(n[k][j], c2, g[k][j]);
      e[j] = a.dh.p ? fma(t, r2, e[j]) : t * r2;
    }
    float f[8];
    split(e, f);
    store8<T, VEC>(static_cast<T*>(a.dx) + row * a.hidden + part.at[k], f, part.step, live ? part.left[k] : 0);
  }
}

// The block's part of dw: its rows are fixed, and with several rows at once
// its slots are added in order.
template <int K, bool VEC>
__device__ __forceinline__ void store_partial(const BwdArgs& a, const Part<K, VEC>& part, const Pair (&acc)[K][4],
                                              float* slots) {
  const int tpr = a.tpr;
  float* to = a.partial + (long long)blockIdx.x * a.hidden;
  if (tpr <= 32) to = slots + (threadIdx.x / tpr) * a.hidden;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float f[8];
    split(acc[k], f);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * part.step < part.left[k]) to[part.at[k] + j * part.step] = f[j];
  }
  if (tpr <= 32) {
    __syncthreads();
    const int per = blockDim.x / tpr;
    for (int col = threadIdx.x; col < a.hidden; col += blockDim.x) {
      float s = 0.0f;
      for (int q = 0; q < per; ++q) s += slots[q * a.hidden + col];
      a.partial[(long long)blockIdx.x * a.hidden + col] = s;
    }
  }
}

template <int K>
__device__ __forceinline__ void clear(Pair (&acc)[K][4]) {
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[k][j] = pair(0.0f, 0.0f);
}

// Each block walks over rows and keeps its columns' part of dw in registers;
// the parts go to `partial` and dw_kernel adds them in block order.
template <typename T, typename W, bool VEC, int K>
__global__ void __launch_bounds__(kRingThreads) norm_backward_kernel(const __grid_constant__ BwdArgs a) {
  __shared__ float red[2][32];
  __shared__ float slots[256 * 8 * K];
  const int tpr = a.tpr;
  const int lane = tpr > 32 ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int per = tpr > 32 ? 1 : blockDim.x / tpr, slot = tpr > 32 ? 0 : threadIdx.x / tpr;
  const Part<K, VEC> part(lane, tpr, a.hidden);
  Pair acc[K][4];
  Load<W, VEC, K> wv;
  wv.load(static_cast<const W*>(a.weight), part);
  clear<K>(acc);
  const long long stride = (long long)gridDim.x * per;
  int turn = 0;
  for (long long row = (long long)blockIdx.x * per + slot; row - slot < a.rows; row += stride, ++turn) {
    const bool live = row < a.rows;
    const long long r = live ? row : a.rows - 1;
    const Row from(r, a.split);
    Load<T, VEC, K> dy, h, dh;
    dy.load(from.of<T>(a.dy), part);
    h.load(from.of<T>(a.h), part);
    if (a.dh.p) dh.load(from.of<T>(a.dh), part);
    finish_grad<T, W, VEC, K>(a, row, live, part, dy, h, dh, a.rstd[r], wv, acc, red[turn & 1]);
  }
  store_partial<K, VEC>(a, part, acc, slots);
}

// A thread's own ring in shared memory: kStages rows of its octets of a 16-bit
// type, brought by 16-byte asynchronous copies. Only the thread itself reads
// them, so a stage needs no barrier: the thread waits for its own copies.
// Copies of later rows are in flight while a row is reduced, without a
// register held for them.
constexpr int kStages = 4;

template <typename T, int K>
struct Ring {
  uint4* base;
  int sources;

  __device__ __forceinline__ uint4* slot(int stage, int source, int k) const {
    return base + ((stage * sources + source) * K + k) * int(blockDim.x) + threadIdx.x;
  }
  __device__ __forceinline__ void fetch(int stage, int source, const T* row, const Part<K, true>& part) const {
#pragma unroll
    for (int k = 0; k < K; ++k)
      if (part.left[k] > 0)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(
                         uint32_t(__cvta_generic_to_shared(slot(stage, source, k)))),
                     "l"(row + part.at[k])
                     : "memory");
  }
  __device__ __forceinline__ void read(int stage, int source, Load<T, true, K>& o) const {
#pragma unroll
    for (int k = 0; k < K; ++k) o.raw[k].o.v[0] = *slot(stage, source, k);
  }
};

// The same with the next rows on their way (octets on their boundary). A
// thread without an octet or a row reads what the ring happens to hold and
// drops it.
template <typename T, typename W, int K>
__global__ void __launch_bounds__(kRingThreads) norm_backward_ring_kernel(const __grid_constant__ BwdArgs a) {
  extern __shared__ uint4 smem[];
  __shared__ float red[2][32];
  const int tpr = a.tpr;
  const int lane = tpr > 32 ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int per = tpr > 32 ? 1 : blockDim.x / tpr, slot = tpr > 32 ? 0 : threadIdx.x / tpr;
  const Part<K, true> part(lane, tpr, a.hidden);
  const Ring<T, K> ring{smem, a.dh.p ? 3 : 2};
  const long long stride = (long long)gridDim.x * per;
  long long ahead = (long long)blockIdx.x * per + slot;
  float rstds[kStages];  // of the rows on their way
  const auto fetch = [&](int stage, float& rstd) {
    rstd = 0.0f;
    if (ahead < a.rows) {
      const Row from(ahead, a.split);
      ring.fetch(stage, 0, from.of<T>(a.dy), part);
      ring.fetch(stage, 1, from.of<T>(a.h), part);
      if (a.dh.p) ring.fetch(stage, 2, from.of<T>(a.dh), part);
      rstd = a.rstd[ahead];
    }
    ahead += stride;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) fetch(s, rstds[s]);
  Pair acc[K][4];
  Load<W, true, K> wv;
  wv.load(static_cast<const W*>(a.weight), part);
  clear<K>(acc);
  for (long long row = (long long)blockIdx.x * per + slot; row - slot < a.rows;) {
#pragma unroll
    for (int s = 0; s < kStages; ++s) {  // the stage is a constant, so rstds stays in registers
      if (row - slot >= a.rows) break;
      // Into the stage of the row before, whose values this thread has used.
      fetch((s + kStages - 1) % kStages, rstds[(s + kStages - 1) % kStages]);
      asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");
      Load<T, true, K> dy, h, dh;
      ring.read(s, 0, dy);
      ring.read(s, 1, h);
      if (a.dh.p) ring.read(s, 2, dh);
      finish_grad<T, W, true, K>(a, row, row < a.rows, part, dy, h, dh, rstds[s], wv, acc, red[s & 1]);
      row += stride;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  store_partial<K, true>(a, part, acc, reinterpret_cast<float*>(smem));
}

// Long rows: dx with two passes over the row (the second from L2) ...
template <typename T, typename W, bool VEC>
__global__ void __launch_bounds__(kLongThreads) norm_backward_long_kernel(const __grid_constant__ BwdArgs a) {
  __shared__ float red[32];
  const long long row = blockIdx.x;
  const Row from(row, a.split);
  const float rstd = a.rstd[row];
  const Pair r2 = pair(rstd, rstd);
  const auto terms = [&](const Part<1, VEC>& part, Pair (&g)[4], Pair (&n)[4]) {
    Load<T, VEC, 1> dy, h;
    Load<W, VEC, 1> wv;
    Pair w[4];
    dy.load(from.of<T>(a.dy), part);
    h.load(from.of<T>(a.h), part);
    wv.load(static_cast<const W*>(a.weight), part);
    dy.get(0, g);
    h.get(0, n);
    wv.get(0, w);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      n[j] = n[j] * r2;
      g[j] = g[j] * w[j];
    }
  };
  Pair sum = pair(0.0f, 0.0f);
  each_turn<VEC>(a.hidden, [&](const Part<1, VEC>& part) {
    if (part.left[0] <= 0) return;
    Pair g[4], n[4];
    terms(part, g, n);
#pragma unroll
    for (int j = 0; j < 4; ++j) sum = fma(g[j], n[j], sum);
  });
  const float c = row_sum(sum_of(sum), kLongThreads, red) * -a.inv_hidden;
  each_turn<VEC>(a.hidden, [&](const Part<1, VEC>& part) {
    if (part.left[0] <= 0) return;
    Pair g[4], n[4], e[4] = {};
    terms(part, g, n);
    if (a.dh.p) {
      Load<T, VEC, 1> dh;
      dh.load(from.of<T>(a.dh), part);
      dh.get(0, e);
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) e[j] = fma(fma(n[j], pair(c, c), g[j]), r2, e[j]);
    float f[8];
    split(e, f);
    store8<T, VEC>(static_cast<T*>(a.dx) + row * a.hidden + part.at[0], f, part.step, part.left[0]);
  });
}

// ... and dw by columns: block (x, y) adds rows y, y + gridDim.y, ... of its columns.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dw_long_kernel(const __grid_constant__ BwdArgs a) {
  Part<1, VEC> part(threadIdx.x, 256, 256 * 8);
  part.at[0] += blockIdx.x * 256 * 8;
  part.left[0] = a.hidden - part.at[0];
  if (part.left[0] <= 0) return;
  Pair acc[4] = {};
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const Row from(row, a.split);
    const float rstd = a.rstd[row];
    Load<T, VEC, 1> dy, h;
    Pair d[4], n[4];
    dy.load(from.of<T>(a.dy), part);
    h.load(from.of<T>(a.h), part);
    dy.get(0, d);
    h.get(0, n);
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[j] = fma(d[j], n[j] * pair(rstd, rstd), acc[j]);
  }
  float* to = a.partial + (long long)blockIdx.y * a.hidden + part.at[0];
  float f[8];
  split(acc, f);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j * part.step < part.left[0]) to[j * part.step] = f[j];
}

// dw[col] = sum of the blocks' parts: a warp-wide strip of 32 columns per
// block, 32 warps over the parts, then the warps in order.
template <typename W>
__global__ void __launch_bounds__(1024) dw_kernel(const float* partial, int parts, int hidden, W* dw) {
  __shared__ float sum[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  if (col < hidden)
    for (int p = threadIdx.y; p < parts; p += 32) s += partial[(long long)p * hidden + col];
  sum[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sum[threadIdx.x][threadIdx.y];  // transposed: a warp adds one column
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  const int at = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && at < hidden) dw[at] = from_float<W>(s);
}

// ---------------------------------------------------------------- host

constexpr int kRingSmem = 220 * 1024;  // of an SM's shared memory, for the rings of its blocks

// How rows are spread over threads and blocks.
struct Shape {
  int tpr = 0, threads = 0, k = 0;  // k 0: the long variant
  bool ring = false;
  size_t smem = 0;
  long long blocks = 0;
};

int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// `k` octets a thread; rows that take up to 32 threads share a block (and a warp).
void spread(Shape& s, int octets, int k) {
  s.k = k;
  if (octets <= 32 * k) {
    s.tpr = pow2_at_least(int(ceil_div(octets, k)));
    s.threads = 256;
  } else {
    s.tpr = s.threads = int(ceil_div(ceil_div(octets, 32), k)) * 32;
  }
}

long long blocks_of(const Shape& s, long long rows) {
  return s.tpr > 32 ? rows : ceil_div(rows, s.threads / s.tpr);
}

Shape shape_fwd(long long rows, int hidden, int most, int sms) {
  Shape s;
  const int octets = int(ceil_div(hidden, 8));
  s.blocks = rows;
  if (octets > 2 * most) return s;
  int k = octets > most || rows > sms ? 2 : 1;
  spread(s, octets, k);
  s.blocks = blocks_of(s, rows);
  return s;
}

Shape shape_bwd(long long rows, int hidden, int es, int sms) {
  Shape s;
  const int octets = int(ceil_div(hidden, 8));
  if (octets > 2 * kRingThreads) {  // blocks that share dw's columns
    const long long columns = ceil_div(octets, 256), splits = ceil_div(8ll * sms, columns);
    s.blocks = splits < rows ? splits : rows;
    return s;
  }
  spread(s, octets, 2);
  // Sized for three sources, so that the parts of dw do not depend on them.
  s.smem = size_t(kStages) * 3u * 2u * size_t(s.threads) * 16u;
  const int by_threads = kRingThreads / s.threads, by_smem = int(size_t(kRingSmem) / s.smem);
  s.ring = es == 2 && by_smem > 0;
  // As many blocks as are resident, but with four rows each before every SM has more than one.
  const long long fit = (long long)sms * (s.ring && by_smem < by_threads ? by_smem : by_threads);
  const long long most = blocks_of(s, rows), few = ceil_div(most, 4);
  s.blocks = most < sms ? most : few < sms ? sms : few < fit ? few : fit;
  return s;
}

RowSplit split_by(long long inner) {
  RowSplit s;
  s.inner = unsigned(inner);
  s.shift = 0;
  while ((1ull << s.shift) < (unsigned long long)inner) ++s.shift;
  s.magic = unsigned(((1ull << 32) * ((1ull << s.shift) - (unsigned long long)inner)) / (unsigned long long)inner + 1);
  return s;
}

template <typename T, typename W, bool F8, bool VEC>
const void* fwd_kernel(int k, bool many) {
  if (k == 1) return many ? reinterpret_cast<const void*>(norm_kernel<T, W, F8, VEC, true, 1>)
                          : reinterpret_cast<const void*>(norm_kernel<T, W, F8, VEC, false, 1>);
  if (k == 2) return many ? reinterpret_cast<const void*>(norm_kernel<T, W, F8, VEC, true, 2>)
                          : reinterpret_cast<const void*>(norm_kernel<T, W, F8, VEC, false, 2>);
  return reinterpret_cast<const void*>(norm_long_kernel<T, W, F8, VEC>);
}

// The kernels of an input and a weight type.
template <typename T, typename W>
struct Kernels {
  static const void* fwd(bool f8, bool vec, int k, bool many) {
    if (f8) return vec ? fwd_kernel<T, W, true, true>(k, many) : fwd_kernel<T, W, true, false>(k, many);
    return vec ? fwd_kernel<T, W, false, true>(k, many) : fwd_kernel<T, W, false, false>(k, many);
  }
  static const void* bwd(bool vec, const Shape& s) {
    if constexpr (sizeof(T) == 2)
      if (s.k && vec && s.ring) return reinterpret_cast<const void*>(norm_backward_ring_kernel<T, W, 2>);
    if (s.k)
      return vec ? reinterpret_cast<const void*>(norm_backward_kernel<T, W, true, 2>)
                 : reinterpret_cast<const void*>(norm_backward_kernel<T, W, false, 2>);
    return vec ? reinterpret_cast<const void*>(norm_backward_long_kernel<T, W, true>)
               : reinterpret_cast<const void*>(norm_backward_long_kernel<T, W, false>);
  }
};

template <typename F>
const void* by_types(int dtype, bool wf32, F f) {
  switch (dtype) {
    case NB_NORM_FLOAT32: return f(Kernels<float, float>());
    case NB_NORM_FLOAT16: return wf32 ? f(Kernels<__half, float>()) : f(Kernels<__half, __half>());
    default: return wf32 ? f(Kernels<__nv_bfloat16, float>()) : f(Kernels<__nv_bfloat16, __nv_bfloat16>());
  }
}

cudaError_t launch(const void* fn, const Shape& s, bool ring, unsigned blocks, void** argv, cudaStream_t stream) {
  size_t smem = 0;
  if (ring) {
    smem = s.smem;
    const cudaError_t e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem));
    if (e != cudaSuccess) return e;
  }
  return cudaLaunchKernel(fn, dim3(blocks), dim3(unsigned(s.k ? s.threads : kLongThreads)), argv, smem, stream);
}

template <typename T>
const void* pick_dw_long(bool vec) {
  return vec ? reinterpret_cast<const void*>(dw_long_kernel<T, true>)
             : reinterpret_cast<const void*>(dw_long_kernel<T, false>);
}

int size_of(int dtype) {
  switch (dtype) {
    case NB_NORM_FLOAT16:
    case NB_NORM_BFLOAT16: return 2;
    case NB_NORM_FLOAT32: return 4;
    default: return 0;
  }
}

constexpr char kNegative[] = "bad arguments: negative stride";

// Whether rows at these strides start on the boundary of an octet (element
// alignment is checked apart).
bool octets_fit(const void* p, long long outer, long long inner, int es) {
  const uintptr_t unit = uintptr_t(es) * 8;
  return reinterpret_cast<uintptr_t>(p) % unit == 0 && outer % 8 == 0 && inner % 8 == 0;
}

bool misplaced(const void* p, int es) { return !p || reinterpret_cast<uintptr_t>(p) % uintptr_t(es); }

// Everything that both directions take. Returns the message of a refusal.
const char* check_common(long long rows, long long inner, int hidden, int dtype, int weight_dtype, const void* weight) {
  if (rows < 0 || inner < 1 || (rows && rows % inner)) return "bad arguments: rows must be a multiple of inner >= 1";
  if (hidden < 1 || hidden > (1 << 24)) return "bad arguments: hidden must be 1 to 16777216";
  if (rows > (1ll << 31) - 1) return "bad arguments: more than 2147483647 rows";
  if (!size_of(dtype)) return "bad arguments: dtype must be ncclFloat16, ncclFloat32 or ncclBfloat16";
  if (weight_dtype != NB_NORM_FLOAT32 && weight_dtype != dtype)
    return "bad arguments: the weight's type is the input's or ncclFloat32";
  if (misplaced(weight, size_of(weight_dtype))) return "bad arguments: null or misaligned weight";
  return nullptr;
}

}  // namespace
}  // namespace nb

using namespace nb;

extern "C" int nb_add_rms_norm(const nb_norm_t* a, void* stream, char* err, size_t errcap) {
  op_message(err, errcap, "");
  if (!a) return op_refuse(err, errcap, "bad arguments: null");
  if (const char* why = check_common(a->rows, a->inner, a->hidden, a->dtype, a->weight_dtype, a->weight))
    return op_refuse(err, errcap, why);
  const int es = size_of(a->dtype);
  const bool f8 = a->out_dtype == NB_NORM_FLOAT8E4M3;
  if (!f8 && a->out_dtype != a->dtype)
    return op_refuse(err, errcap, "bad arguments: the output's type is the input's or ncclFloat8e4m3");
  if (a->parts < 1 || a->parts > 8) return op_refuse(err, errcap, "bad arguments: 1 to 8 partial sums");
  if (f8 ? a->group != 0 && a->group != 32 && a->group != 64 && a->group != 128 : a->group != 0)
    return op_refuse(err, errcap, "bad arguments: group is 0, or with e4m3 output 32, 64 or 128");
  if (!(a->eps > 0.0f) || !std::isfinite(a->eps)) return op_refuse(err, errcap, "bad arguments: eps must be positive");
  if (a->rows == 0) return 0;
  for (int i = 0; i < a->parts; ++i)
    if (misplaced(a->x[i], es)) return op_refuse(err, errcap, "bad arguments: null or misaligned input");
  if (a->residual && misplaced(a->residual, es)) return op_refuse(err, errcap, "bad arguments: misaligned residual");
  if (misplaced(a->y, f8 ? 1 : es) || (a->h && misplaced(a->h, es)) || misplaced(a->rstd, 4) ||
      (f8 && misplaced(a->scale, 4)))
    return op_refuse(err, errcap, "bad arguments: null or misaligned output");
  OpDevice dev(a->device);
  if (dev.error()) return op_refuse(err, errcap, "cannot use the device", int(dev.error()));

  FwdArgs k{};
  bool vec = a->hidden % 8 == 0 && octets_fit(a->weight, 0, 0, size_of(a->weight_dtype));
  for (int i = 0; i < a->parts; ++i) {
    if (a->x_outer[i] < 0 || a->x_inner[i] < 0) return op_refuse(err, errcap, kNegative);
    k.x[i] = {a->x[i], a->x_outer[i], a->x_inner[i]};
    vec = vec && octets_fit(a->x[i], a->x_outer[i], a->x_inner[i], es);
  }
  if (a->r_outer < 0 || a->r_inner < 0) return op_refuse(err, errcap, kNegative);
  k.residual = {a->residual, a->r_outer, a->r_inner};
  if (a->residual) vec = vec && octets_fit(a->residual, a->r_outer, a->r_inner, es);
  vec = vec && octets_fit(a->y, 0, 0, f8 ? 1 : es) && (!a->h || octets_fit(a->h, 0, 0, es));
  const Shape s = shape_fwd(a->rows, a->hidden, max_threads(vec, a->parts > 1), dev.sms());
  k.weight = a->weight;
  k.y = a->y;
  k.scale = a->scale;
  k.h = a->h;
  k.rstd = a->rstd;
  k.rows = a->rows;
  k.split = split_by(a->inner);
  k.hidden = a->hidden;
  k.parts = a->parts;
  k.group = a->group;
  k.groups = a->group ? (a->hidden + a->group - 1) / a->group : 1;
  k.tpr = s.tpr;
  k.eps = a->eps;
  k.inv_hidden = 1.0f / float(a->hidden);
  const void* fn = by_types(a->dtype, a->weight_dtype == NB_NORM_FLOAT32,
                            [&](auto kernels) { return kernels.fwd(f8, vec, s.k, a->parts > 1); });
  void* argv[] = {&k};
  const cudaError_t e = launch(fn, s, false, unsigned(s.blocks), argv, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : op_refuse(err, errcap, "launch of the norm failed", int(e));
}

extern "C" uint64_t nb_add_rms_norm_backward_workspace(int device, int64_t rows, int hidden, int dtype) {
  const int es = size_of(dtype);
  OpDevice dev(device);
  if (dev.error() || rows < 0 || hidden < 1 || !es) return 0;
  return uint64_t(shape_bwd(rows, hidden, es, dev.sms()).blocks) * uint64_t(hidden) * sizeof(float);
}

extern "C" int nb_add_rms_norm_backward(const nb_norm_grad_t* a, void* stream, char* err, size_t errcap) {
  op_message(err, errcap, "");
  if (!a) return op_refuse(err, errcap, "bad arguments: null");
  if (const char* why = check_common(a->rows, a->inner, a->hidden, a->dtype, a->weight_dtype, a->weight))
    return op_refuse(err, errcap, why);
  const int es = size_of(a->dtype), ws = size_of(a->weight_dtype);
  if (misplaced(a->dweight, ws)) return op_refuse(err, errcap, "bad arguments: null or misaligned dweight");
  if (a->rows && (misplaced(a->dy, es) || misplaced(a->h, es) || misplaced(a->dx, es) || misplaced(a->rstd, 4) ||
                  (a->dh && misplaced(a->dh, es))))
    return op_refuse(err, errcap, "bad arguments: null or misaligned tensor");
  OpDevice dev(a->device);
  if (dev.error()) return op_refuse(err, errcap, "cannot use the device", int(dev.error()));
  const Shape s = shape_bwd(a->rows, a->hidden, es, dev.sms());
  const long long parts = s.blocks;
  if (a->rows && (misplaced(a->workspace, 4) || a->workspace_bytes < uint64_t(parts) * uint64_t(a->hidden) * 4))
    return op_refuse(err, errcap, "bad arguments: the workspace is too small");

  BwdArgs k{};
  if (a->dy_outer < 0 || a->dy_inner < 0 || a->h_outer < 0 || a->h_inner < 0 || a->dh_outer < 0 || a->dh_inner < 0)
    return op_refuse(err, errcap, kNegative);
  k.dy = {a->dy, a->dy_outer, a->dy_inner};
  k.h = {a->h, a->h_outer, a->h_inner};
  k.dh = {a->dh, a->dh_outer, a->dh_inner};
  k.weight = a->weight;
  k.rstd = a->rstd;
  k.dx = a->dx;
  k.partial = a->workspace;
  k.rows = a->rows;
  k.split = split_by(a->inner);
  k.hidden = a->hidden;
  k.tpr = s.tpr;
  k.inv_hidden = 1.0f / float(a->hidden);
  const bool vec = a->hidden % 8 == 0 && octets_fit(a->weight, 0, 0, ws) &&
                   octets_fit(a->dy, a->dy_outer, a->dy_inner, es) && octets_fit(a->h, a->h_outer, a->h_inner, es) &&
                   (!a->dh || octets_fit(a->dh, a->dh_outer, a->dh_inner, es)) && octets_fit(a->dx, 0, 0, es);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* argv[] = {&k};
  cudaError_t e = cudaSuccess;
  if (a->rows) {
    const void* fn = by_types(a->dtype, a->weight_dtype == NB_NORM_FLOAT32,
                              [&](auto kernels) { return kernels.bwd(vec, s); });
    e = launch(fn, s, s.ring && vec, unsigned(s.k ? parts : a->rows), argv, st);
    if (e == cudaSuccess && !s.k) {
      fn = a->dtype == NB_NORM_FLOAT32   ? pick_dw_long<float>(vec)
           : a->dtype == NB_NORM_FLOAT16 ? pick_dw_long<__half>(vec)
                                         : pick_dw_long<__nv_bfloat16>(vec);
      const unsigned columns = unsigned(((a->hidden + 7) / 8 + 255) / 256);
      e = cudaLaunchKernel(fn, dim3(columns, unsigned(parts)), dim3(256), argv, 0, st);
    }
  }
  if (e == cudaSuccess) {  // without rows: no parts, dw = 0
    const void* fn = a->weight_dtype == NB_NORM_FLOAT32   ? reinterpret_cast<const void*>(dw_kernel<float>)
                     : a->weight_dtype == NB_NORM_FLOAT16 ? reinterpret_cast<const void*>(dw_kernel<__half>)
                                                          : reinterpret_cast<const void*>(dw_kernel<__nv_bfloat16>);
    const float* partial = a->workspace;
    int count = int(parts), hidden = a->hidden;
    void* dw = a->dweight;
    void* dargv[] = {&partial, &count, &hidden, &dw};
    e = cudaLaunchKernel(fn, dim3(unsigned((hidden + 31) / 32)), dim3(32, 32), dargv, 0, st);
  }
  return e == cudaSuccess ? 0 : op_refuse(err, errcap, "launch of the norm's gradient failed", int(e));
}
