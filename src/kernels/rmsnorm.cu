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

struct Rows {
  const void* p;
  long long outer, inner;
};

struct FwdArgs {
  Rows x[8];
  Rows residual;
  const void* weight;
  void* y;
  float* scale;
  void* h;
  float* rstd;
  long long rows, inner;
  int hidden, parts, wf32, group, tpr, groups;
  float eps;
};

struct BwdArgs {
  Rows dy, h, dh;
  const void* weight;
  const float* rstd;
  void* dx;
  float* partial;  // [blocks][hidden]
  long long rows, inner;
  int hidden, wf32, tpr;
};

template <typename T>
__device__ __forceinline__ const T* row_of(const Rows& r, long long row, long long inner) {
  // One row dimension is the usual case and needs no division.
  if (inner == 1) return static_cast<const T*>(r.p) + row * r.outer;
  const long long o = row / inner;
  return static_cast<const T*>(r.p) + o * r.outer + (row - o * inner) * r.inner;
}

template <typename T, bool VEC>
__device__ __forceinline__ void load_weight(const void* w, int wf32, int col, int left, float (&f)[8]) {
  if (wf32) unpack<float>(load<float, VEC>(static_cast<const float*>(w) + col, left), f);
  else unpack<T>(load<T, VEC>(static_cast<const T*>(w) + col, left), f);
}

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

// The sum of every partial and the residual at one octet.
template <typename T, bool VEC>
__device__ __forceinline__ void sum_octet(const FwdArgs& a, long long row, int col, int left, float (&h)[8]) {
  unpack<T>(load<T, VEC>(row_of<T>(a.x[0], row, a.inner) + col, left), h);
#pragma unroll 1
  for (int s = 1; s < a.parts; ++s) {
    float f[8];
    unpack<T>(load<T, VEC>(row_of<T>(a.x[s], row, a.inner) + col, left), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] += f[j];
  }
  if (a.residual.p) {
    float f[8];
    unpack<T>(load<T, VEC>(row_of<T>(a.residual, row, a.inner) + col, left), f);
#pragma unroll
    for (int j = 0; j < 8; ++j) h[j] += f[j];
  }
}

template <bool VEC>
__device__ __forceinline__ void store_e4m3(uint8_t* p, const float (&f)[8], float inv, int left) {
  float z[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) z[j] = f[j] * inv;
  const uint2 q = to_e4m3(z);
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(p) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = uint8_t((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
  }
}

// The scale of each group of 32, 64 or 128 columns (neighbouring octets are
// held by neighbouring lanes), stored by the group's first lane.
__device__ __forceinline__ float group_scale(const FwdArgs& a, uint32_t top, int tpr, long long row, int col,
                                             bool here) {
  int lanes = a.group >> 3;
  if (lanes > tpr) lanes = tpr;  // the row is shorter than the group
  for (int o = lanes >> 1; o; o >>= 1) top = max(top, __shfl_xor_sync(~0u, top, o));
  const float s = scale_of(top);
  if (here && (col % a.group) == 0) a.scale[row * a.groups + col / a.group] = s;
  return s;
}

// K octets per thread, the row in registers. Octet k of thread t is t + k * tpr.
template <typename T, bool F8, bool VEC, int K>
__global__ void __launch_bounds__(K <= 2 ? 1024 : 512) norm_kernel(const __grid_constant__ FwdArgs a) {
  __shared__ float red[32];
  __shared__ uint32_t top_red[32];
  const int tpr = a.tpr;
  const int lane = tpr > 32 ? threadIdx.x : threadIdx.x & (tpr - 1);
  const long long row = tpr > 32 ? (long long)blockIdx.x
                                 : (long long)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < a.rows;  // every thread stays for the shuffles
  float h[K][8], s = 0.0f;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int col = (lane + k * tpr) * 8, left = live ? a.hidden - col : 0;
    if (left > 0) {
      sum_octet<T, VEC>(a, row, col, left, h[k]);
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) h[k][j] = 0.0f;
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(h[k][j], h[k][j], s);
  }
  float w[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int col = (lane + k * tpr) * 8, left = live ? a.hidden - col : 0;
    if (left > 0) load_weight<T, VEC>(a.weight, a.wf32, col, left, w[k]);
    else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[k][j] = 0.0f;
    }
  }
  if (a.h) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * tpr) * 8, left = live ? a.hidden - col : 0;
      if (left > 0) store<T, VEC>(static_cast<T*>(a.h) + row * a.hidden + col, h[k], left);
    }
  }
  s = row_sum(s, tpr, red);
  const float rstd = 1.0f / sqrtf(s / float(a.hidden) + a.eps);
  if (live && lane == 0) a.rstd[row] = rstd;
  uint32_t top = 0;
#pragma unroll
  for (int k = 0; k < K; ++k)
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      h[k][j] = h[k][j] * rstd * w[k][j];
      if constexpr (F8) top = max(top, magnitude(h[k][j]));
    }
  if constexpr (!F8) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * tpr) * 8, left = live ? a.hidden - col : 0;
      if (left > 0) store<T, VEC>(static_cast<T*>(a.y) + row * a.hidden + col, h[k], left);
    }
  } else {
    float inv = 0.0f;
    if (a.group == 0) {
      const float scale = scale_of(row_max(top, tpr, top_red));
      if (live && lane == 0) a.scale[row] = scale;
      inv = 1.0f / scale;
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * tpr) * 8, left = live ? a.hidden - col : 0;
      if (a.group) {
        top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude(h[k][j]));
        inv = 1.0f / group_scale(a, top, tpr, row, col, left > 0);
      }
      if (left > 0) store_e4m3<VEC>(static_cast<uint8_t*>(a.y) + row * a.hidden + col, h[k], inv, left);
    }
  }
}

// Rows that do not fit the registers of a block: the sum is formed again in
// each pass over the row (from L2), and h is written in the last one, so that
// it may still replace an input.
template <typename T, bool F8, bool VEC>
__global__ void __launch_bounds__(kLongThreads) norm_long_kernel(const __grid_constant__ FwdArgs a) {
  __shared__ float red[32];
  __shared__ uint32_t top_red[32];
  const long long row = blockIdx.x;
  // Whole warps take every turn, for the shuffles of a group's scale.
  const int turns = (a.hidden + 8 * kLongThreads - 1) / (8 * kLongThreads);
  float s = 0.0f;
  for (int k = 0; k < turns; ++k) {
    const int col = (k * kLongThreads + threadIdx.x) * 8, left = a.hidden - col;
    if (left <= 0) continue;
    float h[8];
    sum_octet<T, VEC>(a, row, col, left, h);
#pragma unroll
    for (int j = 0; j < 8; ++j) s = fmaf(h[j], h[j], s);
  }
  s = row_sum(s, kLongThreads, red);
  const float rstd = 1.0f / sqrtf(s / float(a.hidden) + a.eps);
  if (threadIdx.x == 0) a.rstd[row] = rstd;
  float inv = 0.0f;
  if (F8 && a.group == 0) {
    uint32_t top = 0;
    for (int k = 0; k < turns; ++k) {
      const int col = (k * kLongThreads + threadIdx.x) * 8, left = a.hidden - col;
      if (left <= 0) continue;
      float h[8], w[8];
      sum_octet<T, VEC>(a, row, col, left, h);
      load_weight<T, VEC>(a.weight, a.wf32, col, left, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) top = max(top, magnitude(h[j] * rstd * w[j]));
    }
    const float scale = scale_of(row_max(top, kLongThreads, top_red));
    if (threadIdx.x == 0) a.scale[row] = scale;
    inv = 1.0f / scale;
  }
  for (int k = 0; k < turns; ++k) {
    const int col = (k * kLongThreads + threadIdx.x) * 8, left = a.hidden - col;
    float h[8] = {}, w[8];
    if (left > 0) {
      sum_octet<T, VEC>(a, row, col, left, h);
      if (a.h) store<T, VEC>(static_cast<T*>(a.h) + row * a.hidden + col, h, left);
      load_weight<T, VEC>(a.weight, a.wf32, col, left, w);
#pragma unroll
      for (int j = 0; j < 8; ++j) h[j] = h[j] * rstd * w[j];
    }
    if constexpr (F8) {
      if (a.group) {
        uint32_t top = 0;
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, magnitude(h[j]));
        inv = 1.0f / group_scale(a, top, kLongThreads, row, col, left > 0);
      }
      if (left > 0) store_e4m3<VEC>(static_cast<uint8_t*>(a.y) + row * a.hidden + col, h, inv, left);
    } else {
      if (left > 0) store<T, VEC>(static_cast<T*>(a.y) + row * a.hidden + col, h, left);
    }
  }
}

// Each block walks over rows and keeps its columns' part of dw in registers
// (fixed rows per block, so the sum's order is fixed); the parts go to
// `partial` and dw_kernel adds them in block order.
template <typename T, bool VEC, int K>
__global__ void __launch_bounds__(1024) norm_backward_kernel(const __grid_constant__ BwdArgs a) {
  __shared__ float red[2][32];
  __shared__ float slots[256 * 8];
  const int tpr = a.tpr;
  const int lane = tpr > 32 ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int per = tpr > 32 ? 1 : blockDim.x / tpr, slot = tpr > 32 ? 0 : threadIdx.x / tpr;
  float acc[K][8], w[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    const int col = (lane + k * tpr) * 8, left = a.hidden - col;
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[k][j] = w[k][j] = 0.0f;
    if (left > 0) load_weight<T, VEC>(a.weight, a.wf32, col, left, w[k]);
  }
  int turn = 0;
  for (long long base = (long long)blockIdx.x * per; base < a.rows; base += (long long)gridDim.x * per) {
    const long long row = base + slot;
    const bool live = row < a.rows;
    Oct<T> dy[K], h[K], dh[K];
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * tpr) * 8, left = live ? a.hidden - col : 0;
      dy[k] = h[k] = dh[k] = Oct<T>{};
      if (left > 0) {
        dy[k] = load<T, VEC>(row_of<T>(a.dy, row, a.inner) + col, left);
        h[k] = load<T, VEC>(row_of<T>(a.h, row, a.inner) + col, left);
        if (a.dh.p) dh[k] = load<T, VEC>(row_of<T>(a.dh, row, a.inner) + col, left);
      }
    }
    const float rstd = live ? a.rstd[row] : 0.0f;
    float c = 0.0f;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      float d[8], n[8];
      unpack<T>(dy[k], d);
      unpack<T>(h[k], n);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        n[j] *= rstd;
        acc[k][j] = fmaf(d[j], n[j], acc[k][j]);
        c = fmaf(d[j] * w[k][j], n[j], c);
      }
    }
    c = row_sum(c, tpr, red[turn & 1]) / float(a.hidden);
    ++turn;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * tpr) * 8, left = live ? a.hidden - col : 0;
      if (left <= 0) continue;
      float d[8], n[8], e[8], out[8];
      unpack<T>(dy[k], d);
      unpack<T>(h[k], n);
      unpack<T>(dh[k], e);
#pragma unroll
      for (int j = 0; j < 8; ++j) out[j] = fmaf(rstd, d[j] * w[k][j] - n[j] * rstd * c, e[j]);
      store<T, VEC>(static_cast<T*>(a.dx) + row * a.hidden + col, out, left);
    }
  }
  float* to = a.partial + (long long)blockIdx.x * a.hidden;
  if (tpr > 32) {
#pragma unroll
    for (int k = 0; k < K; ++k) {
      const int col = (lane + k * tpr) * 8;
#pragma unroll
      for (int j = 0; j < 8; ++j)
        if (col + j < a.hidden) to[col + j] = acc[k][j];
    }
  } else {  // several rows at once: add the block's slots in order
#pragma unroll
    for (int j = 0; j < 8; ++j) slots[threadIdx.x * 8 + j] = acc[0][j];
    __syncthreads();
    for (int col = threadIdx.x; col < a.hidden; col += blockDim.x) {
      float s = 0.0f;
      for (int q = 0; q < per; ++q) s += slots[q * tpr * 8 + col];
      to[col] = s;
    }
  }
}

// Long rows: dx with two passes over the row (the second from L2) ...
template <typename T, bool VEC>
__global__ void __launch_bounds__(kLongThreads) norm_backward_long_kernel(const __grid_constant__ BwdArgs a) {
  __shared__ float red[32];
  const long long row = blockIdx.x;
  const float rstd = a.rstd[row];
  float c = 0.0f;
  for (int col = threadIdx.x * 8; col < a.hidden; col += kLongThreads * 8) {
    const int left = a.hidden - col;
    float d[8], n[8], w[8];
    unpack<T>(load<T, VEC>(row_of<T>(a.dy, row, a.inner) + col, left), d);
    unpack<T>(load<T, VEC>(row_of<T>(a.h, row, a.inner) + col, left), n);
    load_weight<T, VEC>(a.weight, a.wf32, col, left, w);
#pragma unroll
    for (int j = 0; j < 8; ++j) c = fmaf(d[j] * w[j], n[j] * rstd, c);
  }
  c = row_sum(c, kLongThreads, red) / float(a.hidden);
  for (int col = threadIdx.x * 8; col < a.hidden; col += kLongThreads * 8) {
    const int left = a.hidden - col;
    float d[8], n[8], w[8], e[8] = {}, out[8];
    unpack<T>(load<T, VEC>(row_of<T>(a.dy, row, a.inner) + col, left), d);
    unpack<T>(load<T, VEC>(row_of<T>(a.h, row, a.inner) + col, left), n);
    load_weight<T, VEC>(a.weight, a.wf32, col, left, w);
    if (a.dh.p) unpack<T>(load<T, VEC>(row_of<T>(a.dh, row, a.inner) + col, left), e);
#pragma unroll
    for (int j = 0; j < 8; ++j) out[j] = fmaf(rstd, d[j] * w[j] - n[j] * rstd * c, e[j]);
    store<T, VEC>(static_cast<T*>(a.dx) + row * a.hidden + col, out, left);
  }
}

// ... and dw by columns: block (x, y) adds rows y, y + gridDim.y, ... of its columns.
template <typename T, bool VEC>
__global__ void __launch_bounds__(256) dw_long_kernel(const __grid_constant__ BwdArgs a) {
  const int col = (blockIdx.x * 256 + threadIdx.x) * 8, left = a.hidden - col;
  if (left <= 0) return;
  float acc[8] = {};
  for (long long row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float rstd = a.rstd[row];
    float d[8], n[8];
    unpack<T>(load<T, VEC>(row_of<T>(a.dy, row, a.inner) + col, left), d);
    unpack<T>(load<T, VEC>(row_of<T>(a.h, row, a.inner) + col, left), n);
#pragma unroll
    for (int j = 0; j < 8; ++j) acc[j] = fmaf(d[j], n[j] * rstd, acc[j]);
  }
  float* to = a.partial + (long long)blockIdx.y * a.hidden + col;
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (j < left) to[j] = acc[j];
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

// How a row is spread over threads.
struct Shape {
  int tpr = 0, threads = 0, k = 0;  // k 0: the long variant
  long long rows_per_block = 1;
};

int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

Shape shape_fwd(long long rows, int hidden, int sms) {
  Shape s;
  const int octets = (hidden + 7) / 8;
  if (octets <= 32) {  // several rows per warp or block
    s.tpr = pow2_at_least(octets);
    s.threads = 256;
    s.k = 1;
    s.rows_per_block = 256 / s.tpr;
    return s;
  }
  if (octets > 2048) return s;
  const int need = (octets + 31) / 32 * 32;
  s.k = octets <= 512 || (octets <= 1024 && rows <= sms) ? 1 : octets <= 1024 ? 2 : 4;
  s.tpr = s.threads = (need / 32 + s.k - 1) / s.k * 32;
  return s;
}

Shape shape_bwd(int hidden) {
  Shape s;
  const int octets = (hidden + 7) / 8;
  if (octets <= 32) {
    s.tpr = pow2_at_least(octets);
    s.threads = 256;
    s.k = 1;
    s.rows_per_block = 256 / s.tpr;
    return s;
  }
  if (octets > 2048) return s;
  s.k = octets <= 1024 ? 1 : 2;
  s.tpr = s.threads = ((octets + 31) / 32 + s.k - 1) / s.k * 32;
  return s;
}

// Blocks that share dw, and so the parts of the workspace.
long long backward_blocks(long long rows, int hidden, int sms) {
  const Shape s = shape_bwd(hidden);
  if (!s.k) {
    const long long columns = ((hidden + 7) / 8 + 255) / 256;
    long long splits = (8ll * sms + columns - 1) / columns;
    return splits < rows ? splits : rows;
  }
  const long long want = (rows + s.rows_per_block - 1) / s.rows_per_block;
  const long long fit = (long long)sms * (2048 / s.threads);
  return want < fit ? want : fit;
}

template <typename T, bool F8, bool VEC>
const void* fwd_kernel(int k) {
  switch (k) {
    case 1: return reinterpret_cast<const void*>(norm_kernel<T, F8, VEC, 1>);
    case 2: return reinterpret_cast<const void*>(norm_kernel<T, F8, VEC, 2>);
    case 4: return reinterpret_cast<const void*>(norm_kernel<T, F8, VEC, 4>);
    default: return reinterpret_cast<const void*>(norm_long_kernel<T, F8, VEC>);
  }
}

template <typename T>
const void* pick_fwd(bool f8, bool vec, int k) {
  if (f8) return vec ? fwd_kernel<T, true, true>(k) : fwd_kernel<T, true, false>(k);
  return vec ? fwd_kernel<T, false, true>(k) : fwd_kernel<T, false, false>(k);
}

template <typename T>
const void* pick_bwd(bool vec, int k) {
  if (k == 1) return vec ? reinterpret_cast<const void*>(norm_backward_kernel<T, true, 1>)
                         : reinterpret_cast<const void*>(norm_backward_kernel<T, false, 1>);
  if (k == 2) return vec ? reinterpret_cast<const void*>(norm_backward_kernel<T, true, 2>)
                         : reinterpret_cast<const void*>(norm_backward_kernel<T, false, 2>);
  return vec ? reinterpret_cast<const void*>(norm_backward_long_kernel<T, true>)
             : reinterpret_cast<const void*>(norm_backward_long_kernel<T, false>);
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

  const Shape s = shape_fwd(a->rows, a->hidden, dev.sms());
  FwdArgs k{};
  bool vec = a->hidden % 8 == 0 && octets_fit(a->weight, 0, 0, size_of(a->weight_dtype));
  for (int i = 0; i < a->parts; ++i) {
    k.x[i] = {a->x[i], a->x_outer[i], a->x_inner[i]};
    vec = vec && octets_fit(a->x[i], a->x_outer[i], a->x_inner[i], es);
  }
  k.residual = {a->residual, a->r_outer, a->r_inner};
  if (a->residual) vec = vec && octets_fit(a->residual, a->r_outer, a->r_inner, es);
  vec = vec && octets_fit(a->y, 0, 0, f8 ? 1 : es) && (!a->h || octets_fit(a->h, 0, 0, es));
  k.weight = a->weight;
  k.y = a->y;
  k.scale = a->scale;
  k.h = a->h;
  k.rstd = a->rstd;
  k.rows = a->rows;
  k.inner = a->inner;
  k.hidden = a->hidden;
  k.parts = a->parts;
  k.wf32 = a->weight_dtype == NB_NORM_FLOAT32;
  k.group = a->group;
  k.groups = a->group ? (a->hidden + a->group - 1) / a->group : 1;
  k.tpr = s.k ? s.tpr : kLongThreads;
  k.eps = a->eps;
  const void* fn = a->dtype == NB_NORM_FLOAT32   ? pick_fwd<float>(f8, vec, s.k)
                   : a->dtype == NB_NORM_FLOAT16 ? pick_fwd<__half>(f8, vec, s.k)
                                                 : pick_fwd<__nv_bfloat16>(f8, vec, s.k);
  void* argv[] = {&k};
  const unsigned blocks = unsigned((a->rows + s.rows_per_block - 1) / s.rows_per_block);
  const cudaError_t e = cudaLaunchKernel(fn, dim3(blocks), dim3(s.k ? s.threads : kLongThreads), argv, 0,
                                         static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : op_refuse(err, errcap, "launch of the norm failed", int(e));
}

extern "C" uint64_t nb_add_rms_norm_backward_workspace(int device, int64_t rows, int hidden) {
  OpDevice dev(device);
  if (dev.error() || rows < 0 || hidden < 1) return 0;
  return uint64_t(backward_blocks(rows, hidden, dev.sms())) * uint64_t(hidden) * sizeof(float);
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
  const long long parts = backward_blocks(a->rows, a->hidden, dev.sms());
  if (a->rows && (misplaced(a->workspace, 4) || a->workspace_bytes < uint64_t(parts) * uint64_t(a->hidden) * 4))
    return op_refuse(err, errcap, "bad arguments: the workspace is too small");

  const Shape s = shape_bwd(a->hidden);
  BwdArgs k{};
  k.dy = {a->dy, a->dy_outer, a->dy_inner};
  k.h = {a->h, a->h_outer, a->h_inner};
  k.dh = {a->dh, a->dh_outer, a->dh_inner};
  k.weight = a->weight;
  k.rstd = a->rstd;
  k.dx = a->dx;
  k.partial = a->workspace;
  k.rows = a->rows;
  k.inner = a->inner;
  k.hidden = a->hidden;
  k.wf32 = a->weight_dtype == NB_NORM_FLOAT32;
  k.tpr = s.tpr;
  const bool vec = a->hidden % 8 == 0 && octets_fit(a->weight, 0, 0, ws) &&
                   octets_fit(a->dy, a->dy_outer, a->dy_inner, es) && octets_fit(a->h, a->h_outer, a->h_inner, es) &&
                   (!a->dh || octets_fit(a->dh, a->dh_outer, a->dh_inner, es)) && octets_fit(a->dx, 0, 0, es);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* argv[] = {&k};
  cudaError_t e = cudaSuccess;
  if (a->rows) {
    const void* fn = a->dtype == NB_NORM_FLOAT32   ? pick_bwd<float>(vec, s.k)
                     : a->dtype == NB_NORM_FLOAT16 ? pick_bwd<__half>(vec, s.k)
                                                   : pick_bwd<__nv_bfloat16>(vec, s.k);
    const unsigned blocks = unsigned(s.k ? parts : a->rows);
    e = cudaLaunchKernel(fn, dim3(blocks), dim3(s.k ? s.threads : kLongThreads), argv, 0, st);
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
