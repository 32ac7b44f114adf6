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
#include <type_traits>
#include <cstdio>

#include "kernels/octet.cuh"
#include "kernels/ophost.h"
#include "kernels/rmsnorm.h"

namespace nb {
namespace {

using namespace octet;

constexpr int kLongThreads = 1024;
// A block of the gradient's kernels at most: 128 registers each (with 102 the
// ring's spill, and took 148 us instead of 88); and of the staged ones, whose two
// blocks an SM for up to 5120 columns have 51 or 102.
constexpr int kRingThreads = 512;
constexpr int kStagedThreads = 640;
constexpr int kAll = 1 << 30;  // as what is left of a row: a store to shared memory that has room for everything

// Registers of a thread of the norm's kernel. A row's loads, its sum and its
// stores follow one another, so what keeps HBM busy is how many rows an SM holds,
// and these decide that (see shape_fwd, which picks a variant; times there). es:
// bytes of an input's element.
__host__ __device__ constexpr int norm_registers(int es, int at_once, int k, bool pair, bool lean) {
  if (es == 4 || k == 1) return at_once == 1 ? 64 : 128;
  return at_once == 4 ? (lean ? 72 : 80) : at_once == 2 ? (pair ? 64 : 56) : lean ? 40 : 48;
}

// Where the weight is loaded behind the row's sum. Of 16-bit rows an fp32 one
// takes a third of the registers: 16384 x 5120 bf16 to e4m3 in 93 us, 105 with the
// weight loaded first. A 16-bit one beside a single sum makes 40 registers spill:
// 8192 x 8192 to e4m3 80 against 85 us, 16384 x 7168 136 against 142; with
// several sums it comes first (4096 x 4096, 8 sums to e4m3: 56 us, 60 behind).
template <typename T, typename W, int AT_ONCE, int K>
constexpr bool kLateWeight = sizeof(T) == 2 && K == 2 && (sizeof(W) == 4 || AT_ONCE == 1);

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
  Rows x[9];  // the partial sums, and the residual behind the last
  Rows residual;
  const void* weight;
  void* y;
  float* scale;
  void* h;
  float* rstd;
  long long rows;
  RowSplit split;
  int hidden, parts, group, group_log, tpr, groups;
  int window, windows;  // elements between staged rows, and a row's number of them
  int half;             // columns of a pair's first block
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
  int window;  // elements between staged rows
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
// is, and how much of the row is left from there on. The k-th eight of a
// warp's 32 threads (of a row's `tpr`, if fewer) are 256 (8 tpr) neighbours.
// VEC: a thread has eight of them in a row; without any (left <= 0) it reads
// the row's first ones and drops them. Otherwise it has every 32nd.
template <int K, bool VEC>
struct Part {
  static constexpr int kStep = VEC ? 1 : 32;
  int lane, at[K], left[K];

  __device__ __forceinline__ Part(int lane_, int tpr, int hidden) : lane(lane_) {
    const int in = lane & 31;
#pragma unroll
    for (int k = 0; k < K; ++k) {
      at[k] = VEC ? (lane + k * tpr) * 8 : (lane - in + k * tpr) * 8 + in;
      left[k] = hidden - at[k];
      if (VEC && left[k] <= 0) at[k] = 0;
    }
  }
};

// The threads of one row: a warp's, or the block's.
__device__ __forceinline__ void row_sync(int tpr) {
  if (tpr > 32) __syncthreads();
  else __syncwarp();
}

// A thread's elements of one row of a tensor.
template <typename T, bool VEC, int K>
struct Load {
  Raw<T, VEC> raw[K];

  __device__ __forceinline__ void load(const T* row, const Part<K, VEC>& part) {
#pragma unroll
    for (int k = 0; k < K; ++k) raw[k].load(row + part.at[k], part.kStep, part.left[k]);
  }
  __device__ __forceinline__ void get(int k, Pair (&f)[4]) const { raw[k].get(f); }
};

// The same, loaded where it is used.
template <typename T, int K>
struct LateLoad {
  const T* p[K];
  __device__ __forceinline__ void load(const T* row, const Part<K, true>& part) {
#pragma unroll
    for (int k = 0; k < K; ++k) p[k] = row + part.at[k];
  }
  __device__ __forceinline__ void get(int k, Pair (&f)[4]) const { unpack<T>(load_oct(p[k]), f); }
};

template <typename T, int K>
struct LateElements {
  const T* row;
  const Part<K, false>& part;
  __device__ __forceinline__ void get(int k, Pair (&f)[4]) const {
    Raw<T, false> raw;
    raw.load(row + part.at[k], part.kStep, part.left[k]);
    raw.get(f);
  }
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
__device__ __forceinline__ float reciprocal(float scale) {
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(scale));
  return r;
}

// The reciprocals of the scales of groups of 32, 64 or 128 columns, one for each
// of a thread's eight values; the group's first thread stores its scale. `whole`: the
// largest magnitude of a thread's part, where a group is wider than the row's threads.
template <bool VEC>
__device__ __forceinline__ void group_scales(const FwdArgs& a, const float (&y)[8], uint32_t whole, int tpr,
                                             long long row, int at, int left, float (&inv)[8]) {
  float* to = a.scale + row * a.groups;
  if constexpr (VEC) {  // a thread's values are in one group, with its neighbours
    uint32_t top = left > 0 ? top_of(y) : 0;
    int lanes = a.group >> 3;
    if (lanes > tpr) {
      lanes = tpr;
      top = whole;
    }
    const int in = threadIdx.x & 31;
    top = __reduce_max_sync(((1u << lanes) - 1u) << (in & ~(lanes - 1)), top);
    const float s = scale_of(top), i = reciprocal(s);
    if (left > 0 && (at & (a.group - 1)) == 0) to[at >> a.group_log] = s;
#pragma unroll
    for (int j = 0; j < 8; ++j) inv[j] = i;
  } else {  // a group is one, two or four neighbouring j of a warp's lanes
    uint32_t top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) top[j] = j * 32 < left ? magnitude(y[j]) : 0;
#pragma unroll
    for (int half = 1; half < 4; half *= 2)
      if (a.group > 32 * half) {
        uint32_t other[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) other[j] = top[j ^ half];
#pragma unroll
        for (int j = 0; j < 8; ++j) top[j] = max(top[j], other[j]);
      }
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float s = scale_of(__reduce_max_sync(~0u, top[j]));
      inv[j] = reciprocal(s);
      const int col = at + j * 32;
      if (j * 32 < left && (col & (a.group - 1)) == 0) to[col >> a.group_log] = s;
    }
  }
}

// A row off the vector boundary as it lies in shared memory: the aligned
// 16-byte pieces that hold it, copied asynchronously by the row's threads. What a
// piece holds before the row is the tensor's own (the row's element 0 is at
// `shift` elements); behind the row's end nothing is read.
template <typename T>
struct Window {
  static constexpr int E = 16 / sizeof(T);

  static __device__ __forceinline__ int shift(const T* row) {
    return int(reinterpret_cast<uintptr_t>(row) / sizeof(T)) & (E - 1);
  }
  // `begin`: the tensor's first element. A piece that starts before it (the
  // first row's) is filled one element at a time.
  static __device__ __forceinline__ void fetch(T* to, const T* row, const T* begin, int hidden, int lane, int tpr) {
    const int d = shift(row), whole = (d + hidden) / E, tail = (d + hidden) % E;
    const T* const from = row - d;
    const bool inside = from >= begin;
    const uint32_t at = uint32_t(__cvta_generic_to_shared(to));
    for (int i = lane || inside ? lane : tpr; i < whole; i += tpr)
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at + i * 16), "l"(from + i * E) : "memory");
    if (tail && lane == whole % tpr && (whole || inside))
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(at + whole * 16), "l"(from + whole * E),
                   "r"(tail * int(sizeof(T)))
                   : "memory");
    if (!inside && lane < E - d && lane < hidden) to[d + lane] = row[lane];
  }
};

// The way back: a row of B-byte elements that its threads have put into shared
// memory, at the elements that its place in memory is shifted by. Whole pieces
// are stored as such (stores of single elements off the boundary leave parts of
// 32-byte sectors, and took three times as long).
template <int B>
struct OutWindow {
  static constexpr int E = 16 / B;
  uint8_t* to;     // the row
  uint8_t* stage;  // the window

  __device__ __forceinline__ int shift() const { return int(reinterpret_cast<uintptr_t>(to) & 15) / B; }
  __device__ __forceinline__ uint8_t* element(int i) const { return stage + (shift() + i) * B; }
  __device__ __forceinline__ void put(int i) const {
    if constexpr (B == 1) to[i] = *element(i);
    else if constexpr (B == 2) reinterpret_cast<uint16_t*>(to)[i] = *reinterpret_cast<const uint16_t*>(element(i));
    else reinterpret_cast<uint32_t*>(to)[i] = *reinterpret_cast<const uint32_t*>(element(i));
  }
  __device__ __forceinline__ void flush(int hidden, int lane, int tpr) const {
    const int d = shift(), whole = (d + hidden) / E, tail = (d + hidden) % E;
    uint8_t* const from = to - d * B;  // the first piece's place
    for (int i = lane + (d ? 1 : 0); i < whole; i += tpr)
      *reinterpret_cast<uint4*>(from + i * 16) = *reinterpret_cast<const uint4*>(stage + i * 16);
    if (d && lane < E - d && lane < hidden) put(lane);
    // The end, unless it is in the first piece.
    if (lane < tail && (whole || !d)) put(hidden - tail + lane);
  }
};

// Elements of a row's window, which has room for all that its threads read;
// what lies behind the row is anything.
template <typename T, int K>
struct Staged {
  const T* base;  // the row's element 0
  const Part<K, false>& part;

  __device__ __forceinline__ void get(int k, Pair (&f)[4]) const {
    const T* p = base + part.at[k];
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = pair(to_float<T>(p[j * 64]), to_float<T>(p[j * 64 + 32]));
  }
};

// Zero where a thread's single elements lie behind the row.
__device__ __forceinline__ void clear_behind(Pair (&f)[4], int left) {
  if (left > 7 * 32) return;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    float a, b;
    split(f[j], a, b);
    f[j] = pair(j * 64 < left ? a : 0.0f, j * 64 + 32 < left ? b : 0.0f);
  }
}

// What the other block of a cluster of two gives: each stores its own where
// the other reads it. `box`: a word of shared memory that is not written again before
// both have read it (the next exchange's is another one).
__device__ __forceinline__ uint32_t pair_other(uint32_t mine, float* box, unsigned rank) {
  const uint32_t at = uint32_t(__cvta_generic_to_shared(box));
  if (threadIdx.x == 0) {
    uint32_t far;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(far) : "r"(at), "r"(rank ^ 1u));
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(far), "r"(mine) : "memory");
  }
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
  return *reinterpret_cast<volatile uint32_t*>(box);
}

// The sum of a value of each of the two blocks of a cluster, the same in both.
__device__ __forceinline__ float pair_sum(float s, float* box, unsigned rank, int turn) {
  const float other = __uint_as_float(pair_other(__float_as_uint(s), box + (turn & 1), rank));
  return rank ? other + s : s + other;
}

// A block's half of a row that two share: from which column on, and which of
// the two. Elsewhere all of it.
struct Half {
  int from = 0;
  unsigned rank = 0;
  float* box = nullptr;  // two words, for the sum and the maximum
};

// From the fp32 sum of a row to everything that is stored. part.left is 0 for
// threads without a row. STAGED: the outputs go through `stage`, whose
// contents (the sources) every thread has read.
template <typename T, bool F8, bool VEC, bool STAGED, bool PAIR, int K, typename Weight>
__device__ __forceinline__ void finish_row(const FwdArgs& a, long long row, bool live,
                                           const Part<K, VEC>& part,
                                           const Pair (&h)[K][4], const Weight& wv, float* red, uint32_t* top_red,
                                           const Half& half, T* stage = nullptr) {
  const int tpr = a.tpr;
  Pair sum = pair(0.0f, 0.0f), f[4];
#pragma unroll
  for (int k = 0; k < K; ++k)
    if (part.left[k] > 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sum = fma(h[k][j], h[k][j], sum);
    }
  const long long out = row * a.hidden + (PAIR ? half.from : 0);
  const OutWindow<int(sizeof(T))> hw{reinterpret_cast<uint8_t*>(static_cast<T*>(a.h) + out),
                                     reinterpret_cast<uint8_t*>(stage)};
  const OutWindow<F8 ? 1 : int(sizeof(T))> yw{static_cast<uint8_t*>(a.y) + out * (F8 ? 1 : int(sizeof(T))),
                                              reinterpret_cast<uint8_t*>(a.h ? stage + a.window : stage)};
  const auto put_h = [&] {
    if (a.h) {
#pragma unroll
      for (int k = 0; k < K; ++k) {
        float e[8];
        split(h[k], e);
        T* to = static_cast<T*>(a.h) + out;
        if constexpr (STAGED) to = reinterpret_cast<T*>(hw.element(0));
        store8<T, VEC>(to + part.at[k], e, part.kStep, STAGED ? kAll : part.left[k]);
      }
    }
  };
  if constexpr (!STAGED) put_h();
  float s = row_sum(sum_of(sum), tpr, red);
  if constexpr (PAIR) {
    asm volatile("barrier.cluster.wait.aligned;" ::: "memory");  // the other block has started
    s = pair_sum(s, half.box, half.rank, 0);
  }
  const float rstd = rsqrtf(fmaf(s, a.inv_hidden, a.eps));
  const bool first = live && part.lane == 0 && (!PAIR || half.rank == 0);
  if (first) a.rstd[row] = rstd;
  if constexpr (STAGED) {  // behind every thread's last read of a source
    if (tpr <= 32) __syncwarp();  // else row_sum has a barrier
    put_h();
  }
  const Pair r2 = pair(rstd, rstd);
  float y[K][8];
#pragma unroll
  for (int k = 0; k < K; ++k) {
    wv.get(k, f);
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = h[k][j] * r2 * f[j];
    split(f, y[k]);
  }
  uint8_t* const y0 = STAGED ? yw.element(0) : yw.to;
  if constexpr (!F8) {
#pragma unroll
    for (int k = 0; k < K; ++k)
      store8<T, VEC>(reinterpret_cast<T*>(y0) + part.at[k], y[k], part.kStep, STAGED ? kAll : part.left[k]);
  } else {
    uint32_t most = 0;
    if (a.group == 0 || a.group > 8 * tpr) {
#pragma unroll
      for (int k = 0; k < K; ++k)
        if (part.left[k] > 0) most = max(most, top_of<VEC>(y[k], part.kStep, part.left[k]));
    }
    float inv[8];
    if (a.group == 0) {
      most = row_max(most, tpr, top_red);
      if constexpr (PAIR) most = max(most, pair_other(most, half.box + 1, half.rank));
      const float scale = scale_of(most);
      if (first) a.scale[row] = scale;
#pragma unroll
      for (int j = 0; j < 8; ++j) inv[j] = reciprocal(scale);
    }
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (a.group)
        group_scales<VEC>(a, y[k], most, tpr, row, (PAIR ? half.from : 0) + part.at[k], part.left[k], inv);
      store_e4m3<VEC>(y0 + part.at[k], y[k], inv, part.kStep, STAGED ? kAll : part.left[k]);
    }
  }
  if constexpr (STAGED) {
    row_sync(tpr);
    if (a.h) hw.flush(a.hidden, part.lane, tpr);
    yw.flush(a.hidden, part.lane, tpr);
  }
}

// One row per tpr threads, in registers: every load is issued before the
// first value is used, and a row's threads meet once (twice with one e4m3
// scale per row). Octets on their boundary. W: the weight's type; AT_ONCE:
// partial sums whose loads are issued together.
//
// Two octets a thread share the cost of the row's sum: 8192 x 4096 bf16 with
// residual takes 41.8 us (98 % of the copy bandwidth) against 46 with one octet.
// Blocks that walk over rows with asynchronous copies ahead took 46.5 there, so a
// row has a block. With e4m3 output the arithmetic behind the sum, a chain
// of maximum, scale and conversion, shows: 16384 x 5120 in 93 us, 97 %.
// One row of 8192 takes 2.8 us, most of it the launch.
// PAIR: a row is shared by the two blocks of a cluster. Their part of it is a
// multiple of 128 columns, so that no group of columns is in both.
template <typename T, typename W, bool F8, int AT_ONCE, int K, bool PAIR = false, bool LEAN = false>
__global__ void __maxnreg__(norm_registers(sizeof(T), AT_ONCE, K, PAIR, LEAN))
    norm_kernel(const __grid_constant__ FwdArgs a) {
  __shared__ float red[32];
  __shared__ uint32_t top_red[32];
  __shared__ float box[2];
  Half half;
  int columns = a.hidden;
  if constexpr (PAIR) {
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
    half.rank = blockIdx.x & 1;
    half.box = box;
    half.from = half.rank ? a.half : 0;
    columns = half.rank ? a.hidden - a.half : a.half;
  }
  const int tpr = a.tpr;
  const int lane = tpr > 32 ? threadIdx.x : threadIdx.x & (tpr - 1);
  const long long row = PAIR       ? (long long)(blockIdx.x >> 1)
                        : tpr > 32 ? (long long)blockIdx.x
                                   : (long long)blockIdx.x * (blockDim.x / tpr) + threadIdx.x / tpr;
  const bool live = row < a.rows;  // every thread stays for the shuffles
  const Row from(live ? row : 0, a.split);
  Part<K, true> part(lane, tpr, columns);
  const int at = PAIR ? half.from : 0;
  // AT_ONCE partial sums at a time, with the first of them the residual too.
  constexpr int N = AT_ONCE;
  Load<T, true, K> xv[N], rv;
  std::conditional_t<kLateWeight<T, W, AT_ONCE, K>, LateLoad<W, K>, Load<W, true, K>> wv;
  Pair h[K][4], f[4];
#pragma unroll 1
  for (int s0 = 0; s0 < (N > 1 ? a.parts : 1); s0 += N) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      if (s0 + i < a.parts) xv[i].load(from.of<T>(a.x[s0 + i]) + at, part);
    if (s0 == 0 && a.residual.p) rv.load(from.of<T>(a.residual) + at, part);
    if (s0 == 0) wv.load(static_cast<const W*>(a.weight) + at, part);
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
  finish_row<T, F8, true, false, PAIR, K>(a, row, live, part, h, wv, red, top_red, half);
}

// The same for rows off the vector boundary, which go through shared memory:
// all sources of a row are on their way at once without a register held for
// them, and single elements come out of shared memory. A row has a warp or a block.
// Bound by the instructions that single elements take: 8192 x 4097 bf16 in 74 us
// (76 with the weight loaded ahead of the sum; single elements straight from
// memory: 106; octets cut out of the pieces in registers: 142), four fp16 partials
// of 1013 x 5001 with e4m3 output in 22 us.
template <typename T, typename W, bool F8, int K>
__global__ void __launch_bounds__(kStagedThreads, 2) norm_staged_kernel(const __grid_constant__ FwdArgs a) {
  extern __shared__ uint4 smem[];
  __shared__ float red[32];
  __shared__ uint32_t top_red[32];
  const int tpr = a.tpr, lane = tpr > 32 ? threadIdx.x : threadIdx.x & 31, slot = tpr > 32 ? 0 : threadIdx.x >> 5;
  const long long row = tpr > 32 ? (long long)blockIdx.x : (long long)blockIdx.x * (blockDim.x >> 5) + slot;
  if (row >= a.rows) return;  // a whole warp
  const Row from(row, a.split);
  const int sources = a.parts + (a.residual.p ? 1 : 0);
  T* const stage = reinterpret_cast<T*>(smem) + slot * a.windows * a.window;
  for (int s = 0; s < sources; ++s)
    Window<T>::fetch(stage + s * a.window, from.of<T>(a.x[s]), static_cast<const T*>(a.x[s].p), a.hidden, lane, tpr);
  asm volatile("cp.async.commit_group;" ::: "memory");
  const Part<K, false> part(lane, tpr, a.hidden);
  const LateElements<W, K> wv{static_cast<const W*>(a.weight), part};
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  row_sync(tpr);
  Pair h[K][4], f[4];
  const auto source = [&](int i) {
    return Staged<T, K>{stage + i * a.window + Window<T>::shift(from.of<T>(a.x[i])), part};
  };
  const Staged<T, K> first = source(0);
#pragma unroll
  for (int k = 0; k < K; ++k) first.get(k, h[k]);
#pragma unroll 1
  for (int i = 1; i < sources; ++i) {
    const Staged<T, K> v = source(i);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      v.get(k, f);
      add(h[k], f);
    }
  }
#pragma unroll
  for (int k = 0; k < K; ++k) clear_behind(h[k], part.left[k]);
  finish_row<T, F8, false, true, false, K>(a, row, true, part, h, wv, red, top_red, Half(), stage);
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
    v.load(from.of<T>(a.x[s]), part);
    v.get(0, f);
    add(h, f);
  }
}

// The turns that a block of kLongThreads takes over a long row: turn k is the
// k-th eight elements of its threads. Whole warps take every turn; a thread without
// elements in one gets the row's first place and left <= 0.
template <bool VEC, typename F>
__device__ __forceinline__ void each_turn(int hidden, F f) {
  const int turns = (hidden + 8 * kLongThreads - 1) / (8 * kLongThreads);
  Part<1, VEC> part(threadIdx.x, kLongThreads, hidden);
  const int first = VEC ? int(threadIdx.x) * 8 : part.at[0];
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
      top = max(top, top_of<VEC>(y, part.kStep, part.left[0]));
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
      if (a.h) store8<T, VEC>(static_cast<T*>(a.h) + out + at, e, part.kStep, left);
    }
    if constexpr (F8) {
      if (a.group) group_scales<VEC>(a, y, 0, kLongThreads, row, at, left, inv);
      store_e4m3<VEC>(static_cast<uint8_t*>(a.y) + out + at, y, inv, part.kStep, left);
    } else {
      store8<T, VEC>(static_cast<T*>(a.y) + out + at, y, part.kStep, left);
    }
  });
}

// A row of the gradient, from this thread's elements: adds to dw's part and
// stores the row of dx. `total`: the sum over the row's threads.
template <typename T, typename W, bool VEC, bool STAGED, int K, typename In, typename Total>
__device__ __forceinline__ void finish_grad(const BwdArgs& a, bool live, const Part<K, VEC>& part,
                                            const In& dy, const In& h, const In& dh, float rstd,
                                            const Load<W, VEC, K>& wv, Pair (&acc)[K][4], T* dx, Total total) {
  Pair g[K][4], n[K][4], sum = pair(0.0f, 0.0f);
  const Pair r2 = pair(rstd, rstd);
#pragma unroll
  for (int k = 0; k < K; ++k) {
    Pair w[4];
    dy.get(k, g[k]);
    h.get(k, n[k]);
    wv.get(k, w);
    if constexpr (STAGED) {
      clear_behind(g[k], part.left[k]);
      clear_behind(n[k], part.left[k]);
    }
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
  const float c = total(sum_of(sum)) * -a.inv_hidden;
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
    store8<T, VEC>(dx + part.at[k], f, part.kStep, STAGED ? kAll : live ? part.left[k] : 0);
  }
}

// The block's part of dw: its rows are fixed, and with several rows at once
// its slots are added in order.
template <int K, bool VEC>
__device__ __forceinline__ void store_partial(const BwdArgs& a, const Part<K, VEC>& part, const Pair (&acc)[K][4],
                                              float* slots, float* to) {
  const int tpr = a.tpr;
  op_nearly_done();
  float* const block = to;
  if (tpr <= 32) to = slots + (threadIdx.x / tpr) * a.hidden;
#pragma unroll
  for (int k = 0; k < K; ++k) {
    float f[8];
    split(acc[k], f);
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * part.kStep < part.left[k]) to[part.at[k] + j * part.kStep] = f[j];
  }
  if (tpr <= 32) {
    __syncthreads();
    const int per = blockDim.x / tpr;
    for (int col = threadIdx.x; col < a.hidden; col += blockDim.x) {
      float s = 0.0f;
      for (int q = 0; q < per; ++q) s += slots[q * a.hidden + col];
      block[col] = s;
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
// the parts go to `partial` and dw_kernel adds them in block order. fp32 rows
// use this form: 8192 x 4096 in 88 us (93 % of the copy bandwidth).
template <typename T, typename W, int K>
__global__ void __launch_bounds__(kRingThreads) norm_backward_kernel(const __grid_constant__ BwdArgs a) {
  __shared__ float red[2][32];
  __shared__ float slots[256 * 8 * K];
  const int tpr = a.tpr;
  const int lane = tpr > 32 ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int per = tpr > 32 ? 1 : blockDim.x / tpr, slot = tpr > 32 ? 0 : threadIdx.x / tpr;
  const Part<K, true> part(lane, tpr, a.hidden);
  Pair acc[K][4];
  Load<W, true, K> wv;
  wv.load(static_cast<const W*>(a.weight), part);
  clear<K>(acc);
  const long long stride = (long long)gridDim.x * per;
  int turn = 0;
  for (long long row = (long long)blockIdx.x * per + slot; row - slot < a.rows; row += stride, ++turn) {
    const bool live = row < a.rows;
    const long long r = live ? row : a.rows - 1;
    const Row from(r, a.split);
    Load<T, true, K> dy, h, dh;
    dy.load(from.of<T>(a.dy), part);
    h.load(from.of<T>(a.h), part);
    if (a.dh.p) dh.load(from.of<T>(a.dh), part);
    finish_grad<T, W, true, false, K>(a, live, part, dy, h, dh, a.rstd[r], wv, acc,
                                      static_cast<T*>(a.dx) + row * a.hidden,
                                      [&](float s) { return row_sum(s, tpr, red[turn & 1]); });
  }
  store_partial<K, true>(a, part, acc, slots, a.partial + (long long)blockIdx.x * a.hidden);
}

// A thread's own ring in shared memory: a few rows of its octets of a 16-bit
// type, brought by 16-byte asynchronous copies. Only the thread itself reads
// them, so a stage needs no barrier: the thread waits for its own copies.
// Copies of later rows are in flight while a row is reduced, without a
// register held for them.
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
// drops it. PAIR: a row is shared by the two blocks of a cluster, half of the
// octets each, because one block's registers do not hold it.
//
// A row's sum stands between its loads and its stores, so that without copies
// ahead the memory idles while a block reduces: 16384 x 4096 bf16 in 88 us (92 %
// of the copy bandwidth) against 113 without the ring. Rows of 16384 as pairs: 2048
// of them in 81 us, 105 with two passes over the row.
template <typename T, typename W, bool PAIR, int K, int STAGES>
__global__ void __launch_bounds__(kRingThreads) norm_backward_ring_kernel(const __grid_constant__ BwdArgs a) {
  extern __shared__ uint4 smem[];
  __shared__ float red[2][32];
  __shared__ float box[2];
  const int tpr = a.tpr;
  const int lane = tpr > 32 ? threadIdx.x : threadIdx.x & (tpr - 1);
  const int per = tpr > 32 ? 1 : blockDim.x / tpr, slot = tpr > 32 ? 0 : threadIdx.x / tpr;
  const unsigned rank = PAIR ? blockIdx.x & 1 : 0;
  const long long block = PAIR ? blockIdx.x >> 1 : blockIdx.x, blocks = PAIR ? gridDim.x >> 1 : gridDim.x;
  const int half = (a.hidden / 8 + 1) / 2 * 8, from_col = rank * half;
  const int columns = !PAIR ? a.hidden : rank ? a.hidden - half : half;
  const Part<K, true> part(lane, tpr, columns);
  const Ring<T, K> ring{smem, a.dh.p ? 3 : 2};
  const long long stride = blocks * per;
  long long ahead = block * per + slot;
  float rstds[STAGES];  // of the rows on their way
  const auto fetch = [&](int stage, float& rstd) {
    rstd = 0.0f;
    if (ahead < a.rows) {
      const Row from(ahead, a.split);
      ring.fetch(stage, 0, from.of<T>(a.dy) + from_col, part);
      ring.fetch(stage, 1, from.of<T>(a.h) + from_col, part);
      if (a.dh.p) ring.fetch(stage, 2, from.of<T>(a.dh) + from_col, part);
      rstd = a.rstd[ahead];
    }
    ahead += stride;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < STAGES - 1; ++s) fetch(s, rstds[s]);
  Pair acc[K][4];
  Load<W, true, K> wv;
  wv.load(static_cast<const W*>(a.weight) + from_col, part);
  clear<K>(acc);
  if constexpr (PAIR)  // both blocks have started before either stores into the other
    asm volatile("barrier.cluster.arrive.relaxed.aligned;\n\tbarrier.cluster.wait.aligned;" ::: "memory");
  int turn = 0;
  for (long long row = block * per + slot; row - slot < a.rows;) {
#pragma unroll
    for (int s = 0; s < STAGES; ++s) {  // the stage is a constant, so rstds stays in registers
      if (row - slot >= a.rows) break;
      // Into the stage of the row before, whose values this thread has used.
      fetch((s + STAGES - 1) % STAGES, rstds[(s + STAGES - 1) % STAGES]);
      asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 1) : "memory");
      Load<T, true, K> dy, h, dh;
      ring.read(s, 0, dy);
      ring.read(s, 1, h);
      if (a.dh.p) ring.read(s, 2, dh);
      finish_grad<T, W, true, false, K>(a, row < a.rows, part, dy, h, dh, rstds[s], wv, acc,
                                        static_cast<T*>(a.dx) + row * a.hidden + from_col, [&](float v) {
                                          v = row_sum(v, tpr, red[turn & 1]);
                                          return PAIR ? pair_sum(v, box, rank, turn) : v;
                                        });
      row += stride;
      ++turn;
    }
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  store_partial<K, true>(a, part, acc, reinterpret_cast<float*>(smem), a.partial + block * a.hidden + from_col);
}

// The same for rows off the boundary, a warp or a block to each: the rows on
// their way are windows that the row's threads share, so they meet between a
// stage's copies and its use, and between its use and the next copies. dx has
// a window of its own. 8192 x 4097 bf16 in 102 us (169 with single elements
// straight from and to memory).
constexpr int kStagesOff = 3;

template <typename T, typename W, int K>
__global__ void __launch_bounds__(kStagedThreads) norm_backward_staged_kernel(const __grid_constant__ BwdArgs a) {
  extern __shared__ uint4 smem[];
  __shared__ float red[2][32];
  const int tpr = a.tpr, lane = tpr > 32 ? threadIdx.x : threadIdx.x & 31;
  const int per = tpr > 32 ? 1 : blockDim.x >> 5, slot = tpr > 32 ? 0 : threadIdx.x >> 5;
  const Part<K, false> part(lane, tpr, a.hidden);
  const int sources = a.dh.p ? 3 : 2;
  T* const ring = reinterpret_cast<T*>(smem) + slot * (kStagesOff * sources + 1) * a.window;
  const long long first = (long long)blockIdx.x * per + slot, stride = (long long)gridDim.x * per;
  long long ahead = first;
  const auto fetch = [&](int stage) {
    if (ahead < a.rows) {
      const Row from(ahead, a.split);
      T* to = ring + stage * sources * a.window;
      const auto one = [&](const Rows& t) {
        Window<T>::fetch(to, from.of<T>(t), static_cast<const T*>(t.p), a.hidden, lane, tpr);
        to += a.window;
      };
      one(a.dy);
      one(a.h);
      if (a.dh.p) one(a.dh);
    }
    ahead += stride;
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStagesOff - 1; ++s) fetch(s);
  Pair acc[K][4];
  Load<W, false, K> wv;
  wv.load(static_cast<const W*>(a.weight), part);
  clear<K>(acc);
  int stage = 0, turn = 0;
  for (long long row = first; row < a.rows; row += stride, ++turn) {
    const float rstd = a.rstd[row];
    asm volatile("cp.async.wait_group %0;" ::"n"(kStagesOff - 2) : "memory");
    row_sync(tpr);
    fetch(stage == 0 ? kStagesOff - 1 : stage - 1);  // the stage of the row before
    const Row from(row, a.split);
    const T* at = ring + stage * sources * a.window;
    const Staged<T, K> dy{at + Window<T>::shift(from.of<T>(a.dy)), part},
        h{at + a.window + Window<T>::shift(from.of<T>(a.h)), part},
        dh{at + 2 * a.window + Window<T>::shift(from.of<T>(a.dh)), part};
    const OutWindow<int(sizeof(T))> out{reinterpret_cast<uint8_t*>(static_cast<T*>(a.dx) + row * a.hidden),
                                        reinterpret_cast<uint8_t*>(ring + kStagesOff * sources * a.window)};
    finish_grad<T, W, false, true, K>(a, true, part, dy, h, dh, rstd, wv, acc, reinterpret_cast<T*>(out.element(0)),
                                      [&](float s) { return row_sum(s, tpr, red[turn & 1]); });
    row_sync(tpr);
    out.flush(a.hidden, lane, tpr);  // read before the row's threads meet again
    stage = stage == kStagesOff - 1 ? 0 : stage + 1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  store_partial<K, false>(a, part, acc, reinterpret_cast<float*>(smem),
                          a.partial + (long long)blockIdx.x * a.hidden);
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
    store8<T, VEC>(static_cast<T*>(a.dx) + row * a.hidden + part.at[0], f, part.kStep, part.left[0]);
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
    if (j * part.kStep < part.left[0]) to[j * part.kStep] = f[j];
}

// dw[col] = sum of the blocks' parts: a warp-wide strip of 32 columns per
// block, 32 warps over the parts, then the warps in order.
template <typename W>
__global__ void __launch_bounds__(1024) dw_kernel(const float* partial, int parts, int hidden, W* dw) {
  __shared__ float sum[32][33];
  const int col = blockIdx.x * 32 + threadIdx.x;
  float s = 0.0f;
  op_wait_for_previous();
  if (col < hidden) {
#pragma unroll 8
    for (int p = threadIdx.y; p < parts; p += 32) s += partial[(long long)p * hidden + col];
  }
  sum[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = sum[threadIdx.x][threadIdx.y];  // transposed: a warp adds one column
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  const int at = blockIdx.x * 32 + threadIdx.y;
  if (threadIdx.x == 0 && at < hidden) dw[at] = from_float<W>(s);
}

// ---------------------------------------------------------------- host

constexpr int kStages = 4;  // rows of a ring
constexpr int kRingSmem = 220 * 1024;  // of an SM's shared memory, for the rings of its blocks

// How rows are spread over threads and blocks.
struct Shape {
  int tpr = 0, threads = 0, k = 0;  // k 0: the long variant
  int at_once = 1, half = 0;  // partial sums at a time; columns of a pair's first block
  bool ring = false, staged = false, pair = false, lean = false;
  size_t smem = 0;
  long long blocks = 0;
};

int pow2_at_least(int n) {
  int p = 1;
  while (p < n) p *= 2;
  return p;
}

long long ceil_div(long long a, long long b) { return (a + b - 1) / b; }

// `k` octets a thread; rows of up to 32 threads share a block: `warp` gives each a whole warp.
void spread(Shape& s, int octets, int k, bool warp) {
  s.k = k;
  if (octets <= 32 * k) {
    s.tpr = warp ? 32 : pow2_at_least(int(ceil_div(octets, k)));
    s.threads = 256;
  } else {
    s.tpr = s.threads = int(ceil_div(ceil_div(octets, 32), k)) * 32;
  }
}

int rows_per_block(const Shape& s) { return s.tpr > 32 ? 1 : s.threads / s.tpr; }

// Elements from one staged row to the next: room for every thread's elements, and a piece more for its shift.
int window_of(const Shape& s, int es) { return s.tpr * 8 * s.k + 16 / es; }

// Blocks that an SM's registers hold: each of its four parts has 16384, and
// takes a quarter of a block's warps or one more.
int blocks_by_registers(int threads, int registers) { return 4 * (16384 / (32 * registers)) / (threads / 32); }

// Aligned rows stay in registers; others go through shared memory, `windows`
// (sources or outputs) of them for each row, where two blocks fit an SM. What
// is too long for either is read again in each pass.
//
// Of a row in registers, the variant that lets an SM hold two blocks at least
// (norm_registers; bf16 with residual; "48 -> 40" are registers a thread):
//  - one sum: 40 registers only where they hold more blocks: 4096 x 12288 with
//    e4m3 output 84 -> 63 us, 8192 x 8192 88 -> 79; but 16384 x 5120, where they do
//    not, took 100 instead of 94.
//  - several: four at a time, or two where four leave one block (8192 x 8192, 8 sums:
//    256 -> 226 us) or where there are two (8192 x 7168: 142 -> 92); four in 72
//    registers for 80 where that holds more (8192 x 7168, 4 sums: 163 -> 117).
//  - a pair of blocks for each row where one leaves no room for a second: 4096 x 16384
//    96 -> 91 us, 4096 x 12288 with 8 sums 201 -> 172, and what one block does not hold:
//    2048 x 20480 74 -> 63 (reading it again), 2048 x 16384 fp32 with 4 sums 211 -> 142.
//    Not two sums at a time where a pair holds no more threads (4096 x 12288: 94 us, pairs
//    104), nor one scale a row, whose maximum is a second meeting of the two (4096 x
//    16384: 99 us, pairs 104); nor fp32 with fewer than three sums (2048 x 12288: 96
//    us by reading again, pairs 102).
// Up to a row an SM, one octet a thread is the shortest way.
Shape shape_fwd(long long rows, int hidden, int es, int windows, bool vec, int parts, bool by_row, int sms) {
  Shape s;
  const int octets = int(ceil_div(hidden, 8));
  s.at_once = parts == 1 ? 1 : 4;
  if (!vec) {
    s.blocks = rows;
    if (octets > 2 * 512) return s;
    spread(s, octets, octets > 32 ? 2 : 1, true);
    s.staged = true;
    s.smem = size_t(rows_per_block(s)) * size_t(windows) * size_t(window_of(s, es)) * size_t(es);
    if (s.smem > size_t(kRingSmem) / 2) s = Shape{};
    s.blocks = s.k ? ceil_div(rows, rows_per_block(s)) : rows;
    return s;
  }
  if (rows <= sms && octets <= (parts == 1 ? 1024 : 512)) {
    spread(s, octets, 1, false);
    s.blocks = ceil_div(rows, rows_per_block(s));
    return s;
  }
  // One block a row, if two fit an SM; else a pair's two, where that pays; else one.
  int alone = 0;
  for (const int turn : {0, 1, 2}) {
    s.pair = turn == 1;
    s.half = s.pair ? int(ceil_div(octets, 32)) * 16 * 8 : hidden;
    spread(s, s.half / 8, 2, false);
    const auto fit = [&](int at_once, bool lean) {
      return blocks_by_registers(s.threads, norm_registers(es, at_once, 2, s.pair, lean));
    };
    if (parts > 1 && es == 2)
      s.at_once = parts == 2 || s.threads > 512 || (rows > sms && fit(4, true) < 2) ? 2 : 4;
    s.lean = es == 2 && s.at_once != 2 && fit(s.at_once, true) > fit(s.at_once, false);
    const int blocks = fit(s.at_once, s.lean);
    if (turn == 0 && s.threads <= 1024) alone = blocks * s.threads;
    bool take = s.threads <= 1024 && blocks > (turn == 2 || es == 4 || rows <= sms ? 0 : 1);
    if (s.pair && es == 4) take = take && parts > 2;
    else if (s.pair) take = take && !(by_row && alone) && (s.at_once != 2 || blocks * s.threads > alone);
    if (take) {
      s.blocks = ceil_div(rows, rows_per_block(s));
      return s;
    }
  }
  s = Shape{};
  s.blocks = rows;
  return s;
}

Shape shape_bwd(long long rows, int hidden, int es, bool vec, int sms) {
  Shape s;
  const int octets = int(ceil_div(hidden, 8));
  s.pair = vec && es == 2 && octets > 2 * kRingThreads && octets <= 4 * kRingThreads;
  bool fits = s.pair || octets <= 2 * kRingThreads;
  if (fits) {
    spread(s, s.pair ? (octets + 1) / 2 : octets, 2, !vec);
    // Sized for three sources, so that the parts of dw do not depend on them.
    s.smem = vec ? size_t(kStages) * 3u * 2u * size_t(s.threads) * 16u
                 : size_t(rows_per_block(s)) * (kStagesOff * 3u + 1u) * size_t(window_of(s, es)) * size_t(es);
    const bool room = s.smem <= size_t(kRingSmem);
    s.ring = vec && es == 2 && room;
    s.staged = !vec;
    fits = vec || room;
  }
  if (!fits) {  // blocks that share dw's columns
    s = Shape{};
    const long long columns = ceil_div(octets, 256), splits = ceil_div(8ll * sms, columns);
    s.blocks = splits < rows ? splits : rows;
    return s;
  }
  const int by_threads = (vec ? kRingThreads : kStagedThreads) / s.threads;
  const int by_smem = s.ring || s.staged ? int(size_t(kRingSmem) / s.smem) : by_threads;
  // As many as are resident, but with two rows each before every SM has more
  // than one; of a pair's blocks, half as many.
  const int places = s.pair ? sms / 2 > 0 ? sms / 2 : 1 : sms;
  const long long fit = (long long)places * (by_smem < by_threads ? by_smem : by_threads);
  const long long most = ceil_div(rows, rows_per_block(s)), few = ceil_div(most, 2);
  s.blocks = most < places ? most : few < places ? places : few < fit ? few : fit;
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

template <typename T, typename W, bool F8, bool PAIR>
const void* fwd_kernel2(const Shape& s) {
  if constexpr (sizeof(T) == 2) {
    if (s.at_once == 2) return reinterpret_cast<const void*>(norm_kernel<T, W, F8, 2, 2, PAIR>);
    if (s.lean) return s.at_once == 4 ? reinterpret_cast<const void*>(norm_kernel<T, W, F8, 4, 2, PAIR, true>)
                                      : reinterpret_cast<const void*>(norm_kernel<T, W, F8, 1, 2, PAIR, true>);
  }
  return s.at_once == 4 ? reinterpret_cast<const void*>(norm_kernel<T, W, F8, 4, 2, PAIR>)
                        : reinterpret_cast<const void*>(norm_kernel<T, W, F8, 1, 2, PAIR>);
}

template <typename T, typename W, bool F8>
const void* fwd_kernel(bool vec, const Shape& s) {
  if (s.staged) return s.k == 1 ? reinterpret_cast<const void*>(norm_staged_kernel<T, W, F8, 1>)
                                : reinterpret_cast<const void*>(norm_staged_kernel<T, W, F8, 2>);
  if (s.k == 1) return s.at_once == 4 ? reinterpret_cast<const void*>(norm_kernel<T, W, F8, 4, 1>)
                                      : reinterpret_cast<const void*>(norm_kernel<T, W, F8, 1, 1>);
  if (s.k == 2) return s.pair ? fwd_kernel2<T, W, F8, true>(s) : fwd_kernel2<T, W, F8, false>(s);
  return vec ? reinterpret_cast<const void*>(norm_long_kernel<T, W, F8, true>)
             : reinterpret_cast<const void*>(norm_long_kernel<T, W, F8, false>);
}

// The kernels of an input and a weight type.
template <typename T, typename W>
struct Kernels {
  static const void* fwd(bool f8, bool vec, const Shape& s) {
    return f8 ? fwd_kernel<T, W, true>(vec, s) : fwd_kernel<T, W, false>(vec, s);
  }
  static const void* bwd(bool vec, const Shape& s) {
    if constexpr (sizeof(T) == 2)
      if (s.ring) return s.pair ? reinterpret_cast<const void*>(norm_backward_ring_kernel<T, W, true, 2, kStages>)
                                : reinterpret_cast<const void*>(norm_backward_ring_kernel<T, W, false, 2, kStages>);
    if (s.staged) return reinterpret_cast<const void*>(norm_backward_staged_kernel<T, W, 2>);
    if (s.k) return reinterpret_cast<const void*>(norm_backward_kernel<T, W, 2>);
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

cudaError_t launch(const void* fn, const Shape& s, int device, unsigned blocks, void** argv, cudaStream_t stream) {
  size_t smem = 0;
  if (s.ring || s.staged) {
    smem = s.smem;
    const cudaError_t e = op_allow_smem(fn, device, kRingSmem);
    if (e != cudaSuccess) return e;
  }
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr{};
  cfg.gridDim = dim3(s.pair ? 2 * blocks : blocks);
  cfg.blockDim = dim3(unsigned(s.k ? s.threads : kLongThreads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  if (s.pair) {
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = 2;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
  }
  return cudaLaunchKernelExC(&cfg, fn, argv);
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
  k.x[a->parts] = k.residual;
  if (a->residual) vec = vec && octets_fit(a->residual, a->r_outer, a->r_inner, es);
  vec = vec && octets_fit(a->y, 0, 0, f8 ? 1 : es) && (!a->h || octets_fit(a->h, 0, 0, es));
  const int sources = a->parts + (a->residual ? 1 : 0), outputs = a->h ? 2 : 1;
  k.windows = sources > outputs ? sources : outputs;
  const Shape s = shape_fwd(a->rows, a->hidden, es, k.windows, vec, a->parts, f8 && !a->group, dev.sms());
  k.half = s.half;
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
  k.group_log = a->group == 128 ? 7 : a->group == 64 ? 6 : 5;
  k.groups = a->group ? (a->hidden + a->group - 1) / a->group : 1;
  k.tpr = s.tpr;
  k.window = window_of(s, es);
  k.eps = a->eps;
  k.inv_hidden = 1.0f / float(a->hidden);
  const void* fn = by_types(a->dtype, a->weight_dtype == NB_NORM_FLOAT32,
                            [&](auto kernels) { return kernels.fwd(f8, vec, s); });
  void* argv[] = {&k};
  const cudaError_t e = launch(fn, s, a->device, unsigned(s.blocks), argv, static_cast<cudaStream_t>(stream));
  return e == cudaSuccess ? 0 : op_refuse(err, errcap, "launch of the norm failed", int(e));
}

extern "C" uint64_t nb_add_rms_norm_backward_workspace(int device, int64_t rows, int hidden, int dtype) {
  const int es = size_of(dtype);
  OpDevice dev(device);
  if (dev.error() || rows < 0 || hidden < 1 || !es) return 0;
  const long long on = shape_bwd(rows, hidden, es, true, dev.sms()).blocks;
  const long long off = shape_bwd(rows, hidden, es, false, dev.sms()).blocks;
  return uint64_t(on > off ? on : off) * uint64_t(hidden) * sizeof(float);
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
  const bool vec = a->hidden % 8 == 0 && octets_fit(a->weight, 0, 0, ws) &&
                   octets_fit(a->dy, a->dy_outer, a->dy_inner, es) && octets_fit(a->h, a->h_outer, a->h_inner, es) &&
                   (!a->dh || octets_fit(a->dh, a->dh_outer, a->dh_inner, es)) && octets_fit(a->dx, 0, 0, es);
  const Shape s = shape_bwd(a->rows, a->hidden, es, vec, dev.sms());
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
  k.window = window_of(s, es);
  k.inv_hidden = 1.0f / float(a->hidden);
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  void* argv[] = {&k};
  cudaError_t e = cudaSuccess;
  if (a->rows) {
    const void* fn = by_types(a->dtype, a->weight_dtype == NB_NORM_FLOAT32,
                              [&](auto kernels) { return kernels.bwd(vec, s); });
    e = launch(fn, s, a->device, unsigned(s.k ? parts : a->rows), argv, st);
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
    e = op_launch_after(fn, dim3(unsigned((hidden + 31) / 32)), dim3(32, 32), dargv, st);
  }
  return e == cudaSuccess ? 0 : op_refuse(err, errcap, "launch of the norm's gradient failed", int(e));
}
