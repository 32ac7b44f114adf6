// AdamW and the gradients' norm over many tensors (see optim.h).
//
//   g = scale * (g_0 + ... + g_{n-1})                 (fp32, in order)
//   m = b1 m + (1 - b1) g,   v = b2 v + (1 - b2) g^2
//   p = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v / (1 - b2^t)) + eps)
//
// Bound by HBM: every array is read and written once (28 bytes an element
// with fp32 parameters and states, a 16-bit gradient and a 16-bit copy; 16
// with 8-bit states), so the arithmetic is plain fp32 in the order written.
// 201 M elements of 28 bytes take 845 us (102 % of the copy bandwidth). With 8-bit
// states some 85 instructions an element (the random bits, two roundings, a
// root and a quotient) take as long as the memory: 255 M elements of 18 bytes
// in 870 us, 81 %. The gradients' norm reads at the copy bandwidth: 201 M
// bf16 in 61 us.
//
// States in 8 bits. m and r = sqrt(v) are kept in e4m3, blocks of 256 (one
// warp's eight elements per lane, so a block's maximum is one warp reduction)
// with an fp32 scale that maps the block's largest magnitude to 448. r instead of v
// halves the exponent range that the 8 bits have to cover. They are rounded
// at random, to the neighbour below or above with the odds that keep the
// mean of m and of r: to nearest, a state that moves by less than half a step (3 to 6 %)
// would never move, and beta2 = 0.999 moves v by 0.1 % a step. What three bits of
// mantissa cost: r wanders about its mean, so that v = r^2 is high on average (simulated
// with gradients of one distribution: 5 % at beta2 = 0.999, 2.5 % at 0.95), and single
// ones lie between 0.6 and 1.7 (0.7 and 1.5) of the exact v, 5th to 95th percentile. The random bits
// are a hash of the seed, t, the tensor and the element, so a step is
// reproducible. A positive r never rounds to zero, where m / (r + eps) would
// explode. The update itself uses the unrounded m and v.
#include <cuda_runtime.h>

#include <cmath>
#include <cstring>
#include <memory>
#include <new>
#include <type_traits>
#include <vector>

#include "core/tensor_table.h"
#include "kernels/octet.cuh"
#include "kernels/ophost.h"
#include "kernels/optim.h"

namespace nb {
namespace {

using namespace octet;

constexpr int kThreads = 256;
constexpr unsigned kChunk = kThreads * 8;         // AdamW: eight elements per thread
constexpr int kNormOctets = 4;                    // the norm: four times that, all loaded before the first is used
constexpr unsigned kNormChunk = kChunk * kNormOctets;
constexpr float kLargest = 3.4028235e38f;         // finite in fp32
static_assert(NB_OPTIM_BLOCK == 256, "a block is one warp's elements");

// One tensor of the work list; its gradients' addresses follow the entries.
struct Entry {
  void* param;
  void* copy;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  unsigned long long size;
  unsigned first;  // its first chunk
  unsigned index;  // its place in the caller's list
  float decay;
  int vec;         // every address is on an octet's boundary
};
constexpr int kEntryWords = sizeof(Entry) / 8;

struct GradEntry {
  unsigned long long size;
  unsigned first;
  int vec;
};
constexpr int kGradEntryWords = sizeof(GradEntry) / 8;

// The list's room. A launch with 32 KB of parameters takes about 1 us longer to
// queue than one with 10 KB, which hold some 120 tensors.
constexpr int kSmallWords = 1200, kLargeWords = 4000;

struct StepScalars {
  const long long* t;
  const float* lr;
  const float* scale;
  float t_lr_m;      // lr / (1 - b1^t), where both are the host's
  float t_root;      // 1 / sqrt(1 - b2^t), where t is the host's
  float lr_host, scale_host;
  float inv1;        // 1 / (1 - b1^t), where t is the host's
  unsigned t_host;
};

template <int WORDS>
struct AdamArgs {
  StepScalars s;
  float b1, b1c, b2, b2c, eps, ln_b1, ln_b2;
  unsigned seed, chunks;
  int count, parts;
  unsigned long long words[WORDS];
};
static_assert(sizeof(AdamArgs<kLargeWords>) <= 32764, "kernel parameters");


template <int WORDS>
struct GradArgs {
  double* partial;
  unsigned chunks;
  int count, parts;
  unsigned long long words[WORDS];
};

__device__ __forceinline__ uint32_t mix(uint32_t x) {
  x ^= x >> 16;
  x *= 0xA5CB9243u;
  x ^= x >> 15;
  x *= 0x5D8A37E5u;
  return x ^ x >> 16;
}

// Rounding |z| <= 448 (and an ulp) to e4m3 at random, to the code below
// |z| / step + u steps with u = u16 / 65536. From 2^-6 on, a float whose low 20
// mantissa bits are cut off is that code (the exponent's bias apart), and
// adding u to those bits before the cut is the rounding. Below, neighbours are
// 2^-9 apart, as they are from 2^-6 to 2^-5: 2^-6 is added, and its code
// taken away again. `u24` is u16 << 8; the code plus 192 is in the top byte.
__device__ __forceinline__ uint32_t round_random(float z, uint32_t u24) {
  uint32_t b = __float_as_uint(z);
  if (fabsf(z) < 0x1p-6f) b = __float_as_uint(fabsf(z) + 0x1p-6f) - (8u << 20);
  return (b << 4) + u24;  // the sign is shifted out
}

// The codes of four such words.
__device__ __forceinline__ uint32_t codes4(uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  const uint32_t w = __byte_perm(__byte_perm(a, b, 0x0073), __byte_perm(c, d, 0x0073), 0x5410);
  return ((w & 0x7f7f7f7fu) + 0x40404040u) ^ (w & 0x80808080u);  // 64 added to each byte
}

// The signs of four floats, where e4m3 has them.
__device__ __forceinline__ uint32_t signs4(float a, float b, float c, float d) {
  const uint32_t lo = __byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0073);
  const uint32_t hi = __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0073);
  return __byte_perm(lo, hi, 0x5410) & 0x80808080u;
}

// Where a lane's eight elements are: neighbours, or 32 apart so that single
// elements coalesce. Both cover the warp's 256.
template <bool VEC, typename T>
__device__ __forceinline__ void load8(const T* p, unsigned long long warp_base, int lane, long long left,
                                      float (&f)[8]) {
  if constexpr (VEC) {
    unpack<T>(load_oct(p + warp_base + lane * 8), f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      f[j] = j * 32 + lane < left ? to_float<T>(p[warp_base + j * 32 + lane]) : 0.0f;
  }
}

template <bool VEC, typename T>
__device__ __forceinline__ void store8(T* p, unsigned long long warp_base, int lane, long long left,
                                       const float (&f)[8]) {
  if constexpr (VEC) {
    store_vec<T>(p + warp_base + lane * 8, pack<T>(f));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * 32 + lane < left) p[warp_base + j * 32 + lane] = from_float<T>(f[j]);
  }
}

template <bool VEC>
__device__ __forceinline__ void load8_e4m3(const void* p, unsigned long long warp_base, int lane, long long left,
                                           float (&f)[8]) {
  const uint8_t* b = static_cast<const uint8_t*>(p) + warp_base;
  uint2 q = make_uint2(0, 0);
  if constexpr (VEC) {
    q = *reinterpret_cast<const uint2*>(b + lane * 8);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const uint32_t x = j * 32 + lane < left ? b[j * 32 + lane] : 0;
      if (j < 4) q.x |= x << (8 * j);
      else q.y |= x << (8 * (j - 4));
    }
  }
  from_e4m3(q, f);
}

template <bool VEC>
__device__ __forceinline__ void store8_codes(void* p, unsigned long long warp_base, int lane, long long left, uint2 q) {
  uint8_t* b = static_cast<uint8_t*>(p) + warp_base;
  if constexpr (VEC) {
    *reinterpret_cast<uint2*>(b + lane * 8) = q;
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * 32 + lane < left) b[j * 32 + lane] = uint8_t((j < 4 ? q.x : q.y) >> (8 * (j & 3)));
  }
}

// The step's numbers as the kernel uses them.
struct StepValues {
  float scale, lr, size, root;  // size: lr / (1 - b1^t); root: 1 / sqrt(1 - b2^t)
  unsigned t;
};

// The sum of the partial gradients, times the scale.
template <bool VEC, typename G, typename Args>
__device__ __forceinline__ void load_gradient(const Args& a, const unsigned long long* from, unsigned long long base,
                                              int lane, long long left, float scale, float (&g)[8]) {
  load8<VEC>(reinterpret_cast<const G*>(from[0]), base, lane, left, g);
#pragma unroll 1
  for (int k = 1; k < a.parts; ++k) {
    float f[8];
    load8<VEC>(reinterpret_cast<const G*>(from[k]), base, lane, left, f);
#pragma unroll
    for (int j = 0; j < 8; ++j) g[j] += f[j];
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) g[j] *= scale;
}

// a x + b y: the products and their sum are rounded one by one, so that the
// states do not depend on what a compiler fuses (it fuses paired products and
// sums even where they are written apart).
__device__ __forceinline__ void blend(Pair x, float a, Pair y, float b, float& lo, float& hi) {
  float x0, x1, y0, y1;
  split(x * pair(a, a), x0, x1);
  split(y * pair(b, b), y0, y1);
  lo = __fadd_rn(x0, y0);
  hi = __fadd_rn(x1, y1);
}

// One warp's 256 elements from `base` on. VEC: all there, and every address
// on an octet's boundary. States in fp32.
template <typename P, typename C, typename G, bool VEC, typename Args>
__device__ __forceinline__ void step_tile(const Args& a, const StepValues& r, const Entry& e,
                                          const unsigned long long* from, unsigned long long base, long long left,
                                          int lane) {
  float g[8], m[8], v[8], p[8];
  load8<VEC>(static_cast<const P*>(e.param), base, lane, left, p);
  load8<VEC>(static_cast<const float*>(e.m), base, lane, left, m);
  load8<VEC>(static_cast<const float*>(e.v), base, lane, left, v);
  load_gradient<VEC, G>(a, from, base, lane, left, r.scale, g);
  const float keep = 1.0f - r.lr * e.decay;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const Pair gg = pair(g[j], g[j + 1]);
    blend(pair(m[j], m[j + 1]), a.b1, gg, a.b1c, m[j], m[j + 1]);
    blend(pair(v[j], v[j + 1]), a.b2, gg * gg, a.b2c, v[j], v[j + 1]);
  }
#pragma unroll
  for (int j = 0; j < 8; ++j)  // the quotient is off by two units in the last place at most, and far below p
    p[j] = p[j] * keep - __fdividef(m[j] * r.size, sqrtf(v[j]) * r.root + a.eps);
  store8<VEC>(static_cast<P*>(e.param), base, lane, left, p);
  if constexpr (sizeof(C) != sizeof(P)) store8<VEC>(static_cast<C*>(e.copy), base, lane, left, p);
  store8<VEC>(static_cast<float*>(e.m), base, lane, left, m);
  store8<VEC>(static_cast<float*>(e.v), base, lane, left, v);
}

// sqrt(x) for x = 0 and from 2^-100 to 2^120: one step of Newton's iteration on
// x y, y = 1 / sqrt(x), with the residual x - s^2 exact by a fused product
// (Markstein, "Computation of elementary functions on the IBM RISC System/6000
// processor", 1990). Without a branch, where sqrtf has one an element; it is sqrtf's result but for
// a few in a million, which are its neighbours.
__device__ __forceinline__ Pair root_of(float x0, float x1) {
  const Pair x = pair(x0, x1), y = pair(rsqrtf(fmaxf(x0, 0x1p-100f)), rsqrtf(fmaxf(x1, 0x1p-100f)));
  const Pair s = x * y, half = y * pair(0.5f, 0.5f), minus = s * pair(-1.0f, -1.0f);
  return fma(fma(minus, s, x), half, s);
}

__device__ __forceinline__ float quotient(float n, float d) {  // d a normal number below 2^126
  float r;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(d));
  return n * r;
}

// The same with states in e4m3. v is kept as 2^64 v and its root as 2^32
// sqrt(v) while it is computed, which changes no rounding and keeps the
// smallest ones normal; a block whose v would overflow so takes the plain way.
template <typename P, typename C, typename G, bool VEC, typename Args>
__device__ __forceinline__ void step_tile8(const Args& a, const StepValues& r, const Entry& e,
                                           const unsigned long long* from, unsigned long long base, long long left,
                                           int lane) {
  float g[8], m[8], v[8], p[8];
  load8<VEC>(static_cast<const P*>(e.param), base, lane, left, p);
  float ms = e.m_scale[base >> 8], vs = e.v_scale[base >> 8];
  load8_e4m3<VEC>(e.m, base, lane, left, m);
  load8_e4m3<VEC>(e.v, base, lane, left, v);
  load_gradient<VEC, G>(a, from, base, lane, left, r.scale, g);
  const float big = vs * 0x1p32f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    const Pair gg = pair(g[j], g[j + 1]), gb = gg * pair(0x1p32f, 0x1p32f);
    const Pair q = pair(v[j], v[j + 1]) * pair(big, big);
    blend(pair(m[j], m[j + 1]) * pair(ms, ms), a.b1, gg, a.b1c, m[j], m[j + 1]);
    blend(q * q, a.b2, gb * gb, a.b2c, v[j], v[j + 1]);
  }
  if (__reduce_max_sync(~0u, top_of(v)) < 0x7b800000u) {  // 2^120
#pragma unroll
    for (int j = 0; j < 8; j += 2) split(root_of(v[j], v[j + 1]), v[j], v[j + 1]);
  } else {
    load8_e4m3<VEC>(e.v, base, lane, left, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float q = v[j] * vs;
      v[j] = sqrtf(__fadd_rn(q * q * a.b2, g[j] * g[j] * a.b2c)) * 0x1p32f;
    }
  }
  const float keep = 1.0f - r.lr * e.decay, root = r.root * 0x1p-32f;
#pragma unroll
  for (int j = 0; j < 8; j += 2) {
    float n0, n1, d0, d1, k0, k1;
    split(pair(m[j], m[j + 1]) * pair(r.size, r.size), n0, n1);
    split(fma(pair(v[j], v[j + 1]), pair(root, root), pair(a.eps, a.eps)), d0, d1);
    split(pair(p[j], p[j + 1]) * pair(keep, keep), k0, k1);
    p[j] = k0 - quotient(n0, d0);
    p[j + 1] = k1 - quotient(n1, d1);
  }
  store8<VEC>(static_cast<P*>(e.param), base, lane, left, p);
  if constexpr (sizeof(C) != sizeof(P)) store8<VEC>(static_cast<C*>(e.copy), base, lane, left, p);
  ms = scale_of(__reduce_max_sync(~0u, top_of(m)));
  vs = scale_of(__float_as_uint(__uint_as_float(__reduce_max_sync(~0u, top_of(v))) * 0x1p-32f));
  const float mi = 1.0f / ms, vi = 1.0f / vs * 0x1p-32f;
  const uint32_t key = a.seed + r.t * 0x165667B1u + e.index * 0x3C6EF35Fu + uint32_t(base >> 32) * 0x6A09E667u;
  uint32_t at = (uint32_t(base) + (VEC ? lane * 8 : lane)) * 0x9E3779B9u + key;
  const uint32_t next = VEC ? 0x9E3779B9u : 32u * 0x9E3779B9u;
  uint32_t mw[8], vw[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const uint32_t bits = mix(at);
    at += next;
    mw[j] = round_random(m[j] * mi, __byte_perm(bits, 0, 0x4324));  // the upper half
    // A positive root has the least code at least, which is 2^-9.
    const float y = v[j] * vi;
    vw[j] = round_random(v[j] > 0.0f ? fmaxf(y, 0x1p-9f) : y, __byte_perm(bits, 0, 0x4104));  // the lower half
  }
  store8_codes<VEC>(e.m, base, lane, left,
                    make_uint2(codes4(mw[0], mw[1], mw[2], mw[3]) | signs4(m[0], m[1], m[2], m[3]),
                               codes4(mw[4], mw[5], mw[6], mw[7]) | signs4(m[4], m[5], m[6], m[7])));
  store8_codes<VEC>(e.v, base, lane, left,
                    make_uint2(codes4(vw[0], vw[1], vw[2], vw[3]), codes4(vw[4], vw[5], vw[6], vw[7])));
  if (lane == 0) {
    e.m_scale[base >> 8] = ms;
    e.v_scale[base >> 8] = vs;
  }
}

// P: parameters; C: their copy (P itself: none); G: gradients; S8: states in e4m3.
template <typename P, typename C, typename G, bool S8, int WORDS>
__global__ void __launch_bounds__(kThreads, S8 ? 4 : 3) adamw_kernel(const __grid_constant__ AdamArgs<WORDS> a) {
  float scale = a.s.scale_host;
  if (a.s.scale) scale *= *a.s.scale;
  if (!(fabsf(scale) <= kLargest)) return;  // no step
  float lr = a.s.lr_host, root = a.s.t_root, size = a.s.t_lr_m;
  unsigned t = a.s.t_host;
  if (a.s.t || a.s.lr) {
    if (a.s.lr) lr = *a.s.lr;
    float inv1 = a.s.inv1;
    if (a.s.t) {
      // 1 - b^t = -expm1(t ln b): no cancellation while b^t is near 1.
      const long long td = *a.s.t < 1 ? 1 : *a.s.t;
      t = unsigned(td);
      inv1 = 1.0f / -expm1f(float(td) * a.ln_b1);
      root = 1.0f / sqrtf(-expm1f(float(td) * a.ln_b2));
    }
    size = lr * inv1;
    if (!(fabsf(size) <= kLargest)) return;  // as the host refuses such a step
  }
  const StepValues r{scale, lr, size, root, t};
  const Entry* entries = reinterpret_cast<const Entry*>(a.words);
  const unsigned long long* grads = a.words + (size_t)a.count * kEntryWords;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int i = find_tensor(blockIdx.x, a.count, [&](int k) { return entries[k].first; });
  for (unsigned c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    while (i + 1 < a.count && entries[i + 1].first <= c) ++i;
    const Entry& e = entries[i];
    const unsigned long long base = (unsigned long long)(c - e.first) * kChunk + (unsigned)warp * 256u;
    if (base >= e.size) continue;  // the whole warp
    const long long left = (long long)(e.size - base);
    const unsigned long long* from = grads + (size_t)i * a.parts;
    const bool vec = e.vec && left >= 256;
    if constexpr (S8) {
      if (vec) step_tile8<P, C, G, true>(a, r, e, from, base, left, lane);
      else step_tile8<P, C, G, false>(a, r, e, from, base, left, lane);
    } else {
      if (vec) step_tile<P, C, G, true>(a, r, e, from, base, left, lane);
      else step_tile<P, C, G, false>(a, r, e, from, base, left, lane);
    }
  }
}

// The sum of two doubles over a warp, in a fixed order.
__device__ __forceinline__ double warp_sum(double s) {
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
  return s;
}

template <typename G, bool VEC>
struct NormRaw {
  Oct<G> o[kNormOctets];
  __device__ __forceinline__ void load(const G* p, int lane, long long) {
#pragma unroll
    for (int u = 0; u < kNormOctets; ++u) o[u] = load_oct(p + u * 256 + lane * 8);
  }
  __device__ __forceinline__ void get(int u, float (&f)[8]) const { unpack<G>(o[u], f); }
};

template <typename G>
struct NormRaw<G, false> {
  G e[kNormOctets][8];
  __device__ __forceinline__ void load(const G* p, int lane, long long left) {
#pragma unroll
    for (int u = 0; u < kNormOctets; ++u)
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int at = u * 256 + j * 32 + lane;
        e[u][j] = at < left ? p[at] : from_float<G>(0.0f);
      }
  }
  __device__ __forceinline__ void get(int u, float (&f)[8]) const {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = to_float<G>(e[u][j]);
  }
};

constexpr uint32_t kLeastSum = (127u - 120u) << 23;  // 2^-120 as an integer

// Squares of eight elements are added in fp32 and those sums in fp64: the
// result does not depend on how many elements there are. Where fp32 does not
// hold the squares they are formed again in fp64: above its range, or with a sum
// below 2^-120 (each is off by 2^-150 at most, together by less than 2^-27 of a larger
// sum). The sums of fp16 gradients are never there, unless they are zero.
template <typename G, int WORDS>
__global__ void __launch_bounds__(kThreads, 4) grad_norm_kernel(const __grid_constant__ GradArgs<WORDS> a) {
  __shared__ double sums[kThreads / 32];
  const GradEntry* entries = reinterpret_cast<const GradEntry*>(a.words);
  const unsigned long long* grads = a.words + (size_t)a.count * kGradEntryWords;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double total = 0.0;
  int i = find_tensor(blockIdx.x, a.count, [&](int k) { return entries[k].first; });
  for (unsigned c = blockIdx.x; c < a.chunks; c += gridDim.x) {
    while (i + 1 < a.count && entries[i + 1].first <= c) ++i;
    const GradEntry& e = entries[i];
    const unsigned long long base =
        (unsigned long long)(c - e.first) * kNormChunk + (unsigned)warp * (256u * kNormOctets);
    if (base >= e.size) continue;
    const long long left = (long long)(e.size - base);
    const unsigned long long* from = grads + (size_t)i * a.parts;
    // Octets of neighbours, or single elements 32 apart; either way all of a
    // part's loads are issued before the first is used.
    const auto add = [&](auto raw) {
      float g[kNormOctets][8];
      raw.load(reinterpret_cast<const G*>(from[0]) + base, lane, left);
#pragma unroll
      for (int u = 0; u < kNormOctets; ++u) raw.get(u, g[u]);
#pragma unroll 1
      for (int k = 1; k < a.parts; ++k) {
        raw.load(reinterpret_cast<const G*>(from[k]) + base, lane, left);
#pragma unroll
        for (int u = 0; u < kNormOctets; ++u) {
          float f[8];
          raw.get(u, f);
#pragma unroll
          for (int j = 0; j < 8; ++j) g[u][j] += f[j];
        }
      }
      float s[kNormOctets] = {};
      uint32_t off = 0;  // as integers, so that a NaN is above all
#pragma unroll
      for (int u = 0; u < kNormOctets; ++u) {
#pragma unroll
        for (int j = 0; j < 8; ++j) s[u] = fmaf(g[u][j], g[u][j], s[u]);
        off = max(off, __float_as_uint(s[u]) - kLeastSum);
      }
      if (std::is_same_v<G, __half> || __builtin_expect(off < 0x7f800000u - kLeastSum, 1)) {
#pragma unroll
        for (int u = 0; u < kNormOctets; ++u) total += double(s[u]);
      } else {
#pragma unroll
        for (int u = 0; u < kNormOctets; ++u) {
          double wide = double(s[u]);
          uint32_t any = 0;
#pragma unroll
          for (int j = 0; j < 8; ++j) any |= __float_as_uint(g[u][j]);
          // Not for zeros, which are common (200 M of bf16 took 74 us with it, not 64).
          if (any << 1 && __float_as_uint(s[u]) - kLeastSum >= 0x7f800000u - kLeastSum) {
            wide = 0.0;
#pragma unroll
            for (int j = 0; j < 8; ++j) wide = ::fma(double(g[u][j]), double(g[u][j]), wide);
          }
          total += wide;
        }
      }
    };
    if (e.vec && left >= 256 * kNormOctets) add(NormRaw<G, true>());
    else add(NormRaw<G, false>());
  }
  op_nearly_done();
  total = warp_sum(total);
  if (lane == 0) sums[warp] = total;
  __syncthreads();
  if (warp == 0) {
    total = warp_sum(lane < kThreads / 32 ? sums[lane] : 0.0);
    if (lane == 0) a.partial[blockIdx.x] = total;
  }
}

__global__ void __launch_bounds__(1024) grad_norm_end_kernel(const double* partial, int count, double max_norm,
                                                             double scale, float* out) {
  __shared__ double sums[32];
  double s = 0.0;
  op_wait_for_previous();
  for (int k = threadIdx.x; k < count; k += 1024) s += partial[k];
  s = warp_sum(s);
  if ((threadIdx.x & 31) == 0) sums[threadIdx.x >> 5] = s;
  __syncthreads();
  if (threadIdx.x < 32) {
    s = warp_sum(sums[threadIdx.x]);
    if (threadIdx.x == 0) {
      // Above 2^126 the reciprocal of the norm is no normal fp32 number: an overflow.
      const double root = sqrt(s), norm = scale * (root > 0x1p126 ? HUGE_VAL : root);
      const float shown = float(norm);
      const double clip = max_norm / (norm + 1e-6);
      out[0] = shown;
      out[1] = fabsf(shown) <= kLargest ? float(scale * (clip < 1.0 ? clip : 1.0)) : __int_as_float(0x7fffffff);
    }
  }
}

// ---------------------------------------------------------------- host

int size_of(int dtype) {
  switch (dtype) {
    case NB_OPTIM_FLOAT16:
    case NB_OPTIM_BFLOAT16: return 2;
    case NB_OPTIM_FLOAT32: return 4;
    default: return 0;
  }
}

bool on_boundary(const void* p, size_t unit) { return reinterpret_cast<uintptr_t>(p) % unit == 0; }

template <typename P, typename C, int WORDS>
const void* adamw_by_grad(int grad, bool s8) {
  switch (grad) {
    case NB_OPTIM_FLOAT16:
      return s8 ? reinterpret_cast<const void*>(adamw_kernel<P, C, __half, true, WORDS>)
                : reinterpret_cast<const void*>(adamw_kernel<P, C, __half, false, WORDS>);
    case NB_OPTIM_BFLOAT16:
      return s8 ? reinterpret_cast<const void*>(adamw_kernel<P, C, __nv_bfloat16, true, WORDS>)
                : reinterpret_cast<const void*>(adamw_kernel<P, C, __nv_bfloat16, false, WORDS>);
    default:
      return s8 ? reinterpret_cast<const void*>(adamw_kernel<P, C, float, true, WORDS>)
                : reinterpret_cast<const void*>(adamw_kernel<P, C, float, false, WORDS>);
  }
}

template <int WORDS>
const void* adamw_for(int param, int copy, int grad, bool s8) {
  if (param == NB_OPTIM_FLOAT16) return adamw_by_grad<__half, __half, WORDS>(grad, s8);
  if (param == NB_OPTIM_BFLOAT16) return adamw_by_grad<__nv_bfloat16, __nv_bfloat16, WORDS>(grad, s8);
  if (copy == NB_OPTIM_FLOAT16) return adamw_by_grad<float, __half, WORDS>(grad, s8);
  if (copy == NB_OPTIM_BFLOAT16) return adamw_by_grad<float, __nv_bfloat16, WORDS>(grad, s8);
  return adamw_by_grad<float, float, WORDS>(grad, s8);
}

template <int WORDS>
const void* grad_norm_for(int grad) {
  switch (grad) {
    case NB_OPTIM_FLOAT16: return reinterpret_cast<const void*>(grad_norm_kernel<__half, WORDS>);
    case NB_OPTIM_BFLOAT16: return reinterpret_cast<const void*>(grad_norm_kernel<__nv_bfloat16, WORDS>);
    default: return reinterpret_cast<const void*>(grad_norm_kernel<float, WORDS>);
  }
}

constexpr uint32_t kAdamMagic = 0x6164616d, kNormMagic = 0x6e6f726d;

struct Launch {
  bool large = false;
  unsigned blocks = 0;
  std::vector<unsigned long long> words;
  unsigned chunks = 0;
  int count = 0;
};

struct AdamHandle {
  uint32_t magic = kAdamMagic;
  int device = 0, parts = 1;
  double beta1 = 0, beta2 = 0, eps = 0;
  unsigned seed = 0;
  const void* kernel[2] = {};  // small and large list
  std::vector<Launch> launches;
};

struct NormHandle {
  uint32_t magic = kNormMagic;
  int device = 0, parts = 1, partials = 0;
  const void* kernel[2] = {};
  std::vector<Launch> launches;
};

template <typename E, typename Fill>
std::vector<Launch> build_launches(const uint64_t* sizes, int count, int parts, const void* const* grad,
                                   unsigned most_blocks, unsigned chunk, Fill fill) {
  constexpr int kWords = sizeof(E) / 8;
  std::vector<Launch> out;
  for (const TableLaunch& t : pack_tensors(sizes, size_t(count), kLargeWords / (kWords + parts), chunk)) {
    Launch l;
    l.count = int(t.tensor.size());
    l.chunks = t.chunks;
    l.words.resize(size_t(l.count) * size_t(kWords + parts));
    for (int k = 0; k < l.count; ++k) {
      E e{};
      const int i = t.tensor[size_t(k)];
      e.size = sizes[i];
      e.first = t.first[size_t(k)];
      fill(i, e);
      std::memcpy(&l.words[size_t(k) * kWords], &e, sizeof e);
      for (int p = 0; p < parts; ++p)
        l.words[size_t(l.count) * kWords + size_t(k) * size_t(parts) + size_t(p)] =
            reinterpret_cast<unsigned long long>(grad[size_t(i) * size_t(parts) + size_t(p)]);
    }
    l.large = l.words.size() > size_t(kSmallWords);
    l.blocks = l.chunks < most_blocks ? l.chunks : most_blocks;
    out.push_back(std::move(l));
  }
  return out;
}

template <typename Args>
cudaError_t launch_list(const Launch& l, const void* kernel, Args& args, cudaStream_t stream) {
  args.count = l.count;
  args.chunks = l.chunks;
  std::memcpy(args.words, l.words.data(), l.words.size() * 8);
  void* argv[] = {&args};
  return cudaLaunchKernel(kernel, dim3(l.blocks), dim3(kThreads), argv, 0, stream);
}

// Lists of one launch: null entries and alignment to the element.
const char* check_list(const uint64_t* sizes, int count, int parts, const void* const* grad, int gs) {
  for (int i = 0; i < count; ++i) {
    if (!sizes[i]) continue;
    for (int p = 0; p < parts; ++p) {
      const void* g = grad[size_t(i) * size_t(parts) + size_t(p)];
      if (!g || !on_boundary(g, size_t(gs))) return "bad arguments: null or misaligned gradient";
    }
  }
  return nullptr;
}

}  // namespace
}  // namespace nb

using namespace nb;

extern "C" void* nb_adamw_create(const nb_adamw_t* a, char* err, size_t errcap) {
  op_message(err, errcap, "");
  const auto refuse = [&](const char* why) -> void* {
    op_message(err, errcap, why);
    return nullptr;
  };
  if (!a || a->count < 1 || !a->size || !a->param || !a->grad || !a->m || !a->v || !a->weight_decay)
    return refuse("bad arguments: null or empty list of tensors");
  if (a->parts < 1 || a->parts > 8) return refuse("bad arguments: 1 to 8 partial gradients");
  const int ps = size_of(a->param_dtype), gs = size_of(a->grad_dtype), cs = a->copy_dtype ? size_of(a->copy_dtype) : 0;
  if (!ps || !gs) return refuse("bad arguments: parameters and gradients are ncclFloat16, ncclFloat32 or ncclBfloat16");
  if (a->copy_dtype && (cs != 2 || ps != 4 || !a->copy))
    return refuse("bad arguments: a copy is ncclFloat16 or ncclBfloat16 beside ncclFloat32 parameters");
  const bool s8 = a->state_dtype == NB_OPTIM_FLOAT8E4M3;
  if (!s8 && a->state_dtype != NB_OPTIM_FLOAT32)
    return refuse("bad arguments: states are ncclFloat32 or ncclFloat8e4m3");
  if (s8 && (!a->m_scale || !a->v_scale)) return refuse("bad arguments: 8-bit states need their scales");
  if (!(a->beta1 >= 0 && a->beta1 < 1) || !(a->beta2 >= 0 && a->beta2 < 1) || !(a->eps >= 1.2e-38) || !(a->eps <= 3.4e38))
    return refuse("bad arguments: 0 <= beta < 1 and eps a positive normal fp32 number");
  if (const char* why = check_list(a->size, a->count, a->parts, a->grad, gs)) return refuse(why);
  for (int i = 0; i < a->count; ++i) {
    if (!std::isfinite(a->weight_decay[i])) return refuse("bad arguments: weight_decay must be finite");
    if (!a->size[i]) continue;
    if (!a->param[i] || !on_boundary(a->param[i], size_t(ps)) || !a->m[i] || !a->v[i] ||
        (!s8 && (!on_boundary(a->m[i], 4) || !on_boundary(a->v[i], 4))) ||
        (cs && (!a->copy[i] || !on_boundary(a->copy[i], size_t(cs)))) ||
        (s8 && (!a->m_scale[i] || !a->v_scale[i] || !on_boundary(a->m_scale[i], 4) || !on_boundary(a->v_scale[i], 4))))
      return refuse("bad arguments: null or misaligned tensor");
  }
  OpDevice dev(a->device);
  if (dev.error()) return refuse("cannot use the device");
  try {
    std::unique_ptr<AdamHandle> h(new AdamHandle);
    h->device = a->device;
    h->parts = a->parts;
    h->beta1 = a->beta1;
    h->beta2 = a->beta2;
    h->eps = a->eps;
    h->seed = a->seed * 0x27D4EB2Fu;
    h->kernel[0] = adamw_for<kSmallWords>(a->param_dtype, a->copy_dtype, a->grad_dtype, s8);
    h->kernel[1] = adamw_for<kLargeWords>(a->param_dtype, a->copy_dtype, a->grad_dtype, s8);
    // 32-bit states are bound by HBM, and a block per chunk sweeps it in order
    // (201 M elements: 834 us, against 870 to 966 with 3 to 24 blocks an SM that
    // stride over the chunks); 8-bit ones by their arithmetic, so that a block's
    // setup counts (255 M: 898 us with 12 an SM, 986 with a block per chunk).
    const unsigned most = s8 ? unsigned(dev.sms()) * 12u : ~0u;
    h->launches = build_launches<Entry>(a->size, a->count, a->parts, a->grad, most, kChunk, [&](int i, Entry& e) {
      e.param = a->param[i];
      e.copy = cs ? a->copy[i] : nullptr;
      e.m = a->m[i];
      e.v = a->v[i];
      e.m_scale = s8 ? a->m_scale[i] : nullptr;
      e.v_scale = s8 ? a->v_scale[i] : nullptr;
      e.index = unsigned(i);
      e.decay = a->weight_decay[i];
      bool vec = on_boundary(e.param, size_t(ps) * 8) && (!cs || on_boundary(e.copy, size_t(cs) * 8)) &&
                 on_boundary(e.m, s8 ? 8 : 32) && on_boundary(e.v, s8 ? 8 : 32);
      for (int p = 0; p < a->parts; ++p)
        vec = vec && on_boundary(a->grad[size_t(i) * size_t(a->parts) + size_t(p)], size_t(gs) * 8);
      e.vec = vec;
    });
    return h.release();
  } catch (...) {
    return refuse("out of host memory");
  }
}

extern "C" int nb_adamw_step(const void* handle, int64_t t, const int64_t* t_dev, double lr, const float* lr_dev,
                             double scale, const float* scale_dev, void* stream, char* err, size_t errcap) {
  op_message(err, errcap, "");
  const AdamHandle* h = static_cast<const AdamHandle*>(handle);
  if (!h || h->magic != kAdamMagic) return op_refuse(err, errcap, "bad arguments: not an AdamW handle");
  if (!t_dev && t < 1) return op_refuse(err, errcap, "bad arguments: steps count from 1");
  StepScalars s{};
  s.t = reinterpret_cast<const long long*>(t_dev);
  s.lr = lr_dev;
  s.scale = scale_dev;
  s.lr_host = float(lr);
  s.scale_host = float(scale);
  s.t_host = unsigned(t);
  if (!t_dev) {
    const double inv1 = 1.0 / -std::expm1(double(t) * std::log(h->beta1));
    s.inv1 = float(inv1);
    s.t_lr_m = float(lr * inv1);
    s.t_root = float(1.0 / std::sqrt(-std::expm1(double(t) * std::log(h->beta2))));
  }
  // Checked as the kernel gets them: past fp32's range they would be infinite there.
  if (!lr_dev && (!std::isfinite(s.lr_host) || !std::isfinite(s.t_lr_m)))
    return op_refuse(err, errcap, "bad arguments: lr, and lr / (1 - beta1^t), must be finite in fp32");
  if (!std::isfinite(s.scale_host)) return op_refuse(err, errcap, "bad arguments: scale must be finite in fp32");
  OpDevice dev(h->device);
  if (dev.error()) return op_refuse(err, errcap, "cannot use the device", int(dev.error()));
  const auto fill = [&](auto& k) {
    k.s = s;
    k.b1 = float(h->beta1);
    k.b1c = float(1.0 - h->beta1);
    k.b2 = float(h->beta2);
    k.b2c = float(1.0 - h->beta2);
    k.eps = float(h->eps);
    k.ln_b1 = float(std::log(h->beta1));
    k.ln_b2 = float(std::log(h->beta2));
    k.seed = h->seed;
    k.parts = h->parts;
  };
  for (const Launch& l : h->launches) {
    cudaError_t e;
    if (l.large) {
      AdamArgs<kLargeWords> k;
      fill(k);
      e = launch_list(l, h->kernel[1], k, static_cast<cudaStream_t>(stream));
    } else {
      AdamArgs<kSmallWords> k;
      fill(k);
      e = launch_list(l, h->kernel[0], k, static_cast<cudaStream_t>(stream));
    }
    if (e != cudaSuccess) return op_refuse(err, errcap, "launch of the AdamW step failed", int(e));
  }
  return 0;
}

extern "C" void nb_adamw_destroy(void* handle) {
  AdamHandle* h = static_cast<AdamHandle*>(handle);
  if (h && h->magic == kAdamMagic) {
    h->magic = 0;
    delete h;
  }
}

extern "C" void* nb_grad_norm_create(int device, int count, int parts, int dtype, const uint64_t* size,
                                     const void* const* grad, char* err, size_t errcap) {
  op_message(err, errcap, "");
  const auto refuse = [&](const char* why) -> void* {
    op_message(err, errcap, why);
    return nullptr;
  };
  if (count < 1 || !size || !grad) return refuse("bad arguments: null or empty list of tensors");
  if (parts < 1 || parts > 8) return refuse("bad arguments: 1 to 8 partial gradients");
  const int gs = size_of(dtype);
  if (!gs) return refuse("bad arguments: gradients are ncclFloat16, ncclFloat32 or ncclBfloat16");
  if (const char* why = check_list(size, count, parts, grad, gs)) return refuse(why);
  OpDevice dev(device);
  if (dev.error()) return refuse("cannot use the device");
  try {
    std::unique_ptr<NormHandle> h(new NormHandle);
    h->device = device;
    h->parts = parts;
    h->kernel[0] = grad_norm_for<kSmallWords>(dtype);
    h->kernel[1] = grad_norm_for<kLargeWords>(dtype);
    h->launches = build_launches<GradEntry>(size, count, parts, grad, unsigned(dev.sms()) * 8u, kNormChunk,
                                             [&](int i, GradEntry& e) {
      bool vec = true;
      for (int p = 0; p < parts; ++p)
        vec = vec && on_boundary(grad[size_t(i) * size_t(parts) + size_t(p)], size_t(gs) * 8);
      e.vec = vec;
    });
    for (const Launch& l : h->launches) h->partials += int(l.blocks);
    return h.release();
  } catch (...) {
    return refuse("out of host memory");
  }
}

extern "C" int nb_grad_norm_partials(const void* handle) {
  const NormHandle* h = static_cast<const NormHandle*>(handle);
  return h && h->magic == kNormMagic ? h->partials : -1;
}

extern "C" int nb_grad_norm(const void* handle, double max_norm, double scale, float* out, double* workspace,
                            void* stream, char* err, size_t errcap) {
  op_message(err, errcap, "");
  const NormHandle* h = static_cast<const NormHandle*>(handle);
  if (!h || h->magic != kNormMagic) return op_refuse(err, errcap, "bad arguments: not a gradient norm's handle");
  if (!(max_norm > 0)) return op_refuse(err, errcap, "bad arguments: max_norm must be positive");
  if (!(scale > 0) || !std::isfinite(float(scale)))
    return op_refuse(err, errcap, "bad arguments: scale must be positive, and finite in fp32");
  if (!out || !on_boundary(out, 4) || (h->partials && (!workspace || !on_boundary(workspace, 8))))
    return op_refuse(err, errcap, "bad arguments: null or misaligned output or workspace");
  OpDevice dev(h->device);
  if (dev.error()) return op_refuse(err, errcap, "cannot use the device", int(dev.error()));
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* at = workspace;
  for (const Launch& l : h->launches) {
    cudaError_t e;
    if (l.large) {
      GradArgs<kLargeWords> k;
      k.partial = at;
      k.parts = h->parts;
      e = launch_list(l, h->kernel[1], k, st);
    } else {
      GradArgs<kSmallWords> k;
      k.partial = at;
      k.parts = h->parts;
      e = launch_list(l, h->kernel[0], k, st);
    }
    if (e != cudaSuccess) return op_refuse(err, errcap, "launch of the gradient norm failed", int(e));
    at += l.blocks;
  }
  const double* partial = workspace;
  int count = h->partials;
  double limit = max_norm;
  void* argv[] = {&partial, &count, &limit, &scale, &out};
  const cudaError_t e =
      op_launch_after(reinterpret_cast<const void*>(grad_norm_end_kernel), dim3(1), dim3(1024), argv, st);
  return e == cudaSuccess ? 0 : op_refuse(err, errcap, "launch of the gradient norm failed", int(e));
}

extern "C" void nb_grad_norm_destroy(void* handle) {
  NormHandle* h = static_cast<NormHandle*>(handle);
  if (h && h->magic == kNormMagic) {
    h->magic = 0;
    delete h;
  }
}
