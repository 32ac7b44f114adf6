// Eight neighbouring elements as one thread holds them, and the reductions
// over the threads of a row: shared by the norm and the optimizer kernels.
//
// An octet of a 16-bit type is one 16-byte access, of fp32 one 32-byte access
// (ld/st.global.v8, sm_100).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace nb {
namespace octet {

// For a kernel that was launched while the stream's previous one was running:
// returns when that one has ended and its stores are visible. The previous one
// calls op_nearly_done() when only its last stores are left.
__device__ __forceinline__ void op_wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void op_nearly_done() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

constexpr float kE4m3Max = 448.0f;
// The least scale of a group of 8-bit values (2^-126): its reciprocal is finite.
constexpr float kLeastScale = 1.17549435e-38f;

// Two fp32 operations in one instruction (sm_100), each rounded as usual.
struct Pair {
  unsigned long long v;
};
__device__ __forceinline__ Pair pair(float a, float b) {
  Pair p;
  asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
  return p;
}
__device__ __forceinline__ void split(Pair p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p.v));
}
__device__ __forceinline__ Pair operator*(Pair a, Pair b) {
  Pair r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair operator+(Pair a, Pair b) {
  Pair r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v));
  return r;
}
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) {
  Pair r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return r;
}

template <typename T>
struct Oct {
  uint4 v[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ float to_float(T x) { return float(x); }
template <> __device__ __forceinline__ float to_float<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float to_float<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_float(float x) { return T(x); }
template <> __device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

template <typename T>
__device__ __forceinline__ Oct<T> load_oct(const T* p) {
  Oct<T> o;
  if constexpr (sizeof(T) == 4) {
    asm volatile("ld.global.v8.u32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                 : "=r"(o.v[0].x), "=r"(o.v[0].y), "=r"(o.v[0].z), "=r"(o.v[0].w), "=r"(o.v[1].x), "=r"(o.v[1].y),
                   "=r"(o.v[1].z), "=r"(o.v[1].w)
                 : "l"(p));
  } else {
    asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];"
                 : "=r"(o.v[0].x), "=r"(o.v[0].y), "=r"(o.v[0].z), "=r"(o.v[0].w)
                 : "l"(p));
  }
  return o;
}

// Two neighbours of a 16-bit type at a time.
__device__ __forceinline__ float2 to_float2(__half, uint32_t w) {
  return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
__device__ __forceinline__ float2 to_float2(__nv_bfloat16, uint32_t w) {
  return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ uint32_t from_float2(__half, float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t from_float2(__nv_bfloat16, float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

template <typename T>
__device__ __forceinline__ void unpack(const Oct<T>& o, float (&f)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&o);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = __uint_as_float(w[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 v = to_float2(T(), w[j]);
      f[2 * j] = v.x;
      f[2 * j + 1] = v.y;
    }
  }
}

template <typename T>
__device__ __forceinline__ void unpack(const Oct<T>& o, Pair (&p)[4]) {
  float f[8];
  unpack<T>(o, f);
#pragma unroll
  for (int j = 0; j < 4; ++j) p[j] = pair(f[2 * j], f[2 * j + 1]);
}

__device__ __forceinline__ void split(const Pair (&p)[4], float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) split(p[j], f[2 * j], f[2 * j + 1]);
}

template <typename T>
__device__ __forceinline__ Oct<T> pack(const float (&f)[8]) {
  Oct<T> o;
  uint32_t* w = reinterpret_cast<uint32_t*>(&o);
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int j = 0; j < 8; ++j) w[j] = __float_as_uint(f[j]);
  } else {
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = from_float2(T(), f[2 * j], f[2 * j + 1]);
  }
  return o;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Oct<T>& o) {
  if constexpr (sizeof(T) == 4) {
    asm volatile("st.global.v8.u32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(o.v[0].x), "r"(o.v[0].y),
                 "r"(o.v[0].z), "r"(o.v[0].w), "r"(o.v[1].x), "r"(o.v[1].y), "r"(o.v[1].z), "r"(o.v[1].w)
                 : "memory");
  } else {
    asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(o.v[0].x), "r"(o.v[0].y), "r"(o.v[0].z),
                 "r"(o.v[0].w)
                 : "memory");
  }
}

// Eight elements of a row as they are loaded, and their way back. VEC: an
// octet of neighbours on its boundary. Otherwise single elements `step` apart,
// with the row's other threads between them, so that a warp's accesses are
// neighbours (cutting unaligned octets out of aligned pieces took 92
// instructions an element of a norm, single elements take a fifth of that).
// `left`: elements of the row from the first on; those beyond read as zero.
// Plain (coherent) loads: an output may be one of the inputs.
template <typename T, bool VEC>
struct Raw {
  Oct<T> o;

  __device__ __forceinline__ void load(const T* p, int, int) { o = load_oct(p); }
  __device__ __forceinline__ void get(Pair (&f)[4]) const { unpack<T>(o, f); }
};

template <typename T>
struct Raw<T, false> {
  T e[8];

  __device__ __forceinline__ void load(const T* p, int step, int left) {
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = j * step < left ? p[j * step] : from_float<T>(0.0f);
  }
  __device__ __forceinline__ void get(Pair (&f)[4]) const {
#pragma unroll
    for (int j = 0; j < 4; ++j) f[j] = pair(to_float<T>(e[2 * j]), to_float<T>(e[2 * j + 1]));
  }
};

template <typename T, bool VEC>
__device__ __forceinline__ void store8(T* p, const float (&f)[8], int step, int left) {
  if constexpr (VEC) {
    if (left > 0) store_vec<T>(p, pack<T>(f));
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j * step < left) p[j * step] = from_float<T>(f[j]);
  }
}

// Eight values to e4m3 (round to nearest even, saturating at 448; NaN stays NaN).
__device__ __forceinline__ uint2 to_e4m3(const float (&f)[8]) {
  uint32_t w[4];
#pragma unroll
  for (int j = 0; j < 4; ++j)
    w[j] = __nv_cvt_float2_to_fp8x2(make_float2(f[2 * j], f[2 * j + 1]), __NV_SATFINITE, __NV_E4M3);
  return make_uint2(w[0] | w[1] << 16, w[2] | w[3] << 16);
}

__device__ __forceinline__ void from_e4m3(uint2 q, float (&f)[8]) {
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const uint32_t w = j < 2 ? q.x : q.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(j & 1 ? w >> 16 : w), __NV_E4M3);
    const float2 v = __half22float2(__half2(h));
    f[2 * j] = v.x;
    f[2 * j + 1] = v.y;
  }
}

// The larger magnitude; NaN where one is (fmaxf would drop it). Magnitudes
// compare as their bit patterns do, a NaN above infinity, so that maxima over
// threads may be integer ones.
__device__ __forceinline__ float max_magnitude(float a, float b) {
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
  return r;
}
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }
__device__ __forceinline__ uint32_t top_of(const float (&f)[8]) {
  float m = fabsf(f[0]);
#pragma unroll
  for (int j = 1; j < 8; ++j) m = max_magnitude(m, f[j]);
  return magnitude(m);
}
// The same of those that exist: eight of VEC's, or the ones below `left`.
template <bool VEC>
__device__ __forceinline__ uint32_t top_of(const float (&f)[8], int step, int left) {
  if constexpr (VEC) return top_of(f);
  uint32_t m = 0;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = max(m, j * step < left ? magnitude(f[j]) : 0);
  return m;
}

// The scale of a group whose largest magnitude is `top`; NaN stays NaN.
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float s = __uint_as_float(top) * (1.0f / kE4m3Max);
  return s < kLeastScale ? kLeastScale : s;
}

}  // namespace octet
}  // namespace nb
