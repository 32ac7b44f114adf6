// Eight neighbouring elements as one thread holds them, and the reductions
// over the threads of a row: shared by the norm and the optimizer kernels.
//
// An octet of a 16-bit type is one 16-byte access, of fp32 one 32-byte access
// (ld/st.global.v8, sm_100). Where a pointer, a stride or a length keeps an
// octet off that boundary the same eight elements move one by one, under the
// bounds of their row.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <cstdint>

namespace nb {
namespace octet {

constexpr float kE4m3Max = 448.0f;
// The least scale of a group of 8-bit values (2^-126): its reciprocal is finite.
constexpr float kLeastScale = 1.17549435e-38f;

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

// `left` elements from p on exist; the others read as zero. Plain (coherent)
// loads: an output may be one of the inputs.
template <typename T, bool VEC>
__device__ __forceinline__ Oct<T> load(const T* p, int left) {
  Oct<T> o;
  if constexpr (VEC) {
    if constexpr (sizeof(T) == 4) {
      asm volatile("ld.global.v8.u32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
                   : "=r"(o.v[0].x), "=r"(o.v[0].y), "=r"(o.v[0].z), "=r"(o.v[0].w), "=r"(o.v[1].x),
                     "=r"(o.v[1].y), "=r"(o.v[1].z), "=r"(o.v[1].w)
                   : "l"(p));
    } else {
      asm volatile("ld.global.v4.u32 {%0,%1,%2,%3}, [%4];"
                   : "=r"(o.v[0].x), "=r"(o.v[0].y), "=r"(o.v[0].z), "=r"(o.v[0].w)
                   : "l"(p));
    }
  } else {
    T e[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) e[j] = j < left ? p[j] : from_float<T>(0.0f);
    uint32_t* w = reinterpret_cast<uint32_t*>(&o);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (sizeof(T) == 4) {
        w[j] = __float_as_uint(e[j]);
      } else {
        const uint32_t b = *reinterpret_cast<const uint16_t*>(&e[j]);
        w[j / 2] = j & 1 ? w[j / 2] | b << 16 : b;
      }
    }
  }
  return o;
}

template <typename T>
__device__ __forceinline__ void unpack(const Oct<T>& o, float (&f)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&o);
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if constexpr (sizeof(T) == 4) {
      f[j] = __uint_as_float(w[j]);
    } else {
      const uint16_t b = uint16_t(j & 1 ? w[j / 2] >> 16 : w[j / 2]);
      f[j] = to_float<T>(*reinterpret_cast<const T*>(&b));
    }
  }
}

template <typename T, bool VEC>
__device__ __forceinline__ void store(T* p, const float (&f)[8], int left) {
  if constexpr (VEC) {
    uint32_t w[sizeof(T) * 2];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      if constexpr (sizeof(T) == 4) {
        w[j] = __float_as_uint(f[j]);
      } else {
        const T e = from_float<T>(f[j]);
        const uint32_t b = *reinterpret_cast<const uint16_t*>(&e);
        w[j / 2] = j & 1 ? w[j / 2] | b << 16 : b;
      }
    }
    if constexpr (sizeof(T) == 4) {
      asm volatile("st.global.v8.u32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "r"(w[0]), "r"(w[1]),
                   "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                   : "memory");
    } else {
      asm volatile("st.global.v4.u32 [%0], {%1,%2,%3,%4};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                   "r"(w[3])
                   : "memory");
    }
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (j < left) p[j] = from_float<T>(f[j]);
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

// Magnitudes compare as their bit patterns do, and a NaN is above infinity:
// an integer maximum keeps a NaN that fmaxf would drop.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The scale of a group whose largest magnitude is `top`; NaN stays NaN.
__device__ __forceinline__ float scale_of(uint32_t top) {
  const float s = __uint_as_float(top) * (1.0f / kE4m3Max);
  return s < kLeastScale ? kLeastScale : s;
}

}  // namespace octet
}  // namespace nb
