// Elementwise rows of bf16, fp16 or fp32: eight neighbouring elements of one
// thread, converted to fp32 for the arithmetic and rounded once when stored.
#pragma once

#include <type_traits>

#include "b200_common.cuh"

namespace b200 {

enum ElemType : int { kElemBf16 = 0, kElemF16 = 1, kElemF32 = 2 };

__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(float v) { return v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }

// E neighbouring elements as 32-bit words: unpacked two at a time by a shift and a
// mask (bf16) or one conversion (fp16), packed by one conversion for two.
template <typename T, int E>
struct alignas(sizeof(T) * E >= 16 ? 16 : sizeof(T) * E) Group {
  T e[E];
  __device__ __forceinline__ void unpack(float* f) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < E; ++j) f[j] = e[j];
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(e);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          f[2 * j] = __uint_as_float(w[j] << 16);
          f[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
        } else {
          const float2 v = __half22float2(*reinterpret_cast<const __half2*>(w + j));
          f[2 * j] = v.x;
          f[2 * j + 1] = v.y;
        }
      }
    }
  }
  __device__ __forceinline__ void pack(const float* f) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int j = 0; j < E; ++j) e[j] = f[j];
    } else {
      uint32_t* w = reinterpret_cast<uint32_t*>(e);
#pragma unroll
      for (int j = 0; j < E / 2; ++j) {
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          const __nv_bfloat162 v = __floats2bfloat162_rn(f[2 * j], f[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&v);
        } else {
          const __half2 v = __floats2half2_rn(f[2 * j], f[2 * j + 1]);
          w[j] = *reinterpret_cast<const uint32_t*>(&v);
        }
      }
    }
  }
  // p must be aligned to 16 bytes (or to the group, if that is smaller)
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (sizeof(*this) >= 16) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(*this) / 16); ++i)
        reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (sizeof(*this) >= 16) {
#pragma unroll
      for (int i = 0; i < (int)(sizeof(*this) / 16); ++i)
        reinterpret_cast<uint4*>(p)[i] = reinterpret_cast<const uint4*>(e)[i];
    } else {
      *reinterpret_cast<uint2*>(p) = *reinterpret_cast<const uint2*>(e);
    }
  }
  // The words stay packed up to here: values unpacked before are not kept for use after.
  __device__ __forceinline__ void hold() {
    uint32_t* w = reinterpret_cast<uint32_t*>(e);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(*this) / 4); ++i) asm volatile("" : "+r"(w[i]));
  }
  __device__ __forceinline__ void zero() {
    uint32_t* w = reinterpret_cast<uint32_t*>(e);
#pragma unroll
    for (int i = 0; i < (int)(sizeof(*this) / 4); ++i) w[i] = 0u;
  }
};

// Store to element i of a vector of any of the three types.
__device__ __forceinline__ void store_elem(void* p, int type, int64_t i, float v) {
  if (type == kElemBf16)
    reinterpret_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
  else if (type == kElemF16)
    reinterpret_cast<__half*>(p)[i] = from_f32<__half>(v);
  else
    reinterpret_cast<float*>(p)[i] = v;
}

}  // namespace b200
