// Elementwise rows of bf16, fp16 or fp32: eight neighbouring elements of one
// thread, converted to fp32 for the arithmetic and rounded once when stored.
#pragma once

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

template <typename T>
struct alignas(16) Pack8 {
  T e[8];
};

// p must be 16-byte aligned.
template <typename T>
__device__ __forceinline__ Pack8<T> load_pack(const T* p) {
  Pack8<T> r;
  uint4* d = reinterpret_cast<uint4*>(&r);
  const uint4* s = reinterpret_cast<const uint4*>(p);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r) / 16); ++i) d[i] = s[i];
  return r;
}
template <typename T>
__device__ __forceinline__ void store_pack(T* p, const Pack8<T>& r) {
  uint4* d = reinterpret_cast<uint4*>(p);
  const uint4* s = reinterpret_cast<const uint4*>(&r);
#pragma unroll
  for (int i = 0; i < (int)(sizeof(r) / 16); ++i) d[i] = s[i];
}

// Element i of a vector of any of the three types.
__device__ __forceinline__ float load_elem(const void* p, int type, int64_t i) {
  if (type == kElemBf16) return to_f32(reinterpret_cast<const __nv_bfloat16*>(p)[i]);
  if (type == kElemF16) return to_f32(reinterpret_cast<const __half*>(p)[i]);
  return reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_elem(void* p, int type, int64_t i, float v) {
  if (type == kElemBf16)
    reinterpret_cast<__nv_bfloat16*>(p)[i] = from_f32<__nv_bfloat16>(v);
  else if (type == kElemF16)
    reinterpret_cast<__half*>(p)[i] = from_f32<__half>(v);
  else
    reinterpret_cast<float*>(p)[i] = v;
}

}  // namespace b200
