// Element types of the operators that take fp32, fp16 or bf16 tensors: the
// type ids of the C ABI as C++ types, and conversions of C consecutive elements.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"

namespace btf {

inline bool elem_type_ok(int t) { return t == BTF_F32 || t == BTF_F16 || t == BTF_BF16; }
inline int elem_bytes(int t) { return t == BTF_F32 ? 4 : 2; }

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// C consecutive elements, moved as whole words when C > 1 (the address is then
// aligned to min(16, C * sizeof(T)) bytes).
template <typename T, int C>
struct Pack {
  static constexpr int kBytes = C * (int)sizeof(T);
  static constexpr int kWords = kBytes >= 4 ? kBytes / 4 : 1;
  uint32_t w[kWords];

  __device__ __forceinline__ void load(const T* p) {
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) {
        const uint4 v = reinterpret_cast<const uint4*>(p)[i];
        w[4 * i] = v.x, w[4 * i + 1] = v.y, w[4 * i + 2] = v.z, w[4 * i + 3] = v.w;
      }
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x, w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
      static_assert(kBytes == 2);
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void store(T* p) const {
    if constexpr (kBytes % 16 == 0) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i)
        reinterpret_cast<uint4*>(p)[i] = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
    } else if constexpr (kBytes == 8) {
      *reinterpret_cast<uint2*>(p) = make_uint2(w[0], w[1]);
    } else if constexpr (kBytes == 4) {
      *reinterpret_cast<uint32_t*>(p) = w[0];
    } else {
      *reinterpret_cast<uint16_t*>(p) = (uint16_t)w[0];
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 4) {
      return __uint_as_float(w[i]);
    } else {
      const uint16_t h = (uint16_t)(w[i >> 1] >> (16 * (i & 1)));
      if constexpr (std::is_same_v<T, __half>) return __half2float(__ushort_as_half(h));
      else return __uint_as_float((uint32_t)h << 16);
    }
  }
  __device__ __forceinline__ void set(int i, float v) {
    if constexpr (sizeof(T) == 4) {
      w[i] = __float_as_uint(v);
    } else {
      uint16_t h;
      if constexpr (std::is_same_v<T, __half>) h = __half_as_ushort(__float2half_rn(v));
      else h = __bfloat16_as_ushort(__float2bfloat16_rn(v));
      if ((i & 1) == 0) w[i >> 1] = h;
      else w[i >> 1] |= (uint32_t)h << 16;
    }
  }
};

}  // namespace btf
