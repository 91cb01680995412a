// Runs of N elements of a 32- or 16-bit float type as fp32 values: one or two 16-byte accesses for 8 elements
// (16-byte aligned), scalar otherwise.  Stores round to nearest.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

#include "common.cuh"

namespace swv {

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(__half x) { return __half2float(x); }
template <typename T>
__device__ __forceinline__ T from_f32(float x) {
  if constexpr (sizeof(T) == 4) return x;
  else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(x);
  else return __float2bfloat16_rn(x);
}

template <typename T>
__device__ __forceinline__ void unpack2(uint32_t w, float& a, float& b) {
  if constexpr (std::is_same_v<T, __half>) {
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w));
    a = f.x;
    b = f.y;
  } else {
    a = __uint_as_float(w << 16);
    b = __uint_as_float(w & 0xffff0000u);
  }
}
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __half>) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    return pack_bf16x2(a, b);
  }
}

template <typename T, int N>
__device__ __forceinline__ void load_run(const T* p, float* v) {
  if constexpr (N == 8 && sizeof(T) == 4) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
    v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
  } else if constexpr (N == 8) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    unpack2<T>(a.x, v[0], v[1]);
    unpack2<T>(a.y, v[2], v[3]);
    unpack2<T>(a.z, v[4], v[5]);
    unpack2<T>(a.w, v[6], v[7]);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = to_f32(p[i]);
  }
}
template <typename T, int N>
__device__ __forceinline__ void store_run(T* p, const float* v) {
  if constexpr (N == 8 && sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    *(reinterpret_cast<float4*>(p) + 1) = make_float4(v[4], v[5], v[6], v[7]);
  } else if constexpr (N == 8) {
    *reinterpret_cast<uint4*>(p) =
        make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) p[i] = from_f32<T>(v[i]);
  }
}

// A run of VEC elements as it lies in memory: half the registers of its fp32 values for 16-bit types.
template <typename T, int VEC>
struct Raw {
  static constexpr int kWords = VEC * static_cast<int>(sizeof(T)) / 4 > 0 ? VEC * static_cast<int>(sizeof(T)) / 4 : 1;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (VEC == 8) {
#pragma unroll
      for (int i = 0; i < kWords; i += 4) {
        const uint4 a = __ldcs(reinterpret_cast<const uint4*>(p) + i / 4);      // read once
        w[i] = a.x; w[i + 1] = a.y; w[i + 2] = a.z; w[i + 3] = a.w;
      }
    } else if constexpr (sizeof(T) == 4) {
      w[0] = __float_as_uint(*p);
    } else {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    }
  }
  __device__ __forceinline__ void zero() {
#pragma unroll
    for (int i = 0; i < kWords; ++i) w[i] = 0u;
  }
  __device__ __forceinline__ void values(float* v) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < VEC; ++i) v[i] = __uint_as_float(w[i]);
    } else if constexpr (VEC == 8) {
#pragma unroll
      for (int i = 0; i < kWords; ++i) unpack2<T>(w[i], v[2 * i], v[2 * i + 1]);
    } else {
      float unused;
      unpack2<T>(w[0], v[0], unused);
    }
  }
};

// one element of an array whose type is known at run time
__device__ __forceinline__ float load_as_f32(const void* p, int dtype, int64_t i) {
  if (dtype == SWV_F32) return static_cast<const float*>(p)[i];
  if (dtype == SWV_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
  return __half2float(static_cast<const __half*>(p)[i]);
}
__device__ __forceinline__ void store_from_f32(void* p, int dtype, int64_t i, float x) {
  if (dtype == SWV_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == SWV_BF16) static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
  else static_cast<__half*>(p)[i] = __float2half_rn(x);
}

inline int dtype_bytes(int dtype) { return dtype == SWV_F32 ? 4 : 2; }
inline bool dtype_known(int dtype) { return dtype == SWV_F32 || dtype == SWV_BF16 || dtype == SWV_F16; }
// rows of `es`-byte elements, `stride` elements apart, whose 8-element runs all start on 16 bytes
inline bool rows_vec8(const void* p, int64_t stride, int es) {
  return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && (stride * es) % 16 == 0;
}

}  // namespace swv
