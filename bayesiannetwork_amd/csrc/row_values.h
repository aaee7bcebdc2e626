// What the operators on rows of logits and on gradient tensors share: element types, 16-byte
// loads and stores at any element alignment, reductions over lanes.
#pragma once

#include "../../include/bn_hip.h"

#include <cstdint>

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>

namespace bn_rows {

inline size_t dtype_bytes(int dtype) {
  switch (dtype) {
    case BN_F32: return 4;
    case BN_F64: return 8;
    case BN_F16: return 2;
    case BN_BF16: return 2;
  }
  return 0;
}

// The arithmetic type of a stored type (every conversion to it is exact), and how many make 16 bytes.
template <typename T>
struct Value {
  using Wide = float;
  static constexpr int kVec = 16 / (int)sizeof(T);
  static __device__ __forceinline__ float widen(T v) { return (float)v; }
  static __device__ __forceinline__ T round(float v) { return (T)v; }
};
template <>
struct Value<double> {
  using Wide = double;
  static constexpr int kVec = 2;
  static __device__ __forceinline__ double widen(double v) { return v; }
  static __device__ __forceinline__ double round(double v) { return v; }
};
template <>
struct Value<__hip_bfloat16> {
  using Wide = float;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float widen(__hip_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __hip_bfloat16 round(float v) { return __float2bfloat16(v); }
};
template <>
struct Value<__half> {
  using Wide = float;
  static constexpr int kVec = 8;
  static __device__ __forceinline__ float widen(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half round(float v) { return __float2half(v); }
};

// 16 bytes of T that need no more than T's own alignment: one global_load_dwordx4 /
// global_store_dwordx4 either way (the hardware takes any byte address for these).
template <typename T>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
  T v[Value<T>::kVec];
};

template <typename T>
__device__ __forceinline__ Pack<T> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T>*>(p);
}
template <typename T>
__device__ __forceinline__ void store_pack(T* p, const Pack<T>& v) {
  *reinterpret_cast<Pack<T>*>(p) = v;
}

template <int WIDTH>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int d = 1; d < WIDTH; d <<= 1) v = fmaxf(v, __shfl_xor(v, d, 64));
  return v;
}
template <int WIDTH>
__device__ __forceinline__ double lanes_max(double v) {
#pragma unroll
  for (int d = 1; d < WIDTH; d <<= 1) v = fmax(v, __shfl_xor(v, d, 64));
  return v;
}
// every lane of the group ends with the same sum, taken in the same tree
template <int WIDTH, typename W>
__device__ __forceinline__ W lanes_sum(W v) {
#pragma unroll
  for (int d = 1; d < WIDTH; d <<= 1) v += __shfl_xor(v, d, 64);
  return v;
}

}  // namespace bn_rows
