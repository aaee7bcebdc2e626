// What the operators on rows of logits and on gradient tensors share: element types, 16-byte
// loads and stores at any element alignment, reductions over lanes.
#pragma once

#include "../../include/bn_hip.h"
#include "row_loads.h"

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

// The same past the caches' usual order of replacement, for what this kernel does not read again.
template <typename T>
__device__ __forceinline__ void store_pack_streamed(T* p, const Pack<T>& v) {
  typedef uint32_t Words __attribute__((ext_vector_type(4), aligned(2)));
  __builtin_nontemporal_store(__builtin_bit_cast(Words, v), reinterpret_cast<Words*>(p));
}

// A pack and its registers.  kept() hides where they came from, so that what was unpacked from them
// before (twice the registers for 16-bit types) is not kept alive for later use instead.
template <typename T>
__device__ __forceinline__ Raw raw_of(const Pack<T>& p) {
  return __builtin_bit_cast(Raw, p);
}
template <typename T>
__device__ __forceinline__ Pack<T> pack_of(const Raw& r) {
  return __builtin_bit_cast(Pack<T>, r);
}
__device__ __forceinline__ void kept(Raw& r) {
#pragma unroll
  for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(r.w[i]));
}

// A 32-bit word of the lane whose number differs by MASK, by permutations within the register file: quads and
// mirrors of 8 and 16 lanes, exchanged rows of 16 and halves of 32.  (Through the LDS crossbar each of these
// waits some hundred cycles, and sorts and reductions are chains of them.)
template <int MASK>
__device__ __forceinline__ uint32_t lane_xor(uint32_t v) {
  if constexpr (MASK == 1) return __builtin_amdgcn_mov_dpp(v, 0xB1, 0xF, 0xF, true);
  else if constexpr (MASK == 2) return __builtin_amdgcn_mov_dpp(v, 0x4E, 0xF, 0xF, true);
  else if constexpr (MASK == 3) return __builtin_amdgcn_mov_dpp(v, 0x1B, 0xF, 0xF, true);
  else if constexpr (MASK == 7) return __builtin_amdgcn_mov_dpp(v, 0x141, 0xF, 0xF, true);
  else if constexpr (MASK == 4) return lane_xor<3>(lane_xor<7>(v));
  else if constexpr (MASK == 8) return __builtin_amdgcn_mov_dpp(v, 0x128, 0xF, 0xF, true);
  else if constexpr (MASK == 15) return __builtin_amdgcn_mov_dpp(v, 0x140, 0xF, 0xF, true);
  else if constexpr (MASK == 16) {
    const auto both = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return (threadIdx.x & 16) ? both[0] : both[1];
  } else if constexpr (MASK == 31) return lane_xor<16>(lane_xor<15>(v));
  else if constexpr (MASK == 32) {
    const auto both = __builtin_amdgcn_permlane32_swap(v, v, false, false);
    return (threadIdx.x & 32) ? both[0] : both[1];
  } else {
    static_assert(MASK == 63, "a permutation that the sorts and reductions use");
    return lane_xor<32>(lane_xor<31>(v));
  }
}
template <int MASK>
__device__ __forceinline__ uint64_t lane_xor(uint64_t v) {
  return ((uint64_t)lane_xor<MASK>((uint32_t)(v >> 32)) << 32) | lane_xor<MASK>((uint32_t)v);
}
template <int MASK>
__device__ __forceinline__ int lane_xor(int v) {
  return (int)lane_xor<MASK>((uint32_t)v);
}
template <int MASK>
__device__ __forceinline__ float lane_xor(float v) {
  return __uint_as_float(lane_xor<MASK>(__float_as_uint(v)));
}
template <int MASK>
__device__ __forceinline__ unsigned long long lane_xor(unsigned long long v) {
  return (unsigned long long)lane_xor<MASK>((uint64_t)v);
}
template <int MASK>
__device__ __forceinline__ double lane_xor(double v) {
  return __longlong_as_double((long long)lane_xor<MASK>((uint64_t)__double_as_longlong(v)));
}

// Reductions over groups of WIDTH lanes, the same result in every lane, taken in the same tree.  Once four
// lanes agree, mirroring eight of them is as good as exchanging the fours.
template <int WIDTH, typename W, typename Combine>
__device__ __forceinline__ W lanes_all(W v, Combine combine) {
  if constexpr (WIDTH >= 2) v = combine(v, lane_xor<1>(v));
  if constexpr (WIDTH >= 4) v = combine(v, lane_xor<2>(v));
  if constexpr (WIDTH >= 8) v = combine(v, lane_xor<7>(v));
  if constexpr (WIDTH >= 16) v = combine(v, lane_xor<15>(v));
  if constexpr (WIDTH >= 32) v = combine(v, lane_xor<16>(v));
  if constexpr (WIDTH >= 64) v = combine(v, lane_xor<32>(v));
  return v;
}
template <int WIDTH, typename W>
__device__ __forceinline__ W lanes_max(W v) {
  return lanes_all<WIDTH>(v, [](W p, W q) { return fmax(p, q); });
}
template <int WIDTH, typename W>
__device__ __forceinline__ W lanes_sum(W v) {
  return lanes_all<WIDTH>(v, [](W p, W q) { return p + q; });
}

// Inclusive prefix sums over groups of WIDTH lanes: within rows of 16 lanes by shifts, then each row's last
// lane to the rows behind it.
template <int CONTROL, int ROWS>
__device__ __forceinline__ uint32_t lanes_shifted(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0u, v, CONTROL, ROWS, 0xF, false);  // 0 where no lane is shifted in
}
template <int CONTROL, int ROWS>
__device__ __forceinline__ int lanes_shifted(int v) {
  return (int)lanes_shifted<CONTROL, ROWS>((uint32_t)v);
}
template <int CONTROL, int ROWS>
__device__ __forceinline__ unsigned long long lanes_shifted(unsigned long long v) {
  return ((unsigned long long)lanes_shifted<CONTROL, ROWS>((uint32_t)(v >> 32)) << 32) |
         lanes_shifted<CONTROL, ROWS>((uint32_t)v);
}
template <int CONTROL, int ROWS>
__device__ __forceinline__ double lanes_shifted(double v) {
  return __longlong_as_double((long long)lanes_shifted<CONTROL, ROWS>((unsigned long long)__double_as_longlong(v)));
}
template <int WIDTH, typename U>
__device__ __forceinline__ U lanes_scan(U v) {
  const int lane = threadIdx.x % WIDTH;
  const auto add = [&](U left, int distance) {
    if (WIDTH >= 16 || lane >= distance) v += left;  // narrower groups do not end with their row
  };
  if constexpr (WIDTH >= 2) add(lanes_shifted<0x111, 0xF>(v), 1);
  if constexpr (WIDTH >= 4) add(lanes_shifted<0x112, 0xF>(v), 2);
  if constexpr (WIDTH >= 8) add(lanes_shifted<0x114, 0xF>(v), 4);
  if constexpr (WIDTH >= 16) add(lanes_shifted<0x118, 0xF>(v), 8);
  if constexpr (WIDTH >= 32) add(lanes_shifted<0x142, 0xA>(v), 16);
  if constexpr (WIDTH >= 64) add(lanes_shifted<0x143, 0xC>(v), 32);
  return v;
}
// The value of the lane before, 0 in a group's first.
template <int WIDTH, typename U>
__device__ __forceinline__ U lane_before(U v) {
  const U left = lanes_shifted<0x138, 0xF>(v);
  return threadIdx.x % WIDTH == 0 ? (U)0 : left;
}

}  // namespace bn_rows
