// Element types of the operators that take float32, bfloat16 or float16 tensors (GUNET_DTYPE_*).
#pragma once

#include <initializer_list>

#include "common.h"

namespace gunet {

inline bool dtype_valid(int32_t dtype) { return dtype == GUNET_DTYPE_F32 || dtype == GUNET_DTYPE_BF16 || dtype == GUNET_DTYPE_F16; }
inline size_t dtype_size(int32_t dtype) { return dtype == GUNET_DTYPE_F32 ? 4 : 2; }

template <typename T, int VEC>
struct TypeTag {
  using type = T;
  static constexpr int vec = VEC;
};

// VEC elements moved by one load or store (16 bytes at most).
template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};

template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& v) {
  *reinterpret_cast<Pack<T, VEC>*>(p) = v;
}

// load_pack for what is read once: past the caches, which keep what is read again and written.
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack_once(const T* p) {
  using P = Pack<T, VEC>;
  if constexpr (sizeof(P) == 16)
    return __builtin_bit_cast(P, __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)));
  else
    return load_pack<T, VEC>(p);
}

template <typename T>
__device__ __forceinline__ float to_f32(T v) {
  return static_cast<float>(v);
}
// Rounds to nearest even, once.
template <typename T>
__device__ __forceinline__ T from_f32(float v) {
  return static_cast<T>(v);
}

}  // namespace gunet
