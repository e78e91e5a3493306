// Element types and row access of the dense-head kernels (layer_norm.hip, act8.hip, log_prob.hip): float, bf16 and
// fp16 rows with any leading dimension and any alignment of their elements.
#pragma once

#include "common.hpp"

namespace kgat {

// 16 bytes that lie at any multiple of the element size: gfx950 loads and stores them whole (global_load_dwordx4
// has no alignment of its own under the unaligned access mode that HSA sets), so odd widths and views need no
// scalar path.
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));

template <typename T>
struct Vec {
  static constexpr int N = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte vector
  union {
    u32x4 raw;
    T e[N];
  };
};

// The first `count` elements of a vector at p (count >= N: all of them); the others are `fill`.
template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p, int64_t count, float fill = 0.f) {
  Vec<T> v;
  if (count >= Vec<T>::N) {
    v.raw = *reinterpret_cast<const u32x4_any*>(p);
  } else {
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j) v.e[j] = j < count ? p[j] : static_cast<T>(fill);
  }
  return v;
}

template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& v, int64_t count) {
  if (count >= Vec<T>::N) {
    *reinterpret_cast<u32x4_any*>(p) = v.raw;
  } else {
#pragma unroll
    for (int j = 0; j < Vec<T>::N; ++j)
      if (j < count) p[j] = v.e[j];
  }
}

// Host: calls f(T{}) with the element type of a KGAT_F32 / BF16 / F16 code; an unknown code is KGAT_ERR_INVALID.
template <typename F>
inline int with_dtype(int32_t dtype, F&& f) {
  switch (dtype) {
    case KGAT_F32: return f(float{});
    case KGAT_BF16: return f(__bf16{});
    case KGAT_F16: return f(_Float16{});
    default: return KGAT_ERR_INVALID;
  }
}

inline int dtype_bytes(int32_t dtype) { return dtype == KGAT_F32 ? 4 : 2; }

}  // namespace kgat
