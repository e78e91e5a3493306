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

// Elements [c, c + N) of a row of d; those behind its end are 0.  The row's last vector, where it is cut, is read as the
// row's last N elements and moved down: two shifts in one lane instead of N - 1 loads by all.
template <typename T>
__device__ __forceinline__ Vec<T> load_row(const T* row, int64_t c, int64_t d) {
  constexpr int N = Vec<T>::N;
  Vec<T> v;
  if (c + N <= d) {
    v.raw = *reinterpret_cast<const u32x4_any*>(row + c);
  } else if (c >= d) {
    v.raw = u32x4{0, 0, 0, 0};
  } else if (d >= N) {
    v.raw = *reinterpret_cast<const u32x4_any*>(row + d - N);
    uint64_t lo = static_cast<uint64_t>(v.raw[1]) << 32 | v.raw[0], hi = static_cast<uint64_t>(v.raw[3]) << 32 | v.raw[2];
    const int bits = static_cast<int>(c + N - d) * 8 * static_cast<int>(sizeof(T));  // 16 to 112
    lo = bits >= 64 ? hi >> (bits - 64) : lo >> bits | hi << (64 - bits);
    hi = bits >= 64 ? 0 : hi >> bits;
    v.raw = u32x4{static_cast<uint32_t>(lo), static_cast<uint32_t>(lo >> 32), static_cast<uint32_t>(hi),
                  static_cast<uint32_t>(hi >> 32)};
  } else {
#pragma unroll
    for (int j = 0; j < N; ++j) v.e[j] = c + j < d ? row[c + j] : static_cast<T>(0.f);
  }
  return v;
}

// The other way: elements behind the row's end are left alone.
template <typename T>
__device__ __forceinline__ void store_row(T* row, int64_t c, int64_t d, Vec<T> v) {
  T* p = row + c;
  if (c + Vec<T>::N <= d) {
    *reinterpret_cast<u32x4_any*>(p) = v.raw;
  } else if (c < d) {
    const int count = static_cast<int>(d - c) * static_cast<int>(sizeof(T)) / 2;  // 2-byte units: 1 to 7
    typedef u32x2 u32x2_any __attribute__((aligned(2)));
    typedef uint32_t u32_any __attribute__((aligned(2)));
    char* at = reinterpret_cast<char*>(p);
    if ((count & 4) != 0) {
      *reinterpret_cast<u32x2_any*>(at) = u32x2{v.raw[0], v.raw[1]};
      v.raw[0] = v.raw[2];
      v.raw[1] = v.raw[3];
      at += 8;
    }
    if ((count & 2) != 0) {
      *reinterpret_cast<u32_any*>(at) = v.raw[0];
      v.raw[0] = v.raw[1];
      at += 4;
    }
    if (sizeof(T) == 2 && (count & 1) != 0) *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(v.raw[0]);
  }
}

template <int CTRL>
__device__ __forceinline__ float lane_row(float v) {
  return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), CTRL, 0xF, 0xF, false));
}

// op over the N lanes that share lane / N (N = 2 ... 64), the result in all of them: within a row of 16 by DPP (see
// sum16), then rows and halves against each other (v_permlane16_swap and v_permlane32_swap of a register with itself
// leave the even rows' values in one result and the odd rows' in the other) -- no trip through the LDS crossbar.
// Every level joins the same two parts as lane ^ 1, ^ 2, ^ 4, ... would.  All lanes have to be active.
template <int N, typename F>
__device__ __forceinline__ float lanes_all(float v, F&& op) {
  if constexpr (N >= 2) v = op(v, lane_row<0xB1>(v));
  if constexpr (N >= 4) v = op(v, lane_row<0x4E>(v));
  if constexpr (N >= 8) v = op(v, lane_row<0x141>(v));
  if constexpr (N >= 16) v = op(v, lane_row<0x140>(v));
  if constexpr (N >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if constexpr (N >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}
template <int N>
__device__ __forceinline__ float lanes_sum(float v) {
  return lanes_all<N>(v, [](float a, float b) { return a + b; });
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
