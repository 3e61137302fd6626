// Element types of the token operators (layernorm.hip, rotary.hip, mha.hip): fp32, or bf16 held as uint16_t.  Arithmetic is fp32
// throughout; a bf16 value is widened exactly when it is read and rounded once (nearest even) when it is stored.
#pragma once
#include "common.h"
#include <type_traits>

#define TATT_T_F32 0
#define TATT_T_BF16 1

typedef uint16_t bf16_t;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16_t x) { return __uint_as_float((uint32_t)x << 16); }

template <typename T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16_t from_f32<bf16_t>(float x) {
  const __bf16 b = (__bf16)x;
  return *reinterpret_cast<const bf16_t*>(&b);
}

// elements of 16 bytes
template <typename T>
constexpr int per_chunk() { return 16 / (int)sizeof(T); }

// chunk `c` of a row of D elements, zeros behind its end
template <typename T>
__device__ __forceinline__ uint4 load_chunk(const T* row, int c, int D, int vec) {
  constexpr int E = per_chunk<T>();
  uint4 r = make_uint4(0, 0, 0, 0);
  if (vec) {
    if (c * E < D) r = *reinterpret_cast<const uint4*>(row + c * E);
  } else {
    T t[E];
#pragma unroll
    for (int e = 0; e < E; ++e) t[e] = c * E + e < D ? row[c * E + e] : from_f32<T>(0.f);
    memcpy(&r, t, 16);
  }
  return r;
}

// the same entry point for both types: body with `T` bound to the element type
#define TATT_DISPATCH_TYPE(dtype, ...)    \
  do {                                    \
    if ((dtype) == TATT_T_BF16) {         \
      using T = bf16_t;                   \
      __VA_ARGS__                         \
    } else {                              \
      using T = float;                    \
      __VA_ARGS__                         \
    }                                     \
  } while (0)
