// Element types of the token operators (layernorm.hip, rotary.hip, mha.hip): fp32, or bf16 held as uint16_t.  Arithmetic is fp32
// throughout; a bf16 value is widened exactly when it is read and rounded once (nearest even) when it is stored.
#pragma once
#include "common.h"

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
