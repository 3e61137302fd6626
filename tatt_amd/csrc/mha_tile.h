// Tiles and matrix-core fragments of the attention kernels (mha.hip).
//
// Every product is an MFMA of 32x32 outputs whose B operand sits in registers and whose A operand is read from a row-major tile in LDS:
//   rows(tile) x contraction over the head's dimensions   (scores, dP)          A = 32 tile rows, read as 16-byte chunks
//   dimensions x contraction over the tile's rows         (O, dQ, dK, dV)       A = the tile transposed
// The accumulator of the first kind (lane = column, registers = tile rows 8 (i / 4) + 4 half + i % 4) is, register for register, a B operand of
// the second kind if the contraction visits the tile's rows in that order: no element changes its lane between the two products.
//   bf16: v_mfma_f32_32x32x16_bf16, a chunk pair (16 dimensions) a step; transposed reads are ds_read_b64_tr_b16 (4 rows x 16 dimensions to 16 lanes)
//   fp32: v_mfma_f32_32x32x2_f32, four a step (8 dimensions); transposed reads are 4-byte reads along a row
#pragma once
#include "token_types.h"

__device__ __forceinline__ f32x16 mma(bf16x8 a, bf16x8 b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
__device__ __forceinline__ f32x16 mma(f32x4 a, f32x4 b, f32x16 c) {
#pragma unroll
  for (int t = 0; t < 4; ++t) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[t], b[t], c, 0, 0, 0);
  return c;
}

// accumulator registers [step * n, step * n + n) as the B operand of the transposed product's step (n = 8 bf16, 4 fp32); bf16: rounded to nearest even
template <typename T>
__device__ __forceinline__ typename Elem<T>::Frag pack_step(const f32x16& c, int step);
template <>
__device__ __forceinline__ f32x4 pack_step<float>(const f32x16& c, int step) {
  f32x4 r;
#pragma unroll
  for (int j = 0; j < 4; ++j) r[j] = c[step * 4 + j];
  return r;
}
template <>
__device__ __forceinline__ bf16x8 pack_step<bf16_t>(const f32x16& c, int step) {
  bf16x8 r;
#pragma unroll
  for (int j = 0; j < 8; ++j) r[j] = (__bf16)c[step * 8 + j];
  return r;
}

// A row-major LDS tile of W elements a row (a power of two, 32 to 128).  The 16-byte chunks of row r are stored at chunk ^ swizzle(r): the 16
// rows of a chunk column fall into 16 different 16-byte slots of the 256 bytes that LDS serves at once, and so do the chunks that four
// neighbouring rows of a transposed read take.
template <typename T, int W>
struct Tile {
  static constexpr int NC = W * (int)sizeof(T) / 16;  // chunks of a row: 4, 8, 16 or 32
  static constexpr int ROW = NC * 16;                 // bytes of a row
  __device__ __forceinline__ static int swizzle(int r) {
    if (NC >= 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    if (NC == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return (r >> 2) & 3;
  }
  __device__ __forceinline__ static int offset(int r, int chunk) { return r * ROW + ((chunk ^ swizzle(r)) << 4); }
  __device__ __forceinline__ static void put(char* tile, int r, int chunk, uint4 v) { *reinterpret_cast<uint4*>(tile + offset(r, chunk)) = v; }

  // A operand of a row product: lane (row = lane % 32, half) holds chunk 2 step + half of its row
  __device__ __forceinline__ static typename Elem<T>::Frag rows(const char* tile, int row0, int step, int lane) {
    const int r = row0 + (lane & 31);
    return *reinterpret_cast<const typename Elem<T>::Frag*>(tile + offset(r, 2 * step + (lane >> 5)));
  }

  // A operand of a transposed product: lane (dimension d0 + lane % 32, half) holds the tile rows that accumulator registers of `step` stand for:
  // fp32: row0 + 8 step + 4 half + j;  bf16: row0 + 16 step + 4 half + {0..3, 8..11}.  d0 a multiple of 32, row0 of 32.
  __device__ __forceinline__ static typename Elem<T>::Frag transposed(const char* tile, int row0, int step, int d0, int lane);
};

template <typename T, int W>
__device__ __forceinline__ typename Elem<T>::Frag Tile<T, W>::transposed(const char* tile, int row0, int step, int d0, int lane) {
  const int half = lane >> 5;
  if constexpr (sizeof(T) == 4) {
    const int d = d0 + (lane & 31);
    f32x4 r;
#pragma unroll
    for (int j = 0; j < 4; ++j) r[j] = *reinterpret_cast<const float*>(tile + offset(row0 + 8 * step + 4 * half + j, d >> 2) + 4 * (d & 3));
    return r;
  } else {
    // 16 lanes read four rows x 32 bytes (lane i: row i / 4, 8-byte piece i % 4) and receive column lane % 16 of those four rows
    const int i = lane & 15, piece = i & 3, chunk = (d0 >> 3) + 2 * ((lane >> 4) & 1) + (piece >> 1);
    union {
      s16x4 q[2];
      bf16x8 f;
    } u;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      const char* p = tile + offset(row0 + 16 * step + 4 * half + 8 * s + (i >> 2), chunk) + 8 * (piece & 1);
      u.q[s] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
    }
    return u.f;
  }
}
