// What the attention kernels (mha_fwd.hip, mha_bwd.hip) share: tiles and matrix-core fragments, the way of a tensor's rows into LDS, the
// arguments, their checks and the launch plans.
//
//   S = log2(e) scale q k^T;  lse_i = log2 sum_j 2^S_ij;  P = 2^(S - lse);  O = P V
//   delta_i = dO_i . O_i;  dV = P^T dO;  dS = P (dO V^T - delta);  dQ = scale dS K;  dK = scale dS^T Q
// bf16: delta is formed from O as two bf16 numbers, what is stored and what rounding took from it; without the second that rounding is most of the
// gradients' error where a row sees few keys.
// lse stays in base 2 between the passes: a change of base would round it twice more, and P is off by lse times those roundings.
// H = G * Hkv query heads: head h reads key head h / G.  The G heads of a key head are rows of the same problem (row = query * G + head), so a
// single query of G heads fills G rows of a tile, and a key's gradient sums over its heads as it sums over queries.
// Hidden places: keys whose mask byte is not 0, and, where causal, j > i + Lk - Lq.  A row that sees nothing gives zeros (lse = +inf) and
// takes no part in any gradient; a masked key's K and V are replaced by zeros on their way into LDS, whatever they hold.
//
// Every product is an MFMA of 32x32 outputs whose B operand sits in registers and whose A operand is read from a row-major tile in LDS:
//   rows(tile) x contraction over the head's dimensions   (scores, dP)          A = 32 tile rows, read as 16-byte chunks
//   dimensions x contraction over the tile's rows         (O, dQ, dK, dV)       A = the tile transposed
// The accumulator of the first kind (lane = column, registers = tile rows 8 (i / 4) + 4 half + i % 4) is, register for register, a B operand of
// the second kind if the contraction visits the tile's rows in that order: no element changes its lane between the two products.
// The MFMA is v_mfma_f32_32x32x16_bf16; transposed reads are ds_read_b64_tr_b16 (4 rows x 16 dimensions to 16 lanes).  fp32 tensors go through the
// same products as three bf16 pieces of every operand (fp32 accuracy; 6 bf16 MFMAs of 8 passes against 8 fp32 ones of 16).
// Operands that are computed, P and dS, enter their second product beside bf16 tensors as two bf16 pieces (16 significant bits: 2^-16 of a term, where
// one piece is off by up to 2^-8 of it, as much as the rounding of the stored result); accumulation is fp32.
#pragma once
#include "token_types.h"

namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

// A lane's 8 contraction places of a step, as the matrix core takes them.  bf16 tensors: the values.  fp32 tensors: three bf16 pieces of each value,
// x = x0 + x1 + x2 exactly (3 x 8 significant bits); a product is the six terms a0 b0 + (a0 b1 + a1 b0) + (a0 b2 + a1 b1 + a2 b0), added in fp32,
// smallest first, and what is left out is below the rounding of one fp32 product.  What is computed beside bf16 tensors: two pieces, two products with
// one reading of the other operand.
template <typename T, int N = (sizeof(T) == 2 ? 1 : 3)>
struct Frag {
  static constexpr int PIECES = N;
  bf16x8 p[PIECES];
};
template <typename T>
constexpr int COMPUTED = sizeof(T) == 2 ? 2 : 3;  // pieces of P and dS

template <typename T, int N>
__device__ __forceinline__ f32x16 mma(const Frag<T>& a, const Frag<T, N>& b, f32x16 c) {
  if constexpr (N == 2) c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
  if constexpr (N == 3) {
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[2], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[2], b.p[0], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[1], c, 0, 0, 0);
    c = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[1], b.p[0], c, 0, 0, 0);
  }
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a.p[0], b.p[0], c, 0, 0, 0);
}

// two values as bf16 (nearest even), low half first; and the values that it stands for
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  typedef float f2 __attribute__((ext_vector_type(2)));
  const b2 v = __builtin_convertvector((f2{a, b}), b2);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float low2(uint32_t u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float high2(uint32_t u) { return __uint_as_float(u & 0xFFFF0000u); }

// two fp32 values as three pieces each (of an infinity the remainder is no number: what it reaches is NaN)
__device__ __forceinline__ void split2(float a, float b, uint32_t (&u)[3]) {
  u[0] = pack2(a, b);
  const float ra = a - low2(u[0]), rb = b - high2(u[0]);
  u[1] = pack2(ra, rb);
  u[2] = pack2(ra - low2(u[1]), rb - high2(u[1]));
}

// 8 values, v(0) .. v(7), as a fragment of N pieces
template <typename T, int N, typename V>
__device__ __forceinline__ Frag<T, N> fragment(V v) {
  uint32_t u[N][4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float a = v(2 * j), b = v(2 * j + 1);
    if constexpr (N == 3) {
      uint32_t w[3];
      split2(a, b, w);
#pragma unroll
      for (int x = 0; x < 3; ++x) u[x][j] = w[x];
    } else {
      u[0][j] = pack2(a, b);
      if constexpr (N == 2) u[1][j] = pack2(a - low2(u[0][j]), b - high2(u[0][j]));
    }
  }
  Frag<T, N> f;
  memcpy(&f, u, sizeof(f));
  return f;
}

constexpr int STEP = 16;  // contraction places of an MFMA step (both lane halves)

// accumulator registers 8 step .. 8 step + 7 as the B operand of the transposed product's step
template <typename T>
__device__ __forceinline__ Frag<T, COMPUTED<T>> pack_step(const f32x16& c, int step) {
  return fragment<T, COMPUTED<T>>([&](int j) { return c[8 * step + j]; });
}

// waves a SIMD that the registers are shared out for.  Two (256 registers each) unless what a wave has to hold -- the fragments of its rows, the
// sums, a tile on its way -- would spill: then one (dK and dV of 2 x 2777 tokens, 16 / 4 heads of 128, in bf16: 1129 us with two and 318 spilled registers,
// 408 with one and none).  With one, fp32 dK and dV still spill: heads of 128 and few keys of 64 101 registers, of 96 53, into the accumulators' half of the
// register file but for 58 of the 128's, which go to memory.
template <typename T>
constexpr int fwd_waves(int DK) { return sizeof(T) == 4 && DK > 64 ? 1 : 2; }
template <typename T>
constexpr int dq_waves(int DK) { return sizeof(T) == 4 && DK >= 64 ? 1 : 2; }
template <typename T>
constexpr int dkv_waves(int DK) { return DK > 64 || (sizeof(T) == 4 && DK == 64) ? 1 : 2; }

// head widths the kernels are built for, and the LDS row that holds one
constexpr int row_width(int DK) { return DK <= 32 ? 32 : DK <= 64 ? 64 : 128; }

// A row-major LDS tile of ROWS rows of W bf16 elements (W a power of two, 32 to 128), or three such planes, one for each piece.  The 16-byte chunks
// of row r are stored at chunk ^ swizzle(r): the 16 rows of a chunk column fall into 16 different 16-byte slots of the 256 bytes that LDS serves at
// once, and so do the chunks that four neighbouring rows of a transposed read take (no bank conflict is counted).
template <typename T, int W, int ROWS>
struct Tile {
  static constexpr int NC = W / 8;    // chunks of a row: 4, 8 or 16
  static constexpr int ROW = W * 2;   // bytes of a row
  static constexpr int PLANE = ROWS * ROW, BYTES = PLANE * Frag<T>::PIECES;
  __device__ __forceinline__ static int swizzle(int r) {
    if (NC == 16) return ((r & 3) << 2) | ((r >> 2) & 3);
    if (NC == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return (r >> 2) & 3;
  }
  __device__ __forceinline__ static int offset(int r, int chunk) { return r * ROW + ((chunk ^ swizzle(r)) << 4); }

  // 16 bytes of a row of the tensor, its chunk c (8 bf16 or 4 fp32 elements), into the tile
  __device__ __forceinline__ static void put(char* tile, int r, int c, uint4 v) {
    if constexpr (sizeof(T) == 2) {
      *reinterpret_cast<uint4*>(tile + offset(r, c)) = v;
    } else {
      uint32_t a[3], b[3];
      split2(__uint_as_float(v.x), __uint_as_float(v.y), a);
      split2(__uint_as_float(v.z), __uint_as_float(v.w), b);
#pragma unroll
      for (int x = 0; x < 3; ++x) *reinterpret_cast<uint2*>(tile + x * PLANE + offset(r, c >> 1) + 8 * (c & 1)) = make_uint2(a[x], b[x]);
    }
  }

  // Where a lane reads: (its base ^ a constant) + a constant, so one register serves every fragment of a kind.
  struct Lane {
    int row, col;
    __device__ __forceinline__ explicit Lane(int lane) {
      const int half = lane >> 5, i = lane & 15, piece = i & 3;
      row = offset(lane & 31, half);
      // 16 lanes read four rows x 32 bytes (lane i: row i / 4, 8-byte piece i % 4) and receive column lane % 16 of those four rows
      col = offset(4 * half + (i >> 2), 2 * ((lane >> 4) & 1) + (piece >> 1)) + 8 * (piece & 1);
    }
    // keeps the compiler from holding each base ^ constant in a register of its own across the loop (and spilling them)
    __device__ __forceinline__ void afresh() { asm volatile("" : "+v"(row), "+v"(col)); }
  };

  // A operand of a row product: lane (row = lane % 32, half) holds chunk 2 step + half of its row.  row0 a multiple of 32.
  __device__ __forceinline__ static Frag<T> rows(const char* tile, int row0, int step, const Lane& at) {
    Frag<T> f;
#pragma unroll
    for (int x = 0; x < Frag<T>::PIECES; ++x) f.p[x] = *reinterpret_cast<const bf16x8*>(tile + x * PLANE + row0 * ROW + (at.row ^ (step << 5)));
    return f;
  }

  // A operand of a transposed product: lane (dimension d0 + lane % 32, half) holds the tile rows that accumulator registers of `step` stand for:
  // row0 + 16 step + 4 half + {0..3, 8..11}.  d0 and row0 multiples of 32.
  __device__ __forceinline__ static Frag<T> transposed(const char* tile, int row0, int step, int d0, const Lane& at) {
    union {
      s16x4 q[Frag<T>::PIECES][2];
      Frag<T> f;
    } u;
#pragma unroll
    for (int x = 0; x < Frag<T>::PIECES; ++x)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        const char* p = tile + x * PLANE + (row0 + 16 * step + 8 * s) * ROW + (at.col ^ (((d0 >> 3) ^ (2 * s)) << 4));
        u.q[x][s] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
      }
    return u.f;
  }
};

struct MhaArgs {
  const void *q, *k, *v, *out, *dout;
  const void* out_low;  // bf16: what rounding took from out (contiguous), for delta
  long qs[3], ks[3], vs[3], os[3], dos[3];  // element strides: batch, token, head
  const unsigned char* mask;
  long mask_sb, mask_sl;
  const float* lse;
  float* delta;
  int B, Lq, Lk, H, Hkv, G, D, causal;
  int rows;         // Lq * G
  float scale, c;   // c = |scale| * log2(e), never 0 (a scale of 0: 1e-30)
  int nblk, nsplit, per_split;  // blocks of rows (keys) per key head, splits of the other axis and its length of one split
};

struct Where {
  int blk, split, hk;
  long b;
};
// Workgroups go round the 8 XCDs in turn, and to the CUs in order.
// Causal: blocks differ in length, so the long ones of every problem go first (blocks: the slowest index, w.blk = 0 the longest), and the short ones
// fill up what they leave (4 x 4096, 8 heads of 64, bf16: kernels of a training pass 683 -> 553 us).  With a mask the problems differ too and are turned against the
// XCDs, lest a short sequence leave an XCD idle (two clips, one of them empty: dQ 146 -> 132 us).
// Else each XCD gets a contiguous range of the work, so that the blocks that read one key head share an L2 (fp32, 16 x 4 heads of 1024: 2-6 %
// faster) -- but not where the work of a range may differ, with a mask, or with splits, which share nothing.
__device__ __forceinline__ Where where(const MhaArgs& a) {
  const unsigned problems = (unsigned)a.B * a.Hkv * a.nsplit;
  unsigned id = blockIdx.x;
  Where w;
  if (a.causal) {
    w.blk = id / problems;
    id -= w.blk * problems;
    if (a.mask) id = (id + w.blk) % problems;
  } else {
    if (!a.mask && a.nsplit == 1) {
      const unsigned n = gridDim.x, per = n / 8, rest = n % 8, x = id % 8;
      id = x * per + min(x, rest) + id / 8;
    }
    w.blk = id % a.nblk;
    id /= a.nblk;
  }
  w.split = id % a.nsplit;
  id /= a.nsplit;
  w.hk = id % a.Hkv;
  w.b = id / a.Hkv;
  return w;
}

// One split of the summed axis' places [lo, hi): the split's length, or, where causality has cut that axis differently for every block, an equal share of
// what is left of it in whole tiles (dK and dV of 2 x 2777, 16 / 4 heads of 128: 308 -> 214 us).
__device__ __forceinline__ void take_split(const MhaArgs& a, int split, int tile, int& lo, int& hi) {
  if (a.nsplit == 1) return;
  const int all = max(0, hi - lo), per = a.causal ? ((all + a.nsplit - 1) / a.nsplit + tile - 1) / tile * tile : a.per_split;
  lo += min(all, split * per);
  hi = min(hi, lo + per);
}

// element offset of row r (= query * G + head of the group) of a tensor with these token / head strides
__device__ __forceinline__ long row_offset(int r, int G, long sl, long sh) {
  if (G == 1) return r * sl;
  const int i = (unsigned)r / (unsigned)G;
  return i * sl + (r - i * G) * sh;
}

// B operand of a row product: this lane's row, all steps of the contraction
template <typename T, int DK>
struct RowFrags {
  Frag<T> f[DK / STEP];
  __device__ __forceinline__ void load(const T* row, bool on, int D, int lane) {
#pragma unroll
    for (int s = 0; s < DK / STEP; ++s) {
      T t[8];
      chunk8(row, on, s, D, lane, t);
      if constexpr (sizeof(T) == 2)
        memcpy(&f[s], t, 16);
      else
        f[s] = fragment<T, Frag<T>::PIECES>([&](int j) { return t[j]; });
    }
  }
  // the product with another row
  __device__ __forceinline__ float dot(const T* row, bool on, int D, int lane) const {
    float d = 0.f;
#pragma unroll
    for (int s = 0; s < DK / STEP; ++s) {
      T t[8];
      chunk8(row, on, s, D, lane, t);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        float v = 0.f;
#pragma unroll
        for (int x = Frag<T>::PIECES - 1; x >= 0; --x) v += (float)f[s].p[x][j];
        d += to_f32(t[j]) * v;
      }
    }
    return d;
  }
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int s = 0; s < DK / STEP; ++s)
#pragma unroll
      for (int x = 0; x < Frag<T>::PIECES; ++x) f[s].p[x] = -f[s].p[x];
  }
  // elements 16 s + 8 half .. + 7 of a row
  __device__ __forceinline__ static void chunk8(const T* row, bool on, int s, int D, int lane, T (&t)[8]) {
    constexpr int N = 8 / per_chunk<T>();
    uint4 u[N];
#pragma unroll
    for (int n = 0; n < N; ++n) u[n] = on ? load_chunk<T>(row, (2 * s + (lane >> 5)) * N + n, D, 1) : make_uint4(0, 0, 0, 0);
    memcpy(t, u, 8 * sizeof(T));
  }
};

// ROWS consecutive rows of a tensor on their way into an LDS tile, held in registers by NT threads.  Buffer loads: the tile's first row is a
// scalar base, a thread's places in a tile are offsets that do not change, and a place that does not exist is an offset out of range,
// for which the load returns zeros.  LINEAR: rows are one stride apart (keys), else at places(r) (queries of several heads).
template <typename T, int W, int ROWS, int NT, bool LINEAR>
struct Stage {
  static constexpr int NC = W / per_chunk<T>(), N = (ROWS * NC + NT - 1) / NT, HOP = NT / NC;
  static_assert(NT % NC == 0 && (N == 1 || ROWS * NC % NT == 0), "every thread holds the same chunk of N rows");
  static constexpr int NOWHERE = 0x7FFFFFF0;
  typedef int i32x4 __attribute__((ext_vector_type(4)));
  i32x4 r[N];
  int off[LINEAR ? 1 : N];  // byte offsets from the tile's first row
  int hop;                  // LINEAR: bytes between a thread's rows

  __device__ __forceinline__ static int row(int n) { return n * HOP + (int)threadIdx.x / NC; }
  __device__ __forceinline__ static int chunk() { return (int)threadIdx.x % NC; }

  __device__ __forceinline__ void linear(long stride, int D) {
    static_assert(LINEAR, "");
    off[0] = chunk() * per_chunk<T>() < D && row(0) < ROWS ? (int)(row(0) * stride * (long)sizeof(T)) + chunk() * 16 : NOWHERE;
    hop = (int)(HOP * stride * (long)sizeof(T));
  }
  template <typename Offset>
  __device__ __forceinline__ void places(Offset offset, int D) {
    static_assert(!LINEAR, "");
    const bool on = chunk() * per_chunk<T>() < D && row(0) < ROWS;
#pragma unroll
    for (int n = 0; n < N; ++n) off[n] = on ? (int)(offset(row(n)) * (long)sizeof(T)) + chunk() * 16 : NOWHERE;
  }
  // rows [from, to) of the tile exist
  __device__ __forceinline__ void load(const T* first, int from, int to) {
    const __amdgpu_buffer_rsrc_t rs = __builtin_amdgcn_make_buffer_rsrc((void*)first, 0, NOWHERE, 0x00020000);
    if (from <= 0 && to >= ROWS) {
#pragma unroll
      for (int n = 0; n < N; ++n) r[n] = __builtin_amdgcn_raw_buffer_load_b128(rs, off[LINEAR ? 0 : n], LINEAR ? n * hop : 0, 0);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n)
        r[n] = __builtin_amdgcn_raw_buffer_load_b128(rs, row(n) >= from && row(n) < to ? off[LINEAR ? 0 : n] : NOWHERE, LINEAR ? n * hop : 0, 0);
    }
  }
  __device__ __forceinline__ void put(char* tile) const {
    if (row(0) >= ROWS) return;
#pragma unroll
    for (int n = 0; n < N; ++n) Tile<T, W, ROWS>::put(tile, row(n), chunk(), make_uint4(r[n][0], r[n][1], r[n][2], r[n][3]));
  }
  // zeros in the rows whose bit is not set
  template <int NW>
  __device__ __forceinline__ void hide(const unsigned long (&word)[NW]) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = row(n);
      unsigned long w = word[0];
#pragma unroll
      for (int x = 1; x < NW; ++x) w = i >= 64 * x ? word[x] : w;
      if (!(w >> (i & 63) & 1)) r[n] = i32x4{0, 0, 0, 0};
    }
  }
};

// KT keys from k0 on: bit j of word[j / 64] = key k0 + j is below `kend` and not masked.  The mask's bytes are asked for a tile ahead.
template <int KT>
struct KeyBits {
  static constexpr int NW = (KT + 63) / 64;
  int hidden[NW];
  unsigned long word[NW];
  __device__ __forceinline__ void load(const unsigned char* mask, long stride, int k0, int kend, int lane) {
    if (!mask) return;
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const int j = k0 + 64 * x + lane;
      hidden[x] = j >= kend || mask[j * stride];
    }
  }
  __device__ __forceinline__ void settle(const unsigned char* mask, int k0, int kend) {
#pragma unroll
    for (int x = 0; x < NW; ++x) {
      const int n = min(kend - k0, KT) - 64 * x;
      word[x] = mask ? __ballot(!hidden[x]) : n <= 0 ? 0ul : n >= 64 ? ~0ul : (1ul << n) - 1;
    }
    if (mask && KT < 64) word[0] &= (1ul << (KT & 63)) - 1;
  }
  __device__ __forceinline__ bool full() const {
    bool f = true;
#pragma unroll
    for (int x = 0; x < NW; ++x) f = f && word[x] == (KT % 64 && x == NW - 1 ? (1ul << KT % 64) - 1 : ~0ul);
    return f;
  }
  __device__ __forceinline__ unsigned of(int at) const { return (unsigned)(word[at / 64] >> (at & 63)); }  // 32 keys from `at` on
};

// [lo, hi) shrunk to its first and last key that is not masked (padding at a sequence's end is not even read); `red` = 8 bytes of LDS a wave
template <int NT>
__device__ __forceinline__ void trim_keys(const unsigned char* mask, long stride, int& lo, int& hi, int* red) {
  int first = hi, last = lo - 1;
#pragma unroll 4
  for (int j = lo + (int)threadIdx.x; j < hi; j += NT)
    if (!mask[j * stride]) {
      first = min(first, j);
      last = max(last, j);
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    first = min(first, __shfl_xor(first, o, 64));
    last = max(last, __shfl_xor(last, o, 64));
  }
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = first, red[NT / 64 + (threadIdx.x >> 6)] = last;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < NT / 64; ++x) {
    first = min(first, red[x]);
    last = max(last, red[NT / 64 + x]);
  }
  __syncthreads();
  lo = __builtin_amdgcn_readfirstlane(first);
  hi = __builtin_amdgcn_readfirstlane(last + 1);
}

// the first key below `hi` that is not masked (`hi`: none); `red` = 4 bytes of LDS a wave
template <int NT>
__device__ __forceinline__ int first_key(const unsigned char* mask, long stride, int hi, int* red) {
  int first = hi;
  for (int j = threadIdx.x; j < hi; j += NT)
    if (!mask[j * stride]) {
      first = j;
      break;
    }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
  if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = first;
  __syncthreads();
#pragma unroll
  for (int x = 0; x < NT / 64; ++x) first = min(first, red[x]);
  __syncthreads();
  return __builtin_amdgcn_readfirstlane(first);
}

// the D elements of one row held as accumulators of a transposed product (lane = row, registers = dimensions), times f, to dst
template <typename T, int ND>
__device__ __forceinline__ void store_row(T* dst, const f32x16 (&o)[ND], float f, int D, int lane) {
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * dt + 8 * q + 4 * (lane >> 5);
      if (d >= D) continue;
      if constexpr (sizeof(T) == 2)
        *reinterpret_cast<uint2*>(dst + d) = tatt_pack_bf16x4(o[dt][4 * q] * f, o[dt][4 * q + 1] * f, o[dt][4 * q + 2] * f, o[dt][4 * q + 3] * f);
      else
        *reinterpret_cast<float4*>(dst + d) = make_float4(o[dt][4 * q] * f, o[dt][4 * q + 1] * f, o[dt][4 * q + 2] * f, o[dt][4 * q + 3] * f);
    }
}

// what rounding to bf16 took from that row
template <int ND>
__device__ __forceinline__ void store_low(bf16_t* dst, const f32x16 (&o)[ND], float f, int D, int lane) {
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * dt + 8 * q + 4 * (lane >> 5);
      if (d >= D) continue;
      uint32_t u[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float a = o[dt][4 * q + 2 * e] * f, b = o[dt][4 * q + 2 * e + 1] * f;
        const uint32_t h = pack2(a, b);
        u[e] = pack2(a - low2(h), b - high2(h));
      }
      *reinterpret_cast<uint2*>(dst + d) = make_uint2(u[0], u[1]);
    }
}

// over a lane and the one 32 further: v_permlane32_swap_b32, a register exchange (a shuffle through LDS waits some hundred cycles)
__device__ __forceinline__ float half_max(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}
__device__ __forceinline__ float half_sum(float x) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(p[0]) + __uint_as_float(p[1]);
}
// tile row that accumulator register i of a lane half stands for (+ 4 half)
__device__ __forceinline__ constexpr int acc_row(int i) { return 8 * (i / 4) + i % 4; }

__device__ __forceinline__ void clear(f32x16& o) {
#pragma unroll
  for (int i = 0; i < 16; ++i) o[i] = 0.f;
}
template <int N>
__device__ __forceinline__ void clear(f32x16 (&o)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n) clear(o[n]);
}

// Waits for every load issued so far.  Once before a loop: the fragments loaded for it are then known to be there, and their first use inside the
// loop does not wait for the tile that is on its way (which exposed the whole latency of global memory every iteration).
__device__ __forceinline__ void wait_loads() { __builtin_amdgcn_s_waitcnt(0x0F70); }  // vmcnt(0)

// bits 0 .. n (n < 0: none, n >= 31: all)
__device__ __forceinline__ unsigned bits_to(int n) { return n < 0 ? 0u : n >= 31 ? ~0u : (2u << n) - 1u; }

// ---- launch plans ---------------------------------------------------------------------------------------------------------------------
constexpr float LOG2E = 1.4426950408889634f;

struct Plan {
  int wide, nblk, nsplit, per_split;  // wide: waves side by side along the output axis; else along the summed one
};
// Blocks of 128 along the output axis, 32 if it has no more than 32, and the summed axis in splits of no less than `finest`.
// One tile of rows: where blocks do not fill the chip, as many splits as fill it twice (sequences differ in length), and none where they do: 63 sequences of
// up to 20000 keys, 8 key heads of 128, bf16, take 623 + 5 us in three splits, 64 of them 773 in one.  `whole`, workgroups that work on 128: as few as make the pass
// shortest, with `slots` workgroups at a time, in units of a whole block: the workgroups that a CU gets one after another (of two at a time, the last alone
// takes 0.6), or, where causal, the longest of them and their even share; and the partial sums, written and read, `traffic` / inner of the products' time a
// split.  (bf16, heads of 128, dK and dV: 8 x 1024 x 4 in 58 us unsplit and 84 + 23 in four splits, 2 x 2777 x 16 / 4 in 498 unsplit, 408 + 21 in four and 460
// with the sum still to come in six.)
inline Plan plan(long problems, int outer, int inner, int finest, int causal, int slots, float traffic, bool whole) {
  Plan p;
  p.wide = outer > 32;
  p.nblk = cdiv(outer, p.wide ? 128 : 32);
  const long blocks = problems * p.nblk;
  long n = blocks >= slots ? 1 : (2 * slots + blocks - 1) / blocks, most = inner / finest < 1 ? 1 : inner / finest;
  if (whole) {
    const float load = (float)blocks / slots;
    float best = 0.f;
    long pick = 1;
    for (long i = 1; i <= most && (i <= n || i <= 8); ++i) {
      const float share = 0.55f * load, part = 1.f / i;
      const int each = cdiv(blocks * i, 256);
      const float alone = slots == 256 ? each : each == 1 ? 0.6f : 0.5f * each;
      const float t = (causal ? (part > share ? part : share) : alone * part) + (i > 1 ? i * traffic / inner * load : 0.f);
      if (i == 1 || t < best) best = t, pick = i;
    }
    n = pick;
  }
  if (n > most) n = most;
  p.per_split = cdiv(cdiv(inner, n), 128) * 128;
  p.nsplit = cdiv(inner, p.per_split);
  return p;
}

// workgroups of four waves that the chip holds at once, and plan()'s `traffic`: fp32 products take some four times as long (the measured shapes are split
// alike with 280 for bf16)
inline int slots_of(int waves) { return waves == 1 ? 256 : 512; }
inline float traffic_of(int dtype) { return dtype == TATT_T_BF16 ? 400.f : 80.f; }

// fewer than 2^30 rows of a tensor, factor by factor: three of 31 bits overflow 64
inline bool countable(int B, int H, int L) { return (long)B * H < 1L << 30 && (long)B * H * L < 1L << 30; }

// what the entry points take, and the workspace queries answer (the plans' own products stay within 31 bits)
inline bool sane(int B, int Lq, int Lk, int H, int Hkv, int D) {
  return B > 0 && Lq > 0 && Lk > 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && H / Hkv <= 1 << 16 && D > 0 && D <= 128 && countable(B, H, Lq) && countable(B, Hkv, Lk);
}

// 16-byte rows, and a tile of 128 of them (G heads of 128 / G tokens) within the 31-bit offsets of a buffer load
inline bool reachable(const void* p, const long* s, int size, int G) {
  for (int i = 0; i < 3; ++i)
    if (s[i] < 0 || s[i] >= 1L << 40 || s[i] * size % 16) return false;
  return ((uintptr_t)p & 15) == 0 && ((128 / G + 2) * s[1] + (G - 1) * s[2]) * size < (1L << 31) - 4096;
}

inline int fill(MhaArgs& a, const char* who, const void* q, const void* k, const void* v, const void* out, const void* dout, const long* strides,
                const unsigned char* mask, const long* mask_strides, int B, int Lq, int Lk, int H, int Hkv, int D, float scale, int causal, int dtype,
                const float* workspace) {
  TATT_CHECK_ARG(q && k && v && out && strides && B > 0 && Lq > 0 && Lk > 0 && H > 0 && Hkv > 0, "%s: bad arguments", who);
  TATT_CHECK_ARG(!mask || mask_strides, "%s: a key mask needs its strides", who);
  TATT_CHECK_ARG(H % Hkv == 0, "%s: %d query heads are no multiple of %d key heads", who, H, Hkv);
  TATT_CHECK_ARG(H / Hkv <= 1 << 16, "%s: %d query heads to %d key heads, more than 65536 to one", who, H, Hkv);
  TATT_CHECK_ARG(D > 0 && D <= 128, "%s: built for heads of 1 to 128, got %d", who, D);
  TATT_CHECK_ARG(dtype == TATT_T_F32 || dtype == TATT_T_BF16, "%s: unknown element type %d", who, dtype);
  TATT_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "%s: the workspace is not 16-byte aligned", who);
  TATT_CHECK_ARG(countable(B, H, Lq) && countable(B, Hkv, Lk), "%s: 2^30 rows or more", who);
  a.q = q, a.k = k, a.v = v, a.out = out, a.dout = dout, a.mask = mask;
  a.mask_sb = mask ? mask_strides[0] : 0, a.mask_sl = mask ? mask_strides[1] : 0;
  for (int i = 0; i < 3; ++i) a.qs[i] = strides[i], a.ks[i] = strides[3 + i], a.vs[i] = strides[6 + i];
  if (dout)
    for (int i = 0; i < 3; ++i) a.os[i] = strides[9 + i], a.dos[i] = strides[12 + i];
  const int size = dtype == TATT_T_BF16 ? 2 : 4;
  TATT_CHECK_ARG(D * size % 16 == 0 && reachable(q, a.qs, size, H / Hkv) && reachable(k, a.ks, size, 1) && reachable(v, a.vs, size, 1) &&
                     reachable(out, a.os, size, H / Hkv) && (!dout || reachable(dout, a.dos, size, H / Hkv)),
                 "%s: rows of whole 16 bytes at 16-byte aligned places expected, 128 of them within 2^31 bytes", who);
  a.B = B, a.Lq = Lq, a.Lk = Lk, a.H = H, a.Hkv = Hkv, a.G = H / Hkv, a.D = D, a.causal = causal;
  a.rows = Lq * a.G;
  a.scale = scale;
  a.c = scale == 0.f ? 1e-30f : fabsf(scale) * LOG2E;
  return TATT_OK;
}

// the grid of one workgroup of `threads` per block, key head and split; more LDS than 64 KB has to be asked for
template <typename K>
int prepare_launch(const MhaArgs& a, K kernel, int threads, size_t bytes) {
  TATT_CHECK_ARG((long)a.B * a.Hkv * a.nblk * a.nsplit * threads < (1L << 32), "tatt_mha: %d x %d x %d x %d workgroups exceed the grid", a.B, a.Hkv, a.nblk, a.nsplit);
  if (bytes > 64 * 1024 && hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, (int)bytes) != hipSuccess) {
    (void)hipGetLastError();
    tatt_set_error("tatt_mha: %zu bytes of LDS refused", bytes);
    return TATT_ERR_LAUNCH;
  }
  return TATT_OK;
}

// waves along the summed axis where the other axis has one tile: tiles of 32 of their rows, two buffers of them within 64 KB
template <typename T>
constexpr int narrow_waves(int DK) { return sizeof(T) == 2 ? (DK > 64 ? 2 : 4) : (DK > 64 ? 1 : DK > 32 ? 2 : 4); }

}  // namespace

// body with DK bound to the head width rounded up to what the kernels are built for
#define TATT_DISPATCH_WIDTH(D, ...)             \
  do {                                          \
    if ((D) <= 16) {                            \
      constexpr int DK = 16;                    \
      __VA_ARGS__                               \
    } else if ((D) <= 32) {                     \
      constexpr int DK = 32;                    \
      __VA_ARGS__                               \
    } else if ((D) <= 64) {                     \
      constexpr int DK = 64;                    \
      __VA_ARGS__                               \
    } else if ((D) <= 96) {                     \
      constexpr int DK = 96;                    \
      __VA_ARGS__                               \
    } else {                                    \
      constexpr int DK = 128;                   \
      __VA_ARGS__                               \
    }                                           \
  } while (0)
