// Attention of any lengths, head counts and head widths up to 128, forward and backward (attn.hip is the 26-key, 4 x 16 form).
//   S = log2(e) scale q k^T;  lse_i = log2 sum_j 2^S_ij;  P = 2^(S - lse);  O = P V
//   delta_i = dO_i . O_i;  dV = P^T dO;  dS = P (dO V^T - delta);  dQ = scale dS K;  dK = scale dS^T Q
// lse stays in base 2 between the passes: a change of base would round it twice more, and P is off by lse times those roundings.
// H = G * Hkv query heads: head h reads key head h / G.  The G heads of a key head are rows of the same problem (row = query * G + head), so a
// single query of G heads fills G rows of a tile, and a key's gradient sums over its heads as it sums over queries.
// Hidden places: keys whose mask byte is not 0, and, where causal, j > i + Lk - Lq.  A row that sees nothing gives zeros (lse = +inf) and
// takes no part in any gradient; a masked key's K and V are replaced by zeros on their way into LDS, whatever they hold.
// One pass over the keys with a running maximum and sum (forward), or over keys / rows with P recomputed from lse (backward): no score ever
// leaves the registers.  mha_tile.h has the fragment layouts; operands are rounded to bf16 only where the tensors are bf16 (P and dS enter
// their second product in bf16: 2^-9 of a term, the error that the stored result carries anyway); accumulation is fp32.
#include "mha_tile.h"

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float NO_MAX = -1e30f;  // the running maximum before any visible score; finite, so that differences from it are not NaN
constexpr float LAZY = 8.f;       // the running maximum follows only rises of more than 2^8: P stays below 2^8, and fp32 sums hold that exactly as well

struct MhaArgs {
  const void *q, *k, *v, *out, *dout;
  long qs[3], ks[3], vs[3], os[3], dos[3];  // element strides: batch, token, head
  const unsigned char* mask;
  long mask_sb, mask_sl;
  const float* lse;
  float* delta;
  int B, Lq, Lk, H, Hkv, G, D, causal;
  int rows;         // Lq * G
  float scale, c;   // c = |scale| * log2(e), never 0 (a scale of 0: 1e-30)
  int vec;          // 16-byte loads and stores
  int nblk, nsplit, per_split;  // blocks of rows (keys) per key head, splits of the other axis and its length of one split
};

struct Where {
  int blk, split, hk;
  long b;
};
// Workgroups go round the 8 XCDs in turn; each XCD gets a contiguous range of the work, so that the blocks that read one key head share an L2.
__device__ __forceinline__ Where where(const MhaArgs& a) {
  const unsigned n = gridDim.x, per = n / 8, rest = n % 8, x = blockIdx.x % 8, y = blockIdx.x / 8;
  unsigned id = x * per + min(x, rest) + y;
  Where w;
  w.blk = id % a.nblk;
  id /= a.nblk;
  w.split = id % a.nsplit;
  id /= a.nsplit;
  w.hk = id % a.Hkv;
  w.b = id / a.Hkv;
  return w;
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
  typename Elem<T>::Frag f[DK / Elem<T>::STEP];
  __device__ __forceinline__ void load(const T* row, bool on, int D, int vec, int lane) {
#pragma unroll
    for (int s = 0; s < DK / Elem<T>::STEP; ++s) {
      const uint4 u = on ? load_chunk<T>(row, 2 * s + (lane >> 5), D, vec) : make_uint4(0, 0, 0, 0);
      memcpy(&f[s], &u, 16);
    }
  }
  __device__ __forceinline__ void negate() {
#pragma unroll
    for (int s = 0; s < DK / Elem<T>::STEP; ++s) f[s] = -f[s];
  }
};

// ROWS rows of a tensor on their way into an LDS tile: held in registers by NT threads, zeros where `ok` says so
template <typename T, int DK, int W, int ROWS, int NT>
struct Stage {
  static constexpr int NC = DK / Elem<T>::PER_CHUNK, N = (ROWS * NC + NT - 1) / NT;
  uint4 r[N];
  unsigned ok;
  template <typename Offset, typename Ok>
  __device__ __forceinline__ void load(const T* base, Offset offset, Ok visible, int D, int vec) {
    ok = 0;
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = n * NT + (int)threadIdx.x, row = i / NC;
      if (ROWS * NC % NT && i >= ROWS * NC) break;
      r[n] = load_chunk<T>(base + offset(row), i % NC, D, vec);
      ok |= (visible(row) ? 1u : 0u) << n;
    }
  }
  __device__ __forceinline__ void put(char* tile) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int i = n * NT + (int)threadIdx.x;
      if (ROWS * NC % NT && i >= ROWS * NC) break;
      Tile<T, W>::put(tile, i / NC, i % NC, ok >> n & 1 ? r[n] : make_uint4(0, 0, 0, 0));
    }
  }
};

// the D elements of one row held as accumulators of a transposed product (lane = row, registers = dimensions), times f, to dst
template <typename T, int ND>
__device__ __forceinline__ void store_row(T* dst, const f32x16 (&o)[ND], float f, int D, int vec, int lane) {
#pragma unroll
  for (int dt = 0; dt < ND; ++dt)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int d = 32 * dt + 8 * q + 4 * (lane >> 5);
      const float v[4] = {o[dt][4 * q] * f, o[dt][4 * q + 1] * f, o[dt][4 * q + 2] * f, o[dt][4 * q + 3] * f};
      if (vec) {
        if (d < D) {
          if constexpr (sizeof(T) == 2)
            *reinterpret_cast<uint2*>(dst + d) = tatt_pack_bf16x4(v[0], v[1], v[2], v[3]);
          else
            *reinterpret_cast<float4*>(dst + d) = make_float4(v[0], v[1], v[2], v[3]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (d + e < D) dst[d + e] = from_f32<T>(v[e]);
      }
    }
}

__device__ __forceinline__ float half_max(float x) { return fmaxf(x, __shfl_xor(x, 32, 64)); }
__device__ __forceinline__ float half_sum(float x) { return x + __shfl_xor(x, 32, 64); }
// tile row that accumulator register i of a lane half stands for
__device__ __forceinline__ constexpr int acc_row(int i) { return 8 * (i / 4) + i % 4; }

template <int N>
__device__ __forceinline__ void clear(f32x16 (&o)[N]) {
#pragma unroll
  for (int n = 0; n < N; ++n)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[n][i] = 0.f;
}

// bit j: key k0 + j (32 of them) exists and is not masked; `byte` = the mask byte of key k0 + lane % 32
__device__ __forceinline__ unsigned key_word(int k0, int Lk, int byte, int lane) { return (unsigned)__ballot(k0 + (lane & 31) < Lk && byte == 0); }

// bits 0 .. n (n = -1: none, n >= 31: all)
__device__ __forceinline__ unsigned bits_to(int n) { return n < 0 ? 0u : n >= 31 ? ~0u : (2u << n) - 1u; }

// Forward.  WQ waves along the rows (32 each) x WK along the keys; SUB tiles of 32 keys for a wave at a time.
template <typename T, int DK, int WQ, int WK, int SUB>
__global__ __launch_bounds__(64 * WQ * WK) void mha_fwd_kernel(MhaArgs a, T* __restrict__ out, float* __restrict__ lse, float* __restrict__ part) {
  constexpr int NT = 64 * WQ * WK, W = DK <= 32 ? 32 : DK <= 64 ? 64 : 128, ND = (DK + 31) / 32, KT = 32 * WK * SUB, TILE = KT * Tile<T, W>::ROW;
  constexpr int NS = DK / Elem<T>::STEP, TS = 32 / Elem<T>::STEP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char *kt = lds, *vt = lds + TILE;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wq = wave % WQ, wk = wave / WQ, half = lane >> 5;
  const Where w = where(a);
  const int blk = a.causal ? a.nblk - 1 - w.blk : w.blk;  // causal: the longest blocks first
  const int row0 = blk * 32 * WQ, row = row0 + 32 * wq + (lane & 31);
  const T* kb = (const T*)a.k + w.b * a.ks[0] + w.hk * a.ks[2];
  const T* vb = (const T*)a.v + w.b * a.vs[0] + w.hk * a.vs[2];
  const unsigned char* mb = a.mask ? a.mask + w.b * a.mask_sb : nullptr;
  const int past = a.Lk - a.Lq;
  const int query = (unsigned)row / (unsigned)a.G;
  const int first_query = (row0 + 32 * wq) / a.G, last_query = min(a.rows - 1, row0 + 32 * wq + 31) / a.G;

  RowFrags<T, DK> qf;
  qf.load((const T*)a.q + w.b * a.qs[0] + w.hk * a.G * a.qs[2] + row_offset(min(row, a.rows - 1), a.G, a.qs[1], a.qs[2]), row < a.rows, a.D, a.vec, lane);
  if (a.scale < 0.f) qf.negate();

  const int kbeg = w.split * a.per_split;
  int kend = min(a.Lk, kbeg + a.per_split);
  if (a.causal) kend = min(kend, min(a.rows - 1, row0 + 32 * WQ - 1) / a.G + past + 1);

  f32x16 o[ND];
  clear(o);
  float m = NO_MAX, l = 0.f;

  Stage<T, DK, W, KT, NT> ks, vs;
  int bytes[SUB];
  auto fetch = [&](int k0) {
    auto visible = [&](int r) { return k0 + r < kend && (!mb || mb[(long)(k0 + r) * a.mask_sl] == 0); };
    ks.load(kb, [&](int r) { return min(k0 + r, a.Lk - 1) * a.ks[1]; }, visible, a.D, a.vec);
    vs.load(vb, [&](int r) { return min(k0 + r, a.Lk - 1) * a.vs[1]; }, visible, a.D, a.vec);
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int j = k0 + 32 * (wk * SUB + s) + (lane & 31);
      bytes[s] = mb && j < a.Lk ? mb[(long)j * a.mask_sl] : 0;
    }
  };
  if (kbeg < kend) fetch(kbeg);
  for (int k0 = kbeg; k0 < kend; k0 += KT) {
    __syncthreads();
    ks.put(kt);
    vs.put(vt);
    unsigned word[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) word[s] = key_word(k0 + 32 * (wk * SUB + s), kend, bytes[s], lane);
    __syncthreads();
    if (k0 + KT < kend) fetch(k0 + KT);
    f32x16 sc[SUB];
    bool any = false;
    float tmax = -INFINITY;
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int at = 32 * (wk * SUB + s), limit = a.causal ? query + past - k0 - at : 31;
      if (a.causal && last_query + past - k0 - at < 0) word[s] = 0;
      if (word[s] == 0) continue;
      any = true;
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[s][i] = 0.f;
#pragma unroll
      for (int t = 0; t < NS; ++t) sc[s] = mma(Tile<T, W>::rows(kt, at, t, lane), qf.f[t], sc[s]);
      if (word[s] != ~0u || (a.causal && first_query + past - k0 - at < 31)) {
        const unsigned see = (word[s] & bits_to(limit)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[s][i] = see >> acc_row(i) & 1 ? sc[s][i] : -INFINITY;
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) tmax = fmaxf(tmax, sc[s][i]);
    }
    if (!any) continue;
    tmax = half_max(tmax) * a.c;
    if (__any(tmax > m + LAZY)) {
      const float mn = fmaxf(m, tmax), f = __builtin_amdgcn_exp2f(m - mn);
      m = mn;
      l *= f;
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[dt][i] *= f;
    }
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      if (word[s] == 0) continue;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        sc[s][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s][i], a.c, -m));
        l += sc[s][i];
      }
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        const auto p = pack_step<T>(sc[s], t);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[dt] = mma(Tile<T, W>::transposed(vt, 32 * (wk * SUB + s), t, 32 * dt, lane), p, o[dt]);
      }
    }
  }
  l = half_sum(l);

  if constexpr (WK > 1) {  // join the waves along the keys in LDS: [wk][32 rows][W + 4], and their (m, l)
    float *os = reinterpret_cast<float*>(lds), *ml = os + WK * 32 * (W + 4);
    __syncthreads();
    if (half == 0) ml[(wk * 32 + (lane & 31)) * 2] = m, ml[(wk * 32 + (lane & 31)) * 2 + 1] = l;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q)
        *reinterpret_cast<float4*>(os + (wk * 32 + (lane & 31)) * (W + 4) + 32 * dt + 8 * q + 4 * half) =
            make_float4(o[dt][4 * q], o[dt][4 * q + 1], o[dt][4 * q + 2], o[dt][4 * q + 3]);
    __syncthreads();
    if (wk) return;
    float mm = m, f[WK];
#pragma unroll
    for (int x = 1; x < WK; ++x) mm = fmaxf(mm, ml[(x * 32 + (lane & 31)) * 2]);
    l = 0.f;
#pragma unroll
    for (int x = 0; x < WK; ++x) {
      f[x] = __builtin_amdgcn_exp2f(ml[(x * 32 + (lane & 31)) * 2] - mm);
      l += f[x] * ml[(x * 32 + (lane & 31)) * 2 + 1];
    }
    m = mm;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        o[dt][i] *= f[0];
#pragma unroll
        for (int x = 1; x < WK; ++x) o[dt][i] += f[x] * os[(x * 32 + (lane & 31)) * (W + 4) + 32 * dt + acc_row(i) + 4 * half];
      }
  }
  if (row >= a.rows) return;
  const int g = row - query * a.G, h = w.hk * a.G + g;
  if (part) {  // one of several splits: unnormalised sums and (m, l), joined by mha_fwd_join
    const long R = (long)a.B * a.H * a.Lq, r = (w.b * a.Lq + query) * a.H + h;
    store_row<float, ND>(part + (w.split * R + r) * a.D, o, 1.f, a.D, a.D % 4 == 0, lane);
    if (half == 0) {
      float* ml = part + a.nsplit * R * a.D + (w.split * R + r) * 2;
      ml[0] = m, ml[1] = l;
    }
    return;
  }
  store_row<T, ND>(out + ((w.b * a.Lq + query) * a.H + h) * a.D, o, l == 0.f ? 0.f : 1.f / l, a.D, a.vec, lane);
  if (lse && half == 0) lse[(w.b * a.H + h) * a.Lq + query] = l == 0.f ? INFINITY : m + log2f(l);
}

// the splits of a row: a wave per row
template <typename T>
__global__ __launch_bounds__(256) void mha_fwd_join(const float* __restrict__ part, int nsplit, long R, int D, int H, int Lq, T* __restrict__ out, float* __restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const long r = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= R) return;
  const float* ml = part + nsplit * R * D;
  float m = NO_MAX, l = 0.f;
  for (int s = 0; s < nsplit; ++s) m = fmaxf(m, ml[(s * R + r) * 2]);
  float o0 = 0.f, o1 = 0.f;
  for (int s = 0; s < nsplit; ++s) {
    const float f = __builtin_amdgcn_exp2f(ml[(s * R + r) * 2] - m);
    l += f * ml[(s * R + r) * 2 + 1];
    const float* p = part + (s * R + r) * D;
    if (lane < D) o0 += f * p[lane];
    if (lane + 64 < D) o1 += f * p[lane + 64];
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  if (lane < D) out[r * D + lane] = from_f32<T>(o0 * inv);
  if (lane + 64 < D) out[r * D + lane + 64] = from_f32<T>(o1 * inv);
  if (lse && lane == 0) lse[(r / H / Lq * H + r % H) * Lq + r / H % Lq] = l == 0.f ? INFINITY : m + log2f(l);
}

// dQ and delta.  As the forward pass with WQ waves along the rows; registers hold Q and dO, LDS tiles of 32 SUB keys K and V.
template <typename T, int DK, int WQ, int SUB>
__global__ __launch_bounds__(64 * WQ) void mha_dq_kernel(MhaArgs a, T* __restrict__ dq, float* __restrict__ part) {
  constexpr int NT = 64 * WQ, W = DK <= 32 ? 32 : DK <= 64 ? 64 : 128, ND = (DK + 31) / 32, KT = 32 * SUB, TILE = KT * Tile<T, W>::ROW;
  constexpr int NS = DK / Elem<T>::STEP, TS = 32 / Elem<T>::STEP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char *kt = lds, *vt = lds + TILE;
  const int lane = threadIdx.x & 63, wq = threadIdx.x >> 6, half = lane >> 5;
  const Where w = where(a);
  const int blk = a.causal ? a.nblk - 1 - w.blk : w.blk;
  const int row0 = blk * 32 * WQ, row = row0 + 32 * wq + (lane & 31), past = a.Lk - a.Lq;
  const bool on = row < a.rows;
  const int safe = min(row, a.rows - 1), query = (unsigned)safe / (unsigned)a.G, h = w.hk * a.G + safe - query * a.G;
  const int first_query = (row0 + 32 * wq) / a.G, last_query = min(a.rows - 1, row0 + 32 * wq + 31) / a.G;
  const T* kb = (const T*)a.k + w.b * a.ks[0] + w.hk * a.ks[2];
  const T* vb = (const T*)a.v + w.b * a.vs[0] + w.hk * a.vs[2];
  const unsigned char* mb = a.mask ? a.mask + w.b * a.mask_sb : nullptr;

  RowFrags<T, DK> qf, gf;
  qf.load((const T*)a.q + w.b * a.qs[0] + query * a.qs[1] + h * a.qs[2], on, a.D, a.vec, lane);
  gf.load((const T*)a.dout + w.b * a.dos[0] + query * a.dos[1] + h * a.dos[2], on, a.D, a.vec, lane);
  if (a.scale < 0.f) qf.negate();
  float delta = 0.f;
  {
    const T* orow = (const T*)a.out + w.b * a.os[0] + query * a.os[1] + h * a.os[2];
#pragma unroll
    for (int s = 0; s < NS; ++s) {
      const uint4 u = load_chunk<T>(orow, 2 * s + half, a.D, a.vec);
      T t[Elem<T>::PER_CHUNK];
      memcpy(t, &u, 16);
#pragma unroll
      for (int e = 0; e < Elem<T>::PER_CHUNK; ++e) delta += to_f32(t[e]) * (float)gf.f[s][e];
    }
    delta = half_sum(delta);
  }
  const long stat = (w.b * a.H + h) * a.Lq + query;
  const float lse = on ? a.lse[stat] : INFINITY;
  const bool empty = lse == INFINITY;
  if (empty) delta = 0.f;  // whatever dO holds there
  if (on && half == 0 && w.split == 0) a.delta[stat] = delta;

  const int kbeg = w.split * a.per_split;
  int kend = min(a.Lk, kbeg + a.per_split);
  if (a.causal) kend = min(kend, min(a.rows - 1, row0 + 32 * WQ - 1) / a.G + past + 1);
  f32x16 o[ND];
  clear(o);
  Stage<T, DK, W, KT, NT> ks, vs;
  int bytes[SUB];
  auto fetch = [&](int k0) {
    auto visible = [&](int r) { return k0 + r < kend && (!mb || mb[(long)(k0 + r) * a.mask_sl] == 0); };
    ks.load(kb, [&](int r) { return min(k0 + r, a.Lk - 1) * a.ks[1]; }, visible, a.D, a.vec);
    vs.load(vb, [&](int r) { return min(k0 + r, a.Lk - 1) * a.vs[1]; }, visible, a.D, a.vec);
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int j = k0 + 32 * s + (lane & 31);
      bytes[s] = mb && j < a.Lk ? mb[(long)j * a.mask_sl] : 0;
    }
  };
  if (kbeg < kend) fetch(kbeg);
  for (int k0 = kbeg; k0 < kend; k0 += KT) {
    __syncthreads();
    ks.put(kt);
    vs.put(vt);
    unsigned word[SUB];
#pragma unroll
    for (int s = 0; s < SUB; ++s) word[s] = key_word(k0 + 32 * s, kend, bytes[s], lane);
    __syncthreads();
    if (k0 + KT < kend) fetch(k0 + KT);
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      const int at = 32 * s;
      if (word[s] == 0 || (a.causal && last_query + past - k0 - at < 0)) continue;
      f32x16 sc, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = dp[i] = 0.f;
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        sc = mma(Tile<T, W>::rows(kt, at, t, lane), qf.f[t], sc);
        dp = mma(Tile<T, W>::rows(vt, at, t, lane), gf.f[t], dp);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.c, -lse)) * (dp[i] - delta);
      if (word[s] != ~0u || (a.causal && first_query + past - k0 - at < 31)) {
        const unsigned see = (word[s] & (a.causal ? bits_to(query + past - k0 - at) : ~0u)) >> (4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[i] = see >> acc_row(i) & 1 ? sc[i] : 0.f;
      }
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        const auto p = pack_step<T>(sc, t);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) o[dt] = mma(Tile<T, W>::transposed(kt, at, t, 32 * dt, lane), p, o[dt]);
      }
    }
  }
  if (!on) return;
  if (empty) clear(o);
  const long r = (w.b * a.Lq + query) * a.H + h;
  if (part)
    store_row<float, ND>(part + (w.split * (long)a.B * a.H * a.Lq + r) * a.D, o, a.scale, a.D, a.D % 4 == 0, lane);
  else
    store_row<T, ND>(dq + r * a.D, o, a.scale, a.D, a.vec, lane);
}

// dK and dV.  WN waves along the keys (32 each) x WR along the rows; LDS holds tiles of 32 WR rows of Q and dO, and their lse and delta.
template <typename T, int DK, int WN, int WR>
__global__ __launch_bounds__(64 * WN * WR) void mha_dkv_kernel(MhaArgs a, T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part) {
  constexpr int NT = 64 * WN * WR, W = DK <= 32 ? 32 : DK <= 64 ? 64 : 128, ND = (DK + 31) / 32, RT = 32 * WR, TILE = RT * Tile<T, W>::ROW;
  constexpr int NS = DK / Elem<T>::STEP, TS = 32 / Elem<T>::STEP;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  char *qt = lds, *gt = lds + TILE;
  float *ls = reinterpret_cast<float*>(lds + 2 * TILE), *dl = ls + RT;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wn = wave % WN, wr = wave / WN, half = lane >> 5;
  const Where w = where(a);
  const int key0 = w.blk * 32 * WN, key = key0 + 32 * wn + (lane & 31), past = a.Lk - a.Lq;
  const bool on = key < a.Lk && !(a.mask && a.mask[w.b * a.mask_sb + (long)key * a.mask_sl]);
  const long key_safe = min(key, a.Lk - 1);
  RowFrags<T, DK> kf, vf;
  kf.load((const T*)a.k + w.b * a.ks[0] + key_safe * a.ks[1] + w.hk * a.ks[2], on, a.D, a.vec, lane);
  vf.load((const T*)a.v + w.b * a.vs[0] + key_safe * a.vs[1] + w.hk * a.vs[2], on, a.D, a.vec, lane);
  if (a.scale < 0.f) kf.negate();
  const T* qb = (const T*)a.q + w.b * a.qs[0] + w.hk * a.G * a.qs[2];
  const T* gb = (const T*)a.dout + w.b * a.dos[0] + w.hk * a.G * a.dos[2];
  const float* lse = a.lse + (w.b * a.H + w.hk * a.G) * a.Lq;
  const float* delta = a.delta + (w.b * a.H + w.hk * a.G) * a.Lq;

  // causal: this key is seen from row G (key - past) on; rows before the first query that sees anything hold what they like
  const int first_row = a.causal ? a.G * max(0, key - past) : 0;
  const int empty_rows = a.causal ? a.G * max(0, -past) : 0;
  int rbeg = w.split * a.per_split;
  const int rend = min(a.rows, rbeg + a.per_split);
  if (a.causal) rbeg = max(rbeg, a.G * max(0, key0 - past) / RT * RT);
  f32x16 ok[ND], ov[ND];
  clear(ok);
  clear(ov);
  const bool any = __syncthreads_or(on);  // nothing to do where every key of the block is masked

  Stage<T, DK, W, RT, NT> qs, gs;
  float l0 = 0.f, d0 = 0.f;
  auto fetch = [&](int r0) {
    auto visible = [&](int r) { return r0 + r < rend && r0 + r >= empty_rows; };
    qs.load(qb, [&](int r) { return row_offset(min(r0 + r, a.rows - 1), a.G, a.qs[1], a.qs[2]); }, visible, a.D, a.vec);
    gs.load(gb, [&](int r) { return row_offset(min(r0 + r, a.rows - 1), a.G, a.dos[1], a.dos[2]); }, visible, a.D, a.vec);
    if (threadIdx.x < RT) {
      const int r = r0 + threadIdx.x;
      const bool there = r < rend && r >= empty_rows;
      const int i = (unsigned)min(r, a.rows - 1) / (unsigned)a.G;
      const long at = (long)(min(r, a.rows - 1) - i * a.G) * a.Lq + i;
      l0 = there ? lse[at] : INFINITY;
      d0 = there ? delta[at] : 0.f;
    }
  };
  if (any) {
    if (rbeg < rend) fetch(rbeg);
    for (int r0 = rbeg; r0 < rend; r0 += RT) {
      __syncthreads();
      qs.put(qt);
      gs.put(gt);
      if (threadIdx.x < RT) ls[threadIdx.x] = l0, dl[threadIdx.x] = d0;
      __syncthreads();
      if (r0 + RT < rend) fetch(r0 + RT);
      const int at = 32 * wr;
      f32x16 sc, dp;
#pragma unroll
      for (int i = 0; i < 16; ++i) sc[i] = dp[i] = 0.f;
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        sc = mma(Tile<T, W>::rows(qt, at, t, lane), kf.f[t], sc);
        dp = mma(Tile<T, W>::rows(gt, at, t, lane), vf.f[t], dp);
      }
      const int hidden = first_row - r0 - at - 4 * half;  // accumulator rows below this are causally hidden
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const float4 lq = *reinterpret_cast<const float4*>(ls + at + 8 * q + 4 * half), dq = *reinterpret_cast<const float4*>(dl + at + 8 * q + 4 * half);
        const float lv[4] = {lq.x, lq.y, lq.z, lq.w}, dv4[4] = {dq.x, dq.y, dq.z, dq.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int i = 4 * q + e;
          const float p = on && acc_row(i) >= hidden ? __builtin_amdgcn_exp2f(__builtin_fmaf(sc[i], a.c, -lv[e])) : 0.f;
          sc[i] = p;
          dp[i] = p * (dp[i] - dv4[e]);
        }
      }
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        const auto p = pack_step<T>(sc, t), ds = pack_step<T>(dp, t);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          ov[dt] = mma(Tile<T, W>::transposed(gt, at, t, 32 * dt, lane), p, ov[dt]);
          ok[dt] = mma(Tile<T, W>::transposed(qt, at, t, 32 * dt, lane), ds, ok[dt]);
        }
      }
    }
  }
  if constexpr (WR > 1) {  // sum the waves along the rows in LDS, one of the two gradients at a time: [WN][32 keys][W + 4] added to in wave order
    float* os = reinterpret_cast<float*>(lds) + (wn * 32 + (lane & 31)) * (W + 4);
#pragma unroll
    for (int which = 0; which < 2; ++which)
      for (int x = WR - 1; x >= 0; --x) {
        __syncthreads();
        if (wr != x) continue;
#pragma unroll
        for (int dt = 0; dt < ND; ++dt)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            f32x16& o = which ? ok[dt] : ov[dt];
            float4* p = reinterpret_cast<float4*>(os + 32 * dt + 8 * q + 4 * half);
            float4 s = x == WR - 1 ? make_float4(0, 0, 0, 0) : *p;
            s.x += o[4 * q], s.y += o[4 * q + 1], s.z += o[4 * q + 2], s.w += o[4 * q + 3];
            if (x)
              *p = s;
            else
              o[4 * q] = s.x, o[4 * q + 1] = s.y, o[4 * q + 2] = s.z, o[4 * q + 3] = s.w;
          }
      }
    if (wr) return;
  }
  if (key >= a.Lk) return;
  const long r = (w.b * a.Lk + key) * a.Hkv + w.hk;
  if (part) {
    const long R = (long)a.B * a.Lk * a.Hkv;
    store_row<float, ND>(part + ((w.split * 2L) * R + r) * a.D, ok, a.scale, a.D, a.D % 4 == 0, lane);
    store_row<float, ND>(part + ((w.split * 2L + 1) * R + r) * a.D, ov, 1.f, a.D, a.D % 4 == 0, lane);
  } else {
    store_row<T, ND>(dk + r * a.D, ok, a.scale, a.D, a.vec, lane);
    store_row<T, ND>(dv + r * a.D, ov, 1.f, a.D, a.vec, lane);
  }
}

// y[i] = sum over splits of part[split][i] in split order; two tensors of n values each where y2
template <typename T>
__global__ __launch_bounds__(256) void mha_sum_kernel(const float* __restrict__ part, int nsplit, long n, T* __restrict__ y, T* __restrict__ y2) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, all = y2 ? 2 * n : n;
  if (i >= all) return;
  float s = 0.f;
  for (int k = 0; k < nsplit; ++k) s += part[k * all + i];
  (i < n ? y : y2)[i < n ? i : i - n] = from_f32<T>(s);
}

// ---- launch plans ---------------------------------------------------------------------------------------------------------------------
constexpr int FILL = 512;  // workgroups that fill the 256 CUs twice

struct Plan {
  int wide, nblk, nsplit, per_split;  // wide: waves side by side along the output axis; else along the summed one
};
// blocks of `width` along the output axis (32 if it has no more than 32), and the summed axis split while the chip is not full, no finer than `least`
Plan plan(long problems, int outer, int inner, int width, int least) {
  Plan p;
  p.wide = outer > 32;
  p.nblk = cdiv(outer, p.wide ? width : 32);
  const long blocks = problems * p.nblk;
  long n = blocks >= FILL ? 1 : (2 * FILL + blocks - 1) / blocks;
  if (n > inner / least) n = inner / least;
  if (n < 1) n = 1;
  p.per_split = cdiv(cdiv(inner, n), 128) * 128;
  p.nsplit = cdiv(inner, p.per_split);
  return p;
}
Plan plan_fwd(int B, int Lq, int Lk, int H, int Hkv) { return plan((long)B * Hkv, Lq * (H / Hkv), Lk, 128, 512); }
Plan plan_dq(int B, int Lq, int Lk, int H, int Hkv) { return plan((long)B * Hkv, Lq * (H / Hkv), Lk, 128, 512); }
Plan plan_dkv(int B, int Lq, int Lk, int H, int Hkv) { return plan((long)B * Hkv, Lk, Lq * (H / Hkv), 128, 512); }

int fill(MhaArgs& a, const char* who, const void* q, const void* k, const void* v, const long* strides, const unsigned char* mask, const long* mask_strides,
         int B, int Lq, int Lk, int H, int Hkv, int D, float scale, int causal, int dtype, const float* workspace) {
  TATT_CHECK_ARG(q && k && v && strides && B > 0 && Lq > 0 && Lk > 0 && H > 0 && Hkv > 0, "%s: bad arguments", who);
  TATT_CHECK_ARG(!mask || mask_strides, "%s: a key mask needs its strides", who);
  TATT_CHECK_ARG(H % Hkv == 0, "%s: %d query heads are no multiple of %d key heads", who, H, Hkv);
  TATT_CHECK_ARG(D > 0 && D <= 128, "%s: built for heads of 1 to 128, got %d", who, D);
  TATT_CHECK_ARG(dtype == TATT_T_F32 || dtype == TATT_T_BF16, "%s: unknown element type %d", who, dtype);
  TATT_CHECK_ARG(((uintptr_t)workspace & 15) == 0, "%s: the workspace is not 16-byte aligned", who);
  TATT_CHECK_ARG((long)B * H * Lq < (1L << 30) && (long)B * Hkv * Lk < (1L << 30), "%s: 2^30 rows or more", who);
  a.q = q, a.k = k, a.v = v, a.mask = mask;
  a.mask_sb = mask ? mask_strides[0] : 0, a.mask_sl = mask ? mask_strides[1] : 0;
  for (int i = 0; i < 3; ++i) a.qs[i] = strides[i], a.ks[i] = strides[3 + i], a.vs[i] = strides[6 + i];
  a.B = B, a.Lq = Lq, a.Lk = Lk, a.H = H, a.Hkv = Hkv, a.G = H / Hkv, a.D = D, a.causal = causal;
  a.rows = Lq * a.G;
  a.scale = scale;
  a.c = scale == 0.f ? 1e-30f : fabsf(scale) * LOG2E;
  return TATT_OK;
}

bool aligned(const void* p, const long* s, int size) {
  return ((uintptr_t)p & 15) == 0 && (!s || (s[0] * size % 16 == 0 && s[1] * size % 16 == 0 && s[2] * size % 16 == 0));
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

template <typename T, int DK>
struct Shape {
  static constexpr int W = DK <= 32 ? 32 : DK <= 64 ? 64 : 128;
  static constexpr int ROW = Tile<T, W>::ROW;
  static constexpr int WK = ROW > 256 ? 2 : 4;  // waves along the summed axis: tiles of 32 WK rows, two of them within 64 KB
};

template <typename T, int DK, int WQ, int WK, int SUB>
int launch_fwd(const MhaArgs& a, T* out, float* lse, float* part, hipStream_t st) {
  using S = Shape<T, DK>;
  size_t lds = 2 * 32 * WK * SUB * S::ROW;
  const size_t join = WK > 1 ? (size_t)WK * 32 * (S::W + 4 + 2) * 4 : 0;
  if (join > lds) lds = join;
  if (int rc = prepare_launch(a, mha_fwd_kernel<T, DK, WQ, WK, SUB>, 64 * WQ * WK, lds)) return rc;
  hipLaunchKernelGGL((mha_fwd_kernel<T, DK, WQ, WK, SUB>), dim3((unsigned)((long)a.B * a.Hkv * a.nblk * a.nsplit)), dim3(64 * WQ * WK), lds, st, a, out, lse, part);
  TATT_LAUNCH_CHECK("mha_fwd");
  return TATT_OK;
}

template <typename T, int DK>
int run_fwd(MhaArgs& a, T* out, float* lse, float* part, hipStream_t st) {
  using S = Shape<T, DK>;
  const Plan p = plan_fwd(a.B, a.Lq, a.Lk, a.H, a.Hkv);
  a.nblk = p.nblk, a.nsplit = p.nsplit, a.per_split = p.per_split;
  if (p.nsplit == 1) part = nullptr;
  if (int rc = p.wide ? launch_fwd<T, DK, 4, 1, 2>(a, out, lse, part, st) : launch_fwd<T, DK, 1, S::WK, 1>(a, out, lse, part, st)) return rc;
  if (part) {
    const long R = (long)a.B * a.H * a.Lq;
    hipLaunchKernelGGL(mha_fwd_join<T>, dim3(cdiv(R, 4)), dim3(256), 0, st, part, a.nsplit, R, a.D, a.H, a.Lq, out, lse);
    TATT_LAUNCH_CHECK("mha_fwd_join");
  }
  return TATT_OK;
}

template <typename T, int DK, int WN, int WR>
int launch_dkv(const MhaArgs& a, T* dk, T* dv, float* part, hipStream_t st) {
  using S = Shape<T, DK>;
  size_t lds = 2 * 32 * WR * S::ROW + 2 * 32 * WR * 4;
  const size_t join = WR > 1 ? (size_t)WN * 32 * (S::W + 4) * 4 : 0;
  if (join > lds) lds = join;
  if (int rc = prepare_launch(a, mha_dkv_kernel<T, DK, WN, WR>, 64 * WN * WR, lds)) return rc;
  hipLaunchKernelGGL((mha_dkv_kernel<T, DK, WN, WR>), dim3((unsigned)((long)a.B * a.Hkv * a.nblk * a.nsplit)), dim3(64 * WN * WR), lds, st, a, dk, dv, part);
  TATT_LAUNCH_CHECK("mha_dkv");
  return TATT_OK;
}

template <typename T, int DK>
int run_bwd(MhaArgs& a, T* dq, T* dk, T* dv, float* part, hipStream_t st) {
  using S = Shape<T, DK>;
  Plan p = plan_dq(a.B, a.Lq, a.Lk, a.H, a.Hkv);
  a.nblk = cdiv(a.rows, 128), a.nsplit = p.nsplit, a.per_split = p.per_split;
  {
    constexpr int SUB = 2;
    const size_t lds = 2 * 32 * SUB * S::ROW;
    if (int rc = prepare_launch(a, mha_dq_kernel<T, DK, 4, SUB>, 256, lds)) return rc;
    hipLaunchKernelGGL((mha_dq_kernel<T, DK, 4, SUB>), dim3((unsigned)((long)a.B * a.Hkv * a.nblk * a.nsplit)), dim3(256), lds, st, a, dq,
                       a.nsplit > 1 ? part : nullptr);
    TATT_LAUNCH_CHECK("mha_dq");
    if (a.nsplit > 1) {
      const long n = (long)a.B * a.H * a.Lq * a.D;
      hipLaunchKernelGGL(mha_sum_kernel<T>, dim3(cdiv(n, 256)), dim3(256), 0, st, part, a.nsplit, n, dq, (T*)nullptr);
      TATT_LAUNCH_CHECK("mha_sum");
    }
  }
  p = plan_dkv(a.B, a.Lq, a.Lk, a.H, a.Hkv);
  a.nblk = p.nblk, a.nsplit = p.nsplit, a.per_split = p.per_split;
  float* kv_part = a.nsplit > 1 ? part : nullptr;
  if (int rc = p.wide ? launch_dkv<T, DK, 4, 1>(a, dk, dv, kv_part, st) : launch_dkv<T, DK, 1, S::WK>(a, dk, dv, kv_part, st)) return rc;
  if (kv_part) {
    const long n = (long)a.B * a.Hkv * a.Lk * a.D;
    hipLaunchKernelGGL(mha_sum_kernel<T>, dim3(cdiv(2 * n, 256)), dim3(256), 0, st, part, a.nsplit, n, dk, dv);
    TATT_LAUNCH_CHECK("mha_sum");
  }
  return TATT_OK;
}

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

bool sane(int B, int Lq, int Lk, int H, int Hkv, int D) { return B > 0 && Lq > 0 && Lk > 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && D > 0; }

}  // namespace

extern "C" {

size_t tatt_mha_fwd_workspace(int B, int Lq, int Lk, int H, int Hkv, int D, int dtype) {
  if (!sane(B, Lq, Lk, H, Hkv, D)) return 0;
  const Plan p = plan_fwd(B, Lq, Lk, H, Hkv);
  return p.nsplit == 1 ? 0 : (size_t)p.nsplit * B * H * Lq * (D + 2);
}

int tatt_mha_fwd(const void* q, const void* k, const void* v, const long* strides, const unsigned char* mask, const long* mask_strides,
                 void* out, float* lse, int B, int Lq, int Lk, int H, int Hkv, int D, float scale, int causal, int dtype, float* workspace,
                 hipStream_t st) {
  MhaArgs a = {};
  if (int rc = fill(a, "tatt_mha_fwd", q, k, v, strides, mask, mask_strides, B, Lq, Lk, H, Hkv, D, scale, causal, dtype, workspace)) return rc;
  TATT_CHECK_ARG(out, "tatt_mha_fwd: no output");
  TATT_CHECK_ARG(workspace || tatt_mha_fwd_workspace(B, Lq, Lk, H, Hkv, D, dtype) == 0, "tatt_mha_fwd: needs tatt_mha_fwd_workspace floats");
  const int size = dtype == TATT_T_BF16 ? 2 : 4;
  a.vec = D * size % 16 == 0 && aligned(q, a.qs, size) && aligned(k, a.ks, size) && aligned(v, a.vs, size) && aligned(out, nullptr, size);
  TATT_DISPATCH_TYPE(dtype, TATT_DISPATCH_WIDTH(D, return (run_fwd<T, DK>(a, (T*)out, lse, workspace, st)););;);
  return TATT_OK;
}

size_t tatt_mha_bwd_workspace(int B, int Lq, int Lk, int H, int Hkv, int D, int dtype) {
  if (!sane(B, Lq, Lk, H, Hkv, D)) return 0;
  const Plan p = plan_dq(B, Lq, Lk, H, Hkv), q = plan_dkv(B, Lq, Lk, H, Hkv);
  const size_t a = p.nsplit == 1 ? 0 : (size_t)p.nsplit * B * H * Lq * D, b = q.nsplit == 1 ? 0 : (size_t)q.nsplit * 2 * B * Hkv * Lk * D;
  return ((size_t)B * H * Lq + 3) / 4 * 4 + (a > b ? a : b);  // delta, then the partial sums of one kernel at a time
}

int tatt_mha_bwd(const void* q, const void* k, const void* v, const long* strides, const unsigned char* mask, const long* mask_strides,
                 const void* out, const void* dout, const float* lse, void* dq, void* dk, void* dv, int B, int Lq, int Lk, int H, int Hkv, int D,
                 float scale, int causal, int dtype, float* workspace, hipStream_t st) {
  MhaArgs a = {};
  if (int rc = fill(a, "tatt_mha_bwd", q, k, v, strides, mask, mask_strides, B, Lq, Lk, H, Hkv, D, scale, causal, dtype, workspace)) return rc;
  TATT_CHECK_ARG(out && dout && lse && dq && dk && dv && workspace, "tatt_mha_bwd: bad arguments (workspace: tatt_mha_bwd_workspace floats)");
  a.out = out, a.dout = dout, a.lse = lse, a.delta = workspace;
  for (int i = 0; i < 3; ++i) a.os[i] = strides[9 + i], a.dos[i] = strides[12 + i];
  const int size = dtype == TATT_T_BF16 ? 2 : 4;
  a.vec = D * size % 16 == 0 && aligned(q, a.qs, size) && aligned(k, a.ks, size) && aligned(v, a.vs, size) && aligned(out, a.os, size) &&
          aligned(dout, a.dos, size) && aligned(dq, nullptr, size) && aligned(dk, nullptr, size) && aligned(dv, nullptr, size);
  float* part = workspace + ((size_t)B * H * Lq + 3) / 4 * 4;
  TATT_DISPATCH_TYPE(dtype, TATT_DISPATCH_WIDTH(D, return (run_bwd<T, DK>(a, (T*)dq, (T*)dk, (T*)dv, part, st)););;);
  return TATT_OK;
}

}  // extern "C"
