// Attention of any lengths, head counts and head widths up to 128, forward (attn.hip is the 26-key, 4 x 16 form; mha.h has the mathematics
// and the layouts).  One pass over the keys with a running maximum and sum; no score leaves the registers.
//
// Bound: of a tile of 32 x 32 scores a wave issues D / 16 products of 32 cycles for the scores, D / 8 (P in two pieces, bf16) for the output and some
// 150 vector instructions (maximum, exponential, sum, packing), and the two hardly overlap within a wave; two waves a SIMD share it.  Keys come
// through LDS, 64 a tile, two buffers, loaded a tile ahead.
// 64 rows a wave (R = 2) read every fragment from LDS once for two products; 32 keep more workgroups where rows are few, and the registers of
// heads wider than 64 hold no more.  Measured, at the clock that a busy chip keeps: 4 x 4096 tokens, 8 heads of 64, bf16: 228 us,
// 904 TFLOP/s of executed products (R = 1: 249 us); 16 x 1024, 4 heads of 64, fp32: 92 us, 186 TFLOP/s of fp32 products; 4 x 2816, 16 heads of 128, bf16:
// 401 us, 972 TFLOP/s; one causal clip of 2777 tokens, 16 / 4 heads of 128, in three splits: 62 us, 770 TFLOP/s, and 18 to 22 for the join.
// A single query reads its keys at 3.1 TB/s, half of what reading alone reaches (8 sequences of up to 20000 keys, 8 key heads of 128, bf16: 107 us): the keys
// are split over workgroups, one tile of rows each (the G heads of a key head), with the sums joined afterwards.
#include "mha.h"

namespace {

constexpr float NO_MAX = -3.40282347e38f;  // the running maximum before any visible score: the lowest number, finite so that differences from it are not NaN
// A maximum this far from 0 makes its row NaN: the product of score and scale is rounded in the maximum and not in the difference from it, and past
// 2^31 that residue (2^-24 of it) leaves the range of the exponential, so that the row would come out as zeros or infinities by chance.
constexpr float FAR = 536870912.f;  // 2^29
constexpr float LAZY = 8.f;       // the running maximum follows only rises of more than 2^8: P stays below 2^8, and fp32 sums hold that exactly as well

// WQ waves along the rows (32 R each) x WK along the keys; tiles of 32 SUB keys for a wave, JOINT of them sharing a look at the maximum.
template <typename T, int DK, int WQ, int R, int WK, int SUB, int JOINT>
__global__ __launch_bounds__(64 * WQ * WK, fwd_waves<T>(DK)) void mha_fwd_kernel(MhaArgs a, T* __restrict__ out, bf16_t* __restrict__ low, float* __restrict__ lse, float* __restrict__ part) {
  constexpr int NT = 64 * WQ * WK, W = row_width(DK), ND = (DK + 31) / 32, KT = 32 * WK * SUB, TILE = Tile<T, W, KT>::BYTES;
  constexpr int NS = DK / STEP, TS = 32 / STEP, NB = 4 * TILE <= 64 * 1024 ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wq = wave % WQ, wk = wave / WQ, half = lane >> 5;
  const Where w = where(a);
  const int blk = a.causal ? a.nblk - 1 - w.blk : w.blk;  // causal: the last rows see most keys
  const int row0 = blk * 32 * WQ * R, wrow0 = row0 + 32 * wq * R, row = wrow0 + (lane & 31);  // and row + 32 r
  const T* kb = (const T*)a.k + w.b * a.ks[0] + w.hk * a.ks[2];
  const T* vb = (const T*)a.v + w.b * a.vs[0] + w.hk * a.vs[2];
  const unsigned char* mb = a.mask ? a.mask + w.b * a.mask_sb : nullptr;
  const int past = a.Lk - a.Lq;
  const int first_query = wrow0 / a.G;

  RowFrags<T, DK> qf[R];
  int query[R];
  f32x16 o[R][ND];
  float m[R], l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    query[r] = (unsigned)(row + 32 * r) / (unsigned)a.G;
    qf[r].load((const T*)a.q + w.b * a.qs[0] + w.hk * a.G * a.qs[2] + row_offset(min(row + 32 * r, a.rows - 1), a.G, a.qs[1], a.qs[2]), row + 32 * r < a.rows, a.D, lane);
    if (a.scale < 0.f) qf[r].negate();
    clear(o[r]);
    m[r] = NO_MAX;
    l[r] = 0.f;
  }

  int kbeg = 0, kend = a.Lk;
  if (a.causal) kend = min(kend, min(a.rows - 1, row0 + 32 * WQ * R - 1) / a.G + past + 1);
  take_split(a, w.split, KT, kbeg, kend);
  if (mb && kend - kbeg > 2 * KT) trim_keys<NT>(mb, a.mask_sl, kbeg, kend, reinterpret_cast<int*>(lds));

  Stage<T, W, KT, NT, true> ks, vs;
  KeyBits<KT> next, now;
  ks.linear(a.ks[1], a.D);
  vs.linear(a.vs[1], a.D);
  typename Tile<T, W, KT>::Lane place(lane);
  auto fetch = [&](int k0) {
    ks.load(kb + k0 * a.ks[1], 0, kend - k0);
    vs.load(vb + k0 * a.vs[1], 0, kend - k0);
    next.load(mb, a.mask_sl, k0, kend, lane);
  };
  auto put = [&](char* to, int k0) {
    next.settle(mb, k0, kend);
    if (mb && !next.full()) vs.hide(next.word);  // a masked key's scores are replaced, its V would still meet a probability of 0
    ks.put(to);
    vs.put(to + TILE);
    now = next;
  };
  int at = 0;
  if (kbeg < kend) {
    fetch(kbeg);
    put(lds, kbeg);
    wait_loads();
    if (NB == 2 && kbeg + KT < kend) fetch(kbeg + KT);
    __syncthreads();
  }
  // One version of the loop's body, conditions around single steps only: the accumulators stay where they are (with a version for whole tiles
  // beside one for masked ones the compiler copied them every tile, waiting for the products to do so: 226 us against 190, 4 x 4096, 8 x 64, bf16, P in
  // one piece).
  for (int k0 = kbeg; k0 < kend; k0 += KT) {
    if (NB == 1 && k0 + KT < kend) fetch(k0 + KT);
    const char *kt = lds + at, *vt = kt + TILE;
    place.afresh();
#pragma unroll
    for (int s0 = 0; s0 < SUB; s0 += JOINT) {
      const int j0 = 32 * (wk * SUB + s0);  // of the tile's keys
      f32x16 sc[JOINT][R];
#pragma unroll
      for (int s = 0; s < JOINT; ++s) {
#pragma unroll
        for (int r = 0; r < R; ++r) clear(sc[s][r]);
#pragma unroll
        for (int t = 0; t < NS; ++t) {
          const auto k = Tile<T, W, KT>::rows(kt, j0 + 32 * s, t, place);
#pragma unroll
          for (int r = 0; r < R; ++r) sc[s][r] = mma(k, qf[r].f[t], sc[s][r]);
        }
      }
      if (!now.full() || (a.causal && first_query + past < k0 + j0 + 32 * JOINT - 1)) {
#pragma unroll
        for (int s = 0; s < JOINT; ++s)
#pragma unroll
          for (int r = 0; r < R; ++r) {
            const unsigned see = (now.of(j0 + 32 * s) & (a.causal ? bits_to(query[r] + past - k0 - j0 - 32 * s) : ~0u)) >> (4 * half);
#pragma unroll
            for (int i = 0; i < 16; ++i) sc[s][r][i] = see >> acc_row(i) & 1 ? sc[s][r][i] : -INFINITY;
          }
      }
      float tmax[R];
      bool rise = false;
#pragma unroll
      for (int r = 0; r < R; ++r) {
        tmax[r] = -INFINITY;
#pragma unroll
        for (int s = 0; s < JOINT; ++s)
#pragma unroll
          for (int i = 0; i < 16; ++i) tmax[r] = fmaxf(tmax[r], sc[s][r][i]);
        tmax[r] = half_max(tmax[r]) * a.c;
        rise = rise || tmax[r] > m[r] + LAZY;
      }
      if (__any(rise)) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          float mn = fmaxf(m[r], tmax[r]);
          if (fabsf(mn) >= FAR && mn != NO_MAX) mn = NAN;
          const float f = __builtin_amdgcn_exp2f(m[r] - mn);
          m[r] = mn;
          l[r] *= f;
#pragma unroll
          for (int dt = 0; dt < ND; ++dt)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[r][dt][i] *= f;
        }
      }
#pragma unroll
      for (int s = 0; s < JOINT; ++s) {
        Frag<T, COMPUTED<T>> p[R][TS];
#pragma unroll
        for (int r = 0; r < R; ++r) {
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[s][r][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[s][r][i], a.c, -m[r]));
#pragma unroll
          for (int t = 0; t < TS; ++t) p[r][t] = pack_step<T>(sc[s][r], t);
          float sum = 0.f;
#pragma unroll
          for (int i = 0; i < 16; ++i) sum += sc[s][r][i];
          l[r] += sum;
        }
#pragma unroll
        for (int t = 0; t < TS; ++t)
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) {
            const auto v = Tile<T, W, KT>::transposed(vt, j0 + 32 * s, t, 32 * dt, place);
#pragma unroll
            for (int r = 0; r < R; ++r) o[r][dt] = mma(v, p[r][t], o[r][dt]);
          }
      }
    }
    if (k0 + KT < kend) {
      if (NB == 1) __syncthreads();
      if (NB == 2) at = 2 * TILE - at;
      put(lds + at, k0 + KT);
      if (NB == 2 && k0 + 2 * KT < kend) fetch(k0 + 2 * KT);
      __syncthreads();
    }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) l[r] = half_sum(l[r]);

  if constexpr (WK > 1) {  // join the waves along the keys in LDS: [wk][32 rows][W + 4], and their (m, l)
    static_assert(R == 1, "");
    float *os = reinterpret_cast<float*>(lds), *ml = os + (WK - 1) * 32 * (W + 4), *mine = os + ((wk - 1) * 32 + (lane & 31)) * (W + 4) + 4 * half;
    __syncthreads();
    if (half == 0) ml[(wk * 32 + (lane & 31)) * 2] = m[0], ml[(wk * 32 + (lane & 31)) * 2 + 1] = l[0];
    if (wk) {
#pragma unroll
      for (int dt = 0; dt < ND; ++dt)
#pragma unroll
        for (int q = 0; q < 4; ++q)
          *reinterpret_cast<float4*>(mine + 32 * dt + 8 * q) = make_float4(o[0][dt][4 * q], o[0][dt][4 * q + 1], o[0][dt][4 * q + 2], o[0][dt][4 * q + 3]);
    }
    __syncthreads();
    if (wk) return;
    float mm = m[0], f[WK];
#pragma unroll
    for (int x = 1; x < WK; ++x) mm = fmaxf(mm, ml[(x * 32 + (lane & 31)) * 2]);
    l[0] = 0.f;
#pragma unroll
    for (int x = 0; x < WK; ++x) {
      f[x] = __builtin_amdgcn_exp2f(ml[(x * 32 + (lane & 31)) * 2] - mm);
      l[0] += f[x] * ml[(x * 32 + (lane & 31)) * 2 + 1];
    }
    m[0] = mm;
#pragma unroll
    for (int dt = 0; dt < ND; ++dt)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        f32x16& c = o[0][dt];
        float4 v = make_float4(c[4 * q] * f[0], c[4 * q + 1] * f[0], c[4 * q + 2] * f[0], c[4 * q + 3] * f[0]);
#pragma unroll
        for (int x = 1; x < WK; ++x) {
          const float4 u = *reinterpret_cast<const float4*>(os + ((x - 1) * 32 + (lane & 31)) * (W + 4) + 32 * dt + 8 * q + 4 * half);
          v.x += f[x] * u.x, v.y += f[x] * u.y, v.z += f[x] * u.z, v.w += f[x] * u.w;
        }
        c[4 * q] = v.x, c[4 * q + 1] = v.y, c[4 * q + 2] = v.z, c[4 * q + 3] = v.w;
      }
  }
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (row + 32 * r >= a.rows) break;
    const int h = w.hk * a.G + row + 32 * r - query[r] * a.G;
    const long at = (w.b * a.Lq + query[r]) * a.H + h;
    if (part) {  // one of several splits: unnormalised sums and (m, l), joined by mha_fwd_join
      const long n = (long)a.B * a.H * a.Lq;
      store_row<float, ND>(part + (w.split * n + at) * a.D, o[r], 1.f, a.D, lane);
      if (half == 0) {
        float* ml = part + a.nsplit * n * a.D + (w.split * n + at) * 2;
        ml[0] = m[r], ml[1] = l[r];
      }
    } else {
      const float inv = l[r] == 0.f ? 0.f : 1.f / l[r];
      store_row<T, ND>(out + at * a.D, o[r], inv, a.D, lane);
      if (sizeof(T) == 2 && low) store_low<ND>(low + at * a.D, o[r], inv, a.D, lane);
      if (lse && half == 0) lse[(w.b * a.H + h) * a.Lq + query[r]] = l[r] == 0.f ? INFINITY : m[r] + log2f(l[r]);
    }
  }
}

// The splits of a row, a wave per row.  Lane = split for the weights; then D / 4 lanes (LPR, rounded up to a power of two) hold four dimensions
// each, and as many groups of them as the wave has take the splits in turn.  Bound by memory: 256 rows of 16 splits 5 us, 44432 rows of three splits
// (80 MB) 18 to 22 us.
template <typename T, int LPR>
__global__ __launch_bounds__(256) void mha_fwd_join(const float* __restrict__ part, int nsplit, long R, int D, int H, int Lq, T* __restrict__ out, bf16_t* __restrict__ low,
                                                    float* __restrict__ lse) {
  const int lane = threadIdx.x & 63, group = lane / LPR, d = 4 * (lane % LPR);
  const long r = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (r >= R) return;
  const float* ml = part + nsplit * R * D;
  float m = NO_MAX;
  for (int s = lane; s < nsplit; s += 64) m = fmaxf(m, ml[(s * R + r) * 2]);
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
  float l = 0.f;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int s0 = 0; s0 < nsplit; s0 += 64) {
    float f = 0.f;
    if (s0 + lane < nsplit) {
      const float2 u = *reinterpret_cast<const float2*>(ml + ((s0 + lane) * R + r) * 2);
      f = __builtin_amdgcn_exp2f(u.x - m);
      l += f * u.y;
    }
    const int n = min(64, nsplit - s0);
    constexpr int GROUPS = 64 / LPR, AHEAD = 4;
    for (int s = group; s - group < n; s += GROUPS * AHEAD) {
      float4 p[AHEAD];
#pragma unroll
      for (int e = 0; e < AHEAD; ++e)
        p[e] = s + e * GROUPS < n && d < D ? *reinterpret_cast<const float4*>(part + ((s0 + s + e * GROUPS) * R + r) * D + d) : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int e = 0; e < AHEAD; ++e) {
        const float w = __shfl(f, (s + e * GROUPS) & 63, 64);
        v.x += w * p[e].x, v.y += w * p[e].y, v.z += w * p[e].z, v.w += w * p[e].w;
      }
    }
  }
  l = wave_sum(l);
#pragma unroll
  for (int o = LPR; o < 64; o *= 2) v.x += __shfl_xor(v.x, o, 64), v.y += __shfl_xor(v.y, o, 64), v.z += __shfl_xor(v.z, o, 64), v.w += __shfl_xor(v.w, o, 64);
  if (lse && lane == 0) lse[(r / H / Lq * H + r % H) * Lq + r / H % Lq] = l == 0.f ? INFINITY : m + log2f(l);
  if (group || d >= D) return;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  v.x *= inv, v.y *= inv, v.z *= inv, v.w *= inv;
  if constexpr (sizeof(T) == 2) {
    const uint2 h = make_uint2(pack2(v.x, v.y), pack2(v.z, v.w));
    *reinterpret_cast<uint2*>(out + r * D + d) = h;
    if (low) *reinterpret_cast<uint2*>(low + r * D + d) = make_uint2(pack2(v.x - low2(h.x), v.y - high2(h.x)), pack2(v.z - low2(h.y), v.w - high2(h.y)));
  } else {
    *reinterpret_cast<float4*>(out + r * D + d) = v;
  }
}

// A split costs its partial sums, a second launch and the workspace: with bf16 tiles, done quickly, 512 keys are worth that (8 x 8 heads of 64, one query,
// 1000 keys: 14.6 us unsplit, 9.3 and 3.3 with a launch between in splits of 256), with fp32 ones 128 (17 us in splits
// of 128 and 28 of 512; one query, 4000 keys, 8 key heads of 128: 43 and 92; with two waves, below, 29).
// Workgroups at once: of one wave and 48 KB (fp32 heads past 64, few rows) three a CU (8 sequences of up to 20000 keys, 8 heads of 128, one query: 244 us in
// 23 splits, 424 in the 16 of two a CU; all of them of 20000: 292).
Plan plan_fwd(int B, int Lq, int Lk, int H, int Hkv, int D, int causal, int dtype) {
  const bool bf16 = dtype == TATT_T_BF16;
  const int rows = Lq * (H / Hkv), slots = rows > 32 ? slots_of(bf16 ? fwd_waves<bf16_t>(D) : fwd_waves<float>(D)) : !bf16 && D > 64 ? 768 : 512;
  return plan((long)B * Hkv, rows, Lk, bf16 ? 512 : 128, causal, slots, traffic_of(dtype), rows > 32);
}

template <typename T, int DK, int WQ, int R, int WK, int SUB, int JOINT>
int launch_fwd(const MhaArgs& a, T* out, bf16_t* low, float* lse, float* part, hipStream_t st) {
  const size_t join = WK > 1 ? (size_t)((WK - 1) * 32 * (row_width(DK) + 4) + WK * 32 * 2) * 4 : 0;
  const size_t tiles = 2 * Tile<T, row_width(DK), 32 * WK * SUB>::BYTES;
  size_t lds = 2 * tiles <= 64 * 1024 ? 2 * tiles : tiles;
  if (join > lds) lds = join;
  const auto kernel = mha_fwd_kernel<T, DK, WQ, R, WK, SUB, JOINT>;
  if (int rc = prepare_launch(a, kernel, 64 * WQ * WK, lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((long)a.B * a.Hkv * a.nblk * a.nsplit)), dim3(64 * WQ * WK), lds, st, a, out, low, lse, part);
  TATT_LAUNCH_CHECK("mha_fwd");
  return TATT_OK;
}

template <typename T, int DK>
int run_fwd(MhaArgs& a, T* out, bf16_t* low, float* lse, float* part, hipStream_t st) {
  const Plan p = plan_fwd(a.B, a.Lq, a.Lk, a.H, a.Hkv, a.D, a.causal, sizeof(T) == 2 ? TATT_T_BF16 : TATT_T_F32);
  a.nblk = p.nblk, a.nsplit = p.nsplit, a.per_split = p.per_split;
  if (p.nsplit == 1) part = nullptr;
  constexpr int FSUB = sizeof(T) == 4 && DK > 64 ? 1 : 2;
  int rc;
  constexpr int WK = narrow_waves<T>(DK), MORE = sizeof(T) == 4 && DK > 32 ? 2 * WK : WK;
  if (!p.wide) {
    // fp32 tiles of wide heads leave no room for a second buffer beside more waves.  Where workgroups fill the chip, the others fill a wave's waits;
    // where they do not, more waves do (8 x 32 heads of 128, one query: 300 keys 43 us with 1 wave and 30 with 2, 20000 keys 385 and 440)
    const bool filled = (long)a.B * a.Hkv * p.nblk * p.nsplit >= 512;
    rc = filled ? launch_fwd<T, DK, 1, 1, WK, 1, 1>(a, out, low, lse, part, st) : launch_fwd<T, DK, 1, 1, MORE, 1, 1>(a, out, low, lse, part, st);
  } else if constexpr (sizeof(T) == 2 && DK <= 64) {  // 64 rows a wave where that leaves a workgroup to every CU (228 us against 249, above)
    if ((long)a.B * a.Hkv * a.nsplit * cdiv(a.rows, 256) >= 256) {
      a.nblk = cdiv(a.rows, 256);
      rc = launch_fwd<T, DK, 4, 2, 1, 2, 2>(a, out, low, lse, part, st);
    } else {
      rc = launch_fwd<T, DK, 4, 1, 1, FSUB, FSUB>(a, out, low, lse, part, st);
    }
  } else {
    rc = launch_fwd<T, DK, 4, 1, 1, FSUB, FSUB>(a, out, low, lse, part, st);
  }
  if (rc) return rc;
  if (part) {
    const long R = (long)a.B * a.H * a.Lq;
    hipLaunchKernelGGL((mha_fwd_join<T, (DK <= 16 ? 4 : DK <= 32 ? 8 : DK <= 64 ? 16 : 32)>), dim3(cdiv(R, 4)), dim3(256), 0, st, part, a.nsplit, R, a.D, a.H, a.Lq, out, low, lse);
    TATT_LAUNCH_CHECK("mha_fwd_join");
  }
  return TATT_OK;
}

}  // namespace

extern "C" {

size_t tatt_mha_fwd_workspace(int B, int Lq, int Lk, int H, int Hkv, int D, int dtype) {
  if (!sane(B, Lq, Lk, H, Hkv, D)) return 0;
  const int a = plan_fwd(B, Lq, Lk, H, Hkv, D, 0, dtype).nsplit, b = plan_fwd(B, Lq, Lk, H, Hkv, D, 1, dtype).nsplit, n = a > b ? a : b;
  return n == 1 ? 0 : (size_t)n * B * H * Lq * (D + 2);
}

int tatt_mha_fwd(const void* q, const void* k, const void* v, const long* strides, const unsigned char* mask, const long* mask_strides,
                 void* out, void* out_low, float* lse, int B, int Lq, int Lk, int H, int Hkv, int D, float scale, int causal, int dtype, float* workspace,
                 hipStream_t st) {
  MhaArgs a = {};
  if (int rc = fill(a, "tatt_mha_fwd", q, k, v, out, nullptr, strides, mask, mask_strides, B, Lq, Lk, H, Hkv, D, scale, causal, dtype, workspace)) return rc;
  TATT_CHECK_ARG(!out_low || (dtype == TATT_T_BF16 && ((uintptr_t)out_low & 15) == 0), "tatt_mha_fwd: out_low is a 16-byte aligned bf16 tensor beside bf16 ones");
  TATT_CHECK_ARG(workspace || tatt_mha_fwd_workspace(B, Lq, Lk, H, Hkv, D, dtype) == 0, "tatt_mha_fwd: needs tatt_mha_fwd_workspace floats");
  TATT_DISPATCH_TYPE(dtype, TATT_DISPATCH_WIDTH(D, return (run_fwd<T, DK>(a, (T*)out, (bf16_t*)out_low, lse, workspace, st)););;);
  return TATT_OK;
}

}  // extern "C"
