// Attention of any lengths, head counts and head widths up to 128, backward (mha.h has the mathematics and the layouts).
// The probabilities are recomputed from lse, once in the kernel whose rows are queries (dQ, and delta on the way) and once in the one whose rows
// are keys (dK, dV): seven products instead of the five that atomics into dQ would need, and sums in a fixed order.
//
// Bound like the forward pass: to an exponential, dQ has three products and dK and dV four, those of P and dS by two pieces where tensors are bf16 (four and
// six executed).  Measured, at the clock that a busy chip keeps (executed products): 4 x 4096 tokens, 8 heads of 64, bf16: dQ 264 us, 1040 TFLOP/s (64 rows a
// wave; with 32: 289), dK and dV 391 us, 1055 TFLOP/s (tiles of 128 rows; of 64: 402); 16 x 1024, 4 heads of 64, fp32: 151 us (171, fp32 products) and 192 us
// (179); heads of 128 in bf16, 4 x 2816 tokens of 16 heads: 498 us (1043) and 825 (945); 2 x 2777 of 16 / 4: 268 (942) and 408 + 21 for the sum over four
// splits (929), for one causal clip of them 88 + 16 and 117 + 16.
#include "mha.h"

namespace {

// dQ and delta.  WQ waves of 32 R rows; registers hold Q and dO, LDS tiles of 32 SUB keys K and V.
template <typename T, int DK, int WQ, int R, int SUB>
__global__ __launch_bounds__(64 * WQ, dq_waves<T>(DK)) void mha_dq_kernel(MhaArgs a, T* __restrict__ dq, float* __restrict__ part) {
  constexpr int NT = 64 * WQ, W = row_width(DK), ND = (DK + 31) / 32, KT = 32 * SUB, TILE = Tile<T, W, KT>::BYTES;
  constexpr int NS = DK / STEP, TS = 32 / STEP, NB = 4 * TILE <= 64 * 1024 ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wq = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), half = lane >> 5;
  const Where w = where(a);
  const int blk = a.causal ? a.nblk - 1 - w.blk : w.blk;
  const int row0 = blk * 32 * WQ * R, wrow0 = row0 + 32 * wq * R, row = wrow0 + (lane & 31), past = a.Lk - a.Lq;  // and row + 32 r
  const int first_query = wrow0 / a.G;
  const T* kb = (const T*)a.k + w.b * a.ks[0] + w.hk * a.ks[2];
  const T* vb = (const T*)a.v + w.b * a.vs[0] + w.hk * a.vs[2];
  const unsigned char* mb = a.mask ? a.mask + w.b * a.mask_sb : nullptr;

  RowFrags<T, DK> qf[R], gf[R];
  int query[R];
  long at_row[R];  // row of dQ
  float lse[R], delta[R];
  f32x16 o[R][ND];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const bool on = row + 32 * r < a.rows;
    const int safe = min(row + 32 * r, a.rows - 1);
    query[r] = (unsigned)safe / (unsigned)a.G;
    const int h = w.hk * a.G + safe - query[r] * a.G;
    at_row[r] = (w.b * a.Lq + query[r]) * a.H + h;
    qf[r].load((const T*)a.q + w.b * a.qs[0] + query[r] * a.qs[1] + h * a.qs[2], on, a.D, lane);
    gf[r].load((const T*)a.dout + w.b * a.dos[0] + query[r] * a.dos[1] + h * a.dos[2], on, a.D, lane);
    if (a.scale < 0.f) qf[r].negate();
    const T* orow = (const T*)a.out + w.b * a.os[0] + query[r] * a.os[1] + h * a.os[2];
    float d = gf[r].dot(orow, on, a.D, lane);
    if (sizeof(T) == 2 && a.out_low) d += gf[r].dot((const T*)a.out_low + at_row[r] * a.D, on, a.D, lane);
    const long stat = (w.b * a.H + h) * a.Lq + query[r];
    lse[r] = on ? a.lse[stat] : INFINITY;
    delta[r] = lse[r] == INFINITY ? 0.f : half_sum(d);  // a row that sees nothing: whatever dO holds there
    if (on && half == 0 && w.split == 0) a.delta[stat] = delta[r];
    clear(o[r]);
  }

  int kbeg = 0, kend = a.Lk;
  if (a.causal) kend = min(kend, min(a.rows - 1, row0 + 32 * WQ * R - 1) / a.G + past + 1);
  take_split(a, w.split, KT, kbeg, kend);
  if (mb && kend - kbeg > 2 * KT) trim_keys<NT>(mb, a.mask_sl, kbeg, kend, reinterpret_cast<int*>(lds));
  Stage<T, W, KT, NT, true> ks, vs;
  KeyBits<KT> next, now;
  ks.linear(a.ks[1], a.D);
  vs.linear(a.vs[1], a.D);
  auto fetch = [&](int k0) {
    ks.load(kb + k0 * a.ks[1], 0, kend - k0);
    vs.load(vb + k0 * a.vs[1], 0, kend - k0);
    next.load(mb, a.mask_sl, k0, kend, lane);
  };
  auto put = [&](char* to, int k0) {
    next.settle(mb, k0, kend);
    if (mb && !next.full()) ks.hide(next.word);  // a masked key's dS is replaced, its K would still meet that 0
    ks.put(to);
    vs.put(to + TILE);
    now = next;
  };
  typename Tile<T, W, KT>::Lane place(lane);
  int at = 0;
  if (kbeg < kend) {
    fetch(kbeg);
    put(lds, kbeg);
    wait_loads();
    if (NB == 2 && kbeg + KT < kend) fetch(kbeg + KT);
    __syncthreads();
  }
  for (int k0 = kbeg; k0 < kend; k0 += KT) {
    if (NB == 1 && k0 + KT < kend) fetch(k0 + KT);
    const char *kt = lds + at, *vt = kt + TILE;
    place.afresh();
#pragma unroll
    for (int s = 0; s < SUB; ++s) {
      f32x16 sc[R], dp[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        clear(sc[r]);
        clear(dp[r]);
      }
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        const auto k = Tile<T, W, KT>::rows(kt, 32 * s, t, place);
#pragma unroll
        for (int r = 0; r < R; ++r) sc[r] = mma(k, qf[r].f[t], sc[r]);
      }
#pragma unroll
      for (int t = 0; t < NS; ++t) {
        const auto v = Tile<T, W, KT>::rows(vt, 32 * s, t, place);
#pragma unroll
        for (int r = 0; r < R; ++r) dp[r] = mma(v, gf[r].f[t], dp[r]);
      }
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int i = 0; i < 16; ++i) sc[r][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[r][i], a.c, -lse[r])) * (dp[r][i] - delta[r]);
      if (!now.full() || (a.causal && first_query + past < k0 + 32 * s + 31)) {
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const unsigned see = (now.of(32 * s) & (a.causal ? bits_to(query[r] + past - k0 - 32 * s) : ~0u)) >> (4 * half);
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[r][i] = see >> acc_row(i) & 1 ? sc[r][i] : 0.f;
        }
      }
      Frag<T, COMPUTED<T>> p[R][TS];
#pragma unroll
      for (int r = 0; r < R; ++r)
#pragma unroll
        for (int t = 0; t < TS; ++t) p[r][t] = pack_step<T>(sc[r], t);
#pragma unroll
      for (int t = 0; t < TS; ++t)
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
          const auto k = Tile<T, W, KT>::transposed(kt, 32 * s, t, 32 * dt, place);
#pragma unroll
          for (int r = 0; r < R; ++r) o[r][dt] = mma(k, p[r][t], o[r][dt]);
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
  for (int r = 0; r < R; ++r) {
    if (row + 32 * r >= a.rows) break;
    if (lse[r] == INFINITY) clear(o[r]);
    if (part)
      store_row<float, ND>(part + (w.split * (long)a.B * a.H * a.Lq + at_row[r]) * a.D, o[r], a.scale, a.D, lane);
    else
      store_row<T, ND>(dq + at_row[r] * a.D, o[r], a.scale, a.D, lane);
  }
}

// dK and dV.  WN waves along the keys (32 each) x WR along the rows; LDS holds tiles of 32 WR SUB rows of Q and dO, and their lse and delta.
template <typename T, int DK, int WN, int WR, int SUB>
__global__ __launch_bounds__(64 * WN * WR, dkv_waves<T>(DK)) void mha_dkv_kernel(MhaArgs a, T* __restrict__ dk, T* __restrict__ dv, float* __restrict__ part) {
  constexpr int NT = 64 * WN * WR, W = row_width(DK), ND = (DK + 31) / 32, RT = 32 * WR * SUB, TILE = Tile<T, W, RT>::BYTES, BUF = 2 * TILE + 2 * RT * 4;
  constexpr int NS = DK / STEP, TS = 32 / STEP, NB = 4 * TILE <= 64 * 1024 ? 2 : 1;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), wn = wave % WN, wr = wave / WN, half = lane >> 5;
  const Where w = where(a);
  const int key0 = w.blk * 32 * WN, key = key0 + 32 * wn + (lane & 31), past = a.Lk - a.Lq;
  const bool on = key < a.Lk && !(a.mask && a.mask[w.b * a.mask_sb + (long)key * a.mask_sl]);
  const long key_safe = min(key, a.Lk - 1);
  RowFrags<T, DK> kf, vf;
  kf.load((const T*)a.k + w.b * a.ks[0] + key_safe * a.ks[1] + w.hk * a.ks[2], on, a.D, lane);
  vf.load((const T*)a.v + w.b * a.vs[0] + key_safe * a.vs[1] + w.hk * a.vs[2], on, a.D, lane);
  if (a.scale < 0.f) kf.negate();
  const T* qb = (const T*)a.q + w.b * a.qs[0] + w.hk * a.G * a.qs[2];
  const T* gb = (const T*)a.dout + w.b * a.dos[0] + w.hk * a.G * a.dos[2];
  const float* lse = a.lse + (w.b * a.H + w.hk * a.G) * a.Lq;
  const float* delta = a.delta + (w.b * a.H + w.hk * a.G) * a.Lq;

  // causal: this key is seen from row G (key - past) on; rows before the first query that sees an unmasked key hold what they like
  const int first_row = a.causal ? a.G * max(0, key - past) : 0;
  const int all_rows = a.causal ? a.G * max(0, key0 + 32 * wn + 31 - past) : 0;  // from here on every key of the wave is seen
  const int first_seen = a.causal && a.mask ? first_key<NT>(a.mask + w.b * a.mask_sb, a.mask_sl, min(a.Lk, key0 + 32 * WN), reinterpret_cast<int*>(lds)) : 0;
  const int empty_rows = a.causal ? a.G * max(0, first_seen - past) : 0;
  const bool whole = __all(on);
  int rbeg = a.causal ? a.G * max(0, key0 - past) / RT * RT : 0, rend = a.rows;
  take_split(a, w.split, RT, rbeg, rend);
  f32x16 ok[ND], ov[ND];
  clear(ok);
  clear(ov);
  const bool any = __syncthreads_or(on);  // nothing to do where every key of the block is masked

  Stage<T, W, RT, NT, false> qs, gs;
  float l0 = 0.f, d0 = 0.f;
  const bool steady = 32 % a.G == 0;  // a tile's rows are the same (query, head) places from its first query on
  auto places = [&](int r0) {
    const int i0 = r0 / a.G;
    qs.places([&](int r) { return row_offset(r0 + r, a.G, a.qs[1], a.qs[2]) - i0 * a.qs[1]; }, a.D);
    gs.places([&](int r) { return row_offset(r0 + r, a.G, a.dos[1], a.dos[2]) - i0 * a.dos[1]; }, a.D);
  };
  auto fetch = [&](int r0) {
    if (!steady) places(r0);
    const int i0 = r0 / a.G;
    qs.load(qb + i0 * a.qs[1], empty_rows - r0, rend - r0);
    gs.load(gb + i0 * a.dos[1], empty_rows - r0, rend - r0);
    static_assert(RT <= NT, "");
    if (threadIdx.x < RT) {
      const int r = r0 + threadIdx.x;
      const bool there = r < rend && r >= empty_rows;
      const int i = (unsigned)min(r, a.rows - 1) / (unsigned)a.G;
      const long at = (long)(min(r, a.rows - 1) - i * a.G) * a.Lq + i;
      l0 = there ? lse[at] : INFINITY;
      d0 = there ? delta[at] : 0.f;
    }
  };
  auto put = [&](char* to) {
    qs.put(to);
    gs.put(to + TILE);
    float* ls = reinterpret_cast<float*>(to + 2 * TILE);
    if (threadIdx.x < RT) ls[threadIdx.x] = l0, ls[RT + threadIdx.x] = d0;
  };
  typename Tile<T, W, RT>::Lane place(lane);
  if (any && rbeg < rend) {
    int buf = 0;
    if (steady) places(0);
    fetch(rbeg);
    put(lds);
    wait_loads();
    if (NB == 2 && rbeg + RT < rend) fetch(rbeg + RT);
    __syncthreads();
    for (int r0 = rbeg; r0 < rend; r0 += RT) {
      if (NB == 1 && r0 + RT < rend) fetch(r0 + RT);
      const char *qt = lds + buf, *gt = qt + TILE;
      const float* ls = reinterpret_cast<const float*>(qt + 2 * TILE);
      place.afresh();
#pragma unroll
      for (int s = 0; s < SUB; ++s) {
        const int at = 32 * (wr * SUB + s);
        f32x16 sc, dp;
        clear(sc);
        clear(dp);
#pragma unroll
        for (int t = 0; t < NS; ++t) sc = mma(Tile<T, W, RT>::rows(qt, at, t, place), kf.f[t], sc);
#pragma unroll
        for (int t = 0; t < NS; ++t) dp = mma(Tile<T, W, RT>::rows(gt, at, t, place), vf.f[t], dp);
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 lq = *reinterpret_cast<const f32x4*>(ls + at + 8 * q + 4 * half);
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[4 * q + e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[4 * q + e], a.c, -lq[e]));
        }
        if (!whole || r0 + at < all_rows) {
          const int hidden = on ? first_row - r0 - at - 4 * half : 32;  // accumulator rows below this are causally hidden
#pragma unroll
          for (int i = 0; i < 16; ++i) sc[i] = acc_row(i) >= hidden ? sc[i] : 0.f;
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const f32x4 dq = *reinterpret_cast<const f32x4*>(ls + RT + at + 8 * q + 4 * half);
#pragma unroll
          for (int e = 0; e < 4; ++e) dp[4 * q + e] = sc[4 * q + e] * (dp[4 * q + e] - dq[e]);
        }
#pragma unroll
        for (int t = 0; t < TS; ++t) {
          const auto p = pack_step<T>(sc, t);
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) ov[dt] = mma(Tile<T, W, RT>::transposed(gt, at, t, 32 * dt, place), p, ov[dt]);
        }
#pragma unroll
        for (int t = 0; t < TS; ++t) {
          const auto p = pack_step<T>(dp, t);
#pragma unroll
          for (int dt = 0; dt < ND; ++dt) ok[dt] = mma(Tile<T, W, RT>::transposed(qt, at, t, 32 * dt, place), p, ok[dt]);
        }
      }
      if (r0 + RT < rend) {
        if (NB == 1) __syncthreads();
        if (NB == 2) buf = BUF - buf;
        put(lds + buf);
        if (NB == 2 && r0 + 2 * RT < rend) fetch(r0 + 2 * RT);
        __syncthreads();
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
    store_row<float, ND>(part + ((w.split * 2L) * R + r) * a.D, ok, a.scale, a.D, lane);
    store_row<float, ND>(part + ((w.split * 2L + 1) * R + r) * a.D, ov, 1.f, a.D, lane);
  } else {
    store_row<T, ND>(dk + r * a.D, ok, a.scale, a.D, lane);
    store_row<T, ND>(dv + r * a.D, ov, 1.f, a.D, lane);
  }
}

// y[i] = sum over splits of part[split][i] in split order; two tensors of n values each where y2.  Bound by memory (six splits of 23 MB: 28 us)
template <typename T>
__global__ __launch_bounds__(256) void mha_sum_kernel(const float* __restrict__ part, int nsplit, long n, T* __restrict__ y, T* __restrict__ y2) {
  const long i = (long)blockIdx.x * 256 + threadIdx.x, all = y2 ? 2 * n : n;
  if (i >= all) return;
  float s = 0.f;
  for (int k = 0; k < nsplit; ++k) s += part[k * all + i];
  (i < n ? y : y2)[i < n ? i : i - n] = from_f32<T>(s);
}

// Splits of no less than 256 (2 x 1024 x 1024, 4 heads of 64: kernels fp32 69 us against 103 with 512, bf16 41 against 51; with 128 the same)
Plan plan_dq(int B, int Lq, int Lk, int H, int Hkv, int D, int causal, int dtype) {
  return plan((long)B * Hkv, Lq * (H / Hkv), Lk, 256, causal, slots_of(dtype == TATT_T_BF16 ? dq_waves<bf16_t>(D) : dq_waves<float>(D > 32 ? 64 : D)), traffic_of(dtype), true);
}
Plan plan_dkv(int B, int Lq, int Lk, int H, int Hkv, int D, int causal, int dtype) {
  return plan((long)B * Hkv, Lk, Lq * (H / Hkv), 256, causal, slots_of(dtype == TATT_T_BF16 ? dkv_waves<bf16_t>(D) : dkv_waves<float>(D > 64 ? D : D > 32 ? 64 : D)), traffic_of(dtype), Lk > 32);
}

template <typename T, int DK, int R, int SUB>
int launch_dq(const MhaArgs& a, T* dq, float* part, hipStream_t st) {
  const size_t tiles = 2 * Tile<T, row_width(DK), 32 * SUB>::BYTES, lds = 2 * tiles <= 64 * 1024 ? 2 * tiles : tiles;
  const auto kernel = mha_dq_kernel<T, DK, 4, R, SUB>;
  if (int rc = prepare_launch(a, kernel, 256, lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)((long)a.B * a.Hkv * a.nblk * a.nsplit)), dim3(256), lds, st, a, dq, part);
  TATT_LAUNCH_CHECK("mha_dq");
  return TATT_OK;
}

template <typename T, int DK, int WN, int WR, int SUB>
int launch_dkv(const MhaArgs& a, T* dk, T* dv, float* part, hipStream_t st) {
  const size_t tiles = 2 * Tile<T, row_width(DK), 32 * WR * SUB>::BYTES, buf = tiles + 2 * 32 * WR * SUB * 4, join = WR > 1 ? (size_t)WN * 32 * (row_width(DK) + 4) * 4 : 0;
  size_t lds = 2 * tiles <= 64 * 1024 ? 2 * buf : buf;
  if (join > lds) lds = join;
  if (int rc = prepare_launch(a, mha_dkv_kernel<T, DK, WN, WR, SUB>, 64 * WN * WR, lds)) return rc;
  hipLaunchKernelGGL((mha_dkv_kernel<T, DK, WN, WR, SUB>), dim3((unsigned)((long)a.B * a.Hkv * a.nblk * a.nsplit)), dim3(64 * WN * WR), lds, st, a, dk, dv, part);
  TATT_LAUNCH_CHECK("mha_dkv");
  return TATT_OK;
}

template <typename T, int DK>
int run_bwd(MhaArgs& a, T* dq, T* dk, T* dv, float* part, hipStream_t st) {
  constexpr int dtype = sizeof(T) == 2 ? TATT_T_BF16 : TATT_T_F32;
  Plan p = plan_dq(a.B, a.Lq, a.Lk, a.H, a.Hkv, a.D, a.causal, dtype);
  a.nsplit = p.nsplit, a.per_split = p.per_split;
  float* q_part = a.nsplit > 1 ? part : nullptr;
  int rc = -1;
  if constexpr (sizeof(T) == 2 && DK <= 64)  // 64 rows a wave where that leaves a workgroup to every CU
    if ((long)a.B * a.Hkv * a.nsplit * cdiv(a.rows, 256) >= 256) {
      a.nblk = cdiv(a.rows, 256);
      rc = launch_dq<T, DK, 2, 2>(a, dq, q_part, st);
    }
  if (rc < 0) {
    a.nblk = cdiv(a.rows, 128);
    // tiles of 64 keys (2 x 2777, 16 / 4 heads of 128: 268 us against 277 with 32), of 32 where three pieces of them would not fit
    rc = launch_dq<T, DK, 1, (DK > 64 && sizeof(T) == 4 ? 1 : 2)>(a, dq, q_part, st);
  }
  if (rc) return rc;
  if (q_part) {
    const long n = (long)a.B * a.H * a.Lq * a.D;
    hipLaunchKernelGGL(mha_sum_kernel<T>, dim3(cdiv(n, 256)), dim3(256), 0, st, part, a.nsplit, n, dq, (T*)nullptr);
    TATT_LAUNCH_CHECK("mha_sum");
  }
  p = plan_dkv(a.B, a.Lq, a.Lk, a.H, a.Hkv, a.D, a.causal, dtype);
  a.nblk = p.nblk, a.nsplit = p.nsplit, a.per_split = p.per_split;
  float* kv_part = a.nsplit > 1 ? part : nullptr;
  // Few keys: waves along the rows.  fp32 heads wider than 64 have no registers for that, three of four waves that only bring tiles are better
  // (26 keys, 16 x 1024 queries, 4 heads of 128: 218 us against 361 the pass; 8 heads of 64 with 4 waves 35 us, with 2 that leave room for a second
  // buffer 45)
  if constexpr (sizeof(T) == 4 && DK > 64)
    rc = launch_dkv<T, DK, 4, 1, 1>(a, dk, dv, kv_part, st);
  else if (p.wide)  // row tiles of 128 for narrow bf16 heads, 64 for wide ones (2 x 2777, 16 / 4 of 128: 408 us against 498 with 32), 32 in fp32: what two buffers leave room for
    rc = launch_dkv<T, DK, 4, 1, (sizeof(T) == 4 ? 1 : DK > 64 ? 2 : 4)>(a, dk, dv, kv_part, st);
  else
    rc = launch_dkv<T, DK, 1, (sizeof(T) == 4 ? 4 : narrow_waves<T>(DK)), 1>(a, dk, dv, kv_part, st);
  if (rc) return rc;
  if (kv_part) {
    const long n = (long)a.B * a.Hkv * a.Lk * a.D;
    hipLaunchKernelGGL(mha_sum_kernel<T>, dim3(cdiv(2 * n, 256)), dim3(256), 0, st, part, a.nsplit, n, dk, dv);
    TATT_LAUNCH_CHECK("mha_sum");
  }
  return TATT_OK;
}

}  // namespace

extern "C" {

size_t tatt_mha_bwd_workspace(int B, int Lq, int Lk, int H, int Hkv, int D, int dtype) {
  if (!sane(B, Lq, Lk, H, Hkv, D)) return 0;
  size_t most = 0;  // of either kernel, causal or not
  for (int causal = 0; causal < 2; ++causal) {
    const size_t p = plan_dq(B, Lq, Lk, H, Hkv, D, causal, dtype).nsplit, q = plan_dkv(B, Lq, Lk, H, Hkv, D, causal, dtype).nsplit;
    const size_t a = p == 1 ? 0 : p * B * H * Lq * D, b = q == 1 ? 0 : q * 2 * B * Hkv * Lk * D;
    most = a > most ? a : most;
    most = b > most ? b : most;
  }
  return ((size_t)B * H * Lq + 3) / 4 * 4 + most;  // delta, then the partial sums of one kernel at a time
}

int tatt_mha_bwd(const void* q, const void* k, const void* v, const long* strides, const unsigned char* mask, const long* mask_strides,
                 const void* out, const void* out_low, const void* dout, const float* lse, void* dq, void* dk, void* dv, int B, int Lq, int Lk, int H, int Hkv, int D,
                 float scale, int causal, int dtype, float* workspace, hipStream_t st) {
  MhaArgs a = {};
  TATT_CHECK_ARG(out && dout && lse && dq && dk && dv && workspace, "tatt_mha_bwd: bad arguments (workspace: tatt_mha_bwd_workspace floats)");
  if (int rc = fill(a, "tatt_mha_bwd", q, k, v, out, dout, strides, mask, mask_strides, B, Lq, Lk, H, Hkv, D, scale, causal, dtype, workspace)) return rc;
  TATT_CHECK_ARG((((uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) == 0, "tatt_mha_bwd: dq, dk and dv are 16-byte aligned");
  TATT_CHECK_ARG(!out_low || (dtype == TATT_T_BF16 && ((uintptr_t)out_low & 15) == 0), "tatt_mha_bwd: out_low is a 16-byte aligned bf16 tensor beside bf16 ones");
  a.lse = lse, a.delta = workspace, a.out_low = out_low;
  float* part = workspace + ((size_t)B * H * Lq + 3) / 4 * 4;
  TATT_DISPATCH_TYPE(dtype, TATT_DISPATCH_WIDTH(D, return (run_bwd<T, DK>(a, (T*)dq, (T*)dk, (T*)dv, part, st)););;);
  return TATT_OK;
}

}  // extern "C"
