// LayerNorm over rows of any width, forward and backward (tatt_ln_* in norm.hip is the 64-channel form with dropout in front).
//   s = x (+ res, rounded to the type: the sum is an output, and what is normalised is what was stored)
//   y = (s - mu) rstd * gamma + beta          stat[row] = (mu, rstd)
//   g = dy * gamma,  xhat = (s - mu) rstd,  ds = rstd (g - mean(g) - xhat mean(g xhat)) (+ dsum)
//   dgamma = sum over rows of dy * xhat,  dbeta = sum over rows of dy
// Statistics, sums and parameter gradients are fp32 whatever the tensors' type (sums over the rows of several threads 64 bits).
// Bound by memory, so every tensor is touched once: a row lives in the registers of its TPR threads as NV 16-byte chunks each (mean, then the
// variance of the differences: two passes over registers, no difference of squares), and the backward pass takes dx and the sums over
// rows from the same registers, its threads keeping their columns from row to row.
// Measured: 8192 x 4096, bf16, residual: 49 us forward (268 MB, 5.5 TB/s, some of it from the last cache), 69 backward (268 MB, 3.9 TB/s; the sums over rows
// take registers and with them loads in flight), 11 for the last sum over the workgroups; 65536 x 64, fp32: 8.3, 12 and 7 us.
// Rows that are no whole number of 16-byte chunks, or start at no such border, are read and written element by element, a lane's neighbours 16 bytes on:
// 8192 x 4095, bf16, residual: 255 us forward and 369 backward; 65536 x 63: 18 and 22 us in either type; 8192 x 1001, fp32: 31 and 43 (of 1000: 14 and 22).
// A row has as many threads as it has 16-byte chunks, up to a wave and then up to 256 (two chunks a thread from 128 chunks on), so that narrow rows
// share a wave and wide ones keep their loads in flight; past 2048 chunks a wave reads its row again for each sum (1024 x 20000,
// fp32: 468 us forward, 258 + 67 + 48 backward).
#include "token_types.h"

namespace {

template <typename T, int NV>
struct Row {
  uint4 c[NV];
  template <int TPR>
  __device__ __forceinline__ void load(const T* row, int t, int C, int vec) {
#pragma unroll
    for (int n = 0; n < NV; ++n) c[n] = load_chunk<T>(row, n * TPR + t, C, vec);
  }
  __device__ __forceinline__ void get(int n, float (&f)[per_chunk<T>()]) const {
    T e[per_chunk<T>()];
    memcpy(e, &c[n], 16);
#pragma unroll
    for (int i = 0; i < per_chunk<T>(); ++i) f[i] = to_f32(e[i]);
  }
};

// chunk c of a row from floats, rounded to T
template <typename T>
__device__ __forceinline__ uint4 round_chunk(const float (&f)[per_chunk<T>()]) {
  uint4 u;
  if constexpr (sizeof(T) == 4) {
    u = make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    const uint2 a = tatt_pack_bf16x4(f[0], f[1], f[2], f[3]), b = tatt_pack_bf16x4(f[4], f[5], f[6], f[7]);
    u = make_uint4(a.x, a.y, b.x, b.y);
  }
  return u;
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* row, int c, int C, int vec, uint4 u) {
  constexpr int E = per_chunk<T>();
  if (vec) {
    if (c * E < C) *reinterpret_cast<uint4*>(row + c * E) = u;
  } else {
    T t[E];
    memcpy(t, &u, 16);
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (c * E + e < C) row[c * E + e] = t[e];
  }
}

// whether element e of chunk c is within the row (`vec`: chunks are whole)
__device__ __forceinline__ bool within(int c, int e, int E, int C, int vec) { return vec ? c * E < C : c * E + e < C; }

// the parameters of chunk c (`none` where there are none), zeros behind the row's end
template <int E>
__device__ __forceinline__ void load_params(const float* p, int c, int C, float none, int vec, float (&f)[E]) {
  if (p && vec) {
#pragma unroll
    for (int e = 0; e < E; e += 4) {
      const float4 v = c * E < C ? *reinterpret_cast<const float4*>(p + c * E + e) : make_float4(0.f, 0.f, 0.f, 0.f);
      f[e] = v.x, f[e + 1] = v.y, f[e + 2] = v.z, f[e + 3] = v.w;
    }
    return;
  }
#pragma unroll
  for (int e = 0; e < E; ++e) f[e] = within(c, e, E, C, vec) ? (p ? p[c * E + e] : none) : 0.f;
}

// (a, b) summed over the TPR threads of a row.  TPR >= 256: over the workgroup, red = 32 floats of LDS
template <int TPR>
__device__ __forceinline__ float2 row_sum(float a, float b, float* red) {
#pragma unroll
  for (int o = (TPR > 64 ? 32 : TPR / 2); o > 0; o >>= 1) {
    a += __shfl_xor(a, o, 64);
    b += __shfl_xor(b, o, 64);
  }
  if constexpr (TPR > 64) {
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = a, red[16 + (threadIdx.x >> 6)] = b;
    __syncthreads();
    a = b = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) a += red[i], b += red[16 + i];
  }
  return make_float2(a, b);
}

// threads of a workgroup
constexpr int block_of(int tpr) { return tpr > 256 ? tpr : 256; }

template <typename T, int TPR, int NV, int vec>
__global__ __launch_bounds__(block_of(TPR)) void layernorm_fwd_kernel(const T* __restrict__ x, long ldx, const T* __restrict__ res, long ldr,
                                                            const float* __restrict__ gamma, const float* __restrict__ beta, T* __restrict__ sum,
                                                            T* __restrict__ y, float* __restrict__ stat, long rows, int C, float eps) {
  constexpr int E = per_chunk<T>(), PER = block_of(TPR) / TPR;
  __shared__ float red[32];
  const int t = threadIdx.x % TPR;
  for (long r0 = (long)blockIdx.x * PER; r0 < rows; r0 += (long)gridDim.x * PER) {
    const long row = r0 + threadIdx.x / TPR;
    const bool on = row < rows;
    const long at = on ? row : rows - 1;
    Row<T, NV> s;
    s.template load<TPR>(x + at * ldx, t, C, vec);
    float f[E], a = 0.f, b = 0.f;
    if (res) {
      Row<T, NV> r;
      r.template load<TPR>(res + at * ldr, t, C, vec);
      float g[E];
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        s.get(n, f);
        r.get(n, g);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] += g[e];
        s.c[n] = round_chunk<T>(f);
        if (on) store_chunk<T>(sum + at * C, n * TPR + t, C, vec, s.c[n]);
      }
    }
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      s.get(n, f);
#pragma unroll
      for (int e = 0; e < E; ++e) a += f[e];
    }
    const float mu = row_sum<TPR>(a, 0.f, red).x / C;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      s.get(n, f);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float d = within(n * TPR + t, e, E, C, vec) ? f[e] - mu : 0.f;
        b += d * d;
      }
    }
    const float rstd = rsqrtf(row_sum<TPR>(b, 0.f, red).x / C + eps);
    if (!on) continue;
    if (stat && t == 0) *reinterpret_cast<float2*>(stat + 2 * row) = make_float2(mu, rstd);
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      float w[E], z[E];
      load_params<E>(gamma, n * TPR + t, C, 1.f, vec, w);
      load_params<E>(beta, n * TPR + t, C, 0.f, vec, z);
      s.get(n, f);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = (f[e] - mu) * rstd * w[e] + z[e];
      store_chunk<T>(y + row * C, n * TPR + t, C, vec, round_chunk<T>(f));
    }
  }
}

// dx, and partial[block][2][C] of (dgamma, dbeta) where PARAMS
template <typename T, int TPR, int NV, int vec, bool PARAMS>
__global__ __launch_bounds__(block_of(TPR)) void layernorm_bwd_kernel(const T* __restrict__ s, long lds, const T* __restrict__ dy, long lddy, const T* __restrict__ dsum,
                                                            long ldds, const float* __restrict__ gamma, const float* __restrict__ stat,
                                                            T* __restrict__ dx, float* __restrict__ partial, long rows, int C) {
  constexpr int E = per_chunk<T>(), PER = block_of(TPR) / TPR;
  __shared__ float red[32];
  __shared__ float cols[PARAMS && PER > 1 ? 256 * E : 1];  // one chunk of every thread at a time
  const int t = threadIdx.x % TPR;
  float dg[NV][E], db[NV][E];
#pragma unroll
  for (int n = 0; n < NV; ++n)
#pragma unroll
    for (int e = 0; e < E; ++e) dg[n][e] = db[n][e] = 0.f;
  for (long r0 = (long)blockIdx.x * PER; r0 < rows; r0 += (long)gridDim.x * PER) {
    const long row = r0 + threadIdx.x / TPR;
    const bool on = row < rows;
    const long at = on ? row : rows - 1;
    Row<T, NV> x, d;
    x.template load<TPR>(s + at * lds, t, C, vec);
    d.template load<TPR>(dy + at * lddy, t, C, vec);
    const float2 st = *reinterpret_cast<const float2*>(stat + 2 * at);
    float a = 0.f, b = 0.f, f[E], g[E], w[E];
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      x.get(n, f);
      d.get(n, g);
      load_params<E>(gamma, n * TPR + t, C, 1.f, vec, w);
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float h = (f[e] - st.x) * st.y;
        if (PARAMS && on) dg[n][e] += g[e] * h, db[n][e] += g[e];
        a += g[e] * w[e];
        b += g[e] * w[e] * h;
      }
    }
    const float2 ab = row_sum<TPR>(a, b, red);
    a = ab.x / C;
    b = ab.y / C;
    if (!on) continue;
#pragma unroll
    for (int n = 0; n < NV; ++n) {
      x.get(n, f);
      d.get(n, g);
      load_params<E>(gamma, n * TPR + t, C, 1.f, vec, w);
#pragma unroll
      for (int e = 0; e < E; ++e) f[e] = st.y * (g[e] * w[e] - a - (f[e] - st.x) * st.y * b);
      if (dsum) {
        const uint4 u = load_chunk<T>(dsum + row * ldds, n * TPR + t, C, vec);
        T r[E];
        memcpy(r, &u, 16);
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] += to_f32(r[e]);
      }
      store_chunk<T>(dx + row * C, n * TPR + t, C, vec, round_chunk<T>(f));
    }
  }
  if constexpr (PARAMS) {
    float* p = partial + (long)blockIdx.x * 2 * C;
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
      for (int n = 0; n < NV; ++n) {
        if constexpr (PER > 1) {  // the rows of a pass, in order
          __syncthreads();
#pragma unroll
          for (int e = 0; e < E; ++e) cols[e * 256 + threadIdx.x] = which ? db[n][e] : dg[n][e];
          __syncthreads();
          for (int i = threadIdx.x; i < TPR * E; i += 256) {
            const int c = (n * TPR + i / E) * E + i % E;
            double v = 0.;
#pragma unroll
            for (int r = 0; r < PER; ++r) v += cols[(i % E) * 256 + r * TPR + i / E];
            if (c < C) p[which * C + c] = (float)v;
          }
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e) {
            const int c = (n * TPR + t) * E + e;
            if (c < C) p[which * C + c] = which ? db[n][e] : dg[n][e];
          }
        }
      }
  }
}

// ---- rows too wide for the registers of a workgroup: a wave per row, read again for each of its sums ---------------------------------------
template <typename T>
__global__ __launch_bounds__(256) void layernorm_fwd_wide(const T* __restrict__ x, long ldx, const T* __restrict__ res, long ldr,
                                                          const float* __restrict__ gamma, const float* __restrict__ beta, T* sum, T* __restrict__ y,
                                                          float* __restrict__ stat, long rows, int C, float eps) {
  const int lane = threadIdx.x & 63;
  for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (long)gridDim.x * 4) {
    const T* s = x + row * ldx;
    float t = 0.f;
    if (res) {
      T* so = sum + row * C;
      for (int c = lane; c < C; c += 64) {
        so[c] = from_f32<T>(to_f32(s[c]) + to_f32(res[row * ldr + c]));
        t += to_f32(so[c]);
      }
      s = so;
    } else {
      for (int c = lane; c < C; c += 64) t += to_f32(s[c]);
    }
    const float mu = wave_sum(t) / C;
    float v = 0.f;
    for (int c = lane; c < C; c += 64) {
      const float d = to_f32(s[c]) - mu;
      v += d * d;
    }
    const float rstd = rsqrtf(wave_sum(v) / C + eps);
    if (stat && lane == 0) {
      stat[2 * row] = mu;
      stat[2 * row + 1] = rstd;
    }
    for (int c = lane; c < C; c += 64) {
      const float h = (to_f32(s[c]) - mu) * rstd;
      y[row * C + c] = from_f32<T>((gamma ? h * gamma[c] : h) + (beta ? beta[c] : 0.f));
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void layernorm_dx_wide(const T* __restrict__ s, long lds, const T* __restrict__ dy, long lddy, const T* __restrict__ dsum,
                                                         long ldds, const float* __restrict__ gamma, const float* __restrict__ stat, T* __restrict__ dx,
                                                         long rows, int C) {
  const int lane = threadIdx.x & 63;
  for (long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6); row < rows; row += (long)gridDim.x * 4) {
    const float mu = stat[2 * row], rstd = stat[2 * row + 1];
    float a = 0.f, b = 0.f;
    for (int c = lane; c < C; c += 64) {
      const float g = to_f32(dy[row * lddy + c]) * (gamma ? gamma[c] : 1.f), h = (to_f32(s[row * lds + c]) - mu) * rstd;
      a += g;
      b += g * h;
    }
    a = wave_sum(a) / C;
    b = wave_sum(b) / C;
    for (int c = lane; c < C; c += 64) {
      const float g = to_f32(dy[row * lddy + c]) * (gamma ? gamma[c] : 1.f), h = (to_f32(s[row * lds + c]) - mu) * rstd;
      const float d = rstd * (g - a - h * b);
      dx[row * C + c] = from_f32<T>(dsum ? d + to_f32(dsum[row * ldds + c]) : d);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void layernorm_params_wide(const T* __restrict__ s, long lds, const T* __restrict__ dy, long lddy,
                                                             const float* __restrict__ stat, float* __restrict__ partial, long rows, int C) {
  for (int c = blockIdx.y * 256 + threadIdx.x; c < C; c += gridDim.y * 256) {
    float dg = 0.f, db = 0.f;
    for (long r = blockIdx.x; r < rows; r += gridDim.x) {
      const float d = to_f32(dy[r * lddy + c]);
      dg += d * ((to_f32(s[r * lds + c]) - stat[2 * r]) * stat[2 * r + 1]);
      db += d;
    }
    partial[(blockIdx.x * 2L) * C + c] = dg;
    partial[(blockIdx.x * 2L + 1) * C + c] = db;
  }
}

// partial[block][2][C] -> dgamma, dbeta, in block order: 16 columns of a workgroup by 16 threads each, four loads of a thread in flight.  Sums over
// rows are fp32 only within a thread; past it their roundings would be most of the error (65536 x 64: 1.5e-7 of the result, 7e-8 so).
__global__ __launch_bounds__(256) void layernorm_params_final(const float* __restrict__ partial, int nblk, int C,
                                                              float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ double red[256];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15);
  float* dst = blockIdx.y ? dbeta : dgamma;
  if (!dst) return;
  const float* p = partial + (long)blockIdx.y * C + c;
  double s[4] = {0., 0., 0., 0.};
  int b = threadIdx.x >> 4;
  if (c < C) {
    for (; b + 48 < nblk; b += 64) {
      float t[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) t[i] = p[(b + 16 * i) * 2L * C];
#pragma unroll
      for (int i = 0; i < 4; ++i) s[i] += t[i];
    }
    for (; b < nblk; b += 16) s[0] += p[b * 2L * C];
  }
  red[threadIdx.x] = (s[0] + s[1]) + (s[2] + s[3]);
  __syncthreads();
  if (threadIdx.x >= 16 || c >= C) return;
  double v = 0.;
  for (int j = 0; j < 16; ++j) v += red[16 * j + threadIdx.x];
  dst[c] = (float)v;
}

// how a row of C elements is held: threads of a row and 16-byte chunks of a thread (0: by none, the wide kernels)
struct Held {
  int tpr, nv;
};
Held held(int C, int per_chunk) {
  const int chunks = cdiv(C, per_chunk);
  if (chunks <= 8) return {8, 1};
  if (chunks <= 16) return {16, 1};
  if (chunks <= 32) return {32, 1};
  if (chunks <= 64) return {64, 1};
  if (chunks <= 128) return {64, 2};
  if (chunks <= 256) return {256, 1};
  if (chunks <= 512) return {256, 2};
  if (chunks <= 1024) return {512, 2};
  if (chunks <= 2048) return {1024, 2};
  return {0, 0};
}
#define TATT_DISPATCH_HELD(h, ...)                                                           \
  do {                                                                                       \
    if ((h).tpr == 8) { constexpr int TPR = 8, NV = 1; __VA_ARGS__ }                         \
    else if ((h).tpr == 16) { constexpr int TPR = 16, NV = 1; __VA_ARGS__ }                  \
    else if ((h).tpr == 32) { constexpr int TPR = 32, NV = 1; __VA_ARGS__ }                  \
    else if ((h).tpr == 64 && (h).nv == 1) { constexpr int TPR = 64, NV = 1; __VA_ARGS__ }   \
    else if ((h).tpr == 64) { constexpr int TPR = 64, NV = 2; __VA_ARGS__ }                  \
    else if ((h).tpr == 256 && (h).nv == 1) { constexpr int TPR = 256, NV = 1; __VA_ARGS__ } \
    else if ((h).tpr == 256) { constexpr int TPR = 256, NV = 2; __VA_ARGS__ }                \
    else if ((h).tpr == 512) { constexpr int TPR = 512, NV = 2; __VA_ARGS__ }                \
    else { constexpr int TPR = 1024, NV = 2; __VA_ARGS__ }                                   \
  } while (0)

// one launch, with 16-byte loads or without
template <typename T, int TPR, int NV>
void launch_fwd(bool vec, unsigned n, hipStream_t st, const T* x, long ldx, const T* res, long ldr, const float* gamma, const float* beta, T* sum, T* y,
                float* stat, long rows, int C, float eps) {
  if (vec)
    hipLaunchKernelGGL((layernorm_fwd_kernel<T, TPR, NV, 1>), dim3(n), dim3(block_of(TPR)), 0, st, x, ldx, res, ldr, gamma, beta, sum, y, stat, rows, C, eps);
  else
    hipLaunchKernelGGL((layernorm_fwd_kernel<T, TPR, NV, 0>), dim3(n), dim3(block_of(TPR)), 0, st, x, ldx, res, ldr, gamma, beta, sum, y, stat, rows, C, eps);
}
template <typename T, int TPR, int NV>
void launch_bwd(bool vec, bool params, unsigned n, hipStream_t st, const T* s, long lds, const T* dy, long lddy, const T* dsum, long ldds, const float* gamma,
                const float* stat, T* dx, float* partial, long rows, int C) {
  auto kernel = vec ? (params ? layernorm_bwd_kernel<T, TPR, NV, 1, true> : layernorm_bwd_kernel<T, TPR, NV, 1, false>)
                    : (params ? layernorm_bwd_kernel<T, TPR, NV, 0, true> : layernorm_bwd_kernel<T, TPR, NV, 0, false>);
  hipLaunchKernelGGL(kernel, dim3(n), dim3(block_of(TPR)), 0, st, s, lds, dy, lddy, dsum, ldds, gamma, stat, dx, partial, rows, C);
}

// workgroups of the backward pass: each leaves 2 C partial sums, so no more than fill the chip
int bwd_blocks(long rows, int C, int dtype) {
  const Held h = held(C, dtype == TATT_T_BF16 ? 8 : 4);
  const long per = h.tpr ? block_of(h.tpr) / h.tpr : 1, need = (rows + per - 1) / per, most = h.tpr > 256 ? 512 : 1024;
  return (int)(need < most ? need : most);
}

constexpr long MAX_GRID = 1 << 16;  // workgroups of the forward pass: more rows go round
constexpr int MAX_GRID_Y = 65535;   // and of the grid's second axis: more columns go round
constexpr int MAX_COLUMNS = 1 << 27;  // a column and the loops' steps past it stay within an int, 16 columns a workgroup within the grid

bool lined_up(const void* p, long ld, int size) { return !p || (((uintptr_t)p & 15) == 0 && ld * size % 16 == 0); }

}  // namespace

extern "C" {

int tatt_layernorm_fwd(const void* x, long ldx, const void* res, long ldr, const float* gamma, const float* beta, void* sum, void* y,
                       float* stat, long rows, int C, float eps, int dtype, hipStream_t st) {
  TATT_CHECK_ARG(x && y && rows > 0 && C > 0 && (ldx >= C || ldx == 0) && (!res || (sum && (ldr >= C || ldr == 0))), "tatt_layernorm_fwd: bad arguments (rows %ld, C %d)", rows, C);
  TATT_CHECK_ARG(C < MAX_COLUMNS, "tatt_layernorm_fwd: rows of 2^27 elements or more");
  TATT_CHECK_ARG(dtype == TATT_T_F32 || dtype == TATT_T_BF16, "tatt_layernorm_fwd: unknown element type %d", dtype);
  TATT_CHECK_ARG(((uintptr_t)stat & 7) == 0, "tatt_layernorm_fwd: stat is not 8-byte aligned");
  const int size = dtype == TATT_T_BF16 ? 2 : 4;
  const int vec = C * size % 16 == 0 && lined_up(x, ldx, size) && lined_up(res, ldr, size) && lined_up(sum, C, size) && lined_up(y, C, size) &&
                  lined_up(gamma, 4, 4) && lined_up(beta, 4, 4);
  const Held h = held(C, 16 / size);
  const int per = h.tpr ? block_of(h.tpr) / h.tpr : 4;
  const long need = (rows + per - 1) / per;
  const unsigned n = (unsigned)(need < MAX_GRID ? need : MAX_GRID);
  TATT_DISPATCH_TYPE(
      dtype, if (!h.tpr) hipLaunchKernelGGL(layernorm_fwd_wide<T>, dim3(n), dim3(256), 0, st, (const T*)x, ldx, (const T*)res, ldr, gamma, beta, (T*)sum,
                                            (T*)y, stat, rows, C, eps);
      else TATT_DISPATCH_HELD(h, launch_fwd<T, TPR, NV>(vec, n, st, (const T*)x, ldx, (const T*)res, ldr, gamma, beta, (T*)sum, (T*)y, stat, rows, C, eps););
  );
  TATT_LAUNCH_CHECK("layernorm_fwd");
  return TATT_OK;
}

size_t tatt_layernorm_workspace(long rows, int C, int dtype) { return rows > 0 && C > 0 && C < MAX_COLUMNS ? (size_t)bwd_blocks(rows, C, dtype) * 2 * C : 0; }

int tatt_layernorm_bwd(const void* s, long lds, const void* dy, long lddy, const void* dsum, long ldds, const float* gamma,
                       const float* stat, void* dx, float* dgamma, float* dbeta, long rows, int C, int dtype, float* workspace,
                       hipStream_t st) {
  TATT_CHECK_ARG(s && dy && stat && dx && rows > 0 && C > 0 && (lds >= C || lds == 0) && (lddy >= C || lddy == 0) && (!dsum || ldds >= C || ldds == 0),
                 "tatt_layernorm_bwd: bad arguments (rows %ld, C %d)", rows, C);
  TATT_CHECK_ARG(C < MAX_COLUMNS, "tatt_layernorm_bwd: rows of 2^27 elements or more");
  TATT_CHECK_ARG(dtype == TATT_T_F32 || dtype == TATT_T_BF16, "tatt_layernorm_bwd: unknown element type %d", dtype);
  TATT_CHECK_ARG(workspace || (!dgamma && !dbeta), "tatt_layernorm_bwd: parameter gradients need tatt_layernorm_workspace floats");
  TATT_CHECK_ARG(((uintptr_t)stat & 7) == 0, "tatt_layernorm_bwd: stat is not 8-byte aligned");
  const int size = dtype == TATT_T_BF16 ? 2 : 4, params = dgamma || dbeta, n = bwd_blocks(rows, C, dtype);
  const int vec = C * size % 16 == 0 && lined_up(s, lds, size) && lined_up(dy, lddy, size) && lined_up(dsum, ldds, size) && lined_up(dx, C, size) &&
                  lined_up(gamma, 4, 4);
  const Held h = held(C, 16 / size);
  TATT_DISPATCH_TYPE(
      dtype, if (!h.tpr) {
        hipLaunchKernelGGL(layernorm_dx_wide<T>, dim3((unsigned)((rows + 3) / 4 < MAX_GRID ? (rows + 3) / 4 : MAX_GRID)), dim3(256), 0, st, (const T*)s, lds,
                           (const T*)dy, lddy, (const T*)dsum, ldds, gamma, stat, (T*)dx, rows, C);
        if (params)
          hipLaunchKernelGGL(layernorm_params_wide<T>, dim3(n, cdiv(C, 256) < MAX_GRID_Y ? cdiv(C, 256) : MAX_GRID_Y), dim3(256), 0, st, (const T*)s, lds, (const T*)dy, lddy, stat, workspace, rows, C);
      } else TATT_DISPATCH_HELD(h, launch_bwd<T, TPR, NV>(vec, params, n, st, (const T*)s, lds, (const T*)dy, lddy, (const T*)dsum, ldds, gamma, stat, (T*)dx,
                                                          workspace, rows, C););
  );
  TATT_LAUNCH_CHECK("layernorm_bwd");
  if (params) {
    hipLaunchKernelGGL(layernorm_params_final, dim3(cdiv(C, 16), 2), dim3(256), 0, st, workspace, n, C, dgamma, dbeta);
    TATT_LAUNCH_CHECK("layernorm_params_final");
  }
  return TATT_OK;
}

}  // extern "C"
