// LayerNorm over rows of any width, forward and backward (tatt_ln_* in norm.hip is the 64-channel form with dropout in front).
//   s = x (+ res, rounded to the type: the sum is an output, and what is normalised is what was stored)
//   y = (s - mu) rstd * gamma + beta          stat[row] = (mu, rstd)
//   g = dy * gamma,  xhat = (s - mu) rstd,  ds = rstd (g - mean(g) - xhat mean(g xhat)) (+ dsum)
//   dgamma = sum over rows of dy * xhat,  dbeta = sum over rows of dy
// Statistics, sums and parameter gradients are fp32 whatever the tensors' type.
#include "token_types.h"

namespace {

// a wave per row
template <typename T>
__global__ __launch_bounds__(256) void layernorm_fwd_kernel(const T* __restrict__ x, long ldx, const T* __restrict__ res, long ldr,
                                                            const float* __restrict__ gamma, const float* __restrict__ beta, T* sum,
                                                            T* __restrict__ y, float* __restrict__ stat, long rows, int C, float eps) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
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

template <typename T>
__global__ __launch_bounds__(256) void layernorm_dx_kernel(const T* __restrict__ s, long lds, const T* __restrict__ dy, long lddy,
                                                           const T* __restrict__ dsum, long ldds, const float* __restrict__ gamma,
                                                           const float* __restrict__ stat, T* __restrict__ dx, long rows, int C) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= rows) return;
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

// partial[blk][2][C]: one thread per column walks the block's rows
constexpr int MAX_BLOCKS = 512;

template <typename T>
__global__ __launch_bounds__(256) void layernorm_param_kernel(const T* __restrict__ s, long lds, const T* __restrict__ dy, long lddy,
                                                              const float* __restrict__ stat, float* __restrict__ partial, long rows,
                                                              int C, long rows_per_block) {
  const int c = blockIdx.y * 256 + threadIdx.x;
  if (c >= C) return;
  const long r0 = blockIdx.x * rows_per_block, r1 = min(rows, r0 + rows_per_block);
  float dg = 0.f, db = 0.f;
  for (long r = r0; r < r1; ++r) {
    const float d = to_f32(dy[r * lddy + c]);
    dg += d * ((to_f32(s[r * lds + c]) - stat[2 * r]) * stat[2 * r + 1]);
    db += d;
  }
  partial[(blockIdx.x * 2L) * C + c] = dg;
  partial[(blockIdx.x * 2L + 1) * C + c] = db;
}

__global__ __launch_bounds__(256) void layernorm_param_final(const float* __restrict__ partial, int nblk, int C,
                                                             float* __restrict__ dgamma, float* __restrict__ dbeta) {
  __shared__ float red[256];
  const int c = blockIdx.x * 16 + (threadIdx.x & 15);
  float* dst = blockIdx.y ? dbeta : dgamma;
  const float v = block16_colsum(partial + (long)blockIdx.y * C, nblk, 2L * C, c, c < C, red);
  if (threadIdx.x < 16 && c < C && dst) dst[c] = v;
}

}  // namespace

extern "C" {

int tatt_layernorm_fwd(const void* x, long ldx, const void* res, long ldr, const float* gamma, const float* beta, void* sum, void* y,
                       float* stat, long rows, int C, float eps, int dtype, hipStream_t st) {
  TATT_CHECK_ARG(x && y && rows > 0 && C > 0 && ldx >= C && (!res || (sum && ldr >= C)), "tatt_layernorm_fwd: bad arguments (rows %ld, C %d)", rows, C);
  TATT_CHECK_ARG(dtype == TATT_T_F32 || dtype == TATT_T_BF16, "tatt_layernorm_fwd: unknown element type %d", dtype);
  TATT_CHECK_ARG(rows <= (1L << 32), "tatt_layernorm_fwd: more than 2^32 rows");
  TATT_DISPATCH_TYPE(dtype, hipLaunchKernelGGL(layernorm_fwd_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, (const T*)x, ldx,
                                               (const T*)res, ldr, gamma, beta, (T*)sum, (T*)y, stat, rows, C, eps););
  TATT_LAUNCH_CHECK("layernorm_fwd");
  return TATT_OK;
}

size_t tatt_layernorm_workspace(long rows, int C) { return (size_t)(rows < MAX_BLOCKS ? rows : MAX_BLOCKS) * 2 * C; }

int tatt_layernorm_bwd(const void* s, long lds, const void* dy, long lddy, const void* dsum, long ldds, const float* gamma,
                       const float* stat, void* dx, float* dgamma, float* dbeta, long rows, int C, int dtype, float* workspace,
                       hipStream_t st) {
  TATT_CHECK_ARG(s && dy && stat && dx && rows > 0 && C > 0 && lds >= C && lddy >= C && (!dsum || ldds >= C), "tatt_layernorm_bwd: bad arguments (rows %ld, C %d)", rows, C);
  TATT_CHECK_ARG(dtype == TATT_T_F32 || dtype == TATT_T_BF16, "tatt_layernorm_bwd: unknown element type %d", dtype);
  TATT_CHECK_ARG(workspace || (!dgamma && !dbeta), "tatt_layernorm_bwd: parameter gradients need tatt_layernorm_workspace floats");
  TATT_CHECK_ARG(rows <= (1L << 32), "tatt_layernorm_bwd: more than 2^32 rows");
  TATT_DISPATCH_TYPE(dtype, hipLaunchKernelGGL(layernorm_dx_kernel<T>, dim3((unsigned)((rows + 3) / 4)), dim3(256), 0, st, (const T*)s, lds,
                                               (const T*)dy, lddy, (const T*)dsum, ldds, gamma, stat, (T*)dx, rows, C););
  TATT_LAUNCH_CHECK("layernorm_dx");
  if (dgamma || dbeta) {
    const int nblk = (int)(rows < MAX_BLOCKS ? rows : MAX_BLOCKS);
    const long per = (rows + nblk - 1) / nblk;
    TATT_DISPATCH_TYPE(dtype, hipLaunchKernelGGL(layernorm_param_kernel<T>, dim3(nblk, cdiv(C, 256)), dim3(256), 0, st, (const T*)s, lds,
                                                 (const T*)dy, lddy, stat, workspace, rows, C, per););
    TATT_LAUNCH_CHECK("layernorm_param");
    hipLaunchKernelGGL(layernorm_param_final, dim3(cdiv(C, 16), 2), dim3(256), 0, st, workspace, nblk, C, dgamma, dbeta);
    TATT_LAUNCH_CHECK("layernorm_param_final");
  }
  return TATT_OK;
}

}  // extern "C"
