// Attention of any lengths, head counts and head widths up to 128, forward and backward (attn.hip is the 26-key, 4 x 16 form).
//   S = scale q k^T;  lse_i = log sum_j exp S_ij;  P = exp(S - lse);  O = P V
//   delta_i = dO_i . O_i;  dV = P^T dO;  dS = P (dO V^T - delta);  dQ = scale dS K;  dK = scale dS^T Q
// H = G * Hkv query heads: head h reads key head h / G, and a key head's gradients are the sum over its G query heads.
// Hidden places: keys whose mask byte is not 0, and, where causal, j > i + Lk - Lq.  A row that sees nothing gives zeros (lse = +inf) and
// takes no part in any gradient; a masked key's K and V are never read into a result.
#include "token_types.h"

namespace {

struct MhaArgs {
  const void *q, *k, *v, *out, *dout;
  long qs[3], ks[3], vs[3], os[3], dos[3];  // element strides: batch, token, head
  const unsigned char* mask;
  long mask_sb, mask_sl;
  int B, Lq, Lk, H, Hkv, G, D, causal;
  float scale;
};

// a wave per (batch, head, query); lane = dimensions lane and lane + 64
template <typename T>
__global__ __launch_bounds__(256) void mha_fwd_kernel(MhaArgs a, T* __restrict__ out, float* __restrict__ lse) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (long)a.B * a.H * a.Lq) return;
  const int i = row % a.Lq, h = row / a.Lq % a.H;
  const long b = row / a.Lq / a.H;
  const T* q = (const T*)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T* k = (const T*)a.k + b * a.ks[0] + (h / a.G) * a.ks[2];
  const T* v = (const T*)a.v + b * a.vs[0] + (h / a.G) * a.vs[2];
  const bool on0 = lane < a.D, on1 = lane + 64 < a.D;
  const float q0 = on0 ? to_f32(q[lane]) * a.scale : 0.f, q1 = on1 ? to_f32(q[lane + 64]) * a.scale : 0.f;
  float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
  const int end = a.causal ? min(a.Lk, max(0, i + 1 + a.Lk - a.Lq)) : a.Lk;
  for (int j = 0; j < end; ++j) {
    if (a.mask && a.mask[b * a.mask_sb + j * a.mask_sl]) continue;
    const T *kj = k + j * a.ks[1], *vj = v + j * a.vs[1];
    const float s = wave_sum((on0 ? q0 * to_f32(kj[lane]) : 0.f) + (on1 ? q1 * to_f32(kj[lane + 64]) : 0.f));
    const float mn = fmaxf(m, s), f = expf(m - mn), p = expf(s - mn);
    o0 = o0 * f + (on0 ? p * to_f32(vj[lane]) : 0.f);
    o1 = o1 * f + (on1 ? p * to_f32(vj[lane + 64]) : 0.f);
    l = l * f + p;
    m = mn;
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* o = out + ((b * a.Lq + i) * a.H + h) * a.D;
  if (on0) o[lane] = from_f32<T>(o0 * inv);
  if (on1) o[lane + 64] = from_f32<T>(o1 * inv);
  if (lse && lane == 0) lse[(b * a.H + h) * a.Lq + i] = l == 0.f ? INFINITY : m + logf(l);
}

// dQ: a wave per (batch, head, query)
template <typename T>
__global__ __launch_bounds__(256) void mha_dq_kernel(MhaArgs a, const float* __restrict__ lse, float* __restrict__ delta, T* __restrict__ dq) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (long)a.B * a.H * a.Lq) return;
  const int i = row % a.Lq, h = row / a.Lq % a.H;
  const long b = row / a.Lq / a.H;
  const T* q = (const T*)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
  const T* k = (const T*)a.k + b * a.ks[0] + (h / a.G) * a.ks[2];
  const T* v = (const T*)a.v + b * a.vs[0] + (h / a.G) * a.vs[2];
  const T* o = (const T*)a.out + b * a.os[0] + i * a.os[1] + h * a.os[2];
  const T* g = (const T*)a.dout + b * a.dos[0] + i * a.dos[1] + h * a.dos[2];
  const bool on0 = lane < a.D, on1 = lane + 64 < a.D;
  const float q0 = on0 ? to_f32(q[lane]) * a.scale : 0.f, q1 = on1 ? to_f32(q[lane + 64]) * a.scale : 0.f;
  const float g0 = on0 ? to_f32(g[lane]) : 0.f, g1 = on1 ? to_f32(g[lane + 64]) : 0.f;
  const float dl = wave_sum((on0 ? g0 * to_f32(o[lane]) : 0.f) + (on1 ? g1 * to_f32(o[lane + 64]) : 0.f));
  const float ls = lse[(b * a.H + h) * a.Lq + i];
  if (lane == 0) delta[(b * a.H + h) * a.Lq + i] = dl;
  float d0 = 0.f, d1 = 0.f;
  const int end = a.causal ? min(a.Lk, max(0, i + 1 + a.Lk - a.Lq)) : a.Lk;
  for (int j = 0; j < end; ++j) {
    if (a.mask && a.mask[b * a.mask_sb + j * a.mask_sl]) continue;
    const T *kj = k + j * a.ks[1], *vj = v + j * a.vs[1];
    const float k0 = on0 ? to_f32(kj[lane]) : 0.f, k1 = on1 ? to_f32(kj[lane + 64]) : 0.f;
    const float s = wave_sum(q0 * k0 + q1 * k1);
    const float dp = wave_sum((on0 ? g0 * to_f32(vj[lane]) : 0.f) + (on1 ? g1 * to_f32(vj[lane + 64]) : 0.f));
    const float ds = expf(s - ls) * (dp - dl) * a.scale;
    d0 += ds * k0;
    d1 += ds * k1;
  }
  T* d = dq + ((b * a.Lq + i) * a.H + h) * a.D;
  if (on0) d[lane] = from_f32<T>(d0);
  if (on1) d[lane + 64] = from_f32<T>(d1);
}

// dK, dV: a wave per (batch, key head, key), over the queries of the group's heads
template <typename T>
__global__ __launch_bounds__(256) void mha_dkv_kernel(MhaArgs a, const float* __restrict__ lse, const float* __restrict__ delta,
                                                      T* __restrict__ dk, T* __restrict__ dv) {
  const int lane = threadIdx.x & 63;
  const long row = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (long)a.B * a.Hkv * a.Lk) return;
  const int j = row % a.Lk, hk = row / a.Lk % a.Hkv;
  const long b = row / a.Lk / a.Hkv;
  const bool on0 = lane < a.D, on1 = lane + 64 < a.D;
  const T* k = (const T*)a.k + b * a.ks[0] + j * a.ks[1] + hk * a.ks[2];
  const T* v = (const T*)a.v + b * a.vs[0] + j * a.vs[1] + hk * a.vs[2];
  const float k0 = on0 ? to_f32(k[lane]) * a.scale : 0.f, k1 = on1 ? to_f32(k[lane + 64]) * a.scale : 0.f;
  const float v0 = on0 ? to_f32(v[lane]) : 0.f, v1 = on1 ? to_f32(v[lane + 64]) : 0.f;
  float dk0 = 0.f, dk1 = 0.f, dv0 = 0.f, dv1 = 0.f;
  if (!(a.mask && a.mask[b * a.mask_sb + j * a.mask_sl]))
    for (int h = hk * a.G; h < (hk + 1) * a.G; ++h)
      for (int i = a.causal ? max(0, j - (a.Lk - a.Lq)) : 0; i < a.Lq; ++i) {
        const T* q = (const T*)a.q + b * a.qs[0] + i * a.qs[1] + h * a.qs[2];
        const T* g = (const T*)a.dout + b * a.dos[0] + i * a.dos[1] + h * a.dos[2];
        const float q0 = on0 ? to_f32(q[lane]) : 0.f, q1 = on1 ? to_f32(q[lane + 64]) : 0.f;
        const float g0 = on0 ? to_f32(g[lane]) : 0.f, g1 = on1 ? to_f32(g[lane + 64]) : 0.f;
        const float p = expf(wave_sum(q0 * k0 + q1 * k1) - lse[(b * a.H + h) * a.Lq + i]);
        const float ds = p * (wave_sum(g0 * v0 + g1 * v1) - delta[(b * a.H + h) * a.Lq + i]) * a.scale;
        dk0 += ds * q0, dk1 += ds * q1;
        dv0 += p * g0, dv1 += p * g1;
      }
  const long at = ((b * a.Lk + j) * a.Hkv + hk) * a.D;
  if (on0) dk[at + lane] = from_f32<T>(dk0), dv[at + lane] = from_f32<T>(dv0);
  if (on1) dk[at + lane + 64] = from_f32<T>(dk1), dv[at + lane + 64] = from_f32<T>(dv1);
}

int fill(MhaArgs& a, const char* who, const void* q, const void* k, const void* v, const long* strides, const unsigned char* mask, const long* mask_strides,
         int B, int Lq, int Lk, int H, int Hkv, int D, float scale, int causal, int dtype) {
  TATT_CHECK_ARG(q && k && v && strides && B > 0 && Lq > 0 && Lk > 0 && H > 0 && Hkv > 0, "%s: bad arguments", who);
  TATT_CHECK_ARG(!mask || mask_strides, "%s: a key mask needs its strides", who);
  TATT_CHECK_ARG(H % Hkv == 0, "%s: %d query heads are no multiple of %d key heads", who, H, Hkv);
  TATT_CHECK_ARG(D > 0 && D <= 128, "%s: built for heads of 1 to 128, got %d", who, D);
  TATT_CHECK_ARG(dtype == TATT_T_F32 || dtype == TATT_T_BF16, "%s: unknown element type %d", who, dtype);
  TATT_CHECK_ARG((long)B * H * Lq < (1L << 31) && (long)B * Hkv * Lk < (1L << 31), "%s: 2^31 rows or more", who);
  a.q = q, a.k = k, a.v = v, a.mask = mask;
  a.mask_sb = mask ? mask_strides[0] : 0, a.mask_sl = mask ? mask_strides[1] : 0;
  for (int i = 0; i < 3; ++i) a.qs[i] = strides[i], a.ks[i] = strides[3 + i], a.vs[i] = strides[6 + i];
  a.B = B, a.Lq = Lq, a.Lk = Lk, a.H = H, a.Hkv = Hkv, a.G = H / Hkv, a.D = D, a.scale = scale, a.causal = causal;
  return TATT_OK;
}

}  // namespace

extern "C" {

size_t tatt_mha_fwd_workspace(int B, int Lq, int Lk, int H, int Hkv, int D, int dtype) { return 0; }

int tatt_mha_fwd(const void* q, const void* k, const void* v, const long* strides, const unsigned char* mask, const long* mask_strides,
                 void* out, float* lse, int B, int Lq, int Lk, int H, int Hkv, int D, float scale, int causal, int dtype, float* workspace,
                 hipStream_t st) {
  MhaArgs a = {};
  if (int rc = fill(a, "tatt_mha_fwd", q, k, v, strides, mask, mask_strides, B, Lq, Lk, H, Hkv, D, scale, causal, dtype)) return rc;
  TATT_CHECK_ARG(out, "tatt_mha_fwd: no output");
  TATT_DISPATCH_TYPE(dtype, hipLaunchKernelGGL(mha_fwd_kernel<T>, dim3(cdiv((long)B * H * Lq, 4)), dim3(256), 0, st, a, (T*)out, lse););
  TATT_LAUNCH_CHECK("mha_fwd");
  return TATT_OK;
}

size_t tatt_mha_bwd_workspace(int B, int Lq, int Lk, int H, int Hkv, int D, int dtype) { return (size_t)B * H * Lq; }

int tatt_mha_bwd(const void* q, const void* k, const void* v, const long* strides, const unsigned char* mask, const long* mask_strides,
                 const void* out, const void* dout, const float* lse, void* dq, void* dk, void* dv, int B, int Lq, int Lk, int H, int Hkv, int D, float scale, int causal,
                 int dtype, float* workspace, hipStream_t st) {
  MhaArgs a = {};
  if (int rc = fill(a, "tatt_mha_bwd", q, k, v, strides, mask, mask_strides, B, Lq, Lk, H, Hkv, D, scale, causal, dtype)) return rc;
  TATT_CHECK_ARG(out && dout && lse && dq && dk && dv && workspace, "tatt_mha_bwd: bad arguments (workspace: tatt_mha_bwd_workspace floats)");
  a.out = out, a.dout = dout;
  for (int i = 0; i < 3; ++i) a.os[i] = strides[9 + i], a.dos[i] = strides[12 + i];
  TATT_DISPATCH_TYPE(dtype, hipLaunchKernelGGL(mha_dq_kernel<T>, dim3(cdiv((long)B * H * Lq, 4)), dim3(256), 0, st, a, lse, workspace, (T*)dq););
  TATT_LAUNCH_CHECK("mha_dq");
  TATT_DISPATCH_TYPE(dtype, hipLaunchKernelGGL(mha_dkv_kernel<T>, dim3(cdiv((long)B * Hkv * Lk, 4)), dim3(256), 0, st, a, lse, workspace, (T*)dk, (T*)dv););
  TATT_LAUNCH_CHECK("mha_dkv");
  return TATT_OK;
}

}  // extern "C"
