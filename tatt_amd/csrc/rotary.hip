// Rotary positions over up to four axes (time, height, width ...): section a of a head's dimensions turns by the token's place on axis a.
//   angle = pos[token][a] * freq[pair];   (u, w) -> (u cos - w sin, u sin + w cos);   backward = the rotation by -angle
// A pair is (i, i + section/2) of its section, or (2i, 2i+1) where interleaved; dimensions behind the last section pass through.
// The angle is formed and reduced to a fraction of a turn in fp64 (a position of 10^6 leaves fp32 no correct digit of the sine),
// its sine and cosine and the products are fp32.
// Bound by memory: x is read and y written once.  The fp64 angle and the sine cost some 80 instructions, so a workgroup computes the turns of its
// few tokens once into LDS and applies them to every head of q and k.
// Measured: 36864 tokens, 20 heads of 128, bf16: 82 us a direction (377 MB, 4.6 TB/s); 65536 tokens, 8 heads of 16, fp32: 15-18 us (67 MB).
#include "token_types.h"

namespace {

constexpr int MAX_AXES = 4;
constexpr int TURNS = 512;  // (cos, sin) pairs of a workgroup's tokens in LDS

struct RotaryArgs {
  const void* x[2];      // q, k
  void* y[2];            // contiguous [B][L][H][D]
  long sb[2], sl[2], sh[2];
  int H[2];
  const void* pos;
  int pos_type;          // 0 int64, 1 int32, 2 fp32
  long pb, pl, pa;
  const double* freqs;
  int first_pair[MAX_AXES + 1];  // pairs of axis a: [first_pair[a], first_pair[a + 1])
  int naxes, pairs;
  int tokens;            // B * L
  int per_block;         // tokens of a workgroup
  int L, D;
  float sign;
};

__device__ __forceinline__ double position(const RotaryArgs& a, long b, long l, int axis) {
  const long i = b * a.pb + l * a.pl + axis * a.pa;
  return a.pos_type == 0 ? (double)((const long*)a.pos)[i] : a.pos_type == 1 ? (double)((const int*)a.pos)[i] : (double)((const float*)a.pos)[i];
}

__device__ __forceinline__ float2 turn_of(double angle, float sign) {
  const double turns = angle * 0.15915494309189533577;  // 1 / (2 pi)
  float c, s;
  sincospif((float)(2.0 * (turns - rint(turns))), &s, &c);
  return make_float2(c, s * sign);
}

template <typename T, int V, bool FITS>
struct alignas(sizeof(T) * (FITS ? V : 1)) Vec {
  T e[V];
};

// V neighbouring elements at a time: V = 16 bytes where sections, strides and pointers allow it, else 8 bytes, else (FITS = false) element by element
template <typename T, int V, bool INTERLEAVED, bool FITS>
__global__ __launch_bounds__(256) void rotary_kernel(RotaryArgs a) {
  __shared__ float2 turns[TURNS];
  const int token0 = (int)blockIdx.x * a.per_block, n = min(a.per_block, a.tokens - token0);
  const int rest = a.D - 2 * a.pairs, heads = a.H[0] + a.H[1];
  // units of a head: V pairs each (halves: V elements of either half), then V elements each of what passes through
  constexpr int PAIRS = INTERLEAVED ? V / 2 : V, REST = FITS ? V : 1;
  const int turning = a.pairs / PAIRS, units = turning + rest / REST;
  typedef Vec<T, V, FITS> VT;
  for (int p0 = 0; p0 < n * a.pairs; p0 += TURNS) {  // one pass, unless a single token has more pairs than LDS holds
    __syncthreads();
    for (int i = threadIdx.x; i < min(TURNS, n * a.pairs - p0); i += 256) {
      const int t = (p0 + i) / a.pairs, p = p0 + i - t * a.pairs;
      int axis = 0;
      while (p >= a.first_pair[axis + 1]) ++axis;
      const int token = token0 + t;
      turns[i] = turn_of(position(a, token / a.L, token % a.L, axis) * a.freqs[p], a.sign);
    }
    __syncthreads();
    const int last = p0 + TURNS >= n * a.pairs;
    for (int i = threadIdx.x; i < n * heads * units; i += 256) {
      const int th = i / units, u = i - th * units, t = th / heads, h0 = th - t * heads, w = h0 >= a.H[0], h = w ? h0 - a.H[0] : h0;
      const int token = token0 + t, b = token / a.L, l = token - b * a.L;
      const T* x = (const T*)a.x[w] + b * a.sb[w] + l * a.sl[w] + h * a.sh[w];
      T* y = (T*)a.y[w] + ((long)token * a.H[w] + h) * a.D;
      if (u >= turning) {
        const int d = 2 * a.pairs + (u - turning) * REST;
        if (last) *reinterpret_cast<Vec<T, REST, FITS>*>(y + d) = *reinterpret_cast<const Vec<T, REST, FITS>*>(x + d);
        continue;
      }
      const int p = u * PAIRS, at = t * a.pairs + p - p0;
      if (at < 0 || at >= TURNS) continue;
      if constexpr (INTERLEAVED) {
        VT v = *reinterpret_cast<const VT*>(x + 2 * p);
#pragma unroll
        for (int e = 0; e < V / 2; ++e) {
          const float2 c = turns[at + e];
          const float f = to_f32(v.e[2 * e]), g = to_f32(v.e[2 * e + 1]);
          v.e[2 * e] = from_f32<T>(f * c.x - g * c.y);
          v.e[2 * e + 1] = from_f32<T>(f * c.y + g * c.x);
        }
        *reinterpret_cast<VT*>(y + 2 * p) = v;
      } else {
        int axis = 0;
        while (p >= a.first_pair[axis + 1]) ++axis;
        const int lo = a.first_pair[axis] + p, hi = a.first_pair[axis + 1] + p;  // 2 first + (p - first), and half a section on
        VT v = *reinterpret_cast<const VT*>(x + lo), q = *reinterpret_cast<const VT*>(x + hi);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float2 c = turns[at + e];
          const float f = to_f32(v.e[e]), g = to_f32(q.e[e]);
          v.e[e] = from_f32<T>(f * c.x - g * c.y);
          q.e[e] = from_f32<T>(f * c.y + g * c.x);
        }
        *reinterpret_cast<VT*>(y + lo) = v;
        *reinterpret_cast<VT*>(y + hi) = q;
      }
    }
  }
}

// whether units of V elements fit everything: no unit crosses a half or section, every address is a multiple of its size
bool fits(const RotaryArgs& a, int V, int size, int interleaved) {
  if (a.D % V || 2 * a.pairs % V) return false;
  for (int i = 0; i < a.naxes; ++i)
    if (!interleaved && (a.first_pair[i + 1] - a.first_pair[i]) % V) return false;
  for (int w = 0; w < 2; ++w)
    if (a.x[w] && ((((uintptr_t)a.x[w]) | ((uintptr_t)a.y[w])) % (V * size) || a.sb[w] % V || a.sl[w] % V || a.sh[w] % V)) return false;
  return true;
}

template <typename T, bool INTERLEAVED>
void launch(const RotaryArgs& a, hipStream_t st) {
  const unsigned n = cdiv(a.tokens, a.per_block);
  constexpr int V = 16 / sizeof(T);
  if (fits(a, V, sizeof(T), INTERLEAVED))
    hipLaunchKernelGGL((rotary_kernel<T, V, INTERLEAVED, true>), dim3(n), dim3(256), 0, st, a);
  else if (fits(a, V / 2, sizeof(T), INTERLEAVED))
    hipLaunchKernelGGL((rotary_kernel<T, V / 2, INTERLEAVED, true>), dim3(n), dim3(256), 0, st, a);
  else if constexpr (INTERLEAVED)
    hipLaunchKernelGGL((rotary_kernel<T, 2, true, false>), dim3(n), dim3(256), 0, st, a);
  else
    hipLaunchKernelGGL((rotary_kernel<T, 1, false, false>), dim3(n), dim3(256), 0, st, a);
}

}  // namespace

extern "C" {

int tatt_rotary(const void* q, const long* q_strides, void* q_out, int Hq, const void* k, const long* k_strides, void* k_out, int Hk,
                const void* pos, int pos_type, const long* pos_strides, const double* freqs, const int* sections, int naxes, int B, long L,
                int D, int interleaved, int inverse, int dtype, hipStream_t st) {
  TATT_CHECK_ARG(q && q_strides && q_out && pos && pos_strides && freqs && sections && B > 0 && L > 0 && D > 0 && Hq > 0, "tatt_rotary: bad arguments");
  TATT_CHECK_ARG(!k || (k_strides && k_out && Hk > 0), "tatt_rotary: k without its strides, output or heads");
  TATT_CHECK_ARG(dtype == TATT_T_F32 || dtype == TATT_T_BF16, "tatt_rotary: unknown element type %d", dtype);
  TATT_CHECK_ARG(pos_type >= 0 && pos_type <= 2, "tatt_rotary: unknown position type %d", pos_type);
  TATT_CHECK_ARG(naxes >= 1 && naxes <= MAX_AXES, "tatt_rotary: 1 to %d axes, got %d", MAX_AXES, naxes);
  TATT_CHECK_ARG(L < (1L << 31) && B * L < (1L << 31), "tatt_rotary: 2^31 tokens or more");
  TATT_CHECK_ARG(((long)Hq + (k ? Hk : 0)) * D < (1L << 20), "tatt_rotary: a token of 2^20 elements or more");
  RotaryArgs a = {};
  a.x[0] = q, a.y[0] = q_out, a.sb[0] = q_strides[0], a.sl[0] = q_strides[1], a.sh[0] = q_strides[2], a.H[0] = Hq;
  if (k) a.x[1] = k, a.y[1] = k_out, a.sb[1] = k_strides[0], a.sl[1] = k_strides[1], a.sh[1] = k_strides[2], a.H[1] = Hk;
  a.pos = pos, a.pos_type = pos_type, a.pb = pos_strides[0], a.pl = pos_strides[1], a.pa = pos_strides[2], a.freqs = freqs;
  for (int i = 0; i < naxes; ++i) {
    TATT_CHECK_ARG(sections[i] > 0 && sections[i] % 2 == 0, "tatt_rotary: sections are positive and even, got %d", sections[i]);
    TATT_CHECK_ARG(sections[i] <= D - 2 * a.first_pair[i], "tatt_rotary: the sections exceed the %d dimensions of a head", D);
    a.first_pair[i + 1] = a.first_pair[i] + sections[i] / 2;
  }
  a.naxes = naxes, a.pairs = a.first_pair[naxes], a.tokens = (int)(B * L), a.L = (int)L, a.D = D, a.sign = inverse ? -1.f : 1.f;
  // as many tokens as LDS holds turns for, but no fewer than 1024 workgroups where there are tokens for them: few tokens wait for nothing but latency
  int per = TURNS / a.pairs, most = a.tokens / 1024;
  a.per_block = per < 1 || most < 1 ? 1 : per < most ? per : most;
  while (cdiv(a.tokens, a.per_block) >= 1 << 24) a.per_block *= 2;  // the grid's own limit
  TATT_DISPATCH_TYPE(dtype, if (interleaved) launch<T, true>(a, st); else launch<T, false>(a, st););
  TATT_LAUNCH_CHECK("rotary");
  return TATT_OK;
}

}  // extern "C"
