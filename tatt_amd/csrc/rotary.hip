// Rotary positions over up to four axes (time, height, width ...): section a of a head's dimensions turns by the token's place on axis a.
//   angle = pos[token][a] * freq[pair];   (u, w) -> (u cos - w sin, u sin + w cos);   backward = the rotation by -angle
// A pair is (i, i + section/2) of its section, or (2i, 2i+1) where interleaved; dimensions behind the last section pass through.
// The angle is formed and reduced to a fraction of a turn in fp64 (a position of 10^6 leaves fp32 no correct digit of the sine),
// its sine and cosine and the products are fp32.
#include "token_types.h"

namespace {

constexpr int MAX_AXES = 4;

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
  int naxes;
  long tokens;           // B * L
  long L;
  int D, interleaved;
  float sign;
};

__device__ __forceinline__ double position(const RotaryArgs& a, long b, long l, int axis) {
  const long i = b * a.pb + l * a.pl + axis * a.pa;
  return a.pos_type == 0 ? (double)((const long*)a.pos)[i] : a.pos_type == 1 ? (double)((const int*)a.pos)[i] : (double)((const float*)a.pos)[i];
}

__device__ __forceinline__ void turn_of(double angle, float* c, float* s) {
  const double turns = angle * 0.15915494309189533577;  // 1 / (2 pi)
  sincospif((float)(2.0 * (turns - rint(turns))), s, c);
}

// a workgroup per token: a thread computes its pair's turn once and applies it to every head
template <typename T>
__global__ __launch_bounds__(128) void rotary_kernel(RotaryArgs a) {
  const long token = blockIdx.x, b = token / a.L, l = token - b * a.L;
  const int pairs = a.first_pair[a.naxes];
  for (int p = threadIdx.x; p < pairs; p += 128) {
    int axis = 0;
    while (p >= a.first_pair[axis + 1]) ++axis;
    float c, s;
    turn_of(position(a, b, l, axis) * a.freqs[p], &c, &s);
    s *= a.sign;
    const int f = a.first_pair[axis], n = a.first_pair[axis + 1] - f, i = p - f;
    const int lo = a.interleaved ? 2 * p : 2 * f + i, hi = a.interleaved ? 2 * p + 1 : lo + n;
    for (int w = 0; w < 2; ++w) {
      const T* x = (const T*)a.x[w] + b * a.sb[w] + l * a.sl[w];
      T* y = (T*)a.y[w] + token * a.H[w] * a.D;
      for (int h = 0; h < a.H[w]; ++h) {
        const float u = to_f32(x[h * a.sh[w] + lo]), v = to_f32(x[h * a.sh[w] + hi]);
        y[h * a.D + lo] = from_f32<T>(u * c - v * s);
        y[h * a.D + hi] = from_f32<T>(u * s + v * c);
      }
    }
  }
  const int rest = a.D - 2 * pairs;
  for (int w = 0; w < 2; ++w) {
    const T* x = (const T*)a.x[w] + b * a.sb[w] + l * a.sl[w];
    T* y = (T*)a.y[w] + token * a.H[w] * a.D;
    for (int i = threadIdx.x; i < rest * a.H[w]; i += 128) {
      const int h = i / rest, d = 2 * pairs + i - h * rest;
      y[h * a.D + d] = x[h * a.sh[w] + d];
    }
  }
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
  TATT_CHECK_ARG((long)B * L < (1L << 31), "tatt_rotary: 2^31 tokens or more");
  RotaryArgs a = {};
  a.x[0] = q, a.y[0] = q_out, a.sb[0] = q_strides[0], a.sl[0] = q_strides[1], a.sh[0] = q_strides[2], a.H[0] = Hq;
  if (k) a.x[1] = k, a.y[1] = k_out, a.sb[1] = k_strides[0], a.sl[1] = k_strides[1], a.sh[1] = k_strides[2], a.H[1] = Hk;
  a.pos = pos, a.pos_type = pos_type, a.pb = pos_strides[0], a.pl = pos_strides[1], a.pa = pos_strides[2], a.freqs = freqs;
  for (int i = 0; i < naxes; ++i) {
    TATT_CHECK_ARG(sections[i] > 0 && sections[i] % 2 == 0, "tatt_rotary: sections are positive and even, got %d", sections[i]);
    a.first_pair[i + 1] = a.first_pair[i] + sections[i] / 2;
    TATT_CHECK_ARG(2L * a.first_pair[i + 1] <= D, "tatt_rotary: the sections exceed the %d dimensions of a head", D);
  }
  a.naxes = naxes, a.tokens = (long)B * L, a.L = L, a.D = D, a.interleaved = interleaved, a.sign = inverse ? -1.f : 1.f;
  TATT_DISPATCH_TYPE(dtype, hipLaunchKernelGGL(rotary_kernel<T>, dim3((unsigned)a.tokens), dim3(128), 0, st, a););
  TATT_LAUNCH_CHECK("rotary");
  return TATT_OK;
}

}  // extern "C"
