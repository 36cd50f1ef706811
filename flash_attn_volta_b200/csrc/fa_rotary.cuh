// The angle of a rotary position, shared by the rotation (fa_rotary.cu) and the
// cache append that rotates on the way (fa_kv_cache.cu).
#pragma once
#include <cstdint>
#include <cuda_runtime.h>

#include "fast_div.cuh"

namespace fa_sm100 {

// (M cos a, M sin a) of a = pos * inv_freq.  The angle of a far position is
// large (10^5 rad and more), where an fp32 product is off by 10^-2 rad, so the
// product and its reduction to turns are made in 64 bits: t = a / (2 pi), less
// the whole turns, leaves 2 t in [-1, 1] half turns, exact to 2^-34 at a
// million positions.  The sine and cosine of its fp32 head come from
// sincospif; the tail d (below 2^-24) is added to first order:
// cos(x + d) = cos x - d sin x.
__device__ __forceinline__ float2 rotary_cos_sin(double pos, double inv_freq, float magnitude) {
  const double t = pos * inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  const double half = 2.0 * (t - rint(t));
  const float head = (float)half;
  const float d = (float)(half - (double)head) * 3.14159265358979f;
  float s, c;
  sincospif(head, &s, &c);
  return make_float2(magnitude * fmaf(-d, s, c), magnitude * fmaf(d, c, s));
}

// The same with the sine and cosine in 64 bits, each rounded to fp32 once: for
// keys that are then rounded to 4 bits, where the last bit of a value next to the
// border of two codes decides between values a whole step apart (28.1 against
// 27.4 us for 4 x 1024 tokens of 32 + 2 x 8 heads of 128).
__device__ __forceinline__ float2 rotary_cos_sin_exact(double pos, double inv_freq, float magnitude) {
  const double t = pos * inv_freq * 0.15915494309189533577;  // 1 / (2 pi)
  double s, c;
  sincospi(2.0 * (t - rint(t)), &s, &c);
  return make_float2(magnitude * (float)c, magnitude * (float)s);
}

// N consecutive 16-bit elements as one load or store.
template <int N>
struct alignas(2 * N) Pack16 {
  uint16_t v[N];
};

}  // namespace fa_sm100
