// score.h — how lmh_attend_scored shapes a score before the softmax (device code).
#pragma once

#include "device.h"

namespace lmh {

constexpr float LOG2E = 1.4426950408889634f;

// The largest of x over a row of 16 lanes.
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x121, 0xf, 0xf, true));   // rotated by 1, 2, 4, 8
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x122, 0xf, 0xf, true));
  x = max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x124, 0xf, 0xf, true));
  return max(x, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x128, 0xf, 0xf, true));
}

// cap * tanh(u) of N scores, u = score / cap and cap in the log2 domain (cap * log2(e)). While every |u| of the wave
// is at most 3/4, by a polynomial: tanh(u) = u + u^3 P(u^2), P of degree 4 fitted to the least largest error relative to
// tanh(u), 3.2e-8 of it (2.4 * 2^-24 as evaluated in f32, 0.7 * 2^-24 in the mean): nine multiply-adds. Caps are far above
// most scores, so that is the usual case. Past 3/4, t = e^(-2|u|) and (1 - t) / (1 + t), whose cancellation near 0 (2^-24
// of the cap, 3e-6 at a cap of 50) is why the small ones do not take it too; its two transcendental operations also cost
// as much as eight multiply-adds.
template <int N>
__device__ __forceinline__ void cap_scores(float (&u)[N], float cap) {
  constexpr float C0 = -0.3333306908607483f, C1 = 0.13326521217823029f, C2 = -0.0533902570605278f, C3 = 0.019664909690618515f,
                  C4 = -0.004769487306475639f;
  asm volatile("" : "+v"(u[0]));   // taken behind a test of the launch's cap: not to be computed ahead of it
  float top = fabsf(u[0]);
#pragma unroll
  for (int i = 1; i < N; i++) top = fmaxf(top, fabsf(u[i]));
  const bool far = __ballot(top > 0.75f) != 0;
  float y[N];
#pragma unroll
  for (int i = 0; i < N; i++) {
    const float x = u[i] * u[i], w = u[i] * cap;
    const float p = fmaf(fmaf(fmaf(fmaf(C4, x, C3), x, C2), x, C1), x, C0);
    y[i] = fmaf(w * x, p, w);
  }
  if (__builtin_expect(far, 0)) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const float a = fabsf(u[i]), t = __builtin_amdgcn_exp2f(a * (-2.0f * LOG2E));
      const float z = copysignf((1.0f - t) * __builtin_amdgcn_rcpf(1.0f + t) * cap, u[i]);
      y[i] = a > 0.75f ? z : y[i];
    }
  }
#pragma unroll
  for (int i = 0; i < N; i++) u[i] = y[i];
}

// Less slope * |position of the row - key|, i = 0 .. N - 1: the distance of the lane's first key, `d0` = key - position,
// plus off(i).
template <int N, typename Off>
__device__ __forceinline__ void bias_scores(float (&p)[N], float slope, float d0, Off&& off) {
#pragma unroll
  for (int i = 0; i < N; i++) p[i] = fmaf(-slope, fabsf(d0 + off(i)), p[i]);
}

}  // namespace lmh
