// Normalised and rotated heads, a lane's share of one at a time: rotary.hip (in place) and paged_append.hip (keys on their way to their pages).
//   y = x / (|x|_2 / sqrt(D) + eps) * w;   (a, b) -> (a cos - b sin, b cos + a sin),   in fp32, rounded once.
// D / 8 adjacent lanes hold a head, 8 values each: pairs never leave a lane. Interleaved pairs lie side by side, and a lane holds a stretch of 8; pairs of
// halves: four values of either half of the rotated part. Lanes behind that part hold stretches.
#pragma once
#include <type_traits>

#include "kvx_common.h"

namespace kvx {
namespace {

template <int LPR>
__device__ __forceinline__ float sum_over_row(float v) {
  auto add = [](float x, auto ctrl) {
    return x + __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), decltype(ctrl)::value, 0xf, 0xf, true));
  };
  v = add(v, std::integral_constant<int, 0xB1>{});   // quad_perm [1,0,3,2]
  v = add(v, std::integral_constant<int, 0x4E>{});   // quad_perm [2,3,0,1]
  v = add(v, std::integral_constant<int, 0x141>{});  // row_half_mirror
  if constexpr (LPR >= 16) v = add(v, std::integral_constant<int, 0x140>{});  // row_mirror
  if constexpr (LPR == 32) {
    const u32pair_t r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);  // the other row of the pair
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return v;
}

// x0: values lo .. lo + 3 of a head, x1: hi .. hi + 3. norm: whether there are weights w, uniform; cv, sv: the angles of the lane's pairs if it `turns`; factor: 1 / sqrt(D).
template <int D, bool F16, bool INTERLEAVED>
__device__ __forceinline__ void turn(u32x2_t x0, u32x2_t x1, bool norm, const float* w, int lo, int hi, bool turns, f32x4_t cv, f32x4_t sv, float factor, float eps, u32x2_t& z0,
                                     u32x2_t& z1) {
  float y[8] = {elem_lo<F16>(x0[0]), elem_hi<F16>(x0[0]), elem_lo<F16>(x0[1]), elem_hi<F16>(x0[1]),
                elem_lo<F16>(x1[0]), elem_hi<F16>(x1[0]), elem_lo<F16>(x1[1]), elem_hi<F16>(x1[1])};
  if (norm) {
    float ss = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(y[e], y[e], ss);
    const float n = sqrtf(sum_over_row<D / 8>(ss)) * factor + eps;
    const f32x4_t w0 = *(const f32x4_t*)(w + lo), w1 = *(const f32x4_t*)(w + hi);
    const float inv = 1.0f / n;
    if (__all(n > 0x1p-120f)) {
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = y[e] * inv * (e < 4 ? w0[e] : w1[e - 4]);
    } else {  // some whose inverse is infinite, or NaN
#pragma unroll
      for (int e = 0; e < 8; ++e) y[e] = (n > 0x1p-120f ? y[e] * inv : y[e] / n) * (e < 4 ? w0[e] : w1[e - 4]);
    }
  }
  float z[8];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const int j = INTERLEAVED ? 2 * e : e, k = INTERLEAVED ? 2 * e + 1 : e + 4;
    z[j] = turns ? y[j] * cv[e] - y[k] * sv[e] : y[j];
    z[k] = turns ? y[k] * cv[e] + y[j] * sv[e] : y[k];
  }
  z0 = u32x2_t{pack_pair<F16>(z[0], z[1]), pack_pair<F16>(z[2], z[3])};
  z1 = u32x2_t{pack_pair<F16>(z[4], z[5]), pack_pair<F16>(z[6], z[7])};
}

}  // namespace
}  // namespace kvx
