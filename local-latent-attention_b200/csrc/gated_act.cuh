// gelu's gate to fp32's last bits.
#pragma once

#include "common.cuh"

namespace llattn {
namespace gated {

// phi(g) = erfc(-g / sqrt 2) / 2 and e = exp(-g^2 / 2), by erfc and exp of |g|, whose rounded arguments cost the tail
// 3e-7 of its value at g = -5 and 8e-5 at -13: what the rounding lost comes back to first order.
__device__ __forceinline__ void gaussian(float g, float& phi, float& e) {
  const float b = fminf(fabsf(g), 40.f);  // (e is 0 from 14.4 on; a NaN comes back with g)
  const float h = b * b, x = b * 0.70710678f;
  const float lost_h = fmaf(b, b, -h), lost_x = fmaf(b, 0.70710678f, -x) + b * 1.2101616e-8f;
  e = expf(-0.5f * h);
  e = fmaf(e, -0.5f * lost_h, e);
  const float tail = fmaf(-0.56418958f * e, lost_x, 0.5f * erfcf(x));
  phi = g > 0.f ? 1.f - tail : tail;
}

}  // namespace gated
}  // namespace llattn
