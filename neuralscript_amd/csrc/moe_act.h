// The activations' derivatives of the layer with K experts a token.
#pragma once
#include "common.h"

namespace nship {

// act'(u).  SiLU's is sigma (1 + u (1 - sigma)); the networks' own layers take
// the reference's spelling (act_deriv), which is another function.
__device__ __forceinline__ float act_slope(float u, int act) {
  if (act != kActSilu) return act_deriv(u, act);
  const float s = 1.f / (1.f + expf(-u));
  return s + u * s * (1.f - s);
}

}  // namespace nship
