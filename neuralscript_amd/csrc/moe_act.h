// The activations' derivatives of the layer with K experts a token.
#pragma once
#include "common.h"

namespace nship {

// act(u) and act'(u), what they share computed once.  SiLU's slope is sigma (1 + u
// (1 - sigma)); the networks' own layers take the reference's spelling
// (act_deriv), which is another function.
__device__ __forceinline__ void act_both(float u, int act, float& a, float& slope) {
  switch (act) {
    case kActGelu: {
      const float p = 0.5f * (1.f + erff(u * 0.707106781f));
      a = u * p;
      slope = p + u * expf(-0.5f * u * u) * 0.398942280f;
      break;
    }
    case kActSilu: {
      const float s = 1.f / (1.f + expf(-u));
      a = u * s;
      slope = s + a * (1.f - s);
      break;
    }
    case kActTanh: a = tanhf(u); slope = 1.f - a * a; break;
    case kActSigmoid: a = 1.f / (1.f + expf(-u)); slope = a * (1.f - a); break;
    default: a = act_apply(u, act); slope = act_deriv(u, act); break;
  }
}

}  // namespace nship
