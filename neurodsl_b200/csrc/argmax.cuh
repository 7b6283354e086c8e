// argmax.cuh — the order in which the greedy token is chosen.
#pragma once

namespace nd {

// (v2, i2) replaces (v, i) if larger, equal with a smaller index, or a
// number where v is NaN.
__device__ __forceinline__ void better(float& v, int& i, float v2, int i2) {
  if (v2 > v || (v2 == v && i2 < i) || (v != v && v2 == v2)) {
    v = v2;
    i = i2;
  }
}

}  // namespace nd
