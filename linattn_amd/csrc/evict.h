// Ranking of cached entries by weight, shared by eviction and the decode step.
#pragma once

#include "common.h"

namespace la {

constexpr uint32_t EV_SAFE = 0xffffffffu;  // a protected entry: above every weight

// Monotone map of fp32 weights to 1 and up: -0 ties with +0, a weight that is not a number
// is lowest.
__device__ __forceinline__ uint32_t ev_key(float w) {
  const uint32_t u = __float_as_uint(w + 0.f);  // (-0 + 0 is +0)
  return w != w ? 1u : u ^ ((uint32_t)((int32_t)u >> 31) | 0x80000000u);
}

__device__ __forceinline__ bool ev_safe(int64_t position, int64_t pos, int64_t recent, int64_t sink) {
  return position < sink || position >= pos - recent;
}

}  // namespace la
