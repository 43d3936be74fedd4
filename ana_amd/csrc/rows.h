// Finding a row's sequence in a call's offsets.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace ana {

// the last i < n with off[i] <= r (0 when there is none), for the whole wave:
// 64 of the remaining places at a time
__device__ __forceinline__ uint32_t find_seq(const uint32_t* off, uint32_t n, uint32_t r) {
  const uint32_t lane = threadIdx.x & 63;
  uint32_t lo = 0, cnt = n;
  while (cnt > 1) {
    const uint32_t step = (cnt + 63) / 64, k = lane * step;
    const bool t = k < cnt && off[lo + k] <= r;
    const uint32_t c = __popcll(__ballot(t));
    if (c == 0) break;
    lo += (c - 1) * step;
    cnt = min(step, cnt - (c - 1) * step);
  }
  return lo;
}

// the same for one lane, from a place i at or before the answer: steps that
// double, then halve
__device__ __forceinline__ uint32_t find_from(const uint32_t* off, uint32_t n, uint32_t r, uint32_t i) {
  uint32_t step = 1;
  while (step < n - i && off[i + step] <= r) {
    i += step;
    step *= 2;
  }
  for (; step; step /= 2)
    if (step < n - i && off[i + step] <= r) i += step;
  return i;
}

}  // namespace ana
