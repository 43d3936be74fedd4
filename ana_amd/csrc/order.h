// The order of logits, shared by the kernels that rank them: by value, then
// the lower index, a NaN after every number.
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace ana {

typedef unsigned long long u64;

// a logit's order as a whole number: larger for larger ones, -0 as +0, 0 for NaN
__device__ __forceinline__ uint32_t order_of(float x) {
  if (x != x) return 0;
  const uint32_t u = __builtin_bit_cast(uint32_t, x + 0.0f);
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t o) {
  if (o == 0) return __builtin_nanf("");
  return __builtin_bit_cast(float, (o & 0x80000000u) ? (o & 0x7FFFFFFFu) : ~o);
}
__device__ __forceinline__ u64 key_of(float x, uint32_t i) { return (u64)order_of(x) << 32 | (0xFFFFFFFFu - i); }

}  // namespace ana
