// Norms of queries and keys for each head with the position rotation (rope.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kv4.h"

namespace ana {

constexpr uint32_t kRopeMaxHd = 256;   // heads of 16, 32, .. values

struct RopeArgs {
  Kv4Rows r;            // (seq is not read)
  Kv4Mat q, qo, k, ko;
  uint32_t hq, hk, hd, rot;
  const float* freq;    // [rot / 2]
  const float *gq, *gk; // [hd] or nullptr: no norm
  float eps;
  bool near;            // pairs of neighbours, else one of each half
};
inline bool rope_fits(uint32_t hd) { return hd && hd % 16 == 0 && hd <= kRopeMaxHd; }
// (type: kv4.h's ElemType)
hipError_t launch_rope(const RopeArgs& a, int type, hipStream_t st);

}  // namespace ana
