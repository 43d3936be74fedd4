// Tokens of rows of logits from given random numbers (sample.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

#include "kv4.h"
#include "order.h"

namespace ana {

constexpr uint32_t kSampleMaxVocab = 1u << 21;   // (masses in units of 2^-42 sum to 2^63 at most)
constexpr uint32_t kSampleMaxRows = (1u << 22) - 1;   // (workgroups of 512 threads, counted in 32 bits)

struct SampleArgs {
  const void* logits;
  uint64_t ld;        // elements from row to row
  uint32_t n, vocab;
  const float* u;     // [n]
  // the settings of every row, or [n] of each row's own
  float t, p, q;      // temperature, top-p, min-p
  uint32_t k;         // top-k
  const float *ts, *ps, *qs;
  const uint32_t* ks;
  uint32_t* tok;      // [n]
  float* lp;          // [n]
  u64* part;          // sample_ws_words words
};
// a split row's words in `part`: its bins, the mass of min-p's tokens, how many
// tokens were gathered, S pieces' group maxima, the gathered tokens
constexpr uint32_t kSampleBins = 2048, kSampleGather = 8192;
__host__ __device__ inline uint64_t sample_part_words(uint32_t S) { return kSampleBins + 2 + 32 * (uint64_t)S + kSampleGather; }
// the words of workspace a call takes (0 for none)
uint64_t sample_ws_words(uint32_t n, uint32_t vocab);
// (type: kv4.h's ElemType)
hipError_t launch_sample(const SampleArgs& a, int type, hipStream_t st);

}  // namespace ana
