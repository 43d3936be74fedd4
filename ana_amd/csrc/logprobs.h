// Log probabilities of rows of logits (logprobs.hip).
#pragma once
#include <hip/hip_runtime.h>

#include <cstdint>

namespace ana {

constexpr uint32_t kLpMaxTop = 64;           // alternatives a row
constexpr uint32_t kLpMaxVocab = 64u * 32768;  // (a wave joins up to 64 pieces)

struct LogprobArgs {
  const void* logits;
  uint64_t ld;          // elements from row to row
  uint32_t n, vocab, top;
  const uint32_t* tok;  // [n] given tokens, or nullptr (then lp and rank are not written)
  float *lp, *ent;      // [n]
  uint32_t* rank;       // [n]
  uint32_t* top_tok;    // [n][top]
  float* top_lp;
  uint32_t* part;       // pieces' results, logprobs_part_words words
};
// the words of workspace a call takes (0 for none)
uint64_t logprobs_part_words(uint32_t n, uint32_t vocab, uint32_t top);
// the most rows of a call (a launch's threads are counted in 32 bits)
uint32_t logprobs_max_rows(uint32_t vocab);
// (type: kv4.h's ElemType)
hipError_t launch_logprobs(const LogprobArgs& a, int type, hipStream_t st);

}  // namespace ana
