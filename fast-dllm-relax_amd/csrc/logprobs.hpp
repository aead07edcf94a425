// Launch interface of the token log probabilities (logprobs.hip).
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fdllm {

enum LogitsType : int { LT_BF16 = 0, LT_F16 = 1, LT_F32 = 2 };
constexpr int LP_MAX_TOP = 32;
constexpr int LP_MAX_ROWS = (1 << 24) - 1;      // a launch's x axis holds fewer than 2^32 threads
constexpr int LP_MAX_VOCAB = 0x7fffffff - 4096;  // indices past the end stay in 31 bits
struct LogprobsP {
  const void* logits; long long ld;  // elements from row to row
  int type, rows, vocab, top;
  const int32_t* ids;                // null: no token's log probability
  float *logprob, *entropy;          // [rows] each (logprob null with ids null)
  int32_t* top_ids; float* top_logprob;  // [rows][top]
  int S;                             // vocabulary splits of a row
  void* ws;                          // S > 1: partials of [rows][S]
};
int logprobs_splits(const LogprobsP& a, int cus);
size_t logprobs_bytes(const LogprobsP& a);
hipError_t launch_logprobs(const LogprobsP& a, hipStream_t st);

}  // namespace fdllm
