// Log probabilities of logit rows (logprobs.cu): arguments and launch entry.
#pragma once
#include "common.cuh"

namespace b200mm {

constexpr int kLogprobsMaxTop = 64;

struct LogprobsArgs {
  const void* x; int64_t ldx;  // [M, V]
  const int64_t* tokens;       // [M]
  float* logprob;              // [M]
  float* entropy;              // [M]
  int64_t* top_ids;            // [M, top]
  float* top_logprobs;         // [M, top]
  int64_t M;
  int V, top;
};

int logprobs_launch(const LogprobsArgs& a, int dtype, cudaStream_t st);

}  // namespace b200mm
