// Host-visible declarations of the choice of the next token.
#pragma once

#include <cstdint>
#include <cuda_runtime.h>

namespace ivb {

constexpr long long kSampleMaxVocab = 500000;

struct Sample {
  const void *x;             // [rows][vocab], 16 or 32 bits
  long long rows, stride;
  int vocab, dtype;          // dtype: ivc_dtype
  const float *u, *temperature;
  const int32_t *top_k;
  const float *top_p, *min_p;
  int32_t *tokens;
  float *probs;
  int slice, ranks;          // set by the launch: CTAs a row, and how much of it each has
  bool resident;             // the slice is kept in shared memory
};

cudaError_t launch_sample(Sample a, int sms, cudaStream_t st);

}  // namespace ivb
