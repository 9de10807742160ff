// Launcher of the sampling kernel (csrc/sample.cu). Internal: btf_sample and the
// decoder call it.
#pragma once
#include <cuda_runtime.h>

#include <cstdint>

namespace btf {

// btf_sample's arguments (checked by the caller); tokens2: a second copy of the
// tokens, or null.
struct SampleArgs {
  const void* logits;
  int type;
  int64_t ld;
  int B, V;
  const float *u, *temperature;
  const int32_t* top_k;
  const float *top_p, *min_p;
  int32_t *tokens, *tokens2;
  float* logprobs;
};
cudaError_t launch_sample(const SampleArgs& args, cudaStream_t st);

}  // namespace btf
