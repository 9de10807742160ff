// Launchers of the adapters' prompt kernels (adapters_tc.cu).
#pragma once
#include "adapters.cuh"

namespace btf {
namespace adapt {

int setup_tc();
// y of the plan's large tiles, from h.
int expand_tc(const Params& p, bool half, bool y32, int sms, cudaStream_t st);

}  // namespace adapt
}  // namespace btf
