// Compile-only check: drawn and drafted tokens through the C++ mirror's decoder.
#include <vector>

#include "btf_b200.hpp"

int draft_call_site(btf::cuda::Decoder& dec, int32_t token, float u) {
  const btf_sampling sampling{0.8f, 50, 0.95f, 0.0f};
  float lp = 0.0f;
  const int32_t t = dec.step_sampled(token, sampling, u, nullptr, &lp);
  const std::vector<int32_t> next = dec.verify({t, 1, 2}, {-1, 0, 0});
  dec.accept(0);
  const float us[2] = {u, u};
  return dec.verify({next[0], 3}, {-1, 0}, &sampling, us)[1];
}
