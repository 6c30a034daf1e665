// TEST INFRASTRUCTURE: the serving operators' launches (csrc/kernels.h) as no-ops that record what they were handed.
#include "cuda_runtime.h"
#include "kernels.h"

extern "C" {
extern int fake_launch_count;
int fake_serving_fail = 0;          // the next launches report a failure
uint64_t fake_append_rotary = 0, fake_append_sequences = 0;
}

namespace b200 {
static cudaError_t launched() { ++fake_launch_count; return fake_serving_fail ? cudaErrorNotSupported : cudaSuccess; }
cudaError_t launch_rope_append_pages(const AppendArgs& g, cudaStream_t) {
  fake_append_rotary = g.rotary;
  fake_append_sequences = g.sequences != nullptr;
  return launched();
}
bool attention_pages_dim_ok(uint32_t d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }
size_t attention_pages_scratch_bytes(const AttnPagesArgs& g) { return g.n * 64 + 256; }
cudaError_t launch_attention_pages(const AttnPagesArgs&, void*, int* launches, cudaStream_t) { *launches = 2; return launched(); }
cudaError_t launch_token_logprobs(const LogprobArgs&, cudaStream_t) { return launched(); }
cudaError_t launch_token_logprobs_backward(const LogprobGradArgs&, cudaStream_t) { return launched(); }
}  // namespace b200
