// Log probabilities of given tokens, entropy and the largest alternatives of each row of logits
// (`b200_token_logprobs`), and their gradient (`b200_token_logprobs_backward`).
//
// With y = scale x, m = max y, S = sum e^(y - m) and T = sum e^(y - m) (y - m):
//   lse = m + log S,   log p_j = (y_j - m) - log S,   entropy = log S - T / S.
// Both terms of the entropy are of one sign (T <= 0), so nothing cancels.  Values are ordered as `argmax_row` orders them
// (a NaN above everything, -0 equal to +0, equal values by the lower column): one 64-bit key a value.
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cuda_runtime.h>

#include "device_math.cuh"
#include "kernels.h"
#include "pdl.cuh"

namespace b200 {
namespace {

constexpr int DOMAIN_ERROR = 6;
constexpr int THREADS = 256;

__device__ __forceinline__ float load_float(const void* p, uint64_t i, int bf16) {
  return bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}

// Larger key: larger value, or the same value in a lower column.  Every key lies strictly between 0 and ~0 (a NaN's upper word
// is 0xfffffffe, -inf's 0x007fffff), so both can stand for "none".
__device__ __forceinline__ uint64_t key_of(float v, uint32_t col) {
  uint32_t u = __float_as_uint(v + 0.f);                 // -0 + 0 = +0
  u = v != v ? 0xfffffffeu : (u & 0x80000000u ? ~u : u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~col;
}

template <typename T, typename F>
__device__ __forceinline__ T block_fold(T v, T* sh, F f) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
  __syncthreads();
  v = sh[0];
  for (int w = 1; w < THREADS / 32; ++w) v = f(v, sh[w]);
  return v;
}

// A block a row: the maximum, then the sums under it, then the largest keys one after another.
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(LogprobArgs g) {
  pdl_enter();
  __shared__ float shf[THREADS / 32];
  __shared__ uint64_t shk[THREADS / 32];
  const uint64_t r = blockIdx.x, base = r * g.cols;
  const int tid = threadIdx.x;
  const auto add = [](float a, float b) { return a + b; };
  float m = -FLT_MAX;
  for (uint64_t j = tid; j < g.cols; j += THREADS) m = fmaxf(m, load_float(g.logits, base + j, g.bf16) * g.scale);
  m = block_fold(m, shf, [](float a, float b) { return fmaxf(a, b); });
  float sum = 0.f, dot = 0.f;
  for (uint64_t j = tid; j < g.cols; j += THREADS) {
    const float z = load_float(g.logits, base + j, g.bf16) * g.scale - m, e = expf(z);
    sum += e;
    if (e != 0.f) dot += e * z;                          // an entry of -inf adds nothing
  }
  sum = block_fold(sum, shf, add);
  dot = block_fold(dot, shf, add);
  const bool empty = sum == 0.f;                         // a row of -inf
  const float log_sum = empty ? -INFINITY : logf(sum);
  if (tid == 0) {
    g.lse[r] = empty ? -INFINITY : m + log_sum;
    g.entropy[r] = empty ? 0.f : log_sum - dot / sum;
    const int32_t id = g.ids[r];
    float lp = 0.f;
    if (id < -1 || (id >= 0 && (uint64_t)id >= g.cols)) atomicCAS(g.err, 0, DOMAIN_ERROR);
    else if (id >= 0) lp = empty ? -INFINITY : (load_float(g.logits, base + id, g.bf16) * g.scale - m) - log_sum;
    g.logprob[r] = lp;
  }
  uint64_t last = ~0ull;
  for (uint32_t k = 0; k < g.top; ++k) {
    uint64_t best = 0;
    for (uint64_t j = tid; j < g.cols; j += THREADS) {
      const uint64_t key = key_of(load_float(g.logits, base + j, g.bf16), (uint32_t)j);
      if (key < last && key > best) best = key;
    }
    best = block_fold(best, shk, [](uint64_t a, uint64_t b) { return a > b ? a : b; });
    last = best;
    if (tid == 0) {
      const uint32_t col = ~(uint32_t)best;
      g.top_ids[r * g.top + k] = (int32_t)col;
      g.top_logprobs[r * g.top + k] = empty ? -INFINITY : (load_float(g.logits, base + col, g.bf16) * g.scale - m) - log_sum;
    }
  }
}

// A block a row: scale (g (1[j = id] - p) - h p (y - lse + H)), p = e^(y - lse).
__global__ void __launch_bounds__(THREADS) token_logprobs_backward_kernel(LogprobGradArgs g) {
  pdl_enter();
  const uint64_t r = blockIdx.x, base = r * g.cols;
  const float lse = g.lse[r], h = g.d_entropy ? g.d_entropy[r] : 0.f, H = g.d_entropy ? g.entropy[r] : 0.f;
  int64_t id = g.ids[r];
  if (id < -1 || id >= (int64_t)g.cols) { if (threadIdx.x == 0) atomicCAS(g.err, 0, DOMAIN_ERROR); id = -1; }
  const float up = id >= 0 ? g.d_logprob[r] : 0.f;
  for (uint64_t j = threadIdx.x; j < g.cols; j += THREADS) {
    float v = 0.f;
    if (lse != -INFINITY) {
      const float z = load_float(g.logits, base + j, g.bf16) * g.scale - lse, p = expf(z);
      v = up * ((int64_t)j == id ? 1.f - p : -p);
      if (g.d_entropy && p != 0.f) v -= h * (p * (z + H));
      v *= g.scale;
    }
    if (g.out_bf16) reinterpret_cast<uint16_t*>(g.out)[base + j] = f32_to_bf16_bits(__float_as_uint(v));
    else reinterpret_cast<float*>(g.out)[base + j] = v;
  }
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& g, cudaStream_t stream) {
  if (g.rows == 0) return cudaSuccess;
  launch_pdl(token_logprobs_kernel, dim3((unsigned)g.rows), dim3(THREADS), 0, stream, g);
  return cudaGetLastError();
}

cudaError_t launch_token_logprobs_backward(const LogprobGradArgs& g, cudaStream_t stream) {
  if (g.rows == 0) return cudaSuccess;
  launch_pdl(token_logprobs_backward_kernel, dim3((unsigned)g.rows), dim3(THREADS), 0, stream, g);
  return cudaGetLastError();
}

}  // namespace b200
