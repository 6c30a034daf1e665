// What the serving kernels share: the error word's value, element loads and stores, the exponential, the check of a page number.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "device_math.cuh"
#include "kernels.h"

namespace b200 {
namespace {

constexpr int DOMAIN_ERROR = 6;
__device__ __forceinline__ void set_domain(int* err) { atomicCAS(err, 0, DOMAIN_ERROR); }

__device__ __forceinline__ float load_float(const void* p, uint64_t i, int bf16) {
  return bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_float(void* p, uint64_t i, int bf16, float v) {
  if (bf16) reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(__float_as_uint(v));
  else reinterpret_cast<float*>(p)[i] = v;
}

__device__ __forceinline__ float exp2_fast(float x) {   // the hardware's 2^x: 2 units in the last place, 2^-200 and 2^-inf = 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}

// The pool row of a position, or -1 (with DOMAIN set) where the page is not one of the pool's.  `p` lies within the table.
__device__ __forceinline__ int64_t pool_row(const PageView& c, uint32_t s, uint32_t p, int* err) {
  const int32_t page = c.table[(uint64_t)s * c.width + p / c.page];
  if (page < 0 || (uint32_t)page >= c.pages) { set_domain(err); return -1; }
  return (int64_t)page * c.page + p % c.page;
}

}  // namespace
}  // namespace b200
