// The paged key/value cache: a projection's heads rotated and stored (`b200_rope_append_pages`), and one new token's
// attention over its sequence's pages (`b200_attention_pages`).
//
// Position p of sequence s lies in row table[s, p / page] * page + p % page of the pools.  Every index that comes from
// device memory (a position, a sequence, a page) is checked where it is read: a bad one sets the engine's error word to
// DOMAIN and nothing is read or written through it.
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
__device__ __forceinline__ void set_domain(int* err) { atomicCAS(err, 0, DOMAIN_ERROR); }

__device__ __forceinline__ float load_float(const void* p, uint64_t i, int bf16) {
  return bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(p)[i]) : reinterpret_cast<const float*>(p)[i];
}
__device__ __forceinline__ void store_float(void* p, uint64_t i, int bf16, float v) {
  if (bf16) reinterpret_cast<uint16_t*>(p)[i] = f32_to_bf16_bits(__float_as_uint(v));
  else reinterpret_cast<float*>(p)[i] = v;
}

// The pool row of a position, or -1 (with DOMAIN set) where the page is not one of the pool's.  `p` lies within the table.
__device__ __forceinline__ int64_t pool_row(const PageView& c, uint32_t s, uint32_t p, int* err) {
  const int32_t page = c.table[(uint64_t)s * c.width + p / c.page];
  if (page < 0 || (uint32_t)page >= c.pages) { set_domain(err); return -1; }
  return (int64_t)page * c.page + p % c.page;
}

// ---- append: a block a token.  x cos + swap(x) sin with the two products and the sum each rounded (`rope_blocks`' steps).
__global__ void __launch_bounds__(128) rope_append_kernel(AppendArgs g) {
  pdl_enter();
  const uint64_t i = blockIdx.x;
  const PageView& c = g.cache;
  const int32_t p = g.positions[i];
  const int64_t s = g.sequences ? (int64_t)g.sequences[i] : (int64_t)i;
  const uint32_t q_cols = c.heads * c.dim, kv_cols = c.kv_heads * c.dim;
  const uint32_t kept = q_cols + (g.keys_out ? kv_cols : 0);
  int64_t row = -1;
  if (p >= 0) {
    if (s < 0 || s >= c.sequences || (uint64_t)p >= (uint64_t)c.width * c.page || (g.rotary && (uint64_t)p >= g.table_rows)) set_domain(g.err);
    else row = pool_row(c, (uint32_t)s, (uint32_t)p, g.err);
  } else if (p < -1) set_domain(g.err);
  if (row < 0) {
    for (uint32_t j = threadIdx.x; j < kept; j += blockDim.x) store_float(g.out, i * kept + j, g.out_bf16, 0.f);
    return;
  }
  const uint32_t half = g.rotary / 2;
  for (uint32_t j = threadIdx.x; j < q_cols + kv_cols; j += blockDim.x) {
    const uint32_t e = j % c.dim;
    float v = load_float(g.qkv.p, i * g.qkv.ld + j, g.qkv.bf16);
    if (e < g.rotary) {
      const float w = load_float(g.qkv.p, i * g.qkv.ld + (e < half ? j + half : j - half), g.qkv.bf16);
      v = __fadd_rn(__fmul_rn(v, g.cos[(uint64_t)p * g.rotary + e]), __fmul_rn(w, g.sin[(uint64_t)p * g.rotary + e]));
    }
    if (j < kept) store_float(g.out, i * kept + j, g.out_bf16, v);
    if (j >= q_cols) store_float(c.keys, (uint64_t)row * kv_cols + (j - q_cols), c.bf16, v);
  }
  for (uint32_t j = threadIdx.x; j < kv_cols; j += blockDim.x)
    store_float(c.values, (uint64_t)row * kv_cols + j, c.bf16, load_float(g.qkv.p, i * g.qkv.ld + q_cols + kv_cols + j, g.qkv.bf16));
}

// ---- attention: a block a query head of a sequence, its positions in chunks of a thread each; the running maximum, sum and
// rows of a softmax (a chunk's new maximum scales what was summed before).
constexpr int CHUNK = 128;
__global__ void __launch_bounds__(CHUNK) attention_pages_kernel(AttnPagesArgs g) {
  pdl_enter();
  __shared__ float q[256], prob[CHUNK], red[CHUNK / 32];
  __shared__ int64_t rows[CHUNK];
  const PageView& c = g.cache;
  const uint32_t s = blockIdx.y, h = blockIdx.x, kvh = h / (c.heads / c.kv_heads), d = c.dim;
  const int tid = threadIdx.x;
  const uint64_t kv_cols = (uint64_t)c.kv_heads * d;
  const int32_t p = g.positions[s];
  const uint64_t dst = (uint64_t)s * c.heads * d + (uint64_t)h * d;
  int64_t n = (int64_t)p + 1;                         // positions 0 .. n - 1 are the sequence's
  if (p < -1 || n > (int64_t)c.width * c.page) { if (tid == 0) set_domain(g.err); n = 0; }
  const int64_t first = g.window && n > (int64_t)g.window ? n - g.window : 0;
  for (uint32_t e = tid; e < d; e += CHUNK) q[e] = load_float(g.q.p, (uint64_t)s * g.q.ld + (uint64_t)h * d + e, g.q.bf16);
  float acc[2] = {0.f, 0.f}, top = -FLT_MAX, sum = 0.f;
  for (int64_t at = first; at < n; at += CHUNK) {
    __syncthreads();
    const int64_t j = at + tid;
    float score = -INFINITY;
    int64_t row = -1;
    if (j < n) row = pool_row(c, s, (uint32_t)j, g.err);
    if (row >= 0) {
      float t = 0.f;
      for (uint32_t e = 0; e < d; ++e) t = fmaf(q[e], load_float(c.keys, (uint64_t)row * kv_cols + (uint64_t)kvh * d + e, c.bf16), t);
      score = t * g.scale;
    }
    rows[tid] = row;
    float m = score;
    for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if ((tid & 31) == 0) red[tid >> 5] = m;
    __syncthreads();
    float now = top;
    for (int w = 0; w < CHUNK / 32; ++w) now = fmaxf(now, red[w]);
    const float keep = expf(top - now);
    top = now;
    const float e = row >= 0 ? expf(score - now) : 0.f;
    prob[tid] = e;
    float t = e;
    for (int o = 16; o; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    __syncthreads();
    if ((tid & 31) == 0) red[tid >> 5] = t;
    __syncthreads();
    sum *= keep;
    for (int w = 0; w < CHUNK / 32; ++w) sum += red[w];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      const uint32_t col = tid + u * CHUNK;
      if (col >= d) break;
      float a = acc[u] * keep;
      for (int k = 0; k < CHUNK && at + k < n; ++k)
        if (rows[k] >= 0) a = fmaf(prob[k], load_float(c.values, (uint64_t)rows[k] * kv_cols + (uint64_t)kvh * d + col, c.bf16), a);
      acc[u] = a;
    }
  }
  const float den = sum < FLT_MIN ? FLT_MIN : sum;
#pragma unroll
  for (int u = 0; u < 2; ++u)
    if (tid + u * CHUNK < (int)d) store_float(g.out, dst + tid + u * CHUNK, g.out_bf16, acc[u] / den);
}

}  // namespace

cudaError_t launch_rope_append_pages(const AppendArgs& g, cudaStream_t stream) {
  if (g.n == 0) return cudaSuccess;
  launch_pdl(rope_append_kernel, dim3((unsigned)g.n), dim3(128), 0, stream, g);
  return cudaGetLastError();
}

bool attention_pages_dim_ok(uint32_t d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

cudaError_t launch_attention_pages(const AttnPagesArgs& g, cudaStream_t stream) {
  for (uint64_t at = 0; at < g.n; at += 65535) {
    AttnPagesArgs part = g;
    const uint64_t rows = g.n - at < 65535 ? g.n - at : 65535;
    part.cache.table += at * g.cache.width;
    part.positions += at;
    part.q.p = (const char*)g.q.p + at * g.q.ld * (g.q.bf16 ? 2 : 4);
    part.out = (char*)g.out + at * g.cache.heads * g.cache.dim * (g.out_bf16 ? 2 : 4);
    launch_pdl(attention_pages_kernel, dim3(g.cache.heads, (unsigned)rows), dim3(CHUNK), 0, stream, part);
    const cudaError_t e = cudaGetLastError();
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace b200
