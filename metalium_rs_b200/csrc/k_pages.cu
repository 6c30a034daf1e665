// The paged key/value cache's write: a projection's heads rotated and stored into the pages (`b200_rope_append_pages`).
//
// Position p of sequence s lies in row table[s, p / page] * page + p % page of the pools.  Every index that comes from
// device memory (a position, a sequence, a page) is checked where it is read: a bad one sets the engine's error word to
// DOMAIN and nothing is read or written through it.
#include <cstdint>
#include <cuda_runtime.h>

#include "device_math.cuh"
#include "kernels.h"
#include "pages.cuh"
#include "pdl.cuh"

namespace b200 {
namespace {

// ---- append ---------------------------------------------------------------------
// x cos + swap(x) sin with the two products and the sum each rounded (`rope_blocks`' steps).  Memory-bound: every element of
// the projection is read once and written once or twice.

// Token i's row of the pools; -1 for a padding row, and (with DOMAIN set) for a position or sequence outside its table.
__device__ __forceinline__ int64_t token_row(const AppendArgs& g, uint64_t i, int32_t p) {
  const int64_t s = g.sequences ? (int64_t)g.sequences[i] : (int64_t)i;
  if (p == -1) return -1;
  if (p < 0 || s < 0 || s >= g.cache.sequences || (uint64_t)p >= (uint64_t)g.cache.width * g.cache.page || (g.rotary && (uint64_t)p >= g.table_rows)) {
    set_domain(g.err);
    return -1;
  }
  return pool_row(g.cache, (uint32_t)s, (uint32_t)p, g.err);
}

struct Eight { float f[8]; };
__device__ __forceinline__ Eight load8(const void* p, uint64_t i, int bf16) {
  Eight v;
  if (bf16) {
    const uint4 w = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
    const uint32_t u[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) { v.f[2 * e] = __uint_as_float(u[e] << 16); v.f[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u); }
  } else {
    const float4* q = reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    const float4 a = q[0], b = q[1];
    v.f[0] = a.x; v.f[1] = a.y; v.f[2] = a.z; v.f[3] = a.w; v.f[4] = b.x; v.f[5] = b.y; v.f[6] = b.z; v.f[7] = b.w;
  }
  return v;
}
// Two values as BF16, `f32_to_bf16_bits` of each: the hardware's conversion where that is the same rounding (a zero, or at least
// 2^-126 in magnitude and not a NaN).
__device__ __forceinline__ uint32_t narrow2(float lo, float hi) {
  const uint32_t a = __float_as_uint(lo) & 0x7fffffffu, b = __float_as_uint(hi) & 0x7fffffffu;
  uint32_t w;
  if (min(a - 1u, b - 1u) < 0x007fffffu || max(a, b) > 0x7f800000u)
    return (uint32_t)f32_to_bf16_bits(__float_as_uint(lo)) | ((uint32_t)f32_to_bf16_bits(__float_as_uint(hi)) << 16);
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w) : "f"(hi), "f"(lo));
  return w;
}
__device__ __forceinline__ void store8(void* p, uint64_t i, int bf16, const Eight& v) {
  if (bf16) {
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) =
        make_uint4(narrow2(v.f[0], v.f[1]), narrow2(v.f[2], v.f[3]), narrow2(v.f[4], v.f[5]), narrow2(v.f[6], v.f[7]));
  } else {
    float4* q = reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i);
    q[0] = make_float4(v.f[0], v.f[1], v.f[2], v.f[3]);
    q[1] = make_float4(v.f[4], v.f[5], v.f[6], v.f[7]);
  }
}

struct Four { float f[4]; };
__device__ __forceinline__ Four load4(const void* p, uint64_t i, int bf16) {
  Four v;
  if (bf16) {
    const uint2 w = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
    v.f[0] = __uint_as_float(w.x << 16); v.f[1] = __uint_as_float(w.x & 0xffff0000u);
    v.f[2] = __uint_as_float(w.y << 16); v.f[3] = __uint_as_float(w.y & 0xffff0000u);
  } else {
    const float4 a = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(p) + i);
    v.f[0] = a.x; v.f[1] = a.y; v.f[2] = a.z; v.f[3] = a.w;
  }
  return v;
}
__device__ __forceinline__ void store4(void* p, uint64_t i, int bf16, const Four& v) {
  if (bf16) *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(p) + i) = make_uint2(narrow2(v.f[0], v.f[1]), narrow2(v.f[2], v.f[3]));
  else *reinterpret_cast<float4*>(reinterpret_cast<float*>(p) + i) = make_float4(v.f[0], v.f[1], v.f[2], v.f[3]);
}

// Values that are only moved keep their bits where both sides are of one type.
__device__ __forceinline__ void move8(void* to, uint64_t j, int to_bf16, const void* from, uint64_t i, int from_bf16) {
  if (to_bf16 && from_bf16)
    *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(to) + j) = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(from) + i);
  else store8(to, j, to_bf16, load8(from, i, from_bf16));
}
__device__ __forceinline__ void move4(void* to, uint64_t j, int to_bf16, const void* from, uint64_t i, int from_bf16) {
  if (to_bf16 && from_bf16)
    *reinterpret_cast<uint2*>(reinterpret_cast<uint16_t*>(to) + j) = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(from) + i);
  else store4(to, j, to_bf16, load4(from, i, from_bf16));
}
__device__ __forceinline__ void move1(void* to, uint64_t j, int to_bf16, const void* from, uint64_t i, int from_bf16) {
  if (to_bf16 && from_bf16) reinterpret_cast<uint16_t*>(to)[j] = reinterpret_cast<const uint16_t*>(from)[i];
  else store_float(to, j, to_bf16, load_float(from, i, from_bf16));
}

// Elements as they lie: asked for early, taken apart where they are used.
struct Raw4 {
  uint4 w;
  __device__ __forceinline__ void load(const void* p, uint64_t i, int bf16) {
    if (bf16) {
      const uint2 u = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint16_t*>(p) + i);
      w.x = u.x; w.y = u.y;
    } else w = *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
  }
  __device__ __forceinline__ Four widen(int bf16) const {
    if (bf16) return Four{{__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xffff0000u), __uint_as_float(w.y << 16), __uint_as_float(w.y & 0xffff0000u)}};
    return Four{{__uint_as_float(w.x), __uint_as_float(w.y), __uint_as_float(w.z), __uint_as_float(w.w)}};
  }
};
__device__ __forceinline__ void load_raw8(uint4 (&w)[2], const void* p, uint64_t i, int bf16) {
  if (bf16) w[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const uint16_t*>(p) + i);
  else {
    w[0] = *reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i);
    w[1] = *(reinterpret_cast<const uint4*>(reinterpret_cast<const float*>(p) + i) + 1);
  }
}
__device__ __forceinline__ void store_raw8(void* p, uint64_t i, int to_bf16, const uint4 (&w)[2], int from_bf16) {
  if (from_bf16 && to_bf16) { *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p) + i) = w[0]; return; }
  Eight v;
  const uint32_t u[8] = {w[0].x, w[0].y, w[0].z, w[0].w, w[1].x, w[1].y, w[1].z, w[1].w};
#pragma unroll
  for (int e = 0; e < 8; ++e) v.f[e] = __uint_as_float(from_bf16 ? (e & 1 ? u[e / 2] & 0xffff0000u : u[e / 2] << 16) : u[e]);
  store8(p, i, to_bf16, v);
}

// A block a token: thread (x, y) takes columns 4x of the low half of a rotation and the four across from them -- or, behind the
// rotation, four columns that stay -- in heads y, y + blockDim.y, ..., so that its cos and sin entries are read once for all of
// its heads (read again for every head they were twice the projection's bytes).  Four and not eight columns: the entries of eight
// are 32 registers, and the warps they cost are worth more than the wider loads.  8 prompts of 1000 tokens, 32 and 8 heads of 128
// in BF16: 39.0 us, 4.6 TB/s (eight columns 47.7; four without the early loads 44.7).
__global__ void __launch_bounds__(512) rope_append_kernel(const __grid_constant__ AppendArgs g) {
  pdl_enter();
  const uint64_t i = blockIdx.x;
  const PageView& c = g.cache;
  const uint32_t d = c.dim, half = g.rotary / 2, pairs = half / 4, turned = c.heads + c.kv_heads;
  const uint32_t kept = c.heads + (g.keys_out ? c.kv_heads : 0), threads = blockDim.x * blockDim.y;
  const uint32_t tid = threadIdx.y * blockDim.x + threadIdx.x;
  const bool pair = threadIdx.x < pairs;
  const uint32_t e0 = pair ? threadIdx.x * 4 : g.rotary + (threadIdx.x - pairs) * 4;
  const uint64_t from = i * g.qkv.ld, to = i * (uint64_t)kept * d;
  // Everything that can be asked for is, before the first of it is waited for: the position, the first head and values, then the
  // page and the tables' entries (a token's chain of trips to memory is what a block's time is).
  const int32_t p = g.positions[i];
  const uint64_t kv_cols = (uint64_t)c.kv_heads * d;
  Raw4 a0, b0;
  uint4 v0[2];
  if (threadIdx.y < turned) {
    a0.load(g.qkv.p, from + (uint64_t)threadIdx.y * d + e0, g.qkv.bf16);
    if (pair) b0.load(g.qkv.p, from + (uint64_t)threadIdx.y * d + half + e0, g.qkv.bf16);
  }
  const bool valued = tid < kv_cols / 8;
  if (valued) load_raw8(v0, g.qkv.p, from + (uint64_t)turned * d + tid * 8, g.qkv.bf16);
  Four c0, c1, s0, s1;
  if (pair && p >= 0 && (uint64_t)p < g.table_rows) {
    const uint64_t w = (uint64_t)p * g.rotary;
    c0 = load4(g.cos, w + e0, 0); c1 = load4(g.cos, w + half + e0, 0); s0 = load4(g.sin, w + e0, 0); s1 = load4(g.sin, w + half + e0, 0);
  }
  const int64_t row = token_row(g, i, p);
  if (row < 0) {
    const Eight zero = {{0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}};
    for (uint32_t j = tid; j < kept * d / 8; j += threads) store8(g.out, to + j * 8, g.out_bf16, zero);
    return;
  }
  const uint64_t at = (uint64_t)row * kv_cols;
  if (valued) store_raw8(c.values, at + tid * 8, c.bf16, v0, g.qkv.bf16);
  for (uint32_t j = tid + threads; j < kv_cols / 8; j += threads)
    move8(c.values, at + j * 8, c.bf16, g.qkv.p, from + (uint64_t)turned * d + j * 8, g.qkv.bf16);
  if (pair) {
    for (uint32_t h = threadIdx.y; h < turned; h += blockDim.y) {
      const Four a = a0.widen(g.qkv.bf16), b = b0.widen(g.qkv.bf16);
      if (h + blockDim.y < turned) {     // the next head's, before this one's stores
        a0.load(g.qkv.p, from + (uint64_t)(h + blockDim.y) * d + e0, g.qkv.bf16);
        b0.load(g.qkv.p, from + (uint64_t)(h + blockDim.y) * d + half + e0, g.qkv.bf16);
      }
      Four lo, hi;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        lo.f[e] = __fadd_rn(__fmul_rn(a.f[e], c0.f[e]), __fmul_rn(b.f[e], s0.f[e]));
        hi.f[e] = __fadd_rn(__fmul_rn(b.f[e], c1.f[e]), __fmul_rn(a.f[e], s1.f[e]));
      }
      if (h < kept) {
        store4(g.out, to + (uint64_t)h * d + e0, g.out_bf16, lo);
        store4(g.out, to + (uint64_t)h * d + half + e0, g.out_bf16, hi);
      }
      if (h >= c.heads) {
        store4(c.keys, at + (uint64_t)(h - c.heads) * d + e0, c.bf16, lo);
        store4(c.keys, at + (uint64_t)(h - c.heads) * d + half + e0, c.bf16, hi);
      }
    }
  } else {
    for (uint32_t h = threadIdx.y; h < turned; h += blockDim.y) {
      const uint64_t x = from + (uint64_t)h * d + e0;
      if (h < kept) move4(g.out, to + (uint64_t)h * d + e0, g.out_bf16, g.qkv.p, x, g.qkv.bf16);
      if (h >= c.heads) move4(c.keys, at + (uint64_t)(h - c.heads) * d + e0, c.bf16, g.qkv.p, x, g.qkv.bf16);
    }
  }
}

// Blocks that start at no 16-byte address, and heads or rotations that are not groups of eight columns: an element a thread.  The 8
// prompts of 1000 tokens above, their block one column into a wider buffer: 124 us (39.0 by the kernel above): an element
// costs a division by the head's width and three addresses.
__global__ void __launch_bounds__(128) rope_append_any_kernel(const __grid_constant__ AppendArgs g) {
  pdl_enter();
  const uint64_t i = blockIdx.x;
  const PageView& c = g.cache;
  const uint32_t q_cols = c.heads * c.dim, kv_cols = c.kv_heads * c.dim, half = g.rotary / 2;
  const uint32_t kept = q_cols + (g.keys_out ? kv_cols : 0);
  const int32_t p = g.positions[i];
  const int64_t row = token_row(g, i, p);
  if (row < 0) {
    for (uint32_t j = threadIdx.x; j < kept; j += blockDim.x) store_float(g.out, i * kept + j, g.out_bf16, 0.f);
    return;
  }
  for (uint32_t j = threadIdx.x; j < q_cols + kv_cols; j += blockDim.x) {
    const uint32_t e = j % c.dim;
    if (e >= g.rotary) {
      if (j < kept) move1(g.out, i * kept + j, g.out_bf16, g.qkv.p, i * g.qkv.ld + j, g.qkv.bf16);
      if (j >= q_cols) move1(c.keys, (uint64_t)row * kv_cols + (j - q_cols), c.bf16, g.qkv.p, i * g.qkv.ld + j, g.qkv.bf16);
    } else {
      float v = load_float(g.qkv.p, i * g.qkv.ld + j, g.qkv.bf16);
      const float w = load_float(g.qkv.p, i * g.qkv.ld + (e < half ? j + half : j - half), g.qkv.bf16);
      v = __fadd_rn(__fmul_rn(v, g.cos[(uint64_t)p * g.rotary + e]), __fmul_rn(w, g.sin[(uint64_t)p * g.rotary + e]));
      if (j < kept) store_float(g.out, i * kept + j, g.out_bf16, v);
      if (j >= q_cols) store_float(c.keys, (uint64_t)row * kv_cols + (j - q_cols), c.bf16, v);
    }
  }
  for (uint32_t j = threadIdx.x; j < kv_cols; j += blockDim.x)
    move1(c.values, (uint64_t)row * kv_cols + j, c.bf16, g.qkv.p, i * g.qkv.ld + q_cols + kv_cols + j, g.qkv.bf16);
}

}  // namespace

cudaError_t launch_rope_append_pages(const AppendArgs& g, cudaStream_t stream) {
  if (g.n == 0) return cudaSuccess;
  const uint32_t d = g.cache.dim, lanes = g.rotary / 8 + (d - g.rotary) / 4;    // of a head: pairs of four columns, then fours
  const uintptr_t ends = reinterpret_cast<uintptr_t>(g.qkv.p) | reinterpret_cast<uintptr_t>(g.cos) | reinterpret_cast<uintptr_t>(g.sin) |
                         g.qkv.ld * (g.qkv.bf16 ? 2 : 4);
  if (ends % 16 == 0 && d % 8 == 0 && g.rotary % 8 == 0 && lanes <= 512) {
    // few tokens: a thread for every piece, so that a token's chain of loads is short (one token of 32 and 8 heads of 128 by 512 threads
    // 4.6 us, by 64 8.5; 592 of them 9.1 and 10.3); many: blocks of 64, as many tokens at once (2,400 19.7 us, by 512 29.4)
    const uint32_t want = g.n <= 592 ? 512 : 64, heads = g.cache.heads + g.cache.kv_heads;
    uint32_t y = want / lanes;
    y = y < 1 ? 1 : (y > heads ? heads : y);
    launch_pdl(rope_append_kernel, dim3((unsigned)g.n), dim3(lanes, y), 0, stream, g);
  } else {
    launch_pdl(rope_append_any_kernel, dim3((unsigned)g.n), dim3(128), 0, stream, g);
  }
  return cudaGetLastError();
}

}  // namespace b200
