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
constexpr int CLUSTER = 8;               // blocks that share a row, at most
constexpr int TOP = 32;                  // alternatives a row, at most
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

__device__ __forceinline__ float exp2_fast(float x) {   // the hardware's 2^x: 2 units in the last place, 2^-200 = 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// Larger key: larger value, or the same value in a lower column.  Every key lies strictly between 0 and ~0 (a NaN's upper word
// is 0xfffffffe, -inf's 0x007fffff), so both can stand for "none".
__device__ __forceinline__ uint64_t key_of(float v, uint32_t col) {
  uint32_t u = __float_as_uint(v + 0.f);                 // -0 + 0 = +0
  u = v != v ? 0xfffffffeu : (u & 0x80000000u ? ~u : u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~col;
}
__device__ __forceinline__ uint32_t col_of(uint64_t key) { return ~(uint32_t)key; }

template <typename T> struct Vec;        // a 16-byte piece of a row
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void widen(const uint4& w, float* f) {
    f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
  }
};
template <> struct Vec<uint16_t> {
  static constexpr int N = 8;
  static __device__ __forceinline__ float one(const uint16_t* p) { return bf16_bits_to_f32(*p); }
  static __device__ __forceinline__ void widen(const uint4& w, float* f) {
    f[0] = __uint_as_float(w.x << 16); f[1] = __uint_as_float(w.x & 0xffff0000u);
    f[2] = __uint_as_float(w.y << 16); f[3] = __uint_as_float(w.y & 0xffff0000u);
    f[4] = __uint_as_float(w.z << 16); f[5] = __uint_as_float(w.z & 0xffff0000u);
    f[6] = __uint_as_float(w.w << 16); f[7] = __uint_as_float(w.w & 0xffff0000u);
  }
};

// ---- sorted lists of 32 keys, one a lane, the largest first
__device__ __forceinline__ uint64_t order_pair(uint64_t v, int lane, int apart, bool falling) {
  const uint64_t o = __shfl_xor_sync(0xffffffffu, v, apart);
  return ((lane & apart) == 0) == falling ? (v > o ? v : o) : (v < o ? v : o);
}
__device__ __forceinline__ uint64_t sort32(uint64_t v, int lane) {
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1)
#pragma unroll
    for (int j = k / 2; j; j >>= 1) v = order_pair(v, lane, j, (lane & k) == 0);
  return v;
}
// The largest 32 of two sorted lists: lane i's larger of a[i] and b[31 - i] is a bitonic list of them.
__device__ __forceinline__ uint64_t merge32(uint64_t a, uint64_t b_reversed, int lane) {
  uint64_t v = a > b_reversed ? a : b_reversed;
#pragma unroll
  for (int j = 16; j; j >>= 1) v = order_pair(v, lane, j, true);
  return v;
}

// Sums under a maximum: m in units of log2, s = sum 2^(y - m), t = sum 2^(y - m) (y - m), y = x scale log2 e.
struct Sums { float m, s, t; };
__device__ __forceinline__ Sums under(const Sums& a, float m) {       // a's sums under another, larger maximum
  const float d = a.m - m, f = exp2_fast(d);
  return Sums{m, a.s * f, a.s == 0.f ? 0.f : f * fmaf(a.s, d, a.t)};  // nothing summed stays nothing, however far the maximum moved
}
__device__ __forceinline__ Sums both(const Sums& a, const Sums& b) {
  const float m = fmaxf(a.m, b.m);
  const Sums x = under(a, m), y = under(b, m);
  return Sums{m, x.s + y.s, x.t + y.t};
}

// A block's slice of a row: 16-byte pieces from the address below its start, the pieces of thread i being i, i + THREADS, ...
template <typename T, int THREADS> struct Slice {
  const T* row;                          // the row's first element
  int64_t first, last;                   // the slice's columns
  int64_t origin;                        // the column of piece 0's first element: at most first, aligned in memory
  uint32_t pieces;
  __device__ Slice(const T* r, int64_t a, int64_t b) : row(r), first(a), last(b) {
    const int64_t off = (int64_t)((reinterpret_cast<uintptr_t>(r + a) & 15) / sizeof(T));
    origin = a - off;
    pieces = b > a ? (uint32_t)((b - origin + Vec<T>::N - 1) / Vec<T>::N) : 0;
  }
  __device__ __forceinline__ bool whole(uint32_t u) const {
    const int64_t c = origin + (int64_t)u * Vec<T>::N;
    return c >= first && c + Vec<T>::N <= last;
  }
  __device__ __forceinline__ uint4 raw(uint32_t u) const { return __ldg(reinterpret_cast<const uint4*>(row + origin) + u); }
  // a piece's values; those outside the slice are -inf
  __device__ __forceinline__ void load(uint32_t u, float* x) const {
    if (whole(u)) { Vec<T>::widen(raw(u), x); return; }
#pragma unroll
    for (int e = 0; e < Vec<T>::N; ++e) {
      const int64_t c = origin + (int64_t)u * Vec<T>::N + e;
      x[e] = c >= first && c < last ? Vec<T>::one(row + c) : -INFINITY;
    }
  }
};

// One more group of a thread's values: its largest so far and the sums under it.
template <int N>
__device__ __forceinline__ void take(const float (&x)[N], float c, float& best, Sums& a) {
  float top = x[0];
#pragma unroll
  for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
  if (top > best) {
    best = top;
    a = under(a, fmaxf(top * c, -FLT_MAX));
  }
#pragma unroll
  for (int e = 0; e < N; ++e) {
    const float z = max_nan(fmaf(x[e], c, -a.m), -200.f), p = exp2_fast(z);
    a.s += p;
    a.t = fmaf(p, z, a.t);
  }
}

// The slice's `top` largest keys, one after another: for slices with a NaN or with more candidates than the list holds.
template <typename T, int THREADS>
__device__ void slow_top(const Slice<T, THREADS>& sl, uint32_t top, uint64_t* list, uint64_t* sh) {
  const int tid = threadIdx.x;
  uint64_t bound = ~0ull;
  for (uint32_t k = 0; k < TOP; ++k) {
    uint64_t best = 0;
    if (k < top)
      for (int64_t c = sl.first + tid; c < sl.last; c += THREADS) {
        const uint64_t key = key_of(Vec<T>::one(sl.row + c), (uint32_t)c);
        if (key < bound && key > best) best = key;
      }
#pragma unroll
    for (int o = 16; o; o >>= 1) {
      const uint64_t w = __shfl_xor_sync(0xffffffffu, best, o);
      best = w > best ? w : best;
    }
    __syncthreads();
    if ((tid & 31) == 0) sh[tid >> 5] = best;
    __syncthreads();
    for (int w = 0; w < THREADS / 32; ++w) best = sh[w] > best ? sh[w] : best;
    if (tid == 0) list[k] = best;
    bound = best;                        // 0 once the slice has no more: nothing is below it
  }
  __syncthreads();
}

// A row a block, or a row a cluster of blocks with a slice each (SHARED).  One pass keeps each thread's sums and its largest
// value.  The `top` largest of the threads' largest bound the row's `top` largest from below, and only the threads that hold
// them can hold one: their pieces alone are read again (from L2), what reaches the bound is listed, and the list is sorted.
template <typename T, int THREADS, bool SHARED>
__global__ void __launch_bounds__(THREADS) token_logprobs_kernel(const __grid_constant__ LogprobArgs g) {
  constexpr int WARPS = THREADS / 32, N = Vec<T>::N, HELD = THREADS >= 256 ? 1024 : 512;
  __shared__ uint64_t lists[WARPS][TOP], held[HELD], sh[WARPS], slices[SHARED ? CLUSTER : 1][TOP];
  __shared__ Sums warp_sums[WARPS], slice_sums[SHARED ? CLUSTER : 1];
  __shared__ float warp_best[WARPS], slice_best[SHARED ? CLUSTER : 1];
  __shared__ uint32_t count;
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank = 0, size = 1;
  if constexpr (SHARED) {
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
    asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");   // waited for before another block's memory is written
  }
  const uint64_t r = blockIdx.x / size;
  const T* row = reinterpret_cast<const T*>(g.logits) + r * g.cols;
  const int64_t cols = (int64_t)g.cols, seg = (cols + size - 1) / size;
  const Slice<T, THREADS> sl(row, rank * seg < cols ? rank * seg : cols, (rank + 1) * seg < cols ? (rank + 1) * seg : cols);
  const float c = g.scale * LOG2E;
  if (tid == 0) count = 0;

  // ---- the pass: four pieces of a thread asked for before the first is used; the slice's cut ends by themselves
  Sums a{-FLT_MAX, 0.f, 0.f};
  float best = -INFINITY;
  const uint32_t lo = sl.pieces && !sl.whole(0) ? 1u : 0u, hi = sl.pieces && !sl.whole(sl.pieces - 1) ? sl.pieces - 1 : sl.pieces;
  uint32_t best_piece = (uint32_t)tid;   // the first piece that holds `best`
  const auto edge = [&](uint32_t u) {
    float x[N];
    sl.load(u, x);
    const float was = best;
    take<N>(x, c, best, a);
    if (best > was) best_piece = u;
  };
  if (lo && tid == 0) edge(0);
  for (uint32_t u = lo && tid == 0 ? THREADS : tid; u < hi; u += 4 * THREADS) {
    uint4 w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (u + i * THREADS < hi) w[i] = sl.raw(u + i * THREADS);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (u + i * THREADS < hi) {
        float x[N];
        Vec<T>::widen(w[i], x);
        const float was = best;
        take<N>(x, c, best, a);
        if (best > was) best_piece = u + i * THREADS;
      }
  }
  if (hi < sl.pieces && hi >= lo && sl.pieces > lo && tid == (int)(hi % THREADS)) edge(hi);

  // ---- the slice's sums
  Sums all = a;
  float high = best;
#pragma unroll
  for (int o = 16; o; o >>= 1) {
    const Sums b{__shfl_xor_sync(0xffffffffu, all.m, o), __shfl_xor_sync(0xffffffffu, all.s, o), __shfl_xor_sync(0xffffffffu, all.t, o)};
    all = both(all, b);
    high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  }
  if (lane == 0) { warp_sums[warp] = all; warp_best[warp] = high; }
  const uint32_t top = g.top;
  const uint32_t threads = sl.pieces < (uint32_t)THREADS ? sl.pieces : (uint32_t)THREADS;   // those that hold a piece
  if (top && threads >= top) {
    uint64_t key = 0;
    if (tid < (int)sl.pieces) {
      // the lowest column of the piece with that value; a thread whose values are all -inf has its first
      float x[N];
      sl.load(best_piece, x);
      int at = -1;
#pragma unroll
      for (int e = N - 1; e >= 0; --e) {
        const int64_t col = sl.origin + (int64_t)best_piece * N + e;
        if (x[e] == best && col >= sl.first && col < sl.last) at = e;
      }
      key = at < 0 ? 0 : key_of(best, (uint32_t)(sl.origin + (int64_t)best_piece * N + at));
    }
    lists[warp][lane] = sort32(key, lane);
  }
  __syncthreads();
  all = warp_sums[0];
  high = warp_best[0];
  for (int w = 1; w < WARPS; ++w) { all = both(all, warp_sums[w]); high = fmaxf(high, warp_best[w]); }

  // ---- the slice's largest
  if (top) {
    bool slow = all.s != all.s;          // a NaN or +inf: the maxima above passed over it
    uint64_t bound = 0;
    if (!slow && threads >= top) {
#pragma unroll
      for (int half = WARPS / 2; half; half >>= 1) {
        uint64_t v = 0;
        if (warp < half) v = merge32(lists[warp][lane], lists[warp + half][31 - lane], lane);
        __syncthreads();
        if (warp < half) lists[warp][lane] = v;
        __syncthreads();
      }
      bound = lists[0][top - 1];
    }
    if (!slow) {
      const uint32_t each = (sl.pieces + THREADS - 1) / THREADS, owners = threads >= top ? top : threads;
      for (uint32_t i = tid; i < owners * each; i += THREADS) {
        const uint32_t o = i / each;
        const uint32_t owner = threads >= top ? (uint32_t)(((int64_t)col_of(lists[0][o]) - sl.origin) / N % THREADS) : o;
        const uint32_t u = owner + i % each * THREADS;
        if (u < sl.pieces) {
          float x[N];
          sl.load(u, x);
#pragma unroll
          for (int e = 0; e < N; ++e) {
            const int64_t col = sl.origin + (int64_t)u * N + e;
            if (col >= sl.first && col < sl.last) {
              const uint64_t key = key_of(x[e], (uint32_t)col);
              if (key >= bound) {
                const uint32_t k = atomicAdd(&count, 1u);
                if (k < (uint32_t)HELD) held[k] = key;
              }
            }
          }
        }
      }
      __syncthreads();
      slow = count > (uint32_t)HELD;
    }
    if (slow) {
      slow_top(sl, top, lists[0], sh);
    } else if (warp == 0) {
      // the list's order depends on the atomics, its keys do not, and no two are equal
      uint64_t v = 0;
      for (uint32_t i = 0; i < count; i += 32) {
        const uint64_t x = sort32(i + lane < count ? held[i + lane] : 0, lane);
        v = i ? merge32(v, __shfl_sync(0xffffffffu, x, 31 - lane), lane) : x;
      }
      lists[0][lane] = v;
    }
    __syncthreads();
  }

  // ---- the row, from its slices in their order
  if constexpr (SHARED) {
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const auto there = [](const void* p) {
      uint32_t a;
      asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(p)), "r"(0));
      return a;
    };
    if (tid == 0) {
      const uint32_t at = there(&slice_sums[rank]);
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at), "f"(all.m) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 4), "f"(all.s) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(at + 8), "f"(all.t) : "memory");
      asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(there(&slice_best[rank])), "f"(high) : "memory");
    }
    if (top && warp == 0) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(there(&slices[rank][lane])), "l"(lists[0][lane]) : "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank) return;
    all = slice_sums[0];
    high = slice_best[0];
    for (uint32_t w = 1; w < size; ++w) { all = both(all, slice_sums[w]); high = fmaxf(high, slice_best[w]); }
    if (top && warp == 0) {
      uint64_t v = slices[0][lane];
      for (uint32_t w = 1; w < size; ++w) v = merge32(v, slices[w][31 - lane], lane);
      lists[0][lane] = v;
    }
  }

  // y - lse and the statistics.  The pass's terms are 2^(x c - fl(high c)): the reference's rounding cancels in the results, but it
  // is a factor of up to 2^(|high c| 2^-24) on every term, and a product may leave the type's range (a row masked by the type's
  // lowest value).  Rows with a reference from 1e8 on are taken again from differences to their largest.
  float ref = all.m * LN2, log_sum = logf(all.s), entropy = log_sum - LN2 * all.t / all.s;
  const bool none = high == -INFINITY && all.s == 0.f;     // -inf only
  const bool plain = none || !(fabsf(high) <= FLT_MAX) || fabsf(high * c) < 1e8f;
  if (none) { ref = -INFINITY; log_sum = 0.f; entropy = 0.f; }
  if (!plain) {
    float s = 0.f, t = 0.f;
    for (int64_t j = tid; j < cols; j += THREADS) {
      const float z = (Vec<T>::one(row + j) - high) * g.scale, p = expf(z);
      s += p;
      if (p != 0.f) t += p * z;
    }
#pragma unroll
    for (int o = 16; o; o >>= 1) { s += __shfl_xor_sync(0xffffffffu, s, o); t += __shfl_xor_sync(0xffffffffu, t, o); }
    __syncthreads();
    if (lane == 0) warp_sums[warp] = Sums{0.f, s, t};
    __syncthreads();
    s = t = 0.f;
    for (int w = 0; w < WARPS; ++w) { s += warp_sums[w].s; t += warp_sums[w].t; }
    ref = high * g.scale; log_sum = logf(s); entropy = log_sum - t / s;
  }
  const auto log_prob = [&](float x) {
    if (none) return -INFINITY;
    // a masked logit's product with log2 e may leave the type's range although its product with the scale does not
    return (plain && fabsf(x) < 1e37f ? LN2 * fmaf(x, c, -all.m) : plain ? x * g.scale - ref : (x - high) * g.scale) - log_sum;
  };
  if (tid == 0) {
    g.lse[r] = ref + log_sum;
    g.entropy[r] = entropy;
    const int32_t id = g.ids[r];
    float lp = 0.f;
    if (id < -1 || (id >= 0 && id >= cols)) atomicCAS(g.err, 0, DOMAIN_ERROR);
    else if (id >= 0) lp = log_prob(Vec<T>::one(row + id));
    g.logprob[r] = lp;
  }
  if (warp == 0 && lane < (int)top) {
    const uint32_t col = col_of(lists[0][lane]);
    g.top_ids[r * top + lane] = (int32_t)col;
    g.top_logprobs[r * top + lane] = (int64_t)col < cols ? log_prob(Vec<T>::one(row + col)) : -INFINITY;
  }
}

// scale (g (1[j = id] - p) - h p (y - lse + H)) with p = e^(y - lse).  Both types are read and written in groups of eight
// elements of the whole matrix, whose ends are the result's 16-byte boundaries whatever the row's length; a group that two rows
// share is written by both, an element at a time.  A row's segment of GROUPS * THREADS groups a block, all of a thread's groups
// asked for before the first is used.
constexpr int GROUPS = 2;
// A product whose subnormal results are zero: a BF16 result below 2^-126 is stored as zero (`f32_to_bf16_bits`).
__device__ __forceinline__ float mul_flush(float a, float b) {
  float r;
  asm("mul.ftz.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void load_group(const LogprobGradArgs& g, uint64_t at, bool vec, float* x) {
  if (g.bf16) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(g.logits) + at;
    if (vec) { Vec<uint16_t>::widen(__ldg(reinterpret_cast<const uint4*>(p)), x); return; }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = bf16_bits_to_f32(p[e]);
  } else {
    const float* p = reinterpret_cast<const float*>(g.logits) + at;
    if (vec) {
      Vec<float>::widen(__ldg(reinterpret_cast<const uint4*>(p)), x);
      Vec<float>::widen(__ldg(reinterpret_cast<const uint4*>(p) + 1), x + 4);
      return;
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = p[e];
  }
}
template <bool ENTROPY>
__global__ void __launch_bounds__(256) token_logprobs_backward_kernel(const __grid_constant__ LogprobGradArgs g, uint32_t segments, int vec) {
  pdl_enter();
  const uint64_t r = blockIdx.x / segments, base = r * g.cols, end = base + g.cols;
  const uint64_t group0 = base / 8 + (uint64_t)(blockIdx.x % segments) * GROUPS * blockDim.x + threadIdx.x;
  const float lse = g.lse[r], h = ENTROPY ? g.d_entropy[r] * g.scale : 0.f, H = ENTROPY ? g.entropy[r] : 0.f;
  int64_t id = g.ids[r];
  if (id < -1 || id >= (int64_t)g.cols) {
    if (threadIdx.x == 0) atomicCAS(g.err, 0, DOMAIN_ERROR);
    id = -1;
  }
  const float up = id >= 0 ? g.d_logprob[r] * g.scale : 0.f;
  const uint64_t hot = id >= 0 ? base + (uint64_t)id : ~0ull;
  const bool empty = lse == -INFINITY;
  float x[GROUPS][8];
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const uint64_t at = (group0 + (uint64_t)i * blockDim.x) * 8;
    if (at >= base && at + 8 <= end) load_group(g, at, vec, x[i]);
    else
#pragma unroll
      for (int e = 0; e < 8; ++e)
        x[i][e] = at + e >= base && at + e < end ? (g.bf16 ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(g.logits)[at + e])
                                                           : reinterpret_cast<const float*>(g.logits)[at + e]) : 0.f;
  }
#pragma unroll
  for (int i = 0; i < GROUPS; ++i) {
    const uint64_t at = (group0 + (uint64_t)i * blockDim.x) * 8;
    if (at >= end) break;
    float v[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float z = fmaf(x[i][e], g.scale, -lse), p = exp2_fast(z * LOG2E);
      // an entry of -inf has p = 0 (as everything below -126 log 2 has): its z is kept finite so that their product is 0
      v[e] = mul_flush(p, ENTROPY ? -(up + h * (fmaxf(z, -200.f) + H)) : -up);
    }
    if (hot - at < 8)
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at + e == hot) v[e] += up;
    if (empty)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = 0.f;
    if (at >= base && at + 8 <= end) {
      if (g.out_bf16) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(v[2 * e + 1]), "f"(v[2 * e]));
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(g.out) + at) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(g.out) + at);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (at + e >= base && at + e < end) {
          if (g.out_bf16) reinterpret_cast<uint16_t*>(g.out)[at + e] = f32_to_bf16_bits(__float_as_uint(v[e]));
          else reinterpret_cast<float*>(g.out)[at + e] = v[e];
        }
    }
  }
}

template <typename T, int THREADS, bool SHARED>
cudaError_t launch_form(const LogprobArgs& g, int size, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(g.rows * size)); cfg.blockDim = dim3(THREADS); cfg.stream = stream;
  cudaLaunchAttribute at[2];
  int n = 0;
  if (pdl_enabled()) {
    at[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[n++].val.programmaticStreamSerializationAllowed = 1;
  }
  if (SHARED) {
    at[n].id = cudaLaunchAttributeClusterDimension;
    at[n].val.clusterDim.x = size; at[n].val.clusterDim.y = 1; at[n++].val.clusterDim.z = 1;
  }
  cfg.attrs = at; cfg.numAttrs = n;
  return cudaLaunchKernelEx(&cfg, token_logprobs_kernel<T, THREADS, SHARED>, g);
}

template <typename T>
cudaError_t launch_type(const LogprobArgs& g, cudaStream_t stream) {
  // A row's blocks: as many as leave every block a slice of some thousand values while the rows alone do not fill the GPU.
  int size = 1;
  while (size < CLUSTER && g.rows * size < 296 && g.cols / (size * 2) >= 2048) size *= 2;
  if (size > 1) return launch_form<T, 256, true>(g, size, stream);
  return g.cols <= 1024 ? launch_form<T, 32, false>(g, 1, stream) : launch_form<T, 256, false>(g, 1, stream);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& g, cudaStream_t stream) {
  if (g.rows == 0) return cudaSuccess;
  return g.bf16 ? launch_type<uint16_t>(g, stream) : launch_type<float>(g, stream);
}

cudaError_t launch_token_logprobs_backward(const LogprobGradArgs& g, cudaStream_t stream) {
  if (g.rows == 0) return cudaSuccess;
  const uint64_t groups = (g.cols + 7) / 8 + 1;            // a row that starts inside a group touches one more
  unsigned threads = 32;
  while (threads < 256 && threads * GROUPS < groups) threads *= 2;
  const uint64_t segments = (groups + threads * GROUPS - 1) / (threads * GROUPS), blocks = segments * g.rows;
  if (blocks > 0x7fffffffull) return cudaErrorNotSupported;
  const int vec = (reinterpret_cast<uintptr_t>(g.logits) & 15) == 0;
  launch_pdl(g.d_entropy ? token_logprobs_backward_kernel<true> : token_logprobs_backward_kernel<false>, dim3((unsigned)blocks), dim3(threads), 0, stream,
             g, (uint32_t)segments, vec);
  return cudaGetLastError();
}

}  // namespace b200
