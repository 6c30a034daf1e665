// Log probabilities of given tokens, entropy and the largest alternatives of each row of logits
// (`b200_token_logprobs`), and their gradient (`b200_token_logprobs_backward`).
//
// With y = scale x, m = max y, S = sum e^(y - m) and T = sum e^(y - m) (y - m):
//   lse = m + log S,   log p_j = (y_j - m) - log S,   entropy = log S - T / S.
// Both terms of the entropy are of one sign (T <= 0; m is rounded, so to its last bit), and for a row sure of one token log S is
// as small as that token's log probability: nothing cancels.  Values are ordered as `argmax_row` orders them
// (a NaN above everything, -0 equal to +0, equal values by the lower column): one 64-bit key a value.
#include <cfloat>
#include <cmath>
#include <cstdint>
#include <cuda_runtime.h>

#include "device_math.cuh"
#include "kernels.h"
#include "pages.cuh"
#include "pdl.cuh"

namespace b200 {
namespace {

constexpr int CLUSTER = 8;               // blocks that share a row, at most
constexpr int TOP = 32;                  // alternatives a row, at most
constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

// A product whose subnormal results are zero: a BF16 result below 2^-126 is stored as zero (`f32_to_bf16_bits`).
__device__ __forceinline__ float mul_flush(float a, float b) {
  float r;
  asm("mul.ftz.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float at_least(float x, float low) {   // a NaN stays one
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(x), "f"(low));
  return r;
}
// Two F32 operations an instruction.
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ float2 floats_of(uint64_t v) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(v));
  return r;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
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
__device__ __forceinline__ float value_of(uint64_t key) {      // 0, no key: below every value
  if (key == 0) return -INFINITY;
  const uint32_t u = (uint32_t)(key >> 32);
  return __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}

// A 16-byte piece of a row.  LOW: what -inf (and everything below) counts as in the sums, so that a term of 0 times its
// exponent is 0; nothing above it is touched, a NaN stays one.
constexpr float LOW = -1.0e30f;
template <typename T> struct Vec;
template <> struct Vec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ float one(const float* p) { return *p; }
  static __device__ __forceinline__ void widen(const uint4& w, float* f) {
    f[0] = __uint_as_float(w.x); f[1] = __uint_as_float(w.y); f[2] = __uint_as_float(w.z); f[3] = __uint_as_float(w.w);
  }
  static __device__ __forceinline__ float top(const uint4& w) {
    return fmaxf(fmaxf(__uint_as_float(w.x), __uint_as_float(w.y)), fmaxf(__uint_as_float(w.z), __uint_as_float(w.w)));
  }
  static __device__ __forceinline__ float low(uint32_t w) { return at_least(__uint_as_float(w), LOW); }
  static __device__ __forceinline__ void pairs(const uint4& w, uint64_t* v) { v[0] = pair_of(low(w.x), low(w.y)); v[1] = pair_of(low(w.z), low(w.w)); }
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
  static __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
    uint32_t r;
    asm("max.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
    return r;
  }
  static __device__ __forceinline__ float top(const uint4& w) {
    const uint32_t m = max2(max2(w.x, w.y), max2(w.z, w.w));
    return fmaxf(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u));
  }
  static __device__ __forceinline__ uint64_t low(uint32_t w) {
    uint32_t r;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(w), "r"(0xf14af14au));   // -1.0003e30 twice
    return pair_of(__uint_as_float(r << 16), __uint_as_float(r & 0xffff0000u));
  }
  static __device__ __forceinline__ void pairs(const uint4& w, uint64_t* v) { v[0] = low(w.x); v[1] = low(w.y); v[2] = low(w.z); v[3] = low(w.w); }
};

// Sums under a reference m in units of log2: s = sum 2^(y - m), t = sum 2^(y - m) (y - m), y = x scale log2 e.
struct Sums { float m, s, t; };
__device__ __forceinline__ Sums under(const Sums& a, float m) {       // a's sums under another reference
  if (a.s == 0.f) return Sums{m, 0.f, 0.f};                           // nothing summed stays nothing, however far the reference moved
  const float d = a.m - m, f = exp2_fast(d);
  return Sums{m, a.s * f, f * fmaf(a.s, d, a.t)};
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
  __device__ __forceinline__ uint4 piece(uint32_t u) const {
    if (whole(u)) return raw(u);
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      w[i] = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;
#pragma unroll
      for (int e = 0; e < 4 / (int)sizeof(T); ++e) {
        const int64_t c = origin + (int64_t)u * Vec<T>::N + i * (4 / (int)sizeof(T)) + e;
        if (c >= first && c < last) {
          if constexpr (sizeof(T) == 2) w[i] = e ? (w[i] & 0xffffu) | ((uint32_t)row[c] << 16) : (w[i] & 0xffff0000u) | row[c];
          else w[i] = __float_as_uint(row[c]);
        }
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// The largest of a warp's values, NaN passed over.
__device__ __forceinline__ float warp_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// A thread's running state over its pieces: its largest value and the first piece that has it, the largest of the others, and
// the sums under the reference m = fl(high c).  `high` is the largest value that the warp had met when it last asked (at least
// LOW, and with nothing above that the thread has no reference), and the warp asks before it sums: a reference that stayed
// behind the largest term by z would leave the entropy and a sure token's log probability as differences of two numbers near z.
template <typename T> struct Running {
  float best = -INFINITY, second = -INFINITY, high = LOW, m = 0.f;
  uint32_t piece;
  uint64_t s[2] = {0, 0}, t[2] = {0, 0};
  __device__ __forceinline__ void note(float top, uint32_t u) {
    piece = top > best ? u : piece;
    second = fmaxf(second, fminf(top, best));
    best = fmaxf(best, top);
  }
  __device__ __forceinline__ void add(const uint4& w, uint64_t c2) {
    uint64_t v[Vec<T>::N / 2];
    Vec<T>::pairs(w, v);
    const uint64_t ref = pair_of(-m, -m);
#pragma unroll
    for (int i = 0; i < Vec<T>::N / 2; ++i) {
      const uint64_t z = fma2(v[i], c2, ref);
      const float2 e = floats_of(z);
      const uint64_t p = pair_of(exp2_fast(e.x), exp2_fast(e.y));
      s[i & 1] = add2(s[i & 1], p);
      t[i & 1] = fma2(p, z, t[i & 1]);
    }
  }
  __device__ __forceinline__ Sums sums() const {           // a thread with nothing above LOW has no reference
    const float2 a = floats_of(add2(s[0], s[1])), b = floats_of(add2(t[0], t[1]));
    return Sums{high > LOW ? m : -FLT_MAX, a.x + a.y, b.x + b.y};
  }
  __device__ __forceinline__ void raise(float to, float c) {
    if (!(to > high)) return;
    high = to;
    const Sums a = under(Sums{m, sums().s, sums().t}, fminf(fmaxf(to * c, -FLT_MAX), FLT_MAX));
    s[0] = pair_of(a.s, 0.f); t[0] = pair_of(a.t, 0.f);
    s[1] = t[1] = 0;
    m = a.m;
  }
  __device__ __forceinline__ void alone(const uint4& w, uint32_t u, float c, uint64_t c2) {   // a piece of this thread only
    const float top = Vec<T>::top(w);
    raise(top, c);
    note(top, u);
    add(w, c2);
  }
};

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

// How many of `n` keys are larger than `key`: its place in the sorted list (no two are equal).
__device__ __forceinline__ uint32_t place_of(uint64_t key, const uint64_t* keys, uint32_t n) {
  uint32_t k = 0;
#pragma unroll 8
  for (uint32_t i = 0; i < n; ++i) k += keys[i] > key;
  return k;
}

// A row a block, or a row a cluster of blocks with a slice each (SHARED).  One pass keeps each thread's sums and its largest
// value.  Every warp's few largest of those bound the row's `top` largest from below: a thread that reaches the bound reads the
// piece of its largest again, and only where another of its pieces reaches it too (one thread in ten of those) are all of that
// thread's read by the block.  What reaches the bound is listed and put in order.  Where that is more than the list holds -- rows
// of few distinct values -- the bound is taken again from keys, by value and column.
//
// A thread asks for AHEAD of its pieces before it uses the first, and a warp for its largest value every ASKED of them.  Eight and
// four where rows are long, with the registers of seven blocks an SM: without alternatives 2000 BF16 rows of 50257 take 44.1 us
// (4.6 TB/s), 1000 F32 rows 34.9 (5.8 TB/s); asking every two 43.8 and 34.9, every eight 46.4 and 36.4; with six blocks' registers
// 47.0 and 45.1 (1000 rows are more than one round of blocks then).  Four pieces in the other forms, whose threads have few, and as
// many blocks as the registers allow (0): more of either costs 16000 rows of 2000 59 -> 70 us and above.
// What bounds the pass is neither limit alone: half of the issue slots and of the exponents' rate, two thirds of a copy's bytes
// (2000 x 50257 BF16, 25 warps an SM on average).
template <typename T, int THREADS, bool SHARED>
__global__ void __launch_bounds__(THREADS, THREADS == 128 ? 7 : 0) token_logprobs_kernel(const __grid_constant__ LogprobArgs g) {
  constexpr int WARPS = THREADS / 32, N = Vec<T>::N, HELD = THREADS * 8, AHEAD = THREADS == 128 ? 8 : 4, ASKED = 4;
  __shared__ uint64_t held[HELD], sh[WARPS], slices[SHARED ? CLUSTER * TOP : TOP], list[TOP];
  __shared__ Sums warp_sums[WARPS], slice_sums[SHARED ? CLUSTER : 1];
  __shared__ float warp_best[WARPS], slice_best[SHARED ? CLUSTER : 1];
  __shared__ uint32_t count, owner_count;
  __shared__ uint16_t owners[THREADS];
  __shared__ uint32_t done[THREADS];
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
  const uint64_t c2 = pair_of(c, c);
  const uint32_t top = g.top;
  if (tid == 0) count = owner_count = 0;
  if (tid < TOP) list[tid] = 0;
  const int32_t id = g.ids[r];
  const bool named = id >= 0 && id < cols;
  const float id_logit = named ? Vec<T>::one(row + id) : 0.f;

  // ---- the pass; the slice's cut ends by themselves
  Running<T> a;
  a.piece = (uint32_t)tid;               // a thread whose values are all -inf has its first
  const uint32_t lo = sl.pieces && !sl.whole(0) ? 1u : 0u, hi = sl.pieces && !sl.whole(sl.pieces - 1) ? sl.pieces - 1 : sl.pieces;
  if (lo && tid == 0) a.alone(sl.piece(0), 0, c, c2);
  const uint32_t gone = sizeof(T) == 2 ? 0xff80ff80u : 0xff800000u;           // a lane without a piece: -inf
  for (uint32_t u = tid; u - lane < hi; u += AHEAD * THREADS) {               // the same for a warp's lanes
    uint4 w[AHEAD];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      const uint32_t v = u + i * THREADS;
      w[i] = make_uint4(gone, gone, gone, gone);
      if (v >= lo && v < hi) w[i] = sl.raw(v);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; k += ASKED) {
      if (u - lane + k * THREADS >= hi) break;
      float tops[ASKED], most = -INFINITY;
#pragma unroll
      for (int i = 0; i < ASKED; ++i) {
        tops[i] = Vec<T>::top(w[k + i]);
        most = fmaxf(most, tops[i]);
      }
      if (__any_sync(0xffffffffu, most > a.high)) a.raise(warp_max(most), c);
#pragma unroll
      for (int i = 0; i < ASKED; ++i)
        if (u - lane + (k + i) * THREADS < hi) {
          a.note(tops[i], u + (k + i) * THREADS);
          a.add(w[k + i], c2);
        }
    }
  }
  if (hi < sl.pieces && hi >= lo && sl.pieces > lo && tid == (int)(hi % THREADS)) a.alone(sl.piece(hi), hi, c, c2);

  // ---- the slice's sums: under the largest reference of the warp, then of the block
  Sums all = a.sums();
  float high = a.best;
  {
    float m = all.m;
#pragma unroll
    for (int o = 16; o; o >>= 1) { m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o)); high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o)); }
    all = under(all, m);
#pragma unroll
    for (int o = 16; o; o >>= 1) { all.s += __shfl_xor_sync(0xffffffffu, all.s, o); all.t += __shfl_xor_sync(0xffffffffu, all.t, o); }
  }
  if (lane == 0) { warp_sums[warp] = all; warp_best[warp] = high; }
  const uint32_t threads = sl.pieces < (uint32_t)THREADS ? sl.pieces : (uint32_t)THREADS;   // those that hold a piece
  const bool bounded = threads >= top;
  // the `each`th largest of a warp whose threads all hold a piece, `each` such a warp's share of `top` (with no such warp, the
  // first's `top`th: it has as many)
  const uint32_t whole = threads < 32 ? 1 : threads / 32, each = (top + whole - 1) / whole;
  const auto bound_warp = [&](uint64_t left) {
    uint64_t last = 0;
    for (uint32_t k = 0; k < each; ++k) {
      const uint32_t h = __reduce_max_sync(0xffffffffu, (uint32_t)(left >> 32));
      const uint32_t l = __reduce_max_sync(0xffffffffu, (uint32_t)(left >> 32) == h ? (uint32_t)left : 0u);
      last = ((uint64_t)h << 32) | l;
      if (left == last) left = 0;
    }
    if (lane == 0) sh[warp] = warp < (int)whole ? last : ~0ull;
  };
  // by value alone: a key whose lower word tells the lanes apart and is left out of the bound
  if (top && bounded) bound_warp(tid < (int)threads ? key_of(a.best, (uint32_t)tid) : 0);
  __syncthreads();
  {
    float m = -FLT_MAX;
    high = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) { m = fmaxf(m, warp_sums[w].m); high = fmaxf(high, warp_best[w]); }
    all = Sums{m, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      const Sums b = under(warp_sums[w], m);
      all.s += b.s;
      all.t += b.t;
    }
  }

  // ---- the slice's largest
  if (top) {
    bool slow = all.s != all.s;          // a NaN or +inf: the maxima above passed over it
    const auto bound_of = [&]() {
      uint64_t bound = sh[0];
#pragma unroll
      for (int w = 1; w < WARPS; ++w) bound = sh[w] < bound ? sh[w] : bound;
      return bound;
    };
    const auto collect = [&](uint32_t u, uint64_t bound) {   // a piece's values that reach the bound
      const uint4 w = sl.piece(u);
      const float reach = value_of(bound);
      if (Vec<T>::top(w) < reach) return;
      float x[N];
      Vec<T>::widen(w, x);
#pragma unroll
      for (int e = 0; e < N; ++e)
        if (x[e] >= reach) {
          const int64_t col = sl.origin + (int64_t)u * N + e;
          const uint64_t key = key_of(x[e], (uint32_t)col);
          if (key >= bound && col >= sl.first && col < sl.last) {
            const uint32_t at = atomicAdd(&count, 1u);
            if (at < (uint32_t)HELD) held[at] = key;
          }
        }
    };
    const auto collect_owned = [&](uint64_t bound) {         // all pieces of the listed threads but the one each has done
      const uint32_t rounds = (sl.pieces + THREADS - 1) / THREADS, n = owner_count * rounds;
      for (uint32_t i = tid; i < n; i += THREADS) {
        const uint32_t o = i / rounds, u = owners[o] + i % rounds * THREADS;
        if (u < sl.pieces && u != done[o]) collect(u, bound);
      }
    };
    const auto collect_all = [&](uint64_t bound, bool reaches, bool others) {
      if (tid < (int)threads && reaches) {
        collect(a.piece, bound);
        if (others) {
          const uint32_t at = atomicAdd(&owner_count, 1u);
          owners[at] = (uint16_t)tid;
          done[at] = a.piece;
        }
      }
      __syncthreads();
      collect_owned(bound);
      __syncthreads();
    };
    if (!slow) {
      uint64_t bound = bounded ? bound_of() & 0xffffffff00000000ull : 0;
      collect_all(bound, a.best >= value_of(bound), a.second >= value_of(bound));
      if (count > (uint32_t)HELD && bounded) {
        uint64_t mine = 0;               // this thread's largest key
        if (tid < (int)threads) {
          float x[N];
          Vec<T>::widen(sl.piece(a.piece), x);
          int at = -1;
#pragma unroll
          for (int e = N - 1; e >= 0; --e) {
            const int64_t col = sl.origin + (int64_t)a.piece * N + e;
            if (x[e] == a.best && col >= sl.first && col < sl.last) at = e;
          }
          if (at >= 0) mine = key_of(a.best, (uint32_t)(sl.origin + (int64_t)a.piece * N + at));
        }
        __syncthreads();                 // everyone has seen the count
        if (tid == 0) count = owner_count = 0;
        bound_warp(mine);
        __syncthreads();
        bound = bound_of();
        collect_all(bound, mine >= bound, a.second >= value_of(bound));
      }
      slow = count > (uint32_t)HELD;
      // the list's order depends on the atomics, its keys do not
      if (!slow)
        for (uint32_t i = tid; i < count; i += THREADS) {
          const uint64_t key = held[i];
          const uint32_t k = place_of(key, held, count);
          if (k < top) list[k] = key;
        }
    }
    if (slow) slow_top(sl, top, list, sh);
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
    if (tid < (int)top) asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(there(&slices[rank * top + tid])), "l"(list[tid]) : "memory");
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    if (rank) return;
    float m = -FLT_MAX;
    high = -INFINITY;
    for (uint32_t w = 0; w < size; ++w) { m = fmaxf(m, slice_sums[w].m); high = fmaxf(high, slice_best[w]); }
    all = Sums{m, 0.f, 0.f};
    for (uint32_t w = 0; w < size; ++w) {
      const Sums b = under(slice_sums[w], m);
      all.s += b.s;
      all.t += b.t;
    }
    if (top) {
      for (uint32_t i = tid; i < size * top; i += THREADS) {
        const uint64_t key = slices[i];
        const uint32_t k = key ? place_of(key, slices, size * top) : top;    // 0: a slice with fewer values
        if (k < top) list[k] = key;
      }
      __syncthreads();
    }
  }

  // y - lse and the statistics.  The pass's terms are 2^(x c - fl(high c)): the reference's rounding cancels in the results, but it
  // is a factor of up to 2^(|high c| 2^-24) on every term, and a product may leave the type's range (a row masked by the type's
  // lowest value).  Rows with a reference from 1e8 on, or nothing above LOW, are taken again from differences to their largest.
  if (high == INFINITY) all.s = NAN;
  float ref = all.m * LN2, log_sum = logf(all.s), entropy = log_sum - LN2 * all.t / all.s;
  const bool none = high == -INFINITY && all.s == 0.f;     // -inf only
  const bool plain = none || !(fabsf(high) <= FLT_MAX) || (fabsf(high * c) < 1e8f && high > LOW);
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
    if (!named && id != -1) atomicCAS(g.err, 0, DOMAIN_ERROR);
    g.logprob[r] = named ? log_prob(id_logit) : 0.f;
  }
  if (warp == 0 && lane < (int)top) {
    const uint32_t col = col_of(list[lane]);
    g.top_ids[r * top + lane] = (int32_t)col;
    g.top_logprobs[r * top + lane] = log_prob(value_of(list[lane]));
  }
}

// scale (g (1[j = id] - p) - h p (y - lse + H)) with p = e^(y - lse).  Memory-bound.  Both types are read and written in groups of
// eight elements that start at the result's 16-byte boundaries whatever the row's length; a row's up to seven elements before its
// first such group and behind its last are a thread each.
// What a thread has in flight and how often: registers cost more here than bytes in flight bring (4000 x 32001 BF16: one group
// four times 86 us, two groups four times 84, two once 87, four once 102 on fewer warps; 500 x 49152 F32, twice the bytes a group:
// one once 30.6 us, two once 31.3, two four times 34.2).
template <bool BF> struct Flight { static constexpr int GROUPS = BF ? 2 : 1, STEPS = BF ? 4 : 1; };
template <bool BF>
__device__ __forceinline__ void load_group(const LogprobGradArgs& g, uint64_t at, int vec, uint64_t* v) {
  float x[8];
  if constexpr (BF) {
    const uint16_t* p = reinterpret_cast<const uint16_t*>(g.logits) + at;
    uint4 w;
    if (vec) w = __ldg(reinterpret_cast<const uint4*>(p));
    else w = make_uint4(p[0] | (uint32_t)p[1] << 16, p[2] | (uint32_t)p[3] << 16, p[4] | (uint32_t)p[5] << 16, p[6] | (uint32_t)p[7] << 16);
    Vec<uint16_t>::widen(w, x);
  } else {
    const float* p = reinterpret_cast<const float*>(g.logits) + at;
    uint4 w[2];
    if (vec) { w[0] = __ldg(reinterpret_cast<const uint4*>(p)); w[1] = __ldg(reinterpret_cast<const uint4*>(p) + 1); }
    else {
      const uint32_t* q = reinterpret_cast<const uint32_t*>(p);
      w[0] = make_uint4(q[0], q[1], q[2], q[3]); w[1] = make_uint4(q[4], q[5], q[6], q[7]);
    }
    Vec<float>::widen(w[0], x);
    Vec<float>::widen(w[1], x + 4);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = pair_of(x[2 * i], x[2 * i + 1]);
}
// Part `segment` of a row whose lse is too large to hold the logarithm of its sum (at 4096 F32's step is 2^-11, and in a row masked
// by the type's lowest values nothing of it is left): log p is taken again, from differences to the row's largest as the forward
// takes it.  Rare, so every block of the row reads all of it, and it is out of the way.
constexpr float FAR = 4096.f;
template <bool BF, bool OUT_BF>
__device__ __noinline__ void far_row(const LogprobGradArgs& g, uint64_t base, uint32_t segment, uint32_t segments, float h, float H, float up, uint32_t hot) {
  __shared__ float parts[8];
  const uint32_t cols = (uint32_t)g.cols, tid = threadIdx.x, warps = blockDim.x / 32;
  float high = -INFINITY, s = 0.f;
  for (uint32_t j = tid; j < cols; j += blockDim.x) high = fmaxf(high, load_float(g.logits, base + j, BF));
#pragma unroll
  for (int o = 16; o; o >>= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, o));
  if (tid % 32 == 0) parts[tid / 32] = high;
  __syncthreads();
  for (uint32_t w = 0; w < warps; ++w) high = fmaxf(high, parts[w]);
  __syncthreads();
  for (uint32_t j = tid; j < cols; j += blockDim.x) s += expf((load_float(g.logits, base + j, BF) - high) * g.scale);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (tid % 32 == 0) parts[tid / 32] = s;
  __syncthreads();
  s = 0.f;
  for (uint32_t w = 0; w < warps; ++w) s += parts[w];
  const float log_sum = logf(s);
  const uint32_t each = (cols + segments - 1) / segments, first = segment * each, end = first + each < cols ? first + each : cols;
  for (uint32_t j = first + tid; j < end; j += blockDim.x) {
    const float z = (load_float(g.logits, base + j, BF) - high) * g.scale - log_sum, p = expf(z);
    float v = p == 0.f ? 0.f : p * fmaf(h, z + H, -up);
    v = high == -INFINITY ? 0.f : (j == hot ? v + up : v);                    // -inf only
    store_float(g.out, base + j, OUT_BF, v);
  }
}

template <bool BF, bool OUT_BF, bool ENTROPY>
__global__ void __launch_bounds__(256) token_logprobs_backward_kernel(const __grid_constant__ LogprobGradArgs g, uint32_t segments, int vec) {
  pdl_enter();
  const uint32_t r = blockIdx.x / segments, segment = blockIdx.x % segments, cols = (uint32_t)g.cols;
  const uint64_t base = (uint64_t)r * cols;
  const uint32_t head = (uint32_t)(8 - (base & 7)) & 7, start = head < cols ? head : cols, groups = (cols - start) / 8;
  uint32_t q = segment * (Flight<BF>::GROUPS * Flight<BF>::STEPS) * blockDim.x + threadIdx.x;
  uint64_t x[Flight<BF>::GROUPS][4];
#pragma unroll
  for (int i = 0; i < Flight<BF>::GROUPS; ++i)
    if (q + i * blockDim.x < groups) load_group<BF>(g, base + start + (uint64_t)(q + i * blockDim.x) * 8, vec, x[i]);
  const float lse = g.lse[r], h = ENTROPY ? -g.d_entropy[r] * g.scale : 0.f, H = ENTROPY ? g.entropy[r] : 0.f;
  const float given = g.d_logprob[r] * g.scale;
  const int32_t id = g.ids[r];
  const bool named = id >= 0 && (uint32_t)id < cols;
  if (!named && id != -1 && threadIdx.x == 0) atomicCAS(g.err, 0, DOMAIN_ERROR);
  const float up = named ? given : 0.f;
  const uint32_t hot = named ? (uint32_t)id : 0xffffffffu;
  const bool empty = !named && (!ENTROPY || h == 0.f);       // a padding row, whatever its logits hold (0 * NaN is NaN)
  if (!empty && fabsf(lse) >= FAR) {
    far_row<BF, OUT_BF>(g, base, segment, segments, h, H, up, hot);
    return;
  }
  const float flat = ENTROPY ? fmaf(h, H, -up) : -up;
  // p (h (z + H) - up), z = y - lse; with a z below -1000, where p is 0, its factor stays finite
  const auto value = [&](uint64_t v, float& v0, float& v1) {
    uint64_t z = fma2(v, pair_of(g.scale, g.scale), pair_of(-lse, -lse));
    if constexpr (ENTROPY) z = pair_of(at_least(floats_of(z).x, -1000.f), at_least(floats_of(z).y, -1000.f));
    const float2 e = floats_of(mul2(z, pair_of(LOG2E, LOG2E)));
    const float2 k = floats_of(ENTROPY ? fma2(z, pair_of(h, h), pair_of(flat, flat)) : pair_of(flat, flat));
    v0 = mul_flush(exp2_fast(e.x), k.x);
    v1 = mul_flush(exp2_fast(e.y), k.y);
  };
#pragma unroll 1
  for (int step = 0;; ++step) {
#pragma unroll
    for (int i = 0; i < Flight<BF>::GROUPS; ++i) {
      const uint32_t at = q + i * blockDim.x, col = start + at * 8;
      if (at >= groups) break;
      float v[8];
#pragma unroll
      for (int e = 0; e < 4; ++e) value(x[i][e], v[2 * e], v[2 * e + 1]);
      if (hot - col < 8 || empty)                            // the given token's own term, and an empty row
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = empty ? 0.f : (col + e == hot ? v[e] + up : v[e]);
      if constexpr (OUT_BF) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(w[e]) : "f"(v[2 * e + 1]), "f"(v[2 * e]));
        *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(g.out) + base + col) = make_uint4(w[0], w[1], w[2], w[3]);
      } else {
        float4* o = reinterpret_cast<float4*>(reinterpret_cast<float*>(g.out) + base + col);
        o[0] = make_float4(v[0], v[1], v[2], v[3]);
        o[1] = make_float4(v[4], v[5], v[6], v[7]);
      }
    }
    q += Flight<BF>::GROUPS * blockDim.x;
    if (step + 1 == Flight<BF>::STEPS || q >= groups) break;
#pragma unroll
    for (int i = 0; i < Flight<BF>::GROUPS; ++i)
      if (q + i * blockDim.x < groups) load_group<BF>(g, base + start + (uint64_t)(q + i * blockDim.x) * 8, vec, x[i]);
  }
  if (segment == 0 && threadIdx.x < 16) {
    const uint32_t end = start + groups * 8, col = threadIdx.x < 8 ? threadIdx.x : end + threadIdx.x - 8;
    if (threadIdx.x < 8 ? col < start : col < cols) {
      const float y = BF ? bf16_bits_to_f32(reinterpret_cast<const uint16_t*>(g.logits)[base + col]) : reinterpret_cast<const float*>(g.logits)[base + col];
      float v, other;
      value(pair_of(y, y), v, other);
      v = empty ? 0.f : (col == hot ? v + up : v);
      if constexpr (OUT_BF) reinterpret_cast<uint16_t*>(g.out)[base + col] = f32_to_bf16_bits(__float_as_uint(v));
      else reinterpret_cast<float*>(g.out)[base + col] = v;
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
  // A row's blocks: as many as leave every block a slice of some thousand values while there are fewer than two an SM (one F32 row
  // of 49,152 with five alternatives: 8.7 us by a cluster of eight, 16.1 by one block; of 260,000 with twenty: 16 and 65; 295 BF16
  // rows of 50,257: 13.1 by two blocks a row, 19.5 by four).
  int size = 1;
  while (size < CLUSTER && g.rows * size < 148 * 2 && g.cols / (size * 2) >= 2048) size *= 2;
  if (size > 1) return launch_form<T, 256, true>(g, size, stream);
  // A row's threads: what a row's end costs grows with its block, what a thread has in flight is the same, so blocks are small as
  // long as there are enough of them to fill the GPU.  64 MB of BF16 logits with twenty alternatives by 32 / 64 / 128 / 256
  // threads a row, us: rows of 2,000 67 / 64 / 83 / 137, of 4,000 46 / 41 / 50 / 84, of 8,000 35 / 31 / 33 / 50, of 16,000
  // 49 / 30 / 26 / 33, of 32,000 70 / 35 / 22 / 28; 4,000 rows of 1,000 9 / - / - / 28.  Long rows few enough for blocks of 256
  // to be resident at once, four an SM, take those, by 128 / 256: 400 F32 rows of 49,152 25.9 / 19.4, 592 28.1 / 22.8, 650
  // 28.6 / 32.4; 400 BF16 rows of 11,000 with twenty alternatives 12.0 / 11.7.
  if (g.cols <= 1024) return launch_form<T, 32, false>(g, 1, stream);
  if (g.cols <= 10000) return launch_form<T, 64, false>(g, 1, stream);
  return g.rows <= 148 * 4 ? launch_form<T, 256, false>(g, 1, stream) : launch_form<T, 128, false>(g, 1, stream);
}

}  // namespace

cudaError_t launch_token_logprobs(const LogprobArgs& g, cudaStream_t stream) {
  if (g.rows == 0) return cudaSuccess;
  return g.bf16 ? launch_type<uint16_t>(g, stream) : launch_type<float>(g, stream);
}

cudaError_t launch_token_logprobs_backward(const LogprobGradArgs& g, cudaStream_t stream) {
  if (g.rows == 0) return cudaSuccess;
  const uint64_t groups = g.cols / 8, each = g.bf16 ? Flight<true>::GROUPS * Flight<true>::STEPS : Flight<false>::GROUPS * Flight<false>::STEPS;
  unsigned threads = 32;
  while (threads < 256 && threads * each < groups) threads *= 2;
  const uint64_t segments = groups ? (groups + threads * each - 1) / (threads * each) : 1, blocks = segments * g.rows;
  if (blocks > 0x7fffffffull) return cudaErrorNotSupported;
  const int vec = (reinterpret_cast<uintptr_t>(g.logits) & 15) == 0;
  const auto go = [&](auto kernel) { launch_pdl(kernel, dim3((unsigned)blocks), dim3(threads), 0, stream, g, (uint32_t)segments, vec); };
  const bool h = g.d_entropy != nullptr;
  if (g.bf16) {
    if (g.out_bf16) h ? go(token_logprobs_backward_kernel<true, true, true>) : go(token_logprobs_backward_kernel<true, true, false>);
    else h ? go(token_logprobs_backward_kernel<true, false, true>) : go(token_logprobs_backward_kernel<true, false, false>);
  } else {
    if (g.out_bf16) h ? go(token_logprobs_backward_kernel<false, true, true>) : go(token_logprobs_backward_kernel<false, true, false>);
    else h ? go(token_logprobs_backward_kernel<false, false, true>) : go(token_logprobs_backward_kernel<false, false, false>);
  }
  return cudaGetLastError();
}

}  // namespace b200
