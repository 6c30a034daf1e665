// Attention of one new token a sequence over the pages of its cache (`b200_attention_pages`).
//
// out = softmax(scale q K^T) V over one sequence's positions, up to eight query heads of one key/value head together, so that
// keys and values are read once for all of them.  The bound is that read: HBM.
//
// Split: the batch's positions are one list of tiles of 16, sequence after sequence, cut into equal runs whatever the lengths,
// and a warp takes one run for one key/value head: the warps beside it take the same run for the other heads, so that a cache
// row's heads are read together (a row is one piece of memory).  A run may end inside a sequence and the next one goes on
// there: a warp writes the results of sequences that lie in its run whole, and (maximum, sum, rows) of the at most two that do
// not, which a second kernel joins.  The lengths are on the device, so the list is made there, from a prefix sum.  After that
// sum no warp waits for another.  Where the table leaves room for short sequences only, there is neither list nor second
// kernel: a block, or a cluster of up to eight, has a (sequence, head) to itself, its warps equal shares of the tiles, and
// joins them from shared memory (`cut_of` says when).
//
// A warp's pipeline: it copies its 16 keys and 16 values of a tile to its own shared memory by 16-byte asynchronous copies, as
// many tiles ahead as it has room for (the place of a tile's keys is filled again as soon as its scores are taken, that of its
// values after the product with them; row addresses through the page table, fetched one tile before they are used), and keeps
// its own running maximum, sum and rows.
//
// Precision: keys and values are the cache's own values.  The tensor cores' tile has sixteen rows, and a head takes two of
// them: row r has an operand's leading part and row r + 8 the next one, so one product does both.  On the BF16 path an F32
// query is three BF16 parts (exact, whatever the result's type: a part left out is an error of the score, and a score's error
// is its weight's relative error however large the score), a probability three or, for a BF16 result, two (2^-16 of it); on the
// F32 path every operand is two TF32 parts (2^-22).  A tile's products start from zero and are added to the running rows in
// F32: the tensor cores cut what they add to a sum, which over the thousands of tiles of a long sequence is a bias (160
// sequences of 131,072 positions, values of mean 1: 5.7e-4 of the result summed there, 1.5e-6 summed in F32).
//
// Measured, heads of 128 (32 over 8), BF16 cache: 128 sequences of 500 to 8,192 401 us = 5.7 TB/s of keys and values (the
// copies alone, nothing computed, 378), one of 131,001 106 us = 5.1 TB/s (99), 32 of 5 to 4,100 67 us = 4.0 TB/s (57): what is left
// is the way to the first copy (prefix sum, page, row), the last runs and the join, about 15 us together.  `mma.sync` and not
// tcgen05: its tile could have the positions as its 128 rows and the heads as columns, but what bounds the call is the copies, behind
// which these products lie, and not the products.
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

template <typename KV, int D>
struct Form {
  static constexpr bool BF = sizeof(KV) == 2;
  static constexpr int WARPS = BF ? (D > 192 ? 3 : 4) : (D <= 96 ? 4 : (D == 192 ? 2 : 3));
  static constexpr int THREADS = WARPS * 32;
  // shared-memory row pitches that let eight rows (or the four position pairs of an F32 fragment) fall into distinct banks
  static constexpr int K_PITCH = D * (int)sizeof(KV) + (BF ? 16 : 32);
  static constexpr int V_PITCH = D * (int)sizeof(KV) + 16;
  static constexpr int STAGE = 16 * (K_PITCH + V_PITCH);      // a warp's tile
  // a copy instruction: LANES lanes a row (a whole 128-byte line where rows are whole lines), ROWS rows; a lane's rows of a
  // tile are REST, its pieces of a row PIECES
  static constexpr int CHUNKS = D * (int)sizeof(KV) / 16;     // 16-byte pieces of a row
  static constexpr int LANES = CHUNKS % 8 ? 4 : 8, ROWS = 32 / LANES, REST = 16 / ROWS, PIECES = CHUNKS / LANES;
  // blocks an SM: as many warps as their registers and two or three tiles each leave room for
  static constexpr int BLOCKS = BF ? (D <= 64 ? 3 : 2) : (D <= 64 ? 3 : (D <= 192 ? 2 : 1));
  static __host__ __device__ int prefix_bytes(uint32_t n) { return (int)(((n + 1) * 4 + 127) / 128 * 128); }
};
constexpr uint32_t MAX_SEQUENCES = 512;  // a launch's; its prefix sums lie in shared memory
constexpr int MAX_STAGES = 4;
constexpr int HEADS = 8;                 // query heads a warp
constexpr int CLUSTER = 8;               // blocks that share a (sequence, job), at most

struct AttnPlan {
  AttnPagesArgs g;
  uint64_t page_magic;                   // p / page = p * magic >> (32 + page_shift), exact below 2^31
  uint32_t page_shift;
  uint32_t group, row_tiles;             // query heads a key/value head, and their tiles of HEADS
  uint32_t jobs;                         // kv_heads * row_tiles
  uint32_t runs, slot;                   // runs the tiles are cut into; floats of a piece
  int stages;
  int together;                          // the warps of a cluster of so many blocks share one (sequence, job) and join it themselves; 0: runs
  float scale_log2;
  float* part;                           // [runs][jobs][2] pieces: [rows][D], then (maximum, sum) a row in four floats
  uint32_t* prefix;                      // [n + 1], for the join
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the latest `pending` groups of this thread have arrived
__device__ __forceinline__ void cp_async_wait(int pending) {
  if (pending <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (pending <= 3) asm volatile("cp.async.wait_group 3;" ::: "memory");
  else if (pending <= 5) asm volatile("cp.async.wait_group 5;" ::: "memory");
  else asm volatile("cp.async.wait_group 7;" ::: "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// Shared-memory loads in the order they are written: left to itself the compiler asks for a whole tile's fragments at once and
// spills.
__device__ __forceinline__ float2 lds2(uint32_t at) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(at) : "memory");
  return v;
}
__device__ __forceinline__ float lds1(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}
// a: (row r, first half of the inner index), (row r + 8, first), (r, second), (r + 8, second)
__device__ __forceinline__ void mma_bf16(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// A value's leading TF32 part, to nearest, and what is left of it: exact, and a TF32 value but for its last bit.  (Cut, the left
// would lose two bits, all toward zero: 7.6e-7 of a result in place of 5e-7.)
__device__ __forceinline__ uint32_t tf32_of(float x) { return (__float_as_uint(x) + 0x1000u) & 0xffffe000u; }
__device__ __forceinline__ uint32_t tf32_rest(float x) { return __float_as_uint(x - __uint_as_float(tf32_of(x))); }
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The next BF16 part of `rest`, which keeps what is left: cut, so that each part leaves fewer bits of the same sign, but for the
// last, which is rounded.
__device__ __forceinline__ uint32_t next_part(float& rest, bool last) {
  uint32_t bits = __float_as_uint(rest);
  if (last) bits = (uint32_t)f32_to_bf16_bits(bits) << 16;
  else if (rest != rest) bits = 0x7fc00000u;
  else bits &= 0xffff0000u;
  const float part = __uint_as_float(bits);
  rest = fabsf(part) <= FLT_MAX ? rest - part : 0.f;
  return bits >> 16;
}

// The first tile of run c, and the run that a tile is in: runs of total / runs tiles.
__device__ __forceinline__ uint32_t run_start(uint32_t total, uint32_t c, uint32_t runs) {
  return total / runs * c + (uint32_t)((uint64_t)(total % runs) * c / runs);
}
__device__ __forceinline__ uint32_t run_owner(uint32_t total, uint32_t tile, uint32_t runs) {
  return (uint32_t)((((uint64_t)tile + 1) * runs - 1) / total);
}

// A sequence's positions [lo, lo + count) that are attended to; a position outside the table (or below -1) sets DOMAIN.
__device__ __forceinline__ void span_of(const AttnPagesArgs& g, uint32_t s, uint32_t* lo, uint32_t* count) {
  const int32_t p = g.positions[s];
  uint32_t n = p < 0 ? 0u : (uint32_t)p + 1u;
  if (p < -1 || n > g.cache.width * g.cache.page) { set_domain(g.err); n = 0; }
  *lo = g.window && n > g.window ? n - g.window : 0u;
  *count = n - *lo;
}

// Where a warp's next tile lies.
struct Cursor {
  uint32_t s, tile, tiles, lo, end;
};

// The last sequence that starts at or before a tile of the list: it has tiles.
__device__ __forceinline__ uint32_t sequence_of(const uint32_t* prefix, uint32_t n, uint32_t tile) {
  uint32_t lo = 0, hi = n - 1;
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) / 2;
    if (prefix[mid] <= tile) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// A part [rows][D], or with no `part` the result's rows, again from whole operands: where a value is infinite (or an F32 one too
// large for its parts) the products of the parts hold 0 * inf, which the steps do not.  `top` and `den` are row lane / 4's.  A lane a
// position for the scores, a lane every 32nd column for the rows: rare, so it is simple and out of the way.
template <typename KV, int D>
__device__ __noinline__ void sum_again(const AttnPlan& a, uint32_t s, uint32_t first, uint32_t end, uint32_t kvh, uint32_t head0, uint32_t rows,
                                       float tops, float dens, float* part) {
  const AttnPagesArgs& g = a.g;
  const uint32_t lane = threadIdx.x % 32;
  const uint64_t ld = (uint64_t)g.cache.kv_heads * D, head_at = (uint64_t)kvh * D;
  for (uint32_t r = 0; r < rows; ++r) {
    const float top = __shfl_sync(0xffffffffu, tops, r * 4), den = __shfl_sync(0xffffffffu, dens, r * 4);
    float v[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) v[i] = 0.f;
    for (uint32_t p0 = first; p0 < end; p0 += 32) {
      const int64_t row = p0 + lane < end ? pool_row(g.cache, s, p0 + lane, g.err) : -1;
      float w = 0.f;
      if (row >= 0) {
        for (int i = 0; i < D; ++i)
          w = fmaf(load_float(g.q.p, (uint64_t)s * g.q.ld + (uint64_t)(head0 + r) * D + i, g.q.bf16),
                   load_float(g.cache.keys, (uint64_t)row * ld + head_at + i, sizeof(KV) == 2), w);
        w = exp2_fast(fmaf(w, a.scale_log2, -top));
        w = w > 1.f ? 1.f : w;           // summed in another order than `top`'s, a score may lie a rounding above it
      }
      for (int j = 0; j < 32; ++j) {
        const int64_t from = __shfl_sync(0xffffffffu, row, j);
        const float x = __shfl_sync(0xffffffffu, w, j);
        if (from >= 0)
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
            v[i] = fmaf(x, load_float(g.cache.values, (uint64_t)from * ld + head_at + i * 32 + lane, sizeof(KV) == 2), v[i]);
      }
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
      if (part) part[r * D + i * 32 + lane] = v[i];
      else store_float(g.out, ((uint64_t)s * g.cache.heads + head0 + r) * D + i * 32 + lane, g.out_bf16, v[i] / den);
    }
  }
}

// QP: the queries' parts.  EXACT: an F32 result.
template <typename KV, int D, int QP, bool EXACT>
__global__ void __launch_bounds__(Form<KV, D>::THREADS, Form<KV, D>::BLOCKS) attention_pages_kernel(const __grid_constant__ AttnPlan a) {
  using F = Form<KV, D>;
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t warp_sum[F::WARPS];
  __shared__ uint32_t valid[F::WARPS][MAX_STAGES];
  pdl_enter();
  const AttnPagesArgs& g = a.g;
  const PageView& cache = g.cache;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t n = (uint32_t)g.n;
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem);                       // [n + 1] tiles before a sequence
  unsigned char* stages = smem + F::prefix_bytes(n) + warp * a.stages * F::STAGE;

  // ---- the tile list: a prefix sum over the sequences; rows of sequences without positions are zero
  if (!a.together) {
    const uint32_t each = (n + F::THREADS - 1) / F::THREADS, first = tid * each;
    uint32_t sum = 0;
    for (uint32_t s = first; s < first + each && s < n; ++s) {
      uint32_t lo, count;
      span_of(g, s, &lo, &count);
      prefix[s] = sum;
      sum += (count + 15) / 16;
    }
    uint32_t scan = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const uint32_t up = __shfl_up_sync(0xffffffffu, scan, o);
      if (lane >= o) scan += up;
    }
    if (lane == 31) warp_sum[warp] = scan;
    __syncthreads();
    uint32_t before = scan - sum;
    for (int w = 0; w < warp; ++w) before += warp_sum[w];
    for (uint32_t s = first; s < first + each && s < n; ++s) prefix[s] += before;
    if (tid == F::THREADS - 1) prefix[n] = before + sum;
    __syncthreads();
  }
  const uint32_t total = a.together ? 0 : prefix[n], out_cols = cache.heads * D;
  if (!a.together) {
    if (blockIdx.x == 0)
      for (uint32_t s = tid; s <= n; s += F::THREADS) a.prefix[s] = prefix[s];
    for (uint32_t s = blockIdx.x; s < n; s += gridDim.x)
      if (prefix[s] == prefix[s + 1])
        for (uint32_t j = tid; j < out_cols; j += F::THREADS) store_float(g.out, (uint64_t)s * out_cols + j, g.out_bf16, 0.f);
  }

  const auto enter = [&](Cursor& c) {    // the bounds of sequence c.s
    uint32_t count;
    span_of(g, c.s, &c.lo, &count);
    c.end = c.lo + count;
    c.tiles = (count + 15) / 16;
  };
  const auto seek = [&](Cursor& c, uint32_t tile) {
    c.s = sequence_of(prefix, n, tile);
    enter(c);
    c.tile = tile - prefix[c.s];
  };
  const auto next_sequence = [&](Cursor& c) {
    c.tile = 0;
    do ++c.s; while (c.s < n && prefix[c.s] == prefix[c.s + 1]);
    if (c.s < n) enter(c);
  };
  const int gr = lane >> 2, t4 = lane & 3;
  const uint32_t ld = cache.kv_heads * D * (uint32_t)sizeof(KV);              // bytes of a pool row
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(stages) + (lane % F::LANES) * 16;

  uint32_t rank = 0;                     // this block's in its cluster
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  const uint32_t tasks = a.together ? gridDim.x * F::WARPS : a.runs * a.jobs;
  for (uint32_t task = blockIdx.x * F::WARPS + warp; task < tasks; task += gridDim.x * F::WARPS) {   // the same for a warp's lanes
    uint32_t job, count;                 // its tiles: `count` of them from `ahead`
    Cursor ahead;
    if (a.together) {                    // a share of one sequence's
      job = blockIdx.x / a.together % a.jobs;
      ahead.s = blockIdx.x / a.together / a.jobs;
      enter(ahead);
      const uint32_t warps = a.together * F::WARPS, share = (ahead.tiles + warps - 1) / warps;
      ahead.tile = (rank * F::WARPS + warp) * share;
      count = ahead.tile < ahead.tiles ? min(share, ahead.tiles - ahead.tile) : 0;
    } else {
      const uint32_t run = task / a.jobs, start = run_start(total, run, a.runs), stop = run_start(total, run + 1, a.runs);
      if (start >= stop) continue;
      job = task % a.jobs;
      count = stop - start;
      seek(ahead, start);
    }
    const uint32_t kvh = job / a.row_tiles, r0 = job % a.row_tiles * HEADS;
    const uint32_t rows = a.group - r0 < HEADS ? a.group - r0 : HEADS, head0 = kvh * a.group + r0;

    // ---- the copies' side: the rows of the tile that is issued next
    Cursor here = ahead;                 // the run's other side: the tile that is summed next
    uint32_t to_issue = count;
    int32_t row = -1;                    // lane % 16's pool row of the tile at `ahead`, -1: not attended
    const auto look_up = [&]() {
      row = -1;
      const uint32_t p = ahead.lo + ahead.tile * 16 + (lane & 15);
      if (to_issue && p < ahead.end) {
        const uint32_t at = (uint32_t)(((uint64_t)p * a.page_magic) >> (32 + a.page_shift));
        const int32_t page = cache.table[(uint64_t)ahead.s * cache.width + at];
        if (page >= 0 && (uint32_t)page < cache.pages) row = page * (int32_t)cache.page + (int32_t)(p - at * cache.page);
        else set_domain(g.err);
      }
    };
    look_up();
    const uint64_t head_at = (uint64_t)kvh * D * sizeof(KV) + (lane % F::LANES) * 16;
    const char *key_at = (const char*)cache.keys + head_at, *value_at = (const char*)cache.values + head_at;
    int issue_stage = 0;
    const auto copy = [&](uint32_t at, const char* from_at, int pitch) {
#pragma unroll
      for (int i = 0; i < F::REST; ++i) {
        const int r = i * F::ROWS + lane / F::LANES;
        const int32_t from = __shfl_sync(0xffffffffu, row, r);
        const bool on = from >= 0;
        const char* x = from_at + (uint64_t)(uint32_t)(on ? from : 0) * ld;
#pragma unroll
        for (int c = 0; c < F::PIECES; ++c) cp_async16(at + r * pitch + c * F::LANES * 16, x + c * F::LANES * 16, on);
      }
    };
    const auto issue_keys = [&]() {      // a group of copies each, the keys' and the values' of a tile in turn
      if (to_issue) {
        const uint32_t there = __ballot_sync(0xffffffffu, row >= 0);
        if (lane == 0) valid[warp][issue_stage] = there & 0xffffu;
        copy(to + issue_stage * F::STAGE, key_at, F::K_PITCH);
      }
      cp_async_commit();
    };
    const auto issue_values = [&]() {
      if (to_issue) {
        copy(to + issue_stage * F::STAGE + 16 * F::K_PITCH, value_at, F::V_PITCH);
        if (++ahead.tile == ahead.tiles && to_issue > 1) next_sequence(ahead);
        --to_issue;
        look_up();
      }
      cp_async_commit();
      if (++issue_stage == a.stages) issue_stage = 0;
    };
    for (int i = 0; i < a.stages; ++i) { issue_keys(); issue_values(); }

    // ---- the run's sequences, one after another
    int stage = 0, piece = 0;
    for (uint32_t left = count; left > 0; ++piece) {
      const uint32_t steps = left < here.tiles - here.tile ? left : here.tiles - here.tile;
      const bool whole = here.tile == 0 && steps == here.tiles;

      // the queries' fragments: row gr's leading part and, as row gr + 8, its next one (the third by itself); on the F32 path
      // the queries themselves, which a product takes apart (their parts are too many registers)
      uint32_t qf[D / (F::BF ? 16 : 8)][F::BF ? 2 * QP : 2];
      {
        const uint64_t from = (uint64_t)here.s * g.q.ld + (uint64_t)(head0 + gr) * D;
        const bool live = gr < (int)rows;
        if constexpr (F::BF) {
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              const int e = kk * 16 + hf * 8 + 2 * t4;
              float u = live ? load_float(g.q.p, from + e, g.q.bf16) : 0.f, v = live ? load_float(g.q.p, from + e + 1, g.q.bf16) : 0.f;
#pragma unroll
              for (int p = 0; p < QP; ++p) {
                const uint32_t x = next_part(u, p + 1 == QP), y = next_part(v, p + 1 == QP);
                qf[kk][p * 2 + hf] = x | (y << 16);
              }
            }
        } else {
          // the products' inner index in the order 0, 2, 4, 6, 1, 3, 5, 7 of each eight columns, for both operands
#pragma unroll
          for (int kk = 0; kk < D / 8; ++kk)
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              qf[kk][hf] = live ? __float_as_uint(load_float(g.q.p, from + kk * 8 + 2 * t4 + hf, g.q.bf16)) : 0u;
            }
        }
      }
      float o[D / 8][2];
#pragma unroll
      for (int j = 0; j < D / 8; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) o[j][e] = 0.f;
      float m = -FLT_MAX, l = 0.f;       // row gr's; the sum is this lane's own
      for (uint32_t step = 0; step < steps; ++step) {
        cp_async_wait(2 * a.stages - 1);
        __syncwarp();                    // every lane's copies of the keys are in
        const unsigned char* st = stages + stage * F::STAGE;
        const uint32_t live = valid[warp][stage];
        if (++stage == a.stages) stage = 0;
        const uint32_t k_at = (uint32_t)__cvta_generic_to_shared(st), v_at = k_at + 16 * F::K_PITCH;

        // scores of 8 heads x 16 positions: lane holds row gr and positions 8 nt + 2 t4 + {0, 1}
        float x[2][2];
        if constexpr (F::BF) {
          const uint32_t kb = k_at + ((lane & 7) + ((lane >> 4) & 1) * 8) * F::K_PITCH + ((lane >> 3) & 1) * 16;
          float c[2][2][4];              // two chains of products a score: each waits for the one before it
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i >> 2][(i >> 1) & 1][(i & 1) * 2] = c[i >> 2][(i >> 1) & 1][(i & 1) * 2 + 1] = 0.f;
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk) {
            uint32_t b[4];
            ldmatrix4(b, kb + kk * 32);
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              if constexpr (QP == 1) mma_bf16(c[kk & 1][nt], qf[kk][0], 0u, qf[kk][1], 0u, b[2 * nt], b[2 * nt + 1]);
              else mma_bf16(c[kk & 1][nt], qf[kk][0], qf[kk][2], qf[kk][1], qf[kk][3], b[2 * nt], b[2 * nt + 1]);
              if constexpr (QP == 3) mma_bf16(c[kk & 1][nt], 0u, qf[kk][4], 0u, qf[kk][5], b[2 * nt], b[2 * nt + 1]);
            }
          }
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              x[nt][e] = c[0][nt][e] + c[1][nt][e];
              if constexpr (QP > 1) x[nt][e] += c[0][nt][2 + e] + c[1][nt][2 + e];
            }
        } else {
          float c[2][2][4];
#pragma unroll
          for (int i = 0; i < 8; ++i) c[i >> 2][(i >> 1) & 1][(i & 1) * 2] = c[i >> 2][(i >> 1) & 1][(i & 1) * 2 + 1] = 0.f;
#pragma unroll
          for (int kk = 0; kk < D / 8; ++kk) {
            const uint32_t q0 = tf32_of(__uint_as_float(qf[kk][0])), q1 = tf32_of(__uint_as_float(qf[kk][1]));
            const uint32_t p0 = tf32_rest(__uint_as_float(qf[kk][0])), p1 = tf32_rest(__uint_as_float(qf[kk][1]));
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              const float2 k = lds2(k_at + (nt * 8 + gr) * F::K_PITCH + (kk * 8 + 2 * t4) * 4);
              mma_tf32(c[kk & 1][nt], q0, p0, q1, p1, tf32_rest(k.x), tf32_rest(k.y));
              mma_tf32(c[kk & 1][nt], q0, p0, q1, p1, tf32_of(k.x), tf32_of(k.y));
            }
          }
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[nt][e] = (c[0][nt][e] + c[1][nt][e]) + (c[0][nt][2 + e] + c[1][nt][2 + e]);
        }
        // An infinite key gives 0 * inf among the parts' products: such a score is taken again from whole operands.
        if (__any_sync(0xffffffffu, !(x[0][0] == x[0][0] && x[0][1] == x[0][1] && x[1][0] == x[1][0] && x[1][1] == x[1][1]))) {
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e)
              if (x[nt][e] != x[nt][e] && gr < (int)rows) {
                const unsigned char* k = st + (nt * 8 + 2 * t4 + e) * F::K_PITCH;
                float t = 0.f;
                for (int i = 0; i < D; ++i)
                  t = fmaf(load_float(g.q.p, (uint64_t)here.s * g.q.ld + (uint64_t)(head0 + gr) * D + i, g.q.bf16), load_float(k, i, F::BF), t);
                x[nt][e] = t;
              }
        }

        __syncwarp();                    // every lane is done with the keys
        issue_keys();

        // running softmax: new maximum, the factor of what was summed before, the weights
        const uint32_t off = live == 0xffffu ? 0u : ~live >> (2 * t4);         // bit 8 nt + e: not attended
        float y[2][2];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) y[nt][e] = x[nt][e] * a.scale_log2;
        if (off) {
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) y[nt][e] = (off >> (8 * nt + e)) & 1 ? -INFINITY : y[nt][e];
        }
        float top = fmaxf(fmaxf(y[0][0], y[0][1]), fmaxf(y[1][0], y[1][1]));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        top = fmaxf(top, m);
        const float f = exp2_fast(m - top);
        m = top;
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 2; ++e) x[nt][e] = exp2_fast(fmaf(x[nt][e], a.scale_log2, -m));   // one rounding, of the difference
        if (off) {
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) x[nt][e] = (off >> (8 * nt + e)) & 1 ? 0.f : x[nt][e];
        }
        l = fmaf(l, f, (x[0][0] + x[0][1]) + (x[1][0] + x[1][1]));

        // rows = rows * factor + weights x values
        cp_async_wait(2 * a.stages - 1);
        __syncwarp();                    // every lane's copies of the values are in
        if constexpr (F::BF) {
          uint32_t w[3][2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            float u = x[nt][0], v = x[nt][1];
            w[0][nt] = bf16x2(u, v);
            u -= low_of(w[0][nt]); v -= high_of(w[0][nt]);
            w[1][nt] = bf16x2(u, v);
            if constexpr (EXACT) w[2][nt] = bf16x2(u - low_of(w[1][nt]), v - high_of(w[1][nt]));
          }
          const uint32_t vb = v_at + ((lane & 7) + ((lane >> 3) & 1) * 8) * F::V_PITCH + (lane >> 4) * 16;
#pragma unroll
          for (int j = 0; j < D / 16; ++j) {
            uint32_t b[4];
            ldmatrix4_t(b, vb + j * 32);
#pragma unroll
            for (int hf = 0; hf < 2; ++hf) {
              float* r = o[2 * j + hf];
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              if constexpr (EXACT) mma_bf16(c, 0u, w[2][0], 0u, w[2][1], b[2 * hf], b[2 * hf + 1]);
              mma_bf16(c, w[0][0], w[1][0], w[0][1], w[1][1], b[2 * hf], b[2 * hf + 1]);
              r[0] = fmaf(r[0], f, c[0] + c[2]);
              r[1] = fmaf(r[1], f, c[1] + c[3]);
            }
          }
        } else {
          uint32_t hi[2][2], lo[2][2];
#pragma unroll
          for (int nt = 0; nt < 2; ++nt)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              hi[nt][e] = tf32_of(x[nt][e]);
              lo[nt][e] = tf32_rest(x[nt][e]);
            }
          const uint32_t vs = v_at + 2 * t4 * F::V_PITCH + gr * 4;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int nt = 0; nt < 2; ++nt) {
              const float u = lds1(vs + nt * 8 * F::V_PITCH + j * 32);
              const float v = lds1(vs + (nt * 8 + 1) * F::V_PITCH + j * 32);
              mma_tf32(c, hi[nt][0], lo[nt][0], hi[nt][1], lo[nt][1], tf32_rest(u), tf32_rest(v));
              mma_tf32(c, hi[nt][0], lo[nt][0], hi[nt][1], lo[nt][1], tf32_of(u), tf32_of(v));
            }
            o[j][0] = fmaf(o[j][0], f, c[0] + c[2]);
            o[j][1] = fmaf(o[j][1], f, c[1] + c[3]);
          }
        }
        __syncwarp();                    // every lane is done with the values
        issue_values();
      }

      // ---- the sequence's result, or its part of one
      l += __shfl_xor_sync(0xffffffffu, l, 1);
      l += __shfl_xor_sync(0xffffffffu, l, 2);
      // an infinite largest score: the differences to it leave no weight, where the steps' exp(inf - inf) is NaN
      const float den = m == INFINITY ? NAN : (l < FLT_MIN ? FLT_MIN : l);
      float* part = nullptr;             // (a warp's own tiles are behind it: their room takes its part where the block joins them)
      if (a.together) part = reinterpret_cast<float*>(stages);
      else if (!whole) part = a.part + ((uint64_t)task * 2 + (piece ? 1 : 0)) * a.slot;
      float odd = 0.f;                   // NaN where a sum is no finite number
      if (gr < (int)rows) {
        if (!part) {
          const uint64_t at = (uint64_t)here.s * out_cols + (uint64_t)(head0 + gr) * D + 2 * t4;
#pragma unroll
          for (int j = 0; j < D / 8; ++j) {
            const float u = o[j][0] / den, v = o[j][1] / den;
            if (g.out_bf16)
              *reinterpret_cast<uint32_t*>(reinterpret_cast<uint16_t*>(g.out) + at + j * 8) =
                  (uint32_t)f32_to_bf16_bits(__float_as_uint(u)) | ((uint32_t)f32_to_bf16_bits(__float_as_uint(v)) << 16);
            else *reinterpret_cast<float2*>(reinterpret_cast<float*>(g.out) + at + j * 8) = make_float2(u, v);
          }
        } else {
#pragma unroll
          for (int j = 0; j < D / 8; ++j) *reinterpret_cast<float2*>(part + gr * D + j * 8 + 2 * t4) = make_float2(o[j][0], o[j][1]);
          if (t4 == 0) *reinterpret_cast<float2*>(part + a.slot / (D + 4) * D + gr * 4) = make_float2(m, l);
        }
#pragma unroll
        for (int j = 0; j < D / 8; ++j) odd = fmaf(o[j][0], 0.f, fmaf(o[j][1], 0.f, odd));
      }
      if (__any_sync(0xffffffffu, odd != odd)) {
        __syncwarp();                    // what the lanes have written is written again by others
        const uint32_t first = here.lo + here.tile * 16, end = min(here.end, first + steps * 16);
        sum_again<KV, D>(a, here.s, first, end, kvh, head0, rows, m, den, part);
      }
      left -= steps;
      here.tile += steps;
      if (here.tile == here.tiles && left > 0) next_sequence(here);
    }
    cp_async_wait(0);
    __syncwarp();
    if (a.together) {                    // once a block: its warps' parts, then its cluster's, each in their order
      __syncthreads();
      const uint32_t warps = a.together * F::WARPS, share = (here.tiles + warps - 1) / warps, all = share ? (here.tiles + share - 1) / share : 0;
      const uint32_t held = all > rank * F::WARPS ? min(all - rank * F::WARPS, (uint32_t)F::WARPS) : 0;   // of `all` warps with tiles, this block's
      const uint32_t ml = a.slot / (D + 4) * D;
      const uint64_t at = (uint64_t)here.s * out_cols + (uint64_t)head0 * D;
      unsigned char* parts = smem + F::prefix_bytes(n);
      float* mine = reinterpret_cast<float*>(parts + F::STAGE);       // behind the first warp's part
      for (uint32_t j = tid; j < rows * D; j += F::THREADS) {
        const uint32_t r = j / D;
        float top = -FLT_MAX, v = 0.f, den = 0.f;
        for (uint32_t w = 0; w < held; ++w) top = fmaxf(top, reinterpret_cast<const float*>(parts + w * a.stages * F::STAGE)[ml + r * 4]);
        for (uint32_t w = 0; w < held; ++w) {
          const float* p = reinterpret_cast<const float*>(parts + w * a.stages * F::STAGE);
          const float f = exp2_fast(p[ml + r * 4] - top);
          den = fmaf(p[ml + r * 4 + 1], f, den);
          v = fmaf(p[j], f, v);
        }
        if (a.together == 1) store_float(g.out, at + j, g.out_bf16, v / (den < FLT_MIN ? FLT_MIN : den));
        else {
          mine[j] = v;
          if (j % D == 0) { mine[ml + r * 4] = top; mine[ml + r * 4 + 1] = den; }
        }
      }
      if (a.together > 1) {
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");
        const uint32_t own = (uint32_t)__cvta_generic_to_shared(mine), blocks = (all + F::WARPS - 1) / F::WARPS;
        const auto theirs = [&](uint32_t block, uint32_t i) {
          uint32_t at_block;
          float x;
          asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(at_block) : "r"(own + i * 4), "r"(block));
          asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(x) : "r"(at_block) : "memory");
          return x;
        };
        for (uint32_t j = rank * F::THREADS + tid; j < rows * D; j += a.together * F::THREADS) {
          const uint32_t r = j / D;
          float tops[CLUSTER], dens[CLUSTER], values[CLUSTER], top = -FLT_MAX, v = 0.f, den = 0.f;
#pragma unroll
          for (uint32_t i = 0; i < CLUSTER; ++i) {
            tops[i] = -FLT_MAX; dens[i] = values[i] = 0.f;
            if (i < blocks) { tops[i] = theirs(i, ml + r * 4); dens[i] = theirs(i, ml + r * 4 + 1); values[i] = theirs(i, j); }
          }
#pragma unroll
          for (uint32_t i = 0; i < CLUSTER; ++i) top = fmaxf(top, tops[i]);
#pragma unroll
          for (uint32_t i = 0; i < CLUSTER; ++i) {
            const float f = exp2_fast(tops[i] - top);
            den = fmaf(dens[i], f, den);
            v = fmaf(values[i], f, v);
          }
          store_float(g.out, at + j, g.out_bf16, v / (den < FLT_MIN ? FLT_MIN : den));
        }
        asm volatile("barrier.cluster.arrive.release.aligned;\nbarrier.cluster.wait.acquire.aligned;" ::: "memory");   // no block leaves while it is read
      }
    }
  }
}

// Joins the sequences whose tiles lie in several runs: block (i, h) is query head h of sequence i, or, with fewer runs than
// sequences, of the sequence that run i ends in, if that run is its first.
// rows = sum over the runs, in their order, of rows_c 2^(m_c - m) / sum l_c 2^(m_c - m).
template <int D>
__global__ void __launch_bounds__(1024) attention_pages_join_kernel(const __grid_constant__ AttnPlan a) {
  constexpr int LANES = D / 4;           // a team a run's row, a float4 a lane
  extern __shared__ __align__(16) float sums[];              // [teams][D]
  __shared__ float tops[1024 / LANES], dens[1024 / LANES];
  pdl_enter();
  const AttnPagesArgs& g = a.g;
  const int tid = threadIdx.x, threads = blockDim.x, teams = threads / LANES;
  const uint32_t n = (uint32_t)g.n, total = a.prefix[n], head = blockIdx.y;
  uint32_t s = blockIdx.x;
  if (a.runs < n) {
    const uint32_t mine = run_start(total, blockIdx.x, a.runs), next = run_start(total, blockIdx.x + 1, a.runs);
    if (mine >= next || next >= total) return;               // an empty run, or nothing goes on behind it
    s = sequence_of(a.prefix, n, next);
    if (a.prefix[s] < mine || a.prefix[s] == next) return;   // it began before this run, or begins behind it
  }
  const uint32_t first = a.prefix[s], end = a.prefix[s + 1];
  if (first >= end) return;
  const uint32_t c0 = run_owner(total, first, a.runs), c1 = run_owner(total, end - 1, a.runs);
  if (c0 == c1) return;                                      // written whole
  const uint32_t in = head % a.group, job = head / a.group * a.row_tiles + in / HEADS, r = in % HEADS;
  const uint32_t ml = a.slot / (D + 4) * D + r * 4;
  const bool later = run_start(total, c0, a.runs) != first;  // the sequence is not the first of its first run
  const auto piece = [&](uint32_t c) { return a.part + (((uint64_t)c * a.jobs + job) * 2 + (c == c0 && later ? 1 : 0)) * a.slot; };
  // an empty run lies between two others only where there are fewer tiles than runs: it holds nothing
  const auto there = [&](uint32_t c) { return run_start(total, c, a.runs) < run_start(total, c + 1, a.runs); };
  const int team = tid / LANES, lane = tid % LANES;
  if (team < teams) {
    // every fourth run's part asked for before the first of four is used; the running maximum as in the tiles
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
    float top = -FLT_MAX, den = 0.f;
    for (uint32_t c = c0 + team; c <= c1; c += 4 * teams) {
      float4 x[4];
      float2 w[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        x[i] = make_float4(0.f, 0.f, 0.f, 0.f);
        w[i] = make_float2(-FLT_MAX, 0.f);
        const uint32_t run = c + i * teams;
        if (run <= c1 && there(run)) {
          const float* p = piece(run);
          w[i] = *reinterpret_cast<const float2*>(p + ml);
          x[i] = *reinterpret_cast<const float4*>(p + r * D + lane * 4);
        }
      }
      const float now = fmaxf(fmaxf(fmaxf(w[0].x, w[1].x), fmaxf(w[2].x, w[3].x)), top), keep = exp2_fast(top - now);
      top = now;
      v.x *= keep; v.y *= keep; v.z *= keep; v.w *= keep;
      den *= keep;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = exp2_fast(w[i].x - top);
        den = fmaf(w[i].y, f, den);
        v.x = fmaf(x[i].x, f, v.x); v.y = fmaf(x[i].y, f, v.y); v.z = fmaf(x[i].z, f, v.z); v.w = fmaf(x[i].w, f, v.w);
      }
    }
    *reinterpret_cast<float4*>(sums + team * D + lane * 4) = v;
    if (lane == 0) { tops[team] = top; dens[team] = den; }
  }
  __syncthreads();
  for (int j = tid; j < D; j += threads) {
    float top = -FLT_MAX, t = 0.f, l = 0.f;
    for (int w = 0; w < teams; ++w) top = fmaxf(top, tops[w]);
    for (int w = 0; w < teams; ++w) {
      const float f = exp2_fast(tops[w] - top);
      t = fmaf(sums[w * D + j], f, t);
      l = fmaf(dens[w], f, l);
    }
    store_float(g.out, (uint64_t)s * g.cache.heads * D + (uint64_t)head * D + j, g.out_bf16, t / (l < FLT_MIN ? FLT_MIN : l));
  }
}

// The current device's SMs, asked for once a device.
int sm_count() {
  static const char key = 0;
  int v = 0;
  if (device_value_get(&key, &v)) return v;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&v, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 148;
  device_value_set(&key, v);
  return v;
}

// How a launch of `n` sequences is cut, from the shapes alone.
struct Cut { uint64_t n; uint32_t group, row_tiles, jobs, runs, slot, workers; uint64_t tiles; int together; };
Cut cut_of(const AttnPagesArgs& g, uint64_t left, int dim, int workers, int warps) {
  Cut c;
  c.group = g.cache.heads / g.cache.kv_heads;
  c.row_tiles = (c.group + HEADS - 1) / HEADS;
  c.jobs = g.cache.kv_heads * c.row_tiles;
  c.slot = (c.group < HEADS ? c.group : HEADS) * (dim + 4);
  c.workers = workers;
  uint64_t positions = (uint64_t)g.cache.width * g.cache.page;
  if (g.window && positions > g.window) positions = g.window;
  c.tiles = (positions + 15) / 16;                           // a sequence's, at most (below 2^28)
  c.n = left < MAX_SEQUENCES ? left : MAX_SEQUENCES;
  if (c.tiles && c.n > 0xffffffffull / c.tiles) c.n = 0xffffffffull / c.tiles;
  // Together: the second launch, the list and the sums before it cost 3 to 6 us, an unequal share of the work costs its length.
  // So where a (sequence, job) can have blocks of its own, as many as leave each warp two tiles if there is room for them
  // (7/8 of it: clusters do not fill every SM), and then no warp has more than so many tiles: half an F32 cache's, whose tile
  // takes longer, and half where the blocks leave a quarter of the GPU free, which runs would use.  us by runs / together, 32
  // heads of 128 over 8: one sequence of 100 10.4 / 8.6, of 2,000 13.7 / 12.6, of 4,000 15.9 / 16.8; 8 of 5 to 600 13.9 / 12.5, to
  // 4,000 27.8 / 27.8; 37 to 600 25.0 / 20.2, to 2,000 46.2 / 43.2, to 4,000 71.9 / 75.6; F32, 8 heads of 96, 8 to 1,000 15.9 / 14.0,
  // to 4,000 31.0 / 36.7.
  const uint64_t teams = c.n * c.jobs, resident = (uint64_t)workers / warps;
  c.together = teams <= resident;
  while (c.together && c.together < CLUSTER && teams * c.together * 2 <= resident * 7 / 8 && c.tiles > 2ull * c.together * warps) c.together *= 2;
  const uint64_t most = (g.cache.bf16 ? 8 : 4) * (teams * c.together * 4 >= resident * 3 ? 2 : 1);
  if (c.tiles > most * c.together * warps) c.together = 0;
  // Runs: as many as give every warp one (run, head).  With so many heads that a warp more or less in that division weighs,
  // the count whose last round of warps is fullest (8 sequences to 1,000, 600 heads of 64: 183 us, by one run a head 198).
  uint32_t runs = c.jobs < c.workers ? c.workers / c.jobs : 1;
  if (runs < 8) {
    const auto rounds = [&](uint32_t r) { return (double)(((uint64_t)r * c.jobs + c.workers - 1) / c.workers) / r; };
    for (uint32_t r = runs + 1; r <= 16; ++r)
      if (rounds(r) < 0.95 * rounds(runs)) runs = r;
  }
  if (runs > c.n * c.tiles) runs = (uint32_t)(c.n * c.tiles);
  c.runs = runs < 1 ? 1 : runs;
  return c;
}

template <typename KV, int D, int QP, bool EXACT>
cudaError_t attention_form(const AttnPagesArgs& g, void* scratch, int* launches, cudaStream_t stream) {
  using F = Form<KV, D>;
  const int workers = F::BLOCKS * F::WARPS * sm_count();
  AttnPlan a;
  a.g = g;
  a.page_shift = 31 - __builtin_clz(g.cache.page);
  a.page_magic = (1ull << (32 + a.page_shift)) / g.cache.page + 1;
  a.scale_log2 = g.scale * 1.44269504088896340736f;
  const int limit = 228 * 1024 / F::BLOCKS - 1024 - 256;   // a block's share of an SM's shared memory, less what the launch and the statics take
  cudaError_t e = ensure_dynamic_smem((const void*)attention_pages_kernel<KV, D, QP, EXACT>, limit);
  if (e != cudaSuccess) return e;
  for (uint64_t at = 0; at < g.n;) {
    const Cut c = cut_of(g, g.n - at, D, workers, F::WARPS);
    a.together = c.together;
    a.group = c.group; a.row_tiles = c.row_tiles; a.jobs = c.jobs; a.runs = c.runs; a.slot = c.slot;
    a.prefix = (uint32_t*)scratch;
    a.part = (float*)((char*)scratch + 4096);
    a.g.n = c.n;
    a.g.cache.table = g.cache.table + at * g.cache.width;
    a.g.positions = g.positions + at;
    a.g.q.p = (const char*)g.q.p + at * g.q.ld * (g.q.bf16 ? 2 : 4);
    a.g.out = (char*)g.out + at * g.cache.heads * D * (g.out_bf16 ? 2 : 4);
    const int fixed = F::prefix_bytes((uint32_t)c.n);
    a.stages = (limit - fixed) / (F::WARPS * F::STAGE);
    if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
    if (a.stages < 2) return cudaErrorNotSupported;
    uint64_t blocks = c.together ? c.n * c.jobs * c.together : ((uint64_t)c.runs * c.jobs + F::WARPS - 1) / F::WARPS;
    if (blocks > (uint64_t)F::BLOCKS * sm_count()) blocks = (uint64_t)F::BLOCKS * sm_count();
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)blocks); cfg.blockDim = dim3(F::THREADS); cfg.stream = stream;
    cfg.dynamicSmemBytes = fixed + a.stages * F::WARPS * F::STAGE;
    cudaLaunchAttribute attr[2];
    if (pdl_enabled()) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
      attr[cfg.numAttrs++].val.programmaticStreamSerializationAllowed = 1;
    }
    if (c.together > 1) {
      attr[cfg.numAttrs].id = cudaLaunchAttributeClusterDimension;
      attr[cfg.numAttrs].val.clusterDim.x = c.together; attr[cfg.numAttrs].val.clusterDim.y = 1; attr[cfg.numAttrs++].val.clusterDim.z = 1;
    }
    cfg.attrs = attr;
    e = cudaLaunchKernelEx(&cfg, attention_pages_kernel<KV, D, QP, EXACT>, a);
    if (e != cudaSuccess) return e;
    ++*launches;
    if (!c.together && c.runs > 1 && c.tiles > 1) {                         // a sequence of one tile is never divided
      // a sequence's runs over as many teams as leave each a few (one sequence of 131,001, 148 runs: 105 us by 1,024 threads, 115 by
      // 128; 128 sequences to 8,192, about one run each: 398 by 128, 454 by 1,024)
      constexpr int LANES = D / 4;
      const uint64_t each = c.runs / c.n;
      const int threads = each > 64 ? 1024 : (each > 16 ? 512 : (each > 4 ? 256 : 128));
      launch_pdl(attention_pages_join_kernel<D>, dim3((unsigned)(c.n < c.runs ? c.n : c.runs), g.cache.heads), dim3(threads),
                 threads / LANES * D * sizeof(float), stream, a);
      e = cudaGetLastError();
      if (e != cudaSuccess) return e;
      ++*launches;
    }
    at += c.n;
  }
  return cudaSuccess;
}

// The form for the types: an operand's parts as the precision note says.
template <int D>
cudaError_t attention_dim(const AttnPagesArgs& g, void* scratch, int* launches, cudaStream_t stream) {
  if (!g.cache.bf16) return attention_form<float, D, 2, true>(g, scratch, launches, stream);
  if (g.q.bf16) return g.out_bf16 ? attention_form<uint16_t, D, 1, false>(g, scratch, launches, stream)
                                  : attention_form<uint16_t, D, 1, true>(g, scratch, launches, stream);
  return g.out_bf16 ? attention_form<uint16_t, D, 3, false>(g, scratch, launches, stream)
                    : attention_form<uint16_t, D, 3, true>(g, scratch, launches, stream);
}

template <int D>
size_t scratch_of(const AttnPagesArgs& g) {
  const int warps = g.cache.bf16 ? Form<uint16_t, D>::WARPS : Form<float, D>::WARPS;
  const int blocks = g.cache.bf16 ? Form<uint16_t, D>::BLOCKS : Form<float, D>::BLOCKS;
  const Cut c = cut_of(g, g.n, D, blocks * warps * sm_count(), warps);
  return c.together ? 0 : 4096 + (size_t)c.runs * c.jobs * 2 * c.slot * sizeof(float);
}

}  // namespace

bool attention_pages_dim_ok(uint32_t d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// The prefix sums, and two pieces for every (run, head) of the largest launch; none where no launch leaves pieces.
size_t attention_pages_scratch_bytes(const AttnPagesArgs& g) {
  switch (g.cache.dim) {
    case 32: return scratch_of<32>(g);
    case 64: return scratch_of<64>(g);
    case 96: return scratch_of<96>(g);
    case 128: return scratch_of<128>(g);
    case 192: return scratch_of<192>(g);
    default: return scratch_of<256>(g);
  }
}

cudaError_t launch_attention_pages(const AttnPagesArgs& g, void* scratch, int* launches, cudaStream_t stream) {
  *launches = 0;
  if (g.n == 0) return cudaSuccess;
#define GO(D) case D: return attention_dim<D>(g, scratch, launches, stream)
  switch (g.cache.dim) {
    GO(32); GO(64); GO(96); GO(128); GO(192); GO(256);
    default: return cudaErrorNotSupported;
  }
#undef GO
}

}  // namespace b200
