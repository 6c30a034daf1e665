// Attention of one new token a sequence over the pages of its cache (`b200_attention_pages`).
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

// out = softmax(scale q K^T) V over one sequence's positions, the query heads of one key/value head (up to 16, one
// tensor-core row tile) together, so that keys and values are read once for all of them.  The bound is that read: HBM.
//
// Split: the work is a list of tiles (16 positions a warp) in the order sequence, key/value head, position, and every block
// takes an equal run of it, whatever the lengths: a block's run may end inside a sequence and the next block's goes on there.
// A run's pieces that are whole (sequence, head) results are written at once, the others as (maximum, sum, rows) for the
// second kernel to join, at most two a block.  The lengths are on the device, so the list is made there, from a prefix sum.
//
// A warp's own pipeline: it copies its 16 keys and 16 values of each tile to shared memory by 16-byte asynchronous copies,
// a few tiles ahead (row addresses through the page table, fetched one tile before they are used), and keeps its own
// running maximum, sum and rows; the block's warps meet only at the end of a (sequence, head).  Copies run on across it.
//
// Precision: keys and values are the cache's own values.  On the BF16 path the operands that are F32 are handed to the BF16
// tensor cores as sums of BF16 parts -- an F32 query as three (exact) or, for a BF16 result, two (2^-16), a probability as
// three or two -- since the tensor cores idle while the cache is read.  On the F32 path every operand is two TF32 parts and
// three products are kept (2^-21).  For an F32 result a tile's
// products start from zero and are added to the running rows in F32.
template <typename KV, int D>
struct Form {
  static constexpr bool BF = sizeof(KV) == 2;
  static constexpr int WARPS = !BF && D > 128 ? 2 : 4;        // an F32 tile of a wide head is 33 KB a warp
  static constexpr int THREADS = WARPS * 32;
  static constexpr int TILE = WARPS * 16;                     // positions a block's step
  // shared-memory row pitches that let eight rows (or the four position pairs of an F32 fragment) fall into distinct banks
  static constexpr int K_PITCH = D * (int)sizeof(KV) + (BF ? 16 : 32);
  static constexpr int V_PITCH = D * (int)sizeof(KV) + 16;
  static constexpr int Q_PITCH = K_PITCH;
  static constexpr int STAGE = 16 * (K_PITCH + V_PITCH);      // a warp's stage
  // a copy instruction: LANES lanes a row (a whole 128-byte line where rows are whole lines), ROWS rows; a lane's rows of a
  // tile are REST, its pieces of a row PIECES
  static constexpr int CHUNKS = D * (int)sizeof(KV) / 16;     // 16-byte pieces of a row
  static constexpr int LANES = CHUNKS % 8 ? 4 : 8, ROWS = 32 / LANES, REST = 16 / ROWS, PIECES = CHUNKS / LANES;
  static constexpr int BLOCKS = BF ? (D <= 64 ? 4 : (D <= 128 ? 2 : 1)) : (D <= 64 ? 2 : 1);
  static constexpr int SLAB = 16, SLAB_PITCH = 24;            // columns of the rows merged at a time
  static constexpr int ML = WARPS * 16 * 2 * 4;
  // the queries' parts; the same bytes hold the merged columns once a piece's products are done
  static __host__ __device__ int q_bytes(int parts) {
    const int q = parts * 16 * Q_PITCH, slab = WARPS * 16 * SLAB_PITCH * 4;
    return q > slab ? q : slab;
  }
  static __host__ __device__ int prefix_bytes(uint32_t n) { return (int)(((n + 1) * 4 + 127) / 128 * 128); }
};
constexpr uint32_t MAX_SEQUENCES = 512;  // a launch's; its prefix sums lie in shared memory
constexpr int MAX_STAGES = 4;

struct AttnPlan {
  AttnPagesArgs g;
  uint64_t page_magic;                   // p / page = p * magic >> (32 + page_shift), exact below 2^31
  uint32_t page_shift;
  uint32_t group, row_tiles;             // query heads a key/value head, and their tiles of 16
  uint32_t jobs;                         // kv_heads * row_tiles
  int stages;
  float scale_log2;
  float* part;                           // [blocks][2][16][D + 2]: rows, then (maximum, sum) a row
  uint32_t* prefix;                      // [n + 1], for the join
};

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool there) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
// all but the latest `pending` groups of this thread have arrived
__device__ __forceinline__ void cp_async_wait(int pending) {
  if (pending <= 0) asm volatile("cp.async.wait_group 0;" ::: "memory");
  else if (pending == 1) asm volatile("cp.async.wait_group 1;" ::: "memory");
  else asm volatile("cp.async.wait_group 2;" ::: "memory");
}
__device__ __forceinline__ void ldmatrix4(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldmatrix4_t(uint32_t* r, uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void mma_bf16(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_tf32(float* c, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t tf32_of(float x) {
  uint32_t r;
  asm("cvt.rna.tf32.f32 %0, %1;" : "=r"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ float exp2_fast(float x) {   // the hardware's 2^x: 2 units in the last place, 2^-inf = 0
  float r;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
  return r;
}
__device__ __forceinline__ uint32_t bf16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ float low_of(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float high_of(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// The first tile of block c's run, and the block that a tile is in: runs of total / blocks tiles.
__device__ __forceinline__ uint32_t run_start(uint32_t total, uint32_t c, uint32_t blocks) { return total / blocks * c + total % blocks * c / blocks; }
__device__ __forceinline__ uint32_t run_owner(uint32_t total, uint32_t tile, uint32_t blocks) {
  uint32_t lo = 0, hi = blocks - 1;      // the last c whose run starts at or before `tile`
  while (lo < hi) {
    const uint32_t mid = (lo + hi + 1) / 2;
    if (run_start(total, mid, blocks) <= tile) lo = mid; else hi = mid - 1;
  }
  return lo;
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
  uint32_t s, job, tile, tiles, lo, end;
};

// QP: the queries' parts.  EXACT: an F32 result -- the weights in three parts, and every tile's products added to the rows in
// F32; else two, the rows accumulated by the tensor cores and scaled only when a row's maximum moved.

template <typename KV, int D, int QP, bool EXACT>
__global__ void __launch_bounds__(Form<KV, D>::THREADS, Form<KV, D>::BLOCKS) attention_pages_kernel(const __grid_constant__ AttnPlan a) {
  using F = Form<KV, D>;
  constexpr bool Q_HELD = F::BF && D <= 128 && QP * D <= 256;         // the queries' fragments stay in registers
  extern __shared__ __align__(128) unsigned char smem[];
  __shared__ uint32_t warp_sum[F::WARPS];
  __shared__ uint32_t valid[F::WARPS][MAX_STAGES];
  pdl_enter();
  const AttnPagesArgs& g = a.g;
  const PageView& cache = g.cache;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const uint32_t n = (uint32_t)g.n, block = blockIdx.x, blocks = gridDim.x;
  uint32_t* prefix = reinterpret_cast<uint32_t*>(smem);                       // [n + 1] tiles before a sequence, of all its jobs
  float* ml = reinterpret_cast<float*>(smem + F::prefix_bytes(n));            // [warps][16] (maximum, sum)
  unsigned char* q_sm = reinterpret_cast<unsigned char*>(ml) + F::ML;         // [parts][16] rows
  float* slab = reinterpret_cast<float*>(q_sm);                               // [warps][16][SLAB_PITCH]
  unsigned char* stages = q_sm + F::q_bytes(QP) + warp * a.stages * F::STAGE;

  // ---- the tile list: a prefix sum over the sequences; rows of sequences without positions are zero
  {
    const uint32_t each = (n + F::THREADS - 1) / F::THREADS, first = tid * each;
    uint32_t sum = 0;
    for (uint32_t s = first; s < first + each && s < n; ++s) {
      uint32_t lo, count;
      span_of(g, s, &lo, &count);
      prefix[s] = sum;
      sum += (count + F::TILE - 1) / F::TILE * a.jobs;
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
  const uint32_t total = prefix[n];
  if (block == 0)
    for (uint32_t s = tid; s <= n; s += F::THREADS) a.prefix[s] = prefix[s];
  const uint32_t out_cols = cache.heads * D;
  for (uint32_t s = block; s < n; s += blocks)
    if (prefix[s] == prefix[s + 1])
      for (uint32_t j = tid; j < out_cols; j += F::THREADS) store_float(g.out, (uint64_t)s * out_cols + j, g.out_bf16, 0.f);
  const uint32_t start = run_start(total, block, blocks), stop = run_start(total, block + 1, blocks);
  if (start >= stop) return;             // the same for every thread

  const auto enter = [&](Cursor& c) {    // the bounds of sequence c.s
    uint32_t count;
    span_of(g, c.s, &c.lo, &count);
    c.end = c.lo + count;
    c.tiles = (count + F::TILE - 1) / F::TILE;
  };
  const auto seek = [&](Cursor& c, uint32_t tile) {
    uint32_t lo = 0, hi = n - 1;         // the last sequence that starts at or before the tile: it has tiles
    while (lo < hi) {
      const uint32_t mid = (lo + hi + 1) / 2;
      if (prefix[mid] <= tile) lo = mid; else hi = mid - 1;
    }
    c.s = lo;
    enter(c);
    c.job = (tile - prefix[lo]) / c.tiles;
    c.tile = (tile - prefix[lo]) % c.tiles;
  };
  const auto next_job = [&](Cursor& c) {
    c.tile = 0;
    if (++c.job == a.jobs) {
      c.job = 0;
      do ++c.s; while (c.s < n && prefix[c.s] == prefix[c.s + 1]);
      if (c.s < n) enter(c);
    }
  };

  // ---- the copies' side of the pipeline: rows of the tile that is issued next
  Cursor ahead;
  seek(ahead, start);
  uint32_t to_issue = stop - start;
  int32_t row = -1;                      // lane % 16's pool row of the tile at `ahead`, -1: not attended
  const auto look_up = [&]() {
    row = -1;
    const uint32_t p = ahead.lo + ahead.tile * F::TILE + warp * 16 + (lane & 15);
    if (to_issue && p < ahead.end) {
      const uint32_t at = (uint32_t)(((uint64_t)p * a.page_magic) >> (32 + a.page_shift));
      const int32_t page = cache.table[(uint64_t)ahead.s * cache.width + at];
      if (page >= 0 && (uint32_t)page < cache.pages) row = page * (int32_t)cache.page + (int32_t)(p - at * cache.page);
      else set_domain(g.err);
    }
  };
  look_up();
  const uint32_t ld = cache.kv_heads * D * (uint32_t)sizeof(KV);           // bytes of a pool row
  uint32_t head_at = ahead.job / a.row_tiles * D * (uint32_t)sizeof(KV);   // of the head of the tile at `ahead`
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(stages) + (lane % F::LANES) * 16;
  int issue_stage = 0;
  const auto issue = [&]() {
    if (to_issue) {
      const uint32_t there = __ballot_sync(0xffffffffu, row >= 0);
      if (lane == 0) valid[warp][issue_stage] = there & 0xffffu;
      const uint32_t at = to + issue_stage * F::STAGE;
#pragma unroll
      for (int i = 0; i < F::REST; ++i) {
        const int r = i * F::ROWS + lane / F::LANES;
        const int32_t from = __shfl_sync(0xffffffffu, row, r);
        const bool on = from >= 0;
        const uint64_t off = (uint64_t)(uint32_t)(on ? from : 0) * ld + head_at + (lane % F::LANES) * 16;
        const char *k = (const char*)cache.keys + off, *v = (const char*)cache.values + off;
#pragma unroll
        for (int c = 0; c < F::PIECES; ++c) {
          cp_async16(at + r * F::K_PITCH + c * F::LANES * 16, k + c * F::LANES * 16, on);
          cp_async16(at + 16 * F::K_PITCH + r * F::V_PITCH + c * F::LANES * 16, v + c * F::LANES * 16, on);
        }
      }
      --to_issue;
      if (++ahead.tile == ahead.tiles) {
        next_job(ahead);
        head_at = ahead.job / a.row_tiles * D * (uint32_t)sizeof(KV);
      }
      look_up();
    }
    cp_async_commit();
    if (++issue_stage == a.stages) issue_stage = 0;
  };
  for (int i = 0; i + 1 < a.stages; ++i) issue();

  // ---- the block's (sequence, head) pieces, one after another
  Cursor here;
  seek(here, start);
  const int gr = lane >> 2, t4 = lane & 3;
  int stage = 0, piece_i = 0;
  for (uint32_t left = stop - start; left > 0; ++piece_i) {
    const uint32_t steps = left < here.tiles - here.tile ? left : here.tiles - here.tile;
    const bool whole = here.tile == 0 && steps == here.tiles;
    const uint32_t kvh = here.job / a.row_tiles, r0 = (here.job % a.row_tiles) * 16;
    const uint32_t rows = a.group - r0 < 16 ? a.group - r0 : 16;             // query heads of this tile
    const uint32_t head0 = kvh * a.group + r0;

    // the queries, in the parts the products take; rows without a head are zero
    __syncthreads();                     // the last piece's readers are done
    for (int i = tid; i < 16 * D; i += F::THREADS) {
      const int r = i / D, e = i % D;
      const float q = r < (int)rows ? load_float(g.q.p, (uint64_t)here.s * g.q.ld + (uint64_t)(head0 + r) * D + e, g.q.bf16) : 0.f;
      if constexpr (F::BF) {
        float rest = q;
        for (int p = 0; p < QP; ++p) {
          // all parts but the last are cut, so that each leaves fewer bits of the same sign; the last is rounded
          uint32_t bits = __float_as_uint(rest);
          if (p + 1 == QP) bits = (uint32_t)f32_to_bf16_bits(bits) << 16;
          else if (rest != rest) bits = 0x7fc00000u;
          else bits &= 0xffff0000u;
          *reinterpret_cast<uint16_t*>(q_sm + (p * 16 + r) * F::Q_PITCH + e * 2) = (uint16_t)(bits >> 16);
          const float part = __uint_as_float(bits);
          rest = fabsf(part) <= FLT_MAX ? rest - part : 0.f;
        }
      } else {
        const float hi = __uint_as_float(tf32_of(q));
        *reinterpret_cast<float*>(q_sm + r * F::Q_PITCH + e * 4) = hi;
        *reinterpret_cast<float*>(q_sm + (16 + r) * F::Q_PITCH + e * 4) = fabsf(hi) <= FLT_MAX ? q - hi : 0.f;
      }
    }
    __syncthreads();

    uint32_t qf[Q_HELD ? QP : 1][Q_HELD ? D / 16 : 1][4];
    if constexpr (Q_HELD) {
      const uint32_t qa = (uint32_t)__cvta_generic_to_shared(q_sm) + ((lane & 7) + ((lane >> 3) & 1) * 8) * F::Q_PITCH + (lane >> 4) * 16;
#pragma unroll
      for (int p = 0; p < QP; ++p)
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) ldmatrix4(qf[p][kk], qa + p * 16 * F::Q_PITCH + kk * 32);
    }
    float o[D / 8][4];
#pragma unroll
    for (int j = 0; j < D / 8; ++j) o[j][0] = o[j][1] = o[j][2] = o[j][3] = 0.f;
    float m0 = -FLT_MAX, m1 = -FLT_MAX, l0 = 0.f, l1 = 0.f;      // rows gr and gr + 8; the sums are this lane's own
    for (uint32_t step = 0; step < steps; ++step) {
      cp_async_wait(a.stages - 2);
      __syncwarp();                      // every lane's copies of this stage are in, and every lane is done with the stage before
      issue();
      const unsigned char* st = stages + stage * F::STAGE;
      const uint32_t live = valid[warp][stage];
      if (++stage == a.stages) stage = 0;
      const uint32_t k_at = (uint32_t)__cvta_generic_to_shared(st), v_at = k_at + 16 * F::K_PITCH;
      const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(q_sm);

      // scores of 16 heads x 16 positions: lane holds rows gr, gr + 8 and positions 8 nt + 2 t4 + {0, 1}
      float sc[2][4];
#pragma unroll
      for (int nt = 0; nt < 2; ++nt) sc[nt][0] = sc[nt][1] = sc[nt][2] = sc[nt][3] = 0.f;
      if constexpr (F::BF) {
        const uint32_t kb = k_at + ((lane & 7) + ((lane >> 4) & 1) * 8) * F::K_PITCH + ((lane >> 3) & 1) * 16;
        const uint32_t qa = q_at + ((lane & 7) + ((lane >> 3) & 1) * 8) * F::Q_PITCH + (lane >> 4) * 16;
        float odd_k[2][4];               // two chains of products a score: each waits for the one before it
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) odd_k[nt][0] = odd_k[nt][1] = odd_k[nt][2] = odd_k[nt][3] = 0.f;
#pragma unroll
        for (int kk = 0; kk < D / 16; ++kk) {
          uint32_t b[4];
          ldmatrix4(b, kb + kk * 32);
          auto& to_sum = kk & 1 ? odd_k : sc;
#pragma unroll
          for (int p = 0; p < QP; ++p) {
            if constexpr (Q_HELD) {
              mma_bf16(to_sum[0], qf[p][kk], b[0], b[1]);
              mma_bf16(to_sum[1], qf[p][kk], b[2], b[3]);
            } else {
              uint32_t x[4];
              ldmatrix4(x, qa + p * 16 * F::Q_PITCH + kk * 32);
              mma_bf16(to_sum[0], x, b[0], b[1]);
              mma_bf16(to_sum[1], x, b[2], b[3]);
            }
          }
        }
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e) sc[nt][e] += odd_k[nt][e];
      } else {
        // the products' inner index in the order 0, 2, 4, 6, 1, 3, 5, 7 of each eight columns, for both operands
        const float* qh = reinterpret_cast<const float*>(q_sm + gr * F::Q_PITCH) + 2 * t4;
        constexpr int ROW8 = 8 * F::Q_PITCH / 4, LOW = 16 * F::Q_PITCH / 4;
#pragma unroll 4
        for (int kk = 0; kk < D / 8; ++kk) {
          const float2 h0 = *reinterpret_cast<const float2*>(qh + kk * 8), h1 = *reinterpret_cast<const float2*>(qh + ROW8 + kk * 8);
          const float2 w0 = *reinterpret_cast<const float2*>(qh + LOW + kk * 8), w1 = *reinterpret_cast<const float2*>(qh + LOW + ROW8 + kk * 8);
          const uint32_t hi[4] = {__float_as_uint(h0.x), __float_as_uint(h1.x), __float_as_uint(h0.y), __float_as_uint(h1.y)};
          const uint32_t lo[4] = {__float_as_uint(w0.x), __float_as_uint(w1.x), __float_as_uint(w0.y), __float_as_uint(w1.y)};
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const float2 k = *reinterpret_cast<const float2*>(st + (nt * 8 + gr) * F::K_PITCH + (kk * 8 + 2 * t4) * 4);
            const uint32_t b0 = tf32_of(k.x), b1 = tf32_of(k.y);
            mma_tf32(sc[nt], lo, b0, b1);
            mma_tf32(sc[nt], hi, __float_as_uint(k.x - __uint_as_float(b0)), __float_as_uint(k.y - __uint_as_float(b1)));
            mma_tf32(sc[nt], hi, b0, b1);
          }
        }
      }
      // An infinite key gives 0 * inf among the parts' products: such a score is taken again from whole operands.
      bool odd = false;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 4; ++e) odd |= sc[nt][e] != sc[nt][e];
      if (__any_sync(0xffffffffu, odd)) {
#pragma unroll
        for (int nt = 0; nt < 2; ++nt)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (sc[nt][e] != sc[nt][e]) {
              const int r = gr + (e >> 1) * 8, j = nt * 8 + 2 * t4 + (e & 1);
              float t = 0.f;
              for (int c = 0; c < D; ++c) {
                float q = 0.f;
                for (int p = 0; p < QP; ++p)
                  q += F::BF ? bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(q_sm + (p * 16 + r) * F::Q_PITCH + c * 2))
                             : *reinterpret_cast<const float*>(q_sm + (p * 16 + r) * F::Q_PITCH + c * 4);
                t = fmaf(q, F::BF ? bf16_bits_to_f32(*reinterpret_cast<const uint16_t*>(st + j * F::K_PITCH + c * 2))
                                  : *reinterpret_cast<const float*>(st + j * F::K_PITCH + c * 4), t);
              }
              sc[nt][e] = t;
            }
      }

      // running softmax: new maximum, the factor of what was summed before, the weights
      float x0 = -FLT_MAX, x1 = -FLT_MAX;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const bool on = (live >> (nt * 8 + 2 * t4 + e)) & 1;
          sc[nt][e] = on ? sc[nt][e] * a.scale_log2 : -INFINITY;
          sc[nt][2 + e] = on ? sc[nt][2 + e] * a.scale_log2 : -INFINITY;
          x0 = fmaxf(x0, sc[nt][e]);
          x1 = fmaxf(x1, sc[nt][2 + e]);
        }
      x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 1)); x0 = fmaxf(x0, __shfl_xor_sync(0xffffffffu, x0, 2));
      x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 1)); x1 = fmaxf(x1, __shfl_xor_sync(0xffffffffu, x1, 2));
      x0 = fmaxf(x0, m0); x1 = fmaxf(x1, m1);
      const float f0 = exp2_fast(m0 - x0), f1 = exp2_fast(m1 - x1);
      m0 = x0; m1 = x1;
#pragma unroll
      for (int nt = 0; nt < 2; ++nt)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          sc[nt][e] = exp2_fast(sc[nt][e] - m0);
          sc[nt][2 + e] = exp2_fast(sc[nt][2 + e] - m1);
        }
      l0 = l0 * f0 + ((sc[0][0] + sc[0][1]) + (sc[1][0] + sc[1][1]));
      l1 = l1 * f1 + ((sc[0][2] + sc[0][3]) + (sc[1][2] + sc[1][3]));

      // rows = rows * factor + weights x values
      if constexpr (F::BF) {
        uint32_t w[3][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {          // (row gr, first eight), (gr + 8, first), (gr, second), (gr + 8, second)
          float u = sc[i >> 1][(i & 1) * 2], v = sc[i >> 1][(i & 1) * 2 + 1];
          w[0][i] = bf16x2(u, v);
          u -= low_of(w[0][i]); v -= high_of(w[0][i]);
          w[1][i] = bf16x2(u, v);
          if constexpr (EXACT) w[2][i] = bf16x2(u - low_of(w[1][i]), v - high_of(w[1][i]));
        }
        if constexpr (!EXACT)
          if (__any_sync(0xffffffffu, f0 != 1.f || f1 != 1.f)) {
#pragma unroll
            for (int j = 0; j < D / 8; ++j) { o[j][0] *= f0; o[j][1] *= f0; o[j][2] *= f1; o[j][3] *= f1; }
          }
        const uint32_t vb = v_at + ((lane & 7) + ((lane >> 3) & 1) * 8) * F::V_PITCH + (lane >> 4) * 16;
#pragma unroll
        for (int j = 0; j < D / 16; ++j) {
          uint32_t b[4];
          ldmatrix4_t(b, vb + j * 32);
#pragma unroll
          for (int hf = 0; hf < 2; ++hf) {
            float* r = o[2 * j + hf];
            if constexpr (EXACT) {
              float c[4] = {0.f, 0.f, 0.f, 0.f};
              mma_bf16(c, w[2], b[2 * hf], b[2 * hf + 1]);
              mma_bf16(c, w[1], b[2 * hf], b[2 * hf + 1]);
              mma_bf16(c, w[0], b[2 * hf], b[2 * hf + 1]);
              r[0] = fmaf(r[0], f0, c[0]); r[1] = fmaf(r[1], f0, c[1]);
              r[2] = fmaf(r[2], f1, c[2]); r[3] = fmaf(r[3], f1, c[3]);
            } else {
              mma_bf16(r, w[1], b[2 * hf], b[2 * hf + 1]);
              mma_bf16(r, w[0], b[2 * hf], b[2 * hf + 1]);
            }
          }
        }
      } else {
        uint32_t hi[2][4], lo[2][4];
#pragma unroll
        for (int nt = 0; nt < 2; ++nt) {
          const float v[4] = {sc[nt][0], sc[nt][2], sc[nt][1], sc[nt][3]};   // (gr, even), (gr + 8, even), (gr, odd), (gr + 8, odd)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            hi[nt][i] = tf32_of(v[i]);
            lo[nt][i] = __float_as_uint(v[i] - __uint_as_float(hi[nt][i]));
          }
        }
        const unsigned char* vs = st + 16 * F::K_PITCH + 2 * t4 * F::V_PITCH + gr * 4;
#pragma unroll
        for (int j = 0; j < D / 8; ++j) {
          float c[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int nt = 0; nt < 2; ++nt) {
            const float u = *reinterpret_cast<const float*>(vs + nt * 8 * F::V_PITCH + j * 32);
            const float v = *reinterpret_cast<const float*>(vs + (nt * 8 + 1) * F::V_PITCH + j * 32);
            const uint32_t b0 = tf32_of(u), b1 = tf32_of(v);
            mma_tf32(c, lo[nt], b0, b1);
            mma_tf32(c, hi[nt], __float_as_uint(u - __uint_as_float(b0)), __float_as_uint(v - __uint_as_float(b1)));
            mma_tf32(c, hi[nt], b0, b1);
          }
          float* r = o[j];
          r[0] = fmaf(r[0], f0, c[0]); r[1] = fmaf(r[1], f0, c[1]);
          r[2] = fmaf(r[2], f1, c[2]); r[3] = fmaf(r[3], f1, c[3]);
        }
      }
    }

    // ---- the warps' (maximum, sum, rows) into one, SLAB columns at a time
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    if (t4 == 0) {
      ml[(warp * 16 + gr) * 2] = m0; ml[(warp * 16 + gr) * 2 + 1] = l0;
      ml[(warp * 16 + gr + 8) * 2] = m1; ml[(warp * 16 + gr + 8) * 2 + 1] = l1;
    }
    __syncthreads();
    {
      float t0 = -FLT_MAX, t1 = -FLT_MAX;
      for (int w = 0; w < F::WARPS; ++w) { t0 = fmaxf(t0, ml[(w * 16 + gr) * 2]); t1 = fmaxf(t1, ml[(w * 16 + gr + 8) * 2]); }
      m0 = exp2_fast(m0 - t0); m1 = exp2_fast(m1 - t1);                        // this warp's factors from here on
    }
    float* part = a.part + ((uint64_t)block * 2 + (piece_i ? 1 : 0)) * 16 * (D + 2);
#pragma unroll
    for (int at = 0; at < D; at += F::SLAB) {
      if (at) __syncthreads();
#pragma unroll
      for (int j = 0; j < F::SLAB / 8; ++j) {
        const float* r = o[at / 8 + j];
        float* to = slab + (warp * 16 + gr) * F::SLAB_PITCH + j * 8 + 2 * t4;
        *reinterpret_cast<float2*>(to) = make_float2(r[0] * m0, r[1] * m0);
        *reinterpret_cast<float2*>(to + 8 * F::SLAB_PITCH) = make_float2(r[2] * m1, r[3] * m1);
      }
      __syncthreads();
      for (int i = tid; i < (int)rows * F::SLAB; i += F::THREADS) {
        const int r = i / F::SLAB, c = i % F::SLAB;
        float v = 0.f;
        for (int w = 0; w < F::WARPS; ++w) v += slab[(w * 16 + r) * F::SLAB_PITCH + c];
        if (whole) {
          float top = -FLT_MAX, den = 0.f;
          for (int w = 0; w < F::WARPS; ++w) top = fmaxf(top, ml[(w * 16 + r) * 2]);
          for (int w = 0; w < F::WARPS; ++w) den += ml[(w * 16 + r) * 2 + 1] * exp2_fast(ml[(w * 16 + r) * 2] - top);
          store_float(g.out, (uint64_t)here.s * out_cols + (uint64_t)(head0 + r) * D + at + c, g.out_bf16, v / (den < FLT_MIN ? FLT_MIN : den));
        } else {
          part[r * D + at + c] = v;
        }
      }
    }
    if (!whole && tid < 16) {
      float top = -FLT_MAX, den = 0.f;
      for (int w = 0; w < F::WARPS; ++w) top = fmaxf(top, ml[(w * 16 + tid) * 2]);
      for (int w = 0; w < F::WARPS; ++w) den += ml[(w * 16 + tid) * 2 + 1] * exp2_fast(ml[(w * 16 + tid) * 2] - top);
      part[16 * D + tid * 2] = top;
      part[16 * D + tid * 2 + 1] = den;
    }
    left -= steps;
    here.tile += steps;
    if (here.tile == here.tiles) next_job(here);
  }
  cp_async_wait(0);
}

// Joins a (sequence, head) whose tiles lie in several blocks' runs: block (c, r) is query row r of the piece that ends block
// c's run, if c is the first of its blocks.  rows = sum over the blocks, in their order, of rows_c 2^(m_c - m) / sum l_c 2^(m_c - m).
template <int D>
__global__ void __launch_bounds__(256) attention_pages_join_kernel(const __grid_constant__ AttnPlan a, uint32_t blocks) {
  constexpr int LANES = D / 4, TEAMS = 256 / LANES;          // a team a block's row, a float4 a lane
  __shared__ __align__(16) float sums[TEAMS][D];
  __shared__ float red[256 / 32], dens[TEAMS];
  pdl_enter();
  const AttnPagesArgs& g = a.g;
  const int tid = threadIdx.x;
  const uint32_t c0 = blockIdx.x, r = blockIdx.y, n = (uint32_t)g.n;
  const uint32_t total = a.prefix[n];
  const uint32_t next = run_start(total, c0 + 1, blocks), mine = run_start(total, c0, blocks);
  if (mine >= next || next >= total) return;                 // an empty run, or nothing goes on behind it
  uint32_t s = 0, hi = n - 1;
  while (s < hi) {
    const uint32_t mid = (s + hi + 1) / 2;
    if (a.prefix[mid] <= next) s = mid; else hi = mid - 1;
  }
  const uint32_t tiles = (a.prefix[s + 1] - a.prefix[s]) / a.jobs, job = (next - a.prefix[s]) / tiles;
  const uint32_t first = a.prefix[s] + job * tiles, last = first + tiles - 1;
  if (first == next || first < mine) return;                 // the piece starts behind the run, or before it: another block's
  const uint32_t kvh = job / a.row_tiles, r0 = job % a.row_tiles * 16;
  if (r >= a.group - r0) return;
  const uint32_t c1 = run_owner(total, last, blocks);
  const auto piece = [&](uint32_t c) { return a.part + ((uint64_t)c * 2 + (c == c0 && first != mine ? 1 : 0)) * 16 * (D + 2); };
  // an empty run lies between two others only where there are fewer tiles than blocks: it holds nothing of the piece
  const auto there = [&](uint32_t c) { return run_start(total, c, blocks) < run_start(total, c + 1, blocks); };
  float top = -FLT_MAX;
  for (uint32_t c = c0 + tid; c <= c1; c += 256)
    if (there(c)) top = fmaxf(top, piece(c)[16 * D + r * 2]);
#pragma unroll
  for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
  if ((tid & 31) == 0) red[tid >> 5] = top;
  __syncthreads();
  for (int w = 0; w < 8; ++w) top = fmaxf(top, red[w]);
  const int team = tid / LANES, lane = tid % LANES;
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  float den = 0.f;
  if (team < TEAMS)
    for (uint32_t c = c0 + team; c <= c1; c += TEAMS)
      if (there(c)) {
        const float* p = piece(c);
        const float f = exp2_fast(p[16 * D + r * 2] - top);
        const float4 x = *reinterpret_cast<const float4*>(p + r * D + lane * 4);
        den = fmaf(p[16 * D + r * 2 + 1], f, den);
        v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
      }
  if (team < TEAMS) {
    *reinterpret_cast<float4*>(&sums[team][lane * 4]) = v;
    if (lane == 0) dens[team] = den;
  }
  __syncthreads();
  if (tid < D) {
    float t = 0.f, l = 0.f;
    for (int w = 0; w < TEAMS; ++w) { t += sums[w][tid]; l += dens[w]; }
    const uint32_t head = kvh * a.group + r0 + r;
    store_float(g.out, (uint64_t)s * a.g.cache.heads * D + (uint64_t)head * D + tid, g.out_bf16, t / (l < FLT_MIN ? FLT_MIN : l));
  }
}

// The tiles a sequence can have at most, from the shapes alone.
uint64_t attention_tiles(const AttnPagesArgs& g, int tile) {
  uint64_t p = (uint64_t)g.cache.width * g.cache.page;
  if (g.window && p > g.window) p = g.window;
  return (p + tile - 1) / tile;
}
struct AttnScratch { float* part; uint32_t* prefix; };

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

template <typename KV, int D, int QP, bool EXACT>
cudaError_t attention_form(const AttnPagesArgs& g, int sms, const AttnScratch& scratch, int* launches, cudaStream_t stream) {
  using F = Form<KV, D>;
  AttnPlan a;
  a.g = g;
  a.page_shift = 31 - __builtin_clz(g.cache.page);
  a.page_magic = (1ull << (32 + a.page_shift)) / g.cache.page + 1;
  a.group = g.cache.heads / g.cache.kv_heads;
  a.row_tiles = (a.group + 15) / 16;
  a.jobs = g.cache.kv_heads * a.row_tiles;
  a.scale_log2 = g.scale * 1.44269504088896340736f;
  a.part = scratch.part; a.prefix = scratch.prefix;
  const int limit = 228 * 1024 / F::BLOCKS - 1024 - 256;   // a block's share of an SM's shared memory, less what the launch and the statics take
  const uint64_t per_sequence = attention_tiles(g, F::TILE) * a.jobs;
  if (per_sequence > 0xffffffffull) return cudaErrorNotSupported;
  cudaError_t e = ensure_dynamic_smem((const void*)attention_pages_kernel<KV, D, QP, EXACT>, limit);
  if (e != cudaSuccess) return e;
  for (uint64_t at = 0; at < g.n;) {
    uint64_t rows = g.n - at < MAX_SEQUENCES ? g.n - at : MAX_SEQUENCES;
    if (per_sequence && rows > 0xffffffffull / per_sequence) rows = 0xffffffffull / per_sequence;
    a.g.n = rows;
    a.g.cache.table = g.cache.table + at * g.cache.width;
    a.g.positions = g.positions + at;
    a.g.q.p = (const char*)g.q.p + at * g.q.ld * (g.q.bf16 ? 2 : 4);
    a.g.out = (char*)g.out + at * g.cache.heads * D * (g.out_bf16 ? 2 : 4);
    const int fixed = F::prefix_bytes((uint32_t)rows) + F::ML + F::q_bytes(QP);
    a.stages = (limit - fixed) / (F::WARPS * F::STAGE);
    if (a.stages > MAX_STAGES) a.stages = MAX_STAGES;
    if (a.stages < 2) return cudaErrorNotSupported;
    uint64_t blocks = (uint64_t)F::BLOCKS * sms;
    if (blocks > rows * per_sequence) blocks = rows * per_sequence;   // no more than the tiles there can be
    if (blocks < 1) blocks = 1;
    launch_pdl(attention_pages_kernel<KV, D, QP, EXACT>, dim3((unsigned)blocks), dim3(F::THREADS), fixed + a.stages * F::WARPS * F::STAGE, stream, a);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    ++*launches;
    if (blocks > 1 && per_sequence > a.jobs) {               // a (sequence, head) of one tile is never divided
      launch_pdl(attention_pages_join_kernel<D>, dim3((unsigned)blocks, a.group < 16 ? a.group : 16), dim3(256), 0, stream, a, (uint32_t)blocks);
      e = cudaGetLastError();
      if (e != cudaSuccess) return e;
      ++*launches;
    }
    at += rows;
  }
  return cudaSuccess;
}

// The form for the types: an operand's parts as the precision note says.
template <int D>
cudaError_t attention_dim(const AttnPagesArgs& g, int sms, const AttnScratch& s, int* launches, cudaStream_t stream) {
  if (!g.cache.bf16) return attention_form<float, D, 2, true>(g, sms, s, launches, stream);
  if (g.q.bf16) return g.out_bf16 ? attention_form<uint16_t, D, 1, false>(g, sms, s, launches, stream)
                                  : attention_form<uint16_t, D, 1, true>(g, sms, s, launches, stream);
  return g.out_bf16 ? attention_form<uint16_t, D, 2, false>(g, sms, s, launches, stream)
                    : attention_form<uint16_t, D, 3, true>(g, sms, s, launches, stream);
}

}  // namespace

bool attention_pages_dim_ok(uint32_t d) { return d == 32 || d == 64 || d == 96 || d == 128 || d == 192 || d == 256; }

// Two pieces for every block that may be launched (at most four an SM), and the prefix sums.
size_t attention_pages_scratch_bytes(uint32_t dim) {
  return (size_t)4 * sm_count() * 2 * 16 * (dim + 2) * sizeof(float) + (MAX_SEQUENCES + 1) * sizeof(uint32_t);
}

cudaError_t launch_attention_pages(const AttnPagesArgs& g, void* scratch, int* launches, cudaStream_t stream) {
  *launches = 0;
  if (g.n == 0) return cudaSuccess;
  const int sms = sm_count();
  AttnScratch s;
  s.part = (float*)scratch;
  s.prefix = (uint32_t*)(s.part + (size_t)4 * sms * 2 * 16 * (g.cache.dim + 2));
#define GO(D) case D: return attention_dim<D>(g, sms, s, launches, stream)
  switch (g.cache.dim) {
    GO(32); GO(64); GO(96); GO(128); GO(192); GO(256);
    default: return cudaErrorNotSupported;
  }
#undef GO
}

}  // namespace b200
