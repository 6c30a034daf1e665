// The engine's state, shared by the translation units that hold its entry points (engine.cu: the trait's
// methods; engine_serving.cu: the paged cache and the token log probabilities): the buffer table, the
// device-memory pool, the trace being captured and the error word, and the argument checks both use.
#pragma once
#include <cuda_runtime.h>
#include <stdarg.h>
#include <stdio.h>
#include <string.h>

#include <algorithm>
#include <map>
#include <string>
#include <unordered_map>
#include <unordered_set>
#include <vector>

#include "../../include/b200tt.h"
#include "kernels.h"

namespace b200 {

struct Buf {
  void* ptr = nullptr;
  uint64_t rows = 0, cols = 0;
  int elem = B200_F32;
  uint64_t bytes = 0;       // bytes of the pool block (0 for views / adopted memory)
  b200_buffer parent = 0;   // view of another buffer
  int views = 0;            // live views of this buffer
  bool freed = false;       // free() called while views are alive
  bool adopted = false;
};

inline uint64_t elem_bytes(int elem) { return elem == B200_BF16 ? 2 : 4; }
// Bytes a [rows, cols] buffer of `elem` holds: a BFP8 matrix is a datum byte an element and an exponent byte
// for every sixteen of a row (csrc/k_bfp.cu).
inline uint64_t buffer_bytes(uint64_t rows, uint64_t cols, int elem) {
  return elem == B200_BFP8 ? rows * cols + rows * cols / 16 : rows * cols * elem_bytes(elem);
}

}  // namespace b200

using b200::Buf;
using b200::buffer_bytes;
using b200::elem_bytes;

struct b200_engine {
  int device = 0;
  b200_config cfg{};
  cudaStream_t stream = nullptr;
  cudaEvent_t t0 = nullptr, t1 = nullptr;
  int* d_err = nullptr;
  long long wait_limit_word = 0;   // host copy of the limit kept behind the device error word
  cudaStream_t h2d_stream = nullptr, d2h_stream = nullptr;   // b200_matmul_host_bf16's copy streams
  int matmul_sm_limit = 0;   // b200_set_matmul_sm_limit
  int* h_err = nullptr;  // pinned
  std::string last_error;
  uint64_t oom[3] = {0, 0, 0};
  int sticky = 0;  // first asynchronous failure, reported at every later wait
  std::string sticky_text;
  std::string label;
  const char* matmul_path = "none";
  const char* decode_form = "none";
  b200_traffic traffic{};
  uint64_t next_id = 1;
  uint64_t alloc_calls = 0;
  std::unordered_map<b200_buffer, Buf> bufs;
  std::multimap<uint64_t, void*> cache;  // free blocks by size
  float* full_scratch = nullptr;
  // Traces (CUDA graphs): the counterpart of the reference's begin_trace / end_trace / run_trace
  // (crates/burn-tt/src/server.rs:591-660).  While one is captured, every block the ops take is
  // owned by the trace: a replay writes the same addresses, so they must not go back to the pool
  // before the trace is released.
  struct Trace {
    cudaGraph_t graph = nullptr;
    cudaGraphExec_t exec = nullptr;
    std::vector<std::pair<void*, uint64_t>> blocks;   // every block the capture took
    std::vector<void*> pinned;                        // host copies of block lists the graph re-uploads
    uint64_t launches = 0;
    std::vector<std::pair<std::string, uint64_t>> ops;   // the captured ops in order: (label, kernels)
  };
  bool capturing = false;
  Trace cur;                                          // the trace being captured
  std::multimap<uint64_t, void*> cur_free;            // its blocks free for reuse inside the capture
  std::unordered_map<void*, uint64_t> cur_owned;      // ptr -> size of blocks the capture owns
  std::unordered_map<uint64_t, Trace> traces;
  uint64_t next_trace = 1;
  // Per-op device time (the profile mode, crates/burn-tt/src/profile.rs:1-48): while it is on, every
  // `set_op_label` records an event on the stream, so the device time between two labels is charged to the
  // first one -- the server labels each job before it runs it (server.rs:2370 `timed_job`).
  struct Mark { std::string label; cudaEvent_t at = nullptr; uint64_t launches = 0; };
  bool profiling = false;
  std::vector<Mark> marks;                 // marks[i] opens op i; the next mark (or `prof_end`) closes it
  cudaEvent_t prof_end = nullptr;
  struct Stat { uint64_t calls = 0, launches = 0; double ms = 0; };
  std::vector<std::pair<std::string, Stat>> prof_table;   // in order of first appearance
  void drop_marks() {
    for (auto& m : marks) if (m.at) cudaEventDestroy(m.at);
    marks.clear();
    if (prof_end) { cudaEventDestroy(prof_end); prof_end = nullptr; }
  }

  int fail(int code, const char* fmt, ...) {
    char tmp[512];
    va_list ap;
    va_start(ap, fmt);
    vsnprintf(tmp, sizeof tmp, fmt, ap);
    va_end(ap);
    last_error = label.empty() ? std::string(tmp) : (label + ": " + tmp);
    return code;
  }
  int cuda_fail(cudaError_t e, const char* what) {
    return fail(B200_DEVICE, "%s: %s", what, cudaGetErrorString(e));
  }

  // ---- pool ---------------------------------------------------------------------
  static uint64_t round_size(uint64_t n) {
    if (n == 0) n = 1;
    if (n <= 4096) return (n + 255) & ~255ull;
    if (n <= (1ull << 20)) {
      uint64_t p = 4096;
      while (p < n) p <<= 1;
      return p;
    }
    return (n + (2ull << 20) - 1) & ~((2ull << 20) - 1);
  }
  void release_cache() {
    for (auto& kv : cache) {
      cudaFree(kv.second);
      traffic.pool_reserved -= kv.first;
    }
    cache.clear();
  }
  int alloc(uint64_t bytes, void** out, uint64_t* got) {
    ++alloc_calls;
    const uint64_t sz = round_size(bytes);
    if (cfg.fail_alloc_at > 0 && alloc_calls == (uint64_t)cfg.fail_alloc_at) {
      oom[0] = sz; oom[1] = 0; oom[2] = 0;
      return fail(B200_OUT_OF_MEMORY, "out of device memory: need %llu bytes (injected)", (unsigned long long)sz);
    }
    if (capturing) {
      auto ft = cur_free.lower_bound(sz);
      if (ft != cur_free.end() && ft->first <= sz + sz / 4) {
        *out = ft->second; *got = ft->first;
        cur_free.erase(ft);
        traffic.pool_in_use += *got;
        traffic.pool_high_water = std::max(traffic.pool_high_water, traffic.pool_in_use);
        return B200_OK;
      }
    }
    auto it = cache.lower_bound(sz);
    if (it != cache.end() && it->first <= sz + sz / 4) {
      *out = it->second;
      *got = it->first;
      cache.erase(it);
    } else {
      if (cfg.pool_limit_bytes && traffic.pool_reserved + sz > cfg.pool_limit_bytes) release_cache();
      if (cfg.pool_limit_bytes && traffic.pool_reserved + sz > cfg.pool_limit_bytes) {
        oom[0] = sz; oom[1] = cfg.pool_limit_bytes - traffic.pool_reserved; oom[2] = oom[1];
        return fail(B200_OUT_OF_MEMORY, "out of device memory: need %llu bytes, pool limit leaves %llu",
                    (unsigned long long)sz, (unsigned long long)oom[1]);
      }
      void* p = nullptr;
      cudaError_t e = cudaMalloc(&p, sz);
      if (e != cudaSuccess && !capturing) {   // a synchronise would invalidate an open capture: fail at once there
        cudaGetLastError();
        cudaStreamSynchronize(stream);
        release_cache();
        e = cudaMalloc(&p, sz);
      }
      if (e != cudaSuccess) {
        cudaGetLastError();
        size_t fr = 0, tot = 0;
        cudaMemGetInfo(&fr, &tot);
        oom[0] = sz; oom[1] = fr; oom[2] = fr;
        return fail(B200_OUT_OF_MEMORY, "out of device memory: need %llu bytes, %llu free",
                    (unsigned long long)sz, (unsigned long long)fr);
      }
      *out = p;
      *got = sz;
      traffic.pool_reserved += sz;
    }
    traffic.pool_in_use += *got;
    traffic.pool_high_water = std::max(traffic.pool_high_water, traffic.pool_in_use);
    if (capturing) { cur.blocks.emplace_back(*out, *got); cur_owned.emplace(*out, *got); }
    return B200_OK;
  }
  // Whether a block belongs to a trace (captured or being captured): such a block never
  // returns to the pool while its trace lives.
  std::unordered_set<void*> trace_ptrs;   // blocks of finished traces still alive
  bool trace_owned(void* p) const { return cur_owned.count(p) != 0 || trace_ptrs.count(p) != 0; }
  // The block returns to the cache at once: every user of it was enqueued on the one
  // stream before this call, and so is every later user.
  void release(void* p, uint64_t sz) {
    if (sz == 0) return;                 // a kept block list: the engine's, not the pool's
    traffic.pool_in_use -= sz;
    if (capturing && cur_owned.count(p)) { cur_free.emplace(sz, p); return; }
    if (trace_owned(p)) return;   // its trace keeps it
    cache.emplace(sz, p);
  }

  // ---- buffer table ------------------------------------------------------------
  int new_buffer(uint64_t rows, uint64_t cols, int elem, b200_buffer* id, Buf** out) {
    void* p = nullptr;
    uint64_t got = 0;
    const uint64_t bytes = buffer_bytes(rows, cols, elem);
    int st = alloc(bytes, &p, &got);
    if (st) return st;
    Buf b;
    b.ptr = p; b.rows = rows; b.cols = cols; b.elem = elem; b.bytes = got;
    *id = next_id++;
    auto ins = bufs.emplace(*id, b);
    if (out) *out = &ins.first->second;
    return B200_OK;
  }
  Buf* get(b200_buffer id) {
    auto it = bufs.find(id);
    if (it == bufs.end() || it->second.freed) return nullptr;
    return &it->second;
  }
  // A BFP8 buffer is read only by the ops that say so (`packed_ok`): every other op sees plain 16- or 32-bit
  // elements and is refused a packed one here, before it could misread the bytes.
  int need(b200_buffer id, Buf** out, const char* what, bool packed_ok = false) {
    Buf* b = get(id);
    if (!b) return fail(B200_STALE, "%s: buffer %llu is not live on this engine", what, (unsigned long long)id);
    if (b->elem == B200_BFP8 && !packed_ok)
      return fail(B200_UNSUPPORTED, "%s: buffer %llu is BFP8 storage; a product reads it as its B, cast_bfp widens it, nothing else reads it",
                  what, (unsigned long long)id);
    *out = b;
    return B200_OK;
  }
  void drop(b200_buffer id) {
    auto it = bufs.find(id);
    if (it == bufs.end()) return;
    Buf& b = it->second;
    if (b.views > 0) { b.freed = true; return; }
    const b200_buffer parent = b.parent;
    if (!b.parent && !b.adopted && b.ptr) release(b.ptr, b.bytes);
    bufs.erase(it);
    if (parent) {
      auto pit = bufs.find(parent);
      if (pit != bufs.end()) {
        pit->second.views--;
        if (pit->second.views == 0 && pit->second.freed) { pit->second.freed = false; drop(parent); }
      }
    }
  }
  // Host metadata (block lists, index lists) to a temporary device block.
  // Block lists (batched products, moves, attention heads) go to the device before their kernel.
  // A caller issues the same few lists every step, so lists of up to 64 KB are kept on the device
  // by content: a repeat costs no copy (and adds no copy node to a trace).  A kept list is owned by
  // the engine: *got comes back 0 and release() of it does nothing.
  struct MetaEntry { std::vector<uint8_t> bytes; void* dev = nullptr; };
  std::unordered_multimap<uint64_t, MetaEntry> meta_cache;
  uint64_t meta_hits = 0;
  static uint64_t fnv1a(const void* p, uint64_t n) {
    const uint8_t* b = (const uint8_t*)p;
    uint64_t h = 1469598103934665603ull;
    for (uint64_t i = 0; i < n; ++i) { h ^= b[i]; h *= 1099511628211ull; }
    return h;
  }
  int to_device(const void* host, uint64_t bytes, void** dev, uint64_t* got) {
    const bool keepable = bytes > 0 && bytes <= (64u << 10);
    uint64_t key = 0;
    if (keepable) {
      key = fnv1a(host, bytes);
      auto range = meta_cache.equal_range(key);
      for (auto it = range.first; it != range.second; ++it)
        if (it->second.bytes.size() == bytes && memcmp(it->second.bytes.data(), host, bytes) == 0) {
          *dev = it->second.dev; *got = 0; ++meta_hits;
          return B200_OK;
        }
      if (!capturing && meta_cache.size() < 1024) {
        void* p = nullptr;
        if (cudaMalloc(&p, (bytes + 255) & ~255ull) == cudaSuccess) {
          auto it = meta_cache.emplace(key, MetaEntry());
          it->second.bytes.assign((const uint8_t*)host, (const uint8_t*)host + bytes);
          it->second.dev = p;
          cudaError_t e = cudaMemcpyAsync(p, it->second.bytes.data(), bytes, cudaMemcpyHostToDevice, stream);
          if (e != cudaSuccess) { cudaFree(p); meta_cache.erase(it); return cuda_fail(e, "metadata upload"); }
          traffic.bytes_h2d += bytes;
          *dev = p; *got = 0;
          return B200_OK;
        }
        cudaGetLastError();   // no room for a kept copy: the plain path below
      }
    }
    int st = alloc(bytes, dev, got);
    if (st) return st;
    if (capturing) {
      void* pin = nullptr;
      if (cudaMallocHost(&pin, bytes) != cudaSuccess) { cudaGetLastError(); release(*dev, *got); return fail(B200_OUT_OF_MEMORY, "trace: no pinned memory for a block list"); }
      memcpy(pin, host, bytes);
      cur.pinned.push_back(pin);
      host = pin;
    }
    cudaError_t e = cudaMemcpyAsync(*dev, host, bytes, cudaMemcpyHostToDevice, stream);
    if (e != cudaSuccess) { release(*dev, *got); return cuda_fail(e, "metadata upload"); }
    traffic.bytes_h2d += bytes;
    return B200_OK;
  }
  int launched(cudaError_t e, const char* what, int n = 1) {
    if (e == cudaErrorNotSupported) return fail(B200_UNSUPPORTED, "%s: unsupported", what);
    if (e != cudaSuccess) return cuda_fail(e, what);
    traffic.launches += n;
    if (capturing) { cur.launches += n; cur.ops.emplace_back(label, (uint64_t)n); }
    return B200_OK;
  }
  int wait() {
    if (capturing) return fail(B200_UNSUPPORTED, "a wait (download or sync) inside a trace capture");
    cudaError_t e = cudaMemcpyAsync(h_err, d_err, sizeof(int), cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) {
      sticky = B200_DEVICE;
      sticky_text = std::string("device failure: ") + cudaGetErrorString(e);
    } else if (*h_err != 0 && !sticky) {
      sticky = *h_err;
      sticky_text = sticky == B200_DOMAIN ? "DOMAIN: an index outside its table or a division by zero in an earlier op"
                                          : (sticky == B200_TIMEOUT ? "TIMEOUT: a bounded device wait ran out in an earlier op"
                                                                    : "an earlier op failed on the device");
    }
    if (sticky) { last_error = sticky_text; return sticky; }
    return B200_OK;
  }
};

namespace b200 {

inline void set_dims(uint64_t d[2], uint64_t r, uint64_t c) { if (d) { d[0] = r; d[1] = c; } }

// A block of a buffer.
inline int mat_of_block(b200_engine* e, const b200_block_arg* a, Mat* m, const char* what) {
  Buf* b = nullptr;
  int st = e->need(a->id, &b, what);
  if (st) return st;
  if (a->at[0] + a->dims[0] > b->rows || a->at[1] + a->dims[1] > b->cols)
    return e->fail(B200_UNSUPPORTED, "%s: block [%llu,%llu]+[%llu,%llu] outside [%llu,%llu]", what,
                   (unsigned long long)a->at[0], (unsigned long long)a->at[1], (unsigned long long)a->dims[0],
                   (unsigned long long)a->dims[1], (unsigned long long)b->rows, (unsigned long long)b->cols);
  m->bf16 = b->elem == B200_BF16;
  m->p = (const char*)b->ptr + (a->at[0] * b->cols + a->at[1]) * elem_bytes(b->elem);
  m->ld = b->cols; m->rows = a->dims[0]; m->cols = a->dims[1];
  return B200_OK;
}

inline int index_buf(b200_engine* e, b200_buffer id, Buf** b, const char* what) {
  int st = e->need(id, b, what);
  if (st) return st;
  if ((*b)->elem != B200_I32) return e->fail(B200_UNSUPPORTED, "%s: indices must be I32", what);
  return B200_OK;
}

}  // namespace b200
