// The serving operators' entry points (include/b200tt.h): the paged key/value cache's append and attention, and the
// log probabilities of given tokens with their gradient.  Argument checks, results and launches only; the state is the
// engine's (engine.h), the kernels are k_pages.cu's and k_logprob.cu's.
#include <cmath>
#include <cstring>

#include "engine.h"
#include "kernels.h"

using namespace b200;

namespace {

typedef unsigned long long ull;

// A buffer's memory, for the checks that a result written over a caller's buffer shares none of it.
struct Span { const char* at; uint64_t bytes; };
Span span_of(const Buf* b) { return Span{(const char*)b->ptr, b->rows * b->cols * elem_bytes(b->elem)}; }
struct Spans {
  Span list[12];                         // a call has at most ten operands
  size_t n = 0;
  void push_back(const Span& s) { list[n++] = s; }
};
bool meet(const Span& a, const Span& b) { return a.bytes && b.bytes && a.at < b.at + b.bytes && b.at < a.at + a.bytes; }

// Where a result goes: `into`, checked, or a new buffer.  `made` says whether it is to be dropped when the call fails.
struct Result { void* ptr = nullptr; b200_buffer id = 0; bool made = false; };
int result_of(b200_engine* e, b200_buffer into, uint64_t rows, uint64_t cols, int elem, const Spans& inputs, const char* what, Result* r) {
  Buf* b = nullptr;
  if (!into) {
    int st = e->new_buffer(rows, cols, elem, &r->id, &b);
    if (st) return st;
    r->ptr = b->ptr;
    r->made = true;
    return B200_OK;
  }
  int st = e->need(into, &b, what);
  if (st) return st;
  if (b->rows != rows || b->cols != cols || b->elem != elem)
    return e->fail(B200_UNSUPPORTED, "%s: the result is [%llu, %llu] of element %d, `into` is [%llu, %llu] of %d", what, (ull)rows, (ull)cols,
                   elem, (ull)b->rows, (ull)b->cols, b->elem);
  if (reinterpret_cast<uintptr_t>(b->ptr) & 15) return e->fail(B200_UNSUPPORTED, "%s: `into` does not start at a 16-byte address", what);
  for (size_t i = 0; i < inputs.n; ++i)
    if (meet(inputs.list[i], span_of(b))) return e->fail(B200_UNSUPPORTED, "%s: `into` shares memory with another buffer of the call", what);
  r->ptr = b->ptr;
  r->id = into;
  return B200_OK;
}
void undo(b200_engine* e, const Result& r) { if (r.made) e->drop(r.id); }

// A block of a float buffer, its extent checked without overflow.
int float_block(b200_engine* e, const b200_block_arg* a, Mat* m, Buf** b, const char* what) {
  int st = e->need(a->id, b, what);
  if (st) return st;
  if ((*b)->elem != B200_F32 && (*b)->elem != B200_BF16) return e->fail(B200_UNSUPPORTED, "%s: rows are F32 or BF16", what);
  if (a->at[0] > (*b)->rows || a->dims[0] > (*b)->rows - a->at[0] || a->at[1] > (*b)->cols || a->dims[1] > (*b)->cols - a->at[1])
    return e->fail(B200_UNSUPPORTED, "%s: block [%llu,%llu]+[%llu,%llu] outside [%llu,%llu]", what, (ull)a->at[0], (ull)a->at[1],
                   (ull)a->dims[0], (ull)a->dims[1], (ull)(*b)->rows, (ull)(*b)->cols);
  return mat_of_block(e, a, m, what);
}

// `n` I32 values as one row or one column.
int int_list(b200_engine* e, b200_buffer id, uint64_t n, Buf** b, const char* name, const char* what) {
  int st = e->need(id, b, what);
  if (st) return st;
  if ((*b)->elem != B200_I32) return e->fail(B200_UNSUPPORTED, "%s: %s are I32", what, name);
  if ((*b)->rows * (*b)->cols != n || ((*b)->rows != 1 && (*b)->cols != 1 && n != 0))
    return e->fail(B200_UNSUPPORTED, "%s: %s are [%llu, %llu] for %llu rows", what, name, (ull)(*b)->rows, (ull)(*b)->cols, (ull)n);
  return B200_OK;
}

// The cache both calls read: shape, pages, table.
int page_view(b200_engine* e, const b200_page_shape* shape, b200_buffer key_pages, b200_buffer value_pages, b200_buffer page_table,
              PageView* v, Spans* spans, const char* what) {
  if (!shape) return e->fail(B200_UNSUPPORTED, "%s: no shape", what);
  Buf *K = nullptr, *V = nullptr, *T = nullptr;
  int st = e->need(key_pages, &K, what);
  if (!st) st = e->need(value_pages, &V, what);
  if (!st) st = index_buf(e, page_table, &T, what);
  if (st) return st;
  const uint64_t width = (uint64_t)shape->kv_heads * shape->head_dim;
  if (!shape->heads || !shape->kv_heads || shape->heads % shape->kv_heads || !shape->head_dim || !shape->page_size || shape->heads > 65535 ||
      shape->head_dim > 65535)
    return e->fail(B200_UNSUPPORTED, "%s: %u heads over %u key/value heads of %u columns, pages of %u", what, shape->heads, shape->kv_heads,
                   shape->head_dim, shape->page_size);
  if ((K->elem != B200_F32 && K->elem != B200_BF16) || V->elem != K->elem)
    return e->fail(B200_UNSUPPORTED, "%s: key and value pages are both F32 or both BF16", what);
  if (K->cols != width || V->cols != width || K->rows != V->rows || K->rows % shape->page_size || K->rows > 0x7fffffffull)
    return e->fail(B200_UNSUPPORTED, "%s: key pages [%llu, %llu] and value pages [%llu, %llu] are not pages of %u rows of %llu columns", what,
                   (ull)K->rows, (ull)K->cols, (ull)V->rows, (ull)V->cols, shape->page_size, (ull)width);
  if ((reinterpret_cast<uintptr_t>(K->ptr) | reinterpret_cast<uintptr_t>(V->ptr)) & 15)
    return e->fail(B200_UNSUPPORTED, "%s: the pages do not start at a 16-byte address", what);
  if (T->rows > 0x7fffffffull || T->cols > 0x7fffffffull || T->cols * shape->page_size > 0x7fffffffull)
    return e->fail(B200_UNSUPPORTED, "%s: a page table of [%llu, %llu]", what, (ull)T->rows, (ull)T->cols);
  if (meet(span_of(K), span_of(V)))
    return e->fail(B200_UNSUPPORTED, "%s: key and value pages share memory", what);
  v->table = (const int32_t*)T->ptr;
  v->sequences = (uint32_t)T->rows; v->width = (uint32_t)T->cols;
  v->keys = K->ptr; v->values = V->ptr; v->bf16 = K->elem == B200_BF16;
  v->pages = (uint32_t)(K->rows / shape->page_size); v->page = shape->page_size;
  v->heads = shape->heads; v->kv_heads = shape->kv_heads; v->dim = shape->head_dim;
  spans->push_back(span_of(K)); spans->push_back(span_of(V)); spans->push_back(span_of(T));
  return B200_OK;
}

// What stands for -inf in a row's sums, -1e30, times the scale and log2 e has to stay a finite number far below every term.
bool good_scale(float s) { return s >= 1e-20f && s <= 1e6f; }

// `rows` F32 values as one row or one column (a per-row statistic or gradient).
int row_values(b200_engine* e, b200_buffer id, uint64_t rows, Buf** b, const char* name, const char* what) {
  int st = e->need(id, b, what);
  if (st) return st;
  if ((*b)->elem != B200_F32 || (*b)->rows * (*b)->cols != rows || ((*b)->rows != 1 && (*b)->cols != 1 && rows != 0))
    return e->fail(B200_UNSUPPORTED, "%s: %s is F32, one value a row", what, name);
  return B200_OK;
}

int logits_of(b200_engine* e, b200_buffer logits, Buf** b, const char* what) {
  int st = e->need(logits, b, what);
  if (st) return st;
  if ((*b)->elem != B200_F32 && (*b)->elem != B200_BF16) return e->fail(B200_UNSUPPORTED, "%s: logits are F32 or BF16", what);
  if ((*b)->cols == 0 || (*b)->cols > 0x7fffffffull || (*b)->rows > 0x7fffffffull)
    return e->fail(B200_UNSUPPORTED, "%s: logits [%llu, %llu]", what, (ull)(*b)->rows, (ull)(*b)->cols);
  return B200_OK;
}

}  // namespace

extern "C" {

int32_t b200_rope_append_pages(b200_engine* e, const b200_page_shape* shape, const b200_block_arg* qkv, b200_buffer cos_table,
                               b200_buffer sin_table, b200_buffer positions, b200_buffer sequences, b200_buffer page_table,
                               b200_buffer key_pages, b200_buffer value_pages, int32_t keys_out, int32_t out_bf16, b200_buffer into,
                               b200_buffer* out, uint64_t out_dims[2]) {
  const char* what = "rope_append_pages";
  cudaSetDevice(e->device);
  AppendArgs g;
  Spans spans;
  Buf *X = nullptr, *P = nullptr, *S = nullptr, *C = nullptr, *N = nullptr;
  int st = page_view(e, shape, key_pages, value_pages, page_table, &g.cache, &spans, what);
  if (!st) st = float_block(e, qkv, &g.qkv, &X, what);
  if (st) return st;
  const uint64_t n = g.qkv.rows, d = shape->head_dim;
  if (g.qkv.cols != ((uint64_t)shape->heads + 2ull * shape->kv_heads) * d)
    return e->fail(B200_UNSUPPORTED, "%s: %llu columns are not %u query and 2 x %u key and value heads of %u", what, (ull)g.qkv.cols, shape->heads,
                   shape->kv_heads, shape->head_dim);
  if (n > 0x7fffffffull || g.qkv.cols > 0x7fffffffull) return e->fail(B200_UNSUPPORTED, "%s: [%llu, %llu] rows", what, (ull)n, (ull)g.qkv.cols);
  st = int_list(e, positions, n, &P, "positions", what);
  if (!st && sequences) st = int_list(e, sequences, n, &S, "sequences", what);
  if (st) return st;
  if (!sequences && n > g.cache.sequences)
    return e->fail(B200_UNSUPPORTED, "%s: %llu rows and a page table of %u sequences", what, (ull)n, g.cache.sequences);
  if ((cos_table != 0) != (sin_table != 0)) return e->fail(B200_UNSUPPORTED, "%s: a cos table without a sin table, or the reverse", what);
  if (cos_table) {
    st = e->need(cos_table, &C, what);
    if (!st) st = e->need(sin_table, &N, what);
    if (st) return st;
    if (C->elem != B200_F32 || N->elem != B200_F32 || C->rows != N->rows || C->cols != N->cols || C->cols == 0 || C->cols % 2 || C->cols > d)
      return e->fail(B200_UNSUPPORTED, "%s: cos [%llu, %llu] and sin [%llu, %llu] tables are F32 alike, an even number of columns within a head of %u",
                     what, (ull)C->rows, (ull)C->cols, (ull)N->rows, (ull)N->cols, shape->head_dim);
    g.cos = (const float*)C->ptr; g.sin = (const float*)N->ptr;
    g.table_rows = C->rows; g.rotary = (uint32_t)C->cols;
    spans.push_back(span_of(C)); spans.push_back(span_of(N));
  }
  spans.push_back(span_of(X)); spans.push_back(span_of(P));
  if (S) spans.push_back(span_of(S));
  // the pages are written while the other operands are read
  for (size_t i = 2; i < spans.n; ++i)
    if (meet(spans.list[0], spans.list[i]) || meet(spans.list[1], spans.list[i])) return e->fail(B200_UNSUPPORTED, "%s: the pages share memory with another operand", what);
  const uint64_t cols = ((uint64_t)shape->heads + (keys_out ? shape->kv_heads : 0)) * d;
  Result r;
  st = result_of(e, into, n, cols, out_bf16 ? B200_BF16 : B200_F32, spans, what, &r);
  if (st) return st;
  g.positions = (const int32_t*)P->ptr; g.sequences = S ? (const int32_t*)S->ptr : nullptr;
  g.n = n; g.keys_out = keys_out ? 1 : 0; g.out = r.ptr; g.out_bf16 = out_bf16 ? 1 : 0; g.err = e->d_err;
  st = e->launched(launch_rope_append_pages(g, e->stream), what, n ? 1 : 0);
  if (st) { undo(e, r); return st; }
  *out = r.id;
  set_dims(out_dims, n, cols);
  return B200_OK;
}

int32_t b200_attention_pages(b200_engine* e, const b200_page_shape* shape, const b200_block_arg* q, b200_buffer key_pages, b200_buffer value_pages,
                             b200_buffer page_table, b200_buffer positions, uint32_t window, float scale, int32_t out_bf16, b200_buffer into,
                             b200_buffer* out, uint64_t out_dims[2]) {
  const char* what = "attention_pages";
  cudaSetDevice(e->device);
  AttnPagesArgs g;
  Spans spans;
  Buf *Q = nullptr, *P = nullptr;
  int st = page_view(e, shape, key_pages, value_pages, page_table, &g.cache, &spans, what);
  if (!st) st = float_block(e, q, &g.q, &Q, what);
  if (st) return st;
  const uint64_t n = g.q.rows, cols = (uint64_t)shape->heads * shape->head_dim;
  if (!attention_pages_dim_ok(shape->head_dim)) return e->fail(B200_UNSUPPORTED, "%s: heads of %u columns (32, 64, 96, 128, 192 or 256)", what, shape->head_dim);
  if (g.q.cols != cols) return e->fail(B200_UNSUPPORTED, "%s: %llu query columns for %u heads of %u", what, (ull)g.q.cols, shape->heads, shape->head_dim);
  if (n > g.cache.sequences) return e->fail(B200_UNSUPPORTED, "%s: %llu rows and a page table of %u sequences", what, (ull)n, g.cache.sequences);
  if (!(std::fabs(scale) <= 1e20f)) return e->fail(B200_UNSUPPORTED, "%s: the scale %g is not within -1e20 .. 1e20", what, scale);
  st = int_list(e, positions, n, &P, "positions", what);
  if (st) return st;
  spans.push_back(span_of(Q)); spans.push_back(span_of(P));
  Result r;
  st = result_of(e, into, n, cols, out_bf16 ? B200_BF16 : B200_F32, spans, what, &r);
  if (st) return st;
  g.positions = (const int32_t*)P->ptr;
  g.n = n; g.window = window; g.scale = scale; g.out = r.ptr; g.out_bf16 = out_bf16 ? 1 : 0; g.err = e->d_err;
  int launches = 0;
  void* scratch = nullptr;
  uint64_t got = 0;
  const size_t bytes = n ? attention_pages_scratch_bytes(g) : 0;
  st = bytes ? e->alloc(bytes, &scratch, &got) : B200_OK;
  if (st) { undo(e, r); return st; }
  const cudaError_t ce = launch_attention_pages(g, scratch, &launches, e->stream);
  if (bytes) e->release(scratch, got);
  st = e->launched(ce, what, launches);
  if (st) { undo(e, r); return st; }
  *out = r.id;
  set_dims(out_dims, n, cols);
  return B200_OK;
}

int32_t b200_token_logprobs(b200_engine* e, b200_buffer logits, b200_buffer ids, float scale, uint32_t top, const b200_buffer into[5],
                            b200_buffer out[5], uint64_t out_dims[2]) {
  const char* what = "token_logprobs";
  cudaSetDevice(e->device);
  Buf *X = nullptr, *I = nullptr;
  int st = logits_of(e, logits, &X, what);
  if (st) return st;
  const uint64_t rows = X->rows, cols = X->cols;
  st = int_list(e, ids, rows, &I, "ids", what);
  if (st) return st;
  if (!good_scale(scale)) return e->fail(B200_UNSUPPORTED, "%s: the scale %g is not within 1e-20 .. 1e6", what, scale);
  if (top > 32 || top > cols) return e->fail(B200_UNSUPPORTED, "%s: the %u largest of %llu columns (at most 32)", what, top, (ull)cols);
  LogprobArgs g;
  g.logits = X->ptr; g.bf16 = X->elem == B200_BF16; g.rows = rows; g.cols = cols;
  g.ids = (const int32_t*)I->ptr; g.scale = scale; g.top = top; g.err = e->d_err;
  Spans spans;
  spans.push_back(span_of(X)); spans.push_back(span_of(I));
  Result r[5];
  const int parts = top ? 5 : 3;
  for (int i = 0; i < parts; ++i) {
    st = result_of(e, into ? into[i] : 0, rows, i < 3 ? 1 : top, i == 3 ? B200_I32 : B200_F32, spans, what, &r[i]);
    if (st) { for (int j = 0; j < i; ++j) undo(e, r[j]); return st; }
    spans.push_back(Span{(const char*)r[i].ptr, rows * (i < 3 ? 1 : top) * 4});   // the results share no memory either
  }
  g.logprob = (float*)r[0].ptr; g.entropy = (float*)r[1].ptr; g.lse = (float*)r[2].ptr;
  g.top_ids = (int32_t*)r[3].ptr; g.top_logprobs = (float*)r[4].ptr;
  st = e->launched(launch_token_logprobs(g, e->stream), what, rows ? 1 : 0);
  if (st) { for (int j = 0; j < parts; ++j) undo(e, r[j]); return st; }
  for (int i = 0; i < 5; ++i) out[i] = r[i].id;
  set_dims(out_dims, rows, 1);
  return B200_OK;
}

int32_t b200_token_logprobs_backward(b200_engine* e, b200_buffer logits, b200_buffer ids, b200_buffer lse, b200_buffer entropy,
                                     b200_buffer d_logprob, b200_buffer d_entropy, float scale, int32_t out_bf16, b200_buffer into,
                                     b200_buffer* out, uint64_t out_dims[2]) {
  const char* what = "token_logprobs_backward";
  cudaSetDevice(e->device);
  Buf *X = nullptr, *I = nullptr, *L = nullptr, *H = nullptr, *G = nullptr, *GH = nullptr;
  int st = logits_of(e, logits, &X, what);
  if (st) return st;
  const uint64_t rows = X->rows, cols = X->cols;
  st = int_list(e, ids, rows, &I, "ids", what);
  if (!st) st = row_values(e, lse, rows, &L, "lse", what);
  if (!st) st = row_values(e, d_logprob, rows, &G, "d_logprob", what);
  if (!st && d_entropy) st = row_values(e, d_entropy, rows, &GH, "d_entropy", what);
  if (!st && d_entropy) st = row_values(e, entropy, rows, &H, "entropy", what);
  if (st) return st;
  if (!good_scale(scale)) return e->fail(B200_UNSUPPORTED, "%s: the scale %g is not within 1e-20 .. 1e6", what, scale);
  Spans spans;
  for (const Buf* b : {X, I, L, G}) spans.push_back(span_of(b));
  if (GH) { spans.push_back(span_of(GH)); spans.push_back(span_of(H)); }
  Result r;
  st = result_of(e, into, rows, cols, out_bf16 ? B200_BF16 : B200_F32, spans, what, &r);
  if (st) return st;
  LogprobGradArgs g;
  g.logits = X->ptr; g.bf16 = X->elem == B200_BF16; g.rows = rows; g.cols = cols; g.ids = (const int32_t*)I->ptr;
  g.lse = (const float*)L->ptr; g.d_logprob = (const float*)G->ptr;
  if (GH) { g.d_entropy = (const float*)GH->ptr; g.entropy = (const float*)H->ptr; }
  g.scale = scale; g.out = r.ptr; g.out_bf16 = out_bf16 ? 1 : 0; g.err = e->d_err;
  st = e->launched(launch_token_logprobs_backward(g, e->stream), what, rows ? 1 : 0);
  if (st) { undo(e, r); return st; }
  *out = r.id;
  set_dims(out_dims, rows, cols);
  return B200_OK;
}

int32_t b200_serving_call(b200_engine* e, int32_t call, uint64_t* w, uint64_t n_words) {
  const uint64_t counts[4] = {19, 17, 16, 12};
  if (call < 0 || call > 3 || !w || n_words != counts[call])
    return e->fail(B200_UNSUPPORTED, "serving_call: call %d of %llu words", call, (ull)n_words);
  const auto f32_of = [](uint64_t word) {
    const uint32_t bits = (uint32_t)word;
    float f;
    memcpy(&f, &bits, 4);
    return f;
  };
  const b200_page_shape* shape = reinterpret_cast<const b200_page_shape*>(w[0]);
  const b200_block_arg block = {w[1], {w[2], w[3]}, {w[4], w[5]}};
  switch (call) {
    case B200_ROPE_APPEND_PAGES:
      return b200_rope_append_pages(e, shape, &block, w[6], w[7], w[8], w[9], w[10], w[11], w[12], (int32_t)w[13], (int32_t)w[14], w[15],
                                    (b200_buffer*)&w[16], &w[17]);
    case B200_ATTENTION_PAGES:
      return b200_attention_pages(e, shape, &block, w[6], w[7], w[8], w[9], (uint32_t)w[10], f32_of(w[11]), (int32_t)w[12], w[13],
                                  (b200_buffer*)&w[14], &w[15]);
    case B200_TOKEN_LOGPROBS:
      return b200_token_logprobs(e, w[0], w[1], f32_of(w[2]), (uint32_t)w[3], (const b200_buffer*)&w[4], (b200_buffer*)&w[9], &w[14]);
    default:
      return b200_token_logprobs_backward(e, w[0], w[1], w[2], w[3], w[4], w[5], f32_of(w[6]), (int32_t)w[7], w[8], (b200_buffer*)&w[9],
                                          &w[10]);
  }
}

}  // extern "C"
