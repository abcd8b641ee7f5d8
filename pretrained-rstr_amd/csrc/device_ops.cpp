// device_ops.cpp -- C ABI of the operators on device arrays: the 4-bit paged
// cache (append, read, attention), step maps and draft verification.  They
// queue kernels on the caller's stream and nothing else: no allocation, copy or
// wait, so they may be captured into a graph.
#include <hip/hip_runtime.h>

#include <cmath>
#include <memory>
#include <new>
#include <string>

#include "device_args.h"
#include "kv4.h"
#include "kv4_line.h"
#include "session.h"

using namespace rstr;

struct rstr_kv4 {
  rstr_session* s = nullptr;
  int layers = 0, n_kv = 0, hd = 0, page_size = 0, pages = 0;
  int64_t layer_bytes = 0;
  uint8_t* base = nullptr;
  int plans = 0;  // open attention plans
};
struct rstr_kv4_attn {
  rstr_kv4* p = nullptr;
  int n_q = 0, batch = 0, rows = 0;
  void* ws = nullptr;
};
struct rstr_verify {
  rstr_session* s = nullptr;
  int batch = 0, rows = 0, vocab = 0;
  void* ws = nullptr;
};

namespace {

Kv4Layer layer_of(const rstr_kv4* p, int layer) {
  return Kv4Layer{p->base + (int64_t)layer * p->layer_bytes, p->n_kv, p->hd, p->page_size, p->pages};
}

}  // namespace

// ---------------------------------------------------------------------------
// 4-bit paged cache
// ---------------------------------------------------------------------------
extern "C" int rstr_kv4_open(rstr_session* s, int32_t n_layers, int32_t n_kv, int32_t head_dim, int32_t page_size,
                             int32_t physical_pages, rstr_kv4** out) {
  if (!s) return fail(nullptr, RSTR_E_INVALID, "null session");
  if (!out) return fail(s, RSTR_E_INVALID, "null output pointer");
  *out = nullptr;
  if (n_layers <= 0 || n_kv <= 0 || page_size <= 0 || physical_pages <= 0)
    return fail(s, RSTR_E_INVALID, "4-bit cache extents must be positive integers");
  if (!kv4_head_dim(head_dim)) return fail(s, RSTR_E_INVALID, "4-bit cache head dim must be 64, 128 or 256");
  if (page_size % 16) return fail(s, RSTR_E_INVALID, "4-bit cache page size must be a multiple of 16");
  if ((int64_t)page_size * physical_pages > 0x7FFFFFFF) return fail(s, RSTR_E_INVALID, "4-bit cache slots must fit in 31 bits");
  // offsets inside a page are 32 bits
  if ((double)kv4_record_bytes(head_dim, page_size) * n_kv > 2e9) return fail(s, RSTR_E_INVALID, "4-bit cache pages must be smaller than 2 GB");
  std::unique_ptr<rstr_kv4> p(new (std::nothrow) rstr_kv4());
  if (!p) return fail(s, RSTR_E_OOM, "4-bit cache handle");
  p->s = s;
  p->layers = n_layers;
  p->n_kv = n_kv;
  p->hd = head_dim;
  p->page_size = page_size;
  p->pages = physical_pages;
  const double want = (double)n_layers * n_kv * physical_pages * (double)kv4_record_bytes(head_dim, page_size);
  if (want > 1e15) return fail(s, RSTR_E_OOM, "4-bit cache allocation failed");
  p->layer_bytes = (int64_t)n_kv * physical_pages * kv4_record_bytes(head_dim, page_size);
  const size_t bytes = (size_t)p->layer_bytes * n_layers;
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  if (device_alloc((void**)&p->base, bytes) != hipSuccess) {
    (void)hipGetLastError();
    return fail(s, RSTR_E_OOM, "4-bit cache allocation failed");
  }
  hipError_t e = hipMemsetAsync(p->base, 0, bytes, s->stream);  // scale 0: zeros
  if (e == hipSuccess) e = hipStreamSynchronize(s->stream);
  if (e != hipSuccess) {
    (void)hipFree(p->base);
    HIPCHK(s, e);
  }
  *out = p.release();
  return RSTR_OK;
}

extern "C" int rstr_kv4_close(rstr_kv4* p) {
  if (!p) return RSTR_OK;
  if (p->plans > 0) return fail(p->s, RSTR_E_STATE, "4-bit cache has open attention plans");
  OnDevice dev(p->s->device);
  (void)hipDeviceSynchronize();  // work on it may be queued on any stream
  (void)hipFree(p->base);
  delete p;
  return RSTR_OK;
}

extern "C" int64_t rstr_kv4_bytes(const rstr_kv4* p) { return p ? p->layer_bytes * p->layers : -1; }

static int kv4_rows_args(rstr_kv4* p, int32_t layer, int32_t rows, int32_t dtype, const Rows& k, const Rows& v,
                         const int32_t* slots) {
  rstr_session* s = p->s;
  if (layer < 0 || layer >= p->layers) return fail(s, RSTR_E_INVALID, "layer is outside the 4-bit cache");
  if (rows < 0) return fail(s, RSTR_E_INVALID, "row count must not be negative");
  const int size = elem_size(dtype);
  if (!size) return fail(s, RSTR_E_INVALID, "element type must be f32, f16 or bf16");
  if (rows == 0) return RSTR_OK;
  TRY(check_rows(s, "key", k, size));
  TRY(check_rows(s, "value", v, size));
  TRY(check_ints(s, "slots", slots));
  if (((int64_t)rows / 4 + 8) * p->n_kv * (p->hd / 8) > 0x7FFFFFFF) return fail(s, RSTR_E_INVALID, "too many rows for one call");
  return RSTR_OK;
}

extern "C" int rstr_kv4_append(rstr_kv4* p, int32_t layer, int32_t rows, int32_t dtype, const void* k, int64_t k_row,
                               int64_t k_head, const void* v, int64_t v_row, int64_t v_head, const int32_t* slots,
                               void* stream) {
  if (!p) return fail(nullptr, RSTR_E_INVALID, "null 4-bit cache");
  const Rows kr{(void*)k, k_row, k_head}, vr{(void*)v, v_row, v_head};
  TRY(kv4_rows_args(p, layer, rows, dtype, kr, vr, slots));
  if (rows == 0) return RSTR_OK;
  OnDevice dev(p->s->device);
  HIPCHK(p->s, dev.e);
  HIPCHK(p->s, launch_kv4_append(on_stream(p->s, stream), layer_of(p, layer), dtype, rows, kr, vr, slots));
  return RSTR_OK;
}

extern "C" int rstr_kv4_read(rstr_kv4* p, int32_t layer, int32_t rows, int32_t dtype, const int32_t* slots, void* k,
                             int64_t k_row, int64_t k_head, void* v, int64_t v_row, int64_t v_head, void* stream) {
  if (!p) return fail(nullptr, RSTR_E_INVALID, "null 4-bit cache");
  rstr_session* s = p->s;
  const Rows kr{k, k_row, k_head}, vr{v, v_row, v_head};
  TRY(kv4_rows_args(p, layer, rows, dtype, kr, vr, slots));
  if (rows == 0) return RSTR_OK;
  if (!apart(kr, rows, p->n_kv, p->hd) || !apart(vr, rows, p->n_kv, p->hd))
    return fail(s, RSTR_E_INVALID, "output rows share elements");
  const int size = elem_size(dtype);
  if (share(kr, vr, rows, p->n_kv, p->hd, size)) return fail(s, RSTR_E_INVALID, "output keys and values share elements");
  for (const Rows& o : {kr, vr})
    if (ranges_meet((uintptr_t)slots, (uintptr_t)(slots + rows), (uintptr_t)o.p, rows_end(o, rows, p->n_kv, p->hd, size)))
      return fail(s, RSTR_E_INVALID, "output rows overlap the slots");
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  HIPCHK(s, launch_kv4_read(on_stream(s, stream), layer_of(p, layer), dtype, rows, slots, kr, vr));
  return RSTR_OK;
}

extern "C" int rstr_kv4_attn_open(rstr_kv4* p, int32_t n_q, int32_t max_batch, int32_t max_rows, rstr_kv4_attn** out) {
  if (!p) return fail(nullptr, RSTR_E_INVALID, "null 4-bit cache");
  rstr_session* s = p->s;
  if (!out) return fail(s, RSTR_E_INVALID, "null output pointer");
  *out = nullptr;
  if (n_q <= 0 || n_q % p->n_kv) return fail(s, RSTR_E_INVALID, "query heads must be a multiple of the cache's kv heads");
  if (max_batch <= 0 || max_rows <= 0) return fail(s, RSTR_E_INVALID, "attention plan extents must be positive");
  // a workgroup of up to 256 threads an item joins its pieces, and a grid holds fewer than 2^32 threads
  if ((int64_t)max_rows * n_q > 0x7FFFF000 || attn_items(n_q, p->n_kv, max_batch, max_rows, 16) >= kGridGroups) return fail(s, RSTR_E_INVALID, "attention plan has too many rows");
  std::unique_ptr<rstr_kv4_attn> a(new (std::nothrow) rstr_kv4_attn());
  if (!a) return fail(s, RSTR_E_OOM, "attention plan handle");
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  if (device_alloc(&a->ws, kv4_attn_workspace(n_q, p->n_kv, p->hd, max_batch, max_rows)) != hipSuccess) {
    (void)hipGetLastError();
    return fail(s, RSTR_E_OOM, "attention plan workspace allocation failed");
  }
  a->p = p;
  a->n_q = n_q;
  a->batch = max_batch;
  a->rows = max_rows;
  p->plans++;
  *out = a.release();
  return RSTR_OK;
}

extern "C" int rstr_kv4_attn_close(rstr_kv4_attn* a) {
  if (!a) return RSTR_OK;
  OnDevice dev(a->p->s->device);
  (void)hipDeviceSynchronize();
  (void)hipFree(a->ws);
  a->p->plans--;
  delete a;
  return RSTR_OK;
}

extern "C" int rstr_kv4_attn_run(rstr_kv4_attn* a, int32_t layer, int32_t dtype, int32_t batch, int32_t rows,
                                 int32_t max_rows, int32_t window, float scale, const void* q, int64_t q_row, int64_t q_head,
                                 const int32_t* row_offsets, const int32_t* page_table, int32_t pages_per_seq,
                                 const int32_t* lengths, void* out, int64_t out_row, int64_t out_head, void* stream) {
  if (!a) return fail(nullptr, RSTR_E_INVALID, "null attention plan");
  rstr_kv4* p = a->p;
  rstr_session* s = p->s;
  if (layer < 0 || layer >= p->layers) return fail(s, RSTR_E_INVALID, "layer is outside the 4-bit cache");
  const int size = elem_size(dtype);
  if (!size) return fail(s, RSTR_E_INVALID, "element type must be f32, f16 or bf16");
  if (batch < 0 || batch > a->batch) return fail(s, RSTR_E_INVALID, "batch exceeds the attention plan's");
  if (rows < 0 || rows > a->rows) return fail(s, RSTR_E_INVALID, "rows exceed the attention plan's");
  if (window < 0) return fail(s, RSTR_E_INVALID, "window must not be negative");
  if (!std::isfinite(scale)) return fail(s, RSTR_E_INVALID, "scale must be finite");
  if (batch == 0 || rows == 0) return RSTR_OK;
  if (max_rows <= 0 || max_rows > rows) return fail(s, RSTR_E_INVALID, "rows per sequence must lie between 1 and the rows");
  if (pages_per_seq <= 0) return fail(s, RSTR_E_INVALID, "page table width must be positive");
  const Rows qr{(void*)q, q_row, q_head}, o{out, out_row, out_head};
  TRY(check_rows(s, "query", qr, size));
  TRY(check_rows(s, "output", o, size));
  TRY(check_ints(s, "row offsets", row_offsets));
  TRY(check_ints(s, "page table", page_table));
  TRY(check_ints(s, "lengths", lengths));
  if (!apart(o, rows, a->n_q, p->hd)) return fail(s, RSTR_E_INVALID, "output rows share elements");
  if (ranges_meet((uintptr_t)q, rows_end(qr, rows, a->n_q, p->hd, size), (uintptr_t)out, rows_end(o, rows, a->n_q, p->hd, size)))
    return fail(s, RSTR_E_INVALID, "output overlaps the queries");
  const struct { const int32_t* p; int64_t n; } ints[] = {{row_offsets, batch + (int64_t)1}, {page_table, (int64_t)batch * pages_per_seq}, {lengths, batch}};
  for (const auto& x : ints)
    if (ranges_meet((uintptr_t)x.p, (uintptr_t)(x.p + x.n), (uintptr_t)out, rows_end(o, rows, a->n_q, p->hd, size)))
      return fail(s, RSTR_E_INVALID, "output overlaps the sequences' tables");
  Kv4Attn k{};
  k.c = layer_of(p, layer);
  k.n_q = a->n_q;
  k.batch = batch;
  k.rows = rows;
  k.max_rows = max_rows;
  k.window = window;
  k.pps = pages_per_seq;
  k.scale = scale;
  k.q = qr;
  k.out = o;
  k.row_offsets = row_offsets;
  k.page_table = page_table;
  k.lengths = lengths;
  k.ws = a->ws;
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  HIPCHK(s, launch_kv4_attn(on_stream(s, stream), dtype, k));
  return RSTR_OK;
}

// ---------------------------------------------------------------------------
// step maps
// ---------------------------------------------------------------------------
extern "C" int rstr_step_maps(rstr_session* s, int32_t page_size, int32_t batch, int32_t pages_per_seq, int32_t rows,
                              const int32_t* lengths, const int32_t* counts, const int32_t* start_positions,
                              const int32_t* free_pages, int32_t n_free, int32_t* page_table, int32_t* new_lengths,
                              int32_t* row_offsets, int32_t* positions, int32_t* slots, int32_t* pages_taken, void* stream) {
  if (!s) return fail(nullptr, RSTR_E_INVALID, "null session");
  if (page_size <= 0 || pages_per_seq <= 0) return fail(s, RSTR_E_INVALID, "step map extents must be positive integers");
  if (batch <= 0 || batch > RSTR_STEP_MAPS_BATCH) return fail(s, RSTR_E_INVALID, "step map batch is out of range");
  if (rows < 0 || n_free < 0) return fail(s, RSTR_E_INVALID, "row and free page counts must not be negative");
  TRY(check_ints(s, "lengths", lengths));
  TRY(check_ints(s, "counts", counts));
  TRY(check_ints(s, "page table", page_table));
  TRY(check_ints(s, "new lengths", new_lengths));
  TRY(check_ints(s, "row offsets", row_offsets));
  TRY(check_ints(s, "pages taken", pages_taken));
  if (n_free > 0) TRY(check_ints(s, "free pages", free_pages));
  if (rows > 0) {
    TRY(check_ints(s, "positions", positions));
    TRY(check_ints(s, "slots", slots));
  }
  if (!aligned(start_positions, 4)) return fail(s, RSTR_E_INVALID, "start positions not aligned to its elements");
  // every workgroup reads all inputs while others already write
  const size_t n = (size_t)batch * 4, r = (size_t)rows * 4, f = (size_t)n_free * 4;
  const struct { const void* p; size_t n; } in[] = {{lengths, n}, {counts, n}, {start_positions, start_positions ? n : 0}, {free_pages, f}};
  const struct { const void* p; size_t n; } out[] = {{page_table, n * pages_per_seq}, {new_lengths, n}, {row_offsets, n + 4},
                                                     {positions, r}, {slots, r}, {pages_taken, 4}};
  for (size_t i = 0; i < sizeof(out) / sizeof(out[0]); i++) {
    for (const auto& x : in)
      if (x.n && out[i].n && ranges_meet(x.p, x.n, out[i].p, out[i].n)) return fail(s, RSTR_E_INVALID, "step map outputs overlap its inputs");
    for (size_t j = 0; j < i; j++)
      if (out[i].n && out[j].n && ranges_meet(out[j].p, out[j].n, out[i].p, out[i].n))
        return fail(s, RSTR_E_INVALID, "step map outputs overlap");
  }
  StepMaps m{page_size, batch, pages_per_seq, rows, n_free, lengths, counts, start_positions, free_pages,
             page_table, new_lengths, row_offsets, positions, slots, pages_taken};
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  HIPCHK(s, launch_step_maps(on_stream(s, stream), m));
  return RSTR_OK;
}

// ---------------------------------------------------------------------------
// draft verification
// ---------------------------------------------------------------------------
extern "C" int rstr_verify_open(rstr_session* s, int32_t max_batch, int32_t max_rows, int32_t vocab, rstr_verify** out) {
  if (!s) return fail(nullptr, RSTR_E_INVALID, "null session");
  if (!out) return fail(s, RSTR_E_INVALID, "null output pointer");
  *out = nullptr;
  if (max_batch <= 0 || max_rows <= 0 || vocab <= 0) return fail(s, RSTR_E_INVALID, "verification extents must be positive");
  if (max_batch >= kGridGroups || max_rows >= kGridGroups) return fail(s, RSTR_E_INVALID, "verification has too many rows");
  if (vocab > RSTR_VERIFY_VOCAB) return fail(s, RSTR_E_INVALID, "vocabulary is too large for verification");
  std::unique_ptr<rstr_verify> v(new (std::nothrow) rstr_verify());
  if (!v) return fail(s, RSTR_E_OOM, "verification handle");
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  if (device_alloc(&v->ws, verify_workspace(max_batch, max_rows, vocab)) != hipSuccess) {
    (void)hipGetLastError();
    return fail(s, RSTR_E_OOM, "verification workspace allocation failed");
  }
  v->s = s;
  v->batch = max_batch;
  v->rows = max_rows;
  v->vocab = vocab;
  *out = v.release();
  return RSTR_OK;
}

extern "C" int rstr_verify_close(rstr_verify* v) {
  if (!v) return RSTR_OK;
  OnDevice dev(v->s->device);
  (void)hipDeviceSynchronize();
  (void)hipFree(v->ws);
  delete v;
  return RSTR_OK;
}

extern "C" int rstr_verify_run(rstr_verify* v, int32_t dtype, int32_t batch, int32_t rows, const void* logits,
                               int64_t logits_row, const int32_t* row_offsets, const int32_t* drafts, const float* draft_probs,
                               int64_t probs_row, const float* temperature, const float* u_accept, const float* u_sample,
                               int32_t* accepted, int32_t* tokens, void* stream) {
  if (!v) return fail(nullptr, RSTR_E_INVALID, "null verification handle");
  rstr_session* s = v->s;
  const int size = elem_size(dtype);
  if (!size) return fail(s, RSTR_E_INVALID, "element type must be f32, f16 or bf16");
  if (batch < 0 || batch > v->batch) return fail(s, RSTR_E_INVALID, "batch exceeds the verification handle's");
  if (rows < 0 || rows > v->rows) return fail(s, RSTR_E_INVALID, "rows exceed the verification handle's");
  if (batch == 0) return RSTR_OK;
  TRY(check_ints(s, "row offsets", row_offsets));
  TRY(check_ints(s, "accepted counts", accepted));
  if (rows > 0) {
    const Rows x{(void*)logits, logits_row, 0};
    TRY(check_rows(s, "logit", x, size));
    TRY(check_ints(s, "drafts", drafts));
    TRY(check_ints(s, "tokens", tokens));
    TRY(check_ints(s, "temperatures", (const int32_t*)temperature));
    TRY(check_ints(s, "acceptance numbers", (const int32_t*)u_accept));
    TRY(check_ints(s, "sampling numbers", (const int32_t*)u_sample));
    if (draft_probs) TRY(check_rows(s, "draft probability", Rows{(void*)draft_probs, probs_row, 0}, 4));
    const size_t r = (size_t)rows * 4, n = (size_t)batch * 4;
    const struct { const void* p; size_t n; } in[] = {{row_offsets, n + 4}, {drafts, r}, {temperature, n}, {u_accept, r}, {u_sample, n}};
    for (const auto& x2 : in)
      if (ranges_meet(x2.p, x2.n, accepted, n) || ranges_meet(x2.p, x2.n, tokens, r))
        return fail(s, RSTR_E_INVALID, "verification outputs overlap its inputs");
    const Rows probs{(void*)draft_probs, probs_row, 0};
    const struct { uintptr_t a, b; } wide[] = {{(uintptr_t)logits, rows_end(x, rows, 1, v->vocab, size)},
                                               {(uintptr_t)draft_probs, draft_probs ? rows_end(probs, rows, 1, v->vocab, 4) : 0}};
    for (const auto& y : wide)
      if (ranges_meet(y.a, y.b, (uintptr_t)accepted, (uintptr_t)accepted + n) || ranges_meet(y.a, y.b, (uintptr_t)tokens, (uintptr_t)tokens + r))
        return fail(s, RSTR_E_INVALID, "verification outputs overlap its inputs");
    if (ranges_meet(accepted, n, tokens, r)) return fail(s, RSTR_E_INVALID, "verification outputs overlap");
  }
  Verify a{batch, rows, v->vocab, logits, logits_row, row_offsets, drafts, draft_probs, probs_row, temperature,
           u_accept, u_sample, accepted, tokens, v->ws};
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  HIPCHK(s, launch_verify(on_stream(s, stream), dtype, a));
  return RSTR_OK;
}
