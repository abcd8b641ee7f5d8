// pool_ops.cpp -- C ABI of the operators on device arrays over the fp16 page pool: appends with the position
// rotation, attention of ragged rows, bounds of blocks and the selection of blocks.  As in device_ops.cpp they queue
// kernels on the caller's stream and nothing else, so they may be captured into a graph.
#include <hip/hip_runtime.h>

#include <cmath>
#include <memory>
#include <new>
#include <string>

#include "device_args.h"
#include "pool_ops.h"
#include "session.h"

using namespace rstr;

struct rstr_pool_attn {
  rstr_pool* p = nullptr;
  int n_q = 0, batch = 0, rows = 0;
  void* ws = nullptr;
};
struct rstr_bounds {
  rstr_pool* p = nullptr;
  int64_t layer_elems = 0;
  uint16_t* base = nullptr;
  int plans = 0;  // open selections
};
struct rstr_select {
  rstr_bounds* b = nullptr;
  int n_q = 0, batch = 0, rows = 0, blocks = 0;
  void* ws = nullptr;
};

namespace {

// A [rows][heads][hd] array of which one is written: do the two share an element?  Arrays of one row stride whose heads all lie
// within it (views of one projection's output) do not where their places in it are apart.
bool meet(const Rows& a, int64_t a_heads, const Rows& b, int64_t b_heads, int64_t rows, int64_t hd, int size) {
  if (!ranges_meet((uintptr_t)a.p, rows_end(a, rows, a_heads, hd, size), (uintptr_t)b.p, rows_end(b, rows, b_heads, hd, size))) return false;
  const bool b_behind = (uintptr_t)b.p >= (uintptr_t)a.p;
  const Rows &x = b_behind ? a : b, &y = b_behind ? b : a;
  const int64_t xs = ((b_behind ? a_heads : b_heads) - 1) * x.head + hd, ys = ((b_behind ? b_heads : a_heads) - 1) * y.head + hd;
  const uintptr_t bytes = (uintptr_t)y.p - (uintptr_t)x.p;
  if (x.row != y.row || x.row <= 0 || bytes % size) return true;
  const int64_t d = (int64_t)(bytes / size) % x.row;
  return !(d >= xs && d + ys <= x.row);
}

bool ints_meet(const void* p, int64_t bytes, const Rows& o, int64_t rows, int64_t heads, int64_t hd, int size) {
  return p && ranges_meet((uintptr_t)p, (uintptr_t)p + (uintptr_t)bytes, (uintptr_t)o.p, rows_end(o, rows, heads, hd, size));
}

// Do the rows lie in the pages of the pool's layer?
bool in_pages(const PoolLayer& c, const Rows& r, int64_t rows, int64_t heads, int size) {
  const uintptr_t bytes = (uintptr_t)c.pages * c.page_size * c.n_kv * c.hd * 2, end = rows_end(r, rows, heads, c.hd, size);
  return ranges_meet((uintptr_t)r.p, end, (uintptr_t)c.k, (uintptr_t)c.k + bytes) || ranges_meet((uintptr_t)r.p, end, (uintptr_t)c.v, (uintptr_t)c.v + bytes);
}

constexpr int kMostHeads = 1 << 16;

// What the attention, the bounds and the selection take alike: the sequences of a call.
int sequences_args(rstr_session* s, const int32_t* row_offsets, const int32_t* page_table, int32_t pages_per_seq, const int32_t* lengths) {
  if (pages_per_seq <= 0) return fail(s, RSTR_E_INVALID, "page table width must be positive");
  TRY(check_ints(s, "row offsets", row_offsets));
  TRY(check_ints(s, "page table", page_table));
  TRY(check_ints(s, "lengths", lengths));
  return RSTR_OK;
}

}  // namespace

// ---------------------------------------------------------------------------
// rotated append
// ---------------------------------------------------------------------------
extern "C" int rstr_pool_device(rstr_pool* p, int32_t slab, int32_t layer, void** out) {
  if (!p) return fail(nullptr, RSTR_E_INVALID, "null pool");
  const PoolView v = pool_view(p, 0);
  if (!out) return fail(v.s, RSTR_E_INVALID, "null output pointer");
  *out = nullptr;
  if (slab < 0 || slab > 1 || layer < 0 || layer >= v.layers) return fail(v.s, RSTR_E_INVALID, "slab or layer is outside the pool");
  const PoolLayer c = pool_view(p, layer).c;
  *out = slab ? c.v : c.k;
  pool_shared(p);
  return RSTR_OK;
}

extern "C" int rstr_pool_rope_append(rstr_pool* p, int32_t layer, int32_t rows, int32_t dtype, const void* k, int64_t k_row, int64_t k_head,
                                     const void* v, int64_t v_row, int64_t v_head, int32_t n_q, const void* q, int64_t q_row, int64_t q_head,
                                     void* q_out, int64_t q_out_row, int64_t q_out_head, const float* q_gain, const float* k_gain, float eps,
                                     float gain_offset, int32_t rotary_dim, const double* frequencies, const int32_t* positions,
                                     const int32_t* slots, void* stream) {
  if (!p) return fail(nullptr, RSTR_E_INVALID, "null pool");
  PoolView pv = pool_view(p, 0);
  rstr_session* s = pv.s;
  if (layer < 0 || layer >= pv.layers) return fail(s, RSTR_E_INVALID, "layer is outside the pool");
  pv = pool_view(p, layer);
  const int hd = pv.c.hd, n_kv = pv.c.n_kv;
  if (rows < 0) return fail(s, RSTR_E_INVALID, "row count must not be negative");
  const int size = elem_size(dtype);
  if (!size) return fail(s, RSTR_E_INVALID, "element type must be f32, f16 or bf16");
  if (n_q < 0 || n_q > kMostHeads || n_kv > kMostHeads) return fail(s, RSTR_E_INVALID, "head counts must lie between 0 and 65536");
  if (rotary_dim < 0 || rotary_dim > hd || rotary_dim % 16) return fail(s, RSTR_E_INVALID, "rotary dim must be a multiple of 16 up to the head dim");
  if ((q_gain || k_gain) && !(std::isfinite(eps) && eps >= 0 && std::isfinite(gain_offset)))
    return fail(s, RSTR_E_INVALID, "epsilon and gain offset must be finite and epsilon not negative");
  if (rows >= kGridGroups) return fail(s, RSTR_E_INVALID, "too many rows for one call");
  if (rows == 0) return RSTR_OK;
  const Rows kr{(void*)k, k_row, k_head}, vr{(void*)v, v_row, v_head}, qr{(void*)q, q_row, q_head}, qo{q_out, q_out_row, q_out_head};
  TRY(check_rows(s, "key", kr, size));
  TRY(check_rows(s, "value", vr, size));
  TRY(check_ints(s, "slots", slots));
  if (in_pages(pv.c, kr, rows, n_kv, size) || in_pages(pv.c, vr, rows, n_kv, size)) return fail(s, RSTR_E_INVALID, "rows lie in the layer's pages");
  if (rotary_dim > 0) {
    TRY(check_ints(s, "positions", positions));
    if (!frequencies) return fail(s, RSTR_E_INVALID, "null frequencies");
    if (!aligned(frequencies, 8)) return fail(s, RSTR_E_INVALID, "frequencies not aligned to its elements");
  }
  if (!aligned(q_gain, 4) || !aligned(k_gain, 4)) return fail(s, RSTR_E_INVALID, "gains not aligned to their elements");
  if (n_q > 0) {
    TRY(check_rows(s, "query", qr, size));
    TRY(check_rows(s, "query output", qo, size));
    if (!apart(qo, rows, n_q, hd)) return fail(s, RSTR_E_INVALID, "output rows share elements");
    if (in_pages(pv.c, qr, rows, n_q, size) || in_pages(pv.c, qo, rows, n_q, size)) return fail(s, RSTR_E_INVALID, "rows lie in the layer's pages");
    const bool same = q == q_out && (rows == 1 || q_row == q_out_row) && (n_q == 1 || q_head == q_out_head);
    if (!same && meet(qr, n_q, qo, n_q, rows, hd, size)) return fail(s, RSTR_E_INVALID, "query output overlaps other queries");
    if (meet(qo, n_q, kr, n_kv, rows, hd, size) || meet(qo, n_q, vr, n_kv, rows, hd, size))
      return fail(s, RSTR_E_INVALID, "query output overlaps the keys or values");
    if (ints_meet(slots, (int64_t)rows * 4, qo, rows, n_q, hd, size) || (rotary_dim > 0 && (ints_meet(positions, (int64_t)rows * 4, qo, rows, n_q, hd, size) ||
        ints_meet(frequencies, (int64_t)rotary_dim * 4, qo, rows, n_q, hd, size))) || ints_meet(q_gain, (int64_t)hd * 4, qo, rows, n_q, hd, size) ||
        ints_meet(k_gain, (int64_t)hd * 4, qo, rows, n_q, hd, size))
      return fail(s, RSTR_E_INVALID, "query output overlaps the call's tables");
  }
  RopeAppend a{pv.c, rows, n_q, rotary_dim, qr, qo, kr, vr, n_q > 0 ? q_gain : nullptr, k_gain, eps, gain_offset, frequencies, positions, slots};
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  pool_shared(p);
  HIPCHK(s, launch_rope_append(on_stream(s, stream), dtype, a));
  return RSTR_OK;
}

// ---------------------------------------------------------------------------
// attention
// ---------------------------------------------------------------------------
extern "C" int rstr_pool_attn_open(rstr_pool* p, int32_t n_q, int32_t max_batch, int32_t max_rows, rstr_pool_attn** out) {
  if (!p) return fail(nullptr, RSTR_E_INVALID, "null pool");
  const PoolView v = pool_view(p, 0);
  rstr_session* s = v.s;
  if (!out) return fail(s, RSTR_E_INVALID, "null output pointer");
  *out = nullptr;
  if (n_q <= 0 || n_q % v.c.n_kv) return fail(s, RSTR_E_INVALID, "query heads must be a multiple of the pool's kv heads");
  if (max_batch <= 0 || max_rows <= 0) return fail(s, RSTR_E_INVALID, "attention plan extents must be positive");
  if (n_q > kMostHeads || !pool_attn_fits(n_q, v.c.n_kv, max_batch, max_rows)) return fail(s, RSTR_E_INVALID, "attention plan has too many rows");
  std::unique_ptr<rstr_pool_attn> a(new (std::nothrow) rstr_pool_attn());
  if (!a) return fail(s, RSTR_E_OOM, "attention plan handle");
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  if (device_alloc(&a->ws, pool_attn_workspace(n_q, v.c.n_kv, v.c.hd, max_batch, max_rows)) != hipSuccess) {
    (void)hipGetLastError();
    return fail(s, RSTR_E_OOM, "attention plan workspace allocation failed");
  }
  a->p = p;
  a->n_q = n_q;
  a->batch = max_batch;
  a->rows = max_rows;
  pool_hold(p, 1);
  pool_shared(p);
  *out = a.release();
  return RSTR_OK;
}

extern "C" int rstr_pool_attn_close(rstr_pool_attn* a) {
  if (!a) return RSTR_OK;
  OnDevice dev(pool_view(a->p, 0).s->device);
  (void)hipDeviceSynchronize();
  (void)hipFree(a->ws);
  pool_hold(a->p, -1);
  delete a;
  return RSTR_OK;
}

extern "C" int rstr_pool_attn_run(rstr_pool_attn* a, int32_t layer, int32_t dtype, int32_t batch, int32_t rows, int32_t max_rows,
                                  int32_t window, float scale, const void* q, int64_t q_row, int64_t q_head, const int32_t* row_offsets,
                                  const int32_t* page_table, int32_t pages_per_seq, const int32_t* lengths, const int32_t* blocks,
                                  int32_t blocks_per_row, void* out, int64_t out_row, int64_t out_head, void* stream) {
  if (!a) return fail(nullptr, RSTR_E_INVALID, "null attention plan");
  PoolView v = pool_view(a->p, 0);
  rstr_session* s = v.s;
  if (layer < 0 || layer >= v.layers) return fail(s, RSTR_E_INVALID, "layer is outside the pool");
  v = pool_view(a->p, layer);
  const int hd = v.c.hd, n_kv = v.c.n_kv, size = elem_size(dtype);
  if (!size) return fail(s, RSTR_E_INVALID, "element type must be f32, f16 or bf16");
  if (batch < 0 || batch > a->batch) return fail(s, RSTR_E_INVALID, "batch exceeds the attention plan's");
  if (rows < 0 || rows > a->rows) return fail(s, RSTR_E_INVALID, "rows exceed the attention plan's");
  if (window < 0) return fail(s, RSTR_E_INVALID, "window must not be negative");
  if (!std::isfinite(scale)) return fail(s, RSTR_E_INVALID, "scale must be finite");
  if (batch == 0 || rows == 0) return RSTR_OK;
  if (max_rows <= 0 || max_rows > rows) return fail(s, RSTR_E_INVALID, "rows per sequence must lie between 1 and the rows");
  TRY(sequences_args(s, row_offsets, page_table, pages_per_seq, lengths));
  const Rows qr{(void*)q, q_row, q_head}, o{out, out_row, out_head};
  TRY(check_rows(s, "query", qr, size));
  TRY(check_rows(s, "output", o, size));
  if (blocks) {
    TRY(check_ints(s, "blocks", blocks));
    if (blocks_per_row <= 0) return fail(s, RSTR_E_INVALID, "blocks per row must be positive");
  }
  if (!apart(o, rows, a->n_q, hd)) return fail(s, RSTR_E_INVALID, "output rows share elements");
  if (in_pages(v.c, o, rows, a->n_q, size)) return fail(s, RSTR_E_INVALID, "output lies in the layer's pages");
  if (ranges_meet((uintptr_t)q, rows_end(qr, rows, a->n_q, hd, size), (uintptr_t)out, rows_end(o, rows, a->n_q, hd, size)))
    return fail(s, RSTR_E_INVALID, "output overlaps the queries");
  const struct { const int32_t* p; int64_t n; } ints[] = {{row_offsets, batch + (int64_t)1}, {page_table, (int64_t)batch * pages_per_seq}, {lengths, batch},
                                                           {blocks, blocks ? (int64_t)rows * n_kv * blocks_per_row : 0}};
  for (const auto& x : ints)
    if (ints_meet(x.p, x.n * 4, o, rows, a->n_q, hd, size)) return fail(s, RSTR_E_INVALID, "output overlaps the sequences' tables");
  PoolAttn k{};
  k.c = v.c;
  k.n_q = a->n_q;
  k.batch = batch;
  k.rows = rows;
  k.max_rows = max_rows;
  k.window = window;
  k.pps = pages_per_seq;
  k.top = blocks ? blocks_per_row : 0;
  k.scale = scale;
  k.q = qr;
  k.out = o;
  k.row_offsets = row_offsets;
  k.page_table = page_table;
  k.lengths = lengths;
  k.blocks = blocks;
  k.ws = a->ws;
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  HIPCHK(s, launch_pool_attn(on_stream(s, stream), dtype, k));
  return RSTR_OK;
}

// ---------------------------------------------------------------------------
// bounds of blocks
// ---------------------------------------------------------------------------
extern "C" int rstr_bounds_open(rstr_pool* p, rstr_bounds** out) {
  if (!p) return fail(nullptr, RSTR_E_INVALID, "null pool");
  const PoolView v = pool_view(p, 0);
  rstr_session* s = v.s;
  if (!out) return fail(s, RSTR_E_INVALID, "null output pointer");
  *out = nullptr;
  std::unique_ptr<rstr_bounds> b(new (std::nothrow) rstr_bounds());
  if (!b) return fail(s, RSTR_E_OOM, "block bounds handle");
  b->layer_elems = (int64_t)v.c.pages * v.c.n_kv * 2 * v.c.hd;
  const size_t bytes = (size_t)b->layer_elems * 2 * v.layers;
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  if (device_alloc((void**)&b->base, bytes) != hipSuccess) {
    (void)hipGetLastError();
    return fail(s, RSTR_E_OOM, "block bounds allocation failed");
  }
  hipError_t e = hipMemsetAsync(b->base, 0, bytes, s->stream);
  if (e == hipSuccess) e = hipStreamSynchronize(s->stream);
  if (e != hipSuccess) {
    (void)hipFree(b->base);
    HIPCHK(s, e);
  }
  b->p = p;
  pool_hold(p, 1);
  pool_shared(p);
  *out = b.release();
  return RSTR_OK;
}

extern "C" int rstr_bounds_close(rstr_bounds* b) {
  if (!b) return RSTR_OK;
  rstr_session* s = pool_view(b->p, 0).s;
  if (b->plans > 0) return fail(s, RSTR_E_STATE, "block bounds have open selections");
  OnDevice dev(s->device);
  (void)hipDeviceSynchronize();
  (void)hipFree(b->base);
  pool_hold(b->p, -1);
  delete b;
  return RSTR_OK;
}

extern "C" int rstr_bounds_device(rstr_bounds* b, int32_t layer, void** out) {
  if (!b) return fail(nullptr, RSTR_E_INVALID, "null block bounds");
  const PoolView v = pool_view(b->p, 0);
  if (!out) return fail(v.s, RSTR_E_INVALID, "null output pointer");
  *out = nullptr;
  if (layer < 0 || layer >= v.layers) return fail(v.s, RSTR_E_INVALID, "layer is outside the pool");
  *out = b->base + layer * b->layer_elems;
  return RSTR_OK;
}

extern "C" int rstr_bounds_update(rstr_bounds* b, int32_t layer, int32_t batch, int32_t rows, const int32_t* row_offsets,
                                  const int32_t* page_table, int32_t pages_per_seq, const int32_t* lengths, void* stream) {
  if (!b) return fail(nullptr, RSTR_E_INVALID, "null block bounds");
  PoolView v = pool_view(b->p, 0);
  rstr_session* s = v.s;
  if (layer < 0 || layer >= v.layers) return fail(s, RSTR_E_INVALID, "layer is outside the pool");
  if (batch < 0 || rows < 0) return fail(s, RSTR_E_INVALID, "batch and row counts must not be negative");
  if ((int64_t)rows * v.c.n_kv >= 4 * kGridGroups) return fail(s, RSTR_E_INVALID, "too many rows for one call");
  if (batch == 0 || rows == 0) return RSTR_OK;
  TRY(sequences_args(s, row_offsets, page_table, pages_per_seq, lengths));
  BoundsUpdate a{pool_view(b->p, layer).c, b->base + layer * b->layer_elems, batch, rows, pages_per_seq, row_offsets, page_table, lengths};
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  HIPCHK(s, launch_bounds_update(on_stream(s, stream), a));
  return RSTR_OK;
}

// ---------------------------------------------------------------------------
// selection of blocks
// ---------------------------------------------------------------------------
extern "C" int rstr_select_open(rstr_bounds* b, int32_t n_q, int32_t max_batch, int32_t max_rows, int32_t max_pages, rstr_select** out) {
  if (!b) return fail(nullptr, RSTR_E_INVALID, "null block bounds");
  const PoolView v = pool_view(b->p, 0);
  rstr_session* s = v.s;
  if (!out) return fail(s, RSTR_E_INVALID, "null output pointer");
  *out = nullptr;
  if (n_q <= 0 || n_q % v.c.n_kv) return fail(s, RSTR_E_INVALID, "query heads must be a multiple of the pool's kv heads");
  if (max_batch <= 0 || max_rows <= 0 || max_pages <= 0) return fail(s, RSTR_E_INVALID, "selection extents must be positive");
  if (n_q > kMostHeads || !select_fits(v.c.n_kv, max_rows, max_pages)) return fail(s, RSTR_E_INVALID, "selection has too many rows or pages");
  std::unique_ptr<rstr_select> a(new (std::nothrow) rstr_select());
  if (!a) return fail(s, RSTR_E_OOM, "selection handle");
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  if (device_alloc(&a->ws, select_workspace(v.c.n_kv, max_rows, max_pages)) != hipSuccess) {
    (void)hipGetLastError();
    return fail(s, RSTR_E_OOM, "selection workspace allocation failed");
  }
  a->b = b;
  a->n_q = n_q;
  a->batch = max_batch;
  a->rows = max_rows;
  a->blocks = max_pages;
  b->plans++;
  *out = a.release();
  return RSTR_OK;
}

extern "C" int rstr_select_close(rstr_select* a) {
  if (!a) return RSTR_OK;
  OnDevice dev(pool_view(a->b->p, 0).s->device);
  (void)hipDeviceSynchronize();
  (void)hipFree(a->ws);
  a->b->plans--;
  delete a;
  return RSTR_OK;
}

extern "C" int rstr_select_run(rstr_select* a, int32_t layer, int32_t dtype, int32_t batch, int32_t rows, const void* q, int64_t q_row,
                               int64_t q_head, const int32_t* row_offsets, const int32_t* page_table, int32_t pages_per_seq,
                               const int32_t* lengths, int32_t blocks_per_row, int32_t first, int32_t last, int32_t* blocks, void* stream) {
  if (!a) return fail(nullptr, RSTR_E_INVALID, "null selection handle");
  const PoolView v = pool_view(a->b->p, 0);
  rstr_session* s = v.s;
  if (layer < 0 || layer >= v.layers) return fail(s, RSTR_E_INVALID, "layer is outside the pool");
  const int size = elem_size(dtype);
  if (!size) return fail(s, RSTR_E_INVALID, "element type must be f32, f16 or bf16");
  if (batch < 0 || batch > a->batch) return fail(s, RSTR_E_INVALID, "batch exceeds the selection's");
  if (rows < 0 || rows > a->rows) return fail(s, RSTR_E_INVALID, "rows exceed the selection's");
  if (blocks_per_row <= 0) return fail(s, RSTR_E_INVALID, "blocks per row must be positive");
  if (first < 0 || last < 1 || (int64_t)first + last > blocks_per_row)
    return fail(s, RSTR_E_INVALID, "the first blocks and the last, one at least, must fit in the list");
  if (batch == 0 || rows == 0) return RSTR_OK;
  if (pages_per_seq > a->blocks) return fail(s, RSTR_E_INVALID, "page table is wider than the selection's");
  TRY(sequences_args(s, row_offsets, page_table, pages_per_seq, lengths));
  const Rows qr{(void*)q, q_row, q_head};
  TRY(check_rows(s, "query", qr, size));
  TRY(check_ints(s, "blocks", blocks));
  const size_t n = (size_t)rows * v.c.n_kv * blocks_per_row * 4;
  const struct { const void* p; size_t n; } in[] = {{row_offsets, (size_t)batch * 4 + 4}, {page_table, (size_t)batch * pages_per_seq * 4}, {lengths, (size_t)batch * 4}};
  for (const auto& x : in)
    if (ranges_meet(x.p, x.n, blocks, n)) return fail(s, RSTR_E_INVALID, "blocks overlap the sequences' tables");
  if (ranges_meet(a->b->base, (size_t)a->b->layer_elems * 2 * v.layers, blocks, n)) return fail(s, RSTR_E_INVALID, "blocks overlap the bounds");
  if (ints_meet(blocks, (int64_t)n, qr, rows, a->n_q, v.c.hd, size)) return fail(s, RSTR_E_INVALID, "blocks overlap the queries");
  BlockSelect k{a->b->base + layer * a->b->layer_elems, v.c.n_kv, v.c.hd, v.c.page_size, v.c.pages, a->n_q, batch, rows, pages_per_seq,
                blocks_per_row, first, last, qr, row_offsets, page_table, lengths, blocks, a->ws,
                select_stride(a->blocks)};
  OnDevice dev(s->device);
  HIPCHK(s, dev.e);
  HIPCHK(s, launch_block_select(on_stream(s, stream), dtype, k));
  return RSTR_OK;
}
