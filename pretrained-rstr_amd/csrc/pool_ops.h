// pool_ops.h -- launch interface of the operators on device arrays over the fp16 page pool: appends with the
// position rotation, attention of ragged query rows, and the selection of blocks that it may be limited to.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kv4.h"
#include "pool_line.h"

struct rstr_pool;
struct rstr_session;

namespace rstr {

// One layer of a pool: fp16 [page][page_size][n_kv][hd], keys and values.
struct PoolLayer {
  uint16_t *k, *v;
  int n_kv, hd, page_size, pages;
};
// What the operators need of a pool; k and v are those of `layer` (which exists).
struct PoolView {
  rstr_session* s;
  int layers;
  PoolLayer c;
};
PoolView pool_view(const rstr_pool* p, int layer);
// Handles that read the pool: one more, or one less.  A pool with some does not close.
void pool_hold(rstr_pool* p, int by);
// Work on the pool may be queued on any stream from now on.
void pool_shared(rstr_pool* p);

struct RopeAppend {
  PoolLayer c;
  int rows, n_q, rot;  // rot: dims that are rotated, 0: none
  Rows q, q_out, k, v;
  const float *q_gain, *k_gain;  // null: no norm
  float eps, gain_offset;
  const double* freqs;
  const int32_t *positions, *slots;
};
hipError_t launch_rope_append(hipStream_t st, int dtype, const RopeAppend& a);

struct PoolAttn {
  PoolLayer c;
  int n_q, batch, rows, max_rows, window, pps, top;
  float scale;
  Rows q, out;
  const int32_t *row_offsets, *page_table, *lengths;
  const int32_t* blocks;  // [rows][n_kv][top], or null: all blocks
  void* ws;
};
// Bytes of workspace that every call of up to `rows` query rows and `batch` sequences can need.
size_t pool_attn_workspace(int n_q, int n_kv, int hd, int batch, int rows);
hipError_t launch_pool_attn(hipStream_t st, int dtype, const PoolAttn& a);

// Bounds of one layer's blocks: fp16 [page][n_kv][2][hd], the least and the greatest key element of a channel.
struct BoundsUpdate {
  PoolLayer c;
  uint16_t* bounds;
  int batch, rows, pps;
  const int32_t *row_offsets, *page_table, *lengths;
};
hipError_t launch_bounds_update(hipStream_t st, const BoundsUpdate& a);

struct BlockSelect {
  const uint16_t* bounds;
  int n_kv, hd, page_size, pages;
  int n_q, batch, rows, pps, top, first, last;
  Rows q;
  const int32_t *row_offsets, *page_table, *lengths;
  int32_t* blocks;
  void* ws;
  int64_t ws_blocks;  // scores a row and kv head in the workspace
};
size_t select_workspace(int n_kv, int rows, int blocks);
hipError_t launch_block_select(hipStream_t st, int dtype, const BlockSelect& a);

}  // namespace rstr
