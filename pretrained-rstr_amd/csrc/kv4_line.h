// kv4_line.h -- the line of work of attention over the 4-bit cache: the items that
// the sequences of a call are and how many there can be.  Plain arithmetic, the same on
// the device and on the host.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace rstr {

constexpr int kTile = 32;

__host__ __device__ inline int at_least(int v, int lo) { return v > lo ? v : lo; }
__host__ __device__ inline int at_most(int v, int hi) { return v < hi ? v : hi; }

// a / b for 0 <= a < 2^52 and b > 0, from an estimate r of 1 / b within 2^-20 of it: two Newton steps
// leave it within 2^-52 of itself and a step of its rounding, so that a * r is off by less than 1 where the quotient is below 2^50.
__host__ __device__ inline int64_t quotient_from(int64_t a, int64_t b, double r) {
  const double d = (double)b;
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  r = __builtin_fma(__builtin_fma(-d, r, 1.0), r, r);
  const int64_t q = (int64_t)((double)a * r), rest = a - q * b;
  return rest < 0 ? q - 1 : rest >= b ? q + 1 : q;
}

// The sequences of a call, as every wave sees them.
struct Lines {
  const int32_t *ro, *lens;
  int rows, n_kv, group, window, cols;  // cols: of a column tile
  int cap;                              // tokens that a page table row can hold
  int start;                            // what beginning an item costs, in tiles
  bool whole;                           // one unit an item
  __host__ __device__ inline int per_item(int tiles) const { return whole ? 1 : tiles + start; }
  // tokens that are there of a sequence of `len`: its length gives its rows' positions, the table its end
  __host__ __device__ inline int held(int len) const { return at_most(len, cap); }
};
struct Seq {
  int r0, m, len, lo, tiles, nct;
  bool ordered;  // its rows do not begin behind their end
  int64_t units;
};
// Rows of sequences are apart where every sequence is ordered; a call in which one is not
// has no items (what room they take follows from the rows all together).
__host__ __device__ inline Seq sequence(const Lines& L, int b) {
  Seq s;
  const int begin = L.ro[b], end = L.ro[b + 1];
  s.ordered = begin <= end;
  s.r0 = at_most(at_least(begin, 0), L.rows);
  s.m = at_least(at_most(at_least(end, 0), L.rows) - s.r0, 0);
  s.len = at_least(L.lens[b], 0);
  const int64_t lo = L.window > 0 ? (int64_t)s.len - s.m + 1 - L.window : 0;
  s.lo = lo > 0 ? (int)lo / kTile : 0;  // first tile
  s.tiles = at_least((int)(((int64_t)L.held(s.len) + kTile - 1) / kTile) - s.lo, 0);
  s.nct = (int)(((int64_t)s.m * L.group + L.cols - 1) / L.cols);
  s.units = (int64_t)L.n_kv * s.nct * L.per_item(s.tiles);
  return s;
}

// Items of a call whose sequences are ordered, at most: column tiles that are full, and one a
// sequence that is not.
__host__ __device__ inline int64_t attn_items(int n_q, int n_kv, int batch, int rows, int cols) {
  return n_kv * ((int64_t)rows * (n_q / n_kv) / cols + at_most(batch, rows));
}

// Waves a SIMD that the registers of a form leave room for (head dim 64, one tile of columns, fp16 and bf16: four would
// fit; not tried).  (NT = 1 with two waves and rings of four tiles: 84 us for 128 sequences of one fp16 row, 80 with
// three, and 55 for 51 of three long ones, with a merge of fewer pieces that is as much shorter.)
constexpr int attn_waves(int hd, int nt) { return hd == 256 ? 1 : nt == 1 ? 3 : 2; }
constexpr int kPromptWaves = 8;   // of a workgroup that shares a tile's expansion, 32 columns each
constexpr int kOneTile = 16;      // columns a sequence up to which items have one tile of columns, above it two
constexpr int kManyColumns = 64;  // columns a sequence from which waves may share a tile's expansion

// Workers of a call, at most: waves of a form, workgroups of a prompt.
inline int64_t attn_workers(int hd, int nt, int compute_units) { return (int64_t)compute_units * 4 * attn_waves(hd, nt); }
inline int64_t prompt_workers(int compute_units) { return (int64_t)compute_units * (8 / kPromptWaves); }

// Columns of the pieces, two a worker, that calls of up to `columns` query columns of a kv head leave, at most.
inline int64_t piece_columns(int hd, int64_t columns, int compute_units) {
  int64_t n = attn_workers(hd, 1, compute_units) * 16;
  if (hd != 256 && columns > kOneTile) {
    const int64_t two = attn_workers(hd, 2, compute_units) * 32;
    n = n > two ? n : two;
  }
  if (hd == 128 && columns >= kManyColumns) {
    const int64_t prompt = prompt_workers(compute_units) * 32 * kPromptWaves;
    n = n > prompt ? n : prompt;
  }
  return 2 * n;
}

}  // namespace rstr
