// pool_line.h -- how calls of attention over the fp16 page pool are cut: the forms that they take, the parts of
// their items, the room that pieces need, and the places of tokens in pages.  Plain arithmetic, the same on the device and on
// the host.
#pragma once
#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include "kv4_line.h"

namespace rstr {

constexpr int kStart = 4;        // what beginning an item costs, in tiles
constexpr int kPromptStart = 8;  // the same where waves share tiles
constexpr int kStep = 64;        // tokens at a time there
constexpr int kShareWaves = 8;   // two a SIMD, with half its registers each

constexpr int pool_waves(int hd) { return hd == 256 ? 1 : 2; }  // a SIMD
// Tiles of 16 columns a wave that shares tiles of tokens: what these registers hold.  Four waves of two tiles instead: 167 us for 98 at D = 256, 556 for 449 in
// fp32 at D = 128 (1900 rows at 5000 tokens, 4 and 32 heads).
constexpr int prompt_tiles(int hd, int terms) { return hd * terms >= 256 ? 1 : 2; }

// ---- forms ---------------------------------------------------------------------------
// Tiles of an item that one wave does, without a merge, and twice as many where items occupy half the card: 4 instead costs 34 us for 28 with
// 128 sequences of 250 tokens, 1 instead 14.0 for 11.8 with one of 128; 16 always saves 55 -> 47 with 128 of 500, but costs 37 for 25 with 32.
constexpr int kWhole = 8;
// Tiles a wave takes at least.  1: 17.0 -> 15.6 us for one sequence of 1000 tokens, but 19.3 -> 23.7 for one of 8000; 4: 14.3 -> 18.2 for 300 tokens.
constexpr int kLeast = 2;
// And a workgroup of k_pool_prompt: 8 instead costs 22.8 us for 19.4 with 400 rows of 500 tokens, 16 28.7; all are alike from 2000 tokens on.
constexpr int kPromptLeast = 4;
// Columns a sequence from which waves share tiles.  Both sides, in us, of one sequence of 4000 tokens and of eight of 2000: D = 128 f16
// 25.0 | 26.3 and 39.6 | 38.2 with 32 columns, 31.6 | 26.4 and 46.0 | 41.0 with 64; D = 64 17.2 | 19.4 and 24.4 | 20.9 with 64;
// D = 256 f16 23.4 | 27.9 and 32.0 | 29.9 with 64, 37.7 | 34.4 with 512; D = 256 fp32 40.9 | 46.8 with 128, 38.3 | 44.7 with 512, and with
// 3600 at 5000 tokens 307 | 152.
constexpr int many_columns(int hd, int terms) { return hd < 256 ? 64 : terms == 1 ? 128 : 1024; }
// 16-bit queries: columns a sequence from which items have two tiles of 16 columns, where tables are long enough.  Two tiles | one, in us, 8 rows
// of four heads a kv head: 24.4 | 27.0 for one sequence of 4000 tokens, 36.6 | 43.1 for 16 of 1000, but 67.6 | 59.6 for 128 of 300.  In fp32 one tile is
// never slower (45.9 | 44.0 and 82.3 | 61.5).
constexpr int kTwoTiles = 17, kTwoTilesFrom = 512;

// Tokens that a table row holds for a call: 2^31 - 64 at most, so that the tile behind a position has one too.
__host__ __device__ inline int token_cap(int pps, int page_size) {
  const int64_t n = (int64_t)pps * page_size;
  return n < 0x7FFFFFC0 ? (int)n : 0x7FFFFFC0;
}

// The form of a call over all tokens.
struct PoolForm {
  bool prompt, whole;  // waves share tiles; one unit an item, no join
  int nt, cols;        // tiles of 16 columns a wave; columns an item
  int64_t items, workers;  // items at most; waves, or workgroups that share
};
inline PoolForm pool_form(int hd, int terms, int n_q, int n_kv, int batch, int rows, int max_rows, int cap, int cu) {
  const int64_t group = n_q / n_kv, tiles = ((int64_t)cap + kTile - 1) / kTile;
  const int64_t many = many_columns(hd, terms);
  PoolForm f;
  f.prompt = max_rows * group >= many && rows * group >= many * batch;
  f.nt = f.prompt ? prompt_tiles(hd, terms) : hd != 256 && terms == 1 && max_rows * group >= kTwoTiles && cap > kTwoTilesFrom ? 2 : 1;
  f.cols = 16 * f.nt * (f.prompt ? kShareWaves : 1);
  f.items = attn_items(n_q, n_kv, batch, rows, f.cols);
  const int64_t most = f.prompt ? cu : (int64_t)cu * 4 * pool_waves(hd);
  f.whole = !f.prompt && (tiles <= kWhole || (tiles <= 2 * kWhole && 2 * f.items >= most));
  const int start = f.prompt ? kPromptStart : kStart, least = f.prompt ? kPromptLeast : kLeast;
  const int64_t want = f.whole ? f.items : (f.items * (tiles + start) + least - 1) / least;
  f.workers = f.whole || want < most ? want : most;
  if (!f.prompt) f.workers = (f.workers + 3) / 4 * 4;
  return f;
}

// How the items of lists of blocks are shared out: waves an item, workgroups an item, tiles a wave.
struct Cut {
  int64_t items;
  int waves, parts, tiles;
  int64_t groups() const { return waves > 1 ? items * parts : (items + 3) / 4; }
};
constexpr int listed_waves(int hd) { return hd == 256 ? 4 : 8; }
// A wave an item where these occupy a quarter of the card, and where a list is short (selection and attention together, 100 rows of 8 kv heads: 114 us with
// a wave an item, 134 with a workgroup, for lists of 64 blocks of 16 tokens, 55 and 72 for 16; 60 rows alike); else a workgroup an item, and where
// a wave would have more than kListedTiles tiles several (16 instead of 2: 25 us for 12 + 4 with the join, one row, lists of 128 blocks).
constexpr int kListedTiles = 2;
inline Cut listed_cut(int n_q, int n_kv, int hd, int rows, int top, int pps, int page_size, int cu) {
  // (a row counts no more entries than blocks up to its own)
  int64_t entries = top < pps ? top : pps;
  if (entries > 0x7FFFFFFF / page_size + 1) entries = 0x7FFFFFFF / page_size + 1;
  const int64_t tiles = (entries * page_size + kTile - 1) / kTile, most = (int64_t)cu * 4 * pool_waves(hd);
  const int group = n_q / n_kv, ncts = (group + 15) / 16;
  Cut c{(int64_t)rows * n_kv * ncts, 1, 1, (int)tiles};
  if (tiles <= kLeast || 4 * c.items >= most) return c;
  c.waves = listed_waves(hd);
  const int64_t fit = most / (c.items * c.waves), room = fit > 1 ? fit : 1;
  const int64_t want = (tiles + (int64_t)c.waves * kListedTiles - 1) / (c.waves * kListedTiles), parts = want < room ? want : room;
  c.tiles = (int)((tiles + parts * c.waves - 1) / (parts * c.waves));
  c.parts = (int)((tiles + (int64_t)c.tiles * c.waves - 1) / ((int64_t)c.tiles * c.waves));
  return c;
}

// ---- the workspace ---------------------------------------------------------------------
// Bytes from its beginning of what the parts of items leave: a word (the number of items), `begun` bytes an item that begins,
// four floats and hd of them a column of a piece.
struct PoolRoom {
  size_t begun, ml, acc, end;
};
inline PoolRoom pool_room(size_t begun_bytes, int64_t items, int64_t columns, int hd) {
  PoolRoom r;
  r.begun = 256;
  r.ml = r.begun + align256(begun_bytes * items);
  r.acc = r.ml + align256(16 * columns);
  r.end = r.acc + sizeof(float) * columns * hd;
  return r;
}
// Room for every call of up to `rows` query rows and `batch` sequences: two pieces a worker, of 32 columns at most where each is a wave; a
// list's parts are no more than these.
inline size_t pool_attn_room(size_t begun_bytes, int n_q, int n_kv, int hd, int batch, int rows, int cu) {
  const int64_t waves = (int64_t)cu * 4 * pool_waves(hd) * 32, prompt = (int64_t)cu * 16 * prompt_tiles(hd, 1) * kShareWaves;
  return pool_room(begun_bytes, attn_items(n_q, n_kv, batch, rows, 16), 2 * (waves > prompt ? waves : prompt) + 64, hd).end;
}

// A grid holds fewer than 2^32 threads: of a merge with 256 an item (those with more have few items), and of a wave
// an item of a list.
inline bool pool_attn_fits(int n_q, int n_kv, int batch, int rows) {
  const int64_t dense = attn_items(n_q, n_kv, batch, rows, 16), listed = (int64_t)rows * n_kv * ((n_q / n_kv + 15) / 16);
  return (int64_t)rows * n_q <= 0x7FFFF000 && dense < (1 << 24) && listed < (1 << 24);
}

// ---- selections of blocks -------------------------------------------------------------------
inline int64_t select_stride(int blocks) { return ((int64_t)blocks + 15) / 16 * 16; }  // scores a row and kv head has room for, for tables of that many pages
constexpr int kScoreBlocks = 32;  // blocks that a wave scores, at least
inline bool select_fits(int n_kv, int rows, int blocks) {  // grids hold it
  return (int64_t)rows * n_kv < (1 << 24) && (double)rows * n_kv * (((int64_t)blocks + kScoreBlocks - 1) / kScoreBlocks) < (double)(1 << 26);
}
// Blocks a wave, and waves a row and kv head (`rh` of these).  Twice as many blocks a wave where these waves fill the card (selection and attention of 32
// sequences of up to 1024 blocks: 74.1 us for 77.2; of one sequence of 8192 blocks 46.1 for 45.4).
struct ScoreCut {
  int per, chunks;
};
inline ScoreCut score_cut(int64_t rh, int blocks, int cu) {
  const int64_t twice = ((int64_t)blocks + 2 * kScoreBlocks - 1) / (2 * kScoreBlocks);
  const int per = rh * twice >= 16 * (int64_t)cu ? 2 * kScoreBlocks : kScoreBlocks;
  return ScoreCut{per, (int)(((int64_t)blocks + per - 1) / per)};
}

// ---- places of tokens -------------------------------------------------------------------
// A token's entry of a page table row (or of a list of blocks) and its place in that page.
struct Place {
  int entry, off;
};
__host__ __device__ inline Place place_of(uint32_t token, int page_size) {
  const int e = (int)(token / (uint32_t)page_size);
  return Place{e, (int)(token - (uint32_t)e * page_size)};
}
// `step` tokens on, from the quotient and the rest of step / page_size.
__host__ __device__ inline void forward(Place& p, int step_entries, int step_off, int page_size) {
  p.entry += step_entries;
  p.off += step_off;
  if (p.off >= page_size) p.off -= page_size, p.entry++;
}
// Entries from `from` to that of the last token of the tile that begins at `first`: from 64 on, 64 entries from `from` on do not hold it.
__host__ __device__ inline int entries_to_end(Place first, int from, int page_size) {
  return (int)((uint32_t)first.off + kTile - 1) / page_size + first.entry - from;
}

}  // namespace rstr
