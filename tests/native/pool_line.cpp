// How calls over the fp16 page pool are cut: every form's pieces fit the workspace that a plan opens with, the parts of
// an item cover it once and are joined from where they were left, grids hold the launches, and tokens are found in the pages that
// a wave has looked up.
#include <cstdio>
#include <cstdlib>
#include <set>
#include <vector>

#include "../../pretrained-rstr_amd/csrc/pool_line.h"

using namespace rstr;

static long checks = 0;
#define CHECK(ok, ...)                                      \
  do {                                                      \
    checks++;                                               \
    if (!(ok)) {                                            \
      printf("line %d: %s: ", __LINE__, #ok);               \
      printf(__VA_ARGS__);                                  \
      printf("\n");                                         \
      exit(1);                                              \
    }                                                       \
  } while (0)

static const size_t kBegun = 20;  // bytes that the kernels keep of an item that begins
static const int kHeads[][2] = {{32, 8}, {16, 8}, {4, 1}, {8, 2}, {8, 8}, {24, 1}, {40, 4}, {3, 3}};
static int log_int(int lo, int hi) {  // spread over the logarithm
  double x = lo;
  for (int i = 0; i < 40 && x < hi; i++)
    if (rand() % 40 >= 40 * (i + 1) / 41) x *= 1.0 + (rand() % 1000) / 700.0;
  return x < hi ? (int)x : hi;
}

// ---- forms and the workspace ----
static void call_of(int cu, int hd, int terms, const int* h, int plan_batch, int plan_rows) {
  const size_t plan = pool_attn_room(kBegun, h[0], h[1], hd, plan_batch, plan_rows, cu);
  const int batch = 1 + rand() % plan_batch, rows = 1 + rand() % plan_rows, most = 1 + rand() % rows;
  const int page = 4 * (1 + rand() % 64), pps = log_int(1, 1 << 20), cap = token_cap(pps, page);
  const PoolForm f = pool_form(hd, terms, h[0], h[1], batch, rows, most, cap, cu);
  CHECK(f.items > 0 && f.workers > 0 && f.workers < (1 << 30), "%lld items %lld workers", (long long)f.items, (long long)f.workers);
  CHECK(f.cols == 16 * f.nt * (f.prompt ? kShareWaves : 1) && f.nt <= 2 && (f.prompt || f.workers % 4 == 0), "cols %d", f.cols);
  CHECK((uint64_t)f.workers * (f.prompt ? 64 * kShareWaves : 64) < 1ull << 32 && (uint64_t)f.items * 256 < 1ull << 32, "grid");
  if (!f.whole) {  // (whole items leave no pieces)
    const PoolRoom r = pool_room(kBegun, f.items, 2 * f.workers * f.cols, hd);
    CHECK(r.end <= plan && r.begun < r.ml && r.ml < r.acc, "%zu of %zu bytes: cu %d hd %d heads %d/%d batch %d of %d rows %d of %d most %d cap %d", r.end, plan, cu,
          hd, h[0], h[1], batch, plan_batch, rows, plan_rows, most, cap);
  }
  // lists
  const int top = log_int(1, 1 << 20);
  const Cut c = listed_cut(h[0], h[1], hd, rows, top, pps, page, cu);
  CHECK(c.items == (int64_t)rows * h[1] * ((h[0] / h[1] + 15) / 16) && c.parts >= 1 && c.tiles >= 1, "cut");
  CHECK((uint64_t)c.groups() * 64 * (c.waves > 1 ? c.waves : 4) < 1ull << 32, "%lld groups", (long long)c.groups());
  int64_t entries = top < pps ? top : pps;
  if (entries > 0x7FFFFFFF / page + 1) entries = 0x7FFFFFFF / page + 1;  // up to the block of the last position
  const int64_t tiles = (entries * page + kTile - 1) / kTile;
  CHECK((int64_t)c.parts * c.waves * c.tiles >= tiles, "%d parts of %d waves of %d tiles for %lld", c.parts, c.waves, c.tiles, (long long)tiles);
  if (c.parts > 1) {
    const PoolRoom r = pool_room(kBegun, 0, c.items * c.parts * 16, hd);
    CHECK(r.end <= plan, "lists: %zu of %zu bytes", r.end, plan);
  }
}
static void forms() {
  for (int cu : {1, 64, 256, 304})
    for (int hd : {64, 128, 256})
      for (int terms : {1, 2})
        for (const auto& h : kHeads)
          for (int i = 0; i < 250; i++) {
            const int batch = log_int(1, 4096), rows = log_int(1, 100000);
            if (pool_attn_fits(h[0], h[1], batch, rows)) call_of(cu, hd, terms, h, batch, rows);
          }
}

// ---- parts of items ----
static void parts() {
  for (int i = 0; i < 3000; i++) {
    const int* h = kHeads[rand() % 8];
    const int n_q = h[0], n_kv = h[1], hd = 64 << rand() % 3, terms = 1 + rand() % 2, cu = rand() % 2 ? 256 : 1 + rand() % 20;
    const int batch = 1 + rand() % 70, page = 4 * (1 + rand() % 40), window = rand() % 3 ? 0 : 1 + rand() % 500;
    std::vector<int32_t> ro(batch + 1), lens(batch);
    int most = 0;
    for (int b = 0; b < batch; b++) {
      const int m = rand() % 4 == 0 ? 0 : log_int(1, i % 3 == 0 ? 900 : 6);
      ro[b + 1] = ro[b] + m;
      lens[b] = rand() % 9 == 0 ? rand() % 3 : log_int(1, 4000);
      most = m > most ? m : most;
    }
    const int rows = ro[batch];
    if (rows == 0) continue;
    const int cap = token_cap(log_int(1, 300), page);
    const PoolForm f = pool_form(hd, terms, n_q, n_kv, batch, rows, 1 + rand() % most, cap, cu);
    const int start = f.prompt ? kPromptStart : kStart, least = f.whole ? 1 : f.prompt ? kPromptLeast : kLeast;
    const Lines L{ro.data(), lens.data(), rows, n_kv, n_q / n_kv, window, f.cols, cap, start, f.whole};
    struct Item { int64_t at, units; int tiles; };
    std::vector<Item> items;
    int64_t total = 0;
    for (int b = 0; b < batch; b++) {
      const Seq s = sequence(L, b);
      for (int k = 0; k < n_kv * s.nct; k++) items.push_back({total, L.per_item(s.tiles), s.tiles}), total += L.per_item(s.tiles);
    }
    CHECK((int64_t)items.size() <= f.items, "%zu items in room for %lld", items.size(), (long long)f.items);
    int64_t part = (total + f.workers - 1) / f.workers;
    if (part < least) part = least;
    CHECK(part * f.workers >= total, "%lld parts of %lld", (long long)f.workers, (long long)part);
    if (f.whole) { CHECK(part == 1, "whole items of %lld units a wave", (long long)part); continue; }
    std::set<int64_t> places;
    for (const Item& it : items) {
      const int64_t first = it.at / part, last = (it.at + it.units - 1) / part;
      const int n = first == last ? 0 : pieces_to(last, (int)first);  // as the wave that begins it says
      int64_t seen = 0;
      for (int64_t w = first; w <= last; w++) {
        const int64_t u = it.at > w * part ? it.at : w * part, end = it.at + it.units < (w + 1) * part ? it.at + it.units : (w + 1) * part;
        const int at = (int)(u - it.at), cnt = (int)(end - u), t0 = at > start ? at - start : 0, t1 = at + cnt > start ? at + cnt - start : 0;
        CHECK(t0 == seen && t1 <= it.tiles, "tiles %d to %d behind %lld", t0, t1, (long long)seen);
        seen = t1;
        if (n == 0) continue;
        const int64_t place = piece_place((int)w, w == first), join = w == first ? piece_place((int)first, true) : piece_place((int)first, false) + 2 * (w - first);
        CHECK(place == join && place < 2 * f.workers && places.insert(place).second, "piece %lld", (long long)place);
      }
      CHECK(seen == it.tiles && (n == 0 || n == last - first + 1), "an item's tiles: %lld of %d", (long long)seen, it.tiles);
    }
  }
}

// ---- places of tokens ----
static void places() {
  for (int i = 0; i < 4000; i++) {
    const int ps = i < 512 ? 4 * (1 + i) : 4 * log_int(1, 1 << 20), step_e = kTile / ps, step_off = kTile - step_e * ps;
    int64_t t0 = rand() % 2 ? rand() % 1000 : (int64_t)(rand() % (1 << 26));
    if (t0 > 0x7FFFFFC0 / kTile - 200) t0 = 0x7FFFFFC0 / kTile - 200;
    Place tok[32], first = place_of((uint32_t)t0 * kTile, ps);
    for (int j = 0; j < 32; j++) tok[j] = place_of((uint32_t)t0 * kTile + j, ps);
    int e0 = first.entry;
    for (int64_t t = t0; t < t0 + 180; t++) {
      if (entries_to_end(first, e0, ps) >= 64) e0 = first.entry;
      for (int j = 0; j < 32; j++) {
        CHECK((int64_t)tok[j].entry * ps + tok[j].off == t * kTile + j && tok[j].off >= 0 && tok[j].off < ps, "token %lld in pages of %d", (long long)(t * kTile + j), ps);
        CHECK(tok[j].entry - e0 >= 0 && tok[j].entry - e0 < 64, "entry %d of those from %d on", tok[j].entry, e0);
        if (j % 4) CHECK(tok[j].entry == tok[j - 1].entry && tok[j].off == tok[j - 1].off + 1, "four tokens of two pages");
      }
      for (Place& x : tok) forward(x, step_e, step_off, ps);
      forward(first, step_e, step_off, ps);
    }
    const int se = kStep / ps, so = kStep - se * ps;
    Place four = place_of((uint32_t)t0 * kTile + 4 * (i % 16), ps);
    for (int k = 0; k < 90; k++, forward(four, se, so, ps))
      CHECK((int64_t)four.entry * ps + four.off == t0 * kTile + 4 * (i % 16) + (int64_t)k * kStep && four.off % 4 == 0, "step %d in pages of %d", k, ps);
  }
  CHECK(token_cap(0x7FFFFFFF, 0x7FFFFFFC) == 0x7FFFFFC0 && token_cap(1 << 27, 16) == 0x7FFFFFC0 && token_cap(5, 16) == 80, "cap");
}

// ---- selections ----
static void selections() {
  for (int i = 0; i < 200000; i++) {
    const int n_kv = kHeads[rand() % 8][1], rows = log_int(1, 1 << 22), pages = i % 50 == 0 ? 0x7FFFFFFF - rand() % 70 : log_int(1, 1 << 30);
    if (!select_fits(n_kv, rows, pages)) continue;
    const int64_t stride = select_stride(pages), rh = (int64_t)rows * n_kv;
    CHECK(stride % 16 == 0 && stride >= pages && stride < (int64_t)pages + 16, "stride of %d", pages);
    for (int cu : {1, 256})
      for (int blocks : {pages, 1 + rand() % pages}) {
        const ScoreCut c = score_cut(rh, blocks, cu);
        CHECK((c.per == 32 || c.per == 64) && (int64_t)c.per * c.chunks >= blocks && (int64_t)c.per * (c.chunks - 1) < blocks, "%d waves of %d for %d", c.chunks, c.per, blocks);
        CHECK((uint64_t)((rh * c.chunks + 3) / 4) * 256 < 1ull << 32, "grid of scores");
        CHECK((uint64_t)rh * (blocks <= 1024 ? 256 : 1024) < 1ull << 32, "grid of lists: %lld of %d", (long long)rh, blocks);
      }
  }
  CHECK(!select_fits(1, 1, 0x7FFFFFFF) && !select_fits(8, 1 << 21, 1) && select_fits(8, 1 << 20, 32), "limits");
}

int main() {
  srand(1);
  forms();
  parts();
  places();
  selections();
  printf("ok %ld\n", checks);
  return 0;
}
