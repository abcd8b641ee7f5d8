// The items that attention over the 4-bit cache makes of a call's row offsets, whatever these
// hold: their numbers stay inside the room that the host counts for them.  And the division that cuts
// them into parts, and the room for the pieces of those.
#include <cstdio>
#include <cstdlib>
#include <vector>

#include "../../pretrained-rstr_amd/csrc/kv4_line.h"

using namespace rstr;

static int checks = 0;

// The items of a call, numbered as the kernels number them.  Returns whether it has any.
static bool call(const std::vector<int32_t>& ro, int rows, int n_q, int n_kv, int cols) {
  const int batch = (int)ro.size() - 1;
  std::vector<int32_t> lens(batch, 100);
  const Lines L{ro.data(), lens.data(), rows, n_kv, n_q / n_kv, 0, cols, 1000, 6, false};
  int64_t items = 0, taken = 0;
  bool ordered = true;
  for (int b = 0; b < batch; b++) {
    const Seq s = sequence(L, b);
    ordered = ordered && s.ordered;
    items += (int64_t)n_kv * s.nct;
    taken += s.m;
    if (s.r0 < 0 || s.m < 0 || s.r0 + s.m > rows) { printf("rows %d + %d of %d\n", s.r0, s.m, rows); exit(1); }
  }
  checks++;
  if (!ordered) return false;
  const int64_t room = attn_items(n_q, n_kv, batch, rows, cols);
  if (items > room || taken > rows) {
    printf("batch %d rows %d heads %d/%d cols %d: %lld items in room for %lld, %lld rows\n", batch, rows, n_q, n_kv, cols,
           (long long)items, (long long)room, (long long)taken);
    exit(1);
  }
  return true;
}

// Quotients up to 2^49 from reciprocals as far off as an estimate may be.
static void quotients() {
  const auto random = [](int bits) { return (int64_t)((((uint64_t)rand() << 31 | (uint64_t)rand()) << 2 | (rand() & 3)) >> (64 - bits)); };
  for (int i = 0; i < 2000000; i++) {
    const int bits = 1 + rand() % 49, of = rand() % (52 - bits);
    const int64_t b = 1 + random(of + 1) % ((int64_t)1 << of), q = random(bits);
    const int64_t least = q * b, a = i % 3 == 0 ? least : i % 3 == 1 ? least + b - 1 : least + random(50) % b;
    const double off = (rand() % 2001 - 1000) / 1000.0 * 0x1p-22;
    const int64_t got = quotient_from(a, b, 1.0 / (double)b * (1.0 + off));
    checks++;
    if (got != a / b) {
      printf("%lld / %lld: %lld, not %lld\n", (long long)a, (long long)b, (long long)got, (long long)(a / b));
      exit(1);
    }
  }
}

// The room for pieces covers every form that a call within a plan may take, and is no more than the
// largest of them.
static void pieces() {
  for (int cu : {1, 64, 256, 304})
    for (int hd : {64, 128, 256})
      for (int64_t plan : {1, 4, 16, 17, 63, 64, 65, 100000}) {
        const int64_t room = piece_columns(hd, plan, cu);
        int64_t used = 0;
        for (int64_t call = 1; call <= plan; call += plan > 200 ? 997 : 1) {  // columns of its longest sequence
          const auto form = [&](int64_t workers, int cols) {
            checks++;
            if (2 * workers * cols > used) used = 2 * workers * cols;
          };
          if (hd == 256 || call <= kOneTile) form(attn_workers(hd, 1, cu), 16);
          else form(attn_workers(hd, 2, cu), 32);
          if (hd == 128 && call >= kManyColumns) form(prompt_workers(cu), 32 * kPromptWaves);
        }
        if (used != room) { printf("head dim %d, %lld columns: %lld for %lld\n", hd, (long long)plan, (long long)room, (long long)used); exit(1); }
      }
}

int main() {
  srand(1);
  quotients();
  pieces();
  const int heads[][2] = {{1, 1}, {32, 8}, {8, 8}, {24, 1}, {4, 1}};
  for (const auto& h : heads)
    for (int cols : {16, 32, 256}) {
      for (int rows : {1, 2, 33, 4096}) {
        for (int batch : {1, 2, 3, 64, 65, 200, 4096}) {
          std::vector<int32_t> ro(batch + 1), even(batch + 1);
          for (int b = 0; b <= batch; b++) ro[b] = b % 2 ? rows : 0;  // over and over the same rows
          if (call(ro, rows, h[0], h[1], cols) != (batch == 1)) { printf("offsets that decrease were taken\n"); return 1; }
          for (int b = 0; b <= batch; b++) even[b] = (int32_t)((int64_t)rows * b / batch);
          if (!call(even, rows, h[0], h[1], cols)) { printf("ordered offsets were refused\n"); return 1; }
          for (int i = 0; i < 20; i++) {
            // an ordered line, beginning before the array and ending behind it, with one place disturbed
            int64_t at = rand() % 5 - 2;
            for (int b = 0; b <= batch; b++) {
              ro[b] = at > 0x7FFFFFFF ? 0x7FFFFFFF : (int32_t)at;
              at += i % 4 == 0 ? rand() % 3 : i % 4 == 1 ? rand() % (2 * rows + 1) : i % 4 == 2 ? (rand() % 8 == 0) * rows : (int64_t)rand() * 2;
            }
            if (!call(ro, rows, h[0], h[1], cols)) { printf("ordered offsets were refused\n"); return 1; }
            ro[rand() % (batch + 1)] = rand() % 2 ? -(int32_t)0x7FFFFFFF - 1 : rand() % (rows + 1);
            call(ro, rows, h[0], h[1], cols);
          }
        }
      }
    }
  printf("ok %d\n", checks);
  return 0;
}
