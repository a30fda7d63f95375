// Randomized host test of csrc/paged.h, built with AddressSanitizer and
// UndefinedBehaviorSanitizer by tests/test_paged.py: page lookups at positions and
// with page numbers outside of their ranges touch nothing outside the table, and the
// decoding attention's split covers every tile once, gives every piece a partial slot
// of its own and lets the join find exactly those.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <limits>
#include <random>
#include <set>
#include <vector>

#include "paged.h"

using namespace vafa;

static int fails = 0;
#define CHECK(c)                                                           \
  do {                                                                     \
    if (!(c)) {                                                            \
      std::fprintf(stderr, "check failed at line %d: %s\n", __LINE__, #c); \
      ++fails;                                                             \
    }                                                                      \
  } while (0)

static void lookups(std::mt19937_64 &g) {
  const int page = g() % 2 ? 1 << (g() % 9) : 1 + (int)(g() % 300);
  const int width = (int)(g() % 9), n = 1 + (int)(g() % 4), pages = 1 + (int)(g() % 20);
  const int stride = width + (int)(g() % 3);
  std::vector<int32_t> table((size_t)(n - 1) * stride + width);  // not one entry more
  for (auto &x : table)
    x = g() % 4 ? (int32_t)(g() % pages) : (g() % 2 ? -1 - (int32_t)(g() % 5) : pages + (int32_t)(g() % 5));
  if (!table.empty()) table[g() % table.size()] = g() % 2 ? INT32_MAX : INT32_MIN;
  PageMap m{table.data(), stride, width, page, page_shift(page), pages};
  CHECK(page_shift(page) < 0 || 1 << page_shift(page) == page);
  CHECK(page_capacity(m) == (int64_t)width * page);
  std::vector<int32_t> at = {0, 1, -1, INT32_MAX, INT32_MIN, width * page - 1, width * page};
  for (int i = 0; i < 50; ++i) at.push_back((int32_t)(g() % (width * page + 10)));
  for (int b = 0; b < n; ++b)
    for (int32_t p : at) {
      if (p < 0) {
        CHECK(page_of(m, b, p, PageSlot{0, 0}) == -1);
        continue;
      }
      const PageSlot s = page_slot(m, p);
      CHECK(s.index == p / page && s.slot == p % page);
      const int32_t id = page_of(m, b, p, s);
      if (p >= width * page) {
        CHECK(id == -1);
      } else {
        const int32_t e = table[(size_t)b * stride + p / page];
        CHECK(id == (e >= 0 && e < pages ? e : -1));
      }
    }
  CHECK(clip_len(-5, 10) == 0 && clip_len(INT32_MIN, 10) == 0 && clip_len(11, 10) == 10);
  PageMap huge{nullptr, 0, INT32_MAX, INT32_MAX, -1, 1};
  CHECK(page_capacity(huge) == INT32_MAX && clip_len(INT32_MAX, page_capacity(huge)) == INT32_MAX);
  CHECK(decode_tiles(INT32_MAX, 0) == 1 << 24);
}

static void splits(std::mt19937_64 &g) {
  const int n = 1 + (int)(g() % 40);
  const int chunks = 1 + (int)(g() % (g() % 2 ? 8 : 600)), window = g() % 3 ? 0 : 1 + (int)(g() % 900);
  std::vector<int32_t> tiles(n);
  int32_t total = 0;
  for (auto &t : tiles) {
    const int32_t len = (int32_t)(g() % 4 == 0 ? 0 : g() % (1u << (1 + g() % 17)));
    t = decode_tiles(len, window);
    const int32_t seen = decode_seen(len, window);
    CHECK(seen <= len && (window == 0 || seen <= window) && (t - 1) * kDecodeTile < seen + (seen == 0) &&
          t * kDecodeTile >= seen);
    total += t;
  }
  const int32_t per = decode_per(total, chunks);
  CHECK((int64_t)per * chunks >= total);
  if (total == 0) return;
  std::vector<int> covered(total, 0);
  std::set<int64_t> slots, joined;
  // the chunks' walk
  for (int c = 0; c < chunks; ++c) {
    int64_t cur = (int64_t)c * per;
    const int64_t end = cur + per < total ? cur + per : total;
    while (cur < end) {
      int32_t t0 = 0, nt = 0;
      for (int b = 0; b < n && nt == 0; ++b) {
        if (cur < t0 + tiles[b]) nt = tiles[b];
        else t0 += tiles[b];
      }
      const int64_t stop = t0 + nt < end ? t0 + nt : end;
      for (int64_t t = cur; t < stop; ++t) ++covered[t];
      if (stop - cur < nt) {
        const int64_t s = decode_slot(c, t0, per);
        CHECK(s >= 0 && s < 2 * chunks && slots.insert(s).second);
      }
      cur = stop;
    }
  }
  for (int c : covered) CHECK(c == 1);
  // the join
  int32_t t0 = 0;
  for (int b = 0; b < n; ++b) {
    if (tiles[b] > 0) {
      const int g0 = t0 / per, g1 = (t0 + tiles[b] - 1) / per;
      if (g0 != g1)
        for (int c = g0; c <= g1; ++c) CHECK(joined.insert(decode_slot(c, t0, per)).second);
    }
    t0 += tiles[b];
  }
  CHECK(slots == joined);
}

int main(int argc, char **argv) {
  const int rounds = argc > 1 ? std::atoi(argv[1]) : 100;
  std::mt19937_64 g(argc > 2 ? std::atoll(argv[2]) : 1);
  for (int i = 0; i < rounds; ++i) {
    lookups(g);
    splits(g);
  }
  std::printf("%d failed checks\n", fails);
  return fails != 0;
}
