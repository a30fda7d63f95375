// Randomized host test of the division of paged_chunk_attn's work (csrc/paged.h), built with
// AddressSanitizer and UndefinedBehaviorSanitizer by tests/test_chunk.py: the closed sums over
// tiles are those of the tiles one by one, the chunks' walk covers every unit once, gives every
// piece of a cut tile a partial slot of its own, and the join, started from the chunks'
// borders, finds exactly those.
#include <cstdint>
#include <cstdio>
#include <cstdlib>
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

static int64_t at_least(int64_t x, int64_t low) { return x < low ? low : x; }

static ChunkSeq random_seq(std::mt19937_64 &g, int lt, int window) {
  const int64_t nq = g() % 6 == 0 ? 0 : 1 + (int64_t)(g() % (1u << (1 + g() % 10)));
  const int64_t len = g() % 4 == 0 ? (int64_t)(g() % (nq + 3)) : nq + (int64_t)(g() % 4000);
  return chunk_seq(nq, len, lt, window);
}

static void sums(std::mt19937_64 &g) {
  const int lt = 2 + (int)(g() % 7), window = g() % 2 ? 0 : 1 + (int)(g() % 1500);
  const ChunkSeq s = random_seq(g, lt, window);
  const int64_t m = chunk_tiles(s.nq, lt);
  int64_t total = 0;
  for (int64_t i = 0; i < m; ++i) {
    CHECK(chunk_units_before(s, i) == total && chunk_before(s, i) == total + i * kChunkBegin);
    const int64_t t0 = i << lt, t1 = (i + 1) << lt < s.nq ? (i + 1) << lt : s.nq;
    const int64_t end = at_least(s.len - s.nq + t1, 0);
    const int64_t first = window ? at_least(s.len - s.nq + t0 - window + 1, 0) : 0;
    const int64_t units = end > 0 ? (end + 63) / 64 - first / 64 : 1;
    CHECK(chunk_end(s, i) == end && chunk_start(s, i) == first / 64 * 64);
    CHECK(chunk_units(s, i) == units && units >= 1);
    const int64_t at = chunk_before(s, i), taken = units + kChunkBegin;
    for (int64_t u : {at, at + taken / 2, at + taken - 1}) CHECK(chunk_tile_of(s, u) == i);
    total += units;
  }
  CHECK(chunk_before(s, m) == total + m * kChunkBegin);
}

static void walks(std::mt19937_64 &g) {
  const int lt = 2 + (int)(g() % 6), window = g() % 3 ? 0 : 1 + (int)(g() % 900);
  const int n = 1 + (int)(g() % 12);
  const int64_t chunks = 1 + (int64_t)(g() % (g() % 2 ? 8 : 600));
  std::vector<ChunkSeq> seqs;
  std::vector<int64_t> tile_at, tile_units;  // of every tile of the axis
  int64_t total = 0;
  for (int b = 0; b < n; ++b) {
    seqs.push_back(random_seq(g, lt, window));
    for (int64_t i = 0; i < chunk_tiles(seqs[b].nq, lt); ++i) {
      tile_at.push_back(total + kChunkBegin);  // of its own units
      tile_units.push_back(chunk_units(seqs[b], i));
      total += tile_units.back() + kChunkBegin;
    }
  }
  const int64_t per = at_least((total + chunks - 1) / chunks, kChunkLeast);
  CHECK(per * chunks >= total);
  std::vector<int> covered(total, 0);
  std::set<int64_t> slots, joined;
  auto tile_of = [&](int64_t u) {
    size_t t = 0;
    while (t + 1 < tile_at.size() && tile_at[t + 1] - kChunkBegin <= u) ++t;
    return t;
  };
  for (int64_t c = 0; c < chunks; ++c) {
    int64_t cur = c * per;
    const int64_t end = cur + per < total ? cur + per : total;
    while (cur < end) {
      const size_t t = tile_of(cur);
      const int64_t from = cur > tile_at[t] ? cur : tile_at[t];
      const int64_t stop = tile_at[t] + tile_units[t] < end ? tile_at[t] + tile_units[t] : end;
      if (stop <= from) break;
      for (int64_t u = from; u < stop; ++u) ++covered[u];
      if (stop - from < tile_units[t]) {
        const int64_t s = chunk_slot(c, tile_at[t], per);
        CHECK(s >= 0 && s < 2 * chunks && slots.insert(s).second);
      }
      cur = stop;
    }
  }
  for (int64_t u = 0; u < total; ++u) CHECK(covered[u] == (u >= tile_at[tile_of(u)]));
  for (int64_t c = 1; c < chunks && c * per < total; ++c) {
    const int64_t u = c * per;
    const size_t t = tile_of(u);
    if (tile_at[t] >= u || tile_at[t] < u - per) continue;
    const int64_t last = (tile_at[t] + tile_units[t] - 1) / per;
    CHECK(last < chunks);
    for (int64_t x = c - 1; x <= last; ++x)
      CHECK(joined.insert(chunk_slot(x, tile_at[t], per)).second);
  }
  CHECK(slots == joined);
}

static void ends() {
  // the longest caches and chunks of a call
  for (int lt : {2, 7})
    for (int window : {0, 1, (int)kChunkNoWindow}) {
      const ChunkSeq s = chunk_seq(int64_t{1} << 30, INT32_MAX - 4096, lt, window);
      const int64_t m = chunk_tiles(s.nq, lt), all = chunk_before(s, m);
      CHECK(all >= m && chunk_tile_of(s, 0) == 0 && chunk_tile_of(s, all - 1) == m - 1);
      CHECK(chunk_end(s, m - 1) == s.len);
      const ChunkSeq none = chunk_seq(int64_t{1} << 30, 0, lt, window);
      CHECK(chunk_before(none, m) == m * (1 + kChunkBegin));
    }
}

int main(int argc, char **argv) {
  const int rounds = argc > 1 ? std::atoi(argv[1]) : 100;
  std::mt19937_64 g(argc > 2 ? std::atoll(argv[2]) : 1);
  for (int i = 0; i < rounds; ++i) {
    for (int k = 0; k < 20; ++k) sums(g);
    walks(g);
  }
  ends();
  std::printf("%d failed checks\n", fails);
  return fails != 0;
}
