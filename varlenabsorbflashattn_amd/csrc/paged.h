// Addressing of a paged key-value cache and the work split of the decoding
// attention: plain integer functions shared by the kernels and the host.
#pragma once
#include <stdint.h>

#ifdef __HIP__
#include <hip/hip_runtime.h>
#define VAFA_HD __host__ __device__ __forceinline__
#else
#define VAFA_HD inline
#endif

namespace vafa {

// One sequence's pages: row b of the page table, `width` entries.
struct PageMap {
  const int32_t *table;
  int64_t row_stride;
  int32_t width, page, shift;  // tokens of a page; log2 of it, or -1
  int32_t n_pages;
};

VAFA_HD int page_shift(int64_t page) {
  for (int s = 0; s < 31; ++s)
    if ((int64_t{1} << s) == page) return s;
  return -1;
}

// Tokens that a row of the table can address, and a sequence's length clipped to
// what it can hold (a length is device data: the host cannot refuse it).
VAFA_HD int64_t page_capacity(const PageMap &m) {
  const int64_t c = (int64_t)m.width * m.page;
  return c > INT32_MAX ? INT32_MAX : c;
}
VAFA_HD int32_t clip_len(int32_t len, int64_t capacity) {
  return len < 0 ? 0 : (len > capacity ? (int32_t)capacity : len);
}

struct PageSlot {
  int32_t index, slot;  // entry of the table's row, token in the page
};
VAFA_HD PageSlot page_slot(const PageMap &m, int32_t pos) {
  PageSlot s;
  s.index = m.shift >= 0 ? pos >> m.shift : pos / m.page;
  s.slot = pos - s.index * m.page;
  return s;
}

// The page that holds token `pos` of sequence b, or -1 where the position lies
// outside the table or the entry outside the cache: such a token is neither
// written nor read.
VAFA_HD int32_t page_of(const PageMap &m, int64_t b, int32_t pos, const PageSlot &s) {
  if (pos < 0 || s.index >= m.width) return -1;
  const int32_t id = m.table[b * m.row_stride + s.index];
  return id >= 0 && id < m.n_pages ? id : -1;
}

// ---- decoding attention: tiles of kDecodeTile keys ------------------------------
// The tiles of all sequences, one after another, form one axis, of which chunk c takes
// the tiles [c * per, (c + 1) * per).  A workgroup walks one chunk for one pair (key head,
// block of kDecodeRows query heads).
constexpr int kDecodeTile = 128;
constexpr int kDecodeRows = 16;

// Keys of a sequence that its new token sees, and their tiles.
VAFA_HD int32_t decode_seen(int32_t len, int32_t window) {
  return window > 0 && len > window ? window : len;
}
VAFA_HD int32_t decode_tiles(int32_t len, int32_t window) {
  const int32_t n = decode_seen(len, window);
  return n / kDecodeTile + (n % kDecodeTile != 0);
}
VAFA_HD int32_t decode_per(int32_t total, int32_t chunks) {
  return total / chunks + (total % chunks != 0);
}
// Partial result of the piece that chunk c holds of a sequence whose tiles start at t0
// of the axis: its first piece has slot 2 c, its last 2 c + 1 (pieces between them are
// whole sequences and need none).
VAFA_HD int64_t decode_slot(int32_t c, int32_t t0, int32_t per) {
  return 2 * (int64_t)c + ((int64_t)c * per < t0 ? 1 : 0);
}

// ---- attention of a chunk of new tokens: units of kChunkKeys keys ----------------
// The nq new tokens of a sequence of len cached ones are its last; token t has position
// diag + t, diag = len - nq, and sees the keys up to its own (the last `window` of them).
// Tokens go in tiles of 2^lt; tile i walks units of kChunkKeys keys from start(i), a multiple
// of that, to end(i), one unit at least (a tile without keys writes zeros).  Beginning a tile
// costs as much as kChunkBegin units, which lie in front of its own.  All of them, one tile and
// one sequence after another, form one axis, of which chunk c takes [c * per, (c + 1) * per):
// tiles are cut anywhere among their own units, and their parts joined.
constexpr int kChunkKeys = 64, kChunkShift = 6;
// Of the axis, a chunk has this many at least (one sequence of 1k keys, 4 and 128 new tokens,
// D = 128: 2 19 and 32 us, 4 19 and 30, 8 23 and 33, 24 29 and 50; D = 256: 23 and 34, 27 and
// 36, 37 and 43, 56 and 73)
constexpr int64_t kChunkLeast = 4;
// (24 sequences, 1 to 512 new tokens behind 1 to 16k: chunks of many tiles with few keys held
// the launch; 126 -> 90 us)
constexpr int64_t kChunkBegin = 4;
// as a window, every key: no sum with a position or a tile's rows passes 32 bits
constexpr int32_t kChunkNoWindow = INT32_MAX - 1024;

struct ChunkSeq {
  int64_t nq, len, diag;
  int32_t lt, window;  // window 0: all keys
};
VAFA_HD ChunkSeq chunk_seq(int64_t nq, int64_t len, int32_t lt, int32_t window) {
  return ChunkSeq{nq, len, len - nq, lt, window};
}
VAFA_HD int64_t chunk_tiles(int64_t nq, int32_t lt) {
  return (nq + (int64_t{1} << lt) - 1) >> lt;
}
VAFA_HD int64_t chunk_end(const ChunkSeq &s, int64_t i) {
  const int64_t t = (i + 1) << s.lt, e = (t < s.nq ? t : s.nq) + s.diag;
  return e > 0 ? e : 0;
}
VAFA_HD int64_t chunk_start(const ChunkSeq &s, int64_t i) {
  if (s.window <= 0) return 0;
  const int64_t b = (i << s.lt) + s.diag - s.window + 1;
  return b > 0 ? b >> kChunkShift << kChunkShift : 0;
}
VAFA_HD int64_t chunk_units(const ChunkSeq &s, int64_t i) {
  const int64_t e = chunk_end(s, i);
  return e > 0 ? ((e + kChunkKeys - 1) >> kChunkShift) - (chunk_start(s, i) >> kChunkShift) : 1;
}
// sum of floor((c + (j << lt)) / kChunkKeys) over j in [j0, j1), c + (j0 << lt) >= 0
VAFA_HD int64_t chunk_floors(int64_t c, int32_t lt, int64_t j0, int64_t j1) {
  if (j1 <= j0) return 0;
  if (lt >= kChunkShift)
    return (j1 - j0) * (c >> kChunkShift) +
           ((j1 * (j1 - 1) - j0 * (j0 - 1)) >> 1 << (lt - kChunkShift));
  // floor((c + j 2^lt) / 64) = floor((floor(c / 2^lt) + j) / 2^r): below n, whole runs of 2^r
  const int32_t r = kChunkShift - lt;
  const int64_t n0 = (c >> lt) + j0, n1 = (c >> lt) + j1, q0 = n0 >> r, q1 = n1 >> r;
  return ((q1 * (q1 - 1)) >> 1 << r) + (n1 - (q1 << r)) * q1 -
         (((q0 * (q0 - 1)) >> 1 << r) + (n0 - (q0 << r)) * q0);
}
// Units of the tiles in front of tile i (i up to the sequence's tiles: all of them).
VAFA_HD int64_t chunk_units_before(const ChunkSeq &s, int64_t i) {
  const int64_t m = chunk_tiles(s.nq, s.lt);
  if (s.len <= 0 || i <= 0) return i;
  // tiles whose end is 0; the last has end len > 0
  int64_t none = s.diag < 0 ? -s.diag >> s.lt : 0;
  if (none > m - 1) none = m - 1;
  if (i <= none) return i;
  const int64_t last = i < m ? i : m - 1;
  int64_t n = none + chunk_floors(s.diag + (int64_t{1} << s.lt) + kChunkKeys - 1, s.lt, none, last);
  if (i == m) n += (s.len + kChunkKeys - 1) >> kChunkShift;
  if (s.window > 0) {
    const int64_t back = s.window - 1 - s.diag;  // starts are 0 up to here
    const int64_t w0 = back <= 0 ? 0 : (back + (int64_t{1} << s.lt) - 1) >> s.lt;
    n -= chunk_floors(-back, s.lt, w0, i);
  }
  return n;
}
// What these tiles take of the axis.
VAFA_HD int64_t chunk_before(const ChunkSeq &s, int64_t i) {
  return chunk_units_before(s, i) + i * kChunkBegin;
}
// The tile that holds place u of the sequence's part of the axis.
VAFA_HD int64_t chunk_tile_of(const ChunkSeq &s, int64_t u) {
  int64_t lo = 0, hi = chunk_tiles(s.nq, s.lt) - 1;  // chunk_before(lo) <= u
  while (lo < hi) {
    const int64_t mid = (lo + hi + 1) >> 1;
    if (chunk_before(s, mid) <= u)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}
// Partial result of the piece that chunk c holds of a tile whose own units start at t0 of the
// axis: its first piece has slot 2 c, its last 2 c + 1 (pieces between them are whole tiles).
VAFA_HD int64_t chunk_slot(int64_t c, int64_t t0, int64_t per) {
  return 2 * c + (c * per < t0 ? 1 : 0);
}

}  // namespace vafa
