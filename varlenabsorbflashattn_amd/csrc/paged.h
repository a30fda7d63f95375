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

}  // namespace vafa
