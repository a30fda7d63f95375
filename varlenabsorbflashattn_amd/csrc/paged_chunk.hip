// Attention of several new tokens per sequence over a paged key-value cache, in 16 bits or
// in 8-bit codes, on gfx950 matrix cores (bf16 / f16).
//
// O_i = sum_j softmax_j(s(q_i k_j)) v_j over the keys that token i sees, s the scale, the cap and
// the distance bias, in one pass with a running maximum and sum (masked_tile.h, whose products
// the packed masked forward shares).  A workgroup's 256 rows (128 of 256 features) are tokens of
// up to 32 query heads that share a key head; of a unit of 64 keys the rows are looked up in the
// page table and come to LDS three units ahead.  Lengths are device data, so the work is divided
// here: all units of all tiles form one axis (paged.h), cut into as many even chunks as the GPU
// holds workgroups for each set of heads, and a second launch joins the tiles that were cut.
//
// Few new tokens behind long prefixes are bound by the rows of a cache in 16 bits: 32 sequences
// of 1 to 8 tokens ("drafts" below) behind 1k to 32k keys of 8 heads of 128, 32 query heads, 1.27
// GB, 228 us: 5.6 TB/s, all of it read (a large copy, half written, reaches 5.0); the same inputs
// again and again, of which the last cache keeps a part, 213, and so the comparisons below.  Over
// codes they take 232 for half the bytes, 2.8 TB/s: the units on their way hold half as much, and
// each is converted before it can be used.  Many new tokens are bound by matrix and vector units
// in turn (51% and 41% of the cycles, two waves a SIMD): chunks of 8 prompts, 627 GFLOP, 690 to
// 730 us on different cards, 0.88 PFLOP/s, where the packed kernel on gathered keys takes 652; 14
// of them are the join.  256 rows against 128: the chunks 724 us to 962, 24 turns of 1 to 512
// tokens over codes 90 to 109, the drafts 214 to 215 (a unit is then fetched and, of codes,
// converted for half the rows).
//
// Heads that share a key head share a tile by the largest power of two in their number, and each
// such set walks the keys by itself: the drafts with 16 heads on 4 take 132 us, with 28 on 4, sets
// of one head, 1160 (1500 over codes), with 40 on 8 1740.  Sets whose number is no power of two
// lie unevenly on the XCDs, some of whose workgroups then wait for others to end: the drafts with
// 12 heads on 6 take 275 us for 951 MB, 3.5 TB/s, with 12 on 3 151 for 476, 3.2.
#include <algorithm>
#include <type_traits>

#include "fp8.h"
#include "fwd_tiles.h"
#include "kernels.h"
#include "masked.h"
#include "masked_tile.h"
#include "mfma.h"
#include "paged.h"

namespace vafa {

namespace {

__device__ __forceinline__ int64_t wave_sum_l(int64_t v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((long long)v, o, 64);
  return v;
}
__device__ __forceinline__ int64_t wave_scan_l(int64_t v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int64_t u = __shfl_up((long long)v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}
__device__ __forceinline__ int64_t uniform_l(int64_t v) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)((uint64_t)v >> 32));
  return (int64_t)((uint64_t)hi << 32 | lo);
}

// A sequence's first packed token and its shape.  Lengths that device data have wrong (cu that
// decreases or leaves the rows) give shapes within the rows.
struct SeqAt {
  int q0;
  ChunkSeq s;
};
__device__ __forceinline__ SeqAt seq_at(const ChunkArgs &a, int b) {
  const int T = (int)a.T;
  int q0 = a.cu[b], q1 = a.cu[b + 1], len = a.lens[b];
  asm volatile("" : "+v"(q0), "+v"(q1), "+v"(len));  // (asked for together, used or not)
  q0 = q0 < 0 ? 0 : (q0 > T ? T : q0);
  q1 = q1 < q0 ? q0 : (q1 > T ? T : q1);
  return SeqAt{q0, chunk_seq(q1 - q0, clip_len(len, a.capacity), a.lt, a.window)};
}
// Units of a sequence (tiles where they are not divided).
__device__ __forceinline__ int64_t seq_units(const ChunkArgs &a, int b) {
  if (b >= a.n_seq) return 0;
  const ChunkSeq s = seq_at(a, b).s;
  const int64_t m = chunk_tiles(s.nq, s.lt);
  return a.direct ? m : chunk_before(s, m);
}
// (`mine`: the units of sequence `lane`, which both of these begin with)
__device__ __forceinline__ int64_t all_units(const ChunkArgs &a, int64_t mine, int lane) {
  int64_t total = mine;
  for (int c = 64; c < a.n_seq; c += 64) total += seq_units(a, c + lane);
  return uniform_l(wave_sum_l(total));
}
// The sequence that holds unit `at` of the axis, and the units in front of it.
__device__ __forceinline__ void find_seq(const ChunkArgs &a, int64_t at, int64_t mine, int lane,
                                         int *b, int64_t *base) {
  int64_t before = 0;
  for (int c = 0; c < a.n_seq; c += 64) {
    const int64_t t = c == 0 ? mine : seq_units(a, c + lane), incl = wave_scan_l(t, lane) + before;
    const uint64_t past = __builtin_amdgcn_ballot_w64(incl > at);
    if (past != 0) {
      const int f = __builtin_ctzll(past);
      *b = __builtin_amdgcn_readfirstlane(c + f);
      *base = uniform_l(__shfl((long long)(incl - t), f, 64));
      return;
    }
    before = __shfl((long long)incl, 63, 64);
  }
  *b = a.n_seq;
  *base = uniform_l(before);
}
// n / d by doubles, whose 53 bits hold every axis: the quotient, rounded, is off by one at most.
// (A division of 64-bit integers becomes a branch of the lanes, at whose end the compiler has put
// copies of registers where only the branch's lanes were on.)
__device__ __forceinline__ int64_t quotient(int64_t n, int64_t d) {
  int64_t q = (int64_t)((double)n / (double)d);
  q -= q * d > n;
  return q + ((q + 1) * d <= n);
}
__device__ __forceinline__ int64_t units_per(const ChunkArgs &a, int64_t total) {
  const int64_t per = quotient(total + a.chunks - 1, a.chunks);
  return per < kChunkLeast ? kChunkLeast : per;
}

// A unit's K and V rows in LDS, without padding: 16-byte piece c of row r lies at c ^ f(r), so
// that rows can come by LDS-DMA, which writes whole lines, and are still read without bank
// conflicts: K by 16 rows' same piece at a time (their pieces all over the 64 banks), V by
// transposing reads of 4 rows' 64 bytes.
template <int D>
__device__ __forceinline__ int swizzle_k(int row) {
  return D == 64 ? row >> 1 & 7 : row & 15;
}
template <int D>
__device__ __forceinline__ int swizzle_v(int row) {
  return D == 64 ? (row >> 1 & 1) << 2 : (row & 3) << 2;
}
// Keys of a unit in LDS: the half of an axis unit at D = 256, where 64 leave no room for
// units on their way.
template <int D>
constexpr int kUnitKeys = D == 256 ? 32 : 64;
template <typename T, int D>
struct SwizzledTile {
  static constexpr int kKeys = kUnitKeys<D>;
  static constexpr int kRow = 2 * D, kHalf = kKeys * kRow;  // bytes
  typedef const __attribute__((address_space(3))) u32x4 *lds16;
  typedef __attribute__((address_space(3))) v4s16 *lds8;
  uint32_t ka, va;  // LDS addresses of this lane's first pieces
  static __device__ __forceinline__ SwizzledTile at(uint32_t base, int lane) {
    const int r = lane & 31, i = lane & 15, g = lane >> 4;
    const int vr = 4 * (g >> 1) + (i >> 2);
    SwizzledTile t;
    t.ka = base + r * kRow + (((lane >> 5) ^ swizzle_k<D>(r)) << 4);
    t.va = base + kHalf + vr * kRow +
           ((((g & 1) * 2 + ((i & 3) >> 1)) ^ swizzle_v<D>(vr)) << 4) + (i & 1) * 8;
    return t;
  }
  // (units and rows are multiples of what the exclusive or reaches)
  __device__ __forceinline__ SwizzledTile at_offset(int bytes) const {
    return SwizzledTile{ka + bytes, va + bytes};
  }
  __device__ __forceinline__ u32x4 k(int kt, int cc) const {
    return *(lds16)(uintptr_t)((ka ^ ((cc & 7) << 5)) + (cc >> 3) * 256 + kt * 32 * kRow);
  }
  __device__ __forceinline__ typename Mfma<T>::v8 v(int km, int dt) const {
    const uint32_t p = (va ^ ((dt & 3) << 6)) + (dt >> 2) * 256 + km * 16 * kRow;
    const u32x2 lo = __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds8)(uintptr_t)p));
    const u32x2 hi = __builtin_bit_cast(
        u32x2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds8)(uintptr_t)(p + 8 * kRow)));
    return as_v8<T>(join(lo, hi));
  }
};

// What absent keys hold, and their page.
__device__ const u32x4 kZeroRow[32] = {};
__device__ const int32_t kNoPage = -1;

// Unit u's rows are asked for kAhead units ahead.  16 bits: into one of kAhead + 1 buffers,
// from which the products read them.  Codes: into a raw buffer; they become T in one of two
// buffers a unit ahead.  Beside them, for the units of two blocks of NW: the pages on their way,
// where each key's rows are, which keys there are and, of codes, the words that hold their
// powers of two.
template <int D, int NW, bool kCodes>
struct ChunkSmem {
  static constexpr int kKeys = kUnitKeys<D>, kAhead = D == 64 ? 7 : 3, kRing = 2 * NW;  // units
  static constexpr int kUnit = 2 * kKeys * 2 * D, kRaw = kUnit / 2;       // bytes, K and V
  static constexpr int kBuffers = kCodes ? 2 : kAhead + 1;
  static constexpr int kRawAt = kBuffers * kUnit;
  static constexpr int kRowsAt = kRawAt + (kCodes ? (kAhead + 1) * kRaw : 0);
  static constexpr int kIdsAt = kRowsAt + kRing * kKeys * 16;
  static constexpr int kHereAt = kIdsAt + kRing * 256;
  static constexpr int kWordsAt = kHereAt + kRing * 8;
  static constexpr int kBytes = kWordsAt + (kCodes ? kRing * 512 : 0);
  static_assert(kAhead < NW, "a block's rows are looked up before they are asked for");
};

// 256 rows of 8 waves (D = 256: 128 of 4, which have its registers), one workgroup on a CU.
template <typename T, int D, int NW, bool kCodes, bool kCap, bool kBias, bool kOnce>
__device__ __forceinline__ void chunk_walk(const ChunkArgs &a) {
  using M = Mfma<T>;
  using E = std::conditional_t<kCodes, uint8_t, T>;
  using Tile = SwizzledTile<T, D>;
  using S = ChunkSmem<D, NW, kCodes>;
  constexpr int NC = D / 16, ND = D / 32, NT = 64 * NW, BM = 32 * NW;
  constexpr int kKeys = S::kKeys, kAhead = S::kAhead;
  constexpr int kPiece = 16 / (int)sizeof(E), kPerRow = D / kPiece;  // 16-byte pieces of a row
  constexpr int kHalf = kKeys * kPerRow;                             // of a unit's K
  constexpr int kPieces = 2 * kHalf / NT;                            // of a thread, K and V
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int lg = a.lg, tw = 32 >> lg;  // tokens of a wave
  const HeadSets hs{a.H, a.Hk, lg};

  // the sets of a chunk on one XCD: they read whole token rows of the pages together
  const int sets = hs.sets();
  const int group = blockIdx.x / (kXcds * sets), within = blockIdx.x % (kXcds * sets);
  const int chunk = group * kXcds + within % kXcds, set = within / kXcds;
  const int h0 = set << lg, hk = set / hs.per_key();

  if (chunk >= a.chunks) return;
  ChunkCut *cut = a.cuts + (int64_t)chunk * sets + set;  // at this chunk's end
  if (!a.direct && tid == 0) *cut = ChunkCut{0, 0, 0, 0};
  const int64_t mine = seq_units(a, lane);
  // (tiles dealt in turn go on until there is no sequence for one)
  int64_t total = INT64_MAX, per = 1;
  if (!a.direct) {
    asm volatile("");  // (a branch: not computed aside)
    total = all_units(a, mine, lane);
    per = uniform_l(units_per(a, total));
  }
  int64_t cur = chunk * per;
  const int64_t end = a.direct || total - cur < per ? total : cur + per;
  if (cur >= end) return;
  int b;
  int64_t base;
  find_seq(a, cur, mine, lane, &b, &base);

  ScoreArgs sa{a.c, a.cap2};
  uint32_t qsign = 0;
  if constexpr (!kCap && !kBias) {  // (as in the packed forward)
    if (sa.c < 0.f) qsign = 0x80008000u;
    sa.c = score_factor(sa.c);
  }
  const int window = a.window > 0 ? a.window : kChunkNoWindow;
  const u32x4 *kc = reinterpret_cast<const u32x4 *>((const E *)a.kc + hk * a.kc_head);
  const u32x4 *vc = reinterpret_cast<const u32x4 *>((const E *)a.vc + hk * a.vc_head);
  const uint32_t smem = lds_addr(smem_raw);
  const Tile tile0 = Tile::at(smem, lane);

  while (cur < end) {
    if (b >= a.n_seq) break;
    const SeqAt at = seq_at(a, b);
    const ChunkSeq &s = at.s;
    const int64_t tiles = chunk_tiles(s.nq, s.lt);
    const int64_t all = a.direct ? tiles : chunk_before(s, tiles);
    if (cur - base >= all) {
      base += all;
      ++b;
      continue;
    }
    const int64_t i = a.direct ? cur - base : chunk_tile_of(s, cur - base);
    // the axis from the tile's own units on, and those that are this chunk's
    const int64_t t0 = a.direct ? cur : base + chunk_before(s, i) + kChunkBegin;
    const int64_t units = chunk_units(s, i), from = cur > t0 ? cur : t0;
    const int64_t till = a.direct || t0 + units < end ? t0 + units : end;
    if (till <= from) break;  // the chunk ends in front of them
    const int64_t u0 = from - t0;
    const int part = (int)uniform_l(till - from);
    const bool whole = part == units;
    const int run = part * (kChunkKeys / kKeys);  // in units of LDS
    const int q0 = __builtin_amdgcn_readfirstlane(at.q0 + (int)(i << s.lt));
    const int qn = uniform_clamp((int)(s.nq - (i << s.lt)), BM >> lg), q1 = q0 + qn;
    const int diag = __builtin_amdgcn_readfirstlane((int)(s.diag - at.q0));
    const int kb0 = __builtin_amdgcn_readfirstlane((int)(chunk_start(s, i) + u0 * kChunkKeys));
    const int kend = __builtin_amdgcn_readfirstlane((int)chunk_end(s, i));
    // keys in front of it are of no row's window, though of the first unit: absent
    const int kfirst = a.window > 0 ? q0 + diag - a.window + 1 : 0;

    // A short piece of a tile of few rows: its units lie in the buffers at once, and each is
    // another group of waves' (4 sequences of 2 to 8 tokens behind 17 to 500 keys, 16 heads of
    // 64: 11.8 -> 10.3 us; more features have no room for as many units)
    constexpr bool kShorts = D == 64 && !kCodes;
    int lr = 0;  // log2 of a group's waves
    if (kShorts)
      while ((tw << lr) < qn) ++lr;
    const bool is_short = kShorts && run <= kAhead && run <= NW >> lr;
    const int rw = is_short ? wave & ((1 << lr) - 1) : wave, grp = is_short ? wave >> lr : 0;
    const int w0 = q0 + rw * tw;  // the wave's first token
    const int tok = w0 + (lrow >> lg), h = h0 + (lrow & ((1 << lg) - 1));
    const bool row_ok = tok < q1, wave_active = w0 < q1 && (!is_short || grp < run);
    const int p = tok + diag;
    const int p0 = w0 + diag, p1 = (w0 + tw < q1 ? w0 + tw : q1) - 1 + diag;
    typename M::v8 qf[NC];
    {
      const T *qr = (const T *)a.q + (int64_t)(row_ok ? tok : q0) * a.q_token + h * a.q_head +
                    lhalf * 8;
#pragma unroll
      for (int cc = 0; cc < NC; ++cc) {
        u32x4 x = *reinterpret_cast<const u32x4 *>(qr + cc * 16);
#pragma unroll
        for (int w = 0; w < 4; ++w) x[w] = row_ok ? x[w] ^ qsign : 0u;
        qf[cc] = as_v8<T>(x);
      }
    }
    float slope2 = 0.f;
    if constexpr (kBias) slope2 = a.slopes[h] * kLog2e;

    f32x16 acc[ND];
#pragma unroll
    for (int x = 0; x < ND; ++x)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[x][r] = 0.f;
    float m_run = -kHuge, l_part = 0.f;

    // Each wave looks up the rows of one unit of every block of NW.  First their pages:
    auto ask_ids = [&](int u) {
      const int key = kb0 + u * kKeys + lane % kKeys;
      const int32_t *from = &kNoPage;
      if (u < run && key >= kfirst && key < kend)  // (within the table: kend is)
        from = a.map.table + b * a.map.row_stride + page_slot(a.map, key).index;
      lds_dma4(from, smem + S::kIdsAt + u % S::kRing * 256);
    };
    // then, of each key, where its rows of K and V are, in pieces of 16 bytes from kc and vc
    // (zeros for absent keys); a factor of 16 drops the highest bits, which hold, of codes, the
    // byte of the word that is the row's power of two (0 to 3) and whether there is none (4)
    auto look_up = [&](int u) {
      const int id = reinterpret_cast<const int32_t *>(smem_raw + S::kIdsAt)[u % S::kRing * 64 + lane];
      const bool there = (uint32_t)id < (uint32_t)a.map.n_pages;
      const uint32_t slot = page_slot(a.map, kb0 + u * kKeys + lane % kKeys).slot;
      // (32-bit factors: one instruction each)
      uint64_t k = (uint64_t)(uint32_t)id * a.k_page + (uint64_t)slot * a.kc_token;
      uint64_t v = (uint64_t)(uint32_t)id * a.v_page + (uint64_t)slot * a.vc_token;
      if (!there) {
        k = (uint64_t)((uintptr_t)kZeroRow - (uintptr_t)kc) >> 4;
        v = (uint64_t)((uintptr_t)kZeroRow - (uintptr_t)vc) >> 4;
      }
      if constexpr (kCodes) {
        const RowScales &sc = a.scales;
        const uint32_t i_ = there ? id : 0, s_ = there ? slot : 0;
        const uintptr_t ks = (uintptr_t)(sc.k + hk * sc.k_head) +
                             ((uint64_t)i_ * (uint32_t)sc.k_page + (uint64_t)s_ * (uint32_t)sc.k_token);
        const uintptr_t vs = (uintptr_t)(sc.v + hk * sc.v_head) +
                             ((uint64_t)i_ * (uint32_t)sc.v_page + (uint64_t)s_ * (uint32_t)sc.v_token);
        k |= (uint64_t)((ks & 3) | (there ? 0 : 4)) << 60;
        v |= (uint64_t)((vs & 3) | (there ? 0 : 4)) << 60;
        const uint32_t words = smem + S::kWordsAt + u % S::kRing * 512;
        lds_dma4((const void *)(ks & ~uintptr_t{3}), words);
        lds_dma4((const void *)(vs & ~uintptr_t{3}), words + 256);
      }
      *reinterpret_cast<u32x4 *>(smem_raw + S::kRowsAt + (u % S::kRing * kKeys + lane % kKeys) * 16) =
          u32x4{(uint32_t)k, (uint32_t)(k >> 32), (uint32_t)v, (uint32_t)(v >> 32)};
      const uint64_t here = __builtin_amdgcn_ballot_w64(there);
      if (lane == 0)
        *reinterpret_cast<uint64_t *>(smem_raw + S::kHereAt + u % S::kRing * 8) = here;
    };
    auto present = [&](int u) {  // which keys of unit u there are
      return uniform_l(*reinterpret_cast<const int64_t *>(smem_raw + S::kHereAt + u % S::kRing * 8));
    };
    // where unit u's K and V rows go: 16 bits to where the products read them, piece by piece
    // swizzled, codes as they are
    auto unit_at = [&](int u) { return u % S::kBuffers * S::kUnit; };
    auto raw_at = [&](int u) { return S::kRawAt + u % (kAhead + 1) * S::kRaw; };
    // this thread's pieces of a unit, K's rows and then V's (for some waves' pieces K's, for
    // others' V's where a unit has no more)
    auto row_of = [&](int x) { return (tid + NT * x) % kHalf / kPerRow; };
    auto of_v = [&](int x) { return wave * 64 + NT * x >= kHalf; };
    auto place_of = [&](int u, int x) {
      return smem_raw + S::kRowsAt + (u % S::kRing * kKeys + row_of(x)) * 16 + (of_v(x) ? 8 : 0);
    };
    auto ask_rows = [&](int u) {
      const uint32_t to = smem + (kCodes ? raw_at(u) : unit_at(u)) + wave * 1024;
      const u32x4 *from[kPieces];
#pragma unroll
      for (int x = 0; x < kPieces; ++x) {
        const int piece = tid % kPerRow, row = row_of(x);
        const int col = kCodes ? piece : piece ^ (of_v(x) ? swizzle_v<D>(row) : swizzle_k<D>(row));
        from[x] = (of_v(x) ? vc : kc) + col + *reinterpret_cast<const uint64_t *>(place_of(u, x));
      }
#pragma unroll
      for (int x = 0; x < kPieces; ++x)
        if constexpr (kOnce)
          lds_dma16_once(from[x], to + x * NT * 16);
        else
          lds_dma16(from[x], to + x * NT * 16);
    };
    // codes: unit u's rows, which this thread asked for, become T
    auto convert = [&](int u) {
#pragma unroll
      for (int x = 0; x < kPieces; ++x) {
        const int row = row_of(x), piece = tid % kPerRow;
        const bool is_v = of_v(x);
        const uint32_t top = reinterpret_cast<const uint32_t *>(place_of(u, x))[1] >> 28;
        const uint32_t e = smem_raw[S::kWordsAt + u % S::kRing * 512 + is_v * 256 + row * 4 + (top & 3)];
        // (absent keys are zeros, whatever their power of two)
        const float scale = top < 4 ? row_scale(e) : 1.f;
        const u32x4 codes =
            *reinterpret_cast<const u32x4 *>(smem_raw + raw_at(u) + (tid + NT * x) * 16);
        u32x4 lo, hi;
        from_codes<T>(codes, scale, lo, hi);
        const int c = (2 * piece) ^ (is_v ? swizzle_v<D>(row) : swizzle_k<D>(row));
        unsigned char *to = smem_raw + unit_at(u) + (is_v ? Tile::kHalf : 0) + row * Tile::kRow;
        *reinterpret_cast<u32x4 *>(to + c * 16) = lo;
        *reinterpret_cast<u32x4 *>(to + (c ^ 1) * 16) = hi;
      }
    };

    // Waits count requests, which come in the order they were made: behind unit j + 1's there
    // are those of the kAhead - 1 units after it, and pages and words now and then (the wait is
    // then for a little more).  Past the piece's end the requests go on (for zeros).
    constexpr int kRequests = (kAhead - 1) * kPieces;
    ask_ids(wave);
    ask_ids(NW + wave);
    wait_vmcnt<0>();
    look_up(wave);
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kAhead; ++u) ask_rows(u);
    if (is_short)
      wait_vmcnt<0>();
    else
      wait_vmcnt<kRequests>();
    if constexpr (kCodes) {
      __syncthreads();  // words that other waves asked for
      convert(0);
    }
    __syncthreads();
    const int turns = is_short ? 1 : run;
    for (int j = 0; j < turns; ++j) {
      if (!is_short) {
        if (j % NW == 0) {  // a block's rows before its first are asked for, pages a block ahead
          look_up(j + NW + wave);
          ask_ids(j + 2 * NW + wave);
        }
        ask_rows(j + kAhead);
      }
      const int u = j + grp, kb = kb0 + u * kKeys;
      const int kl = (kb + kKeys < kend ? kb + kKeys : kend) - 1;
      if (wave_active && !none_visible(kb, kl, p0, p1, 0, window)) {
        const uint64_t here = present(u);
        const bool masked = here != ~uint64_t{0} || !all_visible(kb, kl, p0, p1, 0, window);
        masked_tile<T, D, kCap, kBias>(tile0.at_offset(unit_at(u)), qf, acc, m_run, l_part, sa,
                                       slope2, kb, kend, masked, p, 0, window, lane, here);
      }
      if (is_short) break;
      wait_vmcnt<kRequests>();
      if constexpr (kCodes) convert(j + 1);
      __syncthreads();
    }
    wait_vmcnt<0>();  // nothing on its way to what the rows' store takes
    __syncthreads();

    // the groups' rows, each register's 64 lanes beside each other, joined in their order
    if (kShorts && is_short && run > 1) {
      constexpr int kRegs = 16 * ND + 2;
      float *x = reinterpret_cast<float *>(smem_raw) + lane;
      if (wave_active && grp > 0) {
        float *to = x + wave * kRegs * 64;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) to[(d * 16 + r) * 64] = acc[d][r];
        to[16 * ND * 64] = m_run;
        to[(16 * ND + 1) * 64] = l_part;
      }
      __syncthreads();
      if (wave_active && grp == 0) {
        auto part_of = [&](int g) { return x + ((g << lr) + rw) * kRegs * 64; };
        float m_new = m_run;
        for (int g = 1; g < run; ++g) m_new = fmaxf(m_new, part_of(g)[16 * ND * 64]);
        const float f = fast_exp2(m_run - m_new);
        m_run = m_new;
        l_part *= f;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
          for (int r = 0; r < 16; ++r) acc[d][r] *= f;
        for (int g = 1; g < run; ++g) {
          const float *from = part_of(g);
          const float w = fast_exp2(from[16 * ND * 64] - m_new);
          l_part += from[(16 * ND + 1) * 64] * w;
#pragma unroll
          for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[d][r] += from[(d * 16 + r) * 64] * w;
        }
      }
      __syncthreads();
    }
    if (wave_active && grp == 0) {
      // a row that sees no key has l = 0 (output 0, lse -inf); NaN scores stay NaN
      const float l = l_part + __shfl_xor(l_part, 32, 64);
      const float inv = l == 0.f ? 0.f : 1.f / l;
      using RS = RowStore<T, ND>;
      unsigned char *stage = smem_raw + wave * RS::kBytes;
      const int rows = uniform_clamp(q1 - w0, tw) << lg;
      if (whole) {
        RS::rows16_at(acc, [&](float x) { return static_cast<T>(x * inv); }, stage,
                      (T *)a.out + ((int64_t)w0 * a.H + h0) * D,
                      [&](int r) { return (int64_t)hs.row(r) * D; }, rows);
      } else {
        const float lse = l == 0.f ? kNegInf : m_run + fast_log2(l);
        const int64_t row = (chunk_slot(chunk, t0, per) * sets + set) * BM + wave * 32;
        RS::rows32_at(acc, inv, stage, a.part_o + row * D, [&](int r) { return (int64_t)r * D; },
                      rows);
        if (row_ok && lhalf == 0) a.part_lse[row + lrow] = lse;
        if (tid == 0 && u0 == 0)  // the tile's first part
          *cut = ChunkCut{q0, qn, (int)quotient(t0 + units - 1, per),
                          (int)chunk_slot(chunk, t0, per)};
      }
    }
    __syncthreads();  // the staged rows are read: the next piece may write K and V
    if (a.direct) {
      cur += a.chunks;
      if (cur < end) find_seq(a, cur, mine, lane, &b, &base);
    } else {
      cur = till;
    }
  }
}

template <typename T, int D, int NW, bool kCodes, bool kCap, bool kBias, bool kOnce>
__global__ __launch_bounds__(64 * NW, D >= 256 ? 1 : 2) void paged_chunk_kernel(ChunkArgs a) {
  chunk_walk<T, D, NW, kCodes, kCap, kBias, kOnce>(a);
  // rows of no sequence, in front of the first and behind the last
  const int T_ = (int)a.T;
  int lo = a.cu[0], hi = a.cu[a.n_seq];
  lo = lo < 0 ? 0 : (lo > T_ ? T_ : lo);
  hi = hi < lo ? lo : (hi > T_ ? T_ : hi);
  const int64_t edge = (int64_t)lo * a.H * D, pieces = (int64_t)(lo + T_ - hi) * a.H * D / 8;
  for (int64_t e = (int64_t)blockIdx.x * (64 * NW) + threadIdx.x; e < pieces;
       e += (int64_t)gridDim.x * (64 * NW)) {
    const int64_t at = e * 8;
    T *p = (T *)a.out + (at < edge ? at : at - edge + (int64_t)hi * a.H * D);
    *reinterpret_cast<u32x4 *>(p) = u32x4{0, 0, 0, 0};
  }
}

template <typename T, int D, int NW, bool kCodes>
constexpr int chunk_lds() {
  constexpr int kStage = NW * RowStore<T, D / 32>::kBytes;
  static_assert(kStage <= ChunkSmem<D, NW, kCodes>::kBytes, "staged rows");
  return ChunkSmem<D, NW, kCodes>::kBytes;
}

// Joins the parts of a tile that chunks cut: a group of workgroups for each chunk's end and each
// set, of which the tile's first has the work, 4096 outputs a workgroup, 16 neighbouring features
// a thread: m = max lse_g, w_g = 2^(lse_g - m), O = sum w_g O_g / sum w_g.  The first two parts,
// which are all of most tiles, are asked for at once.  Bound by the parts' bytes where tiles are
// full (chunks of 8 prompts: 14 us; finding the tiles again here instead of reading where they
// are cut: 21), else by latency (drafts 7, and 9.5).
template <typename T, int D, int BM>
__global__ __launch_bounds__(256) void paged_chunk_join_kernel(ChunkArgs a) {
  constexpr int kRowsOf = 4096 / D, kParts = BM / kRowsOf;
  const int tid = threadIdx.x, sets = a.H >> a.lg;
  const int part = blockIdx.x % kParts, set = blockIdx.x / kParts % sets;
  const int chunk = blockIdx.x / kParts / sets;
  const ChunkCut cut = a.cuts[(int64_t)chunk * sets + set];
  const int row = part * kRowsOf + tid / (D / 16), f = tid % (D / 16) * 16, tok = row >> a.lg;
  if (tok >= cut.tokens) return;
  auto row_of = [&](int64_t slot) { return (slot * sets + set) * BM + row; };
  auto part_of = [&](int64_t r, f32x4 *x) {
    const f32x4 *src = reinterpret_cast<const f32x4 *>(a.part_o + r * D + f);
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = src[e];
    return a.part_lse[r];
  };
  f32x4 x[4], y[4];
  const float m0 = part_of(row_of(cut.slot), x), m1 = part_of(row_of(2 * (int64_t)chunk + 2), y);
  float m = fmaxf(m0, m1), l = 0.f;
  auto add = [&](float had, float w) {
    l = l * had + w;
#pragma unroll
    for (int e = 0; e < 4; ++e)
#pragma unroll
      for (int t = 0; t < 4; ++t) x[e][t] = x[e][t] * had + y[e][t] * w;
  };
  {
    const float ms = m == kNegInf ? 0.f : m;  // (a part that sees no key is zeros)
    const float w0 = fast_exp2(m0 - ms);
    add(w0, fast_exp2(m1 - ms));
    l += w0;
  }
  for (int g = chunk + 2; g <= cut.last; ++g) {
    const float mg = part_of(row_of(2 * (int64_t)g), y), top = fmaxf(m, mg);
    add(m == kNegInf ? 0.f : fast_exp2(m - top), mg == kNegInf ? 0.f : fast_exp2(mg - top));
    m = top;
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const int head = (set << a.lg) + (row & ((1 << a.lg) - 1));
  T *dst = (T *)a.out + (((int64_t)cut.first + tok) * a.H + head) * D + f;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    typename Mfma<T>::v8 z;
#pragma unroll
    for (int t = 0; t < 8; ++t) z[t] = static_cast<T>(x[2 * e + t / 4][t % 4] * inv);
    *reinterpret_cast<typename Mfma<T>::v8 *>(dst + 8 * e) = z;
  }
}

template <typename T, int D, int NW, bool kCodes, bool kCap, bool kBias, bool kOnce>
void launch_v(const ChunkArgs &a, hipStream_t st) {
  constexpr auto fn = &paged_chunk_kernel<T, D, NW, kCodes, kCap, kBias, kOnce>;
  const int smem = chunk_lds<T, D, NW, kCodes>(), sets = a.H >> a.lg;
  allow_dynamic_lds(reinterpret_cast<const void *>(fn), smem);
  const int64_t wgs = (int64_t)(a.chunks + kXcds - 1) / kXcds * kXcds * sets;
  hipLaunchKernelGGL(fn, dim3((unsigned)wgs), dim3(64 * NW), smem, st, a);
  if (a.direct || a.chunks < 2) return;
  const int64_t joins = (int64_t)(a.chunks - 1) * sets * (32 * NW * D / 4096);
  hipLaunchKernelGGL((paged_chunk_join_kernel<T, D, 32 * NW>), dim3((unsigned)joins), dim3(256), 0,
                     st, a);
}

template <typename T, int D, bool kCodes, bool kOnce>
void launch_d(const ChunkArgs &a, hipStream_t st) {
  constexpr int NW = D <= 128 ? 8 : 4;
  const bool cap = a.cap2 > 0.f, bias = a.slopes != nullptr;
  if (cap && bias) return launch_v<T, D, NW, kCodes, true, true, kOnce>(a, st);
  if (cap) return launch_v<T, D, NW, kCodes, true, false, kOnce>(a, st);
  if (bias) return launch_v<T, D, NW, kCodes, false, true, kOnce>(a, st);
  launch_v<T, D, NW, kCodes, false, false, kOnce>(a, st);
}

}  // namespace

// Rows in 16 bits pass the caches where a sequence has no more than a tile's tokens on average
// and a key head one set, so that most are read once (the drafts 250 -> 213 us; the chunks 718 ->
// 742).  Codes do not: 234 -> 230 us of the drafts, 708 -> 738 of the chunks.
template <typename T, int D>
void launch_paged_chunk(const ChunkArgs &a, hipStream_t st) {
  if (a.scales.k != nullptr) return launch_d<T, D, true, false>(a, st);
  if (a.T <= (int64_t)a.n_seq << a.lt && a.H == a.Hk << a.lg)
    return launch_d<T, D, false, true>(a, st);
  launch_d<T, D, false, false>(a, st);
}

#define VAFA_INST(T, D) template void launch_paged_chunk<T, D>(const ChunkArgs &, hipStream_t);
VAFA_INST(bf16, 64)
VAFA_INST(bf16, 128)
VAFA_INST(bf16, 256)
VAFA_INST(f16, 64)
VAFA_INST(f16, 128)
VAFA_INST(f16, 256)
#undef VAFA_INST

}  // namespace vafa
