// Query and key blocks of the backward kernels: LDS layout, staging by LDS-DMA and
// through registers.
#pragma once
#include "mfma.h"

namespace vafa {

namespace {

constexpr int kRB = 32;  // rows per staged block (queries for dK/dV, keys for dQ)
// LDS layout of a 32-row tile of 16-bit rows that is read both as rows
// (ds_read_b128: 16 lanes take one 16-byte chunk of 16 consecutive rows) and
// transposed (ds_read_b64_tr_b16: 32 lanes take 64 bytes of 4 consecutive
// rows).  With one row stride the two cannot both be conflict-free -- row
// reads want 4 x odd dwords, transposed reads 16 mod 64 dwords -- so rows sit
// in groups of four: P1 elements apart inside a group (P1/2 dwords = 16 mod
// 32: the 4 row pieces of a transposed read fill distinct banks) and P2 =
// 4*P1 + 8 elements from group to group (4 dwords past a multiple of the 64
// banks: 16 consecutive rows start on 16 distinct 4-bank groups).  The
// operand reads add row offsets that are multiples of 4 rows to a per-lane
// base, so those stay compile-time immediates.
template <int D>
struct GTile {
  static constexpr int P1 = (D / 2) % 32 == 16 ? D : D + 32;
  static constexpr int P2 = 4 * P1 + 8;
  static constexpr int kElems = (kRB / 4) * P2;  // 32 rows
  static __device__ __forceinline__ int row(int r) { return (r >> 2) * P2 + (r & 3) * P1; }
};

// A operand of a 32x32x16 MFMA read transposed from a GTile (columns c0 +
// l % 32 as the row index, tile rows k0 .. k0+15 as the reduction index in
// the relabelled order of the C layout; k0 a multiple of 4), as tr_operand
// does for a fixed row stride.
template <typename T, int D>
__device__ __forceinline__ typename Mfma<T>::v8 tr_operand_g(const T *tile, int k0, int c0,
                                                             int lane) {
  using L = GTile<D>;
  const int i = lane & 15, g = lane >> 4;
  const T *p = tile + (k0 >> 2) * L::P2 + L::row(4 * (g >> 1) + (i >> 2)) + c0 + (g & 1) * 16 +
               4 * (i & 3);
  return as_v8<T>(join(lds_tr16(p), lds_tr16(p + 2 * L::P2)));
}

template <int D>
struct DkvSmem {
  static constexpr int kQs = GTile<D>::kElems;                // Q (or dO) rows
  static constexpr int kBufBytes = 2 * kQs * 2 + 2 * kRB * 4;  // Q, dO, LSE, delta
  // + the span of the last full-width DMA instruction past its tile (the
  // instruction's masked lanes write nothing, the slack is never touched)
  static constexpr int kBytes = 2 * kBufBytes + 1024;
};

// Dynamic LDS of the dK/dV kernel: the query-block buffers, or the per-wave
// row-store regions of the epilogue if those are larger (D = 128 on 8 waves).
template <typename T, int D, int NW>
constexpr int dkv_lds_bytes() {
  constexpr int kNDO = D / 32 / (D >= 256 ? 2 : 1);
  constexpr int kStage = NW * StagedRows<T, kNDO>::kBytes;
  constexpr int kBase = DkvSmem<D>::kBytes > kStage ? DkvSmem<D>::kBytes : kStage;
  // D = 256: the partial S / dP exchange region after the query-block buffers
  return D >= 256 ? DkvSmem<D>::kBytes + NW * 64 * 32 * 4 : kBase;
}

// LDS-DMA of one head's rows [r0, r0 + 32) of a [T, H, D] tensor (rows at or
// past r_end read as zero) into a GTile block: wave w of NW moves
// rows RPW*w .. RPW*w + RPW-1 (RPW = 32/NW), one instruction per row with
// lanes < D/8 active.  One buffer descriptor covers the block's valid rows;
// the row sits in the lane offset.
template <typename T, int D, int NW>
__device__ __forceinline__ void dma_rows(const T *src, int r0, int r_end, int H, int h,
                                         uint32_t base, int wave, int lane) {
  constexpr int RPW = kRB / NW;
  const int rows = uniform_clamp(r_end - r0, kRB);
  const u32x4 rs = rsrc_words32(src + (int64_t)r0 * H * D, (uint32_t)(rows * H * D * 2));
  const int off = (wave * RPW * H + h) * D * 2 + lane * 16;
  if (lane < D / 8) {
#pragma unroll
    for (int n = 0; n < RPW; ++n) {
      // one add of a scalar row term (volatile: not hoisted into RPW registers)
      int voff;
      asm volatile("v_add_u32 %0, %1, %2" : "=v"(voff) : "s"(n * H * D * 2), "v"(off));
      lds_dma16(rs, base + GTile<D>::row(wave * RPW + n) * 2, voff);
    }
  }
}

// Query-block staging of the dK/dV and fused kernels: full width at D <= 64.
template <typename T, int D, int NW>
__device__ __forceinline__ void dma_block_rows(const T *src, int r0, int r_end, int H, int h,
                                               uint32_t base, int wave, int lane);

// The same block by full-width LDS-DMA: the instruction with index i writes
// the tile's LDS bytes [1024 i, 1024 i + 1024), lane l the 16 bytes at
// 1024 i + 16 l, so each lane fetches the (row, 16-byte chunk) that the GTile
// layout places there; lanes whose position is row padding or past the tile
// are masked off.  ceil(tile bytes / 1 KiB) instructions per block instead of
// one per row (D = 64: 6 against 32 with 8 of 64 lanes active).  Measured on
// the MI355X (A/B in one call): stage-1 replay (H=4, D=64) fwd+bwd 4.98 ->
// 4.61 ms; C2's D=128 dK/dV kernel (8 waves, 256-key tiles) 0.93 -> 0.97 ms,
// so D >= 128 keeps one instruction per row (16 or 32 active lanes).
template <typename T, int D, int NW>
__device__ __forceinline__ void dma_rows_wide(const T *src, int r0, int r_end, int H, int h,
                                              uint32_t base, int wave, int lane) {
  using L = GTile<D>;
  constexpr int kInstr = (L::kElems / 8 + 63) / 64;
  const int rows = uniform_clamp(r_end - r0, kRB);
  const u32x4 rs = rsrc_words32(src + (int64_t)r0 * H * D, (uint32_t)(rows * H * D * 2));
  for (int i = wave; i < kInstr; i += NW) {
    const int e = (i * 64 + lane) * 8;       // element offset of this lane's 16 bytes
    const int g = e / L::P2, w = e - g * L::P2;
    const int j = w / L::P1, wr = w - j * L::P1;
    if (e < L::kElems && j < 4 && wr < D) {
      // rows at or past `rows` lie past the descriptor's range: zeros
      const int voff = (((4 * g + j) * H + h) * D + wr) * 2;
      lds_dma16(rs, base + i * 1024, voff);
    }
  }
}

template <typename T, int D, int NW>
__device__ __forceinline__ void dma_block_rows(const T *src, int r0, int r_end, int H, int h,
                                               uint32_t base, int wave, int lane) {
  if constexpr (D <= 64)
    dma_rows_wide<T, D, NW>(src, r0, r_end, H, h, base, wave, lane);
  else
    dma_rows<T, D, NW>(src, r0, r_end, H, h, base, wave, lane);
}

// A [kRB x D] block of a [T, H, D] tensor staged through registers: 16-byte
// chunks, rows past the buffer range read as zero.
template <int D, int NT>
struct Rows {
  static constexpr int kChunks = kRB * D / 8;
  static constexpr int kPer = (kChunks + NT - 1) / NT;
  u32x4 v[kPer];
};

template <typename T, int D, int NT>
__device__ __forceinline__ void load_rows(Rows<D, NT> &s, const T *__restrict__ src, int r0,
                                          int r_end, int H, int h, int t) {
  constexpr int CPR = D / 8;
  const int rows = uniform_clamp(r_end - r0, kRB);
  const rsrc_t rs = make_rsrc32(src + (int64_t)r0 * H * D, (uint32_t)(rows * H * D * 2));
#pragma unroll
  for (int i = 0; i < Rows<D, NT>::kPer; ++i) {
    const int ci = t + NT * i;
    const int row = ci < Rows<D, NT>::kChunks ? ci / CPR : kRB;
    s.v[i] = buf_load16(rs, (row * H + h) * D * 2 + (ci % CPR) * 16);
  }
}

template <typename T, int D, int NT>
__device__ __forceinline__ void store_rows(const Rows<D, NT> &s, T *dst, int t) {
  constexpr int CPR = D / 8;
#pragma unroll
  for (int i = 0; i < Rows<D, NT>::kPer; ++i) {
    const int ci = t + NT * i;
    if (ci < Rows<D, NT>::kChunks)
      *reinterpret_cast<u32x4 *>(dst + GTile<D>::row(ci / CPR) + (ci % CPR) * 8) = s.v[i];
  }
}

template <int D>
struct DqSmem {
  static constexpr int kKs = GTile<D>::kElems;
  static constexpr int kBuf = 2 * kKs;  // K and V row-major
  static constexpr int kBytes = 2 * kBuf * 2;
};

}  // namespace

}  // namespace vafa
