// Key / value tiles of the forward kernels: LDS layout and staging through registers.
#pragma once
#include "mfma.h"

namespace vafa {

namespace {

constexpr int kBN = 64;  // keys per LDS tile
// LDS row padding (elements).  K is read by ds_read_b128 (rows as the A
// operand) and V only by ds_read_b64_tr_b16 (V^T operands); measured on
// gfx950 the two want different row strides: 16-byte row reads are
// conflict-free when the stride is 8 * odd elements (D + 24), the transposed
// reads when it is 32 mod 128 elements (D + 32).
constexpr int kKPad = 24;
constexpr int kVPad = 32;

template <int D>
struct FwdSmem {
  static constexpr int KSK = D + kKPad;          // K row stride (elements)
  static constexpr int KSV = D + kVPad;          // V row stride (elements)
  static constexpr int kKs = kBN * KSK;          // elements per K buffer
  static constexpr int kVs = kBN * KSV;          // elements per V buffer
  static constexpr int kBuf = kKs + kVs;         // K then V
  static constexpr int kBytes = 2 * kBuf * 2;    // double buffered, 2 B/elt
};

// Global -> register stage of one K/V tile over NT threads (zero-filled past
// k_end; at D=32 with 512 threads half of them have no chunk).
template <int D, int NT>
struct TileRegs {
  static constexpr int kTotal = kBN * D / 8;                // 16 B chunks per tensor
  static constexpr int kKChunks = (kTotal + NT - 1) / NT;   // per thread
  u32x4 kc[kKChunks];
  u32x4 vc[kKChunks];
};

template <typename T, int D, int NT>
__device__ __forceinline__ void load_tile(TileRegs<D, NT> &r, const T *__restrict__ k,
                                          const T *__restrict__ v, int kbase, int k_end, int H,
                                          int h, int tid) {
  using R = TileRegs<D, NT>;
  constexpr int CPR = D / 8;  // chunks per row
  // one buffer resource per tile: rows past k_end read as zero
  const int64_t row_bytes = (int64_t)H * D * 2;
  const int64_t nbytes = (int64_t)(k_end - kbase < kBN ? k_end - kbase : kBN) * row_bytes;
  const rsrc_t rk = make_rsrc(k + (int64_t)kbase * H * D, nbytes);
  const rsrc_t rv = make_rsrc(v + (int64_t)kbase * H * D, nbytes);
#pragma unroll
  for (int i = 0; i < R::kKChunks; ++i) {
    const int ci = tid + NT * i;
    const int key = ci < R::kTotal ? ci / CPR : kBN, dc = ci % CPR;  // kBN: past the range
    r.kc[i] = buf_load16(rk, (key * H + h) * D * 2 + dc * 16);
  }
#pragma unroll
  for (int i = 0; i < R::kKChunks; ++i) {
    const int ci = tid + NT * i;
    const int key = ci < R::kTotal ? ci / CPR : kBN, dc = ci % CPR;
    r.vc[i] = buf_load16(rv, (key * H + h) * D * 2 + dc * 16);
  }
}

template <typename T, int D, int NT>
__device__ __forceinline__ void store_tile(const TileRegs<D, NT> &r, T *ks, T *vs, int tid) {
  using R = TileRegs<D, NT>;
  constexpr int CPR = D / 8;
#pragma unroll
  for (int i = 0; i < R::kKChunks; ++i) {
    const int ci = tid + NT * i;
    if (R::kTotal % NT == 0 || ci < R::kTotal) {
      const int key = ci / CPR, dc = ci % CPR;
      *reinterpret_cast<u32x4 *>(ks + key * FwdSmem<D>::KSK + dc * 8) = r.kc[i];
      *reinterpret_cast<u32x4 *>(vs + key * FwdSmem<D>::KSV + dc * 8) = r.vc[i];
    }
  }
}

// acc + x[2t] + x[2t+1] on the dot2 unit (fp32 accumulate): the row sum of
// P as rounded for the PV product, half the instructions of fp32 adds.
template <typename T>
__device__ __forceinline__ float dot2_ones(const typename Mfma<T>::v8 &x, int t, float acc);
template <>
__device__ __forceinline__ float dot2_ones<bf16>(const bf16x8 &x, int t, float acc) {
  typedef __bf16 b2 __attribute__((ext_vector_type(2)));
  const b2 v = {x[2 * t], x[2 * t + 1]};
  return __builtin_amdgcn_fdot2_f32_bf16(v, __builtin_bit_cast(b2, 0x3f803f80u), acc, false);
}
template <>
__device__ __forceinline__ float dot2_ones<f16>(const f16x8 &x, int t, float acc) {
  typedef _Float16 h2 __attribute__((ext_vector_type(2)));
  const h2 v = {x[2 * t], x[2 * t + 1]};
  return __builtin_amdgcn_fdot2(v, __builtin_bit_cast(h2, 0x3c003c00u), acc, false);
}

}  // namespace

}  // namespace vafa
