// The forward's step over a tile of keys: scores, online softmax and the product with V for
// a wave's 32 query rows, under the mask and the score transforms of masked.h.
//
// S^T = K Q^T and O^T += V^T P^T over 64 keys in LDS (fwd_tiles.h), with a lazily updated
// running maximum.
#pragma once
#include <cstddef>
#include <type_traits>

#include "fwd_tiles.h"
#include "masked.h"
#include "mfma.h"

namespace vafa {

namespace {

// A tile's K and V rows in LDS as the operands of its products: k(kt, cc), the A operand of
// keys 32 kt + l % 32 and features 16 cc + 8 (l / 32) .. + 7, and v(km, dt), that of
// features 32 dt .. + 31 and keys 16 km .. + 15 in the order of the C layout (mfma.h).
template <typename T, int D>
struct PaddedTile {  // rows with FwdSmem's padding
  static constexpr int kKeys = kBN;
  const T *kp, *vs;
  int lane;
  __device__ __forceinline__ PaddedTile(const T *ks, const T *vs_, int lane_)
      : kp(ks + (lane_ & 31) * FwdSmem<D>::KSK + (lane_ >> 5) * 8), vs(vs_), lane(lane_) {}
  __device__ __forceinline__ u32x4 k(int kt, int cc) const {
    return *reinterpret_cast<const u32x4 *>(kp + kt * 32 * FwdSmem<D>::KSK + cc * 16);
  }
  __device__ __forceinline__ typename Mfma<T>::v8 v(int km, int dt) const {
    return tr_operand<T>(vs, FwdSmem<D>::KSV, km * 16, dt * 32, lane);
  }
};

// One tile (64 keys, or 32) for the wave's 32 query rows; masked: some (row, key) pair is hidden.
// Keys whose bit of `here` (64 bits, where a tile may lack some) is not set are hidden from every
// row (a masked tile's alone).
template <typename T, int D, bool kCap, bool kBias, typename Tile, typename Here = std::nullptr_t>
__device__ __forceinline__ void masked_tile(const Tile &tile,
                                            const typename Mfma<T>::v8 (&qf)[D / 16],
                                            f32x16 (&acc)[D / 32], float &m_run, float &l_part,
                                            const ScoreArgs &sa, float slope2, int kbase,
                                            int k_end, bool masked, int p, int pre, int window,
                                            int lane, Here here = nullptr) {
  using M = Mfma<T>;
  constexpr int NC = D / 16, ND = D / 32, KT = Tile::kKeys / 32;
  constexpr bool kLog2 = kCap || kBias;  // s holds log2-domain scores after the transform
  const int lhalf = lane >> 5;
  constexpr int kPre = 4;
  constexpr int NS = KT * NC;
  f32x16 s[KT];
#pragma unroll
  for (int kt = 0; kt < KT; ++kt)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[kt][r] = 0.f;
  auto kop = [&](int i) { return tile.k(i % KT, i / KT); };
  u32x4 ring[kPre];
#pragma unroll
  for (int i = 0; i < kPre; ++i) ring[i] = kop(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const u32x4 a = ring[i % kPre];
    s[i % KT] = M::mma(as_v8<T>(a), qf[i / KT], s[i % KT]);
    if (i + kPre < NS) ring[i % kPre] = kop(i + kPre);
    __builtin_amdgcn_sched_barrier(0);
  }
  const int k_lane = kbase + lhalf * 4;  // register (kt, r) holds key k_lane + off(kt, r)
  auto off = [](int kt, int r) { return kt * 32 + (r >> 2) * 8 + (r & 3); };
  if constexpr (kLog2) {
    const float back = (float)(p - k_lane);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float z = s[kt][r] * sa.c;
        if constexpr (kCap) z = __builtin_fmaf(-2.f * sa.cap2, cap_e(z), sa.cap2);
        if constexpr (kBias) z = __builtin_fmaf(-slope2, fabsf(back - (float)off(kt, r)), z);
        s[kt][r] = z;
      }
  }
  if (masked) {
    uint64_t seen = seen_keys(k_lane, k_end, p, pre, window);
    if constexpr (!std::is_same_v<Here, std::nullptr_t>) seen &= here >> (lhalf * 4);
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[kt][r] = where_bit((uint32_t)(seen >> 32 * kt), off(0, r), s[kt][r], kNegInf);
  }
  const float c = kLog2 ? 1.f : sa.c;
  typename M::v8 pb[KT][2];
  float ps4[4];
  // P is rounded to T, V's type, for the product; its row sum takes the rounded values, in
  // fp32, so that a constant V comes out as it is (outputs in bf16 1.8e-3 off in the 2-norm,
  // the exact ones rounded 1.7e-3)
  auto build_p = [&]() {
#pragma unroll
    for (int i = 0; i < 4; ++i) ps4[i] = 0.f;
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int mm = 0; mm < 2; ++mm) {
        typename M::v8 x;
#pragma unroll
        for (int t = 0; t < 8; ++t) {
          const float y = s[kt][mm * 8 + t];
          x[t] = static_cast<T>(
              fast_exp2(kLog2 ? y - m_run : __builtin_fmaf(y, c, -m_run)));
        }
        pb[kt][mm] = x;
#pragma unroll
        for (int t = 0; t < 4; ++t) ps4[t] = dot2_ones<T>(x, t, ps4[t]);
      }
  };
  build_p();
  float ps = (ps4[0] + ps4[1]) + (ps4[2] + ps4[3]);
  if (wave_any(!(ps <= kLazyMax))) {
    float m4[4] = {kNegInf, kNegInf, kNegInf, kNegInf};
#pragma unroll
    for (int kt = 0; kt < KT; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) m4[r & 3] = fmaxf(m4[r & 3], s[kt][r]);
    float mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
    mx = max_xor32(mx) * c;
    const float m_new = fmaxf(m_run, mx);
    const float alpha = fast_exp2(m_run - m_new);
    m_run = m_new;
    l_part *= alpha;
#pragma unroll
    for (int i = 0; i < ND; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][r] *= alpha;
    build_p();
    ps = (ps4[0] + ps4[1]) + (ps4[2] + ps4[3]);
  }
  l_part += ps;
  constexpr int NP = 2 * KT * ND;
  auto vop = [&](int i) {  // i = km * ND + dt, km = kt * 2 + mm
    return tile.v(i / ND, i % ND);
  };
  typename M::v8 vring[kPre];
#pragma unroll
  for (int i = 0; i < kPre; ++i) vring[i] = vop(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const typename M::v8 a = vring[i % kPre];
    const int km = i / ND, dt = i % ND;
    acc[dt] = M::mma(a, pb[km >> 1][km & 1], acc[dt]);
    if (i + kPre < NP) vring[i % kPre] = vop(i + kPre);
    __builtin_amdgcn_sched_barrier(0);
  }
}

}  // namespace

}  // namespace vafa
