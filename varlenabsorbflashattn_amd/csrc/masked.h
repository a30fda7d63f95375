// The mask and the score transforms of packed_masked_attn, shared by its forward and
// backward kernels.
//
// Query row r (absolute) has position p = r + diag among the absolute key indexes; it
// sees key j where j < pre or (j <= p and j > p - window).  Without the causal mask
// pre is the segment's end.  The score z = scale q.k passes through cap tanh(z / cap)
// (kCap) and loses slope |p - j| (kBias); everything runs in the log2 domain.
#pragma once
#include <type_traits>

#include "mfma.h"

namespace vafa {

namespace {

// A work item's rows against keys [k0, k1): the keys in front of `pre`, then those of
// the window, which starts at the first row's first key.
struct KeyWalk {
  int a0, a1, na;  // first range and its tiles (0: the ranges join)
  int b0, b1, n;   // second range; tiles of both
};

template <int BN>
__device__ __forceinline__ KeyWalk key_walk(int k0, int k1, int pre, int win0) {
  KeyWalk w;
  w.a0 = k0;
  w.a1 = pre < k1 ? pre : k1;
  w.b1 = k1;
  const int wl = win0 > k0 ? win0 : k0;
  if (w.a1 > k0) {
    w.na = wl > w.a1 ? (w.a1 - k0 + BN - 1) / BN : 0;
    w.b0 = w.na > 0 ? wl : k0;
  } else {
    w.na = 0;
    w.b0 = wl;
  }
  w.n = w.na + (k1 > w.b0 ? (k1 - w.b0 + BN - 1) / BN : 0);
  return w;
}
template <int BN>
__device__ __forceinline__ int walk_key(const KeyWalk &w, int j) {
  return j < w.na ? w.a0 + j * BN : w.b0 + (j - w.na) * BN;
}
__device__ __forceinline__ int walk_end(const KeyWalk &w, int j) { return j < w.na ? w.a1 : w.b1; }

// How keys [j0, j1] meet the rows at positions [p0, p1].
__device__ __forceinline__ bool none_visible(int j0, int j1, int p0, int p1, int pre, int window) {
  return j0 >= pre && (j0 > p1 || j1 <= p0 - window);
}
__device__ __forceinline__ bool all_visible(int j0, int j1, int p0, int p1, int pre, int window) {
  return j1 < pre || (j1 <= p0 && j0 > p1 - window);
}
// The keys [j, j + 64) that the row at position p sees, a bit each, those from `end` on not
// among them: once per tile, and then two instructions per score (where_bit) in place of
// four comparisons and a choice.
__device__ __forceinline__ uint64_t ones(int n) {  // the lowest n bits, none below 0
  return n <= 0 ? 0 : (n >= 64 ? ~uint64_t{0} : (uint64_t{1} << n) - 1);
}
__device__ __forceinline__ uint64_t seen_keys(int j, int end, int p, int pre, int window) {
  const int last = p + 1 < end ? p + 1 : end;
  return ones((pre < end ? pre : end) - j) | (ones(last - j) & ~ones(p - j - window + 1));
}
// x where bit i is set, else y.
__device__ __forceinline__ float where_bit(uint32_t bits, int i, float x, float y) {
  const uint32_t m = (uint32_t)__builtin_amdgcn_sbfe((int)bits, i, 1);
  return __uint_as_float((__float_as_uint(x) & m) | (__float_as_uint(y) & ~m));
}

// Factors of the score transforms.  tanh(x) = 1 - 2 e with e = 1 / (1 + 2^(2 x log2 e)),
// its derivative 4 e (1 - e); infinities of the power give 1 and -1.  The absolute error
// of e, a few 2^-24, reaches the log2-domain score as cap2 times that.
struct ScoreArgs {
  float c;     // kCap: 2 log2e scale / cap, else scale log2e
  float cap2;  // cap log2e
};
// |c| as the factor of scores that may be -inf: not 0, which would make them NaN (2^-126
// times a score below 2^100 is 0 beside any other part of the exponent).
__device__ __forceinline__ float score_factor(float c) {
  // (back to a scalar register: the scalar unit has no float max)
  return __int_as_float(
      __builtin_amdgcn_readfirstlane(__float_as_int(fmaxf(fabsf(c), 0x1p-126f))));
}
__device__ __forceinline__ float cap_e(float z) {
  return __builtin_amdgcn_rcpf(1.f + fast_exp2(z));
}

// Query heads that share a key head are rows of one tile: of the G = H / Hk heads, sets
// of gp = 2^lg (the largest power of two that divides G, at most 32) lie beside each
// other in memory, and row r of a tile is head r % gp of token r / gp.  A tile of 128
// rows then spans 128 / gp tokens: short segments fill it, and the mask's border cuts
// fewer of its (row, key) pairs.
struct HeadSets {
  int H, Hk, lg;
  __device__ __forceinline__ int sets() const { return H >> lg; }       // of all heads
  __device__ __forceinline__ int per_key() const { return (H / Hk) >> lg; }
  // set of workgroup i among an item's: consecutive ones take the same key head every
  // Hk, so that with Hk a multiple of the XCDs one XCD's L2 serves it
  __device__ __forceinline__ int set_of(int i) const { return (i % Hk) * per_key() + i / Hk; }
  // offset of local row r (in heads) from the set's first head of the tile's first token
  __device__ __forceinline__ int row(int r) const {
    return (r >> lg) * H + (r & ((1 << lg) - 1));
  }
};

// delta = rowsum(O dO) takes O better than 16 bits: where few keys carry a row, dP - delta
// is small beside either, and O's rounding shows in the gradients (distance biases of 4
// to 7 a step: dQ and dK 1.7e-2 of their norm off in bf16, 2.2e-3 so; uniform scores 2.45e-3
// and 2.35e-3).  It costs 2 to 3% of a training step.  A byte per element holds the distance of the fp32 value's bits from those of the rounded one, in units of
// 2^kLoShift: 8 more bits of the significand, at any scale.
template <typename T>
constexpr int kLoShift = std::is_same_v<T, bf16> ? 8 : 5;

template <typename T>
__device__ __forceinline__ uint32_t lo_byte(float x) {
  constexpr int S = kLoShift<T>;
  int d = __float_as_int(x) - __float_as_int(to_f(static_cast<T>(x)));
  d = (d + (1 << (S - 1))) >> S;  // (beyond a byte: half a step up, fp16's subnormals)
  return (uint32_t)(d < -128 ? -128 : (d > 127 ? 127 : d)) & 255u;
}
template <typename T>
__device__ __forceinline__ float with_lo(T h, uint32_t word, int byte) {
  const int d = (int)(word << (24 - 8 * byte)) >> 24;
  return __int_as_float(__float_as_int(to_f(h)) + (d << kLoShift<T>));
}

// Where the 8 bytes of features [16 c + 8 half, + 8) of row r lie: the rows that a wave
// takes, `rows` of the tokens from t0 on and one set, are one block, ordered by c, row
// and half, so that the forward writes and dQ reads whole lines.
template <int D>
__device__ __forceinline__ int64_t lo_at(const HeadSets &hs, int64_t t0, int set, int rows, int r,
                                         int c, int half) {
  return (t0 * hs.H + (int64_t)set * rows) * D + ((int64_t)c * rows + r) * 16 + half * 8;
}

}  // namespace

}  // namespace vafa
