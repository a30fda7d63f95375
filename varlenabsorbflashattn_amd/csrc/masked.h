// The mask and the score transforms of packed_masked_attn, shared by its forward and
// backward kernels.
//
// Query row r (absolute) has position p = r + diag among the absolute key indexes; it
// sees key j where j < pre or (j <= p and j > p - window).  Without the causal mask
// pre is the segment's end.  The score z = scale q.k passes through cap tanh(z / cap)
// (kCap) and loses slope |p - j| (kBias); everything runs in the log2 domain.
#pragma once
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
__device__ __forceinline__ bool visible(int j, int p, int pre, int window) {
  return j < pre || (j <= p && j > p - window);
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

}  // namespace

}  // namespace vafa
