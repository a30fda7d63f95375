// Places and rotations of packed tokens: which sequence a token belongs to, where the
// paged cache keeps it, and the turns of its feature pairs.
#pragma once
#include "kernels.h"
#include "mfma.h"

namespace vafa {

namespace {

// Sequence of token t: the number of cu[1..n] that are at most t (n: none, the
// token lies behind the last one).  Every lane of the wave calls it.
__device__ __forceinline__ int seq_of(const int32_t *cu, int n, int t, int lane) {
  int b = 0;
#pragma unroll 4
  for (int c = 0; c < n; c += 64) {  // (several loads on their way)
    const bool le = c + lane < n && cu[1 + c + lane] <= t;
    b += __popcll(__builtin_amdgcn_ballot_w64(le));
  }
  return b;
}

struct TokenAt {
  int pos;           // position, -1: no sequence holds the token
  int64_t k_off, v_off;  // where it goes, in elements (k_off < 0: nowhere)
  int id, slot;          // its page and its place there
};

__device__ __forceinline__ TokenAt token_at(const AppendArgs &a, int t, int lane) {
  TokenAt at{-1, -1, -1, -1, 0};
  int b = t, i = 0;
  if (a.cu != nullptr) {
    b = seq_of(a.cu, a.n_seq, t, lane);
    if (b < a.n_seq) i = t - a.cu[b];
  }
  if (b >= a.n_seq || i < 0) return at;  // (i < 0: a token in front of cu[0])
  const int64_t pos = (int64_t)a.lens[b] + i;
  if (pos < 0 || pos > INT32_MAX) return at;
  at.pos = (int)pos;
  const PageSlot s = page_slot(a.map, at.pos);
  const int id = page_of(a.map, b, at.pos, s);
  if (id >= 0) {
    at.id = id;
    at.slot = s.slot;
    at.k_off = id * a.k_page + s.slot * a.kc_token;
    at.v_off = id * a.v_page + s.slot * a.vc_token;
  }
  return at;
}

__device__ __forceinline__ float2 turn_of(int pos, float inv_freq) {
  const double turns = (double)pos * (double)inv_freq * 0.15915494309189533577;
  float s, c;
  sincospif(2.0f * (float)(turns - rint(turns)), &s, &c);
  return make_float2(c, s);
}

}  // namespace

}  // namespace vafa
