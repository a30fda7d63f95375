// Paged key-value cache: appending keys and values with the position rotation,
// and the attention of one new token over the cache.
#include <algorithm>
#include <type_traits>

#include "fp8.h"
#include "kernels.h"
#include "mfma.h"
#include "paged.h"
#include "paged_rows.h"

namespace vafa {

namespace {

// ---- append -------------------------------------------------------------------
// Token t of sequence b goes to position pos = cache_lens[b] + t - cu[b].  Feature
// pairs (x1, x2) turn by pos * inv_freq: (x1 cos - x2 sin, x2 cos + x1 sin).  The
// angle is formed in turns in 64 bits and reduced there (pos * inv_freq passes what
// 32 bits hold to a part of a turn), sine and cosine of the rest in 32 bits.

// Two 16-byte pieces of one head per unit: the piece of first and the piece of second
// halves of 8 pairs (or 8 pairs of neighbours, or 16 features behind the rotated ones).
// The units of a token are those of q's heads, then k's, then v's; a block takes 256 * R
// neighbouring units, asks for all their pieces, forms place and turns of the tokens that
// it meets while they are on their way, then turns and stores.  Memory-bound, each byte
// moved once: 35k tokens of 32 + 8 heads of 128 (866 MB) in 165 us, 5.2 TB/s, where a
// thread per pair of features takes 351 (a copy moves 4.97 TB/s).  R = 2; R = 1 (171 us
// there) below kAppendWide units, where twice the blocks fill the GPU sooner.
constexpr int64_t kAppendWide = int64_t{1} << 19;

struct AppendSmem {  // of each token: places and position, then the turns
  int64_t k_off, v_off;
  int pos, pad;
};

template <typename T, int R>
__global__ __launch_bounds__(256, 6) void paged_append_kernel(AppendArgs a, int span) {
  using v8 = typename Mfma<T>::v8;
  extern __shared__ __align__(16) unsigned char smem[];
  AppendSmem *tok = reinterpret_cast<AppendSmem *>(smem);
  float2 *turns = reinterpret_cast<float2 *>(tok + span);  // [span][half]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int uh = a.D / 16, U = (a.H + 2 * a.Hk) * uh, half = a.rot / 2, turned = half / 8;
  const int64_t total = a.T * U, first = (int64_t)blockIdx.x * (256 * R);
  const int64_t end = total - first < 256 * R ? total : first + 256 * R;
  const int t0 = (int)(first / U), nt = (int)((end - 1) / U) - t0 + 1;

  struct Unit {
    int t, head, c0, c1;  // token of the block, head of q | k | v, pieces
    bool turn;
  };
  auto unit = [&](int r) {
    // 32-bit division: the block's first unit lies within token t0
    const int at = (int)(first - (int64_t)t0 * U) + r * 256 + tid;
    Unit u;
    u.t = at / U;
    const int w = at - u.t * U;
    u.head = w / uh;
    const int p = w - u.head * uh;
    u.turn = p < turned && u.head < a.H + a.Hk;
    const bool split = p < turned && !a.interleaved;
    u.c0 = split ? p : 2 * p;
    u.c1 = split ? p + turned : 2 * p + 1;
    return u;
  };
  u32x4 x[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (first + r * 256 + tid >= end) continue;
    const Unit u = unit(r);
    const int64_t t = t0 + u.t;
    const T *src = u.head < a.H ? (const T *)a.q + t * a.q_token + u.head * a.q_head
                   : u.head < a.H + a.Hk
                       ? (const T *)a.k + t * a.k_token + (u.head - a.H) * a.k_head
                       : (const T *)a.v + t * a.v_token + (u.head - a.H - a.Hk) * a.v_head;
    x[r][0] = *reinterpret_cast<const u32x4 *>(src + 8 * u.c0);
    x[r][1] = *reinterpret_cast<const u32x4 *>(src + 8 * u.c1);
  }
  for (int i = wave; i < nt; i += 4) {
    const TokenAt at = token_at(a, t0 + i, lane);
    if (lane == 0) tok[i] = AppendSmem{at.k_off, at.v_off, at.pos, 0};
  }
  __syncthreads();
  for (int i = tid; i < nt * half; i += 256) {
    const int t = i / half;
    turns[i] = turn_of(tok[t].pos, a.inv_freq[i - t * half]);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (first + r * 256 + tid >= end) continue;
    const Unit u = unit(r);
    const AppendSmem at = tok[u.t];
    if (u.turn) {
      const float2 *cs = turns + u.t * half + (a.interleaved ? u.c0 / 2 : u.c0) * 8;
      v8 p = as_v8<T>(x[r][0]), q = as_v8<T>(x[r][1]);
      if (a.interleaved) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float2 w = cs[e], z = cs[4 + e];
          const float p0 = to_f(p[2 * e]), p1 = to_f(p[2 * e + 1]);
          const float q0 = to_f(q[2 * e]), q1 = to_f(q[2 * e + 1]);
          p[2 * e] = from_f<T>(p0 * w.x - p1 * w.y);
          p[2 * e + 1] = from_f<T>(p1 * w.x + p0 * w.y);
          q[2 * e] = from_f<T>(q0 * z.x - q1 * z.y);
          q[2 * e + 1] = from_f<T>(q1 * z.x + q0 * z.y);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float2 w = cs[e];
          const float p0 = to_f(p[e]), q0 = to_f(q[e]);
          p[e] = from_f<T>(p0 * w.x - q0 * w.y);
          q[e] = from_f<T>(q0 * w.x + p0 * w.y);
        }
      }
      x[r][0] = __builtin_bit_cast(u32x4, p);
      x[r][1] = __builtin_bit_cast(u32x4, q);
    }
    T *dst;
    if (u.head < a.H) {
      dst = (T *)a.q_out + ((int64_t)(t0 + u.t) * a.H + u.head) * a.D;
      if (at.pos < 0) x[r][0] = x[r][1] = u32x4{0, 0, 0, 0};
    } else if (at.k_off < 0) {
      continue;
    } else if (u.head < a.H + a.Hk) {
      dst = (T *)a.kc + at.k_off + (u.head - a.H) * a.kc_head;
    } else {
      dst = (T *)a.vc + at.v_off + (u.head - a.H - a.Hk) * a.vc_head;
    }
    *reinterpret_cast<u32x4 *>(dst + 8 * u.c0) = x[r][0];
    *reinterpret_cast<u32x4 *>(dst + 8 * u.c1) = x[r][1];
  }
}

// Heads or rotated features that are no multiple of 16: one thread per pair of features
// (of the rotated ones, or two neighbours behind them) of one head: heads of q, then k,
// then v.
template <typename T>
__global__ __launch_bounds__(256) void paged_append_pairs_kernel(AppendArgs a) {
  const int t = blockIdx.x, lane = threadIdx.x & 63, D = a.D, half = a.rot / 2;
  const TokenAt at = token_at(a, t, lane);
  const int per_head = D / 2, n = (a.H + 2 * a.Hk) * per_head;
  for (int u = threadIdx.x; u < n; u += 256) {
    const int head = u / per_head, p = u % per_head;
    int i0, i1;
    if (p < half) {
      i0 = a.interleaved ? 2 * p : p;
      i1 = a.interleaved ? i0 + 1 : p + half;
    } else {
      i0 = 2 * p;
      i1 = i0 + 1;
    }
    const T *src;
    T *dst;
    const bool is_v = head >= a.H + a.Hk;
    if (head < a.H) {
      src = (const T *)a.q + t * a.q_token + head * a.q_head;
      dst = (T *)a.q_out + ((int64_t)t * a.H + head) * D;
    } else if (!is_v) {
      src = (const T *)a.k + t * a.k_token + (head - a.H) * a.k_head;
      dst = (T *)a.kc + at.k_off + (head - a.H) * a.kc_head;
    } else {
      src = (const T *)a.v + t * a.v_token + (head - a.H - a.Hk) * a.v_head;
      dst = (T *)a.vc + at.v_off + (head - a.H - a.Hk) * a.vc_head;
    }
    if (head >= a.H && at.k_off < 0) continue;
    T x0 = src[i0], x1 = src[i1];
    if (head < a.H && at.pos < 0) {
      x0 = x1 = (T)0.f;
    } else if (!is_v && p < half) {
      const float2 cs = turn_of(at.pos, a.inv_freq[p]);
      const float f0 = to_f(x0), f1 = to_f(x1);
      x0 = from_f<T>(f0 * cs.x - f1 * cs.y);
      x1 = from_f<T>(f1 * cs.x + f0 * cs.y);
    }
    dst[i0] = x0;
    dst[i1] = x1;
  }
}

// ---- decode ----------------------------------------------------------------------
// The G query heads of a key head are the columns of 16x16x32 products (lane l:
// head l % 16):
//   S^T = K Q^T: A rows are 16 keys (lane l holds key l % 16, features (l / 16) * 8 of
//     each 32); C row (l / 16) * 4 + r;
//   O^T += V^T P^T over 32 keys: the lane's 8 probabilities are the B operand as they
//     are when slot (l / 16) * 8 + t is key 16 (t / 4) + (l / 16) * 4 + t % 4; V^T in
//     that order comes from transposing reads (over 16 keys: 4 of each, 16x16x16).
// A wave takes 32 of a tile's 128 keys, in one step or two, through registers (the next
// step's are on their way meanwhile) and its own LDS rows, and shares nothing with the
// other waves before the piece's end: no barrier in the loop.  Memory-bound, the products are far from their
// rate even with one head.  What a byte costs: rows are loaded whole (16 lanes a row at
// D = 128) and without keeping them in the caches.  32 heads of 128 on 8 key heads, 64
// sequences of 1k to 32k keys in pages of 16 (2.37 GB), us: K straight into A operands
// (16 rows by 64 bytes per instruction) 473, V by whole rows 453, both 436, both without
// keeping them 391, 6.1 TB/s (without keeping them but by 64 bytes 525: the other half
// of a 128-byte line is read again).  Three waves per SIMD by smaller registers 533.
template <typename T>
struct Mfma16;  // mma: 32 keys or features, mma4: 16 keys
template <>
struct Mfma16<bf16> {
  typedef __attribute__((__vector_size__(4 * sizeof(short)))) short s16x4;
  static __device__ __forceinline__ f32x4 mma4(u32x2 a, bf16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(s16x4, a),
                                                     __builtin_bit_cast(s16x4, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma16<f16> {
  static __device__ __forceinline__ f32x4 mma4(u32x2 a, f16x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

template <int D>
struct DecodeSmem {
  static constexpr int kVS = D + 8;   // K and V row stride (elements)
  static constexpr int kOS = D + 4;   // row stride of the waves' outputs (floats)
  // 16-key groups of a wave's step: by 16 at D = 256, where 32 leave one workgroup on a CU
  // and nothing in flight while it stores its rows (32 sequences of 500 to 8192 keys, 8
  // key heads, 138 -> 115 us); by 32 below (by 16, and more workgroups for it: D = 128 391
  // -> 406 us, D = 64 170 -> 182)
  static constexpr int kGroups = D >= 256 ? 1 : 2;
  static constexpr int kRows = 16 * kGroups;
  static constexpr int kV = 4 * 2 * kRows * kVS * 2;
  static constexpr int kO = 4 * kDecodeRows * kOS * 4;
  static constexpr int kML = kV > kO ? kV : kO;  // then m, l of each wave and row
  static constexpr int kBytes = kML + 2 * 4 * kDecodeRows * 4;
};

__device__ __forceinline__ int wave_sum_i(int v) {
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
__device__ __forceinline__ int wave_scan_i(int v, int lane) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) {
    const int u = __shfl_up(v, o, 64);
    if (lane >= o) v += u;
  }
  return v;
}

__device__ __forceinline__ int seq_tiles(const DecodeArgs &a, int b) {
  return b < a.n_seq ? decode_tiles(clip_len(a.lens[b], a.capacity), a.window) : 0;
}
// Tiles of all sequences (of one pair each).
__device__ __forceinline__ int all_tiles(const DecodeArgs &a, int lane) {
  int total = 0;
  for (int c = 0; c < a.n_seq; c += 64) total += seq_tiles(a, c + lane);
  return wave_sum_i(total);
}
// The sequence whose tiles hold tile `at` of the axis, and the tiles in front of it.
__device__ __forceinline__ void find_seq(const DecodeArgs &a, int at, int lane, int *b, int *base) {
  int before = 0;
  for (int c = 0; c < a.n_seq; c += 64) {
    const int t = seq_tiles(a, c + lane);
    const int incl = wave_scan_i(t, lane) + before;
    const uint64_t past = __builtin_amdgcn_ballot_w64(incl > at);
    if (past != 0) {
      const int f = __builtin_ctzll(past);
      *b = c + f;
      *base = __shfl(incl - t, f, 64);
      return;
    }
    before = __shfl(incl, 63, 64);
  }
  *b = a.n_seq;
  *base = before;
}

// kCodes: rows of 8-bit codes, which become T on the way into LDS.
template <typename T, int D, bool kCodes>
__global__ __launch_bounds__(256, D >= 128 ? 2 : 3) void paged_decode_kernel(DecodeArgs a) {
  using E = std::conditional_t<kCodes, uint8_t, T>;  // of the cache
  using M = Mfma16<T>;
  using S = DecodeSmem<D>;
  using v8 = typename Mfma<T>::v8;
  constexpr int NC = D / 32, ND = D / 16;
  constexpr int kPiece = 16 / (int)sizeof(E);         // features of 16 bytes
  constexpr int kLanes = D / kPiece, kRows = 64 / kLanes;  // of a row, and rows of an instruction
  constexpr int KG = S::kGroups, NI = S::kRows / kRows;  // instructions of a step's K rows
  constexpr int kSteps = 2 / KG;                         // of a tile
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  T *ks = reinterpret_cast<T *>(smem) + wave * 2 * S::kRows * S::kVS, *vs = ks + S::kRows * S::kVS;

  // the pairs of a chunk on one XCD: they read whole token rows of the pages together
  const int group = blockIdx.x / (kXcds * a.pairs), within = blockIdx.x % (kXcds * a.pairs);
  const int chunk = group * kXcds + within % kXcds, pair = within / kXcds;
  if (chunk >= a.chunks) return;
  const int hk = pair / a.head_blocks, hb = pair - hk * a.head_blocks;
  const int h0 = hk * a.G + hb * kDecodeRows;
  const int rows = a.G - hb * kDecodeRows < kDecodeRows ? a.G - hb * kDecodeRows : kDecodeRows;
  int b = chunk, base = 0, cur = 0, end = 0, per = 0;
  if (a.direct) {  // a chunk is a sequence
    end = __builtin_amdgcn_readfirstlane(seq_tiles(a, b));
    if (end == 0) {
      for (int e = tid; e < rows * D; e += 256)
        ((T *)a.out)[((int64_t)b * a.H + h0) * D + e] = (T)0.f;
      return;
    }
  } else {
    const int total = __builtin_amdgcn_readfirstlane(all_tiles(a, lane));
    per = decode_per(total, a.chunks);
    const int64_t first = (int64_t)chunk * per;
    if (first >= total) return;
    cur = (int)first;
    end = total - cur < per ? total : cur + per;
    find_seq(a, cur, lane, &b, &base);
    b = __builtin_amdgcn_readfirstlane(b);
    base = __builtin_amdgcn_readfirstlane(base);
  }

  while (cur < end) {
    const int len = __builtin_amdgcn_readfirstlane(clip_len(a.lens[b], a.capacity));
    const int nt = decode_tiles(len, a.window);
    if (nt == 0) {
      ++b;
      continue;
    }
    const int t0 = cur - base;
    const int run = end - cur < nt - t0 ? end - cur : nt - t0;
    const int lo = len - decode_seen(len, a.window);
    const E *kc = (const E *)a.kc + hk * a.kc_head + lane % kLanes * kPiece;
    const E *vc = (const E *)a.vc + hk * a.vc_head + lane % kLanes * kPiece;

    v8 qf[NC];
    {
      const T *qr = (const T *)a.q + b * a.q_token + (h0 + (l16 < rows ? l16 : 0)) * a.q_head + lg * 8;
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        u32x4 x = *reinterpret_cast<const u32x4 *>(qr + 32 * c);
        if (l16 >= rows) x = u32x4{0, 0, 0, 0};
        qf[c] = as_v8<T>(x);
      }
    }
    float slope2 = 0.f;
    if (a.slopes != nullptr) slope2 = a.slopes[h0 + (l16 < rows ? l16 : 0)] * kLog2e;

    auto keys_at = [&](int u) {  // the first key of step u (of the wave's 32 in tile u / kSteps)
      return lo + u / kSteps * kDecodeTile + wave * 32 + u % kSteps * S::kRows;
    };
    f32x4 acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -kHuge, l_run = 0.f;
    const int u0 = t0 * kSteps, u1 = (t0 + run) * kSteps;
    // the scores, softmax and product with V of step u, whose rows are in LDS; ok: which of
    // its keys there are (bit: key)
    auto attend = [&](int u, uint32_t ok) {
      f32x4 s[KG];
#pragma unroll
      for (int i = 0; i < KG; ++i) {
        s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c)
          s[i] = M::mma(as_v8<T>(*reinterpret_cast<const u32x4 *>(ks + (16 * i + l16) * S::kVS +
                                                                  32 * c + lg * 8)),
                        qf[c], s[i]);
      }
      // scores in the log2 domain; C row (key) 16 i + lg * 4 + r
      float y[4 * KG], mx = kNegInf;
      const int back = len - 1 - keys_at(u);
#pragma unroll
      for (int i = 0; i < KG; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * i + lg * 4 + r;
          float z = s[i][r] * a.c;
          if (a.cap2 > 0.f) z = a.cap2 * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + fast_exp2(z)));
          if (a.slopes != nullptr)
            z -= slope2 * (float)(back - row);
          y[4 * i + r] = ok >> row & 1 ? z : kNegInf;
          mx = fmaxf(mx, y[4 * i + r]);
        }
      mx = max_xor32(max_xor16(mx));
      const float m_new = fmaxf(m_run, mx), alpha = fast_exp2(m_run - m_new);
      m_run = m_new;
      typedef __attribute__((__vector_size__(4 * KG * sizeof(T)))) T VP;
      VP p;
      float ps = 0.f;
#pragma unroll
      for (int e = 0; e < 4 * KG; ++e) {
        const float x = fast_exp2(y[e] - m_run);
        // rounded to T, V's type, for the product; the sum takes the rounded values, in fp32
        // (outputs 0.52 of half a step off in the 2-norm, 0.42 of it their own rounding)
        p[e] = static_cast<T>(x);
        ps += to_f(p[e]);
      }
      l_run = l_run * alpha + ps;
#pragma unroll
      for (int i = 0; i < ND; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= alpha;
        const T *tr = vs + (lg * 4 + (l16 >> 2)) * S::kVS + 16 * i + 4 * (l16 & 3);
        if constexpr (KG == 2)
          acc[i] = M::mma(as_v8<T>(join(lds_tr16(tr), lds_tr16(tr + 16 * S::kVS))), p, acc[i]);
        else
          acc[i] = M::mma4(lds_tr16(tr), p, acc[i]);
      }
    };
    if constexpr (!kCodes) {
      // this lane's key of each group of a step: page and token in it
      struct Keys {
        int id[KG], slot[KG];
      };
      auto keys_of = [&](int u) {
        Keys k;
#pragma unroll
        for (int i = 0; i < KG; ++i) {
          const int t = u / kSteps, key = keys_at(u) + 16 * i + l16;
          const PageSlot s = page_slot(a.map, key);
          k.id[i] = t < t0 + run && key < len ? page_of(a.map, b, key, s) : -1;
          k.slot[i] = s.slot;
        }
        return k;
      };
      // the step's rows of K and V by whole rows: instruction i takes the rows i * kRows +
      // lane / kLanes, whose places the lanes that looked them up hand over
      u32x4 kr[NI], vr[NI];
      auto load = [&](const Keys &k) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = i * kRows + lane / kLanes;
          // (the rows of one instruction lie in one group)
          const int id = __shfl(k.id[i * kRows / 16], row & 15, 64);
          const int slot = __shfl(k.slot[i * kRows / 16], row & 15, 64);
          const int64_t ko = id >= 0 ? id * a.k_page + slot * a.kc_token : 0;
          const int64_t vo = id >= 0 ? id * a.v_page + slot * a.vc_token : 0;
          kr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kc + ko));
          vr[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vc + vo));
        }
      };
      Keys now = keys_of(u0);
      load(now);
      Keys next = keys_of(u0 + 1);
      for (int u = u0; u < u1; ++u) {
        uint32_t ok = 0;
#pragma unroll
        for (int i = 0; i < KG; ++i)
          ok |= (uint32_t)(__builtin_amdgcn_ballot_w64(now.id[i] >= 0) & 0xffffu) << 16 * i;
        if (ok != 0xffffffffu >> (32 - S::kRows)) {
          // values of absent keys are whatever the cache holds: zeros instead, so that
          // their zero probabilities do not meet infinities
#pragma unroll
          for (int i = 0; i < NI; ++i)
            if (!(ok >> (i * kRows + lane / kLanes) & 1)) vr[i] = u32x4{0, 0, 0, 0};
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int at = (i * kRows + lane / kLanes) * S::kVS + lane % kLanes * 8;
          *reinterpret_cast<u32x4 *>(ks + at) = kr[i];
          *reinterpret_cast<u32x4 *>(vs + at) = vr[i];
        }
        now = next;
        if (u + 1 < u1) {
          load(now);
          next = keys_of(u + 2);
        }
        attend(u, ok);
      }
    } else {
      // Codes: rows of half the bytes, so those of two steps are on their way.  Lane l looks
      // up key l % kRows of a step, forms the offsets of its rows, and asks for the power of
      // two of K's row or V's.  Bound by memory: 64 sequences of 1k to 32k keys, 8 heads of
      // 128, 1.19 GB in 227 us, 5.2 TB/s (rows of one step on their way, offsets by the lanes
      // that load: 293); heads of 256, 332 MB in 73 us (84).
      struct Key {
        int id, slot;
      };
      auto key_of = [&](int u) {
        const int key = keys_at(u) + lane % S::kRows;
        const PageSlot s = page_slot(a.map, key);
        return Key{u < u1 && key < len ? page_of(a.map, b, key, s) : -1, s.slot};
      };
      struct Rows {
        u32x4 k[NI], v[NI];
        uint32_t e, ok;
      };
      const bool e_of_v = lane / S::kRows % 2;
      const RowScales &sc = a.scales;
      const uint8_t *es = e_of_v ? sc.v + hk * sc.v_head : sc.k + hk * sc.k_head;
      const uint32_t e_page = (uint32_t)(e_of_v ? sc.v_page : sc.k_page);
      const uint32_t e_token = (uint32_t)(e_of_v ? sc.v_token : sc.k_token);
      // (strides in 16 bytes, 32-bit factors: one instruction each)
      const uint32_t kp = (uint32_t)(a.k_page >> 4), kt = (uint32_t)(a.kc_token >> 4);
      const uint32_t vp = (uint32_t)(a.v_page >> 4), vt = (uint32_t)(a.vc_token >> 4);
      const bool alike = kp == vp && kt == vt;
      auto load = [&](Key k, Rows &r) {
        const bool there = k.id >= 0;
        const uint32_t id = there ? k.id : 0, slot = there ? k.slot : 0;
        r.e = es[(uint64_t)id * e_page + (uint64_t)slot * e_token];
        r.ok = (uint32_t)__builtin_amdgcn_ballot_w64(there) & 0xffffffffu >> (32 - S::kRows);
        const uint64_t ko = (uint64_t)id * kp + (uint64_t)slot * kt;
        const uint64_t vo = (uint64_t)id * vp + (uint64_t)slot * vt;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = i * kRows + lane / kLanes;
          const uint64_t x = __shfl((unsigned long long)ko, row, 64);
          const uint64_t y = alike ? x : (uint64_t)__shfl((unsigned long long)vo, row, 64);
          r.k[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(kc) + x);
          r.v[i] = __builtin_nontemporal_load(reinterpret_cast<const u32x4 *>(vc) + y);
        }
      };
      Key next = key_of(u0 + 2);
      auto step = [&](int u, Rows &r) {
#pragma unroll
        for (int i = 0; i < NI; ++i) {
          const int row = i * kRows + lane / kLanes, at = row * S::kVS + lane % kLanes * kPiece;
          const float ke = row_scale(__shfl(r.e, row, 64));
          const float ve = row_scale(__shfl(r.e, S::kRows + row, 64));
          u32x4 low, high;
          from_codes<T>(r.k[i], ke, low, high);
          *reinterpret_cast<u32x4 *>(ks + at) = low;
          *reinterpret_cast<u32x4 *>(ks + at + 8) = high;
          from_codes<T>(r.v[i], ve, low, high);
          if (!(r.ok >> row & 1)) low = high = u32x4{0, 0, 0, 0};  // (as in 16 bits)
          *reinterpret_cast<u32x4 *>(vs + at) = low;
          *reinterpret_cast<u32x4 *>(vs + at + 8) = high;
        }
        const uint32_t ok = r.ok;
        if (u + 2 < u1) {
          // (the page first: loads come back in order, and the next step needs it while these
          // rows may still be on their way)
          const Key after = key_of(u + 3);
          load(next, r);
          next = after;
        }
        attend(u, ok);
      };
      Rows one, two;
      load(key_of(u0), one);
      load(key_of(u0 + 1), two);
      for (int u = u0; u < u1; u += 2) {
        step(u, one);
        if (u + 1 < u1) step(u + 1, two);
      }
    }
    l_run += __shfl_xor(l_run, 16, 64);
    l_run += __shfl_xor(l_run, 32, 64);

    // the four waves' rows, joined in wave order
    float *ml = reinterpret_cast<float *>(smem + S::kML);
    float *os = reinterpret_cast<float *>(smem);
    __syncthreads();  // every wave is done with its V rows
#pragma unroll
    for (int i = 0; i < ND; ++i)
      *reinterpret_cast<f32x4 *>(os + (wave * kDecodeRows + l16) * S::kOS + 16 * i + 4 * lg) = acc[i];
    if (lg == 0) {
      ml[wave * kDecodeRows + l16] = m_run;
      ml[(4 + wave) * kDecodeRows + l16] = l_run;
    }
    __syncthreads();
    const bool whole = run == nt;
    const int64_t slot = decode_slot(chunk, base, per) * a.pairs + pair;
    for (int e = tid; e < rows * (D / 4); e += 256) {
      const int row = e / (D / 4), col = e % (D / 4) * 4;
      float m = ml[row];
#pragma unroll
      for (int w = 1; w < 4; ++w) m = fmaxf(m, ml[w * kDecodeRows + row]);
      float l = 0.f;
      f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float f = fast_exp2(ml[w * kDecodeRows + row] - m);
        l += f * ml[(4 + w) * kDecodeRows + row];
        const f32x4 x = *reinterpret_cast<const f32x4 *>(os + (w * kDecodeRows + row) * S::kOS + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) o[j] += f * x[j];
      }
      if (whole) {
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        typedef __attribute__((__vector_size__(4 * sizeof(T)))) T T4;
        T4 w;
#pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = static_cast<T>(o[j] * inv);
        *reinterpret_cast<T4 *>((T *)a.out + ((int64_t)b * a.H + h0 + row) * D + col) = w;
      } else {
        *reinterpret_cast<f32x4 *>(a.part_o + (slot * kDecodeRows + row) * D + col) = o;
        if (col == 0) {
          a.part_ml[(slot * kDecodeRows + row) * 2] = m;
          a.part_ml[(slot * kDecodeRows + row) * 2 + 1] = l;
        }
      }
    }
    __syncthreads();  // the rows are read: the next piece may write V
    cur += run;
    if (t0 + run == nt) {
      base += nt;
      ++b;
    }
  }
}

// One workgroup per (sequence, query head): joins the pieces that several workgroups
// formed; a sequence without keys gets zeros.  Threads take 8 features of every 2048 / D-th
// piece (a wave per row, piece after piece, took 20 us for 2 x 131k keys, whose rows have
// 64 pieces each), summed in a fixed order.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(DecodeArgs a) {
  constexpr int C = D / 8, kGroups = 256 / C;  // threads of a piece, pieces at once
  __shared__ __align__(16) float red[kGroups][D + 4];
  __shared__ float red_l[kGroups];
  const int tid = threadIdx.x, lane = tid & 63;
  const int b = blockIdx.x / a.H, h = blockIdx.x % a.H;
  int total = 0, base = 0;  // tiles of all sequences, and of those in front of b
  for (int c = 0; c < a.n_seq; c += 64) {
    const int t = seq_tiles(a, c + lane);
    total += t;
    if (c + lane < b) base += t;
  }
  total = wave_sum_i(total);
  base = wave_sum_i(base);
  const int nt = decode_tiles(clip_len(a.lens[b], a.capacity), a.window);
  T *out = (T *)a.out + (int64_t)blockIdx.x * D;
  if (nt == 0) {
    if (tid < D) out[tid] = (T)0.f;
    return;
  }
  const int per = decode_per(total, a.chunks);
  const int g0 = base / per, g1 = (base + nt - 1) / per;
  if (g0 == g1) return;  // one workgroup had all of it
  const int hk = h / a.G, hr = h % a.G;
  const int pair = hk * a.head_blocks + hr / kDecodeRows, r = hr % kDecodeRows;
  auto row_of = [&](int g) {
    return (decode_slot(g, base, per) * a.pairs + pair) * kDecodeRows + r;
  };
  float m = kNegInf;
  for (int g = g0 + lane; g <= g1; g += 64) m = fmaxf(m, a.part_ml[row_of(g) * 2]);
  m = wave_max(m);
  const int grp = tid / C, col = tid % C * 8;
  float l = 0.f;
  f32x4 x = f32x4{0.f, 0.f, 0.f, 0.f}, y = x;
  for (int g = g0 + grp; g <= g1; g += kGroups) {
    const int64_t at = row_of(g);
    const float f = fast_exp2(a.part_ml[at * 2] - m);
    l += f * a.part_ml[at * 2 + 1];
    const f32x4 u = *reinterpret_cast<const f32x4 *>(a.part_o + at * D + col);
    const f32x4 v = *reinterpret_cast<const f32x4 *>(a.part_o + at * D + col + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] += f * u[e];
      y[e] += f * v[e];
    }
  }
  *reinterpret_cast<f32x4 *>(&red[grp][col]) = x;
  *reinterpret_cast<f32x4 *>(&red[grp][col + 4]) = y;
  if (tid % C == 0) red_l[grp] = l;
  __syncthreads();
  if (tid < D) {
    float o = 0.f;
    l = 0.f;
    const int n = g1 - g0 + 1 < kGroups ? g1 - g0 + 1 : kGroups;
    for (int g = 0; g < n; ++g) {
      o += red[g][tid];
      l += red_l[g];
    }
    out[tid] = from_f<T>(l == 0.f ? 0.f : o / l);
  }
}

template <typename T, int D, bool kCodes>
void launch_decode_d(const DecodeArgs &a, hipStream_t st) {
  const int smem = DecodeSmem<D>::kBytes;
  allow_dynamic_lds(reinterpret_cast<const void *>(&paged_decode_kernel<T, D, kCodes>), smem);
  const int64_t wgs = (int64_t)(a.chunks + kXcds - 1) / kXcds * kXcds * a.pairs;
  hipLaunchKernelGGL((paged_decode_kernel<T, D, kCodes>), dim3((unsigned)wgs), dim3(256), smem, st,
                     a);
  if (a.direct) return;
  hipLaunchKernelGGL((paged_decode_join_kernel<T, D>), dim3((unsigned)((int64_t)a.n_seq * a.H)),
                     dim3(256), 0, st, a);
}

template <typename T, bool kCodes>
void launch_decode(const DecodeArgs &a, int D, hipStream_t st) {
  if (D == 64) return launch_decode_d<T, 64, kCodes>(a, st);
  if (D == 128) return launch_decode_d<T, 128, kCodes>(a, st);
  launch_decode_d<T, 256, kCodes>(a, st);
}

}  // namespace

template <typename T>
void launch_paged_append(const AppendArgs &a, hipStream_t st) {
  if (a.D % 16 == 0 && a.rot % 16 == 0) {
    const int64_t U = (int64_t)(a.H + 2 * a.Hk) * (a.D / 16), units = a.T * U;
    const int R = units >= kAppendWide ? 2 : 1;
    const int span = (int)std::min<int64_t>(a.T, (256 * R + U - 2) / U + 1);
    const int smem = span * ((int)sizeof(AppendSmem) + a.rot / 2 * 8);
    const dim3 grid((unsigned)((units + 256 * R - 1) / (256 * R)));
    if (R == 2)
      hipLaunchKernelGGL((paged_append_kernel<T, 2>), grid, dim3(256), smem, st, a, span);
    else
      hipLaunchKernelGGL((paged_append_kernel<T, 1>), grid, dim3(256), smem, st, a, span);
    return;
  }
  hipLaunchKernelGGL((paged_append_pairs_kernel<T>), dim3((unsigned)a.T), dim3(256), 0, st, a);
}

template <typename T>
void launch_paged_decode(const DecodeArgs &a, int D, hipStream_t st) {
  if (a.scales.k != nullptr) return launch_decode<T, true>(a, D, st);
  launch_decode<T, false>(a, D, st);
}

#define VAFA_INST(T)                                              \
  template void launch_paged_append<T>(const AppendArgs &, hipStream_t); \
  template void launch_paged_decode<T>(const DecodeArgs &, int, hipStream_t);
VAFA_INST(bf16)
VAFA_INST(f16)
#undef VAFA_INST

}  // namespace vafa
