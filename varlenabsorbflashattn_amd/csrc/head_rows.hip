// Rows of heads between a projection and its attention: the norm of queries and keys, the
// position rotation, rounding to 8 bits, forward and backward, and the way back from the
// pages of a cache.
//
// A row x (one token's D features of one head) becomes y = R(x r w): r = 1 / sqrt(mean x^2 +
// eps), w the weights, R the rotation of feature pairs by position * inv_freq, its sine and
// cosine times rot_scale.  All in fp32, rounded once.  Backward, with g = R^T dy and u = x r:
//   dw = sum over rows of g u,   dx = r (g w - u mean(g w u)).
// Each row is read once and written once; D / 16 lanes of a wave hold one, 16 features each, and
// its sums are exchanges between them.  Memory is the bound where rows stay in 16 bits (35k
// tokens of 32 + 8 heads of 128: forward 722 MB, 130 us, 5.6 TB/s; backward 1.08 GB, 241 us, 4.5
// TB/s; with v's 8 heads into a cache 865 MB, 178 us, 4.9 TB/s; those heads back from it 288 MB,
// 55 us, 5.3 TB/s).  Where they become codes the vector units are busy for 77% of the cycles, of
// which there are more for a byte: 794 MB in 170 us, 4.7 TB/s; 41k of such rows back 251 MB in 50
// us, 5.1 TB/s.
#include <algorithm>
#include <type_traits>

#include "fp8.h"
#include "kernels.h"
#include "mfma.h"
#include "paged_rows.h"

namespace vafa {

namespace {

// The weights of q and then k in LDS, fp32 (ones where there are none); they need not be
// aligned.
template <typename T, int D>
__device__ __forceinline__ void stage_weights(float *to, const void *q, const void *k, bool f32,
                                              int tid) {
  for (int i = tid; i < 2 * D; i += 256) {
    const void *w = i < D ? q : k;
    const int at = i < D ? i : i - D;
    to[i] = w == nullptr ? 1.f
            : f32        ? static_cast<const float *>(w)[at]
                         : to_f(static_cast<const T *>(w)[at]);
  }
}
__device__ __forceinline__ void load_weights(const float *w, int at, float *f) {
  const f32x4 x = *reinterpret_cast<const f32x4 *>(w + at);
  const f32x4 y = *reinterpret_cast<const f32x4 *>(w + at + 4);
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    f[e] = x[e];
    f[4 + e] = y[e];
  }
}
// A lane's two pieces x as floats.
template <typename T>
__device__ __forceinline__ void unpack_row(const u32x4 (&x)[2], float *f) {
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const auto v = as_v8<T>(x[h]);
#pragma unroll
    for (int e = 0; e < 8; ++e) f[8 * h + e] = to_f(v[e]);
  }
}
template <typename T>
__device__ __forceinline__ u32x4 pack_row(const float *f) {
  typename Mfma<T>::v8 x;
#pragma unroll
  for (int e = 0; e < 8; ++e) x[e] = from_f<T>(f[e]);
  return __builtin_bit_cast(u32x4, x);
}

// Sum and maximum over the U lanes of a row (4, 8 or 16, rows aligned to them): neighbours,
// pairs, then mirrored halves and rows of 16 lanes, whose partial results are alike on both
// sides; in registers, without the LDS round trip of a shuffle.
template <int U, typename X, typename F>
__device__ __forceinline__ X row_reduce(X x, F f) {
  auto with = [&](auto ctrl) {
    return f(x, __builtin_bit_cast(X, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x),
                                                              decltype(ctrl)::value, 0xf, 0xf, true)));
  };
  x = with(std::integral_constant<int, 0xb1>{});                        // lanes 1 0 3 2 of 4
  x = with(std::integral_constant<int, 0x4e>{});                        // lanes 2 3 0 1 of 4
  if constexpr (U >= 8) x = with(std::integral_constant<int, 0x141>{});   // 8 lanes mirrored
  if constexpr (U >= 16) x = with(std::integral_constant<int, 0x140>{});  // 16 lanes mirrored
  return x;
}
template <int U>
__device__ __forceinline__ float row_sum(float x) {
  return row_reduce<U>(x, [](float a, float b) { return a + b; });
}
template <int U>
__device__ __forceinline__ uint32_t row_max(uint32_t x) {
  return row_reduce<U>(x, [](uint32_t a, uint32_t b) { return a > b ? a : b; });
}

// 1 / sqrt(mean x^2 + eps) of the row, ss its sum of squares in fp32.  Squares of bf16 pass
// fp32's range on both sides (fp16's do not).  Where the mean does not stay below 2^128, or is so
// small that what fell below 2^-149 may count, the row becomes itself times `by`, the power of two
// that brings the larger of max |x| and sqrt(eps) near 1 (exact, but for features that are nothing
// beside those), and the result is that row's.  A row that holds an infinity or NaN stays: its
// result is 0 or NaN.  The branch keeps the backward's loads and sums from running beside the
// norm's (a training step of 35k tokens 369 -> 373 us).
template <typename T, int D>
__device__ __forceinline__ float row_norm(u32x4 (&x)[2], float ss, float eps, float *by) {
  float mean = ss * (1.f / D) + eps;
  *by = 1.f;
  if constexpr (std::is_same_v<T, bf16>) {
    if (!(mean >= 0x1p-90f && mean < __builtin_inff())) {
      float f[16];
      unpack_row<T>(x, f);
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t m = __float_as_uint(f[e]) & 0x7fffffffu;
        top = m > top ? m : top;
      }
      top = row_max<D / 16>(top);
      if (top < 0x7f800000u) {
        asm volatile("" : "+v"(eps));  // (its root is formed here, not kept in a register)
        const uint32_t least = __float_as_uint(sqrtf(eps));
        const uint32_t e2 = (top > least ? top : least) >> 23;
        *by = __uint_as_float((254u - (e2 < 1u ? 1u : (e2 > 253u ? 253u : e2))) << 23);
        ss = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          f[e] *= *by;
          ss += f[e] * f[e];
        }
        x[0] = pack_row<T>(f);
        x[1] = pack_row<T>(f + 8);
        mean = row_sum<D / 16>(ss) * (1.f / D) + eps * *by * *by;
      }
    }
  }
  return rsqrtf(mean);
}

// The lane's 16 features f: pieces of 8 at 8 c0 and 8 c1.  Of the first `turned` lanes of a
// row they are 8 pairs (x[i], x[8 + i]) of the two halves, or neighbours within each piece,
// and turn by cs; `sign` -1 turns back.
struct Pieces {
  int p, c0, c1;
  bool turn;
};
__device__ __forceinline__ Pieces pieces_of(int p, int turned, bool interleaved) {
  Pieces x;
  x.p = p;
  x.turn = p < turned;
  const bool split = x.turn && !interleaved;
  x.c0 = split ? p : 2 * p;
  x.c1 = split ? p + turned : 2 * p + 1;
  return x;
}
__device__ __forceinline__ void turn_pieces(float *f, const float2 *cs, bool interleaved,
                                            float sign) {
  if (interleaved) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 w = cs[e];
      const float a = f[2 * e], b = f[2 * e + 1], s = sign * w.y;
      f[2 * e] = a * w.x - b * s;
      f[2 * e + 1] = b * w.x + a * s;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float2 w = cs[e];
      const float a = f[e], b = f[8 + e], s = sign * w.y;
      f[e] = a * w.x - b * s;
      f[8 + e] = b * w.x + a * s;
    }
  }
}

struct RowPlace {  // of a token: places of its rows and their powers of two, position
  int64_t k_off, v_off, ks_off, vs_off;
  int pos, ok;  // ok: some sequence holds it
};

// The row of head `head` (of q's, then k's, then v's) of the token t behind the bases'.  By value
// and 32-bit factors: a choice between variables or kernel arguments is else made by address,
// over a copy of them in scratch.
struct RowStrides {
  uint32_t token, head;
};
template <typename T>
__device__ __forceinline__ const T *row_source(const T *q, const T *k, const T *v, RowStrides qs,
                                               RowStrides ks, RowStrides vs, int H, int Hk,
                                               uint32_t t, uint32_t head) {
  const bool is_q = head < (uint32_t)H, is_k = head < (uint32_t)(H + Hk);
  const uint32_t token = is_q ? qs.token + 0 : (is_k ? ks.token + 0 : vs.token + 0);
  const uint32_t step = is_q ? qs.head + 0 : (is_k ? ks.head + 0 : vs.head + 0);
  const uint32_t first = is_q ? 0u : (is_k ? (uint32_t)H : (uint32_t)(H + Hk));
  const uint64_t base = is_q ? (uint64_t)q : (is_k ? (uint64_t)k : (uint64_t)v);
  return reinterpret_cast<const T *>(base) + ((uint64_t)t * token + (uint64_t)(head - first) * step);
}

enum RowsTo { kCache16, kCache8, kPackedRows };

// A block takes 256 R neighbouring units of 16 features, heads of q, then k, then v of one
// token after another, asks for all their pieces, forms place and turns of the tokens that it
// meets while they are on their way, then norms, turns and stores.
template <typename T, int D, int R, int kTo>
__global__ __launch_bounds__(256, 4) void head_rows_kernel(HeadRowsArgs s, int span) {
  constexpr int U = D / 16;
  const AppendArgs &a = s.a;
  extern __shared__ __align__(16) unsigned char smem[];
  float *weights = reinterpret_cast<float *>(smem);  // [2][D]
  RowPlace *tok = reinterpret_cast<RowPlace *>(weights + 2 * D);
  float2 *turns = reinterpret_cast<float2 *>(tok + span);  // [span][half]
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int heads = a.H + a.Hk + (kTo == kPackedRows ? 0 : a.Hk), per = heads * U;
  const int half = a.rot / 2, turned = half / 8;
  const int64_t total = a.T * per, first = (int64_t)blockIdx.x * (256 * R);
  const int64_t end = total - first < 256 * R ? total : first + 256 * R;
  const int t0 = (int)(first / per), nt = (int)((end - 1) / per) - t0 + 1;

  struct Unit {
    uint32_t t, head;
    Pieces x;
  };
  const uint32_t at0 = (uint32_t)(first - (int64_t)t0 * per);
  auto unit = [&](int r) {
    const uint32_t at = at0 + r * 256 + tid, p = (uint32_t)per;
    Unit u;
    // (below 2 p + 256 R: compared with few tokens' units instead of divided, mostly)
    u.t = p >= 128 * R ? (uint32_t)(at >= p) + (at >= 2 * p) + (at >= 3 * p) : at / p;
    u.head = (at - u.t * p) / (uint32_t)U;
    u.x = pieces_of(tid % U, u.head < (uint32_t)(a.H + a.Hk) ? turned : 0, a.interleaved);
    return u;
  };
  // (32-bit factors: one instruction each)
  const T *qb = (const T *)a.q + (int64_t)t0 * a.q_token;
  const T *kb = (const T *)a.k + (int64_t)t0 * a.k_token;
  const T *vb = kTo == kPackedRows ? kb : (const T *)a.v + (int64_t)t0 * a.v_token;
  const RowStrides qs{(uint32_t)a.q_token, (uint32_t)a.q_head};
  const RowStrides ks{(uint32_t)a.k_token, (uint32_t)a.k_head};
  const RowStrides vs{(uint32_t)a.v_token, (uint32_t)a.v_head};
  u32x4 x[R][2];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    x[r][0] = x[r][1] = u32x4{0, 0, 0, 0};
    if (first + r * 256 + tid >= end) continue;
    const Unit u = unit(r);
    const T *src = row_source(qb, kb, vb, qs, ks, vs, a.H, a.Hk, u.t, u.head);
    x[r][0] = *reinterpret_cast<const u32x4 *>(src + 8 * u.x.c0);
    x[r][1] = *reinterpret_cast<const u32x4 *>(src + 8 * u.x.c1);
  }
  if constexpr (kTo == kPackedRows) {
    for (int i = tid; i < nt; i += 256)
      tok[i] = RowPlace{(int64_t)(t0 + i) * a.Hk * D, 0, 0, 0, half > 0 ? s.positions[t0 + i] : 0, 1};
  } else {
    for (int i = wave; i < nt; i += 4) {
      const TokenAt at = token_at(a, t0 + i, lane);
      const int64_t id = at.id, slot = at.slot;
      if (lane == 0)
        tok[i] = RowPlace{at.k_off, at.v_off, id * s.scales.k_page + slot * s.scales.k_token,
                          id * s.scales.v_page + slot * s.scales.v_token, at.pos, at.pos >= 0};
    }
  }
  const bool normed = s.q_weight != nullptr || s.k_weight != nullptr;
  if (normed) stage_weights<T, D>(weights, s.q_weight, s.k_weight, s.weights_f32, tid);
  if (half > 0) {
    __syncthreads();
    for (int i = tid; i < nt * half; i += 256) {
      const int t = i / half;
      const float2 w = turn_of(tok[t].pos, a.inv_freq[i - t * half]);
      turns[i] = make_float2(w.x * s.rot_scale, w.y * s.rot_scale);
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    // (rows are whole within a block's units: their lanes stay together)
    if (first + r * 256 + tid >= end) continue;
    const Unit u = unit(r);
    const RowPlace at = tok[u.t];
    const bool is_q = u.head < (uint32_t)a.H, is_k = !is_q && u.head < (uint32_t)(a.H + a.Hk);
    float f[16];
    unpack_row<T>(x[r], f);
    if (normed) {
      float ss = 0.f;
#pragma unroll
      for (int e = 0; e < 16; ++e) ss += f[e] * f[e];
      ss = row_sum<U>(ss);
      if ((is_q ? s.q_weight : is_k ? s.k_weight : nullptr) != nullptr) {
        float g[16], by;
        const float rn = row_norm<T, D>(x[r], ss, s.eps, &by);
        unpack_row<T>(x[r], f);
        load_weights(weights + (is_q ? 0 : D), 8 * u.x.c0, g);
        load_weights(weights + (is_q ? 0 : D), 8 * u.x.c1, g + 8);
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = f[e] * rn * g[e];
      }
    }
    if (u.x.turn)
      turn_pieces(f, turns + u.t * half + (a.interleaved ? u.x.c0 / 2 : u.x.c0) * 8, a.interleaved,
                  1.f);
    if (is_q) {
      T *dst = (T *)a.q_out + ((int64_t)(t0 + u.t) * a.H + u.head) * D;
      const u32x4 z = u32x4{0, 0, 0, 0};
      *reinterpret_cast<u32x4 *>(dst + 8 * u.x.c0) = at.ok ? pack_row<T>(f) : z;
      *reinterpret_cast<u32x4 *>(dst + 8 * u.x.c1) = at.ok ? pack_row<T>(f + 8) : z;
      continue;
    }
    if (at.k_off < 0) continue;
    const int h = is_k ? u.head - a.H : u.head - a.H - a.Hk;
    const int64_t to = is_k ? at.k_off + h * a.kc_head : at.v_off + h * a.vc_head;
    if constexpr (kTo == kCache8) {
      // |x| as integers, which are ordered alike, infinities and NaN behind all others
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const uint32_t m = __float_as_uint(f[e]) & 0x7fffffffu;
        top = m > top ? m : top;
      }
      top = row_max<U>(top);
      float limit;
      int e2 = row_exponent<T>(__uint_as_float(top), &limit);
      uint8_t *dst = (uint8_t *)(is_k ? a.kc : a.vc) + to;
      if (top < 0x7f800000u && limit == 448.f) {
        const float inv = __uint_as_float((uint32_t)(127 - e2) << 23);
        *reinterpret_cast<u32x2 *>(dst + 8 * u.x.c0) = to_codes(f, inv);
        *reinterpret_cast<u32x2 *>(dst + 8 * u.x.c1) = to_codes(f + 8, inv);
      } else {  // something that is not finite, or the type's last binade
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < 16; ++e)
          amax = fabsf(f[e]) < __builtin_inff() ? fmaxf(amax, fabsf(f[e])) : amax;
        amax = __uint_as_float(row_max<U>(__float_as_uint(amax)));
        e2 = row_exponent<T>(amax, &limit);
        const float inv = __uint_as_float((uint32_t)(127 - e2) << 23);
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = to_code_range(f[e], inv, limit);
        *reinterpret_cast<u32x2 *>(dst + 8 * u.x.c0) = to_codes(f, 1.f);
        *reinterpret_cast<u32x2 *>(dst + 8 * u.x.c1) = to_codes(f + 8, 1.f);
      }
      if (u.x.p == 0) {
        uint8_t *sc = is_k ? s.scales.k + at.ks_off + h * s.scales.k_head
                           : s.scales.v + at.vs_off + h * s.scales.v_head;
        *sc = (uint8_t)(e2 + 127);
      }
    } else {
      T *dst = (T *)(is_k ? a.kc : a.vc) + to;
      *reinterpret_cast<u32x4 *>(dst + 8 * u.x.c0) = pack_row<T>(f);
      *reinterpret_cast<u32x4 *>(dst + 8 * u.x.c1) = pack_row<T>(f + 8);
    }
  }
}

// ---- backward of packed rows -------------------------------------------------------
// A block walks runs of 256 units, all blocks beside each other, and sums the weights'
// gradients of its rows in registers (a thread's features are the same in every run, which
// holds whole rows); its sums go to memory as they are, and the blocks' are added in order.
template <typename T, int D>
__global__ __launch_bounds__(256, 4) void head_rows_bwd_kernel(HeadRowsBwdArgs a, int span,
                                                               int runs) {
  constexpr int U = D / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  float *weights = reinterpret_cast<float *>(smem);  // [2][D]
  int *pos = reinterpret_cast<int *>(weights + 2 * D);
  float2 *turns = reinterpret_cast<float2 *>(pos + ((span + 3) & ~3));  // [span][half]
  __shared__ __align__(16) float red[256][17];
  const int tid = threadIdx.x;
  const int per = (a.H + a.Hk) * U, half = a.rot / 2, turned = half / 8;
  const int64_t total = a.T * per;
  const Pieces x = pieces_of(tid % U, turned, a.interleaved);
  float sum_q[16], sum_k[16];
#pragma unroll
  for (int e = 0; e < 16; ++e) sum_q[e] = sum_k[e] = 0.f;

  const bool normed = a.q_weight != nullptr || a.k_weight != nullptr;
  if (normed) stage_weights<T, D>(weights, a.q_weight, a.k_weight, a.weights_f32, tid);
  struct Run {  // of this thread: token of the run's first, head, rows of x and dy
    int t0, nt, t, head;
    bool ok;
    u32x4 x[2], dy[2];
  };
  auto load = [&](int i) {
    Run r;
    const int64_t first = ((int64_t)i * gridDim.x + blockIdx.x) * 256;
    r.ok = i < runs && first + tid < total;
    if (i >= runs || first >= total) {
      r.nt = 0;
      return r;
    }
    const int64_t end = total - first < 256 ? total : first + 256;
    r.t0 = (int)(first / per);
    r.nt = (int)((end - 1) / per) - r.t0 + 1;
    const int at = (int)(first - (int64_t)r.t0 * per) + tid;
    r.t = at / per;
    r.head = (at - r.t * per) / U;
    if (r.ok) {
      const int64_t tt = r.t0 + r.t;
      const bool is_q = r.head < a.H;
      const T *src = is_q ? (const T *)a.q + tt * a.q_token + r.head * a.q_head
                          : (const T *)a.k + tt * a.k_token + (r.head - a.H) * a.k_head;
      const T *dy = is_q ? (const T *)a.dq_out + (tt * a.H + r.head) * D
                         : (const T *)a.dk_out + (tt * a.Hk + r.head - a.H) * D;
      r.x[0] = *reinterpret_cast<const u32x4 *>(src + 8 * x.c0);
      r.x[1] = *reinterpret_cast<const u32x4 *>(src + 8 * x.c1);
      r.dy[0] = *reinterpret_cast<const u32x4 *>(dy + 8 * x.c0);
      r.dy[1] = *reinterpret_cast<const u32x4 *>(dy + 8 * x.c1);
    }
    return r;
  };
  Run next = load(0);
  for (int i = 0; i < runs && next.nt > 0; ++i) {
    Run r = next;
    next = load(i + 1);
    __syncthreads();  // the turns of the run before have been read (at first: the weights are there)
    if (half > 0) {
      for (int j = tid; j < r.nt; j += 256) pos[j] = a.positions[r.t0 + j];
      __syncthreads();
      for (int j = tid; j < r.nt * half; j += 256) {
        const int tj = j / half;
        const float2 w = turn_of(pos[tj], a.inv_freq[j - tj * half]);
        turns[j] = make_float2(w.x * a.rot_scale, w.y * a.rot_scale);
      }
      __syncthreads();
    }
    if (!r.ok) continue;  // (whole rows; the barriers above are met by all)
    const bool is_q = r.head < a.H, of_norm = (is_q ? a.q_weight : a.k_weight) != nullptr;
    float rn = 1.f, by = 1.f;
    if (of_norm) {
      float ss = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const auto v = as_v8<T>(r.x[h]);
#pragma unroll
        for (int e = 0; e < 8; ++e) ss += to_f(v[e]) * to_f(v[e]);
      }
      rn = row_norm<T, D>(r.x, row_sum<U>(ss), a.eps, &by);
    }
    float f[16], g[16];
    unpack_row<T>(r.x, f);
    unpack_row<T>(r.dy, g);
    if (x.turn)
      turn_pieces(g, turns + r.t * half + (a.interleaved ? x.c0 / 2 : x.c0) * 8, a.interleaved,
                  -1.f);
    if (of_norm) {
      float gu = 0.f, ws[16];
      load_weights(weights + (is_q ? 0 : D), 8 * x.c0, ws);
      load_weights(weights + (is_q ? 0 : D), 8 * x.c1, ws + 8);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        f[e] *= rn;
        const float p = g[e] * f[e];
        if (is_q)
          sum_q[e] += p;
        else
          sum_k[e] += p;
        gu += p * ws[e];
      }
      const float mean = row_sum<U>(gu) * (1.f / D);
#pragma unroll
      for (int e = 0; e < 16; ++e) g[e] = rn * (g[e] * ws[e] - f[e] * mean);
      if (by != 1.f) {  // (rn is that of the scaled row)
#pragma unroll
        for (int e = 0; e < 16; ++e) g[e] *= by;
      }
    }
    const int64_t tt = r.t0 + r.t;
    T *dst = is_q ? (T *)a.dq + (tt * a.H + r.head) * D
                  : (T *)a.dk + (tt * a.Hk + r.head - a.H) * D;
    *reinterpret_cast<u32x4 *>(dst + 8 * x.c0) = pack_row<T>(g);
    *reinterpret_cast<u32x4 *>(dst + 8 * x.c1) = pack_row<T>(g + 8);
  }
  if (a.part == nullptr) return;
  // features of the block's rows: thread c sums feature-slot c of the row groups, in order
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 16; ++e) red[tid][e] = side == 0 ? sum_q[e] : sum_k[e];
    __syncthreads();
    for (int c = tid; c < D; c += 256) {
      const int p = c / 16, e = c % 16;
      float sum = 0.f;
      for (int g = 0; g < 256 / U; ++g) sum += red[g * U + p][e];
      const Pieces y = pieces_of(p, turned, a.interleaved);
      a.part[((int64_t)blockIdx.x * 2 + side) * D + 8 * (e < 8 ? y.c0 : y.c1) + e % 8] = sum;
    }
  }
}

// Sums of the blocks' partial gradients, in order: a workgroup per 16 features of one weight.
template <typename T>
__global__ __launch_bounds__(256) void head_rows_dw_kernel(HeadRowsBwdArgs a) {
  __shared__ float red[16][17];
  const int per = a.D / 16, side = blockIdx.x / per, c = blockIdx.x % per * 16 + threadIdx.x % 16;
  const int g = threadIdx.x / 16;
  void *out = side == 0 ? a.dq_weight : a.dk_weight;
  if (out == nullptr) return;
  float sum = 0.f;
#pragma unroll 4
  for (int64_t b = g; b < a.blocks; b += 16) sum += a.part[(b * 2 + side) * a.D + c];
  red[g][threadIdx.x % 16] = sum;
  __syncthreads();
  if (g != 0) return;
  float all = 0.f;
#pragma unroll
  for (int i = 0; i < 16; ++i) all += red[i][threadIdx.x];
  if (a.weights_f32)
    static_cast<float *>(out)[c] = all;
  else
    static_cast<T *>(out)[c] = from_f<T>(all);
}

// ---- rows of a cache ----------------------------------------------------------------
// Output row t of sequence b is the token at starts[b] + t - cu[b], zeros where there is
// none.  256 R units of 16 features, of k's heads, then v's.
template <typename T, int R, bool kCodes>
__global__ __launch_bounds__(256) void paged_gather_kernel(GatherArgs a) {
  extern __shared__ __align__(16) unsigned char smem[];
  int2 *tok = reinterpret_cast<int2 *>(smem);  // page and slot
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  const int U = a.D / 16, per = 2 * a.Hk * U;
  const int64_t total = a.T * per, first = (int64_t)blockIdx.x * (256 * R);
  const int64_t end = total - first < 256 * R ? total : first + 256 * R;
  const int t0 = (int)(first / per), nt = (int)((end - 1) / per) - t0 + 1;
  for (int i = wave; i < nt; i += 4) {
    const int t = t0 + i, b = seq_of(a.cu, a.n_seq, t, lane);
    int id = -1, slot = 0;
    if (b < a.n_seq && t >= a.cu[b]) {
      const int64_t p = (int64_t)(a.starts != nullptr ? a.starts[b] : 0) + t - a.cu[b];
      if (p >= 0 && p <= INT32_MAX) {
        const PageSlot at = page_slot(a.map, (int)p);
        id = page_of(a.map, b, (int)p, at);
        slot = at.slot;
      }
    }
    if (lane == 0) tok[i] = make_int2(id, slot);
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < R; ++r) {
    if (first + r * 256 + tid >= end) continue;
    const int at = (int)(first - (int64_t)t0 * per) + r * 256 + tid;
    const int t = at / per, w = at - t * per, head = w / U, c = (w - head * U) * 16;
    const bool is_k = head < a.Hk;
    const int h = is_k ? head : head - a.Hk;
    const int2 place = tok[t];
    u32x4 lo = u32x4{0, 0, 0, 0}, hi = lo;
    if (place.x >= 0) {
      const int64_t from = is_k ? place.x * a.k_page + place.y * a.kc_token + h * a.kc_head
                                : place.x * a.v_page + place.y * a.vc_token + h * a.vc_head;
      const void *src = is_k ? a.kc : a.vc;
      if constexpr (kCodes) {
        const RowScales &s = a.scales;
        const uint32_t e = is_k ? s.k[place.x * s.k_page + place.y * s.k_token + h * s.k_head]
                                : s.v[place.x * s.v_page + place.y * s.v_token + h * s.v_head];
        const u32x4 codes = *reinterpret_cast<const u32x4 *>((const uint8_t *)src + from + c);
        from_codes<T>(codes, row_scale(e), lo, hi);
      } else {
        lo = *reinterpret_cast<const u32x4 *>((const T *)src + from + c);
        hi = *reinterpret_cast<const u32x4 *>((const T *)src + from + c + 8);
      }
    }
    T *dst = (T *)(is_k ? a.k : a.v) + ((int64_t)(t0 + t) * a.Hk + h) * a.D + c;
    *reinterpret_cast<u32x4 *>(dst) = lo;
    *reinterpret_cast<u32x4 *>(dst + 8) = hi;
  }
}

// Most tokens that `units` neighbouring units meet, of T tokens of `per` units.
int most_tokens(int64_t units, int64_t per, int64_t T) {
  return (int)std::min<int64_t>(T, (units + per - 2) / per + 1);
}

// Units of a thread: two from 2^19 units on, one below, where twice the blocks fill the GPU
// sooner (norms of 40 heads of 128, 5120 units one 3.8 us, two 4.7; 327680 6.8 and 7.1; 655360
// 10.9 and 10.1; 5.2 million 72.5 and 70.3).
constexpr int64_t kRowsWide = int64_t{1} << 19;

template <typename T, int D, int R, int kTo>
void launch_rows_r(const HeadRowsArgs &s, int64_t per, hipStream_t st) {
  const int64_t units = s.a.T * per;
  const int span = most_tokens(256 * R, per, s.a.T);
  const int smem = 2 * D * 4 + span * ((int)sizeof(RowPlace) + s.a.rot / 2 * 8);
  hipLaunchKernelGGL((head_rows_kernel<T, D, R, kTo>),
                     dim3((unsigned)((units + 256 * R - 1) / (256 * R))), dim3(256), smem, st, s,
                     span);
}
template <typename T, int D, int kTo>
void launch_rows_to(const HeadRowsArgs &s, hipStream_t st) {
  const int64_t per = (s.a.H + s.a.Hk + (kTo == kPackedRows ? 0 : s.a.Hk)) * (D / 16);
  if (s.a.T * per >= kRowsWide) return launch_rows_r<T, D, 2, kTo>(s, per, st);
  launch_rows_r<T, D, 1, kTo>(s, per, st);
}

template <typename T, int D>
void launch_rows_d(const HeadRowsArgs &s, hipStream_t st) {
  if (s.packed) return launch_rows_to<T, D, kPackedRows>(s, st);
  if (s.scales.k != nullptr) return launch_rows_to<T, D, kCache8>(s, st);
  launch_rows_to<T, D, kCache16>(s, st);
}

template <typename T, int D>
void launch_rows_bwd_d(const HeadRowsBwdArgs &a, hipStream_t st) {
  const int64_t per = (a.H + a.Hk) * (D / 16), runs = (a.T * per + 255) / 256;
  const int span = most_tokens(256, per, a.T);
  const int smem = 2 * (int)a.D * 4 + ((span + 3) & ~3) * 4 + span * (a.rot / 2) * 8;
  const int each = a.blocks > 0 ? (int)((runs + a.blocks - 1) / a.blocks) : 0;
  if (a.blocks > 0)
    hipLaunchKernelGGL((head_rows_bwd_kernel<T, D>), dim3((unsigned)a.blocks), dim3(256), smem, st,
                       a, span, each);
  if (a.part != nullptr)
    hipLaunchKernelGGL((head_rows_dw_kernel<T>), dim3(2 * D / 16), dim3(256), 0, st, a);
}

}  // namespace

template <typename T>
void launch_head_rows(const HeadRowsArgs &s, hipStream_t st) {
  if (s.a.D == 64) return launch_rows_d<T, 64>(s, st);
  if (s.a.D == 128) return launch_rows_d<T, 128>(s, st);
  launch_rows_d<T, 256>(s, st);
}

// Blocks of the backward: at most four on each of 256 CUs, which every one fills with runs of
// 256 units (a training step of 35k tokens: 512 blocks 442 us, 1024 381, 2048 387).
int64_t head_rows_bwd_blocks(int64_t T, int64_t heads, int64_t D) {
  const int64_t runs = (T * heads * (D / 16) + 255) / 256;
  return std::max<int64_t>(1, std::min<int64_t>(runs, 1024));
}

template <typename T>
void launch_head_rows_bwd(const HeadRowsBwdArgs &a, hipStream_t st) {
  if (a.D == 64) return launch_rows_bwd_d<T, 64>(a, st);
  if (a.D == 128) return launch_rows_bwd_d<T, 128>(a, st);
  launch_rows_bwd_d<T, 256>(a, st);
}

template <typename T, int R>
void launch_gather_r(const GatherArgs &a, int64_t per, hipStream_t st) {
  const int64_t units = a.T * per;
  const int span = most_tokens(256 * R, per, a.T);
  const dim3 grid((unsigned)((units + 256 * R - 1) / (256 * R)));
  if (a.scales.k != nullptr)
    hipLaunchKernelGGL((paged_gather_kernel<T, R, true>), grid, dim3(256), span * 8, st, a);
  else
    hipLaunchKernelGGL((paged_gather_kernel<T, R, false>), grid, dim3(256), span * 8, st, a);
}

template <typename T>
void launch_paged_gather(const GatherArgs &a, hipStream_t st) {
  const int64_t per = 2 * (int64_t)a.Hk * (a.D / 16);
  if (a.T * per >= kRowsWide) return launch_gather_r<T, 2>(a, per, st);
  launch_gather_r<T, 1>(a, per, st);
}

#define VAFA_INST(T)                                                          \
  template void launch_head_rows<T>(const HeadRowsArgs &, hipStream_t);        \
  template void launch_head_rows_bwd<T>(const HeadRowsBwdArgs &, hipStream_t); \
  template void launch_paged_gather<T>(const GatherArgs &, hipStream_t);
VAFA_INST(bf16)
VAFA_INST(f16)
#undef VAFA_INST

}  // namespace vafa
