// Paged key-value cache: appending keys and values with the position rotation,
// and the attention of one new token over the cache.
#include "kernels.h"
#include "mfma.h"
#include "paged.h"

namespace vafa {

namespace {

// ---- append -------------------------------------------------------------------
// Token t of sequence b goes to position pos = cache_lens[b] + t - cu[b].  Feature
// pairs (x1, x2) turn by pos * inv_freq: (x1 cos - x2 sin, x2 cos + x1 sin).  The
// angle is formed in turns in 64 bits and reduced there (pos * inv_freq passes what
// 32 bits hold to a part of a turn), sine and cosine of the rest in 32 bits.

// Sequence of token t: the number of cu[1..n] that are at most t (n: none, the
// token lies behind the last one).  Every lane of the wave calls it.
__device__ __forceinline__ int seq_of(const int32_t *cu, int n, int t, int lane) {
  int b = 0;
  for (int c = 0; c < n; c += 64) {
    const bool le = c + lane < n && cu[1 + c + lane] <= t;
    b += __popcll(__builtin_amdgcn_ballot_w64(le));
  }
  return b;
}

struct TokenAt {
  int pos;           // position, -1: no sequence holds the token
  int64_t k_off, v_off;  // where it goes, in elements (k_off < 0: nowhere)
};

__device__ __forceinline__ TokenAt token_at(const AppendArgs &a, int t, int lane) {
  TokenAt at{-1, -1, -1};
  int b = t, i = 0;
  if (a.cu != nullptr) {
    b = seq_of(a.cu, a.n_seq, t, lane);
    if (b < a.n_seq) i = t - a.cu[b];
  }
  if (b >= a.n_seq) return at;
  const int64_t pos = (int64_t)a.lens[b] + i;
  if (pos < 0 || pos > INT32_MAX) return at;
  at.pos = (int)pos;
  const PageSlot s = page_slot(a.map, at.pos);
  const int id = page_of(a.map, b, at.pos, s);
  if (id >= 0) {
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

// One thread per pair of features (of the rotated ones, or two neighbours behind
// them) of one head: heads of q, then k, then v.
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
//   S^T = K Q^T: A rows are 16 keys (lane l holds key l % 16, features (l / 16) * 8
//     of each 32), straight from the cache into registers; C row (l / 16) * 4 + r;
//   O^T += V^T P^T over 32 keys: the lane's 8 probabilities are the B operand as they
//     are when slot (l / 16) * 8 + t is key 16 (t / 4) + (l / 16) * 4 + t % 4; V^T in
//     that order comes from transposing reads of the wave's own LDS rows.
// A wave takes 32 of a tile's 128 keys and shares nothing with the others before the
// piece's end: no barrier in the loop.
template <typename T>
struct Mfma16;
template <>
struct Mfma16<bf16> {
  static __device__ __forceinline__ f32x4 mma(bf16x8 a, bf16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Mfma16<f16> {
  static __device__ __forceinline__ f32x4 mma(f16x8 a, f16x8 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
};

template <int D>
struct DecodeSmem {
  static constexpr int kVS = D + 8;   // V row stride (elements)
  static constexpr int kOS = D + 4;   // row stride of the waves' outputs (floats)
  static constexpr int kV = 4 * 32 * kVS * 2;
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
    const uint64_t past = __builtin_amdgcn_ballot_w64((int64_t)incl * a.pairs > at);
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

template <typename T, int D>
__global__ __launch_bounds__(256, D >= 256 ? 1 : 2) void paged_decode_kernel(DecodeArgs a) {
  using M = Mfma16<T>;
  using S = DecodeSmem<D>;
  using v8 = typename Mfma<T>::v8;
  constexpr int NC = D / 32, ND = D / 16;
  extern __shared__ __align__(16) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int l16 = lane & 15, lg = lane >> 4;
  T *vs = reinterpret_cast<T *>(smem) + wave * 32 * S::kVS;

  const int total = __builtin_amdgcn_readfirstlane(all_tiles(a, lane)) * a.pairs;
  const int per = decode_per(total, gridDim.x);
  int64_t first = (int64_t)blockIdx.x * per;
  if (first >= total) return;
  int cur = (int)first;
  const int end = total - cur < per ? total : cur + per;
  int b, base;
  find_seq(a, cur, lane, &b, &base);
  b = __builtin_amdgcn_readfirstlane(b);
  base = __builtin_amdgcn_readfirstlane(base);

  while (cur < end) {
    const int len = __builtin_amdgcn_readfirstlane(clip_len(a.lens[b], a.capacity));
    const int nt = decode_tiles(len, a.window);
    if (nt == 0) {
      ++b;
      continue;
    }
    const int rel = cur - base * a.pairs, pair = rel / nt, t0 = rel - pair * nt;
    const int run = end - cur < nt - t0 ? end - cur : nt - t0;
    const int hk = pair / a.head_blocks, hb = pair - hk * a.head_blocks;
    const int h0 = hk * a.G + hb * kDecodeRows;
    const int rows = a.G - hb * kDecodeRows < kDecodeRows ? a.G - hb * kDecodeRows : kDecodeRows;
    const int lo = len - decode_seen(len, a.window);
    const T *kc = (const T *)a.kc + hk * a.kc_head + lg * 8;
    const T *vc = (const T *)a.vc + hk * a.vc_head + lg * 8;

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

    // this lane's two keys of the wave's 32 in tile t: page and token in it
    struct Keys {
      int id[2], slot[2];
    };
    auto keys_of = [&](int t) {
      Keys k;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int key = lo + t * kDecodeTile + wave * 32 + 16 * i + l16;
        const PageSlot s = page_slot(a.map, key);
        k.id[i] = t < t0 + run && key < len ? page_of(a.map, b, key, s) : -1;
        k.slot[i] = s.slot;
      }
      return k;
    };
    u32x4 kr[2][NC], vr[2][NC];
    auto load = [&](const T *p, int64_t page, int64_t token, const Keys &k, u32x4 (&r)[2][NC]) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const T *row = p + (k.id[i] >= 0 ? k.id[i] * page + k.slot[i] * token : 0);
#pragma unroll
        for (int c = 0; c < NC; ++c) r[i][c] = *reinterpret_cast<const u32x4 *>(row + 32 * c);
      }
    };

    f32x4 acc[ND];
#pragma unroll
    for (int i = 0; i < ND; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m_run = -kHuge, l_run = 0.f;
    Keys now = keys_of(t0);
    load(kc, a.k_page, a.kc_token, now, kr);
    load(vc, a.v_page, a.vc_token, now, vr);
    Keys next = keys_of(t0 + 1);
    for (int t = t0; t < t0 + run; ++t) {
      f32x4 s[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int c = 0; c < NC; ++c) s[i] = M::mma(as_v8<T>(kr[i][c]), qf[c], s[i]);
      }
      // which of the 32 keys there are (bit: key)
      const uint32_t ok = (uint32_t)(__builtin_amdgcn_ballot_w64(now.id[0] >= 0) & 0xffffu) |
                          (uint32_t)(__builtin_amdgcn_ballot_w64(now.id[1] >= 0) & 0xffffu) << 16;
      if (ok != 0xffffffffu) {
        // values of absent keys are whatever the cache holds: zeros instead, so that
        // their zero probabilities do not meet infinities
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int c = 0; c < NC; ++c)
            if (now.id[i] < 0) vr[i][c] = u32x4{0, 0, 0, 0};
      }
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int c = 0; c < NC; ++c)
          *reinterpret_cast<u32x4 *>(vs + (16 * i + l16) * S::kVS + 32 * c + lg * 8) = vr[i][c];
      now = next;
      if (t + 1 < t0 + run) {
        load(kc, a.k_page, a.kc_token, now, kr);
        load(vc, a.v_page, a.vc_token, now, vr);
        next = keys_of(t + 2);
      }
      // scores in the log2 domain; C row (key) 16 i + lg * 4 + r
      float y[8], mx = kNegInf;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
          const int row = 16 * i + lg * 4 + r;
          float z = s[i][r] * a.c;
          if (a.cap2 > 0.f) z = a.cap2 * (1.f - 2.f * __builtin_amdgcn_rcpf(1.f + fast_exp2(z)));
          if (a.slopes != nullptr)
            z -= slope2 * (float)(len - 1 - (lo + t * kDecodeTile + wave * 32 + row));
          y[4 * i + r] = ok >> row & 1 ? z : kNegInf;
          mx = fmaxf(mx, y[4 * i + r]);
        }
      mx = max_xor32(max_xor16(mx));
      const float m_new = fmaxf(m_run, mx), alpha = fast_exp2(m_run - m_new);
      m_run = m_new;
      v8 p;
      float ps = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float x = fast_exp2(y[e] - m_run);
        // the sum takes the probabilities as rounded for the product
        p[e] = static_cast<T>(x);
        ps += to_f(p[e]);
      }
      l_run = l_run * alpha + ps;
#pragma unroll
      for (int i = 0; i < ND; ++i) {
#pragma unroll
        for (int r = 0; r < 4; ++r) acc[i][r] *= alpha;
        const T *tr = vs + (lg * 4 + (l16 >> 2)) * S::kVS + 16 * i + 4 * (l16 & 3);
        acc[i] = M::mma(as_v8<T>(join(lds_tr16(tr), lds_tr16(tr + 16 * S::kVS))), p, acc[i]);
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
    const int64_t slot = decode_slot(blockIdx.x, base * a.pairs + pair * nt, per);
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
    if (pair == a.pairs - 1 && t0 + run == nt) {
      base += nt;
      ++b;
    }
  }
}

// One wave per (sequence, query head): joins the pieces that several workgroups
// formed, in their order; a sequence without keys gets zeros.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_decode_join_kernel(DecodeArgs a, int grid) {
  constexpr int E = D / 64;  // features per lane
  const int lane = threadIdx.x & 63;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
  if (row >= (int64_t)a.n_seq * a.H) return;
  const int b = (int)(row / a.H), h = (int)(row % a.H);
  int total = 0, base = 0;  // tiles of all sequences, and of those in front of b
  for (int c = 0; c < a.n_seq; c += 64) {
    const int t = seq_tiles(a, c + lane);
    total += t;
    if (c + lane < b) base += t;
  }
  total = wave_sum_i(total) * a.pairs;
  base = wave_sum_i(base) * a.pairs;
  const int nt = decode_tiles(clip_len(a.lens[b], a.capacity), a.window);
  T *out = (T *)a.out + row * D + lane * E;
  if (nt == 0) {
#pragma unroll
    for (int e = 0; e < E; ++e) out[e] = (T)0.f;
    return;
  }
  const int per = decode_per(total, grid);
  const int hk = h / a.G, hr = h % a.G;
  const int t0 = base + (hk * a.head_blocks + hr / kDecodeRows) * nt;
  const int g0 = t0 / per, g1 = (t0 + nt - 1) / per;
  if (g0 == g1) return;
  const int r = hr % kDecodeRows;
  float m = kNegInf;
  for (int g = g0 + lane; g <= g1; g += 64)
    m = fmaxf(m, a.part_ml[(decode_slot(g, t0, per) * kDecodeRows + r) * 2]);
  m = wave_max(m);
  float l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int g = g0; g <= g1; ++g) {
    const int64_t at = decode_slot(g, t0, per) * kDecodeRows + r;
    const float f = fast_exp2(a.part_ml[at * 2] - m);
    l += f * a.part_ml[at * 2 + 1];
    const float *p = a.part_o + at * D + lane * E;
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] += f * p[e];
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
  for (int e = 0; e < E; ++e) out[e] = from_f<T>(o[e] * inv);
}

template <typename T, int D>
void launch_decode_d(const DecodeArgs &a, int grid, hipStream_t st) {
  const int smem = DecodeSmem<D>::kBytes;
  allow_dynamic_lds(reinterpret_cast<const void *>(&paged_decode_kernel<T, D>), smem);
  hipLaunchKernelGGL((paged_decode_kernel<T, D>), dim3((unsigned)grid), dim3(256), smem, st, a);
  const int64_t rows = (int64_t)a.n_seq * a.H;
  hipLaunchKernelGGL((paged_decode_join_kernel<T, D>), dim3((unsigned)((rows + 3) / 4)), dim3(256),
                     0, st, a, grid);
}

}  // namespace

template <typename T>
void launch_paged_append(const AppendArgs &a, hipStream_t st) {
  hipLaunchKernelGGL((paged_append_pairs_kernel<T>), dim3((unsigned)a.T), dim3(256), 0, st, a);
}

template <typename T>
void launch_paged_decode(const DecodeArgs &a, int D, int grid, hipStream_t st) {
  if (D == 64) return launch_decode_d<T, 64>(a, grid, st);
  if (D == 128) return launch_decode_d<T, 128>(a, grid, st);
  launch_decode_d<T, 256>(a, grid, st);
}

#define VAFA_INST(T)                                              \
  template void launch_paged_append<T>(const AppendArgs &, hipStream_t); \
  template void launch_paged_decode<T>(const DecodeArgs &, int, int, hipStream_t);
VAFA_INST(bf16)
VAFA_INST(f16)
#undef VAFA_INST

}  // namespace vafa
