// Attention of several new tokens per sequence over a paged key-value cache, in 16 bits or
// in 8-bit codes, on gfx950 matrix cores (bf16 / f16).
//
// Tiles and products are those of the packed masked forward (masked_tile.h): 128 rows of a
// workgroup are tokens of up to 32 query heads that share a key head, keys and values come in
// units of 64 through LDS, one unit ahead in registers.  What differs: rows of a unit are
// looked up in the page table, two units ahead; the lengths are device data, so the work is
// divided here: all units of all tiles form one axis (paged.h), cut into as many even chunks
// as the GPU holds workgroups for each set of heads, and a second launch joins the tiles that
// were cut.
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
  int q0 = a.cu[b], q1 = a.cu[b + 1];
  q0 = q0 < 0 ? 0 : (q0 > T ? T : q0);
  q1 = q1 < q0 ? q0 : (q1 > T ? T : q1);
  return SeqAt{q0, chunk_seq(q1 - q0, clip_len(a.lens[b], a.capacity), a.lt, a.window)};
}
// Units of a sequence (tiles where they are not divided).
__device__ __forceinline__ int64_t seq_units(const ChunkArgs &a, int b) {
  if (b >= a.n_seq) return 0;
  const ChunkSeq s = seq_at(a, b).s;
  const int64_t m = chunk_tiles(s.nq, s.lt);
  return a.direct ? m : chunk_before(s, m);
}
__device__ __forceinline__ int64_t all_units(const ChunkArgs &a, int lane) {
  int64_t total = 0;
  for (int c = 0; c < a.n_seq; c += 64) total += seq_units(a, c + lane);
  return uniform_l(wave_sum_l(total));
}
// The sequence that holds unit `at` of the axis, and the units in front of it.
__device__ __forceinline__ void find_seq(const ChunkArgs &a, int64_t at, int lane, int *b,
                                         int64_t *base) {
  int64_t before = 0;
  for (int c = 0; c < a.n_seq; c += 64) {
    const int64_t t = seq_units(a, c + lane), incl = wave_scan_l(t, lane) + before;
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
__device__ __forceinline__ int64_t units_per(const ChunkArgs &a, int64_t total) {
  const int64_t per = (total + a.chunks - 1) / a.chunks;
  return per < kChunkLeast ? kChunkLeast : per;
}

// Pieces of 16 bytes of a unit's rows, by thread, and the rows' powers of two.
template <int D, int NT, bool kCodes>
struct UnitRegs {
  static constexpr int kPerRow = D / (kCodes ? 16 : 8);
  static constexpr int kPieces = kChunkKeys * kPerRow / NT;  // of a thread
  u32x4 k[kPieces], v[kPieces];
  uint32_t ke, ve;  // of this lane's key
};

template <typename T, int D, int NW>
constexpr int chunk_lds() {
  constexpr int kStage = NW * RowStore<T, D / 32>::kBytes;
  return FwdSmem<D>::kBytes > kStage ? FwdSmem<D>::kBytes : kStage;
}

template <typename T, int D, int NW, bool kCodes, bool kCap, bool kBias>
__global__ __launch_bounds__(64 * NW, D >= 256 ? 1 : 2) void paged_chunk_kernel(ChunkArgs a) {
  using M = Mfma<T>;
  using E = std::conditional_t<kCodes, uint8_t, T>;
  using R = UnitRegs<D, 64 * NW, kCodes>;
  constexpr int NC = D / 16, ND = D / 32, NT = 64 * NW, BM = 32 * NW;
  constexpr int kPiece = 16 / (int)sizeof(E);
  extern __shared__ __align__(16) unsigned char smem_raw[];
  T *smem = reinterpret_cast<T *>(smem_raw);
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

  // rows of no sequence
  {
    int lo = a.cu[0], hi = a.cu[a.n_seq];
    const int T_ = (int)a.T;
    lo = lo < 0 ? 0 : (lo > T_ ? T_ : lo);
    hi = hi < lo ? lo : (hi > T_ ? T_ : hi);
    const int64_t n = lo + (T_ - hi), pieces = n * a.H * D / 8;
    for (int64_t e = (int64_t)blockIdx.x * NT + tid; e < pieces; e += (int64_t)gridDim.x * NT) {
      const int64_t at = e * 8, edge = (int64_t)lo * a.H * D;
      T *p = (T *)a.out + (at < edge ? at : at - edge + (int64_t)hi * a.H * D);
      *reinterpret_cast<u32x4 *>(p) = u32x4{0, 0, 0, 0};
    }
  }
  if (chunk >= a.chunks) return;
  const int64_t total = all_units(a, lane);
  const int64_t per = a.direct ? 1 : units_per(a, total);
  int64_t cur = chunk * per;
  const int64_t end = a.direct || total - cur < per ? total : cur + per;
  if (cur >= end) return;
  int b;
  int64_t base;
  find_seq(a, cur, lane, &b, &base);

  ScoreArgs sa{a.c, a.cap2};
  uint32_t qsign = 0;
  if constexpr (!kCap && !kBias) {  // (as in the packed forward)
    if (sa.c < 0.f) qsign = 0x80008000u;
    sa.c = score_factor(sa.c);
  }
  const int window = a.window > 0 ? a.window : kChunkNoWindow;
  const E *kc = (const E *)a.kc + hk * a.kc_head + tid % R::kPerRow * kPiece;
  const E *vc = (const E *)a.vc + hk * a.vc_head + tid % R::kPerRow * kPiece;

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
    const int64_t t0 = a.direct ? cur : base + chunk_before(s, i);
    const int64_t units = chunk_units(s, i);
    const int64_t u0 = a.direct ? 0 : cur - t0;
    const int run = (int)uniform_l(a.direct || units - u0 < end - cur ? units - u0 : end - cur);
    const bool whole = run == units;
    const int q0 = __builtin_amdgcn_readfirstlane(at.q0 + (int)(i << s.lt));
    const int qn = (int)(s.nq - (i << s.lt)), q1 = q0 + uniform_clamp(qn, BM >> lg);
    const int diag = __builtin_amdgcn_readfirstlane((int)(s.diag - at.q0));
    const int kb0 = __builtin_amdgcn_readfirstlane((int)(chunk_start(s, i) + u0 * kChunkKeys));
    const int kend = __builtin_amdgcn_readfirstlane((int)chunk_end(s, i));
    // keys in front of it are of no row's window, though of the first unit: absent
    const int kfirst = a.window > 0 ? q0 + diag - a.window + 1 : 0;

    const int w0 = q0 + wave * tw;  // the wave's first token
    const int tok = w0 + (lrow >> lg), h = h0 + (lrow & ((1 << lg) - 1));
    const bool row_ok = tok < q1, wave_active = w0 < q1;
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

    struct Key {
      int id, slot;  // page (-1: none) and token there of this lane's key of a unit
    };
    auto look_up = [&](int j) {
      const int key = kb0 + j * kChunkKeys + lane;
      Key k{-1, 0};
      if (j < run && key >= kfirst && key < kend) {
        const PageSlot ps = page_slot(a.map, key);
        k.id = page_of(a.map, b, key, ps);
        k.slot = ps.slot;
      }
      return k;
    };
    R regs;
    // rows of the unit whose keys the lanes looked up -> which of them there are
    auto load = [&](Key k) {
      const bool there = k.id >= 0;
      const int64_t id = there ? k.id : 0, slot = there ? k.slot : 0;
      const int64_t ko = id * a.k_page + slot * a.kc_token;
      const int64_t vo = id * a.v_page + slot * a.vc_token;
#pragma unroll
      for (int x = 0; x < R::kPieces; ++x) {
        const int key = (tid + NT * x) / R::kPerRow;
        regs.k[x] = *reinterpret_cast<const u32x4 *>(kc + __shfl((long long)ko, key, 64));
      }
#pragma unroll
      for (int x = 0; x < R::kPieces; ++x) {
        const int key = (tid + NT * x) / R::kPerRow;
        regs.v[x] = *reinterpret_cast<const u32x4 *>(vc + __shfl((long long)vo, key, 64));
      }
      if constexpr (kCodes) {
        const RowScales &sc = a.scales;
        regs.ke = sc.k[id * sc.k_page + slot * sc.k_token + hk * sc.k_head];
        regs.ve = sc.v[id * sc.v_page + slot * sc.v_token + hk * sc.v_head];
      }
      return __builtin_amdgcn_ballot_w64(there);
    };
    auto store = [&](int buf, uint64_t here) {
      T *ks = smem + buf * FwdSmem<D>::kBuf, *vs = ks + FwdSmem<D>::kKs;
#pragma unroll
      for (int x = 0; x < R::kPieces; ++x) {
        const int key = (tid + NT * x) / R::kPerRow, f = tid % R::kPerRow * kPiece;
        u32x4 v = regs.v[x];
        // values of absent keys are whatever the cache holds: zeros, so that their zero
        // probabilities do not meet infinities
        if (!(here >> key & 1)) v = u32x4{0, 0, 0, 0};
        T *kd = ks + key * FwdSmem<D>::KSK + f, *vd = vs + key * FwdSmem<D>::KSV + f;
        if constexpr (kCodes) {
          u32x4 lo, hi;
          from_codes<T>(regs.k[x], row_scale(__shfl(regs.ke, key, 64)), lo, hi);
          *reinterpret_cast<u32x4 *>(kd) = lo;
          *reinterpret_cast<u32x4 *>(kd + 8) = hi;
          const uint32_t ve = __shfl(regs.ve, key, 64);  // (every lane takes part)
          from_codes<T>(v, row_scale(here >> key & 1 ? ve : 127), lo, hi);
          *reinterpret_cast<u32x4 *>(vd) = lo;
          *reinterpret_cast<u32x4 *>(vd + 8) = hi;
        } else {
          *reinterpret_cast<u32x4 *>(kd) = regs.k[x];
          *reinterpret_cast<u32x4 *>(vd) = v;
        }
      }
    };

    uint64_t here = load(look_up(0)), there = 0;
    Key next = look_up(1);
    store(0, here);
    __syncthreads();
    auto step = [&](int j, auto buf) {
      const int B = buf;
      if (j + 1 < run) {
        there = load(next);
        next = look_up(j + 2);
      }
      const T *ks = smem + B * FwdSmem<D>::kBuf;
      const int kb = kb0 + j * kChunkKeys;
      const int kl = (kb + kChunkKeys < kend ? kb + kChunkKeys : kend) - 1;
      if (wave_active && !none_visible(kb, kl, p0, p1, 0, window)) {
        const bool masked = here != ~uint64_t{0} || !all_visible(kb, kl, p0, p1, 0, window);
        masked_tile<T, D, kCap, kBias>(ks, ks + FwdSmem<D>::kKs, qf, acc, m_run, l_part, sa, slope2,
                                       kb, kend, masked, p, 0, window, lane, here);
      }
      if (j + 1 < run) store(1 - B, there);
      here = there;
      __syncthreads();
    };
    for (int j = 0; j < run; ++j) step(j, j & 1);

    if (wave_active) {
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
      }
    }
    __syncthreads();  // the staged rows are read: the next piece may write K and V
    if (a.direct) {
      cur += a.chunks;
      if (cur < end) find_seq(a, cur, lane, &b, &base);
    } else {
      cur += run;
    }
  }
}

// Joins the parts of a tile that chunks cut: a group of workgroups for each border between
// two chunks and each set, of which the tile's first border does the work, 4096 outputs a
// workgroup, 16 neighbouring features a thread: m = max lse_g, w_g = 2^(lse_g - m),
// O = sum w_g O_g / sum w_g.
template <typename T, int D, int BM>
__global__ __launch_bounds__(256) void paged_chunk_join_kernel(ChunkArgs a) {
  constexpr int kRowsOf = 4096 / D, kParts = BM / kRowsOf;
  const int tid = threadIdx.x, lane = tid & 63;
  const HeadSets hs{a.H, a.Hk, a.lg};
  const int sets = hs.sets();
  const int part = blockIdx.x % kParts, set = blockIdx.x / kParts % sets;
  const int64_t c = blockIdx.x / kParts / sets + 1;
  const int64_t total = all_units(a, lane), per = units_per(a, total), u = c * per;
  if (u >= total) return;
  int b;
  int64_t base;
  find_seq(a, u, lane, &b, &base);
  if (b >= a.n_seq) return;
  const SeqAt at = seq_at(a, b);
  const ChunkSeq &s = at.s;
  const int64_t i = chunk_tile_of(s, u - base), t0 = base + chunk_before(s, i);
  if (t0 >= u || t0 < u - per) return;  // no border within a tile, or not its first
  const int g0 = (int)c - 1, g1 = (int)((t0 + chunk_units(s, i) - 1) / per);
  const int row = part * kRowsOf + tid / (D / 16), f = tid % (D / 16) * 16;
  const int64_t tok = (i << s.lt) + (row >> a.lg);
  if (tok >= s.nq) return;
  auto row_of = [&](int g) { return (chunk_slot(g, t0, per) * sets + set) * BM + row; };
  float m = kNegInf;
  for (int g = g0; g <= g1; ++g) m = fmaxf(m, a.part_lse[row_of(g)]);
  const float ms = m == kNegInf ? 0.f : m;  // no part sees a key: zeros
  float l = 0.f;
  f32x4 x[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) x[e] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll 2
  for (int g = g0; g <= g1; ++g) {
    const int64_t r = row_of(g);
    const float w = fast_exp2(a.part_lse[r] - ms);
    l += w;
    const f32x4 *src = reinterpret_cast<const f32x4 *>(a.part_o + r * D + f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const f32x4 y = src[e];
#pragma unroll
      for (int t = 0; t < 4; ++t) x[e][t] += w * y[t];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T *dst = (T *)a.out + ((at.q0 + tok) * a.H + (set << a.lg) + (row & ((1 << a.lg) - 1))) * D + f;
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    typename Mfma<T>::v8 y;
#pragma unroll
    for (int t = 0; t < 8; ++t) y[t] = static_cast<T>(x[2 * e + t / 4][t % 4] * inv);
    *reinterpret_cast<typename Mfma<T>::v8 *>(dst + 8 * e) = y;
  }
}

template <typename T, int D, bool kCodes, bool kCap, bool kBias>
void launch_v(const ChunkArgs &a, hipStream_t st) {
  constexpr int NW = 4;
  constexpr auto fn = &paged_chunk_kernel<T, D, NW, kCodes, kCap, kBias>;
  const int smem = chunk_lds<T, D, NW>(), sets = a.H >> a.lg;
  allow_dynamic_lds(reinterpret_cast<const void *>(fn), smem);
  const int64_t wgs = (int64_t)(a.chunks + kXcds - 1) / kXcds * kXcds * sets;
  hipLaunchKernelGGL(fn, dim3((unsigned)wgs), dim3(64 * NW), smem, st, a);
  if (a.direct || a.chunks < 2) return;
  const int64_t joins = (int64_t)(a.chunks - 1) * sets * (32 * NW * D / 4096);
  hipLaunchKernelGGL((paged_chunk_join_kernel<T, D, 32 * NW>), dim3((unsigned)joins), dim3(256), 0,
                     st, a);
}

template <typename T, int D, bool kCodes>
void launch_d(const ChunkArgs &a, hipStream_t st) {
  const bool cap = a.cap2 > 0.f, bias = a.slopes != nullptr;
  if (cap && bias) return launch_v<T, D, kCodes, true, true>(a, st);
  if (cap) return launch_v<T, D, kCodes, true, false>(a, st);
  if (bias) return launch_v<T, D, kCodes, false, true>(a, st);
  launch_v<T, D, kCodes, false, false>(a, st);
}

}  // namespace

template <typename T, int D>
void launch_paged_chunk(const ChunkArgs &a, hipStream_t st) {
  if (a.scales.k != nullptr) return launch_d<T, D, true>(a, st);
  launch_d<T, D, false>(a, st);
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
