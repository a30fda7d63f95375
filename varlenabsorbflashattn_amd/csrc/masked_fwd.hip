// Forward of packed_masked_attn on gfx950 matrix cores (bf16 / f16).
//
// The layout of products and tiles is that of the packed varlen forward
// (varlen_mfma.hip): 32 query rows per wave, 64-key tiles staged once per workgroup,
// S^T = K Q^T, online softmax against a lazily updated running max, O^T += V^T P^T.
// What differs: the rows of a tile are tokens of several query heads that share a key
// head (HeadSets); a workgroup walks only the keys that some row of its tile sees (key_walk), a wave skips the tiles that none of its
// rows sees, and only tiles that some row does not see whole are masked.
#include <type_traits>

#include "fwd_tiles.h"
#include "kernels.h"
#include "masked.h"
#include "mfma.h"

namespace vafa {

namespace {

// One 64-key tile for the wave's 32 query rows; masked: some (row, key) pair is hidden.
template <typename T, int D, bool kCap, bool kBias>
__device__ __forceinline__ void masked_tile(const T *ks, const T *vs,
                                            const typename Mfma<T>::v8 (&qf)[D / 16],
                                            f32x16 (&acc)[D / 32], float &m_run, float &l_part,
                                            const ScoreArgs &sa, float slope2, int kbase,
                                            int k_end, bool masked, int p, int pre, int window,
                                            int lane) {
  using M = Mfma<T>;
  constexpr int NC = D / 16, ND = D / 32;
  constexpr int KS = FwdSmem<D>::KSK, VS = FwdSmem<D>::KSV;
  constexpr bool kLog2 = kCap || kBias;  // s holds log2-domain scores after the transform
  const int lrow = lane & 31, lhalf = lane >> 5;
  constexpr int kPre = 4;
  constexpr int NS = 2 * NC;
  f32x16 s[2];
#pragma unroll
  for (int kt = 0; kt < 2; ++kt)
#pragma unroll
    for (int r = 0; r < 16; ++r) s[kt][r] = 0.f;
  const T *kbase_p = ks + lrow * KS + lhalf * 8;
  auto kop = [&](int i) {  // i = cc * 2 + kt
    return *reinterpret_cast<const u32x4 *>(kbase_p + (i & 1) * 32 * KS + (i >> 1) * 16);
  };
  u32x4 ring[kPre];
#pragma unroll
  for (int i = 0; i < kPre; ++i) ring[i] = kop(i);
  __builtin_amdgcn_sched_barrier(0);
#pragma unroll
  for (int i = 0; i < NS; ++i) {
    const u32x4 a = ring[i % kPre];
    s[i & 1] = M::mma(as_v8<T>(a), qf[i >> 1], s[i & 1]);
    if (i + kPre < NS) ring[i % kPre] = kop(i + kPre);
    __builtin_amdgcn_sched_barrier(0);
  }
  const int k_lane = kbase + lhalf * 4;  // register (kt, r) holds key k_lane + off(kt, r)
  auto off = [](int kt, int r) { return kt * 32 + (r >> 2) * 8 + (r & 3); };
  if constexpr (kLog2) {
    const float back = (float)(p - k_lane);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        float z = s[kt][r] * sa.c;
        if constexpr (kCap) z = __builtin_fmaf(-2.f * sa.cap2, cap_e(z), sa.cap2);
        if constexpr (kBias) z = __builtin_fmaf(-slope2, fabsf(back - (float)off(kt, r)), z);
        s[kt][r] = z;
      }
  }
  if (masked) {
    const uint64_t seen = seen_keys(k_lane, k_end, p, pre, window);
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
#pragma unroll
      for (int r = 0; r < 16; ++r)
        s[kt][r] = where_bit((uint32_t)(seen >> 32 * kt), off(0, r), s[kt][r], kNegInf);
  }
  const float c = kLog2 ? 1.f : sa.c;
  typename M::v8 pb[2][2];
  float ps4[4];
  // P is rounded to T, V's type, for the product; its row sum takes the rounded values, in
  // fp32, so that a constant V comes out as it is (outputs in bf16 1.8e-3 off in the 2-norm,
  // the exact ones rounded 1.7e-3)
  auto build_p = [&]() {
#pragma unroll
    for (int i = 0; i < 4; ++i) ps4[i] = 0.f;
#pragma unroll
    for (int kt = 0; kt < 2; ++kt)
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
    for (int kt = 0; kt < 2; ++kt)
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
  constexpr int NP = 4 * ND;
  auto vop = [&](int i) {  // i = km * ND + dt, km = kt * 2 + mm
    const int km = i / ND, dt = i % ND;
    return tr_operand<T>(vs, VS, km * 16, dt * 32, lane);
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

template <typename T, int D, int NW, bool kCap, bool kBias>
__global__ __launch_bounds__(64 * NW, D >= 256 ? 1 : 2) void masked_fwd_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    T *__restrict__ o, uint8_t *__restrict__ o_lo, float *__restrict__ lse,
    float *__restrict__ part_o, float *__restrict__ part_lse, const int32_t *__restrict__ items,
    const float *__restrict__ slopes, ScoreArgs sa, HeadSets hs, int window) {
  using M = Mfma<T>;
  constexpr int NC = D / 16, ND = D / 32;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  T *smem = reinterpret_cast<T *>(smem_raw);

  const int H = hs.H, lg = hs.lg, tw = 32 >> lg;  // tokens of a wave
  const int item = blockIdx.x / hs.sets(), set = hs.set_of(blockIdx.x % hs.sets());
  const int h0 = set << lg, hk = set / hs.per_key();
  const PlanItem it = load_item(items, item);
  const int q0 = it.v[0], q1 = it.v[1], pbase = it.v[4], diag = it.v[5], pre = it.v[6];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int t0 = q0 + wave * tw;  // the wave's first token
  const int tok = t0 + (lrow >> lg), h = h0 + (lrow & ((1 << lg) - 1));
  const bool row_ok = tok < q1;
  const bool wave_active = t0 < q1;
  const int p = tok + diag;
  const int p0 = t0 + diag;  // the wave's first and last position
  const int p1 = (t0 + tw < q1 ? t0 + tw : q1) - 1 + diag;
  const KeyWalk kw = key_walk<kBN>(it.v[2], it.v[3], pre, q0 + diag - window + 1);

  // A negative scale is folded into Q (sign flips are exact) where the running max is
  // taken over unscaled scores.
  uint32_t qsign = 0;
  if constexpr (!kCap && !kBias) {
    if (sa.c < 0.f) qsign = 0x80008000u;
    sa.c = score_factor(sa.c);
  }
  typename M::v8 qf[NC];
  {
    const rsrc_t rq = make_rsrc(q + ((int64_t)q0 * H + h0) * D, (int64_t)(q1 - q0) * H * D * 2);
    const int lr = hs.row(wave * 32 + lrow);
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      u32x4 val = buf_load16(rq, lr * D * 2 + cc * 32 + lhalf * 16);
#pragma unroll
      for (int w = 0; w < 4; ++w) val[w] ^= qsign;
      qf[cc] = as_v8<T>(val);
    }
  }
  float slope2 = 0.f;
  if constexpr (kBias) slope2 = slopes[h] * kLog2e;

  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;
  float m_run = -kHuge, l_part = 0.f;

  constexpr int NT = 64 * NW;
  const int nt = kw.n;
  TileRegs<D, NT> regs;
  auto load = [&](int j) {
    load_tile<T, D, NT>(regs, k, v, walk_key<kBN>(kw, j), walk_end(kw, j), hs.Hk, hk, tid);
  };
  if (nt > 0) {
    load(0);
    store_tile<T, D, NT>(regs, smem, smem + FwdSmem<D>::kKs, tid);
  }
  __syncthreads();

  auto step = [&](int j, auto buf) {
    const int B = buf;
    if (j + 1 < nt) load(j + 1);
    const T *ks = smem + B * FwdSmem<D>::kBuf;
    const T *vs = ks + FwdSmem<D>::kKs;
    const int kb = walk_key<kBN>(kw, j), ke = walk_end(kw, j);
    const int kl = (kb + kBN < ke ? kb + kBN : ke) - 1;  // last key of the tile
    if (wave_active && !none_visible(kb, kl, p0, p1, pre, window)) {
      const bool masked = kb + kBN > ke || !all_visible(kb, kl, p0, p1, pre, window);
      masked_tile<T, D, kCap, kBias>(ks, vs, qf, acc, m_run, l_part, sa, slope2, kb, ke, masked, p,
                                     pre, window, lane);
    }
    if (j + 1 < nt) {
      T *nks = smem + (1 - B) * FwdSmem<D>::kBuf;
      store_tile<T, D, NT>(regs, nks, nks + FwdSmem<D>::kKs, tid);
    }
    __syncthreads();
  };
  // the buffer's offset as an immediate where the registers are there for it; at D = 256 ten
  // addresses went to scratch (2215 -> 2200 us of forward and backward)
  if constexpr (D == 128) {
    for (int j = 0; j < nt; j += 2) {
      step(j, std::integral_constant<int, 0>{});
      if (j + 1 < nt) step(j + 1, std::integral_constant<int, 1>{});
    }
  } else {
    for (int j = 0; j < nt; ++j) step(j, j & 1);
  }

  if (!wave_active) return;
  // a row that sees no key has l = 0 (output 0, lse -inf); NaN scores stay NaN
  const float l = l_part + __shfl_xor(l_part, 32, 64);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  const float lse_v = l == 0.f ? kNegInf : m_run + fast_log2(l);
  using RS = RowStore<T, ND>;
  unsigned char *stage = smem_raw + wave * RS::kBytes;
  const int rows = uniform_clamp(q1 - t0, tw) << lg;
  auto off = [&](int r) { return (int64_t)hs.row(r) * D; };
  if (pbase < 0) {
    if (o_lo != nullptr && row_ok) {
      uint8_t *at = o_lo + lo_at<D>(hs, t0, set, rows, lrow, 0, lhalf);
#pragma unroll
      for (int c = 0; c < NC; ++c) {
        // this lane's features 16 c + 4 lhalf + {0..3, 8..11}; with the words of the row's
        // other lane they are 16 c + 8 lhalf + {0..7}
        uint32_t w0 = 0u, w1 = 0u;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w0 |= lo_byte<T>(acc[c >> 1][(c & 1) * 8 + e] * inv) << e * 8;
          w1 |= lo_byte<T>(acc[c >> 1][(c & 1) * 8 + 4 + e] * inv) << e * 8;
        }
        asm volatile("s_nop 1\n\tv_permlane32_swap_b32 %0, %1\n\ts_nop 1" : "+v"(w0), "+v"(w1));
        *reinterpret_cast<u32x2 *>(at) = u32x2{w0, w1};
        at += rows * 16;
        asm volatile("" : "+v"(at));  // one address at a time: D = 256 has no registers for 16
      }
    }
    RS::rows16_at(acc, [&](float x) { return static_cast<T>(x * inv); }, stage,
                  o + ((int64_t)t0 * H + h0) * D, off, rows);
    if (lse != nullptr && row_ok && lhalf == 0) lse[(int64_t)tok * H + h] = lse_v;
  } else {
    // partial rows lie as the outputs do, token pbase + ... of [rows, H, D]
    const int64_t prow = pbase + wave * tw;
    RS::rows32_at(acc, inv, stage, part_o + (prow * H + h0) * D, off, rows);
    if (row_ok && lhalf == 0) part_lse[(prow + (lrow >> lg)) * H + h] = lse_v;
  }
}

// Partial rows of split tiles to o and lse: m = max lse_s, w_s = 2^(lse_s - m), O =
// sum w_s O_s / sum w_s.  An item is {q0, q1, pbase, parts}; its rows lie one after
// another in the output and in each part: a thread takes 8 neighbouring features, which
// moved 4.4 TB/s where one wave per row and 4 bytes a lane moved 2.5.
template <typename T, int D>
__global__ __launch_bounds__(256) void masked_join_kernel(
    const float *__restrict__ part_o, const float *__restrict__ part_lse, T *__restrict__ o,
    uint8_t *__restrict__ o_lo, float *__restrict__ lse, const int32_t *__restrict__ items,
    HeadSets hs, int chunks) {
  const int H = hs.H;
  const PlanItem it = load_item(items, blockIdx.x / chunks);
  const int ns = it.v[3];
  const int64_t rows = (int64_t)(it.v[1] - it.v[0]) * H;  // (token, head) rows of a part
  const int64_t i = ((int64_t)(blockIdx.x % chunks) * 256 + threadIdx.x) * 8;
  const int64_t row = i / D;
  if (row >= rows) return;
  const float *ls = part_lse + (int64_t)it.v[2] * H + row;
  const float *src = part_o + (int64_t)it.v[2] * H * D + i;
  float m = kNegInf;
  for (int s = 0; s < ns; ++s) m = fmaxf(m, ls[s * rows]);
  const float ms = m == kNegInf ? 0.f : m;  // no part sees a key: O = 0, lse = -inf
  float l = 0.f;
  f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll 4
  for (int s = 0; s < ns; ++s) {
    const float w = fast_exp2(ls[s * rows] - ms);
    const f32x4 x = *reinterpret_cast<const f32x4 *>(src + s * rows * D);
    const f32x4 y = *reinterpret_cast<const f32x4 *>(src + s * rows * D + 4);
    l += w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      a[e] += w * x[e];
      b[e] += w * y[e];
    }
  }
  const float inv = l == 0.f ? 0.f : 1.f / l;
  typename Mfma<T>::v8 r;
  u32x2 lo{0u, 0u};
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    r[e] = static_cast<T>(a[e] * inv);
    r[4 + e] = static_cast<T>(b[e] * inv);
    lo[0] |= lo_byte<T>(a[e] * inv) << e * 8;
    lo[1] |= lo_byte<T>(b[e] * inv) << e * 8;
  }
  if (o_lo != nullptr) {
    const int lg = hs.lg, tw = 32 >> lg, f = (int)(i % D);
    const int tok = (int)(row / H), h = (int)(row % H);
    const int w0 = tok / tw * tw, left = it.v[1] - it.v[0] - w0;  // the wave's first token
    *reinterpret_cast<u32x2 *>(
        o_lo + lo_at<D>(hs, it.v[0] + w0, h >> lg, (left < tw ? left : tw) << lg,
                        ((tok - w0) << lg) + (h & ((1 << lg) - 1)), f / 16, f / 8 & 1)) = lo;
  }
  *reinterpret_cast<typename Mfma<T>::v8 *>(o + (int64_t)it.v[0] * H * D + i) = r;
  if (lse != nullptr && i % D == 0)
    lse[(int64_t)it.v[0] * H + row] = l == 0.f ? kNegInf : ms + fast_log2(l);
}

// Dynamic LDS: the K/V buffers, or the per-wave row-store regions if those are larger.
template <typename T, int D, int NW>
constexpr int masked_fwd_lds() {
  constexpr int kStage = NW * RowStore<T, D / 32>::kBytes;
  return FwdSmem<D>::kBytes > kStage ? FwdSmem<D>::kBytes : kStage;
}

template <typename T, int D, int NW, bool kCap, bool kBias>
void launch_v(const MaskedArgs &a, hipStream_t st) {
  constexpr auto fn = &masked_fwd_kernel<T, D, NW, kCap, kBias>;
  const int smem = masked_fwd_lds<T, D, NW>();
  allow_dynamic_lds(reinterpret_cast<const void *>(fn), smem);
  hipLaunchKernelGGL(fn, dim3((unsigned)(a.n_items * (a.H >> a.lg))), dim3(64 * NW), smem, st,
                     (const T *)a.q, (const T *)a.k, (const T *)a.v, (T *)a.o, a.o_lo, a.lse,
                     a.part_o, a.part_lse, a.items, a.slopes, ScoreArgs{a.c, a.cap2},
                     HeadSets{a.H, a.Hk, a.lg}, a.window);
}

template <typename T, int D, int NW>
void launch_nw(const MaskedArgs &a, hipStream_t st) {
  const bool cap = a.cap2 > 0.f, bias = a.slopes != nullptr;
  if (cap && bias) return launch_v<T, D, NW, true, true>(a, st);
  if (cap) return launch_v<T, D, NW, true, false>(a, st);
  if (bias) return launch_v<T, D, NW, false, true>(a, st);
  launch_v<T, D, NW, false, false>(a, st);
}

}  // namespace

template <typename T, int D>
void launch_masked_fwd(const MaskedArgs &a, hipStream_t st) {
  if (a.n_items == 0) return;
  if constexpr (D == 128) {
    if (a.q_tile == kVarlenWideTile) return launch_nw<T, D, 8>(a, st);
  }
  launch_nw<T, D, 4>(a, st);
}

template <typename T, int D>
void launch_masked_join(const MaskedArgs &a, hipStream_t st) {
  if (a.n_comb == 0) return;
  const int64_t chunks = ((int64_t)a.comb_rows * a.H * D + 2047) / 2048;
  hipLaunchKernelGGL((masked_join_kernel<T, D>), dim3((unsigned)(a.n_comb * chunks)), dim3(256),
                     0, st, a.part_o, a.part_lse, (T *)a.o, a.o_lo, a.lse, a.comb_items,
                     HeadSets{a.H, a.Hk, a.lg}, (int)chunks);
}

#define VAFA_INST(T, D)                                                   \
  template void launch_masked_fwd<T, D>(const MaskedArgs &, hipStream_t); \
  template void launch_masked_join<T, D>(const MaskedArgs &, hipStream_t);
VAFA_INST(bf16, 64)
VAFA_INST(bf16, 128)
VAFA_INST(bf16, 256)
VAFA_INST(f16, 64)
VAFA_INST(f16, 128)
VAFA_INST(f16, 256)
#undef VAFA_INST

}  // namespace vafa
