// Backward of packed_masked_attn on gfx950 matrix cores (bf16 / f16).
//
// Deterministic, two kernels that recompute P = 2^(x - LSE) from the forward's LSE, laid
// out as the packed varlen backward (varlen_bwd_mfma.hip):
//   * dQ, query-major over the forward's items: S^T = K Q^T, dP^T = V dO^T,
//     dQ^T += K^T dS^T, and delta = rowsum(O dO) for the other kernel;
//   * dK/dV, key-major: a workgroup owns a key tile of one key head, walks blocks of 32
//     (token, head) rows that see it, of every query head that shares the key head (or a
//     part of those blocks, where one workgroup's walk would outlast the launch: fp32
//     partials, summed in order), and accumulates dV^T += dO^T P, dK^T += Q^T dS.
// P and dS are rounded to T for the products of dV, dQ and dK, formed from fp32 scores, LSE and
// delta: gradients 2.4e-3 (bf16) and 3.0e-4 (fp16) off in the 2-norm, where the exact ones
// rounded are 1.7e-3 and 2.1e-4 off.  Two 16-bit parts each would take half as many products
// again.
// With y = cap tanh(z / cap): dz = dx (1 - tanh^2), formed from e of cap_e as 4 e (1 - e).
#include <algorithm>
#include <type_traits>

#include "bwd_tiles.h"
#include "kernels.h"
#include "masked.h"
#include "mfma.h"

namespace vafa {

namespace {

// ---- dQ ----------------------------------------------------------------------------
template <typename T, int D, int NW, bool kCap, bool kBias>
__global__ __launch_bounds__(64 * NW, D >= 256 ? 1 : 2) void masked_dq_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    const T *__restrict__ dout, const T *__restrict__ o, const uint8_t *__restrict__ o_lo,
    const float *__restrict__ lse, float *__restrict__ delta, float *__restrict__ lse_out, T *__restrict__ dq,
    float *__restrict__ part_dq, const int32_t *__restrict__ items,
    const float *__restrict__ slopes, ScoreArgs sa, HeadSets hs, int window, float scale) {
  using M = Mfma<T>;
  using S = DqSmem<D>;
  using L = GTile<D>;
  constexpr int NC = D / 16, ND = D / 32;
  constexpr int kPre = 4;
  constexpr bool kLog2 = kCap || kBias;
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
  const int p0 = t0 + diag;
  const int p1 = (t0 + tw < q1 ? t0 + tw : q1) - 1 + diag;
  const KeyWalk kw = key_walk<kRB>(it.v[2], it.v[3], pre, q0 + diag - window + 1);

  constexpr int NS = 32 * NW;  // staging threads per tensor
  const bool stage_k = wave < NW / 2;
  const int st = tid & (NS - 1);
  const T *src = stage_k ? k : v;
  Rows<D, NS> stg;
  auto put = [&](int buf) {
    T *ks = smem + buf * S::kBuf;
    store_rows<T, D, NS>(stg, stage_k ? ks : ks + S::kKs, st);
  };
  auto load = [&](int j) {
    load_rows<T, D, NS>(stg, src, walk_key<kRB>(kw, j), walk_end(kw, j), hs.Hk, hk, st);
  };
  const int nblk = kw.n;
  if (nblk > 0) load(0);

  // a negative scale is folded into Q (masked scores are -inf before it)
  uint32_t qsign = 0;
  if constexpr (!kLog2) {
    if (sa.c < 0.f) qsign = 0x80008000u;
    sa.c = score_factor(sa.c);
  }
  typename M::v8 qf[NC], dof[NC];
  float Dr;
  {
    const int64_t nb = (int64_t)(q1 - q0) * H * D * 2;
    const int64_t base = ((int64_t)q0 * H + h0) * D;
    const rsrc_t rq = make_rsrc(q + base, nb);
    const rsrc_t rd = make_rsrc(dout + base, nb);
    const rsrc_t ro = make_rsrc(o + base, nb);
    const int off = hs.row(wave * 32 + lrow) * D * 2 + lhalf * 16;
    const int rows = uniform_clamp(q1 - t0, tw) << lg;
    u32x4 ov[NC];
    u32x2 lo[NC];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      ov[cc] = buf_load16(ro, off + cc * 32);
      lo[cc] = u32x2{0u, 0u};
      if (row_ok)
        lo[cc] = *reinterpret_cast<const u32x2 *>(
            o_lo + lo_at<D>(hs, t0, set, rows, lrow, cc, lhalf));
    }
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      u32x4 a = buf_load16(rq, off + cc * 32), b = buf_load16(rd, off + cc * 32);
      asm volatile("" : "+v"(a), "+v"(b));
#pragma unroll
      for (int w = 0; w < 4; ++w) a[w] ^= qsign;
      qf[cc] = as_v8<T>(a);
      dof[cc] = as_v8<T>(b);
    }
    // delta in fp32: this lane's half of the row, then the other half's
    float sc = 0.f;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      const T *x = reinterpret_cast<const T *>(&ov[cc]);
      float a = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) a = __builtin_fmaf(with_lo(x[e], lo[cc][e >> 2], e & 3), to_f(dof[cc][e]), a);
      sc += a;
    }
    Dr = sc + __shfl_xor(sc, 32, 64);
  }
  // rows past q1, and rows that see no key, get LSE = +inf: their P is 0
  float Lr = row_ok ? lse[(int64_t)tok * H + h] : __builtin_inff();
  const bool dead = !row_ok || Lr == kNegInf;
  if (wave_any(dead)) {  // whatever such a row and its gradient hold, a factor 0 meets no NaN
    if (dead) Lr = __builtin_inff(), Dr = 0.f;
#pragma unroll
    for (int cc = 0; cc < NC; ++cc)
      if (dead) qf[cc] = dof[cc] = as_v8<T>(u32x4{0u, 0u, 0u, 0u});
  }
  if (row_ok && lhalf == 0 && it.v[7] != 0) {  // the item that owns its rows' first keys
    delta[(int64_t)tok * H + h] = Dr;
    lse_out[(int64_t)tok * H + h] = Lr;
  }
  asm volatile("" : "+v"(Lr), "+v"(Dr));
  float slope2 = 0.f;
  if constexpr (kBias) slope2 = slopes[h] * kLog2e;
  // D = 128: dO enters negated and the dP^T chain starts from delta (delta - dP)
  constexpr bool kDeltaInChain = D == 128;
  f32x16 drb;
#pragma unroll
  for (int r = 0; r < 16; ++r) drb[r] = kDeltaInChain ? Dr : 0.f;
  if constexpr (kDeltaInChain) {
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) {
      u32x4 w = __builtin_bit_cast(u32x4, dof[cc]);
#pragma unroll
      for (int e = 0; e < 4; ++e) w[e] ^= 0x80008000u;
      dof[cc] = as_v8<T>(w);
    }
  }
  f32x16 acc[ND];
#pragma unroll
  for (int i = 0; i < ND; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[i][r] = 0.f;

  const int a_off = L::row(lrow) + lhalf * 8;
  const int t_off = L::row(4 * (lane >> 5) + ((lane & 15) >> 2)) + ((lane >> 4) & 1) * 16 +
                    4 * (lane & 3);
  if (nblk > 0) put(0);
  __syncthreads();
  auto block = [&](int j, auto bufc) {
    const int B = bufc;
    const int kb = walk_key<kRB>(kw, j), ke = walk_end(kw, j);
    const int kl = (kb + kRB < ke ? kb + kRB : ke) - 1;
    if (j + 1 < nblk) load(j + 1);
    if (wave_active && !none_visible(kb, kl, p0, p1, pre, window)) {
      const bool masked = kb + kRB > ke || !all_visible(kb, kl, p0, p1, pre, window);
      const lds_cptr<T> ks = as_lds(smem + B * S::kBuf);
      const lds_cptr<T> vs = ks + S::kKs;
      auto aop = [&](int i) { return lds_ld16<T>(((i & 1) ? vs : ks) + a_off + (i >> 1) * 16); };
      f32x16 s, dp = drb;
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = 0.f;
      u32x4 ring[kPre];
#pragma unroll
      for (int i = 0; i < kPre; ++i) ring[i] = aop(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2 * NC; ++i) {
        const typename M::v8 a = as_v8<T>(ring[i % kPre]);
        if (i & 1)
          dp = M::mma(a, dof[i >> 1], dp);
        else
          s = M::mma(a, qf[i >> 1], s);
        if (i + kPre < 2 * NC) ring[i % kPre] = aop(i + kPre);
        __builtin_amdgcn_sched_barrier(0);
      }
      auto top = [&](int i) {
        const lds_cptr<T> tp = ks + t_off + (i / ND) * 4 * L::P2 + (i % ND) * 32;
        return as_v8<T>(join(lds_tr8<T>(tp), lds_tr8<T>(tp + 2 * L::P2)));
      };
      typename M::v8 tring[kPre];
#pragma unroll
      for (int i = 0; i < kPre; ++i) tring[i] = top(i);
      // element r holds key k_lane + off(r) of this lane's row
      const int k_lane = kb + lhalf * 4;
      auto off = [](int r) { return (r >> 2) * 8 + (r & 3); };
      const float back = (float)(p - k_lane);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        if constexpr (!kDeltaInChain) dp[r] -= Dr;
        if constexpr (kLog2) {
          float z = s[r] * sa.c;
          if constexpr (kCap) {
            const float e = cap_e(z), e4 = 4.f * e;
            z = __builtin_fmaf(-2.f * sa.cap2, e, sa.cap2);
            dp[r] *= __builtin_fmaf(-e4, e, e4);
          }
          if constexpr (kBias) z = __builtin_fmaf(-slope2, fabsf(back - (float)off(r)), z);
          s[r] = z;
        }
      }
      if (masked) {
        const uint32_t seen = (uint32_t)seen_keys(k_lane, ke, p, pre, window);
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = where_bit(seen, off(r), s[r], kNegInf);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float pr = fast_exp2(kLog2 ? s[r] - Lr : __builtin_fmaf(s[r], sa.c, -Lr));
        dp[r] = kDeltaInChain ? -(pr * dp[r]) : pr * dp[r];
      }
      typename M::v8 sb[2];
#pragma unroll
      for (int mm = 0; mm < 2; ++mm) sb[mm] = pack8<T>(dp, mm * 8);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2 * ND; ++i) {
        acc[i % ND] = M::mma(tring[i % kPre], sb[i / ND], acc[i % ND]);
        if (i + kPre < 2 * ND) tring[i % kPre] = top(i + kPre);
        __builtin_amdgcn_sched_barrier(0);
      }
    }
    if (j + 1 < nblk) put(1 - B);
    __syncthreads();
  };
  using I0 = std::integral_constant<int, 0>;
  using I1 = std::integral_constant<int, 1>;
  // (one body for both buffers at D = 256: 581 -> 626 us of forward and backward)
  if constexpr (D >= 128) {
    for (int j = 0; j < nblk; j += 2) {
      block(j, I0{});
      if (j + 1 < nblk) block(j + 1, I1{});
    }
  } else {
    for (int j = 0; j < nblk; ++j) block(j, j & 1);
  }

  if (!wave_active) return;
  using RS = RowStore<T, ND>;
  unsigned char *stage = smem_raw + wave * RS::kBytes;
  const int rows = uniform_clamp(q1 - t0, tw) << lg;
  auto off = [&](int r) { return (int64_t)hs.row(r) * D; };
  if (pbase < 0)
    RS::rows16_at(acc, [&](float x) { return static_cast<T>(x * scale); }, stage,
                  dq + ((int64_t)t0 * H + h0) * D, off, rows);
  else
    RS::rows32_at(acc, scale, stage, part_dq + ((int64_t)(pbase + wave * tw) * H + h0) * D, off,
                  rows);
}

// LDS-DMA of 32 rows of a head set (tokens from t0 on, rows at or past `rows` read as
// zero) into a GTile block, as dma_block_rows.
template <typename T, int D, int NW>
__device__ __forceinline__ void dma_set_rows(const T *src, int ntok, const HeadSets &hs,
                                             uint32_t base, int wave, int lane) {
  using L = GTile<D>;
  const u32x4 rs = rsrc_words32(src, (uint32_t)(ntok * hs.H * D * 2));
  if constexpr (D <= 64) {
    constexpr int kInstr = (L::kElems / 8 + 63) / 64;
    for (int i = wave; i < kInstr; i += NW) {
      const int e = (i * 64 + lane) * 8;  // element offset of this lane's 16 bytes
      const int g = e / L::P2, w = e - g * L::P2;
      const int j = w / L::P1, wr = w - j * L::P1;
      if (e < L::kElems && j < 4 && wr < D)
        lds_dma16(rs, base + i * 1024, (hs.row(4 * g + j) * D + wr) * 2);
    }
  } else {
    constexpr int RPW = kRB / NW;
    if (lane < D / 8) {
      int r0 = wave * RPW;
      asm volatile("" : "+s"(r0));  // the rows' offsets are formed here, not held
#pragma unroll
      for (int n = 0; n < RPW; ++n) {
        int voff;
        asm volatile("v_add_u32 %0, %1, %2"
                     : "=v"(voff)
                     : "s"(hs.row(r0 + n) * D * 2), "v"(lane * 16));
        lds_dma16(rs, base + L::row(r0 + n) * 2, voff);
      }
    }
  }
}

// ---- dK / dV -----------------------------------------------------------------------
// Two buffers of a query block: Q and dO rows, then LSE, delta and (with a bias) the
// slopes of its rows; and the last DMA instruction's span past its tile.
template <int D>
struct MDkvSmem {
  static constexpr int kQs = GTile<D>::kElems;
  static constexpr int kVec = 2 * kQs * 2;  // byte offset of the vectors
  static constexpr int kBufBytes = kVec + 3 * kRB * 4;
  static constexpr int kBytes = 2 * kBufBytes + 1024;
};

template <typename T, int D, int NW, bool kCap, bool kBias>
__global__ __launch_bounds__(64 * NW, D >= 256 && NW < 8 ? 1 : 2) void masked_dkv_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    const T *__restrict__ dout, const float *__restrict__ lse, const float *__restrict__ delta,
    T *__restrict__ dk, T *__restrict__ dv, float *__restrict__ part_dk,
    float *__restrict__ part_dv, const int32_t *__restrict__ items,
    const float *__restrict__ slopes, ScoreArgs sa, HeadSets hs, int window, float scale) {
  using M = Mfma<T>;
  using S = MDkvSmem<D>;
  using L = GTile<D>;
  constexpr int ND = D / 32;
  constexpr int kPre = D >= 128 ? 2 : 4;
  // D = 256: waves w and w + 4 share 32 keys, each one half of d (varlen_dkv_kernel)
  constexpr bool kShare = D >= 256;
  static_assert(!kShare || NW == 8, "D = 256 runs on 8 waves");
  constexpr int NDO = kShare ? ND / 2 : ND;
  constexpr int NCS = 2 * NDO;
  constexpr bool kDeltaInChain = D <= 64;
  constexpr bool kLog2 = kCap || kBias;
  extern __shared__ __align__(16) unsigned char smem_raw[];

  const int H = hs.H, Hk = hs.Hk, lg = hs.lg, tb = kRB >> lg;  // tokens of a block
  const int item = blockIdx.x / Hk, hk = blockIdx.x % Hk;
  const PlanItem it = load_item(items, item);
  const int k0 = it.v[0], k1 = it.v[1], q0 = it.v[2], q1 = it.v[3], diag = it.v[4], pre = it.v[5],
            pbase = it.v[6];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kgrp = kShare ? (wave & 3) : wave;
  const int dpart = kShare ? (wave >> 2) : 0;
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int kw0 = k0 + kgrp * 32;  // the wave's first and last key
  const int kw1 = (kw0 + 32 < k1 ? kw0 + 32 : k1) - 1;
  const bool wave_active = kw0 < k1;

  auto issue = [&](int set, int qb, int buf) {
    unsigned char *base = smem_raw + buf * S::kBufBytes;
    const int ntok = uniform_clamp(q1 - qb, tb);
    const int64_t at = (int64_t)qb * H + (set << lg);
    dma_set_rows<T, D, NW>(uniform_ptr(q + at * D), ntok, hs, lds_addr(base), wave, lane);
    dma_set_rows<T, D, NW>(uniform_ptr(dout + at * D), ntok, hs, lds_addr(base + S::kQs * 2), wave,
                           lane);
    // LSE, delta and slopes of the rows: a wave each
    if (wave < 2) {
      const u32x4 rv = rsrc_words32((wave ? delta : lse) + at, (uint32_t)(ntok * H * 4));
      if (lane < kRB) lds_dma4(rv, lds_addr(base + S::kVec + wave * kRB * 4), hs.row(lane) * 4);
    } else if (kBias && wave == 2) {
      const u32x4 rv = rsrc_words32(slopes + (set << lg), 4u << lg);
      if (lane < kRB)
        lds_dma4(rv, lds_addr(base + S::kVec + 2 * kRB * 4), (lane & ((1 << lg) - 1)) * 4);
    }
  };
  // the blocks of the key head's sets, one set after the other; a part of them where the
  // plan divides a key tile's work (v[7]: part << 16 | parts)
  const int nq = (q1 - q0 + tb - 1) / tb, nset = hs.per_key();
  const int64_t all = (int64_t)nq * nset;
  const int part = it.v[7] >> 16, parts = it.v[7] & 0xffff;
  const int f0 = (int)(all * part / parts), nblk = (int)(all * (part + 1) / parts) - f0;
  int set = hk * nset + (nq > 0 ? f0 / nq : 0), qb = q0 + (nq > 0 ? f0 % nq : 0) * tb;
  if (nblk > 0) issue(set, qb, 0);

  uint32_t ksign = 0;  // a negative scale, folded into K's part of the scores
  if constexpr (!kLog2) {
    if (sa.c < 0.f) ksign = 0x80008000u;
    sa.c = score_factor(sa.c);
  }
  typename M::v8 kf[NCS], vf[NCS];
  {
    const int nk = k1 - k0;
    const rsrc_t rk = make_rsrc(k + (int64_t)k0 * Hk * D, (int64_t)nk * Hk * D * 2);
    const rsrc_t rv = make_rsrc(v + (int64_t)k0 * Hk * D, (int64_t)nk * Hk * D * 2);
    const int off = ((kgrp * 32 + lrow) * Hk + hk) * D * 2 + lhalf * 16 + dpart * NDO * 64;
#pragma unroll
    for (int cc = 0; cc < NCS; ++cc) {
      u32x4 a = buf_load16(rk, off + cc * 32), b = buf_load16(rv, off + cc * 32);
      asm volatile("" : "+v"(a), "+v"(b));
#pragma unroll
      for (int w = 0; w < 4; ++w) a[w] ^= ksign;
      kf[cc] = as_v8<T>(a);
      if constexpr (kDeltaInChain) {
#pragma unroll
        for (int w = 0; w < 4; ++w) b[w] ^= 0x80008000u;
      }
      vf[cc] = as_v8<T>(b);
    }
    // a key that no query sees gets zeros, whatever it holds
    const int kj = kw0 + lrow, from = kj - diag, to = from + window;
    const bool seen = kj < pre || (from > q0 ? from : q0) < (to < q1 ? to : q1);
    if (wave_any(!seen)) {
#pragma unroll
      for (int cc = 0; cc < NCS; ++cc)
        if (!seen) kf[cc] = vf[cc] = as_v8<T>(u32x4{0u, 0u, 0u, 0u});
    }
  }
  f32x16 adk[NDO], adv[NDO];
#pragma unroll
  for (int i = 0; i < NDO; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) adk[i][r] = adv[i][r] = 0.f;

  const int a_off = L::row(lrow) + lhalf * 8 + dpart * NDO * 32;
  const int t_off = L::row(4 * (lane >> 5) + ((lane & 15) >> 2)) + ((lane >> 4) & 1) * 16 +
                    4 * (lane & 3);
  auto blk = [&](int j, int B) {
    const int qc = qb;  // the block's first token
    qb += tb;
    if (qb >= q1) {
      qb = q0;
      ++set;
    }
    wait_vmcnt<0>();
    __syncthreads();
    if (j + 1 < nblk) issue(set, qb, 1 - B);
    const unsigned char *base = smem_raw + B * S::kBufBytes;
    const lds_cptr<T> qs = as_lds(reinterpret_cast<const T *>(base));
    const lds_cptr<T> ds_ = qs + S::kQs;
    const float *ls = reinterpret_cast<const float *>(base + S::kVec);
    const int p0 = qc + diag, p1 = (qc + tb < q1 ? qc + tb : q1) - 1 + diag;
    const bool active = wave_active && !none_visible(kw0, kw1, p0, p1, pre, window);
    f32x16 s, dp;
    if (active) {
      auto aop = [&](int i) { return lds_ld16<T>(((i & 1) ? ds_ : qs) + a_off + (i >> 1) * 16); };
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const f32x4 d4 = kDeltaInChain
                             ? *reinterpret_cast<const f32x4 *>(ls + kRB + g * 8 + lhalf * 4)
                             : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          s[4 * g + e] = 0.f;
          dp[4 * g + e] = d4[e];
        }
      }
      u32x4 ring[kPre];
#pragma unroll
      for (int i = 0; i < kPre; ++i) ring[i] = aop(i);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 2 * NCS; ++i) {
        const typename M::v8 a = as_v8<T>(ring[i % kPre]);
        if (i & 1)
          dp = M::mma(a, vf[i >> 1], dp);
        else
          s = M::mma(a, kf[i >> 1], s);
        if (i + kPre < 2 * NCS) ring[i % kPre] = aop(i + kPre);
        __builtin_amdgcn_sched_barrier(0);
      }
      if constexpr (kShare) {
        int eo;
        asm volatile("v_lshl_add_u32 %0, %1, 4, %2"
                     : "=v"(eo)
                     : "v"(lane), "s"(S::kBytes + wave * 8 * 64 * 16));
        f32x4 *ex = reinterpret_cast<f32x4 *>(smem_raw + eo);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          ex[g * 64] = f32x4{s[4 * g], s[4 * g + 1], s[4 * g + 2], s[4 * g + 3]};
          ex[(4 + g) * 64] = f32x4{dp[4 * g], dp[4 * g + 1], dp[4 * g + 2], dp[4 * g + 3]};
        }
      }
    }
    if constexpr (kShare) {
      // the pair w, w ^ 4 holds the same keys: both are active or neither
      __syncthreads();
      if (active) {
        int eo;
        asm volatile("v_lshl_add_u32 %0, %1, 4, %2"
                     : "=v"(eo)
                     : "v"(lane), "s"(S::kBytes + (wave ^ 4) * 8 * 64 * 16));
        const f32x4 *ex = reinterpret_cast<const f32x4 *>(smem_raw + eo);
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          const f32x4 a = ex[g * 64], b = ex[(4 + g) * 64];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            s[4 * g + e] += a[e];
            dp[4 * g + e] += b[e];
          }
          // the partner's registers in two halves: all 32 beside the own 32 would not fit
          if (g == 1) asm volatile("" : "+v"(s), "+v"(dp)::"memory");
        }
      }
    }
    if (active) {
      auto top = [&](int i) {
        const lds_cptr<T> tp = (((i / NDO) & 1) ? qs : ds_) + t_off +
                               ((i / NDO) >> 1) * 4 * L::P2 + (dpart * NDO + i % NDO) * 32;
        return as_v8<T>(join(lds_tr8<T>(tp), lds_tr8<T>(tp + 2 * L::P2)));
      };
      // register r of a lane is row (lane / 32) * 4 + (r / 4) * 8 + r % 4 of the block.  Of
      // the rows that the lane's key sees, one bit each: one register, not 16 tokens
      int ln = lane;
      asm volatile("" : "+v"(ln));  // formed per block
      const int row0 = (ln >> 5) * 4, kj = kw0 + (ln & 31);
      const bool masked = qc + tb > q1 || !all_visible(kw0, kw1, p0, p1, pre, window);
      uint32_t bits = ~0u;
      if (masked) {
        const bool in_pre = kj < pre;
        const int first = kj - diag - qc, last = first + window;
        int lo = in_pre || first < 0 ? 0 : first, hi = q1 - qc;  // tokens of the block
        hi = !in_pre && last < hi ? last : hi;
        hi = hi < tb ? hi : tb;
        bits = lo < hi ? (~0u >> (kRB - (hi << lg)) & ~0u << (lo << lg)) >> row0 : 0u;
      }
      auto row_bit = [](int r) { return (r >> 2) * 8 + (r & 3); };
      if constexpr (!kLog2) {
        if (masked) {
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            s[r] = where_bit(bits, row_bit(r), s[r], kNegInf);
            if (r % 4 == 3) __builtin_amdgcn_sched_barrier(0);
          }
        }
      }
      const int back = qc + diag - kj;
      // P and dS of register r, in place of the score and of dP (delta - dP with
      // kDeltaInChain); hidden pairs are masked above, or here where the score is
      // transformed first
      auto elem = [&](int r, float lr, float dl, float sl) {
        float p, d = dp[r];
        if constexpr (kLog2) {
          float z = s[r] * sa.c;
          if constexpr (kCap) {
            const float e = cap_e(z), e4 = 4.f * e;
            z = __builtin_fmaf(-2.f * sa.cap2, e, sa.cap2);
            if constexpr (!kDeltaInChain) d -= dl;
            d *= __builtin_fmaf(-e4, e, e4);
          } else {
            if constexpr (!kDeltaInChain) d -= dl;
          }
          if constexpr (kBias) {
            const int t = (row0 + (r >> 2) * 8 + (r & 3)) >> lg;
            z = __builtin_fmaf(-kLog2e * sl, fabsf((float)(back + t)), z);
          }
          p = fast_exp2(z - lr);
          p = where_bit(bits, row_bit(r), p, 0.f);
        } else {
          p = fast_exp2(__builtin_fmaf(s[r], sa.c, -lr));
          if constexpr (!kDeltaInChain) d -= dl;
        }
        s[r] = p;
        dp[r] = kDeltaInChain ? -(p * d) : p * d;
      };
      typename M::v8 pb[2], sb[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const float *at = ls + g * 8 + lhalf * 4;
        const f32x4 Lq = *reinterpret_cast<const f32x4 *>(at);
        f32x4 Dl = f32x4{0.f, 0.f, 0.f, 0.f}, Sl = Dl;
        if constexpr (!kDeltaInChain) Dl = *reinterpret_cast<const f32x4 *>(at + kRB);
        if constexpr (kBias) Sl = *reinterpret_cast<const f32x4 *>(at + 2 * kRB);
#pragma unroll
        for (int e = 0; e < 4; ++e) elem(g * 4 + e, Lq[e], Dl[e], Sl[e]);
        if constexpr (kLog2 || D >= 128) __builtin_amdgcn_sched_barrier(0);
      }
      pb[0] = pack8<T>(s, 0);
      sb[0] = pack8<T>(dp, 0);
      __builtin_amdgcn_sched_barrier(0);
      typename M::v8 tring[kPre];
#pragma unroll
      for (int i = 0; i < kPre; ++i) tring[i] = top(i);
      // rows 8..15 under the first half of the chain, which reads rows 0..7 alone
      constexpr int kSteps = 2 * NDO < 8 ? 2 * NDO : 8;
      constexpr int kRowsPer = 8 / kSteps;
      constexpr int kEvery = 2 * NDO / kSteps;
      auto vec_at = [&](int v, int r) { return ls[v * kRB + (r >> 2) * 8 + lhalf * 4 + (r & 3)]; };
      float Ln[kRowsPer], Dn[kRowsPer], Sn[kRowsPer];
      auto next = [&](int r0) {
#pragma unroll
        for (int rr = 0; rr < kRowsPer; ++rr) {
          Ln[rr] = vec_at(0, r0 + rr);
          Dn[rr] = kDeltaInChain ? 0.f : vec_at(1, r0 + rr);
          Sn[rr] = kBias ? vec_at(2, r0 + rr) : 0.f;
        }
      };
      next(8);
      __builtin_amdgcn_sched_barrier(0);
#pragma unroll
      for (int i = 0; i < 4 * NDO; ++i) {
        const int dt = i % NDO, q2 = i / NDO, mm = q2 >> 1;
        const typename M::v8 a = tring[i % kPre];
        if (q2 & 1)
          adk[dt] = M::mma(a, sb[mm], adk[dt]);
        else
          adv[dt] = M::mma(a, pb[mm], adv[dt]);
        if (i + kPre < 4 * NDO) tring[i % kPre] = top(i + kPre);
        if (i < 2 * NDO && i % kEvery == 0) {
          const int g = i / kEvery;
          float Lc[kRowsPer], Dc[kRowsPer], Sc[kRowsPer];
#pragma unroll
          for (int rr = 0; rr < kRowsPer; ++rr) Lc[rr] = Ln[rr], Dc[rr] = Dn[rr], Sc[rr] = Sn[rr];
          if (g + 1 < kSteps) next(8 + (g + 1) * kRowsPer);
#pragma unroll
          for (int rr = 0; rr < kRowsPer; ++rr) elem(8 + g * kRowsPer + rr, Lc[rr], Dc[rr], Sc[rr]);
          if (g == kSteps - 1) {
            pb[1] = pack8<T>(s, 8);
            sb[1] = pack8<T>(dp, 8);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  for (int j = 0; j < nblk; ++j) blk(j, j & 1);
  wait_vmcnt<0>();

  __syncthreads();
  if (!wave_active) return;
  using RS = RowStore<T, NDO>;
  unsigned char *stage = smem_raw + wave * RS::kBytes;
  const int rows = uniform_clamp(k1 - kw0, 32);
  if (pbase < 0) {
    const int64_t off = ((int64_t)kw0 * Hk + hk) * D + dpart * NDO * 32;
    RS::rows16(adk, [&](float x) { return static_cast<T>(x * scale); }, stage, dk + off,
               (int64_t)Hk * D, rows);
    RS::rows16(adv, [](float x) { return static_cast<T>(x); }, stage, dv + off, (int64_t)Hk * D,
               rows);
  } else {
    const int64_t off = ((int64_t)(pbase + kgrp * 32) * Hk + hk) * D + dpart * NDO * 32;
    RS::rows32(adk, scale, stage, part_dk + off, (int64_t)Hk * D, rows);
    RS::rows32(adv, 1.f, stage, part_dv + off, (int64_t)Hk * D, rows);
  }
}

// Partial rows of divided tiles to dq, dk and dv, all in one launch (three cost 4 to 8 us
// more): an item is {r0, r1, pbase, parts}; its rows lie one after another in the
// output and in each part, so a block adds 2048 neighbouring values, part by part in order.
template <typename T>
__global__ __launch_bounds__(256) void masked_sum_kernel(const float *part_dq,
                                                         const float *part_dk,
                                                         const float *part_dv, T *dq, T *dk, T *dv,
                                                         const int32_t *dq_items,
                                                         const int32_t *kv_items, int n_dq,
                                                         int n_kv, int HD, int HkD, int chunks) {
  int y = blockIdx.x / chunks;
  const float *part = part_dq;
  T *out = dq;
  const int32_t *items = dq_items;
  int w = HD;
  if (y >= n_dq) {
    y -= n_dq;
    const bool v = y >= n_kv;
    y -= v ? n_kv : 0;
    part = v ? part_dv : part_dk;
    out = v ? dv : dk;
    items = kv_items;
    w = HkD;
  }
  const PlanItem it = load_item(items, y);
  const int64_t n = (int64_t)(it.v[1] - it.v[0]) * w;
  const int64_t i = ((int64_t)(blockIdx.x % chunks) * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  const float *src = part + (int64_t)it.v[2] * w + i;
  f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll 4
  for (int j = 0; j < it.v[3]; ++j) {
    a += *reinterpret_cast<const f32x4 *>(src + j * n);
    b += *reinterpret_cast<const f32x4 *>(src + j * n + 4);
  }
  typename Mfma<T>::v8 x;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    x[e] = static_cast<T>(a[e]);
    x[4 + e] = static_cast<T>(b[e]);
  }
  *reinterpret_cast<typename Mfma<T>::v8 *>(out + (int64_t)it.v[0] * w + i) = x;
}

// Dynamic LDS: the blocks' buffers, or the per-wave row-store regions if those are larger.
template <typename T, int D, int NW>
constexpr int masked_dq_lds() {
  constexpr int kStage = NW * RowStore<T, D / 32>::kBytes;
  return DqSmem<D>::kBytes > kStage ? DqSmem<D>::kBytes : kStage;
}
template <typename T, int D, int NW>
constexpr int masked_dkv_lds() {
  constexpr int kStage = NW * RowStore<T, D / 32 / (D >= 256 ? 2 : 1)>::kBytes;
  // D = 256: the exchange region behind the buffers
  constexpr int kBase = MDkvSmem<D>::kBytes + (D >= 256 ? NW * 64 * 32 * 4 : 0);
  return kBase > kStage ? kBase : kStage;
}

template <typename T, int D, int NW, bool kCap, bool kBias>
void launch_dq_v(const MaskedArgs &a, hipStream_t st) {
  constexpr auto fn = &masked_dq_kernel<T, D, NW, kCap, kBias>;
  const int smem = masked_dq_lds<T, D, NW>();
  allow_dynamic_lds(reinterpret_cast<const void *>(fn), smem);
  hipLaunchKernelGGL(fn, dim3((unsigned)(a.n_items * (a.H >> a.lg))), dim3(64 * NW), smem, st,
                     (const T *)a.q, (const T *)a.k, (const T *)a.v, (const T *)a.dout,
                     (const T *)a.o_in, a.o_lo_in, a.lse_in, a.delta, a.lse, (T *)a.dq, a.part_o,
                     a.items, a.slopes, ScoreArgs{a.c, a.cap2}, HeadSets{a.H, a.Hk, a.lg},
                     a.window, a.scale);
}
template <typename T, int D, int NW, bool kCap, bool kBias>
void launch_dkv_v(const MaskedArgs &a, hipStream_t st) {
  constexpr auto fn = &masked_dkv_kernel<T, D, NW, kCap, kBias>;
  const int smem = masked_dkv_lds<T, D, NW>();
  allow_dynamic_lds(reinterpret_cast<const void *>(fn), smem);
  hipLaunchKernelGGL(fn, dim3((unsigned)(a.n_kv * a.Hk)), dim3(64 * NW), smem, st,
                     (const T *)a.q, (const T *)a.k, (const T *)a.v, (const T *)a.dout, a.lse,
                     a.delta, (T *)a.dk, (T *)a.dv, a.part_dk, a.part_dv, a.kv_items, a.slopes,
                     ScoreArgs{a.c, a.cap2}, HeadSets{a.H, a.Hk, a.lg}, a.window, a.scale);
}

template <typename T, int D, int NW>
void launch_dq_nw(const MaskedArgs &a, hipStream_t st) {
  const bool cap = a.cap2 > 0.f, bias = a.slopes != nullptr;
  if (cap && bias) return launch_dq_v<T, D, NW, true, true>(a, st);
  if (cap) return launch_dq_v<T, D, NW, true, false>(a, st);
  if (bias) return launch_dq_v<T, D, NW, false, true>(a, st);
  launch_dq_v<T, D, NW, false, false>(a, st);
}
template <typename T, int D, int NW>
void launch_dkv_nw(const MaskedArgs &a, hipStream_t st) {
  const bool cap = a.cap2 > 0.f, bias = a.slopes != nullptr;
  if (cap && bias) return launch_dkv_v<T, D, NW, true, true>(a, st);
  if (cap) return launch_dkv_v<T, D, NW, true, false>(a, st);
  if (bias) return launch_dkv_v<T, D, NW, false, true>(a, st);
  launch_dkv_v<T, D, NW, false, false>(a, st);
}

}  // namespace

template <typename T, int D>
void launch_masked_dq(const MaskedArgs &a, hipStream_t st) {
  if (a.n_items > 0) launch_dq_nw<T, D, 4>(a, st);
}

template <typename T, int D>
void launch_masked_dkv(const MaskedArgs &a, hipStream_t st) {
  if (a.n_kv == 0) return;
  launch_dkv_nw<T, D, D == 256 ? 8 : 4>(a, st);
}

template <typename T>
void launch_masked_sum(const MaskedArgs &a, hipStream_t st) {
  const int64_t n = a.n_comb + 2 * a.n_kvc;
  if (n == 0) return;
  const int HD = a.H * a.D, HkD = a.Hk * a.D;
  const int64_t most = std::max(a.n_comb > 0 ? (int64_t)a.comb_rows * HD : 0,
                                a.n_kvc > 0 ? (int64_t)a.kvc_rows * HkD : 0);
  const int64_t chunks = (most + 2047) / 2048;
  hipLaunchKernelGGL((masked_sum_kernel<T>), dim3((unsigned)(n * chunks)), dim3(256), 0, st,
                     a.part_o, a.part_dk, a.part_dv, (T *)a.dq, (T *)a.dk, (T *)a.dv, a.comb_items,
                     a.kvc_items, (int)a.n_comb, (int)a.n_kvc, HD, HkD, (int)chunks);
}

#define VAFA_INST(T)                                                        \
  template void launch_masked_dq<T, 64>(const MaskedArgs &, hipStream_t);   \
  template void launch_masked_dq<T, 128>(const MaskedArgs &, hipStream_t);  \
  template void launch_masked_dq<T, 256>(const MaskedArgs &, hipStream_t);  \
  template void launch_masked_dkv<T, 64>(const MaskedArgs &, hipStream_t);  \
  template void launch_masked_dkv<T, 128>(const MaskedArgs &, hipStream_t); \
  template void launch_masked_dkv<T, 256>(const MaskedArgs &, hipStream_t); \
  template void launch_masked_sum<T>(const MaskedArgs &, hipStream_t);
VAFA_INST(bf16)
VAFA_INST(f16)
#undef VAFA_INST

}  // namespace vafa
