// Backward of packed_masked_attn on gfx950 matrix cores (bf16 / f16).
//
// Deterministic, two kernels that recompute P = 2^(x - LSE) from the forward's LSE, laid
// out as the packed varlen backward (varlen_bwd_mfma.hip):
//   * dQ, query-major over the forward's items: S^T = K Q^T, dP^T = V dO^T,
//     dQ^T += K^T dS^T, and delta = rowsum(O dO) for the other kernel;
//   * dK/dV, key-major: a workgroup owns a key tile of one key head, walks the queries
//     that see it of every query head that shares the key head (of one of gsplit parts
//     of them, where a launch has few key tiles: fp32 partials, summed in order), and
//     accumulates dV^T += dO^T P, dK^T += Q^T dS.
// With y = cap tanh(z / cap): dz = dx (1 - tanh^2), formed from e of cap_e as 4 e (1 - e).
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
    const T *__restrict__ dout, const T *__restrict__ o, const float *__restrict__ lse,
    float *__restrict__ delta, float *__restrict__ lse_out, T *__restrict__ dq,
    float *__restrict__ part_dq, const int32_t *__restrict__ items,
    const float *__restrict__ slopes, ScoreArgs sa, int H, int Hk, int window, float scale) {
  using M = Mfma<T>;
  using S = DqSmem<D>;
  using L = GTile<D>;
  constexpr int NC = D / 16, ND = D / 32;
  constexpr int kPre = 4;
  constexpr bool kLog2 = kCap || kBias;
  extern __shared__ __align__(16) unsigned char smem_raw[];
  T *smem = reinterpret_cast<T *>(smem_raw);

  const int G = H / Hk;
  const int item = blockIdx.x / H, h = head_of(blockIdx.x % H, Hk, G), hk = h / G;
  const PlanItem it = load_item(items, item);
  const int q0 = it.v[0], q1 = it.v[1], pbase = it.v[4], diag = it.v[5], pre = it.v[6];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int qrow = q0 + wave * 32 + lrow;
  const bool row_ok = qrow < q1;
  const bool wave_active = q0 + wave * 32 < q1;
  const int p = qrow + diag;
  const int p0 = q0 + wave * 32 + diag;
  const int p1 = (q0 + wave * 32 + 31 < q1 ? q0 + wave * 32 + 31 : q1 - 1) + diag;
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
    load_rows<T, D, NS>(stg, src, walk_key<kRB>(kw, j), walk_end(kw, j), Hk, hk, st);
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
    const rsrc_t rq = make_rsrc(q + (int64_t)q0 * H * D, nb);
    const rsrc_t rd = make_rsrc(dout + (int64_t)q0 * H * D, nb);
    const rsrc_t ro = make_rsrc(o + (int64_t)q0 * H * D, nb);
    const int off = ((wave * 32 + lrow) * H + h) * D * 2 + lhalf * 16;
    u32x4 ov[NC];
#pragma unroll
    for (int cc = 0; cc < NC; ++cc) ov[cc] = buf_load16(ro, off + cc * 32);
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
      for (int e = 0; e < 8; ++e) a = __builtin_fmaf(to_f(x[e]), to_f(dof[cc][e]), a);
      sc += a;
    }
    Dr = sc + __shfl_xor(sc, 32, 64);
  }
  // rows past q1, and rows that see no key, get LSE = +inf: their P is 0
  float Lr = row_ok ? lse[(int64_t)qrow * H + h] : __builtin_inff();
  if (Lr == kNegInf) Lr = __builtin_inff();
  if (row_ok && lhalf == 0 && it.v[7] != 0) {  // the item that owns its rows' first keys
    delta[(int64_t)qrow * H + h] = Dr;
    lse_out[(int64_t)qrow * H + h] = Lr;
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
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j2 = k_lane + off(r);
          if (j2 >= ke || !visible(j2, p, pre, window)) s[r] = kNegInf;
        }
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
  const int rows = uniform_clamp(q1 - (q0 + wave * 32), 32);
  if (pbase < 0)
    RS::rows16(acc, [&](float x) { return static_cast<T>(x * scale); }, stage,
               dq + ((int64_t)(q0 + wave * 32) * H + h) * D, (int64_t)H * D, rows);
  else
    RS::rows32(acc, scale, stage, part_dq + ((int64_t)(pbase + wave * 32) * H + h) * D,
               (int64_t)H * D, rows);
}

// ---- dK / dV -----------------------------------------------------------------------
template <typename T, int D, int NW, bool kCap, bool kBias>
__global__ __launch_bounds__(64 * NW, D >= 256 && NW < 8 ? 1 : 2) void masked_dkv_kernel(
    const T *__restrict__ q, const T *__restrict__ k, const T *__restrict__ v,
    const T *__restrict__ dout, const float *__restrict__ lse, const float *__restrict__ delta,
    T *__restrict__ dk, T *__restrict__ dv, float *__restrict__ part_dk,
    float *__restrict__ part_dv, const int32_t *__restrict__ items,
    const float *__restrict__ slopes, ScoreArgs sa, int H, int Hk, int window, int gsplit,
    int64_t T_k, float scale) {
  using M = Mfma<T>;
  using S = DkvSmem<D>;
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

  const int G = H / Hk;
  const int item = blockIdx.x / (Hk * gsplit), part = blockIdx.x % (Hk * gsplit);
  const int hk = part % Hk, gs = part / Hk;
  const int hg0 = hk * G + G * gs / gsplit, hg1 = hk * G + G * (gs + 1) / gsplit;
  const PlanItem it = load_item(items, item);
  const int k0 = it.v[0], k1 = it.v[1], q0 = it.v[2], q1 = it.v[3], diag = it.v[4], pre = it.v[5];
  const int tid = threadIdx.x, lane = tid & 63;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kgrp = kShare ? (wave & 3) : wave;
  const int dpart = kShare ? (wave >> 2) : 0;
  const int lrow = lane & 31, lhalf = lane >> 5;
  const int kw0 = k0 + kgrp * 32;  // the wave's first and last key
  const int kw1 = (kw0 + 32 < k1 ? kw0 + 32 : k1) - 1;
  const bool wave_active = kw0 < k1;

  auto issue = [&](int h, int qb, int buf) {
    unsigned char *base = smem_raw + buf * S::kBufBytes;
    dma_block_rows<T, D, NW>(q, qb, q1, H, h, lds_addr(base), wave, lane);
    dma_block_rows<T, D, NW>(dout, qb, q1, H, h, lds_addr(base + S::kQs * 2), wave, lane);
    const float *vec = (wave & 1) ? delta : lse;
    const int rows = uniform_clamp(q1 - qb, kRB);
    const u32x4 rv = rsrc_words32(vec + (int64_t)qb * H + h, (uint32_t)(rows * H * 4));
    if (lane < kRB) lds_dma4(rv, lds_addr(base + 2 * S::kQs * 2 + (wave & 1) * kRB * 4), lane * H * 4);
  };
  const int nq = (q1 - q0 + kRB - 1) / kRB;  // query blocks of one head
  const int nblk = nq * (hg1 - hg0);
  if (nblk > 0) issue(hg0, q0, 0);

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
  }
  f32x16 adk[NDO], adv[NDO];
#pragma unroll
  for (int i = 0; i < NDO; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) adk[i][r] = adv[i][r] = 0.f;

  const int a_off = L::row(lrow) + lhalf * 8 + dpart * NDO * 32;
  const int t_off = L::row(4 * (lane >> 5) + ((lane & 15) >> 2)) + ((lane >> 4) & 1) * 16 +
                    4 * (lane & 3);
  int h = hg0, qb = q0;  // of the current block
  auto blk = [&](int j, auto bufc) {
    constexpr int B = decltype(bufc)::value;
    const int hc = h, qc = qb;
    qb += kRB;
    if (qb >= q1) {
      qb = q0;
      ++h;
    }
    wait_vmcnt<0>();
    __syncthreads();
    if (j + 1 < nblk) issue(h, qb, 1 - B);
    const unsigned char *base = smem_raw + B * S::kBufBytes;
    const lds_cptr<T> qs = as_lds(reinterpret_cast<const T *>(base));
    const lds_cptr<T> ds_ = qs + S::kQs;
    const float *ls = reinterpret_cast<const float *>(base + 2 * S::kQs * 2);
    const int p0 = qc + diag, p1 = (qc + kRB < q1 ? qc + kRB : q1) - 1 + diag;
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
        }
      }
    }
    if (active) {
      auto top = [&](int i) {
        const lds_cptr<T> tp = (((i / NDO) & 1) ? qs : ds_) + t_off +
                               ((i / NDO) >> 1) * 4 * L::P2 + (dpart * NDO + i % NDO) * 32;
        return as_v8<T>(join(lds_tr8<T>(tp), lds_tr8<T>(tp + 2 * L::P2)));
      };
      typename M::v8 tring[kPre];
#pragma unroll
      for (int i = 0; i < kPre; ++i) tring[i] = top(i);
      // row r of a lane is query q_lane + off(r), its key kw0 + lrow
      const int q_lane = qc + lhalf * 4;
      auto off = [](int r) { return (r >> 2) * 8 + (r & 3); };
      // with a cap, dP - delta is formed (and multiplied by the cap's derivative) here
      constexpr bool kDeltaHere = kCap && !kDeltaInChain;
      if constexpr (kLog2) {
        const float back = (float)(q_lane + diag - kw0 - lrow);
        float slope2 = 0.f;
        if constexpr (kBias) slope2 = slopes[hc] * kLog2e;
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          float z = s[r] * sa.c;
          if constexpr (kCap) {
            const float e = cap_e(z), e4 = 4.f * e;
            z = __builtin_fmaf(-2.f * sa.cap2, e, sa.cap2);
            if constexpr (kDeltaHere) dp[r] -= ls[kRB + off(r) + lhalf * 4];
            dp[r] *= __builtin_fmaf(-e4, e, e4);
          }
          if constexpr (kBias) z = __builtin_fmaf(-slope2, fabsf(back + (float)off(r)), z);
          s[r] = z;
        }
      }
      if (qc + kRB > q1 || !all_visible(kw0, kw1, p0, p1, pre, window)) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int qr = q_lane + off(r);
          if (qr >= q1 || !visible(kw0 + lrow, qr + diag, pre, window)) s[r] = kNegInf;
        }
      }
      auto p_of = [&](float x, float lr) {
        return fast_exp2(kLog2 ? x - lr : __builtin_fmaf(x, sa.c, -lr));
      };
      auto ds_of = [&](float p, float a, float dl) {
        if constexpr (kDeltaInChain)
          return -(p * a);
        else if constexpr (kDeltaHere)
          return p * a;
        else
          return p * (a - dl);
      };
      constexpr bool kDl = !kDeltaInChain && !kDeltaHere;
      typename M::v8 pb[2], sb[2];
#pragma unroll
      for (int g = 0; g < 2; ++g) {
        const f32x4 Lq = *reinterpret_cast<const f32x4 *>(ls + g * 8 + lhalf * 4);
        const f32x4 Dl = kDl ? *reinterpret_cast<const f32x4 *>(ls + kRB + g * 8 + lhalf * 4)
                             : f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = g * 4 + e;
          const float p = p_of(s[r], Lq[e]);
          s[r] = p;
          dp[r] = ds_of(p, dp[r], Dl[e]);
        }
      }
      pb[0] = pack8<T>(s, 0);
      sb[0] = pack8<T>(dp, 0);
      constexpr int kSteps = 2 * NDO < 8 ? 2 * NDO : 8;
      constexpr int kRowsPer = 8 / kSteps;
      constexpr int kEvery = 2 * NDO / kSteps;
      auto lse_at = [&](int r) { return ls[(r >> 2) * 8 + lhalf * 4 + (r & 3)]; };
      auto del_at = [&](int r) {
        return kDl ? ls[kRB + (r >> 2) * 8 + lhalf * 4 + (r & 3)] : 0.f;
      };
      float Ln[kRowsPer], Dn[kRowsPer];
#pragma unroll
      for (int rr = 0; rr < kRowsPer; ++rr) Ln[rr] = lse_at(8 + rr), Dn[rr] = del_at(8 + rr);
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
          float Lc[kRowsPer], Dc[kRowsPer];
#pragma unroll
          for (int rr = 0; rr < kRowsPer; ++rr) {
            Lc[rr] = Ln[rr], Dc[rr] = Dn[rr];
            if (g + 1 < kSteps) {
              const int rn = 8 + (g + 1) * kRowsPer + rr;
              Ln[rr] = lse_at(rn);
              Dn[rr] = del_at(rn);
            }
          }
#pragma unroll
          for (int rr = 0; rr < kRowsPer; ++rr) {
            const int r = 8 + g * kRowsPer + rr;
            const float p = p_of(s[r], Lc[rr]);
            s[r] = p;
            dp[r] = ds_of(p, dp[r], Dc[rr]);
          }
          if (g == kSteps - 1) {
            pb[1] = pack8<T>(s, 8);
            sb[1] = pack8<T>(dp, 8);
          }
        }
        __builtin_amdgcn_sched_barrier(0);
      }
    }
  };
  for (int j = 0; j < nblk; j += 2) {
    blk(j, std::integral_constant<int, 0>{});
    if (j + 1 < nblk) blk(j + 1, std::integral_constant<int, 1>{});
  }
  wait_vmcnt<0>();

  __syncthreads();
  if (!wave_active) return;
  using RS = RowStore<T, NDO>;
  unsigned char *stage = smem_raw + wave * RS::kBytes;
  const int rows = uniform_clamp(k1 - kw0, 32);
  const int64_t off = ((int64_t)kw0 * Hk + hk) * D + dpart * NDO * 32;
  if (gsplit == 1) {
    RS::rows16(adk, [&](float x) { return static_cast<T>(x * scale); }, stage, dk + off,
               (int64_t)Hk * D, rows);
    RS::rows16(adv, [](float x) { return static_cast<T>(x); }, stage, dv + off, (int64_t)Hk * D,
               rows);
  } else {
    const int64_t po = (int64_t)gs * T_k * Hk * D + off;
    RS::rows32(adk, scale, stage, part_dk + po, (int64_t)Hk * D, rows);
    RS::rows32(adv, 1.f, stage, part_dv + po, (int64_t)Hk * D, rows);
  }
}

// dk / dv (blockIdx.y) = sum over the gsplit partials, 8 features per thread.
template <typename T>
__global__ __launch_bounds__(256) void masked_group_sum_kernel(const float *part_dk,
                                                               const float *part_dv, T *dk, T *dv,
                                                               int64_t n, int gsplit) {
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 8;
  if (i >= n) return;
  const float *src = blockIdx.y ? part_dv : part_dk;
  f32x4 a = f32x4{0.f, 0.f, 0.f, 0.f}, b = a;
  for (int g = 0; g < gsplit; ++g) {
    a += *reinterpret_cast<const f32x4 *>(src + g * n + i);
    b += *reinterpret_cast<const f32x4 *>(src + g * n + i + 4);
  }
  typename Mfma<T>::v8 w;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    w[e] = static_cast<T>(a[e]);
    w[4 + e] = static_cast<T>(b[e]);
  }
  *reinterpret_cast<typename Mfma<T>::v8 *>((blockIdx.y ? dv : dk) + i) = w;
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
  constexpr int kBase = dkv_lds_bytes<T, D, NW>();
  return kBase > kStage ? kBase : kStage;
}

template <typename T, int D, int NW, bool kCap, bool kBias>
void launch_dq_v(const MaskedArgs &a, hipStream_t st) {
  constexpr auto fn = &masked_dq_kernel<T, D, NW, kCap, kBias>;
  const int smem = masked_dq_lds<T, D, NW>();
  allow_dynamic_lds(reinterpret_cast<const void *>(fn), smem);
  hipLaunchKernelGGL(fn, dim3((unsigned)(a.n_items * a.H)), dim3(64 * NW), smem, st,
                     (const T *)a.q, (const T *)a.k, (const T *)a.v, (const T *)a.dout,
                     (const T *)a.o_in, a.lse_in, a.delta, a.lse, (T *)a.dq, a.part_o, a.items,
                     a.slopes, ScoreArgs{a.c, a.cap2}, a.H, a.Hk, a.window, a.scale);
}
template <typename T, int D, int NW, bool kCap, bool kBias>
void launch_dkv_v(const MaskedArgs &a, hipStream_t st) {
  constexpr auto fn = &masked_dkv_kernel<T, D, NW, kCap, kBias>;
  const int smem = masked_dkv_lds<T, D, NW>();
  allow_dynamic_lds(reinterpret_cast<const void *>(fn), smem);
  hipLaunchKernelGGL(fn, dim3((unsigned)(a.n_kv * a.Hk * a.gsplit)), dim3(64 * NW), smem, st,
                     (const T *)a.q, (const T *)a.k, (const T *)a.v, (const T *)a.dout, a.lse,
                     a.delta, (T *)a.dk, (T *)a.dv, a.part_dk, a.part_dv, a.kv_items, a.slopes,
                     ScoreArgs{a.c, a.cap2}, a.H, a.Hk, a.window, a.gsplit, a.T_k, a.scale);
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
  if (a.n_items == 0) return;
  if constexpr (D <= 128) {
    if (a.q_tile == kVarlenWideTile) return launch_dq_nw<T, D, 8>(a, st);
  }
  launch_dq_nw<T, D, 4>(a, st);
}

template <typename T, int D>
void launch_masked_dkv(const MaskedArgs &a, hipStream_t st) {
  if (a.n_kv == 0) return;
  if constexpr (D == 256) {
    launch_dkv_nw<T, D, 8>(a, st);
  } else {
    if constexpr (D == 128) {
      if (a.k_tile == kVarlenWideTile) return launch_dkv_nw<T, D, 8>(a, st);
    }
    launch_dkv_nw<T, D, 4>(a, st);
  }
}

template <typename T>
void launch_masked_group_sum(const MaskedArgs &a, hipStream_t st) {
  const int64_t n = a.T_k * a.Hk * a.D;
  if (a.gsplit == 1 || n == 0) return;
  hipLaunchKernelGGL((masked_group_sum_kernel<T>), dim3((unsigned)((n / 8 + 255) / 256), 2),
                     dim3(256), 0, st, a.part_dk, a.part_dv, (T *)a.dk, (T *)a.dv, n, a.gsplit);
}

#define VAFA_INST(T)                                                        \
  template void launch_masked_dq<T, 64>(const MaskedArgs &, hipStream_t);   \
  template void launch_masked_dq<T, 128>(const MaskedArgs &, hipStream_t);  \
  template void launch_masked_dq<T, 256>(const MaskedArgs &, hipStream_t);  \
  template void launch_masked_dkv<T, 64>(const MaskedArgs &, hipStream_t);  \
  template void launch_masked_dkv<T, 128>(const MaskedArgs &, hipStream_t); \
  template void launch_masked_dkv<T, 256>(const MaskedArgs &, hipStream_t); \
  template void launch_masked_group_sum<T>(const MaskedArgs &, hipStream_t);
VAFA_INST(bf16)
VAFA_INST(f16)
#undef VAFA_INST

}  // namespace vafa
