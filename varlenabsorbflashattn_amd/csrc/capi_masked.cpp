// extern "C" entry points of packed_masked_attn: argument checks, workspace carving and
// kernel dispatch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <initializer_list>

#include "../../include/vafa.h"
#include "common.h"
#include "kernels.h"

namespace vafa {
int fail(int code, const char *fmt, ...);

namespace {

int check_plan(const vafa_plan_info *info, int64_t Hk, int64_t D) {
  if (info == nullptr || info->magic != VAFA_PLAN_MAGIC || info->kind != 3)
    return fail(VAFA_ERR_VALUE, "plan does not belong to this operator");
  if (D != 64 && D != 128 && D != 256)
    return fail(VAFA_ERR_ASSERT, "head_dim %lld not supported (64, 128, 256)", (long long)D);
  if (info->H > kMaskedMaxHeads)
    return fail(VAFA_ERR_VALUE, "more than %lld query heads", (long long)kMaskedMaxHeads);
  if (Hk < 1 || info->H < 1 || info->H % Hk != 0)
    return fail(VAFA_ERR_ASSERT, "%lld query heads do not divide among %lld key heads",
                (long long)info->H, (long long)Hk);
  if (info->xcd_heads != masked_set_log2(info->H / Hk))
    return fail(VAFA_ERR_VALUE, "the plan was built for another number of key heads");
  const bool q_ok =
      info->q_tile == kVarlenTile || (info->q_tile == kVarlenWideTile && D == 128);
  if (!q_ok || info->k_tile != kVarlenTile)
    return fail(VAFA_ERR_VALUE, "plan tiles (%lld queries, %lld keys) do not fit head_dim %lld",
                (long long)info->q_tile, (long long)info->k_tile, (long long)D);
  return VAFA_OK;
}

int check_call(const vafa_plan_info *info, int64_t Hk, int64_t D, int32_t dtype, float scale,
               float softcap, int64_t window, std::initializer_list<const void *> ptrs) {
  if (int rc = check_plan(info, Hk, D)) return rc;
  if (dtype != VAFA_BF16 && dtype != VAFA_F16)
    return fail(VAFA_ERR_ASSERT, "dtype not supported (float16, bfloat16)");
  if (!std::isfinite(scale * kLog2e)) return fail(VAFA_ERR_VALUE, "scale must be finite");
  if (!softcap_ok(softcap))
    return fail(VAFA_ERR_VALUE, "softcap must be positive, from %g to %g", (double)kMinSoftcap,
                (double)kMaxSoftcap);
  if (softcap > 0.f && !std::isfinite(2.f * kLog2e * scale / softcap))
    return fail(VAFA_ERR_VALUE, "scale / softcap is not finite");
  if (window < 0) return fail(VAFA_ERR_VALUE, "window must be positive");
  for (const void *p : ptrs)
    if ((uintptr_t)p % 16 != 0) return fail(VAFA_ERR_VALUE, "operands must be 16-byte aligned");
  return VAFA_OK;
}

int check_given(const char *what, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (p == nullptr) return fail(VAFA_ERR_VALUE, "%s: a required pointer is NULL", what);
  return VAFA_OK;
}

inline int64_t up(int64_t x) { return (x + 255) / 256 * 256; }

struct Ws {
  float *part_o, *part_lse, *delta, *lse, *part_dk, *part_dv;
  int64_t bytes;
};

Ws carve(void *ws, const vafa_plan_info *info, int64_t Hk, int64_t D, bool bwd) {
  Ws w{};
  char *base = static_cast<char *>(ws);
  int64_t used = 0;
  auto take = [&](int64_t n) {
    float *p = base != nullptr ? reinterpret_cast<float *>(base + used) : nullptr;
    used += up(n * 4);
    return p;
  };
  const int64_t rows = info->n_part_rows * info->H;
  w.part_o = take(rows * D);
  if (!bwd) {
    w.part_lse = take(rows);
  } else {
    w.delta = take(info->T_q * info->H);
    w.lse = take(info->T_q * info->H);
    w.part_dk = take(info->n_fpart_rows * Hk * D);
    w.part_dv = take(info->n_fpart_rows * Hk * D);
  }
  w.bytes = used;
  return w;
}

MaskedArgs args_of(const vafa_plan_info *info, const int32_t *plan, int64_t Hk, int64_t D,
                   float scale, float softcap, int64_t window, const float *slopes) {
  MaskedArgs a{};
  a.items = plan + info->off_fwd; a.n_items = info->n_fwd;
  a.comb_items = plan + info->off_comb; a.n_comb = info->n_comb;
  a.comb_rows = (int)info->max_comb_rows;
  a.kv_items = plan + info->off_kv; a.n_kv = info->n_kv;
  a.kvc_items = plan + info->off_fcomb; a.n_kvc = info->n_fcomb;
  a.kvc_rows = (int)info->max_fcomb_rows;
  a.H = (int)info->H; a.Hk = (int)Hk; a.D = (int)D;
  a.q_tile = (int)info->q_tile;
  a.window = (int)(window > 0 ? std::min(window, kMaskedMaxTokens) : kMaskedMaxTokens);
  a.lg = masked_set_log2(info->H / Hk);
  a.slopes = slopes;
  a.scale = scale;
  a.c = softcap > 0.f ? 2.f * kLog2e * scale / softcap : scale * kLog2e;
  a.cap2 = softcap * kLog2e;
  return a;
}

int check_ws(int64_t have, const void *ws, int64_t need) {
  if (have < need || (need > 0 && (ws == nullptr || (uintptr_t)ws % 16 != 0)))
    return fail(VAFA_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed (16-byte aligned)",
                (long long)have, (long long)need);
  return VAFA_OK;
}

// Blocks of every launch (rows of sums by 2048 values).
int check_grids(const MaskedArgs &a, const vafa_plan_info *info, bool bwd) {
  const int64_t sets = a.H >> a.lg, HD = (int64_t)a.H * a.D, HkD = (int64_t)a.Hk * a.D;
  auto chunks = [](int64_t values) { return (values + 2047) / 2048; };
  bool ok = grid_ok(a.n_items * sets, !bwd && a.q_tile == kVarlenWideTile ? 512 : 256);
  if (bwd)
    ok = ok && grid_ok(a.n_kv * a.Hk, a.D == 256 ? 512 : 256) &&
         grid_ok((a.n_comb + 2 * a.n_kvc) *
                     std::max(chunks(a.comb_rows * HD), chunks(a.kvc_rows * HkD)), 256);
  else
    ok = ok && grid_ok(a.n_comb * chunks(a.comb_rows * HD), 256);
  return ok ? VAFA_OK
            : fail(VAFA_ERR_VALUE, "more tiles than a launch can have (%lld segments, %lld tokens)",
                   (long long)info->n_seg, (long long)std::max(info->T_q, info->T_k));
}

int check_launch(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return fail(VAFA_ERR_RUNTIME, "%s: kernel launch failed: %s", what, hipGetErrorString(e));
  return VAFA_OK;
}

template <typename T>
void fwd(const MaskedArgs &a, hipStream_t st) {
  if (a.D == 64) launch_masked_fwd<T, 64>(a, st);
  if (a.D == 128) launch_masked_fwd<T, 128>(a, st);
  if (a.D == 256) launch_masked_fwd<T, 256>(a, st);
  if (a.D == 64) launch_masked_join<T, 64>(a, st);
  if (a.D == 128) launch_masked_join<T, 128>(a, st);
  if (a.D == 256) launch_masked_join<T, 256>(a, st);
}

template <typename T>
void bwd(const MaskedArgs &a, hipStream_t st) {
  if (a.D == 64) launch_masked_dq<T, 64>(a, st);
  if (a.D == 128) launch_masked_dq<T, 128>(a, st);
  if (a.D == 256) launch_masked_dq<T, 256>(a, st);
  if (a.D == 64) launch_masked_dkv<T, 64>(a, st);
  if (a.D == 128) launch_masked_dkv<T, 128>(a, st);
  if (a.D == 256) launch_masked_dkv<T, 256>(a, st);
  launch_masked_sum<T>(a, st);
}

}  // namespace
}  // namespace vafa

using namespace vafa;

extern "C" {

int64_t vafa_masked_fwd_workspace(const vafa_plan_info *info, int64_t Hk, int64_t D) {
  if (check_plan(info, Hk, D)) return -1;
  return carve(nullptr, info, Hk, D, false).bytes;
}

int64_t vafa_masked_bwd_workspace(const vafa_plan_info *info, int64_t Hk, int64_t D) {
  if (check_plan(info, Hk, D)) return -1;
  return carve(nullptr, info, Hk, D, true).bytes;
}

int vafa_masked_fwd(const void *q, const void *k, const void *v, void *o, void *o_lo,
                    float *lse, const int32_t *plan_dev, const vafa_plan_info *info, int64_t Hk,
                    int64_t D, int32_t dtype, float scale, float softcap, int64_t window,
                    const float *slopes, void *workspace, int64_t workspace_bytes, void *stream) {
  if (int rc = check_call(info, Hk, D, dtype, scale, softcap, window, {q, k, v, o, o_lo}))
    return rc;
  const char *what = "vafa_masked_fwd";
  if (info->T_q > 0)
    if (int rc = check_given(what, {q, o, plan_dev})) return rc;
  if (info->T_k > 0)
    if (int rc = check_given(what, {k, v})) return rc;
  const Ws w = carve(workspace, info, Hk, D, false);
  if (int rc = check_ws(workspace_bytes, workspace, w.bytes)) return rc;
  MaskedArgs a = args_of(info, plan_dev, Hk, D, scale, softcap, window, slopes);
  a.q = q; a.k = k; a.v = v; a.o = o; a.o_lo = (uint8_t *)o_lo; a.lse = lse;
  a.part_o = w.part_o; a.part_lse = w.part_lse;
  if (int rc = check_grids(a, info, false)) return rc;
  if (dtype == VAFA_BF16)
    fwd<bf16>(a, (hipStream_t)stream);
  else
    fwd<f16>(a, (hipStream_t)stream);
  return check_launch(what);
}

int vafa_masked_bwd(const void *q, const void *k, const void *v, const void *o,
                    const void *o_lo, const void *dout, const float *lse, void *dq, void *dk,
                    void *dv, const int32_t *plan_dev, const vafa_plan_info *info, int64_t Hk,
                    int64_t D, int32_t dtype, float scale, float softcap, int64_t window,
                    const float *slopes, void *workspace, int64_t workspace_bytes, void *stream) {
  if (int rc = check_call(info, Hk, D, dtype, scale, softcap, window,
                          {q, k, v, o, o_lo, dout, dq, dk, dv}))
    return rc;
  const char *what = "vafa_masked_bwd";
  if (o_lo == nullptr && info->T_q > 0)
    return fail(VAFA_ERR_VALUE, "the backward needs the forward's o_lo");
  if (info->T_q > 0)
    if (int rc = check_given(what, {q, o, dout, lse, dq, plan_dev})) return rc;
  if (info->T_k > 0)
    if (int rc = check_given(what, {k, v, dk, dv, plan_dev})) return rc;
  const Ws w = carve(workspace, info, Hk, D, true);
  if (int rc = check_ws(workspace_bytes, workspace, w.bytes)) return rc;
  MaskedArgs a = args_of(info, plan_dev, Hk, D, scale, softcap, window, slopes);
  a.items = plan_dev + info->off_dq; a.n_items = info->n_dq;
  a.comb_items = plan_dev + info->off_dqc; a.n_comb = info->n_dqc;
  a.comb_rows = (int)info->max_dqc_rows;
  a.q = q; a.k = k; a.v = v; a.o_in = o; a.o_lo_in = (const uint8_t *)o_lo; a.dout = dout; a.lse_in = lse;
  a.dq = dq; a.dk = dk; a.dv = dv;
  a.part_o = w.part_o; a.delta = w.delta; a.lse = w.lse;
  a.part_dk = w.part_dk; a.part_dv = w.part_dv;
  if (int rc = check_grids(a, info, true)) return rc;
  if (dtype == VAFA_BF16)
    bwd<bf16>(a, (hipStream_t)stream);
  else
    bwd<f16>(a, (hipStream_t)stream);
  return check_launch(what);
}

}  // extern "C"
