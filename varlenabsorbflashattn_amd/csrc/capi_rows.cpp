// extern "C" entry points of the norms of queries and keys with the position rotation:
// argument checks, dispatch.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cstdint>
#include <initializer_list>

#include "../../include/vafa.h"
#include "common.h"
#include "kernels.h"

namespace vafa {
int fail(int code, const char *fmt, ...);
int check_head_rows(const char *what, int64_t D, int64_t rot, float eps, float rot_scale);

namespace {

constexpr const char *kWhat = "packed_qk_norm_rope";

int check_sizes(int64_t T, int64_t H, int64_t Hk, int64_t D, int64_t rot, float eps,
                float rot_scale) {
  if (int rc = check_head_rows(kWhat, D, rot, eps, rot_scale)) return rc;
  if (H < 1 || H > 4096 || Hk < 1 || Hk > 4096)
    return fail(VAFA_ERR_VALUE, "%s: %lld query heads and %lld key heads", kWhat, (long long)H,
                (long long)Hk);
  if (T < 0 || T > kMaskedMaxTokens || !grid_ok(T * ((H + Hk) * (D / 16)) / 256 + 1, 256))
    return fail(VAFA_ERR_VALUE, "%s: %lld tokens are too many for a call", kWhat, (long long)T);
  return VAFA_OK;
}

int check_dtype(int32_t dtype) {
  if (dtype != VAFA_BF16 && dtype != VAFA_F16)
    return fail(VAFA_ERR_ASSERT, "%s: dtype not supported (float16, bfloat16)", kWhat);
  return VAFA_OK;
}

// Rows of whole 16-byte pieces.
int check_rows(std::initializer_list<const void *> ptrs, std::initializer_list<int64_t> strides) {
  for (const void *p : ptrs)
    if ((uintptr_t)p % 16 != 0)
      return fail(VAFA_ERR_VALUE, "%s: operands must be 16-byte aligned", kWhat);
  for (int64_t s : strides)
    if (s < 0 || s % 8 != 0 || s > UINT32_MAX)
      return fail(VAFA_ERR_VALUE, "%s: strides must be multiples of 8 elements below 2^32, got %lld",
                  kWhat, (long long)s);
  return VAFA_OK;
}

int check_given(std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (p == nullptr) return fail(VAFA_ERR_VALUE, "%s: a required pointer is NULL", kWhat);
  return VAFA_OK;
}

int check_launch() {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return fail(VAFA_ERR_RUNTIME, "%s: kernel launch failed: %s", kWhat, hipGetErrorString(e));
  return VAFA_OK;
}

}  // namespace
}  // namespace vafa

using namespace vafa;

extern "C" {

int vafa_qk_norm_rope_fwd(const void *q, int64_t q_token, int64_t q_head, int64_t H, const void *k,
                          int64_t k_token, int64_t k_head, int64_t Hk, int64_t T, int64_t D,
                          const int32_t *positions, const float *inv_freq, int64_t rot,
                          int32_t interleaved, float rot_scale, const void *q_weight,
                          const void *k_weight, int32_t weights_f32, float eps, void *q_out,
                          void *k_out, int32_t dtype, void *stream) {
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_sizes(T, H, Hk, D, rot, eps, rot_scale)) return rc;
  if (int rc = check_rows({q, k, q_out, k_out}, {q_token, q_head, k_token, k_head})) return rc;
  if (T == 0) return VAFA_OK;
  if (int rc = check_given({q, k, q_out, k_out})) return rc;
  if (rot > 0)
    if (int rc = check_given({positions, inv_freq})) return rc;
  HeadRowsArgs s{};
  s.a.q = q; s.a.k = k; s.a.q_out = q_out; s.a.kc = k_out; s.a.kc_head = D;
  s.a.q_token = q_token; s.a.q_head = q_head; s.a.k_token = k_token; s.a.k_head = k_head;
  s.a.inv_freq = inv_freq; s.a.T = T; s.a.H = (int)H; s.a.Hk = (int)Hk; s.a.D = (int)D;
  s.a.rot = (int)rot; s.a.interleaved = interleaved != 0;
  s.positions = positions; s.q_weight = q_weight; s.k_weight = k_weight;
  s.weights_f32 = weights_f32 != 0; s.packed = 1; s.eps = eps; s.rot_scale = rot_scale;
  if (dtype == VAFA_BF16)
    launch_head_rows<bf16>(s, (hipStream_t)stream);
  else
    launch_head_rows<f16>(s, (hipStream_t)stream);
  return check_launch();
}

int64_t vafa_qk_norm_rope_bwd_workspace(int64_t T, int64_t H, int64_t Hk, int64_t D) {
  if (check_sizes(T, H, Hk, D, 0, 0.f, 1.f)) return -1;
  return head_rows_bwd_blocks(T, H + Hk, D) * 2 * D * 4;
}

int vafa_qk_norm_rope_bwd(const void *q, int64_t q_token, int64_t q_head, int64_t H, const void *k,
                          int64_t k_token, int64_t k_head, int64_t Hk, int64_t T, int64_t D,
                          const int32_t *positions, const float *inv_freq, int64_t rot,
                          int32_t interleaved, float rot_scale, const void *q_weight,
                          const void *k_weight, int32_t weights_f32, float eps,
                          const void *dq_out, const void *dk_out, void *dq, void *dk,
                          void *dq_weight, void *dk_weight, int32_t dtype, void *workspace,
                          int64_t workspace_bytes, void *stream) {
  if (int rc = check_dtype(dtype)) return rc;
  if (int rc = check_sizes(T, H, Hk, D, rot, eps, rot_scale)) return rc;
  if (int rc = check_rows({q, k, dq_out, dk_out, dq, dk}, {q_token, q_head, k_token, k_head}))
    return rc;
  if ((dq_weight != nullptr && q_weight == nullptr) || (dk_weight != nullptr && k_weight == nullptr))
    return fail(VAFA_ERR_VALUE, "%s: a gradient of weights that are not there", kWhat);
  const bool sums = dq_weight != nullptr || dk_weight != nullptr;
  const int64_t bytes = vafa_qk_norm_rope_bwd_workspace(T, H, Hk, D);
  if (sums && (workspace_bytes < bytes || workspace == nullptr || (uintptr_t)workspace % 16 != 0))
    return fail(VAFA_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed (16-byte aligned)",
                (long long)workspace_bytes, (long long)bytes);
  if (T > 0) {
    if (int rc = check_given({q, k, dq_out, dk_out, dq, dk})) return rc;
    if (rot > 0)
      if (int rc = check_given({positions, inv_freq})) return rc;
  }
  HeadRowsBwdArgs a{};
  a.q = q; a.k = k; a.dq_out = dq_out; a.dk_out = dk_out; a.dq = dq; a.dk = dk;
  a.dq_weight = dq_weight; a.dk_weight = dk_weight; a.positions = positions; a.inv_freq = inv_freq;
  a.q_weight = q_weight; a.k_weight = k_weight; a.part = sums ? (float *)workspace : nullptr;
  a.q_token = q_token; a.q_head = q_head; a.k_token = k_token; a.k_head = k_head; a.T = T;
  a.blocks = T > 0 ? head_rows_bwd_blocks(T, H + Hk, D) : 0;
  a.H = (int)H; a.Hk = (int)Hk; a.D = (int)D; a.rot = (int)rot; a.interleaved = interleaved != 0;
  a.weights_f32 = weights_f32 != 0; a.eps = eps; a.rot_scale = rot_scale;
  if (dtype == VAFA_BF16)
    launch_head_rows_bwd<bf16>(a, (hipStream_t)stream);
  else
    launch_head_rows_bwd<f16>(a, (hipStream_t)stream);
  return check_launch();
}

}  // extern "C"
