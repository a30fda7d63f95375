// extern "C" entry points of the paged key-value cache: argument checks, the
// decoding attention's grid and workspace, dispatch.
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
int check_head_rows(const char *what, int64_t D, int64_t rot, float eps, float rot_scale);

namespace {

int check_cache(const char *what, const vafa_paged_cache *c) {
  if (c == nullptr) return fail(VAFA_ERR_VALUE, "%s: no cache", what);
  if (c->n_seq < 0 || c->n_seq > INT32_MAX / 1024 || c->Hk < 1 || c->Hk > 1024)
    return fail(VAFA_ERR_VALUE, "%s: %lld sequences, %lld key heads not supported", what,
                (long long)c->n_seq, (long long)c->Hk);
  if (c->page_size < 1 || c->page_size > INT32_MAX || c->n_pages < 1 || c->n_pages > INT32_MAX)
    return fail(VAFA_ERR_VALUE, "%s: a cache of %lld pages of %lld tokens", what,
                (long long)c->n_pages, (long long)c->page_size);
  if (c->table_width < 0 || c->table_width > INT32_MAX || c->table_stride < 0)
    return fail(VAFA_ERR_VALUE, "%s: page_table with rows of %lld entries, %lld apart", what,
                (long long)c->table_width, (long long)c->table_stride);
  const int64_t strides[] = {c->k_page, c->k_token, c->k_head, c->v_page, c->v_token, c->v_head};
  for (int64_t s : strides)
    if (s < 0 || s % 8 != 0)
      return fail(VAFA_ERR_VALUE, "%s: the cache's strides must be multiples of 8 elements, got %lld",
                  what, (long long)s);
  if ((uintptr_t)c->k % 16 != 0 || (uintptr_t)c->v % 16 != 0)
    return fail(VAFA_ERR_VALUE, "%s: the cache must be 16-byte aligned", what);
  return VAFA_OK;
}

int check_rows(const char *what, const char *name, const void *p, int64_t token, int64_t head) {
  if ((uintptr_t)p % 16 != 0 || token < 0 || token % 8 != 0 || head < 0 || head % 8 != 0)
    return fail(VAFA_ERR_VALUE,
                "%s: %s must be 16-byte aligned with strides that are multiples of 8 elements",
                what, name);
  return VAFA_OK;
}

int check_given(const char *what, std::initializer_list<const void *> ptrs) {
  for (const void *p : ptrs)
    if (p == nullptr) return fail(VAFA_ERR_VALUE, "%s: a required pointer is NULL", what);
  return VAFA_OK;
}

// The cache's pointers, where there are tokens to store or read.
int check_pointers(const char *what, const vafa_paged_cache *c) {
  if (int rc = check_given(what, {c->k, c->v})) return rc;
  if (c->n_seq == 0) return VAFA_OK;
  if (int rc = check_given(what, {c->cache_lens})) return rc;
  return c->table_width > 0 ? check_given(what, {c->page_table}) : VAFA_OK;
}

// The cache and, where it holds codes, their powers of two.
int check_codes(const char *what, const vafa_paged_cache *c, const vafa_row_scales *s) {
  if (int rc = check_cache(what, c)) return rc;
  if (s == nullptr) return VAFA_OK;
  for (int64_t x : {c->k_page, c->k_token, c->k_head, c->v_page, c->v_token, c->v_head})
    if (x % 16 != 0)
      return fail(VAFA_ERR_VALUE, "%s: strides of codes must be multiples of 16, got %lld", what,
                  (long long)x);
  for (int64_t x : {s->k_page, s->k_token, s->k_head, s->v_page, s->v_token, s->v_head})
    if (x < 0 || x > UINT32_MAX)
      return fail(VAFA_ERR_VALUE, "%s: the scales' strides must be below 2^32, got %lld", what,
                  (long long)x);
  // (the kernels' factors: strides in pieces of 16 bytes)
  for (int64_t x : {c->k_page, c->k_token, c->v_page, c->v_token})
    if (x / 16 > UINT32_MAX)
      return fail(VAFA_ERR_VALUE, "%s: strides of codes must be below 2^36, got %lld", what,
                  (long long)x);
  return VAFA_OK;
}

RowScales scales_of(const vafa_row_scales *s) {
  if (s == nullptr) return RowScales{};
  return RowScales{(uint8_t *)s->k, (uint8_t *)s->v, s->k_page, s->k_token, s->k_head,
                   s->v_page, s->v_token, s->v_head};
}

int check_dtype(const char *what, int32_t dtype) {
  if (dtype != VAFA_BF16 && dtype != VAFA_F16)
    return fail(VAFA_ERR_ASSERT, "%s: dtype not supported (float16, bfloat16)", what);
  return VAFA_OK;
}

PageMap map_of(const vafa_paged_cache *c) {
  PageMap m;
  m.table = c->page_table;
  m.row_stride = c->table_stride;
  m.width = (int32_t)c->table_width;
  m.page = (int32_t)c->page_size;
  m.shift = page_shift(c->page_size);
  m.n_pages = (int32_t)c->n_pages;
  return m;
}

int check_launch(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess)
    return fail(VAFA_ERR_RUNTIME, "%s: kernel launch failed: %s", what, hipGetErrorString(e));
  return VAFA_OK;
}

// The decoding attention's launch: the lengths are device data, so chunks and workspace
// go by what the page table could hold.  Workgroups without tiles end at once.
struct DecodePlan {
  int64_t head_blocks = 0, pairs = 0, chunks = 0, bytes = 0, ml_off = 0;
  bool direct = false;
};

// Workgroups resident on the GPU, by registers: 3 (D = 64) or 2 on each of 256 CUs.
int64_t decode_wgs(int64_t D) { return D == 64 ? 768 : 512; }
// Where the page table can hold at most this many tiles a sequence (the lengths are not
// known here), none is divided: a workgroup each, and no launch that joins (4 sequences
// of up to 500 keys: 9.5 -> 6.1 us; 8 of 1000, 8 tiles, the other way round 14 -> 26).
constexpr int64_t kDecodeDirect = 4;

int plan_decode(const vafa_paged_cache *c, int64_t H, int64_t window, DecodePlan *p) {
  if (int rc = check_cache("paged_decode_attn", c)) return rc;
  if (c->D != 64 && c->D != 128 && c->D != 256)
    return fail(VAFA_ERR_ASSERT, "paged_decode_attn: head_dim %lld not supported (64, 128, 256)",
                (long long)c->D);
  if (H < 1 || H % c->Hk != 0 || H > 65536)
    return fail(VAFA_ERR_ASSERT,
                "paged_decode_attn: %lld query heads do not divide among %lld key heads",
                (long long)H, (long long)c->Hk);
  if (window < 0) return fail(VAFA_ERR_VALUE, "paged_decode_attn: window must be positive");
  const int64_t G = H / c->Hk;
  p->head_blocks = (G + kDecodeRows - 1) / kDecodeRows;
  p->pairs = c->Hk * p->head_blocks;
  const int64_t cap = page_capacity(map_of(c));
  const int64_t keys = window > 0 ? std::min(cap, window) : cap;
  const int64_t most = (keys + kDecodeTile - 1) / kDecodeTile;  // tiles of a sequence
  const int64_t tiles = c->n_seq * most;
  if (tiles > INT32_MAX / 2 || !grid_ok((c->n_seq + kXcds) * std::max(H, p->pairs), 256))
    return fail(VAFA_ERR_VALUE, "paged_decode_attn: too many sequences or keys (%lld tiles)",
                (long long)tiles);
  p->direct = most <= kDecodeDirect;
  p->chunks = p->direct ? c->n_seq
                        : std::min(tiles, std::max<int64_t>(1, decode_wgs(c->D) / p->pairs));
  p->chunks = std::max<int64_t>(p->chunks, 1);
  const int64_t rows = p->direct ? 0 : 2 * p->chunks * p->pairs * kDecodeRows;
  p->ml_off = rows * c->D * 4;
  p->bytes = p->ml_off + rows * 2 * 4;
  return VAFA_OK;
}

int check_scores(const char *what, float scale, float softcap) {
  if (!std::isfinite(scale * kLog2e))
    return fail(VAFA_ERR_VALUE, "%s: scale must be finite", what);
  if (!softcap_ok(softcap))
    return fail(VAFA_ERR_VALUE, "%s: softcap must be positive, from %g to %g", what,
                (double)kMinSoftcap, (double)kMaxSoftcap);
  if (softcap > 0.f && !std::isfinite(2.f * kLog2e * scale / softcap))
    return fail(VAFA_ERR_VALUE, "%s: scale / softcap is not finite", what);
  return VAFA_OK;
}

int check_workspace(const void *workspace, int64_t bytes, int64_t needed) {
  if (needed > 0 && (bytes < needed || workspace == nullptr || (uintptr_t)workspace % 16 != 0))
    return fail(VAFA_ERR_WORKSPACE, "workspace of %lld bytes, %lld needed (16-byte aligned)",
                (long long)bytes, (long long)needed);
  return VAFA_OK;
}

// The launch of several new tokens per sequence: lengths and cu are device data, so chunks and
// workspace go by the rows and by what the page table could hold.
struct ChunkPlan {
  int lg = 0, lt = 0;
  int64_t rows = 0, chunks = 0, bytes = 0, lse_off = 0, cut_off = 0;
  bool direct = false;
};

// Where no tile can walk more than this many units, none is divided: no launch that joins (D = 128,
// 8 sequences, 4 and 128 new tokens: of 4 units 14 and 18 us, divided 18 and 33;
// of 8 18 and 26, 21 and 40; of 16 27 and 39, 27 and 49, but of one sequence 27 and 36, 19 and 30).
constexpr int64_t kChunkDirect = 8;

int plan_chunk(const vafa_paged_cache *c, int64_t T, int64_t H, int64_t window, ChunkPlan *p) {
  const char *what = "paged_chunk_attn";
  if (int rc = check_cache(what, c)) return rc;
  if (c->D != 64 && c->D != 128 && c->D != 256)
    return fail(VAFA_ERR_ASSERT, "%s: head_dim %lld not supported (64, 128, 256)", what,
                (long long)c->D);
  if (H < 1 || H % c->Hk != 0 || H > 4096)
    return fail(VAFA_ERR_ASSERT, "%s: %lld query heads do not divide among %lld key heads", what,
                (long long)H, (long long)c->Hk);
  if (T < 0 || T > kMaskedMaxTokens)
    return fail(VAFA_ERR_VALUE, "%s: %lld tokens are too many for a call", what, (long long)T);
  if (window < 0) return fail(VAFA_ERR_VALUE, "%s: window must be positive", what);
  const int64_t G = H / c->Hk;
  while (p->lg < 5 && G % (int64_t{2} << p->lg) == 0) ++p->lg;
  p->rows = c->D <= 128 ? 256 : 128;
  p->lt = (c->D <= 128 ? 8 : 7) - p->lg;
  const int64_t sets = H >> p->lg, tw = int64_t{1} << p->lt;
  const int64_t cap = page_capacity(map_of(c));
  const int64_t keys = window > 0 && window < cap ? std::min(cap, window + tw + kChunkKeys) : cap;
  const int64_t most = std::max<int64_t>(1, (keys + kChunkKeys - 1) / kChunkKeys);
  // (a sequence of nq tokens has at most nq / tw + 1 tiles)
  const int64_t tiles = std::max<int64_t>(1, T / tw + std::min(c->n_seq, T));
  const int64_t slots = 256;  // workgroups that the GPU holds: one on a CU
  p->direct = most <= kChunkDirect;
  if (p->direct)
    p->chunks = std::min<int64_t>(tiles, std::max<int64_t>(slots, 65536 / sets));
  else
    p->chunks = std::max<int64_t>(1, std::min(slots / sets, tiles * most));
  const int64_t rows = p->direct ? 0 : 2 * p->chunks * sets * p->rows;
  p->lse_off = rows * c->D * 4;
  p->cut_off = p->lse_off + rows * 4;  // (a multiple of 16: a tile has 128 rows or more)
  p->bytes = p->cut_off + (p->direct ? 0 : p->chunks * sets * (int64_t)sizeof(ChunkCut));
  return VAFA_OK;
}

// The operands of an append, which both kinds of it take.
int append_args(const char *what, const vafa_paged_cache *c, const void *k, int64_t k_token,
                int64_t k_head, const void *v, int64_t v_token, int64_t v_head, int64_t T,
                const int32_t *cu, const void *q, int64_t q_token, int64_t q_head, int64_t H,
                void *q_out, const float *inv_freq, int64_t rot, int32_t interleaved,
                AppendArgs *out) {
  if (rot < 0 || rot % 2 != 0 || rot > c->D)
    return fail(VAFA_ERR_VALUE, "%s: %lld rotated features of %lld", what, (long long)rot,
                (long long)c->D);
  if (H < 0 || H > 65536) return fail(VAFA_ERR_VALUE, "%s: %lld query heads", what, (long long)H);
  if (T < 0 || T > INT32_MAX || (cu == nullptr && T != c->n_seq))
    return fail(VAFA_ERR_VALUE, "%s: %lld tokens of %lld sequences", what, (long long)T,
                (long long)c->n_seq);
  if (int rc = check_rows(what, "k", k, k_token, k_head)) return rc;
  if (int rc = check_rows(what, "v", v, v_token, v_head)) return rc;
  if (H > 0) {
    if (int rc = check_rows(what, "q", q, q_token, q_head)) return rc;
    if (int rc = check_rows(what, "q_out", q_out, 0, 0)) return rc;
  }
  if (!grid_ok(std::max(T, T * ((H + 2 * c->Hk) * (c->D / 16)) / 256 + 1), 256))
    return fail(VAFA_ERR_VALUE, "%s: %lld tokens are too many for a call", what, (long long)T);
  if (T == 0) return VAFA_OK;
  if (int rc = check_pointers(what, c)) return rc;
  if (int rc = check_given(what, {k, v})) return rc;
  if (H > 0)
    if (int rc = check_given(what, {q, q_out})) return rc;
  if (rot > 0)
    if (int rc = check_given(what, {inv_freq})) return rc;
  AppendArgs &a = *out;
  a.q = q; a.k = k; a.v = v; a.q_out = q_out; a.kc = c->k; a.vc = c->v;
  a.cu = cu; a.lens = c->cache_lens; a.inv_freq = inv_freq;
  a.map = map_of(c);
  a.q_token = q_token; a.q_head = q_head; a.k_token = k_token; a.k_head = k_head;
  a.v_token = v_token; a.v_head = v_head;
  a.k_page = c->k_page; a.kc_token = c->k_token; a.kc_head = c->k_head;
  a.v_page = c->v_page; a.vc_token = c->v_token; a.vc_head = c->v_head;
  a.T = T; a.n_seq = (int)c->n_seq; a.H = (int)H; a.Hk = (int)c->Hk; a.D = (int)c->D;
  a.rot = (int)rot; a.interleaved = interleaved != 0;
  return VAFA_OK;
}

}  // namespace

// What norms and rotations of whole rows take, with or without a cache.
int check_head_rows(const char *what, int64_t D, int64_t rot, float eps, float rot_scale) {
  if (D != 64 && D != 128 && D != 256)
    return fail(VAFA_ERR_ASSERT, "%s: head_dim %lld not supported (64, 128, 256)", what,
                (long long)D);
  if (rot < 0 || rot % 16 != 0 || rot > D)
    return fail(VAFA_ERR_VALUE, "%s: %lld rotated features of %lld (multiples of 16)", what,
                (long long)rot, (long long)D);
  if (!(eps >= 0.f) || !std::isfinite(eps))
    return fail(VAFA_ERR_VALUE, "%s: eps must be finite and not negative", what);
  if (!std::isfinite(rot_scale))
    return fail(VAFA_ERR_VALUE, "%s: rot_scale must be finite", what);
  return VAFA_OK;
}

}  // namespace vafa

using namespace vafa;

extern "C" {

int vafa_paged_append(const vafa_paged_cache *c, const void *k, int64_t k_token, int64_t k_head,
                      const void *v, int64_t v_token, int64_t v_head, int64_t T, const int32_t *cu,
                      const void *q, int64_t q_token, int64_t q_head, int64_t H, void *q_out,
                      const float *inv_freq, int64_t rot, int32_t interleaved, int32_t dtype,
                      void *stream) {
  const char *what = "paged_kv_append";
  if (int rc = check_dtype(what, dtype)) return rc;
  if (int rc = check_cache(what, c)) return rc;
  if (c->D < 8 || c->D > 1024 || c->D % 8 != 0)
    return fail(VAFA_ERR_ASSERT, "%s: head_dim %lld not supported (multiples of 8 up to 1024)", what,
                (long long)c->D);
  AppendArgs a{};
  if (int rc = append_args(what, c, k, k_token, k_head, v, v_token, v_head, T, cu, q, q_token,
                           q_head, H, q_out, inv_freq, rot, interleaved, &a))
    return rc;
  if (T == 0) return VAFA_OK;
  if (dtype == VAFA_BF16)
    launch_paged_append<bf16>(a, (hipStream_t)stream);
  else
    launch_paged_append<f16>(a, (hipStream_t)stream);
  return check_launch(what);
}

int vafa_paged_store(const vafa_paged_cache *c, const vafa_row_scales *scales, const void *k,
                     int64_t k_token, int64_t k_head, const void *v, int64_t v_token,
                     int64_t v_head, int64_t T, const int32_t *cu, const void *q, int64_t q_token,
                     int64_t q_head, int64_t H, void *q_out, const float *inv_freq, int64_t rot,
                     int32_t interleaved, float rot_scale, const void *q_weight,
                     const void *k_weight, int32_t weights_f32, float eps, int32_t dtype,
                     void *stream) {
  const char *what = "paged_kv_append";
  if (int rc = check_dtype(what, dtype)) return rc;
  if (int rc = check_codes(what, c, scales)) return rc;
  if (int rc = check_head_rows(what, c->D, rot, eps, rot_scale)) return rc;
  for (int64_t x : {q_token, q_head, k_token, k_head, v_token, v_head})  // (the kernel's factors)
    if (x > UINT32_MAX)
      return fail(VAFA_ERR_VALUE, "%s: strides of rows must be below 2^32, got %lld", what,
                  (long long)x);
  HeadRowsArgs s{};
  if (int rc = append_args(what, c, k, k_token, k_head, v, v_token, v_head, T, cu, q, q_token,
                           q_head, H, q_out, inv_freq, rot, interleaved, &s.a))
    return rc;
  if (T == 0) return VAFA_OK;
  if (scales != nullptr)
    if (int rc = check_given(what, {scales->k, scales->v})) return rc;
  s.scales = scales_of(scales);
  s.q_weight = q_weight; s.k_weight = k_weight; s.weights_f32 = weights_f32 != 0;
  s.eps = eps; s.rot_scale = rot_scale;
  if (dtype == VAFA_BF16)
    launch_head_rows<bf16>(s, (hipStream_t)stream);
  else
    launch_head_rows<f16>(s, (hipStream_t)stream);
  return check_launch(what);
}

int vafa_paged_gather(const vafa_paged_cache *c, const vafa_row_scales *scales, const int32_t *cu,
                      const int32_t *starts, int64_t T, void *k, void *v, int32_t dtype,
                      void *stream) {
  const char *what = "paged_kv_gather";
  if (int rc = check_dtype(what, dtype)) return rc;
  if (int rc = check_codes(what, c, scales)) return rc;
  if (c->D < 16 || c->D > 1024 || c->D % 16 != 0)
    return fail(VAFA_ERR_ASSERT, "%s: head_dim %lld not supported (multiples of 16 up to 1024)",
                what, (long long)c->D);
  if (T < 0 || T > INT32_MAX || !grid_ok(T * (2 * c->Hk * (c->D / 16)) / 256 + 1, 256))
    return fail(VAFA_ERR_VALUE, "%s: %lld rows are too many for a call", what, (long long)T);
  if (int rc = check_rows(what, "k", k, 0, 0)) return rc;
  if (int rc = check_rows(what, "v", v, 0, 0)) return rc;
  if (T == 0) return VAFA_OK;
  if (int rc = check_given(what, {c->k, c->v, cu, k, v})) return rc;
  if (c->n_seq > 0 && c->table_width > 0)
    if (int rc = check_given(what, {c->page_table})) return rc;
  if (scales != nullptr)
    if (int rc = check_given(what, {scales->k, scales->v})) return rc;
  GatherArgs a{};
  a.kc = c->k; a.vc = c->v; a.scales = scales_of(scales); a.k = k; a.v = v;
  a.cu = cu; a.starts = starts; a.map = map_of(c);
  a.k_page = c->k_page; a.kc_token = c->k_token; a.kc_head = c->k_head;
  a.v_page = c->v_page; a.vc_token = c->v_token; a.vc_head = c->v_head;
  a.T = T; a.n_seq = (int)c->n_seq; a.Hk = (int)c->Hk; a.D = (int)c->D;
  if (dtype == VAFA_BF16)
    launch_paged_gather<bf16>(a, (hipStream_t)stream);
  else
    launch_paged_gather<f16>(a, (hipStream_t)stream);
  return check_launch(what);
}

int64_t vafa_paged_decode_workspace(const vafa_paged_cache *c, int64_t H, int64_t window) {
  DecodePlan p;
  return plan_decode(c, H, window, &p) ? -1 : p.bytes;
}

int vafa_paged_decode(const vafa_paged_cache *c, const void *q, int64_t q_token, int64_t q_head,
                      int64_t H, void *out, float scale, float softcap, int64_t window,
                      const float *slopes, int32_t dtype, void *workspace, int64_t workspace_bytes,
                      void *stream) {
  return vafa_paged_decode_codes(c, nullptr, q, q_token, q_head, H, out, scale, softcap, window,
                                 slopes, dtype, workspace, workspace_bytes, stream);
}

int vafa_paged_decode_codes(const vafa_paged_cache *c, const vafa_row_scales *scales,
                            const void *q, int64_t q_token, int64_t q_head, int64_t H, void *out,
                            float scale, float softcap, int64_t window, const float *slopes,
                            int32_t dtype, void *workspace, int64_t workspace_bytes,
                            void *stream) {
  const char *what = "paged_decode_attn";
  if (int rc = check_dtype(what, dtype)) return rc;
  DecodePlan p;
  if (int rc = plan_decode(c, H, window, &p)) return rc;
  if (int rc = check_codes(what, c, scales)) return rc;
  if (int rc = check_scores(what, scale, softcap)) return rc;
  if (int rc = check_rows(what, "q", q, q_token, q_head)) return rc;
  if (int rc = check_rows(what, "out", out, 0, 0)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes)) return rc;
  if (c->n_seq == 0) return VAFA_OK;
  if (int rc = check_pointers(what, c)) return rc;
  if (int rc = check_given(what, {q, out})) return rc;
  if (scales != nullptr)
    if (int rc = check_given(what, {scales->k, scales->v})) return rc;
  DecodeArgs a{};
  a.scales = scales_of(scales);
  a.q = q; a.kc = c->k; a.vc = c->v; a.out = out; a.lens = c->cache_lens; a.slopes = slopes;
  a.part_o = (float *)workspace;
  a.part_ml = (float *)((char *)workspace + p.ml_off);
  a.map = map_of(c);
  a.q_token = q_token; a.q_head = q_head;
  a.k_page = c->k_page; a.kc_token = c->k_token; a.kc_head = c->k_head;
  a.v_page = c->v_page; a.vc_token = c->v_token; a.vc_head = c->v_head;
  a.capacity = page_capacity(a.map);
  a.n_seq = (int)c->n_seq; a.H = (int)H; a.G = (int)(H / c->Hk); a.pairs = (int)p.pairs;
  a.head_blocks = (int)p.head_blocks; a.chunks = (int)p.chunks; a.direct = p.direct;
  a.window = (int)std::min<int64_t>(window, INT32_MAX);
  // capped: tanh(x) = 1 - 2 / (1 + 2^(2 x log2 e)), x = scale q.k / cap
  a.c = softcap > 0.f ? 2.f * kLog2e * scale / softcap : scale * kLog2e;
  a.cap2 = softcap * kLog2e;
  if (dtype == VAFA_BF16)
    launch_paged_decode<bf16>(a, (int)c->D, (hipStream_t)stream);
  else
    launch_paged_decode<f16>(a, (int)c->D, (hipStream_t)stream);
  return check_launch(what);
}

int64_t vafa_paged_chunk_workspace(const vafa_paged_cache *c, int64_t T, int64_t H,
                                   int64_t window) {
  ChunkPlan p;
  return plan_chunk(c, T, H, window, &p) ? -1 : p.bytes;
}

int vafa_paged_chunk(const vafa_paged_cache *c, const vafa_row_scales *scales, const void *q,
                     int64_t q_token, int64_t q_head, int64_t T, int64_t H, const int32_t *cu,
                     void *out, float scale, float softcap, int64_t window, const float *slopes,
                     int32_t dtype, void *workspace, int64_t workspace_bytes, void *stream) {
  const char *what = "paged_chunk_attn";
  if (int rc = check_dtype(what, dtype)) return rc;
  ChunkPlan p;
  if (int rc = plan_chunk(c, T, H, window, &p)) return rc;
  if (int rc = check_codes(what, c, scales)) return rc;
  // (codes: as far as check_codes lets them)
  const int64_t piece = scales != nullptr ? 16 : 8;
  for (int64_t x : {c->k_page, c->k_token, c->v_page, c->v_token})
    if (x / piece > UINT32_MAX)
      return fail(VAFA_ERR_VALUE, "%s: the cache's strides must be below 2^35, got %lld", what,
                  (long long)x);
  if (int rc = check_scores(what, scale, softcap)) return rc;
  if (int rc = check_rows(what, "q", q, q_token, q_head)) return rc;
  if (int rc = check_rows(what, "out", out, 0, 0)) return rc;
  if (int rc = check_workspace(workspace, workspace_bytes, p.bytes)) return rc;
  if (T == 0) return VAFA_OK;
  if (int rc = check_pointers(what, c)) return rc;
  if (int rc = check_given(what, {q, out, cu})) return rc;
  if (scales != nullptr)
    if (int rc = check_given(what, {scales->k, scales->v})) return rc;
  ChunkArgs a{};
  a.q = q; a.kc = c->k; a.vc = c->v; a.out = out; a.cu = cu; a.lens = c->cache_lens;
  a.slopes = slopes; a.part_o = (float *)workspace;
  a.part_lse = (float *)((char *)workspace + p.lse_off);
  a.cuts = (ChunkCut *)((char *)workspace + p.cut_off);
  a.map = map_of(c); a.q_token = q_token; a.q_head = q_head;
  a.kc_head = c->k_head; a.vc_head = c->v_head;
  a.k_page = (uint32_t)(c->k_page / piece); a.kc_token = (uint32_t)(c->k_token / piece);
  a.v_page = (uint32_t)(c->v_page / piece); a.vc_token = (uint32_t)(c->v_token / piece);
  a.scales = scales_of(scales); a.T = T;
  // (so that a key behind the last unit still has a number)
  a.capacity = std::min<int64_t>(page_capacity(a.map), INT32_MAX - 4096);
  a.n_seq = (int)c->n_seq; a.H = (int)H; a.Hk = (int)c->Hk;
  a.window = (int)std::min<int64_t>(window, kChunkNoWindow);
  a.lg = p.lg; a.lt = p.lt; a.chunks = (int)p.chunks; a.direct = p.direct;
  // (as for one token: tanh(x) = 1 - 2 / (1 + 2^(2 x log2 e)), x = scale q.k / cap)
  a.c = softcap > 0.f ? 2.f * kLog2e * scale / softcap : scale * kLog2e;
  a.cap2 = softcap * kLog2e;
  const hipStream_t st = (hipStream_t)stream;
  const bool bf = dtype == VAFA_BF16;
  if (c->D == 64)
    bf ? launch_paged_chunk<bf16, 64>(a, st) : launch_paged_chunk<f16, 64>(a, st);
  else if (c->D == 128)
    bf ? launch_paged_chunk<bf16, 128>(a, st) : launch_paged_chunk<f16, 128>(a, st);
  else
    bf ? launch_paged_chunk<bf16, 256>(a, st) : launch_paged_chunk<f16, 256>(a, st);
  return check_launch(what);
}

}  // extern "C"
