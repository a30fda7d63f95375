// Allocation and launch of one operator pass per call, for the Python layer:
// each function allocates outputs and workspace with torch's allocator, takes
// the current stream of the operands' device and calls one entry point of
// libvafa.so (include/vafa.h).  The plan cache is in Python, and so are autograd and the
// argument checks of packed_varlen_attn and packed_target_attn; packed_masked_attn and the
// paged cache, whose small calls have less time for them, have theirs here.  With tensor
// factories, ctypes conversions and stream lookups
// there too, host time held every small call: us a call with cu_seqlens seen before
// (the plan cached), before -> now, 4 short sequences forward 31 -> 17 (host
// cu_seqlens), forward + backward 150 -> 93; 16 absorb samples forward 34 -> 25,
// forward + backward 220 -> 171.  With new lengths in every call planning adds 15 to
// 50 us: 4 sequences 73 -> 62, 16 absorb samples 84 -> 85.
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <dlfcn.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/extension.h>

#include <initializer_list>
#include <mutex>
#include <string>
#include <tuple>
#include <unordered_map>
#include <vector>

#include "../../include/vafa.h"

namespace {

using at::Tensor;

// Entry points of the library the Python layer loaded.
struct Api {
#define VAFA_FN(name) decltype(&::vafa_##name) name = nullptr;
#define VAFA_FNS(X)                                                                       \
  X(last_error) X(varlen_fwd_workspace) X(varlen_fwd) X(varlen_bwd_workspace)             \
  X(varlen_bwd) X(absorb_fwd_workspace) X(absorb_fwd) X(absorb_bwd_workspace)             \
  X(absorb_bwd) X(absorb_fwd_full_workspace) X(absorb_fwd_full) X(absorb_bwd_full)        \
  X(absorb_bwd_full_workspace)                                                            \
  X(absorb_project_workspace) X(absorb_project_fwd) X(absorb_project_bwd)                 \
  X(absorb_project_f32_workspace) X(absorb_project_f32_fwd) X(absorb_project_f32_bwd)      \
  X(paged_append) X(paged_decode_workspace) X(paged_decode) X(masked_fwd_workspace)        \
  X(masked_fwd) X(masked_bwd_workspace) X(masked_bwd)
  VAFA_FNS(VAFA_FN)
#undef VAFA_FN
} api;

void bind_library(const std::string &path) {
  void *h = dlopen(path.c_str(), RTLD_NOW | RTLD_LOCAL);
  TORCH_CHECK(h != nullptr, "cannot load ", path, ": ", dlerror());
#define VAFA_SYM(name)                                                                    \
  api.name = reinterpret_cast<decltype(api.name)>(dlsym(h, "vafa_" #name));               \
  TORCH_CHECK(api.name != nullptr, path, " lacks vafa_" #name);
  VAFA_FNS(VAFA_SYM)
#undef VAFA_SYM
}

struct AssertionFailed : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int rc) {
  if (rc == VAFA_OK) return;
  const std::string msg = api.last_error();
  if (rc == VAFA_ERR_VALUE) throw py::value_error(msg);
  if (rc == VAFA_ERR_ASSERT) throw AssertionFailed(msg);
  throw std::runtime_error("vafa error " + std::to_string(rc) + ": " + msg);
}

int32_t dtype_of(const Tensor &t) {
  switch (t.scalar_type()) {
    case at::kFloat: return VAFA_F32;
    case at::kHalf: return VAFA_F16;
    case at::kBFloat16: return VAFA_BF16;
    default: throw AssertionFailed("dtype not supported (float32, float16, bfloat16)");
  }
}

// One call's device, stream and workspace.
struct Call {
  c10::DeviceGuard guard;
  at::TensorOptions opt;
  void *stream;
  Tensor ws;
  explicit Call(const Tensor &t)
      : guard(t.device()), opt(t.options()),
        stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream()) {}
  Tensor empty(at::IntArrayRef shape) const { return at::empty(shape, opt); }
  Tensor empty_f32(at::IntArrayRef shape) const { return at::empty(shape, opt.dtype(at::kFloat)); }
  Tensor like(const Tensor &t) const { return at::empty(t.sizes(), opt); }
  // a workspace of n bytes (none for 0); a negative size is the query's error
  void *workspace(int64_t n) {
    if (n < 0) check(VAFA_ERR_VALUE);
    if (n == 0) return nullptr;
    ws = at::empty({n}, opt.dtype(at::kByte));
    return ws.data_ptr();
  }
  int64_t ws_bytes() const { return ws.defined() ? ws.numel() : 0; }
};

// A device plan: its items and info struct.
struct Plan {
  Tensor items;
  vafa_plan_info info;
  Plan(Tensor t, const std::string &bytes) : items(std::move(t)) {
    TORCH_CHECK(bytes.size() == sizeof(info), "plan info of ", bytes.size(), " bytes");
    std::memcpy(&info, bytes.data(), sizeof(info));
  }
  // The items as a launch of call c reads them.  A launch that a graph records reads them
  // again in every replay, without a call that could look the plan up: such a plan stays for
  // the process's life (32 bytes an item), whatever the cache and the autograd nodes drop.
  const int32_t *dev(const Call &c) const {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    const bool known =
        hipStreamIsCapturing(static_cast<hipStream_t>(c.stream), &status) == hipSuccess;
    if (!known) (void)hipGetLastError();  // not this call's error
    if (!known || status != hipStreamCaptureStatusNone) {
      static std::mutex lock;
      // (never destroyed: at exit the GPU may be gone before it)
      static auto *kept = new std::unordered_map<const void *, Tensor>;
      const std::lock_guard<std::mutex> hold(lock);
      kept->emplace(items.unsafeGetTensorImpl(), items);
    }
    return items.data_ptr<int32_t>();
  }
};

void *ptr(const Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }
const float *f32(const Tensor &t) { return static_cast<const float *>(ptr(t)); }
float *f32w(const Tensor &t) { return static_cast<float *>(ptr(t)); }

// An upstream gradient as the kernels read it: the operands' dtype,
// contiguous, 16-byte aligned.
Tensor grad_in(Tensor g, const Tensor &like) {
  g = g.contiguous();
  if (g.scalar_type() != like.scalar_type()) g = g.to(like.scalar_type());
  if (reinterpret_cast<uintptr_t>(g.data_ptr()) % 16 != 0) g = g.clone();
  return g;
}

std::tuple<Tensor, Tensor> varlen_fwd(const Tensor &q, const Tensor &k, const Tensor &v,
                                      const Plan &p, double scale) {
  Call c(q);
  const int64_t D = q.size(2);
  Tensor o = c.like(q), lse = c.empty_f32({q.size(0), q.size(1)});
  void *ws = c.workspace(api.varlen_fwd_workspace(&p.info, D));
  check(api.varlen_fwd(ptr(q), ptr(k), ptr(v), ptr(o), f32w(lse), p.dev(c), &p.info, D, dtype_of(q),
                       (float)scale, ws, c.ws_bytes(), c.stream));
  return {o, lse};
}

std::tuple<Tensor, Tensor, Tensor> varlen_bwd(const Tensor &q, const Tensor &k, const Tensor &v,
                                              const Tensor &o, const Tensor &lse, const Tensor &g,
                                              const Plan &p, double scale) {
  Call c(q);
  const int64_t D = q.size(2);
  const Tensor dout = grad_in(g, q);
  Tensor dq = c.like(q), dk = c.like(k), dv = c.like(v);
  void *ws = c.workspace(api.varlen_bwd_workspace(&p.info, D));
  check(api.varlen_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(dout), f32(lse), ptr(dq), ptr(dk),
                       ptr(dv), p.dev(c), &p.info, D, dtype_of(q), (float)scale, ws, c.ws_bytes(),
                       c.stream));
  return {dq, dk, dv};
}

std::tuple<Tensor, Tensor> absorb_fwd(const Tensor &u, const Tensor &X, const Tensor &W_V,
                                      const Plan &p, double scale) {
  Call c(u);
  const int64_t T_q = u.size(0), H = u.size(1), F = u.size(2), DH = W_V.size(2);
  Tensor O = c.empty({T_q, H, DH}), lse = c.empty_f32({T_q, H});
  void *ws = c.workspace(api.absorb_fwd_workspace(&p.info, F, DH));
  check(api.absorb_fwd(ptr(u), ptr(X), ptr(W_V), ptr(O), f32w(lse), p.dev(c), &p.info, F, DH,
                       dtype_of(u), (float)scale, ws, c.ws_bytes(), c.stream));
  return {O, lse};
}

std::tuple<Tensor, Tensor, Tensor> absorb_bwd(const Tensor &u, const Tensor &X, const Tensor &W_V,
                                              const Tensor &O, const Tensor &lse, const Tensor &g,
                                              const Plan &p, double scale) {
  Call c(u);
  const int64_t F = u.size(2), DH = W_V.size(2);
  const Tensor dO = grad_in(g, u);
  Tensor du = c.like(u), dX = c.like(X), dW = c.like(W_V);
  void *ws = c.workspace(api.absorb_bwd_workspace(&p.info, F, DH));
  check(api.absorb_bwd(ptr(u), ptr(X), ptr(W_V), ptr(O), ptr(dO), f32(lse), ptr(du), ptr(dX),
                       ptr(dW), p.dev(c), &p.info, F, DH, dtype_of(u), (float)scale, ws,
                       c.ws_bytes(), c.stream));
  return {du, dX, dW};
}

// The whole 16-bit forward: (q_proj, O, lse).
std::tuple<Tensor, Tensor, Tensor> absorb_full_fwd(const Tensor &q_raw, const Tensor &X,
                                                   const Tensor &W_Q, const Tensor &W_K,
                                                   const Tensor &W_V, const Plan &p,
                                                   double scale) {
  Call c(q_raw);
  const int64_t T_q = q_raw.size(0), DQ = q_raw.size(1), F = X.size(1), H = W_Q.size(1),
                DH = W_Q.size(2);
  Tensor q_proj = c.empty({T_q, H * DH}), O = c.empty({T_q, H, DH}), lse = c.empty_f32({T_q, H});
  void *ws = c.workspace(api.absorb_fwd_full_workspace(&p.info, DQ, F, DH));
  check(api.absorb_fwd_full(ptr(q_raw), ptr(X), ptr(W_Q), ptr(W_K), ptr(W_V), ptr(q_proj), ptr(O),
                            f32w(lse), T_q, p.dev(c), &p.info, DQ, F, DH, dtype_of(q_raw),
                            (float)scale, ws, c.ws_bytes(), c.stream));
  return {q_proj, O, lse};
}

// Projections in 16 bits or fp32: (q_proj, u).
std::tuple<Tensor, Tensor> project_fwd(const Tensor &q_raw, const Tensor &W_Q, const Tensor &W_K) {
  Call c(q_raw);
  const int64_t T_q = q_raw.size(0), DQ = q_raw.size(1), H = W_Q.size(1), DH = W_Q.size(2),
                F = W_K.size(0);
  Tensor q_proj = c.empty({T_q, H * DH}), u = c.empty({T_q, H, F});
  if (q_raw.scalar_type() == at::kFloat) {
    check(api.absorb_project_f32_fwd(f32(q_raw), f32(W_Q), f32(W_K), f32w(q_proj), f32w(u), T_q, H,
                                     DQ, F, DH, c.stream));
  } else {
    void *ws = c.workspace(api.absorb_project_workspace(T_q, H, DQ, F, DH, 0));
    check(api.absorb_project_fwd(ptr(q_raw), ptr(W_Q), ptr(W_K), ptr(q_proj), ptr(u), T_q, H, DQ,
                                 F, DH, dtype_of(q_raw), ws, c.ws_bytes(), c.stream));
  }
  return {q_proj, u};
}

// (dq_raw, dW_Q, dW_K), None where not asked for.
using Grads3 = std::tuple<std::optional<Tensor>, std::optional<Tensor>, std::optional<Tensor>>;
Grads3 project_bwd(const Tensor &q_raw, const Tensor &W_Q, const Tensor &W_K, const Tensor &q_proj,
                   const Tensor &g, bool need_q, bool need_wq, bool need_wk) {
  Call c(q_raw);
  const int64_t T_q = q_raw.size(0), DQ = q_raw.size(1), H = W_Q.size(1), DH = W_Q.size(2),
                F = W_K.size(0);
  const Tensor du = grad_in(g, q_raw);
  Tensor dq, dwq, dwk;
  if (need_q) dq = c.like(q_raw);
  if (need_wq) dwq = c.like(W_Q);
  if (need_wk) dwk = c.like(W_K);
  if (q_raw.scalar_type() == at::kFloat) {
    void *ws = c.workspace(api.absorb_project_f32_workspace(T_q, H, DQ, F, DH));
    check(api.absorb_project_f32_bwd(f32(q_raw), f32(W_Q), f32(W_K), f32(q_proj), f32(du),
                                     f32w(dq), f32w(dwq), f32w(dwk), T_q, H, DQ, F, DH, ws,
                                     c.ws_bytes(), c.stream));
  } else {
    void *ws = c.workspace(api.absorb_project_workspace(T_q, H, DQ, F, DH, 1));
    check(api.absorb_project_bwd(ptr(q_raw), ptr(W_Q), ptr(W_K), ptr(q_proj), ptr(du), ptr(dq),
                                 ptr(dwq), ptr(dwk), T_q, H, DQ, F, DH, dtype_of(q_raw), ws,
                                 c.ws_bytes(), c.stream));
  }
  auto opt = [](const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
  return {opt(dq), opt(dwq), opt(dwk)};
}

// Backward of the whole 16-bit op: (dq_raw, dX, dW_Q, dW_K, dW_V).
std::tuple<std::optional<Tensor>, Tensor, std::optional<Tensor>, std::optional<Tensor>, Tensor>
absorb_full_bwd(const Tensor &q_raw, const Tensor &W_Q, const Tensor &W_K, const Tensor &q_proj,
                const Tensor &X, const Tensor &W_V, const Tensor &O, const Tensor &lse,
                const Tensor &g, const Plan &p, double scale, bool need_q, bool need_wq,
                bool need_wk) {
  Call c(q_raw);
  const int64_t T_q = q_raw.size(0), DQ = q_raw.size(1), F = X.size(1), DH = W_Q.size(2);
  const Tensor dO = grad_in(g, q_raw);
  Tensor dX = c.like(X), dW_V = c.like(W_V), dq, dwq, dwk;
  if (need_q) dq = c.like(q_raw);
  if (need_wq) dwq = c.like(W_Q);
  if (need_wk) dwk = c.like(W_K);
  void *ws = c.workspace(api.absorb_bwd_full_workspace(&p.info, T_q, DQ, F, DH));
  check(api.absorb_bwd_full(ptr(q_raw), ptr(X), ptr(W_Q), ptr(W_K), ptr(W_V), ptr(q_proj), ptr(O),
                            ptr(dO), f32(lse), ptr(dq), ptr(dX), ptr(dwq), ptr(dwk), ptr(dW_V),
                            T_q, p.dev(c), &p.info, DQ, F, DH, dtype_of(q_raw), (float)scale, ws,
                            c.ws_bytes(), c.stream));
  auto opt = [](const Tensor &t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; };
  return {opt(dq), dX, opt(dwq), opt(dwk), dW_V};
}

// ---- paged cache: argument checks here, where a call of a few us can afford them ----

void need(bool ok, const char *what, const char *msg) {
  if (!ok) throw AssertionFailed(std::string(what) + ": " + msg);
}

// The stride of a dimension as the kernels use it: one of size 1 is never stepped over.
int64_t stride_of(const Tensor &t, int64_t dim) { return t.size(dim) > 1 ? t.stride(dim) : 0; }

// Neighbours in memory along a dimension, which the kernels read as such: an expanded
// dimension (stride 0) holds one element where they would read size of them.
bool dense(const Tensor &t, int64_t dim) { return t.size(dim) <= 1 || t.stride(dim) == 1; }

bool rows_ok(const Tensor &t) {
  bool ok = dense(t, t.dim() - 1) && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0;
  for (int64_t d = 0; d + 1 < t.dim(); ++d) ok = ok && stride_of(t, d) % 8 == 0;
  return ok;
}

// [T, H, D] as the kernels read it (any token and head stride of whole 16 bytes);
// other layouts are copied.
Tensor rows_in(const Tensor &t) {
  return rows_ok(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

// Forward-mode derivatives and traces follow torch's own operations, of which a call here
// shows them none but the allocation of its output: the tangent would be dropped, and the
// trace would return memory that nothing wrote.
void direct_only(const char *what, std::initializer_list<Tensor> ts) {
  if (torch::jit::tracer::isTracing())
    throw py::value_error(std::string(what) + " cannot be traced by torch.jit");
  for (const Tensor &t : ts)
    if (t.defined() && t._fw_grad(0).defined())
      throw py::value_error(std::string(what) +
                            " has no forward-mode derivative: unpack its dual tensors first");
}

void no_grad_only(const char *what, std::initializer_list<Tensor> ts) {
  direct_only(what, ts);
  if (!at::GradMode::is_enabled()) return;
  for (const Tensor &t : ts)
    if (t.defined() && t.requires_grad())
      throw py::value_error(std::string(what) +
                            " has no backward: call it under torch.no_grad() or detach its inputs");
}

// (last of the checks: the others refuse the same calls without a GPU)
void on_gpu(const char *what, const Tensor &t) {
  need(t.is_cuda(), what, "requires GPU tensors on one device");
}

vafa_paged_cache cache_of(const char *what, const Tensor &kc, const Tensor &vc,
                          const Tensor &table, const Tensor &lens) {
  need(kc.dim() == 4 && vc.sizes() == kc.sizes(), what,
       "k_cache and v_cache must be [n_pages, page_size, H_k, D] alike");
  const auto dt = kc.scalar_type();
  need(dt == at::kHalf || dt == at::kBFloat16, what, "dtype not supported (float16, bfloat16)");
  need(vc.scalar_type() == dt, what, "k_cache and v_cache must share dtype");
  need(table.dim() == 2 && lens.dim() == 1 && table.size(0) == lens.size(0), what,
       "page_table must be [n_seq, pages] and cache_lens [n_seq]");
  need(table.scalar_type() == at::kInt && lens.scalar_type() == at::kInt, what,
       "page_table and cache_lens must be int32");
  if (!dense(table, 1) || !dense(lens, 0))
    throw py::value_error(std::string(what) +
                          ": the rows of page_table and cache_lens must be contiguous");
  if (!rows_ok(kc) || !rows_ok(vc))
    throw py::value_error(std::string(what) +
                          ": the caches must be 16-byte aligned, features contiguous and other "
                          "strides multiples of 8 elements");
  for (const Tensor *t : {&kc, &vc})
    for (int64_t d = 0; d < 4; ++d)
      if (t->size(d) > 1 && t->stride(d) == 0)
        throw py::value_error(std::string(what) + ": the caches must not be expanded views");
  need(vc.device() == kc.device() && table.device() == kc.device() &&
           lens.device() == kc.device(),
       what, "requires GPU tensors on one device");
  vafa_paged_cache c{};
  c.k = kc.data_ptr(); c.v = vc.data_ptr();
  c.n_pages = kc.size(0); c.page_size = kc.size(1); c.Hk = kc.size(2); c.D = kc.size(3);
  c.k_page = stride_of(kc, 0); c.k_token = stride_of(kc, 1); c.k_head = stride_of(kc, 2);
  c.v_page = stride_of(vc, 0); c.v_token = stride_of(vc, 1); c.v_head = stride_of(vc, 2);
  c.page_table = table.data_ptr<int32_t>();
  c.table_stride = stride_of(table, 0); c.table_width = table.size(1);
  c.cache_lens = lens.data_ptr<int32_t>(); c.n_seq = lens.size(0);
  return c;
}

// [T, heads, D] of the cache's type and device.
void check_tokens(const char *what, const char *name, const Tensor &t, const Tensor &kc) {
  if (t.dim() != 3 || t.size(2) != kc.size(3))
    throw AssertionFailed(std::string(what) + ": " + name + " must be [T, heads, " +
                          std::to_string(kc.size(3)) + "]");
  if (t.scalar_type() != kc.scalar_type() || t.device() != kc.device())
    throw AssertionFailed(std::string(what) + ": " + name +
                          " must have the cache's dtype and device");
}

std::optional<Tensor> paged_append(const Tensor &k_in, const Tensor &v_in, const Tensor &kc,
                                   const Tensor &vc, const Tensor &table, const Tensor &lens,
                                   const std::optional<Tensor> &cu,
                                   const std::optional<Tensor> &q_in,
                                   const std::optional<Tensor> &inv_freq, bool interleaved) {
  const char *what = "paged_kv_append";
  no_grad_only(what, {k_in, v_in, kc, vc, q_in.value_or(Tensor()), inv_freq.value_or(Tensor())});
  const vafa_paged_cache c = cache_of(what, kc, vc, table, lens);
  check_tokens(what, "k", k_in, kc);
  check_tokens(what, "v", v_in, kc);
  need(k_in.size(1) == c.Hk && v_in.sizes() == k_in.sizes(), what,
       "k and v must be [T, H_k, D] with the cache's heads");
  const int64_t T = k_in.size(0);
  if (cu) {
    need(cu->dim() == 1 && cu->size(0) == c.n_seq + 1, what, "cu_seqlens must be [n_seq + 1]");
    need(cu->scalar_type() == at::kInt && cu->device() == kc.device(), what,
         "cu_seqlens must be int32 on the cache's device");
    if (!dense(*cu, 0))
      throw py::value_error(std::string(what) + ": cu_seqlens must be contiguous");
  } else {
    need(T == c.n_seq, what, "without cu_seqlens there must be one token per sequence");
  }
  int64_t rot = 0;
  if (inv_freq) {
    need(inv_freq->dim() == 1 && 2 * inv_freq->size(0) <= c.D, what,
         "inv_freq must be [rotated features / 2]");
    need(inv_freq->scalar_type() == at::kFloat && inv_freq->device() == kc.device(), what,
         "inv_freq must be float32 on the cache's device");
    if (!dense(*inv_freq, 0))
      throw py::value_error(std::string(what) + ": inv_freq must be contiguous");
    rot = 2 * inv_freq->size(0);
  }
  int64_t H = 0;
  if (q_in) {
    check_tokens(what, "q", *q_in, kc);
    need(q_in->size(0) == T, what, "q must have as many tokens as k");
    H = q_in->size(1);
  }
  on_gpu(what, kc);
  Call call(kc);
  const Tensor k = rows_in(k_in), v = rows_in(v_in);
  Tensor q, out;
  if (q_in) {
    q = rows_in(*q_in);
    out = call.empty({T, H, c.D});
  }
  check(api.paged_append(&c, ptr(k), stride_of(k, 0), stride_of(k, 1), ptr(v), stride_of(v, 0),
                         stride_of(v, 1), T, cu ? cu->data_ptr<int32_t>() : nullptr, ptr(q),
                         q_in ? stride_of(q, 0) : 0, q_in ? stride_of(q, 1) : 0, H, ptr(out),
                         inv_freq ? f32(*inv_freq) : nullptr, rot, interleaved, dtype_of(kc),
                         call.stream));
  for (const Tensor *t : {&kc, &vc})
    if (!t->is_inference()) t->unsafeGetTensorImpl()->bump_version();
  return q_in ? std::optional<Tensor>(out) : std::nullopt;
}

// slopes [H] of the distance bias, float32 on q's device.
const float *slopes_of(const char *what, const std::optional<Tensor> &slopes, int64_t H,
                       const Tensor &q) {
  if (!slopes) return nullptr;
  need(slopes->dim() == 1 && slopes->size(0) == H, what, "alibi_slopes must be [H]");
  need(slopes->scalar_type() == at::kFloat && slopes->device() == q.device(), what,
       "alibi_slopes must be float32 on q's device");
  if (!dense(*slopes, 0))
    throw py::value_error(std::string(what) + ": alibi_slopes must be contiguous");
  return f32(*slopes);
}

Tensor paged_decode(const Tensor &q_in, const Tensor &kc, const Tensor &vc, const Tensor &table,
                    const Tensor &lens, double scale, std::optional<double> softcap,
                    std::optional<int64_t> window, const std::optional<Tensor> &slopes) {
  const char *what = "paged_decode_attn";
  no_grad_only(what, {q_in, kc, vc, slopes.value_or(Tensor())});
  // (1e-50 would be 0 in 32 bits, which means none)
  if (softcap && !(*softcap > 0 && (float)*softcap > 0.f))
    throw py::value_error("softcap must be positive");
  if (window && *window < 1) throw py::value_error("window must be positive");
  const vafa_paged_cache c = cache_of(what, kc, vc, table, lens);
  check_tokens(what, "q", q_in, kc);
  need(q_in.size(0) == c.n_seq, what, "q must hold one token per sequence");
  const int64_t H = q_in.size(1);
  const float *sl = slopes_of(what, slopes, H, q_in);
  on_gpu(what, kc);
  Call call(kc);
  const Tensor q = rows_in(q_in);
  Tensor out = call.empty({c.n_seq, H, c.D});
  void *ws = call.workspace(api.paged_decode_workspace(&c, H, window.value_or(0)));
  check(api.paged_decode(&c, ptr(q), stride_of(q, 0), stride_of(q, 1), H, ptr(out), (float)scale,
                         (float)softcap.value_or(0.0), window.value_or(0), sl, dtype_of(kc), ws,
                         call.ws_bytes(), call.stream));
  return out;
}

// dtype and content of an integer tensor on the host, for a plan's key (tensor.numpy()
// alone takes 5 to 10 us).
py::bytes cu_key(const Tensor &t) {
  if (!t.is_cpu() || !t.is_contiguous()) throw py::value_error("cu_key: a contiguous host tensor");
  std::string s(1, (char)t.scalar_type());
  s.append(static_cast<const char *>(t.data_ptr()), (size_t)t.nbytes());
  return py::bytes(s);
}

// Rows that the plan does not reach (possible where validation is off) as zeros.
void clear_rest(const Tensor &t, int64_t rows) {
  if (t.size(0) > rows) t.slice(0, rows).zero_();
}

// packed_masked_attn's operands as the kernels read them: [T, heads, D], contiguous,
// 16-byte aligned; with the checks of everything but the lengths.
std::tuple<Tensor, Tensor, Tensor> masked_operands(const Tensor &q_in, const Tensor &k_in,
                                                   const Tensor &v_in,
                                                   const std::optional<Tensor> &slopes) {
  auto rows = [](const Tensor &x, const char *name) {
    if (x.dim() != 3 && x.dim() != 4)
      throw py::value_error(std::string(name) + ": expected 3-D [T,H,D] or 4-D [1,T,H,D], got " +
                            std::to_string(x.dim()) + "-D");
    if (x.dim() == 4 && x.size(0) != 1)
      throw py::value_error(std::string(name) + ": 4-D input must have batch=1 (packed varlen)");
    Tensor t = x.dim() == 4 ? x.squeeze(0) : x;
    if (!t.is_contiguous()) t = t.contiguous();
    // (a view: the copy stays in the autograd graph)
    return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 != 0 ? t.clone() : t;
  };
  const char *what = "packed_masked_attn";
  direct_only(what, {q_in, k_in, v_in, slopes.value_or(Tensor())});
  const Tensor q = rows(q_in, "q"), k = rows(k_in, "k"), v = rows(v_in, "v");
  const int64_t H = q.size(1), D = q.size(2), Hk = k.size(1);
  need(k.size(2) == D && v.sizes() == k.sizes(), what, "k and v must be [T_k, H_k, D] alike");
  if (Hk < 1 || H < 1 || H % Hk != 0)
    throw AssertionFailed(std::to_string(H) + " query heads do not divide among " +
                          std::to_string(Hk) + " key heads");
  const auto dt = q.scalar_type();
  need(k.scalar_type() == dt && v.scalar_type() == dt, what, "q/k/v must share dtype");
  need(dt == at::kHalf || dt == at::kBFloat16, what, "dtype not supported (float16, bfloat16)");
  if (D != 64 && D != 128 && D != 256)
    throw AssertionFailed("head_dim " + std::to_string(D) + " not supported (64, 128, 256)");
  slopes_of(what, slopes, H, q);
  if (slopes && slopes->requires_grad() && at::GradMode::is_enabled())
    throw py::value_error("alibi_slopes get no gradient: detach them");
  need(q.is_cuda() && k.device() == q.device() && v.device() == q.device(), what,
       "requires GPU tensors on one device");
  return {q, k, v};
}

// o, and for a backward its low bytes and LSE.
std::tuple<Tensor, Tensor, Tensor> masked_fwd(const Tensor &q, const Tensor &k, const Tensor &v,
                                              const Plan &p, double scale, double softcap,
                                              int64_t window,
                                              const std::optional<Tensor> &slopes, bool train) {
  Call c(q);
  // evicted from the cache while a kernel of this stream still reads it, the plan keeps
  // its memory until the stream's work is done
  p.items.record_stream(c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(q.device().index()).unwrap());
  const int64_t H = q.size(1), D = q.size(2);
  const float *sl = slopes_of("packed_masked_attn", slopes, H, q);
  Tensor o = c.like(q), lo, lse;
  if (train) {
    lo = at::empty(q.sizes(), q.options().dtype(at::kByte));
    lse = c.empty_f32({q.size(0), H});
  }
  void *ws = c.workspace(api.masked_fwd_workspace(&p.info, k.size(1), D));
  check(api.masked_fwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lo), f32w(lse), p.dev(c), &p.info,
                       k.size(1), D, dtype_of(q), (float)scale, (float)softcap, window, sl, ws,
                       c.ws_bytes(), c.stream));
  clear_rest(o, p.info.T_q);
  return {o, lo, lse};
}

std::tuple<Tensor, Tensor, Tensor> masked_bwd(const Tensor &q, const Tensor &k, const Tensor &v,
                                              const Tensor &o, const Tensor &lo,
                                              const Tensor &lse, const Tensor &g,
                                              const Plan &p, double scale, double softcap,
                                              int64_t window,
                                              const std::optional<Tensor> &slopes) {
  Call c(q);
  const int64_t H = q.size(1), D = q.size(2), Hk = k.size(1);
  const float *sl = slopes_of("packed_masked_attn", slopes, H, q);
  const Tensor dout = grad_in(g, q);
  Tensor dq = c.like(q), dk = c.like(k), dv = c.like(v);
  void *ws = c.workspace(api.masked_bwd_workspace(&p.info, Hk, D));
  check(api.masked_bwd(ptr(q), ptr(k), ptr(v), ptr(o), ptr(lo), ptr(dout), f32(lse), ptr(dq),
                       ptr(dk), ptr(dv), p.dev(c), &p.info, Hk, D, dtype_of(q), (float)scale,
                       (float)softcap, window, sl, ws, c.ws_bytes(), c.stream));
  clear_rest(dq, p.info.T_q);
  clear_rest(dk, p.info.T_k);
  clear_rest(dv, p.info.T_k);
  return {dq, dk, dv};
}

// The operator with its backward as a native autograd node: no Python runs in the engine's
// thread (forward + backward of a small call 110 -> 81 us of host time).
struct PlanHolder : torch::CustomClassHolder {
  Plan plan;
  explicit PlanHolder(const Plan &p) : plan(p) {}
};

struct MaskedAttn : torch::autograd::Function<MaskedAttn> {
  static Tensor forward(torch::autograd::AutogradContext *ctx, const Tensor &q, const Tensor &k,
                        const Tensor &v, const Plan &p, double scale, double softcap,
                        int64_t window, const std::optional<Tensor> &slopes) {
    auto [o, lo, lse] = masked_fwd(q, k, v, p, scale, softcap, window, slopes, true);
    ctx->save_for_backward({q, k, v, o, lo, lse, slopes.value_or(Tensor())});
    ctx->saved_data["plan"] = c10::IValue::make_capsule(c10::make_intrusive<PlanHolder>(p));
    ctx->saved_data["scale"] = scale;
    ctx->saved_data["softcap"] = softcap;
    ctx->saved_data["window"] = window;
    return o;
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext *ctx,
                                                 torch::autograd::variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const auto holder = ctx->saved_data["plan"].toCapsule();
    const Plan &p = static_cast<PlanHolder *>(holder.get())->plan;
    const Tensor &sl = saved[6];
    Tensor dq, dk, dv;
    std::tie(dq, dk, dv) =
        masked_bwd(saved[0], saved[1], saved[2], saved[3], saved[4], saved[5], grads[0], p,
                   ctx->saved_data["scale"].toDouble(), ctx->saved_data["softcap"].toDouble(),
                   ctx->saved_data["window"].toInt(),
                   sl.defined() ? std::optional<Tensor>(sl) : std::nullopt);
    if (at::GradMode::is_enabled()) {  // create_graph: the gradients depend on these four
      const auto no_second = std::make_shared<torch::autograd::Error>(
          "packed_masked_attn has no second derivative",
          torch::autograd::collect_next_edges(saved[0], saved[1], saved[2], grads[0]));
      for (Tensor *t : {&dq, &dk, &dv}) torch::autograd::set_history(*t, no_second);
    }
    return {dq, dk, dv, Tensor(), Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor masked_attn(const Tensor &q, const Tensor &k, const Tensor &v, const Plan &p, double scale,
                   double softcap, int64_t window, const std::optional<Tensor> &slopes) {
  if (at::GradMode::is_enabled() &&
      (q.requires_grad() || k.requires_grad() || v.requires_grad()))
    return MaskedAttn::apply(q, k, v, p, scale, softcap, window, slopes);
  return std::get<0>(masked_fwd(q, k, v, p, scale, softcap, window, slopes, false));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  py::register_exception_translator([](std::exception_ptr e) {
    try {
      if (e) std::rethrow_exception(e);
    } catch (const AssertionFailed &x) {
      PyErr_SetString(PyExc_AssertionError, x.what());
    }
  });
  py::class_<Plan>(m, "Plan").def(py::init([](Tensor items, const py::bytes &info) {
    return Plan(std::move(items), std::string(info));
  }));
  // allocation and launch may wait (a full queue, an allocator retry): other
  // Python threads run meanwhile, as they do under a ctypes call
  py::call_guard<py::gil_scoped_release> no_gil;
  m.def("bind", &bind_library);
  m.def("varlen_fwd", &varlen_fwd, no_gil);
  m.def("varlen_bwd", &varlen_bwd, no_gil);
  m.def("absorb_fwd", &absorb_fwd, no_gil);
  m.def("absorb_bwd", &absorb_bwd, no_gil);
  m.def("absorb_full_fwd", &absorb_full_fwd, no_gil);
  m.def("absorb_full_bwd", &absorb_full_bwd, no_gil);
  m.def("project_fwd", &project_fwd, no_gil);
  m.def("project_bwd", &project_bwd, no_gil);
  m.def("cu_key", &cu_key);
  m.def("masked_operands", &masked_operands, no_gil);
  m.def("masked_attn", &masked_attn, no_gil);
  m.def("paged_append", &paged_append, no_gil);
  m.def("paged_decode", &paged_decode, no_gil);
}
