// Host side of the operators around attention: argument checks, outputs and
// workspaces from torch's allocator, autograd nodes and the calls into libsolattn,
// as a Python extension (_native.so). A call of one launch takes 5.5-6.5 us of host time,
// what one of torch's own elementwise kernels takes, of two 9-10, where the same steps in
// Python and ctypes took 25-33; a forward and backward pass 45-95 us, most of it torch's
// engine, where Python nodes took 95-175.
//
// Nothing here links against libsolattn: init() takes the addresses that the ctypes
// binding has loaded, so both always call the same library.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <c10/util/StringUtil.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/csrc/utils/pybind.h>

#include <algorithm>
#include <cmath>
#include <string>
#include <utility>
#include <vector>

#include "../../include/solattn.h"

namespace py = pybind11;
using at::Tensor;
using OptTensor = std::optional<Tensor>;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

namespace {

struct Library {
  decltype(&solattn_last_error) last_error = nullptr;
  decltype(&solattn_qk_norm_rope) qk_norm_rope = nullptr;
  decltype(&solattn_qk_norm_rope_append) qk_norm_rope_append = nullptr;
  decltype(&solattn_qk_norm_rope_bwd) qk_norm_rope_bwd = nullptr;
  decltype(&solattn_qk_norm_rope_bwd_workspace_bytes) qk_norm_rope_bwd_workspace_bytes = nullptr;
  decltype(&solattn_window_attn) window_attn = nullptr;
  decltype(&solattn_window_attn_workspace_bytes) window_attn_workspace_bytes = nullptr;
  decltype(&solattn_window_attn_bwd) window_attn_bwd = nullptr;
  decltype(&solattn_window_attn_bwd_workspace_bytes) window_attn_bwd_workspace_bytes = nullptr;
  decltype(&solattn_paged_attn_shared) paged_attn_shared = nullptr;
  decltype(&solattn_paged_attn_shared_workspace_bytes) paged_attn_shared_workspace_bytes = nullptr;
  decltype(&solattn_qk_norm_rope_append8) qk_norm_rope_append8 = nullptr;
  decltype(&solattn_cache_append) cache_append = nullptr;
  decltype(&solattn_cache_read) cache_read = nullptr;
} lib;

// A libsolattn call that returned a status; raised as _capi.SolAttnError.
struct LibraryError : std::runtime_error {
  using std::runtime_error::runtime_error;
};

void check(int rc, const char* name) {
  if (rc != 0) throw LibraryError(c10::str(name, " failed (", rc, "): ", lib.last_error()));
}

template <typename... A>
[[noreturn]] void refuse(const A&... a) {
  throw py::value_error(c10::str(a...));
}

std::string shape(const Tensor& t) { return c10::str(t.sizes()); }

constexpr int64_t kMaxHeadDim = 128;

// A recorder of torch operators sees the outputs' allocation and nothing of the kernels,
// so what it records would return memory that nobody wrote.
void refuse_recording(const char* what) {
  using Mode = c10::impl::TorchDispatchModeKey;
  bool on = torch::jit::tracer::isTracing();
  for (const Mode m : {Mode::FAKE, Mode::PROXY, Mode::FUNCTIONAL})
    on = on || c10::impl::TorchDispatchModeTLS::get_mode(m).has_value();
  if (on) refuse(what, " cannot be traced: its kernels are no torch operators");
}

// Inputs of one call: 4-dimensional, of one type and device, one head dim.
struct Named {
  const char* name;
  const Tensor& t;
};
void check_rows(const Tensor& q, std::initializer_list<Named> others, bool fp32, const char* name = "q") {
  if (!q.is_cuda()) refuse(name, " is not a GPU tensor");
  const auto type = q.scalar_type();
  if (type != at::kBFloat16 && type != at::kHalf && !(fp32 && type == at::kFloat))
    refuse(name, " dtype ", type, "; bfloat16", fp32 ? ", float16 or float32" : " or float16");
  if (q.dim() != 4) refuse(name, " must have 4 dimensions, got shape ", shape(q));
  const int64_t D = q.size(3);
  for (const auto& o : others) {
    if (o.t.dim() != 4) refuse(o.name, " must have 4 dimensions, got shape ", shape(o.t));
    if (o.t.scalar_type() != type) refuse(o.name, " dtype ", o.t.scalar_type(), " differs from ", name, "'s ", type);
    if (o.t.device() != q.device()) refuse(o.name, " is on ", o.t.device(), ", ", name, " on ", q.device());
    if (o.t.size(3) != D) refuse(o.name, " has head_dim ", o.t.size(3), ", ", name, " ", D);
  }
  if (D < 8 || D > kMaxHeadDim || D % 8)
    refuse("head_dim ", D, " not supported (multiples of 8 up to ", kMaxHeadDim, ")");
}

int type_code(const Tensor& t) {
  return t.scalar_type() == at::kBFloat16 ? SOLATTN_BF16 : t.scalar_type() == at::kHalf ? SOLATTN_FP16 : SOLATTN_FP32;
}

bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

// A contiguous last dim and every row 16-byte aligned.
bool rows_aligned(const Tensor& t) {
  const int64_t whole = 16 / t.element_size();
  const auto s = t.strides();
  return s[3] == 1 && aligned16(t) && (s[0] | s[1] | s[2]) % whole == 0;
}
// Whether the kernels read t in place: aligned rows, token strides in their range.
bool row_ready(const Tensor& t) { return rows_aligned(t) && t.stride(1) < (1 << 24); }
Tensor as_rows(const Tensor& t) {
  // (a contiguous tensor may be misaligned, so contiguous() alone is not enough)
  return row_ready(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

void check_kv_heads(int64_t heads, int64_t kv_heads) {
  if (kv_heads < 1 || heads < 1 || heads % kv_heads)
    refuse(heads, " query heads cannot share ", kv_heads, " kv heads");
}

void check_int32(const Tensor& t, const char* name, at::IntArrayRef want, const at::Device& device) {
  if (t.scalar_type() != at::kInt || t.sizes() != want || t.device() != device)
    refuse(name, " must be an int32 tensor of shape ", want, " on ", device, ", got ", t.scalar_type(), " ", t.sizes(),
           " on ", t.device());
}

void check_window(const std::optional<int64_t>& window, int64_t sinks, double scale) {
  if (window && *window < 1) refuse("window ", *window, "; at least 1, or None");
  if (sinks < 0) refuse("sinks ", sinks);
  if (!(static_cast<float>(scale) > 0.f) || !std::isfinite(static_cast<float>(scale)))
    refuse("scale ", scale, " is not a positive float");
}

// A paged cache: k_cache and v_cache [pages, page_size, Hkv, D], page_table int32
// [B, pages of a sequence], lengths int32 [B].
void check_cache(const Tensor& k, const Tensor& v, const Tensor& table, const Tensor& lengths, int64_t B,
                 const at::Device& device) {
  if (k.sizes() != v.sizes()) refuse("cache shapes differ: ", shape(k), " ", shape(v));
  if (!rows_aligned(k) || !rows_aligned(v))  // read and written in place: a copy would not be the cache
    refuse("cache rows must be contiguous and 16-byte aligned, strides ", k.strides(), " ", v.strides());
  if (k.size(1) % 8 || k.size(1) == 0) refuse("page size ", k.size(1), " is not a multiple of 8");
  if (table.dim() != 2 || table.size(0) != B)
    refuse("page_table must be [", B, ", pages of a sequence], got ", shape(table));
  check_int32(table, "page_table", table.sizes(), device);
  check_int32(lengths, "lengths", {B}, device);
}

// (the stride of a dim of one says nothing)
int64_t scale_stride(const Tensor& t, int d) { return t.defined() && t.size(d) > 1 ? t.stride(d) : 0; }

// A cache of codes: k_cache and v_cache of int8 or float8_e4m3fn, each with the rows'
// powers of two, float8_e8m0fnu [pages, Hkv, page_size]. Returns the library's cache_type.
int check_codes(const Tensor& k, const Tensor& v, const OptTensor& ks, const OptTensor& vs, int64_t D,
                const at::Device& device) {
  if (!ks || !vs) refuse("k_scale and v_scale go together");
  const auto type = k.scalar_type();
  if (type != at::kChar && type != at::kFloat8_e4m3fn)
    refuse("k_cache dtype ", type, " with scales; int8 or float8_e4m3fn");
  if (v.scalar_type() != type) refuse("v_cache dtype ", v.scalar_type(), " differs from k_cache's ", type);
  if (k.dim() != 4 || v.dim() != 4) refuse("caches must have 4 dimensions, got ", shape(k), " ", shape(v));
  if (k.device() != device || v.device() != device)
    refuse("caches are on ", k.device(), " and ", v.device(), ", the call on ", device);
  if (k.size(3) != D) refuse("k_cache has head_dim ", k.size(3), ", the call ", D);
  if (D < 16 || D > kMaxHeadDim || D % 16)
    refuse("head_dim ", D, " of an 8-bit cache (multiples of 16 up to ", kMaxHeadDim, ")");
  for (const Tensor& t : {*ks, *vs}) {
    const int64_t want[3] = {k.size(0), k.size(2), k.size(1)};
    if (t.scalar_type() != at::kFloat8_e8m0fnu || t.sizes() != at::IntArrayRef(want, 3) || t.device() != device)
      refuse("scales must be float8_e8m0fnu of shape ", at::IntArrayRef(want, 3), " on ", device, ", got ",
             t.scalar_type(), " ", t.sizes(), " on ", t.device());
    if (t.stride(2) != 1 || (scale_stride(t, 0) | scale_stride(t, 1)) % 8 ||
        reinterpret_cast<uintptr_t>(t.data_ptr()) % 8)
      refuse("a page's scales of a head must be contiguous and 8-byte aligned, strides ", t.strides());
  }
  return type == at::kChar ? SOLATTN_INT8 : SOLATTN_E4M3;
}

// k's and v's tensors that a call writes to in place.
void check_written(const Tensor& k, const Tensor& v) {
  for (const Tensor& c : {k, v})
    for (int64_t d = 0; d + 1 < c.dim(); ++d)
      if (c.stride(d) == 0 && c.size(d) > 1) refuse("a cache to write to is expanded: strides ", c.strides());
}
void check_apart(const Tensor& k, const Tensor& v) {
  if (k.numel() && k.data_ptr() == v.data_ptr()) refuse("k_cache and v_cache are the same memory");
}
void written(std::initializer_list<Tensor> ts) {  // (a backward pass that has kept the cache finds it changed)
  for (const Tensor& c : ts)
    if (!c.is_inference()) c.unsafeGetTensorImpl()->bump_version();
}

// (a table without pages is never read, but its address must not be null)
Tensor page_rows(const Tensor& table, const Tensor& lengths) {
  if (table.size(1) == 0) return lengths;
  return table.size(1) > 1 && table.stride(1) != 1 ? table.contiguous() : table;
}

Tensor tensor(const OptTensor& t) { return t.value_or(Tensor()); }

bool wants_grad(std::initializer_list<Tensor> ts) {
  if (!at::GradMode::is_enabled()) return false;
  for (const auto& t : ts)
    if (t.defined() && t.requires_grad()) return true;
  return false;
}

void refuse_grad(const char* what, std::initializer_list<Tensor> ts) {
  if (wants_grad(ts)) refuse(what, " has no gradient; call it under torch.no_grad()");
}

// Forward-mode derivatives: the nodes below have backward passes only, and without a
// node a tangent would be dropped.
void refuse_tangents(const char* what, std::initializer_list<Tensor> ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const auto& t : ts)
    if (t.defined() && t._fw_grad(0).defined()) refuse(what, " has no forward-mode derivative");
}

// backward() under create_graph=True would return gradients cut off from the graph.
void once_only(const char* what) {
  TORCH_CHECK(!at::GradMode::is_enabled(), what, " can be differentiated once only");
}

Tensor workspace(int64_t bytes, const Tensor& like) {
  return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor();
}

solattn_stream_t stream_of(const Tensor& t) {
  return reinterpret_cast<solattn_stream_t>(
      at::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream());
}

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T>
T* ptr_as(const Tensor& t) {
  return static_cast<T*>(ptr(t));
}
using U16 = uint16_t;

#define STRIDES(t) (t).stride(0), (t).stride(1), (t).stride(2)

// ------------------------------------------------------- norms and rotation
struct RopePlan {
  Tensor qw, kw, cos, sin, positions;
  int64_t P = 0, R = 0, pos_b = 0;
  bool interleaved = false;
  double eps = 0;
};

Tensor weight_of(const OptTensor& w, const char* name, const Tensor& q) {
  if (!w) return {};
  if (w->dim() != 1 || w->size(0) != q.size(3) || w->device() != q.device() || !w->is_floating_point())
    refuse(name, " must be a float tensor of shape [", q.size(3), "] on ", q.device(), ", got ", w->scalar_type(), " ",
           w->sizes(), " on ", w->device());
  Tensor f = w->to(at::kFloat).contiguous();
  return aligned16(f) ? f : f.clone(at::MemoryFormat::Contiguous);
}

Tensor table_of(const Tensor& t, const char* name, const Tensor& q) {
  if (t.scalar_type() != at::kFloat || t.device() != q.device())
    refuse(name, " must be float32 on ", q.device(), ", got ", t.scalar_type(), " on ", t.device());
  return t.is_contiguous() && aligned16(t) ? t : t.clone(at::MemoryFormat::Contiguous);
}

RopePlan rope_plan(const Tensor& q, const OptTensor& qw, const OptTensor& kw, const OptTensor& cos, const OptTensor& sin,
                   double eps, bool interleaved) {
  RopePlan p;
  p.qw = weight_of(qw, "q_weight", q);
  p.kw = weight_of(kw, "k_weight", q);
  if (!(eps >= 0.0) || !std::isfinite(static_cast<float>(eps))) refuse("eps ", eps, " is not a float from 0 on");
  p.eps = eps;
  p.interleaved = interleaved;
  if (!cos && !sin) return p;
  if (!cos || !sin) refuse("cos and sin go together");
  if (wants_grad({*cos, *sin})) refuse("cos and sin have no gradient; detach them");
  if (cos->dim() != 2 || cos->sizes() != sin->sizes() || cos->size(0) == 0)
    refuse("cos and sin must be [positions, pairs], got ", cos->sizes(), " ", sin->sizes());
  p.P = cos->size(0);
  p.R = 2 * cos->size(1);
  const int64_t whole = interleaved ? 8 : 16;
  if (p.R > q.size(3) || p.R % whole) refuse(p.R, " rotated channels of ", q.size(3), "; a multiple of ", whole);
  p.cos = table_of(*cos, "cos", q);
  p.sin = table_of(*sin, "sin", q);
  return p;
}

std::pair<Tensor, Tensor> rope_forward(const Tensor& q, const Tensor& k, const RopePlan& p) {
  Tensor qo = at::empty(q.sizes(), q.options()), ko = at::empty(k.sizes(), k.options());
  if (q.numel() == 0) return {qo, ko};
  const c10::OptionalDeviceGuard guard(q.device());
  check(lib.qk_norm_rope(ptr(q), STRIDES(q), ptr(k), STRIDES(k), q.size(0), q.size(1), q.size(2), k.size(2), q.size(3),
                         type_code(q), ptr_as<float>(p.qw), ptr_as<float>(p.kw), ptr_as<float>(p.cos),
                         ptr_as<float>(p.sin), p.P, p.R, p.interleaved, ptr_as<int32_t>(p.positions), p.pos_b,
                         static_cast<float>(p.eps), ptr(qo), STRIDES(qo), ptr(ko), STRIDES(ko), stream_of(q)),
        "solattn_qk_norm_rope");
  return {qo, ko};
}

struct NormRope : torch::autograd::Function<NormRope> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const OptTensor& q_weight,
                               const OptTensor& k_weight, const RopePlan& plan) {
    const Tensor qw = tensor(q_weight), kw = tensor(k_weight);
    ctx->save_for_backward({q, k, qw, kw, plan.cos, plan.sin, plan.positions});
    ctx->saved_data["P"] = plan.P;
    ctx->saved_data["R"] = plan.R;
    ctx->saved_data["pos_b"] = plan.pos_b;
    ctx->saved_data["interleaved"] = plan.interleaved;
    ctx->saved_data["eps"] = plan.eps;
    ctx->saved_data["need_qw"] = qw.defined() && qw.requires_grad();
    ctx->saved_data["need_kw"] = kw.defined() && kw.requires_grad();
    RopePlan p = plan;
    p.qw = qw;
    p.kw = kw;
    auto out = rope_forward(q, k, p);
    return {out.first, out.second};
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only("qk_norm_rope");
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &qw = s[2], &kw = s[3], &cos = s[4], &sin = s[5], &positions = s[6];
    auto& data = ctx->saved_data;
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options());
    const int64_t D = q.size(3);
    const auto f32 = q.options().dtype(at::kFloat);
    Tensor dqw = data["need_qw"].toBool() ? at::empty({D}, f32) : Tensor();
    Tensor dkw = data["need_kw"].toBool() ? at::empty({D}, f32) : Tensor();
    if (q.numel() == 0) {
      if (dqw.defined()) dqw.zero_();
      if (dkw.defined()) dkw.zero_();
      return {dq, dk, dqw, dkw, Tensor()};
    }
    const c10::OptionalDeviceGuard guard(q.device());
    const Tensor gq = as_rows(grads[0].defined() ? grads[0] : at::zeros(q.sizes(), q.options()));
    const Tensor gk = as_rows(grads[1].defined() ? grads[1] : at::zeros(k.sizes(), k.options()));
    const Tensor ws = workspace(dqw.defined() || dkw.defined() ? lib.qk_norm_rope_bwd_workspace_bytes(D) : 0, q);
    check(lib.qk_norm_rope_bwd(
              ptr(q), STRIDES(q), ptr(k), STRIDES(k), ptr(gq), STRIDES(gq), ptr(gk), STRIDES(gk), q.size(0), q.size(1),
              q.size(2), k.size(2), D, type_code(q), ptr_as<float>(qw), ptr_as<float>(kw), ptr_as<float>(cos),
              ptr_as<float>(sin), data["P"].toInt(), data["R"].toInt(), data["interleaved"].toBool(),
              ptr_as<int32_t>(positions), data["pos_b"].toInt(), static_cast<float>(data["eps"].toDouble()), ptr(dq),
              STRIDES(dq), ptr(dk), STRIDES(dk), ptr_as<float>(dqw), ptr_as<float>(dkw), ptr(ws),
              ws.defined() ? ws.numel() : 0, stream_of(q)),
          "solattn_qk_norm_rope_bwd");
    return {dq, dk, dqw, dkw, Tensor()};
  }
};

std::pair<Tensor, Tensor> qk_norm_rope(const Tensor& q0, const Tensor& k0, const OptTensor& qw, const OptTensor& kw,
                                       const OptTensor& cos, const OptTensor& sin, double eps,
                                       const OptTensor& positions, bool interleaved) {
  refuse_recording("qk_norm_rope");
  refuse_tangents("qk_norm_rope", {q0, k0, tensor(qw), tensor(kw), tensor(cos), tensor(sin)});
  check_rows(q0, {{"k", k0}}, true);
  const int64_t B = q0.size(0), T = q0.size(1);
  if (k0.size(0) != B || k0.size(1) != T) refuse("q and k hold different tokens: ", shape(q0), " ", shape(k0));
  if (q0.size(2) < 1 || k0.size(2) < 1) refuse("no heads: ", shape(q0), " ", shape(k0));
  RopePlan p = rope_plan(q0, qw, kw, cos, sin, eps, interleaved);
  if (positions) {
    const Tensor& t = *positions;
    if ((t.scalar_type() != at::kInt && t.scalar_type() != at::kLong) || t.device() != q0.device())
      refuse("positions must be int32 or int64 on ", q0.device(), ", got ", t.scalar_type(), " on ", t.device());
    const bool batch = t.dim() == 2 && t.size(0) == B && t.size(1) == T;
    if (!batch && !(t.dim() == 1 && t.size(0) == T))
      refuse("positions must be [", T, "] or [", B, ", ", T, "], got ", shape(t));
    // (int64 positions beyond 32 bits clamp to the table, as the kernel does)
    p.positions = (t.scalar_type() == at::kLong ? t.clamp(0, std::max<int64_t>(p.P - 1, 0)) : t).to(at::kInt).contiguous();
    p.pos_b = batch ? T : 0;
  } else if (p.R && T > p.P) {
    refuse(T, " tokens, a table of ", p.P, " positions");
  }
  const Tensor q = as_rows(q0), k = as_rows(k0);
  if (wants_grad({q, k, p.qw, p.kw})) {
    const auto optional = [](const Tensor& t) { return t.defined() ? OptTensor(t) : std::nullopt; };
    auto out = NormRope::apply(q, k, optional(p.qw), optional(p.kw), p);
    return {out[0], out[1]};
  }
  return rope_forward(q, k, p);
}

#define SCALES(t) ptr_as<uint8_t>(t), scale_stride(t, 0), scale_stride(t, 1)

Tensor qk_norm_rope_append(const Tensor& q0, const Tensor& k0, const Tensor& v0, const Tensor& k_cache,
                           const Tensor& v_cache, const Tensor& table0, const Tensor& lengths0, const OptTensor& qw,
                           const OptTensor& kw, const OptTensor& cos, const OptTensor& sin, double eps,
                           bool interleaved, const OptTensor& k_scale, const OptTensor& v_scale) {
  const char* what = "qk_norm_rope_append";
  refuse_recording(what);
  refuse_tangents(what, {q0, k0, v0, k_cache, v_cache, tensor(qw), tensor(kw), tensor(cos), tensor(sin)});
  refuse_grad(what, {q0, k0, v0, k_cache, v_cache, tensor(qw), tensor(kw)});
  const bool codes = k_scale || v_scale;
  int cache_type = 0;
  if (codes) {
    check_rows(q0, {{"k", k0}, {"v", v0}}, true);
    cache_type = check_codes(k_cache, v_cache, k_scale, v_scale, q0.size(3), q0.device());
  } else {
    check_rows(q0, {{"k", k0}, {"v", v0}, {"k_cache", k_cache}, {"v_cache", v_cache}}, true);
  }
  const int64_t B = q0.size(0), T = q0.size(1), H = q0.size(2), Hkv = k0.size(2);
  if (k0.size(0) != B || k0.size(1) != T || k0.sizes() != v0.sizes() || k_cache.size(2) != Hkv)
    refuse("shapes do not match: q ", shape(q0), " k ", shape(k0), " v ", shape(v0), " cache ", shape(k_cache));
  check_kv_heads(H, Hkv);
  check_cache(k_cache, v_cache, table0, lengths0, B, q0.device());
  check_written(k_cache, v_cache);
  if (codes) check_written(*k_scale, *v_scale);
  const RopePlan p = rope_plan(q0, qw, kw, cos, sin, eps, interleaved);
  check_apart(k_cache, v_cache);
  if (codes) check_apart(*k_scale, *v_scale);
  const Tensor q = as_rows(q0), k = as_rows(k0), v = as_rows(v0);
  const Tensor lengths = lengths0.contiguous(), table = page_rows(table0, lengths);
  Tensor qo = at::empty(q.sizes(), q.options());
  if (q.numel() == 0) return qo;
  // a cache without pages is never written, but its address must not be null
  const bool none = k_cache.numel() == 0;
  const Tensor &kc = none ? k : k_cache, &vc = none ? v : v_cache;
  const int64_t pages = none ? 0 : k_cache.size(0), page = k_cache.size(1);
  const c10::OptionalDeviceGuard guard(q.device());
  if (codes) {
    const Tensor &ks = none ? q : *k_scale, &vs = none ? q : *v_scale;
    const auto stride = [none](const Tensor& t, int d) { return none ? 0 : t.stride(d); };
    check(lib.qk_norm_rope_append8(
              ptr(q), STRIDES(q), ptr(k), STRIDES(k), ptr(v), STRIDES(v), B, T, H, Hkv, q.size(3), type_code(q),
              ptr_as<float>(p.qw), ptr_as<float>(p.kw), ptr_as<float>(p.cos), ptr_as<float>(p.sin), p.P, p.R,
              interleaved, static_cast<float>(eps), ptr(qo), STRIDES(qo), ptr(kc), stride(kc, 0), stride(kc, 1),
              stride(kc, 2), ptr(vc), stride(vc, 0), stride(vc, 1), stride(vc, 2), pages, page, cache_type,
              SCALES(ks), SCALES(vs),
              ptr_as<int32_t>(table), table.stride(0), table0.size(1), ptr_as<int32_t>(lengths), stream_of(q)),
          "solattn_qk_norm_rope_append8");
    written({k_cache, v_cache, *k_scale, *v_scale});
    return qo;
  }
  check(lib.qk_norm_rope_append(
            ptr(q), STRIDES(q), ptr(k), STRIDES(k), ptr(v), STRIDES(v), B, T, H, Hkv, q.size(3), type_code(q),
            ptr_as<float>(p.qw), ptr_as<float>(p.kw), ptr_as<float>(p.cos), ptr_as<float>(p.sin), p.P, p.R, interleaved,
            static_cast<float>(eps), ptr(qo), STRIDES(qo), ptr(kc), STRIDES(kc), ptr(vc), STRIDES(vc), pages, page,
            ptr_as<int32_t>(table), table.stride(0), table0.size(1), ptr_as<int32_t>(lengths), stream_of(q)),
        "solattn_qk_norm_rope_append");
  written({k_cache, v_cache});
  return qo;
}

// -------------------------------------------------------------- 8-bit caches
void cache_append(const Tensor& k0, const Tensor& v0, const Tensor& k_cache, const Tensor& v_cache,
                  const Tensor& table0, const Tensor& lengths0, const OptTensor& k_scale, const OptTensor& v_scale) {
  const char* what = "cache_append";
  refuse_recording(what);
  refuse_tangents(what, {k0, v0, k_cache, v_cache});
  refuse_grad(what, {k0, v0, k_cache, v_cache});
  check_rows(k0, {{"v", v0}}, true, "k");
  const int64_t B = k0.size(0), T = k0.size(1), Hkv = k0.size(2), D = k0.size(3);
  const int cache_type = check_codes(k_cache, v_cache, k_scale, v_scale, D, k0.device());
  if (k0.sizes() != v0.sizes() || k_cache.size(2) != Hkv)
    refuse("shapes do not match: k ", shape(k0), " v ", shape(v0), " cache ", shape(k_cache));
  check_cache(k_cache, v_cache, table0, lengths0, B, k0.device());
  check_written(k_cache, v_cache);
  check_written(*k_scale, *v_scale);
  check_apart(k_cache, v_cache);
  check_apart(*k_scale, *v_scale);
  if (k0.numel() == 0 || k_cache.numel() == 0) return;
  const Tensor k = as_rows(k0), v = as_rows(v0), lengths = lengths0.contiguous(), table = page_rows(table0, lengths);
  const c10::OptionalDeviceGuard guard(k.device());
  check(lib.cache_append(ptr(k), STRIDES(k), ptr(v), STRIDES(v), B, T, Hkv, D, type_code(k), ptr(k_cache),
                         STRIDES(k_cache), ptr(v_cache), STRIDES(v_cache), k_cache.size(0), k_cache.size(1), cache_type,
                         SCALES(*k_scale), SCALES(*v_scale), ptr_as<int32_t>(table), table.stride(0), table0.size(1),
                         ptr_as<int32_t>(lengths), stream_of(k)),
        "solattn_cache_append");
  written({k_cache, v_cache, *k_scale, *v_scale});
}

std::pair<Tensor, Tensor> cache_read(const Tensor& k_cache, const Tensor& v_cache, const Tensor& table0,
                                     const Tensor& lengths0, const OptTensor& k_scale, const OptTensor& v_scale,
                                     int64_t tokens, const OptTensor& start0, at::ScalarType dtype) {
  const char* what = "cache_read";
  refuse_recording(what);
  refuse_tangents(what, {k_cache, v_cache});
  refuse_grad(what, {k_cache, v_cache});
  if (!k_cache.is_cuda()) refuse("k_cache is not a GPU tensor");
  if (k_cache.dim() != 4) refuse("k_cache must have 4 dimensions, got shape ", shape(k_cache));
  const auto device = k_cache.device();
  const int64_t D = k_cache.size(3), Hkv = k_cache.size(2);
  const int cache_type = check_codes(k_cache, v_cache, k_scale, v_scale, D, device);
  if (dtype != at::kBFloat16 && dtype != at::kHalf) refuse("dtype ", dtype, "; bfloat16 or float16");
  if (tokens < 0) refuse(tokens, " tokens");
  if (table0.dim() != 2) refuse("page_table must be [sequences, pages of a sequence], got ", shape(table0));
  const int64_t B = table0.size(0);
  check_cache(k_cache, v_cache, table0, lengths0, B, device);
  if (start0) check_int32(*start0, "start", {B}, device);
  const auto options = k_cache.options().dtype(dtype);
  Tensor k = at::empty({B, tokens, Hkv, D}, options), v = at::empty({B, tokens, Hkv, D}, options);
  if (k.numel() == 0) return {k, v};
  if (k_cache.numel() == 0) return {k.zero_(), v.zero_()};
  const Tensor lengths = lengths0.contiguous(), table = page_rows(table0, lengths);
  const Tensor start = start0 ? start0->contiguous() : Tensor();
  const c10::OptionalDeviceGuard guard(device);
  check(lib.cache_read(ptr(k_cache), STRIDES(k_cache), ptr(v_cache), STRIDES(v_cache), k_cache.size(0), k_cache.size(1),
                       cache_type, SCALES(*k_scale), SCALES(*v_scale), ptr_as<int32_t>(table), table.stride(0),
                       table0.size(1), ptr_as<int32_t>(lengths), ptr_as<int32_t>(start), B, tokens, Hkv, D, type_code(k),
                       ptr_as<U16>(k), STRIDES(k), ptr_as<U16>(v), STRIDES(v), stream_of(k)),
        "solattn_cache_read");
  return {k, v};
}

// ------------------------------------------------------------------- windows
struct WindowPlan {
  Tensor lengths;
  int64_t window = 1, sinks = 0, q_start = 0;
  bool causal = true;
  double scale = 1;
};

Tensor window_forward(const Tensor& q, const Tensor& k, const Tensor& v, const WindowPlan& p, const Tensor& lse,
                      const Tensor& o_lo) {
  const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), D = q.size(3), Tk = k.size(1), Hkv = k.size(2);
  Tensor out = at::empty({B, Tq, H, D}, q.options());
  const c10::OptionalDeviceGuard guard(q.device());
  const int64_t need = lib.window_attn_workspace_bytes(B, Tq, Tk, H, Hkv, D, p.q_start, p.window, p.sinks, p.causal,
                                                       lse.defined());
  const Tensor ws = workspace(need, q);
  check(lib.window_attn(ptr_as<U16>(q), STRIDES(q), ptr_as<U16>(k), STRIDES(k), ptr_as<U16>(v), STRIDES(v), B, Tq, Tk,
                        H, Hkv, D, type_code(q), p.q_start, ptr_as<int32_t>(p.lengths), p.window, p.sinks, p.causal,
                        static_cast<float>(p.scale), ptr_as<U16>(out), STRIDES(out), ptr_as<float>(lse),
                        ptr_as<U16>(o_lo), ptr(ws), need, stream_of(q)),
        "solattn_window_attn");
  return out;
}

struct WindowAttn : torch::autograd::Function<WindowAttn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& v,
                        const WindowPlan& p) {
    const Tensor lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    const Tensor o_lo = at::empty(q.sizes(), q.options());
    Tensor out = window_forward(q, k, v, p, lse, o_lo);
    ctx->save_for_backward({q, k, v, out, lse, p.lengths, o_lo});
    ctx->saved_data["window"] = p.window;
    ctx->saved_data["sinks"] = p.sinks;
    ctx->saved_data["q_start"] = p.q_start;
    ctx->saved_data["causal"] = p.causal;
    ctx->saved_data["scale"] = p.scale;
    return out;
  }
  static variable_list backward(AutogradContext* ctx, const variable_list& grads) {
    once_only("window_attn");
    const auto s = ctx->get_saved_variables();
    const Tensor &q = s[0], &k = s[1], &v = s[2], &out = s[3], &lse = s[4], &lengths = s[5], &o_lo = s[6];
    auto& data = ctx->saved_data;
    const int64_t B = q.size(0), Tq = q.size(1), H = q.size(2), D = q.size(3), Tk = k.size(1), Hkv = k.size(2);
    const int64_t window = data["window"].toInt(), sinks = data["sinks"].toInt();
    const bool causal = data["causal"].toBool();
    Tensor dq = at::empty(q.sizes(), q.options()), dk = at::empty(k.sizes(), k.options()),
           dv = at::empty(v.sizes(), v.options());
    const c10::OptionalDeviceGuard guard(q.device());
    const Tensor g = as_rows(grads[0]);
    const Tensor ws = workspace(lib.window_attn_bwd_workspace_bytes(B, Tq, Tk, H, Hkv, D, window, sinks, causal), q);
    check(lib.window_attn_bwd(ptr_as<U16>(q), STRIDES(q), ptr_as<U16>(k), STRIDES(k), ptr_as<U16>(v), STRIDES(v),
                              ptr_as<U16>(out), STRIDES(out), ptr_as<U16>(g), STRIDES(g), ptr_as<float>(lse),
                              ptr_as<U16>(o_lo), B, Tq, Tk, H, Hkv, D, type_code(q), data["q_start"].toInt(),
                              ptr_as<int32_t>(lengths), window, sinks, causal, static_cast<float>(data["scale"].toDouble()), ptr_as<U16>(dq), STRIDES(dq),
                              ptr_as<U16>(dk), STRIDES(dk), ptr_as<U16>(dv), STRIDES(dv), ptr(ws),
                              ws.defined() ? ws.numel() : 0, stream_of(q)),
          "solattn_window_attn_bwd");
    return {dq, dk, dv, Tensor()};
  }
};

Tensor window_attn(const Tensor& q0, const Tensor& k0, const Tensor& v0, std::optional<int64_t> window, int64_t sinks,
                   bool causal, std::optional<double> scale, const OptTensor& lengths, std::optional<int64_t> q_start) {
  refuse_recording("window_attn");
  refuse_tangents("window_attn", {q0, k0, v0});
  check_rows(q0, {{"k", k0}, {"v", v0}}, false);
  const int64_t B = q0.size(0), Tq = q0.size(1), H = q0.size(2), D = q0.size(3), Tk = k0.size(1);
  WindowPlan p;
  p.scale = scale ? *scale : 1.0 / std::sqrt(static_cast<double>(D));
  check_window(window, sinks, p.scale);
  if (k0.sizes() != v0.sizes() || k0.size(0) != B)
    refuse("q/k/v shapes do not match: ", shape(q0), " ", shape(k0), " ", shape(v0));
  check_kv_heads(H, k0.size(2));
  p.q_start = q_start ? *q_start : Tk - Tq;
  if (Tq > Tk || p.q_start < 0 || p.q_start > Tk - Tq) refuse(Tq, " rows from ", p.q_start, " on of ", Tk, " keys");
  if (lengths) {
    check_int32(*lengths, "lengths", {B}, q0.device());
    p.lengths = lengths->contiguous();
  }
  p.window = window ? std::min(*window, Tk) : Tk;
  p.sinks = std::min(sinks, Tk);
  p.causal = causal;
  const bool grad = wants_grad({q0, k0, v0});
  if (q0.numel() == 0)  // no rows: nothing to run, gradients of zeros
    return grad ? q0 * 1 + 0 * (k0.narrow(0, 0, 0).sum() + v0.narrow(0, 0, 0).sum()) : at::empty(q0.sizes(), q0.options());
  if (D != 64 && D != 128 && (grad || Tq > 1 || !causal)) {
    // zero channels add exact zeros to every product; the pad's gradient is a slice
    const int64_t pad[2] = {0, (D < 64 ? 64 : 128) - D};
    const Tensor q = at::constant_pad_nd(q0, pad), k = at::constant_pad_nd(k0, pad), v = at::constant_pad_nd(v0, pad);
    return (grad ? WindowAttn::apply(q, k, v, p) : window_forward(q, k, v, p, {}, {})).narrow(3, 0, D).contiguous();
  }
  const Tensor q = as_rows(q0), k = as_rows(k0), v = as_rows(v0);
  return grad ? WindowAttn::apply(q, k, v, p) : window_forward(q, k, v, p, {}, {});
}

// --------------------------------------------------------------------- pages
Tensor paged_attn(const Tensor& q0, const Tensor& k, const Tensor& v, const Tensor& table0, const Tensor& lengths0,
                  std::optional<int64_t> window, int64_t sinks, std::optional<double> scale0, const OptTensor& k_scale,
                  const OptTensor& v_scale, int64_t shared, int64_t groups) {
  refuse_recording("paged_attn");
  refuse_tangents("paged_attn", {q0, k, v});
  refuse_grad("paged_attn", {q0, k, v});
  int cache_type = 0;
  if (k_scale || v_scale) {
    check_rows(q0, {}, false);
    cache_type = check_codes(k, v, k_scale, v_scale, q0.size(3), q0.device());
  } else {
    check_rows(q0, {{"k_cache", k}, {"v_cache", v}}, false);
  }
  const int64_t B = q0.size(0), H = q0.size(2), D = q0.size(3), Hkv = k.size(2), pages = k.size(0), page = k.size(1);
  const double scale = scale0 ? *scale0 : 1.0 / std::sqrt(static_cast<double>(D));
  check_window(window, sinks, scale);
  if (q0.size(1) != 1) refuse("q holds ", q0.size(1), " tokens of a sequence; one");
  check_kv_heads(H, Hkv);
  check_cache(k, v, table0, lengths0, B, q0.device());
  if (shared < 0) refuse("shared ", shared);
  if (groups < 1 || B % groups) refuse(B, " sequences in ", groups, " groups");
  if (shared && (window || sinks)) refuse("shared keys and a window: what windows leave of them differs");
  Tensor out = at::empty({B, 1, H, D}, q0.options());
  if (B == 0) return out;
  const int64_t max_pages = table0.size(1);
  if (pages == 0 || max_pages == 0) return out.zero_();
  const Tensor q = as_rows(q0);
  const Tensor lengths = lengths0.contiguous(), table = page_rows(table0, lengths);
  const int64_t top = (1ll << 31) - 1, w = window ? std::min(*window, top) : 0;
  sinks = std::min(sinks, top);
  shared = std::min(shared, top);
  const c10::OptionalDeviceGuard guard(q.device());
  const int64_t need =
      lib.paged_attn_shared_workspace_bytes(B, H, Hkv, D, max_pages, page, w, sinks, cache_type, shared, groups);
  const Tensor ws = workspace(need, q);
  const Tensor ks = tensor(k_scale), vs = tensor(v_scale);
  check(lib.paged_attn_shared(
            ptr_as<U16>(q), q.stride(0), q.stride(2), ptr(k), STRIDES(k), ptr(v), STRIDES(v), pages, page, cache_type,
            SCALES(ks), SCALES(vs), ptr_as<int32_t>(table), table.stride(0), max_pages, ptr_as<int32_t>(lengths), B, H,
            Hkv, D, type_code(q), w, sinks, shared, groups, static_cast<float>(scale), ptr(ws), need, ptr_as<U16>(out),
            out.stride(0), out.stride(2), stream_of(q)),
        "solattn_paged_attn");
  return out;
}

template <typename F>
void take(F& f, const py::dict& addresses, const char* name) {
  f = reinterpret_cast<F>(addresses[name].cast<uintptr_t>());
}

}  // namespace

PYBIND11_MODULE(_native, m) {
  static PyObject* library_error = PyExc_RuntimeError;  // (kept for the life of the process)
  m.def("init", [](const py::dict& at, py::object error) {
    library_error = error.release().ptr();
    take(lib.last_error, at, "solattn_last_error");
    take(lib.qk_norm_rope, at, "solattn_qk_norm_rope");
    take(lib.qk_norm_rope_append, at, "solattn_qk_norm_rope_append");
    take(lib.qk_norm_rope_bwd, at, "solattn_qk_norm_rope_bwd");
    take(lib.qk_norm_rope_bwd_workspace_bytes, at, "solattn_qk_norm_rope_bwd_workspace_bytes");
    take(lib.window_attn, at, "solattn_window_attn");
    take(lib.window_attn_workspace_bytes, at, "solattn_window_attn_workspace_bytes");
    take(lib.window_attn_bwd, at, "solattn_window_attn_bwd");
    take(lib.window_attn_bwd_workspace_bytes, at, "solattn_window_attn_bwd_workspace_bytes");
    take(lib.paged_attn_shared, at, "solattn_paged_attn_shared");
    take(lib.paged_attn_shared_workspace_bytes, at, "solattn_paged_attn_shared_workspace_bytes");
    take(lib.qk_norm_rope_append8, at, "solattn_qk_norm_rope_append8");
    take(lib.cache_append, at, "solattn_cache_append");
    take(lib.cache_read, at, "solattn_cache_read");
  });
  py::register_local_exception_translator([](std::exception_ptr p) {
    try {
      if (p) std::rethrow_exception(p);
    } catch (const LibraryError& e) {
      PyErr_SetString(library_error, e.what());
    }
  });
  m.def("qk_norm_rope", &qk_norm_rope);
  m.def("qk_norm_rope_append", &qk_norm_rope_append);
  m.def("window_attn", &window_attn);
  m.def("paged_attn", &paged_attn);
  m.def("cache_append", &cache_append);
  m.def("cache_read", &cache_read);
}
