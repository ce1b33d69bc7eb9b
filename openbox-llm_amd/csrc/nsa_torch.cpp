// The torch side of the operators around the attention (nsa_lm.py,
// nsa_paged.py): argument checks, output allocation and the autograd nodes, in
// C++.  A generation step or a small training step spends more time in these
// than in its kernels: with the same work in Python over ctypes a norm took
// 9.6 us of host time, a paged step 16.3, and a norm forward and backward 63 to
// 128 (the backward runs on the engine's own thread).
//
// The kernels stay behind the C-ABI of libnsa_hip.so, whose addresses bind()
// takes from the loaded library: this module links against torch alone.
// Refusals are AssertionErrors; every launch goes to the current stream of the
// tensors' device; nothing waits for the host.
#include <ATen/ops/empty.h>
#include <ATen/ops/zeros_like.h>
#include <c10/core/AutogradState.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/utils/pybind.h>

#include <initializer_list>
#include <optional>
#include <string>
#include <tuple>
#include <vector>

#include "nsa_hip.h"

namespace py = pybind11;
using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

namespace {

// --- the library ------------------------------------------------------------
#define NSA_ENTRY(name) decltype(&name) p_##name = nullptr
NSA_ENTRY(nsa_norm_fwd);
NSA_ENTRY(nsa_norm_bwd);
NSA_ENTRY(nsa_norm_bwd_workspace);
NSA_ENTRY(nsa_logprob_fwd);
NSA_ENTRY(nsa_logprob_bwd);
NSA_ENTRY(nsa_logprob_workspace);
NSA_ENTRY(nsa_paged_attend_max);
NSA_ENTRY(nsa_paged_workspace);
#undef NSA_ENTRY

void bind(const py::dict& at) {
#define NSA_BIND(name) p_##name = reinterpret_cast<decltype(&name)>(at[#name].cast<uintptr_t>())
  NSA_BIND(nsa_norm_fwd);
  NSA_BIND(nsa_norm_bwd);
  NSA_BIND(nsa_norm_bwd_workspace);
  NSA_BIND(nsa_logprob_fwd);
  NSA_BIND(nsa_logprob_bwd);
  NSA_BIND(nsa_logprob_workspace);
  NSA_BIND(nsa_paged_attend_max);
  NSA_BIND(nsa_paged_workspace);
#undef NSA_BIND
}

// --- checks -----------------------------------------------------------------
[[noreturn]] void refuse(const std::string& why) {
  PyErr_SetString(PyExc_AssertionError, why.c_str());
  throw py::error_already_set();
}
#define NSA_ASSERT(cond, why) \
  do {                        \
    if (!(cond)) refuse(why); \
  } while (0)

// A status of the library: its refusals as assertions (with the interpreter's
// lock held), the rest as runtime errors.
void check_status(int rc, const char* what) {
  if (rc == NSA_OK) return;
  if (rc == NSA_ERR_SHAPE || rc == NSA_ERR_DTYPE)
    refuse(std::string(what) + ": unsupported shape or dtype (code " + std::to_string(rc) + ")");
  throw std::runtime_error(std::string(what) + ": HIP library error code " + std::to_string(rc));
}
// The same on the autograd engine's thread, without the lock.
void check_backward(int rc, const char* what) {
  TORCH_CHECK(rc == NSA_OK, what, ": HIP library error code ", rc);
}

bool is_float(const Tensor& t) { return t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16; }
void check_tensor(const Tensor& t, const char* what) {
  NSA_ASSERT(t.is_cuda(), std::string(what) + ": a GPU tensor is needed");
  NSA_ASSERT(is_float(t), std::string(what) + ": dtype " + c10::toString(t.scalar_type()) +
                              " is not supported (float32 or bfloat16)");
}
// Forward-mode derivatives: none of these operators has one, and the raw path
// would drop a dual tensor's tangent (it does not need requires_grad, and
// no_grad does not turn it off).
bool has_tangent(const Tensor& t) {
  return t.defined() && c10::AutogradState::get_tls_state().get_fw_grad_mode() && t._fw_grad(/*level=*/0).defined();
}
bool has_tangent(const OptTensor& t) { return t && has_tangent(*t); }
void no_tangent(bool found, const char* what) {
  NSA_ASSERT(!found, std::string(what) + " has no forward-mode derivative");
}
int code_of(at::ScalarType t) {
  return t == at::kFloat ? NSA_F32 : t == at::kBFloat16 ? NSA_BF16 : NSA_E4M3;
}

// --- plumbing ---------------------------------------------------------------
// t's device as the current one, and its current stream.
struct On {
  c10::DeviceIndex was, dev;
  void* stream;
  explicit On(const Tensor& t) : was(c10::hip::current_device()), dev(t.device().index()) {
    if (dev != was) c10::hip::set_device(dev);
    stream = static_cast<void*>(c10::hip::getCurrentHIPStream(dev).stream());
  }
  ~On() {
    if (dev != was) c10::hip::set_device(was);
  }
  On(const On&) = delete;
};
Tensor fresh(at::IntArrayRef sizes, const Tensor& like, at::ScalarType type) {
  return at::empty(sizes, like.options().dtype(type));
}
void* at_of(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
template <typename T> T* at_as(const Tensor& t) { return static_cast<T*>(at_of(t)); }
Tensor aligned(const Tensor& t) {   // dense, on 16 bytes
  Tensor c = t.contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}
bool wants_grad(const Tensor& a, const OptTensor& b, const Tensor& c) {
  return at::GradMode::is_enabled() && (a.requires_grad() || (b && b->requires_grad()) || c.requires_grad());
}

// A backward's gradients under create_graph: taking a second derivative raises.
variable_list once(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "trying to differentiate twice an operator that gives first derivatives only", (int64_t)grads.size());
  variable_list in = grads;
  for (auto& g : in)
    if (g.defined()) g = g.detach().requires_grad_();
  return node->apply(std::move(in));
}

// --- residual addition with root-mean-square norm -----------------------------
struct NormOut {
  Tensor y, h, scale, rstd;
};

NormOut norm_forward(const Tensor& x_, const OptTensor& res_, const Tensor& w_, double eps, at::ScalarType out,
                     bool want_rstd) {
  const Tensor x = x_.contiguous(), w = w_.contiguous(), res = res_ ? res_->contiguous() : Tensor();
  const int64_t D = x.size(-1), rows = x.numel() / D;
  NormOut o;
  o.h = res.defined() ? fresh(res.sizes(), res, res.scalar_type()) : x;
  o.y = fresh(x.sizes(), x, out);
  if (out == at::kFloat8_e4m3fn) o.scale = fresh(x.sizes().slice(0, x.dim() - 1), x, at::kFloat);
  if (want_rstd) o.rstd = fresh({rows}, x, at::kFloat);
  On on(x);
  check_status(p_nsa_norm_fwd(x.data_ptr(), at_of(res), w.data_ptr(), res.defined() ? o.h.data_ptr() : nullptr,
                              o.y.data_ptr(), at_as<float>(o.scale), at_as<float>(o.rstd), rows, (int)D, (float)eps,
                              code_of(x.scalar_type()), code_of(o.h.scalar_type()), code_of(w.scalar_type()),
                              code_of(out), on.stream),
               "nsa_norm_fwd");
  return o;
}

struct NormFn : torch::autograd::Function<NormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const OptTensor& res, const Tensor& w, double eps,
                               int64_t out) {
    ctx->set_materialize_grads(false);
    NormOut o = norm_forward(x, res, w, eps, static_cast<at::ScalarType>(out), true);
    ctx->save_for_backward({o.h, w.contiguous(), o.rstd});
    ctx->saved_data["x"] = static_cast<int64_t>(x.scalar_type());
    ctx->saved_data["added"] = res.has_value();
    if (res) return {o.y, o.h};
    return {o.y};
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor h = saved[0].contiguous(), &w = saved[1], &rstd = saved[2];
    const auto xt = static_cast<at::ScalarType>(ctx->saved_data["x"].toInt());
    const bool added = ctx->saved_data["added"].toBool();
    const bool need_w = ctx->needs_input_grad(added ? 2 : 1);
    Tensor dy = grads[0], dh = added ? grads[1] : Tensor(), dx, dr, dw;
    TORCH_CHECK(!has_tangent(dy) && !has_tangent(dh), "nsa_norm_bwd has no forward-mode derivative");
    if (!dy.defined()) {   // only the sum was used: its gradient passes through
      if (dh.defined()) {
        dx = dh.to(xt);
        dr = dh;
        if (need_w) dw = at::zeros_like(w);
      }
      return once({dx, dr, dw, Tensor(), Tensor()});
    }
    const int64_t D = h.size(-1), rows = h.numel() / D;
    dy = dy.contiguous();
    if (dh.defined()) dh = dh.contiguous();
    dx = fresh(h.sizes(), h, xt);
    const bool two = added && xt != h.scalar_type();
    if (two) dr = fresh(h.sizes(), h, h.scalar_type());
    if (need_w) dw = rows > 0 ? fresh(w.sizes(), w, w.scalar_type()) : at::zeros_like(w);
    if (rows > 0) {
      On on(h);
      Tensor ws;
      size_t bytes = 0;
      if (need_w) {
        bytes = p_nsa_norm_bwd_workspace(rows, (int)D, on.stream);
        ws = fresh({(int64_t)bytes}, h, at::kByte);
      }
      check_backward(p_nsa_norm_bwd(dy.data_ptr(), at_of(dh), h.data_ptr(), w.data_ptr(), at_as<float>(rstd),
                                    dx.data_ptr(), at_of(dr), at_of(dw), at_of(ws), bytes, rows, (int)D, code_of(xt),
                                    code_of(h.scalar_type()), code_of(w.scalar_type()), code_of(dy.scalar_type()),
                                    on.stream),
                     "nsa_norm_bwd");
    }
    if (added && !two) dr = dx;
    return once({dx, dr, dw, Tensor(), Tensor()});
  }
};

double norm_args(const Tensor& x, const OptTensor& res, const Tensor& w, std::optional<double> eps, const char* what) {
  const std::string at = std::string(what) + ": ";
  no_tangent(has_tangent(x) || has_tangent(res) || has_tangent(w), what);
  check_tensor(x, what);
  check_tensor(w, what);
  NSA_ASSERT(x.dim() >= 1 && x.size(-1) >= 1 && x.size(-1) <= (1 << 24), at + "x must be [..., D]");
  NSA_ASSERT(w.dim() == 1 && w.size(0) == x.size(-1), at + "weight must be [D]");
  NSA_ASSERT(w.device() == x.device(), at + "x and weight on different devices");
  if (res) {
    check_tensor(*res, what);
    NSA_ASSERT(res->sizes() == x.sizes() && res->device() == x.device(), at + "residual must be like x");
  }
  // (float32's epsilon for bf16 too: torch.nn.RMSNorm takes that of the type it computes in)
  const double e = eps ? *eps : 0x1p-23;
  NSA_ASSERT(e >= 0.0, at + "eps must not be negative");
  return e;
}

std::tuple<Tensor, Tensor> add_rms_norm(const Tensor& x, const OptTensor& res, const Tensor& w,
                                        std::optional<double> eps, std::optional<at::ScalarType> out_) {
  const double e = norm_args(x, res, w, eps, "add_rms_norm");
  const auto out = out_ ? *out_ : res ? res->scalar_type() : x.scalar_type();
  NSA_ASSERT(out == at::kFloat || out == at::kBFloat16, "add_rms_norm: out_dtype must be float32 or bfloat16");
  if (!wants_grad(x, res, w)) {
    NormOut o = norm_forward(x, res, w, e, out, false);
    return {o.y, res ? o.h : x};
  }
  auto o = NormFn::apply(x, res, w, e, static_cast<int64_t>(out));
  return {o[0], res ? o[1] : x};
}

std::tuple<Tensor, Tensor, Tensor> add_rms_norm_q8(const Tensor& x, const OptTensor& res, const Tensor& w,
                                                   std::optional<double> eps) {
  const double e = norm_args(x, res, w, eps, "add_rms_norm_q8");
  NSA_ASSERT(!wants_grad(x, res, w), "add_rms_norm_q8 has no gradient: call it under torch.no_grad()");
  NormOut o = norm_forward(x, res, w, e, at::kFloat8_e4m3fn, false);
  return {o.y, o.scale, res ? o.h : x};
}

// --- log probabilities of tokens ----------------------------------------------
struct LpOut {
  Tensor logp, ent, top_logp, top_idx, stat;
};

LpOut logprob_forward(const Tensor& z, const OptTensor& targets, int64_t top, bool want_stat) {
  const int64_t rows = z.size(0), V = z.size(1);
  LpOut o;
  if (targets) o.logp = fresh({rows}, z, at::kFloat);
  o.ent = fresh({rows}, z, at::kFloat);
  if (want_stat) o.stat = fresh({rows, 2}, z, at::kFloat);
  if (top > 0) {
    o.top_logp = fresh({rows, top}, z, at::kFloat);
    o.top_idx = fresh({rows, top}, z, at::kLong);
  }
  On on(z);
  const size_t bytes = p_nsa_logprob_workspace(rows, (int)V, (int)top, on.stream);
  NSA_ASSERT(bytes > 0, "token_logprobs: unsupported shape");
  const Tensor ws = bytes > 16 ? fresh({(int64_t)bytes}, z, at::kByte) : Tensor();
  check_status(p_nsa_logprob_fwd(z.data_ptr(), targets ? targets->const_data_ptr<int64_t>() : nullptr,
                                 at_as<float>(o.logp), at_as<float>(o.ent), at_as<float>(o.stat),
                                 at_as<float>(o.top_logp), at_as<int64_t>(o.top_idx), at_of(ws), bytes, rows, (int)V,
                                 (int)top, code_of(z.scalar_type()), on.stream),
               "nsa_logprob_fwd");
  return o;
}

struct LogprobFn : torch::autograd::Function<LogprobFn> {
  // Outputs: logp (with targets), entropy, top_logp and top_idx (with top)
  static variable_list forward(AutogradContext* ctx, const Tensor& z, const OptTensor& targets, int64_t top) {
    ctx->set_materialize_grads(false);
    LpOut o = logprob_forward(z, targets, top, true);
    ctx->save_for_backward({z, targets ? *targets : Tensor(), o.stat, o.ent});
    ctx->saved_data["targets"] = targets.has_value();
    variable_list out;
    if (targets) out.push_back(o.logp);
    out.push_back(o.ent);
    if (top > 0) {
      ctx->mark_non_differentiable({o.top_logp, o.top_idx});
      out.push_back(o.top_logp);
      out.push_back(o.top_idx);
    }
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &z = saved[0], &targets = saved[1], &stat = saved[2], &ent = saved[3];
    const bool t = ctx->saved_data["targets"].toBool();
    Tensor dlogp = t ? grads[0] : Tensor(), dent = grads[t ? 1 : 0];
    TORCH_CHECK(!has_tangent(dlogp) && !has_tangent(dent), "nsa_logprob_bwd has no forward-mode derivative");
    if (!dlogp.defined() && !dent.defined()) return {Tensor(), Tensor(), Tensor()};
    if (dlogp.defined()) dlogp = dlogp.contiguous();
    if (dent.defined()) dent = dent.contiguous();
    Tensor dz = fresh(z.sizes(), z, z.scalar_type());
    On on(z);
    check_backward(p_nsa_logprob_bwd(z.data_ptr(), at_as<int64_t>(targets), at_as<float>(stat), at_as<float>(ent),
                                     at_as<float>(dlogp), at_as<float>(dent), dz.data_ptr(), z.size(0),
                                     (int)z.size(1), code_of(z.scalar_type()), on.stream),
                   "nsa_logprob_bwd");
    return once({dz, Tensor(), Tensor()});
  }
};

std::tuple<OptTensor, Tensor, OptTensor, OptTensor> token_logprobs(const Tensor& logits, const OptTensor& targets_,
                                                                   int64_t top) {
  no_tangent(has_tangent(logits), "token_logprobs");
  check_tensor(logits, "token_logprobs: logits");
  NSA_ASSERT(logits.dim() >= 1 && logits.size(-1) >= 1 && logits.size(-1) <= (1 << 28),
             "token_logprobs: logits must be [..., V]");
  const int64_t V = logits.size(-1);
  const auto lead = logits.sizes().slice(0, logits.dim() - 1);
  NSA_ASSERT(top >= 0 && top <= 64 && top <= V, "token_logprobs: top must be 0 .. min(64, V)");
  OptTensor targets;
  if (targets_) {
    NSA_ASSERT(targets_->device() == logits.device(), "token_logprobs: targets on the logits' device");
    const auto tt = targets_->scalar_type();
    NSA_ASSERT(at::isIntegralType(tt, /*includeBool=*/false), "token_logprobs: targets must be integers");
    NSA_ASSERT(targets_->sizes() == lead, "token_logprobs: one target for each row");
    targets = targets_->reshape({-1}).to(at::kLong).contiguous();
  }
  const Tensor z = logits.dim() == 2 ? logits.contiguous() : logits.reshape({-1, V}).contiguous();
  LpOut o;
  if (at::GradMode::is_enabled() && logits.requires_grad()) {
    auto out = LogprobFn::apply(z, targets, top);
    size_t i = 0;
    if (targets) o.logp = out[i++];
    o.ent = out[i++];
    if (top > 0) {
      o.top_logp = out[i++];
      o.top_idx = out[i];
    }
  } else {
    o = logprob_forward(z, targets, top, false);
  }
  auto shaped = [&](const Tensor& t, bool wide) -> OptTensor {
    if (!t.defined()) return std::nullopt;
    if (lead.size() == 1) return t;
    std::vector<int64_t> sizes(lead.begin(), lead.end());
    if (wide) sizes.push_back(top);
    return t.view(sizes);
  };
  return {shaped(o.logp, false), *shaped(o.ent, false), shaped(o.top_logp, true), shaped(o.top_idx, true)};
}

// --- one new token over a paged cache -----------------------------------------
void check_pages(const Tensor& kp, const Tensor& vp, const Tensor& table, const Tensor& lens) {
  NSA_ASSERT(kp.dim() == 4 && kp.is_cuda(), "paged: pages must be [n_pages, Hkv, page, D] on the GPU");
  NSA_ASSERT(vp.sizes() == kp.sizes() && vp.scalar_type() == kp.scalar_type() && vp.device() == kp.device(),
             "paged: key and value pages differ in shape, dtype or device");
  const int64_t P = kp.size(2), D = kp.size(3);
  NSA_ASSERT(kp.size(0) >= 1 && kp.size(0) <= INT32_MAX && kp.size(1) >= 1 && P >= 16 && P % 16 == 0,
             "paged: the page size must be a multiple of 16");
  NSA_ASSERT(D == 16 || D == 32 || D == 64 || D == 128, "head dim must be a power of two <= 128");
  NSA_ASSERT(is_float(kp), std::string("dtype ") + c10::toString(kp.scalar_type()) +
                               " is not supported (float32 or bfloat16)");
  NSA_ASSERT(kp.is_contiguous() && vp.is_contiguous() && reinterpret_cast<uintptr_t>(kp.data_ptr()) % 16 == 0 &&
                 reinterpret_cast<uintptr_t>(vp.data_ptr()) % 16 == 0,
             "paged: pages must be dense and 16-byte aligned");
  NSA_ASSERT(table.dim() == 2 && table.scalar_type() == at::kInt && table.device() == kp.device(),
             "paged: table int32 [B, max_pages] on the pages' device");
  NSA_ASSERT(table.size(1) >= 1 && table.size(1) * P <= (1 << 30), "paged: table of 1 page to 2^30 positions");
  NSA_ASSERT(lens.scalar_type() == at::kInt && lens.dim() == 1 && lens.size(0) == table.size(0) &&
                 lens.device() == kp.device(),
             "paged: lens int32 [B] on the pages' device");
}

// -> (out, lse or None, new lengths or None)
std::tuple<Tensor, OptTensor, OptTensor> paged(const Tensor& q_, const OptTensor& k_new, const OptTensor& v_new,
                                               const Tensor& kp, const Tensor& vp, const Tensor& table_,
                                               const Tensor& lens_, std::optional<double> scale, bool want_lse,
                                               std::optional<int64_t> max_len) {
  NSA_ASSERT(k_new.has_value() == v_new.has_value(), "paged: a new key row needs its value row, and the other way round");
  no_tangent(has_tangent(q_) || has_tangent(k_new) || has_tangent(v_new) || has_tangent(kp) || has_tangent(vp),
             "paged attention");
  check_pages(kp, vp, table_, lens_);
  const int64_t n = kp.size(0), Hkv = kp.size(1), P = kp.size(2), D = kp.size(3), B = table_.size(0);
  const int64_t mp = table_.size(1);
  NSA_ASSERT(q_.dim() == 3 && q_.size(0) == B && q_.size(2) == D, "paged: q must be [B, Hq, D]");
  NSA_ASSERT(q_.scalar_type() == kp.scalar_type() && q_.device() == kp.device(),
             "paged: q in the pages' dtype and device");
  const int64_t Hq = q_.size(1);
  NSA_ASSERT(Hq >= 1 && Hq % Hkv == 0, "GQA needs n_q_heads divisible by n_kv_heads");
  NSA_ASSERT(Hq <= 4096 && B <= 65536, "paged: at most 4096 heads and 65536 sequences");
  if (at::GradMode::is_enabled())
    NSA_ASSERT(!q_.requires_grad() && !(k_new && (k_new->requires_grad() || v_new->requires_grad())) &&
                   !kp.requires_grad() && !vp.requires_grad(),
               "paged: attention over pages has no gradient: call it under torch.no_grad()");
  NSA_ASSERT(!max_len || *max_len >= 0, "paged: max_len must not be negative");
  const int end = max_len && *max_len < INT32_MAX ? (int)*max_len : INT32_MAX;
  const Tensor q = aligned(q_), table = table_.contiguous(), lens = lens_.contiguous();
  Tensor kn, vn, lens_out, lse;
  if (k_new) {
    for (const Tensor* r : {&*k_new, &*v_new})
      NSA_ASSERT(r->dim() == 3 && r->size(0) == B && r->size(1) == Hkv && r->size(2) == D &&
                     r->scalar_type() == kp.scalar_type() && r->device() == kp.device(),
                 "paged: new rows must be [B, Hkv, D] in the pages' dtype");
    kn = aligned(*k_new);
    vn = aligned(*v_new);
    lens_out = fresh({B}, lens, at::kInt);
  }
  Tensor out = fresh({B, Hq, D}, q, q.scalar_type());
  if (want_lse) lse = fresh({B, Hq}, q, at::kFloat);
  if (B > 0) {
    On on(q);
    const int code = code_of(q.scalar_type());
    const size_t bytes = p_nsa_paged_workspace((int)B, (int)Hq, (int)Hkv, (int)D, (int)P, (int)mp, code, on.stream);
    const Tensor ws = bytes > 16 ? fresh({(int64_t)bytes}, q, at::kByte) : Tensor();
    const double s = scale ? *scale : 1.0 / std::sqrt((double)D);
    check_status(p_nsa_paged_attend_max(q.data_ptr(), at_of(kn), at_of(vn), kp.data_ptr(), vp.data_ptr(),
                                    static_cast<const int32_t*>(table.data_ptr()),
                                    static_cast<const int32_t*>(lens.data_ptr()), at_as<int32_t>(lens_out),
                                    out.data_ptr(), at_as<float>(lse), at_of(ws), bytes, (int)B, (int)Hq, (int)Hkv,
                                    (int)D, (int)P, (int)mp, (int)n, end, (float)s, code, on.stream),
                 "nsa_paged_attend");
  }
  return {out, want_lse ? OptTensor(lse) : std::nullopt, k_new ? OptTensor(lens_out) : std::nullopt};
}

}  // namespace

PYBIND11_MODULE(_nsa_torch, m) {
  m.def("bind", &bind);
  m.def("add_rms_norm", &add_rms_norm);
  m.def("add_rms_norm_q8", &add_rms_norm_q8);
  m.def("token_logprobs", &token_logprobs);
  m.def("check_pages", &check_pages);
  m.def("no_tangent", [](const std::vector<Tensor>& ts, const std::string& what) {
    for (const Tensor& t : ts) no_tangent(has_tangent(t), what.c_str());
  });
  m.def("paged", &paged);
}
