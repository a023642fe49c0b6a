// Torch operators over the token-block entry points of lncc.h: allocation, strides, streams, and autograd.
//
// The operators' kernels take a few microseconds at small sizes, and a Python autograd function costs several times
// that: its backward pass alone waits for the interpreter on the engine's thread. So these are C++: checks, outputs and
// scratch from torch's allocator, the caller's current stream, and nodes that the engine runs without Python. For each
// operator there are fused_<name> (checks, and autograd where a gradient is wanted; eager Python calls it as a function of
// this module, which takes a microsecond less than a call through torch.ops), and <name> and <name>_backward, which
// torch.compile sees (their shapes for it are in fused_lncc/_native.py).
#include "lncc.h"

#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <ATen/record_function.h>
#include <c10/core/AutogradState.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/utils/pybind.h>
#include <torch/library.h>

namespace {

using at::Tensor;
using std::optional;
using torch::autograd::AutogradContext;
using torch::autograd::Variable;
using torch::autograd::variable_list;

int dtype_code(at::ScalarType t) {
  return t == at::kFloat ? LNCC_F32 : t == at::kBFloat16 ? LNCC_BF16 : t == at::kHalf ? LNCC_F16 : -1;
}
void check_tensor(const char* what, const char* name, const Tensor& t) {
  TORCH_CHECK(t.is_cuda(), "fused_lncc: ", what, ": ", name, " must be a CUDA tensor");
  TORCH_CHECK(dtype_code(t.scalar_type()) >= 0, "fused_lncc: ", what, ": float32, bfloat16 or float16 only, got ", name,
              " of ", t.scalar_type());
}
void check_like(const char* what, const char* name, const Tensor& t, const Tensor& x, bool same_type) {
  check_tensor(what, name, t);
  TORCH_CHECK(t.device() == x.device(), "fused_lncc: ", what, ": ", name, " must be on ", x.device(), ", got ", t.device());
  TORCH_CHECK(!same_type || t.scalar_type() == x.scalar_type(), "fused_lncc: ", what, ": ", name, " must be ",
              x.scalar_type(), ", got ", t.scalar_type());
}
void check_status(int status, const char* what) {
  TORCH_CHECK(status == LNCC_OK, "fused_lncc ", what, ": ", lncc_strerror(status), " (status ", status, ")");
}

std::string shape_of(const Tensor& t) {
  std::string s = "(";
  for (int64_t i = 0; i < t.dim(); i++) {
    const c10::SymInt n = t.sym_size(i);
    const auto known = n.maybe_as_int();
    s += (i ? ", " : "") + (known ? std::to_string(*known) : std::string("?"));
  }
  return s + ")";
}

c10::DispatchKeySet keys_of(const Tensor& t) { return t.defined() ? t.key_set() : c10::DispatchKeySet(); }
c10::DispatchKeySet keys_of(const optional<Tensor>& t) { return t ? keys_of(*t) : c10::DispatchKeySet(); }
// Whether a call on these tensors, all that it takes, may go straight to the function below, as it does in eager mode: nothing
// (tracing, functional, Python or negated tensors, a dispatch mode, a profiler) stands between it and the CUDA kernel. A call
// through the dispatcher costs a microsecond.
template <typename... Ts> bool straight(const Ts&... ts) {
  const c10::impl::LocalDispatchKeySet tls = c10::impl::tls_local_dispatch_key_set();
  const c10::DispatchKeySet keys = ((keys_of(ts) | ...) | tls.included_) - tls.excluded_ -
                                   c10::autograd_dispatch_keyset_with_ADInplaceOrView -
                                   c10::DispatchKeySet(c10::DispatchKey::BackendSelect);
  return keys.highestPriorityTypeId() == c10::DispatchKey::CUDA && !at::hasCallbacks();
}
// An operator as torch sees it, so that a compiled graph records the call.
template <typename F> auto op_of(const char* name, F*) {
  return c10::Dispatcher::singleton().findSchemaOrThrow(name, "").typed<F>();
}

// t (..., C) as (rows, C) with contiguous rows at one stride of at least C: a view where its strides allow it.
Tensor rows_of(const Tensor& t) {
  const int64_t c = t.size(-1);
  if (t.is_contiguous()) return t.dim() == 2 ? t : t.view({-1, c});
  if (t.dim() == 1) return t.contiguous().view({1, c});
  Tensor r = t;
  if (t.dim() != 2) {
    // leading axes that follow one another collapse into one
    int64_t stride = t.stride(-2), next = stride * t.size(-2);
    bool collapses = true;
    for (int64_t d = t.dim() - 3; d >= 0 && collapses; d--) {
      if (t.size(d) != 1) collapses = t.stride(d) == next;
      next *= t.size(d);
    }
    r = collapses ? t.as_strided({t.numel() / c, c}, {stride, t.stride(-1)}) : t.reshape({-1, c});
  }
  if (r.size(0) == 1 || (r.stride(1) == 1 && r.stride(0) >= c)) {
    if (r.stride(1) == 1 || c == 1) return r;
  }
  return r.contiguous();
}
// channels contiguous, other strides as they are
Tensor channels_last_axis(const Tensor& t) { return t.size(-1) == 1 || t.stride(-1) == 1 ? t : t.contiguous(); }
// The memory of t; null, which the entry points take as "not given", only where there is none to read or write.
const void* ptr(const Tensor& t) {
  if (!t.defined() || !t.numel()) return nullptr;
  const void* const p = t.const_data_ptr();
  TORCH_CHECK(p, "fused_lncc: a tensor without memory of its own (a subclass?) reached a kernel call");
  return p;
}
void* mut(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
// A call's scratch, from torch's allocator and on the current stream like a tensor's memory.
struct Scratch {
  c10::DataPtr at;
  explicit Scratch(size_t n) {
    if (n) at = c10::cuda::CUDACachingAllocator::get()->allocate(n);
  }
  void* get() const { return at.get(); }
};
Tensor new_tensor(at::IntArrayRef sizes, const at::TensorOptions& options) { return at::detail::empty_cuda(sizes, options); }
cudaStream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.device().index()).stream(); }
// The operators have no forward-mode derivative. Below the autograd keys a tangent would be lost, and torch takes a missing one
// for zero.
template <typename... Ts> void refuse_tangents(const char* what, const Ts&... ts) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  TORCH_CHECK_NOT_IMPLEMENTED(!((ts.defined() && ts._fw_grad(0).defined()) || ...), "fused_lncc: ", what,
                              ": forward-mode derivatives are not implemented");
}
bool wants_grad(const Tensor& t) { return t.defined() && t.requires_grad(); }
Tensor or_undefined(const optional<Tensor>& t) { return t.has_value() ? *t : Tensor(); }
optional<Tensor> or_none(const Tensor& t) { return t.defined() ? optional<Tensor>(t) : std::nullopt; }

// ---- layer norm -------------------------------------------------------------------------------------------------------
// y, and the statistics where they are wanted
Tensor norm_rows(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps, float* mean, float* rstd) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Tensor y = new_tensor(x.sizes(), x.options());
  if (rows) {
    const Tensor xr = rows_of(x);
    const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
    const at::ScalarType wt = weight ? weight->scalar_type() : bias ? bias->scalar_type() : x.scalar_type();
    check_status(lncc_layer_norm_forward(ptr(xr), xr.stride(0), ptr(w), ptr(b), dtype_code(x.scalar_type()), dtype_code(wt),
                                         rows, width, float(eps), mut(y), mean, rstd, stream_of(x)),
                 "layer_norm forward");
  }
  return y;
}
std::tuple<Tensor, Tensor, Tensor> layer_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                                              double eps, bool keep) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t rows = keep ? x.numel() / x.size(-1) : 0;
  const auto f32 = x.options().dtype(at::kFloat);
  const Tensor mean = new_tensor({rows}, f32), rstd = new_tensor({rows}, f32);
  const Tensor y = norm_rows(x, weight, bias, eps, static_cast<float*>(mut(mean)), static_cast<float*>(mut(rstd)));
  return {y, mean, rstd};
}

std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& dy, const Tensor& x, const optional<Tensor>& weight,
                                                       const Tensor& mean, const Tensor& rstd, at::ScalarType wdtype,
                                                       bool need_x, bool need_params) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t width = x.size(-1), rows = x.numel() / width;
  Tensor dx = need_x ? new_tensor(x.sizes(), x.options()) : new_tensor({0}, x.options());
  const auto params = x.options().dtype(wdtype);
  Tensor dw = new_tensor({need_params ? width : 0}, params), db = new_tensor({need_params ? width : 0}, params);
  const Tensor xr = rows ? rows_of(x) : x, dr = rows ? rows_of(dy) : dy, w = weight ? weight->contiguous() : Tensor();
  const size_t n = need_params ? lncc_layer_norm_scratch_bytes(rows, width) : 0;
  const Scratch ws(n);
  check_status(lncc_layer_norm_backward(ptr(dr), rows ? dr.stride(0) : width, ptr(xr), rows ? xr.stride(0) : width, ptr(w),
                                        dtype_code(x.scalar_type()), dtype_code(wdtype), rows, width,
                                        static_cast<const float*>(ptr(mean)), static_cast<const float*>(ptr(rstd)),
                                        need_x ? mut(dx) : nullptr, mut(dw), mut(db), ws.get(), n, stream_of(x)),
               "layer_norm backward");
  return {dx, dw, db};
}

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias,
                        double eps) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = op_of("fused_lncc::layer_norm", layer_norm);
    auto [y, mean, rstd] = straight(x, weight, bias) ? layer_norm(x, weight, bias, eps, true) : op.call(x, weight, bias, eps, true);
    ctx->save_for_backward({x, or_undefined(weight), mean, rstd});
    const optional<Tensor>& p = weight ? weight : bias;
    ctx->saved_data["wdtype"] = int64_t(p ? p->scalar_type() : x.scalar_type());
    ctx->saved_data["weight"] = weight.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = op_of("fused_lncc::layer_norm_backward", layer_norm_backward);
    const auto saved = ctx->get_saved_variables();
    // only tensors that were given have an edge
    const bool has_w = ctx->saved_data["weight"].toBool(), has_b = ctx->saved_data["bias"].toBool();
    const bool need_x = ctx->needs_input_grad(0), need_w = has_w && ctx->needs_input_grad(1),
               need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
    at::AutoDispatchBelowADInplaceOrView below;
    const auto wdtype = at::ScalarType(ctx->saved_data["wdtype"].toInt());
    auto [dx, dw, db] = straight(grads[0], saved[0], saved[1], saved[2], saved[3])
                            ? layer_norm_backward(grads[0], saved[0], or_none(saved[1]), saved[2], saved[3], wdtype, need_x, need_w || need_b)
                            : op.call(grads[0], saved[0], or_none(saved[1]), saved[2], saved[3], wdtype, need_x, need_w || need_b);
    return {need_x ? dx : Tensor(), need_w ? dw : Tensor(), need_b ? db : Tensor(), Tensor()};
  }
};

Tensor fused_layer_norm(const Tensor& x, const optional<Tensor>& weight, const optional<Tensor>& bias, double eps) {
  const char* what = "layer_norm";
  check_tensor(what, "x", x);
  TORCH_CHECK(x.dim() >= 1 && x.sym_size(-1) >= 1, "fused_lncc: layer_norm: expect x (..., C) with C >= 1");
  const Tensor w = or_undefined(weight), b = or_undefined(bias);
  const Tensor* const params[2] = {&w, &b};
  for (int i = 0; i < 2; i++) {
    const Tensor& p = *params[i];
    if (!p.defined()) continue;
    const char* name = i ? "bias" : "weight";
    check_like(what, name, p, x, false);
    TORCH_CHECK(p.scalar_type() == x.scalar_type() || p.scalar_type() == at::kFloat, "fused_lncc: layer_norm: ", name,
                " must be ", x.scalar_type(), " or Float, got ", p.scalar_type());
    TORCH_CHECK(p.dim() == 1 && p.sym_size(0) == x.sym_size(-1), "fused_lncc: layer_norm: ", name, " must have x's last size, got ",
                shape_of(p), " for x ", shape_of(x));
  }
  TORCH_CHECK(!w.defined() || !b.defined() || w.scalar_type() == b.scalar_type(),
              "fused_lncc: layer_norm: weight and bias must have one type");
  refuse_tangents(what, x, w, b);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w) || wants_grad(b)))
    return LayerNormNode::apply(x, weight, bias, eps);
  at::AutoDispatchBelowADInplaceOrView below;
  if (straight(x, weight, bias)) return norm_rows(x, weight, bias, eps, nullptr, nullptr);
  static const auto op = op_of("fused_lncc::layer_norm", layer_norm);
  return std::get<0>(op.call(x, weight, bias, eps, false));
}

// ---- gated scan -------------------------------------------------------------------------------------------------------
std::tuple<Tensor, Tensor, Tensor> gated_scan(const Tensor& x_, const Tensor& gate_, const optional<Tensor>& state,
                                              bool reverse, bool keep) {
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = channels_last_axis(x_), gate = channels_last_axis(gate_), s = state ? state->contiguous() : Tensor();
  const int64_t B = x.size(0), T = x.size(1), C = x.size(2);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor h = new_tensor({B, T, C}, x.options()), last = new_tensor({B, C}, f32);
  Tensor kept = new_tensor({keep ? int64_t(lncc_gated_scan_kept_bytes(B, T, C) / 4) : 0}, f32);
  const size_t n = lncc_gated_scan_scratch_bytes(B, T, C);
  const Scratch ws(n);
  check_status(lncc_gated_scan_forward(ptr(x), x.stride(0), x.stride(1), ptr(gate), gate.stride(0), gate.stride(1),
                                       static_cast<const float*>(ptr(s)), dtype_code(x.scalar_type()), B, T, C, reverse,
                                       mut(h), static_cast<float*>(mut(last)), static_cast<float*>(mut(kept)), ws.get(), n,
                                       stream_of(x)),
               "gated_scan forward");
  return {h, last, kept};
}

std::tuple<Tensor, Tensor, Tensor> gated_scan_backward(const Tensor& dh_, const optional<Tensor>& dlast, const Tensor& x_,
                                                       const Tensor& gate_, const Tensor& kept, bool reverse,
                                                       bool need_state) {
  const c10::cuda::CUDAGuard guard(x_.device());
  const Tensor x = channels_last_axis(x_), gate = channels_last_axis(gate_), dh = channels_last_axis(dh_);
  const Tensor dl = dlast ? dlast->contiguous() : Tensor();
  const int64_t B = x.size(0), T = x.size(1), C = x.size(2);
  const auto f32 = x.options().dtype(at::kFloat);
  Tensor dx = new_tensor({B, T, C}, x.options()), dgate = new_tensor({B, T, C}, x.options());
  Tensor dstate = need_state ? new_tensor({B, C}, f32) : new_tensor({0}, f32);
  const size_t n = lncc_gated_scan_scratch_bytes(B, T, C);
  const Scratch ws(n);
  check_status(lncc_gated_scan_backward(ptr(dh), dh.stride(0), dh.stride(1), static_cast<const float*>(ptr(dl)), ptr(x),
                                        x.stride(0), x.stride(1), ptr(gate), gate.stride(0), gate.stride(1),
                                        static_cast<const float*>(ptr(kept)), dtype_code(x.scalar_type()), B, T, C, reverse,
                                        mut(dx), mut(dgate), static_cast<float*>(mut(dstate)), ws.get(), n, stream_of(x)),
               "gated_scan backward");
  return {dx, dgate, dstate};
}

struct GatedScanNode : torch::autograd::Function<GatedScanNode> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const optional<Tensor>& state,
                               bool reverse) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = op_of("fused_lncc::gated_scan", gated_scan);
    auto [h, last, kept] = straight(x, gate, state) ? gated_scan(x, gate, state, reverse, true) : op.call(x, gate, state, reverse, true);
    ctx->save_for_backward({x, gate, kept});
    ctx->saved_data["reverse"] = reverse;
    ctx->saved_data["state"] = state.has_value();
    ctx->set_materialize_grads(false);
    return {h, last};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = op_of("fused_lncc::gated_scan_backward", gated_scan_backward);
    if (!grads[0].defined() && !grads[1].defined()) return {Tensor(), Tensor(), Tensor(), Tensor()};
    const auto saved = ctx->get_saved_variables();
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor dh = grads[0].defined() ? grads[0] : at::zeros_like(saved[0], at::MemoryFormat::Contiguous);
    const bool need_state = ctx->saved_data["state"].toBool() && ctx->needs_input_grad(2);  // edges of given tensors alone
    const bool reverse = ctx->saved_data["reverse"].toBool();
    auto [dx, dgate, dstate] = straight(dh, grads[1], saved[0], saved[1], saved[2])
                                   ? gated_scan_backward(dh, or_none(grads[1]), saved[0], saved[1], saved[2], reverse, need_state)
                                   : op.call(dh, or_none(grads[1]), saved[0], saved[1], saved[2], reverse, need_state);
    return {ctx->needs_input_grad(0) ? dx : Tensor(), ctx->needs_input_grad(1) ? dgate : Tensor(),
            need_state ? dstate : Tensor(), Tensor()};
  }
};

std::tuple<Tensor, Tensor> fused_gated_scan(const Tensor& x, const Tensor& gate, const optional<Tensor>& state_, bool reverse) {
  const char* what = "gated_scan";
  check_tensor(what, "x", x);
  TORCH_CHECK(x.dim() == 3 && x.sym_size(2) >= 1, "fused_lncc: gated_scan: expect x (B, T, C) with C >= 1, got ", shape_of(x));
  check_like(what, "gate", gate, x, true);
  TORCH_CHECK(gate.sym_sizes().equals(x.sym_sizes()), "fused_lncc: gated_scan: gate must be ", shape_of(x), ", got ", shape_of(gate));
  Tensor state = or_undefined(state_);
  if (state.defined()) {
    check_like(what, "state", state, x, false);
    TORCH_CHECK(state.dim() == 2 && state.sym_size(0) == x.sym_size(0) && state.sym_size(1) == x.sym_size(2),
                "fused_lncc: gated_scan: state must be (B, C), got ", shape_of(state), " for x ", shape_of(x));
    state = state.to(at::kFloat);
  }
  refuse_tangents(what, x, gate, state);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(gate) || wants_grad(state))) {
    const variable_list r = GatedScanNode::apply(x, gate, or_none(state), reverse);
    return {r[0], r[1]};
  }
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = op_of("fused_lncc::gated_scan", gated_scan);
  auto [h, last, kept] =
      straight(x, gate, state) ? gated_scan(x, gate, or_none(state), reverse, false) : op.call(x, gate, or_none(state), reverse, false);
  return {h, last};
}

// ---- gated feed-forward -----------------------------------------------------------------------------------------------
Tensor gated_ffn(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, int64_t act) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t F = w_gate.size(0), K = w_gate.size(1), N = w_down.size(0), M = x.numel() / K;
  auto shape = x.sizes().vec();
  shape.back() = N;
  Tensor y = new_tensor(shape, x.options());
  if (!M) return y;
  const Tensor xr = rows_of(x), wg = w_gate.contiguous(), wu = w_up.contiguous(), wd = w_down.contiguous();
  const int dt = dtype_code(x.scalar_type());
  const size_t n = lncc_gated_ffn_scratch_bytes(M, K, F, N, dt, 0);
  const Scratch ws(n);
  check_status(lncc_gated_ffn_forward(ptr(xr), xr.stride(0), ptr(wg), ptr(wu), ptr(wd), dt, int(act), M, K, F, N, mut(y),
                                      ws.get(), n, stream_of(x)),
               "gated_ffn forward");
  return y;
}

std::tuple<Tensor, Tensor, Tensor, Tensor> gated_ffn_backward(const Tensor& dy, const Tensor& x, const Tensor& w_gate,
                                                              const Tensor& w_up, const Tensor& w_down, int64_t act,
                                                              bool need_x, bool need_gate, bool need_up, bool need_down) {
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t F = w_gate.size(0), K = w_gate.size(1), N = w_down.size(0), M = x.numel() / K;
  const auto out = [&](bool need, const Tensor& of) {
    return need ? new_tensor(of.sizes(), x.options()) : new_tensor({0}, x.options());
  };
  Tensor dx = out(need_x, x), dwg = out(need_gate, w_gate), dwu = out(need_up, w_up), dwd = out(need_down, w_down);
  const Tensor xr = M ? rows_of(x) : x, dr = M ? rows_of(dy) : dy;
  const Tensor wg = w_gate.contiguous(), wu = w_up.contiguous(), wd = w_down.contiguous();
  const int dt = dtype_code(x.scalar_type());
  const size_t n = M ? lncc_gated_ffn_scratch_bytes(M, K, F, N, dt, 1) : 0;
  const Scratch ws(n);
  check_status(lncc_gated_ffn_backward(ptr(dr), M ? dr.stride(0) : N, ptr(xr), M ? xr.stride(0) : K, ptr(wg), ptr(wu), ptr(wd),
                                       dt, int(act), M, K, F, N, need_x ? mut(dx) : nullptr, need_gate ? mut(dwg) : nullptr,
                                       need_up ? mut(dwu) : nullptr, need_down ? mut(dwd) : nullptr, ws.get(), n, stream_of(x)),
               "gated_ffn backward");
  return {dx, dwg, dwu, dwd};
}

struct GatedFFNNode : torch::autograd::Function<GatedFFNNode> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down,
                        int64_t act) {
    at::AutoDispatchBelowADInplaceOrView below;
    static const auto op = op_of("fused_lncc::gated_ffn", gated_ffn);
    ctx->save_for_backward({x, w_gate, w_up, w_down});
    ctx->saved_data["act"] = act;
    return straight(x, w_gate, w_up, w_down) ? gated_ffn(x, w_gate, w_up, w_down, act) : op.call(x, w_gate, w_up, w_down, act);
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    static const auto op = op_of("fused_lncc::gated_ffn_backward", gated_ffn_backward);
    const auto saved = ctx->get_saved_variables();
    bool need[4];
    for (int i = 0; i < 4; i++) need[i] = ctx->needs_input_grad(i);
    at::AutoDispatchBelowADInplaceOrView below;
    const int64_t act = ctx->saved_data["act"].toInt();
    auto [dx, dwg, dwu, dwd] =
        straight(grads[0], saved[0], saved[1], saved[2], saved[3])
            ? gated_ffn_backward(grads[0], saved[0], saved[1], saved[2], saved[3], act, need[0], need[1], need[2], need[3])
            : op.call(grads[0], saved[0], saved[1], saved[2], saved[3], act, need[0], need[1], need[2], need[3]);
    return {need[0] ? dx : Tensor(), need[1] ? dwg : Tensor(), need[2] ? dwu : Tensor(), need[3] ? dwd : Tensor(), Tensor()};
  }
};

Tensor fused_gated_ffn(const Tensor& x, const Tensor& w_gate, const Tensor& w_up, const Tensor& w_down, int64_t act) {
  const char* what = "gated_ffn";
  check_tensor(what, "x", x);
  const Tensor* const weights[3] = {&w_gate, &w_up, &w_down};
  const char* const names[3] = {"w_gate", "w_up", "w_down"};
  for (int i = 0; i < 3; i++) {
    check_like(what, names[i], *weights[i], x, true);
    TORCH_CHECK(weights[i]->dim() == 2 && weights[i]->sym_numel() > 0, "fused_lncc: gated_ffn: ", names[i],
                " must be a matrix, got ", shape_of(*weights[i]));
  }
  TORCH_CHECK(x.dim() >= 1 && x.sym_size(-1) == w_gate.sym_size(1) && w_up.sym_sizes().equals(w_gate.sym_sizes()) &&
                  w_down.sym_size(1) == w_gate.sym_size(0),
              "fused_lncc: gated_ffn: expect x (..., K), w_gate and w_up (F, K), w_down (N, F), got ", shape_of(x), ", ",
              shape_of(w_gate), ", ", shape_of(w_up), ", ", shape_of(w_down));
  refuse_tangents(what, x, w_gate, w_up, w_down);
  if (at::GradMode::is_enabled() && (wants_grad(x) || wants_grad(w_gate) || wants_grad(w_up) || wants_grad(w_down)))
    return GatedFFNNode::apply(x, w_gate, w_up, w_down, act);
  at::AutoDispatchBelowADInplaceOrView below;
  static const auto op = op_of("fused_lncc::gated_ffn", gated_ffn);
  return straight(x, w_gate, w_up, w_down) ? gated_ffn(x, w_gate, w_up, w_down, act) : op.call(x, w_gate, w_up, w_down, act);
}

}  // namespace

TORCH_LIBRARY_FRAGMENT(fused_lncc, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, bool keep) -> (Tensor, Tensor, Tensor)");
  m.def("layer_norm_backward(Tensor dy, Tensor x, Tensor? weight, Tensor mean, Tensor rstd, ScalarType wdtype, bool need_x, "
        "bool need_params) -> (Tensor, Tensor, Tensor)");
  m.def("gated_scan(Tensor x, Tensor gate, Tensor? state, bool reverse, bool keep) -> (Tensor, Tensor, Tensor)");
  m.def("gated_scan_backward(Tensor dh, Tensor? dlast, Tensor x, Tensor gate, Tensor kept, bool reverse, bool need_state) -> "
        "(Tensor, Tensor, Tensor)");
  m.def("gated_ffn(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int act) -> Tensor");
  m.def("gated_ffn_backward(Tensor dy, Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int act, bool need_x, bool "
        "need_gate, bool need_up, bool need_down) -> (Tensor, Tensor, Tensor, Tensor)");
  m.def("fused_layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps) -> Tensor", fused_layer_norm);
  m.def("fused_gated_scan(Tensor x, Tensor gate, Tensor? state, bool reverse) -> (Tensor, Tensor)", fused_gated_scan);
  m.def("fused_gated_ffn(Tensor x, Tensor w_gate, Tensor w_up, Tensor w_down, int act) -> Tensor", fused_gated_ffn);
}
TORCH_LIBRARY_IMPL(fused_lncc, CUDA, m) {
  m.impl("layer_norm", layer_norm);
  m.impl("layer_norm_backward", layer_norm_backward);
  m.impl("gated_scan", gated_scan);
  m.impl("gated_scan_backward", gated_scan_backward);
  m.impl("gated_ffn", gated_ffn);
  m.impl("gated_ffn_backward", gated_ffn_backward);
}

PYBIND11_MODULE(libfused_lncc_torch, m) {
  const auto no_gil = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.def("layer_norm", fused_layer_norm, no_gil);
  m.def("gated_scan", fused_gated_scan, no_gil);
  m.def("gated_ffn", fused_gated_ffn, no_gil);
}
