// The torch side of rms_norm, linear and gated_linear: what a call of layers.* does on the host besides the launch, in C++.
//
// A decoding step calls these operators a few times a layer with kernels of a few microseconds, and a small training step's
// gradients come back through autograd's device thread: there the host bounds the call. Argument checks, output
// allocation and autograd nodes in Python cost 14 us a call of rms_norm, and 110 us with its gradients; here they cost 5 and 65, of
// which 40 are autograd's own hand-over between threads.
//
// The kernels are reached through the C ABI (include/jla_b200.h) of the library that the Python side has loaded: bind() gets
// the addresses of its entry points. A call that these functions do not take comes back as None, and the Python side
// says what is wrong with it.
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <string>
#include <unordered_set>
#include <vector>

#include "../../include/jla_b200.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

constexpr at::ScalarType kNone = at::ScalarType::Undefined;  // "no dtype asked for"

struct Abi {
  decltype(&jla_last_error) last_error;
  decltype(&jla_rms_norm_fwd) rms_norm_fwd;
  decltype(&jla_rms_norm_bwd_scratch_bytes) rms_norm_bwd_scratch_bytes;
  decltype(&jla_rms_norm_bwd) rms_norm_bwd;
  decltype(&jla_linear_fwd) linear_fwd;
  decltype(&jla_gated_linear_fwd) gated_linear_fwd;
  decltype(&jla_activation_bwd_scratch_bytes) activation_bwd_scratch_bytes;
  decltype(&jla_activation_bwd) activation_bwd;
  decltype(&jla_gated_activation_bwd) gated_activation_bwd;
  decltype(&jla_linear_bwd_input) linear_bwd_input;
  decltype(&jla_linear_bwd_weight) linear_bwd_weight;
} abi;

void bind(const py::dict& addresses) {
  auto at = [&](const char* name) { return reinterpret_cast<void*>(addresses[name].cast<uintptr_t>()); };
#define JLA_BIND(name) abi.name = reinterpret_cast<decltype(abi.name)>(at("jla_" #name))
  JLA_BIND(last_error);
  JLA_BIND(rms_norm_fwd);
  JLA_BIND(rms_norm_bwd_scratch_bytes);
  JLA_BIND(rms_norm_bwd);
  JLA_BIND(linear_fwd);
  JLA_BIND(gated_linear_fwd);
  JLA_BIND(activation_bwd_scratch_bytes);
  JLA_BIND(activation_bwd);
  JLA_BIND(gated_activation_bwd);
  JLA_BIND(linear_bwd_input);
  JLA_BIND(linear_bwd_weight);
#undef JLA_BIND
}

void check(int rc, const char* what) {
  if (rc == JLA_OK) return;
  const std::string text = std::string(what) + ": " + abi.last_error();
  TORCH_CHECK_NOT_IMPLEMENTED(rc != JLA_ERR_UNSUPPORTED, text);
  TORCH_CHECK_VALUE(rc != JLA_ERR_BAD_ARGUMENT && rc != JLA_ERR_WORKSPACE, text);
  TORCH_CHECK(false, text, " (status ", rc, ")");
}

int code(at::ScalarType t) {
  switch (t) {
    case at::kBFloat16: return JLA_DTYPE_BF16;
    case at::kHalf: return JLA_DTYPE_F16;
    case at::kFloat: return JLA_DTYPE_F32;
    case at::kFloat8_e4m3fn: return JLA_DTYPE_E4M3;
    default: return -1;
  }
}
bool sixteen(at::ScalarType t) { return t == at::kBFloat16 || t == at::kHalf; }

void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
const float* fptr(const Tensor& t) { return static_cast<const float*>(ptr(t)); }
float* fmut(const Tensor& t) { return static_cast<float*>(ptr(t)); }
jla_stream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }

// Contiguous, no lazily negated view, and on a 16-byte boundary (a slice of another tensor may start anywhere).
Tensor aligned(const Tensor& t) {
  if (!t.defined()) return t;
  Tensor c = t.contiguous().resolve_neg();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) & 15 ? c.clone() : c;
}

// x [..., width] as rows that start `stride` elements apart, without a copy where they allow 16-byte loads.
struct Rows {
  Tensor t;
  int64_t rows, stride;
};
Rows rows_of(const Tensor& x, int64_t width) {
  const int64_t rows = x.numel() / width, last = x.dim() - 1;
  if (!x.is_contiguous() && x.stride(last) == 1 && !x.is_neg()) {
    int64_t stride = -1, next = 0;
    bool even = true;
    for (int64_t i = last - 1; i >= 0 && even; --i) {
      if (x.size(i) == 1) continue;
      if (stride < 0) stride = x.stride(i), next = stride * x.size(i);
      else if (x.stride(i) == next) next *= x.size(i);
      else even = false;
    }
    if (stride < 0) stride = width;
    if (even && stride >= width && !((stride * x.element_size() | reinterpret_cast<intptr_t>(x.data_ptr())) & 15)) {
      return {x, rows, stride};
    }
  }
  return {aligned(x), rows, width};
}

// Whether a gradient would be recorded, of any order or mode, for a call with these tensors.
bool differentiated(std::initializer_list<const Tensor*> tensors) {
  for (const Tensor* t : tensors) {
    if (!t->defined()) continue;
    if (t->requires_grad() && at::GradMode::is_enabled()) return true;
    if (t->_fw_grad(0).defined()) return true;
  }
  return false;
}

// Gradients that cannot be differentiated again: an attempt raises, as torch's once_differentiable does.
variable_list once(variable_list grads) {
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    auto error = std::make_shared<torch::autograd::DelayedError>("the gradients of this operator cannot be differentiated again", 1);
    g = (*error)(variable_list{g.detach().requires_grad_(true)})[0];
  }
  return grads;
}

// A saved tensor as a backward pass gets it. Saved-tensor hooks (offloading, compression) may hand back another tensor than
// the one that was saved: its strides and its alignment count for nothing here, and what else differs is refused, since the
// kernels would read outside of it or read it wrongly.
Tensor restored(const Tensor& t, at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  TORCH_CHECK_VALUE(t.defined() && t.layout() == at::kStrided && t.sizes() == shape && t.scalar_type() == type &&
                        t.device() == like.device(),
                    "a saved tensor came back from its hook with another shape, dtype or device");
  return t;
}

// Called by a node's backward pass. Autograd hands a gradient over on the stream of the node that takes it. Where that is the
// default stream, which takes no part in a capture, the hand-over breaks the capture: a leaf's node, while an eager graph of the
// leaf lives, or a node of this graph that was made before the capture. So all nodes are looked at that this one's gradients go
// to, directly or by way of others (a cast of a bias, a transposed or padded weight). Only a captured pass pays for it.
void refuse_broken_capture() {
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto node = torch::autograd::get_current_node();
  if (!node) return;
  std::vector<torch::autograd::Node*> open{node.get()};
  std::unordered_set<torch::autograd::Node*> seen{node.get()};
  while (!open.empty()) {
    torch::autograd::Node* from = open.back();
    open.pop_back();
    for (size_t i = 0; i < from->num_outputs(); ++i) {
      torch::autograd::Node* next = from->next_edge(i).function.get();
      if (!next || !from->task_should_compute_output(i) || !seen.insert(next).second) continue;
      const auto stream = next->stream();
      TORCH_CHECK(!stream || c10::cuda::CUDAStream(*stream) != c10::cuda::getDefaultCUDAStream(stream->device_index()),
                  "an eager autograd graph of one of these leaves is alive on the default stream, or a part of this graph was made "
                  "there: drop its outputs before the backward pass is captured, and make the whole graph in the capture");
      open.push_back(next);
    }
  }
}

// A tensor, None (undefined) or something else (false).
bool take(const py::handle& h, Tensor& t) {
  if (h.is_none()) return true;
  if (!THPVariable_Check(h.ptr())) return false;
  t = THPVariable_Unpack(h.ptr());
  return true;
}
// None or a torch.dtype.
bool take_dtype(const py::handle& h, at::ScalarType& t) {
  if (h.is_none()) return true;
  if (!THPDtype_Check(h.ptr())) return false;
  t = reinterpret_cast<THPDtype*>(h.ptr())->scalar_type;
  return true;
}
bool on(const Tensor& t, const Tensor& like) { return t.is_cuda() && t.get_device() == like.get_device(); }

// (a node's inputs that are not there are left out of its edges: needs_input_grad counts the others only)
std::optional<Tensor> maybe(const Tensor& t) { return t.defined() ? std::optional<Tensor>(t) : std::nullopt; }

Tensor make(at::IntArrayRef shape, at::ScalarType type, const Tensor& like) {
  return at::empty(shape, like.options().dtype(type).requires_grad(false));
}

// ---- rms_norm -----------------------------------------------------------------------------------------------------------

struct Norm {
  Tensor y, stream, rstd, scale;
};

Norm norm_fwd(const Tensor& x, const Tensor& residual, const Tensor& weight, double eps, bool e4m3, bool keep) {
  c10::cuda::OptionalCUDAGuard guard(x.device());
  Norm n;
  const int64_t dim = x.size(-1), rows = x.numel() / dim;
  n.y = make(x.sizes(), e4m3 ? at::kFloat8_e4m3fn : x.scalar_type(), x);
  if (residual.defined()) n.stream = make(x.sizes(), x.scalar_type(), x);
  if (keep) n.rstd = make({rows}, at::kFloat, x);
  if (e4m3) n.scale = make(x.sizes().slice(0, x.dim() - 1), at::kFloat, x);
  check(abi.rms_norm_fwd(code(x.scalar_type()), rows, (int)dim, ptr(x), ptr(residual), fptr(weight), (float)eps, e4m3, ptr(n.y),
                         ptr(n.stream), fmut(n.rstd), fmut(n.scale), stream_of(x)),
        "jla_rms_norm_fwd");
  return n;
}

struct RmsNorm : torch::autograd::Function<RmsNorm> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& residual_,
                               double eps) {
    const Tensor residual = residual_.value_or(Tensor());
    Norm n = norm_fwd(x, residual, weight, eps, false, true);
    ctx->save_for_backward({x, residual, weight, n.rstd});
    ctx->saved_data["residual"] = residual.defined();
    ctx->set_materialize_grads(false);
    if (!residual.defined()) return {n.y};
    if (!x.requires_grad() && !residual.requires_grad()) ctx->mark_non_differentiable({n.stream});  // the weight is not in it
    return {n.y, n.stream};
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_broken_capture();
    const bool again = at::GradMode::is_enabled();
    variable_list out;
    {
      at::AutoGradMode off(false);
      const variable_list saved = ctx->get_saved_variables();
      const bool has_residual = ctx->saved_data["residual"].toBool();
      Tensor dx, dw, dy = grads[0], ds = grads.size() > 1 ? grads[1] : Tensor();
      if (!dy.defined()) {
        dx = ds;  // only the stream was used
      } else {
        c10::cuda::OptionalCUDAGuard guard(dy.device());
        dy = aligned(dy), ds = aligned(ds);
        const int64_t dim = dy.size(-1), rows = dy.numel() / dim;
        const Tensor x = aligned(restored(saved[0], dy.sizes(), dy.scalar_type(), dy));
        const Tensor residual = has_residual ? aligned(restored(saved[1], dy.sizes(), dy.scalar_type(), dy)) : Tensor();
        const Tensor weight = aligned(restored(saved[2], {dim}, at::kFloat, dy));
        const Tensor rstd = aligned(restored(saved[3], {rows}, at::kFloat, dy));
        dx = make(x.sizes(), x.scalar_type(), x);
        Tensor scratch;
        size_t bytes = 0;
        if (ctx->needs_input_grad(1)) {
          dw = make({dim}, at::kFloat, x);
          bytes = abi.rms_norm_bwd_scratch_bytes(rows, (int)dim);
          scratch = make({(int64_t)bytes}, at::kByte, x);
        }
        check(abi.rms_norm_bwd(code(x.scalar_type()), rows, (int)dim, ptr(x), ptr(residual), fptr(rstd), fptr(weight), ptr(dy),
                               ptr(ds), ptr(dx), fmut(dw), ptr(scratch), bytes, stream_of(x)),
              "jla_rms_norm_bwd");
      }
      out = {dx, dw, has_residual ? dx : Tensor(), Tensor()};
    }
    return again ? once(out) : out;
  }
};

// y, (y, stream), (q, scale) or (q, scale, stream); None for a call that the Python side has to refuse.
py::object rms_norm(const py::handle& x_, const py::handle& weight_, const py::handle& residual_, double eps,
                    const py::handle& dtype_) {
  Tensor x, weight, residual;
  at::ScalarType out = kNone;
  if (!take(x_, x) || !take(weight_, weight) || !take(residual_, residual) || !take_dtype(dtype_, out)) return py::none();
  if (!x.defined() || !weight.defined() || !x.is_cuda() || x.dim() < 1) return py::none();
  const int64_t dim = x.size(-1);
  const at::ScalarType type = x.scalar_type();
  if (dim < 1 || dim > 16384 || code(type) < 0 || code(type) == JLA_DTYPE_E4M3 || weight.dim() != 1 || weight.size(0) != dim ||
      !on(weight, x) || !weight.is_floating_point()) {
    return py::none();
  }
  if (residual.defined() && (residual.scalar_type() != type || !on(residual, x) || residual.sizes() != x.sizes())) return py::none();
  const bool e4m3 = out == at::kFloat8_e4m3fn, grads = differentiated({&x, &weight, &residual});
  if ((out != kNone && !e4m3 && out != type) || (e4m3 && grads)) return py::none();
  variable_list made;
  {
    py::gil_scoped_release unlocked;
    x = aligned(x), residual = aligned(residual);
    weight = aligned(weight.scalar_type() == at::kFloat ? weight : weight.to(at::kFloat));
    if (grads) {
      made = RmsNorm::apply(x, weight, maybe(residual), eps);
    } else {
      Norm n = norm_fwd(x, residual, weight, eps, e4m3, false);
      made.push_back(n.y);
      if (e4m3) made.push_back(n.scale);
      if (n.stream.defined()) made.push_back(n.stream);
    }
  }
  if (made.size() == 1) return py::cast(made[0]);
  if (made.size() == 2) return py::make_tuple(made[0], made[1]);
  return py::make_tuple(made[0], made[1], made[2]);
}

// ---- linear and gated_linear ------------------------------------------------------------------------------------------------

std::vector<int64_t> out_shape(const Tensor& x, int64_t out) {
  std::vector<int64_t> s(x.sizes().begin(), x.sizes().end());
  s.back() = out;
  return s;
}

Tensor linear_fwd(const Rows& x, const Tensor& weight, const Tensor& x_scale, const Tensor& w_scale, const Tensor& bias, int64_t act,
                  const Tensor& residual, at::IntArrayRef shape, at::ScalarType type, Tensor* z) {
  c10::cuda::OptionalCUDAGuard guard(weight.device());
  Tensor y = make(shape, type, weight);
  if (z) *z = make({x.rows, weight.size(0)}, at::kFloat, weight);
  check(abi.linear_fwd(code(weight.scalar_type()), code(type), x.rows, (int)weight.size(1), (int)weight.size(0), ptr(x.t), x.stride,
                       ptr(weight), fptr(x_scale), fptr(w_scale), fptr(bias), (int)act, ptr(residual), ptr(y), z ? fmut(*z) : nullptr,
                       stream_of(weight)),
        "jla_linear_fwd");
  return y;
}

Tensor gated_fwd(const Rows& x, const Tensor& gate, const Tensor& up, const Tensor& x_scale, const Tensor& g_scale,
                 const Tensor& u_scale, int64_t act, at::IntArrayRef shape, at::ScalarType type, Tensor* g, Tensor* u) {
  c10::cuda::OptionalCUDAGuard guard(gate.device());
  Tensor h = make(shape, type, gate);
  if (g) *g = make({x.rows, gate.size(0)}, at::kFloat, gate), *u = make({x.rows, gate.size(0)}, at::kFloat, gate);
  check(abi.gated_linear_fwd(code(gate.scalar_type()), code(type), x.rows, (int)gate.size(1), (int)gate.size(0), ptr(x.t), x.stride,
                             ptr(gate), ptr(up), fptr(x_scale), fptr(g_scale), fptr(u_scale), (int)act, ptr(h),
                             g ? fmut(*g) : nullptr, g ? fmut(*u) : nullptr, stream_of(gate)),
        "jla_gated_linear_fwd");
  return h;
}

Tensor input_grad(at::IntArrayRef shape, int64_t rows, const Tensor& dz, const Tensor& w, const Tensor& dz2, const Tensor& w2) {
  Tensor dx = make(shape, w.scalar_type(), w);
  check(abi.linear_bwd_input(code(w.scalar_type()), rows, (int)w.size(1), (int)w.size(0), ptr(dz), ptr(w), ptr(dz2), ptr(w2), ptr(dx),
                             stream_of(w)),
        "jla_linear_bwd_input");
  return dx;
}

// dw [out, in] of dz, and dw2 of dz2 in the same launch where there is one
void weight_grads(const Rows& x, const Tensor& dz, int64_t out, Tensor& dw, const Tensor& dz2, Tensor* dw2) {
  const int64_t in = x.t.size(-1);
  dw = make({out, in}, dz.scalar_type(), dz);
  if (dw2) *dw2 = make({out, in}, dz.scalar_type(), dz);
  check(abi.linear_bwd_weight(code(dz.scalar_type()), x.rows, (int)in, (int)out, ptr(dz), ptr(dz2), ptr(x.t), x.stride, ptr(dw),
                              dw2 ? ptr(*dw2) : nullptr, stream_of(dz)),
        "jla_linear_bwd_weight");
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const std::optional<Tensor>& bias_,
                        const std::optional<Tensor>& residual_, int64_t act) {
    const Tensor bias = bias_.value_or(Tensor()), residual = residual_.value_or(Tensor());
    const Rows rows = rows_of(x, weight.size(1));
    const bool keep_z = act != JLA_ACT_NONE && (x.requires_grad() || weight.requires_grad() || (bias.defined() && bias.requires_grad()));
    Tensor z;
    Tensor y = linear_fwd(rows, weight, {}, {}, bias, act, aligned(residual), out_shape(x, weight.size(0)), x.scalar_type(),
                          keep_z ? &z : nullptr);
    // what the gradients that are wanted read, and nothing else: a frozen weight keeps no x alive
    ctx->save_for_backward({weight.requires_grad() ? rows.t : Tensor(), x.requires_grad() ? weight : Tensor(), z});
    ctx->saved_data["cfg"] = std::vector<int64_t>{act, bias.defined(), residual.defined()};
    ctx->saved_data["shape"] = x.sizes().vec();
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_broken_capture();
    const bool again = at::GradMode::is_enabled();
    variable_list out;
    {
      at::AutoGradMode off(false);
      const variable_list saved = ctx->get_saved_variables();
      const std::vector<int64_t> cfg = ctx->saved_data["cfg"].toIntVector(), shape = ctx->saved_data["shape"].toIntVector();
      const int64_t act = cfg[0];
      const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_b = cfg[1] && ctx->needs_input_grad(2);
      c10::cuda::OptionalCUDAGuard guard(grads[0].device());
      const Tensor dy = aligned(grads[0]);
      const int64_t depth = shape.back(), n = dy.size(-1), rows = dy.numel() / n;
      Tensor z, dz = dy, db, dx, dw;
      if (act != JLA_ACT_NONE && (need_x || need_w || need_b)) z = aligned(restored(saved[2], {rows, n}, at::kFloat, dy));
      if (need_b || z.defined()) {
        if (z.defined()) dz = make({rows, n}, dy.scalar_type(), dy);
        Tensor scratch;
        size_t bytes = 0;
        if (need_b) {
          bytes = abi.activation_bwd_scratch_bytes(rows, (int)n);
          db = make({n}, at::kFloat, dy);
          scratch = make({(int64_t)bytes}, at::kByte, dy);
        }
        check(abi.activation_bwd(code(dy.scalar_type()), rows, (int)n, (int)act, fptr(z), ptr(dy), z.defined() ? ptr(dz) : nullptr,
                                 fmut(db), ptr(scratch), bytes, stream_of(dy)),
              "jla_activation_bwd");
      }
      if (need_x) dx = input_grad(shape, rows, dz, aligned(restored(saved[1], {n, depth}, dy.scalar_type(), dy)), {}, {});
      if (need_w) weight_grads(rows_of(restored(saved[0], shape, dy.scalar_type(), dy), depth), dz, n, dw, {}, nullptr);
      out = {dx, dw, db, cfg[2] && ctx->needs_input_grad(cfg[1] ? 3 : 2) ? grads[0] : Tensor(), Tensor()};
    }
    return again ? once(out) : out;
  }
};

struct GatedLinear : torch::autograd::Function<GatedLinear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate, const Tensor& up, int64_t act) {
    const Rows rows = rows_of(x, gate.size(1));
    Tensor g, u;
    Tensor h = gated_fwd(rows, gate, up, {}, {}, {}, act, out_shape(x, gate.size(0)), x.scalar_type(), &g, &u);
    const bool x_too = gate.requires_grad() || up.requires_grad(), weights_too = x.requires_grad();
    ctx->save_for_backward({x_too ? rows.t : Tensor(), weights_too ? gate : Tensor(), weights_too ? up : Tensor(), g, u});
    ctx->saved_data["act"] = act;
    ctx->saved_data["shape"] = x.sizes().vec();
    return h;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    refuse_broken_capture();
    const bool again = at::GradMode::is_enabled();
    variable_list out;
    {
      at::AutoGradMode off(false);
      const variable_list saved = ctx->get_saved_variables();
      const std::vector<int64_t> shape = ctx->saved_data["shape"].toIntVector();
      const int64_t act = ctx->saved_data["act"].toInt();
      c10::cuda::OptionalCUDAGuard guard(grads[0].device());
      const Tensor dh = aligned(grads[0]);
      const int64_t depth = shape.back(), n = dh.size(-1), rows = dh.numel() / n;
      const Tensor g = aligned(restored(saved[3], {rows, n}, at::kFloat, dh));
      const Tensor u = aligned(restored(saved[4], {rows, n}, at::kFloat, dh));
      const Tensor dg = make({rows, n}, dh.scalar_type(), dh), du = make({rows, n}, dh.scalar_type(), dh);
      check(abi.gated_activation_bwd(code(dh.scalar_type()), rows, (int)n, (int)act, fptr(g), fptr(u), ptr(dh), ptr(dg), ptr(du),
                                     stream_of(dh)),
            "jla_gated_activation_bwd");
      Tensor dx, d_gate, d_up;
      const bool need_g = ctx->needs_input_grad(1), need_u = ctx->needs_input_grad(2);
      if (ctx->needs_input_grad(0)) {
        const Tensor gate = aligned(restored(saved[1], {n, depth}, dh.scalar_type(), dh));
        dx = input_grad(shape, rows, dg, gate, du, aligned(restored(saved[2], {n, depth}, dh.scalar_type(), dh)));
      }
      if (need_g || need_u) {
        const Rows x = rows_of(restored(saved[0], shape, dh.scalar_type(), dh), depth);
        if (need_g) weight_grads(x, dg, n, d_gate, need_u ? du : Tensor(), need_u ? &d_up : nullptr);
        else weight_grads(x, du, n, d_up, {}, nullptr);
      }
      out = {dx, d_gate, d_up, Tensor()};
    }
    return again ? once(out) : out;
  }
};

// Widths that the kernels do not take as they are: zeros to the next multiple, in copies that autograd sees through.
struct Padding {
  int64_t out, more_in, more_out;
  Padding(const Tensor& w) {
    const int64_t step = w.scalar_type() == at::kFloat8_e4m3fn ? 16 : 8;
    out = w.size(0), more_in = (step - w.size(1) % step) % step, more_out = (8 - out % 8) % 8;
  }
  bool needed() const { return more_in || more_out; }
  static Tensor wider(const Tensor& t, int64_t cols, int64_t rows = 0) {
    if (!t.defined() || (!cols && !rows)) return t;
    const std::vector<int64_t> by = rows ? std::vector<int64_t>{0, cols, 0, rows} : std::vector<int64_t>{0, cols};
    if (t.scalar_type() != at::kFloat8_e4m3fn) return at::constant_pad_nd(t, by, 0);
    return at::constant_pad_nd(t.view(at::kByte), by, 0).view(at::kFloat8_e4m3fn);
  }
  Tensor cut(const Tensor& y) const { return more_out ? y.narrow(-1, 0, out).contiguous() : y; }
};

// The checks that both products share; `type` becomes the output's dtype.
bool operands(const Tensor& x, const Tensor& w, const Tensor& x_scale, std::initializer_list<const Tensor*> scales,
              const py::handle& dtype_, at::ScalarType& type) {
  if (!x.defined() || !w.defined() || !x.is_cuda() || !on(w, x) || x.dim() < 1 || w.dim() != 2) return false;
  const at::ScalarType t = x.scalar_type();
  const int64_t out = w.size(0), depth = w.size(1);
  if (w.scalar_type() != t || x.size(-1) != depth || depth < 1 || out < 1 || depth > (1 << 24) || out > (1 << 24)) return false;
  type = kNone;
  if (!take_dtype(dtype_, type)) return false;
  if (t != at::kFloat8_e4m3fn) {
    for (const Tensor* s : scales) {
      if (s->defined()) return false;
    }
    if (!sixteen(t) || x_scale.defined() || (type != kNone && type != t)) return false;
    type = t;
    return true;
  }
  for (const Tensor* s : scales) {
    if (!s->defined() || s->scalar_type() != at::kFloat || s->dim() != 1 || s->size(0) != out || !on(*s, x)) return false;
  }
  if (!x_scale.defined() || x_scale.scalar_type() != at::kFloat || x_scale.sizes() != x.sizes().slice(0, x.dim() - 1) || !on(x_scale, x)) {
    return false;
  }
  if (type == kNone) type = at::kBFloat16;
  return sixteen(type);
}

py::object linear(const py::handle& x_, const py::handle& weight_, const py::handle& bias_, int64_t act, const py::handle& residual_,
                  const py::handle& x_scale_, const py::handle& w_scale_, const py::handle& dtype_) {
  Tensor x, w, bias, residual, x_scale, w_scale;
  at::ScalarType type;
  if (!take(x_, x) || !take(weight_, w) || !take(bias_, bias) || !take(residual_, residual) || !take(x_scale_, x_scale) ||
      !take(w_scale_, w_scale) || !operands(x, w, x_scale, {&w_scale}, dtype_, type)) {
    return py::none();
  }
  if (bias.defined() && (bias.dim() != 1 || bias.size(0) != w.size(0) || !on(bias, x) || !bias.is_floating_point())) return py::none();
  const std::vector<int64_t> shape = out_shape(x, w.size(0));
  if (residual.defined() && (residual.scalar_type() != type || !on(residual, x) || residual.sizes() != at::IntArrayRef(shape))) {
    return py::none();
  }
  const bool grads = differentiated({&x, &w, &bias, &residual, &x_scale, &w_scale});
  if (grads && x.scalar_type() == at::kFloat8_e4m3fn) return py::none();
  Tensor y;
  {
    py::gil_scoped_release unlocked;
    if (bias.defined() && bias.scalar_type() != at::kFloat) bias = bias.to(at::kFloat);
    const Padding pad(w);
    if (pad.needed()) {
      x = pad.wider(x, pad.more_in), w = pad.wider(w, pad.more_in, pad.more_out), bias = pad.wider(bias, pad.more_out);
      residual = pad.wider(residual, pad.more_out), w_scale = pad.wider(w_scale, pad.more_out);
    }
    w = aligned(w), bias = aligned(bias);
    y = grads ? Linear::apply(x, w, maybe(bias), maybe(residual), act)
              : linear_fwd(rows_of(x, w.size(1)), w, aligned(x_scale), aligned(w_scale), bias, act, aligned(residual),
                           out_shape(x, w.size(0)), type, nullptr);
    y = pad.cut(y);
  }
  return py::cast(y);
}

py::object gated_linear(const py::handle& x_, const py::handle& gate_, const py::handle& up_, int64_t act, const py::handle& x_scale_,
                        const py::handle& g_scale_, const py::handle& u_scale_, const py::handle& dtype_) {
  Tensor x, gate, up, x_scale, g_scale, u_scale;
  at::ScalarType type;
  if (!take(x_, x) || !take(gate_, gate) || !take(up_, up) || !take(x_scale_, x_scale) || !take(g_scale_, g_scale) ||
      !take(u_scale_, u_scale) || !operands(x, gate, x_scale, {&g_scale, &u_scale}, dtype_, type) || !up.defined() || !on(up, x) ||
      up.scalar_type() != gate.scalar_type() || up.sizes() != gate.sizes()) {
    return py::none();
  }
  const bool grads = differentiated({&x, &gate, &up, &x_scale, &g_scale, &u_scale});
  if (grads && x.scalar_type() == at::kFloat8_e4m3fn) return py::none();
  Tensor h;
  {
    py::gil_scoped_release unlocked;
    const Padding pad(gate);
    if (pad.needed()) {
      x = pad.wider(x, pad.more_in);
      gate = pad.wider(gate, pad.more_in, pad.more_out), up = pad.wider(up, pad.more_in, pad.more_out);
      g_scale = pad.wider(g_scale, pad.more_out), u_scale = pad.wider(u_scale, pad.more_out);
    }
    gate = aligned(gate), up = aligned(up);
    h = grads ? GatedLinear::apply(x, gate, up, act)
              : gated_fwd(rows_of(x, gate.size(1)), gate, up, aligned(x_scale), aligned(g_scale), aligned(u_scale), act,
                          out_shape(x, gate.size(0)), type, nullptr, nullptr);
    h = pad.cut(h);
  }
  return py::cast(h);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("bind", &bind);
  m.def("rms_norm", &rms_norm);
  m.def("linear", &linear);
  m.def("gated_linear", &gated_linear);
}
