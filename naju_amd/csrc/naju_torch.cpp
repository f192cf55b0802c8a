// naju_torch.cpp -- the autograd side of layer norm, of the gated feed-forward
// product and of the vocabulary head's loss, over the C ABI of
// include/naju_mixer.h and include/naju_loss.h: torch.ops.naju.*, which
// naju_amd/layernorm.py, gated.py and linear_xent.py call after their checks.
//
// The forward and the backward of a small call take 10 to 60 us on the GPU; an
// autograd function in Python spends twice that on the host, most of it in the
// engine's device thread, which waits for the interpreter at every step (layer
// norm of 3063 x 771 both ways: 141 us in Python, 24 us on the GPU). Here neither
// direction enters the interpreter.
//
// Operands are brought to the kernels' row form here (RowOperand), on the
// current stream; all memory comes from torch's allocator, on that stream too.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/library.h>

#include "naju_loss.h"
#include "naju_mixer.h"
#include "naju_scan.h"

namespace {

using at::Tensor;
using c10::optional;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return NAJU_DTYPE_F32;
    case at::kBFloat16: return NAJU_DTYPE_BF16;
    case at::kHalf: return NAJU_DTYPE_F16;
    default: TORCH_CHECK(false, "naju: unsupported dtype ", t);
  }
}
at::ScalarType type_of(int64_t code) {
  return code == NAJU_DTYPE_F32 ? at::kFloat : code == NAJU_DTYPE_BF16 ? at::kBFloat16 : at::kHalf;
}

void* stream_of(const Tensor& t) {
  return (void*)c10::hip::getCurrentHIPStreamMasqueradingAsCUDA(t.device().index()).stream();
}
void check_mixer(int rc) { TORCH_CHECK(rc == NAJU_OK, "naju error ", rc, ": ", naju_mixer_last_error()); }
void check_loss(int rc) { TORCH_CHECK(rc == NAJU_OK, "naju error ", rc, ": ", naju_loss_last_error()); }

// Whether a graph is being recorded through t. Where it is not, the operators
// make their call alone: no node, nothing kept for a backward.
bool records(const Tensor& t) { return at::GradMode::is_enabled() && t.requires_grad(); }
bool records(const optional<Tensor>& t) { return t && records(*t); }

// A forward-mode tangent of an operand is refused, whether a graph is recorded
// or not: the kernels know nothing of it, and a result without a tangent counts
// as constant.
void no_tangent(const Tensor& t) {
  TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), "naju: forward-mode derivatives (jvp) are not served");
}
void no_tangent(const optional<Tensor>& t) {
  if (t) no_tangent(*t);
}

// What a backward that may itself be differentiated (create_graph) hands its
// gradients on with: it leads to all that they depend on, and raises when a
// second derivative is taken through it, whichever way and for whichever of
// them. Without it their dependence would count as zero.
struct Refusal : torch::autograd::Node {
  explicit Refusal(const char* of) : of_(of) {}
  variable_list apply(variable_list&&) override {
    TORCH_CHECK(false, "naju: ", of_, " has no second derivative (its gradient does not require grad further)");
  }
  std::string name() const override { return "NajuSecondDerivative"; }
  const char* of_;
};
variable_list once_differentiable(const char* of, const variable_list& incoming, variable_list grads) {
  const auto self = torch::autograd::get_current_node();
  if (!at::GradMode::is_enabled() || !self) return grads;
  // the way to the operator's own inputs, and to what the incoming gradients came from
  torch::autograd::edge_list next = self->next_edges();
  for (const Tensor& g : incoming)
    if (g.defined() && g.requires_grad()) next.push_back(torch::autograd::impl::gradient_edge(g));
  const std::shared_ptr<Refusal> node(new Refusal(of), torch::autograd::deleteNode);
  node->set_next_edges(std::move(next));
  for (Tensor& g : grads) {
    if (!g.defined()) continue;
    g = g.detach();
    torch::autograd::create_gradient_edge(g, node);
  }
  return grads;
}

// t [..., d] as [rows, d] with d fastest and rows at least d apart: a view where there is one.
Tensor row_matrix(const Tensor& t) {
  const int64_t d = t.size(-1);
  Tensor m = t.dim() == 2 ? t : (t.numel() ? t.reshape({-1, d}) : t.reshape({0, d}));
  if (m.stride(1) != 1 || (m.size(0) > 1 && m.stride(0) < d)) m = m.contiguous();
  return m;
}
int64_t row_stride(const Tensor& m) { return m.size(0) > 1 ? m.stride(0) : m.size(1); }

// m [rows, d], 16 bits, as the tile kernels read it: 16-byte aligned rows a
// multiple of 8 elements and at most 2^21 apart (their offsets within a tile are
// 32 bits), zeros from d to the next multiple of 8. m itself where it lies so,
// else a copy padded to 64: the last token of each of a batch of long sequences.
Tensor aligned_rows(const Tensor& m, bool copy = false) {
  const int64_t rows = m.size(0), d = m.size(1);
  if (!copy && d % 8 == 0 && m.stride(1) == 1 && ((uintptr_t)m.data_ptr() & 15) == 0 &&
      (rows <= 1 || (m.stride(0) >= d && m.stride(0) % 8 == 0 && m.stride(0) <= (1 << 21))))
    return m;
  const Tensor s = m.stride(1) != 1 || (rows > 1 && m.stride(0) < d) ? m.contiguous() : m;
  Tensor out = at::empty({rows, (d + 63) / 64 * 64}, m.options());
  check_mixer(naju_pack_rows(s.data_ptr(), row_stride(s), rows, d, out.data_ptr(), out.size(1), stream_of(m)));
  return out;
}
int64_t operand_stride(const Tensor& m) {
  const int64_t d8 = (m.size(1) + 7) / 8 * 8, s = row_stride(m);
  return s > d8 ? s : d8;
}

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}
// Uninitialised where the kernels write it, zeros where no row does.
Tensor grad_buffer(at::IntArrayRef shape, at::ScalarType type, const Tensor& like, bool zero) {
  const auto opt = like.options().dtype(type);
  return zero ? at::zeros(shape, opt) : at::empty(shape, opt);
}
// The type a weight's gradient is formed in: the weight's own where it is the
// products' 16-bit type, else float32.
at::ScalarType weight_grad_type(at::ScalarType weight, at::ScalarType compute) {
  return weight == compute ? compute : at::kFloat;
}
Tensor as(const Tensor& t, at::ScalarType type) { return t.scalar_type() == type ? t : t.to(type); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// ------------------------------------------------------------ layer norm

variable_list norm_backward(AutogradContext* ctx, const Tensor& grad, const Tensor& dres_in) {
  const auto saved = ctx->get_saved_variables();
  const Tensor &x = saved[0], &w = saved[1], &stats = saved[2];
  const int64_t rows = x.size(0), d = x.size(1);
  const c10::DeviceGuard guard(x.device());
  const auto& data = ctx->saved_data;
  const bool has_w = data.at("w").toBool(), has_b = data.at("b").toBool();
  const bool need_w = has_w && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
  Tensor dw, db, dx = at::empty({rows, d}, x.options());
  if (need_w) dw = grad_buffer({d}, at::kFloat, x, rows == 0);
  if (need_b) db = grad_buffer({d}, at::kFloat, x, rows == 0);
  if (rows) {
    const Tensor dy = row_matrix(grad);
    const Tensor dres = dres_in.defined() ? as(dres_in, x.scalar_type()).contiguous() : Tensor();
    Tensor ws;
    size_t bytes = 0;
    if (need_w || need_b) {
      bytes = naju_layernorm_workspace_bytes(rows, d);
      ws = workspace(bytes, x);
    }
    const float* mean = (const float*)stats.data_ptr();
    check_mixer(naju_layernorm_bwd(x.data_ptr(), row_stride(x), (const float*)ptr(w), mean, mean + rows, dy.data_ptr(),
                                   row_stride(dy), ptr(dres), dx.data_ptr(), (float*)ptr(dw), (float*)ptr(db), rows, d,
                                   code_of(x.scalar_type()), code_of(dy.scalar_type()), ptr(ws), bytes,
                                   stream_of(x)));
  }
  return {dx.view(data.at("shape").toIntVector()), dw, db, Tensor(), Tensor()};
}

Tensor norm_forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                    double eps, int64_t out) {
  const Tensor m = row_matrix(x);
  const int64_t rows = m.size(0), d = m.size(1);
  const c10::DeviceGuard guard(x.device());
  Tensor y = at::empty(x.sizes(), x.options().dtype(type_of(out)).memory_format(at::MemoryFormat::Contiguous));
  Tensor stats;
  if (ctx) stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
  float* mean = ctx && rows ? (float*)stats.data_ptr() : nullptr;
  check_mixer(naju_layernorm_fwd(m.data_ptr(), row_stride(m), w ? (const float*)w->data_ptr() : nullptr,
                                 b ? (const float*)b->data_ptr() : nullptr, (float)eps, y.data_ptr(), mean,
                                 mean ? mean + rows : nullptr, rows, d, code_of(x.scalar_type()), (int)out,
                                 stream_of(x)));
  if (ctx) {
    ctx->save_for_backward({m, w ? *w : Tensor(), stats});
    ctx->saved_data["w"] = w.has_value();
    ctx->saved_data["b"] = b.has_value();
    ctx->saved_data["shape"] = x.sizes();
  }
  return y;
}

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                        double eps, int64_t out) {
    return norm_forward(ctx, x, w, b, eps, out);
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    return once_differentiable("layer_norm", g, norm_backward(ctx, g[0], Tensor()));
  }
};

// (x, norm(x)): the gradients of both meet in the norm's backward kernel.
struct LayerNormFork : torch::autograd::Function<LayerNormFork> {
  static variable_list forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w,
                               const optional<Tensor>& b, double eps, int64_t out) {
    ctx->set_materialize_grads(false);
    Tensor y = norm_forward(ctx, x, w, b, eps, out);
    return {x.view(x.sizes()), y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (g[1].defined()) return once_differentiable("layer_norm", g, norm_backward(ctx, g[1], g[0]));
    // only the stream was used: its gradient as it is
    return {g[0], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor layer_norm(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps, int64_t out) {
  no_tangent(x), no_tangent(w), no_tangent(b);
  if (!records(x) && !records(w) && !records(b)) return norm_forward(nullptr, x, w, b, eps, out);
  return LayerNorm::apply(x, w, b, eps, out);
}
std::tuple<Tensor, Tensor> layer_norm_fork(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                                           double eps, int64_t out) {
  no_tangent(x), no_tangent(w), no_tangent(b);
  auto r = LayerNormFork::apply(x, w, b, eps, out);
  return {r[0], r[1]};
}

// ------------------------------------------------------------ gated product

struct Gated : torch::autograd::Function<Gated> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        const optional<Tensor>& pair, int64_t act) {
    const auto type = x.scalar_type();
    const int64_t f = wg.size(0), d = wg.size(1);
    const c10::DeviceGuard guard(x.device());
    const Tensor m = aligned_rows(row_matrix(x));
    // the weights in x's type: from one 16-bit matrix of both, or cast here
    const Tensor gt = pair ? pair->narrow(0, 0, f) : as(wg, type), ut = pair ? pair->narrow(0, f, f) : as(wu, type);
    Tensor gw = aligned_rows(gt), uw = aligned_rows(ut);
    if (operand_stride(gw) != operand_stride(uw)) {
      // the kernels take one stride: both copied to the same one
      gw = aligned_rows(gt, true);
      uw = aligned_rows(ut, true);
    }
    auto shape = x.sizes().vec();
    shape.back() = f;
    Tensor h = at::empty(shape, x.options().memory_format(at::MemoryFormat::Contiguous));
    check_mixer(naju_gated_fwd(m.data_ptr(), operand_stride(m), gw.data_ptr(), uw.data_ptr(), operand_stride(gw),
                               h.data_ptr(), f, m.size(0), d, f, (int)act, code_of(type), stream_of(x)));
    if (!ctx) return h;
    ctx->save_for_backward({m, gw, uw});
    ctx->saved_data["shape"] = x.sizes();
    ctx->saved_data["act"] = act;
    ctx->saved_data["f"] = f;
    ctx->saved_data["g_type"] = (int64_t)wg.scalar_type();
    ctx->saved_data["u_type"] = (int64_t)wu.scalar_type();
    return h;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &m = saved[0], &gw = saved[1], &uw = saved[2];
    const auto type = m.scalar_type();
    const auto& data = ctx->saved_data;
    const auto shape = data.at("shape").toIntVector();
    const int64_t rows = m.size(0), d = shape.back(), f = data.at("f").toInt();
    const auto g_type = (at::ScalarType)data.at("g_type").toInt(), u_type = (at::ScalarType)data.at("u_type").toInt();
    const c10::DeviceGuard guard(m.device());
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const auto w_type = g_type == type && u_type == type ? type : at::kFloat;
    Tensor dx, dg, du;
    if (need_x) dx = at::empty({rows, d}, m.options());
    if (need_w) {
      dg = grad_buffer({f, d}, w_type, m, rows == 0);
      du = grad_buffer({f, d}, w_type, m, rows == 0);
    }
    if (rows && (need_x || need_w)) {
      const Tensor dh = row_matrix(as(grads[0], type));
      const size_t bytes = naju_gated_workspace_bytes(rows, d, f);
      const Tensor ws = workspace(bytes, m);
      check_mixer(naju_gated_bwd(m.data_ptr(), operand_stride(m), gw.data_ptr(), uw.data_ptr(), operand_stride(gw),
                                 dh.data_ptr(), row_stride(dh), ptr(dx), ptr(dg), ptr(du), rows, d, f,
                                 (int)data.at("act").toInt(), code_of(type), code_of(w_type), ws.data_ptr(), bytes,
                                 stream_of(m)));
    }
    return once_differentiable("gated_linear", grads, {need_x ? dx.view(shape) : dx, need_w ? as(dg, g_type) : dg,
                                                       need_w ? as(du, u_type) : du, Tensor(), Tensor()});
  }
};

Tensor gated_linear(const Tensor& x, const Tensor& wg, const Tensor& wu, const optional<Tensor>& pair, int64_t act) {
  no_tangent(x), no_tangent(wg), no_tangent(wu);
  if (!records(x) && !records(wg) && !records(wu)) return Gated::forward(nullptr, x, wg, wu, pair, act);
  return Gated::apply(x, wg, wu, pair, act);
}

// ------------------------------------------------------------ head and loss

enum { kMean, kSum, kNone };

struct LinearXent : torch::autograd::Function<LinearXent> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& target,
                        const optional<Tensor>& w16, int64_t ignore, int64_t reduction) {
    const auto type = x.scalar_type();
    const int64_t v = weight.size(0), d = weight.size(1);
    const c10::DeviceGuard guard(x.device());
    const Tensor m = aligned_rows(row_matrix(x));
    const Tensor w = aligned_rows(w16 ? w16->narrow(0, 0, v) : as(weight, type));
    const int64_t rows = m.size(0);
    const auto f32 = x.options().dtype(at::kFloat).memory_format(at::MemoryFormat::Contiguous);
    Tensor lse = at::empty({rows}, f32), row_loss = at::empty(target.sizes(), f32), loss, scale;
    if (reduction != kNone) {
      loss = at::empty({}, f32);
      scale = at::empty({}, f32);
    }
    const size_t bytes = naju_linear_xent_workspace_bytes(rows, d, v, 0);
    const Tensor ws = workspace(bytes, x);
    check_loss(naju_linear_xent_fwd(m.data_ptr(), operand_stride(m), w.data_ptr(), operand_stride(w),
                                    (const int64_t*)target.data_ptr(), rows, d, v, code_of(type), ignore,
                                    (float*)lse.data_ptr(), (float*)row_loss.data_ptr(), reduction == kMean,
                                    (float*)ptr(loss), (float*)ptr(scale), ws.data_ptr(), bytes, stream_of(x)));
    if (ctx) {
      ctx->save_for_backward({m, w, target, lse, scale});
      ctx->saved_data["shape"] = x.sizes();
      ctx->saved_data["v"] = v;
      ctx->saved_data["ignore"] = ignore;
      ctx->saved_data["w_type"] = (int64_t)weight.scalar_type();
    }
    return reduction == kNone ? row_loss : loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &m = saved[0], &w = saved[1], &target = saved[2], &lse = saved[3], &scale = saved[4];
    const auto type = m.scalar_type();
    const auto& data = ctx->saved_data;
    const auto shape = data.at("shape").toIntVector();
    const int64_t rows = m.size(0), d = shape.back(), v = data.at("v").toInt();
    const auto w_type = (at::ScalarType)data.at("w_type").toInt();
    const c10::DeviceGuard guard(m.device());
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    const auto dw_type = weight_grad_type(w_type, type);
    Tensor dx, dw;
    if (need_x) dx = at::empty({rows, d}, m.options());
    if (need_w) dw = grad_buffer({v, d}, dw_type, m, rows == 0);
    if (rows && (need_x || need_w)) {
      const Tensor dloss = as(grads[0], at::kFloat).contiguous();
      const size_t bytes = naju_linear_xent_workspace_bytes(rows, d, v, 1);
      const Tensor ws = workspace(bytes, m);
      check_loss(naju_linear_xent_bwd(m.data_ptr(), operand_stride(m), w.data_ptr(), operand_stride(w),
                                      (const int64_t*)target.data_ptr(), rows, d, v, code_of(type),
                                      data.at("ignore").toInt(), (const float*)lse.data_ptr(),
                                      (const float*)ptr(scale), (const float*)dloss.data_ptr(), !scale.defined(),
                                      ptr(dx), ptr(dw), code_of(dw_type), ws.data_ptr(), bytes, stream_of(m)));
    }
    return once_differentiable("linear_cross_entropy", grads, {need_x ? dx.view(shape) : dx,
                                                               need_w ? as(dw, w_type) : dw, Tensor(), Tensor(),
                                                               Tensor(), Tensor()});
  }
};

Tensor linear_cross_entropy(const Tensor& x, const Tensor& weight, const Tensor& target, const optional<Tensor>& w16,
                            int64_t ignore, int64_t reduction) {
  no_tangent(x), no_tangent(weight);
  if (!records(x) && !records(weight)) return LinearXent::forward(nullptr, x, weight, target, w16, ignore, reduction);
  return LinearXent::apply(x, weight, target, w16, ignore, reduction);
}

}  // namespace

// Composite: autograd is the functions above, whatever the dispatch mode.
TORCH_LIBRARY(naju, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, int out_dtype) -> Tensor",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(layer_norm)));
  m.def("layer_norm_fork(Tensor x, Tensor? weight, Tensor? bias, float eps, int out_dtype) -> (Tensor, Tensor)",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(layer_norm_fork)));
  m.def("gated_linear(Tensor x, Tensor w_gate, Tensor w_up, Tensor? pair, int act) -> Tensor",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(gated_linear)));
  m.def("linear_cross_entropy(Tensor x, Tensor weight, Tensor target, Tensor? w16, int ignore_index, int reduction) "
        "-> Tensor",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(linear_cross_entropy)));
}
