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
// Three layers, each an operator that torch's dispatcher knows:
//   layer_norm, gated_linear, linear_cross_entropy   what the Python modules
//     call; at the autograd key the native function below where a graph is
//     recorded, else on to the kernel;
//   _layer_norm_fwd / _bwd, _gated_fwd / _bwd, _linear_xent_fwd / _bwd   what
//     those functions call, with what the backward needs among the results;
//   layer_norm_fork   a composite of the function and a view.
// The kernels stand at the CUDA key and the results' shapes at the Meta key, so
// that whatever stands between (tracers, fake tensors, torch.compile, dispatch
// modes) sees operators and never their insides.
//
// Operands are brought to the kernels' row form here, on the current stream;
// all memory comes from torch's allocator, on that stream too.
#include <ATen/ATen.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>
#include <c10/core/DeviceGuard.h>
#include <c10/core/impl/TorchDispatchModeTLS.h>
#include <torch/csrc/autograd/autograd_not_implemented_fallback.h>
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

// Whether t is an ordinary tensor on the GPU that no dispatch mode stands
// before: its sizes are numbers, and its memory can be read here unseen.
bool plain(const Tensor& t) {
  return t.is_cuda() && !t.key_set().has(c10::DispatchKey::Python) && !c10::impl::dispatch_mode_enabled();
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
// else a copy padded to 64 (the last token of each of a batch of long sequences,
// say): its first d columns, or all of it where d is no multiple of 8.
Tensor aligned_rows(const Tensor& m, bool copy = false) {
  const int64_t rows = m.size(0), d = m.size(1);
  if (!copy && d % 8 == 0 && m.stride(1) == 1 && ((uintptr_t)m.data_ptr() & 15) == 0 &&
      (rows <= 1 || (m.stride(0) >= d && m.stride(0) % 8 == 0 && m.stride(0) <= (1 << 21))))
    return m;
  const Tensor s = m.stride(1) != 1 || (rows > 1 && m.stride(0) < d) ? m.contiguous() : m;
  Tensor out = at::empty({rows, (d + 63) / 64 * 64}, m.options());
  check_mixer(naju_pack_rows(s.data_ptr(), row_stride(s), rows, d, out.data_ptr(), out.size(1), stream_of(m)));
  return d % 8 ? out : out.narrow(1, 0, d);
}
// Two weights, in rows of one stride.
void align_pair(Tensor& a, Tensor& b) {
  const Tensor a0 = a, b0 = b;
  a = aligned_rows(a0);
  b = aligned_rows(b0);
  if (row_stride(a) != row_stride(b)) {
    // the kernels take one stride: both copied to the same one
    a = aligned_rows(a0, true);
    b = aligned_rows(b0, true);
  }
}

// For the functions below, which keep operands from the forward to the
// backward: x as rows, brought to the kernels' form once. Where that may not be
// looked into (plain), the kernels do so themselves, each time.
Tensor rows_of(const Tensor& x) {
  if (plain(x)) return row_matrix(x);
  const c10::SymInt d = x.sym_size(-1);
  return x.dim() == 2 ? x : x.reshape_symint({x.sym_numel() / d, d});
}
// The `width` with which operands so kept are passed on: their d where they are
// padded past it, else 0.
int64_t kept_width(const Tensor& x) { return plain(x) && x.size(-1) % 8 ? x.size(-1) : 0; }

Tensor workspace(size_t bytes, const Tensor& like) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte));
}
Tensor none_of(at::ScalarType type, const Tensor& like) { return at::empty({0}, like.options().dtype(type)); }
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
void* ptr(const Tensor& t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
// like's shape but for a last axis of n
c10::SymDimVector with_last(c10::SymIntArrayRef like, const c10::SymInt& n) {
  c10::SymDimVector s(like.begin(), like.end());
  s.back() = n;
  return s;
}
auto contiguous_like(const Tensor& t, at::ScalarType type) {
  return t.options().dtype(type).memory_format(at::MemoryFormat::Contiguous);
}

// Operator NAME of F's type, looked up once.
#define NAJU_OP(NAME, F)                                                                                    \
  ([]() -> const c10::TypedOperatorHandle<decltype(F)>& {                                                   \
    static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("naju::" NAME, "").typed<decltype(F)>(); \
    return op;                                                                                              \
  }())
// Calls within it go to the kernels, or to what stands before them, without autograd's own steps.
using Below = at::AutoDispatchBelowADInplaceOrView;

// ------------------------------------------------------------ layer norm

void check_norm(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b) {
  TORCH_CHECK(x.dim() > 0 && x.size(-1) > 0, "naju: x must have a last axis");
  for (const auto* t : {&w, &b})
    TORCH_CHECK(!*t || ((*t)->dim() == 1 && (*t)->size(0) == x.size(-1) && (*t)->scalar_type() == at::kFloat &&
                        (*t)->is_contiguous() && (*t)->device() == x.device()),
                "naju: the weight and the bias must be contiguous float32 of x's width, on its device");
}
Tensor norm_cuda(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps, int64_t out,
                 Tensor* stats) {
  check_norm(x, w, b);
  const c10::DeviceGuard guard(x.device());
  const Tensor m = row_matrix(x);
  const int64_t rows = m.size(0), d = m.size(1);
  Tensor y = at::empty(x.sizes(), contiguous_like(x, type_of(out)));
  if (stats) *stats = at::empty({2, rows}, x.options().dtype(at::kFloat));
  float* mean = stats && rows ? (float*)stats->data_ptr() : nullptr;
  check_mixer(naju_layernorm_fwd(m.data_ptr(), row_stride(m), w ? (const float*)w->data_ptr() : nullptr,
                                 b ? (const float*)b->data_ptr() : nullptr, (float)eps, y.data_ptr(), mean,
                                 mean ? mean + rows : nullptr, rows, d, code_of(x.scalar_type()), (int)out,
                                 stream_of(x)));
  return y;
}
Tensor layer_norm_cuda(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps,
                       int64_t out) {
  return norm_cuda(x, w, b, eps, out, nullptr);
}
Tensor layer_norm_meta(const Tensor& x, const optional<Tensor>&, const optional<Tensor>&, double, int64_t out) {
  return at::empty_symint(x.sym_sizes(), contiguous_like(x, type_of(out)));
}

// (y, the rows' means and reciprocal deviations [2, rows])
std::tuple<Tensor, Tensor> norm_fwd_cuda(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                                         double eps, int64_t out) {
  Tensor stats;
  Tensor y = norm_cuda(x, w, b, eps, out, &stats);
  return {y, stats};
}
std::tuple<Tensor, Tensor> norm_fwd_meta(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                                         double eps, int64_t out) {
  return {layer_norm_meta(x, w, b, eps, out),
          at::empty_symint({2, x.sym_numel() / x.sym_size(-1)}, x.options().dtype(at::kFloat))};
}

// x as rows [rows, d], dy of any shape of as many. (dx, dw, db), those not wanted of no elements.
std::tuple<Tensor, Tensor, Tensor> norm_bwd_cuda(const Tensor& grad, const optional<Tensor>& dres_in, const Tensor& x,
                                                 const optional<Tensor>& w, const Tensor& stats, bool need_w,
                                                 bool need_b) {
  check_norm(x, w, optional<Tensor>());
  const int64_t rows = x.size(0), d = x.size(1);
  TORCH_CHECK(x.dim() == 2 && grad.numel() == rows * d && grad.size(-1) == d && stats.numel() == 2 * rows &&
                  (!dres_in || dres_in->numel() == rows * d),
              "naju: the gradients must have x's shape");
  const c10::DeviceGuard guard(x.device());
  const Tensor m = row_matrix(x);
  Tensor dx = at::empty({rows, d}, contiguous_like(x, x.scalar_type()));
  Tensor dw = need_w ? grad_buffer({d}, at::kFloat, x, rows == 0) : none_of(at::kFloat, x);
  Tensor db = need_b ? grad_buffer({d}, at::kFloat, x, rows == 0) : none_of(at::kFloat, x);
  if (rows) {
    const Tensor dy = row_matrix(grad);
    const Tensor dres = dres_in ? as(*dres_in, x.scalar_type()).contiguous() : Tensor();
    Tensor ws;
    size_t bytes = 0;
    if (need_w || need_b) {
      bytes = naju_layernorm_workspace_bytes(rows, d);
      ws = workspace(bytes, x);
    }
    const float* mean = (const float*)stats.data_ptr();
    check_mixer(naju_layernorm_bwd(m.data_ptr(), row_stride(m), w ? (const float*)w->data_ptr() : nullptr, mean,
                                   mean + rows, dy.data_ptr(), row_stride(dy), ptr(dres), dx.data_ptr(),
                                   (float*)ptr(dw), (float*)ptr(db), rows, d, code_of(x.scalar_type()),
                                   code_of(dy.scalar_type()), ptr(ws), bytes, stream_of(x)));
  }
  return {dx, dw, db};
}
std::tuple<Tensor, Tensor, Tensor> norm_bwd_meta(const Tensor&, const optional<Tensor>&, const Tensor& x,
                                                 const optional<Tensor>&, const Tensor&, bool need_w, bool need_b) {
  const auto f32 = x.options().dtype(at::kFloat);
  const c10::SymInt d = x.sym_size(1);
  return {at::empty_symint(x.sym_sizes(), contiguous_like(x, x.scalar_type())),
          at::empty_symint({need_w ? d : c10::SymInt(0)}, f32), at::empty_symint({need_b ? d : c10::SymInt(0)}, f32)};
}

Tensor norm_forward(AutogradContext* ctx, const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                    double eps, int64_t out) {
  const Tensor m = rows_of(x);
  const Below below;
  auto [y, stats] = NAJU_OP("_layer_norm_fwd", norm_fwd_cuda).call(m, w, b, eps, out);
  ctx->save_for_backward({m, w ? *w : Tensor(), stats});
  ctx->saved_data["w"] = w.has_value();
  ctx->saved_data["b"] = b.has_value();
  return x.dim() == 2 ? y : y.view_symint(x.sym_sizes());
}

variable_list norm_backward(AutogradContext* ctx, const Tensor& grad, const Tensor& dres) {
  const auto saved = ctx->get_saved_variables();
  const Tensor &m = saved[0], &w = saved[1], &stats = saved[2];
  const bool has_w = ctx->saved_data.at("w").toBool(), has_b = ctx->saved_data.at("b").toBool();
  const bool need_w = has_w && ctx->needs_input_grad(1), need_b = has_b && ctx->needs_input_grad(has_w ? 2 : 1);
  const Below below;
  auto [dx, dw, db] = NAJU_OP("_layer_norm_bwd", norm_bwd_cuda)
                          .call(grad, dres.defined() ? optional<Tensor>(dres) : optional<Tensor>(), m,
                                w.defined() ? optional<Tensor>(w) : optional<Tensor>(), stats, need_w, need_b);
  return {grad.dim() == 2 ? dx : dx.view_symint(grad.sym_sizes()), need_w ? dw : Tensor(), need_b ? db : Tensor(),
          Tensor(), Tensor()};
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
    return {x.view_symint(x.sym_sizes()), y};
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    if (g[1].defined()) return once_differentiable("layer_norm", g, norm_backward(ctx, g[1], g[0]));
    // only the stream was used: its gradient as it is
    return {g[0], Tensor(), Tensor(), Tensor(), Tensor()};
  }
};

Tensor layer_norm_autograd(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b, double eps,
                           int64_t out) {
  no_tangent(x), no_tangent(w), no_tangent(b);
  if (records(x) || records(w) || records(b)) return LayerNorm::apply(x, w, b, eps, out);
  const Below below;
  return NAJU_OP("layer_norm", layer_norm_cuda).call(x, w, b, eps, out);
}
std::tuple<Tensor, Tensor> layer_norm_fork(const Tensor& x, const optional<Tensor>& w, const optional<Tensor>& b,
                                           double eps, int64_t out) {
  no_tangent(x), no_tangent(w), no_tangent(b);
  if (!records(x) && !records(w) && !records(b))
    return {x.view_symint(x.sym_sizes()), NAJU_OP("layer_norm", layer_norm_cuda).call(x, w, b, eps, out)};
  auto r = LayerNormFork::apply(x, w, b, eps, out);
  return {r[0], r[1]};
}

// ------------------------------------------------------------ gated product

// The 16-bit operands of a call: d columns of each, from operands as they come
// (width 0) or padded to rows of more (width d).
struct GatedOperands {
  Tensor x, wg, wu;
  int64_t d;
  GatedOperands(const Tensor& x_, const Tensor& wg_, const Tensor& wu_, int64_t width) : x(x_), wg(wg_), wu(wu_) {
    TORCH_CHECK(x.dim() == 2 && wg.dim() == 2 && wg.sizes() == wu.sizes() && wg.size(1) == x.size(1) &&
                    wg.scalar_type() == x.scalar_type() && wu.scalar_type() == x.scalar_type() &&
                    wg.device() == x.device() && wu.device() == x.device(),
                "naju: gated_linear's operands do not fit together");
    d = width ? width : x.size(1);
    if (width) {
      TORCH_CHECK(d <= x.size(1), "naju: width past the operands");
      return;
    }
    x = aligned_rows(x);
    align_pair(wg, wu);
  }
};

Tensor gated_fwd_cuda(const Tensor& x, const Tensor& wg, const Tensor& wu, int64_t width, int64_t act) {
  const c10::DeviceGuard guard(x.device());
  const GatedOperands o(x, wg, wu, width);
  const int64_t rows = x.size(0), f = wg.size(0);
  Tensor h = at::empty({rows, f}, contiguous_like(x, x.scalar_type()));
  check_mixer(naju_gated_fwd(o.x.data_ptr(), row_stride(o.x), o.wg.data_ptr(), o.wu.data_ptr(), row_stride(o.wg),
                             h.data_ptr(), f, rows, o.d, f, (int)act, code_of(x.scalar_type()), stream_of(x)));
  return h;
}
Tensor gated_fwd_meta(const Tensor& x, const Tensor& wg, const Tensor&, int64_t, int64_t) {
  return at::empty_symint({x.sym_size(0), wg.sym_size(0)}, contiguous_like(x, x.scalar_type()));
}

// (dx [rows, d], dw_gate, dw_up [f, d] of type dw_dtype), those not wanted of no elements
std::tuple<Tensor, Tensor, Tensor> gated_bwd_cuda(const Tensor& grad, const Tensor& x, const Tensor& wg,
                                                  const Tensor& wu, int64_t width, int64_t act, bool need_x,
                                                  bool need_w, int64_t dw_dtype) {
  const c10::DeviceGuard guard(x.device());
  const GatedOperands o(x, wg, wu, width);
  const int64_t rows = x.size(0), f = wg.size(0);
  TORCH_CHECK(grad.numel() == rows * f && grad.size(-1) == f, "naju: the gradient must have h's shape");
  const auto type = x.scalar_type(), w_type = type_of(dw_dtype);
  Tensor dx = need_x ? at::empty({rows, o.d}, contiguous_like(x, type)) : none_of(type, x);
  Tensor dg = need_w ? grad_buffer({f, o.d}, w_type, x, rows == 0) : none_of(w_type, x);
  Tensor du = need_w ? grad_buffer({f, o.d}, w_type, x, rows == 0) : none_of(w_type, x);
  if (rows && (need_x || need_w)) {
    const Tensor dh = row_matrix(as(grad, type));
    const size_t bytes = naju_gated_workspace_bytes(rows, o.d, f);
    const Tensor ws = workspace(bytes, x);
    check_mixer(naju_gated_bwd(o.x.data_ptr(), row_stride(o.x), o.wg.data_ptr(), o.wu.data_ptr(), row_stride(o.wg),
                               dh.data_ptr(), row_stride(dh), ptr(dx), ptr(dg), ptr(du), rows, o.d, f, (int)act,
                               code_of(type), (int)dw_dtype, ws.data_ptr(), bytes, stream_of(x)));
  }
  return {dx, dg, du};
}
std::tuple<Tensor, Tensor, Tensor> gated_bwd_meta(const Tensor&, const Tensor& x, const Tensor& wg, const Tensor&,
                                                  int64_t width, int64_t, bool need_x, bool need_w, int64_t dw_dtype) {
  const c10::SymInt d = width ? c10::SymInt(width) : x.sym_size(1);
  auto of = [&](bool need, const c10::SymInt& rows, at::ScalarType type) {
    return need ? at::empty_symint({rows, d}, contiguous_like(x, type)) : none_of(type, x);
  };
  const auto w_type = type_of(dw_dtype);
  return {of(need_x, x.sym_size(0), x.scalar_type()), of(need_w, wg.sym_size(0), w_type),
          of(need_w, wg.sym_size(0), w_type)};
}

// The weights in x's type: from one 16-bit matrix of both, or cast here.
std::pair<Tensor, Tensor> gated_weights(const Tensor& wg, const Tensor& wu, const optional<Tensor>& pair,
                                        at::ScalarType type) {
  if (!pair) return {as(wg, type), as(wu, type)};
  const c10::SymInt f = wg.sym_size(0);
  return {pair->narrow_symint(0, 0, f), pair->narrow_symint(0, f, f)};
}

struct Gated : torch::autograd::Function<Gated> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& wg, const Tensor& wu,
                        const optional<Tensor>& pair, int64_t act) {
    Tensor m = rows_of(x);
    auto [gw, uw] = gated_weights(wg, wu, pair, x.scalar_type());
    const int64_t width = kept_width(x);
    if (plain(x)) {
      const c10::DeviceGuard guard(x.device());
      m = aligned_rows(m);
      align_pair(gw, uw);
    }
    const Below below;
    const Tensor h = NAJU_OP("_gated_fwd", gated_fwd_cuda).call(m, gw, uw, width, act);
    ctx->save_for_backward({m, gw, uw});
    auto& data = ctx->saved_data;
    data["width"] = width;
    data["act"] = act;
    data["g_type"] = (int64_t)wg.scalar_type();
    data["u_type"] = (int64_t)wu.scalar_type();
    return x.dim() == 2 ? h : h.view_symint(with_last(x.sym_sizes(), h.sym_size(1)));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &m = saved[0], &gw = saved[1], &uw = saved[2], &dh = grads[0];
    const auto type = m.scalar_type();
    const auto& data = ctx->saved_data;
    const auto g_type = (at::ScalarType)data.at("g_type").toInt(), u_type = (at::ScalarType)data.at("u_type").toInt();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1) || ctx->needs_input_grad(2);
    const auto w_type = g_type == type && u_type == type ? type : at::kFloat;
    variable_list out(5);
    {
      const Below below;
      auto [dx, dg, du] = NAJU_OP("_gated_bwd", gated_bwd_cuda)
                              .call(dh, m, gw, uw, data.at("width").toInt(), data.at("act").toInt(), need_x, need_w,
                                    code_of(w_type));
      if (need_x) out[0] = dh.dim() == 2 ? dx : dx.view_symint(with_last(dh.sym_sizes(), dx.sym_size(1)));
      if (need_w) {
        out[1] = as(dg, g_type);
        out[2] = as(du, u_type);
      }
    }
    return once_differentiable("gated_linear", grads, std::move(out));
  }
};

Tensor gated_linear_cuda(const Tensor& x, const Tensor& wg, const Tensor& wu, const optional<Tensor>& pair,
                         int64_t act) {
  auto [gw, uw] = gated_weights(wg, wu, pair, x.scalar_type());
  const Tensor h = gated_fwd_cuda(row_matrix(x), gw, uw, 0, act);
  return x.dim() == 2 ? h : h.view_symint(with_last(x.sym_sizes(), h.sym_size(1)));
}
Tensor gated_linear_meta(const Tensor& x, const Tensor& wg, const Tensor&, const optional<Tensor>&, int64_t) {
  return at::empty_symint(with_last(x.sym_sizes(), wg.sym_size(0)), contiguous_like(x, x.scalar_type()));
}
Tensor gated_linear_autograd(const Tensor& x, const Tensor& wg, const Tensor& wu, const optional<Tensor>& pair,
                             int64_t act) {
  no_tangent(x), no_tangent(wg), no_tangent(wu);
  if (records(x) || records(wg) || records(wu)) return Gated::apply(x, wg, wu, pair, act);
  const Below below;
  return NAJU_OP("gated_linear", gated_linear_cuda).call(x, wg, wu, pair, act);
}

// ------------------------------------------------------------ head and loss

enum { kMean, kSum, kNone };

struct HeadOperands {
  Tensor x, w;
  int64_t d;
  HeadOperands(const Tensor& x_, const Tensor& w_, const Tensor& target, int64_t width) : x(x_), w(w_) {
    TORCH_CHECK(x.dim() == 2 && w.dim() == 2 && w.size(1) == x.size(1) && w.scalar_type() == x.scalar_type() &&
                    target.numel() == x.size(0) && target.scalar_type() == at::kLong && target.is_contiguous() &&
                    w.device() == x.device() && target.device() == x.device(),
                "naju: linear_cross_entropy's operands do not fit together");
    d = width ? width : x.size(1);
    if (width) {
      TORCH_CHECK(d <= x.size(1), "naju: width past the operands");
      return;
    }
    x = aligned_rows(x);
    w = aligned_rows(w);
  }
};

// (the loss, the rows' logsumexp, the factor of the rows' losses in it; none where a loss for each row is asked for)
std::tuple<Tensor, Tensor, Tensor> xent_fwd_cuda(const Tensor& x, const Tensor& weight, const Tensor& target,
                                                 int64_t width, int64_t ignore, int64_t reduction) {
  const c10::DeviceGuard guard(x.device());
  const HeadOperands o(x, weight, target, width);
  const int64_t rows = x.size(0), v = weight.size(0);
  const auto f32 = contiguous_like(x, at::kFloat);
  Tensor lse = at::empty({rows}, f32), row_loss = at::empty(target.sizes(), f32), loss, scale;
  if (reduction != kNone) {
    loss = at::empty({}, f32);
    scale = at::empty({}, f32);
  } else {
    scale = none_of(at::kFloat, x);
  }
  const size_t bytes = naju_linear_xent_workspace_bytes(rows, o.d, v, 0);
  const Tensor ws = workspace(bytes, x);
  check_loss(naju_linear_xent_fwd(o.x.data_ptr(), row_stride(o.x), o.w.data_ptr(), row_stride(o.w),
                                  (const int64_t*)target.data_ptr(), rows, o.d, v, code_of(x.scalar_type()), ignore,
                                  (float*)lse.data_ptr(), (float*)row_loss.data_ptr(), reduction == kMean,
                                  (float*)ptr(loss), (float*)ptr(scale), ws.data_ptr(), bytes, stream_of(x)));
  return {reduction == kNone ? row_loss : loss, lse, scale};
}
std::tuple<Tensor, Tensor, Tensor> xent_fwd_meta(const Tensor& x, const Tensor&, const Tensor& target, int64_t,
                                                 int64_t, int64_t reduction) {
  const auto f32 = contiguous_like(x, at::kFloat);
  return {reduction == kNone ? at::empty_symint(target.sym_sizes(), f32) : at::empty({}, f32),
          at::empty_symint({x.sym_size(0)}, f32), reduction == kNone ? none_of(at::kFloat, x) : at::empty({}, f32)};
}

// (dx [rows, d], dw [v, d] of type dw_dtype), that not wanted of no elements
std::tuple<Tensor, Tensor> xent_bwd_cuda(const Tensor& grad, const Tensor& x, const Tensor& weight,
                                         const Tensor& target, const Tensor& lse, const Tensor& scale, int64_t width,
                                         int64_t ignore, bool need_x, bool need_w, int64_t dw_dtype) {
  const c10::DeviceGuard guard(x.device());
  const HeadOperands o(x, weight, target, width);
  const int64_t rows = x.size(0), v = weight.size(0);
  TORCH_CHECK(grad.numel() == (scale.numel() ? 1 : rows) && lse.numel() == rows,
              "naju: the gradient must have the loss's shape");
  const auto type = x.scalar_type(), w_type = type_of(dw_dtype);
  Tensor dx = need_x ? at::empty({rows, o.d}, contiguous_like(x, type)) : none_of(type, x);
  Tensor dw = need_w ? grad_buffer({v, o.d}, w_type, x, rows == 0) : none_of(w_type, x);
  if (rows && (need_x || need_w)) {
    const Tensor dloss = as(grad, at::kFloat).contiguous();
    const size_t bytes = naju_linear_xent_workspace_bytes(rows, o.d, v, 1);
    const Tensor ws = workspace(bytes, x);
    check_loss(naju_linear_xent_bwd(o.x.data_ptr(), row_stride(o.x), o.w.data_ptr(), row_stride(o.w),
                                    (const int64_t*)target.data_ptr(), rows, o.d, v, code_of(type), ignore,
                                    (const float*)lse.data_ptr(), (const float*)ptr(scale),
                                    (const float*)dloss.data_ptr(), scale.numel() == 0, ptr(dx), ptr(dw),
                                    (int)dw_dtype, ws.data_ptr(), bytes, stream_of(x)));
  }
  return {dx, dw};
}
std::tuple<Tensor, Tensor> xent_bwd_meta(const Tensor&, const Tensor& x, const Tensor& w, const Tensor&, const Tensor&,
                                         const Tensor&, int64_t width, int64_t, bool need_x, bool need_w,
                                         int64_t dw_dtype) {
  const c10::SymInt d = width ? c10::SymInt(width) : x.sym_size(1);
  auto of = [&](bool need, const c10::SymInt& rows, at::ScalarType type) {
    return need ? at::empty_symint({rows, d}, contiguous_like(x, type)) : none_of(type, x);
  };
  return {of(need_x, x.sym_size(0), x.scalar_type()), of(need_w, w.sym_size(0), type_of(dw_dtype))};
}

// The weight in x's type: the first rows of a 16-bit copy, or cast here.
Tensor head_weight(const Tensor& weight, const optional<Tensor>& w16, at::ScalarType type) {
  return w16 ? w16->narrow_symint(0, 0, weight.sym_size(0)) : as(weight, type);
}

struct LinearXent : torch::autograd::Function<LinearXent> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& weight, const Tensor& target,
                        const optional<Tensor>& w16, int64_t ignore, int64_t reduction) {
    Tensor m = rows_of(x), w = head_weight(weight, w16, x.scalar_type());
    const int64_t width = kept_width(x);
    if (plain(x)) {
      const c10::DeviceGuard guard(x.device());
      m = aligned_rows(m);
      w = aligned_rows(w);
    }
    const Below below;
    auto [loss, lse, scale] =
        NAJU_OP("_linear_xent_fwd", xent_fwd_cuda).call(m, w, target, width, ignore, reduction);
    ctx->save_for_backward({m, w, target, lse, scale});
    auto& data = ctx->saved_data;
    data["width"] = width;
    data["ignore"] = ignore;
    data["w_type"] = (int64_t)weight.scalar_type();
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &m = saved[0], &w = saved[1], &target = saved[2], &lse = saved[3], &scale = saved[4];
    const auto& data = ctx->saved_data;
    const auto w_type = (at::ScalarType)data.at("w_type").toInt();
    const bool need_x = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1);
    variable_list out(6);
    {
      const Below below;
      auto [dx, dw] = NAJU_OP("_linear_xent_bwd", xent_bwd_cuda)
                          .call(grads[0], m, w, target, lse, scale, data.at("width").toInt(),
                                data.at("ignore").toInt(), need_x, need_w,
                                code_of(weight_grad_type(w_type, m.scalar_type())));
      if (need_x) {
        c10::SymDimVector shape(target.sym_sizes().begin(), target.sym_sizes().end());
        shape.push_back(dx.sym_size(1));
        out[0] = shape.size() == 2 ? dx : dx.view_symint(shape);
      }
      if (need_w) out[1] = as(dw, w_type);
    }
    return once_differentiable("linear_cross_entropy", grads, std::move(out));
  }
};

Tensor xent_cuda(const Tensor& x, const Tensor& weight, const Tensor& target, const optional<Tensor>& w16,
                 int64_t ignore, int64_t reduction) {
  return std::get<0>(
      xent_fwd_cuda(row_matrix(x), head_weight(weight, w16, x.scalar_type()), target, 0, ignore, reduction));
}
Tensor xent_meta(const Tensor& x, const Tensor&, const Tensor& target, const optional<Tensor>&, int64_t,
                 int64_t reduction) {
  const auto f32 = contiguous_like(x, at::kFloat);
  return reduction == kNone ? at::empty_symint(target.sym_sizes(), f32) : at::empty({}, f32);
}
Tensor xent_autograd(const Tensor& x, const Tensor& weight, const Tensor& target, const optional<Tensor>& w16,
                     int64_t ignore, int64_t reduction) {
  no_tangent(x), no_tangent(weight);
  if (records(x) || records(weight)) return LinearXent::apply(x, weight, target, w16, ignore, reduction);
  const Below below;
  return NAJU_OP("linear_cross_entropy", xent_cuda).call(x, weight, target, w16, ignore, reduction);
}

}  // namespace

TORCH_LIBRARY(naju, m) {
  m.def("layer_norm(Tensor x, Tensor? weight, Tensor? bias, float eps, int out_dtype) -> Tensor");
  m.def("_layer_norm_fwd(Tensor x, Tensor? weight, Tensor? bias, float eps, int out_dtype) -> (Tensor, Tensor)");
  m.def("_layer_norm_bwd(Tensor dy, Tensor? dres, Tensor x, Tensor? weight, Tensor stats, bool need_w, bool need_b) "
        "-> (Tensor, Tensor, Tensor)");
  // whatever the dispatch mode, the operators above and a view
  m.def("layer_norm_fork(Tensor x, Tensor? weight, Tensor? bias, float eps, int out_dtype) -> (Tensor, Tensor)",
        torch::dispatch(c10::DispatchKey::CompositeImplicitAutograd, TORCH_FN(layer_norm_fork)));
  m.def("gated_linear(Tensor x, Tensor w_gate, Tensor w_up, Tensor? pair, int act) -> Tensor");
  m.def("_gated_fwd(Tensor x, Tensor w_gate, Tensor w_up, int width, int act) -> Tensor");
  m.def("_gated_bwd(Tensor dh, Tensor x, Tensor w_gate, Tensor w_up, int width, int act, bool need_x, bool need_w, "
        "int dw_dtype) -> (Tensor, Tensor, Tensor)");
  m.def("linear_cross_entropy(Tensor x, Tensor weight, Tensor target, Tensor? w16, int ignore_index, int reduction) "
        "-> Tensor");
  m.def("_linear_xent_fwd(Tensor x, Tensor w, Tensor target, int width, int ignore_index, int reduction) "
        "-> (Tensor, Tensor, Tensor)");
  m.def("_linear_xent_bwd(Tensor dloss, Tensor x, Tensor w, Tensor target, Tensor lse, Tensor scale, int width, "
        "int ignore_index, bool need_x, bool need_w, int dw_dtype) -> (Tensor, Tensor)");
}
TORCH_LIBRARY_IMPL(naju, CUDA, m) {
  m.impl("layer_norm", TORCH_FN(layer_norm_cuda));
  m.impl("_layer_norm_fwd", TORCH_FN(norm_fwd_cuda));
  m.impl("_layer_norm_bwd", TORCH_FN(norm_bwd_cuda));
  m.impl("gated_linear", TORCH_FN(gated_linear_cuda));
  m.impl("_gated_fwd", TORCH_FN(gated_fwd_cuda));
  m.impl("_gated_bwd", TORCH_FN(gated_bwd_cuda));
  m.impl("linear_cross_entropy", TORCH_FN(xent_cuda));
  m.impl("_linear_xent_fwd", TORCH_FN(xent_fwd_cuda));
  m.impl("_linear_xent_bwd", TORCH_FN(xent_bwd_cuda));
}
TORCH_LIBRARY_IMPL(naju, Meta, m) {
  m.impl("layer_norm", TORCH_FN(layer_norm_meta));
  m.impl("_layer_norm_fwd", TORCH_FN(norm_fwd_meta));
  m.impl("_layer_norm_bwd", TORCH_FN(norm_bwd_meta));
  m.impl("gated_linear", TORCH_FN(gated_linear_meta));
  m.impl("_gated_fwd", TORCH_FN(gated_fwd_meta));
  m.impl("_gated_bwd", TORCH_FN(gated_bwd_meta));
  m.impl("linear_cross_entropy", TORCH_FN(xent_meta));
  m.impl("_linear_xent_fwd", TORCH_FN(xent_fwd_meta));
  m.impl("_linear_xent_bwd", TORCH_FN(xent_bwd_meta));
}
TORCH_LIBRARY_IMPL(naju, Autograd, m) {
  m.impl("layer_norm", TORCH_FN(layer_norm_autograd));
  m.impl("gated_linear", TORCH_FN(gated_linear_autograd));
  m.impl("linear_cross_entropy", TORCH_FN(xent_autograd));
  // the functions' own steps have no derivative: asked for one they raise
  for (const char* step : {"_layer_norm_fwd", "_layer_norm_bwd", "_gated_fwd", "_gated_bwd", "_linear_xent_fwd",
                           "_linear_xent_bwd"})
    m.impl(step, torch::autograd::autogradNotImplementedFallback());
}
