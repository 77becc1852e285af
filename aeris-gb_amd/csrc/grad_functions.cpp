// The differentiable calls of grad.py as nodes of torch's autograd graph: argument checks, outputs, what is kept for the backward pass, and
// the C ABI's calls on the current stream.  In C++ because a pass of a small block is bound by the host: written as
// torch.autograd.Function in Python, forward and backward pass of a [2048, 128] norm took 113 us, and its kernels 15.
#include <ATen/ATen.h>
#include <c10/hip/HIPFunctions.h>
#include <c10/hip/HIPStream.h>
#include <hip/hip_runtime.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/utils/pybind.h>

#include <unordered_set>

#include "../../include/aeris_hip.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::Node;
using torch::autograd::variable_list;
using Optional = std::optional<Tensor>;

constexpr auto BF16 = at::kBFloat16;
constexpr auto F32 = at::kFloat;

void check(int code) { TORCH_CHECK(code == AERIS_OK, "libaeris_hip error ", code, ": ", aeris_last_error()); }
int dtype_of(const Tensor& t) { return t.scalar_type() == F32 ? AERIS_F32 : AERIS_BF16; }
bool known(const Tensor& t) { return t.scalar_type() == BF16 || t.scalar_type() == F32; }
Tensor value(const Optional& t) { return t.has_value() ? *t : Tensor(); }
void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* stream() { return c10::hip::getCurrentHIPStream().stream(); }

// every tensor of a call lives on the current GPU, whose stream the call goes to
void on_current_device(std::initializer_list<std::pair<const char*, const Tensor*>> all) {
  for (const auto& [name, t] : all)
    if (t->defined()) TORCH_CHECK(t->is_cuda(), name, " must live on the GPU (the HIP kernels have no CPU fallback)");
  const auto current = c10::hip::current_device();
  for (const auto& [name, t] : all)
    if (t->defined())
      TORCH_CHECK(t->device().index() == current, name, " is on ", t->device(), "; every tensor of the call must be on the current device (cuda:", (int)current, ")");
}
bool capturing() {
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  return hipStreamIsCapturing(c10::hip::getCurrentHIPStream().stream(), &status) == hipSuccess && status != hipStreamCaptureStatusNone;
}
constexpr const char* REVERSE_ONLY = "these operators are differentiable in reverse mode only";
bool has_tangent(const Tensor& t) { return t.defined() && t._fw_grad(0).defined(); }
bool wants_grad(std::initializer_list<const Tensor*> inputs) {
  for (const Tensor* t : inputs) TORCH_CHECK(!has_tangent(*t), REVERSE_ONLY);
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor* t : inputs)
    if (t->defined() && t->requires_grad()) return true;
  return false;
}

// A captured backward pass whose graph has nodes of another stream ends the process: torch makes the streams wait for each other.  Such nodes
// are what an eager graph that is still alive has of a leaf, or what an input was made with outside the capture.
void refuse_other_streams(std::initializer_list<const Tensor*> inputs) {
  if (!capturing()) return;
  const c10::Stream here = c10::hip::getCurrentHIPStream().unwrap();
  std::vector<std::shared_ptr<Node>> todo;
  for (const Tensor* t : inputs) {
    if (!t->defined() || !t->requires_grad()) continue;
    if (t->grad_fn()) todo.push_back(t->grad_fn());
    else if (auto leaf = torch::autograd::impl::try_get_grad_accumulator(*t)) todo.push_back(leaf);
  }
  std::unordered_set<Node*> seen;
  while (!todo.empty()) {
    const std::shared_ptr<Node> node = todo.back();
    todo.pop_back();
    if (!seen.insert(node.get()).second) continue;
    const auto s = node->stream();
    TORCH_CHECK(!s || (s->id() == here.id() && s->device_index() == here.device_index()),
                "an eager graph of a tensor of this captured call is still alive on another stream (or the tensor was made there): release its result before the "
                "capture, or make it where the capture runs (torch ties that stream to the capture in the backward pass, which ends the process)");
    for (const auto& edge : node->next_edges())
      if (edge.function) todo.push_back(edge.function);
  }
}

// a result's gradient as the kernels read it: contiguous, its address a multiple of 16, without a tangent, which they would drop
Tensor incoming(const Tensor& dy) {
  TORCH_CHECK(!has_tangent(dy), REVERSE_ONLY);
  Tensor g = dy.contiguous();
  return reinterpret_cast<uintptr_t>(g.data_ptr()) & 15 ? g.clone() : g;
}
std::vector<int64_t> rows_of(const Tensor& t, int64_t columns) {
  std::vector<int64_t> shape = t.sizes().vec();
  shape.back() = columns;
  return shape;
}

// What is kept for the backward pass may come back from hooks of the caller's (torch.autograd.graph.saved_tensors_hooks).  The kernels read it by its
// address and by sizes that follow from those of dy, so it is held to them.
void check_kept(const Tensor& t, const Tensor& dy, at::IntArrayRef sizes, bool right_type) {
  TORCH_CHECK(right_type && t.device() == dy.device() && t.sizes() == sizes && t.is_contiguous(), "a tensor kept for the backward pass came back as ", t.scalar_type(), " ", t.sizes(),
              " with strides ", t.strides(), " on ", t.device(), ", not as contiguous ", sizes, " on ", dy.device(), " in the type that it was kept in");
}
void check_kept(const Tensor& t, const Tensor& dy, at::IntArrayRef sizes, at::ScalarType type = BF16) { check_kept(t, dy, sizes, t.scalar_type() == type); }

// Gradients that themselves have none: where a graph of the backward pass is asked for, they refuse to be differentiated.  Behind the node that
// refuses lie the operator's inputs and the result's gradient dy: autograd, asked for the gradients of a few tensors, runs only what leads to
// those, and would leave the term out without a word.
variable_list outgoing(variable_list grads, const Tensor& dy) {
  if (!at::GradMode::is_enabled()) return grads;
  torch::autograd::edge_list behind;
  if (const auto node = torch::autograd::get_current_node()) behind = node->next_edges();
  behind.push_back(torch::autograd::impl::gradient_edge(dy));
  const auto refusal = std::make_shared<torch::autograd::Error>("these operators are differentiable once", std::move(behind));
  for (const Tensor& t : grads)
    if (t.defined()) torch::autograd::set_history(t, refusal);
  return grads;
}
Tensor scratch(int64_t bytes, const Tensor& like) { return bytes ? at::empty({bytes}, like.options().dtype(at::kByte)) : Tensor(); }

// ---- norm and modulation

struct NormHow { int64_t kind, order; double eps; };

Tensor norm_forward(const Tensor& x, const Tensor& gamma, const Tensor& beta, const Tensor& shift, const Tensor& scale, const NormHow& how, at::ScalarType out) {
  Tensor y = at::empty(x.sizes(), x.options().dtype(out));
  if (!x.numel()) return y;
  const Tensor& mod = shift.defined() ? shift : scale;
  const int64_t stride = mod.defined() && mod.size(0) > 1 ? mod.stride(0) : 0;
  check(aeris_norm_modulate_fwd(x.data_ptr(), dtype_of(x), y.data_ptr(), dtype_of(y), gamma.data_ptr(), ptr(beta), dtype_of(gamma),
                                static_cast<const float*>(ptr(shift)), static_cast<const float*>(ptr(scale)), stride, x.size(0), x.size(1), (int)x.size(2),
                                (int)how.kind, (int)how.order, (float)how.eps, stream()));
  return y;
}

struct NormModulate : torch::autograd::Function<NormModulate> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gamma, const Optional& beta_, const Optional& shift_, const Optional& scale_, int64_t kind,
                        int64_t order, double eps, int64_t out) {
    // (a modulation row expanded over the members is copied: each member has a gradient)
    auto rows = [](const Tensor& t) { return t.defined() && t.size(0) > 1 && t.stride(0) == 0 ? t.contiguous() : t; };
    const Tensor beta = value(beta_), shift = rows(value(shift_)), scale = rows(value(scale_));
    ctx->save_for_backward({x, gamma, beta, shift, scale});
    ctx->saved_data["kind"] = kind;
    ctx->saved_data["order"] = order;
    ctx->saved_data["eps"] = eps;
    return norm_forward(x, gamma, beta, shift, scale, {kind, order, eps}, out ? F32 : BF16);
  }
  static variable_list backward(AutogradContext* ctx, variable_list given) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &gamma = saved[1];
    const Tensor dy = incoming(given[0]);
    const int64_t d = dy.size(2);
    check_kept(x, dy, dy.sizes(), known(x));
    check_kept(gamma, dy, {d}, known(gamma));
    if (saved[2].defined()) check_kept(saved[2], dy, {d}, gamma.scalar_type());
    // (modulation rows are columns of one matrix, unless a hook gave them memory of their own)
    Tensor shift = saved[3], scale = saved[4];
    for (Tensor* t : {&shift, &scale})
      if (t->defined()) {
        const bool member_rows = t->dim() == 2 && t->size(0) > 1, both = shift.defined() && scale.defined();
        if (member_rows && (t->stride(1) != 1 || t->stride(0) < d || (both && shift.strides() != scale.strides()))) *t = t->contiguous();
        TORCH_CHECK(t->device() == dy.device() && t->scalar_type() == F32 && t->dim() == 2 && t->size(1) == d && (d == 1 || t->stride(1) == 1) &&
                        (t->size(0) == 1 || t->size(0) == dy.size(0)) && (!both || shift.size(0) == scale.size(0)),
                    "modulation rows kept for the backward pass came back as ", t->scalar_type(), " ", t->sizes(), " with strides ", t->strides(), " on ", t->device());
      }
    Tensor grads[5];
    for (size_t i = 0, edge = 0; i < 5; ++i)  // (only inputs that are there have an edge)
      if (saved[i].defined() && ctx->needs_input_grad(edge++))
        grads[i] = x.numel() ? at::empty_like(saved[i], at::MemoryFormat::Contiguous) : at::zeros_like(saved[i], at::MemoryFormat::Contiguous);
    if (x.numel()) {
      const Tensor& mod = shift.defined() ? shift : scale;
      aeris_norm_modulate_grad a;
      a.x = x.data_ptr();
      a.dy = dy.data_ptr();
      a.gamma = gamma.data_ptr();
      a.beta = ptr(saved[2]);
      a.shift = static_cast<const float*>(ptr(shift));
      a.scale = static_cast<const float*>(ptr(scale));
      a.dx = ptr(grads[0]);
      a.dgamma = ptr(grads[1]);
      a.dbeta = ptr(grads[2]);
      a.dshift = static_cast<float*>(ptr(grads[3]));
      a.dscale = static_cast<float*>(ptr(grads[4]));
      a.B = x.size(0);
      a.rows_per_batch = x.size(1);
      a.d = x.size(2);
      a.mod_batch_stride = mod.defined() && mod.size(0) > 1 ? mod.stride(0) : 0;
      a.x_dtype = dtype_of(x);
      a.dy_dtype = dtype_of(dy);
      a.param_dtype = dtype_of(gamma);
      a.kind = ctx->saved_data["kind"].toInt();
      a.order = ctx->saved_data["order"].toInt();
      a.eps = ctx->saved_data["eps"].toDouble();
      const int64_t need = aeris_norm_modulate_grad_workspace_bytes(&a);
      const Tensor ws = scratch(need, x);
      check(aeris_norm_modulate_bwd(&a, ptr(ws), need, stream()));
    }
    return outgoing({grads[0], grads[1], grads[2], grads[3], grads[4], Tensor(), Tensor(), Tensor(), Tensor()}, given[0]);
  }
};

Tensor norm_modulate(const Tensor& x, const Tensor& gamma, const Optional& beta_, const Optional& shift_, const Optional& scale_, int64_t kind, int64_t order, double eps,
                     bool out_f32) {
  const Tensor beta = value(beta_), shift = value(shift_), scale = value(scale_);
  on_current_device({{"x", &x}, {"gamma", &gamma}, {"beta", &beta}, {"shift", &shift}, {"scale", &scale}});
  TORCH_CHECK(known(x) && known(gamma), "x and gamma must be bf16 or f32, got ", x.scalar_type(), " and ", gamma.scalar_type());
  TORCH_CHECK(x.dim() == 3 && x.is_contiguous(), "x must be contiguous [B, S, d], got ", x.sizes());
  const int64_t B = x.size(0), d = x.size(2);
  TORCH_CHECK(gamma.dim() == 1 && gamma.size(0) == d && gamma.is_contiguous(), "gamma must be contiguous [", d, "], got ", gamma.sizes());
  if (beta.defined())
    TORCH_CHECK(beta.dim() == 1 && beta.size(0) == d && beta.is_contiguous() && beta.scalar_type() == gamma.scalar_type(), "beta must be contiguous [", d, "] of gamma's type, got ",
                beta.scalar_type(), " ", beta.sizes());
  for (const Tensor* t : {&shift, &scale})
    if (t->defined())
      TORCH_CHECK(t->scalar_type() == F32 && t->dim() == 2 && t->size(1) == d && (t->size(0) == 1 || t->size(0) == B) && (d <= 1 || t->stride(1) == 1),
                  "shift and scale must be f32 [1, ", d, "] or [", B, ", ", d, "] with unit column stride, got ", t->scalar_type(), " ", t->sizes());
  if (shift.defined() && scale.defined())
    TORCH_CHECK(shift.sizes() == scale.sizes() && (shift.size(0) == 1 || shift.stride(0) == scale.stride(0)), "shift and scale must be of one shape and layout, got ", shift.sizes(),
                " and ", scale.sizes());
  if (!wants_grad({&x, &gamma, &beta, &shift, &scale})) return norm_forward(x, gamma, beta, shift, scale, {kind, order, eps}, out_f32 ? F32 : BF16);
  const Tensor& mod = shift.defined() ? shift : scale;
  TORCH_CHECK(!mod.defined() || mod.size(0) == 1 || (B <= 65535 && B * (d / 8) < 1 << 22), "no gradients of ", B, " members of ", d, " channels with modulation rows of their own");
  refuse_other_streams({&x, &gamma, &beta, &shift, &scale});
  return NormModulate::apply(x, gamma, beta_, shift_, scale_, kind, order, eps, (int64_t)out_f32);
}

// ---- projection

struct Sizes { int64_t M, N, K; };

// what aeris_linear_bwd and aeris_feed_forward_bwd take, so that a call whose gradients would be refused is refused itself
void check_gradients_sizes(const Sizes& s) {
  constexpr int64_t WIDE = 1 << 20, PRODUCT = 1 << 30, TILES = 1 << 24;
  TORCH_CHECK(s.M < int64_t(1) << 31 && s.N <= WIDE && s.K <= WIDE && s.N * s.K < PRODUCT && (s.M + 63) / 64 * ((s.N + 31) / 32) < TILES && (s.M + 63) / 64 * ((s.K + 63) / 64) < TILES,
              "no gradients of ", s.M, " rows of ", s.K, " -> ", s.N, " (widths up to 2^20, their product below 2^30, fewer than 2^31 rows, and fewer than 2^24 tiles of 64 x 32 of the result and of 64 x 64 of what is projected)");
}

Tensor linear_forward(const Tensor& a, const Tensor& w, const Tensor& bias, const Tensor& residual, int64_t act, at::ScalarType out, const Sizes& s, Tensor* z) {
  Tensor y = at::empty(rows_of(a, s.N), a.options().dtype(out));
  const bool bent = act == AERIS_ACT_GELU || act == AERIS_ACT_SILU;
  if (z && bent) *z = at::empty({3 * s.M * s.N}, a.options().dtype(at::kByte));
  if (!s.M) return y;
  if (!bent) {
    check(aeris_gemm_fwd(a.data_ptr(), w.data_ptr(), y.data_ptr(), ptr(bias), nullptr, ptr(residual), s.M, (int)s.N, (int)s.K, s.N, AERIS_ACT_NONE,
                         residual.defined() ? dtype_of(residual) : 0, dtype_of(y), 0, s.M, stream()));
    return y;
  }
  aeris_linear_train c;
  c.x = a.data_ptr();
  c.w = w.data_ptr();
  c.bias = ptr(bias);
  c.residual = ptr(residual);
  c.y = y.data_ptr();
  c.z = z ? ptr(*z) : nullptr;
  c.M = s.M;
  c.N = s.N;
  c.K = s.K;
  c.act = act;
  c.res_dtype = residual.defined() ? dtype_of(residual) : 0;
  c.y_dtype = dtype_of(y);
  check(aeris_linear_train_fwd(&c, stream()));
  return y;
}

struct Linear : torch::autograd::Function<Linear> {
  static Tensor forward(AutogradContext* ctx, const Tensor& a, const Tensor& w, const Optional& bias_, const Optional& residual_, int64_t act, int64_t out, int64_t M) {
    const Tensor bias = value(bias_), residual = value(residual_);
    const bool keep = a.requires_grad() || w.requires_grad() || (bias.defined() && bias.requires_grad());
    Tensor z;
    Tensor y = linear_forward(a, w, bias, residual, act, out ? F32 : BF16, {M, w.size(0), w.size(1)}, keep ? &z : nullptr);
    ctx->save_for_backward({a, w, z});
    ctx->saved_data["act"] = act;
    ctx->saved_data["bias"] = bias.defined();
    if (residual.defined()) {
      ctx->saved_data["residual_f32"] = residual.scalar_type() == F32;
      ctx->saved_data["residual_shape"] = residual.sizes().vec();
    }
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list given) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &a = saved[0], &w = saved[1], &z = saved[2];
    const int64_t act = ctx->saved_data["act"].toInt(), N = given[0].size(-1), K = w.size(-1), M = given[0].numel() / N;
    const bool has_bias = ctx->saved_data["bias"].toBool(), has_res = ctx->saved_data.count("residual_f32") != 0;  // (only inputs that are there have an edge)
    const bool need_a = ctx->needs_input_grad(0), need_w = ctx->needs_input_grad(1), need_bias = has_bias && ctx->needs_input_grad(2),
               need_res = has_res && ctx->needs_input_grad(has_bias ? 3 : 2);
    const Tensor dy = need_a || need_w || need_bias ? incoming(given[0]) : given[0].contiguous();
    check_kept(w, dy, {N, K});
    check_kept(a, dy, rows_of(dy, K));
    if (z.defined()) check_kept(z, dy, {3 * M * N}, at::kByte);
    const auto res_dtype = need_res && ctx->saved_data["residual_f32"].toBool() ? F32 : BF16;
    // dy rounded to bf16 is what the products read of an f32 dy, and what a bf16 residual gets
    // (made beside the products; alone, or where a graph of the backward pass is asked for, by torch's own cast, which is differentiable)
    const bool round_res = need_res && res_dtype == BF16 && dy.scalar_type() == F32 && act == AERIS_ACT_NONE && M && (need_a || need_w || need_bias) && !at::GradMode::is_enabled();
    Tensor da, dw, dbias, dz, dres;
    if (need_a) da = at::empty_like(a, at::MemoryFormat::Contiguous);
    if (need_w) dw = M ? at::empty_like(w) : at::zeros_like(w);
    if (need_bias) dbias = M ? at::empty({N}, w.options()) : at::zeros({N}, w.options());
    if (round_res) dz = at::empty_like(dy, dy.options().dtype(BF16));
    if (M && (need_a || need_w || need_bias)) {
      aeris_linear_grad c;
      c.dy = dy.data_ptr();
      c.x = a.data_ptr();
      c.w = w.data_ptr();
      c.z = ptr(z);
      c.dx = ptr(da);
      c.dw = ptr(dw);
      c.dbias = ptr(dbias);
      c.dz = ptr(dz);
      c.M = M;
      c.N = N;
      c.K = K;
      c.act = act;
      c.dy_dtype = dtype_of(dy);
      const int64_t need = aeris_linear_grad_workspace_bytes(&c);
      const Tensor ws = scratch(need, a);
      check(aeris_linear_bwd(&c, ptr(ws), need, stream()));
    }
    if (need_res) {
      // dy itself where it has the residual's type and shape, as torch's own addition returns it; otherwise memory of its own.  Never a view of dy: the
      // accumulation takes a tensor that nobody else holds for its own and adds the next pass's gradient into it
      const auto shape = ctx->saved_data["residual_shape"].toIntVector();
      dres = round_res ? dz : dy.to(res_dtype);
      if (dres.sizes() != at::IntArrayRef(shape)) dres = (dres.is_same(dy) ? dres.clone() : dres).view(shape);
    }
    variable_list grads = outgoing({da, dw, dbias}, given[0]);
    grads.insert(grads.end(), {dres, Tensor(), Tensor(), Tensor()});
    return grads;
  }
};

Tensor linear(const Tensor& a, const Tensor& w, const Optional& bias_, int64_t act, const Optional& residual_, bool out_f32) {
  const Tensor bias = value(bias_), residual = value(residual_);
  on_current_device({{"a", &a}, {"w", &w}, {"bias", &bias}, {"residual", &residual}});
  TORCH_CHECK(a.scalar_type() == BF16 && w.scalar_type() == BF16 && w.dim() == 2 && a.dim() >= 1 && a.is_contiguous() && w.is_contiguous() && a.size(-1) == w.size(1),
              "a must be contiguous bf16 [.., K] and w [N, K], got ", a.scalar_type(), " ", a.sizes(), " and ", w.scalar_type(), " ", w.sizes());
  const int64_t N = w.size(0), K = w.size(1);
  TORCH_CHECK(N > 0 && K > 0 && N % 8 == 0 && K % 8 == 0, "widths must be positive multiples of 8 for the gradients' products, got ", N, " and ", K);
  const int64_t M = a.numel() / K;
  if (bias.defined())
    TORCH_CHECK(bias.dim() == 1 && bias.size(0) == N && bias.scalar_type() == BF16 && bias.is_contiguous(), "bias must be contiguous bf16 [", N, "], got ", bias.scalar_type(), " ", bias.sizes());
  if (residual.defined())
    TORCH_CHECK(known(residual) && residual.numel() == M * N && residual.dim() >= 1 && residual.size(-1) == N && residual.is_contiguous(),
                "residual must be contiguous bf16 or f32 [", M, ", ", N, "], got ", residual.scalar_type(), " ", residual.sizes());
  if (!wants_grad({&a, &w, &bias, &residual})) return linear_forward(a, w, bias, residual, act, out_f32 ? F32 : BF16, {M, N, K}, nullptr);
  check_gradients_sizes({M, N, K});
  refuse_other_streams({&a, &w, &bias, &residual});
  return Linear::apply(a, w, bias_, residual_, act, (int64_t)out_f32, M);
}

// ---- gated MLP

Tensor feed_forward_forward(const Tensor& x, const Tensor& w1, const Tensor& w2, Tensor* gate_up, Tensor* h) {
  const int64_t d = w2.size(0), H = w2.size(1), M = x.numel() / d;
  Tensor y = at::empty_like(x, at::MemoryFormat::Contiguous);
  if (gate_up) *gate_up = at::empty({6 * M * H}, x.options().dtype(at::kByte));
  *h = at::empty({(M > AERIS_FEW_TOKENS ? 1 : 2) * M * H}, x.options());
  if (!M) return y;
  aeris_feed_forward c;
  c.x = x.data_ptr();
  c.w1 = w1.data_ptr();
  c.w2 = w2.data_ptr();
  c.gate_up = gate_up ? ptr(*gate_up) : nullptr;
  c.h = h->data_ptr();
  c.y = y.data_ptr();
  c.M = M;
  c.d = d;
  c.H = H;
  const int64_t need = aeris_feed_forward_workspace_bytes(&c);
  const Tensor ws = scratch(need, x);
  check(aeris_feed_forward_train_fwd(&c, ptr(ws), need, stream()));
  return y;
}

struct FeedForward : torch::autograd::Function<FeedForward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& w1, const Tensor& w2) {
    Tensor gate_up, h;
    Tensor y = feed_forward_forward(x, w1, w2, &gate_up, &h);
    ctx->save_for_backward({x, w1, w2, gate_up, h});
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list given) {
    const auto saved = ctx->get_saved_variables();
    const Tensor &x = saved[0], &w2 = saved[2];
    const Tensor dy = incoming(given[0]);
    const int64_t d = dy.size(-1), H = w2.size(-1), M = dy.numel() / d;
    check_kept(x, dy, dy.sizes());
    check_kept(saved[1], dy, {2 * H, d});
    check_kept(w2, dy, {d, H});
    check_kept(saved[3], dy, {6 * M * H}, at::kByte);
    check_kept(saved[4], dy, {(M > AERIS_FEW_TOKENS ? 1 : 2) * M * H});
    Tensor grads[3];
    for (int i = 0; i < 3; ++i)
      if (ctx->needs_input_grad(i)) grads[i] = M ? at::empty_like(saved[i], at::MemoryFormat::Contiguous) : at::zeros_like(saved[i], at::MemoryFormat::Contiguous);
    if (M) {
      aeris_feed_forward_grad c;
      c.dy = dy.data_ptr();
      c.x = x.data_ptr();
      c.w1 = saved[1].data_ptr();
      c.w2 = w2.data_ptr();
      c.gate_up = ptr(saved[3]);
      c.h = ptr(saved[4]);
      c.dx = ptr(grads[0]);
      c.dw1 = ptr(grads[1]);
      c.dw2 = ptr(grads[2]);
      c.M = M;
      c.d = d;
      c.H = H;
      const int64_t need = aeris_feed_forward_grad_workspace_bytes(&c);
      const Tensor ws = scratch(need, x);
      check(aeris_feed_forward_bwd(&c, ptr(ws), need, stream()));
    }
    return outgoing({grads[0], grads[1], grads[2]}, given[0]);
  }
};

Tensor feed_forward(const Tensor& x, const Tensor& w1, const Tensor& w2) {
  on_current_device({{"x", &x}, {"w1", &w1}, {"w2", &w2}});
  TORCH_CHECK(w2.dim() == 2 && w1.dim() == 2 && x.dim() >= 1 && x.size(-1) == w2.size(0) && w1.size(0) == 2 * w2.size(1) && w1.size(1) == w2.size(0) && x.scalar_type() == BF16 &&
                  w1.scalar_type() == BF16 && w2.scalar_type() == BF16 && x.is_contiguous() && w1.is_contiguous() && w2.is_contiguous(),
              "x must be [.., d], w1 [2H, d] and w2 [d, H], bf16 and contiguous, got ", x.scalar_type(), " ", x.sizes(), ", ", w1.scalar_type(), " ", w1.sizes(), " and ", w2.scalar_type(),
              " ", w2.sizes());
  const int64_t d = w2.size(0), H = w2.size(1);
  TORCH_CHECK(d > 0 && H > 0 && d % 8 == 0 && H % 8 == 0, "widths must be positive multiples of 8 for the gradients' products, got ", d, " and ", H);
  if (!wants_grad({&x, &w1, &w2})) {
    Tensor h;
    return feed_forward_forward(x, w1, w2, nullptr, &h);
  }
  refuse_other_streams({&x, &w1, &w2});
  return FeedForward::apply(x, w1, w2);
}

}  // namespace

PYBIND11_MODULE(aeris_grad, m) {
  const auto free = pybind11::call_guard<pybind11::gil_scoped_release>();
  m.attr("marker") = AERIS_GRAD_MARKER;  // the torch that this was built against, which build.py and grad.py look for in the file
  m.def("norm_modulate", &norm_modulate, free);
  m.def("linear", &linear, free);
  m.def("feed_forward", &feed_forward, free);
}
