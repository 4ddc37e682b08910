// torch side of the operators between and behind the quantized layers (rotary positions, query / key norms,
// linear cross entropy): argument checks, outputs and autograd nodes over the C ABI, in C++.
//
// A decoding step's rotation is 5 us of GPU work and an image batch's training step a few tens; through
// ctypes and Python autograd functions their host side took 23 and 145 to 200 us.  Nothing here
// computes: every result comes from the kernels of libfp4t.so, on torch's current stream of the tensors'
// device, and nothing synchronises.
#include <ATen/autocast_mode.h>
#include <c10/cuda/CUDAGraphsC10Utils.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/accumulate_grad.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/extension.h>

#include <array>
#include <atomic>
#include <unordered_set>

#include "../../include/fp4t.h"

namespace {

using at::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
using OptTensor = std::optional<Tensor>;

std::atomic<int64_t> g_rotary_launches{0}, g_xent_launches{0};

void check(int rc, const char* what) {
  if (rc == FP4T_OK) return;
  TORCH_CHECK_VALUE(rc != FP4T_ERR_ARG, what, ": ", fp4t_last_error());
  TORCH_CHECK(false, what, " failed (", rc, "): ", fp4t_last_error());
}
void need_cuda(const Tensor& t) {
  TORCH_CHECK_NOT_IMPLEMENTED(t.is_cuda(), "fp4t operators run on CUDA tensors only (no CPU implementation)");
}
fp4t_stream_t stream_of(const Tensor& t) { return c10::cuda::getCurrentCUDAStream(t.get_device()).stream(); }
int code(at::ScalarType t) { return t == at::kFloat ? FP4T_DT_F32 : FP4T_DT_BF16; }
bool aligned16(const Tensor& t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }
Tensor packed16(const Tensor& t) {      // contiguous and 16-byte aligned
  Tensor c = t.contiguous();
  return aligned16(c) ? c : c.clone();
}

std::string shape(const Tensor& t) {
  std::string s = "[";
  for (int64_t i = 0; i < t.dim(); ++i) s += (i ? ", " : "") + std::to_string(t.size(i));
  return s + "]";
}

// A function that differentiates once: gradients of its gradients raise when they are asked for.
variable_list once(variable_list grads, const variable_list& out_grads) {
  if (!at::GradMode::is_enabled()) return grads;
  bool wanted = false;
  for (const auto& g : out_grads) wanted = wanted || (g.defined() && g.requires_grad());
  if (!wanted) return grads;
  variable_list defined;
  for (auto& g : grads)
    if (g.defined()) {
      g = g.detach();
      g.set_requires_grad(true);
      defined.push_back(g);
    }
  auto node = std::make_shared<torch::autograd::DelayedError>("trying to differentiate twice a function that differentiates once",
                                                              (int64_t)defined.size());
  auto marked = (*node)(std::move(defined));
  size_t i = 0;
  for (auto& g : grads)
    if (g.defined()) g = marked[i++];
  return grads;
}

// A captured backward pass must not reach a leaf whose gradient accumulator belongs to the default stream, which it does
// while an eager graph of that leaf lives: that stream would be made to wait for the capturing one, which CUDA
// forbids; the capture is lost and the process can end with it.  Looked for along the edges that this pass takes,
// once per node and capture.
void refuse_eager_leaves(const Tensor& like) {
  const c10::cuda::OptionalCUDAGuard guard(like.device());
  const auto standard = c10::cuda::getDefaultCUDAStream(like.get_device());
  if (c10::cuda::getCurrentCUDAStream(like.get_device()) == standard) return;          // it cannot be captured
  if (c10::cuda::currentStreamCaptureStatusMayInitCtx() == c10::cuda::CaptureStatus::None) return;
  const auto start = torch::autograd::get_current_node();
  std::vector<torch::autograd::Node*> open{start.get()};
  std::unordered_set<torch::autograd::Node*> seen{start.get()};
  while (!open.empty()) {
    torch::autograd::Node* node = open.back();
    open.pop_back();
    for (size_t i = 0; i < node->num_outputs(); ++i) {
      torch::autograd::Node* next = node->next_edge(i).function.get();
      if (!next || !node->task_should_compute_output(i) || !seen.insert(next).second) continue;
      if (dynamic_cast<torch::autograd::AccumulateGrad*>(next)) {
        const auto stream = next->stream();
        TORCH_CHECK(!stream.has_value() || *stream != standard.unwrap(),
                    "a backward pass is captured while an eager graph of the same leaves, built on the default stream, is alive: drop the eager "
                    "graph's results first, or build it on another stream");
      }
      open.push_back(next);
    }
  }
}

// ------------------------------------------------------------------ rotary positions, query / key norms
struct Heads {
  std::array<Tensor, 2> t;
  std::array<fp4t_heads_t, 2> h{};
  int count = 0;
};

fp4t_heads_t heads_of(const Tensor& t) { return fp4t_heads_t{t.data_ptr(), t.size(2), t.stride(0), t.stride(1), t.stride(2)}; }

Heads take_heads(const char* what, at::ArrayRef<Tensor> x, const Tensor* like = nullptr) {
  TORCH_CHECK_VALUE(x.size() == 1 || x.size() == 2, what, " takes one or two tensors");
  const Tensor& first = like ? *like : x[0];
  Heads r;
  for (const Tensor& t : x) {
    need_cuda(t);
    TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat || t.scalar_type() == at::kBFloat16, what, " runs on float32 / bfloat16 tensors");
    TORCH_CHECK_VALUE(t.dim() == 4, what, " takes [batch, tokens, heads, head_dim] tensors");
    TORCH_CHECK_VALUE(t.scalar_type() == first.scalar_type() && t.device() == first.device(), what,
                      ": all tensors must have one dtype and one device");
    TORCH_CHECK_VALUE(t.size(0) == first.size(0) && t.size(1) == first.size(1) && t.size(3) == first.size(3), what,
                      ": tensors must agree in batch, tokens and head_dim");
    r.t[r.count] = t.stride(3) == 1 ? t : t.contiguous();
    r.h[r.count] = heads_of(r.t[r.count]);
    ++r.count;
  }
  const int64_t dim = first.size(3);
  TORCH_CHECK_VALUE(dim % 2 == 0 && dim >= 2 && dim <= 512, what, " needs an even head_dim of 2 to 512, got ", dim);
  return r;
}
Heads like_heads(const Heads& x) {
  Heads r;
  r.count = x.count;
  for (int i = 0; i < x.count; ++i) {
    r.t[i] = at::empty(x.t[i].sizes(), x.t[i].options());
    r.h[i] = heads_of(r.t[i]);
  }
  return r;
}

// The table of turning pairs as the modules hold it; undefined tensors: no rotation.
struct Table {
  Tensor positions, turns, axis;
  int64_t axes = 0;
  bool interleaved = false;
};
Table table_of(const OptTensor& positions, const OptTensor& turns, const OptTensor& axis, int64_t axes, bool interleaved) {
  return Table{positions.value_or(Tensor()), turns.value_or(Tensor()), axis.value_or(Tensor()), axes, interleaved};
}

fp4t_rotary_t rotary_args(const char* what, const Tensor& x, const Table& t) {
  fp4t_rotary_t r{};
  if (!t.turns.defined()) {
    TORCH_CHECK_VALUE(!t.positions.defined(), what, ": positions without a rotary table");
    return r;
  }
  TORCH_CHECK_VALUE(t.positions.defined(), what, ": a rotary table needs positions");
  const Tensor& p = t.positions;
  need_cuda(p);
  need_cuda(t.turns);
  need_cuda(t.axis);
  TORCH_CHECK_VALUE(p.scalar_type() == at::kLong || p.scalar_type() == at::kInt, what, ": positions must be int32 or int64");
  TORCH_CHECK_VALUE(p.device() == x.device() && t.turns.device() == x.device() && t.axis.device() == x.device(), what,
                    ": positions and the rotary table must be on the tensors' device");
  TORCH_CHECK_VALUE(t.turns.scalar_type() == at::kLong && t.axis.scalar_type() == at::kInt && t.turns.dim() == 1 &&
                        t.axis.sizes() == t.turns.sizes() && t.turns.is_contiguous() && t.axis.is_contiguous(),
                    what, ": the rotary table is an int64 and an int32 vector of one length");
  const int64_t batch = x.size(0), tokens = x.size(1), dim = x.size(3), turned = t.turns.numel();
  const bool flat = p.dim() == 1 && t.axes == 1;      // one axis: [tokens] will do
  const int64_t n = p.dim();
  const bool fits = flat ? p.size(0) == tokens
                         : (n == 2 || n == 3) && p.size(n - 1) == t.axes && p.size(n - 2) == tokens && (n == 2 || p.size(0) == batch || p.size(0) == 1);
  TORCH_CHECK_VALUE(fits, what, ": positions must be [tokens, ", t.axes, "] or [batch, tokens, ", t.axes, "], got ", shape(p), " for ", batch,
                    " x ", tokens, " tokens");
  TORCH_CHECK_VALUE(2 * turned <= dim, what, ": ", turned, " turning pairs do not fit head_dim ", dim);
  r.positions = p.data_ptr();
  r.positions_i64 = p.scalar_type() == at::kLong;
  r.stride_batch = n == 3 && p.size(0) > 1 ? p.stride(0) : 0;
  r.stride_token = flat ? p.stride(0) : p.stride(n - 2);
  r.stride_axis = flat ? 1 : p.stride(n - 1);
  r.axes = (int)t.axes;
  r.turned = (int)turned;
  r.interleaved = t.interleaved;
  r.turns = reinterpret_cast<const uint64_t*>(t.turns.data_ptr());
  r.axis = static_cast<const int32_t*>(t.axis.data_ptr());
  return r;
}

Heads rotate(at::ArrayRef<Tensor> in, const Table& table, bool inverse) {
  const Heads x = take_heads("rotary", in);
  const fp4t_rotary_t r = rotary_args("rotary", x.t[0], table);
  const c10::cuda::OptionalCUDAGuard guard(x.t[0].device());
  Heads y = like_heads(x);
  check(fp4t_rotary(x.h.data(), y.h.data(), x.count, code(x.t[0].scalar_type()), x.t[0].size(0), x.t[0].size(1), x.t[0].size(3), &r, inverse,
                    stream_of(x.t[0])),
        "fp4t_rotary");
  g_rotary_launches += 1;
  return y;
}

Tensor norm_weight(const Tensor& w, const Tensor& x) {
  TORCH_CHECK_VALUE(w.dim() == 1 && w.size(0) == x.size(3) && w.device() == x.device(),
                    "qk_norm_rotary: weights must be [head_dim] vectors on the tensors' device");
  return w.scalar_type() == at::kFloat && w.is_contiguous() && aligned16(w) ? w : packed16(w.to(at::kFloat));
}

Heads norm_forward(at::ArrayRef<Tensor> in, at::ArrayRef<Tensor> weights, double eps, const Table& table) {
  const Heads x = take_heads("qk_norm_rotary", in);
  TORCH_CHECK_VALUE((int)weights.size() == x.count, "qk_norm_rotary: one weight per tensor");
  const fp4t_rotary_t r = rotary_args("qk_norm_rotary", x.t[0], table);
  const c10::cuda::OptionalCUDAGuard guard(x.t[0].device());
  std::array<Tensor, 2> w;
  std::array<const float*, 2> wp{};
  for (int i = 0; i < x.count; ++i) {
    w[i] = norm_weight(weights[i], x.t[i]);
    wp[i] = static_cast<const float*>(w[i].data_ptr());
  }
  Heads y = like_heads(x);
  check(fp4t_qk_norm_rotary_forward(x.h.data(), wp.data(), (float)eps, y.h.data(), x.count, code(x.t[0].scalar_type()), x.t[0].size(0),
                                    x.t[0].size(1), x.t[0].size(3), &r, stream_of(x.t[0])),
        "fp4t_qk_norm_rotary_forward");
  g_rotary_launches += 1;
  return y;
}

std::pair<Heads, std::array<Tensor, 2>> norm_backward(at::ArrayRef<Tensor> grads, at::ArrayRef<Tensor> in, at::ArrayRef<Tensor> weights, double eps,
                                                      const Table& table) {
  const Heads x = take_heads("qk_norm_rotary", in);
  std::vector<Tensor> cast;
  for (const Tensor& g : grads) {
    need_cuda(g);
    cast.push_back(g.to(x.t[0].scalar_type()));
  }
  TORCH_CHECK_VALUE(cast.size() == in.size() && weights.size() == in.size(), "qk_norm_rotary: one gradient and one weight per tensor");
  const Heads dy = take_heads("qk_norm_rotary", cast, &x.t[0]);
  for (int i = 0; i < x.count; ++i) TORCH_CHECK_VALUE(dy.t[i].sizes() == x.t[i].sizes(), "dy must have the shapes of x");
  const fp4t_rotary_t r = rotary_args("qk_norm_rotary", x.t[0], table);
  const c10::cuda::OptionalCUDAGuard guard(x.t[0].device());
  const int64_t dim = x.t[0].size(3);
  std::array<Tensor, 2> w, dw;
  std::array<const float*, 2> wp{};
  std::array<float*, 2> dwp{};
  const auto f32 = x.t[0].options().dtype(at::kFloat);
  for (int i = 0; i < x.count; ++i) {
    w[i] = norm_weight(weights[i], x.t[i]);
    wp[i] = static_cast<const float*>(w[i].data_ptr());
    dw[i] = at::empty({dim}, f32);
    dwp[i] = static_cast<float*>(dw[i].data_ptr());
  }
  Heads dx = like_heads(x);
  const int64_t bytes = fp4t_qk_norm_rotary_backward_workspace_bytes(dim);
  TORCH_CHECK(bytes >= 0, "fp4t_qk_norm_rotary_backward_workspace_bytes: unsupported shape or device");
  const Tensor ws = at::empty({bytes}, f32.dtype(at::kByte));
  check(fp4t_qk_norm_rotary_backward(dy.h.data(), x.h.data(), wp.data(), (float)eps, dx.h.data(), dwp.data(), x.count, code(x.t[0].scalar_type()),
                                     x.t[0].size(0), x.t[0].size(1), dim, &r, ws.data_ptr(), bytes, stream_of(x.t[0])),
        "fp4t_qk_norm_rotary_backward");
  g_rotary_launches += 2;
  return {dx, dw};
}

struct RotaryFn : public torch::autograd::Function<RotaryFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const OptTensor& k, const Tensor& positions, const Tensor& turns,
                               const Tensor& axis, int64_t axes, bool interleaved) {
    std::array<Tensor, 2> x{q, k.value_or(Tensor())};
    const size_t n = k.has_value() ? 2 : 1;
    Heads y = rotate(at::ArrayRef<Tensor>(x.data(), n), Table{positions, turns, axis, axes, interleaved}, false);
    ctx->save_for_backward({positions, turns, axis});
    ctx->saved_data["layout"] = 2 * axes + interleaved;
    return n == 2 ? variable_list{y.t[0], y.t[1]} : variable_list{y.t[0]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto saved = ctx->get_saved_variables();
    const int64_t layout = ctx->saved_data["layout"].toInt();
    refuse_eager_leaves(saved[0]);
    // a rotation's transpose is the rotation back
    Heads dx = rotate(dy, Table{saved[0], saved[1], saved[2], layout / 2, (layout & 1) != 0}, true);
    return once({dx.t[0], dx.t[1], Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, dy);
  }
};

struct QKNormFn : public torch::autograd::Function<QKNormFn> {
  static variable_list forward(AutogradContext* ctx, const Tensor& q, const Tensor& k, const Tensor& wq, const Tensor& wk, const OptTensor& positions,
                               const OptTensor& turns, const OptTensor& axis, int64_t axes, bool interleaved, double eps) {
    const Table table = table_of(positions, turns, axis, axes, interleaved);
    Heads y = norm_forward({q, k}, {wq, wk}, eps, table);
    ctx->save_for_backward({q, k, wq, wk, table.positions, table.turns, table.axis});
    ctx->saved_data["layout"] = 2 * axes + interleaved;
    ctx->saved_data["eps"] = eps;
    return {y.t[0], y.t[1]};
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    const auto s = ctx->get_saved_variables();
    const int64_t layout = ctx->saved_data["layout"].toInt();
    refuse_eager_leaves(s[0]);
    auto [dx, dw] = norm_backward(dy, {s[0], s[1]}, {s[2], s[3]}, ctx->saved_data["eps"].toDouble(),
                                  Table{s[4], s[5], s[6], layout / 2, (layout & 1) != 0});
    for (int i = 0; i < 2; ++i) dw[i] = dw[i].to(s[2 + i].scalar_type());
    return once({dx.t[0], dx.t[1], dw[0], dw[1], Tensor(), Tensor(), Tensor(), Tensor(), Tensor(), Tensor()}, dy);
  }
};

variable_list list_of(const Heads& h) { return h.count == 2 ? variable_list{h.t[0], h.t[1]} : variable_list{h.t[0]}; }

// The modules' calls.  3-D tensors are [tokens, heads, head_dim].
variable_list rotary_call(Tensor q, OptTensor k, const Tensor& positions, const Tensor& turns, const Tensor& axis, int64_t axes, bool interleaved) {
  const bool flat = q.dim() == 3;
  if (flat) {
    q = q.unsqueeze(0);
    if (k.has_value()) k = k->unsqueeze(0);
  }
  variable_list y = RotaryFn::apply(q, k, positions, turns, axis, axes, interleaved);
  if (flat)
    for (auto& t : y) t = t.squeeze(0);
  return y;
}
variable_list qk_norm_call(Tensor q, Tensor k, const Tensor& wq, const Tensor& wk, const OptTensor& positions, const OptTensor& turns,
                           const OptTensor& axis, int64_t axes, bool interleaved, double eps) {
  const bool flat = q.dim() == 3;
  if (flat) {
    q = q.unsqueeze(0);
    k = k.unsqueeze(0);
  }
  variable_list y = QKNormFn::apply(q, k, wq, wk, positions, turns, axis, axes, interleaved, eps);
  if (flat)
    for (auto& t : y) t = t.squeeze(0);
  return y;
}

// ------------------------------------------------------------------ linear cross entropy
struct Rows {
  Tensor t;
  int64_t ld;
};
Rows take_rows(const Tensor& t, const char* name) {
  need_cuda(t);
  TORCH_CHECK_VALUE(t.dim() == 2 && t.scalar_type() == at::kBFloat16, "linear_cross_entropy: ", name, " must be a 2-D bfloat16 tensor");
  const int64_t dim = t.size(1), ld = t.size(0) > 1 ? t.stride(0) : dim;
  if (t.stride(1) == 1 && ld % 8 == 0 && ld >= dim && aligned16(t)) return {t, ld};
  return {packed16(t), dim};
}
struct XentArgs {
  Rows h, w;
  Tensor bias, target;
  int64_t T, D, V;
};
XentArgs xent_args(const Tensor& hidden, const Tensor& weight, const Tensor& bias, const Tensor& target, int64_t reduction) {
  XentArgs a{take_rows(hidden, "hidden"), take_rows(weight, "weight"), Tensor(), Tensor(), hidden.size(0), hidden.size(1), weight.size(0)};
  need_cuda(target);
  TORCH_CHECK_VALUE(weight.size(1) == a.D, "linear_cross_entropy: hidden is ", a.D, " wide, weight ", weight.size(1));
  TORCH_CHECK_VALUE(a.D % 8 == 0 && a.D > 0, "linear_cross_entropy needs a width that is a multiple of 8, got ", a.D);
  TORCH_CHECK_VALUE(a.V > 0, "linear_cross_entropy: the vocabulary is empty");
  TORCH_CHECK_VALUE(target.dim() == 1 && target.size(0) == a.T && target.scalar_type() == at::kLong, "linear_cross_entropy: target must be int64 [",
                    a.T, "]");
  TORCH_CHECK_VALUE(reduction >= FP4T_XENT_NONE && reduction <= FP4T_XENT_SUM, "linear_cross_entropy: unknown reduction");
  if (bias.defined()) {
    need_cuda(bias);
    TORCH_CHECK_VALUE(bias.dim() == 1 && bias.size(0) == a.V && (bias.scalar_type() == at::kFloat || bias.scalar_type() == at::kBFloat16),
                      "linear_cross_entropy: bias must be float32 or bfloat16 [", a.V, "]");
    TORCH_CHECK_VALUE(bias.device() == hidden.device(), "linear_cross_entropy: all tensors must be on one device");
    a.bias = packed16(bias);
  }
  TORCH_CHECK_VALUE(weight.device() == hidden.device() && target.device() == hidden.device(),
                    "linear_cross_entropy: all tensors must be on one device");
  a.target = target.contiguous();
  return a;
}
const void* ptr(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

// -> loss ([] or, without a reduction, [T]), lse [T], count []
std::array<Tensor, 3> xent_forward(const Tensor& hidden, const Tensor& weight, const Tensor& bias, const Tensor& target, int64_t ignore,
                                   int64_t reduction, int64_t status) {
  const XentArgs a = xent_args(hidden, weight, bias, target, reduction);
  const c10::cuda::OptionalCUDAGuard guard(hidden.device());
  const auto f32 = hidden.options().dtype(at::kFloat);
  Tensor lse = at::empty({a.T}, f32), count = at::empty({}, f32);
  const std::vector<int64_t> dims = reduction == FP4T_XENT_NONE ? std::vector<int64_t>{a.T} : std::vector<int64_t>{};
  if (a.T == 0) {
    count.zero_();
    return {at::full(dims, reduction == FP4T_XENT_MEAN ? NAN : 0.0, f32), lse, count};
  }
  Tensor loss = at::empty(dims, f32);
  const int64_t bytes = fp4t_linear_xent_forward_workspace_bytes(a.T, a.D, a.V);
  if (bytes < 0) check(FP4T_ERR_ARG, "fp4t_linear_xent_forward_workspace_bytes");
  const Tensor ws = at::empty({bytes}, f32.dtype(at::kByte));
  check(fp4t_linear_xent_forward(a.h.t.data_ptr(), a.h.ld, a.w.t.data_ptr(), a.w.ld, ptr(a.bias), a.bias.defined() ? code(a.bias.scalar_type()) : 0,
                                 static_cast<const int64_t*>(a.target.data_ptr()), a.T, a.D, a.V, ignore, (int)reduction,
                                 static_cast<float*>(loss.data_ptr()), static_cast<float*>(lse.data_ptr()), static_cast<float*>(count.data_ptr()),
                                 ws.data_ptr(), bytes, reinterpret_cast<int32_t*>(status), stream_of(hidden)),
        "fp4t_linear_xent_forward");
  g_xent_launches += 1 + 2 * ((a.T + 16383) / 16384);
  return {loss, lse, count};
}

// -> dh, dw, db in the dtypes given; undefined where none is
std::array<Tensor, 3> xent_backward(Tensor grad, const Tensor& hidden, const Tensor& weight, const Tensor& bias, const Tensor& target,
                                    const Tensor& lse, int64_t ignore, int64_t reduction, std::array<std::optional<at::ScalarType>, 3> want,
                                    int64_t status) {
  const XentArgs a = xent_args(hidden, weight, bias, target, reduction);
  need_cuda(grad);
  need_cuda(lse);
  grad = grad.to(at::kFloat).contiguous();
  TORCH_CHECK_VALUE(grad.numel() == (reduction == FP4T_XENT_NONE ? a.T : 1) && lse.numel() == a.T && lse.scalar_type() == at::kFloat &&
                        lse.is_contiguous(),
                    "linear_cross_entropy: grad_loss must have the shape of the loss, lse that of the forward's");
  const c10::cuda::OptionalCUDAGuard guard(hidden.device());
  const std::array<std::vector<int64_t>, 3> shapes{std::vector<int64_t>{a.T, a.D}, std::vector<int64_t>{a.V, a.D}, std::vector<int64_t>{a.V}};
  std::array<Tensor, 3> out;
  std::array<int, 3> dt{};
  int wanted = 0;
  for (int i = 0; i < 3; ++i) {
    if (!want[i].has_value()) continue;
    TORCH_CHECK_VALUE(*want[i] == at::kFloat || *want[i] == at::kBFloat16, "linear_cross_entropy: gradients are float32 or bfloat16");
    const auto opt = hidden.options().dtype(*want[i]);
    out[i] = a.T == 0 ? at::zeros(shapes[i], opt) : at::empty(shapes[i], opt);
    dt[i] = code(*want[i]);
    ++wanted;
  }
  if (a.T == 0 || wanted == 0) return out;
  const int64_t bytes = fp4t_linear_xent_backward_workspace_bytes(a.T, a.D, a.V, out[0].defined(), out[1].defined(), out[2].defined());
  TORCH_CHECK(bytes >= 0, "fp4t_linear_xent_backward_workspace_bytes: unsupported shape or device");
  const Tensor ws = at::empty({bytes}, hidden.options().dtype(at::kByte));
  check(fp4t_linear_xent_backward(static_cast<const float*>(grad.data_ptr()), a.h.t.data_ptr(), a.h.ld, a.w.t.data_ptr(), a.w.ld, ptr(a.bias),
                                  a.bias.defined() ? code(a.bias.scalar_type()) : 0, static_cast<const int64_t*>(a.target.data_ptr()),
                                  static_cast<const float*>(lse.data_ptr()), a.T, a.D, a.V, ignore, (int)reduction, const_cast<void*>(ptr(out[0])),
                                  dt[0], const_cast<void*>(ptr(out[1])), dt[1], const_cast<void*>(ptr(out[2])), dt[2], ws.data_ptr(), bytes,
                                  reinterpret_cast<int32_t*>(status), stream_of(hidden)),
        "fp4t_linear_xent_backward");
  g_xent_launches += 2 + wanted;
  return out;
}

Tensor operand(const Tensor& t, const char* name) {
  if (t.scalar_type() == at::kBFloat16) return t;
  TORCH_CHECK_VALUE(t.scalar_type() == at::kFloat && at::autocast::is_autocast_enabled(at::kCUDA) &&
                        at::autocast::get_autocast_dtype(at::kCUDA) == at::kBFloat16,
                    "linear_cross_entropy: ", name, " is ", t.scalar_type(), "; it takes bfloat16 (float32 too under bfloat16 autocast)");
  need_cuda(t);
  return t.to(at::kBFloat16);
}

struct XentFn : public torch::autograd::Function<XentFn> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const OptTensor& bias, const Tensor& target, int64_t ignore,
                        int64_t reduction, int64_t status) {
    const Tensor h = operand(hidden, "hidden").reshape({-1, hidden.size(-1)}), w = operand(weight, "weight"), t = target.reshape({-1});
    const Tensor b = bias.value_or(Tensor());
    auto [loss, lse, count] = xent_forward(h, w, b, t, ignore, reduction, status);
    ctx->save_for_backward({h, w, b, t, lse});
    ctx->saved_data["shape"] = hidden.sizes().vec();
    ctx->saved_data["args"] = std::vector<int64_t>{ignore, reduction, status, (int64_t)hidden.scalar_type(), (int64_t)weight.scalar_type()};
    return reduction == FP4T_XENT_NONE && target.dim() != 1 ? loss.view(target.sizes()) : loss;
  }
  static variable_list backward(AutogradContext* ctx, variable_list grad) {
    const auto s = ctx->get_saved_variables();
    const auto args = ctx->saved_data["args"].toIntVector();
    refuse_eager_leaves(s[0]);
    std::array<std::optional<at::ScalarType>, 3> want;
    if (ctx->needs_input_grad(0)) want[0] = (at::ScalarType)args[3];
    if (ctx->needs_input_grad(1)) want[1] = (at::ScalarType)args[4];
    if (s[2].defined() && ctx->needs_input_grad(2)) want[2] = s[2].scalar_type();
    auto out = xent_backward(grad[0].reshape({-1}), s[0], s[1], s[2], s[3], s[4], args[0], args[1], want, args[2]);
    if (out[0].defined()) out[0] = out[0].view(ctx->saved_data["shape"].toIntVector());
    return once({out[0], out[1], out[2], Tensor(), Tensor(), Tensor(), Tensor()}, grad);
  }
};

Tensor xent_call(const Tensor& hidden, const Tensor& weight, const OptTensor& bias, const Tensor& target, int64_t ignore, int64_t reduction,
                 int64_t status) {
  TORCH_CHECK_VALUE(hidden.dim() >= 1 && weight.dim() == 2 && target.sizes() == hidden.sizes().slice(0, hidden.dim() - 1),
                    "linear_cross_entropy takes hidden [..., D], weight [V, D] and target [...], got ", shape(hidden), ", ", shape(weight), " and ",
                    shape(target), " (", target.dim(), " dimensions)");
  return XentFn::apply(hidden, weight, bias, target, ignore, reduction, status);
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  using Release = py::call_guard<py::gil_scoped_release>;
  m.def("rotary_call", &rotary_call, Release());
  m.def("qk_norm_call", &qk_norm_call, Release());
  m.def("xent_call", &xent_call, Release());
  m.def("rotary", [](const variable_list& x, const OptTensor& positions, const OptTensor& turns, const OptTensor& axis, int64_t axes, bool interleaved,
                     bool inverse) {
    at::AutoGradMode off(false);
    return list_of(rotate(x, table_of(positions, turns, axis, axes, interleaved), inverse));
  }, Release());
  m.def("qk_norm_forward", [](const variable_list& x, const variable_list& w, double eps, const OptTensor& positions, const OptTensor& turns,
                              const OptTensor& axis, int64_t axes, bool interleaved) {
    at::AutoGradMode off(false);
    return list_of(norm_forward(x, w, eps, table_of(positions, turns, axis, axes, interleaved)));
  }, Release());
  m.def("qk_norm_backward", [](const variable_list& dy, const variable_list& x, const variable_list& w, double eps, const OptTensor& positions,
                               const OptTensor& turns, const OptTensor& axis, int64_t axes, bool interleaved) {
    at::AutoGradMode off(false);
    auto [dx, dw] = norm_backward(dy, x, w, eps, table_of(positions, turns, axis, axes, interleaved));
    return std::make_pair(list_of(dx), variable_list(dw.begin(), dw.begin() + dx.count));
  }, Release());
  m.def("xent_forward", [](const Tensor& h, const Tensor& w, const OptTensor& b, const Tensor& t, int64_t ignore, int64_t reduction, int64_t status) {
    at::AutoGradMode off(false);
    auto r = xent_forward(h, w, b.value_or(Tensor()), t, ignore, reduction, status);
    return std::make_tuple(r[0], r[1], r[2]);
  }, Release());
  m.def("xent_backward", [](const Tensor& grad, const Tensor& h, const Tensor& w, const OptTensor& b, const Tensor& t, const Tensor& lse, int64_t ignore,
                            int64_t reduction, std::optional<at::ScalarType> dh, std::optional<at::ScalarType> dw, std::optional<at::ScalarType> db,
                            int64_t status) {
    at::AutoGradMode off(false);
    auto r = xent_backward(grad, h, w, b.value_or(Tensor()), t, lse, ignore, reduction, {dh, dw, db}, status);
    std::array<OptTensor, 3> out;
    for (int i = 0; i < 3; ++i)
      if (r[i].defined()) out[i] = r[i];
    return std::make_tuple(out[0], out[1], out[2]);
  }, Release());
  m.def("launches", [] { return std::make_pair(g_rotary_launches.load(), g_xent_launches.load()); });
}
