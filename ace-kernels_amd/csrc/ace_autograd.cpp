// The autograd node of hip_mi355x in C++: the host side of one loss call
// (output allocation, the ace_forward launch, the backward node and its
// ace_backward launch) without the Python autograd Function, for call
// signatures whose arguments are fixed (ace_kernels/impls/hip_mi355x.py:
// _Call); and the same for several levels in one launch per direction
// (ace_kernels/levels.py).  It mirrors the reference's `_V6Loss` autograd Function
// (src/ace_kernels/impls/v6_triton.py:93-111): saved for backward are the
// input, the target and coef / d / jac; the backward returns d input only.
//
// The kernels are reached through the C-ABI of libace_hip.so, by the entry
// points that the Python loader hands over (set_entry_points), so that this
// module and the ctypes binding drive the same loaded library.  Host code
// only: it builds with g++ against torch's headers.
//
// The vocabulary losses (ace_kernels/vocab.py), the balance loss
// (ace_kernels/balance.py), the token log probabilities (ace_kernels/logprobs.py) and
// the experts' operators (ace_kernels/experts.py) have their calls and nodes here
// too, for any arguments: the Python side checks them, nothing is remembered between
// calls.
#include <ATen/DeviceGuard.h>
#include <c10/core/AutogradState.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/extension.h>

#include <c10/hip/HIPStream.h>

#include <atomic>
#include <initializer_list>
#include <memory>
#include <stdexcept>
#include <string>
#include <vector>

#include "ace_hip.h"

namespace {

using torch::autograd::Node;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

using ForwardFn = decltype(&ace_forward);
using BackwardFn = decltype(&ace_backward);
using ErrorFn = decltype(&ace_error_string);

std::atomic<ForwardFn> g_forward{nullptr};
std::atomic<BackwardFn> g_backward{nullptr};
std::atomic<ErrorFn> g_error{nullptr};

// The arguments of ace_forward / ace_backward that a call signature fixes.
// Device pointers (tables, class weights, workspace) belong to buffers the
// Python side keeps for the life of the process.
struct Signature {
  int x_dtype = 0, target_kind = 0, num_bins = 0, binning = 0, activation = 0;
  int include_background = 0, ignore_empty = 0, reduction = 0, right = 0;
  int64_t batch = 0, channels = 0, voxels = 0;
  float empty_weight = 0.0f;
  const float* class_weight = nullptr;
  const float* bin_table = nullptr;
  const float* centre_table = nullptr;
  void* workspace = nullptr;
  size_t workspace_bytes = 0;
  // `saved` (float32): coef [B, C', K] at 0, d at o_d ([B, C', K], soft
  // [2, B, C', K]: its float32 rounding and remainder), jac [B, C'] at o_jac,
  // and the per-class errors at o_pc unless they are the returned loss
  int64_t n_saved = 0, o_d = 0, o_jac = 0, o_pc = 0;
  bool reduced = true, soft = false;
  std::vector<int64_t> loss_shape;
};

[[noreturn]] void fail(int rc, const char* what) {
  const ErrorFn err = g_error.load(std::memory_order_relaxed);
  throw std::runtime_error(std::string(what) + " failed with code " + std::to_string(rc) + ": " +
                           (err ? err(rc) : "unknown error"));
}

hipStream_t current_stream(const at::Tensor& t) {
  return c10::hip::getCurrentHIPStream(t.device().index()).stream();
}

float* at_offset(const at::Tensor& base, int64_t bytes) {
  return reinterpret_cast<float*>(static_cast<char*>(base.data_ptr()) + bytes);
}

struct AceLossBackward : public Node {
  explicit AceLossBackward(std::shared_ptr<const Signature> s) : sig(std::move(s)) {}

  std::string name() const override { return "AceLossBackward"; }

  variable_list apply(variable_list&& grads) override {
    const Signature& s = *sig;
    at::Tensor x = x_.unpack();
    at::Tensor saved = saved_.unpack();
    at::Tensor target = s.soft ? target_.unpack() : at::Tensor();
    const at::Tensor& g = grads[0];
    if (!g.defined()) return {at::Tensor()};
    at::Tensor go = g;
    if (go.scalar_type() != at::kFloat || !go.is_contiguous()) go = go.to(at::kFloat).contiguous();
    at::Tensor dx = at::empty_like(x, at::MemoryFormat::Contiguous);
    const BackwardFn bwd = g_backward.load(std::memory_order_relaxed);
    if (!bwd) throw std::runtime_error("ace_autograd: entry points not set");
    const int rc = bwd(x.data_ptr(), s.x_dtype, s.soft ? target.data_ptr() : nullptr, s.target_kind,
                       s.batch, s.channels, s.voxels, s.num_bins, s.binning, s.activation,
                       s.include_background, s.right, s.bin_table, s.centre_table,
                       at_offset(saved, 0), at_offset(saved, s.o_d), at_offset(saved, s.o_jac),
                       go.data_ptr<float>(), s.reduced ? 0 : 1, dx.data_ptr(), current_stream(x));
    if (rc) fail(rc, "ace_backward");
    return {dx};
  }

  void release_variables() override {
    x_.reset_data();
    target_.reset_data();
    saved_.reset_data();
  }

  std::shared_ptr<const Signature> sig;
  SavedVariable x_, target_, saved_;
};

// The loss of one call of signature `s` (input and target contiguous, of
// the signature's shapes and dtypes: the Python caller checks), with a
// backward node when the input needs a gradient.
at::Tensor ace_loss(const at::Tensor& x, const at::Tensor& target,
                    const std::shared_ptr<Signature>& sig) {
  const Signature& s = *sig;
  const ForwardFn fwd = g_forward.load(std::memory_order_relaxed);
  if (!fwd) throw std::runtime_error("ace_autograd: entry points not set");
  const c10::DeviceGuard guard(x.device());  // the C-ABI launches on the current device
  const auto opts = x.options().dtype(at::kFloat).requires_grad(false);
  at::Tensor saved = at::empty({s.n_saved}, opts);
  at::Tensor loss = at::empty(s.loss_shape, opts);
  float* lp = loss.data_ptr<float>();
  const int rc = fwd(x.data_ptr(), s.x_dtype, target.data_ptr(), s.target_kind, s.batch, s.channels,
                     s.voxels, s.num_bins, s.binning, s.activation, s.include_background,
                     s.ignore_empty, s.reduction, s.right, s.empty_weight, s.class_weight,
                     s.bin_table, s.centre_table, s.workspace, s.workspace_bytes,
                     at_offset(saved, 0), at_offset(saved, s.o_d), at_offset(saved, s.o_jac),
                     s.reduced ? at_offset(saved, s.o_pc) : lp, s.reduced ? lp : nullptr, nullptr,
                     current_stream(x));
  if (rc) fail(rc, "ace_forward");
  if (torch::autograd::compute_requires_grad(x)) {
    auto node = std::shared_ptr<AceLossBackward>(new AceLossBackward(sig),
                                                 torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->x_ = SavedVariable(x, false);
    if (s.soft) node->target_ = SavedVariable(target, false);
    node->saved_ = SavedVariable(saved, false);
    torch::autograd::set_history(loss, node);
  }
  return loss;
}

// ---------------------------------------------------------------- levels
// Several levels of one loss in one launch per direction (the Python
// counterpart is ace_kernels/levels.py: _HipLevelsLoss): the arguments of
// ace_forward_levels / ace_backward_levels that a levels signature fixes.
// Every level has the same batch, channels and configuration; `voxels`
// holds each level's count.  Each level's coef / d / jac (and per-class
// errors unless they are its loss) sit in one float32 allocation, `n_saved`
// floats per level at the same offsets as in Signature.
struct LevelSignature {
  int x_dtype = 0, num_bins = 0, binning = 0, include_background = 0, ignore_empty = 0;
  int reduction = 0, right = 0;
  int64_t batch = 0, channels = 0;
  float empty_weight = 0.0f;
  const float* class_weight = nullptr;
  const float* bin_table = nullptr;
  const float* centre_table = nullptr;
  void* workspace = nullptr;
  size_t workspace_bytes = 0;
  std::vector<int64_t> voxels;
  int64_t n_saved = 0, o_d = 0, o_jac = 0, o_pc = 0;
  bool reduced = true, soft = false;
  std::vector<int64_t> loss_shape;
};

using ForwardLevelsFn = decltype(&ace_forward_levels);
using BackwardLevelsFn = decltype(&ace_backward_levels);
std::atomic<ForwardLevelsFn> g_forward_levels{nullptr};
std::atomic<BackwardLevelsFn> g_backward_levels{nullptr};

struct AceLevelsBackward : public Node {
  explicit AceLevelsBackward(std::shared_ptr<const LevelSignature> s) : sig(std::move(s)) {}

  std::string name() const override { return "AceLevelsBackward"; }

  variable_list apply(variable_list&& grads) override {
    const LevelSignature& s = *sig;
    const size_t n = s.voxels.size();
    const BackwardLevelsFn bwd = g_backward_levels.load(std::memory_order_relaxed);
    if (!bwd) throw std::runtime_error("ace_autograd: entry points not set");
    at::Tensor saved = saved_.unpack();
    std::vector<at::Tensor> xs(n), keep(n);
    std::vector<AceBwdLevel> lv(n);
    variable_list out(n);
    const at::Tensor* ref = nullptr;  // a defined upstream gradient: the shape of any missing one
    for (const at::Tensor& g : grads)
      if (g.defined()) ref = &g;
    if (!ref) return out;
    for (size_t i = 0; i < n; ++i) {
      xs[i] = xs_[i].unpack();
      at::Tensor target = s.soft ? ts_[i].unpack() : at::Tensor();
      at::Tensor go = grads[i].defined() ? grads[i] : at::zeros_like(*ref);
      if (go.scalar_type() != at::kFloat || !go.is_contiguous()) go = go.to(at::kFloat).contiguous();
      keep[i] = go;
      out[i] = at::empty_like(xs[i], at::MemoryFormat::Contiguous);
      const int64_t base = (int64_t)i * s.n_saved * 4;
      lv[i] = AceBwdLevel{xs[i].data_ptr(), s.soft ? target.data_ptr() : nullptr, s.voxels[i],
                          at_offset(saved, base), at_offset(saved, base + s.o_d),
                          at_offset(saved, base + s.o_jac), go.data_ptr<float>(),
                          out[i].data_ptr()};
    }
    const int rc = bwd((int)n, lv.data(), s.x_dtype, s.batch, s.channels, s.num_bins, s.binning,
                       s.include_background, s.right, s.reduced ? 0 : 1, s.bin_table,
                       s.centre_table, current_stream(xs[0]));
    if (rc) fail(rc, "ace_backward_levels");
    for (size_t i = 0; i < n; ++i)
      if (!should_compute_output(i)) out[i] = at::Tensor();
    return out;
  }

  void release_variables() override {
    for (auto& v : xs_) v.reset_data();
    for (auto& v : ts_) v.reset_data();
    saved_.reset_data();
  }

  std::shared_ptr<const LevelSignature> sig;
  std::vector<SavedVariable> xs_, ts_;
  SavedVariable saved_;
};

// The loss of every level from one ace_forward_levels launch, with one
// backward node for all of them when an input needs a gradient.  Inputs and
// targets are contiguous, of the signature's shapes and dtypes (the Python
// caller checks).
std::vector<at::Tensor> ace_loss_levels(const std::vector<at::Tensor>& xs,
                                        const std::vector<at::Tensor>& targets,
                                        const std::shared_ptr<LevelSignature>& sig) {
  const LevelSignature& s = *sig;
  const size_t n = s.voxels.size();
  if (xs.size() != n || targets.size() != n)
    throw std::invalid_argument("ace_loss_levels: one input and one target per level");
  const ForwardLevelsFn fwd = g_forward_levels.load(std::memory_order_relaxed);
  if (!fwd) throw std::runtime_error("ace_autograd: entry points not set");
  const c10::DeviceGuard guard(xs[0].device());
  const auto opts = xs[0].options().dtype(at::kFloat).requires_grad(false);
  at::Tensor saved = at::empty({(int64_t)n * s.n_saved}, opts);
  std::vector<at::Tensor> losses(n);
  std::vector<AceFwdLevel> lv(n);
  for (size_t i = 0; i < n; ++i) {
    losses[i] = at::empty(s.loss_shape, opts);
    float* lp = losses[i].data_ptr<float>();
    const int64_t base = (int64_t)i * s.n_saved * 4;
    lv[i] = AceFwdLevel{xs[i].data_ptr(), targets[i].data_ptr(), s.voxels[i],
                        at_offset(saved, base), at_offset(saved, base + s.o_d),
                        at_offset(saved, base + s.o_jac),
                        s.reduced ? at_offset(saved, base + s.o_pc) : lp,
                        s.reduced ? lp : nullptr};
  }
  const int rc = fwd((int)n, lv.data(), s.x_dtype, s.batch, s.channels, s.num_bins, s.binning,
                     s.include_background, s.ignore_empty, s.reduction, s.right, s.empty_weight,
                     s.class_weight, s.bin_table, s.centre_table, s.workspace, s.workspace_bytes,
                     current_stream(xs[0]));
  if (rc) fail(rc, "ace_forward_levels");
  if (torch::autograd::compute_requires_grad(at::ArrayRef<at::Tensor>(xs))) {
    auto node = std::shared_ptr<AceLevelsBackward>(new AceLevelsBackward(sig),
                                                   torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(at::ArrayRef<at::Tensor>(xs)));
    for (size_t i = 0; i < n; ++i) {
      node->xs_.emplace_back(xs[i], false);
      node->ts_.emplace_back(s.soft ? targets[i] : at::Tensor(), false);
    }
    node->saved_ = SavedVariable(saved, false);
    torch::autograd::set_history(losses, node);
  }
  return losses;
}

// ------------------------------------------------- language-model losses
std::atomic<decltype(&ace_vocab_saved_bytes)> g_vocab_saved{nullptr};
std::atomic<decltype(&ace_vocab_workspace_bytes)> g_vocab_workspace{nullptr};
std::atomic<decltype(&ace_vocab_forward)> g_vocab_forward{nullptr};
std::atomic<decltype(&ace_vocab_backward)> g_vocab_backward{nullptr};
std::atomic<decltype(&ace_balance_workspace_bytes)> g_balance_workspace{nullptr};
std::atomic<decltype(&ace_balance_forward)> g_balance_forward{nullptr};
std::atomic<decltype(&ace_balance_backward)> g_balance_backward{nullptr};

int dtype_code(const at::Tensor& t) {
  switch (t.scalar_type()) {
    case at::kFloat: return ACE_F32;
    case at::kBFloat16: return ACE_BF16;
    case at::kHalf: return ACE_F16;
    default: throw std::invalid_argument("float32, bfloat16 or float16 tensors only");
  }
}

// t contiguous, its memory holding its values: not their negatives, as the memory of
// a tensor with the negative bit (the imaginary part of a conjugate) does.
at::Tensor plain(const at::Tensor& t) {
  return t.is_neg() ? t.resolve_neg().contiguous() : t.contiguous();
}

// That and starting at a multiple of 16 bytes.
at::Tensor dense(const at::Tensor& t) {
  at::Tensor c = plain(t);
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 ? c.clone() : c;
}

at::Tensor scratch(const at::Tensor& like, size_t bytes) {
  return at::empty({(int64_t)bytes}, like.options().dtype(at::kByte).requires_grad(false));
}

at::Tensor float32(const at::Tensor& g) {
  return g.defined() ? plain(g.to(at::kFloat)) : at::Tensor();
}

// Gradients of a backward that is itself recorded (create_graph) refuse to be
// differentiated again, rather than pass as constants.
void refuse_second_derivative(variable_list& out, torch::autograd::edge_list inputs,
                              const char* what) {
  if (!at::GradMode::is_enabled()) return;
  auto node = std::make_shared<torch::autograd::Error>(
      std::string(what) + " can be differentiated only once", std::move(inputs));
  for (at::Tensor& t : out)
    if (t.defined()) torch::autograd::set_history(t, node);
}
void refuse_second_derivative(variable_list& out, const variable_list& inputs, const char* what) {
  if (!at::GradMode::is_enabled()) return;
  refuse_second_derivative(out, torch::autograd::collect_next_edges(inputs), what);
}

// The nodes know no forward-mode derivative: a tensor that carries a tangent is
// refused, as its result would come without one.
void refuse_tangents(std::initializer_list<at::Tensor> inputs, const char* what) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  for (const at::Tensor& t : inputs)
    TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !t._fw_grad(/*level=*/0).defined(), what,
                                " has no forward-mode derivative");
}

struct VocabLossBackward : public Node {
  std::string name() const override { return "VocabLossBackward"; }

  variable_list apply(variable_list&& grads) override {
    variable_list out(2);
    const at::Tensor& gl = grads[0];
    const at::Tensor gc = grads.size() > 1 ? grads[1] : at::Tensor();
    if (!gl.defined() && !gc.defined()) return out;
    refuse_tangents({gl, gc}, "vocab_loss's gradient");
    const at::Tensor hidden = hidden_.unpack(), weight = weight_.unpack(), saved = saved_.unpack();
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(hidden.device());
      const at::Tensor x = dense(hidden.reshape({-1, size})), w = dense(weight);
      const at::Tensor go = float32(gl), co = float32(gc);
      if (task_should_compute_output(0))
        out[0] = at::empty(hidden.sizes(), hidden.options().requires_grad(false));
      if (task_should_compute_output(1))
        out[1] = at::empty(weight.sizes(), weight.options().requires_grad(false));
      const int code = dtype_code(hidden);
      const at::Tensor ws = scratch(hidden, g_vocab_workspace.load()(code, tokens, size, vocab, 1));
      const int rc = g_vocab_backward.load()(
          x.data_ptr(), w.data_ptr(), code, tokens, size, vocab, reduction, saved.data_ptr(),
          go.defined() ? go.data_ptr<float>() : nullptr,
          co.defined() ? co.data_ptr<float>() : nullptr,
          out[0].defined() ? out[0].data_ptr() : nullptr,
          out[1].defined() ? out[1].data_ptr() : nullptr, ws.data_ptr(), (size_t)ws.numel(),
          current_stream(hidden));
      if (rc) fail(rc, "ace_vocab_backward");
    }
    refuse_second_derivative(out, {hidden, weight, gl, gc}, "vocab_loss");
    return out;
  }

  void release_variables() override {
    hidden_.reset_data();
    weight_.reset_data();
    saved_.reset_data();
  }

  int64_t tokens = 0, size = 0, vocab = 0;
  int reduction = 0;
  SavedVariable hidden_, weight_, saved_;
};

// (loss) or (loss, confidence, correct) of checked arguments.
std::vector<at::Tensor> vocab_loss(const at::Tensor& hidden, const at::Tensor& weight,
                                   const at::Tensor& labels, int64_t ignore_index, int reduction,
                                   bool scores) {
  if (!g_vocab_forward.load()) throw std::runtime_error("ace_autograd: entry points not set");
  refuse_tangents({hidden, weight}, "vocab_loss");
  const bool record = torch::autograd::compute_requires_grad(hidden, weight);
  const c10::DeviceGuard guard(hidden.device());
  std::vector<at::Tensor> out;
  at::Tensor saved;
  const int64_t size = weight.size(1), vocab = weight.size(0), tokens = labels.numel();
  {
    const at::NoGradGuard no_grad;
    const at::Tensor x = dense(hidden.reshape({-1, size})), w = dense(weight);
    const at::Tensor y = plain(labels.to(at::kLong));
    const auto f32 = hidden.options().dtype(at::kFloat).requires_grad(false);
    const int code = dtype_code(hidden);
    out.push_back(reduction == ACE_RED_NONE ? at::empty(labels.sizes(), f32) : at::empty({}, f32));
    if (scores)
      for (int i = 0; i < 2; ++i) out.push_back(at::empty(labels.sizes(), f32));
    saved = scratch(hidden, g_vocab_saved.load()(tokens));
    const at::Tensor ws = scratch(hidden, g_vocab_workspace.load()(code, tokens, size, vocab, 0));
    const int rc = g_vocab_forward.load()(
        x.data_ptr(), w.data_ptr(), code, y.data_ptr<int64_t>(), tokens, size, vocab, ignore_index,
        reduction, saved.data_ptr(), out[0].data_ptr<float>(),
        scores ? out[1].data_ptr<float>() : nullptr, scores ? out[2].data_ptr<float>() : nullptr,
        ws.data_ptr(), (size_t)ws.numel(), current_stream(hidden));
    if (rc) fail(rc, "ace_vocab_forward");
  }
  if (record) {
    auto node = std::shared_ptr<VocabLossBackward>(new VocabLossBackward(),
                                                   torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(hidden, weight));
    node->tokens = tokens;
    node->size = size;
    node->vocab = vocab;
    node->reduction = reduction;
    node->hidden_ = SavedVariable(hidden, false);
    node->weight_ = SavedVariable(weight, false);
    node->saved_ = SavedVariable(saved, false);
    torch::autograd::set_history(out[0], node);
    if (scores) torch::autograd::set_history(out[1], node);
  }
  return out;
}

struct BalanceLossBackward : public Node {
  std::string name() const override { return "BalanceLossBackward"; }

  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    if (!grads[0].defined()) return out;
    refuse_tangents({grads[0]}, "balance_loss's gradient");
    const at::Tensor logits = logits_.unpack(), share = share_.unpack(), mask = mask_.unpack();
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(logits.device());
      const at::Tensor x = plain(logits), go = float32(grads[0]);
      const at::Tensor m = mask.defined() ? mask.contiguous() : mask;
      out[0] = at::empty(logits.sizes(), logits.options().requires_grad(false));
      const int rc = g_balance_backward.load()(
          x.data_ptr(), dtype_code(logits),
          m.defined() ? static_cast<const uint8_t*>(m.data_ptr()) : nullptr, groups, tokens,
          experts, reduction, share.data_ptr<float>(), go.data_ptr<float>(), out[0].data_ptr(),
          current_stream(logits));
      if (rc) fail(rc, "ace_balance_backward");
    }
    refuse_second_derivative(out, {logits, grads[0]}, "balance_loss");
    return out;
  }

  void release_variables() override {
    logits_.reset_data();
    mask_.reset_data();
    share_.reset_data();
  }

  int64_t groups = 0, tokens = 0, experts = 0;
  int reduction = 0;
  SavedVariable logits_, mask_, share_;
};

// (loss, counts) of checked arguments; `tickets`: zero, left zero.
std::vector<at::Tensor> balance_loss(const at::Tensor& logits, const std::optional<at::Tensor>& mask,
                                     int64_t groups, int top_k, int reduction,
                                     const at::Tensor& tickets) {
  if (!g_balance_forward.load()) throw std::runtime_error("ace_autograd: entry points not set");
  refuse_tangents({logits}, "balance_loss");
  const bool record = torch::autograd::compute_requires_grad(logits);
  const c10::DeviceGuard guard(logits.device());
  const int64_t tokens = logits.size(-2), experts = logits.size(-1);
  at::Tensor loss, counts, share;
  {
    const at::NoGradGuard no_grad;
    const at::Tensor x = plain(logits);
    const at::Tensor m = mask ? mask->contiguous() : at::Tensor();
    const auto options = logits.options().requires_grad(false);
    std::vector<int64_t> lead(logits.sizes().begin(), logits.sizes().end() - 2);
    loss = at::empty(reduction == ACE_RED_NONE ? lead : std::vector<int64_t>{},
                     options.dtype(at::kFloat));
    lead.push_back(experts);
    counts = at::empty(lead, options.dtype(at::kLong));
    share = at::empty({groups, experts}, options.dtype(at::kFloat));
    const at::Tensor ws = scratch(logits, g_balance_workspace.load()(groups, tokens, experts));
    const int rc = g_balance_forward.load()(
        x.data_ptr(), dtype_code(logits),
        m.defined() ? static_cast<const uint8_t*>(m.data_ptr()) : nullptr, groups, tokens, experts,
        top_k, reduction, loss.data_ptr<float>(), counts.data_ptr<int64_t>(),
        share.data_ptr<float>(), tickets.data_ptr(), (size_t)tickets.numel(), ws.data_ptr(),
        (size_t)ws.numel(), current_stream(logits));
    if (rc) fail(rc, "ace_balance_forward");
  }
  if (record) {
    auto node = std::shared_ptr<BalanceLossBackward>(new BalanceLossBackward(),
                                                     torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->groups = groups;
    node->tokens = tokens;
    node->experts = experts;
    node->reduction = reduction;
    node->logits_ = SavedVariable(logits, false);
    if (mask) node->mask_ = SavedVariable(*mask, false);
    node->share_ = SavedVariable(share, false);
    torch::autograd::set_history(loss, node);
  }
  return {loss, counts};
}

void set_lm_entry_points(uintptr_t vocab_saved, uintptr_t vocab_workspace, uintptr_t vocab_forward,
                         uintptr_t vocab_backward, uintptr_t balance_workspace,
                         uintptr_t balance_forward, uintptr_t balance_backward) {
  g_vocab_saved.store(reinterpret_cast<decltype(&ace_vocab_saved_bytes)>(vocab_saved));
  g_vocab_workspace.store(reinterpret_cast<decltype(&ace_vocab_workspace_bytes)>(vocab_workspace));
  g_vocab_forward.store(reinterpret_cast<decltype(&ace_vocab_forward)>(vocab_forward));
  g_vocab_backward.store(reinterpret_cast<decltype(&ace_vocab_backward)>(vocab_backward));
  g_balance_workspace.store(
      reinterpret_cast<decltype(&ace_balance_workspace_bytes)>(balance_workspace));
  g_balance_forward.store(reinterpret_cast<decltype(&ace_balance_forward)>(balance_forward));
  g_balance_backward.store(reinterpret_cast<decltype(&ace_balance_backward)>(balance_backward));
}

// ------------------------------------------------ token log probabilities
std::atomic<decltype(&ace_logprob_saved_bytes)> g_logprob_saved{nullptr};
std::atomic<decltype(&ace_logprob_workspace_bytes)> g_logprob_workspace{nullptr};
std::atomic<decltype(&ace_logprob_forward)> g_logprob_forward{nullptr};
std::atomic<decltype(&ace_logprob_backward)> g_logprob_backward{nullptr};

// t as rows of its last dimension, whose elements are neighbours: a view wherever the
// strides allow one.
at::Tensor as_rows(const at::Tensor& t) {
  at::Tensor r = (t.is_neg() ? t.resolve_neg() : t).reshape({-1, t.size(-1)});
  return r.size(1) == 1 || r.stride(1) == 1 ? r : r.contiguous();
}

struct TokenLogprobsBackward : public Node {
  std::string name() const override { return "TokenLogprobsBackward"; }

  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    const at::Tensor &gl = grads[0], &ge = grads[1];
    if (!gl.defined() && !ge.defined()) return out;
    refuse_tangents({gl, ge}, "token_logprobs's gradient");
    const at::Tensor logits = logits_.unpack(), saved = saved_.unpack();
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(logits.device());
      const at::Tensor x = as_rows(logits), l = float32(gl), e = float32(ge);
      out[0] = at::empty(logits.sizes(), logits.options().requires_grad(false));
      const int rc = g_logprob_backward.load()(
          x.data_ptr(), dtype_code(logits), x.stride(0), x.size(0), x.size(1), temperature,
          saved.data_ptr(), l.defined() ? l.data_ptr<float>() : nullptr,
          e.defined() ? e.data_ptr<float>() : nullptr, out[0].data_ptr(), current_stream(logits));
      if (rc) fail(rc, "ace_logprob_backward");
    }
    refuse_second_derivative(out, {logits, gl, ge}, "token_logprobs");
    return out;
  }

  void release_variables() override {
    logits_.reset_data();
    saved_.reset_data();
  }

  float temperature = 1.f;
  SavedVariable logits_, saved_;
};

// (logprob, entropy), and with top > 0 (.., top_logprobs, top_tokens), of checked
// arguments; `tickets`: zero, left zero, where the sizes need them.
std::vector<at::Tensor> token_logprobs(const at::Tensor& logits, const at::Tensor& tokens,
                                       int64_t ignore_index, float temperature, int top,
                                       const std::optional<at::Tensor>& tickets) {
  if (!g_logprob_forward.load()) throw std::runtime_error("ace_autograd: entry points not set");
  refuse_tangents({logits}, "token_logprobs");
  const bool record = torch::autograd::compute_requires_grad(logits);
  const c10::DeviceGuard guard(logits.device());
  std::vector<at::Tensor> out;
  at::Tensor saved;
  {
    const at::NoGradGuard no_grad;
    const at::Tensor x = as_rows(logits), y = plain(tokens.to(at::kLong));
    const int64_t rows = x.size(0), vocab = x.size(1);
    const int code = dtype_code(logits);
    const auto f32 = logits.options().dtype(at::kFloat).requires_grad(false);
    for (int i = 0; i < 2; ++i) out.push_back(at::empty(tokens.sizes(), f32));
    if (top > 0) {
      std::vector<int64_t> shape(tokens.sizes().begin(), tokens.sizes().end());
      shape.push_back(top);
      out.push_back(at::empty(shape, f32));
      out.push_back(at::empty(shape, f32.dtype(at::kLong)));
    }
    saved = scratch(logits, g_logprob_saved.load()(rows));
    const size_t need = g_logprob_workspace.load()(code, rows, vocab, top);
    const at::Tensor ws = need ? scratch(logits, need) : at::Tensor();
    const int rc = g_logprob_forward.load()(
        x.data_ptr(), code, x.stride(0), y.data_ptr<int64_t>(), rows, vocab, ignore_index,
        temperature, top, saved.data_ptr(), out[0].data_ptr<float>(), out[1].data_ptr<float>(),
        top > 0 ? out[2].data_ptr<float>() : nullptr,
        top > 0 ? out[3].data_ptr<int64_t>() : nullptr, tickets ? tickets->data_ptr() : nullptr,
        tickets ? (size_t)tickets->numel() : 0, ws.defined() ? ws.data_ptr() : nullptr, need,
        current_stream(logits));
    if (rc) fail(rc, "ace_logprob_forward");
  }
  if (record) {
    auto node = std::shared_ptr<TokenLogprobsBackward>(new TokenLogprobsBackward(),
                                                       torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->temperature = temperature;
    node->logits_ = SavedVariable(logits, false);
    node->saved_ = SavedVariable(saved, false);
    for (int i = 0; i < 2; ++i) torch::autograd::set_history(out[i], node);
  }
  return out;
}

void set_logprob_entry_points(uintptr_t saved, uintptr_t workspace, uintptr_t forward,
                              uintptr_t backward) {
  g_logprob_saved.store(reinterpret_cast<decltype(&ace_logprob_saved_bytes)>(saved));
  g_logprob_workspace.store(reinterpret_cast<decltype(&ace_logprob_workspace_bytes)>(workspace));
  g_logprob_forward.store(reinterpret_cast<decltype(&ace_logprob_forward)>(forward));
  g_logprob_backward.store(reinterpret_cast<decltype(&ace_logprob_backward)>(backward));
}

// ------------------------------------------------------------------ experts
std::atomic<decltype(&ace_route_forward)> g_route_forward{nullptr};
std::atomic<decltype(&ace_route_backward)> g_route_backward{nullptr};
std::atomic<decltype(&ace_expert_order_workspace_bytes)> g_order_workspace{nullptr};
std::atomic<decltype(&ace_expert_order)> g_order{nullptr};
std::atomic<decltype(&ace_to_experts)> g_to_experts{nullptr};
std::atomic<decltype(&ace_from_experts)> g_from_experts{nullptr};
std::atomic<decltype(&ace_from_experts_backward)> g_from_experts_backward{nullptr};

struct RouteTokensBackward : public Node {
  std::string name() const override { return "RouteTokensBackward"; }

  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    if (!grads[0].defined()) return out;
    refuse_tangents({grads[0]}, "route_tokens's gradient");
    const at::Tensor logits = logits_.unpack(), chosen = chosen_.unpack(),
                     weights = weights_.unpack();
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(chosen.device());
      const at::Tensor g = float32(grads[0]);
      out[0] = at::empty(sizes, options);
      // without kept scores any address will do
      const at::Tensor x = logits.defined() ? plain(logits) : out[0];
      const int rc = g_route_backward.load()(
          x.data_ptr(), dtype_code(out[0]), tokens, sizes.back(), top_k, normalize,
          chosen.data_ptr<int64_t>(), weights.data_ptr<float>(), g.data_ptr<float>(),
          out[0].data_ptr(), current_stream(out[0]));
      if (rc) fail(rc, "ace_route_backward");
    }
    refuse_second_derivative(out, {next_edge(0), torch::autograd::impl::gradient_edge(grads[0])},
                             "route_tokens");
    return out;
  }

  void release_variables() override {
    logits_.reset_data();
    chosen_.reset_data();
    weights_.reset_data();
  }

  int64_t tokens = 0;
  int top_k = 0, normalize = 0;
  std::vector<int64_t> sizes;
  at::TensorOptions options;
  SavedVariable logits_, chosen_, weights_;
};

// (experts, weights) of checked arguments.
std::vector<at::Tensor> route_tokens(const at::Tensor& logits, const std::optional<at::Tensor>& mask,
                                     int top_k, bool normalize) {
  if (!g_route_forward.load()) throw std::runtime_error("ace_autograd: entry points not set");
  refuse_tangents({logits}, "route_tokens");
  const bool record = torch::autograd::compute_requires_grad(logits);
  const c10::DeviceGuard guard(logits.device());
  at::Tensor chosen, weights;
  int64_t tokens = 0;
  {
    const at::NoGradGuard no_grad;
    const at::Tensor x = plain(logits);
    const at::Tensor m = mask ? mask->contiguous() : at::Tensor();
    std::vector<int64_t> shape(logits.sizes().begin(), logits.sizes().end());
    shape.back() = top_k;
    const auto options = logits.options().requires_grad(false);
    chosen = at::empty(shape, options.dtype(at::kLong));
    weights = at::empty(shape, options.dtype(at::kFloat));
    tokens = weights.numel() / top_k;
    const int rc = g_route_forward.load()(
        x.data_ptr(), dtype_code(logits),
        m.defined() ? static_cast<const uint8_t*>(m.data_ptr()) : nullptr, tokens, logits.size(-1),
        top_k, normalize, chosen.data_ptr<int64_t>(), weights.data_ptr<float>(),
        current_stream(logits));
    if (rc) fail(rc, "ace_route_forward");
  }
  if (record) {
    auto node = std::shared_ptr<RouteTokensBackward>(new RouteTokensBackward(),
                                                     torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(logits));
    node->tokens = tokens;
    node->top_k = top_k;
    node->normalize = normalize;
    node->sizes.assign(logits.sizes().begin(), logits.sizes().end());
    node->options = logits.options().requires_grad(false);
    // the gradient of normalised weights reads no score
    if (!normalize) node->logits_ = SavedVariable(logits, false);
    node->chosen_ = SavedVariable(chosen, false);
    // not the result itself, which will hold the node; it shares the version that
    // tells of changes in place
    node->weights_ = SavedVariable(weights.detach(), false);
    torch::autograd::set_history(weights, node);
  }
  return {chosen, weights};
}

// (offsets, source, place) of checked arguments.
std::vector<at::Tensor> expert_order(const at::Tensor& experts, int64_t num_experts) {
  if (!g_order.load()) throw std::runtime_error("ace_autograd: entry points not set");
  const at::NoGradGuard no_grad;
  const c10::DeviceGuard guard(experts.device());
  const at::Tensor chosen = plain(experts.to(at::kLong));
  const auto options = chosen.options();
  const int64_t slots = chosen.numel();
  const at::Tensor offsets = at::empty({num_experts + 1}, options);
  const at::Tensor source = at::empty({slots}, options), place = at::empty(experts.sizes(), options);
  const size_t need = g_order_workspace.load()(slots, num_experts);
  const at::Tensor ws = need ? scratch(chosen, need) : at::Tensor();
  const int rc = g_order.load()(chosen.data_ptr<int64_t>(), slots, num_experts,
                                offsets.data_ptr<int64_t>(), source.data_ptr<int64_t>(),
                                place.data_ptr<int64_t>(), ws.defined() ? ws.data_ptr() : nullptr,
                                need, current_stream(chosen));
  if (rc) fail(rc, "ace_expert_order");
  return {offsets, source, place};
}

struct ToExpertsBackward : public Node {
  std::string name() const override { return "ToExpertsBackward"; }

  variable_list apply(variable_list&& grads) override {
    variable_list out(1);
    const at::Tensor& g = grads[0];
    if (!g.defined()) return out;
    refuse_tangents({g}, "to_experts's gradient");
    const at::Tensor source = source_.unpack(), place = place_.unpack();
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(g.device());
      const at::Tensor rows = plain(g);
      out[0] = at::empty(shape, g.options().requires_grad(false));
      const int64_t top_k = place.size(-1);
      const int rc = g_from_experts.load()(rows.data_ptr(), dtype_code(g), place.numel() / top_k,
                                           shape.back(), top_k, source.data_ptr<int64_t>(),
                                           place.data_ptr<int64_t>(), nullptr, out[0].data_ptr(),
                                           current_stream(g));
      if (rc) fail(rc, "ace_from_experts");
    }
    refuse_second_derivative(out, {g}, "to_experts");
    return out;
  }

  void release_variables() override {
    source_.reset_data();
    place_.reset_data();
  }

  std::vector<int64_t> shape;
  SavedVariable source_, place_;
};

// The rows of checked arguments.
at::Tensor to_experts(const at::Tensor& x, const at::Tensor& source, const at::Tensor& place) {
  if (!g_to_experts.load()) throw std::runtime_error("ace_autograd: entry points not set");
  refuse_tangents({x}, "to_experts");
  const bool record = torch::autograd::compute_requires_grad(x);
  const c10::DeviceGuard guard(x.device());
  at::Tensor rows, of, at;
  {
    const at::NoGradGuard no_grad;
    const at::Tensor in = plain(x);
    of = source.contiguous();
    at = place.contiguous();
    const int64_t top_k = at.size(-1), width = x.size(-1);
    rows = at::empty({at.numel(), width}, x.options().requires_grad(false));
    const int rc = g_to_experts.load()(in.data_ptr(), dtype_code(x), at.numel() / top_k, width,
                                       top_k, of.data_ptr<int64_t>(), at.data_ptr<int64_t>(),
                                       rows.data_ptr(), current_stream(x));
    if (rc) fail(rc, "ace_to_experts");
  }
  if (record) {
    auto node = std::shared_ptr<ToExpertsBackward>(new ToExpertsBackward(),
                                                   torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x));
    node->shape.assign(x.sizes().begin(), x.sizes().end());
    node->source_ = SavedVariable(of, false);
    node->place_ = SavedVariable(at, false);
    torch::autograd::set_history(rows, node);
  }
  return rows;
}

struct FromExpertsBackward : public Node {
  std::string name() const override { return "FromExpertsBackward"; }

  variable_list apply(variable_list&& grads) override {
    variable_list out(2);
    const at::Tensor& g = grads[0];
    if (!g.defined()) return out;
    refuse_tangents({g}, "from_experts's gradient");
    const at::Tensor place = place_.unpack(), source = source_.unpack(), rows = rows_.unpack(),
                     weights = weights_.unpack();
    {
      const at::NoGradGuard no_grad;
      const c10::DeviceGuard guard(g.device());
      const at::Tensor up = plain(g), w = weights.defined() ? plain(weights) : weights;
      const int64_t top_k = place.size(-1), slots = place.numel(), width = g.size(-1);
      if (task_should_compute_output(0))
        out[0] = at::empty({slots, width}, g.options().requires_grad(false));
      at::Tensor in;
      if (rows.defined() && task_should_compute_output(1)) {
        in = plain(rows);
        out[1] = at::empty(place.sizes(), g.options().dtype(at::kFloat).requires_grad(false));
      }
      const int rc = g_from_experts_backward.load()(
          in.defined() ? in.data_ptr() : nullptr, up.data_ptr(), dtype_code(g), slots / top_k,
          width, top_k, source.data_ptr<int64_t>(), place.data_ptr<int64_t>(),
          w.defined() ? w.data_ptr<float>() : nullptr,
          out[0].defined() ? out[0].data_ptr() : nullptr,
          out[1].defined() ? out[1].data_ptr<float>() : nullptr, current_stream(g));
      if (rc) fail(rc, "ace_from_experts_backward");
    }
    refuse_second_derivative(out, {rows, weights, g}, "from_experts");
    return out;
  }

  void release_variables() override {
    rows_.reset_data();
    weights_.reset_data();
    source_.reset_data();
    place_.reset_data();
  }

  SavedVariable rows_, weights_, source_, place_;
};

// The tokens' rows of checked arguments.
at::Tensor from_experts(const at::Tensor& rows, const at::Tensor& source, const at::Tensor& place,
                        const std::optional<at::Tensor>& weights) {
  if (!g_from_experts.load()) throw std::runtime_error("ace_autograd: entry points not set");
  const at::Tensor factor = weights ? *weights : at::Tensor();
  refuse_tangents({rows, factor}, "from_experts");
  const bool record = torch::autograd::compute_requires_grad(rows, factor);
  const c10::DeviceGuard guard(rows.device());
  at::Tensor out, of, at;
  {
    const at::NoGradGuard no_grad;
    const at::Tensor in = plain(rows), w = factor.defined() ? plain(factor) : factor;
    of = source.contiguous();
    at = place.contiguous();
    const int64_t top_k = at.size(-1), width = rows.size(-1);
    std::vector<int64_t> shape(at.sizes().begin(), at.sizes().end());
    shape.back() = width;
    out = at::empty(shape, rows.options().requires_grad(false));
    const int rc = g_from_experts.load()(in.data_ptr(), dtype_code(rows), at.numel() / top_k, width,
                                         top_k, of.data_ptr<int64_t>(), at.data_ptr<int64_t>(),
                                         w.defined() ? w.data_ptr<float>() : nullptr,
                                         out.data_ptr(), current_stream(rows));
    if (rc) fail(rc, "ace_from_experts");
  }
  if (record) {
    auto node = std::shared_ptr<FromExpertsBackward>(new FromExpertsBackward(),
                                                     torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(rows, factor));
    // the rows only for the weights' gradient
    if (factor.defined() && factor.requires_grad()) node->rows_ = SavedVariable(rows, false);
    if (factor.defined()) node->weights_ = SavedVariable(factor, false);
    node->source_ = SavedVariable(of, false);
    node->place_ = SavedVariable(at, false);
    torch::autograd::set_history(out, node);
  }
  return out;
}

void set_expert_entry_points(uintptr_t route_forward, uintptr_t route_backward,
                             uintptr_t order_workspace, uintptr_t order, uintptr_t to,
                             uintptr_t from, uintptr_t from_backward) {
  g_route_forward.store(reinterpret_cast<decltype(&ace_route_forward)>(route_forward));
  g_route_backward.store(reinterpret_cast<decltype(&ace_route_backward)>(route_backward));
  g_order_workspace.store(
      reinterpret_cast<decltype(&ace_expert_order_workspace_bytes)>(order_workspace));
  g_order.store(reinterpret_cast<decltype(&ace_expert_order)>(order));
  g_to_experts.store(reinterpret_cast<decltype(&ace_to_experts)>(to));
  g_from_experts.store(reinterpret_cast<decltype(&ace_from_experts)>(from));
  g_from_experts_backward.store(
      reinterpret_cast<decltype(&ace_from_experts_backward)>(from_backward));
}

std::shared_ptr<LevelSignature> make_level_signature(
    int x_dtype, int64_t batch, int64_t channels, int num_bins, int binning, int include_background,
    int ignore_empty, int reduction, int right, float empty_weight, uintptr_t class_weight,
    uintptr_t bin_table, uintptr_t centre_table, uintptr_t workspace, size_t workspace_bytes,
    std::vector<int64_t> voxels, int64_t n_saved, int64_t o_d, int64_t o_jac, int64_t o_pc,
    bool reduced, bool soft, std::vector<int64_t> loss_shape) {
  if (voxels.empty() || voxels.size() > 4)
    throw std::invalid_argument("make_level_signature: 1 to 4 levels");
  auto s = std::make_shared<LevelSignature>();
  s->x_dtype = x_dtype;
  s->batch = batch;
  s->channels = channels;
  s->num_bins = num_bins;
  s->binning = binning;
  s->include_background = include_background;
  s->ignore_empty = ignore_empty;
  s->reduction = reduction;
  s->right = right;
  s->empty_weight = empty_weight;
  s->class_weight = reinterpret_cast<const float*>(class_weight);
  s->bin_table = reinterpret_cast<const float*>(bin_table);
  s->centre_table = reinterpret_cast<const float*>(centre_table);
  s->workspace = reinterpret_cast<void*>(workspace);
  s->workspace_bytes = workspace_bytes;
  s->voxels = std::move(voxels);
  s->n_saved = n_saved;
  s->o_d = o_d;
  s->o_jac = o_jac;
  s->o_pc = o_pc;
  s->reduced = reduced;
  s->soft = soft;
  s->loss_shape = std::move(loss_shape);
  return s;
}

std::shared_ptr<Signature> make_signature(
    int x_dtype, int target_kind, int64_t batch, int64_t channels, int64_t voxels, int num_bins,
    int binning, int activation, int include_background, int ignore_empty, int reduction,
    int right, float empty_weight, uintptr_t class_weight, uintptr_t bin_table,
    uintptr_t centre_table, uintptr_t workspace, size_t workspace_bytes, int64_t n_saved,
    int64_t o_d, int64_t o_jac, int64_t o_pc, bool reduced, bool soft,
    std::vector<int64_t> loss_shape) {
  auto s = std::make_shared<Signature>();
  s->x_dtype = x_dtype;
  s->target_kind = target_kind;
  s->batch = batch;
  s->channels = channels;
  s->voxels = voxels;
  s->num_bins = num_bins;
  s->binning = binning;
  s->activation = activation;
  s->include_background = include_background;
  s->ignore_empty = ignore_empty;
  s->reduction = reduction;
  s->right = right;
  s->empty_weight = empty_weight;
  s->class_weight = reinterpret_cast<const float*>(class_weight);
  s->bin_table = reinterpret_cast<const float*>(bin_table);
  s->centre_table = reinterpret_cast<const float*>(centre_table);
  s->workspace = reinterpret_cast<void*>(workspace);
  s->workspace_bytes = workspace_bytes;
  s->n_saved = n_saved;
  s->o_d = o_d;
  s->o_jac = o_jac;
  s->o_pc = o_pc;
  s->reduced = reduced;
  s->soft = soft;
  s->loss_shape = std::move(loss_shape);
  return s;
}

void set_entry_points(uintptr_t forward, uintptr_t backward, uintptr_t forward_levels,
                      uintptr_t backward_levels, uintptr_t error_string) {
  g_forward.store(reinterpret_cast<ForwardFn>(forward));
  g_backward.store(reinterpret_cast<BackwardFn>(backward));
  g_forward_levels.store(reinterpret_cast<ForwardLevelsFn>(forward_levels));
  g_backward_levels.store(reinterpret_cast<BackwardLevelsFn>(backward_levels));
  g_error.store(reinterpret_cast<ErrorFn>(error_string));
}

}  // namespace

PYBIND11_MODULE(_ace_autograd, m) {
  m.doc() = "hip_mi355x's loss call and backward node in C++ over libace_hip.so";
  pybind11::class_<Signature, std::shared_ptr<Signature>>(m, "Signature");
  pybind11::class_<LevelSignature, std::shared_ptr<LevelSignature>>(m, "LevelSignature");
  m.def("make_signature", &make_signature);
  m.def("make_level_signature", &make_level_signature);
  m.def("set_entry_points", &set_entry_points);
  m.def("ace_loss", &ace_loss);
  m.def("ace_loss_levels", &ace_loss_levels);
  m.def("set_lm_entry_points", &set_lm_entry_points);
  m.def("vocab_loss", &vocab_loss);
  m.def("balance_loss", &balance_loss, pybind11::arg(), pybind11::arg().none(true), pybind11::arg(),
        pybind11::arg(), pybind11::arg(), pybind11::arg());
  m.def("set_logprob_entry_points", &set_logprob_entry_points);
  m.def("token_logprobs", &token_logprobs, pybind11::arg(), pybind11::arg(), pybind11::arg(),
        pybind11::arg(), pybind11::arg(), pybind11::arg().none(true));
  m.def("set_expert_entry_points", &set_expert_entry_points);
  m.def("route_tokens", &route_tokens, pybind11::arg(), pybind11::arg().none(true), pybind11::arg(),
        pybind11::arg());
  m.def("expert_order", &expert_order);
  m.def("to_experts", &to_experts);
  m.def("from_experts", &from_experts, pybind11::arg(), pybind11::arg(), pybind11::arg(),
        pybind11::arg().none(true));
}
