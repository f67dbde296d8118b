// Autograd nodes of the small training operators (layer norm, the router's
// auxiliary loss) in C++, over the C ABI of libpmoe.
//
// Autograd runs a node's backward on a thread of its own. A node written in Python
// first takes the interpreter's lock there, and its calls are the larger part of a
// small call's time; these do not touch the interpreter: layer norm of 1531 x 1001,
// forward and backward, 119 -> 66 us (torch's own 71; the kernels are 20), the
// auxiliary loss of one layer 131 -> 59 us, of 48 layers 466 -> 288 us. Arguments
// are checked by the Python entry points (layernorm.py, router_aux.py), sizes and
// pointers again by the C ABI.
#include <torch/extension.h>
#include <torch/csrc/autograd/custom_function.h>
#include <torch/csrc/autograd/functions/basic_ops.h>
#include <torch/csrc/autograd/functions/utils.h>

#include "../../include/pmoe.h"

namespace {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::SavedVariable;
using torch::autograd::variable_list;
using MaybeTensor = c10::optional<Tensor>;

int code_of(at::ScalarType t) {
  switch (t) {
    case at::kFloat: return PMOE_F32;
    case at::kBFloat16: return PMOE_BF16;
    case at::kHalf: return PMOE_F16;
    default: TORCH_CHECK_TYPE(false, "pmoe supports bf16, fp16 and fp32 tensors, got ", t);
  }
}

void check(int rc, const char* name) {
  TORCH_CHECK(rc == PMOE_OK, name, " failed (status ", rc, "): ", pmoe_last_error_string());
}

// The handle of the stream that was current when the forward ran; autograd makes it
// current again for the node's backward.
void* stream_of(int64_t handle) { return reinterpret_cast<void*>(handle); }

void refuse_capture(int64_t stream, const char* op) {
  TORCH_CHECK(!pmoe_stream_capturing(stream_of(stream)), "pmoe::", op,
              ": the backward is not supported under HIP graph capture (capture the forward only)");
}

// What a saved-tensor hook gave back, as the kernels read it.
Tensor ready(const Tensor& t) {
  if (!t.defined()) return t;
  TORCH_CHECK(t.is_cuda(), "pluggy_amd runs on ROCm GPU tensors only (there is no CPU fallback); got a tensor on ",
              t.device());
  return t.contiguous();
}

void* data(const Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }

Tensor bytes(size_t n, const Tensor& like) {
  return at::empty({(int64_t)std::max<size_t>(1, n)}, like.options().dtype(at::kByte));
}

// Whether a gradient can be asked of a call on these tensors. Forward-mode derivatives are refused.
bool differentiated(at::TensorList ts) {
  bool any = false;
  for (const Tensor& t : ts) {
    if (!t.defined()) continue;
    TORCH_CHECK(!t._fw_grad(/*level=*/0).defined(), "pmoe: forward-mode differentiation is not supported");
    any = any || t.requires_grad();
  }
  return any && torch::GradMode::is_enabled();
}

// There is no second derivative: gradients that could be differentiated raise when they are.
variable_list refuse_second(variable_list grads, const Tensor& grad) {
  if (!torch::GradMode::is_enabled() || !grad.requires_grad()) return grads;
  variable_list defined;
  for (const Tensor& g : grads)
    if (g.defined()) defined.push_back(g.detach().set_requires_grad(true));
  auto node = std::make_shared<torch::autograd::DelayedError>(
      "pmoe: a second derivative of this operator is not supported", (int64_t)defined.size());
  const variable_list out = (*node)(std::move(defined));
  size_t k = 0;
  for (Tensor& g : grads)
    if (g.defined()) g = out[k++];
  return grads;
}

// --------------------------------------------------------------- layer norm

struct LayerNorm : torch::autograd::Function<LayerNorm> {
  static int param_code(const Tensor& w, const Tensor& b) {
    return w.defined() ? code_of(w.scalar_type()) : b.defined() ? code_of(b.scalar_type()) : PMOE_F32;
  }

  // stats: (2, T) fp32, the rows' means and reciprocal deviations; undefined: not wanted.
  static Tensor launch(const Tensor& x, const Tensor& w, const Tensor& b, double eps, at::ScalarType out_dtype,
                       int64_t stream, const Tensor& stats) {
    c10::DeviceGuard guard(x.device());
    const int64_t H = x.size(-1), T = x.numel() / H;
    Tensor out = at::empty(x.sizes(), x.options().dtype(out_dtype));
    float* mean = stats.defined() ? stats.data_ptr<float>() : nullptr;
    check(pmoe_layernorm_forward(data(x), code_of(x.scalar_type()), data(w), data(b), param_code(w, b), (float)eps, T,
                                 H, data(out), code_of(out_dtype), mean, mean != nullptr ? mean + T : nullptr,
                                 stream_of(stream)),
          "pmoe_layernorm_forward");
    return out;
  }

  static Tensor forward(AutogradContext* ctx, const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias,
                        double eps, at::ScalarType out_dtype, int64_t stream) {
    at::AutoDispatchBelowADInplaceOrView below;
    const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
    Tensor stats = at::empty({2, x.numel() / x.size(-1)}, x.options().dtype(at::kFloat));
    Tensor out = launch(x, w, b, eps, out_dtype, stream, stats);
    ctx->save_for_backward({x, w, b, stats});
    ctx->saved_data["stream"] = stream;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    const int64_t stream = ctx->saved_data["stream"].toInt();
    refuse_capture(stream, "layer_norm_bwd");
    const auto saved = ctx->get_saved_variables();
    variable_list out(6);
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const Tensor x = ready(saved[0]), w = ready(saved[1]), b = saved[2], stats = ready(saved[3]);
      const Tensor g = grads[0].contiguous();
      c10::DeviceGuard guard(x.device());
      const int64_t H = x.size(-1), T = x.numel() / H;
      TORCH_CHECK(stats.numel() == 2 * T && g.sizes() == x.sizes(), "pmoe::layer_norm_bwd: saved tensors of other sizes");
      // the edges are those of the tensors that were given
      size_t edge = 1;
      const bool need_w = w.defined() && ctx->needs_input_grad(edge++);
      const bool need_b = b.defined() && ctx->needs_input_grad(edge);
      if (ctx->needs_input_grad(0)) out[0] = at::empty(x.sizes(), x.options());
      if (need_w) out[1] = at::empty({H}, w.options());
      if (need_b) out[2] = at::empty({H}, x.options().dtype(b.scalar_type()));
      const size_t need = need_w || need_b ? pmoe_layernorm_backward_workspace_size(T, H) : 0;
      const Tensor ws = need > 0 ? bytes(need, x) : Tensor();
      const float* mean = stats.data_ptr<float>();
      check(pmoe_layernorm_backward(data(g), code_of(g.scalar_type()), data(x), code_of(x.scalar_type()), data(w),
                                    param_code(w, b), mean, mean + T, T, H, data(out[0]), data(out[1]), data(out[2]),
                                    data(ws), need, stream_of(stream)),
            "pmoe_layernorm_backward");
    }
    return refuse_second(std::move(out), grads[0]);
  }
};

Tensor layer_norm(const Tensor& x, const MaybeTensor& weight, const MaybeTensor& bias, double eps,
                  at::ScalarType out_dtype, int64_t stream) {
  const Tensor w = weight.value_or(Tensor()), b = bias.value_or(Tensor());
  const std::array<Tensor, 3> in = {x, w, b};
  if (differentiated(in)) return LayerNorm::apply(x, weight, bias, eps, out_dtype, stream);
  at::AutoDispatchBelowADInplaceOrView below;
  return LayerNorm::launch(x, w, b, eps, out_dtype, stream, Tensor());
}

// ---------------------------------------------------- router auxiliary loss

template <typename P>
std::vector<P> pointers(at::TensorList ts) {
  std::vector<P> out;
  out.reserve(ts.size());
  for (const Tensor& t : ts) out.push_back(static_cast<P>(data(t)));
  return out;
}

// A node of its own: a Function does not follow the tensors of a list.
struct AuxLossBackward : torch::autograd::Node {
  std::vector<SavedVariable> logits;
  SavedVariable coef, mask;
  float aux_coef = 0.0f, z_coef = 0.0f;
  int64_t stream = 0;

  std::string name() const override { return "RouterAuxLossBackward"; }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (SavedVariable& s : logits) s.reset_data();
    coef.reset_data();
    mask.reset_data();
  }

  variable_list apply(variable_list&& grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    const size_t L = logits.size();
    variable_list out(L);
    if (!grads[0].defined()) return out;
    refuse_capture(stream, "aux_loss_bwd");
    std::vector<Tensor> ls(L);
    for (size_t i = 0; i < L; ++i) ls[i] = logits[i].unpack();
    const Tensor saved_coef = coef.unpack(), saved_mask = mask.unpack();
    {
      at::AutoDispatchBelowADInplaceOrView below;
      const Tensor c = ready(saved_coef), m = ready(saved_mask);
      const int64_t E = c.size(0) - 1;
      std::vector<int64_t> rows(L), sizes(L);
      int64_t total = 0;
      for (size_t i = 0; i < L; ++i) {
        ls[i] = ready(ls[i]);
        TORCH_CHECK(ls[i].dim() == 2 && ls[i].size(1) == E && ls[i].scalar_type() == ls[0].scalar_type() &&
                        ls[i].device() == c.device(),
                    "pmoe::aux_loss_bwd: saved logits unlike the forward's");
        rows[i] = ls[i].size(0);
        sizes[i] = task_should_compute_output(i) ? rows[i] : 0;
        total += sizes[i];
      }
      c10::DeviceGuard guard(c.device());
      const Tensor g = grads[0].to(at::kFloat).contiguous();
      // one allocation for all layers; each gradient is its rows
      const std::vector<Tensor> parts = at::empty({total, E}, ls[0].options()).split_with_sizes(sizes);
      for (size_t i = 0; i < L; ++i)
        if (task_should_compute_output(i)) out[i] = parts[i];
      check(pmoe_aux_loss_backward(pointers<const void*>(ls).data(), pointers<void*>(out).data(), rows.data(),
                                   (int64_t)L, code_of(ls[0].scalar_type()), static_cast<const uint8_t*>(data(m)),
                                   m.defined() ? m.numel() : 0, E, c.data_ptr<float>(), g.data_ptr<float>(), aux_coef,
                                   z_coef, stream_of(stream)),
            "pmoe_aux_loss_backward");
    }
    return refuse_second(std::move(out), grads[0]);
  }
};

// -> loss (with the logits' gradient), load balance, z-loss, expert_counts. The
// statistics of the fused routers (one entry a layer), or empty lists.
std::tuple<Tensor, Tensor, Tensor, Tensor> aux_loss(const std::vector<Tensor>& logits, const MaybeTensor& token_mask,
                                                    const std::vector<Tensor>& counts,
                                                    const std::vector<Tensor>& prob_sums,
                                                    const std::vector<Tensor>& lse_sq_sums, int64_t top_k,
                                                    double aux_coef, double z_coef, int64_t stream) {
  const bool wanted = differentiated(logits);
  const Tensor mask = token_mask.value_or(Tensor());
  const int64_t L = (int64_t)logits.size(), E = logits[0].size(1);
  Tensor loss, balance, z, picks, coef;
  {
    at::AutoDispatchBelowADInplaceOrView below;
    c10::DeviceGuard guard(logits[0].device());
    std::vector<int64_t> rows(L);
    int64_t total = 0;
    for (int64_t i = 0; i < L; ++i) total += rows[i] = logits[i].size(0);
    const auto f32 = logits[0].options().dtype(at::kFloat);
    loss = at::empty({}, f32);
    balance = at::empty({}, f32);
    z = at::empty({}, f32);
    coef = at::empty({E + 1}, f32);
    picks = at::empty({L, E}, f32.dtype(at::kInt));
    const bool from_stats = !counts.empty();
    const size_t need = from_stats ? pmoe_aux_loss_from_stats_workspace_size(L, E)
                                   : pmoe_aux_loss_forward_workspace_size(rows.data(), L, E);
    const Tensor ws = bytes(need, logits[0]);
    float *pl = loss.data_ptr<float>(), *pb = balance.data_ptr<float>(), *pz = z.data_ptr<float>();
    if (from_stats)
      check(pmoe_aux_loss_from_stats(pointers<const int32_t*>(counts).data(), pointers<const float*>(prob_sums).data(),
                                     pointers<const float*>(lse_sq_sums).data(), L, total, E, top_k, (float)aux_coef,
                                     (float)z_coef, pl, pb, pz, picks.data_ptr<int32_t>(), coef.data_ptr<float>(),
                                     data(ws), need, stream_of(stream)),
            "pmoe_aux_loss_from_stats");
    else
      check(pmoe_aux_loss_forward(pointers<const void*>(logits).data(), rows.data(), L, code_of(logits[0].scalar_type()),
                                  static_cast<const uint8_t*>(data(mask)), mask.defined() ? mask.numel() : 0, E, top_k,
                                  (float)aux_coef, (float)z_coef, pl, pb, pz, picks.data_ptr<int32_t>(),
                                  coef.data_ptr<float>(), data(ws), need, stream_of(stream)),
            "pmoe_aux_loss_forward");
  }
  if (wanted) {
    std::shared_ptr<AuxLossBackward> node(new AuxLossBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(at::TensorList(logits)));
    node->logits.reserve(L);
    for (const Tensor& t : logits) node->logits.emplace_back(t, false);
    node->coef = SavedVariable(coef, false);
    node->mask = SavedVariable(mask, false);
    node->aux_coef = (float)aux_coef;
    node->z_coef = (float)z_coef;
    node->stream = stream;
    torch::autograd::set_history(loss, node);
  }
  return {loss, balance, z, picks};
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  // errors come out as torch's own classes (out of memory among them), a hook's as they were raised
  m.def("layer_norm", torch::wrap_pybind_function_no_gil(layer_norm));
  m.def("aux_loss", torch::wrap_pybind_function_no_gil(aux_loss));
}
