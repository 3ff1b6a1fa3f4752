// The gated feed-forward block as an autograd function over the HIP kernels
// (rhip_gated_*), and its layer on sparse tensors.
#include <cmath>

#include "transformer.hpp"

namespace riemann {

namespace {

int32_t activation_of(const std::string &name) {
  TORCH_CHECK(name == "silu" || name == "gelu", "activation must be \"silu\" or \"gelu\", got \"",
              name, "\"");
  return name == "silu" ? RHIP_ACT_SILU : RHIP_ACT_GELU;
}

rhip_gated gated_desc(const at::Tensor &x, const at::Tensor &gate, const at::Tensor &up,
                      const at::Tensor &down, int64_t activation) {
  rhip_gated d{};
  d.n = x.size(0);
  d.x = x.data_ptr(), d.gate = gate.data_ptr(), d.up = up.data_ptr(), d.down = down.data_ptr();
  d.x_row = x.stride(0), d.gate_row = gate.stride(0), d.up_row = up.stride(0);
  d.down_row = down.stride(0);
  d.channels = static_cast<int32_t>(x.size(1)), d.hidden = static_cast<int32_t>(gate.size(0));
  d.outputs = static_cast<int32_t>(down.size(0));
  d.activation = static_cast<int32_t>(activation);
  d.dtype = hip_dtype(x, "feed-forward input");
  return d;
}

at::Tensor run_gated(const at::Tensor &x, const at::Tensor &gate, const at::Tensor &up,
                     const at::Tensor &down, int64_t activation, at::Tensor *saved) {
  const auto dev = x.device();
  at::DeviceGuard guard(dev);
  const rhip_gated d = gated_desc(x, gate, up, down, activation);
  auto y = torch::empty({x.size(0), down.size(0)}, x.options());
  size_t bytes = 0;
  if (saved) {
    check_rhip(rhip_gated_saved_bytes(&d, &bytes), "rhip_gated_saved_bytes");
    *saved = byte_buffer(bytes, dev);
  }
  check_rhip(rhip_gated_workspace_bytes(&d, saved ? RHIP_GATED_FORWARD : RHIP_GATED_INFERENCE,
                                        &bytes),
             "rhip_gated_workspace_bytes");
  auto ws = byte_buffer(bytes, dev);
  check_rhip(rhip_gated_forward(&d, y.data_ptr(), saved ? saved->data_ptr() : nullptr,
                                saved ? saved->numel() : 0, ws.data_ptr(), ws.numel(),
                                stream_of(dev)),
             "rhip_gated_forward");
  return y;
}

struct HipGatedFunction : public torch::autograd::Function<HipGatedFunction> {
  static at::Tensor forward(AutogradContext *ctx, at::Tensor x, at::Tensor gate, at::Tensor up,
                            at::Tensor down, int64_t activation) {
    at::Tensor saved;
    auto y = run_gated(x, gate, up, down, activation, &saved);
    ctx->save_for_backward({x, gate, up, down, saved});
    ctx->saved_data["activation"] = activation;
    return y;
  }

  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    first_derivative_only("the gated feed-forward block");
    auto s = ctx->get_saved_variables();
    const auto dev = s[0].device();
    at::DeviceGuard guard(dev);
    rhip_gated d = gated_desc(s[0], s[1], s[2], s[3], ctx->saved_data["activation"].toInt());
    auto gy = dense_last(grads[0]);
    d.grad_y = gy.data_ptr(), d.grad_y_row = gy.stride(0);
    at::Tensor g[4]; // of x, gate, up, down
    auto want = [&](int i) { g[i] = torch::empty(s[i].sizes(), s[i].options()); };
    if (ctx->needs_input_grad(0))
      want(0);
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
      want(1);
      want(2);
    }
    if (ctx->needs_input_grad(3))
      want(3);
    size_t bytes = 0;
    check_rhip(rhip_gated_workspace_bytes(&d, RHIP_GATED_BACKWARD, &bytes),
               "rhip_gated_workspace_bytes");
    auto ws = byte_buffer(bytes, dev);
    check_rhip(rhip_gated_backward(&d, s[4].data_ptr(), s[4].numel(), vptr_mut(g[0]),
                                   vptr_mut(g[1]), vptr_mut(g[2]), vptr_mut(g[3]), ws.data_ptr(),
                                   ws.numel(), stream_of(dev)),
               "rhip_gated_backward");
    return {g[0], g[1], g[2], g[3], {}};
  }
};

} // namespace

at::Tensor hip_gated_feed_forward(const at::Tensor &input, const at::Tensor &gate,
                                  const at::Tensor &up, const at::Tensor &down,
                                  const std::string &activation) {
  TORCH_CHECK(input.is_cuda(), "feed-forward input must be a device tensor (no CPU path)");
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) > 0,
              "the gated feed-forward block needs at least one channel");
  hip_dtype(input, "feed-forward input");
  for (const auto *w : {&gate, &up, &down})
    TORCH_CHECK(w->device() == input.device() && w->scalar_type() == input.scalar_type() &&
                    w->dim() == 2,
                "feed-forward weights must be matrices of the input's dtype and device");
  const int64_t C = input.size(-1), H = gate.size(0);
  TORCH_CHECK(H > 0 && gate.size(1) == C && up.sizes() == gate.sizes(),
              "gate and up must be [hidden, ", C, "] both, got ", gate.sizes(), " and ",
              up.sizes());
  TORCH_CHECK(down.size(1) == H && down.size(0) > 0, "down must be [outputs, ", H, "], got ",
              down.sizes());
  for (const int64_t wide : {C, H, down.size(0)})
    TORCH_CHECK(wide <= int64_t(1) << 20, "the gated feed-forward block takes widths up to 2^20, got ",
                wide);
  const int64_t kind = activation_of(activation);
  // the rows of the last axis; a 2-D view keeps its row stride
  auto x = dense_last(input.dim() == 2 ? input : input.reshape({-1, C}));
  auto g = dense_last(gate), u = dense_last(up), d = dense_last(down);
  auto y = through_autograd({input, gate, up, down})
               ? HipGatedFunction::apply(x, g, u, d, kind)
               : run_gated(x, g, u, d, kind, nullptr);
  if (input.dim() == 2)
    return y;
  auto shape = input.sizes().vec();
  shape.back() = down.size(0);
  return y.reshape(shape);
}

RiemannGatedFeedForwardImpl::RiemannGatedFeedForwardImpl(int64_t channels, int64_t hidden,
                                                         const std::string &activation)
    : channels_(channels), hidden_(hidden), activation_(activation) {
  TORCH_CHECK(channels > 0 && hidden > 0, "RiemannGatedFeedForward needs channels and hidden ones");
  activation_of(activation);
  reset();
}

void RiemannGatedFeedForwardImpl::reset() {
  // as torch's linear layers begin
  auto weight = [&](const char *name, int64_t out, int64_t in) {
    const double bound = 1.0 / std::sqrt(static_cast<double>(in));
    return register_parameter(name, torch::empty({out, in}).uniform_(-bound, bound));
  };
  gate_ = weight("gate", hidden_, channels_);
  up_ = weight("up", hidden_, channels_);
  down_ = weight("down", channels_, hidden_);
}

at::Tensor RiemannGatedFeedForwardImpl::forward(const at::Tensor &input) {
  return hip_gated_feed_forward(input, gate_, up_, down_, activation_);
}

SparseTensor RiemannGatedFeedForwardImpl::forward(const SparseTensor &input) {
  const auto &x = input.F();
  TORCH_CHECK(x.dim() == 2 && x.size(1) == channels_, "RiemannGatedFeedForward expects [N, ",
              channels_, "] features, got ", x.sizes());
  return SparseTensor(forward(x), input.coordinate_map_key(), input.coordinate_manager());
}

} // namespace riemann
