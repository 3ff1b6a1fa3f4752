// The rotation of heads by positions, with the heads' norm before it or
// without, as an autograd function over the HIP kernels (rhip_rotary_*).
#include <cmath>

#include "transformer.hpp"

namespace riemann {

namespace {

using Sections = std::vector<int64_t>;
constexpr int64_t kMaxHeads = int64_t(1) << 20;

struct Rotation {
  at::Tensor positions, frequencies;
  Sections sections;
  bool interleaved, norm;
  double eps;

  rhip_rotary desc(const at::Tensor &q) const {
    rhip_rotary r{};
    r.n = q.size(0), r.dim = static_cast<int32_t>(q.size(2));
    r.positions = positions.data_ptr();
    r.position_row = positions.stride(0);
    r.position_type = positions.scalar_type() == torch::kInt    ? RHIP_POSITION_I32
                      : positions.scalar_type() == torch::kLong ? RHIP_POSITION_I64
                                                                : RHIP_POSITION_F32;
    r.frequencies = frequencies.data_ptr<double>();
    r.axes = static_cast<int32_t>(sections.size());
    for (size_t i = 0; i < sections.size(); ++i)
      r.sections[i] = static_cast<int32_t>(sections[i]);
    r.interleaved = interleaved, r.norm = norm;
    r.dtype = hip_dtype(q, "rotated heads");
    r.eps = eps;
    return r;
  }

  // y of q and, where it has heads, of k
  tensor_list forward(const at::Tensor &q, const at::Tensor &k, const at::Tensor &wq,
                      const at::Tensor &wk) const {
    const auto dev = q.device();
    at::DeviceGuard guard(dev);
    const rhip_rotary r = desc(q);
    tensor_list out;
    rhip_rotary_heads h[2]{};
    for (const auto *x : {&q, &k}) {
      if (!x->defined())
        continue;
      const size_t i = out.size();
      out.push_back(torch::empty(x->sizes(), x->options()));
      h[i].x = x->data_ptr(), h[i].x_row = x->stride(0), h[i].x_head = x->stride(1);
      h[i].weight = fptr(i ? wk : wq);
      h[i].y = out[i].data_ptr();
      h[i].heads = static_cast<int32_t>(x->size(1));
    }
    check_rhip(rhip_rotary_forward(&r, &h[0], k.defined() ? &h[1] : nullptr, stream_of(dev)),
               "rhip_rotary_forward");
    return out;
  }
};

struct HipRotaryFunction : public torch::autograd::Function<HipRotaryFunction> {
  // k, wq and wk may be empty
  static tensor_list forward(AutogradContext *ctx, at::Tensor q, at::Tensor k, at::Tensor wq,
                             at::Tensor wk, at::Tensor positions, at::Tensor frequencies,
                             Sections sections, bool two, bool interleaved, bool norm,
                             double eps) {
    const Rotation r{positions, frequencies, sections, interleaved, norm, eps};
    // without the norm the gradient does not need x
    ctx->save_for_backward({norm ? q : at::Tensor(), norm ? k : at::Tensor(), wq, wk, positions,
                            frequencies});
    ctx->saved_data["sections"] = sections;
    ctx->saved_data["two"] = two;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["norm"] = norm;
    ctx->saved_data["eps"] = eps;
    return r.forward(q, two ? k : at::Tensor(), wq, wk);
  }

  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    first_derivative_only("the rotation of heads");
    auto s = ctx->get_saved_variables();
    const bool two = ctx->saved_data["two"].toBool(), norm = ctx->saved_data["norm"].toBool();
    const Rotation r{s[4],
                     s[5],
                     ctx->saved_data["sections"].toIntVector(),
                     ctx->saved_data["interleaved"].toBool(),
                     norm,
                     ctx->saved_data["eps"].toDouble()};
    const auto dev = grads[0].device();
    at::DeviceGuard guard(dev);
    const rhip_rotary d = r.desc(grads[0]);
    rhip_rotary_heads h[2]{};
    at::Tensor gy[2], gx[2], gw[2];
    bool weights = false;
    for (int i = 0; i < (two ? 2 : 1); ++i) {
      gy[i] = dense_last(grads[i]);
      h[i].heads = static_cast<int32_t>(gy[i].size(1));
      h[i].grad_y = gy[i].data_ptr();
      h[i].grad_y_row = gy[i].stride(0), h[i].grad_y_head = gy[i].stride(1);
      if (norm) {
        h[i].x = s[i].data_ptr(), h[i].x_row = s[i].stride(0), h[i].x_head = s[i].stride(1);
        h[i].weight = fptr(s[2 + i]);
      }
      if (ctx->needs_input_grad(i))
        gx[i] = torch::empty(gy[i].sizes(), gy[i].options());
      if (norm && present(s[2 + i]) && ctx->needs_input_grad(2 + i)) {
        gw[i] = torch::empty(s[2 + i].sizes(), s[2 + i].options());
        weights = true;
      }
      h[i].grad_x = vptr_mut(gx[i]);
      h[i].grad_weight = fptr_mut(gw[i]);
    }
    at::Tensor ws;
    if (weights) {
      size_t bytes = 0;
      check_rhip(rhip_rotary_workspace_bytes(&d, &bytes), "rhip_rotary_workspace_bytes");
      ws = byte_buffer(bytes, dev);
    }
    check_rhip(rhip_rotary_backward(&d, &h[0], two ? &h[1] : nullptr, vptr_mut(ws),
                                    ws.defined() ? ws.numel() : 0, stream_of(dev)),
               "rhip_rotary_backward");
    return {gx[0], gx[1], gw[0], gw[1], {}, {}, {}, {}, {}, {}, {}};
  }
};

at::Tensor checked_positions(const at::Tensor &positions, const at::Tensor &query,
                             const Sections &sections) {
  TORCH_CHECK(positions.device() == query.device(), "positions must be on the heads' device");
  TORCH_CHECK(positions.scalar_type() == torch::kInt || positions.scalar_type() == torch::kLong ||
                  positions.scalar_type() == torch::kFloat,
              "positions must be int32, int64 or fp32, got ", positions.scalar_type());
  auto p = positions.dim() == 1 ? positions.unsqueeze(1) : positions;
  TORCH_CHECK(p.dim() == 2 && p.size(0) == query.size(0) &&
                  p.size(1) == static_cast<int64_t>(sections.size()),
              "positions must be [", query.size(0), " rows, ", sections.size(),
              " axes, one for each section], got ", positions.sizes());
  return dense_last(p);
}

Rotation checked_rotation(const at::Tensor &query, const at::Tensor &positions,
                          const at::Tensor &frequencies, const Sections &sections,
                          bool interleaved, bool norm, double eps) {
  TORCH_CHECK(query.is_cuda(), "heads must be device tensors (the HIP path has no CPU fallback)");
  TORCH_CHECK(query.dim() == 3 && query.size(1) > 0 && query.size(2) > 0,
              "heads must be [rows, heads, width], got ", query.sizes());
  TORCH_CHECK(query.size(2) <= 256, "rotation takes head widths up to 256, got ", query.size(2));
  TORCH_CHECK(query.size(1) <= kMaxHeads, "rotation takes up to 2^20 heads, got ", query.size(1));
  hip_dtype(query, "rotated heads");
  TORCH_CHECK(!sections.empty() && sections.size() <= RHIP_ROTARY_MAX_AXES,
              "rotation takes 1 to ", RHIP_ROTARY_MAX_AXES, " sections, got ", sections.size());
  int64_t pairs = 0;
  for (const int64_t s : sections) {
    TORCH_CHECK(s >= 0 && s <= query.size(2), "sections must lie between 0 and the head width, got ",
                s);
    pairs += s;
  }
  TORCH_CHECK(pairs > 0 && 2 * pairs <= query.size(2), "sections hold ", pairs,
              " pairs; heads of width ", query.size(2), " have 1 to ", query.size(2) / 2);
  TORCH_CHECK(frequencies.device() == query.device() &&
                  frequencies.scalar_type() == torch::kDouble && frequencies.dim() == 1 &&
                  frequencies.size(0) == pairs,
              "frequencies must be an fp64 vector of ", pairs, " pairs on the heads' device");
  for (const auto *t : {&positions, &frequencies})
    TORCH_CHECK(!t->requires_grad() && !t->_fw_grad(0).defined(),
                "positions and frequencies of a rotation have no gradients");
  return {checked_positions(positions, query, sections),
          frequencies.contiguous(),
          sections,
          interleaved,
          norm,
          eps};
}

} // namespace

at::Tensor hip_rotate_heads(const at::Tensor &input, const at::Tensor &positions,
                            const at::Tensor &frequencies, const std::vector<int64_t> &sections,
                            bool interleaved) {
  const Rotation r =
      checked_rotation(input, positions, frequencies, sections, interleaved, false, 1.0);
  auto x = dense_last(input);
  if (!through_autograd({input}))
    return r.forward(x, at::Tensor(), at::Tensor(), at::Tensor())[0];
  const auto none = or_empty(at::Tensor(), x);
  return HipRotaryFunction::apply(x, none, none, none, r.positions, r.frequencies, sections, false,
                                  interleaved, false, 1.0)[0];
}

std::tuple<at::Tensor, at::Tensor>
hip_norm_rotate_heads(const at::Tensor &query, const at::Tensor &key, const at::Tensor &positions,
                      const at::Tensor &frequencies, const std::vector<int64_t> &sections,
                      const at::Tensor &query_weight, const at::Tensor &key_weight, double eps,
                      bool interleaved) {
  const Rotation r =
      checked_rotation(query, positions, frequencies, sections, interleaved, true, eps);
  TORCH_CHECK(key.dim() == 3 && key.size(0) == query.size(0) && key.size(1) > 0 &&
                  key.size(1) <= kMaxHeads && key.size(2) == query.size(2) &&
                  key.device() == query.device() && key.scalar_type() == query.scalar_type(),
              "keys must be [", query.size(0), " rows, up to 2^20 heads, ", query.size(2),
              "] of the queries' dtype and device, got ", key.sizes());
  for (const auto *w : {&query_weight, &key_weight})
    TORCH_CHECK(!w->defined() || (w->device() == query.device() &&
                                  w->scalar_type() == torch::kFloat && w->dim() == 1 &&
                                  w->size(0) == query.size(2)),
                "the heads' norm weights must be fp32 vectors of ", query.size(2),
                " on the queries' device");
  auto q = dense_last(query), k = dense_last(key);
  auto wq = query_weight.defined() ? query_weight.contiguous() : query_weight;
  auto wk = key_weight.defined() ? key_weight.contiguous() : key_weight;
  tensor_list y;
  if (through_autograd({query, key, query_weight, key_weight}))
    y = HipRotaryFunction::apply(q, k, or_empty(wq, q), or_empty(wk, q), r.positions,
                                 r.frequencies, sections, true, interleaved, true, eps);
  else
    y = r.forward(q, k, wq, wk);
  return {y[0], y[1]};
}

at::Tensor rotary_frequencies(const std::vector<int64_t> &sections, double base,
                              const at::Device &device) {
  TORCH_CHECK(std::isfinite(base) && base > 0, "the base must be positive and finite");
  std::vector<at::Tensor> parts;
  for (const int64_t s : sections) {
    TORCH_CHECK(s >= 0, "sections must not be negative");
    parts.push_back(torch::pow(
        base, -torch::arange(s, torch::kDouble) / static_cast<double>(std::max<int64_t>(s, 1))));
  }
  TORCH_CHECK(!parts.empty(), "rotation needs a section");
  return torch::cat(parts).to(device);
}

} // namespace riemann
