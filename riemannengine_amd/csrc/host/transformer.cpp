// Transformer stages over packed rows: attention inside every sequence, layer
// norm and embedding lookup as autograd functions over the HIP kernels
// (rhip_attn_*, rhip_ln_*, rhip_embed_*), and the layers that put them on
// sparse tensors (a sequence = the rows of one batch). These layers have no
// counterpart in the reference; they follow its layers' conventions.
#include <cmath>
#include <limits>

#include <ATen/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include "riemann.hpp"

namespace riemann {

namespace {

using torch::autograd::AutogradContext;
using torch::autograd::tensor_list;

hipStream_t stream_of(const at::Device &dev) {
  return c10::hip::getCurrentHIPStream(dev.index()).stream();
}

at::Tensor byte_buffer(size_t bytes, const at::Device &dev) {
  return torch::empty({static_cast<int64_t>(bytes)},
                      torch::TensorOptions().dtype(torch::kUInt8).device(dev));
}

int32_t hip_dtype(const at::Tensor &t, const char *what) {
  if (t.scalar_type() == torch::kBFloat16)
    return RHIP_BF16;
  TORCH_CHECK(t.scalar_type() == torch::kFloat, what, " must be fp32 or bf16, got ",
              t.scalar_type());
  return RHIP_F32;
}

// Optional tensors travel through autograd as empty tensors.
bool present(const at::Tensor &t) { return t.defined() && t.numel() > 0; }
at::Tensor or_empty(const at::Tensor &t, const at::Tensor &like) {
  return t.defined() ? t : torch::empty({0}, like.options());
}
const float *fptr(const at::Tensor &t) { return present(t) ? t.data_ptr<float>() : nullptr; }
float *fptr_mut(at::Tensor &t) { return t.defined() ? t.data_ptr<float>() : nullptr; }
void *vptr_mut(at::Tensor &t) { return t.defined() ? t.data_ptr() : nullptr; }

// The kernels take any strides but a strided last axis.
at::Tensor dense_last(const at::Tensor &t) {
  return t.size(-1) <= 1 || t.stride(-1) == 1 ? t : t.contiguous();
}

at::Tensor int_vector(const at::Tensor &t, const at::Device &dev, const char *what) {
  TORCH_CHECK(t.device() == dev, what, " must be on the queries' device");
  TORCH_CHECK(t.dim() == 1 && (t.scalar_type() == torch::kInt || t.scalar_type() == torch::kLong),
              what, " must be a vector of int32 or int64");
  return t.to(torch::kInt).contiguous();
}

// Whether a call goes through its autograd function: an input is recorded, or
// carries a forward-mode tangent (which the function refuses; without it the
// result would lose the tangent).
bool through_autograd(std::initializer_list<at::Tensor> ts) {
  for (const auto &t : ts)
    if (t.defined() && ((torch::GradMode::is_enabled() && t.requires_grad()) ||
                        t._fw_grad(0).defined()))
      return true;
  return false;
}

// ------------------------------------------------------------- attention

struct Attention {
  at::Tensor q, k, v, q_offsets, k_offsets, k_lengths;
  bool causal;
  double scale;

  rhip_attn desc() const {
    rhip_attn d{};
    d.n_q = q.size(0), d.n_k = k.size(0);
    d.q_row = q.stride(0), d.q_head = q.stride(1);
    d.k_row = k.stride(0), d.k_head = k.stride(1);
    d.v_row = v.stride(0), d.v_head = v.stride(1);
    d.q_offsets = q_offsets.data_ptr<int32_t>();
    d.k_offsets = k_offsets.data_ptr<int32_t>();
    d.k_lengths = present(k_lengths) ? k_lengths.data_ptr<int32_t>() : nullptr;
    d.n_seq = static_cast<int32_t>(q_offsets.numel() - 1);
    d.heads = static_cast<int32_t>(q.size(1));
    d.kv_heads = static_cast<int32_t>(k.size(1));
    d.dim = static_cast<int32_t>(q.size(2));
    d.causal = causal ? 1 : 0;
    d.dtype = hip_dtype(q, "queries");
    d.scale = static_cast<float>(scale);
    return d;
  }

  // With lse, also what the backward pass needs of bf16 results: out's
  // rounding error.
  at::Tensor forward(at::Tensor *lse, at::Tensor *rest) const {
    const auto dev = q.device();
    at::DeviceGuard guard(dev);
    const rhip_attn d = desc();
    auto out = torch::empty(q.sizes(), q.options());
    if (lse) {
      *lse = torch::empty({q.size(1), q.size(0)}, q.options().dtype(torch::kFloat));
      if (d.dtype == RHIP_BF16)
        *rest = torch::empty(q.sizes(), q.options());
      else
        *rest = torch::empty({0}, q.options());
    }
    size_t bytes = 0;
    check_rhip(rhip_attn_workspace_bytes(&d, 0, &bytes), "rhip_attn_workspace_bytes");
    auto ws = byte_buffer(bytes, dev);
    check_rhip(rhip_attn_forward(&d, q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(),
                                 lse && present(*rest) ? rest->data_ptr() : nullptr,
                                 lse ? lse->data_ptr<float>() : nullptr, ws.data_ptr(),
                                 ws.numel(), stream_of(dev)),
               "rhip_attn_forward");
    return out;
  }
};

struct HipAttentionFunction : public torch::autograd::Function<HipAttentionFunction> {
  static at::Tensor forward(AutogradContext *ctx, at::Tensor q, at::Tensor k, at::Tensor v,
                            at::Tensor q_offsets, at::Tensor k_offsets, at::Tensor k_lengths,
                            bool causal, double scale) {
    const Attention a{q, k, v, q_offsets, k_offsets, k_lengths, causal, scale};
    at::Tensor lse, rest;
    auto out = a.forward(&lse, &rest);
    ctx->save_for_backward({q, k, v, out, lse, q_offsets, k_offsets, k_lengths, rest});
    ctx->saved_data["causal"] = causal;
    ctx->saved_data["scale"] = scale;
    return out;
  }

  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    auto s = ctx->get_saved_variables();
    const Attention a{s[0], s[1], s[2], s[5], s[6], s[7], ctx->saved_data["causal"].toBool(),
                      ctx->saved_data["scale"].toDouble()};
    const auto dev = a.q.device();
    at::DeviceGuard guard(dev);
    const rhip_attn d = a.desc();
    auto go = dense_last(grads[0].to(a.q.scalar_type()));
    at::Tensor gq, gk, gv;
    if (ctx->needs_input_grad(0))
      gq = torch::empty(a.q.sizes(), a.q.options());
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
      gk = torch::empty(a.k.sizes(), a.k.options());
      gv = torch::empty(a.v.sizes(), a.v.options());
    }
    size_t bytes = 0;
    check_rhip(rhip_attn_workspace_bytes(&d, 1, &bytes), "rhip_attn_workspace_bytes");
    auto ws = byte_buffer(bytes, dev);
    check_rhip(rhip_attn_backward(&d, go.data_ptr(), go.stride(0), go.stride(1), a.q.data_ptr(),
                                  a.k.data_ptr(), a.v.data_ptr(), s[3].data_ptr(),
                                  present(s[8]) ? s[8].data_ptr() : nullptr,
                                  s[4].data_ptr<float>(), vptr_mut(gq), vptr_mut(gk),
                                  vptr_mut(gv), ws.data_ptr(), ws.numel(), stream_of(dev)),
               "rhip_attn_backward");
    return {gq, gk, gv, {}, {}, {}, {}, {}};
  }
};

// ------------------------------------------------------------ layer norm

at::Tensor run_layer_norm(const at::Tensor &x, const at::Tensor &weight, const at::Tensor &bias,
                          double eps, at::Tensor *mean, at::Tensor *rstd) {
  const auto dev = x.device();
  at::DeviceGuard guard(dev);
  const int64_t n = x.size(0), C = x.size(1);
  auto y = torch::empty({n, C}, x.options());
  if (mean) {
    const auto f32 = x.options().dtype(torch::kFloat);
    *mean = torch::empty({n}, f32);
    *rstd = torch::empty({n}, f32);
  }
  check_rhip(rhip_ln_forward(x.data_ptr(), x.stride(0), n, static_cast<int32_t>(C), fptr(weight),
                             fptr(bias), eps, y.data_ptr(),
                             mean ? mean->data_ptr<float>() : nullptr,
                             mean ? rstd->data_ptr<float>() : nullptr,
                             hip_dtype(x, "layer norm input"), stream_of(dev)),
             "rhip_ln_forward");
  return y;
}

struct HipLayerNormFunction : public torch::autograd::Function<HipLayerNormFunction> {
  static at::Tensor forward(AutogradContext *ctx, at::Tensor x, at::Tensor weight,
                            at::Tensor bias, double eps) {
    at::Tensor mean, rstd;
    auto y = run_layer_norm(x, weight, bias, eps, &mean, &rstd);
    ctx->save_for_backward({x, weight, mean, rstd});
    return y;
  }

  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    auto s = ctx->get_saved_variables();
    auto x = s[0], weight = s[1], mean = s[2], rstd = s[3];
    const auto dev = x.device();
    at::DeviceGuard guard(dev);
    const int64_t n = x.size(0), C = x.size(1);
    auto gy = dense_last(grads[0].to(x.scalar_type()));
    at::Tensor gx, gw, gb, ws;
    const auto f32 = x.options().dtype(torch::kFloat);
    if (ctx->needs_input_grad(0))
      gx = torch::empty({n, C}, x.options());
    if (ctx->needs_input_grad(1))
      gw = torch::empty({C}, f32);
    if (ctx->needs_input_grad(2))
      gb = torch::empty({C}, f32);
    if (gw.defined() || gb.defined()) {
      size_t bytes = 0;
      check_rhip(rhip_ln_workspace_bytes(n, static_cast<int32_t>(C), &bytes),
                 "rhip_ln_workspace_bytes");
      ws = byte_buffer(bytes, dev);
    }
    check_rhip(rhip_ln_backward(gy.data_ptr(), gy.stride(0), x.data_ptr(), x.stride(0), n,
                                static_cast<int32_t>(C), fptr(mean), fptr(rstd), fptr(weight),
                                vptr_mut(gx), fptr_mut(gw), fptr_mut(gb),
                                hip_dtype(x, "layer norm input"), vptr_mut(ws),
                                ws.defined() ? ws.numel() : 0, stream_of(dev)),
               "rhip_ln_backward");
    return {gx, gw, gb, {}};
  }
};

// ------------------------------------------------------------- embedding

at::Tensor run_embedding(const at::Tensor &ids, const at::Tensor &weight, double scale) {
  const auto dev = weight.device();
  at::DeviceGuard guard(dev);
  const int64_t n = ids.numel(), V = weight.size(0), C = weight.size(1);
  auto y = torch::empty({n, C}, weight.options());
  check_rhip(rhip_embed_forward(ids.data_ptr(), ids.scalar_type() == torch::kInt ? 1 : 0, n,
                                weight.data_ptr(), weight.stride(0), V, static_cast<int32_t>(C),
                                static_cast<float>(scale), y.data_ptr(),
                                hip_dtype(weight, "embedding weight"), stream_of(dev)),
             "rhip_embed_forward");
  return y;
}

struct HipEmbeddingFunction : public torch::autograd::Function<HipEmbeddingFunction> {
  static at::Tensor forward(AutogradContext *ctx, at::Tensor ids, at::Tensor weight,
                            double scale) {
    ctx->save_for_backward({ids});
    ctx->saved_data["rows"] = weight.size(0);
    ctx->saved_data["scale"] = scale;
    return run_embedding(ids, weight, scale);
  }

  static tensor_list backward(AutogradContext *ctx, tensor_list grads) {
    auto ids = ctx->get_saved_variables()[0];
    auto gy = dense_last(grads[0]);
    const auto dev = gy.device();
    at::DeviceGuard guard(dev);
    const int64_t n = gy.size(0), V = ctx->saved_data["rows"].toInt(), C = gy.size(1);
    auto gw = torch::empty({V, C}, gy.options());
    size_t bytes = 0;
    check_rhip(rhip_embed_workspace_bytes(n, V, static_cast<int32_t>(C), &bytes),
               "rhip_embed_workspace_bytes");
    auto ws = byte_buffer(bytes, dev);
    check_rhip(rhip_embed_backward(gy.data_ptr(), gy.stride(0), ids.data_ptr(),
                                   ids.scalar_type() == torch::kInt ? 1 : 0, n, V,
                                   static_cast<int32_t>(C),
                                   static_cast<float>(ctx->saved_data["scale"].toDouble()),
                                   gw.data_ptr(), hip_dtype(gy, "embedding gradient"),
                                   ws.data_ptr(), ws.numel(), stream_of(dev)),
               "rhip_embed_backward");
    return {{}, gw, {}};
  }
};

// The rows of a sparse tensor grouped by batch: `members` (int64) in batch
// order, seg the sequences' offsets. Rows of negative batches follow the last.
struct Scenes {
  at::Tensor members, seg;
};
Scenes scenes_of(const SparseTensor &input) {
  const auto coords = input.C().contiguous();
  const auto dev = coords.device();
  at::DeviceGuard guard(dev);
  const hipStream_t st = stream_of(dev);
  const int64_t n = coords.size(0);
  const int32_t ncol = static_cast<int32_t>(coords.size(1));
  size_t bytes = 0;
  check_rhip(rhip_global_pool_workspace_bytes(n, 1, 0, &bytes),
             "rhip_global_pool_workspace_bytes");
  auto ws = byte_buffer(bytes, dev);
  int32_t n_batches = 0;
  check_rhip(rhip_batch_count(coords.data_ptr<int32_t>(), n, ncol, ws.data_ptr(), ws.numel(),
                              &n_batches, st),
             "rhip_batch_count");
  auto iopt = torch::TensorOptions().dtype(torch::kInt32).device(dev);
  auto members = torch::empty({std::max<int64_t>(n, 1)}, iopt);
  auto seg = torch::empty({n_batches + 1}, iopt);
  check_rhip(rhip_batch_segments(coords.data_ptr<int32_t>(), n, ncol, n_batches, ws.data_ptr(),
                                 ws.numel(), members.data_ptr<int32_t>(),
                                 seg.data_ptr<int32_t>(), st),
             "rhip_batch_segments");
  return {members.slice(0, 0, n).to(torch::kLong), seg};
}

} // namespace

// ------------------------------------------------------------- functions

at::Tensor hip_packed_attention(const at::Tensor &query, const at::Tensor &key,
                                const at::Tensor &value, const at::Tensor &query_offsets,
                                const at::Tensor &key_offsets, const at::Tensor &key_lengths,
                                bool causal, c10::optional<double> scale) {
  TORCH_CHECK(query.is_cuda() && key.device() == query.device() &&
                  value.device() == query.device(),
              "query, key and value must be on one device (the HIP path has no CPU fallback)");
  TORCH_CHECK(query.dim() == 3 && key.dim() == 3 && value.dim() == 3,
              "query must be [rows, heads, width], key and value [rows, key heads, width]");
  TORCH_CHECK(key.sizes() == value.sizes(), "key ", key.sizes(), " and value ", value.sizes(),
              " must have the same shape");
  TORCH_CHECK(key.size(2) == query.size(2), "query width ", query.size(2), " != key width ",
              key.size(2));
  TORCH_CHECK(key.size(1) > 0 && query.size(1) > 0 && query.size(1) % key.size(1) == 0,
              "query heads ", query.size(1), " must be a multiple of key heads ", key.size(1));
  hip_dtype(query, "query");
  TORCH_CHECK(key.scalar_type() == query.scalar_type() &&
                  value.scalar_type() == query.scalar_type(),
              "query, key and value must share their dtype");
  const auto dev = query.device();
  auto qo = int_vector(query_offsets, dev, "query offsets");
  auto ko = key_offsets.defined() && !key_offsets.is_same(query_offsets)
                ? int_vector(key_offsets, dev, "key offsets")
                : qo;
  TORCH_CHECK(qo.numel() >= 1 && ko.numel() == qo.numel(),
              "query and key offsets must hold one value more than there are sequences");
  TORCH_CHECK(key_offsets.defined() || key.size(0) == query.size(0),
              "without key offsets, keys and queries must have the same rows");
  at::Tensor kl;
  if (key_lengths.defined()) {
    kl = int_vector(key_lengths, dev, "key lengths");
    TORCH_CHECK(kl.numel() == qo.numel() - 1, "key lengths must hold one value per sequence");
  }
  const double s = scale.value_or(1.0 / std::sqrt(static_cast<double>(query.size(2))));
  auto q = dense_last(query), k = dense_last(key), v = dense_last(value);
  if (through_autograd({query, key, value}))
    return HipAttentionFunction::apply(q, k, v, qo, ko, or_empty(kl, qo), causal, s);
  return Attention{q, k, v, qo, ko, kl, causal, s}.forward(nullptr, nullptr);
}

at::Tensor hip_layer_norm(const at::Tensor &input, const at::Tensor &weight,
                          const at::Tensor &bias, double eps) {
  TORCH_CHECK(input.is_cuda(), "layer norm input must be a device tensor (no CPU path)");
  TORCH_CHECK(input.dim() >= 1 && input.size(-1) > 0, "layer norm needs at least one channel");
  hip_dtype(input, "layer norm input");
  const int64_t C = input.size(-1);
  TORCH_CHECK(C < INT32_MAX, "layer norm takes fewer than 2^31 - 1 channels, got ", C);
  for (const auto *p : {&weight, &bias})
    TORCH_CHECK(!p->defined() || (p->device() == input.device() &&
                                  p->scalar_type() == torch::kFloat && p->dim() == 1 &&
                                  p->size(0) == C),
                "layer norm weight and bias must be fp32 vectors of ", C, " on the input's device");
  // the rows of the last axis; a 2-D view keeps its row stride
  auto x = dense_last(input.dim() == 2 ? input : input.reshape({-1, C}));
  auto w = weight.defined() ? weight.contiguous() : weight;
  auto b = bias.defined() ? bias.contiguous() : bias;
  auto y = through_autograd({input, weight, bias})
               ? HipLayerNormFunction::apply(x, or_empty(w, x), or_empty(b, x), eps)
               : run_layer_norm(x, w, b, eps, nullptr, nullptr);
  return input.dim() == 2 ? y : y.reshape(input.sizes());
}

at::Tensor hip_embedding(const at::Tensor &ids, const at::Tensor &weight, double scale) {
  TORCH_CHECK(weight.is_cuda() && ids.device() == weight.device(),
              "ids and embedding weight must be on one device (no CPU path)");
  TORCH_CHECK(ids.scalar_type() == torch::kInt || ids.scalar_type() == torch::kLong,
              "ids must be int32 or int64");
  TORCH_CHECK(weight.dim() == 2 && weight.size(1) > 0, "embedding weight must be [rows, channels]");
  TORCH_CHECK(weight.size(1) < INT32_MAX, "embedding takes fewer than 2^31 - 1 channels, got ",
              weight.size(1));
  TORCH_CHECK(std::abs(scale) <= std::numeric_limits<float>::max(), "scale must be finite in fp32");
  hip_dtype(weight, "embedding weight");
  auto flat = ids.reshape({-1}).contiguous();
  auto w = dense_last(weight);
  auto y = through_autograd({weight}) ? HipEmbeddingFunction::apply(flat, w, scale)
                                : run_embedding(flat, w, scale);
  if (ids.dim() == 1)
    return y;
  auto shape = ids.sizes().vec();
  shape.push_back(weight.size(1));
  return y.reshape(shape);
}

// ---------------------------------------------------------------- layers

RiemannLayerNormImpl::RiemannLayerNormImpl(int64_t num_features, double eps, bool affine)
    : num_features_(num_features), eps_(eps), affine_(affine) {
  TORCH_CHECK(num_features > 0, "RiemannLayerNorm needs at least one feature");
  reset();
}

void RiemannLayerNormImpl::reset() {
  if (!affine_)
    return;
  weight_ = register_parameter("weight", torch::ones({num_features_}));
  bias_ = register_parameter("bias", torch::zeros({num_features_}));
}

void RiemannLayerNormImpl::to(torch::Dtype, bool) {}

void RiemannLayerNormImpl::to(torch::Device device, torch::Dtype, bool non_blocking) {
  torch::nn::Module::to(device, non_blocking);
}

SparseTensor RiemannLayerNormImpl::forward(const SparseTensor &input) {
  const auto &x = input.F();
  TORCH_CHECK(x.dim() == 2 && x.size(1) == num_features_, "RiemannLayerNorm expects [N, ",
              num_features_, "] features, got ", x.sizes());
  return SparseTensor(hip_layer_norm(x, weight_, bias_, eps_), input.coordinate_map_key(),
                      input.coordinate_manager());
}

RiemannEmbeddingImpl::RiemannEmbeddingImpl(int64_t num_embeddings, int64_t channels, double scale)
    : num_embeddings_(num_embeddings), channels_(channels), scale_(scale) {
  TORCH_CHECK(num_embeddings > 0 && channels > 0, "RiemannEmbedding needs rows and channels");
  reset();
}

void RiemannEmbeddingImpl::reset() {
  weight_ = register_parameter("weight", torch::randn({num_embeddings_, channels_}) /
                                             std::sqrt(static_cast<double>(channels_)));
}

at::Tensor RiemannEmbeddingImpl::forward(const at::Tensor &ids) {
  return hip_embedding(ids, weight_, scale_);
}

SparseTensor RiemannEmbeddingImpl::forward(const at::Tensor &ids, const SparseTensor &rows) {
  TORCH_CHECK(ids.dim() == 1 && ids.size(0) == rows.F().size(0),
              "RiemannEmbedding expects one id per row");
  return SparseTensor(hip_embedding(ids, weight_, scale_), rows.coordinate_map_key(),
                      rows.coordinate_manager());
}

RiemannAttentionImpl::RiemannAttentionImpl(int64_t channels, int64_t heads, int64_t kv_heads,
                                           bool causal, bool bias)
    : channels_(channels), heads_(heads), kv_heads_(kv_heads == 0 ? heads : kv_heads),
      causal_(causal), has_bias_(bias) {
  TORCH_CHECK(channels > 0 && heads > 0 && channels % heads == 0,
              "RiemannAttention needs a multiple of ", heads, " channels, got ", channels);
  TORCH_CHECK(kv_heads_ > 0 && heads % kv_heads_ == 0, "heads ", heads, " must be a multiple of key heads ",
              kv_heads_);
  reset();
}

void RiemannAttentionImpl::reset() {
  const int64_t dim = channels_ / heads_;
  projection_ = register_module(
      "projection", torch::nn::Linear(torch::nn::LinearOptions(
                                          channels_, (heads_ + 2 * kv_heads_) * dim)
                                          .bias(has_bias_)));
  output_ = register_module(
      "output",
      torch::nn::Linear(torch::nn::LinearOptions(channels_, channels_).bias(has_bias_)));
}

SparseTensor RiemannAttentionImpl::forward(const SparseTensor &input) {
  const auto &x = input.F();
  TORCH_CHECK(x.dim() == 2 && x.size(1) == channels_, "RiemannAttention expects [N, ", channels_,
              "] features, got ", x.sizes());
  TORCH_CHECK(x.is_cuda(), "features must be device tensors (no CPU attention path)");
  const int64_t n = x.size(0), dim = channels_ / heads_;
  const Scenes scenes = scenes_of(input);
  auto rows = projection_->forward(x.index_select(0, scenes.members))
                  .view({n, heads_ + 2 * kv_heads_, dim});
  auto mixed = hip_packed_attention(rows.narrow(1, 0, heads_),
                                    rows.narrow(1, heads_, kv_heads_),
                                    rows.narrow(1, heads_ + kv_heads_, kv_heads_), scenes.seg,
                                    scenes.seg, at::Tensor(), causal_, c10::nullopt);
  auto out = output_->forward(mixed.view({n, channels_}));
  // back to the tensor's own row order
  auto back = torch::empty_like(scenes.members)
                  .index_copy_(0, scenes.members, torch::arange(n, scenes.members.options()));
  return SparseTensor(out.index_select(0, back), input.coordinate_map_key(),
                      input.coordinate_manager());
}

AttentionBlockImpl::AttentionBlockImpl(int64_t channels, int64_t heads, int64_t kv_heads,
                                       int64_t expansion, bool causal)
    : channels_(channels), heads_(heads), kv_heads_(kv_heads), expansion_(expansion),
      causal_(causal) {
  TORCH_CHECK(expansion > 0, "AttentionBlock expansion must be positive");
  reset();
}

void AttentionBlockImpl::reset() {
  norm1_ = register_module("norm1", RiemannLayerNorm(channels_));
  attention_ =
      register_module("attention", RiemannAttention(channels_, heads_, kv_heads_, causal_));
  norm2_ = register_module("norm2", RiemannLayerNorm(channels_));
  up_ = register_module("up", torch::nn::Linear(channels_, channels_ * expansion_));
  down_ = register_module("down", torch::nn::Linear(channels_ * expansion_, channels_));
}

SparseTensor AttentionBlockImpl::forward(const SparseTensor &input) {
  auto x = input.F() + attention_->forward(norm1_->forward(input)).F();
  SparseTensor mid(x, input.coordinate_map_key(), input.coordinate_manager());
  x = x + down_->forward(torch::gelu(up_->forward(norm2_->forward(mid).F())));
  return SparseTensor(std::move(x), input.coordinate_map_key(), input.coordinate_manager());
}

} // namespace riemann
