// The eager autograd nodes of the layers (attnres.layers), in C++ over the C ABI
// (attnres_layers_hip.h): layer norm, embedding, the loss over a vocabulary and the gated feed-forward block.
//
// Each layer has a forward and a backward function that allocate and launch; the nodes
// call them without Python, and so do the torch.library ops that stand for the nodes
// under torch.compile, so both give the same bits.

#include <torch/extension.h>

#include <torch/csrc/autograd/functions/basic_ops.h>

#include <algorithm>

#include "attnres_layers_hip.h"
#include "attnres_nodes.h"

namespace attnres_nodes {
namespace {

using OptionalTensor = std::optional<Tensor>;

int dtype_of(at::ScalarType type) {
  switch (type) {
    case at::kBFloat16: return ATTNRES_BF16;
    case at::kHalf: return ATTNRES_F16;
    case at::kFloat: return ATTNRES_F32;
    default: TORCH_CHECK_TYPE(false, "attnres layers take BF16, FP16 and FP32 tensors, not ", type);
  }
}

bool wants_grad(at::TensorList tensors) {
  if (!at::GradMode::is_enabled()) return false;
  for (const Tensor& tensor : tensors) {
    if (tensor.defined() && tensor.requires_grad()) return true;
  }
  return false;
}

Tensor value_of(const OptionalTensor& tensor) { return tensor ? *tensor : Tensor(); }
const void* data_of(const Tensor& tensor) { return tensor.defined() && tensor.numel() > 0 ? tensor.data_ptr() : nullptr; }

// Rows a kernel can address: the tensor itself where its rows are evenly spaced and
// unit-stride, else a contiguous copy.
struct Rows {
  Tensor tensor;
  int64_t stride;
};
Rows rows_view(const Tensor& tensor) {
  if (const std::optional<int64_t> stride = row_stride(tensor)) return {tensor, *stride};
  Tensor copy = tensor.contiguous();
  return {copy, copy.size(-1)};
}

// First-order gradients: in a backward pass that is itself recorded (create_graph), differentiating the
// gradients again raises instead of leaving these layers' terms out.
variable_list once_differentiable(variable_list grads) {
  if (!at::GradMode::is_enabled()) return grads;
  variable_list defined;
  for (const Tensor& grad : grads) {
    if (grad.defined()) defined.push_back(grad.detach().requires_grad_(true));
  }
  torch::autograd::DelayedError error("attnres layers have first-order gradients only", static_cast<int64_t>(defined.size()));
  const variable_list marked = error.apply(std::move(defined));
  size_t next = 0;
  for (Tensor& grad : grads) {
    if (grad.defined()) grad = marked[next++];
  }
  return grads;
}

// -------------------------------------------------------------- layer norm

std::tuple<Tensor, Tensor> layer_norm_forward(const Tensor& x, const OptionalTensor& weight, const OptionalTensor& bias,
                                              double eps, bool save) {
  refuse_tangents("layer_norm", x, weight, bias);
  const c10::DeviceGuard guard(x.device());
  const Rows rows = rows_view(x);
  const int64_t width = x.size(-1), count = x.numel() / width;
  const Tensor w = weight ? weight->contiguous() : Tensor(), b = bias ? bias->contiguous() : Tensor();
  const at::ScalarType param = w.defined() ? w.scalar_type() : b.defined() ? b.scalar_type() : x.scalar_type();
  Tensor out = torch::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous));
  Tensor stats = torch::empty({2, save ? count : 0}, x.options().dtype(torch::kFloat32));
  check(attnres_hip_layer_norm_forward(rows.tensor.data_ptr(), rows.stride, count, width, dtype_of(x.scalar_type()), data_of(w),
                                       data_of(b), dtype_of(param), static_cast<float>(eps), out.data_ptr(),
                                       save ? stats.data_ptr<float>() : nullptr, current_stream(x)),
        "layer norm forward");
  return {out, stats};
}

// Gradients that are not wanted come back empty.
std::tuple<Tensor, Tensor, Tensor> layer_norm_backward(const Tensor& grad_out, const Tensor& x, const OptionalTensor& weight,
                                                       at::ScalarType param, const Tensor& stats, bool want_x, bool want_weight,
                                                       bool want_bias) {
  refuse_tangents("layer_norm's backward", grad_out, x, weight);
  const c10::DeviceGuard guard(x.device());
  const Rows rows = rows_view(x);
  const int64_t width = x.size(-1), count = x.numel() / width;
  const Tensor w = weight ? weight->contiguous() : Tensor();
  const Tensor grad = grad_out.to(x.scalar_type()).contiguous(), saved = stats.contiguous();
  const auto params = x.options().dtype(param);
  Tensor grad_x = want_x ? torch::empty(x.sizes(), x.options().memory_format(at::MemoryFormat::Contiguous))
                         : torch::empty({0}, x.options());
  Tensor grad_weight = torch::empty({want_weight ? width : 0}, params), grad_bias = torch::empty({want_bias ? width : 0}, params);
  Tensor workspace;
  if (want_weight || want_bias) {
    workspace = torch::empty({attnres_hip_layer_norm_workspace_elems(count, width)}, x.options().dtype(torch::kFloat32));
  }
  check(attnres_hip_layer_norm_backward(grad.data_ptr(), rows.tensor.data_ptr(), rows.stride, count, width,
                                        dtype_of(x.scalar_type()), data_of(w), dtype_of(param), saved.data_ptr<float>(),
                                        want_x && count > 0 ? grad_x.data_ptr() : nullptr,
                                        want_weight ? grad_weight.data_ptr() : nullptr,
                                        want_bias ? grad_bias.data_ptr() : nullptr,
                                        workspace.defined() ? workspace.data_ptr<float>() : nullptr,
                                        workspace.defined() ? workspace.numel() : 0, current_stream(x)),
        "layer norm backward");
  return {grad_x, grad_weight, grad_bias};
}

struct LayerNorm : public torch::autograd::Function<LayerNorm> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const OptionalTensor& weight, const OptionalTensor& bias,
                        double eps) {
    auto [out, stats] = layer_norm_forward(x, weight, bias, eps, true);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, value_of(weight), stats});
    const at::ScalarType param = weight ? weight->scalar_type() : bias ? bias->scalar_type() : x.scalar_type();
    ctx->saved_data["param"] = static_cast<int64_t>(param);
    ctx->saved_data["weight"] = weight.has_value();
    ctx->saved_data["bias"] = bias.has_value();
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(4);
    if (!grads[0].defined()) return result;
    const bool has_weight = ctx->saved_data["weight"].toBool(), has_bias = ctx->saved_data["bias"].toBool();
    const bool want_x = ctx->needs_input_grad(0), want_weight = has_weight && ctx->needs_input_grad(1);
    const bool want_bias = has_bias && ctx->needs_input_grad(has_weight ? 2 : 1);
    const variable_list saved = ctx->get_saved_variables();
    const auto [grad_x, grad_weight, grad_bias] = layer_norm_backward(
        grads[0], saved[0], has_weight ? OptionalTensor(saved[1]) : std::nullopt,
        static_cast<at::ScalarType>(ctx->saved_data["param"].toInt()), saved[2], want_x, want_weight, want_bias);
    if (want_x) result[0] = grad_x;
    if (want_weight) result[1] = grad_weight;
    if (want_bias) result[2] = grad_bias;
    return once_differentiable(std::move(result));
  }
};

Tensor layer_norm(const Tensor& x, const OptionalTensor& weight, const OptionalTensor& bias, double eps) {
  if (!wants_grad({x, value_of(weight), value_of(bias)})) return std::get<0>(layer_norm_forward(x, weight, bias, eps, false));
  return LayerNorm::apply(x, weight, bias, eps);
}

// --------------------------------------------------------------- embedding

// tokens [..., length]: all leading axes are the batch.
int64_t length_of(const Tensor& tokens) { return tokens.dim() > 0 ? tokens.size(-1) : 1; }
int64_t batch_of(const Tensor& tokens) {
  const int64_t length = length_of(tokens);
  return length > 0 ? tokens.numel() / length : 0;
}

Tensor embedding_forward(const Tensor& tokens, const Tensor& weight, const OptionalTensor& positions, double scale,
                         at::ScalarType dtype) {
  refuse_tangents("embedding", weight, positions);
  const c10::DeviceGuard guard(weight.device());
  const Tensor ids = tokens.contiguous(), table = weight.contiguous();
  const Tensor places = positions ? positions->contiguous() : Tensor();
  std::vector<int64_t> shape = tokens.sizes().vec();
  shape.push_back(weight.size(1));
  Tensor out = torch::empty(shape, weight.options().dtype(dtype));
  check(attnres_hip_embedding_forward(data_of(ids), static_cast<int>(ids.element_size()), batch_of(ids), length_of(ids),
                                      table.data_ptr(), weight.size(0), weight.size(1), dtype_of(weight.scalar_type()),
                                      data_of(places), static_cast<float>(scale), out.data_ptr(), dtype_of(dtype),
                                      current_stream(weight)),
        "embedding forward");
  return out;
}

// position_rows: of the positions' gradient; gradients that are not wanted come back empty.
std::tuple<Tensor, Tensor> embedding_backward(const Tensor& grad_out, const Tensor& tokens, int64_t vocab, int64_t position_rows,
                                              at::ScalarType table, double scale, bool want_weight, bool want_positions) {
  refuse_tangents("embedding's backward", grad_out);
  const c10::DeviceGuard guard(grad_out.device());
  const Tensor grad = grad_out.contiguous(), ids = tokens.contiguous();
  const int64_t width = grad.size(-1), batch = batch_of(ids), length = length_of(ids);
  const auto options = grad.options().dtype(table);
  Tensor grad_weight = torch::empty({want_weight ? vocab : 0, width}, options);
  Tensor grad_positions = torch::empty({want_positions ? position_rows : 0, width}, options);
  Tensor workspace;
  if (want_weight || want_positions) {
    const int64_t bytes = want_weight ? attnres_hip_embedding_workspace_bytes(batch, length, vocab, width)
                                      : attnres_hip_embedding_positions_workspace_bytes(batch, length, width);
    TORCH_CHECK_VALUE(bytes >= 0, "embedding backward: shape outside the supported envelope");
    workspace = torch::empty({bytes}, grad.options().dtype(torch::kUInt8));
  }
  check(attnres_hip_embedding_backward(data_of(grad), dtype_of(grad.scalar_type()), data_of(ids),
                                       static_cast<int>(ids.element_size()), batch, length, vocab, width, dtype_of(table),
                                       static_cast<float>(scale), want_weight ? grad_weight.data_ptr() : nullptr,
                                       want_positions ? grad_positions.data_ptr() : nullptr, position_rows,
                                       workspace.defined() ? workspace.data_ptr() : nullptr,
                                       workspace.defined() ? workspace.numel() : 0, current_stream(grad)),
        "embedding backward");
  return {grad_weight, grad_positions};
}

struct Embedding : public torch::autograd::Function<Embedding> {
  static Tensor forward(AutogradContext* ctx, const Tensor& weight, const OptionalTensor& positions, const Tensor& tokens,
                        double scale, int64_t dtype) {
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({tokens});
    ctx->saved_data["vocab"] = weight.size(0);
    ctx->saved_data["position_rows"] = positions ? positions->size(0) : 0;
    ctx->saved_data["positions"] = positions.has_value();
    ctx->saved_data["table"] = static_cast<int64_t>(weight.scalar_type());
    ctx->saved_data["scale"] = scale;
    return embedding_forward(tokens, weight, positions, scale, static_cast<at::ScalarType>(dtype));
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(5);
    if (!grads[0].defined()) return result;
    const bool want_weight = ctx->needs_input_grad(0);
    const bool want_positions = ctx->saved_data["positions"].toBool() && ctx->needs_input_grad(1);
    const auto [grad_weight, grad_positions] = embedding_backward(
        grads[0], ctx->get_saved_variables()[0], ctx->saved_data["vocab"].toInt(), ctx->saved_data["position_rows"].toInt(),
        static_cast<at::ScalarType>(ctx->saved_data["table"].toInt()), ctx->saved_data["scale"].toDouble(), want_weight,
        want_positions);
    if (want_weight) result[0] = grad_weight;
    if (want_positions) result[1] = grad_positions;
    return once_differentiable(std::move(result));
  }
};

Tensor embedding(const Tensor& tokens, const Tensor& weight, const OptionalTensor& positions, double scale,
                 at::ScalarType dtype) {
  if (!wants_grad({weight, value_of(positions)})) return embedding_forward(tokens, weight, positions, scale, dtype);
  return Embedding::apply(weight, positions, tokens, scale, static_cast<int64_t>(dtype));
}

// -------------------------------------------------------------------- loss

// The vocabulary's rows as the kernels take them: 16-bit rows of whole 32-element steps are
// multiplied where they lie and have to start at multiples of 16 bytes; a copy does.
Rows weight_rows(const Tensor& weight) {
  Rows rows = rows_view(weight);
  if (weight.size(0) == 1 && rows.stride < weight.size(1)) rows.stride = weight.size(1);
  const bool in_place = weight.scalar_type() != at::kFloat && weight.size(1) % 32 == 0;
  if (in_place && (reinterpret_cast<uintptr_t>(rows.tensor.data_ptr()) % 16 != 0 || rows.stride % 8 != 0 ||
                   rows.stride < weight.size(1) || rows.stride > (int64_t{1} << 22))) {
    Tensor copy = torch::empty(weight.sizes(), weight.options().memory_format(at::MemoryFormat::Contiguous));
    copy.copy_(weight);
    rows = {copy, copy.size(-1)};
  }
  return rows;
}

// backward: as attnres_hip_loss_workspace_bytes takes it.
Tensor loss_workspace(const Tensor& hidden, const Tensor& weight, int64_t rows, bool keep, int backward) {
  const int64_t bytes =
      attnres_hip_loss_workspace_bytes(rows, weight.size(0), weight.size(1), dtype_of(weight.scalar_type()), keep, backward);
  TORCH_CHECK_VALUE(bytes >= 0, "linear cross entropy: shape outside the supported envelope");
  return torch::empty({bytes}, hidden.options().dtype(torch::kUInt8));
}

// (loss, saved): the loss has the targets' shape for ATTNRES_REDUCE_NONE, else none.
std::tuple<Tensor, Tensor> loss_forward(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore_index,
                                        int64_t reduction, bool keep) {
  refuse_tangents("linear_cross_entropy", hidden, weight);
  const c10::DeviceGuard guard(hidden.device());
  const at::NoGradGuard no_grad;
  const Rows h = rows_view(hidden), w = weight_rows(weight);
  const Tensor ids = targets.contiguous();
  const int64_t rows = ids.numel();
  const auto floats = hidden.options().dtype(torch::kFloat32);
  Tensor loss = reduction == ATTNRES_REDUCE_NONE ? torch::empty(targets.sizes(), floats) : torch::empty({}, floats);
  Tensor workspace = loss_workspace(hidden, weight, rows, keep, 0);
  Tensor saved = torch::empty(
      {attnres_hip_loss_saved_bytes(rows, weight.size(0), weight.size(1), dtype_of(weight.scalar_type()), keep)},
      hidden.options().dtype(torch::kUInt8));
  if (rows == 0 && reduction == ATTNRES_REDUCE_NONE) return {loss, saved};
  check(attnres_hip_loss_forward(h.tensor.data_ptr(), h.stride, w.tensor.data_ptr(), w.stride, data_of(ids),
                                 static_cast<int>(ids.element_size()), rows, weight.size(0), weight.size(1),
                                 dtype_of(hidden.scalar_type()), ignore_index, static_cast<int>(reduction), keep,
                                 loss.data_ptr<float>(), saved.data_ptr(), workspace.data_ptr(), workspace.numel(),
                                 current_stream(hidden)),
        "linear cross entropy forward");
  return {loss, saved};
}

std::tuple<Tensor, Tensor> loss_backward(const Tensor& grad_loss, const Tensor& hidden, const Tensor& weight, const Tensor& saved,
                                         int64_t reduction, bool keep, bool want_hidden, bool want_weight) {
  refuse_tangents("linear_cross_entropy's backward", grad_loss, hidden, weight);
  const c10::DeviceGuard guard(hidden.device());
  const at::NoGradGuard no_grad;
  const Rows h = rows_view(hidden), w = weight_rows(weight);
  const int64_t rows = hidden.numel() / hidden.size(-1);
  const Tensor grad = grad_loss.to(torch::kFloat32).contiguous();
  const auto contiguous = at::MemoryFormat::Contiguous;
  Tensor grad_hidden = want_hidden ? torch::empty(hidden.sizes(), hidden.options().memory_format(contiguous))
                                   : torch::empty({0}, hidden.options());
  if (rows == 0) {
    return {grad_hidden, want_weight ? torch::zeros(weight.sizes(), weight.options().memory_format(contiguous))
                                     : torch::empty({0}, weight.options())};
  }
  Tensor grad_weight = want_weight ? torch::empty(weight.sizes(), weight.options().memory_format(contiguous))
                                   : torch::empty({0}, weight.options());
  Tensor workspace = loss_workspace(hidden, weight, rows, keep, reduction == ATTNRES_REDUCE_NONE ? 1 : 2);
  check(attnres_hip_loss_backward(h.tensor.data_ptr(), h.stride, w.tensor.data_ptr(), w.stride, rows, weight.size(0),
                                  weight.size(1), dtype_of(hidden.scalar_type()), static_cast<int>(reduction), keep, saved.data_ptr(),
                                  grad.data_ptr<float>(), want_hidden ? grad_hidden.data_ptr() : nullptr,
                                  want_weight ? grad_weight.data_ptr() : nullptr, workspace.data_ptr(), workspace.numel(),
                                  current_stream(hidden)),
        "linear cross entropy backward");
  return {grad_hidden, grad_weight};
}

struct LinearCrossEntropy : public torch::autograd::Function<LinearCrossEntropy> {
  static Tensor forward(AutogradContext* ctx, const Tensor& hidden, const Tensor& weight, const Tensor& targets,
                        int64_t ignore_index, int64_t reduction, bool keep) {
    auto [loss, saved] = loss_forward(hidden, weight, targets, ignore_index, reduction, keep);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({hidden, weight, saved});
    ctx->saved_data["reduction"] = reduction;
    ctx->saved_data["keep"] = keep;
    return loss;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(6);
    if (!grads[0].defined()) return result;
    const variable_list saved = ctx->get_saved_variables();
    const bool want_hidden = ctx->needs_input_grad(0), want_weight = ctx->needs_input_grad(1);
    const auto [grad_hidden, grad_weight] = loss_backward(grads[0], saved[0], saved[1], saved[2],
                                                          ctx->saved_data["reduction"].toInt(), ctx->saved_data["keep"].toBool(),
                                                          want_hidden, want_weight);
    if (want_hidden) result[0] = grad_hidden;
    if (want_weight) result[1] = grad_weight;
    return once_differentiable(std::move(result));
  }
};

Tensor linear_cross_entropy(const Tensor& hidden, const Tensor& weight, const Tensor& targets, int64_t ignore_index,
                            int64_t reduction, bool keep) {
  if (!wants_grad({hidden, weight})) return std::get<0>(loss_forward(hidden, weight, targets, ignore_index, reduction, false));
  return LinearCrossEntropy::apply(hidden, weight, targets, ignore_index, reduction, keep);
}

// ----------------------------------------------------- gated feed-forward

// Rows as the products take them: rows of whole 32-element steps are multiplied where they lie and have to
// start at multiples of 16 bytes, `least` to `most` elements apart; a copy does.
Rows product_rows(const Tensor& tensor, bool in_place, int64_t least, int64_t most) {
  Rows rows = rows_view(tensor);
  if (rows_of(tensor) == 1 && rows.stride < least) rows.stride = least;
  if (in_place && (reinterpret_cast<uintptr_t>(rows.tensor.data_ptr()) % 16 != 0 || rows.stride % 8 != 0 ||
                   rows.stride < least || rows.stride > most)) {
    Tensor copy = torch::empty(tensor.sizes(), tensor.options().memory_format(at::MemoryFormat::Contiguous));
    copy.copy_(tensor);
    rows = {copy, copy.size(-1)};
  }
  return rows;
}

struct FeedForward {
  Rows x, gate_up, down;
  int64_t rows, width, hidden, out_width;
  int dtype;
  FeedForward(const Tensor& input, const Tensor& weights, const Tensor& last)
      : rows(input.numel() / input.size(-1)), width(weights.size(1)), hidden(last.size(1)), out_width(last.size(0)),
        dtype(dtype_of(input.scalar_type())) {
    const bool even = hidden % 32 == 0;
    constexpr int64_t kMost = int64_t{1} << 22;
    const int64_t second = int64_t{1} << (dtype == ATTNRES_F32 ? 29 : 30);
    x = product_rows(input, width % 32 == 0, 0, kMost);
    gate_up = product_rows(weights, width % 32 == 0 && even, width, std::min(kMost, second / hidden));
    down = product_rows(last, even, hidden, kMost);
  }
  Tensor workspace(const Tensor& like, int backward) const {
    const int64_t bytes = attnres_hip_gated_ffn_workspace_bytes(rows, width, hidden, out_width, dtype, backward);
    TORCH_CHECK_VALUE(bytes >= 0, "gated feed-forward: shape outside the supported envelope");
    return torch::empty({bytes}, like.options().dtype(torch::kUInt8));
  }
};

// (out, saved): saved is empty where it is not kept.
std::tuple<Tensor, Tensor> feed_forward_forward(const Tensor& x, const Tensor& gate_up, const Tensor& down, int64_t activation,
                                                bool keep) {
  refuse_tangents("gated_feed_forward", x, gate_up, down);
  const c10::DeviceGuard guard(x.device());
  const at::NoGradGuard no_grad;
  const FeedForward f(x, gate_up, down);
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = f.out_width;
  Tensor out = torch::empty(shape, x.options().memory_format(at::MemoryFormat::Contiguous));
  const auto bytes = x.options().dtype(torch::kUInt8);
  if (f.rows == 0) return {out, torch::empty({0}, bytes)};
  const Tensor workspace = f.workspace(x, 0);
  Tensor saved = torch::empty({keep ? attnres_hip_gated_ffn_saved_bytes(f.rows, f.width, f.hidden, f.out_width, f.dtype) : 0}, bytes);
  check(attnres_hip_gated_ffn_forward(f.x.tensor.data_ptr(), f.x.stride, f.gate_up.tensor.data_ptr(), f.gate_up.stride,
                                      f.down.tensor.data_ptr(), f.down.stride, f.rows, f.width, f.hidden, f.out_width, f.dtype,
                                      static_cast<int>(activation), out.data_ptr(), keep ? saved.data_ptr() : nullptr,
                                      workspace.data_ptr(), workspace.numel(), current_stream(x)),
        "gated feed-forward forward");
  return {out, saved};
}

// saved: empty where the backward forms it again; gradients that are not wanted come back empty.
std::tuple<Tensor, Tensor, Tensor> feed_forward_backward(const Tensor& grad_out, const Tensor& x, const Tensor& gate_up,
                                                         const Tensor& down, const Tensor& saved, int64_t activation, bool want_x,
                                                         bool want_gate_up, bool want_down) {
  refuse_tangents("gated_feed_forward's backward", grad_out, x, gate_up, down);
  const c10::DeviceGuard guard(x.device());
  const at::NoGradGuard no_grad;
  const FeedForward f(x, gate_up, down);
  const auto result = [&](const Tensor& like, bool wanted) {
    if (!wanted) return torch::empty({0}, like.options());
    const auto options = like.options().memory_format(at::MemoryFormat::Contiguous);
    return f.rows == 0 ? torch::zeros(like.sizes(), options) : torch::empty(like.sizes(), options);
  };
  Tensor grad_x = result(x, want_x), grad_gate_up = result(gate_up, want_gate_up), grad_down = result(down, want_down);
  if (f.rows == 0) return {grad_x, grad_gate_up, grad_down};
  Tensor grad = grad_out.to(x.scalar_type()).contiguous();
  if (reinterpret_cast<uintptr_t>(grad.data_ptr()) % 16 != 0) grad = grad.clone();
  const Tensor workspace = f.workspace(x, saved.numel() > 0 ? 1 : 2);
  check(attnres_hip_gated_ffn_backward(grad.data_ptr(), f.x.tensor.data_ptr(), f.x.stride, f.gate_up.tensor.data_ptr(),
                                       f.gate_up.stride, f.down.tensor.data_ptr(), f.down.stride, f.rows, f.width, f.hidden,
                                       f.out_width, f.dtype, static_cast<int>(activation),
                                       saved.numel() > 0 ? saved.data_ptr() : nullptr, want_x ? grad_x.data_ptr() : nullptr,
                                       want_gate_up ? grad_gate_up.data_ptr() : nullptr,
                                       want_down ? grad_down.data_ptr() : nullptr, workspace.data_ptr(), workspace.numel(),
                                       current_stream(x)),
        "gated feed-forward backward");
  return {grad_x, grad_gate_up, grad_down};
}

struct GatedFeedForward : public torch::autograd::Function<GatedFeedForward> {
  static Tensor forward(AutogradContext* ctx, const Tensor& x, const Tensor& gate_up, const Tensor& down, int64_t activation,
                        bool keep) {
    auto [out, saved] = feed_forward_forward(x, gate_up, down, activation, keep);
    ctx->set_materialize_grads(false);
    ctx->save_for_backward({x, gate_up, down, saved});
    ctx->saved_data["activation"] = activation;
    return out;
  }

  static variable_list backward(AutogradContext* ctx, variable_list grads) {
    variable_list result(5);
    if (!grads[0].defined()) return result;
    const variable_list saved = ctx->get_saved_variables();
    const bool want[3] = {ctx->needs_input_grad(0), ctx->needs_input_grad(1), ctx->needs_input_grad(2)};
    const auto [grad_x, grad_gate_up, grad_down] =
        feed_forward_backward(grads[0], saved[0], saved[1], saved[2], saved[3], ctx->saved_data["activation"].toInt(), want[0],
                              want[1], want[2]);
    if (want[0]) result[0] = grad_x;
    if (want[1]) result[1] = grad_gate_up;
    if (want[2]) result[2] = grad_down;
    return once_differentiable(std::move(result));
  }
};

Tensor gated_feed_forward(const Tensor& x, const Tensor& gate_up, const Tensor& down, int64_t activation, bool keep) {
  if (!wants_grad({x, gate_up, down})) return std::get<0>(feed_forward_forward(x, gate_up, down, activation, false));
  return GatedFeedForward::apply(x, gate_up, down, activation, keep);
}

}  // namespace

void bind_layers(pybind11::module_& m) {
  m.def("layer_norm", &layer_norm, "layer norm (eager autograd node)");
  m.def("layer_norm_forward", &layer_norm_forward, "(out, stats [2, rows])");
  m.def("layer_norm_backward", &layer_norm_backward, "(grad_x, grad_weight, grad_bias)");
  m.def("embedding", &embedding, "embedding (eager autograd node)");
  m.def("embedding_forward", &embedding_forward, "rows by token");
  m.def("embedding_backward", &embedding_backward, "(grad_weight, grad_positions)");
  m.def("linear_cross_entropy", &linear_cross_entropy, "loss over a vocabulary (eager autograd node)");
  m.def("loss_forward", &loss_forward, "(loss, saved)");
  m.def("loss_backward", &loss_backward, "(grad_hidden, grad_weight)");
  m.def("gated_feed_forward", &gated_feed_forward, "gated feed-forward block (eager autograd node)");
  m.def("feed_forward_forward", &feed_forward_forward, "(out, saved)");
  m.def("feed_forward_backward", &feed_forward_backward, "(grad_x, grad_gate_up, grad_down)");
}

}  // namespace attnres_nodes
