// attnres_nodes.h - what the eager autograd nodes share: errors, streams and row
// layouts (attnres_autograd.cpp: the reads and the source bank;
// attnres_layers_autograd.cpp: the layers around them).
#ifndef ATTNRES_NODES_H
#define ATTNRES_NODES_H

#include <torch/extension.h>

#include <c10/core/AutogradState.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPStream.h>

#include <optional>
#include <vector>

#include "attnres_hip.h"

namespace attnres_nodes {

using torch::Tensor;
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// A failing status raises as the Python binding does: ValueError for argument
// errors, RuntimeError otherwise, with the library's own message.
inline void check(int status, const char* what) {
  if (status == ATTNRES_OK) return;
  const char* message = attnres_hip_last_error();
  if (status == ATTNRES_ERR_SHAPE || status == ATTNRES_ERR_STRIDE || status == ATTNRES_ERR_SCALAR ||
      status == ATTNRES_ERR_WORKSPACE) {
    TORCH_CHECK_VALUE(false, what, ": ", message);
  }
  TORCH_CHECK(false, what, ": ", message, " (status ", status, ")");
}

inline hipStream_t current_stream(const Tensor& tensor) {
  return c10::hip::getCurrentHIPStream(tensor.device().index()).stream();
}

// Element stride between consecutive rows of tensor[..., D] flattened to
// [rows, D], or nothing when the rows are not evenly spaced or a row is not
// unit-stride (the Python `row_stride`, after fla_full_sources.py:164-178).
inline std::optional<int64_t> row_stride(const Tensor& tensor) {
  const int64_t last = tensor.dim() - 1;
  if (tensor.size(last) > 1 && tensor.stride(last) != 1) return std::nullopt;
  std::optional<int64_t> stride;
  int64_t rows = 1;
  for (int64_t d = last - 1; d >= 0; --d) {
    if (tensor.size(d) == 1) continue;
    if (!stride) {
      stride = tensor.stride(d);
    } else if (tensor.stride(d) != rows * *stride) {
      return std::nullopt;
    }
    rows *= tensor.size(d);
  }
  return stride.value_or(0);
}

// Nothing here carries a forward-mode derivative: a launch refuses inputs that have a tangent instead of returning outputs
// without one (a node's forward, within which forward mode is off, is refused by the node itself).  Where forward mode
// is off (inference mode) tangents are dropped, as everywhere.
inline bool has_tangent(const Tensor& tensor) { return tensor.defined() && tensor._fw_grad(/*level=*/0).defined(); }
inline bool has_tangent(const std::optional<Tensor>& tensor) { return tensor && has_tangent(*tensor); }
inline bool has_tangent(const std::vector<Tensor>& tensors) {
  for (const Tensor& tensor : tensors) {
    if (has_tangent(tensor)) return true;
  }
  return false;
}
template <class... T>
void refuse_tangents(const char* what, const T&... tensors) {
  if (!c10::AutogradState::get_tls_state().get_fw_grad_mode()) return;
  TORCH_CHECK_NOT_IMPLEMENTED(!(has_tangent(tensors) || ...), what, " has no forward-mode derivative");
}

inline int64_t rows_of(const Tensor& tensor) { return tensor.dim() > 1 ? tensor.numel() / tensor.size(-1) : 1; }

// Registers the layers' functions in the extension module.
void bind_layers(pybind11::module_& m);

}  // namespace attnres_nodes

#endif  // ATTNRES_NODES_H
