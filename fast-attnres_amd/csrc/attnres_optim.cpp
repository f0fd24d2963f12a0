// The optimizer step over lists of tensors (attnres.optim), in C++ over the C ABI
// (attnres_optim_hip.h): checks every tensor, lays out gradients that lie in another order, and launches.

#include <torch/extension.h>

#include <algorithm>

#include "attnres_nodes.h"
#include "attnres_optim_hip.h"

namespace attnres_nodes {
namespace {

using Tensors = std::vector<Tensor>;
using OptionalTensors = std::optional<Tensors>;
using OptionalTensor = std::optional<Tensor>;

int dtype_of(at::ScalarType type, const char* what) {
  switch (type) {
    case at::kBFloat16: return ATTNRES_BF16;
    case at::kHalf: return ATTNRES_F16;
    case at::kFloat: return ATTNRES_F32;
    default: TORCH_CHECK_TYPE(false, what, " must be BF16, FP16 or FP32 tensors, not ", type);
  }
}

// Whether the elements of both lie in one order, without gaps.
bool same_order(const Tensor& a, const Tensor& b) {
  return a.strides() == b.strides() || (a.is_contiguous() && b.is_contiguous());
}

struct Range {
  uintptr_t begin, end;
  bool written;
};

// What is written overlaps nothing else.
void check_ranges(std::vector<Range>& ranges) {
  std::sort(ranges.begin(), ranges.end(), [](const Range& a, const Range& b) { return a.begin < b.begin; });
  uintptr_t any = 0, written = 0;
  for (const Range& r : ranges) {
    TORCH_CHECK_VALUE(r.begin >= (r.written ? any : written), "the tensors of a step must not overlap (is one given twice?)");
    any = std::max(any, r.end);
    if (r.written) written = std::max(written, r.end);
  }
}

void check_one(const OptionalTensor& tensor, at::ScalarType type, const Tensor& like, const char* name) {
  if (!tensor) return;
  TORCH_CHECK_TYPE(tensor->scalar_type() == type, name, " must be a tensor of ", type);
  TORCH_CHECK_VALUE(tensor->numel() == 1, name, " must have one element");
  TORCH_CHECK_TYPE(tensor->device() == like.device(), name, " must be on the parameters' device");
}

void adamw_step(const Tensors& params, const Tensors& grads, const Tensors& exp_avgs, const Tensors& exp_avg_sqs,
                const OptionalTensors& exp_avg_scales, const OptionalTensors& exp_avg_sq_scales, const OptionalTensors& masters,
                double lr, const OptionalTensor& lr_device, double beta1, double beta2, double eps, double weight_decay, int64_t step,
                const OptionalTensor& step_device, const OptionalTensor& grad_scale) {
  const size_t count = params.size();
  const auto check_list = [&](const Tensors& list, const char* name) {
    TORCH_CHECK_VALUE(list.size() == count, "expected as many ", name, " as params");
  };
  check_list(grads, "grads");
  check_list(exp_avgs, "exp_avgs");
  check_list(exp_avg_sqs, "exp_avg_sqs");
  TORCH_CHECK_VALUE(exp_avg_scales.has_value() == exp_avg_sq_scales.has_value(),
                    "exp_avg_scales and exp_avg_sq_scales go together");
  const bool eighth = exp_avg_scales.has_value();
  if (eighth) {
    check_list(*exp_avg_scales, "exp_avg_scales");
    check_list(*exp_avg_sq_scales, "exp_avg_sq_scales");
  }
  if (masters) check_list(*masters, "masters");
  if (count == 0) return;
  const Tensor& first = params[0];
  const int param_dtype = dtype_of(first.scalar_type(), "params"), grad_dtype = dtype_of(grads[0].scalar_type(), "grads");
  TORCH_CHECK_TYPE(grad_dtype == param_dtype || grad_dtype == ATTNRES_F32, "grads must have the dtype of params or FP32");
  TORCH_CHECK_TYPE(!masters || param_dtype != ATTNRES_F32, "FP32 params have no masters");
  const at::ScalarType state = eighth ? at::kFloat8_e4m3fn : at::kFloat;
  const at::NoGradGuard no_grad;
  Tensors copies;  // of gradients in another order, held until the launches are made
  std::vector<attnres_adamw_tensor> table;
  std::vector<Range> ranges;
  table.reserve(count);
  ranges.reserve(7 * count);
  const auto place = [&](const Tensor& tensor, bool written) {
    const uintptr_t begin = reinterpret_cast<uintptr_t>(tensor.data_ptr());
    ranges.push_back({begin, begin + tensor.numel() * tensor.element_size(), written});
    return tensor.data_ptr();
  };
  const auto check_like = [&](const Tensor& tensor, const Tensor& param, at::ScalarType type, const char* name, size_t i) {
    TORCH_CHECK_TYPE(tensor.scalar_type() == type, name, "[", i, "] must be of ", type);
    TORCH_CHECK_VALUE(tensor.sizes() == param.sizes() && same_order(tensor, param), name, "[", i,
                      "] must have the shape and strides of its parameter");
    TORCH_CHECK_TYPE(tensor.device() == first.device(), name, "[", i, "] must be on the parameters' device");
  };
  for (size_t i = 0; i < count; ++i) {
    const Tensor& p = params[i];
    TORCH_CHECK_TYPE(p.scalar_type() == first.scalar_type(), "params must have one dtype");
    TORCH_CHECK_TYPE(p.device() == first.device(), "params must be on one device");
    TORCH_CHECK_VALUE(p.is_non_overlapping_and_dense(), "params[", i, "] must be dense: no gaps and no element twice");
    const Tensor& grad = grads[i];
    TORCH_CHECK_TYPE(grad.layout() == at::kStrided && grad.scalar_type() == grads[0].scalar_type(),
                     "grads must be dense tensors of one dtype");
    TORCH_CHECK_VALUE(grad.sizes() == p.sizes(), "grads[", i, "] must have the shape of its parameter");
    TORCH_CHECK_TYPE(grad.device() == first.device(), "grads[", i, "] must be on the parameters' device");
    check_like(exp_avgs[i], p, state, "exp_avgs", i);
    check_like(exp_avg_sqs[i], p, state, "exp_avg_sqs", i);
    if (masters) check_like((*masters)[i], p, at::kFloat, "masters", i);
    if (eighth) {
      const int64_t blocks = (p.numel() + ATTNRES_ADAMW_BLOCK - 1) / ATTNRES_ADAMW_BLOCK;
      for (const Tensor* scales : {&(*exp_avg_scales)[i], &(*exp_avg_sq_scales)[i]}) {
        TORCH_CHECK_TYPE(scales->scalar_type() == at::kFloat, "scales must be FP32");
        TORCH_CHECK_VALUE(scales->dim() == 1 && scales->numel() == blocks && scales->is_contiguous(), "scales of params[", i,
                          "] must be contiguous, one per ", ATTNRES_ADAMW_BLOCK, " elements");
        TORCH_CHECK_TYPE(scales->device() == first.device(), "scales must be on the parameters' device");
      }
    }
  }
  check_one(lr_device, at::kFloat, first, "lr");
  check_one(step_device, at::kLong, first, "step");
  check_one(grad_scale, at::kFloat, first, "grad_scale");
  TORCH_CHECK(first.is_cuda(), "adamw_step requires CUDA (ROCm/HIP) device tensors");
  const c10::DeviceGuard guard(first.device());
  for (size_t i = 0; i < count; ++i) {
    const Tensor& p = params[i];
    if (p.numel() == 0) continue;
    Tensor grad = grads[i];
    if (!same_order(grad, p)) {
      grad = torch::empty_like(p, p.options().dtype(grad.scalar_type())).copy_(grad);
      copies.push_back(grad);
    }
    table.push_back({place(p, true), place(grad, false), place(exp_avgs[i], true), place(exp_avg_sqs[i], true),
                     eighth ? static_cast<float*>(place((*exp_avg_scales)[i], true)) : nullptr,
                     eighth ? static_cast<float*>(place((*exp_avg_sq_scales)[i], true)) : nullptr,
                     masters ? static_cast<float*>(place((*masters)[i], true)) : nullptr, p.numel()});
  }
  check_ranges(ranges);
  check(attnres_hip_adamw(table.data(), static_cast<int64_t>(table.size()), param_dtype, grad_dtype, eighth ? 8 : 32, lr,
                          lr_device ? lr_device->data_ptr<float>() : nullptr, beta1, beta2, eps, weight_decay, step,
                          step_device ? step_device->data_ptr<int64_t>() : nullptr,
                          grad_scale ? grad_scale->data_ptr<float>() : nullptr, current_stream(first)),
        "AdamW step");
  // autograd's check of values that a backward still needs
  const auto changed = [](const Tensors& list) {
    for (const Tensor& tensor : list) {
      if (!tensor.is_inference()) tensor.unsafeGetTensorImpl()->bump_version();
    }
  };
  changed(params);
  changed(exp_avgs);
  changed(exp_avg_sqs);
  if (eighth) {
    changed(*exp_avg_scales);
    changed(*exp_avg_sq_scales);
  }
  if (masters) changed(*masters);
}

}  // namespace

void bind_optim(pybind11::module_& m) { m.def("adamw_step", &adamw_step, "an AdamW step over lists of tensors, in place"); }

}  // namespace attnres_nodes
