// The operators over lists of tensors (grad_norm, adamw_step) as functions of libmxs_nf4_torch.so,
// for py_lists.cpp, which hands them Python lists without the dispatcher.
#pragma once

#include <ATen/ATen.h>

#include <optional>

namespace mxs_lists {

struct StepOptions {
  double lr, beta1, beta2, eps, weight_decay, max_norm;
  std::optional<at::Tensor> lr_dev, norm, grad_scale, found_inf;
};

at::Tensor grad_norm(at::TensorList grads, const std::optional<at::Tensor>& grad_scale);

void adamw_step(at::TensorList params, at::TensorList grads, at::TensorList avgs,
                at::TensorList avg_sqs, at::TensorList avg_scales, at::TensorList avg_sq_scales,
                const at::Tensor& step, const StepOptions& options);

}  // namespace mxs_lists
