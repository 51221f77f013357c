// FGMS.backend's functions for what goes around attention in a block (fgms_torch_block.cpp), for the module's definition.
#pragma once

#include <torch/extension.h>

#include <tuple>

std::tuple<at::Tensor, at::Tensor> add_norm(const at::Tensor &x, const c10::optional<at::Tensor> &residual, const c10::optional<at::Tensor> &scale,
                                            double eps, double p, const c10::optional<at::Tensor> &seed);
at::Tensor dropout_add(const at::Tensor &x, const c10::optional<at::Tensor> &residual, double p, const c10::optional<at::Tensor> &seed);
std::tuple<at::Tensor, at::Tensor> quantize_rows(const at::Tensor &x, bool gated);
std::tuple<at::Tensor, at::Tensor, at::Tensor> add_norm_int8(const at::Tensor &x, const c10::optional<at::Tensor> &residual,
                                                             const c10::optional<at::Tensor> &scale, double eps);
at::Tensor int8_linear(const at::Tensor &x, const at::Tensor &x_scales, const at::Tensor &weight, const at::Tensor &weight_scales,
                       const c10::optional<at::Tensor> &bias, at::ScalarType dtype);
