// FGMS.backend's attention functions (fgms_torch_attention.cpp), for the module's definition.
#pragma once

#include <torch/extension.h>

#include <tuple>
#include <vector>

std::tuple<at::Tensor, at::Tensor> norm_rotary(const at::Tensor &q, const at::Tensor &k, const c10::optional<at::Tensor> &q_scale,
                                               const c10::optional<at::Tensor> &k_scale, const at::Tensor &coords, const at::Tensor &freqs,
                                               const std::vector<int64_t> &sections, double eps, bool interleaved);
at::Tensor segment_attention(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &q_offsets,
                             const at::Tensor &k_offsets, const c10::optional<at::Tensor> &k_lengths, bool causal, double scale);
