// What the native autograd nodes of FGMS.backend share: checks of tensors, streams, and what is kept between the passes.
#pragma once

#include <torch/extension.h>
#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/autograd/variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/library.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <initializer_list>
#include <memory>
#include <stdexcept>
#include <string>

#include "fgms.h"

namespace fgms_nodes {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

inline void check(int rc) {
  if (rc == FGMS_OK) return;
  if (rc == FGMS_E_INVALID) throw std::invalid_argument(fgms_last_error());
  throw std::runtime_error(fgms_last_error());
}

// (the message is only put together where it is wanted: a small call takes six microseconds)
#define FGMS_NEED(ok, what) \
  do {                      \
    if (!(ok)) throw std::invalid_argument(what); \
  } while (0)

inline int dtype_of(const at::Tensor &t, const char *of = "FGMS attention") {
  switch (t.scalar_type()) {
    case at::ScalarType::Float: return FGMS_F32;
    case at::ScalarType::Half: return FGMS_F16;
    case at::ScalarType::BFloat16: return FGMS_BF16;
    default: throw std::invalid_argument(std::string(of) + " handles float32, float16 and bfloat16 tensors");
  }
}

inline void need_features(const at::Tensor &t, const at::Tensor &like, const char *name, const char *of = "q") {
  FGMS_NEED(t.is_cuda(), std::string(name) + " must be a GPU tensor");
  FGMS_NEED(t.device() == like.device(), std::string(name) + " must be on the device of " + of);
  FGMS_NEED(t.scalar_type() == like.scalar_type(), std::string(name) + " must have the dtype of " + of);
}

// (a slice of a wider tensor, such as the coordinates of a batched cloud, is copied)
inline at::Tensor need_ints(const at::Tensor &t, const at::Tensor &like, int dims, const char *name) {
  FGMS_NEED(t.scalar_type() == at::ScalarType::Int && t.is_cuda() && t.dim() == dims,
       std::string(name) + " must be an int32 tensor of " + std::to_string(dims) + " dimension(s) on the GPU");
  FGMS_NEED(t.device() == like.device(), std::string(name) + " must be on the device of q");
  return t.is_contiguous() ? t : t.clone(at::MemoryFormat::Contiguous);
}

inline void refuse_tangent(const at::Tensor &t, const char *op, const char *name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !torch::autograd::isFwGradDefined(t), op, " has no forward-mode derivative, but ", name,
                              " carries a tangent");
}

// [rows, heads, channels] as the kernels read it: the channels of a head side by side, every head of a row on 16 bytes.
// Slices of one projection and heads expanded from one are taken as they lie; anything else is copied.  (A tile's rows are reached
// by 32-bit offsets, rows of keys and values end where the next begins or before: see fgms_segment_attention_fwd's checks.)
inline at::Tensor by_rows(const at::Tensor &t, int64_t group = 1) {
  const int64_t size = t.element_size(), row = t.size(0) > 1 ? t.stride(0) : t.size(2), head = t.size(1) > 1 ? t.stride(1) : t.size(2);
  const bool fits = t.stride(2) == 1 && row * size % 16 == 0 && head * size % 16 == 0 && t.stride(0) * size % 16 == 0 &&
                    t.stride(1) * size % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && row >= t.size(2) &&
                    row * size <= 16 << 20 && t.stride(0) * size <= 16 << 20 && t.stride(1) * size * group <= 512 << 20;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
// ... and a tensor that has to be contiguous.
inline at::Tensor packed(const at::Tensor &t) {
  return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

inline void *data(const at::Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
inline const int32_t *ints(const at::Tensor &t) { return t.defined() && t.numel() ? t.data_ptr<int>() : nullptr; }
inline hipStream_t current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
inline at::Tensor result(at::IntArrayRef shape, const at::Tensor &like) { return at::empty(shape, like.options().requires_grad(false)); }

// A saved tensor's shape, type and place, and the tensor as it came back from whatever hooks it went through.
struct Saved {
  SavedVariable variable;
  std::vector<int64_t> shape;
  at::TensorOptions options;

  void save(const at::Tensor &t, bool is_output = false) {
    variable = SavedVariable(t, is_output);
    shape = t.sizes().vec();
    options = t.options();
  }
  at::Tensor unpack(const std::shared_ptr<torch::autograd::Node> &node, const char *op, const char *name) {
    const at::Tensor t = variable.unpack(node);
    if (shape.empty() && !t.defined()) return t;
    TORCH_CHECK_VALUE(t.defined() && t.sizes() == at::IntArrayRef(shape) && t.dtype() == options.dtype() && t.device() == options.device(), op,
                      ": the saved ", name, " came back with another shape, dtype or device than it was saved with");
    refuse_tangent(t, op, name);
    return t.detach();
  }
};

// A tensor that both passes read and that has no gradient: the backward pass refuses it where it was written to in between.  (Kept as it is, not
// as a saved tensor, which those of inference mode cannot be; they count no changes.)
struct Index {
  at::Tensor tensor;
  int64_t version = 0;

  Index() = default;
  explicit Index(const at::Tensor &t) : tensor(t), version(version_of(t)) {}
  static int64_t version_of(const at::Tensor &t) { return t.is_inference() ? 0 : (int64_t)t._version(); }
  const at::Tensor &unchanged(const char *op, const char *name) const {
    TORCH_CHECK(version_of(tensor) == version, op, ": ", name, " has been modified by an inplace operation between the forward and the backward pass");
    return tensor;
  }
};

// Gradients are formed outside of any graph.  Where a graph of them is asked for (create_graph), one that depends on an input or an output gradient
// that has a graph itself becomes the result of a node that refuses to be passed: without its part a second derivative would look right and not be.
struct NoSecondDerivative final : public torch::autograd::Node {
  const char *op;

  explicit NoSecondDerivative(const char *op_) : op(op_) {}
  variable_list apply(variable_list &&grads) override {
    TORCH_CHECK_NOT_IMPLEMENTED(!grads[0].defined(), op, " has no second derivatives");
    return variable_list(num_outputs());      // (no gradient came)
  }
  std::string name() const override { return "NoSecondDerivative"; }
};

// (made before the gradients are, while the pass's own mode holds)
struct Once {
  const torch::autograd::Node &node;
  const char *op;
  bool graph = at::GradMode::is_enabled();

  Once(const torch::autograd::Node &node_, const char *op_) : node(node_), op(op_) {}
  // `grad`, a tensor of the node's own making, depends on these output gradients and on the node's inputs at these places.
  void operator()(const at::Tensor &grad, std::initializer_list<const at::Tensor *> output_grads, std::initializer_list<size_t> inputs) const {
    if (!graph || !grad.defined()) return;
    torch::autograd::edge_list edges;
    for (const at::Tensor *t : output_grads)
      if (t->defined() && t->requires_grad()) edges.push_back(torch::autograd::impl::gradient_edge(*t));
    for (size_t i : inputs)
      if (node.next_edge(i).is_valid()) edges.push_back(node.next_edge(i));
    if (edges.empty()) return;
    const std::shared_ptr<NoSecondDerivative> refusal(new NoSecondDerivative(op), torch::autograd::deleteNode);
    refusal->set_next_edges(std::move(edges));
    torch::autograd::set_history(grad, refusal);
  }
};

// A gradient that is handed on under stream capture is waited for on the stream that its receiver was made on, which joins the capture and
// never leaves it if it is none of the capture's: the capture's end then takes the process with it.  That is so where an eager graph of the
// same leaves is still alive (its nodes receive their gradients): refused before anything is queued.  (A gradient that the pass does not ask for is handed
// to nobody.)
inline void refuse_receivers_outside_the_capture(const torch::autograd::Node &node, const char *op) {
  const auto capturing = [](hipStream_t stream) {
    hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
    return stream && hipStreamIsCapturing(stream, &status) == hipSuccess && status != hipStreamCaptureStatusNone;
  };
  if (!capturing(current_stream())) return;
  for (size_t i = 0; i < node.num_outputs(); ++i) {
    if (!node.task_should_compute_output(i)) continue;
    const auto &receiver = node.next_edge(i).function;
    const auto stream = receiver ? receiver->stream() : std::nullopt;
    TORCH_CHECK(!stream || capturing(c10::hip::HIPStreamMasqueradingAsCUDA(*stream).stream()), op,
                ": a backward pass is being captured whose leaves belong to a graph of an eager pass too: drop that pass's results first");
  }
}

}  // namespace fgms_nodes
