// FGMS.backend's attention over voxel clouds: norm_rotary and segment_attention as native autograd nodes over the C ABI.
// As sparse_conv: work goes to torch's current stream, outputs are allocated here, a gradient that nobody needs is not
// computed, tangents are refused, and tensors that saved-tensor hooks hand back are checked before a kernel sees them.
#include "fgms_torch_attention.h"

#include <torch/csrc/autograd/function.h>
#include <torch/csrc/autograd/functions/utils.h>
#include <torch/csrc/autograd/saved_variable.h>
#include <torch/csrc/jit/frontend/tracer.h>
#include <torch/library.h>

#include <ATen/hip/impl/HIPGuardImplMasqueradingAsCUDA.h>
#include <ATen/hip/impl/HIPStreamMasqueradingAsCUDA.h>

#include <algorithm>
#include <memory>
#include <stdexcept>
#include <string>

#include "fgms.h"

namespace {

using torch::autograd::SavedVariable;
using torch::autograd::variable_list;

void check(int rc) {
  if (rc == FGMS_OK) return;
  if (rc == FGMS_E_INVALID) throw std::invalid_argument(fgms_last_error());
  throw std::runtime_error(fgms_last_error());
}

// (the message is only put together where it is wanted: a small call takes six microseconds)
#define FGMS_NEED(ok, what) \
  do {                      \
    if (!(ok)) throw std::invalid_argument(what); \
  } while (0)

int dtype_of(const at::Tensor &t) {
  switch (t.scalar_type()) {
    case at::ScalarType::Float: return FGMS_F32;
    case at::ScalarType::Half: return FGMS_F16;
    case at::ScalarType::BFloat16: return FGMS_BF16;
    default: throw std::invalid_argument("FGMS attention handles float32, float16 and bfloat16 tensors");
  }
}

void need_features(const at::Tensor &t, const at::Tensor &like, const char *name) {
  FGMS_NEED(t.is_cuda(), std::string(name) + " must be a GPU tensor");
  FGMS_NEED(t.device() == like.device(), std::string(name) + " must be on the device of q");
  FGMS_NEED(t.scalar_type() == like.scalar_type(), std::string(name) + " must have the dtype of q");
}

// (a slice of a wider tensor, such as the coordinates of a batched cloud, is copied)
at::Tensor need_ints(const at::Tensor &t, const at::Tensor &like, int dims, const char *name) {
  FGMS_NEED(t.scalar_type() == at::ScalarType::Int && t.is_cuda() && t.dim() == dims,
       std::string(name) + " must be an int32 tensor of " + std::to_string(dims) + " dimension(s) on the GPU");
  FGMS_NEED(t.device() == like.device(), std::string(name) + " must be on the device of q");
  return t.is_contiguous() ? t : t.clone(at::MemoryFormat::Contiguous);
}

void refuse_tangent(const at::Tensor &t, const char *op, const char *name) {
  TORCH_CHECK_NOT_IMPLEMENTED(!t.defined() || !torch::autograd::isFwGradDefined(t), op, " has no forward-mode derivative, but ", name,
                              " carries a tangent");
}

// [rows, heads, channels] as the kernels read it: the channels of a head side by side, every head of a row on 16 bytes.
// Slices of one projection and heads expanded from one are taken as they lie; anything else is copied.  (A tile's rows are reached
// by 32-bit offsets, rows of keys and values end where the next begins or before: see fgms_segment_attention_fwd's checks.)
at::Tensor by_rows(const at::Tensor &t, int64_t group = 1) {
  const int64_t size = t.element_size(), row = t.size(0) > 1 ? t.stride(0) : t.size(2), head = t.size(1) > 1 ? t.stride(1) : t.size(2);
  const bool fits = t.stride(2) == 1 && row * size % 16 == 0 && head * size % 16 == 0 && t.stride(0) * size % 16 == 0 &&
                    t.stride(1) * size % 16 == 0 && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 && row >= t.size(2) &&
                    row * size <= 16 << 20 && t.stride(0) * size <= 16 << 20 && t.stride(1) * size * group <= 512 << 20;
  return fits ? t : t.clone(at::MemoryFormat::Contiguous);
}
// ... and a tensor that has to be contiguous.
at::Tensor packed(const at::Tensor &t) {
  return t.is_contiguous() && reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0 ? t : t.clone(at::MemoryFormat::Contiguous);
}

void *data(const at::Tensor &t) { return t.defined() && t.numel() ? t.data_ptr() : nullptr; }
const int32_t *ints(const at::Tensor &t) { return t.defined() && t.numel() ? t.data_ptr<int>() : nullptr; }
hipStream_t current_stream() { return c10::hip::getCurrentHIPStreamMasqueradingAsCUDA().stream(); }
at::Tensor result(at::IntArrayRef shape, const at::Tensor &like) { return at::empty(shape, like.options().requires_grad(false)); }

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

// ------------------------------------------------------------------------------------------------ norms and rotation
struct Turn {
  Index coords, freqs;
  std::vector<int> sections;
  double eps = 0;
  bool interleaved = false;
};

struct NormRotaryBackward final : public torch::autograd::Node {
  Saved q, k, q_scale, k_scale;
  Turn turn;

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    static const char op[] = "norm_rotary";
    if (!grads[0].defined() && !grads[1].defined()) return variable_list(4);
    const auto self = shared_from_this();
    at::Tensor x[2] = {q.unpack(self, op, "q"), k.unpack(self, op, "k")};
    at::Tensor w[2] = {q_scale.unpack(self, op, "q_scale"), k_scale.unpack(self, op, "k_scale")};
    at::NoGradGuard no_grad;
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x[0].device());
    at::Tensor g[2], gx[2], gw[2];
    for (int i = 0; i < 2; ++i) {
      refuse_tangent(grads[i], op, "the output gradient");
      x[i] = by_rows(x[i]);
      if (w[i].defined()) w[i] = packed(w[i]);
      // (no gradient reaches this output: its part of all sums is zero)
      g[i] = grads[i].defined() ? packed(grads[i]) : at::zeros(x[i].sizes(), x[i].options().requires_grad(false));
      FGMS_NEED(g[i].scalar_type() == x[i].scalar_type(), "the output gradient must have the dtype of q");
      if (task_should_compute_output(i)) gx[i] = result(x[i].sizes(), x[i]);
      if (w[i].defined() && task_should_compute_output(2 + i)) gw[i] = result(w[i].sizes(), w[i]);
    }
    check(fgms_norm_rotary_bwd(data(g[0]), data(g[1]), data(x[0]), data(x[1]), data(w[0]), data(w[1]), ints(turn.coords.unchanged(op, "coords")),
                               (const float *)data(turn.freqs.unchanged(op, "freqs")), data(gx[0]), data(gx[1]), data(gw[0]), data(gw[1]), x[0].size(0),
                               (int)x[0].size(1), (int)x[1].size(1), (int)x[0].size(2), x[0].stride(0), x[0].stride(1), x[1].stride(0),
                               x[1].stride(1), (int)turn.sections.size(), turn.sections.data(), turn.interleaved, (float)turn.eps,
                               dtype_of(x[0]), current_stream()));
    return {gx[0], gx[1], gw[0], gw[1]};
  }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (Saved *s : {&q, &k, &q_scale, &k_scale}) s->variable.reset_data();
  }

  std::string name() const override { return "NormRotaryBackward"; }
};

std::tuple<at::Tensor, at::Tensor> norm_rotary_node(const at::Tensor &q, const at::Tensor &k, const c10::optional<at::Tensor> &q_scale_,
                                                    const c10::optional<at::Tensor> &k_scale_, const at::Tensor &coords_,
                                                    const at::Tensor &freqs_, at::IntArrayRef sections, double eps, bool interleaved) {
  static const char op[] = "norm_rotary";
  const at::Tensor scale[2] = {q_scale_.value_or(at::Tensor()), k_scale_.value_or(at::Tensor())};
  FGMS_NEED(q.dim() == 3 && k.dim() == 3 && q.size(0) == k.size(0) && q.size(2) == k.size(2),
       "expected q [N, heads, D] and k [N, key heads, D]");
  need_features(q, q, "q");
  need_features(k, q, "k");
  const int dtype = dtype_of(q);
  for (const at::Tensor &s : scale)
    if (s.defined()) {
      need_features(s, q, "a scale");
      FGMS_NEED(s.dim() == 1 && s.size(0) == q.size(2), "a scale must have one value for each channel of a head");
    }
  const at::Tensor coords = need_ints(coords_, q, 2, "coords");
  FGMS_NEED(coords.size(0) == q.size(0) && coords.size(1) == (int64_t)sections.size(),
       "coords must be [N, axes], with one of the sections for each axis");
  int64_t pairs = 0;
  std::vector<int> each;
  for (int64_t s : sections) {
    FGMS_NEED(s >= 0 && s <= 64, "a section must be between 0 and half the channels of a head");
    each.push_back((int)s);
    pairs += s;
  }
  FGMS_NEED(freqs_.scalar_type() == at::ScalarType::Float && freqs_.is_cuda() && freqs_.device() == q.device() && freqs_.dim() == 1 &&
           freqs_.size(0) == pairs,
       "freqs must be a float32 tensor on the device of q, with a value for each pair of the sections");
  const bool grad_mode = at::GradMode::is_enabled();
  FGMS_NEED(!(grad_mode && freqs_.requires_grad()), "norm_rotary forms no gradient of freqs");
  refuse_tangent(q, op, "q");
  refuse_tangent(k, op, "k");
  refuse_tangent(freqs_, op, "freqs");
  const at::Tensor freqs = freqs_.is_contiguous() ? freqs_ : freqs_.clone(at::MemoryFormat::Contiguous);
  const Turn turn{Index(coords), Index(freqs), each, eps, interleaved};
  at::Tensor x[2], w[2], y[2];
  {
    at::AutoGradMode no_grad(false);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    x[0] = by_rows(q), x[1] = by_rows(k);
    for (int i = 0; i < 2; ++i) {
      refuse_tangent(scale[i], op, "a scale");
      if (scale[i].defined()) w[i] = packed(scale[i]);
      y[i] = result(x[i].sizes(), x[i]);
    }
    check(fgms_norm_rotary_fwd(data(x[0]), data(x[1]), data(w[0]), data(w[1]), ints(coords), (const float *)data(freqs), data(y[0]),
                               data(y[1]), q.size(0), (int)q.size(1), (int)k.size(1), (int)q.size(2), x[0].stride(0), x[0].stride(1),
                               x[1].stride(0), x[1].stride(1), (int)turn.sections.size(), turn.sections.data(), interleaved, (float)eps,
                               dtype, current_stream()));
  }
  const auto wants = [](const at::Tensor &t) { return t.defined() && t.requires_grad(); };
  if (grad_mode && (wants(q) || wants(k) || wants(scale[0]) || wants(scale[1]))) {
    auto node = std::shared_ptr<NormRotaryBackward>(new NormRotaryBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, scale[0], scale[1]));
    node->q.save(x[0]);
    node->k.save(x[1]);
    if (w[0].defined()) node->q_scale.save(w[0]);
    if (w[1].defined()) node->k_scale.save(w[1]);
    node->turn = turn;
    torch::autograd::set_history({y[0], y[1]}, node);
  }
  return {y[0], y[1]};
}

// ------------------------------------------------------------------------------------------------ attention
struct Segments {
  Index q_offsets, k_offsets;
  bool causal = false;
  double scale = 1;
};

struct SegmentAttentionBackward final : public torch::autograd::Node {
  Saved q, k, v, out, lse;
  Segments segments;

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    static const char op[] = "segment_attention";
    if (!grads[0].defined()) return variable_list(3);
    const auto self = shared_from_this();
    at::Tensor x[3] = {q.unpack(self, op, "q"), k.unpack(self, op, "k"), v.unpack(self, op, "v")};
    at::Tensor o = out.unpack(self, op, "result"), l = lse.unpack(self, op, "log-sums");
    refuse_tangent(grads[0], op, "the output gradient");
    at::NoGradGuard no_grad;
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x[0].device());
    at::Tensor gx[3];
    for (int i = 0; i < 3; ++i) {
      x[i] = by_rows(x[i], i ? 1 : x[0].size(1) / std::max<int64_t>(x[1].size(1), 1));
      if (task_should_compute_output(i)) gx[i] = result(x[i].sizes(), x[i]);
    }
    o = packed(o);
    l = packed(l);
    const at::Tensor g = packed(grads[0]), &q_offsets = segments.q_offsets.unchanged(op, "q_offsets"),
                     &k_offsets = segments.k_offsets.unchanged(op, "k_offsets");
    FGMS_NEED(g.scalar_type() == x[0].scalar_type(), "the output gradient must have the dtype of q");
    check(fgms_segment_attention_bwd(data(g), data(x[0]), data(x[1]), data(x[2]), data(o), (const float *)data(l), data(gx[0]), data(gx[1]),
                                     data(gx[2]), ints(q_offsets), ints(k_offsets), x[0].size(0), x[1].size(0),
                                     (int)q_offsets.numel() - 1, (int)x[0].size(1), (int)x[1].size(1), (int)x[0].size(2),
                                     x[0].stride(0), x[0].stride(1), x[1].stride(0), x[1].stride(1), x[2].stride(0), x[2].stride(1),
                                     segments.causal, (float)segments.scale, dtype_of(x[0]), current_stream()));
    return {gx[0], gx[1], gx[2]};
  }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    for (Saved *s : {&q, &k, &v, &out, &lse}) s->variable.reset_data();
  }

  std::string name() const override { return "SegmentAttentionBackward"; }
};

at::Tensor segment_attention_node(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &q_offsets_,
                                  const at::Tensor &k_offsets_, const c10::optional<at::Tensor> &k_lengths_, bool causal, double scale) {
  static const char op[] = "segment_attention";
  at::Tensor k_lengths = k_lengths_.value_or(at::Tensor());
  FGMS_NEED(q.dim() == 3 && k.dim() == 3 && v.dim() == 3 && k.sizes() == v.sizes() && q.size(2) == k.size(2),
       "expected q [Nq, heads, D], k and v [Nk, key heads, D]");
  need_features(q, q, "q");
  need_features(k, q, "k");
  need_features(v, q, "v");
  const int dtype = dtype_of(q);
  const at::Tensor q_offsets = need_ints(q_offsets_, q, 1, "q_offsets"), k_offsets = need_ints(k_offsets_, q, 1, "k_offsets");
  FGMS_NEED(q_offsets.numel() >= 1 && q_offsets.numel() == k_offsets.numel(), "q_offsets and k_offsets must have one more entry than there are segments");
  if (k_lengths.defined()) {
    k_lengths = need_ints(k_lengths, q, 1, "k_lengths");
    FGMS_NEED(k_lengths.numel() == q_offsets.numel() - 1, "k_lengths must have an entry for each segment");
  }
  const bool wants_grad = at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad() || v.requires_grad());
  FGMS_NEED(!(wants_grad && k_lengths.defined()), "segment_attention forms no gradients over caches (k_lengths)");
  refuse_tangent(q, op, "q");
  refuse_tangent(k, op, "k");
  refuse_tangent(v, op, "v");
  at::Tensor x[3], out, lse;
  {
    at::AutoGradMode no_grad(false);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(q.device());
    x[0] = by_rows(q, q.size(1) / std::max<int64_t>(k.size(1), 1)), x[1] = by_rows(k), x[2] = by_rows(v);
    out = result(q.sizes(), q);
    if (wants_grad) lse = at::empty({q.size(0), q.size(1)}, q.options().dtype(at::kFloat).requires_grad(false));
    check(fgms_segment_attention_fwd(data(x[0]), data(x[1]), data(x[2]), data(out), (float *)data(lse), ints(q_offsets), ints(k_offsets),
                                     ints(k_lengths), q.size(0), k.size(0), (int)q_offsets.numel() - 1, (int)q.size(1), (int)k.size(1),
                                     (int)q.size(2), x[0].stride(0), x[0].stride(1), x[1].stride(0), x[1].stride(1), x[2].stride(0),
                                     x[2].stride(1), causal, (float)scale, dtype, current_stream()));
  }
  if (wants_grad) {
    auto node = std::shared_ptr<SegmentAttentionBackward>(new SegmentAttentionBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(q, k, v));
    node->q.save(x[0]);
    node->k.save(x[1]);
    node->v.save(x[2]);
    node->lse.save(lse);
    node->segments = Segments{Index(q_offsets), Index(k_offsets), causal, scale};
    torch::autograd::set_history(out, node);
    node->out.save(out, true);
  }
  return out;
}

}  // namespace

// Under torch.jit.trace both go through torch's dispatcher, as sparse_conv does.
std::tuple<at::Tensor, at::Tensor> norm_rotary(const at::Tensor &q, const at::Tensor &k, const c10::optional<at::Tensor> &q_scale,
                                               const c10::optional<at::Tensor> &k_scale, const at::Tensor &coords, const at::Tensor &freqs,
                                               const std::vector<int64_t> &sections, double eps, bool interleaved) {
  if (!torch::jit::tracer::isTracing()) return norm_rotary_node(q, k, q_scale, k_scale, coords, freqs, sections, eps, interleaved);
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fgms::norm_rotary", "").typed<decltype(norm_rotary_node)>();
  return op.call(q, k, q_scale, k_scale, coords, freqs, sections, eps, interleaved);
}

at::Tensor segment_attention(const at::Tensor &q, const at::Tensor &k, const at::Tensor &v, const at::Tensor &q_offsets,
                             const at::Tensor &k_offsets, const c10::optional<at::Tensor> &k_lengths, bool causal, double scale) {
  if (!torch::jit::tracer::isTracing()) return segment_attention_node(q, k, v, q_offsets, k_offsets, k_lengths, causal, scale);
  static const auto op = c10::Dispatcher::singleton().findSchemaOrThrow("fgms::segment_attention", "").typed<decltype(segment_attention_node)>();
  return op.call(q, k, v, q_offsets, k_offsets, k_lengths, causal, scale);
}

TORCH_LIBRARY_FRAGMENT(fgms, m) {
  m.def("norm_rotary(Tensor q, Tensor k, Tensor? q_scale, Tensor? k_scale, Tensor coords, Tensor freqs, int[] sections, float eps, "
        "bool interleaved) -> (Tensor, Tensor)", &norm_rotary_node);
  m.def("segment_attention(Tensor q, Tensor k, Tensor v, Tensor q_offsets, Tensor k_offsets, Tensor? k_lengths, bool causal, "
        "float scale) -> Tensor", &segment_attention_node);
}
