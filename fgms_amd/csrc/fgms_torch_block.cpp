// FGMS.backend's functions for what goes around attention in a block, over the C ABI: add_norm and dropout_add as native autograd nodes,
// rows in eight bits and their products, which have no gradients.
#include "fgms_torch_block.h"
#include "fgms_torch_nodes.h"

#include <cmath>

namespace {

using namespace fgms_nodes;
using MaybeTensor = c10::optional<at::Tensor>;

constexpr char kOf[] = "FGMS.nn's rows";

at::Tensor or_none(const MaybeTensor &t) { return t.value_or(at::Tensor()); }

// [rows, channels] with the channels of a row side by side, rows as far apart as they are (a slice of wider rows is read as it lies).
at::Tensor by_row(const at::Tensor &t) { return t.size(1) <= 1 || t.stride(1) == 1 ? t : t.clone(at::MemoryFormat::Contiguous); }
int64_t row_stride(const at::Tensor &t) { return t.defined() && t.size(0) > 1 ? t.stride(0) : 0; }

void need_rows(const at::Tensor &x) {
  FGMS_NEED(x.dim() == 2, "expected x [N, channels]");
  need_features(x, x, "x", "x");
}
void need_residual(const at::Tensor &residual, const at::Tensor &x) {
  if (!residual.defined()) return;
  FGMS_NEED(residual.dim() == 2 && residual.sizes() == x.sizes(), "residual must have the shape of x");
  need_features(residual, x, "residual", "x");
}
void need_scale(const at::Tensor &scale, const at::Tensor &x) {
  if (!scale.defined()) return;
  need_features(scale, x, "scale", "x");
  FGMS_NEED(scale.dim() == 1 && scale.size(0) == x.size(1), "scale must have one value for each channel");
}

struct Dropout {
  Index seed;
  double p = 0;
  bool falls = false;      // whether any element does

  Dropout() = default;
  Dropout(const MaybeTensor &given, double p_, const at::Tensor &x) : p(p_) {
    FGMS_NEED(p >= 0 && p < 1, "p must be at least 0 and less than 1");
    falls = std::rint(p * 65536) > 0;
    if (p <= 0) return;
    FGMS_NEED(given.has_value() && given->defined(), "dropout takes a seed");
    FGMS_NEED(given->scalar_type() == at::ScalarType::Long && given->dim() == 1 && given->size(0) == 2 && given->device() == x.device(),
              "seed must be two int64 numbers on the device of x");
    seed = Index(given->is_contiguous() ? *given : given->clone(at::MemoryFormat::Contiguous));
  }
  const int64_t *data() const { return seed.tensor.defined() ? seed.tensor.data_ptr<int64_t>() : nullptr; }
  const int64_t *unchanged(const char *op) const { return seed.tensor.defined() ? seed.unchanged(op, "seed").data_ptr<int64_t>() : nullptr; }
};

at::Tensor drop(const at::Tensor &x, const at::Tensor &residual, const Dropout &dropout, const int64_t *seed);
at::Tensor dropout_add_node(const at::Tensor &x, const MaybeTensor &residual, double p, const MaybeTensor &seed);

// The gradient of a sum on its way to the branch that was dropped from: the same map again, whose gradient is the same map.
at::Tensor dropped_grad(const at::Tensor &g, const Dropout &dropout, const char *op) {
  if (!dropout.falls) return g;
  const int64_t *const seed = dropout.unchanged(op);
  if (at::GradMode::is_enabled() && g.requires_grad()) return dropout_add_node(g, {}, dropout.p, dropout.seed.tensor);
  at::NoGradGuard no_grad;
  return drop(by_row(g), at::Tensor(), dropout, seed);
}

// ------------------------------------------------------------------------------------------------ sums and norms
struct AddNormBackward final : public torch::autograd::Node {
  Saved sum, scale;
  Dropout dropout;
  double eps = 0;
  bool both = false;      // outputs: the norm and the sum (else the sum is x)

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    static const char op[] = "add_norm";
    const bool given = both && grads[1].defined();
    if (!grads[0].defined() && !given) return variable_list(3);
    refuse_receivers_outside_the_capture(*this, op);
    const bool wants_x = task_should_compute_output(0), wants_residual = task_should_compute_output(1);
    if (!grads[0].defined()) {      // (the norm has no part in it, whatever its rows hold)
      refuse_tangent(grads[1], op, "the output gradient");
      c10::hip::HIPGuardMasqueradingAsCUDA guard(grads[1].device());
      return {wants_x ? dropped_grad(grads[1], dropout, op) : at::Tensor(), wants_residual ? grads[1] : at::Tensor(),
              task_should_compute_output(2) ? at::zeros(scale.shape, scale.options.requires_grad(false)) : at::Tensor()};
    }
    const Once once(*this, op);
    const auto self = shared_from_this();
    const at::Tensor h = by_row(sum.unpack(self, op, "sum"));
    at::Tensor w = scale.unpack(self, op, "scale");
    at::NoGradGuard no_grad;
    c10::hip::HIPGuardMasqueradingAsCUDA guard(h.device());
    if (w.defined()) w = packed(w);
    at::Tensor g[2];
    for (int i = 0; i < (both ? 2 : 1); ++i) {
      refuse_tangent(grads[i], op, "the output gradient");
      if (grads[i].defined()) g[i] = packed(grads[i]);
      FGMS_NEED(!g[i].defined() || g[i].scalar_type() == h.scalar_type(), "the output gradient must have the dtype of x");
    }
    at::Tensor gx, g_residual, gw, sums;
    if (dropout.falls && wants_x) gx = result(h.sizes(), h);
    if (wants_residual || (wants_x && !dropout.falls)) g_residual = result(h.sizes(), h);
    if (w.defined() && task_should_compute_output(2)) {
      gw = result(w.sizes(), w);
      sums = at::empty({fgms_add_norm_bwd_sums(h.size(0), (int)h.size(1))}, h.options().dtype(at::kFloat).requires_grad(false));
    }
    check(fgms_add_norm_bwd(data(g[0]), data(g[1]), data(h), data(w), data(gx), data(g_residual), data(gw), (float *)data(sums), h.size(0),
                            (int)h.size(1), row_stride(h), (float)eps, (float)dropout.p, dropout.unchanged(op),
                            dtype_of(h, kOf), current_stream()));
    const at::Tensor &g_y = grads[0], &g_h = both ? grads[1] : grads[0];
    once(g_residual, {&g_y, &g_h}, {0, 1, 2});
    once(gx, {&g_y, &g_h}, {0, 1, 2});
    once(gw, {&g_y}, {0, 1});
    if (!dropout.falls && wants_x) gx = g_residual;      // (the sum's own)
    return {gx, wants_residual ? g_residual : at::Tensor(), gw};
  }

  void release_variables() override {
    std::lock_guard<std::mutex> lock(mutex_);
    sum.variable.reset_data();
    scale.variable.reset_data();
  }

  std::string name() const override { return "AddNormBackward"; }
};

std::tuple<at::Tensor, at::Tensor> add_norm_node(const at::Tensor &x_, const MaybeTensor &residual_, const MaybeTensor &scale_, double eps, double p,
                                                 const MaybeTensor &seed) {
  static const char op[] = "add_norm";
  const at::Tensor residual = or_none(residual_), scale = or_none(scale_);
  need_rows(x_);
  const int dtype = dtype_of(x_, kOf);
  need_residual(residual, x_);
  need_scale(scale, x_);
  const Dropout dropout(seed, p, x_);
  for (const at::Tensor *t : {&x_, &residual, &scale}) refuse_tangent(*t, op, "an input");
  const bool both = residual.defined() || dropout.falls;
  at::Tensor x, r, w, y, h;
  {
    at::AutoGradMode no_grad(false);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x_.device());
    x = by_row(x_);
    if (residual.defined()) r = by_row(residual);
    if (scale.defined()) w = packed(scale);
    y = result(x.sizes(), x);
    if (both) h = result(x.sizes(), x);
    check(fgms_add_norm_fwd(data(x), data(r), data(w), data(h), data(y), x.size(0), (int)x.size(1), row_stride(x), row_stride(r), (float)eps,
                            (float)p, dropout.data(), dtype, current_stream()));
  }
  const auto wants = [](const at::Tensor &t) { return t.defined() && t.requires_grad(); };
  if (at::GradMode::is_enabled() && (wants(x_) || wants(residual) || wants(scale))) {
    auto node = std::shared_ptr<AddNormBackward>(new AddNormBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x_, residual, scale));
    if (w.defined()) node->scale.save(w);
    node->dropout = dropout;
    node->eps = eps;
    node->both = both;
    if (both) {
      torch::autograd::set_history({y, h}, node);
      node->sum.save(h, true);
    } else {
      torch::autograd::set_history(y, node);
      node->sum.save(x);
    }
  }
  return {y, both ? h : x_};
}

// ------------------------------------------------------------------------------------------------ dropout
at::Tensor drop(const at::Tensor &x, const at::Tensor &residual, const Dropout &dropout, const int64_t *seed) {
  const at::Tensor out = result(x.sizes(), x);
  check(fgms_dropout_add(data(x), data(residual), data(out), x.size(0), (int)x.size(1), row_stride(x), row_stride(residual), (float)dropout.p, seed,
                         dtype_of(x, kOf), current_stream()));
  return out;
}

struct DropoutAddBackward final : public torch::autograd::Node {
  Dropout dropout;

  variable_list apply(variable_list &&grads) override {
    std::lock_guard<std::mutex> lock(mutex_);
    static const char op[] = "dropout_add";
    if (!grads[0].defined()) return variable_list(2);
    refuse_receivers_outside_the_capture(*this, op);
    refuse_tangent(grads[0], op, "the output gradient");
    c10::hip::HIPGuardMasqueradingAsCUDA guard(grads[0].device());
    const at::Tensor gx = task_should_compute_output(0) ? dropped_grad(grads[0], dropout, op) : at::Tensor();
    return {gx, task_should_compute_output(1) ? grads[0] : at::Tensor()};
  }

  std::string name() const override { return "DropoutAddBackward"; }
};

at::Tensor dropout_add_node(const at::Tensor &x, const MaybeTensor &residual_, double p, const MaybeTensor &seed) {
  static const char op[] = "dropout_add";
  const at::Tensor residual = or_none(residual_);
  need_rows(x);
  (void)dtype_of(x, kOf);
  need_residual(residual, x);
  const Dropout dropout(seed, p, x);
  for (const at::Tensor *t : {&x, &residual}) refuse_tangent(*t, op, "an input");
  at::Tensor out;
  {
    at::AutoGradMode no_grad(false);
    c10::hip::HIPGuardMasqueradingAsCUDA guard(x.device());
    out = drop(by_row(x), residual.defined() ? by_row(residual) : residual, dropout, dropout.data());
  }
  if (at::GradMode::is_enabled() && (x.requires_grad() || (residual.defined() && residual.requires_grad()))) {
    auto node = std::shared_ptr<DropoutAddBackward>(new DropoutAddBackward(), torch::autograd::deleteNode);
    node->set_next_edges(torch::autograd::collect_next_edges(x, residual));
    node->dropout = dropout;
    torch::autograd::set_history(out, node);
  }
  return out;
}

// ------------------------------------------------------------------------------------------------ eight bits
// [rows, channels], every row on 16 bytes (what lies behind its channels is not read as anything).
int64_t padded_row(int64_t channels) { return (channels + 15) / 16 * 16; }
at::Tensor eighths(int64_t n, int64_t channels, const at::Tensor &like) {
  const at::Tensor all = at::empty({n, padded_row(channels)}, like.options().dtype(at::kChar).requires_grad(false));
  return padded_row(channels) == channels ? all : all.narrow(1, 0, channels);
}
at::Tensor on_sixteen_bytes(const at::Tensor &t) {
  const int64_t least = padded_row(t.size(1)), row = t.size(0) > 1 ? t.stride(0) : least;
  const int64_t room = (int64_t)t.storage().nbytes() - t.storage_offset() - (t.size(0) - 1) * row;      // (the last row's)
  if (t.numel() == 0 || (t.stride(1) == 1 && row % 16 == 0 && row >= least && row <= 4 << 20 && room >= least &&
                         reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0))
    return t;
  const at::Tensor to = eighths(t.size(0), t.size(1), t);
  to.copy_(t);
  return to;
}
int64_t eighths_stride(const at::Tensor &t) { return t.size(0) > 1 ? t.stride(0) : padded_row(t.size(1)); }

void refuse_gradients(const char *op, std::initializer_list<const at::Tensor *> inputs) {
  for (const at::Tensor *t : inputs) {
    FGMS_NEED(!(at::GradMode::is_enabled() && t->defined() && t->requires_grad()),
              std::string(op) + " forms no gradients: call it under torch.no_grad()");
    refuse_tangent(*t, op, "an input");
  }
}

std::tuple<at::Tensor, at::Tensor> quantize_rows_op(const at::Tensor &x_, bool gated) {
  static const char op[] = "quantize_rows";
  need_rows(x_);
  const int dtype = dtype_of(x_, kOf);
  FGMS_NEED(!gated || x_.size(1) % 2 == 0, "gated rows hold two halves");
  refuse_gradients(op, {&x_});
  at::AutoGradMode no_grad(false);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x_.device());
  const at::Tensor x = by_row(x_);
  const int64_t n = x.size(0), channels = gated ? x.size(1) / 2 : x.size(1);
  const at::Tensor q = eighths(n, channels, x), scales = at::empty({n}, x.options().dtype(at::kFloat).requires_grad(false));
  check(fgms_quantize_rows(data(x), (int8_t *)data(q), (float *)data(scales), n, (int)channels, row_stride(x), padded_row(channels), gated, dtype,
                           current_stream()));
  return {q, scales};
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> add_norm_int8_op(const at::Tensor &x_, const MaybeTensor &residual_, const MaybeTensor &scale_,
                                                                double eps) {
  static const char op[] = "add_norm_int8";
  const at::Tensor residual = or_none(residual_), scale = or_none(scale_);
  need_rows(x_);
  const int dtype = dtype_of(x_, kOf);
  need_residual(residual, x_);
  need_scale(scale, x_);
  refuse_gradients(op, {&x_, &residual, &scale});
  at::AutoGradMode no_grad(false);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x_.device());
  const at::Tensor x = by_row(x_), r = residual.defined() ? by_row(residual) : residual, w = scale.defined() ? packed(scale) : scale;
  const int64_t n = x.size(0), channels = x.size(1);
  const at::Tensor q = eighths(n, channels, x), scales = at::empty({n}, x.options().dtype(at::kFloat).requires_grad(false));
  const at::Tensor h = r.defined() ? result(x.sizes(), x) : at::Tensor();
  check(fgms_add_norm_int8(data(x), data(r), data(w), data(h), (int8_t *)data(q), (float *)data(scales), n, (int)channels, row_stride(x), row_stride(r),
                           padded_row(channels), (float)eps, dtype, current_stream()));
  return {q, scales, h.defined() ? h : x_};
}

at::Tensor int8_linear_op(const at::Tensor &x_, const at::Tensor &x_scales, const at::Tensor &weight_, const at::Tensor &weight_scales,
                          const MaybeTensor &bias_, at::ScalarType dtype) {
  static const char op[] = "int8_linear";
  const at::Tensor bias = or_none(bias_);
  FGMS_NEED(x_.dim() == 2 && weight_.dim() == 2 && x_.size(1) == weight_.size(1), "expected x [N, channels] and weight [outputs, channels]");
  FGMS_NEED(x_.is_cuda(), "x must be a GPU tensor");
  FGMS_NEED(x_.scalar_type() == at::ScalarType::Char && weight_.scalar_type() == at::ScalarType::Char, "x and weight must be int8 tensors");
  FGMS_NEED(weight_.device() == x_.device(), "weight must be on the device of x");
  const at::Tensor *const scales[2] = {&x_scales, &weight_scales};
  const int64_t rows[2] = {x_.size(0), weight_.size(0)};
  for (int i = 0; i < 2; ++i)
    FGMS_NEED(scales[i]->scalar_type() == at::ScalarType::Float && scales[i]->device() == x_.device() && scales[i]->dim() == 1 && scales[i]->size(0) == rows[i],
              "x_scales and weight_scales must be float32 tensors on the device of x, with one value for each row of x and of weight");
  const at::Tensor out = at::empty({x_.size(0), weight_.size(0)}, x_.options().dtype(dtype).requires_grad(false));
  const int type = dtype_of(out, kOf);
  if (bias.defined()) {
    need_features(bias, out, "bias", "the result");
    FGMS_NEED(bias.dim() == 1 && bias.size(0) == weight_.size(0), "bias must have one value for each output");
  }
  refuse_gradients(op, {&x_scales, &weight_scales, &bias});
  at::AutoGradMode no_grad(false);
  c10::hip::HIPGuardMasqueradingAsCUDA guard(x_.device());
  const at::Tensor x = on_sixteen_bytes(x_), weight = on_sixteen_bytes(weight_);
  const at::Tensor sx = x_scales.contiguous(), sw = weight_scales.contiguous(), b = bias.defined() ? bias.contiguous() : bias;
  check(fgms_int8_linear((const int8_t *)data(x), (const float *)data(sx), (const int8_t *)data(weight), (const float *)data(sw), data(b), data(out),
                         x.size(0), (int)weight.size(0), (int)x.size(1), eighths_stride(x), eighths_stride(weight), type, current_stream()));
  return out;
}

}  // namespace

// Under torch.jit.trace all go through torch's dispatcher, as sparse_conv does.  An operator's results there are tensors of its own: where the sum is x itself,
// the norm's own operators are recorded and x is handed on beside them; the others, called by name, leave a copy of it.
namespace {

std::tuple<at::Tensor, at::Tensor> add_norm_op(const at::Tensor &x, const MaybeTensor &residual, const MaybeTensor &scale, double eps, double p,
                                               const MaybeTensor &seed) {
  const auto [y, h] = add_norm_node(x, residual, scale, eps, p, seed);
  return {y, h.is_same(x) ? x.clone() : h};
}
at::Tensor norm_op(const at::Tensor &x, const MaybeTensor &scale, double eps) { return std::get<0>(add_norm_node(x, {}, scale, eps, 0, {})); }

std::tuple<at::Tensor, at::Tensor, at::Tensor> add_norm_int8_own(const at::Tensor &x, const MaybeTensor &residual, const MaybeTensor &scale, double eps) {
  const auto [q, scales, h] = add_norm_int8_op(x, residual, scale, eps);
  return {q, scales, h.is_same(x) ? x.clone() : h};
}
std::tuple<at::Tensor, at::Tensor> norm_int8_op(const at::Tensor &x, const MaybeTensor &scale, double eps) {
  const auto all = add_norm_int8_op(x, {}, scale, eps);
  return {std::get<0>(all), std::get<1>(all)};
}

}  // namespace

#define FGMS_TRACED(name, f) \
  static const auto traced = c10::Dispatcher::singleton().findSchemaOrThrow("fgms::" name, "").typed<decltype(f)>()

std::tuple<at::Tensor, at::Tensor> add_norm(const at::Tensor &x, const MaybeTensor &residual, const MaybeTensor &scale, double eps, double p,
                                            const MaybeTensor &seed) {
  if (!torch::jit::tracer::isTracing()) return add_norm_node(x, residual, scale, eps, p, seed);
  if (!or_none(residual).defined() && !Dropout(seed, p, x).falls) {
    FGMS_TRACED("norm", norm_op);
    return {traced.call(x, scale, eps), x};
  }
  FGMS_TRACED("add_norm", add_norm_op);
  return traced.call(x, residual, scale, eps, p, seed);
}

at::Tensor dropout_add(const at::Tensor &x, const MaybeTensor &residual, double p, const MaybeTensor &seed) {
  if (!torch::jit::tracer::isTracing()) return dropout_add_node(x, residual, p, seed);
  FGMS_TRACED("dropout_add", dropout_add_node);
  return traced.call(x, residual, p, seed);
}

std::tuple<at::Tensor, at::Tensor> quantize_rows(const at::Tensor &x, bool gated) {
  if (!torch::jit::tracer::isTracing()) return quantize_rows_op(x, gated);
  FGMS_TRACED("quantize_rows", quantize_rows_op);
  return traced.call(x, gated);
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> add_norm_int8(const at::Tensor &x, const MaybeTensor &residual, const MaybeTensor &scale, double eps) {
  if (!torch::jit::tracer::isTracing()) return add_norm_int8_op(x, residual, scale, eps);
  if (!or_none(residual).defined()) {
    FGMS_TRACED("norm_int8", norm_int8_op);
    const auto [q, scales] = traced.call(x, scale, eps);
    return {q, scales, x};
  }
  FGMS_TRACED("add_norm_int8", add_norm_int8_own);
  return traced.call(x, residual, scale, eps);
}

at::Tensor int8_linear(const at::Tensor &x, const at::Tensor &x_scales, const at::Tensor &weight, const at::Tensor &weight_scales,
                       const MaybeTensor &bias, at::ScalarType dtype) {
  if (!torch::jit::tracer::isTracing()) return int8_linear_op(x, x_scales, weight, weight_scales, bias, dtype);
  FGMS_TRACED("int8_linear", int8_linear_op);
  return traced.call(x, x_scales, weight, weight_scales, bias, dtype);
}

TORCH_LIBRARY_FRAGMENT(fgms, m) {
  m.def("add_norm(Tensor x, Tensor? residual, Tensor? scale, float eps, float p, Tensor? seed) -> (Tensor, Tensor)", &add_norm_op);
  m.def("norm(Tensor x, Tensor? scale, float eps) -> Tensor", &norm_op);
  m.def("dropout_add(Tensor x, Tensor? residual, float p, Tensor? seed) -> Tensor", &dropout_add_node);
  m.def("quantize_rows(Tensor x, bool gated) -> (Tensor, Tensor)", &quantize_rows_op);
  m.def("add_norm_int8(Tensor x, Tensor? residual, Tensor? scale, float eps) -> (Tensor, Tensor, Tensor)", &add_norm_int8_own);
  m.def("norm_int8(Tensor x, Tensor? scale, float eps) -> (Tensor, Tensor)", &norm_int8_op);
  m.def("int8_linear(Tensor x, Tensor x_scales, Tensor weight, Tensor weight_scales, Tensor? bias, ScalarType dtype) -> Tensor", &int8_linear_op);
}
