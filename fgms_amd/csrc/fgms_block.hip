// extern "C" entry points of what goes around attention in a block: argument checks.
#include <math.h>

#include <initializer_list>

#include "fgms_int8_linear.h"
#include "fgms_internal.h"
#include "fgms_rows.h"

namespace fgms {
namespace {

int refuse(const char *what, const char *why) {
  set_error("%s: %s", what, why);
  return FGMS_E_INVALID;
}

constexpr int64_t kMostRowBytes = 4 << 20;      // 256 rows of a tile: below 2^31

int element_bytes(int dtype) { return dtype == FGMS_F32 ? 4 : 2; }
bool on(const void *p, int bytes) { return reinterpret_cast<uintptr_t>(p) % bytes == 0; }

int check_shape(const char *what, int64_t n, int channels, int dtype) {
  if (dtype != FGMS_F32 && dtype != FGMS_F16 && dtype != FGMS_BF16) return refuse(what, "dtype must be FGMS_F32, FGMS_F16 or FGMS_BF16");
  if (n < 0 || n > INT32_MAX) return refuse(what, "between 0 and 2^31 - 1 rows");
  if (channels < 1 || channels > kMostChannels) return refuse(what, "between 1 and 16384 channels");
  return FGMS_OK;
}

// A tensor that has to be there if there are rows, and one that may be.
int check_rows(const char *what, const void *p, bool there, int64_t row, int dtype) {
  if (there && !p) return refuse(what, "null pointer");
  if (!on(p, element_bytes(dtype))) return refuse(what, "tensors have to begin on an element");
  if (row < 0 || row > (int64_t)1 << 40) return refuse(what, "a row stride is out of range");
  return FGMS_OK;
}

int check_eps(const char *what, float eps) {
  return eps >= 0.f && eps < 1e30f ? FGMS_OK : refuse(what, "eps must be finite and not negative");
}

// The share of words that fall, and what makes up for it.  (The factor goes by the share that is met, so that means are kept exactly.)
int take_dropout(const char *what, float p, const int64_t *seed, RowsArgs &a) {
  if (!(p >= 0.f) || !(p < 1.f)) return refuse(what, "p must be at least 0 and less than 1");
  a.dropped = (unsigned)rint((double)p * 65536);
  if (a.dropped > 65535) return refuse(what, "p must not round to 1 in steps of 2^-16");
  if (p > 0.f && (!seed || !on(seed, 8))) return refuse(what, "dropout takes a seed, two 64-bit numbers on the device");
  a.back = (float)(65536.0 / (65536 - a.dropped));
  a.seed = seed;
  return FGMS_OK;
}

int check_eighths(const char *what, const int8_t *out, const float *scales, int64_t row, int channels, bool there) {
  if (there && (!out || !scales)) return refuse(what, "null pointer");
  if (!on(scales, 4)) return refuse(what, "tensors have to begin on an element");
  return row >= channels && row <= (int64_t)1 << 40 ? FGMS_OK : refuse(what, "rows of the result overlap");
}

RowsArgs rows_args(int64_t n, int channels, int dtype, void *stream) {
  RowsArgs a{};
  a.n = n, a.channels = channels, a.dtype = dtype, a.stream = (hipStream_t)stream;
  a.back = 1.f;
  return a;
}

}  // namespace
}  // namespace fgms

using namespace fgms;

extern "C" int fgms_add_norm_fwd(const void *x, const void *residual, const void *scale, void *sum, void *out, int64_t n, int channels,
                                 int64_t x_row, int64_t residual_row, float eps, float p, const int64_t *seed, int dtype, void *stream) {
  static const char what[] = "fgms_add_norm_fwd";
  RowsArgs a = rows_args(n, channels, dtype, stream);
  int rc = check_shape(what, n, channels, dtype);
  if (rc || (rc = check_eps(what, eps)) || (rc = take_dropout(what, p, seed, a)) || (rc = check_rows(what, x, n > 0, x_row, dtype)) ||
      (rc = check_rows(what, residual, false, residual_row, dtype)) || (rc = check_rows(what, out, n > 0, 0, dtype)) ||
      (rc = check_rows(what, sum, false, 0, dtype)) || (rc = check_rows(what, scale, false, 0, dtype)) || n == 0)
    return rc;
  a.x = x, a.x_row = x_row, a.residual = residual, a.residual_row = residual_row, a.scale = scale, a.sum = sum, a.out = out, a.eps = eps;
  return launch_rows(a, kRowsNorm);
}

extern "C" int64_t fgms_add_norm_bwd_sums(int64_t n, int channels) {
  return n < 1 || n > INT32_MAX || channels < 1 || channels > kMostChannels ? 0 : scale_grad_groups(n, channels) * channels;
}

extern "C" int fgms_add_norm_bwd(const void *out_grad, const void *sum_grad, const void *sum, const void *scale, void *x_grad,
                                 void *residual_grad, void *scale_grad, float *scale_sums, int64_t n, int channels, int64_t sum_row, float eps,
                                 float p, const int64_t *seed, int dtype, void *stream) {
  static const char what[] = "fgms_add_norm_bwd";
  RowsArgs a = rows_args(n, channels, dtype, stream);
  int rc = check_shape(what, n, channels, dtype);
  if (rc || (rc = check_eps(what, eps)) || (rc = take_dropout(what, p, seed, a)) || (rc = check_rows(what, sum, n > 0, sum_row, dtype)) ||
      (rc = check_rows(what, out_grad, n > 0, 0, dtype)))
    return rc;
  for (const void *t : {sum_grad, scale, (const void *)x_grad, (const void *)residual_grad, (const void *)scale_grad})
    if ((rc = check_rows(what, t, false, 0, dtype))) return rc;
  if (n == 0) return scale_grad ? launch_fill_zero(scale_grad, (size_t)channels * element_bytes(dtype), a.stream) : FGMS_OK;
  if (scale_grad && (!scale_sums || !on(scale_sums, 4))) return refuse(what, "the scale's gradient takes room for its sums");
  a.sum = const_cast<void *>(sum), a.x_row = sum_row, a.scale = scale, a.eps = eps, a.g_out = out_grad, a.g_sum = sum_grad;
  a.gx = x_grad, a.g_residual = residual_grad, a.g_scale = scale_grad, a.scale_sums = scale_grad ? scale_sums : nullptr;
  return launch_add_norm_bwd(a);
}

extern "C" int fgms_dropout_add(const void *x, const void *residual, void *out, int64_t n, int channels, int64_t x_row, int64_t residual_row,
                                float p, const int64_t *seed, int dtype, void *stream) {
  static const char what[] = "fgms_dropout_add";
  RowsArgs a = rows_args(n, channels, dtype, stream);
  int rc = check_shape(what, n, channels, dtype);
  if (rc || (rc = take_dropout(what, p, seed, a)) || (rc = check_rows(what, x, n > 0, x_row, dtype)) ||
      (rc = check_rows(what, residual, false, residual_row, dtype)) || (rc = check_rows(what, out, n > 0, 0, dtype)) || n == 0)
    return rc;
  a.x = x, a.x_row = x_row, a.residual = residual, a.residual_row = residual_row, a.out = out;
  return launch_dropout_add(a);
}

extern "C" int fgms_quantize_rows(const void *x, int8_t *out, float *scales, int64_t n, int channels, int64_t x_row, int64_t out_row, int gated,
                                  int dtype, void *stream) {
  static const char what[] = "fgms_quantize_rows";
  RowsArgs a = rows_args(n, channels, dtype, stream);
  int rc = check_shape(what, n, channels, dtype);
  if (rc || (rc = check_rows(what, x, n > 0, x_row, dtype)) || (rc = check_eighths(what, out, scales, out_row, channels, n > 0)) || n == 0) return rc;
  a.x = x, a.x_row = x_row, a.eighths = out, a.eighths_row = out_row, a.scales = scales;
  return launch_rows(a, gated ? kRowsGatedEighths : kRowsEighths);
}

extern "C" int fgms_add_norm_int8(const void *x, const void *residual, const void *scale, void *sum, int8_t *out, float *scales, int64_t n,
                                  int channels, int64_t x_row, int64_t residual_row, int64_t out_row, float eps, int dtype, void *stream) {
  static const char what[] = "fgms_add_norm_int8";
  RowsArgs a = rows_args(n, channels, dtype, stream);
  int rc = check_shape(what, n, channels, dtype);
  if (rc || (rc = check_eps(what, eps)) || (rc = check_rows(what, x, n > 0, x_row, dtype)) ||
      (rc = check_rows(what, residual, false, residual_row, dtype)) || (rc = check_rows(what, sum, false, 0, dtype)) ||
      (rc = check_rows(what, scale, false, 0, dtype)) || (rc = check_eighths(what, out, scales, out_row, channels, n > 0)) || n == 0)
    return rc;
  a.x = x, a.x_row = x_row, a.residual = residual, a.residual_row = residual_row, a.scale = scale, a.sum = sum, a.eps = eps;
  a.eighths = out, a.eighths_row = out_row, a.scales = scales;
  return launch_rows(a, kRowsNormEighths);
}

extern "C" int fgms_int8_linear(const int8_t *x, const float *x_scales, const int8_t *weight, const float *weight_scales, const void *bias,
                                void *out, int64_t n, int outputs, int channels, int64_t x_row, int64_t weight_row, int dtype, void *stream) {
  static const char what[] = "fgms_int8_linear";
  if (dtype != FGMS_F32 && dtype != FGMS_F16 && dtype != FGMS_BF16) return refuse(what, "dtype must be FGMS_F32, FGMS_F16 or FGMS_BF16");
  if (n < 0 || n > INT32_MAX) return refuse(what, "between 0 and 2^31 - 1 rows");
  if (channels < 1 || channels > kMostDepth) return refuse(what, "between 1 and 131071 channels");
  if (outputs < 1 || outputs > 1 << 20) return refuse(what, "between 1 and 2^20 outputs");
  const int64_t least = (channels + 15) / 16 * 16;
  for (const int64_t row : {x_row, weight_row})
    if (row < least || row % 16 || row > kMostRowBytes) return refuse(what, "rows of x and weight take a multiple of 16 bytes each, 4 MB at most");
  if (!on(x, 16) || !on(weight, 16)) return refuse(what, "rows of x and weight have to begin on 16 bytes");
  if (!weight || !weight_scales || (n > 0 && (!x || !x_scales || !out))) return refuse(what, "null pointer");
  if (!on(x_scales, 4) || !on(weight_scales, 4) || !on(bias, element_bytes(dtype)) || !on(out, element_bytes(dtype)))
    return refuse(what, "tensors have to begin on an element");
  if (n == 0) return FGMS_OK;
  Int8LinearArgs a{};
  a.x = x, a.weight = weight, a.x_scales = x_scales, a.weight_scales = weight_scales, a.bias = bias, a.out = out, a.n = n, a.x_row = x_row;
  a.weight_row = weight_row, a.outputs = outputs, a.depth = channels, a.dtype = dtype, a.stream = (hipStream_t)stream;
  return launch_int8_linear(a);
}
