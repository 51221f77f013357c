// Rows of features on their way from one branch of a block to the next (sums with dropout, norms, eight bits): arguments.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fgms {

// What a forward launch leaves behind besides the sum.
enum { kRowsNorm = 0, kRowsNormEighths = 1, kRowsEighths = 2, kRowsGatedEighths = 3 };
constexpr int kMostChannels = 16384;

struct RowsArgs {
  int64_t n;
  int channels;
  const void *x, *residual, *scale;      // residual, scale [channels]: or nullptr
  int64_t x_row, residual_row;           // strides in elements (kRowsGatedEighths: rows of x have twice the channels)
  float eps;
  // dropout: words below `dropped` (of 65536; 0: none) fall, the others' elements are multiplied with `back`
  unsigned dropped;
  float back;
  const int64_t *seed;                   // [2]: key, upper half of the counter
  int64_t first;                         // which row of the caller's the first is (a launch may have a part of them)
  void *sum, *out;                       // [n, channels]; sum may be nullptr
  int8_t *eighths;                       // rows of `eighths_row`
  int64_t eighths_row;
  float *scales;                         // [n]
  // backward
  const void *g_out, *g_sum;             // [n, channels]; g_sum may be nullptr
  void *gx, *g_residual, *g_scale;       // written, any of them may be nullptr
  float *scale_sums;                     // [scale_grad_groups()][channels], with g_scale
  int dtype;
  hipStream_t stream;
};

int launch_rows(const RowsArgs &a, int what);
int launch_add_norm_bwd(const RowsArgs &a);
int launch_dropout_add(const RowsArgs &a);
// Workgroups of the backward launch, each of which leaves sums of the scale's gradient behind.
int64_t scale_grad_groups(int64_t n, int channels);

}  // namespace fgms
