// Norms of queries and keys for each head and their rotation by coordinates: arguments.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fgms {

constexpr int kMaxAxes = 4;

struct NormRotaryArgs {
  // index 0: queries, 1: keys (heads 0: none)
  const void *x[2], *scale[2];      // scale [dim] or nullptr (ones)
  int heads[2];
  int64_t row[2], head[2];          // x's strides in elements
  void *y[2];                       // forward: written, [n, heads, dim]
  const void *gy[2];                // backward: read, [n, heads, dim]
  void *gx[2], *gscale[2];          // backward: written, [n, heads, dim] and [dim], any of them may be nullptr
  const int32_t *coords;            // [n, axes]
  const float *freqs;               // [sum of sections], radians a step
  int axes, sections[kMaxAxes];
  int64_t n;
  int dim;
  int interleaved;
  float eps;
  int dtype;
  hipStream_t stream;
};

int launch_norm_rotary(const NormRotaryArgs &a, bool backward);

}  // namespace fgms
