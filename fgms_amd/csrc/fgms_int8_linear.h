// Products of rows in eight bits with weights in eight bits: arguments.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace fgms {

// (127^2 and 128^2 times so many are whole numbers of 32 bits)
constexpr int kMostDepth = 131071;

struct Int8LinearArgs {
  const int8_t *x, *weight;          // [n, depth], [outputs, depth]; rows begin on 16 bytes and are 16 bytes long or a multiple of it
  const float *x_scales, *weight_scales;
  const void *bias;                  // [outputs] or nullptr
  void *out;                         // [n, outputs]
  int64_t n, x_row, weight_row;      // strides in bytes
  int outputs, depth;
  int dtype;
  hipStream_t stream;
};

int launch_int8_linear(const Int8LinearArgs &a);

}  // namespace fgms
