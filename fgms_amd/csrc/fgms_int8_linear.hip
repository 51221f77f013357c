// out[i][o] = x_scales[i] weight_scales[o] sum_k x[i][k] weight[o][k] + bias[o], x and weight in eight bits.
//
// The sums are whole numbers in 32 bits and exact, whatever their order; what is rounded is their conversion to float, the two scales, the bias
// (fp32) and the result.
#include "fgms_int8_linear.h"

#include "fgms_device.h"
#include "fgms_internal.h"
#include "fgms_mma.h"

namespace fgms {
namespace {

typedef int int16v __attribute__((ext_vector_type(16)));

constexpr int kDepth = 128, kChunks = kDepth / 16;      // bytes of a row, and 16-byte chunks, to a tile in LDS

// Where chunk c of a tile's row lies (a fragment is read by 32 lanes that ask 32 rows for the same chunk).
__device__ __forceinline__ int chunk_at(int row, int c) { return row * kChunks + (c ^ (((row & 2) << 1) | ((row >> 2) & 3))); }

// Rows of a tensor on their way to a tile in LDS.
template <int ROWS, int THREADS>
struct Tile {
  static constexpr int PER = ROWS * kChunks / THREADS;
  const int8_t *base;
  unsigned range, offset[PER];
  int chunk[PER];
  __device__ __forceinline__ void open(const int8_t *from, int64_t first, int64_t count, int64_t stride, int depth) {
    base = from + first * stride;
    const int there = (int)min((int64_t)ROWS, count - first);
    range = (unsigned)(there - 1) * (unsigned)stride + (unsigned)((depth + 15) & ~15);
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = threadIdx.x + i * THREADS, row = e / kChunks;
      chunk[i] = chunk_at(row, e % kChunks) - row * kChunks;
      offset[i] = (unsigned)row * (unsigned)stride + chunk[i] * 16;
    }
  }
  __device__ __forceinline__ void load(int4v *tile, int k, int depth) const {
    const __amdgpu_buffer_rsrc_t rows = rows_resource(base + k, range - k);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      tile[threadIdx.x + i * THREADS] = __builtin_bit_cast(
          int4v, __builtin_amdgcn_raw_buffer_load_b128(rows, k + chunk[i] * 16 < depth ? offset[i] : kAbsentRow, 0, 0));
  }
};

// 64 rows by 64 outputs to a workgroup, 32 by 32 to a wave.
template <typename T>
__global__ __launch_bounds__(256) void int8_linear_kernel(const Int8LinearArgs a) {
  __shared__ int4v x_tile[64 * kChunks], w_tile[64 * kChunks];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64;
  const int64_t row0 = (int64_t)blockIdx.x * 64;
  const int out0 = blockIdx.y * 64;
  Tile<64, 256> x, w;
  x.open(a.x, row0, a.n, a.x_row, a.depth);
  w.open(a.weight, out0, a.outputs, a.weight_row, a.depth);
  int16v acc = {};
  for (int k = 0; k < a.depth; k += kDepth) {
    __syncthreads();
    x.load(x_tile, k, a.depth);
    w.load(w_tile, k, a.depth);
    __syncthreads();
    if (a.depth - k < kDepth && a.depth % 16) {
      // (what lies behind a row is not known: zeros on one side are enough)
      int8_t *const last = (int8_t *)&x_tile[chunk_at(threadIdx.x % 64, (a.depth - k) / 16)];
      if (threadIdx.x < 64)
        for (int b = a.depth % 16; b < 16; ++b) last[b] = 0;
      __syncthreads();
    }
#pragma unroll
    for (int s = 0; s < kDepth / 32; ++s) {
      const int4v wf = w_tile[chunk_at(wave / 2 * 32 + lane % 32, 2 * s + lane / 32)];
      const int4v xf = x_tile[chunk_at(wave % 2 * 32 + lane % 32, 2 * s + lane / 32)];
      acc = __builtin_amdgcn_mfma_i32_32x32x32_i8(wf, xf, acc, 0, 0, 0);
    }
  }
  const int64_t row = row0 + wave % 2 * 32 + lane % 32;
  if (row >= a.n) return;
  const float by = a.x_scales[row];
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int o = out0 + wave / 2 * 32 + 8 * (r / 4) + 4 * (lane / 32) + r % 4;
    if (o < a.outputs) ((T *)a.out)[row * a.outputs + o] = (T)((float)acc[r] * by * a.weight_scales[o] + (a.bias ? (float)((const T *)a.bias)[o] : 0.f));
  }
}

}  // namespace

int launch_int8_linear(const Int8LinearArgs &a) {
  const dim3 grid((unsigned)((a.n + 63) / 64), (unsigned)((a.outputs + 63) / 64));
  if (a.dtype == FGMS_F32) int8_linear_kernel<float><<<grid, 256, 0, a.stream>>>(a);
  else if (a.dtype == FGMS_F16) int8_linear_kernel<_Float16><<<grid, 256, 0, a.stream>>>(a);
  else int8_linear_kernel<__bf16><<<grid, 256, 0, a.stream>>>(a);
  FGMS_HIP_TRY(hipGetLastError());
  return FGMS_OK;
}

}  // namespace fgms
