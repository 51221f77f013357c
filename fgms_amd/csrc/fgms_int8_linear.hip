// out[i][o] = x_scales[i] weight_scales[o] sum_k x[i][k] weight[o][k] + bias[o], x and weight in eight bits.
//
// The sums are whole numbers in 32 bits and exact, whatever their order; what is rounded is their conversion to float, the two scales, the bias
// (fp32) and the result.  The weights are the matrix unit's left operand, so that a lane has neighbouring outputs of one row of x.
#include "fgms_int8_linear.h"

#include "fgms_device.h"
#include "fgms_internal.h"
#include "fgms_mma.h"

namespace fgms {
namespace {

typedef int int16v __attribute__((ext_vector_type(16)));

constexpr int kDepth = 128, kChunks = kDepth / 16;      // bytes of a row, and 16-byte chunks, to a tile in LDS

// Where chunk c of a tile's row lies.  A fragment is read by 32 lanes that ask 32 rows for the same chunk: this way they cover all banks.  (The
// same for rows 32 apart.)
__device__ __forceinline__ int swizzle(int row) { return ((row & 2) << 1) | ((row >> 2) & 3); }
__device__ __forceinline__ int chunk_at(int row, int c) { return row * kChunks + (c ^ swizzle(row)); }

// 16 bytes a lane from a buffer to LDS, one lane's behind the other's from `to` on (the same for all lanes).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, int4v *to, unsigned offset) {
  typedef __attribute__((address_space(3))) void lds_any;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_any *)to, 16, offset, 0, 0, 0);
}

// Rows of a tensor on their way to a tile in LDS, past the registers: every lane asks for the chunk that belongs where its 16 bytes land; rows
// behind the last are out of the buffer's range and arrive as zeros, and so do chunks behind the channels, which are asked for out of range.
template <int ROWS, int THREADS>
struct Stager {
  static constexpr int PER = ROWS * kChunks / THREADS;
  const int8_t *base;
  unsigned range, offset[PER];
  int wave, chunk;      // (rows of a lane lie THREADS / kChunks apart, a multiple of 16: their chunks are the same)
  __device__ __forceinline__ void open(const int8_t *from, int64_t first, int64_t count, int64_t stride, int depth) {
    static_assert(THREADS / kChunks % 16 == 0, "");
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
    base = from + first * stride;
    const int there = (int)min((int64_t)ROWS, count - first);
    range = (unsigned)(there - 1) * (unsigned)stride + (unsigned)((depth + 15) & ~15);
    const int row = threadIdx.x / kChunks;
    chunk = (threadIdx.x % kChunks) ^ swizzle(row);
#pragma unroll
    for (int i = 0; i < PER; ++i) offset[i] = (unsigned)(row + i * (THREADS / kChunks)) * (unsigned)stride + chunk * 16;
  }
  // shares [from, to) of PER
  __device__ __forceinline__ void load(int4v *tile, int k, int depth, int from = 0, int to = PER) const {
    // (a range that the compiler does not know to be the wave's would have every load looped over lane by lane)
    const __amdgpu_buffer_rsrc_t rows = rows_resource(base + k, (unsigned)__builtin_amdgcn_readfirstlane(max((int)range - k, 0)));
    const bool there = k + chunk * 16 < depth;
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (i >= from && i < to) load_to_lds(rows, tile + wave * 64 + i * THREADS, there ? offset[i] : kAbsentRow);
  }
};

// Everything asked for has landed, for all waves.
__device__ __forceinline__ void tiles_ready() {
  __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0)
  __syncthreads();
}

// The tile of a workgroup: workgroups b mod 8 run on the same XCD, which takes a run of tiles that share rows in its L2: eight tiles of
// rows by all tiles of outputs after another.
__device__ __forceinline__ void place_of(unsigned block, unsigned x_tiles, unsigned w_tiles, unsigned &x_tile, unsigned &w_tile) {
  constexpr unsigned kPanel = 8;
  const unsigned tiles = x_tiles * w_tiles, each = tiles / 8, more = tiles % 8, xcd = block % 8;
  const unsigned at = xcd * each + min(xcd, more) + block / 8;
  const unsigned panel = at / (kPanel * w_tiles), in = at % (kPanel * w_tiles), height = min(kPanel, x_tiles - panel * kPanel);
  x_tile = panel * kPanel + in % height;
  w_tile = in / height;
}

// The upper lanes' a for the lower lanes' b, lane by lane.
__device__ __forceinline__ void swap_halves(int &a, int &b) {
  const auto r = __builtin_amdgcn_permlane32_swap((unsigned)a, (unsigned)b, false, false);
  a = (int)r[0], b = (int)r[1];
}

// Results of a block of 32 outputs by 32 rows of x (register 4 p + e of lane l: output 8 p + 4 (l / 32) + e, row l % 32).
template <typename T>
__device__ __forceinline__ void store_block(T *to, const int16v &acc, float by, const float4v (&w)[4], const float4v (&b)[4], int there, bool whole, int lane) {
  float4v v[4];
#pragma unroll
  for (int p = 0; p < 4; ++p)
#pragma unroll
    for (int e = 0; e < 4; ++e) v[p][e] = (float)acc[4 * p + e] * by * w[p][e] + b[p][e];
  if (!whole) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (8 * p + 4 * (lane / 32) + e < there) to[8 * p + 4 * (lane / 32) + e] = (T)v[p][e];
  } else if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int p = 0; p < 4; ++p)
      if (8 * p + 4 * (lane / 32) < there) *reinterpret_cast<float4v *>(to + 8 * p + 4 * (lane / 32)) = v[p];
  } else {
    // eight outputs side by side: a lane takes its partner's four for one pair of p, and gives it four of the other
    typedef T T4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int p = 0; p < 4; p += 2) {
      const int2v lo = __builtin_bit_cast(int2v, __builtin_convertvector(v[p], T4)), hi = __builtin_bit_cast(int2v, __builtin_convertvector(v[p + 1], T4));
      int a = lo[0], b = lo[1], c = hi[0], d = hi[1];
      swap_halves(a, c);
      swap_halves(b, d);
      const int at = 8 * p + 8 * (lane / 32);
      if (at < there) *reinterpret_cast<int4v *>(to + at) = int4v{a, b, c, d};
    }
  }
}

// A lane's chunks of 32 of a tile's 128 bytes, for 32 MB rows of x and 32 NB outputs.
template <int MB, int NB>
struct Fragments {
  int4v x[MB], w[NB];
  __device__ __forceinline__ void read(const int4v *x_tile, const int4v *w_tile, int at) {
#pragma unroll
    for (int i = 0; i < MB; ++i) x[i] = x_tile[32 * i * kChunks + at];
#pragma unroll
    for (int j = 0; j < NB; ++j) w[j] = w_tile[32 * j * kChunks + at];
  }
  __device__ __forceinline__ void multiply(int16v (&acc)[NB][MB]) const {
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[j], x[i], acc[j][i], 0, 0, 0);
  }
};

// The next chunks are read while these are multiplied, and LOADS loads asked for: one of each between every few products.
template <int LOADS, int MB, int NB, typename L>
__device__ __forceinline__ void step(int16v (&acc)[NB][MB], const Fragments<MB, NB> &now, Fragments<MB, NB> &next, const int4v *x_tile, const int4v *w_tile,
                                     int at, const L &load) {
  next.read(x_tile, w_tile, at);
  load();
  now.multiply(acc);
#pragma unroll
  for (int i = 0; i < MB + NB; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                              // a read of LDS
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                              // a product
    if (i < LOADS) __builtin_amdgcn_sched_group_barrier(0x020, 1, 0);               // a load
    if (MB * NB > 8) __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
  }
  __builtin_amdgcn_sched_barrier(0);
}

// A tile of 128 bytes of depth, whose first chunks are in `first` already, and the next one's first chunks.  load(0) and load(1) ask for the
// halves of the one after the next: x's rows into this one's place as soon as all waves have read theirs, the weights' during the next one's first step.
template <int MB, int NB, typename L0, typename L1>
__device__ __forceinline__ void turn(int16v (&acc)[NB][MB], Fragments<MB, NB> &first, const int4v *x_now, const int4v *w_now, const int4v *x_next,
                                     const int4v *w_next, const int (&at)[kDepth / 32], const L0 &load_rest, const L1 &load) {
  const auto none = [] {};
  Fragments<MB, NB> other;
  step<2 * NB>(acc, first, other, x_now, w_now, at[1], load_rest);
  step<0>(acc, other, first, x_now, w_now, at[2], none);
  step<0>(acc, first, other, x_now, w_now, at[3], none);
  tiles_ready();
  __builtin_amdgcn_sched_barrier(0);
  step<2 * MB>(acc, other, first, x_next, w_next, at[0], load);
}

// 64 MB rows of x by 64 NB outputs to a workgroup of four waves, 32 MB by 32 NB to a wave.
template <typename T, int MB, int NB>
__global__ __launch_bounds__(256, (MB * NB >= 16 ? 1 : 2)) void int8_linear_kernel(const Int8LinearArgs a, unsigned x_tiles, unsigned w_tiles) {
  constexpr int XR = 64 * MB, WR = 64 * NB;
  __shared__ int4v x_tile0[XR * kChunks], w_tile0[WR * kChunks], x_tile1[XR * kChunks], w_tile1[WR * kChunks];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  unsigned xt, wt;
  place_of(blockIdx.x, x_tiles, w_tiles, xt, wt);
  const int64_t row0 = (int64_t)xt * XR;
  const int out0 = (int)wt * WR;
  Stager<XR, 256> x;
  Stager<WR, 256> w;
  x.open(a.x, row0, a.n, a.x_row, a.depth);
  w.open(a.weight, out0, a.outputs, a.weight_row, a.depth);
  // The last tile goes first: what lies behind a row in its last 16 bytes is not known (zeros on one side are enough), and is out of the way
  // then.  Tiles behind the last are zeros.
  const int tiles = (a.depth + kDepth - 1) / kDepth, last = (tiles - 1) * kDepth;
  x.load(x_tile0, last, a.depth);
  w.load(w_tile0, last, a.depth);
  const int x0 = wave % 2 * 32 * MB, w0 = wave / 2 * 32 * NB;
  int at[kDepth / 32];
#pragma unroll
  for (int s = 0; s < kDepth / 32; ++s) at[s] = chunk_at(lane % 32, 2 * s + lane / 32);
  int16v acc[NB][MB] = {};
  tiles_ready();
  if (a.depth % 16) {
    for (int row = threadIdx.x; row < XR; row += 256) {
      int8_t *const end = (int8_t *)&x_tile0[chunk_at(row, (a.depth - last) / 16)];
      for (int b = a.depth % 16; b < 16; ++b) end[b] = 0;
    }
    __syncthreads();
  }
  // (no choice in the loop: the accumulators would be moved from registers to registers)
  const int4v *const x0_now = x_tile0 + x0 * kChunks, *const w0_now = w_tile0 + w0 * kChunks;
  const int4v *const x1_now = x_tile1 + x0 * kChunks, *const w1_now = w_tile1 + w0 * kChunks;
  const auto k_of = [&](int tile) { return tile < tiles ? (tile - 1) * kDepth : a.depth; };
  x.load(x_tile1, k_of(1), a.depth);
  Fragments<MB, NB> first;
  first.read(x0_now, w0_now, at[0]);
  int i = 0;
  for (; i + 1 < tiles; i += 2) {
    turn(acc, first, x0_now, w0_now, x1_now, w1_now, at, [&] { w.load(w_tile1, k_of(i + 1), a.depth); }, [&] { x.load(x_tile0, k_of(i + 2), a.depth); });
    turn(acc, first, x1_now, w1_now, x0_now, w0_now, at, [&] { w.load(w_tile0, k_of(i + 2), a.depth); }, [&] { x.load(x_tile1, k_of(i + 3), a.depth); });
  }
  if (i < tiles) {
    const auto none = [] {};
    Fragments<MB, NB> other;
    step<0>(acc, first, other, x0_now, w0_now, at[1], none);
    step<0>(acc, other, first, x0_now, w0_now, at[2], none);
    step<0>(acc, first, other, x0_now, w0_now, at[3], none);
    other.multiply(acc);
  }
  __builtin_amdgcn_s_waitcnt(0x0f70);      // (the zeros asked for behind the last tile: their place is used again)
  // scales and bias of the workgroup's outputs by way of LDS
  __syncthreads();
  float *const scales = (float *)w_tile0, *const biases = scales + WR;
  for (int o = threadIdx.x; o < WR; o += 256) {
    const bool there = out0 + o < a.outputs;
    scales[o] = there ? a.weight_scales[out0 + o] : 0.f;
    biases[o] = there && a.bias ? (float)((const T *)a.bias)[out0 + o] : 0.f;
  }
  float by[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t row = row0 + x0 + 32 * i + lane % 32;
    by[i] = row < a.n ? a.x_scales[row] : 0.f;
  }
  __syncthreads();
  const bool whole = a.outputs % (16 / (int)sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(a.out) % 16 == 0;
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    const int o = w0 + 32 * j;
    float4v wb[4], bb[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      wb[p] = *reinterpret_cast<const float4v *>(scales + o + 8 * p + 4 * (lane / 32));
      bb[p] = *reinterpret_cast<const float4v *>(biases + o + 8 * p + 4 * (lane / 32));
    }
    const int there = a.outputs - out0 - o;
#pragma unroll
    for (int i = 0; i < MB; ++i) {
      const int64_t row = row0 + x0 + 32 * i + lane % 32;
      __builtin_amdgcn_sched_barrier(0);      // (block by block: there are no registers for two)
      // (a lane whose row is not there keeps its partner company in the exchange)
      store_block<T>((T *)a.out + row * a.outputs + out0 + o, acc[j][i], by[i], wb, bb, row < a.n ? there : 0, whole, lane);
    }
  }
}

// Few rows of x: the weights' way from memory counts.  A workgroup has 16 outputs, its waves take turns along the depth, 256 bytes of each row at
// a time, straight into registers, and add their sums up in LDS.
template <typename T, int MB>
__global__ __launch_bounds__(512) void int8_linear_few_kernel(const Int8LinearArgs a) {
  constexpr int kWaves = 8, kSteps = 4;
  __shared__ int4v sums[kWaves][MB][64];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int out0 = blockIdx.x * 16;
  // (rows behind the last are read as the last one, and left)
  const int8_t *const w = a.weight + min(out0 + lane % 16, a.outputs - 1) * a.weight_row + lane / 16 * 16;
  const int8_t *x[MB];
#pragma unroll
  for (int i = 0; i < MB; ++i) x[i] = a.x + min((int64_t)(16 * i + lane % 16), a.n - 1) * a.x_row + lane / 16 * 16;
  int4v acc[MB] = {};
  for (int k = wave * 64 * kSteps; k < a.depth; k += kWaves * 64 * kSteps) {
    int4v wf[kSteps], xf[kSteps][MB];
    if (k + 64 * kSteps <= a.depth) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        wf[s] = *reinterpret_cast<const int4v *>(w + k + 64 * s);
#pragma unroll
        for (int i = 0; i < MB; ++i) xf[s][i] = *reinterpret_cast<const int4v *>(x[i] + k + 64 * s);
      }
    } else {
      // (what lies behind a row in its last 16 bytes is not known: zeros on one side are enough)
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
        const int left = a.depth - (k + 64 * s + lane / 16 * 16);      // bytes of the chunk that count
        const int4v none = {0, 0, 0, 0};
        int4v keep;
#pragma unroll
        for (int q = 0; q < 4; ++q) keep[q] = left >= 4 * q + 4 ? -1 : left <= 4 * q ? 0 : (int)((1u << (8 * (left - 4 * q))) - 1);
        wf[s] = left > 0 ? *reinterpret_cast<const int4v *>(w + k + 64 * s) : none;
#pragma unroll
        for (int i = 0; i < MB; ++i) xf[s][i] = left > 0 ? *reinterpret_cast<const int4v *>(x[i] + k + 64 * s) & keep : none;
      }
    }
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[i] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[s], xf[s][i], acc[i], 0, 0, 0);
  }
#pragma unroll
  for (int i = 0; i < MB; ++i) sums[wave][i][lane] = acc[i];
  __syncthreads();
  // value e of lane l: output 4 (l / 16) + e, row l % 16
  for (int v = threadIdx.x; v < MB * 256; v += 64 * kWaves) {
    const int i = v / 256, l = v % 64, e = v / 64 % 4;
    int sum = 0;
#pragma unroll
    for (int u = 0; u < kWaves; ++u) sum += ((const int *)&sums[u][i][l])[e];
    const int row = 16 * i + l % 16, o = out0 + 4 * (l / 16) + e;
    if (row < a.n && o < a.outputs)
      ((T *)a.out)[(int64_t)row * a.outputs + o] = (T)((float)sum * a.x_scales[row] * a.weight_scales[o] + (a.bias ? (float)((const T *)a.bias)[o] : 0.f));
  }
}

template <typename T, int MB, int NB>
int launch_tiles(const Int8LinearArgs &a) {
  const int64_t x_tiles = (a.n + 64 * MB - 1) / (64 * MB), w_tiles = (a.outputs + 64 * NB - 1) / (64 * NB);
  if (x_tiles * w_tiles > 0x7fffffff) {
    set_error("products in eight bits: more results than one launch takes");
    return FGMS_E_INVALID;
  }
  int8_linear_kernel<T, MB, NB><<<(unsigned)(x_tiles * w_tiles), 256, 0, a.stream>>>(a, (unsigned)x_tiles, (unsigned)w_tiles);
  return FGMS_OK;
}

template <typename T, int MB>
int launch_few(const Int8LinearArgs &a) {
  int8_linear_few_kernel<T, MB><<<(unsigned)((a.outputs + 15) / 16), 512, 0, a.stream>>>(a);
  return FGMS_OK;
}

template <typename T>
int launch(const Int8LinearArgs &a) {
  if (a.n <= 16) return launch_few<T, 1>(a);
  if (a.n <= 32) return launch_few<T, 2>(a);
  if (a.n <= 64) return launch_few<T, 4>(a);
  const auto tiles = [&](int64_t side) { return ((a.n + side - 1) / side) * ((a.outputs + side - 1) / side); };
  if (tiles(256) >= num_cus()) return launch_tiles<T, 4, 4>(a);
  if (tiles(128) >= num_cus()) return launch_tiles<T, 2, 2>(a);
  return launch_tiles<T, 1, 1>(a);
}

}  // namespace

int launch_int8_linear(const Int8LinearArgs &a) {
  const int rc = a.dtype == FGMS_F32 ? launch<float>(a) : a.dtype == FGMS_F16 ? launch<_Float16>(a) : launch<__bf16>(a);
  if (rc != FGMS_OK) return rc;
  FGMS_HIP_TRY(hipGetLastError());
  return FGMS_OK;
}

}  // namespace fgms
