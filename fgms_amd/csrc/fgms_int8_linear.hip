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

// Where chunk c of a tile's row of DEPTH bytes lies.  A fragment is read by 32 lanes that ask 32 rows for the same chunk: this way they cover all
// banks.  (The same for rows 32 apart.)
template <int DEPTH>
__device__ __forceinline__ int swizzle(int row) { return DEPTH == 128 ? ((row & 2) << 1) | ((row >> 2) & 3) : (row >> 2) & 3; }
template <int DEPTH>
__device__ __forceinline__ int chunk_at(int row, int c) { return row * (DEPTH / 16) + (c ^ swizzle<DEPTH>(row)); }

// 16 bytes a lane from a buffer to LDS, one lane's behind the other's from `to` on (the same for all lanes).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, int4v *to, unsigned offset) {
  typedef __attribute__((address_space(3))) void lds_any;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_any *)to, 16, offset, 0, 0, 0);
}

// Rows of a tensor on their way to a tile in LDS, past the registers: every lane asks for the chunk that belongs where its 16 bytes land; rows
// behind the last are out of the buffer's range and arrive as zeros, and so do chunks behind the channels, which are asked for out of range.
template <int ROWS, int DEPTH>
struct Stager {
  static constexpr int THREADS = 256, kChunks = DEPTH / 16, PER = ROWS * kChunks / THREADS;
  const int8_t *base;
  unsigned range, offset[PER];
  int wave, chunk;      // (rows of a lane lie THREADS / kChunks apart, a multiple of 16: their chunks are the same)
  __device__ __forceinline__ void open(const int8_t *from, int64_t first, int64_t count, int64_t stride, int depth) {
    static_assert(THREADS / kChunks % 16 == 0, "");
    wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 % (THREADS / 64));
    base = from + first * stride;
    const int there = (int)min((int64_t)ROWS, count - first);
    range = (unsigned)(there - 1) * (unsigned)stride + (unsigned)((depth + 15) & ~15);
    const int row = threadIdx.x % THREADS / kChunks;
    chunk = (threadIdx.x % kChunks) ^ swizzle<DEPTH>(row);
#pragma unroll
    for (int i = 0; i < PER; ++i) offset[i] = (unsigned)(row + i * (THREADS / kChunks)) * (unsigned)stride + chunk * 16;
  }
  __device__ __forceinline__ void load(int4v *tile, int k, int depth) const {
    // (a range that the compiler does not know to be the wave's would have every load looped over lane by lane)
    const __amdgpu_buffer_rsrc_t rows = rows_resource(base + k, (unsigned)__builtin_amdgcn_readfirstlane(max((int)range - k, 0)));
    const bool there = k + chunk * 16 < depth;
#pragma unroll
    for (int i = 0; i < PER; ++i) load_to_lds(rows, tile + wave * 64 + i * THREADS, there ? offset[i] : kAbsentRow);
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

// Results of a block of 32 outputs by 32 rows of x (register 4 p + e of lane l: output 8 p + 4 (l / 32) + e, row l % 32): `scales` and `biases` are the
// block's.  16-bit types: a lane takes its partner's four for one p and gives it four of the other, which makes chunks of eight outputs side by side, the
// first from output 8 (l / 32) on, the second 16 behind it; float: chunks of four, eight apart.
template <typename T>
struct Results {
  static constexpr int N = 16 / (int)sizeof(T), CHUNKS = 32 / (2 * N);
  int4v chunk[CHUNKS];
  __device__ __forceinline__ void form(const int16v &acc, float by, const float *scales, const float *biases, int lane) {
    float4v v[4];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float4v w = *reinterpret_cast<const float4v *>(scales + 8 * p + 4 * (lane / 32)), b = *reinterpret_cast<const float4v *>(biases + 8 * p + 4 * (lane / 32));
#pragma unroll
      for (int e = 0; e < 4; ++e) v[p][e] = (float)acc[4 * p + e] * by * w[e] + b[e];
    }
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      if constexpr (N == 4) {
        chunk[i] = __builtin_bit_cast(int4v, v[i]);
      } else {
        typedef T T4 __attribute__((ext_vector_type(4)));
        const int2v lo = __builtin_bit_cast(int2v, __builtin_convertvector(v[2 * i], T4)), hi = __builtin_bit_cast(int2v, __builtin_convertvector(v[2 * i + 1], T4));
        int a = lo[0], b = lo[1], c = hi[0], d = hi[1];
        swap_halves(a, c);
        swap_halves(b, d);
        chunk[i] = int4v{a, b, c, d};
      }
    }
  }
  static __device__ __forceinline__ int place(int i, int lane) { return 2 * N * i + N * (lane / 32); }
};

// `left` outputs from `to` on are there; those of a chunk from its element `from` on.  (Places are compared as what is left of a row against numbers that
// the instruction holds: sums of a place and a number would each take a register.)
template <typename T>
__device__ __forceinline__ void store_elements(T *to, int left, const int4v &chunk, int from) {
  typedef T Tn __attribute__((ext_vector_type(16 / sizeof(T))));
  const Tn all = __builtin_bit_cast(Tn, chunk);
#pragma unroll
  for (int e = 0; e < 16 / (int)sizeof(T); ++e)
    if (e >= from && e < left) to[e] = all[e];
}

// 16 bytes at a time, wherever an element or two begin.
template <typename T, int MB, int NB, int CHUNKS = Results<T>::CHUNKS>
__device__ __forceinline__ void store_row(T *to, const int16v (&acc)[NB][MB], int i, float by, const float *scales, const float *biases, int there, int lane) {
  typedef int4v Anywhere __attribute__((aligned(4)));
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    __builtin_amdgcn_sched_barrier(0);      // (block by block: there are no registers for two)
    Results<T> r;
    r.form(acc[j][i], by, scales + 32 * j, biases + 32 * j, lane);
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c) {
      const int at = 32 * j + r.place(c, lane);
      if (r.N <= there - at) *reinterpret_cast<Anywhere *>(to + at) = r.chunk[c];
      else store_elements<T>(to + at, there - at, r.chunk[c], 0);
    }
  }
}

// ... where rows may begin half-way through four bytes (an odd number of outputs): such a row's chunks are shifted by an element, whose place the next
// chunk's first fills.  (50000 rows of 256 to 767, bf16, from memory: 37.2 us over three sets of tensors, with stores of 16 bytes beside four-byte boundaries
// 47.6; to 768 31.0.)
template <typename T, int MB, int NB>
__device__ __forceinline__ void store_odd_row(T *to, const int16v (&acc)[NB][MB], int i, float by, const float *scales, const float *biases, int there, int lane) {
  typedef int4v Four __attribute__((aligned(4)));
  typedef int int3v __attribute__((ext_vector_type(3)));
  typedef int3v Three __attribute__((aligned(4)));
  const unsigned odd = (unsigned)(reinterpret_cast<uintptr_t>(to) >> 1 & 1), shift = 16 * odd;
  Results<T> now, next;
  now.form(acc[0][i], by, scales, biases, lane);
  if (lane < 32 && odd && there > 0) to[0] = __builtin_bit_cast(T, (unsigned short)now.chunk[0][0]);
#pragma unroll
  for (int j = 0; j < NB; ++j) {
    __builtin_amdgcn_sched_barrier(0);
    if (j + 1 < NB) next.form(acc[j + 1 < NB ? j + 1 : 0][i], by, scales + 32 * (j + 1), biases + 32 * (j + 1), lane);
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int4v d = now.chunk[c];
      const int at = 32 * j + now.place(c, lane), left = there - at;
      // the next chunk is the partner's: the same for the lower lanes, for the upper ones the one after
      int a = d[0], b = c == 0 ? now.chunk[1][0] : j + 1 < NB ? next.chunk[0][0] : 0;
      swap_halves(a, b);
      const int follows = lane < 32 ? b : a;
      const bool last = c == 1 && j == NB - 1 && lane >= 32;      // (what follows is another wave's)
      const int4v s = {(int)__builtin_amdgcn_alignbit((unsigned)d[1], (unsigned)d[0], shift), (int)__builtin_amdgcn_alignbit((unsigned)d[2], (unsigned)d[1], shift),
                       (int)__builtin_amdgcn_alignbit((unsigned)d[3], (unsigned)d[2], shift), (int)__builtin_amdgcn_alignbit((unsigned)follows, (unsigned)d[3], shift)};
      if (8 + (int)odd <= left && !(last && odd)) {
        *reinterpret_cast<Four *>(to + at + odd) = s;
      } else if (last && odd && 8 <= left) {
        *reinterpret_cast<Three *>(to + at + 1) = int3v{s[0], s[1], s[2]};
        to[at + 7] = __builtin_bit_cast(T, (unsigned short)((unsigned)d[3] >> 16));
      } else {
        store_elements<T>(to + at, left, d, (int)odd);
      }
    }
    now = next;
  }
}

// A lane's chunks of 32 bytes of a tile's depth, for 32 MB rows of x and 32 NB outputs.
template <int MB, int NB, int DEPTH>
struct Fragments {
  int4v x[MB], w[NB];
  __device__ __forceinline__ void read(const int4v *x_tile, const int4v *w_tile, int at) {
#pragma unroll
    for (int i = 0; i < MB; ++i) x[i] = x_tile[2 * i * DEPTH + at];
#pragma unroll
    for (int j = 0; j < NB; ++j) w[j] = w_tile[2 * j * DEPTH + at];
  }
  __device__ __forceinline__ void multiply(int16v (&acc)[NB][MB]) const {
#pragma unroll
    for (int j = 0; j < NB; ++j)
#pragma unroll
      for (int i = 0; i < MB; ++i) acc[j][i] = __builtin_amdgcn_mfma_i32_32x32x32_i8(w[j], x[i], acc[j][i], 0, 0, 0);
  }
};

struct Nothing {
  __device__ __forceinline__ void operator()() const {}
};

// The next chunks are read while these are multiplied, and LOADS loads asked for: one of each between every few products.  (All 16 loads of a tile
// in a row keep the wave from its products: 8192^3 478 us, this way 443.)
template <int LOADS, int MB, int NB, int DEPTH, typename L>
__device__ __forceinline__ void step(int16v (&acc)[NB][MB], const Fragments<MB, NB, DEPTH> &now, Fragments<MB, NB, DEPTH> &next, const int4v *x_tile,
                                     const int4v *w_tile, int at, const L &load) {
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

// The chunks of a tile behind its first two, of which the second are in `other`, to its last (in `other` then), whose products are left.
template <int MB, int NB, int DEPTH>
__device__ __forceinline__ void rest_of(int16v (&acc)[NB][MB], Fragments<MB, NB, DEPTH> &first, Fragments<MB, NB, DEPTH> &other, const int4v *x_tile,
                                        const int4v *w_tile, const int (&at)[DEPTH / 32]) {
  if constexpr (DEPTH == 128) {
    step<0>(acc, other, first, x_tile, w_tile, at[2], Nothing());
    step<0>(acc, first, other, x_tile, w_tile, at[3], Nothing());
  }
}

// ... and the first two of the next one.  load_x and load_w ask for the tile after that, into this one's place, as soon as all waves have read theirs.
template <int MB, int NB, int DEPTH, typename L0, typename L1>
__device__ __forceinline__ void turn(int16v (&acc)[NB][MB], Fragments<MB, NB, DEPTH> &first, Fragments<MB, NB, DEPTH> &other, const int4v *x_now,
                                     const int4v *w_now, const int4v *x_next, const int4v *w_next, const int (&at)[DEPTH / 32], const L0 &load_x,
                                     const L1 &load_w) {
  rest_of(acc, first, other, x_now, w_now, at);
  tiles_ready();
  __builtin_amdgcn_sched_barrier(0);
  step<MB * DEPTH / 64>(acc, other, first, x_next, w_next, at[0], load_x);
  step<NB * DEPTH / 64>(acc, first, other, x_next, w_next, at[1], load_w);
}

// 64 MB rows of x by 64 NB outputs to a workgroup, 32 MB by 32 NB to a wave.  Four waves have a tile of LDS after another, from the last on; with KW
// above one, as many fours take turns at the tiles and add their sums up at the end.
// 256 by 256: four waves of 128 by 128, as the fragments of a step are then 8 KB to 16 products of 32 cycles, half of what LDS can give, and the tiles'
// way into it another quarter; one wave a SIMD, whose reads and loads go between its products.  8192^3, bf16: 432 to 444 us, 2.47 to 2.55 POP/s where a large
// library product has 2.16; the matrix pipe is busy 73 % of the time, at 1.6 GHz: what bounds it is power.
template <typename T, int MB, int NB, int KW, int DEPTH>
__global__ __launch_bounds__(256 * KW, (MB * NB >= 16 ? 1 : KW > 1 ? KW : DEPTH == 128 ? 2 : 4)) void int8_linear_kernel(const Int8LinearArgs a, unsigned x_tiles, unsigned w_tiles) {
  constexpr int XR = 64 * MB, WR = 64 * NB, CH = DEPTH / 16;
  __shared__ int4v x_tiles0[KW * XR * CH], w_tiles0[KW * WR * CH], x_tiles1[KW * XR * CH], w_tiles1[KW * WR * CH];
  __shared__ float scales[WR], biases[WR], row_scales[XR];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64 % 4), four = __builtin_amdgcn_readfirstlane(threadIdx.x / 256);
  unsigned xt, wt;
  place_of(blockIdx.x, x_tiles, w_tiles, xt, wt);
  const int64_t row0 = (int64_t)xt * XR;
  const int out0 = (int)wt * WR;
  const int x0 = wave % 2 * 32 * MB, w0 = wave / 2 * 32 * NB;
  int4v *const x_tile0 = x_tiles0 + four * XR * CH, *const w_tile0 = w_tiles0 + four * WR * CH;
  int4v *const x_tile1 = x_tiles1 + four * XR * CH, *const w_tile1 = w_tiles1 + four * WR * CH;
  Stager<XR, DEPTH> x;
  Stager<WR, DEPTH> w;
  x.open(a.x, row0, a.n, a.x_row, a.depth);
  w.open(a.weight, out0, a.outputs, a.weight_row, a.depth);
  // Tile i of this four: the last goes first.  (What lies behind a row in its last 16 bytes is not known, and is out of the way then: zeros on
  // one side are enough.)  Tiles in front of the first are zeros.
  const int all = (a.depth + DEPTH - 1) / DEPTH, tiles = (all + KW - 1) / KW;
  const auto k_of = [&](int i) {
    const int tile = all - 1 - four - i * KW;
    return tile < 0 ? a.depth : tile * DEPTH;
  };
  x.load(x_tile0, k_of(0), a.depth);
  w.load(w_tile0, k_of(0), a.depth);
  x.load(x_tile1, k_of(1), a.depth);
  w.load(w_tile1, k_of(1), a.depth);
  // scales and bias of the workgroup's outputs, scales of its rows: to LDS when all products are done
  static_assert(XR == WR && 256 * KW >= WR, "");
  const int mine = min(out0 + (int)threadIdx.x, a.outputs - 1);
  const float scale = a.weight_scales[mine], row_scale = a.x_scales[min(row0 + (int)threadIdx.x, a.n - 1)];
  const T bias = a.bias ? ((const T *)a.bias)[mine] : (T)0.f;
  int at[DEPTH / 32];
#pragma unroll
  for (int s = 0; s < DEPTH / 32; ++s) at[s] = chunk_at<DEPTH>(lane % 32, 2 * s + lane / 32);
  int16v acc[NB][MB] = {};
  // the first tile is there, the second may be on its way
  constexpr int kBehind = x.PER + w.PER;
  __builtin_amdgcn_s_waitcnt(0x0f70 | (kBehind & 15) | (kBehind & 48) << 10);
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();      // (__syncthreads waits for all loads)
  asm volatile("" ::: "memory");
  if (a.depth % 16) {
    for (int row = threadIdx.x; row < XR; row += 256 * KW) {
      int8_t *const end = (int8_t *)&x_tiles0[chunk_at<DEPTH>(row, a.depth % DEPTH / 16)];
      for (int b = a.depth % 16; b < 16; ++b) end[b] = 0;
    }
    __syncthreads();
  }
  // (no choice in the loop: the accumulators would be moved from registers to registers)
  const int4v *const x0_now = x_tile0 + x0 * CH, *const w0_now = w_tile0 + w0 * CH, *const x1_now = x_tile1 + x0 * CH, *const w1_now = w_tile1 + w0 * CH;
  Fragments<MB, NB, DEPTH> first, other;
  first.read(x0_now, w0_now, at[0]);
  step<0>(acc, first, other, x0_now, w0_now, at[1], Nothing());
  int i = 0;
  for (; i + 2 < tiles; i += 2) {
    turn(acc, first, other, x0_now, w0_now, x1_now, w1_now, at, [&] { x.load(x_tile0, k_of(i + 2), a.depth); }, [&] { w.load(w_tile0, k_of(i + 2), a.depth); });
    turn(acc, first, other, x1_now, w1_now, x0_now, w0_now, at, [&] { x.load(x_tile1, k_of(i + 3), a.depth); }, [&] { w.load(w_tile1, k_of(i + 3), a.depth); });
  }
  rest_of(acc, first, other, x0_now, w0_now, at);
  if (i + 1 < tiles) {
    tiles_ready();
    step<0>(acc, other, first, x1_now, w1_now, at[0], Nothing());
    step<0>(acc, first, other, x1_now, w1_now, at[1], Nothing());
    rest_of(acc, first, other, x1_now, w1_now, at);
  }
  other.multiply(acc);
  tiles_ready();      // (zeros asked for behind the last tile have landed before their place or the workgroup's LDS is used again)
  if (threadIdx.x < WR) scales[threadIdx.x] = scale, biases[threadIdx.x] = (float)bias, row_scales[threadIdx.x] = row_scale;
  if constexpr (KW == 1) __syncthreads();
  if constexpr (KW > 1) {
    static_assert(MB == 1 && NB == 1 && KW <= 4 && DEPTH == 128, "");
    // 16 KB a four: two in x's first tiles, the third in the weights'
    const auto place = [&](int f) { return (f < 3 ? x_tiles0 : w_tiles0) + (f - 1) % 2 * 1024 + threadIdx.x % 256; };
    if (four > 0)
#pragma unroll
      for (int q = 0; q < 4; ++q) place(four)[q * 256] = int4v{acc[0][0][4 * q], acc[0][0][4 * q + 1], acc[0][0][4 * q + 2], acc[0][0][4 * q + 3]};
    __syncthreads();
    if (four > 0) return;
#pragma unroll
    for (int f = 1; f < KW; ++f)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int4v more = place(f)[q * 256];
#pragma unroll
        for (int e = 0; e < 4; ++e) acc[0][0][4 * q + e] += more[e];
      }
  }
  const bool odd = sizeof(T) == 2 && (a.outputs % 2 || reinterpret_cast<uintptr_t>(a.out) % 4);
#pragma unroll
  for (int i = 0; i < MB; ++i) {
    const int64_t row = row0 + x0 + 32 * i + lane % 32;
    const int there = row < a.n ? a.outputs - out0 - w0 : 0;      // (a lane whose row is not there keeps its partner company in the exchange)
    T *const to = (T *)a.out + row * a.outputs + out0 + w0;
    const float by = row_scales[x0 + 32 * i + lane % 32];
    if constexpr (sizeof(T) == 2) {
      if (odd) {
        store_odd_row<T, MB, NB>(to, acc, i, by, scales + w0, biases + w0, there, lane);
        continue;
      }
    }
    store_row<T, MB, NB>(to, acc, i, by, scales + w0, biases + w0, there, lane);
  }
}

// Few rows of x: the weights' way from memory counts.  A workgroup has 16 outputs, its waves take turns along the depth, 256 bytes of each row at
// a time, straight into registers, and add their sums up in LDS.  (16 rows of 11008 to 4096: 45 MB in 14.6 us from memory, 12.8 where a cache holds
// the weights; one of 4096 to 4096: 17 MB in 6.9 and 4.9.)
template <typename T, int MB>
__global__ __launch_bounds__(512) void int8_linear_few_kernel(const Int8LinearArgs a) {
  constexpr int kWaves = 8, kSteps = 4;
  __shared__ int4v sums[kWaves][MB][64];
  const int lane = threadIdx.x % 64, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / 64);
  const int out0 = blockIdx.x * 16;
  // (rows behind the last are read as the last one, and left)
  const int8_t *const w = a.weight + min(out0 + lane % 16, a.outputs - 1) * a.weight_row + lane / 16 * 16, *x[MB];
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

template <typename T, int MB, int NB, int KW, int DEPTH>
int launch_tiles(const Int8LinearArgs &a) {
  const int64_t x_tiles = (a.n + 64 * MB - 1) / (64 * MB), w_tiles = (a.outputs + 64 * NB - 1) / (64 * NB);
  if (x_tiles * w_tiles > 0xffffffffll / (256 * KW)) {
    set_error("products in eight bits: more results than one launch takes");
    return FGMS_E_INVALID;
  }
  int8_linear_kernel<T, MB, NB, KW, DEPTH><<<(unsigned)(x_tiles * w_tiles), 256 * KW, 0, a.stream>>>(a, (unsigned)x_tiles, (unsigned)w_tiles);
  return FGMS_OK;
}

template <typename T, int MB>
int launch_few(const Int8LinearArgs &a) {
  int8_linear_few_kernel<T, MB><<<(unsigned)((a.outputs + 15) / 16), 512, 0, a.stream>>>(a);
  return FGMS_OK;
}

// Up to 32 rows: sixteen outputs a workgroup where that leaves a CU no more than two (32 rows of 4096 to 4096 outputs 8.0 us, tiles of 64 by four
// fours 9.9; to 11008 outputs 17 to 19 and 11.5).  Otherwise the widest tiles that fill the chip: 256 in lives of more than eight tiles (24000 rows, 4096
// outputs, 1024 deep: 128 us with 256 as with 128, 2048 deep 201 and 220, 512 deep 104 and 85), 128, and 64 with two fours along the depth, or four
// where the tiles are not even one a CU (256 x 4096 x 4096: 12.7 us with two, 11.1 with four, 21.6 with tiles of 128; 512 rows 14.9, 21.3, 22.3).  Up to 128
// deep a tile has 64 bytes of depth and a CU twice the workgroups, which hide each other's ends (120000 rows of 128 to 384: 25.6 -> 22.9 us; 50000
// of 256 to 768 the other way, 25.9 -> 29.4), up to 64 outputs in tiles that these fill (200000 rows of 64 to 64: 11.5 -> 10.1).  All of these with one set of
// tensors, which the last-level cache holds where it can; from memory 256 x 4096 x 4096 takes 15.2 us, 120000 of 128 to 384 36, 50000 of 256 to 768 33, 200000 of
// 64 to 64 14.  The rule goes by the number of tiles and not by how far rows fill them: one row of 4096 to 128256 outputs runs in tiles of 256 (526 MB of
// weights in 136 us).
template <typename T>
int launch(const Int8LinearArgs &a) {
  const auto tiles = [&](int64_t side) { return ((a.n + side - 1) / side) * ((a.outputs + side - 1) / side); };
  const int64_t cus = num_cus();
  if (a.n <= 32 && a.outputs <= 32 * cus) return a.n <= 16 ? launch_few<T, 1>(a) : launch_few<T, 2>(a);
  if (a.depth <= 128) return a.outputs <= 64 || tiles(128) < cus ? launch_tiles<T, 1, 1, 1, 64>(a) : launch_tiles<T, 2, 2, 1, 64>(a);
  if (a.depth > 1024 && tiles(256) >= cus) return launch_tiles<T, 4, 4, 1, 128>(a);
  if (tiles(128) >= cus) return launch_tiles<T, 2, 2, 1, 128>(a);
  return a.depth >= 2048 && tiles(64) <= cus ? launch_tiles<T, 1, 1, 4, 128>(a) : launch_tiles<T, 1, 1, 2, 128>(a);
}

}  // namespace

int launch_int8_linear(const Int8LinearArgs &a) {
  const int rc = a.dtype == FGMS_F32 ? launch<float>(a) : a.dtype == FGMS_F16 ? launch<_Float16>(a) : launch<__bf16>(a);
  if (rc != FGMS_OK) return rc;
  FGMS_HIP_TRY(hipGetLastError());
  return FGMS_OK;
}

}  // namespace fgms
