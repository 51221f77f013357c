// Rows of features on their way from one branch of a block to the next:
//
//   h = x factor + residual          factor: 1, or with dropout 0 or 1 / (1 - p), from a generator that counts the elements
//   y = h r w,  r = 1 / sqrt(mean h^2 + eps)
//   s = max |v| / 127, q = round(v / s)      of a row v: the norm, x itself or silu(a) b
//   backward:  gs = g_h + r (w g_y - h r^2 mean(w g_y h));  g_residual = gs;  g_x = gs factor;  g_w = sum g_y h r
//
// A dozen operations an element: memory is what the kernels have to wait for.  h is rounded to the type before its norm is taken: it is a
// result, and the backward pass, which reads it, then forms the gradient of the very values that were computed.
#include "fgms_rows.h"

#include "fgms_internal.h"
#include "fgms_mma.h"

namespace fgms {
namespace {

// (an array, whose elements the compiler keeps apart)
struct Eight {
  float v[8];
  __device__ __forceinline__ float &operator[](int e) { return v[e]; }
  __device__ __forceinline__ float operator[](int e) const { return v[e]; }
  template <typename F>
  __device__ __forceinline__ void each(F f) {
#pragma unroll
    for (int e = 0; e < 8; ++e) f(v[e], e);
  }
};
typedef int8_t byte8v __attribute__((ext_vector_type(8)));
typedef byte8v Byte8Anywhere __attribute__((aligned(1)));

// Sixteen random bits for each of eight neighbouring elements: Philox4x32 with ten rounds (Salmon, Moraes, Dror, Shaw, "Parallel random
// numbers: as easy as 1, 2, 3", SC 2011), counter (chunk, seed[1]), key seed[0].  Word e of a chunk is half e % 2 of the call's number e / 2.
// (16 bits a word: a call of ten rounds takes some 90 instructions, half of them at a quarter of the rate; with a call for four elements
// the multiplier, and not memory, would set the pace of 16-bit tensors.  p is met to 2^-17.)
struct Words {
  unsigned v[4];
  __device__ __forceinline__ bool falls(int e, unsigned below) const { return (v[e / 2] >> (16 * (e % 2)) & 0xffffu) < below; }
};
__device__ __forceinline__ Words words_of(int64_t chunk, const int64_t *__restrict__ seed) {
  unsigned k0 = (unsigned)seed[0], k1 = (unsigned)((uint64_t)seed[0] >> 32);
  unsigned c0 = (unsigned)chunk, c1 = (unsigned)((uint64_t)chunk >> 32), c2 = (unsigned)seed[1], c3 = (unsigned)((uint64_t)seed[1] >> 32);
#pragma unroll
  for (int round = 0; round < 10; ++round) {
    const uint64_t p = (uint64_t)0xD2511F53u * c0, q = (uint64_t)0xCD9E8D57u * c2;
    c0 = (unsigned)(q >> 32) ^ c1 ^ k0;
    c1 = (unsigned)q;
    c2 = (unsigned)(p >> 32) ^ c3 ^ k1;
    c3 = (unsigned)p;
    k0 += 0x9E3779B9u, k1 += 0xBB67AE85u;
  }
  return Words{{c0, c1, c2, c3}};
}

// Eight channels of a row from `c` on, zeros behind the last.  WHOLE: there are eight, and they begin on 16 bytes; other rows are read and written
// 16 bytes at a time too, wherever these begin, and by elements where they end.
template <typename T, bool WHOLE>
struct Chunk {
  static constexpr int N = 16 / (int)sizeof(T);
  typedef T Aligned __attribute__((ext_vector_type(N)));
  typedef Aligned Vector __attribute__((aligned(WHOLE ? 16 : sizeof(T))));
};
// ... as they come from memory, in half the registers of their values where these have 16 bits.
template <typename T>
struct Raw {
  int4v part[sizeof(T) / 2];
  __device__ __forceinline__ Eight values() const {
    constexpr int N = 16 / (int)sizeof(T);
    typedef T Tn __attribute__((ext_vector_type(N)));
    Eight to;
#pragma unroll
    for (int i = 0; i < 8 / N; ++i) {
      const Tn from = __builtin_bit_cast(Tn, part[i]);
#pragma unroll
      for (int e = 0; e < N; ++e) to[i * N + e] = (float)from[e];
    }
    return to;
  }
};
template <typename T, bool WHOLE>
__device__ __forceinline__ Raw<T> load_raw(const T *__restrict__ row, int c, int channels, bool there = true) {
  typedef Chunk<T, WHOLE> C;
  Raw<T> to = {};
  if (!there || c >= channels) return to;
  if (WHOLE || c + 8 <= channels) {
#pragma unroll
    for (int i = 0; i < 8 / C::N; ++i) to.part[i] = __builtin_bit_cast(int4v, (typename C::Aligned)reinterpret_cast<const typename C::Vector *>(row + c)[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8 / C::N; ++i) {
      typename C::Aligned v;
#pragma unroll
      for (int e = 0; e < C::N; ++e) v[e] = c + i * C::N + e < channels ? row[c + i * C::N + e] : (T)0.f;
      to.part[i] = __builtin_bit_cast(int4v, v);
    }
  }
  return to;
}
template <typename T, bool WHOLE>
__device__ __forceinline__ void store8(T *__restrict__ row, int c, int channels, const Eight &v) {
  typedef Chunk<T, WHOLE> C;
  if (WHOLE || c + 8 <= channels) {
#pragma unroll
    for (int i = 0; i < 8 / C::N; ++i) {
      typename C::Aligned to;
#pragma unroll
      for (int e = 0; e < C::N; ++e) to[e] = (T)v[i * C::N + e];
      reinterpret_cast<typename C::Vector *>(row + c)[i] = to;
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < channels) row[c + e] = (T)v[e];
  }
}
__device__ __forceinline__ void add(Eight &to, const Eight &v) {
  to.each([&](float &t, int e) { t += v[e]; });
}

// How a row lies on its lanes: lane l of `lanes` (a power of two) has chunks l, l + lanes, ... of eight channels, `chunks` of them.  Up to 2048
// channels a row is a wave's or less and is summed by exchanges between lanes alone; the widest take 1024 threads, whose registers
// hold two chunks.  Gradients have rows of 2049 to 8192 channels on a chunk a thread, which leaves room to ask for the next row (4096 rows of 8192, fp32, the
// norm's gradient, the sum's, the sum and the result, 537 MB, with the scale's second launch: 121 us on 256 threads, 110 so; fp16 76 and 72).
struct Share {
  int lanes, chunks, threads;
};
inline Share share_of(int channels, bool gradient = false) {
  const int all = (channels + 7) / 8;
  if (gradient && all > 256 && all <= 1024) return all > 512 ? Share{1024, 1, 1024} : Share{512, 1, 512};
  if (all > 1024) return Share{1024, 2, 1024};
  if (all > 256) return Share{256, all > 512 ? 4 : 2, 256};
  int lanes = 1;
  while (lanes < 64 && lanes < all) lanes *= 2;
  return Share{lanes, (all + lanes - 1) / lanes, 256};
}

// Sum over / largest of the lanes of a row.  `part`: a number for each wave, not in use by another exchange.
template <typename V, typename F>
__device__ __forceinline__ V over_row(V v, int lanes, V *part, F join) {
  for (int d = 1; d < lanes && d < 64; d *= 2) v = join(v, __shfl_xor(v, d));
  if (lanes > 64) {
    const int wave = threadIdx.x / 64, waves = lanes / 64, first = wave / waves * waves;
    if (threadIdx.x % 64 == 0) part[wave] = v;
    __syncthreads();
    v = part[first];
    for (int w = 1; w < waves; ++w) v = join(v, part[first + w]);
  }
  return v;
}
__device__ __forceinline__ float sum_of(float a, float b) { return a + b; }
// (of the bits of numbers without their sign, which are in the numbers' order, infinity and then NaN behind the others)
__device__ __forceinline__ unsigned larger_of(unsigned a, unsigned b) { return a > b ? a : b; }

// A row to each group of lanes, once: what a launch of any kind (WHAT) reads and writes is all that memory moves.  (50000 rows of 256, fp32: 205 MB in
// 41 us, 5.0 TB/s; 16384 of 2048, fp16: 268 MB in 46 us, 5.8 TB/s; 120000 of 128, fp16, with dropout: 123 MB in 25 us; a norm of 200000 of 64 to eight bits:
// 90 MB in 19 to 21 us; 200000 of 64 as they are, fp16 to eight bits: 39 MB in 12 us; 16 gated rows of 11008: 5.7 us.)
template <typename T, int CHUNKS, int THREADS, bool WHOLE, int WHAT>
__global__ __launch_bounds__(THREADS) void rows_kernel(const RowsArgs a, int lanes) {
  constexpr bool NORM = WHAT == kRowsNorm || WHAT == kRowsNormEighths;
  __shared__ float sums[THREADS / 64];
  __shared__ unsigned tops[THREADS / 64];
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t row = (int64_t)blockIdx.x * (THREADS / lanes) + threadIdx.x / lanes;
  const bool there = row < a.n;
  const int per_row = (a.channels + 7) / 8;
  // (all that is read, before any of it is waited for)
  const T *const x = (const T *)a.x + row * a.x_row;
  Raw<T> x_raw[CHUNKS], other[CHUNKS];
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) x_raw[i] = load_raw<T, WHOLE>(x, 8 * (lane + i * lanes), a.channels, there);
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int c = 8 * (lane + i * lanes);
    if constexpr (WHAT == kRowsGatedEighths) other[i] = load_raw<T, WHOLE>(x + a.channels, c, a.channels, there);
    if constexpr (NORM) other[i] = load_raw<T, WHOLE>((const T *)a.residual + row * a.residual_row, c, a.channels, there && a.residual);
  }
  Eight v[CHUNKS];
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) v[i] = x_raw[i].values();
  if constexpr (WHAT == kRowsGatedEighths) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const Eight b = other[i].values();
      // (the exponential and the reciprocal as the unit gives them: of 2 M values two fall to the other side of a border, as many as with divisions; where the
      // exponential's reciprocal is no normal number, a below -87.3, silu counts as zero.  50000 rows of 256, fp16: 16.1 us, 18.3 with the argument's rest and a
      // Newton step; fp32 21.6 and 22.0)
      v[i].each([&](float &t, int e) { t = t * __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * t)) * b[e]; });
    }
  }
  if constexpr (NORM) {
    Raw<T> w[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) w[i] = load_raw<T, WHOLE>((const T *)a.scale, 8 * (lane + i * lanes), a.channels, a.scale);
    float square = 0.f;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = 8 * (lane + i * lanes);
      if (!there || c >= a.channels) continue;
      if (a.dropped) {
        const Words words = words_of((a.first + row) * per_row + c / 8, a.seed);
        v[i].each([&](float &t, int e) { t = words.falls(e, a.dropped) ? 0.f : t * a.back; });
      }
      add(v[i], other[i].values());
      v[i].each([](float &t, int) { t = (float)(T)t; });      // (x itself stays what it is)
      if (a.sum) store8<T, WHOLE>((T *)a.sum + row * a.channels, c, a.channels, v[i]);
      v[i].each([&](float &t, int) { square = __builtin_fmaf(t, t, square); });
    }
    square = over_row(square, lanes, sums, sum_of);
    const float r = 1.f / __builtin_sqrtf(square / (float)a.channels + a.eps);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = 8 * (lane + i * lanes);
      if (!there || c >= a.channels) continue;
      v[i].each([&](float &t, int) { t *= r; });
      if (a.scale) {
        const Eight wv = w[i].values();
        v[i].each([&](float &t, int e) { t *= wv[e]; });
      }
      if constexpr (WHAT == kRowsNorm) store8<T, WHOLE>((T *)a.out + row * a.channels, c, a.channels, v[i]);
    }
  }
  if constexpr (WHAT != kRowsNorm) {
    unsigned top = 0;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float value = v[i][e];
        top = larger_of(top, __builtin_bit_cast(unsigned, value) & 0x7fffffffu);
      }
    top = over_row(top, lanes, tops, larger_of);
    // A row with an infinity or NaN stands for NaN in every channel, one whose step would be no normal number for zeros.
    const bool finite = top < 0x7f800000u;
    const float most = __builtin_bit_cast(float, top), step = most / 127.f;
    const bool some = finite && step >= 0x1p-126f;
    const float by = some ? 1.f / step : 0.f;
    if (there && lane == 0) a.scales[row] = some ? step : finite ? 0.f : __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = 8 * (lane + i * lanes);
      if (!there || c >= a.channels) continue;
      byte8v q;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        // The quotient by the step, rounded as a division rounds it (halves are met where they are meant): its remainder is exact, the first correction
        // brings it within its last bit, the second is right with a reciprocal that is (P. Markstein, IBM J. Res. Dev. 34, 1990).  A division's own
        // steps take 10 to 25 % longer (200000 rows of 64 that a cache holds 12.4 us, this 10.5 to 10.8; from memory this takes 12.2).
        const float value = v[i][e], near = value * by, nearer = __builtin_fmaf(__builtin_fmaf(-near, step, value), by, near);
        const float quotient = __builtin_fmaf(__builtin_fmaf(-nearer, step, value), by, nearer);
        q[e] = some ? (int8_t)(int)__builtin_rintf(quotient) : (int8_t)0;
      }
      int8_t *const to = a.eighths + row * a.eighths_row + c;
      if (WHOLE || c + 8 <= a.channels) {
        *reinterpret_cast<Byte8Anywhere *>(to) = q;
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (c + e < a.channels) to[e] = q[e];
      }
    }
  }
}

// A workgroup goes through the rows in steps of the grid and keeps its lanes' sums of the scale's gradient in registers.  The next row is asked for
// before this one is worked on: the registers of three chunks leave two waves a SIMD, whose loads alone would not keep memory busy.  (120000 rows of 128,
// fp16, with dropout: 154 MB in 32 to 34 us; 10007 of 1096, bf16: 88 MB in 21 to 23 us; 50000 of 256, fp32: 205 MB in 42 us; 4096 of 16384, fp16, where
// nothing is asked for ahead: 537 MB in 117 us.)
template <typename T, int CHUNKS, int THREADS, bool WHOLE>
__global__ __launch_bounds__(THREADS) void add_norm_grad_kernel(const RowsArgs a, int lanes) {
  __shared__ float parts[2][2][THREADS / 64];
  __shared__ Eight all[THREADS == 256 ? CHUNKS * 256 : 1];
  const int lane = threadIdx.x & (lanes - 1), group = threadIdx.x / lanes, groups = THREADS / lanes, per_row = (a.channels + 7) / 8;
  Raw<T> w[CHUNKS];
  Eight gw[CHUNKS] = {};
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) w[i] = load_raw<T, WHOLE>((const T *)a.scale, 8 * (lane + i * lanes), a.channels, a.scale);
  Raw<T> next_h[CHUNKS], next_g[CHUNKS], next_gs[CHUNKS];
  const auto ask = [&](int64_t row) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = 8 * (lane + i * lanes);
      next_h[i] = load_raw<T, WHOLE>((const T *)a.sum + row * a.x_row, c, a.channels, row < a.n);
      next_g[i] = load_raw<T, WHOLE>((const T *)a.g_out + row * a.channels, c, a.channels, row < a.n);
      next_gs[i] = load_raw<T, WHOLE>((const T *)a.g_sum + row * a.channels, c, a.channels, row < a.n && a.g_sum);
    }
  };
  int64_t row = (int64_t)blockIdx.x * groups + group;
  const int64_t stride = (int64_t)gridDim.x * groups;
  constexpr bool kAhead = THREADS * CHUNKS < 2048;      // (two chunks of 1024 threads have no registers for it)
  if (kAhead) ask(row);
  int turn = 0;      // (a row's exchanges and the next one's do not share their places)
  for (int64_t first = (int64_t)blockIdx.x * groups; first < a.n; first += stride, row += stride, turn ^= 1) {
    if (!kAhead) ask(row);
    Raw<T> h[CHUNKS], g[CHUNKS], gs_raw[CHUNKS];
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) h[i] = next_h[i], g[i] = next_g[i], gs_raw[i] = next_gs[i];
    if (kAhead) ask(row + stride);
    const bool there = row < a.n;
    float square = 0.f, along = 0.f;
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const Eight hv = h[i].values(), gv = g[i].values();
      Eight wv = w[i].values();
      wv.each([&](float &t, int e) {
        square = __builtin_fmaf(hv[e], hv[e], square);
        along = __builtin_fmaf((a.scale ? t : 1.f) * gv[e], hv[e], along);
      });
    }
    square = over_row(square, lanes, parts[turn][0], sum_of);
    along = over_row(along, lanes, parts[turn][1], sum_of);
    const float r = 1.f / __builtin_sqrtf(square / (float)a.channels + a.eps), back = r * r * (along / (float)a.channels);
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) {
      const int c = 8 * (lane + i * lanes);
      if (!there || c >= a.channels) continue;
      const Eight hv = h[i].values(), gv = g[i].values(), wv = w[i].values(), more = gs_raw[i].values();
      gw[i].each([&](float &t, int e) { t = __builtin_fmaf(gv[e] * r, hv[e], t); });
      Eight gs;
      gs.each([&](float &t, int e) { t = __builtin_fmaf(r, (a.scale ? wv[e] : 1.f) * gv[e] - hv[e] * back, more[e]); });
      if (a.g_residual) store8<T, WHOLE>((T *)a.g_residual + row * a.channels, c, a.channels, gs);
      if (a.gx) {
        if (a.dropped) {
          const Words words = words_of(row * per_row + c / 8, a.seed);
          gs.each([&](float &t, int e) { t = words.falls(e, a.dropped) ? 0.f : t * a.back; });
        }
        store8<T, WHOLE>((T *)a.gx + row * a.channels, c, a.channels, gs);
      }
    }
  }
  if (!a.scale_sums) return;
  // the groups of lanes, in their order
  float *const to = a.scale_sums + (int64_t)blockIdx.x * a.channels;
  if (groups > 1) {
#pragma unroll
    for (int i = 0; i < CHUNKS; ++i) all[i * 256 + threadIdx.x] = gw[i];
    __syncthreads();
    if (group) return;
    for (int other = 1; other < groups; ++other)
#pragma unroll
      for (int i = 0; i < CHUNKS; ++i) add(gw[i], all[i * 256 + other * lanes + lane]);
  }
#pragma unroll
  for (int i = 0; i < CHUNKS; ++i) {
    const int c = 8 * (lane + i * lanes);
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (c + e < a.channels) to[c + e] = gw[i][e];
  }
}

// out[channel] = the workgroups' sums, eight channels a workgroup, 32 threads each, in a fixed order.  (1250 sums of 128: 5.5 us, 501 of 1096: 4.4, 256 of 16384:
// 11.8.)
template <typename T>
__global__ __launch_bounds__(256) void column_sums_kernel(const float *__restrict__ sums, int64_t groups, int channels, T *__restrict__ out) {
  __shared__ float part[4][8];
  const int c = threadIdx.x % 8, column = blockIdx.x * 8 + c;
  float sum = 0.f;
  if (column < channels)
#pragma unroll 8
    for (int64_t b = threadIdx.x / 8; b < groups; b += 32) sum += sums[b * channels + column];
  for (int d = 8; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if (threadIdx.x % 64 < 8) part[threadIdx.x / 64][c] = sum;
  __syncthreads();
  if (threadIdx.x < 8 && column < channels) out[column] = (T)(part[0][c] + part[1][c] + part[2][c] + part[3][c]);
}

// Eight elements a thread, counted through the rows; their words while they are on their way.  (200000 rows of 64, fp32: 154 MB in 28 us; 16384 of 4096,
// bf16: 403 MB in 70 to 72 us, 5.7 TB/s.)
template <typename T, bool WHOLE>
__global__ __launch_bounds__(256) void dropout_add_kernel(const RowsArgs a, int64_t chunks) {
  const int per_row = (a.channels + 7) / 8;
  const int64_t at = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (at >= chunks) return;
  const int64_t row = at / per_row;
  const int c = 8 * (int)(at - row * per_row);
  const Raw<T> x = load_raw<T, WHOLE>((const T *)a.x + row * a.x_row, c, a.channels);
  const Raw<T> residual = load_raw<T, WHOLE>((const T *)a.residual + row * a.residual_row, c, a.channels, a.residual);
  Words words = {};
  if (a.dropped) words = words_of(a.first * per_row + at, a.seed);
  Eight v = x.values();
  if (a.dropped) v.each([&](float &t, int e) { t = words.falls(e, a.dropped) ? 0.f : t * a.back; });
  if (a.residual) add(v, residual.values());
  store8<T, WHOLE>((T *)a.out + row * a.channels, c, a.channels, v);
}

// --- launches --------------------------------------------------------------------------------------------------
template <int N> struct Number { static constexpr int value = N; };
template <int CHUNKS, int THREADS> struct Shape {
  static constexpr int chunks = CHUNKS, threads = THREADS;
};
template <typename F>
void by_share(const Share &s, F f) {
  if (s.threads == 1024) return f(Shape<2, 1024>());
  return s.chunks == 1 ? f(Shape<1, 256>()) : s.chunks == 2 ? f(Shape<2, 256>()) : s.chunks == 3 ? f(Shape<3, 256>()) : f(Shape<4, 256>());
}
template <typename F>
void by_grad_share(const Share &s, F f) {
  if (s.threads == 512) return f(Shape<1, 512>());
  if (s.threads == 1024 && s.chunks == 1) return f(Shape<1, 1024>());
  by_share(s, f);
}
template <typename F>
void by_type(int dtype, F f) {
  return dtype == FGMS_F32 ? f(float()) : dtype == FGMS_F16 ? f((_Float16)0) : f((__bf16)0);
}

// Launches over all rows, `rows` at most in one (a grid has fewer than 2^32 threads): f(the rows of one).
constexpr int64_t kMostThreads = (int64_t)1 << 31;
template <typename F>
void by_parts(const RowsArgs &a, int64_t rows, F f) {
  const int64_t size = a.dtype == FGMS_F32 ? 4 : 2;
  for (int64_t first = 0; first < a.n; first += rows) {
    const auto moved = [&](const void *p, int64_t row) { return p ? (const char *)p + first * row * size : nullptr; };
    RowsArgs part = a;
    part.first = first, part.n = a.n - first < rows ? a.n - first : rows;
    part.x = moved(a.x, a.x_row), part.residual = moved(a.residual, a.residual_row);
    part.sum = (void *)moved(a.sum, a.channels), part.out = (void *)moved(a.out, a.channels);
    if (a.eighths) part.eighths = a.eighths + first * a.eighths_row;
    if (a.scales) part.scales = a.scales + first;
    f(part);
  }
}

// Whether all rows begin on 16 bytes and are whole chunks of eight channels.
bool whole(const void *p, int64_t row, int size) { return reinterpret_cast<uintptr_t>(p) % 16 == 0 && row * size % 16 == 0; }
bool whole_rows(const RowsArgs &a) {
  const int size = a.dtype == FGMS_F32 ? 4 : 2;
  bool ok = a.channels % 8 == 0 && whole(a.x, a.x_row, size) && whole(a.sum, a.x_row, size) && (!a.residual || whole(a.residual, a.residual_row, size));
  for (const void *p : {a.scale, (const void *)a.out, a.g_out, a.g_sum, (const void *)a.gx, (const void *)a.g_residual}) ok = ok && whole(p, 0, size);
  return ok;
}

}  // namespace

int launch_rows(const RowsArgs &a, int what) {
  const Share s = share_of(a.channels);
  const int at_once = s.threads / s.lanes;
  const bool w = whole_rows(a);
  by_parts(a, kMostThreads / s.lanes, [&](const RowsArgs &part) {
    const unsigned grid = (unsigned)((part.n + at_once - 1) / at_once);
    by_type(a.dtype, [&](auto t) {
      using T = decltype(t);
      by_share(s, [&](auto shape) {
        constexpr int K = decltype(shape)::chunks, N = decltype(shape)::threads;
        const auto launch = [&](auto kind) {
          constexpr int WHAT = decltype(kind)::value;
          if (w) rows_kernel<T, K, N, true, WHAT><<<grid, N, 0, a.stream>>>(part, s.lanes);
          else rows_kernel<T, K, N, false, WHAT><<<grid, N, 0, a.stream>>>(part, s.lanes);
        };
        if (what == kRowsNorm) launch(Number<kRowsNorm>());
        else if (what == kRowsNormEighths) launch(Number<kRowsNormEighths>());
        else if (what == kRowsEighths) launch(Number<kRowsEighths>());
        else launch(Number<kRowsGatedEighths>());
      });
    });
  });
  FGMS_HIP_TRY(hipGetLastError());
  return FGMS_OK;
}

// About as many as run at once on 256 CUs, or fewer that all have as many rows: the last round of a grid is as long as the others.  (10007 rows of 1096, two
// at once: 1024 workgroups 24.8 us, 501 21.0.)  The counts are those of 16-bit rows of one to three chunks, whose registers leave a SIMD five, three or two
// waves; fp32 rows on 16 bytes leave four, two and one, rows of four chunks one in every type, so that some of their workgroups start behind the others.
int64_t scale_grad_groups(int64_t n, int channels) {
  const Share s = share_of(channels, true);
  const int at_once = s.threads / s.lanes;
  const int64_t all = (n + at_once - 1) / at_once, most = 256 * (s.threads == 1024 ? 1 : s.threads == 512 ? 2 : s.chunks == 1 ? 5 : s.chunks == 2 ? 3 : 2);
  const int64_t rounds = (all + most - 1) / most;
  return rounds ? (all + rounds - 1) / rounds : 0;
}

int launch_add_norm_bwd(const RowsArgs &a) {
  const Share s = share_of(a.channels, true);
  const unsigned grid = (unsigned)scale_grad_groups(a.n, a.channels);
  const bool w = whole_rows(a);
  by_type(a.dtype, [&](auto t) {
    using T = decltype(t);
    by_grad_share(s, [&](auto shape) {
      constexpr int K = decltype(shape)::chunks, N = decltype(shape)::threads;
      if (w) add_norm_grad_kernel<T, K, N, true><<<grid, N, 0, a.stream>>>(a, s.lanes);
      else add_norm_grad_kernel<T, K, N, false><<<grid, N, 0, a.stream>>>(a, s.lanes);
      if (a.g_scale) column_sums_kernel<T><<<(a.channels + 7) / 8, 256, 0, a.stream>>>(a.scale_sums, grid, a.channels, (T *)a.g_scale);
    });
  });
  FGMS_HIP_TRY(hipGetLastError());
  return FGMS_OK;
}

int launch_dropout_add(const RowsArgs &a) {
  const int per_row = (a.channels + 7) / 8;
  const bool w = whole_rows(a);
  by_parts(a, kMostThreads / per_row, [&](const RowsArgs &part) {
    const int64_t chunks = part.n * per_row;
    const unsigned grid = (unsigned)((chunks + 255) / 256);
    by_type(a.dtype, [&](auto t) {
      using T = decltype(t);
      if (w) dropout_add_kernel<T, true><<<grid, 256, 0, a.stream>>>(part, chunks);
      else dropout_add_kernel<T, false><<<grid, 256, 0, a.stream>>>(part, chunks);
    });
  });
  FGMS_HIP_TRY(hipGetLastError());
  return FGMS_OK;
}

}  // namespace fgms
