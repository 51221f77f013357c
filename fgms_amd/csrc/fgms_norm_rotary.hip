// Norms of queries and keys for each head, and their rotation by the rows' coordinates, in one pass; and its gradients.
//
//   z = x r w,  r = 1 / sqrt(mean x^2 + eps);   pair (a, b) of channels: y = (z_a cos f - z_b sin f, z_a sin f + z_b cos f)
//   h = the output gradient turned back;   gw = sum h x r;   gx = r (w h - x r^2 mean(w h x))
// A dozen operations an element: memory is what it has to wait for.  (50 k rows of 8 + 8 heads of 32, fp32: 205 MB in 33 us out of the caches, 45
// with inputs that change, 40 at the rate of a copy; 120 k rows of 4 + 4 heads of 32, fp16: 25 us forward, 41 + 3.5 back.)
#include "fgms_norm_rotary.h"

#include <optional>

#include "fgms_internal.h"
#include "fgms_mma.h"

namespace fgms {
namespace {

template <typename T, int V> using Vec = T __attribute__((ext_vector_type(V)));

// sin and cos of coordinate * frequency.  The angle of a far voxel has thousands of turns, of which 32 bits would leave the fraction a
// few digits only: the product and the reduction to an eighth of a turn are taken in 64 (a handful of operations a pair of
// channels, shared by all heads), the Taylor sums of the rest in 32 (up to pi / 4; the first terms left out are x^11 / 11!, below
// 2^-29, and x^12 / 12!, below 2^-33).
__device__ __forceinline__ void sine_cosine(int coordinate, float frequency, float &sine, float &cosine) {
  const double turns = (double)coordinate * (double)frequency * 0.15915494309189535;
  const double quarters = __builtin_rint(turns * 4.0);
  const float x = (float)((turns - quarters * 0.25) * 6.283185307179586);
  const int quadrant = (int)(quarters - 4.0 * __builtin_floor(quarters * 0.25));
  const float xx = x * x;
  const float s = x * (1.f + xx * (-1.f / 6 + xx * (1.f / 120 + xx * (-1.f / 5040 + xx * (1.f / 362880)))));
  const float c = 1.f + xx * (-0.5f + xx * (1.f / 24 + xx * (-1.f / 720 + xx * (1.f / 40320 - xx * (1.f / 3628800)))));
  const float a = quadrant & 1 ? c : s, b = quadrant & 1 ? s : c;
  sine = quadrant & 2 ? -a : a;
  cosine = quadrant == 1 || quadrant == 2 ? -b : b;
}

// The angles of `rows` rows from `first` on: turn[row][pair] = (cos, sin), (1, 0) for pairs that stay.
__device__ __forceinline__ void fill_angles(float2 *turn, const NormRotaryArgs &a, int64_t first, int rows) {
  const int pairs = a.dim / 2;
  for (int e = threadIdx.x; e < rows * pairs; e += 256) {
    const int row = e / pairs, pair = e % pairs;
    int axis = -1, end = 0;
#pragma unroll
    for (int i = kMaxAxes - 1; i >= 0; --i) {
      int upto = 0;
      for (int j = 0; j <= i; ++j) upto += a.sections[j];
      if (pair < upto) axis = i;
      end = max(end, upto);
    }
    float s = 0.f, c = 1.f;
    if (pair < end) sine_cosine(a.coords[(first + row) * a.axes + axis], a.freqs[pair], s, c);
    turn[e] = make_float2(c, s);
  }
}

template <typename T, int V>
__device__ __forceinline__ void load(float (&to)[V], const T *from) {
  const Vec<T, V> v = *reinterpret_cast<const Vec<T, V> *>(from);
#pragma unroll
  for (int i = 0; i < V; ++i) to[i] = (float)v[i];
}
template <typename T, int V>
__device__ __forceinline__ void store(T *to, const float (&from)[V]) {
  Vec<T, V> v;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = (T)from[i];
  *reinterpret_cast<Vec<T, V> *>(to) = v;
}

// A workgroup takes `tile` rows at a time: their angles to LDS once, then one head of one row to a group of `lanes` lanes (a power of
// two), heads next to each other.  A lane has V pairs of its head: channels p and p + dim / 2, or 2p and 2p + 1.
template <typename T, int V, bool NEXT, bool BACKWARD>
__global__ __launch_bounds__(256) void norm_rotary_kernel(const NormRotaryArgs a, int tile, int lanes, float *__restrict__ partial) {
  extern __shared__ int4v angles[];      // (16-byte reads)
  float2 *const turn = reinterpret_cast<float2 *>(angles);
  const int c = threadIdx.x & (lanes - 1), pairs = a.dim / 2;
  const bool there = c * V < pairs;
  const int at0 = there ? NEXT ? 2 * V * c : V * c : 0, at1 = NEXT ? at0 + V : pairs + at0;
  const float mean = 1.f / a.dim;
  float sums[2][2][V] = {};      // of h x r, this lane's channels
  const int64_t tiles = (a.n + tile - 1) / tile;
  for (int64_t t = blockIdx.x; t < tiles; t += gridDim.x) {
    const int64_t first = t * tile;
    const int rows = (int)min((int64_t)tile, a.n - first);
    __syncthreads();
    fill_angles(turn, a, first, rows);
    __syncthreads();
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      const int heads = a.heads[which];
      if (!heads) continue;
      const T *const scale = (const T *)a.scale[which];
      float w0[V], w1[V];
#pragma unroll
      for (int i = 0; i < V; ++i) w0[i] = w1[i] = 1.f;
      if (scale) {
        load<T, V>(w0, scale + at0);
        load<T, V>(w1, scale + at1);
      }
      for (int e = threadIdx.x / lanes; e < rows * heads; e += 256 / lanes) {
        const int row = e / heads, head = e % heads;
        const T *const x = (const T *)a.x[which] + (first + row) * a.row[which] + head * a.head[which];
        const int64_t to = ((first + row) * heads + head) * a.dim;
        float x0[V], x1[V], g0[V], g1[V];
        load<T, V>(x0, x + at0);
        load<T, V>(x1, x + at1);
        if constexpr (BACKWARD) {
          load<T, V>(g0, (const T *)a.gy[which] + to + at0);
          load<T, V>(g1, (const T *)a.gy[which] + to + at1);
        }
        float square = 0.f, along = 0.f;
#pragma unroll
        for (int i = 0; i < V; ++i) square = __builtin_fmaf(x0[i], x0[i], __builtin_fmaf(x1[i], x1[i], square));
        // turns pair p of (u, v) by its angle, or back
        const float2 *const angle = turn + row * pairs + V * (there ? c : 0);
        const auto rotate = [&](float (&u)[V], float (&v)[V]) {
#pragma unroll
          for (int i = 0; i < V; ++i) {
            const float cosine = angle[i].x, sine = BACKWARD ? -angle[i].y : angle[i].y;
            float &p = NEXT ? (2 * i < V ? u[2 * i % V] : v[2 * i % V]) : u[i], &q = NEXT ? (2 * i < V ? u[2 * i % V + 1] : v[2 * i % V + 1]) : v[i];
            const float p_ = p * cosine - q * sine;
            q = p * sine + q * cosine;
            p = p_;
          }
        };
        if constexpr (BACKWARD) {
          rotate(g0, g1);
#pragma unroll
          for (int i = 0; i < V; ++i) along = __builtin_fmaf(w0[i] * g0[i], x0[i], __builtin_fmaf(w1[i] * g1[i], x1[i], along));
        }
        if (!there) square = along = 0.f;
        for (int d = 1; d < lanes; d *= 2) {
          square += __shfl_xor(square, d);
          if constexpr (BACKWARD) along += __shfl_xor(along, d);
        }
        const float r = 1.f / __builtin_sqrtf(__builtin_fmaf(square, mean, a.eps));
        if constexpr (!BACKWARD) {
#pragma unroll
          for (int i = 0; i < V; ++i) x0[i] *= r * w0[i], x1[i] *= r * w1[i];
          rotate(x0, x1);
          if (there) {
            store<T, V>((T *)a.y[which] + to + at0, x0);
            store<T, V>((T *)a.y[which] + to + at1, x1);
          }
        } else {
          const float back = r * r * along * mean;
#pragma unroll
          for (int i = 0; i < V; ++i) {
            sums[which][0][i] = __builtin_fmaf(g0[i] * r, x0[i], sums[which][0][i]);
            sums[which][1][i] = __builtin_fmaf(g1[i] * r, x1[i], sums[which][1][i]);
            x0[i] = r * (w0[i] * g0[i] - x0[i] * back);
            x1[i] = r * (w1[i] * g1[i] - x1[i] * back);
          }
          if (there && a.gx[which]) {
            store<T, V>((T *)a.gx[which] + to + at0, x0);
            store<T, V>((T *)a.gx[which] + to + at1, x1);
          }
        }
      }
    }
  }
  if constexpr (BACKWARD) {
    if (!partial) return;
    // partial[workgroup][which][channel]: lanes of the same channels in a fixed order
    float *const all = reinterpret_cast<float *>(turn);      // [256 / lanes][dim]
    const int group = threadIdx.x / lanes, groups = 256 / lanes;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
      __syncthreads();
      if (there)
#pragma unroll
        for (int i = 0; i < V; ++i) all[group * a.dim + at0 + i] = sums[which][0][i], all[group * a.dim + at1 + i] = sums[which][1][i];
      __syncthreads();
      for (int d = threadIdx.x; d < a.dim; d += 256) {
        float sum = 0.f;
        for (int g = 0; g < groups; ++g) sum += all[g * a.dim + d];
        partial[((int64_t)blockIdx.x * 2 + which) * a.dim + d] = sum;
      }
    }
  }
}

// gscale[which][channel] = the workgroups' sums, eight channels a workgroup, 128 threads each.
template <typename T>
__global__ __launch_bounds__(1024) void scale_grad_kernel(const float *__restrict__ partial, int blocks, int dim, T *gq, T *gk) {
  __shared__ float part[16][8];
  const int c = threadIdx.x % 8, column = blockIdx.x * 8 + c, slice = threadIdx.x / 8;      // (dim is a multiple of 8)
  float sum = 0.f;
#pragma unroll 8
  for (int b = slice; b < blocks; b += 128) sum += partial[(int64_t)b * 2 * dim + column];
  for (int d = 8; d < 64; d *= 2) sum += __shfl_xor(sum, d);
  if (threadIdx.x % 64 < 8) part[threadIdx.x / 64][c] = sum;
  __syncthreads();
  if (threadIdx.x >= 8) return;
  sum = 0.f;
  for (int s = 0; s < 16; ++s) sum += part[s][c];
  T *const to = column < dim ? gq : gk;
  if (to) to[column % dim] = (T)sum;
}

template <typename T, int V, bool NEXT, bool BACKWARD>
int launch(const NormRotaryArgs &a) {
  int lanes = 1;
  while (lanes * V < a.dim / 2) lanes *= 2;
  // Rows to a tile: four heads a lane group and tile, fewer where the tiles would not fill the chip.
  const int heads = a.heads[0] + a.heads[1], at_once = 256 / lanes;
  int64_t tile = (4 * at_once + heads - 1) / heads;
  const int64_t even = a.n / (4 * num_cus());
  tile = tile < even ? tile : even;
  tile = tile < 1 ? 1 : tile > 32 ? 32 : tile;
  int64_t blocks = (a.n + tile - 1) / tile;
  float *partial = nullptr;
  size_t lds = (size_t)tile * (a.dim / 2) * sizeof(float2);
  const bool scales = BACKWARD && (a.gscale[0] || a.gscale[1]);
  std::optional<StreamTurn> turn;
  if (scales) turn.emplace(a.stream);
  if (BACKWARD) {
    const int64_t most = 4 * num_cus();      // (each leaves sums behind)
    blocks = blocks < most ? blocks : most;
    if (scales) {
      const int rc = workspace_get(a.stream, kSlotScaleSums, (size_t)blocks * 2 * a.dim * sizeof(float), (void **)&partial);
      if (rc != FGMS_OK) return rc;
      const size_t need = (size_t)at_once * a.dim * sizeof(float);
      lds = lds > need ? lds : need;
    }
  }
  if (blocks > 0x7fffffff) {
    set_error("norm and rotation: %lld rows are more than one launch takes", (long long)a.n);
    return FGMS_E_INVALID;
  }
  norm_rotary_kernel<T, V, NEXT, BACKWARD><<<(unsigned)blocks, 256, lds, a.stream>>>(a, (int)tile, lanes, partial);
  if (scales) scale_grad_kernel<T><<<2 * a.dim / 8, 1024, 0, a.stream>>>(partial, (int)blocks, a.dim, (T *)a.gscale[0], (T *)a.gscale[1]);
  FGMS_HIP_TRY(hipGetLastError());
  return FGMS_OK;
}

template <typename T, int V>
int launch_vec(const NormRotaryArgs &a, bool backward) {
  if (a.interleaved) return backward ? launch<T, V, true, true>(a) : launch<T, V, true, false>(a);
  return backward ? launch<T, V, false, true>(a) : launch<T, V, false, false>(a);
}

// 16 bytes a load, eight where half a head is no whole number of those.
template <typename T>
int launch_type(const NormRotaryArgs &a, bool backward) {
  if constexpr (sizeof(T) == 2)
    if (a.dim % 16 == 0) return launch_vec<T, 8>(a, backward);
  return launch_vec<T, 4>(a, backward);
}

}  // namespace

int launch_norm_rotary(const NormRotaryArgs &a, bool backward) {
  return a.dtype == FGMS_F32 ? launch_type<float>(a, backward)
         : a.dtype == FGMS_F16 ? launch_type<_Float16>(a, backward) : launch_type<__bf16>(a, backward);
}

}  // namespace fgms
