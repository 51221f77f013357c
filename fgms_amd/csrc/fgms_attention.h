// Attention over ragged segments: arguments, and the pieces its kernels share.
//
// A segment is a range of rows of q and a range of rows of k and v (a window of a cloud, a scan, a cache);
// where they begin is read on the device, so that no size comes back to the host.  Query heads come in
// groups of `group` that share a key head.  For one segment and key head the queries of a group are
// group * Lq rows of one matrix, row r being head r % group of token r / group: the keys are then read once
// for the whole group, and a single new token still fills several rows of a tile.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "fgms_internal.h"
#include "fgms_mma.h"

namespace fgms {

struct AttentionArgs {
  const void *q, *k, *v;
  const int32_t *q_offsets, *k_offsets, *k_lengths;      // [segments + 1], [segments + 1], [segments] or nullptr
  int n_q, n_k;
  int segments, heads, kv_heads, dim;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;   // strides in elements
  float scale;
  int causal;
  int dtype;
  hipStream_t stream;
  // forward: written; backward: read
  void *out;             // [n_q, heads, dim]
  float *lse;            // [n_q, heads]: log of the row's sum of exponentials, -inf for a row without keys
  // backward
  const void *g_out;     // [n_q, heads, dim]
  float *delta;          // [n_q, heads]: g_out . out
  void *gq, *gk, *gv;    // contiguous, any of them may be nullptr
  int slots;             // tiles of each key head
  bool by_xcd;           // order of the workgroups (place_of)
  // a long axis cut into `parts` pieces, joined by a second launch
  int parts;
  float *part_sum;       // [slot][kv head][part][tile row][dim]
  float *part_lse;       // [slot][kv head][part][tile row]
};

int launch_attention_fwd(AttentionArgs a);
int launch_attention_bwd(AttentionArgs a);
// For one type (fgms_attention_f16.hip, _bf16.hip, _f32.hip).
template <typename T> int attention_fwd(const AttentionArgs &a);
template <typename T> int attention_bwd(const AttentionArgs &a);

// Tiles of `rows` rows, numbered segment by segment without their lengths being known: segment s begins at slot
// offset[s] / rows + s, which leaves it ceil(length / rows) slots at least; a slot behind its segment's last row has
// nothing to do.  Rows behind the last segment are a segment of their own (number `segments`), without partners.
__host__ __device__ inline int64_t attention_slots(int64_t n, int64_t segments, int rows) { return n / rows + segments + 1; }

#ifdef __HIPCC__

// Row at which segment s begins, whatever stands in the offsets.  (One load for any s, and no branch around it.)
__device__ __forceinline__ int segment_begin(const int32_t *__restrict__ offsets, int s, int segments, int n) {
  const int at = offsets[min(max(s, 0), segments)];
  return s <= 0 ? 0 : s > segments ? n : min(max(at, 0), n);
}

// A value that the compiler does not know to be the wave's: what follows from it goes to the scalar unit (and a buffer's address that does
// not is looped over lane by lane).
__device__ __forceinline__ int same_for_all(int v) { return __builtin_amdgcn_readfirstlane(v); }

struct Slot {
  int segment;
  int begin, tokens;      // the segment's rows in the tensor
  int length;             // ... in the tile's matrix: times `group`
  int first;              // the tile's first row, in the segment
};

// x / by for 0 <= x < 2^22, from by's reciprocal: (x + 1/2) / by is at least 1 / (2 by) from a whole number, and the product off by
// less than (x + 1/2) 2^-23 / by.
__device__ __forceinline__ int divide(int x, float reciprocal) { return (int)(((float)x + 0.5f) * reciprocal); }

// The slot's segment: 64 of them are asked at a time, first those around the place it has if all are of one length (windows of a cloud are
// near enough: one round of loads), then by steps.  `group`: rows of the matrix to a row of the tensor; all rows of the tensor times
// `group` are less than 2^31.  Whatever stands in the offsets, the segment found is one that begins at or before the slot.
__device__ __forceinline__ Slot find_slot(const int32_t *__restrict__ offsets, int segments, int n, int group, int rows, int slot, int slots) {
  const int lane = threadIdx.x % 64;
  // segments [lo, hi) are in question, and lo begins at or before the slot
  int lo = 0, hi = segments + 1, step = 1;
  int first = (int)((float)slot * (float)hi / (float)slots) - 32;
  first = max(min(first, hi - 64), 0);
  int count, value;
  for (;;) {
    const int at = (int)min((unsigned)first + (unsigned)lane * (unsigned)step, (unsigned)hi);
    value = segment_begin(offsets, at, segments, n);
    const unsigned long long after = ~__builtin_amdgcn_ballot_w64(at < hi && value * group / rows + at <= slot);
    count = after ? __builtin_ctzll(after) : 64;
    if (count == 0) {      // (all behind the slot: only if the first guess was)
      hi = first;
      first = lo;
    } else {
      lo = first + (count - 1) * step;
      hi = count < 64 ? min(hi, lo + step) : hi;
      if (hi - lo <= 1 && step == 1) break;
      first = lo;
    }
    step = (int)(((unsigned)(hi - lo) + 63u) / 64u);
  }
  Slot r;
  r.segment = same_for_all(lo);
  r.begin = __builtin_amdgcn_readlane(value, count - 1);
  const int end = count < 64 ? __builtin_amdgcn_readlane(value, count) : same_for_all(segment_begin(offsets, r.segment + 1, segments, n));
  r.tokens = max(end - r.begin, 0);
  r.length = r.tokens * group;
  r.first = (slot - (r.begin * group / rows + r.segment)) * rows;
  return r;
}

// The rows of the other side that go with segment s.
__device__ __forceinline__ void partner_rows(const int32_t *__restrict__ offsets, const int32_t *__restrict__ lengths, int s,
                                             int segments, int n, int &begin, int &length) {
  begin = same_for_all(segment_begin(offsets, s, segments, n));
  const int end = same_for_all(segment_begin(offsets, s + 1, segments, n));
  length = s < segments && end > begin ? end - begin : 0;
  if (lengths && s < segments) length = min(max(same_for_all(lengths[s]), 0), length);
}

// acc += a x b, 16 bytes of the contracted axis a lane: 16 deep for 16-bit types, 8 for float.
template <typename T>
__device__ __forceinline__ void multiply(float16v &acc, const int4v &a, const int4v &b) {
  if constexpr (__is_same(T, _Float16)) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8, a), __builtin_bit_cast(half8, b), acc, 0, 0, 0);
  } else if constexpr (__is_same(T, __bf16)) {
    acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), acc, 0, 0, 0);
  } else {
    const float4v fa = __builtin_bit_cast(float4v, a), fb = __builtin_bit_cast(float4v, b);
#pragma unroll
    for (int e = 0; e < 4; ++e) acc = __builtin_amdgcn_mfma_f32_32x32x2f32(fa[e], fb[e], acc, 0, 0, 0);
  }
}

// A tile of rows in LDS, DP channels each, in 16-byte chunks.  A fragment of rows is read by 32 lanes that ask 32 rows
// for the same chunk, one of columns (16-bit types: the transposing read) by 16 lanes that ask four rows for four chunks,
// two rows' worth beside it.  Chunk c of a row lies at c ^ swizzle(row): both kinds then cover all banks, the first over 16 rows,
// the second over its four (rows of 256 bytes: the row's lowest two bits move groups of four chunks, the next two the chunks
// in them; of 128, or 384: bit 1 moves groups, as two rows share 256 bytes; of 64, or 192: the groups move by themselves).
template <typename T, int DP>
struct RowTile {
  static constexpr int E = 16 / (int)sizeof(T), CH = DP / E;
  static __device__ __forceinline__ int swizzle(int row) {
    if constexpr (CH % 16 == 0) return ((row & 3) << 2) | ((row >> 2) & 3);
    else if constexpr (CH % 8 == 0) return ((row & 2) << 1) | ((row >> 2) & 3);
    else return (row >> 2) & 3;
  }
  static __device__ __forceinline__ int at(int row, int c) { return row * CH + (c ^ swizzle(row)); }

  // Where a lane reads, in bytes from a tile's first row: a tile's own place, and rows by 16s, go into the instructions.
  static constexpr int STEPS = CH / 2, BLOCKS = DP / 32, COLUMNS = sizeof(T) == 2 ? 2 * BLOCKS : 8;
  int row_at[STEPS], column_at[COLUMNS];
  __device__ __forceinline__ void aim(int lane) {
#pragma unroll
    for (int i = 0; i < STEPS; ++i) row_at[i] = at(lane % 32, 2 * i + lane / 32) * 16;
    if constexpr (sizeof(T) == 2) {
      const int i = lane & 15, row = 4 * (lane >> 5) + (i >> 2), c = ((lane >> 4) & 1) * 2 + ((i & 3) >> 1);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) {
        column_at[2 * b] = at(row, 4 * b + c) * 16 + (i & 1) * 8;
        column_at[2 * b + 1] = at(row + 8, 4 * b + c) * 16 + (i & 1) * 8;
      }
    } else {
      const int col = (BLOCKS == 3 ? 1 : BLOCKS) * (lane % 32);
#pragma unroll
      for (int r = 0; r < 8; ++r) column_at[r] = at(8 * (r / 4) + 4 * (lane / 32) + r % 4, col / 4) * 16 + col % 4 * 4;
    }
  }
  template <typename V>
  static __device__ __forceinline__ V read(const int4v *tile, int from, int bytes) {
    typedef __attribute__((address_space(3))) const char lds_char;
    typedef __attribute__((address_space(3))) const V lds_v;
    return *(lds_v *)((lds_char *)tile + from + bytes);
  }
  // operand with the tile's rows as its outer index: lane l has row row0 + l % 32, chunk 2 * step + l / 32
  __device__ __forceinline__ int4v rows(const int4v *tile, int row0, int step) const { return read<int4v>(tile, row_at[step], row0 * CH * 16); }
  // 16-bit types: operand with the tile's columns as its outer index, contracted over its rows: lane l has column
  // 32 b + l % 32 of rows row0 + 4 * (l / 32) + {0 .. 3} and, 8 further down, four more -- the rows whose products the
  // accumulator registers 8 i .. 8 i + 7 of that lane hold, so that these are the other operand as they are
  __device__ __forceinline__ int4v columns(const int4v *tile, int row0, int b) const {
    typedef short short4v __attribute__((ext_vector_type(4)));
    typedef short short8v __attribute__((ext_vector_type(8)));
    typedef __attribute__((address_space(3))) const char lds_char;
    typedef __attribute__((address_space(3))) short4v lds_v4;
    const short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4 *)((lds_char *)tile + column_at[2 * b] + row0 * CH * 16));
    const short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4 *)((lds_char *)tile + column_at[2 * b + 1] + row0 * CH * 16));
    const short8v v = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    return __builtin_bit_cast(int4v, v);
  }
  // float: channels BLOCKS * (l % 32) + {0 .. BLOCKS - 1}, one for each block of 32, of the row whose product register r holds (three
  // blocks: 32 b + l % 32, as three floats in a row may lie in two chunks)
  __device__ __forceinline__ void channels(float (&to)[BLOCKS], const int4v *tile, int row0, int r) const {
    typedef float V __attribute__((ext_vector_type(BLOCKS)));
    if constexpr (BLOCKS == 1 || BLOCKS == 3) {
      // (32 channels on: eight chunks, which the swizzle of such rows leaves alone)
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) to[b] = read<float>(tile, column_at[r % 8], (row0 + r / 8 * 16) * CH * 16 + b * 128);
    } else {
      const V v = read<V>(tile, column_at[r % 8], (row0 + r / 8 * 16) * CH * 16);
#pragma unroll
      for (int b = 0; b < BLOCKS; ++b) to[b] = v[b];
    }
  }
};

// out[channel][lane's row] += sum over 32 rows of the tile from row0 on of tile[row][channel] * w[row][lane's row]; w as an
// accumulator holds it (register r of lane l: row 8 (r / 4) + 4 (l / 32) + r % 4, column l % 32), rounded to T.  Which channels the rows
// of out[b] are is free: 32 b + {0 .. 31} with the transposing read; float takes DP / 32 neighbouring ones a lane in one read (96: as 16-bit types).
template <typename T, int DP>
__device__ __forceinline__ void add_weighted_rows(float16v (&out)[DP / 32], const RowTile<T, DP> &at, const int4v *tile, int row0, const float16v &w) {
  if constexpr (sizeof(T) == 2) {
    typedef T T8 __attribute__((ext_vector_type(8)));
    typedef float float8v __attribute__((ext_vector_type(8)));
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float8v part = {w[8 * i], w[8 * i + 1], w[8 * i + 2], w[8 * i + 3], w[8 * i + 4], w[8 * i + 5], w[8 * i + 6], w[8 * i + 7]};
      const int4v b = __builtin_bit_cast(int4v, __builtin_convertvector(part, T8));
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) multiply<T>(out[db], at.columns(tile, row0 + 16 * i, db), b);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float rows[DP / 32];
      at.channels(rows, tile, row0, r);
#pragma unroll
      for (int db = 0; db < DP / 32; ++db) out[db] = __builtin_amdgcn_mfma_f32_32x32x2f32(rows[db], w[r], out[db], 0, 0, 0);
    }
  }
}

// The larger of / the sum over lanes l and l ^ 32.
__device__ __forceinline__ float both_max(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return __builtin_fmaxf(__builtin_bit_cast(float, (unsigned)r[0]), __builtin_bit_cast(float, (unsigned)r[1]));
}
__device__ __forceinline__ float both_sum(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return __builtin_bit_cast(float, (unsigned)r[0]) + __builtin_bit_cast(float, (unsigned)r[1]);
}
// Lane l % 32 + 32's.
__device__ __forceinline__ float of_upper(float v) {
  const auto r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), __builtin_bit_cast(unsigned, v), false, false);
  return __builtin_bit_cast(float, (unsigned)r[1]);
}

// Row `row` (or nullptr) of `dim` channels into fragments, zeros where there is nothing.
template <typename T, int DP>
__device__ __forceinline__ void load_row(int4v (&to)[DP / (32 / (int)sizeof(T))], const T *row, int dim, int lane) {
  constexpr int E = 16 / (int)sizeof(T);
#pragma unroll
  for (int s = 0; s < DP / (2 * E); ++s) {
    const int c = (2 * s + lane / 32) * E;
    to[s] = row && c < dim ? *reinterpret_cast<const int4v *>(row + c) : int4v{0, 0, 0, 0};
  }
}

// A lane's row of a result, from accumulators of T's products that hold it as columns, times `by`.
template <typename T, typename To, int DP>
__device__ __forceinline__ void store_row(To *row, const float16v (&acc)[DP / 32], float by, int dim, int lane) {
  if constexpr (sizeof(T) == 2 || DP == 96) {
    typedef To To4 __attribute__((ext_vector_type(4)));
#pragma unroll
    for (int db = 0; db < DP / 32; ++db)
#pragma unroll
      for (int p = 0; p < 4; ++p) {
        const int c = db * 32 + 8 * p + 4 * (lane / 32);
        const float4v v = {acc[db][4 * p] * by, acc[db][4 * p + 1] * by, acc[db][4 * p + 2] * by, acc[db][4 * p + 3] * by};
        if (c < dim) *reinterpret_cast<To4 *>(row + c) = __builtin_convertvector(v, To4);
      }
  } else {
    // four rows of all blocks: 4 * DP / 32 neighbouring channels, of which dim, a multiple of 8, may end inside
#pragma unroll
    for (int p = 0; p < 4; ++p)
#pragma unroll
      for (int e = 0; e < DP / 32; ++e) {
        const int first = 4 * e, c = DP / 32 * (8 * p + 4 * (lane / 32)) + first;
        float4v v;
#pragma unroll
        for (int i = 0; i < 4; ++i) v[i] = acc[(first + i) % (DP / 32)][4 * p + (first + i) / (DP / 32)] * by;
        if (c < dim) *reinterpret_cast<float4v *>(row + c) = v;
      }
  }
}

template <int N> struct Number { static constexpr int value = N; };

constexpr float kLog2e = 1.4426950408889634f;

#endif

}  // namespace fgms
