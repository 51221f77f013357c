// The attention kernels, for one type (included by fgms_attention_f16.hip, _bf16.hip and _f32.hip).
#pragma once

#include "fgms_attention.h"
#include "fgms_device.h"

namespace fgms {
namespace {

// Channels of a tile in LDS, heads of up to DP: the products whose columns these are come in 32s (heads of up to 16 are contracted over 16).
template <int DP> constexpr int tile_width() { return DP < 32 ? 32 : DP; }
// Keys (queries in the keys' gradients) to a tile: 64 where the four of them then take no more than 16 KB of LDS a wave.
template <typename T, int DP, int NW> constexpr int tile_rows() { return sizeof(T) == 4 || 64 * tile_width<DP>() / NW > 2048 ? 32 : 64; }

// Waves to a SIMD that the registers are to leave room for.
template <typename T, int DP> constexpr int waves_of_queries() { return (DP <= 32 ? 4 : DP == 64 ? 3 : 2) - (sizeof(T) == 4 ? 1 : 0); }
template <typename T, int DP> constexpr int waves_of_keys() { return sizeof(T) == 4 ? (DP >= 96 ? 1 : 2) : DP <= 32 ? 3 : DP == 128 ? 1 : 2; }

// 16 bytes a lane from a buffer to LDS, one lane's behind the other's from `to` on (the same for all lanes).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, int4v *to, unsigned offset) {
  typedef __attribute__((address_space(3))) void lds_any;
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (lds_any *)to, 16, offset, 0, 0, 0);
}

// Rows of a strided tensor on their way to a tile in LDS, past the registers: every lane asks for the chunk that belongs where
// its 16 bytes land.  Chunks behind the channels, and rows behind the last, are out of the buffer's range and arrive as zeros.
// (KEEP: chunks behind the channels stay as they are.)
template <typename T, int DP, int ROWS, int NW, bool KEEP = false>
struct Stager {
  using Rows = RowTile<T, DP>;
  static constexpr int PER = ROWS * Rows::CH / (64 * NW);
  const char *base;
  int64_t stride;              // bytes
  unsigned offset[PER];
  // (`like`: the other tensor's, whose lanes ask for the same places if its rows lie as far apart)
  template <bool K2 = KEEP>
  __device__ __forceinline__ void open(const T *from, int64_t row_stride, int dim, int wave, int lane, const Stager<T, DP, ROWS, NW, K2> *like = nullptr) {
    base = (const char *)from;
    stride = row_stride * (int)sizeof(T);
    if (like && like->stride == stride) {
#pragma unroll
      for (int i = 0; i < PER; ++i) offset[i] = like->offset[i];
      return;
    }
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (wave + i * NW) * 64 + lane, row = e / Rows::CH, c = (e % Rows::CH) ^ Rows::swizzle(row);
      offset[i] = c * Rows::E < dim ? (unsigned)row * (unsigned)stride + c * 16 : kAbsentRow;
    }
  }
  // rows [first, first + ROWS) of `count`
  __device__ __forceinline__ void load(int4v *tile, int first, int count, int wave) const {
    const int there = same_for_all(min(max(count - first, 0), ROWS));
    const __amdgpu_buffer_rsrc_t rows = rows_resource(base + first * stride, (unsigned)there * (unsigned)stride);
#pragma unroll
    for (int i = 0; i < PER; ++i)
      if (!KEEP || offset[i] != kAbsentRow) load_to_lds(rows, tile + (wave + i * NW) * 64, offset[i]);
  }
};

// Everything asked for has landed, for all waves.
__device__ __forceinline__ void tiles_ready() {
  __builtin_amdgcn_s_waitcnt(0x0f70);      // vmcnt(0)
  __syncthreads();
}

// Where a launch's workgroup stands: the heads of a tile one after the other, tiles with most partners where the order is causal first (the
// last queries, the first keys): workgroups start in this order, and the long ones are then not the last to end.  (Three causal scans
// of 12 k rows together, 16 heads of 64, both passes: 619 us; head by head, as few of them share the L2s then, 795.)
// Short segments: the heads of a tile share lines of memory (a row's heads lie side by side), so they and three neighbouring tiles go
// to one XCD (workgroup b runs on XCD b mod 8); not where that leaves XCDs without work.
struct Place {
  int slot, kv_head, part;
};
constexpr int kPlaceTiles = 4;
template <bool LAST_FIRST = true>
__device__ __forceinline__ Place place_of(unsigned block, int kv_heads, int parts, bool by_xcd, int slots) {
  Place p;
  p.part = (int)(block % parts);
  block /= parts;
  if (by_xcd) {
    const unsigned per = kPlaceTiles * kv_heads, i = block / 8;
    block = (i / per * 8 + block % 8) * per + i % per;
  }
  p.kv_head = (int)(block % kv_heads);
  p.slot = (int)(block / kv_heads);
  if (LAST_FIRST && p.slot < slots) p.slot = slots - 1 - p.slot;
  return p;
}

// --- forward --------------------------------------------------------------------------------------------------
// A wave holds 32 query rows as columns: scores come out of the matrix unit transposed (keys down the registers, a query a
// lane and its partner 32 lanes on), so that a row's maximum and sum are taken inside two lanes, and the exponentials are
// the right operand of the second product as they stand, with no exchange between lanes.  Tiles of keys and values pass through
// two pairs of buffers: the next one is on its way while this one is worked on.  ONES: a head has fewer channels than the tile (16-bit types);
// the values' last column then holds ones, and the rows' sums come out of the second product, a sixth of the vector instructions less
// (of the probabilities as rounded for it, so that a row's weights add up to one).
// 16/4 heads of 128, two causal scans of 24 k rows together, bf16: 1.33 to 1.38 ms, 1.10 to 1.14 PFLOP/s where a large library product has 1.14; 16
// heads of 64 over three of 12 k together 142 us, 815 TFLOP/s: the vector pipe is busy 75 % of the time, the matrix pipe 46 % (heads of 128: 54 %
// and 65 %; an exponential takes two turns).  Windows of 160 voxels on average, 4 heads of 16, 200 k voxels: 64 us, 20 for its bytes.
template <typename T, int DP, int NW, bool PARTS, bool ONES>
__global__ __launch_bounds__(NW * 64, (waves_of_queries<T, DP>())) void segment_attention_kernel(const AttentionArgs a) {
  constexpr int W = tile_width<DP>(), NK = tile_rows<T, DP, NW>(), STEPS = DP / (32 / (int)sizeof(T)), T_ROWS = 32 * NW;
  using Rows = RowTile<T, W>;
  __shared__ int4v k_tile0[NK * Rows::CH], v_tile0[NK * Rows::CH], k_tile1[NK * Rows::CH], v_tile1[NK * Rows::CH];
  const int lane = threadIdx.x % 64, wave = same_for_all(threadIdx.x / 64), group = a.heads / a.kv_heads;
  Rows rows_at;
  rows_at.aim(lane);
  const Place at = place_of(blockIdx.x, a.kv_heads, PARTS ? a.parts : 1, a.by_xcd, a.slots);
  if (at.slot >= a.slots) return;
  const Slot slot = find_slot(a.q_offsets, a.segments, a.n_q, group, T_ROWS, at.slot, a.slots);
  int k_begin, k_count;
  partner_rows(a.k_offsets, a.k_lengths, slot.segment, a.segments, a.n_k, k_begin, k_count);
  if (slot.first >= slot.length) return;
  const int ahead = k_count - slot.tokens;      // the last query sees the last key

  // keys that the rows see: those below `seen` for this lane's, of the workgroup's rows the last sees most, of a wave's the first least
  const int token0 = group == 1 ? slot.first : slot.first / group, head0 = slot.first - token0 * group;      // the tile's first row
  const float per_group = 1.f / group;
  const auto token_of = [&](int local) { return token0 + divide(head0 + local, per_group); };
  const int local = wave * 32 + lane % 32, token = token_of(local), head = at.kv_head * group + head0 + local - (token - token0) * group;
  const bool mine = slot.first + local < slot.length;
  const bool awake = slot.first + wave * 32 < slot.length;
  const int last = min(T_ROWS, slot.length - slot.first) - 1, wave_last = min(wave * 32 + 31, last);
  int begin = 0, end = a.causal ? min(k_count, token_of(last) + ahead + 1) : k_count;
  if constexpr (PARTS) {
    const int piece = ((max(end, 0) + a.parts - 1) / a.parts + NK - 1) / NK * NK;      // (of the keys that are seen)
    begin = at.part * piece;
    end = min(end, begin + piece);
  }
  const int seen = a.causal ? min(k_count, token + ahead + 1) : k_count;
  const int whole = min(end, a.causal ? token_of(wave * 32) + ahead + 1 : k_count);
  const int wave_end = same_for_all(!awake ? begin : a.causal ? min(end, token_of(wave_last) + ahead + 1) : end);

  Stager<T, W, NK, NW> k;
  k.open((const T *)a.k + k_begin * a.k_row + at.kv_head * a.k_head, a.k_row, a.dim, wave, lane);
  Stager<T, W, NK, NW, ONES> v;
  v.open((const T *)a.v + k_begin * a.v_row + at.kv_head * a.v_head, a.v_row, a.dim, wave, lane, &k);
  if (begin < end) {
    k.load(k_tile0, begin, k_count, wave);
    v.load(v_tile0, begin, k_count, wave);
  }
  if constexpr (ONES) {
    // (chunks behind the channels: zeros, and a one at the end of a row; no load touches them)
    const int4v last = {0, 0, 0, (int)((unsigned)__builtin_bit_cast(unsigned short, (T)1.f) << 16)};
    for (int row = threadIdx.x; row < NK; row += 64 * NW)
      for (int c = a.dim / Rows::E; c < Rows::CH; ++c) v_tile0[Rows::at(row, c)] = v_tile1[Rows::at(row, c)] = c == Rows::CH - 1 ? last : int4v{0, 0, 0, 0};
  }
  int4v q[STEPS];
  load_row<T, DP>(q, mine ? (const T *)a.q + (slot.begin + token) * a.q_row + head * a.q_head : nullptr, a.dim, lane);

  const float by = a.scale * kLog2e;
  const float inf = __builtin_inff();
  // of the scores so far, times `by`: a number that none exceeds by more than kSlack, -inf before the first (and what is subtracted from them).
  // fp16 holds the probabilities times 2^7: they grow to 2^15 within the slack, and half a step of the smallest is 2^-32 of the largest instead
  // of 2^-25 (of 65 k keys beside one that is 2^25 times each, 0.2 % of the row).
  constexpr float kSlack = 8.f, kUp = __is_same(T, _Float16) ? 7.f : 0.f;
  float most = -inf, base = 0.f, sum = 0.f;
  float16v o[W / 32] = {};
  // KB blocks of 32 keys, all seen by all rows or not
  const auto take = [&](auto blocks, auto masked, const int4v *k_tile, const int4v *v_tile, int j) __attribute__((always_inline)) {
    constexpr int KB = decltype(blocks)::value;
    float16v s[KB] = {};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int i = 0; i < STEPS; ++i)
        if (sizeof(T) == 2 || i * 2 * Rows::E < a.dim) multiply<T>(s[kb], rows_at.rows(k_tile, kb * 32, i), q[i]);
    if constexpr (decltype(masked)::value != 0) {
      const int left = seen - j - 4 * (lane / 32);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[kb][r] = left > kb * 32 + 8 * (r / 4) + r % 4 ? s[kb][r] : -inf;
    }
    float top = s[0][0];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, s[kb][r]);
    top = both_max(top) * by;
    // a new maximum is taken only where the old one is left behind by 2^8, which fp32 sums and 16-bit probabilities bear
    if (__builtin_amdgcn_ballot_w64(top > most + kSlack)) {
      const bool mine = top > most + kSlack;
      const float keep = mine ? __builtin_amdgcn_exp2f(most - top) : 1.f;
      most = mine ? top : most;
      base = mine ? top - kUp : base;
      if constexpr (!ONES) sum *= keep;
#pragma unroll
      for (int db = 0; db < W / 32; ++db) o[db] *= keep;
    }
    float add[2] = {0.f, 0.f};
#pragma unroll
    for (int kb = 0; kb < KB; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], by, -base));
        if constexpr (!ONES) add[r % 2] += s[kb][r];
      }
    if constexpr (!ONES) sum += add[0] + add[1];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) add_weighted_rows<T, W>(o, rows_at, v_tile, kb * 32, s[kb]);
  };
  const auto load_next = [&](int4v *k_next, int4v *v_next, int j) __attribute__((always_inline)) {
    tiles_ready();
    if (j + NK < end) {
      k.load(k_next, j + NK, k_count, wave);
      v.load(v_next, j + NK, k_count, wave);
    }
  };
  const auto all_of = [&](const int4v *k_tile, const int4v *v_tile, int4v *k_next, int4v *v_next, int j) __attribute__((always_inline)) {
    load_next(k_next, v_next, j);
    take(Number<NK / 32>(), Number<0>(), k_tile, v_tile, j);
  };
  const auto some_of = [&](const int4v *k_tile, const int4v *v_tile, int4v *k_next, int4v *v_next, int j) __attribute__((always_inline)) {
    load_next(k_next, v_next, j);
    if (NK == 64 && j + 32 < wave_end) take(Number<NK / 32>(), Number<1>(), k_tile, v_tile, j);
    else if (j < wave_end) take(Number<1>(), Number<1>(), k_tile, v_tile, j);
  };
  // Tiles that all rows of the wave see whole have a loop of their own: with a choice in it the accumulators are moved from
  // registers to registers at its end, which waits for their last product.
  int j = begin;
  const int all_end = same_for_all(begin + max(min(whole, wave_end) - begin, 0) / NK * NK);
  bool second = false;      // whose turn it is
  while (j < all_end) {
    all_of(k_tile0, v_tile0, k_tile1, v_tile1, j);
    j += NK;
    second = j >= all_end;
    if (second) break;
    all_of(k_tile1, v_tile1, k_tile0, v_tile0, j);
    j += NK;
  }
  for (; j < end; j += NK) {
    if (second) some_of(k_tile1, v_tile1, k_tile0, v_tile0, j);
    else some_of(k_tile0, v_tile0, k_tile1, v_tile1, j);
    second = !second;
  }

  // (the last column's products: row 31 of the last block, register 15 of the upper lanes)
  sum = ONES ? of_upper(o[W / 32 - 1][15]) : both_sum(sum);
  const bool none = sum == 0.f;      // no key for this row (here), or none with a score above -inf: the largest adds one or more
  const float inverse = none ? 0.f : 1.f / sum;
  if (a.causal && __builtin_amdgcn_ballot_w64(none))      // (zeros, whatever values of the tile they were multiplied with)
#pragma unroll
    for (int db = 0; db < W / 32; ++db) o[db] = none ? float16v{} : o[db];
  const float lse = none ? -inf : (base + __builtin_log2f(sum)) * (1.f / kLog2e);
  if constexpr (PARTS) {
    const int64_t tile = (((int64_t)at.slot * a.kv_heads + at.kv_head) * a.parts + at.part) * T_ROWS + local;
    if (mine && !none) store_row<T, float, W>(a.part_sum + tile * a.dim, o, inverse, a.dim, lane);
    if (mine && lane < 32) a.part_lse[tile] = lse;
  } else if (mine) {
    const int64_t to = (int64_t)(slot.begin + token) * a.heads + head;
    store_row<T, T, W>((T *)a.out + to * a.dim, o, inverse, a.dim, lane);
    if (a.lse && lane < 32) a.lse[to] = lse;
  }
}

// --- joining the parts -----------------------------------------------------------------------------------------
// SUMS: the parts add up (gradients); else they are averages over their keys, to be weighted by their sums of exponentials.  A workgroup
// has eight rows of a tile: the parts' weights first, then a thread four channels of a row, eight parts under way at a time.
// (38 parts of 64 tiles, heads of 128: 13 us.)
constexpr int kMostParts = 256, kJoinRows = 8;
template <typename T, int NW, bool SUMS>
__global__ __launch_bounds__(256) void join_parts_kernel(const AttentionArgs a, const int32_t *__restrict__ offsets, int n, int group,
                                                         const float *__restrict__ sums, T *__restrict__ out) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  constexpr int T_ROWS = 32 * NW;
  __shared__ float weight[kJoinRows][kMostParts + 1];      // (rows in different banks)
  const int per_row = a.dim / 4;
  const Place at = place_of<false>(blockIdx.x, a.kv_heads, T_ROWS / kJoinRows, false, a.slots);      // (its rows: a part of the tile)
  const Slot slot = find_slot(offsets, a.segments, n, group, T_ROWS, at.slot, a.slots);
  const int row0 = at.part * kJoinRows, rows = min(kJoinRows, slot.length - slot.first - row0);
  if (rows <= 0) return;
  const int64_t first = ((int64_t)at.slot * a.kv_heads + at.kv_head) * a.parts * T_ROWS + row0;
  const auto place = [&](int local) {
    const int row = slot.first + row0 + local;
    return ((int64_t)(slot.begin + row / group) * a.kv_heads + at.kv_head) * group + row % group;
  };
  if constexpr (!SUMS) {
    // eight threads a row
    const int local = threadIdx.x / 8, lane = threadIdx.x % 8;
    const float inf = __builtin_inff();
    float most = -inf, total = 0.f;
    if (local < rows)
      for (int p = lane; p < a.parts; p += 8) {
        const float lse = a.part_lse[first + (int64_t)p * T_ROWS + local];
        weight[local][p] = lse;
        most = __builtin_fmaxf(most, lse);
      }
    for (int d = 1; d < 8; d *= 2) most = __builtin_fmaxf(most, __shfl_xor(most, d));
    if (local < rows)
      for (int p = lane; p < a.parts; p += 8) {
        // (a part without keys has nothing written)
        const float w = weight[local][p] == -inf ? 0.f : __builtin_amdgcn_exp2f((weight[local][p] - most) * kLog2e);
        weight[local][p] = w;
        total += w;
      }
    for (int d = 1; d < 8; d *= 2) total += __shfl_xor(total, d);
    const bool any = most != -inf || total != 0.f;      // (not a number: kept)
    if (local < rows) {
      for (int p = lane; p < a.parts; p += 8) weight[local][p] = any ? weight[local][p] / total : 0.f;
      if (a.lse && lane == 0) a.lse[place(local)] = any ? most + __builtin_log2f(total) * (1.f / kLog2e) : -inf;
    }
    __syncthreads();
  }
  for (int e = threadIdx.x; e < rows * per_row; e += 256) {
    const int local = e / per_row, c = e % per_row * 4;
    const float *const from = sums + (first + local) * a.dim + c;
    const int64_t step = (int64_t)T_ROWS * a.dim;
    float4v total = {0.f, 0.f, 0.f, 0.f};
    for (int p0 = 0; p0 < a.parts; p0 += 8) {
      float4v v[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool there = p0 + i < a.parts && (SUMS || weight[local][p0 + i] != 0.f);
        v[i] = there ? *reinterpret_cast<const float4v *>(from + (p0 + i) * step) : float4v{0.f, 0.f, 0.f, 0.f};
      }
#pragma unroll
      for (int i = 0; i < 8; ++i) total += SUMS ? v[i] : v[i] * (p0 + i < a.parts ? weight[local][p0 + i] : 0.f);
    }
    *reinterpret_cast<T4 *>(out + place(local) * a.dim + c) = __builtin_convertvector(total, T4);
  }
}

// --- backward -------------------------------------------------------------------------------------------------
// ds = p (g_out . v - delta) is rounded to T for its two products, p for its one.  In fp16 a power of two goes with them, taken out
// of the sums again: p is 1 / N in a row of N like keys and would lose bits from 2^-14 on, with 2^10 from 2^-24 on; ds has 2^4
// (steps of 2^-28; it may reach 4094).  Where ds reaches further, the sums of its row (its key) come out infinite or as no number in every
// channel; these rows alone are then formed again with 2^-11, and with 2^-26 where that is not enough, which bears the 2^40 of two
// products of 128 channels of 65504.  (Half a step of such a row is 2^-26 of its largest ds.)
template <typename T> constexpr int p_shift() { return __is_same(T, _Float16) ? 10 : 0; }
template <typename T> constexpr int ds_shift() { return __is_same(T, _Float16) ? 4 : 0; }
template <typename T> constexpr bool ds_shifted() { return ds_shift<T>() != 0; }
constexpr int kShiftDown = 15, kLeastShift = 4 - 2 * kShiftDown;
constexpr float pow2(int e) { return e >= 0 ? (float)(1 << e) : 1.f / (float)(1 << -e); }

// Whether a lane of the workgroup says so, by way of a tile that all waves are done with when they have come here (16 bytes of their own
// would leave room for a workgroup less on a CU).
template <int NW>
__device__ __forceinline__ bool any_lane(bool mine, int4v *tile) {
  const bool here = __builtin_amdgcn_ballot_w64(mine) != 0;
  if constexpr (NW == 1) return here;
  int *const says = (int *)tile;
  __syncthreads();
  if (threadIdx.x % 64 == 0) says[threadIdx.x / 64] = here;
  __syncthreads();
  int any = 0;
#pragma unroll
  for (int w = 0; w < NW; ++w) any |= says[w];
  return same_for_all(any) != 0;
}

// A round that forms rows again is a function of its own, so that nothing of it is kept while the first one runs (as a loop around that one
// it took 8 to 23 % of the gradients' time, in registers; as it is, 0 to 4).  It is given the kernel's arguments where they lie; what a call passes is the
// same for all lanes here, which the compiler has to be told again.
typedef __attribute__((address_space(4))) const AttentionArgs args_in_place;
template <typename E> using Lds = __attribute__((address_space(3))) E;
__device__ __forceinline__ AttentionArgs same_args(args_in_place *args) {
  const unsigned long long at = (unsigned long long)args;
  const unsigned lo = __builtin_amdgcn_readfirstlane((unsigned)at), hi = __builtin_amdgcn_readfirstlane((unsigned)(at >> 32));
  args_in_place *const there = (args_in_place *)((unsigned long long)hi << 32 | lo);
  AttentionArgs a;
  __builtin_memcpy(&a, (const AttentionArgs *)there, sizeof(a));
  return a;
}
template <typename E>
__device__ __forceinline__ E *same_tile(Lds<E> *p) {
  return (E *)(Lds<E> *)(uintptr_t)(unsigned)__builtin_amdgcn_readfirstlane((unsigned)(uintptr_t)p);
}

// delta = g_out . out of a lane's row, shared with its partner.
template <typename T, int DP>
__device__ __forceinline__ float row_delta(const int4v (&g)[DP / (32 / (int)sizeof(T))], const T *out, int dim, int lane) {
  constexpr int E = 16 / (int)sizeof(T), STEPS = DP / (2 * E);
  typedef T Te __attribute__((ext_vector_type(E)));
  int4v o[STEPS];
  load_row<T, DP>(o, out, dim, lane);
  float delta = 0.f;
#pragma unroll
  for (int i = 0; i < STEPS; ++i)
#pragma unroll
    for (int e = 0; e < E; ++e) delta = __builtin_fmaf((float)__builtin_bit_cast(Te, o[i])[e], (float)__builtin_bit_cast(Te, g[i])[e], delta);
  return both_sum(delta);
}

// All rows' delta, where the queries' gradient, which has them on its way, is not wanted.
template <typename T, int DP>
__global__ __launch_bounds__(256) void attention_delta_kernel(const T *__restrict__ g_out, const T *__restrict__ out,
                                                              float *__restrict__ delta, int64_t rows, int dim) {
  const int lane = threadIdx.x % 64;
  const int64_t row = (int64_t)blockIdx.x * 128 + threadIdx.x / 64 * 32 + lane % 32;
  int4v g[DP / (32 / (int)sizeof(T))];
  load_row<T, DP>(g, row < rows ? g_out + row * dim : nullptr, dim, lane);
  const float sum = row_delta<T, DP>(g, row < rows ? out + row * dim : nullptr, dim, lane);
  if (row < rows && lane < 32) delta[row] = sum;
}

// Queries' gradients.  As the forward kernel: a wave's 32 query rows are columns, so that a row's log-sum and delta are one value a lane,
// and ds the right operand of dq^T = k^T ds as it stands.  Three products (16 heads of 64, three causal scans of 12 k rows together, bf16:
// 178 us, 975 TFLOP/s); a kernel of its own and not a by-product of the keys' gradients, whose sums over key tiles would need atomics.
template <typename T, int DP, int NW, bool PARTS>
__device__ __forceinline__ bool query_grad_rows(const AttentionArgs &a, int4v *k_tile0, int4v *v_tile0, int4v *k_tile1, int4v *v_tile1,
                                                unsigned block, int shift, bool open) {
  constexpr int W = tile_width<DP>(), NK = tile_rows<T, DP, NW>(), STEPS = DP / (32 / (int)sizeof(T)), T_ROWS = 32 * NW;
  using Rows = RowTile<T, W>;
  const int lane = threadIdx.x % 64, wave = same_for_all(threadIdx.x / 64), group = a.heads / a.kv_heads;
  Rows rows_at;
  rows_at.aim(lane);
  const Place at = place_of(block, a.kv_heads, PARTS ? a.parts : 1, a.by_xcd, a.slots);
  if (at.slot >= a.slots) return false;
  const Slot slot = find_slot(a.q_offsets, a.segments, a.n_q, group, T_ROWS, at.slot, a.slots);
  int k_begin, k_count;
  partner_rows(a.k_offsets, a.k_lengths, slot.segment, a.segments, a.n_k, k_begin, k_count);
  if (slot.first >= slot.length) return false;
  const int ahead = k_count - slot.tokens;

  const int token0 = group == 1 ? slot.first : slot.first / group, head0 = slot.first - token0 * group;
  const float per_group = 1.f / group;
  const auto token_of = [&](int local) { return token0 + divide(head0 + local, per_group); };
  const int local = wave * 32 + lane % 32, token = token_of(local), head = at.kv_head * group + head0 + local - (token - token0) * group;
  const bool mine = slot.first + local < slot.length;
  const bool awake = slot.first + wave * 32 < slot.length;
  const int last = min(T_ROWS, slot.length - slot.first) - 1, wave_last = min(wave * 32 + 31, last);
  int begin = 0, end = a.causal ? min(k_count, token_of(last) + ahead + 1) : k_count;
  if constexpr (PARTS) {
    const int piece = ((max(end, 0) + a.parts - 1) / a.parts + NK - 1) / NK * NK;      // (of the keys that are seen)
    begin = at.part * piece;
    end = min(end, begin + piece);
  }
  const int seen = a.causal ? min(k_count, token + ahead + 1) : k_count;
  const int whole = min(end, a.causal ? token_of(wave * 32) + ahead + 1 : k_count);
  const int wave_end = same_for_all(!awake ? begin : a.causal ? min(end, token_of(wave_last) + ahead + 1) : end);

  Stager<T, W, NK, NW> k;
  k.open((const T *)a.k + k_begin * a.k_row + at.kv_head * a.k_head, a.k_row, a.dim, wave, lane);
  Stager<T, W, NK, NW> v;
  v.open((const T *)a.v + k_begin * a.v_row + at.kv_head * a.v_head, a.v_row, a.dim, wave, lane, &k);
  if (begin < end) {
    k.load(k_tile0, begin, k_count, wave);
    v.load(v_tile0, begin, k_count, wave);
  }
  const int64_t to = (int64_t)(slot.begin + token) * a.heads + head;
  int4v q[STEPS], g[STEPS];
  load_row<T, DP>(q, mine ? (const T *)a.q + (slot.begin + token) * a.q_row + head * a.q_head : nullptr, a.dim, lane);
  load_row<T, DP>(g, mine ? (const T *)a.g_out + to * a.dim : nullptr, a.dim, lane);
  const float inf = __builtin_inff();
  float lse = mine ? a.lse[to] : inf;
  lse = lse == -inf ? inf : lse * kLog2e - shift;      // (no keys: all probabilities 0)
  const float delta = row_delta<T, DP>(g, mine ? (const T *)a.out + to * a.dim : nullptr, a.dim, lane);
  if (mine && lane < 32 && (!PARTS || at.part == 0)) a.delta[to] = delta;      // (for the keys' gradients)

  const float by = a.scale * kLog2e;
  float16v dq[W / 32] = {};
  const auto take = [&](auto masked, const int4v *k_tile, const int4v *v_tile, int kb, int j) __attribute__((always_inline)) {
    float16v s = {}, dp = {};
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (sizeof(T) == 2 || i * 2 * Rows::E < a.dim) multiply<T>(s, rows_at.rows(k_tile, kb * 32, i), q[i]);
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (sizeof(T) == 2 || i * 2 * Rows::E < a.dim) multiply<T>(dp, rows_at.rows(v_tile, kb * 32, i), g[i]);
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], by, -lse)) * (dp[r] - delta);
    if constexpr (decltype(masked)::value != 0) {
      const int left = seen - j - kb * 32 - 4 * (lane / 32);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = left > 8 * (r / 4) + r % 4 ? s[r] : 0.f;
    }
    add_weighted_rows<T, W>(dq, rows_at, k_tile, kb * 32, s);
  };
  const auto load_next = [&](int4v *k_next, int4v *v_next, int j) __attribute__((always_inline)) {
    tiles_ready();
    if (j + NK < end) {
      k.load(k_next, j + NK, k_count, wave);
      v.load(v_next, j + NK, k_count, wave);
    }
  };
  const auto all_of = [&](const int4v *k_tile, const int4v *v_tile, int4v *k_next, int4v *v_next, int j) __attribute__((always_inline)) {
    load_next(k_next, v_next, j);
#pragma unroll
    for (int kb = 0; kb < NK / 32; ++kb) take(Number<0>(), k_tile, v_tile, kb, j);
  };
  const auto some_of = [&](const int4v *k_tile, const int4v *v_tile, int4v *k_next, int4v *v_next, int j) __attribute__((always_inline)) {
    load_next(k_next, v_next, j);
#pragma unroll
    for (int kb = 0; kb < NK / 32; ++kb)
      if (j + kb * 32 < wave_end) take(Number<1>(), k_tile, v_tile, kb, j);
  };
  int j = begin;
  const int all_end = same_for_all(begin + max(min(whole, wave_end) - begin, 0) / NK * NK);
  bool second = false;
  while (j < all_end) {
    all_of(k_tile0, v_tile0, k_tile1, v_tile1, j);
    j += NK;
    second = j >= all_end;
    if (second) break;
    all_of(k_tile1, v_tile1, k_tile0, v_tile0, j);
    j += NK;
  }
  for (; j < end; j += NK) {
    if (second) some_of(k_tile1, v_tile1, k_tile0, v_tile0, j);
    else some_of(k_tile0, v_tile0, k_tile1, v_tile1, j);
    second = !second;
  }
  if (a.causal && __builtin_amdgcn_ballot_w64(lse == inf))      // (no keys: as the forward pass)
#pragma unroll
    for (int db = 0; db < W / 32; ++db) dq[db] = lse == inf ? float16v{} : dq[db];
  const bool fits = !ds_shifted<T>() || shift <= kLeastShift || __builtin_fabsf(dq[0][0]) < inf, ends = mine && open && fits;
  const float scale = a.scale * __builtin_amdgcn_ldexpf(1.f, -shift);
  if constexpr (PARTS) {
    const int64_t tile = (((int64_t)at.slot * a.kv_heads + at.kv_head) * a.parts + at.part) * T_ROWS + local;
    if (ends) store_row<T, float, W>(a.part_sum + tile * a.dim, dq, scale, a.dim, lane);
  } else if (ends) {
    store_row<T, T, W>((T *)a.gq + to * a.dim, dq, scale, a.dim, lane);
  }
  return mine && open && !fits;
}

template <typename T, int DP, int NW, bool PARTS>
__device__ __attribute__((noinline)) void query_grad_again(args_in_place *args, Lds<int4v> *k_tile0, Lds<int4v> *v_tile0, Lds<int4v> *k_tile1,
                                                           Lds<int4v> *v_tile1, unsigned block, bool open) {
  const AttentionArgs a = same_args(args);
  block = same_for_all((int)block);
  int4v *const k0 = same_tile<int4v>(k_tile0), *const v0 = same_tile<int4v>(v_tile0);
  int4v *const k1 = same_tile<int4v>(k_tile1), *const v1 = same_tile<int4v>(v_tile1);
  int shift = ds_shift<T>();
  do {
    shift -= kShiftDown;
    open = query_grad_rows<T, DP, NW, PARTS>(a, k0, v0, k1, v1, block, shift, open);
  } while (any_lane<NW>(open, k1));
}

template <typename T, int DP, int NW, bool PARTS>
__global__ __launch_bounds__(NW * 64, (waves_of_queries<T, DP>())) void attention_query_grad_kernel(const AttentionArgs a) {
  constexpr int CHUNKS = tile_rows<T, DP, NW>() * RowTile<T, tile_width<DP>()>::CH;
  __shared__ int4v k_tile0[CHUNKS], v_tile0[CHUNKS], k_tile1[CHUNKS], v_tile1[CHUNKS];
  const bool open = query_grad_rows<T, DP, NW, PARTS>(a, k_tile0, v_tile0, k_tile1, v_tile1, blockIdx.x, ds_shift<T>(), true);
  if constexpr (ds_shifted<T>())
    if (any_lane<NW>(open, k_tile1))
      query_grad_again<T, DP, NW, PARTS>((args_in_place *)__builtin_amdgcn_kernarg_segment_ptr(), (Lds<int4v> *)k_tile0, (Lds<int4v> *)v_tile0,
                                         (Lds<int4v> *)k_tile1, (Lds<int4v> *)v_tile1, blockIdx.x, open);
}

// Keys' and values' gradients: a wave's 32 keys are columns, the queries of all heads of the group pass by as rows, and
// dk^T = q^T ds, dv^T = g_out^T p take ds and p as they stand.  Four products, 266 us of the same scans (870 TFLOP/s): keys, values and two
// sums fill 254 registers at heads of 64, and every fragment of q and g_out comes out of LDS twice.  (A second block of keys to a wave halves
// those reads and leaves one wave a SIMD: 389 us.)
template <typename T, int DP, int NW, bool PARTS>
__device__ __forceinline__ bool key_grad_rows(const AttentionArgs &a, int4v *q_tile0, int4v *g_tile0, int4v *q_tile1, int4v *g_tile1, float4v *lse_tile0,
                                              float4v *delta_tile0, float4v *lse_tile1, float4v *delta_tile1, unsigned block, int shift, bool open) {
  constexpr int W = tile_width<DP>(), NQ = tile_rows<T, DP, NW>(), STEPS = DP / (32 / (int)sizeof(T)), T_ROWS = 32 * NW;
  using Rows = RowTile<T, W>;
  constexpr int PER = NQ * Rows::CH / (64 * NW);
  const int lane = threadIdx.x % 64, wave = same_for_all(threadIdx.x / 64), group = a.heads / a.kv_heads;
  Rows rows_at;
  rows_at.aim(lane);
  const Place at = place_of<false>(block, a.kv_heads, PARTS ? a.parts : 1, a.by_xcd, a.slots);
  if (at.slot >= a.slots) return false;
  const Slot slot = find_slot(a.k_offsets, a.segments, a.n_k, 1, T_ROWS, at.slot, a.slots);
  int q_begin, q_count;
  partner_rows(a.q_offsets, nullptr, slot.segment, a.segments, a.n_q, q_begin, q_count);
  if (slot.first >= slot.length) return false;
  const int ahead = slot.length - q_count, rows = q_count * group;

  const int local = wave * 32 + lane % 32, key = slot.first + local;
  const bool mine = key < slot.length;
  const bool awake = slot.first + wave * 32 < slot.length;

  // rows from which on this lane's key is seen, the workgroup's first key (first of all), the wave's first and last
  int begin = 0, end = rows;
  const int from = a.causal ? max(0, key - ahead) * group : 0;
  const int wave_from = awake ? a.causal ? max(0, slot.first + wave * 32 - ahead) * group : 0 : rows;
  const int whole = a.causal ? max(0, slot.first + wave * 32 + 31 - ahead) * group : 0;
  if (a.causal) begin = max(0, slot.first - ahead) * group / NQ * NQ;
  if constexpr (PARTS) {
    const int piece = ((max(rows - begin, 0) + a.parts - 1) / a.parts + NQ - 1) / NQ * NQ;
    begin += at.part * piece;
    end = min(end, begin + piece);
  }

  // Rows on their way to LDS: row r is head r % group of token r / group.  Where a lane's rows lie behind their tile's first token is the same
  // for all tiles if these begin with a group's first head, which tiles of NQ rows do where the group divides NQ.
  const int64_t q_row = a.q_row * (int)sizeof(T), q_head = a.q_head * (int)sizeof(T), g_row = (int64_t)a.heads * a.dim * (int)sizeof(T);
  const char *const q_base = (const char *)a.q + q_begin * q_row + at.kv_head * group * q_head;
  const char *const g_base = (const char *)a.g_out + q_begin * g_row + (int64_t)at.kv_head * group * a.dim * (int)sizeof(T);
  const float *const lse_base = a.lse + (int64_t)q_begin * a.heads + at.kv_head * group;
  const float *const delta_base = a.delta + (int64_t)q_begin * a.heads + at.kv_head * group;
  const float per_group = 1.f / group, inf = __builtin_inff();
  const bool steady = NQ % group == 0;
  unsigned q_at[PER], g_at[PER], row_sum_at;
  const auto aim = [&](int head0) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < PER; ++i) {
      const int e = (wave + i * NW) * 64 + lane, row = e / Rows::CH, c = (e % Rows::CH) ^ Rows::swizzle(row);
      const int token = divide(head0 + row, per_group), head = head0 + row - token * group;
      const bool there = c * Rows::E < a.dim;
      q_at[i] = there ? (unsigned)token * (unsigned)q_row + (unsigned)head * (unsigned)q_head + c * 16 : kAbsentRow;
      g_at[i] = there ? (unsigned)token * (unsigned)g_row + (unsigned)(head * a.dim * (int)sizeof(T)) + c * 16 : kAbsentRow;
    }
    const int token = divide(head0 + lane, per_group);
    row_sum_at = (unsigned)token * a.heads + (head0 + lane - token * group);
  };
  aim(steady ? 0 : same_for_all(begin % group));
  float next_lse = 0.f, next_delta = 0.f;
  const auto load = [&](int4v *q_tile, int4v *g_tile, int first) __attribute__((always_inline)) {
    const int token0 = same_for_all(group == 1 ? first : first / group);
    if (!steady) aim(first - token0 * group);
    const __amdgpu_buffer_rsrc_t qs = rows_resource(q_base + token0 * q_row, kMaxBufferBytes), gs = rows_resource(g_base + token0 * g_row, kMaxBufferBytes);
    if (first + NQ <= rows) {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        load_to_lds(qs, q_tile + (wave + i * NW) * 64, q_at[i]);
        load_to_lds(gs, g_tile + (wave + i * NW) * 64, g_at[i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const bool there = first + ((wave + i * NW) * 64 + lane) / Rows::CH < rows;
        load_to_lds(qs, q_tile + (wave + i * NW) * 64, there ? q_at[i] : kAbsentRow);
        load_to_lds(gs, g_tile + (wave + i * NW) * 64, there ? g_at[i] : kAbsentRow);
      }
    }
    if (wave == 0) {
      const bool there = lane < NQ && first + lane < rows;
      const int64_t to = (int64_t)token0 * a.heads + (there ? row_sum_at : 0);
      next_lse = lse_base[to], next_delta = delta_base[to];
      next_lse = there ? next_lse : -inf;      // (no such row: all probabilities 0)
      next_delta = there ? next_delta : 0.f;
    }
  };
  const auto keep = [&](float4v *lse_tile, float4v *delta_tile) __attribute__((always_inline)) {
    if (wave == 0 && lane < NQ) {
      reinterpret_cast<float *>(lse_tile)[lane] = next_lse == -inf ? inf : next_lse * kLog2e - p_shift<T>();
      reinterpret_cast<float *>(delta_tile)[lane] = next_delta;
    }
  };
  if (begin < end) {
    load(q_tile0, g_tile0, begin);
    keep(lse_tile0, delta_tile0);
  }
  int4v k[STEPS], v[STEPS];
  load_row<T, DP>(k, mine ? (const T *)a.k + (slot.begin + key) * a.k_row + at.kv_head * a.k_head : nullptr, a.dim, lane);
  load_row<T, DP>(v, mine ? (const T *)a.v + (slot.begin + key) * a.v_row + at.kv_head * a.v_head : nullptr, a.dim, lane);
  const float by = a.scale * kLog2e;
  const float ds_by = __builtin_amdgcn_ldexpf(1.f, shift - p_shift<T>());      // (p's power of two taken out)
  float16v dk[W / 32] = {}, dv[W / 32] = {};
  const auto take = [&](auto masked, const int4v *q_tile, const int4v *g_tile, const float4v *lse_tile, const float4v *delta_tile, int qb,
                        int r0) __attribute__((always_inline)) {
    float16v p = {}, ds = {};
    // (heads of 96: what one step reads is not fetched during the one before, which the registers have no room for: both gradients of
    // two scans of 9 k rows together, 16/4 heads, bf16, 1278 -> 1228 us)
    const auto phase = []() __attribute__((always_inline)) { if constexpr (DP == 96) __builtin_amdgcn_sched_barrier(0); };
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (sizeof(T) == 2 || i * 2 * Rows::E < a.dim) multiply<T>(p, rows_at.rows(q_tile, qb * 32, i), k[i]);
    phase();
#pragma unroll
    for (int i = 0; i < STEPS; ++i)
      if (sizeof(T) == 2 || i * 2 * Rows::E < a.dim) multiply<T>(ds, rows_at.rows(g_tile, qb * 32, i), v[i]);
    phase();
#pragma unroll
    for (int r4 = 0; r4 < 4; ++r4) {
      const float4v lse = lse_tile[qb * 8 + 2 * r4 + lane / 32], delta = delta_tile[qb * 8 + 2 * r4 + lane / 32];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 4 * r4 + e;
        p[r] = __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], by, -lse[e]));
        ds[r] = p[r] * ((ds[r] - delta[e]) * ds_by);
      }
    }
    if constexpr (decltype(masked)::value != 0) {
      const int hidden = from - r0 - qb * 32 - 4 * (lane / 32);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        p[r] = hidden > 8 * (r / 4) + r % 4 ? 0.f : p[r];
        ds[r] = hidden > 8 * (r / 4) + r % 4 ? 0.f : ds[r];
      }
    }
    phase();
    add_weighted_rows<T, W>(dv, rows_at, g_tile, qb * 32, p);
    phase();
    add_weighted_rows<T, W>(dk, rows_at, q_tile, qb * 32, ds);
  };
  const auto all_of = [&](auto masked, const int4v *q_tile, const int4v *g_tile, const float4v *lse_tile, const float4v *delta_tile, int4v *q_next, int4v *g_next,
                          float4v *lse_next, float4v *delta_next, int r0) __attribute__((always_inline)) {
    tiles_ready();
    const bool more = r0 + NQ < end;
    if (more) load(q_next, g_next, r0 + NQ);
#pragma unroll
    for (int qb = 0; qb < NQ / 32; ++qb) take(masked, q_tile, g_tile, lse_tile, delta_tile, qb, r0);
    if (more) keep(lse_next, delta_next);
  };
  const auto rest_of = [&](const int4v *q_tile, const int4v *g_tile, const float4v *lse_tile, const float4v *delta_tile, int r0) __attribute__((always_inline)) {
    tiles_ready();
    if (!awake) return;
    take(Number<1>(), q_tile, g_tile, lse_tile, delta_tile, 0, r0);
    if (NQ == 64 && r0 + 32 < end) take(Number<1>(), q_tile, g_tile, lse_tile, delta_tile, NQ / 32 - 1, r0);
  };
  // Tiles that no key of the wave is seen from, tiles that some are not seen from (even numbers of both: the loops behind start with the
  // first pair of buffers), whole tiles, and what is left.  As in the forward kernel the loops have no choice in them that the
  // accumulators depend on.
  int r0 = begin;
  const int wave_begin = same_for_all(awake ? min(begin + max(wave_from - begin, 0) / (2 * NQ) * (2 * NQ), end) : end);
  for (bool second = false; r0 < wave_begin; r0 += NQ) {
    tiles_ready();
    second = !second;      // (the pair to be filled)
    if (r0 + NQ >= end) continue;
    load(second ? q_tile1 : q_tile0, second ? g_tile1 : g_tile0, r0 + NQ);
    keep(second ? lse_tile1 : lse_tile0, second ? delta_tile1 : delta_tile0);
  }
  bool second = false;
  const auto all_until = [&](auto masked, int stop) __attribute__((always_inline)) {
    while (r0 < stop) {
      all_of(masked, q_tile0, g_tile0, lse_tile0, delta_tile0, q_tile1, g_tile1, lse_tile1, delta_tile1, r0);
      r0 += NQ;
      second = r0 >= stop;
      if (second) break;
      all_of(masked, q_tile1, g_tile1, lse_tile1, delta_tile1, q_tile0, g_tile0, lse_tile0, delta_tile0, r0);
      r0 += NQ;
    }
  };
  const int all_end = begin + max(end - begin, 0) / NQ * NQ;
  const int masked_end = same_for_all(min(r0 + (max(whole - r0, 0) + 2 * NQ - 1) / (2 * NQ) * (2 * NQ), all_end));
  all_until(Number<1>(), masked_end);
  all_until(Number<0>(), all_end);
  if (r0 < end) {
    if (second) rest_of(q_tile1, g_tile1, lse_tile1, delta_tile1, r0);
    else rest_of(q_tile0, g_tile0, lse_tile0, delta_tile0, r0);
  }
  const bool fits = !ds_shifted<T>() || !a.gk || shift <= kLeastShift || __builtin_fabsf(dk[0][0]) < inf;
  const float k_by = a.scale * __builtin_amdgcn_ldexpf(1.f, -shift), v_by = pow2(-p_shift<T>());
  if (mine && open && fits) {
    if constexpr (PARTS) {
      const int64_t tile = (((int64_t)at.slot * a.kv_heads + at.kv_head) * a.parts + at.part) * T_ROWS + local;
      const int64_t all = (int64_t)a.slots * a.kv_heads * a.parts * T_ROWS * a.dim;
      store_row<T, float, W>(a.part_sum + tile * a.dim, dk, k_by, a.dim, lane);
      store_row<T, float, W>(a.part_sum + all + tile * a.dim, dv, v_by, a.dim, lane);
    } else {
      const int64_t to = ((int64_t)(slot.begin + key) * a.kv_heads + at.kv_head) * a.dim;
      if (a.gk) store_row<T, T, W>((T *)a.gk + to, dk, k_by, a.dim, lane);
      if (a.gv) store_row<T, T, W>((T *)a.gv + to, dv, v_by, a.dim, lane);
    }
  }
  return mine && open && !fits;
}

template <typename T, int DP, int NW, bool PARTS>
__device__ __attribute__((noinline)) void key_grad_again(args_in_place *args, Lds<int4v> *q_tile0, Lds<int4v> *g_tile0, Lds<int4v> *q_tile1,
                                                         Lds<int4v> *g_tile1, Lds<float4v> *lse_tile0, Lds<float4v> *delta_tile0,
                                                         Lds<float4v> *lse_tile1, Lds<float4v> *delta_tile1, unsigned block, bool open) {
  const AttentionArgs a = same_args(args);
  block = same_for_all((int)block);
  int4v *const q0 = same_tile<int4v>(q_tile0), *const g0 = same_tile<int4v>(g_tile0);
  int4v *const q1 = same_tile<int4v>(q_tile1), *const g1 = same_tile<int4v>(g_tile1);
  float4v *const lse0 = same_tile<float4v>(lse_tile0), *const delta0 = same_tile<float4v>(delta_tile0);
  float4v *const lse1 = same_tile<float4v>(lse_tile1), *const delta1 = same_tile<float4v>(delta_tile1);
  int shift = ds_shift<T>();
  do {
    shift -= kShiftDown;
    open = key_grad_rows<T, DP, NW, PARTS>(a, q0, g0, q1, g1, lse0, delta0, lse1, delta1, block, shift, open);
  } while (any_lane<NW>(open, q1));
}

template <typename T, int DP, int NW, bool PARTS>
__global__ __launch_bounds__(NW * 64, (waves_of_keys<T, DP>())) void attention_key_grad_kernel(const AttentionArgs a) {
  constexpr int NQ = tile_rows<T, DP, NW>(), CHUNKS = NQ * RowTile<T, tile_width<DP>()>::CH;
  __shared__ int4v q_tile0[CHUNKS], g_tile0[CHUNKS], q_tile1[CHUNKS], g_tile1[CHUNKS];
  __shared__ float4v lse_tile0[NQ / 4], delta_tile0[NQ / 4], lse_tile1[NQ / 4], delta_tile1[NQ / 4];
  const bool open = key_grad_rows<T, DP, NW, PARTS>(a, q_tile0, g_tile0, q_tile1, g_tile1, lse_tile0, delta_tile0, lse_tile1, delta_tile1, blockIdx.x,
                                                    ds_shift<T>(), true);
  if constexpr (ds_shifted<T>())
    if (any_lane<NW>(open, q_tile1))
      key_grad_again<T, DP, NW, PARTS>((args_in_place *)__builtin_amdgcn_kernarg_segment_ptr(), (Lds<int4v> *)q_tile0, (Lds<int4v> *)g_tile0,
                                       (Lds<int4v> *)q_tile1, (Lds<int4v> *)g_tile1, (Lds<float4v> *)lse_tile0, (Lds<float4v> *)delta_tile0,
                                       (Lds<float4v> *)lse_tile1, (Lds<float4v> *)delta_tile1, blockIdx.x, open);
}

// --- launches --------------------------------------------------------------------------------------------------
inline int launched(const char *what) {
  const hipError_t e = hipGetLastError();
  if (e == hipSuccess) return FGMS_OK;
  set_error("%s: %s", what, hipGetErrorString(e));
  return FGMS_E_HIP;
}

inline int grid_of(int64_t blocks, unsigned *grid) {
  if (blocks > 0x7fffffff) {
    set_error("segment attention: %lld workgroups are more than one launch takes", (long long)blocks);
    return FGMS_E_INVALID;
  }
  *grid = (unsigned)blocks;
  return FGMS_OK;
}

// Rows of a workgroup's tile go by the average segment: four waves of 32 share the staged tiles of the other side, over segments of up to 256 rows
// two, which leave fewer idle behind a segment's last row, and one where segments have hardly more than 32.
// (Windows of 120 k voxels, 90 on average, both passes: four waves 201 us, two 183, one 232; scans of 24 k rows 1.68 ms, 2.67, 6.9.)
inline int waves_for(int64_t rows, int64_t segments) {
  return rows > 256 * segments ? 4 : rows > 48 * segments ? 2 : 1;
}

// Pieces of a long axis: until a CU has 16 waves (fp32, and single waves: twelve workgroups, more than run at once, as segments and so
// their pieces differ in length), none shorter than 128 rows on average, and only where a segment has four such (fp32: two): the join is a
// launch of five to ten microseconds, in which a workgroup gets through 300 to 500 rows.  (fp32, 37 segments of 540 keys, heads of
// 40, forward: two pieces 79 us, four 68, seven 75; bf16, two of 1185, heads of 72: four 36, five 35, nine 43.)
inline int parts_for(int64_t workgroups, int waves, int64_t partners, int64_t segments, int dtype) {
  const int64_t least = 128, each = partners / (segments > 0 ? segments : 1);
  if (each < (dtype == FGMS_F32 ? 2 : 4) * least) return 1;
  const int64_t per_cu = dtype == FGMS_F32 || waves == 1 ? 12 : 16 / waves;
  const int64_t want = per_cu * num_cus() / (workgroups > 0 ? workgroups : 1), most = each / least;
  const int64_t parts = want < most ? want : most;
  return parts < 2 || workgroups > 2 * num_cus() ? 1 : parts > kMostParts ? kMostParts : (int)parts;
}

// Workgroups of a launch over tiles of `rows` rows: slots, parts and order go into `a`.
inline int plan_grid(AttentionArgs &a, int64_t rows, int tile, int64_t partners, unsigned *grid, int64_t *tiles) {
  const int64_t slots = attention_slots(rows, a.segments, tile), segments = a.segments > 0 ? a.segments : 1;
  a.parts = parts_for((rows / tile + a.segments) * a.kv_heads, tile / 32, partners, a.segments, a.dtype);
  // (short: the partners of a segment, all heads, are less than half of an XCD's L2)
  const int64_t element = a.dtype == FGMS_F32 ? 4 : 2;
  a.by_xcd = a.parts == 1 && slots >= 64 * kPlaceTiles && partners / segments * 2 * a.kv_heads * a.dim * element <= (2 << 20);
  *tiles = slots * a.kv_heads;
  const int64_t per = (int64_t)kPlaceTiles * a.kv_heads * 8;
  const int rc = grid_of((a.by_xcd ? (*tiles + per - 1) / per * per : *tiles) * a.parts, grid);
  a.slots = (int)slots;
  return rc;
}

template <typename T, int DP, int NW, bool ONES>
int forward(AttentionArgs a) {
  const int group = a.heads / a.kv_heads;
  unsigned grid;
  int64_t tiles;
  int rc = plan_grid(a, (int64_t)a.n_q * group, 32 * NW, a.n_k, &grid, &tiles);
  if (rc != FGMS_OK) return rc;
  if (a.parts == 1) {
    segment_attention_kernel<T, DP, NW, false, ONES><<<grid, NW * 64, 0, a.stream>>>(a);
    return launched("segment attention");
  }
  const StreamTurn turn(a.stream);
  const size_t rows = (size_t)tiles * a.parts * 32 * NW;
  rc = workspace_get(a.stream, kSlotAttention, rows * (a.dim + 1) * sizeof(float), (void **)&a.part_sum);
  if (rc != FGMS_OK) return rc;
  a.part_lse = a.part_sum + rows * a.dim;
  segment_attention_kernel<T, DP, NW, true, ONES><<<grid, NW * 64, 0, a.stream>>>(a);
  join_parts_kernel<T, NW, false><<<(unsigned)tiles * (32 * NW / kJoinRows), 256, 0, a.stream>>>(a, a.q_offsets, a.n_q, group, a.part_sum, (T *)a.out);
  return launched("segment attention");
}

template <typename T, int DP, int NW>
int query_grad(AttentionArgs a) {
  const int group = a.heads / a.kv_heads;
  unsigned grid;
  int64_t tiles;
  int rc = plan_grid(a, (int64_t)a.n_q * group, 32 * NW, a.n_k, &grid, &tiles);
  if (rc != FGMS_OK) return rc;
  if (a.parts == 1) {
    attention_query_grad_kernel<T, DP, NW, false><<<grid, NW * 64, 0, a.stream>>>(a);
    return launched("segment attention, queries' gradient");
  }
  rc = workspace_get(a.stream, kSlotAttention, (size_t)tiles * a.parts * 32 * NW * a.dim * sizeof(float), (void **)&a.part_sum);
  if (rc != FGMS_OK) return rc;
  attention_query_grad_kernel<T, DP, NW, true><<<grid, NW * 64, 0, a.stream>>>(a);
  join_parts_kernel<T, NW, true><<<(unsigned)tiles * (32 * NW / kJoinRows), 256, 0, a.stream>>>(a, a.q_offsets, a.n_q, group, a.part_sum, (T *)a.gq);
  return launched("segment attention, queries' gradient");
}

template <typename T, int DP, int NW>
int key_grad(AttentionArgs a) {
  unsigned grid;
  int64_t tiles;
  int rc = plan_grid(a, a.n_k, 32 * NW, (int64_t)a.n_q * (a.heads / a.kv_heads), &grid, &tiles);
  if (rc != FGMS_OK) return rc;
  if (a.parts == 1) {
    attention_key_grad_kernel<T, DP, NW, false><<<grid, NW * 64, 0, a.stream>>>(a);
    return launched("segment attention, keys' gradients");
  }
  const size_t all = (size_t)tiles * a.parts * 32 * NW * a.dim;
  rc = workspace_get(a.stream, kSlotAttention, 2 * all * sizeof(float), (void **)&a.part_sum);
  if (rc != FGMS_OK) return rc;
  attention_key_grad_kernel<T, DP, NW, true><<<grid, NW * 64, 0, a.stream>>>(a);
  if (a.gk) join_parts_kernel<T, NW, true><<<(unsigned)tiles * (32 * NW / kJoinRows), 256, 0, a.stream>>>(a, a.k_offsets, a.n_k, 1, a.part_sum, (T *)a.gk);
  if (a.gv) join_parts_kernel<T, NW, true><<<(unsigned)tiles * (32 * NW / kJoinRows), 256, 0, a.stream>>>(a, a.k_offsets, a.n_k, 1, a.part_sum + all, (T *)a.gv);
  return launched("segment attention, keys' gradients");
}

template <typename F>
int by_waves(int waves, F f) {
  return waves == 4 ? f(Number<4>()) : waves == 2 ? f(Number<2>()) : f(Number<1>());
}

template <typename T, int DP>
int forward_any(const AttentionArgs &a) {
  return by_waves(waves_for((int64_t)a.n_q * (a.heads / a.kv_heads), a.segments), [&](auto w) {
    if constexpr (DP < 32) return forward<T, DP, decltype(w)::value, true>(a);
    else if constexpr (sizeof(T) == 4) return forward<T, DP, decltype(w)::value, false>(a);
    else return a.dim < DP ? forward<T, DP, decltype(w)::value, true>(a) : forward<T, DP, decltype(w)::value, false>(a);
  });
}

template <typename T, int DP>
int backward_any(const AttentionArgs &a) {
  const int64_t rows = (int64_t)a.n_q * a.heads;
  int rc = FGMS_OK;
  if (a.gq && a.n_q > 0) {
    rc = by_waves(waves_for((int64_t)a.n_q * (a.heads / a.kv_heads), a.segments), [&](auto w) { return query_grad<T, DP, decltype(w)::value>(a); });
  } else if (rows > 0) {
    unsigned grid;
    if ((rc = grid_of((rows + 127) / 128, &grid)) != FGMS_OK) return rc;
    attention_delta_kernel<T, DP><<<grid, 256, 0, a.stream>>>((const T *)a.g_out, (const T *)a.out, a.delta, rows, a.dim);
    rc = launched("segment attention, backward");
  }
  if (rc == FGMS_OK && (a.gk || a.gv) && a.n_k > 0)
    rc = by_waves(waves_for(a.n_k, a.segments), [&](auto w) { return key_grad<T, DP, decltype(w)::value>(a); });
  return rc;
}

}  // namespace

template <typename T>
int attention_fwd(const AttentionArgs &a) {
  if constexpr (sizeof(T) == 2)
    if (a.dim <= 16) return forward_any<T, 16>(a);
  return a.dim <= 32 ? forward_any<T, 32>(a) : a.dim <= 64 ? forward_any<T, 64>(a) : a.dim <= 96 ? forward_any<T, 96>(a) : forward_any<T, 128>(a);
}

template <typename T>
int attention_bwd(const AttentionArgs &a) {
  if constexpr (sizeof(T) == 2)
    if (a.dim <= 16) return backward_any<T, 16>(a);
  return a.dim <= 32 ? backward_any<T, 32>(a) : a.dim <= 64 ? backward_any<T, 64>(a) : a.dim <= 96 ? backward_any<T, 96>(a) : backward_any<T, 128>(a);
}

}  // namespace fgms
