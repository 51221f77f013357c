// The attention kernels, for one type (included by fgms_attention_f16.hip, _bf16.hip and _f32.hip).
#pragma once

#include "fgms_attention.h"

namespace fgms {
namespace {

// Keys (queries in the keys' gradients) to a tile.
template <typename T, int DP> constexpr int tile_rows() { return sizeof(T) * DP > 256 ? 32 : 64; }

// Rows [first, first + ROWS) of a strided tensor to LDS, zeros from row `end` on and behind the channels.
template <typename T, int DP, int ROWS, int THREADS>
__device__ __forceinline__ void stage_rows(int4v *tile, const T *base, int64_t stride, int64_t first, int64_t end, int dim) {
  using Rows = RowTile<T, DP>;
  constexpr int PER = ROWS * Rows::CH / THREADS;
  int4v v[PER];
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = threadIdx.x + i * THREADS, row = e / Rows::CH, c = e % Rows::CH;
    v[i] = first + row < end && c * Rows::E < dim ? *reinterpret_cast<const int4v *>(base + (first + row) * stride + c * Rows::E)
                                                  : int4v{0, 0, 0, 0};
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int e = threadIdx.x + i * THREADS;
    tile[Rows::at(e / Rows::CH, e % Rows::CH)] = v[i];
  }
}

// Where a launch's workgroup stands.
struct Place {
  int64_t slot;
  int kv_head, part;
};
__device__ __forceinline__ Place place_of(int64_t block, int kv_heads, int parts) {
  Place p;
  p.part = (int)(block % parts);
  p.kv_head = (int)(block / parts % kv_heads);
  p.slot = block / parts / kv_heads;
  return p;
}

// --- forward --------------------------------------------------------------------------------------------------
// A wave holds 32 query rows as columns: scores come out of the matrix unit transposed (keys down the registers, a query a
// lane and its partner 32 lanes on), so that a row's maximum and sum are taken inside two lanes, and the exponentials are
// the right operand of the second product as they stand, with no exchange between lanes.
template <typename T, int DP, int NW, bool PARTS>
__global__ __launch_bounds__(NW * 64) void segment_attention_kernel(const AttentionArgs a) {
  constexpr int NK = tile_rows<T, DP>(), STEPS = DP / (32 / (int)sizeof(T)), T_ROWS = 32 * NW;
  __shared__ int4v k_tile[NK * RowTile<T, DP>::CH], v_tile[NK * RowTile<T, DP>::CH];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, group = a.heads / a.kv_heads;
  const Place at = place_of(blockIdx.x, a.kv_heads, PARTS ? a.parts : 1);
  const Slot slot = find_slot(a.q_offsets, a.segments, a.n_q, group, T_ROWS, at.slot);
  if (slot.first >= slot.length) return;
  int64_t k_begin, k_count;
  partner_rows(a.k_offsets, a.k_lengths, slot.segment, a.segments, a.n_k, k_begin, k_count);
  const int64_t ahead = k_count - slot.length / group;      // the last query sees the last key

  const int64_t row = slot.first + wave * 32 + lane % 32;
  const bool mine = row < slot.length;
  const int64_t token = row / group;
  const int head = at.kv_head * group + (int)(row % group);
  int4v q[STEPS];
  load_row<T, DP>(q, mine ? (const T *)a.q + (slot.begin + token) * a.q_row + head * a.q_head : nullptr, a.dim, lane);

  // keys this lane's row sees: those below `seen`; of a workgroup's rows the last sees most, of a wave's the first least
  const int64_t seen = a.causal ? min(k_count, token + ahead + 1) : k_count;
  const int64_t last_row = min(slot.first + T_ROWS, slot.length) - 1;
  int64_t begin = 0, end = a.causal ? min(k_count, last_row / group + ahead + 1) : k_count;
  const int64_t whole = a.causal ? min(k_count, (slot.first + wave * 32) / group + ahead + 1) : k_count;
  if constexpr (PARTS) {
    const int64_t piece = ((k_count + a.parts - 1) / a.parts + NK - 1) / NK * NK;
    begin = at.part * piece;
    end = min(end, begin + piece);
  }

  const T *const k = (const T *)a.k + k_begin * a.k_row + at.kv_head * a.k_head;
  const T *const v = (const T *)a.v + k_begin * a.v_row + at.kv_head * a.v_head;
  const float by = a.scale * kLog2e;
  const float inf = __builtin_inff();
  float most = -inf, sum = 0.f;      // of the scores so far, times `by`; this lane's part of the sum
  float16v o[DP / 32] = {};
  for (int64_t j = begin; j < end; j += NK) {
    __syncthreads();
    stage_rows<T, DP, NK, NW * 64>(k_tile, k, a.k_row, j, k_count, a.dim);
    stage_rows<T, DP, NK, NW * 64>(v_tile, v, a.v_row, j, k_count, a.dim);
    __syncthreads();
    float16v s[NK / 32] = {};
#pragma unroll
    for (int kb = 0; kb < NK / 32; ++kb)
#pragma unroll
      for (int i = 0; i < STEPS; ++i) multiply<T>(s[kb], RowTile<T, DP>::rows(k_tile, kb * 32, i, lane), q[i]);
    if (j + NK > whole) {
      const int left = (int)max((int64_t)-1, min((int64_t)NK, seen - j));
#pragma unroll
      for (int kb = 0; kb < NK / 32; ++kb)
#pragma unroll
        for (int r = 0; r < 16; ++r)
          if (kb * 32 + 8 * (r / 4) + 4 * (lane / 32) + r % 4 >= left) s[kb][r] = -inf;
    }
    float top = -inf;
#pragma unroll
    for (int kb = 0; kb < NK / 32; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = __builtin_fmaxf(top, s[kb][r]);
    top = __builtin_fmaxf(most, both_max(top) * by);
    const float from = top == -inf ? 0.f : top;      // (a row that has met no key yet)
    const float keep = __builtin_amdgcn_exp2f(most - from);
    most = top;
    float add = 0.f;
#pragma unroll
    for (int kb = 0; kb < NK / 32; ++kb)
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        s[kb][r] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[kb][r], by, -from));
        add += s[kb][r];
      }
    sum = __builtin_fmaf(sum, keep, add);
#pragma unroll
    for (int db = 0; db < DP / 32; ++db) o[db] *= keep;
#pragma unroll
    for (int kb = 0; kb < NK / 32; ++kb) add_weighted_rows<T, DP>(o, v_tile, kb * 32, s[kb], lane);
  }

  sum = both_sum(sum);
  const bool none = seen <= begin || end <= begin;      // no key for this row (here)
  const float inverse = none ? 0.f : 1.f / sum;
  const float lse = none ? -inf : (most + __builtin_log2f(sum)) * (1.f / kLog2e);
  if constexpr (PARTS) {
    const int64_t tile = ((at.slot * a.kv_heads + at.kv_head) * a.parts + at.part) * T_ROWS + wave * 32 + lane % 32;
    if (mine && !none) store_row<float, DP>(a.part_sum + tile * a.dim, o, inverse, a.dim, lane);
    if (mine && lane < 32) a.part_lse[tile] = lse;
  } else if (mine) {
    const int64_t to = (slot.begin + token) * a.heads + head;
    store_row<T, DP>((T *)a.out + to * a.dim, o, inverse, a.dim, lane);
    if (a.lse && lane < 32) a.lse[to] = lse;
  }
}

// --- joining the parts -----------------------------------------------------------------------------------------
// A thread four channels of a row; SUMS: the parts add up (gradients, times `by`), else they are averages over their keys, to be
// weighted by their sums of exponentials.
template <typename T, int NW, bool SUMS>
__global__ __launch_bounds__(256) void join_parts_kernel(const AttentionArgs a, const int32_t *__restrict__ offsets, int64_t n, int group,
                                                         const float *__restrict__ sums, T *__restrict__ out, float by) {
  typedef T T4 __attribute__((ext_vector_type(4)));
  constexpr int T_ROWS = 32 * NW;
  const int per_row = a.dim / 4;
  const Place at = place_of(blockIdx.x, a.kv_heads, 1);
  const Slot slot = find_slot(offsets, a.segments, n, group, T_ROWS, at.slot);
  const int64_t first = (at.slot * a.kv_heads + at.kv_head) * a.parts * T_ROWS;
  for (int e = threadIdx.x; e < T_ROWS * per_row; e += 256) {
    const int local = e / per_row, c = e % per_row * 4;
    const int64_t row = slot.first + local;
    if (row >= slot.length) break;
    const int64_t to = ((slot.begin + row / group) * a.kv_heads + at.kv_head) * group + row % group;
    float4v total = {0.f, 0.f, 0.f, 0.f};
    if constexpr (SUMS) {
      for (int p = 0; p < a.parts; ++p) total += *reinterpret_cast<const float4v *>(sums + (first + (int64_t)p * T_ROWS + local) * a.dim + c);
      total *= by;
    } else {
      const float *const lse = a.part_lse + first + local;
      float most = -__builtin_inff();
      for (int p = 0; p < a.parts; ++p) most = __builtin_fmaxf(most, lse[(int64_t)p * T_ROWS]);
      float weight = 0.f;
      bool any = false;
      for (int p = 0; p < a.parts; ++p) {
        const float l = lse[(int64_t)p * T_ROWS];
        if (l == -__builtin_inff()) continue;      // (no keys there, and nothing written)
        any = true;
        const float w = __builtin_amdgcn_exp2f((l - most) * kLog2e);
        weight += w;
        total += w * *reinterpret_cast<const float4v *>(sums + (first + (int64_t)p * T_ROWS + local) * a.dim + c);
      }
      if (any) total /= weight;
      if (a.lse && c == 0) a.lse[to] = any ? most + __builtin_log2f(weight) * (1.f / kLog2e) : -__builtin_inff();
    }
    *reinterpret_cast<T4 *>(out + to * a.dim + c) = __builtin_convertvector(total, T4);
  }
}


// --- backward -------------------------------------------------------------------------------------------------
// ds = p (g_out . v - delta) is rounded to T for its two products, p for its one.  In fp16 a power of two goes with them, taken out
// of the sums again: p is 1 / N in a row of N like keys and would lose bits from 2^-14 on, with 2^10 from 2^-24 on; ds has 2^4
// (steps of 2^-28; it may reach 4094).
template <typename T> constexpr int p_shift() { return __is_same(T, _Float16) ? 10 : 0; }
template <typename T> constexpr int ds_shift() { return __is_same(T, _Float16) ? 4 : 0; }
constexpr float pow2(int e) { return e >= 0 ? (float)(1 << e) : 1.f / (float)(1 << -e); }

// delta = g_out . out of each row and head: eight lanes a row.
template <typename T>
__global__ __launch_bounds__(256) void attention_delta_kernel(const T *__restrict__ g_out, const T *__restrict__ out,
                                                              float *__restrict__ delta, int64_t rows, int dim) {
  typedef T T8 __attribute__((ext_vector_type(8)));
  const int64_t row = (int64_t)blockIdx.x * 32 + threadIdx.x / 8;
  float sum = 0.f;
  if (row < rows)
    for (int c = threadIdx.x % 8 * 8; c < dim; c += 64) {
      const T8 x = *reinterpret_cast<const T8 *>(g_out + row * dim + c), y = *reinterpret_cast<const T8 *>(out + row * dim + c);
#pragma unroll
      for (int e = 0; e < 8; ++e) sum = __builtin_fmaf((float)x[e], (float)y[e], sum);
    }
#pragma unroll
  for (int d = 1; d < 8; d *= 2) sum += __shfl_xor(sum, d);
  if (row < rows && threadIdx.x % 8 == 0) delta[row] = sum;
}

// Queries' gradients.  As the forward kernel: a wave's 32 query rows are columns, so that a row's log-sum and delta are one value a lane,
// and ds the right operand of dq^T = k^T ds as it stands.
template <typename T, int DP, int NW, bool PARTS>
__global__ __launch_bounds__(NW * 64) void attention_query_grad_kernel(const AttentionArgs a) {
  constexpr int NK = tile_rows<T, DP>(), STEPS = DP / (32 / (int)sizeof(T)), T_ROWS = 32 * NW;
  __shared__ int4v k_tile[NK * RowTile<T, DP>::CH], v_tile[NK * RowTile<T, DP>::CH];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, group = a.heads / a.kv_heads;
  const Place at = place_of(blockIdx.x, a.kv_heads, PARTS ? a.parts : 1);
  const Slot slot = find_slot(a.q_offsets, a.segments, a.n_q, group, T_ROWS, at.slot);
  if (slot.first >= slot.length) return;
  int64_t k_begin, k_count;
  partner_rows(a.k_offsets, a.k_lengths, slot.segment, a.segments, a.n_k, k_begin, k_count);
  const int64_t ahead = k_count - slot.length / group;

  const int64_t row = slot.first + wave * 32 + lane % 32;
  const bool mine = row < slot.length;
  const int64_t token = row / group;
  const int head = at.kv_head * group + (int)(row % group);
  const int64_t to = (slot.begin + token) * a.heads + head;
  int4v q[STEPS], g[STEPS];
  load_row<T, DP>(q, mine ? (const T *)a.q + (slot.begin + token) * a.q_row + head * a.q_head : nullptr, a.dim, lane);
  load_row<T, DP>(g, mine ? (const T *)a.g_out + to * a.dim : nullptr, a.dim, lane);
  const float inf = __builtin_inff();
  float lse = mine ? a.lse[to] : inf;
  lse = lse == -inf ? inf : lse * kLog2e - ds_shift<T>();      // (no keys: all probabilities 0)
  const float delta = mine ? a.delta[to] : 0.f;

  const int64_t seen = a.causal ? min(k_count, token + ahead + 1) : k_count;
  const int64_t last_row = min(slot.first + T_ROWS, slot.length) - 1;
  int64_t begin = 0, end = a.causal ? min(k_count, last_row / group + ahead + 1) : k_count;
  const int64_t whole = a.causal ? min(k_count, (slot.first + wave * 32) / group + ahead + 1) : k_count;
  if constexpr (PARTS) {
    const int64_t piece = ((k_count + a.parts - 1) / a.parts + NK - 1) / NK * NK;
    begin = at.part * piece;
    end = min(end, begin + piece);
  }
  const T *const k = (const T *)a.k + k_begin * a.k_row + at.kv_head * a.k_head;
  const T *const v = (const T *)a.v + k_begin * a.v_row + at.kv_head * a.v_head;
  const float by = a.scale * kLog2e;
  float16v dq[DP / 32] = {};
  for (int64_t j = begin; j < end; j += NK) {
    __syncthreads();
    stage_rows<T, DP, NK, NW * 64>(k_tile, k, a.k_row, j, k_count, a.dim);
    stage_rows<T, DP, NK, NW * 64>(v_tile, v, a.v_row, j, k_count, a.dim);
    __syncthreads();
    const int left = j + NK > whole ? (int)max((int64_t)-1, min((int64_t)NK, seen - j)) : NK;
#pragma unroll
    for (int kb = 0; kb < NK / 32; ++kb) {
      float16v s = {}, dp = {};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) multiply<T>(s, RowTile<T, DP>::rows(k_tile, kb * 32, i, lane), q[i]);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) multiply<T>(dp, RowTile<T, DP>::rows(v_tile, kb * 32, i, lane), g[i]);
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const float ds = __builtin_amdgcn_exp2f(__builtin_fmaf(s[r], by, -lse)) * (dp[r] - delta);
        s[r] = kb * 32 + 8 * (r / 4) + 4 * (lane / 32) + r % 4 < left ? ds : 0.f;
      }
      add_weighted_rows<T, DP>(dq, k_tile, kb * 32, s, lane);
    }
  }
  const float scale = a.scale * pow2(-ds_shift<T>());
  if constexpr (PARTS) {
    const int64_t tile = ((at.slot * a.kv_heads + at.kv_head) * a.parts + at.part) * T_ROWS + wave * 32 + lane % 32;
    if (mine) store_row<float, DP>(a.part_sum + tile * a.dim, dq, scale, a.dim, lane);
  } else if (mine) {
    store_row<T, DP>((T *)a.gq + to * a.dim, dq, scale, a.dim, lane);
  }
}

// Keys' and values' gradients: a wave's 32 keys are columns, the queries of all heads of the group pass by as rows, and
// dk^T = q^T ds, dv^T = g_out^T p take ds and p as they stand.
template <typename T, int DP, int NW, bool PARTS>
__global__ __launch_bounds__(NW * 64) void attention_key_grad_kernel(const AttentionArgs a) {
  constexpr int NQ = tile_rows<T, DP>(), STEPS = DP / (32 / (int)sizeof(T)), T_ROWS = 32 * NW, THREADS = NW * 64;
  using Rows = RowTile<T, DP>;
  __shared__ int4v q_tile[NQ * Rows::CH], g_tile[NQ * Rows::CH];
  __shared__ float4v lse_tile[NQ / 4], delta_tile[NQ / 4];
  const int lane = threadIdx.x % 64, wave = threadIdx.x / 64, group = a.heads / a.kv_heads;
  const Place at = place_of(blockIdx.x, a.kv_heads, PARTS ? a.parts : 1);
  const Slot slot = find_slot(a.k_offsets, a.segments, a.n_k, 1, T_ROWS, at.slot);
  if (slot.first >= slot.length) return;
  int64_t q_begin, q_count;
  partner_rows(a.q_offsets, nullptr, slot.segment, a.segments, a.n_q, q_begin, q_count);
  const int64_t ahead = slot.length - q_count, rows = q_count * group;

  const int64_t key = slot.first + wave * 32 + lane % 32;
  const bool mine = key < slot.length;
  int4v k[STEPS], v[STEPS];
  load_row<T, DP>(k, mine ? (const T *)a.k + (slot.begin + key) * a.k_row + at.kv_head * a.k_head : nullptr, a.dim, lane);
  load_row<T, DP>(v, mine ? (const T *)a.v + (slot.begin + key) * a.v_row + at.kv_head * a.v_head : nullptr, a.dim, lane);

  // rows from which on this lane's key is seen, the workgroup's first key (first of all), the wave's last
  int64_t begin = 0, end = rows;
  const int64_t from = a.causal ? max((int64_t)0, key - ahead) * group : 0;
  const int64_t whole = a.causal ? max((int64_t)0, slot.first + wave * 32 + 31 - ahead) * group : 0;
  if constexpr (PARTS) {
    const int64_t piece = ((rows + a.parts - 1) / a.parts + NQ - 1) / NQ * NQ;
    begin = at.part * piece;
    end = min(end, begin + piece);
  }
  if (a.causal) {
    const int64_t first = max((int64_t)0, slot.first - ahead) * group / NQ * NQ;
    begin = max(begin, first);
  }
  const float by = a.scale * kLog2e, inf = __builtin_inff();
  float16v dk[DP / 32] = {}, dv[DP / 32] = {};
  for (int64_t r0 = begin; r0 < end; r0 += NQ) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < NQ * Rows::CH / THREADS; ++i) {
      const int e = threadIdx.x + i * THREADS, c = e % Rows::CH;
      const int64_t row = r0 + e / Rows::CH, token = q_begin + row / group;
      const int head = at.kv_head * group + (int)(row % group);
      int4v x = {0, 0, 0, 0}, y = {0, 0, 0, 0};
      if (row < rows && c * Rows::E < a.dim) {
        x = *reinterpret_cast<const int4v *>((const T *)a.q + token * a.q_row + head * a.q_head + c * Rows::E);
        y = *reinterpret_cast<const int4v *>((const T *)a.g_out + (token * a.heads + head) * a.dim + c * Rows::E);
      }
      q_tile[Rows::at(e / Rows::CH, c)] = x;
      g_tile[Rows::at(e / Rows::CH, c)] = y;
    }
    for (int e = threadIdx.x; e < NQ; e += THREADS) {
      const int64_t row = r0 + e, to = (q_begin + row / group) * a.heads + at.kv_head * group + row % group;
      const float lse = row < rows ? a.lse[to] : -inf;      // (no keys, no such row: all probabilities 0)
      reinterpret_cast<float *>(lse_tile)[e] = lse == -inf ? inf : lse * kLog2e - p_shift<T>();
      reinterpret_cast<float *>(delta_tile)[e] = row < rows ? a.delta[to] : 0.f;
    }
    __syncthreads();
    const int hidden = r0 < whole ? (int)min((int64_t)NQ, max((int64_t)0, from - r0)) : 0;
#pragma unroll
    for (int qb = 0; qb < NQ / 32; ++qb) {
      float16v p = {}, ds = {};
#pragma unroll
      for (int i = 0; i < STEPS; ++i) multiply<T>(p, Rows::rows(q_tile, qb * 32, i, lane), k[i]);
#pragma unroll
      for (int i = 0; i < STEPS; ++i) multiply<T>(ds, Rows::rows(g_tile, qb * 32, i, lane), v[i]);
#pragma unroll
      for (int r4 = 0; r4 < 4; ++r4) {
        const float4v lse = lse_tile[qb * 8 + 2 * r4 + lane / 32], delta = delta_tile[qb * 8 + 2 * r4 + lane / 32];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * r4 + e;
          p[r] = qb * 32 + 8 * r4 + 4 * (lane / 32) + e < hidden ? 0.f : __builtin_amdgcn_exp2f(__builtin_fmaf(p[r], by, -lse[e]));
          ds[r] = qb * 32 + 8 * r4 + 4 * (lane / 32) + e < hidden ? 0.f : p[r] * ((ds[r] - delta[e]) * pow2(ds_shift<T>() - p_shift<T>()));
        }
      }
      add_weighted_rows<T, DP>(dv, g_tile, qb * 32, p, lane);
      add_weighted_rows<T, DP>(dk, q_tile, qb * 32, ds, lane);
    }
  }
  const float k_by = a.scale * pow2(-ds_shift<T>()), v_by = pow2(-p_shift<T>());
  if (!mine) return;
  if constexpr (PARTS) {
    const int64_t tile = ((at.slot * a.kv_heads + at.kv_head) * a.parts + at.part) * T_ROWS + wave * 32 + lane % 32;
    const int64_t all = attention_slots(a.n_k, a.segments, T_ROWS) * a.kv_heads * a.parts * T_ROWS * a.dim;
    store_row<float, DP>(a.part_sum + tile * a.dim, dk, k_by, a.dim, lane);
    store_row<float, DP>(a.part_sum + all + tile * a.dim, dv, v_by, a.dim, lane);
  } else {
    const int64_t to = ((slot.begin + key) * a.kv_heads + at.kv_head) * a.dim;
    if (a.gk) store_row<T, DP>((T *)a.gk + to, dk, k_by, a.dim, lane);
    if (a.gv) store_row<T, DP>((T *)a.gv + to, dv, v_by, a.dim, lane);
  }
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

// Rows of a workgroup's tile go by the average segment: four waves of 32 share the staged tiles of the other side; where
// segments have hardly more than 32 rows one wave a workgroup leaves none idle.
inline int waves_for(int64_t rows, int64_t segments) { return rows > 48 * segments ? 4 : 1; }

// Pieces of a long axis: until the chip has four workgroups to a CU, none shorter than 256 rows on average.
inline int parts_for(int64_t workgroups, int64_t partners, int64_t segments) {
  const int64_t want = 4 * (int64_t)num_cus() / (workgroups > 0 ? workgroups : 1), most = partners / (segments > 0 ? segments : 1) / 256;
  const int64_t parts = want < most ? want : most;
  return parts < 2 ? 1 : parts > 1024 ? 1024 : (int)parts;
}

template <typename T, int DP, int NW>
int forward(AttentionArgs a) {
  const int group = a.heads / a.kv_heads;
  const int64_t tiles = attention_slots(a.n_q * group, a.segments, 32 * NW) * a.kv_heads;
  a.parts = parts_for((a.n_q * group / (32 * NW) + a.segments) * a.kv_heads, a.n_k, a.segments);
  unsigned grid;
  int rc = grid_of(tiles * a.parts, &grid);
  if (rc != FGMS_OK) return rc;
  if (a.parts == 1) {
    segment_attention_kernel<T, DP, NW, false><<<grid, NW * 64, 0, a.stream>>>(a);
    return launched("segment attention");
  }
  const size_t rows = (size_t)tiles * a.parts * 32 * NW;
  rc = workspace_get(a.stream, kSlotAttention, rows * (a.dim + 1) * sizeof(float), (void **)&a.part_sum);
  if (rc != FGMS_OK) return rc;
  a.part_lse = a.part_sum + rows * a.dim;
  segment_attention_kernel<T, DP, NW, true><<<grid, NW * 64, 0, a.stream>>>(a);
  join_parts_kernel<T, NW, false><<<(unsigned)tiles, 256, 0, a.stream>>>(a, a.q_offsets, a.n_q, group, a.part_sum, (T *)a.out, 1.f);
  return launched("segment attention");
}

template <typename T, int DP, int NW>
int query_grad(AttentionArgs a) {
  const int group = a.heads / a.kv_heads;
  const int64_t tiles = attention_slots(a.n_q * group, a.segments, 32 * NW) * a.kv_heads;
  a.parts = parts_for((a.n_q * group / (32 * NW) + a.segments) * a.kv_heads, a.n_k, a.segments);
  unsigned grid;
  int rc = grid_of(tiles * a.parts, &grid);
  if (rc != FGMS_OK) return rc;
  if (a.parts == 1) {
    attention_query_grad_kernel<T, DP, NW, false><<<grid, NW * 64, 0, a.stream>>>(a);
    return launched("segment attention, queries' gradient");
  }
  rc = workspace_get(a.stream, kSlotAttention, (size_t)tiles * a.parts * 32 * NW * a.dim * sizeof(float), (void **)&a.part_sum);
  if (rc != FGMS_OK) return rc;
  attention_query_grad_kernel<T, DP, NW, true><<<grid, NW * 64, 0, a.stream>>>(a);
  join_parts_kernel<T, NW, true><<<(unsigned)tiles, 256, 0, a.stream>>>(a, a.q_offsets, a.n_q, group, a.part_sum, (T *)a.gq, 1.f);
  return launched("segment attention, queries' gradient");
}

template <typename T, int DP, int NW>
int key_grad(AttentionArgs a) {
  const int64_t tiles = attention_slots(a.n_k, a.segments, 32 * NW) * a.kv_heads;
  a.parts = parts_for((a.n_k / (32 * NW) + a.segments) * a.kv_heads, a.n_q * (a.heads / a.kv_heads), a.segments);
  unsigned grid;
  int rc = grid_of(tiles * a.parts, &grid);
  if (rc != FGMS_OK) return rc;
  if (a.parts == 1) {
    attention_key_grad_kernel<T, DP, NW, false><<<grid, NW * 64, 0, a.stream>>>(a);
    return launched("segment attention, keys' gradients");
  }
  const size_t all = (size_t)tiles * a.parts * 32 * NW * a.dim;
  rc = workspace_get(a.stream, kSlotAttention, 2 * all * sizeof(float), (void **)&a.part_sum);
  if (rc != FGMS_OK) return rc;
  attention_key_grad_kernel<T, DP, NW, true><<<grid, NW * 64, 0, a.stream>>>(a);
  if (a.gk) join_parts_kernel<T, NW, true><<<(unsigned)tiles, 256, 0, a.stream>>>(a, a.k_offsets, a.n_k, 1, a.part_sum, (T *)a.gk, 1.f);
  if (a.gv) join_parts_kernel<T, NW, true><<<(unsigned)tiles, 256, 0, a.stream>>>(a, a.k_offsets, a.n_k, 1, a.part_sum + all, (T *)a.gv, 1.f);
  return launched("segment attention, keys' gradients");
}

template <typename T, int DP>
int forward_any(const AttentionArgs &a) {
  return waves_for(a.n_q * (a.heads / a.kv_heads), a.segments) == 4 ? forward<T, DP, 4>(a) : forward<T, DP, 1>(a);
}

template <typename T, int DP>
int backward_any(const AttentionArgs &a) {
  const int64_t rows = a.n_q * a.heads;
  unsigned grid;
  int rc = grid_of((rows + 31) / 32, &grid);
  if (rc == FGMS_OK && rows > 0) {
    attention_delta_kernel<T><<<grid, 256, 0, a.stream>>>((const T *)a.g_out, (const T *)a.out, a.delta, rows, a.dim);
    rc = launched("segment attention, backward");
  }
  if (rc == FGMS_OK && a.gq && a.n_q > 0)
    rc = waves_for(a.n_q * (a.heads / a.kv_heads), a.segments) == 4 ? query_grad<T, DP, 4>(a) : query_grad<T, DP, 1>(a);
  if (rc == FGMS_OK && (a.gk || a.gv) && a.n_k > 0)
    rc = waves_for(a.n_k, a.segments) == 4 ? key_grad<T, DP, 4>(a) : key_grad<T, DP, 1>(a);
  return rc;
}

}  // namespace

template <typename T>
int attention_fwd(const AttentionArgs &a) {
  return a.dim <= 32 ? forward_any<T, 32>(a) : a.dim <= 64 ? forward_any<T, 64>(a) : forward_any<T, 128>(a);
}

template <typename T>
int attention_bwd(const AttentionArgs &a) {
  return a.dim <= 32 ? backward_any<T, 32>(a) : a.dim <= 64 ? backward_any<T, 64>(a) : backward_any<T, 128>(a);
}

}  // namespace fgms
