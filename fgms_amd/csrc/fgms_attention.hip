// extern "C" entry points of attention over ragged segments and of the norms and rotations in front of it:
// argument checks and the choice of a type.
#include "fgms_attention.h"

#include <math.h>

#include "fgms_norm_rotary.h"

namespace fgms {
namespace {

bool known_dtype(int dtype) { return dtype == FGMS_F32 || dtype == FGMS_F16 || dtype == FGMS_BF16; }
int64_t element_bytes(int dtype) { return dtype == FGMS_F32 ? 4 : 2; }

int refuse(const char *what, const char *why) {
  set_error("%s: %s", what, why);
  return FGMS_E_INVALID;
}

constexpr int64_t kMostRowBytes = 16 << 20;      // 64 rows of a tile, and 512 MB between the heads of a group: below 2^31
constexpr int64_t kMostRows = INT32_MAX - (1 << 25);

bool aligned(const void *p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

// A strided [rows, heads, dim] tensor that the kernels read 16 bytes at a time (`there`: it has elements).
int check_rows(const char *what, const void *p, bool there, int64_t row, int64_t head, int dtype) {
  if (!there) return FGMS_OK;
  if (!p) return refuse(what, "null pointer");
  const int64_t bytes = element_bytes(dtype);
  if (!aligned(p) || row < 0 || head < 0 || row * bytes % 16 || head * bytes % 16)
    return refuse(what, "rows and heads have to begin on 16 bytes");
  // (a tile's rows are reached by 32-bit offsets)
  if (row * bytes > kMostRowBytes) return refuse(what, "rows lie too far apart");
  return FGMS_OK;
}

int check_shape(const char *what, int heads, int kv_heads, int dim, int dtype) {
  if (!known_dtype(dtype)) return refuse(what, "dtype must be FGMS_F32, FGMS_F16 or FGMS_BF16");
  if (dim < 8 || dim > 128 || dim % 8) return refuse(what, "the channels of a head must be a multiple of 8 from 8 to 128");
  if (heads < 1 || kv_heads < 0 || heads > 65536 || kv_heads > 65536) return refuse(what, "there must be 1 to 65536 heads");
  return FGMS_OK;
}

int check_norm_rotary(const char *what, const NormRotaryArgs &a) {
  int rc = check_shape(what, a.heads[0], a.heads[1], a.dim, a.dtype);
  if (rc != FGMS_OK) return rc;
  if (a.n < 0 || a.n > INT32_MAX) return refuse(what, "between 0 and 2^31 - 1 rows");
  if (!(a.eps >= 0.f) || !(a.eps < 1e30f)) return refuse(what, "eps must be finite and not negative");
  if (a.axes < 1 || a.axes > kMaxAxes) return refuse(what, "one to four axes");
  int64_t pairs = 0;
  for (int i = 0; i < a.axes; ++i) {
    if (a.sections[i] < 0) return refuse(what, "a section is negative");
    pairs += a.sections[i];
  }
  if (pairs > a.dim / 2) return refuse(what, "the sections add up to more than half the channels of a head");
  if (a.n > 0 && pairs > 0 && (!a.coords || !a.freqs)) return refuse(what, "null pointer");
  for (int i = 0; i < 2; ++i) {
    if ((rc = check_rows(what, a.x[i], a.n > 0 && a.heads[i] > 0, a.row[i], a.head[i], a.dtype))) return rc;
    if (!aligned(a.scale[i])) return refuse(what, "scales have to begin on 16 bytes");
  }
  return FGMS_OK;
}

int check_attention(const char *what, const AttentionArgs &a, int64_t n_q, int64_t n_k) {
  int rc = check_shape(what, a.heads, a.kv_heads, a.dim, a.dtype);
  if (rc != FGMS_OK) return rc;
  if (a.kv_heads < 1 || a.heads % a.kv_heads) return refuse(what, "the query heads must be a multiple of the key heads");
  if (n_q < 0 || n_k < 0 || n_k > kMostRows || n_q > kMostRows / (a.heads / a.kv_heads))
    return refuse(what, "the rows, times the heads of a group, must be fewer than 2^31 - 2^25");
  if (a.segments < 0 || a.segments > kMostRows) return refuse(what, "the number of segments is out of range");
  if (!a.q_offsets || !a.k_offsets) return refuse(what, "null offsets");
  if (!(a.scale > 0.f) || !(a.scale < 1e30f)) return refuse(what, "scale must be positive and finite");
  if ((rc = check_rows(what, a.q, n_q > 0, a.q_row, a.q_head, a.dtype))) return rc;
  if ((rc = check_rows(what, a.k, n_k > 0, a.k_row, a.k_head, a.dtype))) return rc;
  if ((rc = check_rows(what, a.v, n_k > 0, a.v_row, a.v_head, a.dtype))) return rc;
  // (a tile's rows end where the buffer over them does)
  if ((n_k > 1 && (a.k_row < a.dim || a.v_row < a.dim))) return refuse(what, "rows of k and v overlap");
  if (a.q_head > ((int64_t)512 << 20) / element_bytes(a.dtype) / (a.heads / a.kv_heads))
    return refuse(what, "the heads of a group lie too far apart");
  return FGMS_OK;
}

AttentionArgs attention_args(const void *q, const void *k, const void *v, const int32_t *q_offsets, const int32_t *k_offsets,
                             const int32_t *k_lengths, int64_t n_q, int64_t n_k, int segments, int heads, int kv_heads, int dim,
                             int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int64_t v_row, int64_t v_head,
                             int causal, float scale, int dtype, void *stream) {
  AttentionArgs a{};
  a.q = q, a.k = k, a.v = v;
  a.q_offsets = q_offsets, a.k_offsets = k_offsets, a.k_lengths = k_lengths;
  a.n_q = (int)n_q, a.n_k = (int)n_k, a.segments = segments, a.heads = heads, a.kv_heads = kv_heads, a.dim = dim;
  a.q_row = q_row, a.q_head = q_head, a.k_row = k_row, a.k_head = k_head, a.v_row = v_row, a.v_head = v_head;
  // (a single row may carry any stride, 0 where it was expanded; the kernels end a row of k and v where its stride does)
  if (n_k == 1) a.k_row = a.v_row = dim;
  a.causal = causal, a.scale = scale, a.dtype = dtype, a.stream = (hipStream_t)stream, a.parts = 1;
  return a;
}

NormRotaryArgs norm_rotary_args(const void *q, const void *k, const void *q_scale, const void *k_scale, const int32_t *coords,
                                const float *freqs, int64_t n, int q_heads, int k_heads, int dim, int64_t q_row, int64_t q_head,
                                int64_t k_row, int64_t k_head, int axes, const int *sections, int interleaved, float eps, int dtype,
                                void *stream) {
  NormRotaryArgs a{};
  a.x[0] = q, a.x[1] = k, a.scale[0] = q_scale, a.scale[1] = k_scale;
  a.heads[0] = q_heads, a.heads[1] = k_heads;
  a.row[0] = q_row, a.row[1] = k_row, a.head[0] = q_head, a.head[1] = k_head;
  a.coords = coords, a.freqs = freqs, a.axes = axes;
  for (int i = 0; sections && i < axes && i < kMaxAxes; ++i) a.sections[i] = sections[i];
  a.n = n, a.dim = dim, a.interleaved = interleaved, a.eps = eps, a.dtype = dtype, a.stream = (hipStream_t)stream;
  return a;
}

}  // namespace
}  // namespace fgms

using namespace fgms;

extern "C" int fgms_norm_rotary_fwd(const void *q, const void *k, const void *q_scale, const void *k_scale, const int32_t *coords,
                                    const float *freqs, void *q_out, void *k_out, int64_t n, int q_heads, int k_heads, int head_dim,
                                    int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int axes, const int *sections,
                                    int interleaved, float eps, int dtype, void *stream) {
  static const char what[] = "fgms_norm_rotary_fwd";
  if (!sections) return refuse(what, "null pointer");
  NormRotaryArgs a = norm_rotary_args(q, k, q_scale, k_scale, coords, freqs, n, q_heads, k_heads, head_dim, q_row, q_head, k_row, k_head,
                                      axes, sections, interleaved, eps, dtype, stream);
  const int rc = check_norm_rotary(what, a);
  if (rc != FGMS_OK || n == 0) return rc;
  if (!q_out || (k_heads > 0 && !k_out) || !aligned(q_out) || !aligned(k_out)) return refuse(what, "results have to begin on 16 bytes");
  a.y[0] = q_out, a.y[1] = k_out;
  return launch_norm_rotary(a, false);
}

extern "C" int fgms_norm_rotary_bwd(const void *q_out_grad, const void *k_out_grad, const void *q, const void *k, const void *q_scale,
                                    const void *k_scale, const int32_t *coords, const float *freqs, void *q_grad, void *k_grad,
                                    void *q_scale_grad, void *k_scale_grad, int64_t n, int q_heads, int k_heads, int head_dim,
                                    int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int axes, const int *sections,
                                    int interleaved, float eps, int dtype, void *stream) {
  static const char what[] = "fgms_norm_rotary_bwd";
  if (!sections) return refuse(what, "null pointer");
  NormRotaryArgs a = norm_rotary_args(q, k, q_scale, k_scale, coords, freqs, n, q_heads, k_heads, head_dim, q_row, q_head, k_row, k_head,
                                      axes, sections, interleaved, eps, dtype, stream);
  const int rc = check_norm_rotary(what, a);
  if (rc != FGMS_OK) return rc;
  a.gscale[0] = q_scale_grad, a.gscale[1] = k_scale_grad;      // (without key heads: zeros)
  if (n == 0) {
    const size_t bytes = (size_t)head_dim * element_bytes(dtype);
    int filled = FGMS_OK;
    for (int i = 0; i < 2 && filled == FGMS_OK; ++i)
      if (a.gscale[i]) filled = launch_fill_zero(a.gscale[i], bytes, a.stream);
    return filled;
  }
  a.gy[0] = q_out_grad, a.gy[1] = k_out_grad, a.gx[0] = q_grad, a.gx[1] = k_grad;
  for (int i = 0; i < 2; ++i) {
    if (a.heads[i] > 0 && !a.gy[i]) return refuse(what, "null pointer");
    if (!aligned(a.gy[i]) || !aligned(a.gx[i])) return refuse(what, "gradients have to begin on 16 bytes");
  }
  return launch_norm_rotary(a, true);
}

extern "C" int fgms_segment_attention_fwd(const void *q, const void *k, const void *v, void *out, float *lse, const int32_t *q_offsets,
                                          const int32_t *k_offsets, const int32_t *k_lengths, int64_t n_q, int64_t n_k, int segments,
                                          int heads, int kv_heads, int head_dim, int64_t q_row, int64_t q_head, int64_t k_row,
                                          int64_t k_head, int64_t v_row, int64_t v_head, int causal, float scale, int dtype, void *stream) {
  static const char what[] = "fgms_segment_attention_fwd";
  AttentionArgs a = attention_args(q, k, v, q_offsets, k_offsets, k_lengths, n_q, n_k, segments, heads, kv_heads, head_dim, q_row, q_head,
                                   k_row, k_head, v_row, v_head, causal, scale, dtype, stream);
  const int rc = check_attention(what, a, n_q, n_k);
  if (rc != FGMS_OK || n_q == 0) return rc;
  if (!out || !aligned(out)) return refuse(what, "the result has to begin on 16 bytes");
  a.out = out, a.lse = lse;
  return launch_attention_fwd(a);
}

extern "C" int fgms_segment_attention_bwd(const void *out_grad, const void *q, const void *k, const void *v, const void *out,
                                          const float *lse, void *q_grad, void *k_grad, void *v_grad, const int32_t *q_offsets,
                                          const int32_t *k_offsets, int64_t n_q, int64_t n_k, int segments, int heads, int kv_heads,
                                          int head_dim, int64_t q_row, int64_t q_head, int64_t k_row, int64_t k_head, int64_t v_row,
                                          int64_t v_head, int causal, float scale, int dtype, void *stream) {
  static const char what[] = "fgms_segment_attention_bwd";
  AttentionArgs a = attention_args(q, k, v, q_offsets, k_offsets, nullptr, n_q, n_k, segments, heads, kv_heads, head_dim, q_row, q_head,
                                   k_row, k_head, v_row, v_head, causal, scale, dtype, stream);
  const int rc = check_attention(what, a, n_q, n_k);
  if (rc != FGMS_OK) return rc;
  if (n_q > 0 && (!out_grad || !out || !lse)) return refuse(what, "null pointer");
  if (!aligned(out_grad) || !aligned(out) || !aligned(q_grad) || !aligned(k_grad) || !aligned(v_grad))
    return refuse(what, "gradients and the result have to begin on 16 bytes");
  a.g_out = out_grad, a.out = const_cast<void *>(out), a.lse = const_cast<float *>(lse);
  a.gq = q_grad, a.gk = k_grad, a.gv = v_grad;
  return launch_attention_bwd(a);
}

namespace fgms {

int launch_attention_fwd(AttentionArgs a) {
  return a.dtype == FGMS_F32 ? attention_fwd<float>(a) : a.dtype == FGMS_F16 ? attention_fwd<_Float16>(a) : attention_fwd<__bf16>(a);
}

int launch_attention_bwd(AttentionArgs a) {
  const StreamTurn turn(a.stream);
  const int rc = workspace_get(a.stream, kSlotAttentionDelta, (size_t)a.n_q * a.heads * sizeof(float), (void **)&a.delta);
  if (rc != FGMS_OK) return rc;
  return a.dtype == FGMS_F32 ? attention_bwd<float>(a) : a.dtype == FGMS_F16 ? attention_bwd<_Float16>(a) : attention_bwd<__bf16>(a);
}

}  // namespace fgms
