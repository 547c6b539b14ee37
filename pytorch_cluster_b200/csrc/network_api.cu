// extern "C" entry points of gather_rows, norm_rotate and attention: argument checks and kernel selection.
#include <float.h>
#include <math.h>

#include <atomic>
#include <initializer_list>

#include "attention.cuh"
#include "common.cuh"
#include "launchers.h"

namespace b200c {

int check_device();  // api.cu

static bool is_network_type(int dtype) { return dtype == B200C_F32 || dtype == B200C_F16 || dtype == B200C_BF16; }
static size_t elem_bytes(int dtype) { return dtype == B200C_F32 ? 4 : 2; }
constexpr int64_t MOST_ROWS = 0x7fffffffLL;
constexpr int64_t MOST_GATHER_CHANNELS = 65536;
constexpr int64_t MOST_SEGMENTS = 1ll << 30;  // segments are bisected with 32-bit numbers
// Scores are divided by a cap and multiplied by it again.  Above 2^100 it bends no score below 2^88, and those quotients
// would leave the normal numbers of fp32: such a cap is none.
constexpr float MOST_CAP = 1.2676506e30f;

static std::atomic<int32_t *> attention_report{nullptr};

// what every workspace is carved from
static bool aligned_workspace(const void *p) { return ((uintptr_t)p & 15) == 0; }
// whether all pointers lie at multiples of their elements
static bool aligned_to(size_t bytes, std::initializer_list<const void *> pointers) {
  for (const void *p : pointers)
    if ((uintptr_t)p & (bytes - 1)) return false;
  return true;
}

static int check_gather(const void *in, const int64_t *index, int64_t rows, int64_t edges, int64_t channels, int dtype,
                        const void *out) {
  B200C_CHECK_ARG(is_network_type(dtype), "unsupported dtype");
  B200C_CHECK_ARG(rows >= 0 && edges >= 0 && channels >= 1, "Input mismatch");
  B200C_CHECK_ARG(rows <= MOST_ROWS && edges <= MOST_ROWS, "more than 2^31-1 rows or edges are not supported");
  B200C_CHECK_ARG(channels <= MOST_GATHER_CHANNELS, "more than 65536 channels are not supported");
  B200C_CHECK_ARG((edges == 0 || index != nullptr) && (rows == 0 || edges == 0 || (in != nullptr && out != nullptr)),
                  "null pointer");
  B200C_CHECK_ARG(aligned_to(elem_bytes(dtype), {in, out}) && aligned_to(8, {index}), "misaligned pointer");
  return check_device();
}

static int check_rotate(const b200c_norm_rotate_side_t *q, const b200c_norm_rotate_side_t *k, const void *freq, int dims,
                        int channels, int pos_f64, int freq_f64, float eps, int dtype, bool forward,
                        cudaStream_t stream, NormRotateArgs &a) {
  B200C_CHECK_ARG(q != nullptr && k != nullptr && freq != nullptr, "null pointer");
  B200C_CHECK_ARG(is_network_type(dtype), "unsupported dtype");
  B200C_CHECK_ARG(channels >= 2 && channels <= 256 && channels % 2 == 0, "channels must be even and at most 256");
  B200C_CHECK_ARG(dims >= 1 && dims <= 8, "1 to 8 coordinates are supported");
  B200C_CHECK_ARG(aligned_to(freq_f64 ? 8 : 4, {freq}), "misaligned pointer");
  const b200c_norm_rotate_side_t *sides[2] = {q, k};
  for (int i = 0; i < 2; ++i) {
    const b200c_norm_rotate_side_t &s = *sides[i];
    B200C_CHECK_ARG(s.rows >= 0 && s.rows <= MOST_ROWS, "more than 2^31-1 rows are not supported");
    B200C_CHECK_ARG(s.heads >= 1 && s.heads <= 1024, "1 to 1024 heads are supported");
    if (s.rows > 0) {
      B200C_CHECK_ARG(s.x && s.pos, "null pointer");
      B200C_CHECK_ARG(forward ? s.y != nullptr : (s.dy && s.dx), "null pointer");
      B200C_CHECK_ARG(aligned_to(elem_bytes(dtype), {s.x, forward ? s.y : s.dx, forward ? nullptr : s.dy}) &&
                          aligned_to(pos_f64 ? 8 : 4, {s.pos}),
                      "misaligned pointer");
    }
    B200C_CHECK_ARG(aligned_to(4, {s.weight, forward ? nullptr : s.dweight}), "misaligned pointer");
    a.side[i] = s;
    if (s.rows == 0) a.side[i].x = a.side[i].y = a.side[i].dx = nullptr, a.side[i].dy = nullptr;
    a.dweight[i] = forward ? nullptr : s.dweight;
  }
  a.freq = freq;
  a.dims = dims;
  a.half = channels / 2;
  a.pos_f64 = pos_f64;
  a.freq_f64 = freq_f64;
  a.eps = eps;
  a.dtype = dtype;
  a.joint = q->rows == k->rows && q->pos == k->pos;
  a.stream = stream;
  return check_device();
}

static int check_attention(const b200c_attention_t *a) {
  B200C_CHECK_ARG(a != nullptr, "null pointer");
  B200C_CHECK_ARG(is_network_type(a->dtype), "unsupported dtype");
  B200C_CHECK_ARG(a->m >= 0 && a->n >= 0 && a->m <= MOST_ROWS && a->n <= MOST_ROWS,
                  "more than 2^31-1 rows are not supported");
  B200C_CHECK_ARG(a->channels >= 1 && a->channels <= AT_MAX_CHANNELS, "1 to 128 channels are supported");
  B200C_CHECK_ARG(a->groups >= 1 && a->heads >= a->groups && a->heads % a->groups == 0 && a->heads <= 1024,
                  "heads must be a multiple of the key heads, at most 1024");
  B200C_CHECK_ARG(a->dims >= 0 && a->dims <= AT_MAX_DIMS, "0 to 8 coordinates are supported");
  B200C_CHECK_ARG(a->m * a->heads <= (1ll << 33), "more than 2^33 rows of all heads are not supported");
  B200C_CHECK_ARG((a->ptr_q == nullptr) == (a->ptr_k == nullptr), "Input mismatch");
  B200C_CHECK_ARG(a->ptr_q == nullptr ? a->num_segments == 1 : a->num_segments >= 1, "Input mismatch");
  B200C_CHECK_ARG(a->num_segments <= MOST_SEGMENTS, "more than 2^30 segments are not supported");
  B200C_CHECK_ARG(a->m == 0 || a->q, "null pointer");
  B200C_CHECK_ARG(a->n == 0 || (a->k && a->v), "null pointer");
  B200C_CHECK_ARG(a->dims == 0 || (a->slope && (a->m == 0 || a->pos_q) && (a->n == 0 || a->pos_k)), "null pointer");
  B200C_CHECK_ARG(isfinite(a->scale) && isfinite(a->cap), "scale and cap must be finite numbers");
  B200C_CHECK_ARG(!(a->cap > 0.f) || (a->cap >= FLT_MIN && isfinite(2.f * AT_LOG2E * fabsf(a->scale) / a->cap)),
                  "cap must be at least 2^-126, and scale / cap a number of 32 bits");
  B200C_CHECK_ARG(aligned_to(elem_bytes(a->dtype), {a->q, a->k, a->v}) && aligned_to(8, {a->ptr_q, a->ptr_k}) &&
                      (a->dims == 0 || aligned_to(4, {a->pos_q, a->pos_k, a->slope})),
                  "misaligned pointer");
  return B200C_OK;
}

static b200c_attention_t without_idle_cap(const b200c_attention_t &a) {
  b200c_attention_t p = a;
  if (p.cap > MOST_CAP) p.cap = 0.f;
  return p;
}

}  // namespace b200c

using namespace b200c;

extern "C" int b200c_gather_rows(const void *x, const int64_t *index, int64_t rows, int64_t edges, int64_t channels,
                                 float scale, int dtype, void *out, b200c_stream_t stream) {
  const int st = check_gather(x, index, rows, edges, channels, dtype, out);
  if (st != B200C_OK || edges == 0) return st;
  B200C_CHECK_ARG(out != nullptr, "null pointer");
  return launch_gather_rows(x, index, rows, edges, channels, scale, dtype, out, (cudaStream_t)stream);
}

extern "C" size_t b200c_gather_rows_workspace_bytes(int64_t rows, int64_t edges, int64_t channels) {
  if (rows < 0 || edges <= 0 || channels < 1 || rows > MOST_ROWS || edges > MOST_ROWS || channels > MOST_GATHER_CHANNELS)
    return 0;  // such calls are refused, or need none
  return gather_rows_workspace_bytes(rows, edges, channels);
}

extern "C" int b200c_gather_rows_backward(const void *dout, const int64_t *index, int64_t rows, int64_t edges,
                                          int64_t channels, float scale, int dtype, void *dx, void *workspace,
                                          size_t workspace_bytes, b200c_stream_t stream) {
  const int st = check_gather(dout, index, rows, edges, channels, dtype, dx);
  if (st != B200C_OK || rows == 0) return st;
  B200C_CHECK_ARG(dx != nullptr, "null pointer");
  B200C_CHECK_ARG(aligned_workspace(workspace), "misaligned workspace");
  if (edges == 0) {
    B200C_CUDA(cudaMemsetAsync(dx, 0, (size_t)rows * channels * elem_bytes(dtype), (cudaStream_t)stream));
    return B200C_OK;
  }
  const size_t need = gather_rows_workspace_bytes(rows, edges, channels);
  if (workspace == nullptr || workspace_bytes < need) {
    set_error("gather_rows workspace too small: %zu < %zu", workspace_bytes, need);
    return B200C_ERR_WORKSPACE;
  }
  return launch_gather_rows_backward(dout, index, rows, edges, channels, scale, dtype, dx, workspace,
                                     (cudaStream_t)stream);
}

extern "C" int b200c_norm_rotate(const b200c_norm_rotate_side_t *q, const b200c_norm_rotate_side_t *k, const void *freq,
                                 int dims, int channels, int pos_f64, int freq_f64, float eps, int dtype,
                                 b200c_stream_t stream) {
  NormRotateArgs a{};
  const int st = check_rotate(q, k, freq, dims, channels, pos_f64, freq_f64, eps, dtype, true, (cudaStream_t)stream, a);
  if (st != B200C_OK || (q->rows == 0 && k->rows == 0)) return st;
  return launch_norm_rotate(a, true, nullptr);
}

extern "C" size_t b200c_norm_rotate_workspace_bytes(int channels) {
  return channels < 2 || channels > 256 ? 0 : norm_rotate_workspace_bytes(channels);
}

extern "C" int b200c_norm_rotate_backward(const b200c_norm_rotate_side_t *q, const b200c_norm_rotate_side_t *k,
                                          const void *freq, int dims, int channels, int pos_f64, int freq_f64, float eps,
                                          int dtype, void *workspace, size_t workspace_bytes, b200c_stream_t stream) {
  NormRotateArgs a{};
  const int st = check_rotate(q, k, freq, dims, channels, pos_f64, freq_f64, eps, dtype, false, (cudaStream_t)stream, a);
  if (st != B200C_OK) return st;
  B200C_CHECK_ARG(aligned_workspace(workspace), "misaligned workspace");
  const size_t need = norm_rotate_workspace_bytes(channels);
  if ((a.dweight[0] || a.dweight[1]) && (workspace == nullptr || workspace_bytes < need)) {
    set_error("norm_rotate workspace too small: %zu < %zu", workspace_bytes, need);
    return B200C_ERR_WORKSPACE;
  }
  if (q->rows == 0 && k->rows == 0) {
    for (float *dw : a.dweight)
      if (dw) B200C_CUDA(cudaMemsetAsync(dw, 0, (size_t)channels * 4, a.stream));
    return B200C_OK;
  }
  return launch_norm_rotate(a, false, (float *)workspace);
}

extern "C" void b200c_attention_set_report(int32_t *word) { attention_report.store(word); }
extern "C" int32_t *b200c_attention_report(void) { return attention_report.load(); }

static size_t align256(size_t v) { return (v + 255) / 256 * 256; }

extern "C" size_t b200c_attention_workspace_bytes(const b200c_attention_t *a) {
  if (check_attention(a) != B200C_OK) return 0;
  const b200c_attention_t p = without_idle_cap(*a);
  const size_t few = attention_few_workspace_bytes(p);
  if (few > 0) return few;
  const int splits = attention_tensor_splits(p);
  if (splits > 1) return (size_t)p.m * p.heads * splits * (p.channels + 2) * 4;
  return attention_tensor_order_bytes(p);
}

extern "C" int b200c_attention_forward(const b200c_attention_t *args, void *out, void *rest, float *lse, void *workspace,
                                       size_t workspace_bytes, b200c_stream_t stream) {
  int st = check_attention(args);
  if (st != B200C_OK) return st;
  const b200c_attention_t effective = without_idle_cap(*args), *p = &effective;
  B200C_CHECK_ARG(aligned_workspace(workspace), "misaligned workspace");
  B200C_CHECK_ARG(aligned_to(elem_bytes(p->dtype), {out, rest}) && aligned_to(4, {lse}), "misaligned pointer");
  if ((st = check_device()) != B200C_OK || p->m == 0) return st;
  B200C_CHECK_ARG(out != nullptr, "null output pointer");
  const size_t need = b200c_attention_workspace_bytes(p);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    set_error("attention workspace too small: %zu < %zu", workspace_bytes, need);
    return B200C_ERR_WORKSPACE;
  }
  AttnArgs a;
  a.p = *p;
  a.out = out;
  a.rest = rest;
  a.lse = lse;
  a.stream = (cudaStream_t)stream;
  a.report = attention_report.load();
  const int splits = attention_few_splits(*p);
  if (splits > 0) return launch_attention_few(a, splits, workspace);
  if (attention_tensor_applicable(*p) && (((uintptr_t)out | (uintptr_t)rest) & 15) == 0) {
    // the statistics of a training step need the exact sums, which the joined parts do not carry
    if (lse == nullptr && rest == nullptr) a.splits = attention_tensor_splits(*p);
    if (a.splits > 1)
      a.parts = (float *)workspace;
    else if (attention_tensor_splits(*p) == 1 && need > 0)
      a.order = (int *)workspace;
    return launch_attention_tensor_forward(a);
  }
  return launch_attention_plain_forward(a);
}

extern "C" size_t b200c_attention_backward_workspace_bytes(const b200c_attention_t *a) {
  if (check_attention(a) != B200C_OK) return 0;
  // D, the largest norms, order; never 0
  return align256((size_t)a->m * a->heads * 4) + align256(attention_norms_bytes(*a) + 1) +
         attention_tensor_order_bytes(without_idle_cap(*a));
}

extern "C" int b200c_attention_backward(const b200c_attention_t *args, const void *out, const void *rest,
                                        const float *lse, const void *dout, void *dq, void *dk, void *dv, void *workspace,
                                        size_t workspace_bytes, b200c_stream_t stream) {
  int st = check_attention(args);
  if (st != B200C_OK) return st;
  const b200c_attention_t effective = without_idle_cap(*args), *p = &effective;
  B200C_CHECK_ARG(aligned_workspace(workspace), "misaligned workspace");
  B200C_CHECK_ARG(aligned_to(elem_bytes(p->dtype), {out, rest, dout, dq, dk, dv}) && aligned_to(4, {lse}),
                  "misaligned pointer");
  if ((st = check_device()) != B200C_OK) return st;
  B200C_CHECK_ARG(p->m == 0 || (out && lse && dout), "null pointer");
  B200C_CHECK_ARG((dk == nullptr) == (dv == nullptr), "dk and dv come together");
  const size_t need = b200c_attention_backward_workspace_bytes(p);
  if (need > 0 && (workspace == nullptr || workspace_bytes < need)) {
    set_error("attention workspace too small: %zu < %zu", workspace_bytes, need);
    return B200C_ERR_WORKSPACE;
  }
  AttnArgs a;
  a.p = *p;
  a.out = (void *)out;
  a.rest = (void *)rest;
  a.lse = (float *)lse;
  a.dout = dout;
  a.delta = (const float *)workspace;
  a.dq = dq;
  a.dk = dk;
  a.dv = dv;
  a.stream = (cudaStream_t)stream;
  a.report = attention_report.load();
  float *norms = (float *)((char *)workspace + align256((size_t)p->m * p->heads * 4));
  a.norms = norms;
  if (attention_tensor_order_bytes(*p) > 0) a.order = (int *)((char *)norms + align256(attention_norms_bytes(*p) + 1));
  if ((st = launch_attention_delta(a, (float *)workspace, norms)) != B200C_OK) return st;
  if (attention_tensor_applicable(*p) &&
      (((uintptr_t)dout | (uintptr_t)dq | (uintptr_t)dk | (uintptr_t)dv) & 15) == 0)
    return launch_attention_tensor_backward(a);
  return launch_attention_plain_backward(a);
}
