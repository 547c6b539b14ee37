// Softmax attention inside the examples of a ragged batch (shared by the attention_*.cu kernels).
//
// For query i (row of q, head h) and every key j of the same example (segment of ptr_q / ptr_k):
//   t_ij = scale q_i . k_j           with a cap: t_ij = cap tanh(scale q_i . k_j / cap)
//   z_ij = t_ij - slope_h |pos_i - pos_j|
//   o_i  = sum_j p_ij v_j,  p_ij = exp(z_ij) / sum_j exp(z_ij)
// Head h reads key/value head h / (heads / groups).  A row without keys (its example has none, or it belongs
// to no example) and a row whose scores are all -inf give zeros.
//
// Backward, with D_i = do_i . o_i:  dp_ij = do_i . v_j,  ds_ij = p_ij (dp_ij - D_i) (1 - (t_ij / cap)^2),
//   dv_j = sum_i p_ij do_i,  dq_i = scale sum_j ds_ij k_j,  dk_j = scale sum_i ds_ij q_i,
// the sums over i running over all heads of the key's group.  p is formed again from the forward pass's
//   lse_i = log2 sum_j exp(z_ij)      (+inf for rows that give zeros, so that p = 0),
// stored [heads, m].  D is a small difference of what the rounded outputs give where few keys share the weight, so the
// forward pass of a training step also keeps what rounding took from out, in out's type.  Scores are kept in units of
// log 2: exp(z) = 2^(z log2 e).
#pragma once

#include "common.cuh"

namespace b200c {

constexpr float AT_LOG2E = 1.4426950408889634f;
constexpr int AT_MAX_CHANNELS = 128;
constexpr int AT_MAX_DIMS = 8;
// The kernels for 16-bit types form tanh(y) as 1 - 2 / (e^2y + 1), right to 4e-7 absolutely, which the cap multiplies;
// above this cap (1e-4 of a score) CUDA's tanh is called, in the plain kernels.
constexpr float AT_MAX_FAST_CAP = 256.f;

struct AttnArgs {
  b200c_attention_t p;
  void *out = nullptr;           // [m, heads, channels]
  float *lse = nullptr;          // [heads, m]; forward: may be null
  void *rest = nullptr;          // [m, heads, channels]: what rounding took from out, in out's type; may be null
  const void *dout = nullptr;    // [m, heads, channels]
  const float *delta = nullptr;  // [heads, m]: D_i
  void *dq = nullptr, *dk = nullptr, *dv = nullptr;  // [m, heads, channels], [n, groups, channels] x 2
  const float *norms = nullptr;  // fp16: [segments, groups, 2], the largest |do|^2 and |v|^2 of a row (at_sigma)
  // forward, split over the columns: [m, heads, splits, channels + 2] (maximum, sum, result)
  float *parts = nullptr;
  int splits = 1;
  int *report = nullptr;         // host memory, set to 1 where a bounded wait ran out; may be null
  int *order = nullptr;          // place for the tiles' order (attention_tensor_order_bytes), queries' and keys' in turn
  cudaStream_t stream = nullptr;
};

template <typename T>
__device__ __forceinline__ float at_float(T v) { return (float)v; }
template <>
__device__ __forceinline__ float at_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float at_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T at_round(float v) { return (T)v; }
template <>
__device__ __forceinline__ __half at_round<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 at_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Rows [lo, hi) of one side that belong to segment b, clipped to the rows there are: an unsorted batch vector gives
// wrong segments, never an access out of range.
__device__ __forceinline__ void at_clip(int64_t from, int64_t to, int64_t rows, int64_t &lo, int64_t &hi) {
  lo = from < 0 ? 0 : from;
  hi = to > rows ? rows : to;
  if (hi < lo) hi = lo;
}
__device__ __forceinline__ void at_segment(const int64_t *__restrict__ ptr, int64_t rows, int64_t b, int64_t &lo,
                                           int64_t &hi) {
  lo = 0;
  hi = rows;
  if (ptr != nullptr) at_clip(ptr[b], ptr[b + 1], rows, lo, hi);
}

int launch_attention_plain_forward(const AttnArgs &a);
int launch_attention_plain_backward(const AttnArgs &a);
size_t attention_norms_bytes(const b200c_attention_t &p);  // of `norms`: fp16 only
int launch_attention_delta(const AttnArgs &a, float *delta, float *norms);
bool attention_tensor_applicable(const b200c_attention_t &p);
int launch_attention_tensor_forward(const AttnArgs &a);
int launch_attention_tensor_backward(const AttnArgs &a);
int attention_few_splits(const b200c_attention_t &p);  // 0: not for this call
size_t attention_few_workspace_bytes(const b200c_attention_t &p);
int launch_attention_few(const AttnArgs &a, int splits, void *workspace);
int launch_attention_join(const AttnArgs &a);          // a.parts of a.splits splits to out, rest and lse
int attention_tensor_splits(const b200c_attention_t &p);  // of a forward pass without statistics
size_t attention_tensor_order_bytes(const b200c_attention_t &p);  // of `order`, 0: tiles are taken as they come

}  // namespace b200c
