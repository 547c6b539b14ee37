// Dispatch of the tensor-core attention over channels, coordinates and cap.  Channel counts are padded to 64 or 128
// with zeros by the copies; coordinates to 1, 3 or 8.
#pragma once

#include "attention_backward.cuh"
#include "attention_forward.cuh"

namespace b200c {

template <typename T, int CP, int DIM, bool CAP>
struct AtForwardCall {
  static int run(const AttnArgs &a) {
    using F = AtForward<CP>;
    const b200c_attention_t &p = a.p;
    AtForwardMaps maps;
    int st = attention_tensor_map(&maps.q, p.q, p.dtype, p.m, p.heads, p.channels, p.q_row, p.q_head, AT_ROWS);
    if (st == B200C_OK)
      st = attention_tensor_map(&maps.k, p.k, p.dtype, p.n, p.groups, p.channels, p.k_row, p.k_head, AT_COLS);
    if (st == B200C_OK)
      st = attention_tensor_map(&maps.v, p.v, p.dtype, p.n, p.groups, p.channels, p.v_row, p.v_head, AT_COLS);
    if (st != B200C_OK) return st;
    const dim3 grid((unsigned)((p.m + AT_ROWS - 1) / AT_ROWS * p.heads), 1, (unsigned)a.splits);
    static unsigned long long configured = 0ull;
    B200C_CUDA(opt_in_shared_memory(attention_forward_kernel<T, CP, DIM, CAP>, F::SMEM, configured));
    attention_forward_kernel<T, CP, DIM, CAP><<<grid, F::THREADS, F::SMEM, a.stream>>>(maps, a, (T *)a.rest);
    B200C_LAUNCH_CHECK("attention_forward_kernel");
    return B200C_OK;
  }
};

template <typename T, int CP, int DIM, bool CAP, bool KV>
struct AtBackwardCall {
  static int run(const AttnArgs &a) {
    using F = AtBackward<CP, KV>;
    const b200c_attention_t &p = a.p;
    const int64_t row = (int64_t)p.heads * p.channels;
    const int q_box = KV ? AT_COLS : AT_ROWS, k_box = KV ? AT_ROWS : AT_COLS;
    AtBackwardMaps maps;
    CUtensorMap *q = KV ? &maps.col0 : &maps.row0, *dout = KV ? &maps.col1 : &maps.row1;
    CUtensorMap *k = KV ? &maps.row0 : &maps.col0, *v = KV ? &maps.row1 : &maps.col1;
    int st = attention_tensor_map(q, p.q, p.dtype, p.m, p.heads, p.channels, p.q_row, p.q_head, q_box);
    if (st == B200C_OK)
      st = attention_tensor_map(dout, a.dout, p.dtype, p.m, p.heads, p.channels, row, p.channels, q_box);
    if (st == B200C_OK)
      st = attention_tensor_map(k, p.k, p.dtype, p.n, p.groups, p.channels, p.k_row, p.k_head, k_box);
    if (st == B200C_OK)
      st = attention_tensor_map(v, p.v, p.dtype, p.n, p.groups, p.channels, p.v_row, p.v_head, k_box);
    if (st != B200C_OK) return st;
    const dim3 grid((unsigned)(((KV ? p.n : p.m) + AT_ROWS - 1) / AT_ROWS * (KV ? p.groups : p.heads)));
    static unsigned long long configured = 0ull;
    B200C_CUDA(opt_in_shared_memory(attention_backward_kernel<T, CP, DIM, CAP, KV>, F::SMEM, configured));
    attention_backward_kernel<T, CP, DIM, CAP, KV><<<grid, F::THREADS, F::SMEM, a.stream>>>(maps, a, a.norms);
    B200C_LAUNCH_CHECK("attention_backward_kernel");
    return B200C_OK;
  }
};

template <typename T, int CP, int DIM, bool CAP>
using AtQueriesCall = AtBackwardCall<T, CP, DIM, CAP, false>;
template <typename T, int CP, int DIM, bool CAP>
using AtKeysCall = AtBackwardCall<T, CP, DIM, CAP, true>;

template <template <typename, int, int, bool> class Call, typename T, int CP, bool CAP>
int at_dims(const AttnArgs &a) {
  if (a.p.dims == 0) return Call<T, CP, 0, CAP>::run(a);
  if (a.p.dims == 1) return Call<T, CP, 1, CAP>::run(a);
  if (a.p.dims <= 3) return Call<T, CP, 3, CAP>::run(a);
  return Call<T, CP, 8, CAP>::run(a);
}

template <template <typename, int, int, bool> class Call, typename T>
int at_dispatch(const AttnArgs &a) {
  if (a.p.channels <= 64) return a.p.cap > 0.f ? at_dims<Call, T, 64, true>(a) : at_dims<Call, T, 64, false>(a);
  return a.p.cap > 0.f ? at_dims<Call, T, 128, true>(a) : at_dims<Call, T, 128, false>(a);
}

}  // namespace b200c
