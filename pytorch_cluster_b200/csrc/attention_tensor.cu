// Host side of the tensor-core attention: which calls it takes, tensor maps, dispatch over types.
#include "attention_tensor.cuh"
#include "attention_tensor_launch.h"

namespace b200c {

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

int attention_tensor_map(CUtensorMap *map, const void *base, int dtype, int64_t rows, int heads, int channels,
                         int64_t row_stride, int64_t head_stride, int box_rows) {
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) {
    set_error("the driver has no cuTensorMapEncodeTiled");
    return B200C_ERR_CUDA;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)channels, (cuuint64_t)heads, (cuuint64_t)rows};
  // a stride that no coordinate uses still has to be a valid one
  const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? head_stride : 128) * 2,
                                 (cuuint64_t)(rows > 1 ? row_stride : 128) * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, dtype == B200C_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            3, (void *)base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed: %d", (int)r);
    return B200C_ERR_CUDA;
  }
  return B200C_OK;
}

// 16-byte rows that a tensor map can describe
static bool at_side(const void *base, int64_t rows, int heads, int64_t row_stride, int64_t head_stride) {
  const auto fits = [](int64_t s) { return s > 0 && s % 8 == 0 && s < (1ll << 38); };
  return ((uintptr_t)base & 15) == 0 && (rows <= 1 || fits(row_stride)) && (heads <= 1 || fits(head_stride));
}

bool attention_tensor_applicable(const b200c_attention_t &p) {
  constexpr int64_t most = 0x7fffffffLL - 1024;  // column numbers of a step past the last stay in 32 bits
  return p.dtype != B200C_F32 && p.channels % 8 == 0 && !(p.cap > AT_MAX_FAST_CAP) &&
         p.m > 0 && p.n > 0 && p.m < most && p.n < most &&
         at_side(p.q, p.m, p.heads, p.q_row, p.q_head) && at_side(p.k, p.n, p.groups, p.k_row, p.k_head) &&
         at_side(p.v, p.n, p.groups, p.v_row, p.v_head);
}

// Up to 32 channels and 128 rows per example on average (either side) the kernels of attention_short.cuh are taken.
// Measured on 60000 rows, 8 heads, three coordinates, bfloat16, forward / gradient in us, 128-row tiles against 16-row
// ones:
//   32 channels: 16 rows 185 / 437, 125 / 254;  64 rows 220 / 488, 151 / 331;  128 rows 251 / 567, 208 / 463;
//                192 rows 277 / 633, 266 / 594
//   64 channels: 16 rows 188 / 465, 198 / 471;  64 rows 220 / 510, 250 / 602
constexpr int64_t AT_SHORT_ROWS = 128;
constexpr int AT_SHORT_CHANNELS = 32;
static bool is_short(const b200c_attention_t &p) {
  return p.channels <= AT_SHORT_CHANNELS && p.m <= AT_SHORT_ROWS * p.num_segments &&
         p.n <= AT_SHORT_ROWS * p.num_segments;
}

// A small call leaves most SMs without a block of 128 rows: the columns are dealt out to several, 128 and more to each,
// as long as that fills the SMs, and a second kernel joins them (one cloud of 1024 points, 4 heads: 33 -> 25 us).
int attention_tensor_splits(const b200c_attention_t &p) {
  if (!attention_tensor_applicable(p) || is_short(p)) return 1;
  const int64_t blocks = (p.m + AT_ROWS - 1) / AT_ROWS * p.heads;
  int64_t splits = 148 / blocks;
  const int64_t most = p.n / p.num_segments / 128;
  if (splits > most) splits = most;
  return (int)(splits < 1 ? 1 : splits > 16 ? 16 : splits);
}

// Tiles of long examples come to the SMs most columns first.  An order costs a launch of some 5 us and is made where
// blocks outnumber what the GPU holds at once, take long (1024 columns and more) and are not so many that the last ones
// hardly count.
constexpr int AT_ORDER_TILES = 4096, AT_ORDER_BINS = 256;
static bool at_ordered(const b200c_attention_t &p, int64_t rows, int64_t cols, int per_tile) {
  const int64_t tiles = (rows + AT_ROWS - 1) / AT_ROWS;
  return p.num_segments > 1 && tiles <= AT_ORDER_TILES && tiles * per_tile > 2 * 148 && cols >= 1024 * p.num_segments;
}
size_t attention_tensor_order_bytes(const b200c_attention_t &p) {
  if (!attention_tensor_applicable(p) || is_short(p)) return 0;
  const bool any = at_ordered(p, p.m, p.n, p.heads) || at_ordered(p, p.n, p.m, p.groups);
  return any ? (size_t)AT_ORDER_TILES * 4 : 0;
}

__global__ void __launch_bounds__(1024) attention_order_kernel(const int64_t *__restrict__ ptr_r,
                                                              const int64_t *__restrict__ ptr_c, int64_t rows,
                                                              int64_t cols, int segments, int tiles,
                                                              int *__restrict__ order) {
  __shared__ int most, at[AT_ORDER_BINS + 1];
  const int tid = threadIdx.x;
  if (tid == 0) most = 1;
  if (tid <= AT_ORDER_BINS) at[tid] = 0;
  __syncthreads();
  int cost[AT_ORDER_TILES / 1024];
#pragma unroll
  for (int i = 0; i < AT_ORDER_TILES / 1024; ++i) {
    const int64_t t0 = ((int64_t)i * 1024 + tid) * AT_ROWS;
    cost[i] = -1;
    if (i * 1024 + tid >= tiles) continue;
    int64_t lo, hi, unused;
    at_segment(ptr_c, cols, segment_of(ptr_r, segments, t0), lo, unused);
    at_segment(ptr_c, cols, segment_of(ptr_r, segments, t0 + AT_ROWS < rows ? t0 + AT_ROWS - 1 : rows - 1), unused, hi);
    cost[i] = hi > lo ? (int)(hi - lo) : 0;
    atomicMax(&most, cost[i]);
  }
  __syncthreads();
  // a counting sort, dearest bin first; the order within a bin is whatever it is: it moves blocks, not results
  const float to_bin = (float)(AT_ORDER_BINS - 1) / (float)most;
#pragma unroll
  for (int i = 0; i < AT_ORDER_TILES / 1024; ++i)
    if (cost[i] >= 0) {
      const int bin = (int)((float)cost[i] * to_bin);
      cost[i] = AT_ORDER_BINS - 1 - (bin < AT_ORDER_BINS ? bin : AT_ORDER_BINS - 1);
      atomicAdd(&at[cost[i] + 1], 1);
    }
  __syncthreads();
  if (tid < 32) {
    int before = 0;
    for (int b0 = 0; b0 < AT_ORDER_BINS; b0 += 32) {
      int v = at[b0 + tid + 1];
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(FULL_MASK, v, o);
        if (tid >= o) v += u;
      }
      at[b0 + tid + 1] = before + v;
      before += __shfl_sync(FULL_MASK, v, 31);
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < AT_ORDER_TILES / 1024; ++i)
    if (cost[i] >= 0) order[atomicAdd(&at[cost[i]], 1)] = i * 1024 + tid;
}

// a with its tiles' order, or without
static int at_order(AttnArgs &a, bool keys) {
  const b200c_attention_t &p = a.p;
  const int64_t rows = keys ? p.n : p.m, cols = keys ? p.m : p.n;
  if (a.order == nullptr || !at_ordered(p, rows, cols, keys ? p.groups : p.heads)) {
    a.order = nullptr;
    return B200C_OK;
  }
  attention_order_kernel<<<1, 1024, 0, a.stream>>>(keys ? p.ptr_k : p.ptr_q, keys ? p.ptr_q : p.ptr_k, rows, cols,
                                                   (int)p.num_segments, (int)((rows + AT_ROWS - 1) / AT_ROWS), a.order);
  B200C_LAUNCH_CHECK("attention_order_kernel");
  return B200C_OK;
}

int launch_attention_tensor_forward(const AttnArgs &args) {
  AttnArgs a = args;
  const bool bf16 = a.p.dtype == B200C_BF16;
  if (a.splits > 1) {
    const int st = bf16 ? attention_tensor_forward_bf16(a) : attention_tensor_forward_f16(a);
    return st != B200C_OK ? st : launch_attention_join(a);
  }
  if (is_short(a.p)) return bf16 ? attention_short_forward_bf16(a) : attention_short_forward_f16(a);
  const int st = at_order(a, false);
  if (st != B200C_OK) return st;
  return bf16 ? attention_tensor_forward_bf16(a) : attention_tensor_forward_f16(a);
}

int launch_attention_tensor_backward(const AttnArgs &args) {
  AttnArgs a = args;
  const bool bf16 = a.p.dtype == B200C_BF16;
  int st = B200C_OK;
  if (is_short(a.p)) {
    if (a.dq) st = bf16 ? attention_short_dq_bf16(a) : attention_short_dq_f16(a);
    if (st != B200C_OK || !a.dk) return st;
    return bf16 ? attention_short_dkv_bf16(a) : attention_short_dkv_f16(a);
  }
  if (a.dq) {
    if ((st = at_order(a, false)) == B200C_OK) st = bf16 ? attention_tensor_dq_bf16(a) : attention_tensor_dq_f16(a);
    if (st != B200C_OK) return st;
  }
  if (!a.dk) return B200C_OK;
  a.order = args.order;
  if ((st = at_order(a, true)) != B200C_OK) return st;
  return bf16 ? attention_tensor_dkv_bf16(a) : attention_tensor_dkv_f16(a);
}

}  // namespace b200c
