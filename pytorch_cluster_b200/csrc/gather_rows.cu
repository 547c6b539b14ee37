// Rows of a feature matrix by index, scaled, and the gradient of that.
//   out[e] = scale x[index[e]],   dx[n] = scale sum_{e : index[e] = n} dout[e]
// An index outside [0, rows) is padding (knn's -1): it gives a row of zeros and receives no gradient.
//
// Both directions are bound by memory: the forward pass is one copy with 16-byte accesses.  The backward pass has to
// bring equal indices together.  It sorts (index, e) pairs with a stable radix sort — as few passes of up to 9 bits as the
// row count needs, each a histogram, a scan and a scatter of 8 bytes per pair — and then adds dout's
// rows in that order, in fp32, each thread owning 16 bytes of the channels over a fixed number of consecutive pairs.
// Sums that cross such a piece's border go to the workspace and are joined in order.  No atomics touch a sum, so
// the result is the same from run to run, and an index that occurs a million times costs no more than a million
// different ones.
#include "common.cuh"
#include "launchers.h"

namespace b200c {

constexpr int GR_THREADS = 256;
constexpr int GR_WARPS = GR_THREADS / 32;
constexpr int GR_ITEMS = 16;                       // pairs per thread of a sort block
constexpr int GR_TILE = GR_THREADS * GR_ITEMS;     // pairs per sort block
constexpr int GR_MAX_BITS = 9;
constexpr int GR_SHORT = 16;                       // pieces a single thread joins; longer runs get a block

template <typename T, int VL>
struct alignas(sizeof(T) * VL) GrVec {
  T v[VL];
};

template <typename T>
__device__ __forceinline__ float gr_float(T v) { return (float)v; }
template <>
__device__ __forceinline__ float gr_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float gr_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T gr_round(float v) { return (T)v; }
template <>
__device__ __forceinline__ __half gr_round<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 gr_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VL>
__global__ void __launch_bounds__(GR_THREADS) gather_rows_kernel(const T *__restrict__ x,
                                                                 const int64_t *__restrict__ index, int64_t rows,
                                                                 int64_t edges, int units, float scale,
                                                                 T *__restrict__ out) {
  const int64_t i = (int64_t)blockIdx.x * GR_THREADS + threadIdx.x;
  if (i >= edges * units) return;
  const int64_t e = i / units, u = i - e * units;
  const int64_t row = index[e];
  GrVec<T, VL> r;
  if (row >= 0 && row < rows) {
    r = reinterpret_cast<const GrVec<T, VL> *>(x)[row * units + u];
#pragma unroll
    for (int c = 0; c < VL; ++c) r.v[c] = gr_round<T>(gr_float(r.v[c]) * scale);
  } else {
#pragma unroll
    for (int c = 0; c < VL; ++c) r.v[c] = gr_round<T>(0.f);
  }
  reinterpret_cast<GrVec<T, VL> *>(out)[i] = r;
}

// ---- stable radix sort of (key, edge) ------------------------------------------------------------------------
// The first pass reads the indices themselves (keys == nullptr); an index outside [0, rows) becomes the key `rows`.
__device__ __forceinline__ uint32_t gr_key(const int64_t *index, const uint32_t *keys, int64_t rows, int64_t i) {
  if (keys) return keys[i];
  const int64_t v = index[i];
  return (uint32_t)(v >= 0 && v < rows ? v : rows);
}

__global__ void __launch_bounds__(GR_THREADS) gather_sort_count_kernel(const int64_t *__restrict__ index,
                                                                       const uint32_t *__restrict__ keys, int64_t rows,
                                                                       int64_t edges, int shift, int bits,
                                                                       int32_t *__restrict__ counts) {
  __shared__ int hist[1 << GR_MAX_BITS];
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < bins; i += GR_THREADS) hist[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * GR_TILE;
#pragma unroll 4
  for (int r = 0; r < GR_ITEMS; ++r) {
    const int64_t i = base + r * GR_THREADS + threadIdx.x;
    if (i < edges) atomicAdd(&hist[(gr_key(index, keys, rows, i) >> shift) & (bins - 1)], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += GR_THREADS) counts[(int64_t)i * gridDim.x + blockIdx.x] = hist[i];
}

__global__ void __launch_bounds__(GR_THREADS) gather_sort_scatter_kernel(
    const int64_t *__restrict__ index, const uint32_t *__restrict__ keys, const uint32_t *__restrict__ vals,
    int64_t rows, int64_t edges, int shift, int bits, const int64_t *__restrict__ offsets,
    uint32_t *__restrict__ keys_out, uint32_t *__restrict__ vals_out) {
  // next[w][d]: where warp w puts its next pair of digit d (32 bits: at most 2^31 - 1 pairs)
  __shared__ uint32_t next[GR_WARPS][1 << GR_MAX_BITS];
  const int bins = 1 << bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < GR_WARPS * bins; i += GR_THREADS) next[i / bins][i % bins] = 0u;
  __syncthreads();
  // a warp owns GR_ITEMS * 32 consecutive pairs, so that warp, round and lane together keep the order
  const int64_t base = (int64_t)blockIdx.x * GR_TILE + warp * (GR_ITEMS * 32) + lane;
  uint32_t key[GR_ITEMS];
#pragma unroll
  for (int r = 0; r < GR_ITEMS; ++r) {
    const int64_t i = base + r * 32;
    key[r] = i < edges ? gr_key(index, keys, rows, i) : 0u;
    if (i < edges) atomicAdd(&next[warp][(key[r] >> shift) & (bins - 1)], 1u);
  }
  __syncthreads();
  for (int d = threadIdx.x; d < bins; d += GR_THREADS) {
    uint32_t at = (uint32_t)offsets[(int64_t)d * gridDim.x + blockIdx.x];
#pragma unroll
    for (int w = 0; w < GR_WARPS; ++w) {
      const uint32_t c = next[w][d];
      next[w][d] = at;
      at += c;
    }
  }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < GR_ITEMS; ++r) {
    const int64_t i = base + r * 32;
    const bool have = i < edges;
    const uint32_t digit = have ? (key[r] >> shift) & (bins - 1) : (uint32_t)bins;
    const unsigned same = __match_any_sync(FULL_MASK, digit);
    const int rank = __popc(same & ((1u << lane) - 1u));
    uint32_t at = 0u;
    if (have) at = next[warp][digit] + rank;
    __syncwarp();
    if (have && rank == 0) next[warp][digit] += __popc(same);
    __syncwarp();
    if (have) {
      keys_out[at] = key[r];
      vals_out[at] = vals ? vals[i] : (uint32_t)i;
    }
  }
}

// ---- sums over runs of equal keys ----------------------------------------------------------------------------
// Piece g covers the sorted pairs [g G, g G + G).  part[2 g] holds the sum of a run that reaches the piece's start from
// before or begins there and leaves its end; part[2 g + 1] that of a run that begins inside and leaves the end.
template <typename T, int VL>
__global__ void __launch_bounds__(GR_THREADS) gather_sum_kernel(const T *__restrict__ dout,
                                                                const uint32_t *__restrict__ keys,
                                                                const uint32_t *__restrict__ vals, int64_t rows,
                                                                int64_t edges, int units, int piece, int64_t pieces,
                                                                float scale, T *__restrict__ dx,
                                                                float *__restrict__ part) {
  constexpr int AHEAD = 8;
  const int64_t id = (int64_t)blockIdx.x * GR_THREADS + threadIdx.x;
  const int64_t g = id / units, u = id - g * units;
  if (g >= pieces) return;
  const int64_t lo = g * piece, hi = lo + piece < edges ? lo + piece : edges;
  const GrVec<T, VL> *src = reinterpret_cast<const GrVec<T, VL> *>(dout);
  float acc[VL] = {};
  uint32_t run = keys[lo];
  bool whole = lo == 0 || keys[lo - 1] != run;  // the run began at or after this piece's start
  bool first = true;                            // and is the piece's first
  auto flush = [&](bool ends) {
    if (whole && ends) {
      if (run < rows) {
        GrVec<T, VL> r;
#pragma unroll
        for (int c = 0; c < VL; ++c) r.v[c] = gr_round<T>(acc[c] * scale);
        reinterpret_cast<GrVec<T, VL> *>(dx)[(int64_t)run * units + u] = r;
      }
    } else {
      float *dst = part + ((2 * g + (first ? 0 : 1)) * units + u) * VL;
#pragma unroll
      for (int c = 0; c < VL; ++c) dst[c] = acc[c];
    }
  };
  for (int64_t i0 = lo; i0 < hi; i0 += AHEAD) {
    uint32_t key[AHEAD];
    GrVec<T, VL> row[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
      const int64_t i = i0 + n < hi ? i0 + n : hi - 1;
      key[n] = keys[i];
      row[n] = src[(int64_t)vals[i] * units + u];
    }
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
      if (i0 + n < hi) {
        if (key[n] != run) {
          flush(true);
          run = key[n];
          whole = true;
          first = false;
#pragma unroll
          for (int c = 0; c < VL; ++c) acc[c] = 0.f;
        }
#pragma unroll
        for (int c = 0; c < VL; ++c) acc[c] += gr_float(row[n].v[c]);
      }
    }
  }
  flush(hi == edges || keys[hi] != run);
}

// Where the run that leaves piece g began in g: its pieces are g .. last; returns last, or -1 if none does.
__device__ __forceinline__ int64_t gr_run(const uint32_t *keys, int64_t edges, int piece, int64_t pieces, int64_t g,
                                          uint32_t &run, int &slot) {
  const int64_t lo = g * piece, hi = lo + piece;
  if (hi >= edges) return -1;
  run = keys[hi - 1];
  if (keys[hi] != run) return -1;
  slot = keys[lo] == run ? 0 : 1;
  if (slot == 0 && lo > 0 && keys[lo - 1] == run) return -1;  // began earlier
  int64_t a = g + 1, b = pieces - 1;  // the last piece whose first key is the run's
  while (a < b) {
    const int64_t mid = (a + b + 1) >> 1;
    if (keys[mid * piece] == run)
      a = mid;
    else
      b = mid - 1;
  }
  return a;
}

template <typename T, int VL>
__global__ void __launch_bounds__(GR_THREADS) gather_join_kernel(const uint32_t *__restrict__ keys, int64_t rows,
                                                                 int64_t edges, int units, int piece, int64_t pieces,
                                                                 float scale, T *__restrict__ dx,
                                                                 const float *__restrict__ part,
                                                                 int *__restrict__ num_long,
                                                                 uint32_t *__restrict__ long_runs) {
  const int64_t id = (int64_t)blockIdx.x * GR_THREADS + threadIdx.x;
  const int64_t g = id / units, u = id - g * units;
  if (g >= pieces) return;
  uint32_t run;
  int slot;
  const int64_t last = gr_run(keys, edges, piece, pieces, g, run, slot);
  if (last < 0 || run >= rows) return;
  if (last - g > GR_SHORT) {
    if (u == 0) long_runs[atomicAdd(num_long, 1)] = (uint32_t)g;
    return;
  }
  float acc[VL];
#pragma unroll
  for (int c = 0; c < VL; ++c) acc[c] = part[((2 * g + slot) * units + u) * VL + c];
  for (int64_t h = g + 1; h <= last; ++h)
#pragma unroll
    for (int c = 0; c < VL; ++c) acc[c] += part[(2 * h * units + u) * VL + c];
  GrVec<T, VL> r;
#pragma unroll
  for (int c = 0; c < VL; ++c) r.v[c] = gr_round<T>(acc[c] * scale);
  reinterpret_cast<GrVec<T, VL> *>(dx)[(int64_t)run * units + u] = r;
}

// A block per (long run, 32 channels): 8 warps add contiguous shares of its pieces, then one adds the shares in order.
template <typename T>
__global__ void __launch_bounds__(GR_THREADS) gather_join_long_kernel(const uint32_t *__restrict__ keys, int64_t rows,
                                                                      int64_t edges, int channels, int piece,
                                                                      int64_t pieces, float scale, T *__restrict__ dx,
                                                                      const float *__restrict__ part,
                                                                      const int *__restrict__ num_long,
                                                                      const uint32_t *__restrict__ long_runs) {
  __shared__ float share[GR_WARPS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slabs = (channels + 31) / 32;
  const int64_t tasks = (int64_t)*num_long * slabs;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const int64_t g = long_runs[t / slabs];
    const int c = (int)(t % slabs) * 32 + lane;
    uint32_t run = 0;
    int slot = 0;
    const int64_t last = gr_run(keys, edges, piece, pieces, g, run, slot);
    const int64_t n = last - g + 1, each = (n + GR_WARPS - 1) / GR_WARPS;
    const int64_t a = warp * each, b = a + each < n ? a + each : n;
    float acc = 0.f;
    if (c < channels) {
#pragma unroll 8
      for (int64_t h = a; h < b; ++h) acc += part[(2 * (g + h) + (h == 0 ? slot : 0)) * channels + c];
    }
    share[warp][lane] = acc;
    __syncthreads();
    if (warp == 0 && c < channels) {
      acc = 0.f;
#pragma unroll
      for (int w = 0; w < GR_WARPS; ++w) acc += share[w][lane];
      dx[(int64_t)run * channels + c] = gr_round<T>(acc * scale);
    }
    __syncthreads();
  }
}

// ---- host ----------------------------------------------------------------------------------------------------
static size_t gr_align(size_t v) { return (v + 255) / 256 * 256; }

struct GrPlan {
  int bits, passes, piece;
  int64_t blocks, pieces;
  size_t keys, counts, offsets, scan, part, runs, total;
};

static GrPlan gr_plan(int64_t rows, int64_t edges, int64_t channels) {
  GrPlan p{};
  int bits = 1;
  while ((1ll << bits) <= rows) ++bits;  // keys 0 .. rows
  p.passes = (bits + GR_MAX_BITS - 1) / GR_MAX_BITS;
  p.bits = (bits + p.passes - 1) / p.passes;
  p.blocks = (edges + GR_TILE - 1) / GR_TILE;
  // 64 pairs a piece: the borders' sums then cost an eighth of dout's bytes (16-bit types) at most
  p.piece = 64;
  p.pieces = (edges + p.piece - 1) / p.piece;
  const int64_t bins = (1ll << p.bits) * p.blocks;
  p.keys = gr_align((size_t)edges * 4);
  p.counts = gr_align((size_t)bins * 4);
  p.offsets = gr_align((size_t)(bins + 1) * 8);
  p.scan = gr_align(b200c_scan_workspace_bytes(bins));
  p.part = gr_align((size_t)p.pieces * 2 * channels * 4);
  p.runs = gr_align((size_t)(p.pieces + 1) * 4);
  p.total = 4 * p.keys + p.counts + p.offsets + p.scan + p.part + p.runs;
  return p;
}

template <typename T, int VL>
static int gr_forward(const void *x, const int64_t *index, int64_t rows, int64_t edges, int64_t channels, float scale,
                      void *out, cudaStream_t stream) {
  const int64_t threads = edges * (channels / VL);
  gather_rows_kernel<T, VL><<<(unsigned)((threads + GR_THREADS - 1) / GR_THREADS), GR_THREADS, 0, stream>>>(
      (const T *)x, index, rows, edges, (int)(channels / VL), scale, (T *)out);
  B200C_LAUNCH_CHECK("gather_rows_kernel");
  return B200C_OK;
}

template <typename T, int VL>
static int gr_backward(const void *dout, const int64_t *index, int64_t rows, int64_t edges, int64_t channels,
                       float scale, void *dx, void *workspace, cudaStream_t stream) {
  const GrPlan p = gr_plan(rows, edges, channels);
  char *ws = (char *)workspace;
  uint32_t *keys[2], *vals[2];
  for (int i = 0; i < 2; ++i) {
    keys[i] = (uint32_t *)ws, ws += p.keys;
    vals[i] = (uint32_t *)ws, ws += p.keys;
  }
  int32_t *counts = (int32_t *)ws;
  ws += p.counts;
  int64_t *offsets = (int64_t *)ws;
  ws += p.offsets;
  void *scan = ws;
  ws += p.scan;
  float *part = (float *)ws;
  ws += p.part;
  int *num_long = (int *)ws;
  uint32_t *long_runs = (uint32_t *)ws + 1;

  B200C_CUDA(cudaMemsetAsync(dx, 0, (size_t)rows * channels * sizeof(T), stream));  // rows that no index names
  const uint32_t *k = nullptr, *v = nullptr;
  for (int pass = 0; pass < p.passes; ++pass) {
    gather_sort_count_kernel<<<(unsigned)p.blocks, GR_THREADS, 0, stream>>>(index, k, rows, edges, pass * p.bits,
                                                                            p.bits, counts);
    B200C_LAUNCH_CHECK("gather_sort_count_kernel");
    int st = b200c_exclusive_scan(counts, (1ll << p.bits) * p.blocks, offsets, scan, p.scan, stream);
    if (st != B200C_OK) return st;
    gather_sort_scatter_kernel<<<(unsigned)p.blocks, GR_THREADS, 0, stream>>>(
        index, k, v, rows, edges, pass * p.bits, p.bits, offsets, keys[pass & 1], vals[pass & 1]);
    B200C_LAUNCH_CHECK("gather_sort_scatter_kernel");
    k = keys[pass & 1];
    v = vals[pass & 1];
  }
  B200C_CUDA(cudaMemsetAsync(num_long, 0, 4, stream));
  const int units = (int)(channels / VL);
  const unsigned blocks = (unsigned)((p.pieces * units + GR_THREADS - 1) / GR_THREADS);
  gather_sum_kernel<T, VL><<<blocks, GR_THREADS, 0, stream>>>((const T *)dout, k, v, rows, edges, units, p.piece,
                                                              p.pieces, scale, (T *)dx, part);
  B200C_LAUNCH_CHECK("gather_sum_kernel");
  gather_join_kernel<T, VL><<<blocks, GR_THREADS, 0, stream>>>(k, rows, edges, units, p.piece, p.pieces, scale,
                                                               (T *)dx, part, num_long, long_runs);
  B200C_LAUNCH_CHECK("gather_join_kernel");
  gather_join_long_kernel<T><<<296, GR_THREADS, 0, stream>>>(k, rows, edges, (int)channels, p.piece, p.pieces, scale,
                                                             (T *)dx, part, num_long, long_runs);
  B200C_LAUNCH_CHECK("gather_join_long_kernel");
  return B200C_OK;
}

struct GrCall {
  const void *in;
  const int64_t *index;
  int64_t rows, edges, channels;
  float scale;
  void *out, *workspace;
  cudaStream_t stream;
  bool forward;
};

template <typename T, int VL>
static int gr_run_call(const GrCall &c) {
  return c.forward ? gr_forward<T, VL>(c.in, c.index, c.rows, c.edges, c.channels, c.scale, c.out, c.stream)
                   : gr_backward<T, VL>(c.in, c.index, c.rows, c.edges, c.channels, c.scale, c.out, c.workspace,
                                        c.stream);
}

// the widest access that the channels and both arrays' alignment allow, 16 bytes at most
template <typename T>
static int gr_width(const GrCall &c) {
  const uintptr_t at = (uintptr_t)c.in | (uintptr_t)c.out;
  constexpr int MOST = 16 / (int)sizeof(T);
  if (c.channels % MOST == 0 && at % 16 == 0) return gr_run_call<T, MOST>(c);
  if (c.channels % (MOST / 2) == 0 && at % 8 == 0) return gr_run_call<T, MOST / 2>(c);
  return gr_run_call<T, 1>(c);
}

static int gr_type(const GrCall &c, int dtype) {
  if (dtype == B200C_F32) return gr_width<float>(c);
  if (dtype == B200C_F16) return gr_width<__half>(c);
  return gr_width<__nv_bfloat16>(c);
}

size_t gather_rows_workspace_bytes(int64_t rows, int64_t edges, int64_t channels) {
  return edges > 0 ? gr_plan(rows, edges, channels).total : 0;
}

int launch_gather_rows(const void *x, const int64_t *index, int64_t rows, int64_t edges, int64_t channels, float scale,
                       int dtype, void *out, cudaStream_t stream) {
  return gr_type({x, index, rows, edges, channels, scale, out, nullptr, stream, true}, dtype);
}

int launch_gather_rows_backward(const void *dout, const int64_t *index, int64_t rows, int64_t edges, int64_t channels,
                                float scale, int dtype, void *dx, void *workspace, cudaStream_t stream) {
  return gr_type({dout, index, rows, edges, channels, scale, dx, workspace, stream, false}, dtype);
}

}  // namespace b200c
