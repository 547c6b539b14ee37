// Rows of a feature matrix by index, scaled, and the gradient of that.
//   out[e] = scale x[index[e]],   dx[n] = scale sum_{e : index[e] = n} dout[e]
// An index outside [0, rows) is padding (knn's -1): it gives a row of zeros and receives no gradient.
//
// Both directions are bound by memory: the forward pass is one copy with 16-byte accesses, four edges per thread so
// that enough loads are on their way behind the indices.  The backward pass has to bring equal indices together.  It
// sorts (index, e) pairs with a stable radix sort — as few passes of up to 9 bits as the row count needs, each a
// histogram per block, a scan of the blocks' counts per digit, and a scatter of 8 bytes per pair by way of shared
// memory, where a block's pairs are put in order first, so that they leave in runs — and then adds dout's rows in that
// order, in fp32, each thread owning 16 bytes of the channels over 64 or more consecutive pairs. Sums that cross such a
// piece's border go to the workspace and are joined in order.  No atomics touch a sum, so the result is the same from
// run to run, and an index that occurs a million times costs no more than a million different ones.
#include "common.cuh"
#include "launchers.h"

namespace b200c {

constexpr int GR_THREADS = 256;
constexpr int GR_WARPS = GR_THREADS / 32;
// pairs per thread of a sort block: 16 leave 2.6e6 edges in two waves of blocks (85 us of sort, 77 so)
constexpr int GR_ITEMS = 10;
constexpr int GR_TILE = GR_THREADS * GR_ITEMS;     // pairs per sort block
constexpr int GR_MAX_BITS = 9;
constexpr int GR_EDGES = 4;                        // edges per thread of the forward pass
constexpr int GR_LONG_WARPS = 32;                  // of a block that joins a long run
constexpr int GR_SHORT = 16;                       // pieces a single thread joins; longer runs get a block
// Calls of up to GR_ONE pairs sort in one block and leave every join to a thread: 4 launches for 11, 75 -> 66 us of a
// training step of 1100 edges, which the host's launches bound.  Up to GR_FEW blocks the scatter adds up the counts
// that it needs itself, in place of a launch per pass.
constexpr int GR_ONE_THREADS = 1024;
constexpr int GR_ONE_ITEMS = 16;
constexpr int GR_ONE = GR_ONE_THREADS * GR_ONE_ITEMS;
constexpr int GR_FEW = 32;
// Up to GR_ROWS rows and edges the sort leaves every row's place too, and one kernel writes all rows, zeros included: 2
// launches for 4 (1100 edges 66 -> 63 us).
constexpr int GR_ROWS = 4096;
constexpr int GR_SLOTS = 8;  // warps that share the edges of a row

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
                                                                 int64_t total, int units, float scale,
                                                                 T *__restrict__ out) {
  // thread t of a block takes units t, t + 256, t + 512, ... of the block's share
  const int64_t base = (int64_t)blockIdx.x * (GR_THREADS * GR_EDGES) + threadIdx.x;
  int64_t from[GR_EDGES];
#pragma unroll
  for (int n = 0; n < GR_EDGES; ++n) {
    const int64_t i = base + n * GR_THREADS;
    from[n] = -1;
    if (i < total) {
      const int64_t e = total <= 0xffffffffLL ? (int64_t)((uint32_t)i / (uint32_t)units) : i / units;
      const int64_t row = index[e];
      if (row >= 0 && row < rows) from[n] = row * units + (i - e * units);
    }
  }
  GrVec<T, VL> r[GR_EDGES];
#pragma unroll
  for (int n = 0; n < GR_EDGES; ++n) {
    if (from[n] >= 0) {
      r[n] = reinterpret_cast<const GrVec<T, VL> *>(x)[from[n]];
    } else {
#pragma unroll
      for (int c = 0; c < VL; ++c) r[n].v[c] = gr_round<T>(0.f);
    }
  }
#pragma unroll
  for (int n = 0; n < GR_EDGES; ++n) {
    const int64_t i = base + n * GR_THREADS;
    if (i >= total) break;
    if (from[n] >= 0) {
#pragma unroll
      for (int c = 0; c < VL; ++c) r[n].v[c] = gr_round<T>(gr_float(r[n].v[c]) * scale);
    }
    reinterpret_cast<GrVec<T, VL> *>(out)[i] = r[n];
  }
}

// ---- stable radix sort of (key, edge) ------------------------------------------------------------------------
// The first pass reads the indices themselves (pairs == nullptr); an index outside [0, rows) becomes the key `rows`.
__device__ __forceinline__ uint2 gr_pair(const int64_t *index, const uint2 *pairs, int64_t rows, int64_t i) {
  if (pairs) return pairs[i];
  const int64_t v = index[i];
  return make_uint2((uint32_t)(v >= 0 && v < rows ? v : rows), (uint32_t)i);
}

// counts[digit][block]
__global__ void __launch_bounds__(GR_THREADS) gather_sort_count_kernel(const int64_t *__restrict__ index,
                                                                       const uint2 *__restrict__ pairs, int64_t rows,
                                                                       int64_t edges, int shift, int bits,
                                                                       uint32_t *__restrict__ counts,
                                                                       int *__restrict__ num_long) {
  if (pairs == nullptr && blockIdx.x == 0 && threadIdx.x == 0) *num_long = 0;  // for the joins
  __shared__ int hist[1 << GR_MAX_BITS];
  const int bins = 1 << bits;
  for (int i = threadIdx.x; i < bins; i += GR_THREADS) hist[i] = 0;
  __syncthreads();
  const int64_t base = (int64_t)blockIdx.x * GR_TILE;
#pragma unroll 8
  for (int r = 0; r < GR_ITEMS; ++r) {
    const int64_t i = base + r * GR_THREADS + threadIdx.x;
    if (i < edges) atomicAdd(&hist[(gr_pair(index, pairs, rows, i).x >> shift) & (bins - 1)], 1);
  }
  __syncthreads();
  for (int i = threadIdx.x; i < bins; i += GR_THREADS) counts[(int64_t)i * gridDim.x + blockIdx.x] = hist[i];
}

// exclusive sum over one warp-sized batch per warp of the block; returns this thread's, and the block's total
template <int WARPS = GR_WARPS>
__device__ __forceinline__ uint32_t gr_block_scan(uint32_t v, uint32_t *warp_sums, uint32_t &total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  uint32_t in = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const uint32_t t = __shfl_up_sync(FULL_MASK, in, o);
    if (lane >= o) in += t;
  }
  __syncthreads();
  if (lane == 31) warp_sums[warp] = in;
  __syncthreads();
  uint32_t before = 0u;
  total = 0u;
#pragma unroll
  for (int w = 0; w < WARPS; ++w) {
    if (w < warp) before += warp_sums[w];
    total += warp_sums[w];
  }
  return before + in - v;
}

// a block per digit: its counts become exclusive sums over the blocks, totals[digit] their total
__global__ void __launch_bounds__(GR_THREADS) gather_sort_scan_kernel(uint32_t *__restrict__ counts, int64_t blocks,
                                                                      uint32_t *__restrict__ totals) {
  __shared__ uint32_t warp_sums[GR_WARPS];
  uint32_t *mine = counts + (int64_t)blockIdx.x * blocks;
  uint32_t run = 0u;
  for (int64_t i0 = 0; i0 < blocks; i0 += GR_THREADS * 4) {
    uint32_t v[4], sum = 0u, total;
    const int64_t i = i0 + threadIdx.x * 4;
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      v[n] = i + n < blocks ? mine[i + n] : 0u;
      sum += v[n];
    }
    uint32_t at = run + gr_block_scan(sum, warp_sums, total);
#pragma unroll
    for (int n = 0; n < 4; ++n) {
      if (i + n < blocks) mine[i + n] = at;
      at += v[n];
    }
    run += total;
  }
  if (threadIdx.x == 0) totals[blockIdx.x] = run;
}

// The place of this lane's pair: those of a digit follow one another in the order of the lanes.  next[digit] is the
// warp's next place and moves on.  The lanes with one digit are found by a ballot per bit (match_any takes three times
// as long where digits differ).
__device__ __forceinline__ uint32_t gr_place(bool have, uint32_t digit, int bits, uint32_t *next) {
  unsigned same = __ballot_sync(FULL_MASK, have);
  if (!have) same = ~same;
  for (int b = 0; b < bits; ++b) {
    const bool one = (digit >> b) & 1u;
    const unsigned ones = __ballot_sync(FULL_MASK, one);
    same &= one ? ones : ~ones;
  }
  const int rank = __popc(same & ((1u << (threadIdx.x & 31)) - 1u));
  uint32_t at = 0u;
  if (have) at = next[digit];
  __syncwarp();
  if (have && rank == 0) next[digit] = at + __popc(same);
  __syncwarp();
  return at + rank;
}

__global__ void __launch_bounds__(GR_THREADS) gather_sort_scatter_kernel(
    const int64_t *__restrict__ index, const uint2 *__restrict__ pairs, int64_t rows, int64_t edges, int shift,
    int bits, const uint32_t *__restrict__ counts, const uint32_t *__restrict__ totals, uint2 *__restrict__ out) {
  constexpr int MOST = 1 << GR_MAX_BITS;
  extern __shared__ __align__(16) unsigned char gr_smem[];
  uint2 *sorted = reinterpret_cast<uint2 *>(gr_smem);                          // the block's pairs, by digit
  // where warp w puts its next pair of digit d; out position - position in `sorted`, per digit
  uint32_t(*next)[MOST] = reinterpret_cast<uint32_t(*)[MOST]>(sorted + GR_TILE);
  uint32_t *shift_to = reinterpret_cast<uint32_t *>(next + GR_WARPS);
  __shared__ uint32_t warp_sums[GR_WARPS];
  const int bins = 1 << bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int i = threadIdx.x; i < GR_WARPS * MOST; i += GR_THREADS) next[0][i] = 0u;
  __syncthreads();
  // a warp owns GR_ITEMS * 32 consecutive pairs, so that warp, round and lane together keep the order
  const int64_t base = (int64_t)blockIdx.x * GR_TILE + warp * (GR_ITEMS * 32) + lane;
  uint2 pair[GR_ITEMS];
#pragma unroll
  for (int r = 0; r < GR_ITEMS; ++r) {
    const int64_t i = base + r * 32;
    pair[r] = i < edges ? gr_pair(index, pairs, rows, i) : make_uint2(0u, 0u);
  }
#pragma unroll
  for (int r = 0; r < GR_ITEMS; ++r)
    if (base + r * 32 < edges) atomicAdd(&next[warp][(pair[r].x >> shift) & (bins - 1)], 1u);
  __syncthreads();
  // two digits per thread: the block's and all blocks' exclusive sums over the digits
  const int d0 = threadIdx.x * 2;
  uint32_t here[2] = {}, all[2] = {}, earlier[2] = {}, unused;
#pragma unroll
  for (int n = 0; n < 2; ++n)
    if (d0 + n < bins) {
      for (int w = 0; w < GR_WARPS; ++w) here[n] += next[w][d0 + n];
      const uint32_t *mine = counts + (int64_t)(d0 + n) * gridDim.x;
      if (totals) {
        all[n] = totals[d0 + n];
        earlier[n] = mine[blockIdx.x];
      } else {
#pragma unroll 8
        for (unsigned b = 0; b < gridDim.x; ++b) {
          const uint32_t c = mine[b];
          all[n] += c;
          if (b < blockIdx.x) earlier[n] += c;
        }
      }
    }
  uint32_t at_here = gr_block_scan(here[0] + here[1], warp_sums, unused);
  uint32_t at_all = gr_block_scan(all[0] + all[1], warp_sums, unused);
#pragma unroll
  for (int n = 0; n < 2; ++n)
    if (d0 + n < bins) {
      shift_to[d0 + n] = at_all + earlier[n] - at_here;
      uint32_t at = at_here;
      for (int w = 0; w < GR_WARPS; ++w) {
        const uint32_t c = next[w][d0 + n];
        next[w][d0 + n] = at;
        at += c;
      }
      at_here += here[n];
      at_all += all[n];
    }
  __syncthreads();
#pragma unroll
  for (int r = 0; r < GR_ITEMS; ++r) {
    const bool have = base + r * 32 < edges;
    const uint32_t digit = have ? (pair[r].x >> shift) & (bins - 1) : (uint32_t)bins;
    const uint32_t at = gr_place(have, digit, bits, next[warp]);
    if (have) sorted[at] = pair[r];
  }
  __syncthreads();
  const int64_t left = edges - (int64_t)blockIdx.x * GR_TILE;
  const int count = left < GR_TILE ? (int)left : GR_TILE;
#pragma unroll 4
  for (int i = threadIdx.x; i < count; i += GR_THREADS) {
    const uint2 p = sorted[i];
    out[(uint32_t)i + shift_to[(p.x >> shift) & (bins - 1)]] = p;
  }
}

// All passes in one block; the pairs stay in shared memory between them.
__global__ void __launch_bounds__(GR_ONE_THREADS) gather_sort_one_kernel(const int64_t *__restrict__ index, int64_t rows,
                                                                        int edges, int passes, int bits,
                                                                        uint2 *__restrict__ out,
                                                                        int *__restrict__ starts) {
  constexpr int MOST = 1 << GR_MAX_BITS, WARPS = GR_ONE_THREADS / 32;
  extern __shared__ __align__(16) unsigned char gr_smem[];
  uint2 *sorted = reinterpret_cast<uint2 *>(gr_smem);
  uint32_t(*next)[MOST] = reinterpret_cast<uint32_t(*)[MOST]>(sorted + GR_ONE);
  __shared__ uint32_t warp_sums[WARPS];
  const int bins = 1 << bits, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int items = (edges + GR_ONE_THREADS - 1) / GR_ONE_THREADS;  // a warp owns items * 32 consecutive pairs
  const int base = warp * items * 32 + lane;
  for (int pass = 0; pass < passes; ++pass) {
    const int shift = pass * bits;
    for (int i = threadIdx.x; i < WARPS * MOST; i += GR_ONE_THREADS) next[0][i] = 0u;
    __syncthreads();
    uint2 pair[GR_ONE_ITEMS];
#pragma unroll
    for (int r = 0; r < GR_ONE_ITEMS; ++r) {
      const int i = base + r * 32;
      const bool have = r < items && i < edges;
      pair[r] = !have ? make_uint2(0u, 0u) : pass == 0 ? gr_pair(index, nullptr, rows, i) : sorted[i];
      if (have) atomicAdd(&next[warp][(pair[r].x >> shift) & (bins - 1)], 1u);
    }
    __syncthreads();
    const int d = threadIdx.x;  // a digit per thread
    uint32_t here = 0u, unused;
    if (d < bins)
      for (int w = 0; w < WARPS; ++w) here += next[w][d];
    uint32_t at = gr_block_scan<WARPS>(here, warp_sums, unused);
    if (d < bins)
      for (int w = 0; w < WARPS; ++w) {
        const uint32_t c = next[w][d];
        next[w][d] = at;
        at += c;
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < GR_ONE_ITEMS; ++r) {
      if (r >= items) break;
      const bool have = base + r * 32 < edges;
      const uint32_t digit = have ? (pair[r].x >> shift) & (bins - 1) : (uint32_t)bins;
      const uint32_t to = gr_place(have, digit, bits, next[warp]);
      if (have) sorted[to] = pair[r];
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < edges; i += GR_ONE_THREADS) out[i] = sorted[i];
  if (starts)
    for (int64_t row = threadIdx.x; row <= rows; row += GR_ONE_THREADS) {
      int lo = 0, hi = edges;  // the first pair of this row or a later one
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (sorted[mid].x < row)
          lo = mid + 1;
        else
          hi = mid;
      }
      starts[row] = lo;
    }
}

// A lane per (row, 16 bytes of channels); GR_SLOTS warps take contiguous shares of the row's pairs, which are added in
// order.
template <typename T, int VL>
__global__ void __launch_bounds__(32 * GR_SLOTS) gather_sum_rows_kernel(const T *__restrict__ dout,
                                                                        const uint2 *__restrict__ keys,
                                                                        const int *__restrict__ starts, int64_t total,
                                                                        int units, float scale, T *__restrict__ dx) {
  constexpr int AHEAD = 4;
  __shared__ float share[GR_SLOTS][VL][32];
  const int lane = threadIdx.x & 31, slot = threadIdx.x >> 5;
  const int64_t i = (int64_t)blockIdx.x * 32 + lane;
  const bool have = i < total;
  const int64_t row = i / units, u = i - row * units;
  int lo = 0, hi = 0;
  if (have) {
    const int first = starts[row], count = starts[row + 1] - first;
    lo = first + (int)((int64_t)count * slot / GR_SLOTS);
    hi = first + (int)((int64_t)count * (slot + 1) / GR_SLOTS);
  }
  const GrVec<T, VL> *src = reinterpret_cast<const GrVec<T, VL> *>(dout);
  float acc[VL] = {};
  for (int j = lo; j < hi; j += AHEAD) {
    GrVec<T, VL> v[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) v[n] = src[(int64_t)keys[j + n < hi ? j + n : hi - 1].y * units + u];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n)
      if (j + n < hi) {
#pragma unroll
        for (int c = 0; c < VL; ++c) acc[c] += gr_float(v[n].v[c]);
      }
  }
#pragma unroll
  for (int c = 0; c < VL; ++c) share[slot][c][lane] = acc[c];
  __syncthreads();
  if (slot != 0 || !have) return;
  GrVec<T, VL> r;
#pragma unroll
  for (int c = 0; c < VL; ++c) {
    for (int s = 1; s < GR_SLOTS; ++s) acc[c] += share[s][c][lane];
    r.v[c] = gr_round<T>(acc[c] * scale);
  }
  reinterpret_cast<GrVec<T, VL> *>(dx)[i] = r;
}

// ---- sums over runs of equal keys ----------------------------------------------------------------------------
// Piece g covers the sorted pairs [g G, g G + G).  part[2 g] holds the sum of a run that reaches the piece's start from
// before or begins there and leaves its end; part[2 g + 1] that of a run that begins inside and leaves the end.
template <typename T, int VL>
__global__ void __launch_bounds__(GR_THREADS) gather_sum_kernel(const T *__restrict__ dout,
                                                                const uint2 *__restrict__ keys, int64_t rows,
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
  uint32_t run = keys[lo].x;
  bool whole = lo == 0 || keys[lo - 1].x != run;  // the run began at or after this piece's start
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
  // the pairs of the next rows are on their way while these rows are
  uint2 pair[AHEAD];
#pragma unroll
  for (int n = 0; n < AHEAD; ++n) pair[n] = keys[lo + n < hi ? lo + n : hi - 1];
  for (int64_t i0 = lo; i0 < hi; i0 += AHEAD) {
    uint32_t key[AHEAD];
    GrVec<T, VL> row[AHEAD];
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) {
      key[n] = pair[n].x;
      row[n] = src[(int64_t)pair[n].y * units + u];
    }
#pragma unroll
    for (int n = 0; n < AHEAD; ++n) pair[n] = keys[i0 + AHEAD + n < hi ? i0 + AHEAD + n : hi - 1];
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
  flush(hi == edges || keys[hi].x != run);
}

// Where the run that leaves piece g began in g: its pieces are g .. last; returns last, or -1 if none does.
__device__ __forceinline__ int64_t gr_run(const uint2 *keys, int64_t edges, int piece, int64_t pieces, int64_t g,
                                          uint32_t &run, int &slot) {
  const int64_t lo = g * piece, hi = lo + piece;
  if (hi >= edges) return -1;
  run = keys[hi - 1].x;
  if (keys[hi].x != run) return -1;
  slot = keys[lo].x == run ? 0 : 1;
  if (slot == 0 && lo > 0 && keys[lo - 1].x == run) return -1;  // began earlier
  // the last piece whose first key is the run's: in steps of twice the size as far as it goes, then of half (most end
  // at once)
  int64_t a = g + 1, step = 1;
  while (a + step < pieces && keys[(a + step) * piece].x == run) a += step, step *= 2;
  for (step /= 2; step > 0; step /= 2)
    if (a + step < pieces && keys[(a + step) * piece].x == run) a += step;
  return a;
}

template <typename T, int VL>
__global__ void __launch_bounds__(GR_THREADS) gather_join_kernel(const uint2 *__restrict__ keys, int64_t rows,
                                                                 int64_t edges, int units, int piece, int64_t pieces,
                                                                 float scale, T *__restrict__ dx,
                                                                 const float *__restrict__ part, int most,
                                                                 int *__restrict__ num_long,
                                                                 uint2 *__restrict__ long_runs) {
  const int64_t id = (int64_t)blockIdx.x * GR_THREADS + threadIdx.x;
  const int64_t g = id / units, u = id - g * units;
  if (g >= pieces) return;
  uint32_t run;
  int slot;
  const int64_t last = gr_run(keys, edges, piece, pieces, g, run, slot);
  if (last < 0 || run >= rows) return;
  if (last - g > most) {
    if (u == 0) long_runs[atomicAdd(num_long, 1)] = make_uint2((uint32_t)g, (uint32_t)last);
    return;
  }
  float acc[VL];
#pragma unroll
  for (int c = 0; c < VL; ++c) acc[c] = part[((2 * g + slot) * units + u) * VL + c];
#pragma unroll 8
  for (int64_t h = g + 1; h <= last; ++h)
#pragma unroll
    for (int c = 0; c < VL; ++c) acc[c] += part[(2 * h * units + u) * VL + c];
  GrVec<T, VL> r;
#pragma unroll
  for (int c = 0; c < VL; ++c) r.v[c] = gr_round<T>(acc[c] * scale);
  reinterpret_cast<GrVec<T, VL> *>(dx)[(int64_t)run * units + u] = r;
}

// A block per (long run, 32 channels): its warps add contiguous shares of its pieces, then one adds the shares in
// order.
template <typename T>
__global__ void __launch_bounds__(32 * GR_LONG_WARPS) gather_join_long_kernel(const uint2 *__restrict__ keys, int64_t rows,
                                                                      int64_t edges, int channels, int piece,
                                                                      int64_t pieces, float scale, T *__restrict__ dx,
                                                                      const float *__restrict__ part,
                                                                      const int *__restrict__ num_long,
                                                                      const uint2 *__restrict__ long_runs) {
  __shared__ float share[GR_LONG_WARPS][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int slabs = (channels + 31) / 32;
  const int64_t tasks = (int64_t)*num_long * slabs;
  for (int64_t t = blockIdx.x; t < tasks; t += gridDim.x) {
    const uint2 pieces_of = long_runs[t / slabs];
    const int64_t g = pieces_of.x, n = (int64_t)pieces_of.y - g + 1;
    const uint32_t run = keys[(g + 1) * piece].x;
    const int c = (int)(t % slabs) * 32 + lane;
    const int64_t each = (n + GR_LONG_WARPS - 1) / GR_LONG_WARPS;
    int64_t a = warp * each;
    const int64_t b = a + each < n ? a + each : n;
    float acc = 0.f;
    if (c < channels) {
      const float *src = part + 2 * g * channels + c;
      if (a == 0) {  // the run's first piece, where it need not begin at the start
        acc = src[keys[g * piece].x == run ? 0 : channels];
        a = 1;
      }
      // 16 loads on their way, whole or not: the longest run sets the time
      for (int64_t h = a; h < b; h += 16) {
        const int count = b - h < 16 ? (int)(b - h) : 16;
        const float *at = src + 2 * h * channels;
        float v[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = at[(int64_t)(i < count ? i : 0) * 2 * channels];
#pragma unroll
        for (int i = 0; i < 16; ++i) acc += i < count ? v[i] : 0.f;
      }
    }
    share[warp][lane] = acc;
    __syncthreads();
    if (warp == 0 && c < channels) {
      acc = 0.f;
#pragma unroll
      for (int w = 0; w < GR_LONG_WARPS; ++w) acc += share[w][lane];
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
  size_t pairs, counts, totals, part, runs, total;
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
  // Where rows are named thousands of times (node types), longer pieces leave less to join, as long as there are enough
  // of them: 1000003 edges of 128 channels on 100 rows, a third of them on one, 139 us of sums and joins -> 127.
  while (p.piece < 256 && rows > 0 && edges / rows >= 8 * p.piece &&
         edges / (2 * p.piece) * channels >= 148 * 2048)
    p.piece *= 2;
  p.pieces = (edges + p.piece - 1) / p.piece;
  const int64_t bins = (1ll << p.bits) * p.blocks;
  p.pairs = gr_align((size_t)edges * 8);
  if (edges <= GR_ROWS && rows <= GR_ROWS) p.pairs += gr_align((size_t)(rows + 1) * 4);  // the rows' places
  p.counts = gr_align((size_t)bins * 4);
  p.totals = gr_align((size_t)4 << p.bits);
  p.part = gr_align((size_t)p.pieces * 2 * channels * 4);
  p.runs = gr_align((size_t)(p.pieces + 1) * 8);
  p.total = 2 * p.pairs + p.counts + p.totals + p.part + p.runs;
  return p;
}

template <typename T, int VL>
static int gr_forward(const void *x, const int64_t *index, int64_t rows, int64_t edges, int64_t channels, float scale,
                      void *out, cudaStream_t stream) {
  const int64_t total = edges * (channels / VL);
  constexpr int SHARE = GR_THREADS * GR_EDGES;
  gather_rows_kernel<T, VL><<<(unsigned)((total + SHARE - 1) / SHARE), GR_THREADS, 0, stream>>>(
      (const T *)x, index, rows, total, (int)(channels / VL), scale, (T *)out);
  B200C_LAUNCH_CHECK("gather_rows_kernel");
  return B200C_OK;
}

template <typename T, int VL>
static int gr_backward(const void *dout, const int64_t *index, int64_t rows, int64_t edges, int64_t channels,
                       float scale, void *dx, void *workspace, cudaStream_t stream) {
  const GrPlan p = gr_plan(rows, edges, channels);
  char *ws = (char *)workspace;
  uint2 *pairs[2];
  for (int i = 0; i < 2; ++i) pairs[i] = (uint2 *)ws, ws += p.pairs;
  uint32_t *counts = (uint32_t *)ws;
  ws += p.counts;
  uint32_t *totals = (uint32_t *)ws;
  ws += p.totals;
  float *part = (float *)ws;
  ws += p.part;
  int *num_long = (int *)ws;
  uint2 *long_runs = (uint2 *)ws + 1;

  const bool one = edges <= GR_ONE, whole = edges <= GR_ROWS && rows <= GR_ROWS;
  if (!whole) B200C_CUDA(cudaMemsetAsync(dx, 0, (size_t)rows * channels * sizeof(T), stream));  // rows of no index
  const uint2 *k = nullptr;
  if (one) {
    constexpr size_t smem = (size_t)GR_ONE * 8 + (size_t)(GR_ONE_THREADS / 32) * (4 << GR_MAX_BITS);
    static unsigned long long configured = 0ull;
    B200C_CUDA(opt_in_shared_memory(gather_sort_one_kernel, smem, configured));
    gather_sort_one_kernel<<<1, GR_ONE_THREADS, smem, stream>>>(index, rows, (int)edges, p.passes, p.bits, pairs[0],
                                                                 whole ? (int *)pairs[1] : nullptr);
    B200C_LAUNCH_CHECK("gather_sort_one_kernel");
    k = pairs[0];
    if (whole) {
      const int64_t total = rows * (channels / VL);
      gather_sum_rows_kernel<T, VL><<<(unsigned)((total + 31) / 32), 32 * GR_SLOTS, 0, stream>>>(
          (const T *)dout, k, (const int *)pairs[1], total, (int)(channels / VL), scale, (T *)dx);
      B200C_LAUNCH_CHECK("gather_sum_rows_kernel");
      return B200C_OK;
    }
  } else {
    constexpr size_t smem = (size_t)GR_TILE * 8 + (size_t)(GR_WARPS + 1) * (4 << GR_MAX_BITS);
    static unsigned long long configured = 0ull;
    B200C_CUDA(opt_in_shared_memory(gather_sort_scatter_kernel, smem, configured));
    const bool few = p.blocks <= GR_FEW;
    for (int pass = 0; pass < p.passes; ++pass) {
      gather_sort_count_kernel<<<(unsigned)p.blocks, GR_THREADS, 0, stream>>>(index, k, rows, edges, pass * p.bits,
                                                                              p.bits, counts, num_long);
      B200C_LAUNCH_CHECK("gather_sort_count_kernel");
      if (!few) {
        gather_sort_scan_kernel<<<1u << p.bits, GR_THREADS, 0, stream>>>(counts, p.blocks, totals);
        B200C_LAUNCH_CHECK("gather_sort_scan_kernel");
      }
      gather_sort_scatter_kernel<<<(unsigned)p.blocks, GR_THREADS, smem, stream>>>(
          index, k, rows, edges, pass * p.bits, p.bits, counts, few ? nullptr : totals, pairs[pass & 1]);
      B200C_LAUNCH_CHECK("gather_sort_scatter_kernel");
      k = pairs[pass & 1];
    }
  }
  const int units = (int)(channels / VL);
  const unsigned blocks = (unsigned)((p.pieces * units + GR_THREADS - 1) / GR_THREADS);
  gather_sum_kernel<T, VL><<<blocks, GR_THREADS, 0, stream>>>((const T *)dout, k, rows, edges, units, p.piece, p.pieces,
                                                              scale, (T *)dx, part);
  B200C_LAUNCH_CHECK("gather_sum_kernel");
  gather_join_kernel<T, VL><<<blocks, GR_THREADS, 0, stream>>>(k, rows, edges, units, p.piece, p.pieces, scale,
                                                               (T *)dx, part, one ? GR_ONE : GR_SHORT, num_long,
                                                               long_runs);
  B200C_LAUNCH_CHECK("gather_join_kernel");
  if (one) return B200C_OK;
  gather_join_long_kernel<T><<<296, 32 * GR_LONG_WARPS, 0, stream>>>(k, rows, edges, (int)channels, p.piece, p.pieces, scale,
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
