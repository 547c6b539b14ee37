// Attention for every type and channel count, on the FP32 pipe (see attention.cuh for the formulas).
//
// A block of 256 threads owns 64 rows of one head and walks the other side's rows of the same example in tiles of
// 64: one pass over the keys with the running maximum and sum of the softmax.  Operands are widened to fp32 and kept
// transposed in shared memory ([channel][row], rows padded to 68 so that the 16-byte reads of both products are
// free of bank conflicts); a thread holds a 4 x 4 tile of the scores and 4 x channels/16 of the result.  Where shared
// memory has room for two blocks per SM all the same, the next tile is on its way (asynchronous copies for fp32) while
// this one is worked on.  tanh is CUDA's: an error of the hardware's form would be multiplied by the cap. Tiles begin
// with an example, so that a block walks one example's columns (fp32, 8 clouds of 256 to 676 points: forward 223 -> 136
// us, dq 264 -> 165, dk and dv 317 -> 196 against 64 rows wherever they fall).  Where examples are shorter than 16
// rows, tiles hold rows of several; those are processed one example after the other, so that a NaN in one example never
// meets another one's zeros. The backward pass is two kernels of the same shape: one owns 64 queries and sums dq over
// the keys, one owns 64 keys and sums dk and dv over the queries of all heads of its group.  Scores are formed twice,
// but nothing is added atomically: the result does not depend on the order of the blocks.
#include <type_traits>

#include "attention_tensor.cuh"

namespace b200c {

constexpr int AP_T = 64;        // rows and columns of a tile
constexpr int AP_LD = AP_T + 4;
constexpr int AP_THREADS = 256;

__device__ __forceinline__ void ap_copy(float *dst, const float *src, bool there) {
  const unsigned bytes = there ? 4u : 0u;  // nothing is read where there is nothing: zeros are written
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;\n" ::"r"((unsigned)__cvta_generic_to_shared(dst)), "l"(src),
               "r"(bytes)
               : "memory");
}

// rows [row0, row0 + 64) of src (rows outside [lo, hi) are zero) to dst[channel][row]; fp32 asynchronously.  A thread
// keeps its channel and adds up its address: worked out for every element, addresses were a third of all instructions
// (forward of 8 clouds of 500 points, 44 channels: 136 -> 119 us).
template <typename T, int CP>
__device__ __forceinline__ void ap_load(float *dst, const T *__restrict__ src, int64_t row_stride, int64_t row0,
                                        int64_t lo, int64_t hi, int channels, int tid) {
  constexpr int WIDTH = CP <= 32 ? 32 : CP <= 64 ? 64 : 128, STEP = AP_THREADS / WIDTH;
  const int c = tid % WIDTH, r0 = tid / WIDTH;
  if (c >= CP) return;
  const int64_t from = lo - row0, to = hi - row0;
  const int r_lo = from < 0 ? 0 : from > AP_T ? AP_T : (int)from;
  const int r_hi = c >= channels || to < 0 ? 0 : to > AP_T ? AP_T : (int)to;
  const T *at = src + (row0 + r0) * row_stride + c;
  const int64_t step = STEP * row_stride;
  float *to_at = dst + c * AP_LD + r0;
#pragma unroll 8
  for (int r = r0; r < AP_T; r += STEP, at += step, to_at += STEP) {
    const bool there = r >= r_lo && r < r_hi;
    if constexpr (sizeof(T) == 4)
      ap_copy(to_at, there ? at : src, there);
    else
      *to_at = there ? at_float(*at) : 0.f;
  }
}

__device__ __forceinline__ void ap_load_pos(float *dst, const float *__restrict__ src, int dims, int64_t row0,
                                            int64_t lo, int64_t hi, int tid) {
  for (int i = tid; i < AP_T * dims; i += AP_THREADS) {
    const int r = i / dims, d = i - r * dims;
    const int64_t row = row0 + r;
    const bool there = row >= lo && row < hi;
    ap_copy(dst + d * AP_LD + r, there ? src + row * dims + d : src, there);
  }
}

// acc[i][j] += sum_c a[c][4 ty + i] b[c][4 tx + j]
__device__ __forceinline__ void ap_scores(const float *a, const float *b, int channels, int ty, int tx,
                                          float (&acc)[4][4]) {
#pragma unroll 4
  for (int c = 0; c < channels; ++c) {
    const float4 x = *reinterpret_cast<const float4 *>(a + c * AP_LD + 4 * ty);
    const float4 y = *reinterpret_cast<const float4 *>(b + c * AP_LD + 4 * tx);
    const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(xs[i], ys[j], acc[i][j]);
  }
}

// acc[i][n] += sum_j w[4 ty + i][j] b[tx + 16 n][j]
template <int NC>
__device__ __forceinline__ void ap_accumulate(const float *w, const float *b, int ty, int tx, float (&acc)[4][NC]) {
  for (int j = 0; j < AP_T; j += 4) {
    float4 x[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const float4 *>(w + (4 * ty + i) * AP_LD + j);
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const float4 y = *reinterpret_cast<const float4 *>(b + (tx + 16 * n) * AP_LD + j);
#pragma unroll
      for (int i = 0; i < 4; ++i)
        acc[i][n] = fmaf(x[i].x, y.x, fmaf(x[i].y, y.y, fmaf(x[i].z, y.z, fmaf(x[i].w, y.w, acc[i][n]))));
    }
  }
}

// log2 e (t - slope |pos_a - pos_b|) of the 4 x 4 tile; bend[i][j] = 1 - (t / cap)^2.  Coordinates are read four
// rows and four columns at a time (forward 119 -> 102 us).
template <bool BEND>
__device__ __forceinline__ void ap_logits(float (&s)[4][4], float (&bend)[4][4], const float *pa, const float *pb,
                                          int dims, int ty, int tx, float scale, float cap, float slope) {
  const float inv_cap = cap > 0.f ? 1.f / cap : 0.f;
  float d2[4][4] = {};
  for (int d = 0; d < dims; ++d) {
    const float4 x = *reinterpret_cast<const float4 *>(pa + d * AP_LD + 4 * ty);
    const float4 y = *reinterpret_cast<const float4 *>(pb + d * AP_LD + 4 * tx);
    const float xs[4] = {x.x, x.y, x.z, x.w}, ys[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float df = xs[i] - ys[j];
        d2[i][j] = fmaf(df, df, d2[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float t = s[i][j] * scale;
      if (BEND) bend[i][j] = 1.f;
      if (cap > 0.f) {
        const float u = tanhf(t * inv_cap);
        t = cap * u;
        if (BEND) bend[i][j] = 1.f - u * u;
      }
      if (dims > 0) t = fmaf(-slope, t5_sqrt(d2[i][j]), t);
      s[i][j] = t * AT_LOG2E;
    }
}

__device__ __forceinline__ float ap_max16(float v) {
  for (int o = 8; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(FULL_MASK, v, o));
  return v;
}
__device__ __forceinline__ float ap_sum16(float v) {
  for (int o = 8; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  return v;
}

// floats of shared memory: `own` tiles of the block's rows, two of the columns in BUFS sets (with coordinates and
// statistics), the weights.  Two sets where two blocks then still fit an SM.
template <int CP, int OWN>
struct ApSmem {
  static constexpr int TILE = CP * AP_LD, W = AP_T * AP_LD, POS = AT_MAX_DIMS * AP_LD, STAT = 2 * AP_T;
  static constexpr int SET = 2 * TILE + POS + STAT;
  static constexpr int BUFS = (OWN * TILE + POS + W + 2 * SET) * 4 <= 113 * 1024 ? 2 : 1;
  static constexpr int FLOATS = OWN * TILE + POS + W + BUFS * SET;
};

// Whether tiles begin with an example; the blocks of a launch then.
__host__ __device__ __forceinline__ bool ap_aligned(const int64_t *ptr, int64_t rows, int64_t segments) {
  return ptr != nullptr && segments <= rows / 16;
}
static unsigned ap_blocks(const int64_t *ptr, int64_t rows, int64_t segments) {
  return (unsigned)(ap_aligned(ptr, rows, segments) ? rows / AP_T + segments : (rows + AP_T - 1) / AP_T);
}
// The rows [t0, t1) of tile i, or false where there are none.  The tiles of segment b are numbered from (first row of
// b) / 64 + b, which leaves room for all of them; rows outside every segment go with the first or the last.
__device__ __forceinline__ bool ap_tile(const int64_t *__restrict__ ptr, int64_t rows, int segments, int64_t i,
                                        int64_t &t0, int64_t &t1) {
  t0 = i * AP_T;
  int64_t end = rows;
  if (ap_aligned(ptr, rows, segments)) {
    const auto first = [&](int b) {
      const int64_t at = b == 0 ? 0 : ptr[b];
      return at < 0 ? 0 : at > rows ? rows : at;
    };
    int lo = 0, hi = segments - 1;  // the last segment whose number is not above i
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (first(mid) / AP_T + mid <= i)
        lo = mid;
      else
        hi = mid - 1;
    }
    t0 = first(lo) + (i - first(lo) / AP_T - lo) * AP_T;
    if (lo + 1 < segments) end = first(lo + 1);
  }
  t1 = t0 + AP_T < end ? t0 + AP_T : end;
  return t0 < t1;
}

template <typename T, int CP>
__global__ void __launch_bounds__(AP_THREADS) attention_plain_forward_kernel(AttnArgs a) {
  constexpr int NC = CP / 16;
  using S = ApSmem<CP, 1>;
  extern __shared__ __align__(16) float ap_smem[];
  float *sq = ap_smem, *sw = sq + S::TILE, *spq = sw + S::W, *sets = spq + S::POS;
  const b200c_attention_t &p = a.p;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int head = blockIdx.y, group = head / (p.heads / p.groups);
  const T *q = (const T *)p.q + (int64_t)head * p.q_head;
  const T *k = (const T *)p.k + (int64_t)group * p.k_head;
  const T *v = (const T *)p.v + (int64_t)group * p.v_head;
  const float slope = p.dims > 0 ? p.slope[head] : 0.f;
  int64_t t0, t1;
  if (!ap_tile(p.ptr_q, p.m, (int)p.num_segments, blockIdx.x, t0, t1)) return;
  T *out = (T *)a.out, *rest = (T *)a.rest;

  ap_load<T, CP>(sq, q, p.q_row, t0, t0, t1, p.channels, tid);
  if (p.dims > 0) ap_load_pos(spq, p.pos_q, p.dims, t0, t0, t1, tid);
  // rows of no example stay at zero
  for (int64_t row = t0; row < t1; ++row) {
    const int b = segment_of(p.ptr_q, p.num_segments, row);
    int64_t lo, hi;
    at_segment(p.ptr_q, p.m, b, lo, hi);
    if (row >= lo && row < hi) {
      row = hi - 1;
      continue;
    }
    for (int c = tid; c < p.channels; c += AP_THREADS) {
      out[(row * p.heads + head) * p.channels + c] = at_round<T>(0.f);
      if (rest) rest[(row * p.heads + head) * p.channels + c] = at_round<T>(0.f);
    }
    if (a.lse && tid == 0) a.lse[(int64_t)head * p.m + row] = pos_inf<float>();
  }
  const int b_first = segment_of(p.ptr_q, p.num_segments, t0), b_last = segment_of(p.ptr_q, p.num_segments, t1 - 1);
  for (int b = b_first; b <= b_last; ++b) {
    int64_t q_lo, q_hi, k_lo, k_hi;
    at_segment(p.ptr_q, p.m, b, q_lo, q_hi);
    at_segment(p.ptr_k, p.n, b, k_lo, k_hi);
    if (q_lo < t0) q_lo = t0;
    if (q_hi > t1) q_hi = t1;
    if (q_lo >= q_hi) continue;
    float o[4][NC] = {}, top[4], sum[4] = {};
#pragma unroll
    for (int i = 0; i < 4; ++i) top[i] = -pos_inf<float>();
    auto fetch = [&](int64_t c0, int set) {
      float *sk = sets + set * S::SET, *sv = sk + S::TILE, *spk = sv + S::TILE;
      ap_load<T, CP>(sk, k, p.k_row, c0, k_lo, k_hi, p.channels, tid);
      ap_load<T, CP>(sv, v, p.v_row, c0, k_lo, k_hi, p.channels, tid);
      if (p.dims > 0) ap_load_pos(spk, p.pos_k, p.dims, c0, k_lo, k_hi, tid);
    };
    int set = 0;
    __syncthreads();
    if (S::BUFS == 2 && k_lo < k_hi) fetch(k_lo, 0);
    for (int64_t c0 = k_lo; c0 < k_hi; c0 += AP_T) {
      // this tile is in; nobody reads the other set any more
      if (S::BUFS == 1) {
        __syncthreads();
        fetch(c0, 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
      __syncthreads();
      const float *sk = sets + set * S::SET, *sv = sk + S::TILE, *spk = sv + S::TILE;
      if (S::BUFS == 2) {
        set ^= 1;
        if (c0 + AP_T < k_hi) fetch(c0 + AP_T, set);
      }
      float s[4][4] = {}, unused[4][4];
      ap_scores(sq, sk, p.channels, ty, tx, s);
      ap_logits<false>(s, unused, spq, spk, p.dims, ty, tx, p.scale, p.cap, slope);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float m = top[i];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          if (c0 + 4 * tx + j >= k_hi) s[i][j] = -pos_inf<float>();
          m = fmaxf(m, s[i][j]);
        }
        m = ap_max16(m);
        const float base = m == -pos_inf<float>() ? 0.f : m;
        const float shrink = t5_ex2(top[i] - base);
        top[i] = m;
        float part = 0.f;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          s[i][j] = t5_ex2(s[i][j] - base);
          part += s[i][j];
        }
        sum[i] = fmaf(sum[i], shrink, ap_sum16(part));
#pragma unroll
        for (int n = 0; n < NC; ++n) o[i][n] *= shrink;
        *reinterpret_cast<float4 *>(sw + (4 * ty + i) * AP_LD + 4 * tx) =
            make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
      }
      __syncwarp();  // a row of the weights is written and read by the same half warp
      ap_accumulate<NC>(sw, sv, ty, tx, o);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = t0 + 4 * ty + i;
      if (row < q_lo || row >= q_hi) continue;
      const float inv = sum[i] == 0.f ? 0.f : 1.f / sum[i];  // NaN sums stay NaN
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int c = tx + 16 * n;
        if (c >= p.channels) continue;
        const T r = at_round<T>(o[i][n] * inv);
        out[(row * p.heads + head) * p.channels + c] = r;
        if (rest) rest[(row * p.heads + head) * p.channels + c] = at_round<T>(o[i][n] * inv - at_float(r));
      }
      if (a.lse && tx == 0)
        a.lse[(int64_t)head * p.m + row] = sum[i] == 0.f ? pos_inf<float>() : top[i] + log2f(sum[i]);
    }
  }
  cp_async_wait<0>();  // a block without a tile still has its own rows' copies under way
}

// dq of 64 queries of one head
template <typename T, int CP>
__global__ void __launch_bounds__(AP_THREADS) attention_plain_dq_kernel(AttnArgs a) {
  constexpr int NC = CP / 16;
  using S = ApSmem<CP, 2>;
  extern __shared__ __align__(16) float ap_smem[];
  float *sq = ap_smem, *sdo = sq + S::TILE, *sw = sdo + S::TILE, *spq = sw + S::W, *sets = spq + S::POS;
  const b200c_attention_t &p = a.p;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int head = blockIdx.y, group = head / (p.heads / p.groups);
  const int64_t qrow = (int64_t)p.heads * p.channels;
  const T *q = (const T *)p.q + (int64_t)head * p.q_head;
  const T *k = (const T *)p.k + (int64_t)group * p.k_head;
  const T *v = (const T *)p.v + (int64_t)group * p.v_head;
  const T *dout = (const T *)a.dout + (int64_t)head * p.channels;
  T *dq = (T *)a.dq + (int64_t)head * p.channels;
  const float slope = p.dims > 0 ? p.slope[head] : 0.f;
  int64_t t0, t1;
  if (!ap_tile(p.ptr_q, p.m, (int)p.num_segments, blockIdx.x, t0, t1)) return;

  ap_load<T, CP>(sq, q, p.q_row, t0, t0, t1, p.channels, tid);
  ap_load<T, CP>(sdo, dout, qrow, t0, t0, t1, p.channels, tid);
  if (p.dims > 0) ap_load_pos(spq, p.pos_q, p.dims, t0, t0, t1, tid);
  for (int64_t row = t0; row < t1; ++row) {
    const int b = segment_of(p.ptr_q, p.num_segments, row);
    int64_t lo, hi;
    at_segment(p.ptr_q, p.m, b, lo, hi);
    if (row >= lo && row < hi) {
      row = hi - 1;
      continue;
    }
    for (int c = tid; c < p.channels; c += AP_THREADS) dq[row * qrow + c] = at_round<T>(0.f);
  }
  float lse[4], delta[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int64_t row = t0 + 4 * ty + i;
    lse[i] = row < t1 ? a.lse[(int64_t)head * p.m + row] : pos_inf<float>();
    delta[i] = row < t1 ? a.delta[(int64_t)head * p.m + row] : 0.f;
  }
  const int b_first = segment_of(p.ptr_q, p.num_segments, t0), b_last = segment_of(p.ptr_q, p.num_segments, t1 - 1);
  for (int b = b_first; b <= b_last; ++b) {
    int64_t q_lo, q_hi, k_lo, k_hi;
    at_segment(p.ptr_q, p.m, b, q_lo, q_hi);
    at_segment(p.ptr_k, p.n, b, k_lo, k_hi);
    if (q_lo < t0) q_lo = t0;
    if (q_hi > t1) q_hi = t1;
    if (q_lo >= q_hi) continue;
    float acc[4][NC] = {};
    auto fetch = [&](int64_t c0, int set) {
      float *sk = sets + set * S::SET, *sv = sk + S::TILE, *spk = sv + S::TILE;
      ap_load<T, CP>(sk, k, p.k_row, c0, k_lo, k_hi, p.channels, tid);
      ap_load<T, CP>(sv, v, p.v_row, c0, k_lo, k_hi, p.channels, tid);
      if (p.dims > 0) ap_load_pos(spk, p.pos_k, p.dims, c0, k_lo, k_hi, tid);
    };
    int set = 0;
    __syncthreads();
    if (S::BUFS == 2 && k_lo < k_hi) fetch(k_lo, 0);
    for (int64_t c0 = k_lo; c0 < k_hi; c0 += AP_T) {
      // this tile is in; nobody reads the other set any more
      if (S::BUFS == 1) {
        __syncthreads();
        fetch(c0, 0);
      }
      cp_async_commit();
      cp_async_wait<0>();
      __syncthreads();
      const float *sk = sets + set * S::SET, *sv = sk + S::TILE, *spk = sv + S::TILE;
      if (S::BUFS == 2) {
        set ^= 1;
        if (c0 + AP_T < k_hi) fetch(c0 + AP_T, set);
      }
      float s[4][4] = {}, dp[4][4] = {}, bend[4][4];
      ap_scores(sq, sk, p.channels, ty, tx, s);
      ap_scores(sdo, sv, p.channels, ty, tx, dp);
      ap_logits<true>(s, bend, spq, spk, p.dims, ty, tx, p.scale, p.cap, slope);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const bool there = c0 + 4 * tx + j < k_hi && lse[i] < pos_inf<float>();
          const float w = t5_ex2(s[i][j] - lse[i]) * (dp[i][j] - delta[i]) * bend[i][j];
          s[i][j] = there || lse[i] != lse[i] ? w : 0.f;
          if (c0 + 4 * tx + j >= k_hi) s[i][j] = 0.f;
        }
        *reinterpret_cast<float4 *>(sw + (4 * ty + i) * AP_LD + 4 * tx) =
            make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
      }
      __syncwarp();
      ap_accumulate<NC>(sw, sk, ty, tx, acc);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = t0 + 4 * ty + i;
      if (row < q_lo || row >= q_hi) continue;
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int c = tx + 16 * n;
        if (c < p.channels) dq[row * qrow + c] = at_round<T>(acc[i][n] * p.scale);
      }
    }
  }
  cp_async_wait<0>();  // a block without a tile still has its own rows' copies under way
}

// dk and dv of 64 keys of one group
template <typename T, int CP>
__global__ void __launch_bounds__(AP_THREADS) attention_plain_dkv_kernel(AttnArgs a) {
  constexpr int NC = CP / 16;
  using S = ApSmem<CP, 2>;
  extern __shared__ __align__(16) float ap_smem[];
  float *sk = ap_smem, *sv = sk + S::TILE, *sw = sv + S::TILE, *spk = sw + S::W, *sets = spk + S::POS;
  const b200c_attention_t &p = a.p;
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int group = blockIdx.y, per_group = p.heads / p.groups;
  const int64_t qrow = (int64_t)p.heads * p.channels, krow = (int64_t)p.groups * p.channels;
  const T *k = (const T *)p.k + (int64_t)group * p.k_head;
  const T *v = (const T *)p.v + (int64_t)group * p.v_head;
  T *dk = (T *)a.dk + (int64_t)group * p.channels, *dv = (T *)a.dv + (int64_t)group * p.channels;
  int64_t t0, t1;
  if (!ap_tile(p.ptr_k, p.n, (int)p.num_segments, blockIdx.x, t0, t1)) return;

  ap_load<T, CP>(sk, k, p.k_row, t0, t0, t1, p.channels, tid);
  ap_load<T, CP>(sv, v, p.v_row, t0, t0, t1, p.channels, tid);
  if (p.dims > 0) ap_load_pos(spk, p.pos_k, p.dims, t0, t0, t1, tid);
  for (int64_t row = t0; row < t1; ++row) {
    const int b = segment_of(p.ptr_k, p.num_segments, row);
    int64_t lo, hi;
    at_segment(p.ptr_k, p.n, b, lo, hi);
    if (row >= lo && row < hi) {
      row = hi - 1;
      continue;
    }
    for (int c = tid; c < p.channels; c += AP_THREADS) dk[row * krow + c] = dv[row * krow + c] = at_round<T>(0.f);
  }
  const int b_first = segment_of(p.ptr_k, p.num_segments, t0), b_last = segment_of(p.ptr_k, p.num_segments, t1 - 1);
  for (int b = b_first; b <= b_last; ++b) {
    int64_t q_lo, q_hi, k_lo, k_hi;
    at_segment(p.ptr_q, p.m, b, q_lo, q_hi);
    at_segment(p.ptr_k, p.n, b, k_lo, k_hi);
    if (k_lo < t0) k_lo = t0;
    if (k_hi > t1) k_hi = t1;
    if (k_lo >= k_hi) continue;
    float gk[4][NC] = {}, gv[4][NC] = {};
    for (int e = 0; e < per_group; ++e) {
      const int head = group * per_group + e;
      const float slope = p.dims > 0 ? p.slope[head] : 0.f;
      const T *q = (const T *)p.q + (int64_t)head * p.q_head, *dout = (const T *)a.dout + (int64_t)head * p.channels;
      auto fetch = [&](int64_t c0, int set) {
        float *sq = sets + set * S::SET, *sdo = sq + S::TILE, *spq = sdo + S::TILE, *stat = spq + S::POS;
        ap_load<T, CP>(sq, q, p.q_row, c0, q_lo, q_hi, p.channels, tid);
        ap_load<T, CP>(sdo, dout, qrow, c0, q_lo, q_hi, p.channels, tid);
        if (p.dims > 0) ap_load_pos(spq, p.pos_q, p.dims, c0, q_lo, q_hi, tid);
        if (tid < AP_T) {
          const bool there = c0 + tid < q_hi;
          stat[tid] = there ? a.lse[(int64_t)head * p.m + c0 + tid] : pos_inf<float>();
          stat[AP_T + tid] = there ? a.delta[(int64_t)head * p.m + c0 + tid] : 0.f;
        }
      };
      int set = 0;
      __syncthreads();
      if (S::BUFS == 2 && q_lo < q_hi) fetch(q_lo, 0);
      for (int64_t c0 = q_lo; c0 < q_hi; c0 += AP_T) {
        if (S::BUFS == 1) {
          __syncthreads();
          fetch(c0, 0);
        }
        cp_async_commit();
        cp_async_wait<0>();
        __syncthreads();
        const float *sq = sets + set * S::SET, *sdo = sq + S::TILE, *spq = sdo + S::TILE, *slse = spq + S::POS,
                    *sdelta = slse + AP_T;
        if (S::BUFS == 2) {
          set ^= 1;
          if (c0 + AP_T < q_hi) fetch(c0 + AP_T, set);
        }
        float s[4][4] = {}, dp[4][4] = {}, bend[4][4];
        ap_scores(sk, sq, p.channels, ty, tx, s);
        ap_scores(sv, sdo, p.channels, ty, tx, dp);
        ap_logits<true>(s, bend, spk, spq, p.dims, ty, tx, p.scale, p.cap, slope);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float lse = slse[4 * tx + j], delta = sdelta[4 * tx + j];
          const bool none = lse == pos_inf<float>();
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            s[i][j] = none ? 0.f : t5_ex2(s[i][j] - lse);
            dp[i][j] = none ? 0.f : s[i][j] * (dp[i][j] - delta) * bend[i][j];
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4 *>(sw + (4 * ty + i) * AP_LD + 4 * tx) =
              make_float4(s[i][0], s[i][1], s[i][2], s[i][3]);
        __syncwarp();
        ap_accumulate<NC>(sw, sdo, ty, tx, gv);
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 4; ++i)
          *reinterpret_cast<float4 *>(sw + (4 * ty + i) * AP_LD + 4 * tx) =
              make_float4(dp[i][0], dp[i][1], dp[i][2], dp[i][3]);
        __syncwarp();
        ap_accumulate<NC>(sw, sq, ty, tx, gk);
      }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t row = t0 + 4 * ty + i;
      if (row < k_lo || row >= k_hi) continue;
#pragma unroll
      for (int n = 0; n < NC; ++n) {
        const int c = tx + 16 * n;
        if (c < p.channels) {
          dk[row * krow + c] = at_round<T>(gk[i][n] * p.scale);
          dv[row * krow + c] = at_round<T>(gv[i][n]);
        }
      }
    }
  }
  cp_async_wait<0>();  // a block without a tile still has its own rows' copies under way
}

// What the backward pass needs beforehand: D_i = do_i . o_i per (row, head), and for fp16 the largest |do_i|^2 and
// |v_j|^2 of any finite row of an example and key head (norms[b][group][0], [1]; non-negative floats order like their
// bits, and a maximum does not depend on the order).  LP lanes share a row, VL channels at a time; the blocks past the
// first `do_blocks` take the rows of v.  A block has consecutive rows, mostly of a few examples, and collects their
// maxima in shared memory: one at a time they were as many atomics as rows.
constexpr int AP_NORMS = 1024;  // (example, key head) pairs of a block that are collected
template <typename T, int VL>
struct alignas(sizeof(T) * VL) ApVec {
  T v[VL];
};
template <typename T, int VL, int LP, bool NORMS>
__global__ void __launch_bounds__(256, NORMS ? 6 : 1) attention_prepare_kernel(AttnArgs a, float *__restrict__ delta,
                                                                unsigned *__restrict__ norms, int64_t do_rows,
                                                                unsigned do_blocks) {
  using V = ApVec<T, VL>;
  constexpr int SLOTS = 256 / LP;
  __shared__ unsigned s_most[NORMS ? AP_NORMS : 1];
  const b200c_attention_t &p = a.p;
  const int part = threadIdx.x % LP, units = p.channels / VL;
  const bool values = NORMS && blockIdx.x >= do_blocks;
  const unsigned block = values ? blockIdx.x - do_blocks : blockIdx.x;
  const unsigned blocks = values ? gridDim.x - do_blocks : do_blocks;
  const int64_t rows = values ? p.n * p.groups : do_rows;
  const int heads = values ? p.groups : p.heads;
  const V *dout = (const V *)a.dout, *out = (const V *)a.out, *rest = (const V *)a.rest;
  int64_t from = (int64_t)block * SLOTS, to = rows, step = (int64_t)blocks * SLOTS;
  // NORMS: the place of example b, relative to row0
  const int64_t *ptr = values ? p.ptr_k : p.ptr_q;
  const int64_t side = values ? p.n : p.m;
  int64_t row0 = 0;
  int b_first = 0, b = 0, lo = 0, hi = 0;
  if (NORMS) {
    step = SLOTS;
    const int64_t each = ((rows + blocks - 1) / blocks + SLOTS - 1) / SLOTS * SLOTS;
    from = (int64_t)block * each;
    if (from + each < to) to = from + each;
    for (int i = threadIdx.x; i < AP_NORMS; i += 256) s_most[i] = 0u;
    row0 = from / heads;
    if (from < to) b = b_first = at_segment_of_warp(ptr, (int)p.num_segments, row0, threadIdx.x & 31);
    __syncthreads();
  }
  // whole warps take the same number of steps (the sums are shuffles)
  for (int64_t i0 = from; i0 < to; i0 += step) {
    const int64_t i = i0 + threadIdx.x / LP;
    float s = 0.f, sq = 0.f;
    if (i < to) {
      const V *v = dout + i * units;
      if (values) v = reinterpret_cast<const V *>((const T *)p.v + (i / p.groups) * p.v_row + (i % p.groups) * p.v_head);
      for (int u = part; u < units; u += LP) {
        const V g = v[u];
        if (values) {
#pragma unroll
          for (int c = 0; c < VL; ++c) sq = fmaf(at_float(g.v[c]), at_float(g.v[c]), sq);
        } else {
          const V o = out[i * units + u];
          V r{};
          if (rest) r = rest[i * units + u];
#pragma unroll
          for (int c = 0; c < VL; ++c) {
            const float x = at_float(g.v[c]);
            s = fmaf(x, at_float(o.v[c]), s);
            if (rest) s = fmaf(x, at_float(r.v[c]), s);
            if (NORMS) sq = fmaf(x, x, sq);
          }
        }
      }
    }
#pragma unroll
    for (int o = LP / 2; o > 0; o >>= 1) {
      s += __shfl_xor_sync(FULL_MASK, s, o);
      if (NORMS) sq += __shfl_xor_sync(FULL_MASK, sq, o);
    }
    if (part == 0 && i < to) {
      const int64_t row = i / heads;
      const int head = (int)(i - row * heads);
      if (!values) delta[(int64_t)head * p.m + row] = s;
      if (NORMS && sq < pos_inf<float>()) {  // not of NaN either
        const int at = (int)(row - row0), group = values ? head : head / (p.heads / p.groups);
        if (at < lo || at >= hi) {
          // most often the next example's
          int64_t l, h;
          if (hi > 0 && b + 1 < p.num_segments) ++b;
          at_segment(ptr, side, b, l, h);
          if (row < l || row >= h) {
            b = segment_of(ptr, (int)p.num_segments, row);
            at_segment(ptr, side, b, l, h);
          }
          lo = l > row0 ? (int)(l - row0) : 0;
          hi = h > row0 ? (int)(h - row0) : 0;
        }
        if (at >= lo && at < hi) {  // else of no example
          const int64_t place = (int64_t)(b - b_first) * p.groups + group;
          if (place >= 0 && place < AP_NORMS)
            atomicMax(&s_most[place], __float_as_uint(sq));
          else
            atomicMax(norms + 2 * ((int64_t)b * p.groups + group) + (values ? 1 : 0), __float_as_uint(sq));
        }
      }
    }
  }
  if (NORMS) {
    __syncthreads();
    for (int i = threadIdx.x; i < AP_NORMS; i += 256)
      if (s_most[i] != 0u) atomicMax(norms + 2 * ((int64_t)b_first * p.groups + i) + (values ? 1 : 0), s_most[i]);
  }
}

template <typename T, int CP>
static int ap_forward(const AttnArgs &a) {
  constexpr size_t smem = ApSmem<CP, 1>::FLOATS * 4;
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  static unsigned long long configured = 0ull;
  B200C_CUDA(opt_in_shared_memory(attention_plain_forward_kernel<T, CP>, smem, configured));
  const dim3 grid(ap_blocks(a.p.ptr_q, a.p.m, a.p.num_segments), (unsigned)a.p.heads);
  attention_plain_forward_kernel<T, CP><<<grid, AP_THREADS, smem, a.stream>>>(a);
  B200C_LAUNCH_CHECK("attention_plain_forward_kernel");
  return B200C_OK;
}

template <typename T, int CP>
static int ap_backward(const AttnArgs &a) {
  constexpr size_t smem = ApSmem<CP, 2>::FLOATS * 4;
  static_assert(smem <= 227 * 1024, "shared memory of a block");
  static unsigned long long configured_q = 0ull, configured_kv = 0ull;
  if (a.dq && a.p.m > 0) {
    B200C_CUDA(opt_in_shared_memory(attention_plain_dq_kernel<T, CP>, smem, configured_q));
    const dim3 grid(ap_blocks(a.p.ptr_q, a.p.m, a.p.num_segments), (unsigned)a.p.heads);
    attention_plain_dq_kernel<T, CP><<<grid, AP_THREADS, smem, a.stream>>>(a);
    B200C_LAUNCH_CHECK("attention_plain_dq_kernel");
  }
  if (a.dk && a.p.n > 0) {
    B200C_CUDA(opt_in_shared_memory(attention_plain_dkv_kernel<T, CP>, smem, configured_kv));
    const dim3 grid(ap_blocks(a.p.ptr_k, a.p.n, a.p.num_segments), (unsigned)a.p.groups);
    attention_plain_dkv_kernel<T, CP><<<grid, AP_THREADS, smem, a.stream>>>(a);
    B200C_LAUNCH_CHECK("attention_plain_dkv_kernel");
  }
  return B200C_OK;
}

template <typename T>
static int ap_dispatch(const AttnArgs &a, bool forward) {
  if (a.p.channels <= 32) return forward ? ap_forward<T, 32>(a) : ap_backward<T, 32>(a);
  if (a.p.channels <= 48) return forward ? ap_forward<T, 48>(a) : ap_backward<T, 48>(a);
  if (a.p.channels <= 64) return forward ? ap_forward<T, 64>(a) : ap_backward<T, 64>(a);
  return forward ? ap_forward<T, 128>(a) : ap_backward<T, 128>(a);
}

static int ap_any(const AttnArgs &a, bool forward) {
  if (a.p.dtype == B200C_F32) return ap_dispatch<float>(a, forward);
  if (a.p.dtype == B200C_F16) return ap_dispatch<__half>(a, forward);
  return ap_dispatch<__nv_bfloat16>(a, forward);
}

int launch_attention_plain_forward(const AttnArgs &a) { return ap_any(a, true); }
int launch_attention_plain_backward(const AttnArgs &a) { return ap_any(a, false); }

template <typename T, int VL, int LP>
static int ap_prepare_launch(const AttnArgs &a, float *delta, float *norms) {
  const int64_t rows = a.p.m * a.p.heads, values = norms ? a.p.n * a.p.groups : 0;
  constexpr bool NORMS = std::is_same<T, __half>::value;
  const auto blocks = [](int64_t r, int per_sm) {
    const int64_t want = (r + 256 / LP - 1) / (256 / LP), most = 148 * per_sm;
    return (unsigned)(want < most ? want : most);
  };
  // with norms six blocks fit an SM (2048 molecules: D and norms 57 us in blocks of fewer rows, 46 so)
  const unsigned b0 = blocks(rows, NORMS ? 3 : 8), b1 = blocks(values, 3);
  if (norms) B200C_CUDA(cudaMemsetAsync(norms, 0, attention_norms_bytes(a.p), a.stream));
  if (b0 + b1 == 0) return B200C_OK;
  attention_prepare_kernel<T, VL, LP, NORMS><<<b0 + b1, 256, 0, a.stream>>>(a, delta, (unsigned *)norms, rows, b0);
  B200C_LAUNCH_CHECK("attention_prepare_kernel");
  return B200C_OK;
}

template <typename T>
static int ap_delta(const AttnArgs &a, float *delta, float *norms) {
  constexpr int VL = 16 / (int)sizeof(T);
  const b200c_attention_t &p = a.p;
  const bool vec = p.channels % VL == 0 && p.v_row % VL == 0 && p.v_head % VL == 0 &&
                   (((uintptr_t)a.dout | (uintptr_t)a.out | (uintptr_t)a.rest | (uintptr_t)p.v) & 15) == 0;
  if (!vec) return ap_prepare_launch<T, 1, 32>(a, delta, norms);
  if (p.channels <= 4 * VL) return ap_prepare_launch<T, VL, 4>(a, delta, norms);
  if (p.channels <= 8 * VL) return ap_prepare_launch<T, VL, 8>(a, delta, norms);
  return ap_prepare_launch<T, VL, 16>(a, delta, norms);
}

size_t attention_norms_bytes(const b200c_attention_t &p) {
  return p.dtype == B200C_F16 ? (size_t)p.num_segments * p.groups * 8 : 0;
}

int launch_attention_delta(const AttnArgs &a, float *delta, float *norms) {
  if (a.p.dtype == B200C_F32) return ap_delta<float>(a, delta, nullptr);
  if (a.p.dtype == B200C_F16) return ap_delta<__half>(a, delta, norms);
  return ap_delta<__nv_bfloat16>(a, delta, nullptr);
}

}  // namespace b200c
