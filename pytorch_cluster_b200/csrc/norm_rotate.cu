// RMS norm of every head of the queries and keys, and their rotation by the points' coordinates, in one pass.
//   r = 1 / sqrt(mean_c x_c^2 + eps),  u = w x r,  a_p = sum_d pos_d freq_dp,
//   y_p = u_p cos a_p - u_{p+h} sin a_p,  y_{p+h} = u_{p+h} cos a_p + u_p sin a_p   (p < h = channels / 2)
// Backward: g = the rotation of dy by -a, dw = sum g x r over rows and heads, t = g w,
//   dx = r t - x r^3 mean_c(t x).
//
// Memory bounds both directions (2 and 3 bytes-per-value passes); the rotation's angles are shared by all heads of a row, so a
// block forms the sines and cosines of its rows once, in shared memory, and uses them for every head of q and, where
// both have the same positions, of k.  Positions may be far from zero (whole numbers up to millions, in
// either type): the angle is a sum of products in 64 bits, reduced to [-pi, pi] there, and only then rounded to 32.
// LP lanes hold a head's row, 16 bytes of either half each; sums over a row are shuffles.  The gradient of the weights is
// summed in registers over a block's rows, then over the blocks in a fixed order: no atomics.
#include "common.cuh"
#include "launchers.h"

namespace b200c {

constexpr int NR_THREADS = 256;
constexpr int NR_MAX_HALF = 128;
constexpr int NR_PARTS = 148 * 4;  // blocks of the backward pass: each leaves one part of the weights' gradient

template <typename T>
__device__ __forceinline__ float nr_float(T v) { return (float)v; }
template <>
__device__ __forceinline__ float nr_float<__half>(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float nr_float<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T>
__device__ __forceinline__ T nr_round(float v) { return (T)v; }
template <>
__device__ __forceinline__ __half nr_round<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 nr_round<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T, int VL>
struct alignas(sizeof(T) * VL) NrVec {
  T v[VL];
};

template <typename T, int VL>
__device__ __forceinline__ void nr_load(const T *p, float (&f)[VL]) {
  const NrVec<T, VL> r = *reinterpret_cast<const NrVec<T, VL> *>(p);
#pragma unroll
  for (int c = 0; c < VL; ++c) f[c] = nr_float(r.v[c]);
}
template <typename T, int VL>
__device__ __forceinline__ void nr_store(T *p, const float (&f)[VL]) {
  NrVec<T, VL> r;
#pragma unroll
  for (int c = 0; c < VL; ++c) r.v[c] = nr_round<T>(f[c]);
  *reinterpret_cast<NrVec<T, VL> *>(p) = r;
}

template <int LP>
__device__ __forceinline__ float nr_sum(float v) {
#pragma unroll
  for (int o = LP / 2; o > 0; o >>= 1) v += __shfl_xor_sync(FULL_MASK, v, o);
  return v;
}

// sines and cosines of rows [row0, row0 + count)
__device__ __forceinline__ void nr_angles(const b200c_norm_rotate_side_t &s, const NormRotateArgs &a, int64_t row0,
                                          int count, float *cs, float *sn) {
  for (int i = threadIdx.x; i < count * a.half; i += NR_THREADS) {
    const int r = i / a.half, p = i - r * a.half;
    const int64_t at = (row0 + r) * a.dims;
    double angle = 0.0;
    for (int d = 0; d < a.dims; ++d) {
      const double x = a.pos_f64 ? ((const double *)s.pos)[at + d] : (double)((const float *)s.pos)[at + d];
      const double f = a.freq_f64 ? ((const double *)a.freq)[d * a.half + p] : (double)((const float *)a.freq)[d * a.half + p];
      angle = fma(x, f, angle);
    }
    // 2 pi in two parts: exact to about 1e-16 of the turns taken
    const double turns = rint(angle * 0.15915494309189535);
    angle = fma(-turns, 6.283185307179586, angle);
    angle = fma(-turns, 2.4492935982947064e-16, angle);
    sincosf((float)angle, sn + i, cs + i);
  }
}

// IT > 1 (VL = 1, LP = 32) is the form for rows without 16-byte alignment
template <typename T, int VL, int LP, int IT>
__global__ void __launch_bounds__(NR_THREADS) norm_rotate_kernel(NormRotateArgs a, int rows_per_block) {
  extern __shared__ float nr_smem[];
  float *cs = nr_smem, *sn = nr_smem + rows_per_block * a.half;
  constexpr int SLOTS = NR_THREADS / LP;
  const int slot = threadIdx.x / LP, part = threadIdx.x % LP;
  const b200c_norm_rotate_side_t &pos_side = a.joint ? a.side[0] : a.side[blockIdx.y];
  const int64_t row0 = (int64_t)blockIdx.x * rows_per_block;
  if (row0 >= pos_side.rows) return;
  const int count = (int)(pos_side.rows - row0 < rows_per_block ? pos_side.rows - row0 : rows_per_block);
  nr_angles(pos_side, a, row0, count, cs, sn);
  __syncthreads();
  const int s_first = a.joint ? 0 : (int)blockIdx.y, s_last = a.joint ? 1 : (int)blockIdx.y;
  for (int si = s_first; si <= s_last; ++si) {
    const b200c_norm_rotate_side_t &s = a.side[si];
    const int tasks = count * s.heads;
    // whole warps take the same number of steps (the sums are warp-wide shuffles)
    for (int t0 = 0; t0 < tasks; t0 += SLOTS) {
      const bool have = t0 + slot < tasks;
      const int t = have ? t0 + slot : tasks - 1;
      const int r = t / s.heads, head = t - r * s.heads;
      const int64_t row = row0 + r;
      const T *x = (const T *)s.x + row * s.row_stride + head * s.head_stride;
      float lo[IT][VL], hi[IT][VL], sq = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (part + LP * i) * VL;
#pragma unroll
        for (int e = 0; e < VL; ++e) lo[i][e] = hi[i][e] = 0.f;
        if (c < a.half) {
          nr_load<T, VL>(x + c, lo[i]);
          nr_load<T, VL>(x + a.half + c, hi[i]);
        }
#pragma unroll
        for (int e = 0; e < VL; ++e) sq = fmaf(lo[i][e], lo[i][e], fmaf(hi[i][e], hi[i][e], sq));
      }
      sq = nr_sum<LP>(sq);
      const float inv = 1.f / sqrtf(sq / (float)(2 * a.half) + a.eps);
      T *y = (T *)s.y + (row * s.heads + head) * (2 * (int64_t)a.half);
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (part + LP * i) * VL;
        if (have && c < a.half) {
#pragma unroll
          for (int e = 0; e < VL; ++e) {
            const float wl = s.weight ? s.weight[c + e] : 1.f, wh = s.weight ? s.weight[a.half + c + e] : 1.f;
            const float co = cs[r * a.half + c + e], si2 = sn[r * a.half + c + e];
            const float u = lo[i][e] * inv * wl, w = hi[i][e] * inv * wh;
            lo[i][e] = u * co - w * si2;
            hi[i][e] = w * co + u * si2;
          }
          nr_store<T, VL>(y + c, lo[i]);
          nr_store<T, VL>(y + a.half + c, hi[i]);
        }
      }
    }
  }
}

template <typename T, int VL, int LP, int IT>
__global__ void __launch_bounds__(NR_THREADS) norm_rotate_backward_kernel(NormRotateArgs a, int rows_per_block,
                                                                          float *__restrict__ parts) {
  extern __shared__ float nr_smem[];
  float *cs = nr_smem, *sn = nr_smem + rows_per_block * a.half;
  __shared__ float s_dw[NR_THREADS / 32][2 * NR_MAX_HALF];
  constexpr int SLOTS = NR_THREADS / LP;
  const int slot = threadIdx.x / LP, part = threadIdx.x % LP, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int s_first = a.joint ? 0 : (int)blockIdx.y, s_last = a.joint ? 1 : (int)blockIdx.y;
  float dwl[2][IT][VL] = {}, dwh[2][IT][VL] = {};
  const b200c_norm_rotate_side_t &pos_side = a.side[s_first];
  for (int64_t row0 = (int64_t)blockIdx.x * rows_per_block; row0 < pos_side.rows;
       row0 += (int64_t)gridDim.x * rows_per_block) {
    const int count = (int)(pos_side.rows - row0 < rows_per_block ? pos_side.rows - row0 : rows_per_block);
    __syncthreads();
    nr_angles(pos_side, a, row0, count, cs, sn);
    __syncthreads();
#pragma unroll
    for (int si = 0; si < 2; ++si) {
      if (si < s_first || si > s_last) continue;
      const b200c_norm_rotate_side_t &s = a.side[si];
      const int tasks = count * s.heads;
      for (int t0 = 0; t0 < tasks; t0 += SLOTS) {
        const bool have = t0 + slot < tasks;
        const int t = have ? t0 + slot : tasks - 1;
        const int r = t / s.heads, head = t - r * s.heads;
        const int64_t row = row0 + r;
        const T *x = (const T *)s.x + row * s.row_stride + head * s.head_stride;
        const T *dy = (const T *)s.dy + (row * s.heads + head) * (2 * (int64_t)a.half);
        float xl[IT][VL], xh[IT][VL], gl[IT][VL], gh[IT][VL], sq = 0.f, tx = 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int c = (part + LP * i) * VL;
#pragma unroll
          for (int e = 0; e < VL; ++e) xl[i][e] = xh[i][e] = gl[i][e] = gh[i][e] = 0.f;
          if (c < a.half) {
            nr_load<T, VL>(x + c, xl[i]);
            nr_load<T, VL>(x + a.half + c, xh[i]);
            nr_load<T, VL>(dy + c, gl[i]);
            nr_load<T, VL>(dy + a.half + c, gh[i]);
#pragma unroll
            for (int e = 0; e < VL; ++e) {
              const float co = cs[r * a.half + c + e], si2 = sn[r * a.half + c + e];
              const float l = gl[i][e] * co + gh[i][e] * si2, h = gh[i][e] * co - gl[i][e] * si2;
              gl[i][e] = l;
              gh[i][e] = h;
              const float wl = s.weight ? s.weight[c + e] : 1.f, wh = s.weight ? s.weight[a.half + c + e] : 1.f;
              sq = fmaf(xl[i][e], xl[i][e], fmaf(xh[i][e], xh[i][e], sq));
              tx = fmaf(l * wl, xl[i][e], fmaf(h * wh, xh[i][e], tx));
            }
          }
        }
        sq = nr_sum<LP>(sq);
        tx = nr_sum<LP>(tx);
        const float mean = 1.f / (float)(2 * a.half);
        const float inv = 1.f / sqrtf(sq * mean + a.eps);
        const float back = inv * inv * inv * (tx * mean);
        T *dx = (T *)s.dx + (row * s.heads + head) * (2 * (int64_t)a.half);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int c = (part + LP * i) * VL;
          if (have && c < a.half) {
#pragma unroll
            for (int e = 0; e < VL; ++e) {
              const float wl = s.weight ? s.weight[c + e] : 1.f, wh = s.weight ? s.weight[a.half + c + e] : 1.f;
              dwl[si][i][e] = fmaf(gl[i][e], xl[i][e] * inv, dwl[si][i][e]);
              dwh[si][i][e] = fmaf(gh[i][e], xh[i][e] * inv, dwh[si][i][e]);
              gl[i][e] = gl[i][e] * wl * inv - xl[i][e] * back;
              gh[i][e] = gh[i][e] * wh * inv - xh[i][e] * back;
            }
            nr_store<T, VL>(dx + c, gl[i]);
            nr_store<T, VL>(dx + a.half + c, gh[i]);
          }
        }
      }
    }
  }
  // this block's part of the weights' gradients: lane groups of a warp, then warps in order
#pragma unroll
  for (int si = 0; si < 2; ++si) {
    if (si < s_first || si > s_last || parts == nullptr) continue;
#pragma unroll
    for (int i = 0; i < IT; ++i)
#pragma unroll
      for (int e = 0; e < VL; ++e) {
        float l = dwl[si][i][e], h = dwh[si][i][e];
#pragma unroll
        for (int o = LP; o < 32; o <<= 1) {
          l += __shfl_xor_sync(FULL_MASK, l, o);
          h += __shfl_xor_sync(FULL_MASK, h, o);
        }
        const int c = (part + LP * i) * VL + e;
        if (lane < LP && c < a.half) {
          s_dw[warp][c] = l;
          s_dw[warp][a.half + c] = h;
        }
      }
    __syncthreads();
    for (int c = threadIdx.x; c < 2 * a.half; c += NR_THREADS) {
      float v = 0.f;
#pragma unroll
      for (int w = 0; w < NR_THREADS / 32; ++w) v += s_dw[w][c];
      parts[((int64_t)si * gridDim.x + blockIdx.x) * (2 * a.half) + c] = v;
    }
    __syncthreads();
  }
}

// one block per (side, 32 channels): the parts in a fixed order
__global__ void __launch_bounds__(NR_THREADS) norm_rotate_weights_kernel(const float *__restrict__ parts, int blocks,
                                                                         int channels, float *__restrict__ dw0,
                                                                         float *__restrict__ dw1) {
  __shared__ float share[NR_THREADS / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float *dw = blockIdx.y == 0 ? dw0 : dw1;
  if (dw == nullptr) return;
  float v = 0.f;
  if (c < channels) {
#pragma unroll 8
    for (int b = warp; b < blocks; b += NR_THREADS / 32) v += parts[((int64_t)blockIdx.y * blocks + b) * channels + c];
  }
  share[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < channels) {
    v = 0.f;
#pragma unroll
    for (int w = 0; w < NR_THREADS / 32; ++w) v += share[w][lane];
    dw[c] = v;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------
static int nr_rows_per_block(const NormRotateArgs &a, int lanes) {
  // enough rows that every lane group has two heads to work on, at most 32 (shared memory)
  const int slots = NR_THREADS / lanes, heads = a.joint ? a.side[0].heads + a.side[1].heads : a.side[0].heads;
  const int rows = (2 * slots + heads - 1) / heads;
  return rows < 1 ? 1 : rows > 32 ? 32 : rows;
}

template <typename T, int VL, int LP, int IT>
static int nr_launch(const NormRotateArgs &a, bool forward, float *parts) {
  int rpb = nr_rows_per_block(a, LP);
  const int64_t most = a.side[0].rows > a.side[1].rows ? a.side[0].rows : a.side[1].rows;
  while (rpb > 1 && (most + rpb - 1) / rpb < 296) rpb /= 2;  // small calls: more blocks rather than fuller ones
  const size_t smem = (size_t)rpb * a.half * 8;
  const int64_t chunks = (most + rpb - 1) / rpb;
  const unsigned sides = a.joint ? 1u : 2u;
  if (forward) {
    norm_rotate_kernel<T, VL, LP, IT><<<dim3((unsigned)chunks, sides), NR_THREADS, smem, a.stream>>>(a, rpb);
    B200C_LAUNCH_CHECK("norm_rotate_kernel");
    return B200C_OK;
  }
  const unsigned blocks = chunks < NR_PARTS ? (unsigned)chunks : (unsigned)NR_PARTS;
  const bool weights = a.dweight[0] || a.dweight[1];
  norm_rotate_backward_kernel<T, VL, LP, IT><<<dim3(blocks, sides), NR_THREADS, smem, a.stream>>>(
      a, rpb, weights ? parts : nullptr);
  B200C_LAUNCH_CHECK("norm_rotate_backward_kernel");
  if (weights) {
    norm_rotate_weights_kernel<<<dim3((unsigned)((2 * a.half + 31) / 32), 2u), NR_THREADS, 0, a.stream>>>(
        parts, (int)blocks, 2 * a.half, a.dweight[0], a.dweight[1]);
    B200C_LAUNCH_CHECK("norm_rotate_weights_kernel");
  }
  return B200C_OK;
}

template <typename T>
static int nr_type(const NormRotateArgs &a, bool forward, float *parts) {
  constexpr int VL = 16 / (int)sizeof(T);
  bool vec = a.half % VL == 0;
  for (const auto &s : a.side)
    vec = vec && s.row_stride % VL == 0 && s.head_stride % VL == 0 &&
          (((uintptr_t)s.x | (uintptr_t)s.y | (uintptr_t)s.dy | (uintptr_t)s.dx) & 15) == 0;
  if (!vec) return nr_launch<T, 1, 32, NR_MAX_HALF / 32>(a, forward, parts);
  const int lanes = a.half / VL;
  if (lanes <= 2) return nr_launch<T, VL, 2, 1>(a, forward, parts);
  if (lanes <= 4) return nr_launch<T, VL, 4, 1>(a, forward, parts);
  if (lanes <= 8) return nr_launch<T, VL, 8, 1>(a, forward, parts);
  if (lanes <= 16) return nr_launch<T, VL, 16, 1>(a, forward, parts);
  return nr_launch<T, VL, 32, 1>(a, forward, parts);
}

size_t norm_rotate_workspace_bytes(int64_t channels) { return (size_t)2 * NR_PARTS * channels * 4; }

int launch_norm_rotate(const NormRotateArgs &a, bool forward, float *parts) {
  if (a.dtype == B200C_F32) return nr_type<float>(a, forward, parts);
  if (a.dtype == B200C_F16) return nr_type<__half>(a, forward, parts);
  return nr_type<__nv_bfloat16>(a, forward, parts);
}

}  // namespace b200c
