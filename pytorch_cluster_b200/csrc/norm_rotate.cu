// RMS norm of every head of the queries and keys, and their rotation by the points' coordinates, in one pass.
//   r = 1 / sqrt(mean_c x_c^2 + eps),  u = w x r,  a_p = sum_d pos_d freq_dp,
//   y_p = u_p cos a_p - u_{p+h} sin a_p,  y_{p+h} = u_{p+h} cos a_p + u_p sin a_p   (p < h = channels / 2)
// Backward: g = the rotation of dy by -a, dw = sum g x r over rows and heads, t = g w,
//   dx = r t - x r^3 mean_c(t x).
//
// Memory bounds both directions (2 and 3 bytes-per-value passes); the rotation's angles are shared by all heads of a
// row, so a block forms the sines and cosines of its rows once, in shared memory, and uses them for every head of q
// and, where both have the same positions, of k.  Positions may be far from zero (whole numbers up to millions, in
// either type): the angle is a sum of products in 64 bits, reduced to [-pi, pi] there, and only then rounded to 32. LP
// lanes hold a head's row, 16 bytes of either half each; sums over a row are shuffles.  Next to memory it is
// instructions that cost: offsets are added up from step to step, the root is the hardware's reciprocal root.  The
// gradient of the weights is summed in registers over a block's rows, then over the blocks in a fixed order: no
// atomics.
#include "common.cuh"
#include "launchers.h"

namespace b200c {

constexpr int NR_THREADS = 256;
constexpr int NR_JOIN_THREADS = 1024;
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
// VL floats of shared memory
template <int VL>
__device__ __forceinline__ void nr_floats(const float *p, float (&f)[VL]) {
  if constexpr (VL % 4 == 0) {
#pragma unroll
    for (int c = 0; c < VL; c += 4) {
      const float4 v = *reinterpret_cast<const float4 *>(p + c);
      f[c] = v.x, f[c + 1] = v.y, f[c + 2] = v.z, f[c + 3] = v.w;
    }
  } else {
#pragma unroll
    for (int c = 0; c < VL; ++c) f[c] = p[c];
  }
}
// the weights of both sides, [2][channels], once per block
__device__ __forceinline__ void nr_weights(const NormRotateArgs &a, float *sw) {
  for (int i = threadIdx.x; i < 4 * a.half; i += NR_THREADS) {
    const b200c_norm_rotate_side_t &s = a.side[i >= 2 * a.half];
    sw[i] = s.weight ? s.weight[i >= 2 * a.half ? i - 2 * a.half : i] : 1.f;
  }
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

// The frequencies in 64 bits, [dims][half], once per block.
__device__ __forceinline__ void nr_frequencies(const NormRotateArgs &a, double *fr) {
  for (int i = threadIdx.x; i < a.dims * a.half; i += NR_THREADS)
    fr[i] = a.freq_f64 ? ((const double *)a.freq)[i] : (double)((const float *)a.freq)[i];
}
// Sines and cosines of rows [row0, row0 + count).  The reduced angle is at most pi, where the hardware's sine and
// cosine are off by 2^-21 at most: a thousandth of the 16-bit types' steps, but several of fp32's, which calls the
// exact ones and brings in what rounding took from the angle (error of a rotation of 1024 rows 1.7e-7 -> 0.7e-7).
template <typename T>
__device__ __forceinline__ void nr_angles(const b200c_norm_rotate_side_t &s, const NormRotateArgs &a, int64_t row0,
                                          int count, const double *fr, float *cs, float *sn) {
  for (int i = threadIdx.x; i < count * a.half; i += NR_THREADS) {
    const int r = i / a.half, p = i - r * a.half;
    const int64_t at = (row0 + r) * a.dims;
    double angle = 0.0;
    for (int d = 0; d < a.dims; ++d) {
      const double x = a.pos_f64 ? ((const double *)s.pos)[at + d] : (double)((const float *)s.pos)[at + d];
      angle = fma(x, fr[d * a.half + p], angle);
    }
    // 2 pi in two parts: exact to about 1e-16 of the turns taken
    const double turns = rint(angle * 0.15915494309189535);
    angle = fma(-turns, 6.283185307179586, angle);
    angle = fma(-turns, 2.4492935982947064e-16, angle);
    const float f = (float)angle;
    if constexpr (sizeof(T) == 4) {
      const float rest = (float)(angle - (double)f);
      float si, co;
      sincosf(f, &si, &co);
      cs[i] = fmaf(-si, rest, co);
      sn[i] = fmaf(co, rest, si);
    } else {
      cs[i] = __cosf(f);
      sn[i] = __sinf(f);
    }
  }
}

// Where a lane group's (row, head) lies and how far its next one is: offsets are added up, not multiplied out.
template <typename T>
struct NrTask {
  int64_t x0, y0, x_step, x_wrap;  // elements
  int y_step, angle, angle_step, half, head, head_step, heads;
  __device__ __forceinline__ NrTask(const b200c_norm_rotate_side_t &s, int half_, int64_t row0, int slot, int slots)
      : half(half_), heads(s.heads) {
    const int r = slot / heads, r_step = slots / heads;
    head = slot - r * heads;
    head_step = slots - r_step * heads;
    x0 = (row0 + r) * s.row_stride + head * s.head_stride;
    y0 = ((row0 + r) * heads + head) * (2 * (int64_t)half);
    x_step = r_step * s.row_stride + head_step * s.head_stride;
    x_wrap = s.row_stride - heads * s.head_stride;
    y_step = slots * 2 * half;
    angle = r * half;
    angle_step = r_step * half;
  }
  __device__ __forceinline__ int64_t move() {
    int64_t by = x_step;
    head += head_step;
    angle += angle_step;
    if (head >= heads) {
      head -= heads;
      angle += half;
      by += x_wrap;
    }
    return by;
  }
};

// IT > 1 (VL = 1, LP = 32) is the form for rows without 16-byte alignment
template <typename T, int VL, int LP, int IT>
__global__ void __launch_bounds__(NR_THREADS, 4) norm_rotate_kernel(NormRotateArgs a, int rows_per_block) {
  extern __shared__ __align__(16) double nr_smem[];
  double *fr = nr_smem;
  float *sw = reinterpret_cast<float *>(fr + a.dims * a.half), *cs = sw + 4 * a.half, *sn = cs + rows_per_block * a.half;
  constexpr int SLOTS = NR_THREADS / LP;
  const int slot = threadIdx.x / LP, part = threadIdx.x % LP;
  const float mean = 1.f / (float)(2 * a.half);
  const b200c_norm_rotate_side_t &pos_side = a.joint ? a.side[0] : a.side[blockIdx.y];
  const int64_t row0 = (int64_t)blockIdx.x * rows_per_block;
  if (row0 >= pos_side.rows) return;
  const int count = (int)(pos_side.rows - row0 < rows_per_block ? pos_side.rows - row0 : rows_per_block);
  nr_frequencies(a, fr);
  nr_weights(a, sw);
  __syncthreads();
  nr_angles<T>(pos_side, a, row0, count, fr, cs, sn);
  __syncthreads();
  const int s_first = a.joint ? 0 : (int)blockIdx.y, s_last = a.joint ? 1 : (int)blockIdx.y;
  for (int si = s_first; si <= s_last; ++si) {
    const b200c_norm_rotate_side_t &s = a.side[si];
    const float *weight = sw + si * 2 * a.half;
    NrTask<T> at(s, a.half, row0, slot, SLOTS);
    const T *x = (const T *)s.x + at.x0;
    T *y = (T *)s.y + at.y0;
    // whole warps take the same number of steps (the sums are warp-wide shuffles)
    for (int left = count * s.heads - slot, n = (count * s.heads + SLOTS - 1) / SLOTS; n > 0; --n, left -= SLOTS) {
      const bool have = left > 0;
      float lo[IT][VL], hi[IT][VL], sq = 0.f;
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (part + LP * i) * VL;
#pragma unroll
        for (int e = 0; e < VL; ++e) lo[i][e] = hi[i][e] = 0.f;
        if (have && c < a.half) {
          nr_load<T, VL>(x + c, lo[i]);
          nr_load<T, VL>(x + a.half + c, hi[i]);
        }
#pragma unroll
        for (int e = 0; e < VL; ++e) sq = fmaf(lo[i][e], lo[i][e], fmaf(hi[i][e], hi[i][e], sq));
      }
      sq = nr_sum<LP>(sq);
      const float inv = rsqrtf(fmaf(sq, mean, a.eps));
#pragma unroll
      for (int i = 0; i < IT; ++i) {
        const int c = (part + LP * i) * VL;
        if (have && c < a.half) {
          float co[VL], si2[VL], wl[VL], wh[VL];
          nr_floats<VL>(cs + at.angle + c, co);
          nr_floats<VL>(sn + at.angle + c, si2);
          nr_floats<VL>(weight + c, wl);
          nr_floats<VL>(weight + a.half + c, wh);
#pragma unroll
          for (int e = 0; e < VL; ++e) {
            const float u = lo[i][e] * inv * wl[e], w = hi[i][e] * inv * wh[e];
            lo[i][e] = u * co[e] - w * si2[e];
            hi[i][e] = w * co[e] + u * si2[e];
          }
          nr_store<T, VL>(y + c, lo[i]);
          nr_store<T, VL>(y + a.half + c, hi[i]);
        }
      }
      x += at.move();
      y += at.y_step;
    }
  }
}

template <typename T, int VL, int LP, int IT>
__global__ void __launch_bounds__(NR_THREADS, 2) norm_rotate_backward_kernel(NormRotateArgs a, int rows_per_block,
                                                                          float *__restrict__ parts) {
  extern __shared__ __align__(16) double nr_smem[];
  double *fr = nr_smem;
  float *sw = reinterpret_cast<float *>(fr + a.dims * a.half), *cs = sw + 4 * a.half, *sn = cs + rows_per_block * a.half;
  __shared__ float s_dw[NR_THREADS / 32][2 * NR_MAX_HALF];
  constexpr int SLOTS = NR_THREADS / LP;
  const int slot = threadIdx.x / LP, part = threadIdx.x % LP, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const float mean = 1.f / (float)(2 * a.half);
  const int s_first = a.joint ? 0 : (int)blockIdx.y, s_last = a.joint ? 1 : (int)blockIdx.y;
  float dwl[2][IT][VL] = {}, dwh[2][IT][VL] = {};
  const b200c_norm_rotate_side_t &pos_side = a.side[s_first];
  nr_frequencies(a, fr);
  nr_weights(a, sw);
  for (int64_t row0 = (int64_t)blockIdx.x * rows_per_block; row0 < pos_side.rows;
       row0 += (int64_t)gridDim.x * rows_per_block) {
    const int count = (int)(pos_side.rows - row0 < rows_per_block ? pos_side.rows - row0 : rows_per_block);
    __syncthreads();
    nr_angles<T>(pos_side, a, row0, count, fr, cs, sn);
    __syncthreads();
#pragma unroll
    for (int si = 0; si < 2; ++si) {
      if (si < s_first || si > s_last) continue;
      const b200c_norm_rotate_side_t &s = a.side[si];
      const float *weight = sw + si * 2 * a.half;
      NrTask<T> at(s, a.half, row0, slot, SLOTS);
      const T *x = (const T *)s.x + at.x0, *dy = (const T *)s.dy + at.y0;
      T *dx = (T *)s.dx + at.y0;
      for (int left = count * s.heads - slot, n = (count * s.heads + SLOTS - 1) / SLOTS; n > 0; --n, left -= SLOTS) {
        const bool have = left > 0;
        float xl[IT][VL], xh[IT][VL], gl[IT][VL], gh[IT][VL], sq = 0.f, tx = 0.f;
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int c = (part + LP * i) * VL;
#pragma unroll
          for (int e = 0; e < VL; ++e) xl[i][e] = xh[i][e] = gl[i][e] = gh[i][e] = 0.f;
          if (have && c < a.half) {
            nr_load<T, VL>(x + c, xl[i]);
            nr_load<T, VL>(x + a.half + c, xh[i]);
            nr_load<T, VL>(dy + c, gl[i]);
            nr_load<T, VL>(dy + a.half + c, gh[i]);
            float co[VL], si2[VL], wl[VL], wh[VL];
            nr_floats<VL>(cs + at.angle + c, co);
            nr_floats<VL>(sn + at.angle + c, si2);
            nr_floats<VL>(weight + c, wl);
            nr_floats<VL>(weight + a.half + c, wh);
#pragma unroll
            for (int e = 0; e < VL; ++e) {
              const float l = gl[i][e] * co[e] + gh[i][e] * si2[e], h = gh[i][e] * co[e] - gl[i][e] * si2[e];
              gl[i][e] = l;
              gh[i][e] = h;
              sq = fmaf(xl[i][e], xl[i][e], fmaf(xh[i][e], xh[i][e], sq));
              tx = fmaf(l * wl[e], xl[i][e], fmaf(h * wh[e], xh[i][e], tx));
            }
          }
        }
        sq = nr_sum<LP>(sq);
        tx = nr_sum<LP>(tx);
        const float inv = rsqrtf(fmaf(sq, mean, a.eps));
        // in an order in which rows of 1e16 and of 1e-14 pass (the cube of inv would leave the range of fp32)
        const float back = inv * inv * (inv * tx * mean);
#pragma unroll
        for (int i = 0; i < IT; ++i) {
          const int c = (part + LP * i) * VL;
          if (have && c < a.half) {
            float wl[VL], wh[VL];
            nr_floats<VL>(weight + c, wl);
            nr_floats<VL>(weight + a.half + c, wh);
#pragma unroll
            for (int e = 0; e < VL; ++e) {
              // g / norm: its product with x is the weight's gradient, with the weight the row's
              const float l = gl[i][e] * inv, h = gh[i][e] * inv;
              dwl[si][i][e] = fmaf(l, xl[i][e], dwl[si][i][e]);
              dwh[si][i][e] = fmaf(h, xh[i][e], dwh[si][i][e]);
              gl[i][e] = fmaf(l, wl[e], -xl[i][e] * back);
              gh[i][e] = fmaf(h, wh[e], -xh[i][e] * back);
            }
            nr_store<T, VL>(dx + c, gl[i]);
            nr_store<T, VL>(dx + a.half + c, gh[i]);
          }
        }
        x += at.move();
        dy += at.y_step;
        dx += at.y_step;
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
__global__ void __launch_bounds__(NR_JOIN_THREADS) norm_rotate_weights_kernel(const float *__restrict__ parts, int blocks,
                                                                         int channels, float *__restrict__ dw0,
                                                                         float *__restrict__ dw1) {
  __shared__ float share[NR_JOIN_THREADS / 32][32];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int c = blockIdx.x * 32 + lane;
  float *dw = blockIdx.y == 0 ? dw0 : dw1;
  if (dw == nullptr) return;
  float v = 0.f;
  if (c < channels) {
#pragma unroll 4
    for (int b = warp; b < blocks; b += NR_JOIN_THREADS / 32) v += parts[((int64_t)blockIdx.y * blocks + b) * channels + c];
  }
  share[warp][lane] = v;
  __syncthreads();
  if (warp == 0 && c < channels) {
    v = 0.f;
#pragma unroll
    for (int w = 0; w < NR_JOIN_THREADS / 32; ++w) v += share[w][lane];
    dw[c] = v;
  }
}

// ---- host ----------------------------------------------------------------------------------------------------
static int nr_rows_per_block(const NormRotateArgs &a, int lanes) {
  // enough rows that every lane group has eight heads to work on, so that the angles, which all wait for, are a small
  // part of the time; at most 32 (shared memory)
  const int slots = NR_THREADS / lanes, heads = a.joint ? a.side[0].heads + a.side[1].heads : a.side[0].heads;
  const int rows = (8 * slots + heads - 1) / heads;
  return rows < 1 ? 1 : rows > 32 ? 32 : rows;
}

template <typename T, int VL, int LP, int IT>
static int nr_launch(const NormRotateArgs &a, bool forward, float *parts) {
  int rpb = nr_rows_per_block(a, LP);
  const int64_t most = a.side[0].rows > a.side[1].rows ? a.side[0].rows : a.side[1].rows;
  while (rpb > 1 && (most + rpb - 1) / rpb < 296) rpb /= 2;  // small calls: more blocks rather than fuller ones
  // with the 8 KB of the weights' sums, below the 48 KB that a block has without asking
  while (rpb > 1 && (size_t)(rpb + a.dims + 2) * a.half * 8 > 40 * 1024) --rpb;
  const size_t smem = (size_t)(rpb + a.dims + 2) * a.half * 8;  // sines and cosines, frequencies, weights
  const int64_t chunks = (most + rpb - 1) / rpb;
  const unsigned sides = a.joint ? 1u : 2u;
  static_assert(NR_MAX_HALF <= 4 * 32, "a row's half fits the lanes");
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
    norm_rotate_weights_kernel<<<dim3((unsigned)((2 * a.half + 31) / 32), 2u), NR_JOIN_THREADS, 0, a.stream>>>(
        parts, (int)blocks, 2 * a.half, a.dweight[0], a.dweight[1]);
    B200C_LAUNCH_CHECK("norm_rotate_weights_kernel");
  }
  return B200C_OK;
}

template <typename T, int VL>
static int nr_lanes(const NormRotateArgs &a, bool forward, float *parts) {
  bool vec = a.half % VL == 0;
  for (const auto &s : a.side)
    vec = vec && s.row_stride % VL == 0 && s.head_stride % VL == 0 &&
          (((uintptr_t)s.x | (uintptr_t)s.y | (uintptr_t)s.dy | (uintptr_t)s.dx) & (VL * sizeof(T) - 1)) == 0;
  if (!vec) return nr_launch<T, 1, 32, NR_MAX_HALF / 32>(a, forward, parts);
  const int lanes = a.half / VL;
  if (lanes <= 2) return nr_launch<T, VL, 2, 1>(a, forward, parts);
  if (lanes <= 4) return nr_launch<T, VL, 4, 1>(a, forward, parts);
  if (lanes <= 8) return nr_launch<T, VL, 8, 1>(a, forward, parts);
  if (lanes <= 16) return nr_launch<T, VL, 16, 1>(a, forward, parts);
  return nr_launch<T, VL, 32, 1>(a, forward, parts);
}
template <typename T>
static int nr_type(const NormRotateArgs &a, bool forward, float *parts) {
  return nr_lanes<T, 16 / (int)sizeof(T)>(a, forward, parts);
}

size_t norm_rotate_workspace_bytes(int64_t channels) { return (size_t)2 * NR_PARTS * channels * 4; }

int launch_norm_rotate(const NormRotateArgs &a, bool forward, float *parts) {
  if (a.dtype == B200C_F32) return nr_type<float>(a, forward, parts);
  if (a.dtype == B200C_F16) return nr_type<__half>(a, forward, parts);
  return nr_type<__nv_bfloat16>(a, forward, parts);
}

}  // namespace b200c
