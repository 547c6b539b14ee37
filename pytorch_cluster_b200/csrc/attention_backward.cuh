// Backward attention on the tensor cores (see attention_tensor.cuh): KV = false sums dq of 128 queries of a head
// over the keys, KV = true sums dk and dv of 128 keys of a group over the queries of all its heads.
//
// Forming the scores once per direction costs two products more than one kernel for both would, which the tensor
// cores have to spare here (exponentials and roots bound these kernels); in return no sum is shared
// between blocks, so there are no atomics.  The statistics of the softmax are known, so a row's columns need no
// reduction: two groups of four warps take 32 columns of a step each.
// P and dS enter the second products in the 16-bit type.  In fp16, whose range is small, P is kept times 2^12 and dS times a
// power of two that brings the largest value that |do| and |v| allow to 2^14; both are taken out of the fp32 sums.
#pragma once

#include "attention_tensor.cuh"

namespace b200c {

template <int CP>
struct AtBackward {
  static constexpr int EL_WARPS = 8;
  static constexpr int THREADS = 32 * (EL_WARPS + 2);
  static constexpr int EL_THREADS = 32 * EL_WARPS;
  static constexpr int NB = CP == 64 ? 1 : 2;      // score accumulators
  static constexpr int BLOCKS = CP == 64 ? 2 : 1;  // resident blocks per SM: tensor memory and shared memory
  static constexpr int STAGES = CP == 64 ? 3 : 4;
  static constexpr int ROW_BYTES = AT_ROWS * CP * 2, TILE_BYTES = AT_COLS * CP * 2;
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int SIDE_FLOATS = (AT_MAX_DIMS + 2) * AT_COLS;  // coordinates, lse, D of a step's columns
  static constexpr int SMEM = 2 * ROW_BYTES + STAGES * (STAGE_BYTES + SIDE_FLOATS * 4) + 1024;
  static constexpr int TMEM = CP == 64 ? 256 : 512;
};

struct AtBackwardMaps {
  CUtensorMap row0, row1, col0, col1;  // q, do, k, v or k, v, q, do
};

// the power of two that dS is kept times (see above); norms: the largest |do|^2 and |v|^2 of a row
template <typename T>
__device__ __forceinline__ float at_sigma(const float *norms) {
  if constexpr (AtType<T>::BF16) {
    return 1.f;
  } else {
    const float most = 2.f * sqrtf(norms[0]) * sqrtf(norms[1]);
    if (!(most > 1e-30f && most < 1e30f)) return 1.f;
    return exp2f(14.f - ceilf(log2f(most)));
  }
}

template <typename T, int CP, int DIM, bool CAP, bool KV>
__global__ void __launch_bounds__(AtBackward<CP>::THREADS, AtBackward<CP>::BLOCKS)
attention_backward_kernel(const __grid_constant__ AtBackwardMaps maps, const __grid_constant__ AttnArgs a,
                          const float *__restrict__ norms) {
  using F = AtBackward<CP>;
  using A = AtType<T>;
  constexpr int ATOMS = CP / 64;
  extern __shared__ unsigned char at_raw[];
  unsigned char *smem = at_raw + ((1024u - (t5_smem(at_raw) & 1023u)) & 1023u);
  unsigned char *rows0 = smem, *rows1 = smem + F::ROW_BYTES, *stages = smem + 2 * F::ROW_BYTES;
  float *side = reinterpret_cast<float *>(stages + F::STAGES * F::STAGE_BYTES);
  __shared__ __align__(8) uint64_t r_full, full[F::STAGES], empty[F::STAGES], s_full[F::NB], w_ready[F::NB], done,
      drained;
  __shared__ uint32_t tmem_s;
  __shared__ int failed_s, bad_s;
  volatile int *failed = &failed_s;

  const b200c_attention_t &p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int per_group = p.heads / p.groups;
  const int head0 = KV ? (int)blockIdx.y * per_group : (int)blockIdx.y;
  const int group = KV ? (int)blockIdx.y : head0 / per_group;
  const int heads = KV ? per_group : 1;  // heads whose columns are walked
  AtTile tile;
  if (KV)
    tile.init((int64_t)blockIdx.x * AT_ROWS, p.ptr_k, p.ptr_q, p.n, p.m, p.num_segments);
  else
    tile.init((int64_t)blockIdx.x * AT_ROWS, p.ptr_q, p.ptr_k, p.m, p.n, p.num_segments);

  if (tid == 0) {
    t5_mbar_init(&r_full, 1);
    for (int i = 0; i < F::STAGES; ++i) {
      t5_mbar_init(&full[i], 1);
      t5_mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < F::NB; ++i) {
      t5_mbar_init(&s_full[i], 1);
      t5_mbar_init(&w_ready[i], F::EL_THREADS);
    }
    t5_mbar_init(&done, 1);
    t5_mbar_init(&drained, 1);
    failed_s = 0;
    bad_s = 0;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == F::EL_WARPS) t5_alloc(&tmem_s, F::TMEM);
  t5_fence_before();
  __syncthreads();
  t5_fence_after();
  const uint32_t tmem = tmem_s;
  const uint32_t t_acc = tmem + F::NB * 2 * AT_COLS;  // dq, or dv and dk side by side

  // element threads: a row and half of a step's columns each
  const bool element = warp < F::EL_WARPS;
  const int half = warp >> 2;
  const int64_t row = tile.t0 + (tid & (AT_ROWS - 1));
  int64_t row_lo = 0, row_hi = 0;
  int row_segment = -1;
  float pos[DIM == 0 ? 1 : DIM], lse = 0.f, delta = 0.f;
  if (element && row < tile.t1) {
    row_segment = segment_of(tile.ptr_r, tile.segments, row);
    int64_t lo, hi;
    at_segment(tile.ptr_r, tile.rows, row_segment, lo, hi);
    if (row >= lo && row < hi) at_segment(tile.ptr_c, tile.cols, row_segment, row_lo, row_hi);
    if (!KV) {
      lse = a.lse[(int64_t)head0 * p.m + row] - A::SHIFT;
      delta = a.delta[(int64_t)head0 * p.m + row];
    }
  }
  if constexpr (DIM > 0) {
    const float *src = KV ? p.pos_k : p.pos_q;
#pragma unroll
    for (int d = 0; d < DIM; ++d) pos[d] = element && row < tile.t1 && d < p.dims ? src[row * p.dims + d] : 0.f;
  }
  const float pre = CAP ? 2.f * AT_LOG2E * p.scale / p.cap : p.scale * AT_LOG2E, post = p.cap * AT_LOG2E;
  const float sigma = at_sigma<T>(norms);
  const float sig = A::BF16 ? 1.f : sigma * (1.f / 4096.f);  // P carries 2^SHIFT already

  if (warp == F::EL_WARPS && lane == 0) {
    t5_mbar_expect(&r_full, 2 * F::ROW_BYTES);
    for (int at = 0; at < ATOMS; ++at) {
      t5_tma_3d(rows0 + at * (AT_ROWS * 128), &maps.row0, at * 64, KV ? group : head0, (int)tile.t0, &r_full);
      t5_tma_3d(rows1 + at * (AT_ROWS * 128), &maps.row1, at * 64, KV ? group : head0, (int)tile.t0, &r_full);
    }
    t5_mbar_arrive(&r_full);
  }

  bool by_example = false;
  int64_t next_row = tile.t0;
  AtPass pass = tile.all();
  const bool mixed = tile.b_first != tile.b_last;
  uint32_t it = 0, issued = 0, passes = 0;
  bool ok = true;
  if (warp == F::EL_WARPS + 1) ok = __all_sync(FULL_MASK, t5_mbar_wait(&r_full, 0, failed));

  for (;;) {
    const int64_t count = pass.c_hi - pass.c_lo;
    const uint32_t each = (uint32_t)((count + AT_COLS - 1) / AT_COLS);  // steps per head
    const uint32_t steps = each * heads;
    if (warp == F::EL_WARPS) {
      // ---- copies
      uint32_t e = 0, c = 0;
      for (uint32_t s = 0; s < steps && ok; ++s) {
        const uint32_t g = it + s, st = g % F::STAGES, round = g / F::STAGES;
        if (round > 0) ok = __all_sync(FULL_MASK, t5_mbar_wait(&empty[st], (round - 1) & 1, failed));
        if (!ok) break;
        const int64_t c0 = pass.c_lo + (int64_t)c * AT_COLS;
        const int head = KV ? head0 + (int)e : group;
        unsigned char *dst = stages + st * F::STAGE_BYTES;
        if (lane == 0) {
          t5_mbar_expect(&full[st], F::STAGE_BYTES);
          for (int at = 0; at < ATOMS; ++at) {
            t5_tma_3d(dst + at * (AT_COLS * 128), &maps.col0, at * 64, head, (int)c0, &full[st]);
            t5_tma_3d(dst + F::TILE_BYTES + at * (AT_COLS * 128), &maps.col1, at * 64, head, (int)c0, &full[st]);
          }
        }
        float *sd = side + st * F::SIDE_FLOATS;
        if constexpr (DIM > 0) {
          const float *src = KV ? p.pos_q : p.pos_k;
          for (int i = lane; i < AT_COLS * DIM; i += 32) {
            const int j = i / DIM, d = i - j * DIM;
            sd[d * AT_COLS + j] = c0 + j < pass.c_hi && d < p.dims ? src[(c0 + j) * p.dims + d] : 0.f;
          }
        }
        if constexpr (KV) {
          for (int j = lane; j < AT_COLS; j += 32) {
            const bool there = c0 + j < pass.c_hi;
            sd[AT_MAX_DIMS * AT_COLS + j] = there ? a.lse[(int64_t)head * p.m + c0 + j] - A::SHIFT : pos_inf<float>();
            sd[(AT_MAX_DIMS + 1) * AT_COLS + j] = there ? a.delta[(int64_t)head * p.m + c0 + j] : 0.f;
          }
        }
        __syncwarp();
        if (lane == 0) t5_mbar_arrive(&full[st]);
        issued = g + 1;
        if (++c == each) {
          c = 0;
          ++e;
        }
      }
    } else if (warp == F::EL_WARPS + 1) {
      // ---- products
      const uint32_t id_s = t5_idesc(A::BF16, AT_COLS, false), id_a = t5_idesc(A::BF16, CP, true);
      constexpr uint32_t LAG = F::NB - 1;
      for (uint32_t s = 0; s < steps + LAG && steps > 0 && ok; ++s) {
        if (s < steps) {
          const uint32_t g = it + s, st = g % F::STAGES, nb = g % F::NB;
          ok = __all_sync(FULL_MASK, t5_mbar_wait(&full[st], (g / F::STAGES) & 1, failed));
          // the accumulators hold the weights of NB steps ago: products of different accumulators are not ordered
          if (ok && s >= F::NB) {
            const uint32_t b = g - F::NB;
            ok = __all_sync(FULL_MASK, t5_mbar_wait(&empty[b % F::STAGES], (b / F::STAGES) & 1, failed));
          }
          if (!ok) break;
          t5_fence_after();
          if (lane == 0) {
            const uint32_t c0 = t5_smem(stages + st * F::STAGE_BYTES), c1 = c0 + F::TILE_BYTES;
#pragma unroll
            for (int ks = 0; ks < CP / 16; ++ks) {
              const uint32_t ro = (ks >> 2) * (AT_ROWS * 128) + (ks & 3) * 32, co = (ks >> 2) * (AT_COLS * 128) + (ks & 3) * 32;
              t5_mma_ss(tmem + nb * 2 * AT_COLS, t5_desc(t5_smem(rows0) + ro), t5_desc(c0 + co), id_s, ks > 0);
            }
#pragma unroll
            for (int ks = 0; ks < CP / 16; ++ks) {
              const uint32_t ro = (ks >> 2) * (AT_ROWS * 128) + (ks & 3) * 32, co = (ks >> 2) * (AT_COLS * 128) + (ks & 3) * 32;
              t5_mma_ss(tmem + nb * 2 * AT_COLS + AT_COLS, t5_desc(t5_smem(rows1) + ro), t5_desc(c1 + co), id_s, ks > 0);
            }
            t5_commit(&s_full[nb]);
          }
          __syncwarp();
        }
        if (s >= LAG) {
          const uint32_t g = it + s - LAG, st = g % F::STAGES, nb = g % F::NB;
          ok = __all_sync(FULL_MASK, t5_mbar_wait(&w_ready[nb], (g / F::NB) & 1, failed));
          if (!ok) break;
          t5_fence_after();
          if (lane == 0) {
            const uint32_t c0 = t5_smem(stages + st * F::STAGE_BYTES), c1 = c0 + F::TILE_BYTES;
            const uint32_t w = tmem + nb * 2 * AT_COLS;
            const bool more = s > LAG;
#pragma unroll
            for (int ks = 0; ks < AT_COLS / 16; ++ks) {
              const uint32_t wo = (ks >> 1) * 32 + (ks & 1) * 8;
              if constexpr (KV) {
                t5_mma_ts(t_acc, w + wo, t5_desc(c1 + ks * 2048, AT_COLS * 128), id_a, more || ks > 0);
                t5_mma_ts(t_acc + CP, w + AT_COLS + wo, t5_desc(c0 + ks * 2048, AT_COLS * 128), id_a, more || ks > 0);
              } else {
                t5_mma_ts(t_acc, w + AT_COLS + wo, t5_desc(c0 + ks * 2048, AT_COLS * 128), id_a, more || ks > 0);
              }
            }
            t5_commit(&empty[st]);
            if (s == steps + LAG - 1) t5_commit(&done);
          }
          __syncwarp();
        }
      }
    } else {
      // ---- elements
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      const bool mine = pass.segment < 0 || pass.segment == row_segment;
      const int64_t lo64 = mine ? row_lo - pass.c_lo : 0, hi64 = mine ? row_hi - pass.c_lo : 0;
      const int lo = (int)(lo64 < 0 ? 0 : lo64 > count ? count : lo64), hi = (int)(hi64 < 0 ? 0 : hi64 > count ? count : hi64);
      uint32_t bad = 0u, e = 0, c = 0;
      for (uint32_t s = 0; s < steps && ok; ++s) {
        const uint32_t g = it + s, st = g % F::STAGES, nb = g % F::NB;
        const int step_base = (int)(c * AT_COLS), base = step_base + half * 32;
        const bool last = step_base + AT_COLS > (int)count;
        unsigned char *stage = stages + st * F::STAGE_BYTES;
        const float *sd = side + st * F::SIDE_FLOATS + half * 32;
        float slope2 = 0.f;
        if constexpr (DIM > 0) slope2 = __ldg(p.slope + head0 + e) * AT_LOG2E;
        ok = __all_sync(FULL_MASK, t5_mbar_wait(&full[st], (g / F::STAGES) & 1, failed));
        if (mixed && !by_example && ok) {
          bad |= at_scan<T, CP>(stage, tid, F::EL_THREADS);
          if constexpr (KV) bad |= at_scan<T, CP>(stage + F::TILE_BYTES, tid, F::EL_THREADS);
        }
        if (ok) ok = __all_sync(FULL_MASK, t5_mbar_wait(&s_full[nb], (g / F::NB) & 1, failed));
        if (!ok) break;
        t5_fence_after();
        const uint32_t t_s = tmem + nb * 2 * AT_COLS + half * 32 + lane_base, t_dp = t_s + AT_COLS;
        uint32_t w[16], wp[KV ? 16 : 1];
        const bool any = __any_sync(FULL_MASK, hi > base && lo < base + 32 && lo < hi);
        if (any) {
          float x[32], dp[32], u[CAP ? 32 : 1];
          t5_ld32(t_s, x);
          t5_ld32(t_dp, dp);
          t5_wait_ld32(x);
          t5_wait_ld32(dp);
          at_logits<DIM, CAP, CAP>(x, u, sd, pos, slope2, pre, post);
          const bool whole = __all_sync(FULL_MASK, lo <= base && hi >= base + 32);
#pragma unroll
          for (int j4 = 0; j4 < 32; j4 += 4) {
            float ls[4] = {lse, lse, lse, lse}, de[4] = {delta, delta, delta, delta};
            if constexpr (KV) {
              const float4 l4 = *reinterpret_cast<const float4 *>(sd + AT_MAX_DIMS * AT_COLS + j4);
              const float4 d4 = *reinterpret_cast<const float4 *>(sd + (AT_MAX_DIMS + 1) * AT_COLS + j4);
              ls[0] = l4.x, ls[1] = l4.y, ls[2] = l4.z, ls[3] = l4.w;
              de[0] = d4.x, de[1] = d4.y, de[2] = d4.z, de[3] = d4.w;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float pr = t5_ex2(x[j4 + j] - ls[j]);
              float ds = pr * (dp[j4 + j] - de[j]);
              if constexpr (CAP) ds *= fmaf(-u[j4 + j], u[j4 + j], 1.f);
              if constexpr (!A::BF16) ds *= sig;
              x[j4 + j] = pr;
              dp[j4 + j] = ds;
            }
          }
          if (!whole) {
#pragma unroll
            for (int j = 0; j < 32; ++j)
              if (base + j < lo || base + j >= hi) x[j] = dp[j] = 0.f;
          }
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            w[j] = A::pack(dp[2 * j], dp[2 * j + 1]);
            if constexpr (KV) wp[j] = A::pack(x[2 * j], x[2 * j + 1]);
          }
        } else {
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            w[j] = 0u;
            if constexpr (KV) wp[j] = 0u;
          }
        }
        t5_st16(t_dp, w);
        if constexpr (KV) t5_st16(t_s, wp);
        t5_wait_st();
        if (last) {
          at_clear<CP>(stage, (int)count - step_base, tid, F::EL_THREADS);
          if constexpr (KV) at_clear<CP>(stage + F::TILE_BYTES, (int)count - step_base, tid, F::EL_THREADS);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        t5_fence_before();
        t5_mbar_arrive(&w_ready[nb]);
        if (++c == each) {
          c = 0;
          ++e;
        }
      }
      if (ok && steps > 0) {
        ok = __all_sync(FULL_MASK, t5_mbar_wait(&done, passes & 1, failed));
        t5_fence_after();
      }
      if (bad) bad_s = 1;
      const bool redo = mixed && !by_example;
      if (redo) asm volatile("bar.sync 1, 256;" ::: "memory");
      if (!(redo && *(volatile int *)&bad_s)) {
        const bool store = mine && row < tile.t1;
        const float nan = __int_as_float(0x7fffffff);
        // the first half of the warps takes dv (or the first channels of dq), the second dk (or the others)
        T *dst;
        float times;
        int c_first, c_count;
        if constexpr (KV) {
          dst = (half == 0 ? (T *)a.dv : (T *)a.dk) + (row * p.groups + group) * p.channels;
          times = half == 0 ? (A::BF16 ? 1.f : 1.f / 4096.f) : p.scale / sigma;
          c_first = 0;
          c_count = CP;
        } else {
          dst = (T *)a.dq + (row * p.heads + head0) * p.channels;
          times = p.scale / sigma;
          c_first = half * (CP / 2);
          c_count = CP / 2;
        }
        if (!ok) times = nan;
        for (int cc = c_first; cc < c_first + c_count; cc += 32) {
          float o[32];
          if (steps > 0 && ok) {
            t5_ld32(t_acc + (KV && half ? CP : 0) + lane_base + cc, o);
            t5_wait_ld32(o);
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i) o[i] = 0.f;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 out;
            uint32_t *po = reinterpret_cast<uint32_t *>(&out);
#pragma unroll
            for (int k = 0; k < 4; ++k) po[k] = A::pack(o[i + 2 * k] * times, o[i + 2 * k + 1] * times);
            if (store && cc + i < p.channels) *reinterpret_cast<uint4 *>(dst + cc + i) = out;
          }
        }
      }
    }
    it += steps;
    if (steps > 0) ++passes;
    t5_fence_before();
    __syncthreads();
    t5_fence_after();
    if (*failed) break;
    if (!by_example) {
      if (!mixed || !*(volatile int *)&bad_s) break;
      by_example = true;
    }
    if (!tile.next(next_row, pass)) break;
  }
  if (*failed && element && row < tile.t1 && half == 0) {
    // a wait ran out: nothing of this block is to be trusted
    for (int c = 0; c < p.channels; ++c) {
      const T nan = at_round<T>(__int_as_float(0x7fffffff));
      if (KV) {
        ((T *)a.dk)[(row * p.groups + group) * p.channels + c] = nan;
        ((T *)a.dv)[(row * p.groups + group) * p.channels + c] = nan;
      } else {
        ((T *)a.dq)[(row * p.heads + head0) * p.channels + c] = nan;
      }
    }
  }
  if (*failed && warp == F::EL_WARPS) {
    at_drain(&r_full, 1, 1);
    at_drain(full, F::STAGES, issued);
  }
  if (*failed && warp == F::EL_WARPS + 1) {
    if (lane == 0) t5_commit(&drained);
    __syncwarp();
    at_drain(&drained, 1, 1);
  }
  __syncthreads();
  if (warp == F::EL_WARPS) t5_dealloc(tmem, F::TMEM);
}

}  // namespace b200c
