// Forward attention on the tensor cores: 128 queries of one head per block, see attention_tensor.cuh.
//
// Two score accumulators, so that the product of the next step's scores runs while this step's softmax does; the weights
// go back into the accumulator they came from.  The running maximum is only raised (and the result in tensor memory
// rescaled) when a row's maximum rises by more than 8 powers of two: until then weights up to 2^8 are exact enough in
// either type, and the rescaling, a round trip through tensor memory, is rare.
// Sums and the result are fp32; the weights are rounded to the 16-bit type as operands of the second product.
#pragma once

#include "attention_tensor.cuh"

namespace b200c {

template <int CP>
struct AtForward {
  static constexpr int STAGES = CP == 64 ? 3 : 2;
  static constexpr int THREADS = 192;  // 4 softmax warps, 1 copy warp, 1 product warp
  static constexpr int Q_BYTES = AT_ROWS * CP * 2, TILE_BYTES = AT_COLS * CP * 2;
  static constexpr int POS_BYTES = AT_MAX_DIMS * AT_COLS * 4;
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int SMEM = Q_BYTES + STAGES * (STAGE_BYTES + POS_BYTES) + 1024;
  static constexpr int TMEM = 256;
  static constexpr float RAISE = 8.f;
};

struct AtForwardMaps {
  CUtensorMap q, k, v;
};

template <typename T, int CP, int DIM, bool CAP>
__global__ void __launch_bounds__(AtForward<CP>::THREADS, 2)
attention_forward_kernel(const __grid_constant__ AtForwardMaps maps, const __grid_constant__ AttnArgs a,
                         T *__restrict__ rest) {
  using F = AtForward<CP>;
  using A = AtType<T>;
  constexpr int ATOMS = CP / 64;
  extern __shared__ unsigned char at_raw[];
  unsigned char *smem = at_raw + ((1024u - (t5_smem(at_raw) & 1023u)) & 1023u);
  unsigned char *sq = smem;
  unsigned char *stages = smem + F::Q_BYTES;
  float *spos = reinterpret_cast<float *>(stages + F::STAGES * F::STAGE_BYTES);
  __shared__ __align__(8) uint64_t q_full, full[F::STAGES], empty[F::STAGES], s_full[2], p_ready[2], o_done, done, drained;
  __shared__ uint32_t tmem_s;
  __shared__ int failed_s, bad_s;
  volatile int *failed = &failed_s;

  const b200c_attention_t &p = a.p;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int head = blockIdx.y, group = head / (p.heads / p.groups);
  AtTile tile;
  tile.init((int64_t)blockIdx.x * AT_ROWS, p.ptr_q, p.ptr_k, p.m, p.n, p.num_segments);

  if (tid == 0) {
    t5_mbar_init(&q_full, 1);
    for (int i = 0; i < F::STAGES; ++i) {
      t5_mbar_init(&full[i], 1);
      t5_mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      t5_mbar_init(&s_full[i], 1);
      t5_mbar_init(&p_ready[i], AT_ROWS);
    }
    t5_mbar_init(&o_done, 1);
    t5_mbar_init(&done, 1);
    t5_mbar_init(&drained, 1);
    failed_s = 0;
    bad_s = 0;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == 4) t5_alloc(&tmem_s, F::TMEM);
  t5_fence_before();
  __syncthreads();
  t5_fence_after();
  const uint32_t tmem = tmem_s;
  const uint32_t t_o = tmem + 2 * AT_COLS;

  // softmax threads: a row each
  const int64_t row = tile.t0 + tid;
  int64_t row_lo = 0, row_hi = 0;  // the columns it sees
  int row_segment = -1;
  float pos[DIM == 0 ? 1 : DIM], slope2 = 0.f;
  if (warp < 4 && row < tile.t1) {
    row_segment = segment_of(tile.ptr_r, tile.segments, row);
    int64_t lo, hi;
    at_segment(tile.ptr_r, p.m, row_segment, lo, hi);
    if (row >= lo && row < hi) at_segment(tile.ptr_c, p.n, row_segment, row_lo, row_hi);
  }
  if constexpr (DIM > 0) {
    slope2 = p.slope[head] * AT_LOG2E;
#pragma unroll
    for (int d = 0; d < DIM; ++d) pos[d] = warp < 4 && row < tile.t1 && d < p.dims ? p.pos_q[row * p.dims + d] : 0.f;
  }
  const float pre = CAP ? 2.f * AT_LOG2E * p.scale / p.cap : p.scale * AT_LOG2E, post = p.cap * AT_LOG2E;

  // the copy warp: the queries once
  if (warp == 4 && lane == 0) {
    t5_mbar_expect(&q_full, F::Q_BYTES);
    for (int at = 0; at < ATOMS; ++at)
      t5_tma_3d(sq + at * (AT_ROWS * 128), &maps.q, at * 64, head, (int)tile.t0, &q_full);
    t5_mbar_arrive(&q_full);
  }

  bool by_example = false;
  int64_t next_row = tile.t0;
  AtPass pass = tile.all();
  const bool mixed = tile.b_first != tile.b_last;
  uint32_t it = 0;      // steps so far, over all passes
  uint32_t passes = 0;  // passes with steps
  uint32_t issued = 0;  // copy warp: steps whose copies were issued
  bool ok = true;
  if (warp == 5) ok = __all_sync(FULL_MASK, t5_mbar_wait(&q_full, 0, failed));

  for (;;) {
    const int64_t count = pass.c_hi - pass.c_lo;
    const uint32_t steps = (uint32_t)((count + AT_COLS - 1) / AT_COLS);
    if (warp == 4) {
      // ---- copies
      for (uint32_t s = 0; s < steps && ok; ++s) {
        const uint32_t g = it + s, st = g % F::STAGES, round = g / F::STAGES;
        if (round > 0) ok = __all_sync(FULL_MASK, t5_mbar_wait(&empty[st], (round - 1) & 1, failed));
        if (!ok) break;
        const int64_t c0 = pass.c_lo + (int64_t)s * AT_COLS;
        unsigned char *dst = stages + st * F::STAGE_BYTES;
        if (lane == 0) {
          t5_mbar_expect(&full[st], F::STAGE_BYTES);
          for (int at = 0; at < ATOMS; ++at) {
            t5_tma_3d(dst + at * (AT_COLS * 128), &maps.k, at * 64, group, (int)c0, &full[st]);
            t5_tma_3d(dst + F::TILE_BYTES + at * (AT_COLS * 128), &maps.v, at * 64, group, (int)c0, &full[st]);
          }
        }
        if constexpr (DIM > 0) {
          float *sp = spos + st * (AT_MAX_DIMS * AT_COLS);
          for (int i = lane; i < AT_COLS * DIM; i += 32) {
            const int c = i / DIM, d = i - c * DIM;
            sp[d * AT_COLS + c] = c0 + c < pass.c_hi && d < p.dims ? p.pos_k[(c0 + c) * p.dims + d] : 0.f;
          }
          __syncwarp();
        }
        if (lane == 0) t5_mbar_arrive(&full[st]);
        issued = g + 1;
      }
    } else if (warp == 5) {
      // ---- products
      const uint32_t id_s = t5_idesc(A::BF16, AT_COLS, false), id_o = t5_idesc(A::BF16, CP, true);
      for (uint32_t s = 0; s <= steps && steps > 0 && ok; ++s) {
        if (s < steps) {
          const uint32_t g = it + s, st = g % F::STAGES;
          ok = __all_sync(FULL_MASK, t5_mbar_wait(&full[st], (g / F::STAGES) & 1, failed));
          // the accumulator holds the weights of two steps ago: products of different accumulators are not ordered
          if (ok && s > 1) ok = __all_sync(FULL_MASK, t5_mbar_wait(&o_done, (g - 2) & 1, failed));
          if (!ok) break;
          t5_fence_after();
          if (lane == 0) {
            const uint32_t sk = t5_smem(stages + st * F::STAGE_BYTES);
#pragma unroll
            for (int ks = 0; ks < CP / 16; ++ks) {
              const uint64_t da = t5_desc(t5_smem(sq) + (ks >> 2) * (AT_ROWS * 128) + (ks & 3) * 32);
              const uint64_t db = t5_desc(sk + (ks >> 2) * (AT_COLS * 128) + (ks & 3) * 32);
              t5_mma_ss(tmem + (g & 1) * AT_COLS, da, db, id_s, ks > 0);
            }
            t5_commit(&s_full[g & 1]);
          }
          __syncwarp();
        }
        if (s > 0) {
          const uint32_t g = it + s - 1, st = g % F::STAGES;
          ok = __all_sync(FULL_MASK, t5_mbar_wait(&p_ready[g & 1], (g >> 1) & 1, failed));
          if (!ok) break;
          t5_fence_after();
          if (lane == 0) {
            const uint32_t sv = t5_smem(stages + st * F::STAGE_BYTES + F::TILE_BYTES);
#pragma unroll
            for (int ks = 0; ks < AT_COLS / 16; ++ks)
              t5_mma_ts(t_o, tmem + (g & 1) * AT_COLS + ks * 8, t5_desc(sv + ks * 2048, AT_COLS * 128), id_o,
                        s > 1 || ks > 0);
            t5_commit(&empty[st]);
            t5_commit(&o_done);
            if (s == steps) t5_commit(&done);
          }
          __syncwarp();
        }
      }
    } else {
      // ---- softmax
      const uint32_t lane_base = (uint32_t)(warp * 32) << 16;
      const bool mine = pass.segment < 0 || pass.segment == row_segment;
      // the row's columns relative to the pass's first; 64 columns fit an int many times over
      const int64_t lo64 = mine ? row_lo - pass.c_lo : 0, hi64 = mine ? row_hi - pass.c_lo : 0;
      const int lo = (int)(lo64 < 0 ? 0 : lo64 > count ? count : lo64), hi = (int)(hi64 < 0 ? 0 : hi64 > count ? count : hi64);
      float top = -pos_inf<float>(), sum = 0.f;
      uint32_t bad = 0u;
      for (uint32_t s = 0; s < steps && ok; ++s) {
        const uint32_t g = it + s, st = g % F::STAGES;
        const int base = (int)(s * AT_COLS);
        const bool last = base + AT_COLS > (int)count;
        if (DIM > 0 || mixed || last)
          ok = __all_sync(FULL_MASK, t5_mbar_wait(&full[st], (g / F::STAGES) & 1, failed));
        if (mixed && !by_example && ok)
          bad |= at_scan<T, CP>(stages + st * F::STAGE_BYTES + F::TILE_BYTES, tid, AT_ROWS);
        if (ok) ok = __all_sync(FULL_MASK, t5_mbar_wait(&s_full[g & 1], (g >> 1) & 1, failed));
        if (!ok) break;
        t5_fence_after();
        const uint32_t t_s = tmem + (g & 1) * AT_COLS + lane_base;
        uint32_t w[32];
        const bool any = __any_sync(FULL_MASK, hi > base && lo < base + AT_COLS && lo < hi);
        if (any) {
          float x[AT_COLS];
          t5_ld32(t_s, x);
          t5_ld32(t_s + 32, x + 32);
          t5_wait_ld32(x);
          t5_wait_ld32(x + 32);
          const float *cp = spos + st * (AT_MAX_DIMS * AT_COLS);
          at_logits<DIM, CAP, false>(x, nullptr, cp, pos, slope2, pre, post);
          at_logits<DIM, CAP, false>(x + 32, nullptr, cp + 32, pos, slope2, pre, post);
          if (!__all_sync(FULL_MASK, lo <= base && hi >= base + AT_COLS)) {
#pragma unroll
            for (int j = 0; j < AT_COLS; ++j)
              if (base + j < lo || base + j >= hi) x[j] = -pos_inf<float>();
          }
          float m0 = top, m1 = x[0], m2 = x[1], m3 = x[2];
#pragma unroll
          for (int j = 3; j + 3 < AT_COLS; j += 4) {
            m0 = fmaxf(m0, x[j]);
            m1 = fmaxf(m1, x[j + 1]);
            m2 = fmaxf(m2, x[j + 2]);
            m3 = fmaxf(m3, x[j + 3]);
          }
          m0 = fmaxf(fmaxf(m0, m1), fmaxf(fmaxf(m2, m3), x[AT_COLS - 1]));
          const bool raise = m0 > top + F::RAISE || (top == -pos_inf<float>() && m0 > top);
          if (__any_sync(FULL_MASK, raise)) {
            const float to = raise ? m0 : top;
            const float shrink = raise ? t5_ex2(top - to) : 1.f;  // from -inf: 0
            top = to;
            sum *= shrink;
            if (s > 0) {
              // the product of the step before has to be in
              ok = __all_sync(FULL_MASK, t5_mbar_wait(&o_done, (g - 1) & 1, failed));
              if (!ok) break;
              t5_fence_after();
#pragma unroll
              for (int c = 0; c < CP; c += 32) {
                float o[32];
                t5_ld32(t_o + lane_base + c, o);
                t5_wait_ld32(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= shrink;
                t5_st32(t_o + lane_base + c, reinterpret_cast<const uint32_t *>(o));
              }
            }
          }
          const float sub = top == -pos_inf<float>() ? 0.f : top;
          float l0 = 0.f, l1 = 0.f;
#pragma unroll
          for (int j = 0; j < AT_COLS; j += 2) {
            const float e0 = t5_ex2(x[j] - sub), e1 = t5_ex2(x[j + 1] - sub);
            l0 += e0;
            l1 += e1;
            w[j >> 1] = A::pack(e0, e1);
          }
          sum += l0 + l1;
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) w[j] = 0u;
        }
        t5_st32(t_s, w);
        t5_wait_st();
        if (last) {
          at_clear<CP>(stages + st * F::STAGE_BYTES + F::TILE_BYTES, (int)count - base, tid, AT_ROWS);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        t5_fence_before();
        t5_mbar_arrive(&p_ready[g & 1]);
      }
      if (ok && steps > 0) {
        ok = __all_sync(FULL_MASK, t5_mbar_wait(&done, passes & 1, failed));
        t5_fence_after();
      }
      if (bad) bad_s = 1;
      const bool redo = mixed && !by_example;
      if (redo) {  // the softmax warps agree on whether this pass counts
        asm volatile("bar.sync 1, 128;" ::: "memory");
      }
      if (!(redo && *(volatile int *)&bad_s)) {
        const bool store = mine && row < tile.t1;
        const float nan = __int_as_float(0x7fffffff);
        const float inv = !ok ? nan : sum == 0.f ? 0.f : 1.f / sum;
        T *dst = (T *)a.out + (row * p.heads + head) * p.channels;
        T *dst2 = rest ? rest + (row * p.heads + head) * p.channels : nullptr;
#pragma unroll
        for (int c = 0; c < CP; c += 32) {
          float o[32];
          if (steps > 0 && ok) {
            t5_ld32(t_o + lane_base + c, o);
            t5_wait_ld32(o);
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 out, low;
            uint32_t *po = reinterpret_cast<uint32_t *>(&out), *pl = reinterpret_cast<uint32_t *>(&low);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x0 = 0.f, x1 = 0.f;
              if (steps > 0 && (sum != 0.f || !ok)) {
                x0 = o[i + 2 * e] * inv;
                x1 = o[i + 2 * e + 1] * inv;
              }
              if (!ok) x0 = x1 = nan;
              po[e] = A::pack(x0, x1);
              const T *h = reinterpret_cast<const T *>(&po[e]);
              pl[e] = A::pack(x0 - at_float(h[0]), x1 - at_float(h[1]));
            }
            if (store && c + i < p.channels) {
              *reinterpret_cast<uint4 *>(dst + c + i) = out;
              if (dst2) *reinterpret_cast<uint4 *>(dst2 + c + i) = low;
            }
          }
        }
        if (a.lse && store) a.lse[(int64_t)head * p.m + row] = sum == 0.f ? pos_inf<float>() : top + log2f(sum);
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
  if (*failed && warp < 4 && row < tile.t1) {
    // a wait ran out: nothing of this block is to be trusted
    T *dst = (T *)a.out + (row * p.heads + head) * p.channels;
    for (int c = 0; c < p.channels; ++c) dst[c] = at_round<T>(__int_as_float(0x7fffffff));
  }
  if (*failed && warp == 4) {
    at_drain(&q_full, 1, 1);
    at_drain(full, F::STAGES, issued);
  }
  if (*failed && warp == 5) {
    if (lane == 0) t5_commit(&drained);
    __syncwarp();
    at_drain(&drained, 1, 1);
  }
  __syncthreads();
  if (warp == 4) t5_dealloc(tmem, F::TMEM);
}

}  // namespace b200c
