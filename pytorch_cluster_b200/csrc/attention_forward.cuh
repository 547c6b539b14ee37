// Forward attention on the tensor cores: 128 queries of one head per block, see attention_tensor.cuh.
//
// Each group of warps has its own running maximum, sum and result of its steps; they are joined at the end.  The
// maximum is not looked for in every step: weights are formed against the one in use, and only where their sum over the
// step's 32 columns passes 2^10 in bf16, 2^6 in fp16 (or no maximum is known yet) is it raised to the step's and the
// result in tensor memory, the sum and the step's weights brought to it.  bf16 holds weights up to 2^10 as exactly as
// weights up to 1; fp16 keeps them times 2^9, below 2^15, and loses less than 2^-34 of the row's sum with each.
// Sums and the result are fp32; the weights are rounded to the 16-bit type as operands of the second product.
// The result is divided by the sum of the rounded weights, not of the exact ones (which the statistics keep): where few
// keys share the weight their roundings then cancel, and D = do . o, which the gradients need, is as much better.
#pragma once

#include "attention_tensor.cuh"

namespace b200c {

template <int CP>
struct AtForward {
  static constexpr int G = 2;
  static constexpr int BLOCKS = CP == 64 ? 2 : 1;  // resident blocks per SM: tensor memory
  static constexpr int STAGES = CP == 64 ? 3 : 4;
  static constexpr int EL_WARPS = 4 * G, EL_THREADS = 32 * EL_WARPS;
  static constexpr int THREADS = EL_THREADS + 96;  // the groups, a copy warp, two product warps
  static constexpr int Q_BYTES = AT_ROWS * CP * 2, TILE_BYTES = AT_COLS * CP * 2;
  static constexpr int POS_BYTES = AT_MAX_DIMS * AT_COLS * 4;
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int SMEM = Q_BYTES + STAGES * (STAGE_BYTES + POS_BYTES) + 1024;
  static constexpr int PAIRS = G / 2, PAIR_COLS = AT_COLS + AT_SUB;  // scores of a stage, two groups' weights
  static constexpr int TMEM = CP == 64 ? 256 : 512;
  static_assert(STAGES * STAGE_BYTES >= 2 * Q_BYTES, "the ring takes the block's rows");
  static_assert(PAIRS * PAIR_COLS + G * CP <= TMEM, "tensor memory");
};

struct AtForwardMaps {
  CUtensorMap q, k, v;
};

template <typename T, int CP, int DIM, bool CAP>
__global__ void __launch_bounds__(AtForward<CP>::THREADS, AtForward<CP>::BLOCKS)
attention_forward_kernel(const __grid_constant__ AtForwardMaps maps, const __grid_constant__ AttnArgs a,
                         T *__restrict__ rest) {
  using F = AtForward<CP>;
  using A = AtType<T>;
  constexpr int ATOMS = CP / 64, G = F::G, COPY = F::EL_WARPS, SCORE = F::EL_WARPS + 1, SUM = F::EL_WARPS + 2;
  extern __shared__ unsigned char at_raw[];
  unsigned char *smem = at_raw + ((1024u - (t5_smem(at_raw) & 1023u)) & 1023u);
  unsigned char *sq = smem;
  unsigned char *stages = smem + F::Q_BYTES;
  float *spos = reinterpret_cast<float *>(stages + F::STAGES * F::STAGE_BYTES);
  // s_full / s_free: a pair's scores are in / have been read; w_ready: a group's weights are in; a_done: their product
  // is
  __shared__ __align__(8) uint64_t q_full, full[F::STAGES], empty[F::STAGES], s_full[F::PAIRS], s_free[F::PAIRS],
      w_ready[G], a_done[G], done, drained[2];
  __shared__ uint32_t tmem_s;
  __shared__ int failed_s, bad_s;
  __shared__ AtTileShared shared_tile;
  __shared__ float s_top[G][AT_ROWS], s_sum[G][AT_ROWS], s_sum16[G][AT_ROWS];
  volatile int *failed = &failed_s;

  const b200c_attention_t &p = a.p;
  const int tid = threadIdx.x, warp = t5_warp(), lane = tid & 31;
  const int head = (int)(blockIdx.x % (unsigned)p.heads), group = head / (p.heads / p.groups);
  AtTile tile;
  tile.init(at_tile_of(a.order, p.heads) * AT_ROWS, p.ptr_q, p.ptr_k, p.m, p.n, p.num_segments);

  // element threads: a row each
  const bool element = warp < F::EL_WARPS;
  const int grp = warp >> 2, lrow = tid & (AT_ROWS - 1);
  const int64_t row = tile.t0 + lrow;
  float pos[DIM == 0 ? 1 : DIM], slope2 = 0.f;
  if constexpr (DIM > 0) {
    slope2 = p.slope[head] * AT_LOG2E;
#pragma unroll
    for (int d = 0; d < DIM; ++d) pos[d] = element && row < tile.t1 && d < p.dims ? p.pos_q[row * p.dims + d] : 0.f;
  }

  if (tid == 64) {
    t5_mbar_init(&q_full, 1);
    for (int i = 0; i < F::STAGES; ++i) {
      t5_mbar_init(&full[i], 1);
      t5_mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < F::PAIRS; ++i) {
      t5_mbar_init(&s_full[i], 1);
      t5_mbar_init(&s_free[i], 8);
    }
    for (int i = 0; i < G; ++i) {
      t5_mbar_init(&w_ready[i], 4);
      t5_mbar_init(&a_done[i], 1);
    }
    t5_mbar_init(&done, 1);
    t5_mbar_init(&drained[0], 1);
    t5_mbar_init(&drained[1], 1);
    failed_s = 0;
    bad_s = 0;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
  }
  if (warp == COPY) t5_alloc(&tmem_s, F::TMEM);
  tile.search(shared_tile, warp, lane);
  t5_fence_before();
  __syncthreads();
  t5_fence_after();
  const uint32_t tmem = tmem_s;
  const uint32_t t_o = tmem + F::PAIRS * F::PAIR_COLS;  // G results
  // the copy warp: the queries once
  if (warp == COPY && lane == 0) {
    t5_mbar_expect(&q_full, F::Q_BYTES);
    for (int at = 0; at < ATOMS; ++at)
      t5_tma_3d(sq + at * (AT_ROWS * 128), &maps.q, at * 64, head, (int)tile.t0, &q_full);
    t5_mbar_arrive(&q_full);
  }
  tile.found(shared_tile);
  if (tile.listed()) {
    tile.list(shared_tile, tid);
    __syncthreads();
  }

  // element threads: the columns that the row sees
  int64_t row_lo = 0, row_hi = 0;
  int row_segment = -1;
  if (element && row < tile.t1) {
    row_segment = tile.segment(shared_tile, row);
    int64_t lo, hi;
    tile.rows_of(shared_tile, row_segment, lo, hi);
    if (row >= lo && row < hi) tile.cols_of(shared_tile, row_segment, row_lo, row_hi);
    if (grp == 0) shared_tile.segment[lrow] = row_segment;
  }
  const float pre = CAP ? 2.f * AT_LOG2E * p.scale / p.cap : p.scale * AT_LOG2E, post = p.cap * AT_LOG2E;

  bool by_example = false;
  int64_t next_row = tile.t0;
  AtPass pass = tile.all(shared_tile);
  // This block's share of the tile's columns, in whole stages.  A pass over one example takes what of it lies in the share
  // of the whole tile: each block decides by itself whether it goes example by example, and the others' columns must not
  // depend on that.
  __shared__ int64_t share_s[2];
  if (a.splits > 1) {
    const int64_t unit = (int64_t)a.splits * AT_COLS;
    const int64_t each = (pass.c_hi - pass.c_lo + unit - 1) / unit * AT_COLS;
    pass.c_lo += each * blockIdx.z;
    if (pass.c_lo > pass.c_hi) pass.c_lo = pass.c_hi;
    if (pass.c_lo + each < pass.c_hi) pass.c_hi = pass.c_lo + each;
    if (tid == 0) share_s[0] = pass.c_lo, share_s[1] = pass.c_hi;  // read after a barrier, at the end of this pass
  }
  const bool mixed = tile.b_first != tile.b_last;
  uint32_t stage0 = 0, passes = 0;  // stages, and passes with any, so far
  uint32_t issued = 0;              // copy warp: stages whose copies were issued
  bool ok = true;
  if (warp == SCORE) ok = t5_mbar_wait_warp(&q_full, 0, failed);

  for (;;) {
    const int64_t count = pass.c_hi - pass.c_lo;
    const uint32_t each = at_stages(count), stages_now = each;
    if (warp == COPY) {
      // ---- copies
      AtRing<F::STAGES> ring(stage0);
      uint32_t c = 0;
      for (uint32_t g = stage0; g < stage0 + stages_now && ok; ++g, ring.next()) {
        const uint32_t st = ring.st;
        const int64_t c0 = pass.c_lo + (int64_t)c * AT_COLS;
        // the columns' coordinates are on their way while the stage is waited for
        float place[DIM == 0 ? 1 : 2 * DIM];
        at_fetch_places<DIM>(place, p.pos_k, p.dims, c0, pass.c_hi, lane);
        // the stage's round before this one is through
        if (g >= F::STAGES) ok = t5_mbar_wait_idle(&empty[st], ring.parity ^ 1u, failed);
        if (!ok) break;
        unsigned char *dst = stages + st * F::STAGE_BYTES;
        if (lane == 0) {
          t5_mbar_expect(&full[st], F::STAGE_BYTES);
          for (int at = 0; at < ATOMS; ++at) {
            t5_tma_3d(dst + at * (AT_COLS * 128), &maps.k, at * 64, group, (int)c0, &full[st]);
            t5_tma_3d(dst + F::TILE_BYTES + at * (AT_COLS * 128), &maps.v, at * 64, group, (int)c0, &full[st]);
          }
        }
        if constexpr (DIM > 0) {
          at_put_places<DIM>(spos + st * (AT_MAX_DIMS * AT_COLS), place, lane);
          __syncwarp();
        }
        if (lane == 0) t5_mbar_arrive(&full[st]);
        issued = g + 1;
        ++c;
      }
    } else if (warp == SCORE) {
      // ---- scores
      const uint32_t id = t5_idesc(A::BF16, AT_COLS, false);
      const uint64_t d_q = t5_desc(t5_smem(sq)), d_k = t5_desc(t5_smem(stages));
      AtRing<F::STAGES> ring(stage0);
      for (uint32_t g = stage0; g < stage0 + stages_now && ok; ++g, ring.next()) {
        const uint32_t pair = g % F::PAIRS, k = g / F::PAIRS;
        ok = t5_mbar_wait_idle(&full[ring.st], ring.parity, failed);
        if (ok && k > 0) ok = t5_mbar_wait_idle(&s_free[pair], (k - 1) & 1, failed);
        if (!ok) break;
        t5_fence_after();
        const uint64_t d = d_k + ring.st * (F::STAGE_BYTES / 16);
        if (t5_elect()) {
#pragma unroll
          for (int ks = 0; ks < CP / 16; ++ks)
            t5_mma_ss(tmem + pair * F::PAIR_COLS, d_q + ((ks >> 2) * (AT_ROWS * 128) + (ks & 3) * 32) / 16,
                      d + ((ks >> 2) * (AT_COLS * 128) + (ks & 3) * 32) / 16, id, ks > 0);
          t5_commit(&s_full[pair]);
        }
        __syncwarp();
      }
    } else if (warp == SUM) {
      // ---- products with the weights
      const uint32_t id = t5_idesc(A::BF16, CP, true);
      const uint64_t d_v = t5_desc(t5_smem(stages + F::TILE_BYTES), AT_COLS * 128);
      AtRing<F::STAGES> ring(stage0);
      for (uint32_t g = stage0; g < stage0 + stages_now && ok; ++g, ring.next()) {
        const uint32_t pair = g % F::PAIRS, k = g / F::PAIRS;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t gr = 2 * pair + h;
          if (ok) ok = t5_mbar_wait_idle(&w_ready[gr], k & 1, failed);
          if (!ok) break;
          t5_fence_after();
          const uint64_t d = d_v + ring.st * (F::STAGE_BYTES / 16) + h * (AT_SUB * 128 / 16);
          const uint32_t w = tmem + pair * F::PAIR_COLS + AT_COLS + h * (AT_SUB / 2);
          if (t5_elect()) {
#pragma unroll
            for (int ks = 0; ks < AT_SUB / 16; ++ks)
              t5_mma_ts(t_o + gr * CP, w + ks * 8, d + ks * (2048 / 16), id, g - stage0 >= F::PAIRS || ks > 0);
            t5_commit(&a_done[gr]);
            if (h == 1) t5_commit(&empty[ring.st]);
            if (h == 1 && g + 1 == stage0 + stages_now) t5_commit(&done);
          }
          __syncwarp();
        }
      }
    } else {
      // ---- softmax
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t pair = grp >> 1, half = grp & 1, t_pair = tmem + pair * F::PAIR_COLS + lane_base;
      const uint32_t t_s = t_pair + half * AT_SUB, t_p = t_pair + AT_COLS + half * (AT_SUB / 2),
                     t_r = t_o + grp * CP + lane_base;
      const bool mine = pass.segment < 0 || pass.segment == row_segment;
      const AtSeen seen(row_lo, row_hi, pass, mine);
      const bool scan = mixed && !by_example;
      // sub: what the scores are taken relative to (0 as long as no maximum is known, then RAISED below it); sums of the
      // weights, exact and rounded
      float top = -pos_inf<float>(), sub = 0.f, sum = 0.f, sum16 = 0.f;
      uint32_t bad = 0u;
      const uint32_t c0 = (pair + F::PAIRS - stage0 % F::PAIRS) % F::PAIRS;  // the pair's first stage
      for (uint32_t c = c0; c < each && ok; c += F::PAIRS) {
        const uint32_t g = stage0 + c, st = g % F::STAGES, k = g / F::PAIRS;
        const int base = (int)(c * AT_COLS + half * AT_SUB);
        const bool tail = base + AT_SUB > (int)count, first = g - stage0 < F::PAIRS;
        unsigned char *values = stages + st * F::STAGE_BYTES + F::TILE_BYTES + half * (AT_SUB * 128);
        // the scores in, and what came with the columns, where it is read here
        ok = t5_mbar_wait_both(&s_full[pair], k & 1, &full[st], (g / F::STAGES) & 1, DIM > 0 || scan || tail, failed);
        if (!ok) break;
        if (scan) bad |= at_scan<T, CP>(values, lrow);
        t5_fence_after();
        uint32_t w[AT_SUB / 2];
        // asked here, answered when the weights are there to be stored
        bool taken = first || t5_mbar_try(&a_done[grp], (k - 1) & 1);
        if (seen.any(base)) {
          float x[AT_SUB];
          t5_ld32(t_s, x);
          t5_wait_ld32(x);
          t5_fence_before();
          __syncwarp();
          if (lane == 0) t5_mbar_arrive(&s_free[pair]);
          at_logits<DIM, CAP, false, false>(x, nullptr, spos + st * (AT_MAX_DIMS * AT_COLS) + half * AT_SUB, pos, slope2,
                                            pre, post, sub, nullptr);
          if (!seen.all(base)) {
#pragma unroll
            for (int j = 0; j < AT_SUB; ++j)
              if (base + j < seen.lo || base + j >= seen.hi) x[j] = -pos_inf<float>();
          }
          // rows that see their first columns here (sub is 0): the maximum is looked for
          const bool fresh = top == -pos_inf<float>() && seen.lo < base + AT_SUB && seen.hi > base && seen.lo < seen.hi;
          if (__any_sync(FULL_MASK, fresh)) {
            float m = x[0];
#pragma unroll
            for (int j = 1; j < AT_SUB; ++j) m = fmaxf(m, x[j]);
            if (fresh && m > -pos_inf<float>()) {
              top = m;
              sub = m - A::RAISED;
#pragma unroll
              for (int j = 0; j < AT_SUB; ++j) x[j] -= sub;
            }
          }
          float l0 = 0.f, l1 = 0.f, r0 = 0.f, r1 = 0.f;
#pragma unroll
          for (int j = 0; j < AT_SUB; j += 2) {
            const float e0 = t5_ex2(x[j]), e1 = t5_ex2(x[j + 1]);
            l0 += e0;
            l1 += e1;
            w[j >> 1] = A::pack(e0, e1);
            r0 += A::low(w[j >> 1]);
            r1 += A::high(w[j >> 1]);
          }
          l0 += l1;
          const bool raise = !(l0 <= A::MOST);
          if (__any_sync(FULL_MASK, raise)) {
            float m = x[0];
#pragma unroll
            for (int j = 1; j < AT_SUB; ++j) m = fmaxf(m, x[j]);
            m += sub;
            const float to = raise && m > top ? m : top;
            const float to_sub = to == -pos_inf<float>() ? 0.f : to - A::RAISED;
            const float shrink = top == -pos_inf<float>() ? 0.f : t5_ex2(sub - to_sub);
            l0 = l1 = r0 = r1 = 0.f;
#pragma unroll
            for (int j = 0; j < AT_SUB; j += 2) {
              const float e0 = t5_ex2(x[j] + (sub - to_sub)), e1 = t5_ex2(x[j + 1] + (sub - to_sub));
              l0 += e0;
              l1 += e1;
              w[j >> 1] = A::pack(e0, e1);
              r0 += A::low(w[j >> 1]);
              r1 += A::high(w[j >> 1]);
            }
            l0 += l1;
            top = to;
            sub = to_sub;
            sum *= shrink;
            sum16 *= shrink;
            if (!first) {
              // the product of the group's step before has to be in
              ok = t5_mbar_wait_warp(&a_done[grp], (k - 1) & 1, failed);
              if (!ok) break;
              t5_fence_after();
#pragma unroll
              for (int c = 0; c < CP; c += 32) {
                float o[32];
                t5_ld32(t_r + c, o);
                t5_wait_ld32(o);
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] *= shrink;
                t5_st32(t_r + c, o);
              }
            }
          }
          sum += l0;
          sum16 += r0 + r1;
        } else {
          if (lane == 0) t5_mbar_arrive(&s_free[pair]);
#pragma unroll
          for (int j = 0; j < AT_SUB / 2; ++j) w[j] = 0u;
        }
        // the weights of the group's step before have been taken
        if (!__all_sync(FULL_MASK, taken)) ok = t5_mbar_wait_warp(&a_done[grp], (k - 1) & 1, failed);
        if (!ok) break;
        t5_fence_after();
        t5_st16(t_p, w);
        t5_wait_st();
        if (tail) {
          at_clear<CP>(values, (int)count > base ? (int)count - base : 0, lrow);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        }
        t5_fence_before();
        __syncwarp();
        if (lane == 0) t5_mbar_arrive(&w_ready[grp]);
      }
      if (ok && count > 0) {
        ok = t5_mbar_wait_warp(&done, passes & 1, failed);
        t5_fence_after();
      }
      if (bad) bad_s = 1;
      s_top[grp][lrow] = top == -pos_inf<float>() ? top : sub;  // what the sums are relative to
      s_sum[grp][lrow] = sum;
      s_sum16[grp][lrow] = sum16;
      asm volatile("bar.sync 1, %0;" ::"n"(F::EL_THREADS) : "memory");
      if (!(scan && *(volatile int *)&bad_s)) {
        // join the groups: each takes CP / G channels of the row
        float all_top = -pos_inf<float>(), all_sum = 0.f, all_sum16 = 0.f, part[G];
#pragma unroll
        for (int g = 0; g < G; ++g) all_top = fmaxf(all_top, s_top[g][lrow]);
        const float all_sub = all_top == -pos_inf<float>() ? 0.f : all_top;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          part[g] = t5_ex2(s_top[g][lrow] - all_sub);
          all_sum = fmaf(part[g], s_sum[g][lrow], all_sum);
          all_sum16 = fmaf(part[g], s_sum16[g][lrow], all_sum16);
        }
        const bool none = all_sum == 0.f;
        const float nan = __int_as_float(0x7fffffff), inv = none ? 0.f : 1.f / all_sum16;
        unsigned char *tile_out = stages, *tile_rest = stages + AT_ROWS * CP * 2;
#pragma unroll
        for (int cc = 0; cc < CP / G; cc += 32) {
          const int c = grp * (CP / G) + cc;
          float r[32] = {};
#pragma unroll
          for (int g = 0; g < G; ++g) {
            // a group without a stage in this pass has no result
            if ((g / 2 + F::PAIRS - (stage0 % F::PAIRS)) % F::PAIRS < each && ok) {
              float o[32];
              t5_ld32(t_o + g * CP + lane_base + c, o);
              t5_wait_ld32(o);
#pragma unroll
              for (int i = 0; i < 32; ++i) r[i] = fmaf(o[i], part[g], r[i]);
            }
          }
          if (a.splits > 1) {
            if (mine && row < tile.t1) {
              float *dst = a.parts + ((row * p.heads + head) * a.splits + blockIdx.z) * (p.channels + 2);
              if (c == 0) {
                dst[0] = ok ? all_top : nan;
                dst[1] = all_sum16;
              }
#pragma unroll
              for (int i = 0; i < 32; ++i)
                if (c + i < p.channels) dst[2 + c + i] = ok ? r[i] : nan;
            }
            continue;
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 out, low;
            uint32_t *po = reinterpret_cast<uint32_t *>(&out), *pl = reinterpret_cast<uint32_t *>(&low);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float x0 = !ok ? nan : none ? 0.f : r[i + 2 * e] * inv;
              const float x1 = !ok ? nan : none ? 0.f : r[i + 2 * e + 1] * inv;
              po[e] = A::pack(x0, x1);
              const T *h = reinterpret_cast<const T *>(&po[e]);
              pl[e] = A::pack(x0 - at_float(h[0]), x1 - at_float(h[1]));
            }
            at_put<CP>(tile_out, lrow, (c + i) / 8, out);
            if (rest) at_put<CP>(tile_rest, lrow, (c + i) / 8, low);
          }
        }
        if (a.lse && mine && row < tile.t1 && grp == 0)
          a.lse[(int64_t)head * p.m + row] = none ? pos_inf<float>() : all_top + log2f(all_sum);
        asm volatile("bar.sync 1, %0;" ::"n"(F::EL_THREADS) : "memory");
        const int64_t stride = (int64_t)p.heads * p.channels;
        if (a.splits == 1)
          at_write_rows<T, CP>(tile_out, shared_tile, tile, pass, (T *)a.out + (int64_t)head * p.channels, stride,
                               p.channels, tid, F::EL_THREADS);
        if (rest)
          at_write_rows<T, CP>(tile_rest, shared_tile, tile, pass, rest + (int64_t)head * p.channels, stride, p.channels,
                               tid, F::EL_THREADS);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");  // the ring takes copies again
      }
    }
    stage0 += stages_now;
    if (count > 0) ++passes;
    t5_fence_before();
    __syncthreads();
    t5_fence_after();
    if (*failed) break;
    if (!by_example) {
      if (!mixed || !*(volatile int *)&bad_s) break;
      by_example = true;
    }
    if (!tile.next(next_row, pass)) break;
    if (a.splits > 1) {
      if (pass.c_lo < share_s[0]) pass.c_lo = share_s[0];
      if (pass.c_hi > share_s[1]) pass.c_hi = share_s[1];
      if (pass.c_hi < pass.c_lo) pass.c_hi = pass.c_lo;
    }
  }
  if (*failed && element && grp == 0 && row < tile.t1 && a.splits > 1) {
    a.parts[((row * p.heads + head) * a.splits + blockIdx.z) * (p.channels + 2) + 1] = __int_as_float(0x7fffffff);
  } else if (*failed && element && grp == 0 && row < tile.t1) {
    // a wait ran out: nothing of this block is to be trusted
    const float nan = __int_as_float(0x7fffffff);
    const int64_t at = (row * p.heads + head) * p.channels;
    for (int c = 0; c < p.channels; ++c) {
      ((T *)a.out)[at + c] = at_round<T>(nan);
      if (rest) rest[at + c] = at_round<T>(nan);
    }
    if (a.lse) a.lse[(int64_t)head * p.m + row] = nan;
  }
  if (*failed && tid == 0) t5_report(a.report);
  if (*failed && warp == COPY) {
    at_drain(&q_full, 1, 1);
    at_drain(full, F::STAGES, issued);
  }
  if (*failed && (warp == SCORE || warp == SUM)) {
    uint64_t *bar = &drained[warp == SUM];
    if (t5_elect()) t5_commit(bar);
    __syncwarp();
    at_drain(bar, 1, 1);
  }
  __syncthreads();
  if (warp == COPY) t5_dealloc(tmem, F::TMEM);
}

}  // namespace b200c
