// Backward attention on the tensor cores (see attention_tensor.cuh): KV = false sums dq of 128 queries of a head
// over the keys, KV = true sums dk and dv of 128 keys of a group over the queries of all its heads.
//
// Forming the scores once per direction costs two products more than one kernel for both would, which the tensor
// cores have to spare here; in return no sum is shared between blocks, so there are no atomics.  The statistics of the
// softmax are known, so the groups' steps need nothing of one another and share one accumulator.
// P and dS enter the second products in the 16-bit type.  dq takes dS in two parts, rounded and what rounding left,
// because the rows of dS sum to zero and a rounded one does not: dq's error was 1.5 times that of its own rounding, now
// it is that (for dk and dv, 1.4 times, tensor memory has no room left).  In fp16, whose range is small, P is kept
// times 2^12 and dS times a power of two of its example (at_sigma); both are taken out of the fp32 sums.  What vanishes
// there is below 2^-37 as a weight, and below 2^-39 of the largest value that dS can have in its example.
#pragma once

#include "attention_tensor.cuh"

namespace b200c {

template <int CP, bool KV>
struct AtBackward {
  // groups and resident blocks per SM, as tensor memory allows: 16 warps per SM, 8 where two results of 128 channels
  // fill it
  static constexpr int BLOCKS = CP == 64 && !KV ? 2 : 1;
  static constexpr int G = CP == 64 && !KV ? 2 : CP == 128 && KV ? 2 : 4;
  static constexpr int EL_WARPS = 4 * G, EL_THREADS = 32 * EL_WARPS;
  static constexpr int THREADS = EL_THREADS + 96;
  static constexpr int STAGES = BLOCKS == 2 ? 3 : 4;
  static constexpr int ROW_BYTES = AT_ROWS * CP * 2, TILE_BYTES = AT_COLS * CP * 2;
  static constexpr int STAGE_BYTES = 2 * TILE_BYTES;
  static constexpr int SIDE_FLOATS = (AT_MAX_DIMS + 2) * AT_COLS;  // coordinates, lse, D of a stage's columns
  static constexpr int SMEM = 2 * ROW_BYTES + STAGES * (STAGE_BYTES + SIDE_FLOATS * 4) + 1024;
  static constexpr int W_COLS = AT_SUB;  // a group's dS and P, or dS in two parts
  static constexpr int PAIRS = G / 2, PAIR_COLS = 2 * AT_COLS + 2 * W_COLS;  // S, dP of a stage, two groups' weights
  static constexpr int TMEM = BLOCKS == 2 ? 256 : 512;
  static_assert(STAGES * STAGE_BYTES >= 2 * ROW_BYTES, "the ring takes the block's rows");
  static_assert(PAIRS * PAIR_COLS + (KV ? 2 : 1) * CP <= TMEM, "tensor memory");
  static_assert(BLOCKS * (SMEM + 1024) <= 228 * 1024, "shared memory");
};

struct AtBackwardMaps {
  CUtensorMap row0, row1, col0, col1;  // q, do, k, v or k, v, q, do
};

template <typename T, int CP, int DIM, bool CAP, bool KV>
__global__ void __launch_bounds__(AtBackward<CP, KV>::THREADS, AtBackward<CP, KV>::BLOCKS)
attention_backward_kernel(const __grid_constant__ AtBackwardMaps maps, const __grid_constant__ AttnArgs a,
                          const float *__restrict__ norms) {
  using F = AtBackward<CP, KV>;
  using A = AtType<T>;
  constexpr int ATOMS = CP / 64, G = F::G, COPY = F::EL_WARPS, SCORE = F::EL_WARPS + 1, SUM = F::EL_WARPS + 2;
  extern __shared__ unsigned char at_raw[];
  unsigned char *smem = at_raw + ((1024u - (t5_smem(at_raw) & 1023u)) & 1023u);
  unsigned char *rows0 = smem, *rows1 = smem + F::ROW_BYTES, *stages = smem + 2 * F::ROW_BYTES;
  float *side = reinterpret_cast<float *>(stages + F::STAGES * F::STAGE_BYTES);
  // s_full / s_free: a pair's scores are in / have been read; w_ready: a group's weights are in; a_done: their product
  // is
  __shared__ __align__(8) uint64_t r_full, full[F::STAGES], empty[F::STAGES], s_full[F::PAIRS], s_free[F::PAIRS],
      w_ready[G], a_done[G], done, drained[2];
  __shared__ uint32_t tmem_s;
  __shared__ int failed_s, bad_s;
  __shared__ AtTileShared shared_tile;
  volatile int *failed = &failed_s;

  const b200c_attention_t &p = a.p;
  const int tid = threadIdx.x, warp = t5_warp(), lane = tid & 31;
  const int per_group = p.heads / p.groups;
  const int per_tile = KV ? p.groups : p.heads, which = (int)(blockIdx.x % (unsigned)per_tile);
  const int head0 = KV ? which * per_group : which;
  const int group = KV ? which : head0 / per_group;
  const int heads = KV ? per_group : 1;  // heads whose columns are walked
  AtTile tile;
  if (KV)
    tile.init(at_tile_of(a.order, per_tile) * AT_ROWS, p.ptr_k, p.ptr_q, p.n, p.m, p.num_segments);
  else
    tile.init(at_tile_of(a.order, per_tile) * AT_ROWS, p.ptr_q, p.ptr_k, p.m, p.n, p.num_segments);

  // element threads: a row each
  const bool element = warp < F::EL_WARPS;
  const int grp = warp >> 2, lrow = tid & (AT_ROWS - 1);
  const int64_t row = tile.t0 + lrow;
  float pos[DIM == 0 ? 1 : DIM], lse = 0.f, delta = 0.f;
  if constexpr (DIM > 0) {
    const float *src = KV ? p.pos_k : p.pos_q;
#pragma unroll
    for (int d = 0; d < DIM; ++d) pos[d] = element && row < tile.t1 && d < p.dims ? src[row * p.dims + d] : 0.f;
  }
  if (!KV && element && row < tile.t1) {
    lse = a.lse[(int64_t)head0 * p.m + row] - A::SHIFT;
    delta = a.delta[(int64_t)head0 * p.m + row];
  }

  if (tid == 64) {
    t5_mbar_init(&r_full, 1);
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
  const uint32_t t_acc = tmem + F::PAIRS * F::PAIR_COLS;  // dq, or dv and dk side by side
  if (warp == COPY && lane == 0) {
    t5_mbar_expect(&r_full, 2 * F::ROW_BYTES);
    for (int at = 0; at < ATOMS; ++at) {
      t5_tma_3d(rows0 + at * (AT_ROWS * 128), &maps.row0, at * 64, KV ? group : head0, (int)tile.t0, &r_full);
      t5_tma_3d(rows1 + at * (AT_ROWS * 128), &maps.row1, at * 64, KV ? group : head0, (int)tile.t0, &r_full);
    }
    t5_mbar_arrive(&r_full);
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
  const float sigma = at_sigma<T>(norms, p.groups, row_segment, group);  // of the row
  const float sig = A::BF16 ? 1.f : sigma * (1.f / 4096.f);  // P carries 2^SHIFT already

  bool by_example = false;
  int64_t next_row = tile.t0;
  AtPass pass = tile.all(shared_tile);
  const bool mixed = tile.b_first != tile.b_last;
  uint32_t stage0 = 0, passes = 0, issued = 0;
  bool ok = true;
  if (warp == SCORE) ok = t5_mbar_wait_warp(&r_full, 0, failed);

  for (;;) {
    const int64_t count = pass.c_hi - pass.c_lo;
    const uint32_t each = at_stages(count), stages_now = each * heads;
    if (warp == COPY) {
      // ---- copies
      AtRing<F::STAGES> ring(stage0);
      uint32_t e = 0, c = 0;
      for (uint32_t g = stage0; g < stage0 + stages_now && ok; ++g, ring.next()) {
        const uint32_t st = ring.st;
        const int64_t c0 = pass.c_lo + (int64_t)c * AT_COLS;
        const int head = KV ? head0 + (int)e : group;
        // what the columns bring beside the operands is on its way while the stage is waited for
        float place[DIM == 0 ? 1 : 2 * DIM], col_lse[2], col_delta[2];
        at_fetch_places<DIM>(place, KV ? p.pos_q : p.pos_k, p.dims, c0, pass.c_hi, lane);
        if constexpr (KV) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            const bool there = c0 + n * 32 + lane < pass.c_hi;
            const int64_t at = (int64_t)head * p.m + c0 + n * 32 + lane;
            col_lse[n] = there ? a.lse[at] - A::SHIFT : pos_inf<float>();
            col_delta[n] = there ? a.delta[at] : 0.f;
          }
        }
        // the stage's round before this one is through
        if (g >= F::STAGES) ok = t5_mbar_wait_idle(&empty[st], ring.parity ^ 1u, failed);
        if (!ok) break;
        unsigned char *dst = stages + st * F::STAGE_BYTES;
        if (lane == 0) {
          t5_mbar_expect(&full[st], F::STAGE_BYTES);
          for (int at = 0; at < ATOMS; ++at) {
            t5_tma_3d(dst + at * (AT_COLS * 128), &maps.col0, at * 64, head, (int)c0, &full[st]);
            t5_tma_3d(dst + F::TILE_BYTES + at * (AT_COLS * 128), &maps.col1, at * 64, head, (int)c0, &full[st]);
          }
        }
        float *sd = side + st * F::SIDE_FLOATS;
        at_put_places<DIM>(sd, place, lane);
        if constexpr (KV) {
#pragma unroll
          for (int n = 0; n < 2; ++n) {
            sd[AT_MAX_DIMS * AT_COLS + n * 32 + lane] = col_lse[n];
            sd[(AT_MAX_DIMS + 1) * AT_COLS + n * 32 + lane] = col_delta[n];
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
    } else if (warp == SCORE) {
      // ---- scores
      const uint32_t id = t5_idesc(A::BF16, AT_COLS, false);
      const uint64_t d_r0 = t5_desc(t5_smem(rows0)), d_r1 = t5_desc(t5_smem(rows1)), d_c0 = t5_desc(t5_smem(stages)),
                     d_c1 = t5_desc(t5_smem(stages + F::TILE_BYTES));
      AtRing<F::STAGES> ring(stage0);
      for (uint32_t g = stage0; g < stage0 + stages_now && ok; ++g, ring.next()) {
        const uint32_t pair = g % F::PAIRS, k = g / F::PAIRS;
        ok = t5_mbar_wait_idle(&full[ring.st], ring.parity, failed);
        if (ok && k > 0) ok = t5_mbar_wait_idle(&s_free[pair], (k - 1) & 1, failed);
        if (!ok) break;
        t5_fence_after();
        const uint32_t off = ring.st * (F::STAGE_BYTES / 16), t_s = tmem + pair * F::PAIR_COLS;
        if (t5_elect()) {
#pragma unroll
          for (int ks = 0; ks < CP / 16; ++ks)
            t5_mma_ss(t_s, d_r0 + ((ks >> 2) * (AT_ROWS * 128) + (ks & 3) * 32) / 16,
                      d_c0 + off + ((ks >> 2) * (AT_COLS * 128) + (ks & 3) * 32) / 16, id, ks > 0);
#pragma unroll
          for (int ks = 0; ks < CP / 16; ++ks)
            t5_mma_ss(t_s + AT_COLS, d_r1 + ((ks >> 2) * (AT_ROWS * 128) + (ks & 3) * 32) / 16,
                      d_c1 + off + ((ks >> 2) * (AT_COLS * 128) + (ks & 3) * 32) / 16, id, ks > 0);
          t5_commit(&s_full[pair]);
        }
        __syncwarp();
      }
    } else if (warp == SUM) {
      // ---- products with the weights
      const uint32_t id = t5_idesc(A::BF16, CP, true);
      const uint64_t d_c0 = t5_desc(t5_smem(stages), AT_COLS * 128),
                     d_c1 = t5_desc(t5_smem(stages + F::TILE_BYTES), AT_COLS * 128);
      AtRing<F::STAGES> ring(stage0);
      for (uint32_t g = stage0; g < stage0 + stages_now && ok; ++g, ring.next()) {
        const uint32_t pair = g % F::PAIRS, k = g / F::PAIRS;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t gr = 2 * pair + h;
          if (ok) ok = t5_mbar_wait_idle(&w_ready[gr], k & 1, failed);
          if (!ok) break;
          t5_fence_after();
          const uint32_t off = ring.st * (F::STAGE_BYTES / 16) + h * (AT_SUB * 128 / 16);
          const uint32_t w = tmem + pair * F::PAIR_COLS + 2 * AT_COLS + h * F::W_COLS;
          const bool more = g != stage0 || h > 0;
          if (t5_elect()) {
#pragma unroll
            for (int ks = 0; ks < AT_SUB / 16; ++ks) {
              t5_mma_ts(t_acc + (KV ? CP : 0), w + ks * 8, d_c0 + off + ks * (2048 / 16), id, more || ks > 0);
              if constexpr (KV)
                t5_mma_ts(t_acc, w + AT_SUB / 2 + ks * 8, d_c1 + off + ks * (2048 / 16), id, more || ks > 0);
              else
                t5_mma_ts(t_acc, w + AT_SUB / 2 + ks * 8, d_c0 + off + ks * (2048 / 16), id, true);
            }
            t5_commit(&a_done[gr]);
            if (h == 1) t5_commit(&empty[ring.st]);
            if (h == 1 && g + 1 == stage0 + stages_now) t5_commit(&done);
          }
          __syncwarp();
        }
      }
    } else {
      // ---- elements
      const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16;
      const uint32_t pair = grp >> 1, half = grp & 1, t_pair = tmem + pair * F::PAIR_COLS + lane_base;
      const uint32_t t_s = t_pair + half * AT_SUB, t_w = t_pair + 2 * AT_COLS + half * F::W_COLS;
      const bool mine = pass.segment < 0 || pass.segment == row_segment;
      const AtSeen seen(row_lo, row_hi, pass, mine);
      const bool scan = mixed && !by_example;
      uint32_t bad = 0u;
      uint32_t e = 0, c = (pair + F::PAIRS - stage0 % F::PAIRS) % F::PAIRS;  // the pair's first stage
      for (uint32_t g = stage0 + c; g < stage0 + stages_now && ok; g += F::PAIRS, c += F::PAIRS) {
        while (c >= each) {
          c -= each;
          ++e;
        }
        const uint32_t st = g % F::STAGES, k = g / F::PAIRS;
        const int base = (int)(c * AT_COLS + half * AT_SUB);
        const bool tail = base + AT_SUB > (int)count;
        unsigned char *stage = stages + st * F::STAGE_BYTES + half * (AT_SUB * 128);
        const float *sd = side + st * F::SIDE_FLOATS + half * AT_SUB;
        float slope2 = 0.f;
        if constexpr (DIM > 0) slope2 = __ldg(p.slope + head0 + e) * AT_LOG2E;
        // the scores in, and what came with the columns
        ok = t5_mbar_wait_both(&s_full[pair], k & 1, &full[st], (g / F::STAGES) & 1, true, failed);
        if (!ok) break;
        if (scan) {
          bad |= at_scan<T, CP>(stage, lrow);
          if constexpr (KV) bad |= at_scan<T, CP>(stage + F::TILE_BYTES, lrow);
        }
        t5_fence_after();
        uint32_t w[AT_SUB / 2], w2[AT_SUB / 2];  // dS; P, or the rest of dS
        // asked here, answered when the weights are there to be stored
        bool taken = g - stage0 < F::PAIRS || t5_mbar_try(&a_done[grp], (k - 1) & 1);
        if (seen.any(base)) {
          float x[AT_SUB], dp[AT_SUB], u[CAP ? AT_SUB : 1];
          t5_ld32(t_s, x);
          t5_ld32(t_s + AT_COLS, dp);
          t5_wait_ld32(x);
          t5_wait_ld32(dp);
          t5_fence_before();
          __syncwarp();
          if (lane == 0) t5_mbar_arrive(&s_free[pair]);
          at_logits<DIM, CAP, CAP, KV>(x, u, sd, pos, slope2, pre, post, lse, sd + AT_MAX_DIMS * AT_COLS);
#pragma unroll
          for (int j4 = 0; j4 < AT_SUB; j4 += 4) {
            float de[4] = {delta, delta, delta, delta};
            if constexpr (KV) {
              const float4 d4 = *reinterpret_cast<const float4 *>(sd + (AT_MAX_DIMS + 1) * AT_COLS + j4);
              de[0] = d4.x, de[1] = d4.y, de[2] = d4.z, de[3] = d4.w;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
              const float pr = t5_ex2(x[j4 + j]);
              float ds = pr * (dp[j4 + j] - de[j]);
              if constexpr (CAP) ds *= fmaf(-u[j4 + j], u[j4 + j], 1.f);
              if constexpr (!A::BF16) ds *= sig;
              x[j4 + j] = pr;
              dp[j4 + j] = ds;
            }
          }
          if (!seen.all(base)) {
#pragma unroll
            for (int j = 0; j < AT_SUB; ++j)
              if (base + j < seen.lo || base + j >= seen.hi) x[j] = dp[j] = 0.f;
          }
#pragma unroll
          for (int j = 0; j < AT_SUB / 2; ++j) {
            w[j] = A::pack(dp[2 * j], dp[2 * j + 1]);
            if constexpr (KV)
              w2[j] = A::pack(x[2 * j], x[2 * j + 1]);
            else
              w2[j] = A::pack(dp[2 * j] - A::low(w[j]), dp[2 * j + 1] - A::high(w[j]));
          }
        } else {
          if (lane == 0) t5_mbar_arrive(&s_free[pair]);
#pragma unroll
          for (int j = 0; j < AT_SUB / 2; ++j) w[j] = w2[j] = 0u;
        }
        // the weights of the group's step before have been taken
        if (!__all_sync(FULL_MASK, taken)) ok = t5_mbar_wait_warp(&a_done[grp], (k - 1) & 1, failed);
        if (!ok) break;
        t5_fence_after();
        t5_st16(t_w, w);
        t5_st16(t_w + AT_SUB / 2, w2);
        t5_wait_st();
        if (tail) {
          at_clear<CP>(stage, (int)count > base ? (int)count - base : 0, lrow);
          if constexpr (KV) at_clear<CP>(stage + F::TILE_BYTES, (int)count > base ? (int)count - base : 0, lrow);
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
      if (scan) asm volatile("bar.sync 1, %0;" ::"n"(F::EL_THREADS) : "memory");
      if (!(scan && *(volatile int *)&bad_s)) {
        const float nan = __int_as_float(0x7fffffff);
        // the results' channels in chunks of 32, dealt out to the groups
        constexpr int CHUNKS = (KV ? 2 : 1) * CP / 32;
#pragma unroll 1
        for (int ch = grp; ch < CHUNKS; ch += G) {
          const int c = ch * 32 % CP;
          const bool is_dv = KV && ch * 32 < CP;
          const float times = !ok ? nan : is_dv ? (A::BF16 ? 1.f : 1.f / 4096.f) : p.scale / sigma;
          float o[32] = {};
          if (count > 0 && ok) {
            t5_ld32(t_acc + lane_base + ch * 32, o);
            t5_wait_ld32(o);
            // a row that sees no column (of no example, or of one without) shares the pass of its neighbours, where 0
            // times a NaN or an infinity of the columns would stay
            if (row_lo >= row_hi) {
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = 0.f;
            }
          }
#pragma unroll
          for (int i = 0; i < 32; i += 8) {
            uint4 out;
            uint32_t *po = reinterpret_cast<uint32_t *>(&out);
#pragma unroll
            for (int k = 0; k < 4; ++k) po[k] = A::pack(o[i + 2 * k] * times, o[i + 2 * k + 1] * times);
            at_put<CP>(is_dv || !KV ? stages : stages + F::ROW_BYTES, lrow, (c + i) / 8, out);
          }
        }
        asm volatile("bar.sync 1, %0;" ::"n"(F::EL_THREADS) : "memory");
        if constexpr (KV) {
          const int64_t stride = (int64_t)p.groups * p.channels;
          at_write_rows<T, CP>(stages, shared_tile, tile, pass, (T *)a.dv + (int64_t)group * p.channels, stride, p.channels,
                               tid, F::EL_THREADS);
          at_write_rows<T, CP>(stages + F::ROW_BYTES, shared_tile, tile, pass, (T *)a.dk + (int64_t)group * p.channels,
                               stride, p.channels, tid, F::EL_THREADS);
        } else {
          at_write_rows<T, CP>(stages, shared_tile, tile, pass, (T *)a.dq + (int64_t)head0 * p.channels,
                               (int64_t)p.heads * p.channels, p.channels, tid, F::EL_THREADS);
        }
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
  }
  if (*failed && element && row < tile.t1 && grp == 0) {
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
  if (*failed && tid == 0) t5_report(a.report);
  if (*failed && warp == COPY) {
    at_drain(&r_full, 1, 1);
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
