// Attention and its gradients where examples are a few dozen rows (molecules): 16-bit types, up to 32 channels.
//
// The tcgen05 kernels work on 128 rows against 64 columns; with examples of 30 rows three quarters of that is masked.
// Here a warp owns 16 rows and walks the columns of their example 32 at a time with warp-wide products of 16 x 8 x 16,
// so little is padded, and takes several heads one after the other, for which it looks its rows' examples up once.  The
// scheme is that of the tcgen05 kernels:
//   forward: rows = queries, columns = keys;     S = R0 C0^T, O += P C1           (R0 = q; C0, C1 = k, v)
//   dq:      rows = queries, columns = keys;     S = R0 C0^T, dP = R1 C1^T, dq += dS C0   (R = q, do; C = k, v)
//   dk, dv:  rows = keys,    columns = queries;  S = R0 C0^T, dP = R1 C1^T, dv += P C1, dk += dS C0   (R = k, v; C = q, do)
// Operands come by asynchronous 16-byte copies into the warp's own tiles, the next step's while this one is
// worked on; there is no barrier between warps.  16 rows that lie in several examples are taken example by example, and
// only the example's rows are stored, so that a NaN of one never meets another one's zeros; columns past
// the example's end are cleared in shared memory for the same reason.
// Weights are rounded to the type as operands (fp16: times 2^15, see AtType; dS of dq in two parts, see
// attention_backward.cuh); statistics and sums are fp32.
#pragma once

#include "attention_tensor.cuh"
#include "attention_warp.cuh"

namespace b200c {

constexpr int AS_ROWS = 16, AS_COLS = 32, AS_WARPS = 4;
constexpr int AS_HEADS = 4;  // heads (or groups) that a warp takes one after the other

enum AsRole { AS_FORWARD, AS_DQ, AS_DKV };

template <int CP, int DIM, AsRole ROLE>
struct AsTiles {
  static constexpr int ROWS = AS_ROWS * CP * 2, COLS = AS_COLS * CP * 2;
  // coordinates of the columns and, where rows are keys, lse and D
  static constexpr int SIDE = (DIM + (ROLE == AS_DKV ? 2 : 0)) * AS_COLS * 4;
  static constexpr int STAGE = 2 * COLS + SIDE;
  static constexpr int WARP = 2 * 2 * ROWS + 2 * STAGE;  // two sets of both rows' tiles, two stages
  static constexpr int SMEM = AS_WARPS * WARP;
};

// Blocks per SM: shared memory has room for four, which leave 128 registers; dk and dv do not fit in them (2048
// molecules, three blocks -> four: forward 126 -> 117 us, dq 128 -> 122, dk and dv 138 -> 164).
template <int DIM, AsRole ROLE>
constexpr int as_blocks() {
  return ROLE != AS_DKV && DIM <= 3 ? 4 : 3;
}

// [rows, heads, channels] of one operand
struct AsOperand {
  const void *base;
  int64_t row, head;
};

template <typename T, int CP, int DIM, bool CAP, AsRole ROLE>
__global__ void __launch_bounds__(32 * AS_WARPS, (as_blocks<DIM, ROLE>())) attention_short_kernel(const __grid_constant__ AttnArgs a) {
  using S = AsTiles<CP, DIM, ROLE>;
  using A = AtType<T>;
  constexpr bool KV = ROLE == AS_DKV, FORWARD = ROLE == AS_FORWARD;
  constexpr int KT = CP / 16, CT = CP / 8, NT = AS_COLS / 8, CHUNKS = CP / 8;
  extern __shared__ __align__(128) unsigned char as_smem[];
  const b200c_attention_t &p = a.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int gr = lane >> 2, gc = (lane & 3) * 2;  // rows gr, gr + 8 and columns gc, gc + 1 of every 8 are this lane's
  const int per_group = p.heads / p.groups, chunks = p.channels / 8;
  unsigned char *mine = as_smem + warp * S::WARP;
  const uint32_t at_mine = t5_smem(mine);
  AtTile tile;
  const int64_t t0 = ((int64_t)blockIdx.x * AS_WARPS + warp) * AS_ROWS;
  if (KV)
    tile.init(t0, p.ptr_k, p.ptr_q, p.n, p.m, p.num_segments);
  else
    tile.init(t0, p.ptr_q, p.ptr_k, p.m, p.n, p.num_segments);
  if (t0 >= tile.rows) return;
  tile.t1 = t0 + AS_ROWS < tile.rows ? t0 + AS_ROWS : tile.rows;
  const int64_t q_row = (int64_t)p.heads * p.channels;
  const AsOperand q{p.q, p.q_row, p.q_head}, k{p.k, p.k_row, p.k_head}, v{p.v, p.v_row, p.v_head},
      dout{a.dout, q_row, p.channels};
  const AsOperand rows0 = KV ? k : q, rows1 = KV ? v : dout, cols0 = KV ? q : k, cols1 = KV ? dout : v;
  const int units = KV ? p.groups : p.heads;  // what the warp's rows have: groups of k and v, or heads of q
  const int u_lo = blockIdx.y * AS_HEADS, u_hi = u_lo + AS_HEADS < units ? u_lo + AS_HEADS : units;
  const int inner = KV ? per_group : 1;  // heads whose columns are walked per unit
  const float pre = CAP ? 2.f * AT_LOG2E * p.scale / p.cap : p.scale * AT_LOG2E, post = p.cap * AT_LOG2E;

  float pos[2][DIM == 0 ? 1 : DIM];
  if constexpr (DIM > 0) {
    const float *src = KV ? p.pos_k : p.pos_q;
#pragma unroll
    for (int e = 0; e < 2; ++e)
#pragma unroll
      for (int d = 0; d < DIM; ++d)
        pos[e][d] = t0 + gr + 8 * e < tile.t1 && d < p.dims ? src[(t0 + gr + 8 * e) * p.dims + d] : 0.f;
  }

  for (int64_t at = t0; at < tile.t1;) {
    // the rows [at, to) of one example and its columns (none for rows of no example)
    const int b = at_segment_of_warp(tile.ptr_r, tile.segments, at, lane);
    int64_t lo, hi, c_lo = 0, c_hi = 0, to;
    at_segment(tile.ptr_r, tile.rows, b, lo, hi);
    if (at >= lo && at < hi) {
      to = hi;
      at_segment(tile.ptr_c, tile.cols, b, c_lo, c_hi);
    } else {
      to = at < lo ? lo : b == tile.segments - 1 ? tile.t1 : at + 1;
    }
    if (to > tile.t1) to = tile.t1;
    const int64_t count = c_hi - c_lo;
    const int blocks = (int)((count + AS_COLS - 1) / AS_COLS);  // per head

    // copies of step (u, e, j): the unit's rows with its first step, the columns' tiles and what belongs to them.  A
    // lane copies chunk my_c of rows my_r, my_r + PER, ...
    constexpr int PER = 32 / CHUNKS;
    const int my_r = lane / CHUNKS, my_c = lane % CHUNKS;
    const T *r0_at = (const T *)rows0.base + (t0 + my_r) * rows0.row + my_c * 8;
    const T *r1_at = (const T *)rows1.base + (t0 + my_r) * rows1.row + my_c * 8;
    const T *c0_at = (const T *)cols0.base + (c_lo + my_r) * cols0.row + my_c * 8;
    const T *c1_at = (const T *)cols1.base + (c_lo + my_r) * cols1.row + my_c * 8;
    const int my_rows = my_c < chunks ? (int)(tile.t1 - t0) - my_r : 0;  // this lane's rows lie below that
    auto copy = [&](uint32_t dst, const T *src, bool there) {  // nothing is read where there is nothing: zeros are written
      asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(dst), "l"(there ? src : (const T *)cols0.base),
                   "r"(there ? 16u : 0u)
                   : "memory");
    };
    auto fetch = [&](int u, int e, int64_t j, int stage) {
      if (u < u_hi) {
        const int head = KV ? u * per_group + e : u, col_head = KV ? head : u / per_group;
        if (e == 0 && j == 0) {
          const uint32_t dst = at_mine + (u & 1) * (2 * S::ROWS);
          const T *s0 = r0_at + u * rows0.head, *s1 = r1_at + u * rows1.head;
#pragma unroll
          for (int n = 0; n < AS_ROWS / PER; ++n) {
            const uint32_t off = aw_at<CP>(n * PER + my_r, my_c);
            copy(dst + off, s0 + n * PER * rows0.row, n * PER < my_rows);
            if (!FORWARD) copy(dst + S::ROWS + off, s1 + n * PER * rows1.row, n * PER < my_rows);
          }
        }
        const int64_t j0 = c_lo + j * AS_COLS;
        const int my_cols = my_c < chunks ? (int)(c_hi - j0 < AS_COLS ? c_hi - j0 : AS_COLS) - my_r : 0;
        unsigned char *st = mine + 4 * S::ROWS + stage * S::STAGE;
        const uint32_t at_st = at_mine + 4 * S::ROWS + stage * S::STAGE;
        const T *s0 = c0_at + j * AS_COLS * cols0.row + col_head * cols0.head;
        const T *s1 = c1_at + j * AS_COLS * cols1.row + col_head * cols1.head;
#pragma unroll
        for (int n = 0; n < AS_COLS / PER; ++n) {
          const uint32_t off = aw_at<CP>(n * PER + my_r, my_c);
          copy(at_st + off, s0 + n * PER * cols0.row, n * PER < my_cols);
          copy(at_st + S::COLS + off, s1 + n * PER * cols1.row, n * PER < my_cols);
        }
        float *side = reinterpret_cast<float *>(st + 2 * S::COLS);
        if constexpr (DIM > 0) {
          const float *src = KV ? p.pos_q : p.pos_k;
#pragma unroll
          for (int n = 0; n < DIM; ++n) {  // [dims][32 columns]
            const int i = n * 32 + lane, c = i / DIM, d = i - c * DIM;
            if (j0 + c < c_hi && d < p.dims)
              cp_async_4(side + d * AS_COLS + c, src + (j0 + c) * p.dims + d);
            else
              side[d * AS_COLS + c] = 0.f;
          }
        }
        if constexpr (KV) {
          float *stat = side + DIM * AS_COLS;
          const int64_t col = (int64_t)head * p.m + j0 + lane;
          if (j0 + lane < c_hi) {
            cp_async_4(stat + lane, a.lse + col);
            cp_async_4(stat + AS_COLS + lane, a.delta + col);
          } else {
            stat[lane] = pos_inf<float>();
            stat[AS_COLS + lane] = 0.f;
          }
        }
      }
      cp_async_commit();
    };

    int stage = 0;
    if (blocks > 0) fetch(u_lo, 0, 0, 0);
    // a lane finds one unit's power of two while that is on its way
    float sigmas = 1.f;
    if (!FORWARD && u_lo + (lane & (AS_HEADS - 1)) < u_hi)
      sigmas = at_sigma<T>(a.norms, p.groups, b, (u_lo + (lane & (AS_HEADS - 1))) / (KV ? 1 : per_group));
    for (int u = u_lo; u < u_hi; ++u) {
      const int head0 = KV ? u * per_group : u;
      const float sigma = FORWARD || A::BF16 ? 1.f : __shfl_sync(FULL_MASK, sigmas, u - u_lo);
      const float sig = A::BF16 ? 1.f : sigma * (1.f / 4096.f);  // P carries 2^SHIFT already
      float top[2] = {-pos_inf<float>(), -pos_inf<float>()}, sum[2] = {}, lse[2] = {}, delta[2] = {};
      float acc[CT][4] = {}, acc2[KV ? CT : 1][4] = {};
      if constexpr (ROLE == AS_DQ) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int64_t row = t0 + gr + 8 * e;
          lse[e] = row < tile.t1 ? a.lse[(int64_t)head0 * p.m + row] - A::SHIFT : pos_inf<float>();
          delta[e] = row < tile.t1 ? a.delta[(int64_t)head0 * p.m + row] : 0.f;
        }
      }
      const uint32_t at_rows = at_mine + (u & 1) * (2 * S::ROWS);
      uint32_t r0[KT][4], r1[FORWARD ? 1 : KT][4];
      for (int e = 0; e < inner && blocks > 0; ++e) {
        const float slope2 = DIM > 0 ? p.slope[head0 + e] * AT_LOG2E : 0.f;
        for (int j = 0; j < blocks; ++j, stage ^= 1) {
          // the next step's copies, then this step's have landed
          if (j + 1 < blocks)
            fetch(u, e, j + 1, stage ^ 1);
          else if (e + 1 < inner)
            fetch(u, e + 1, 0, stage ^ 1);
          else
            fetch(u + 1, 0, 0, stage ^ 1);
          cp_async_wait<1>();
          __syncwarp();
          if (e == 0 && j == 0) {
#pragma unroll
            for (int t = 0; t < KT; ++t) {
              aw_rows<CP>(r0[t], at_rows, t, lane);
              if constexpr (!FORWARD) aw_rows<CP>(r1[t], at_rows + S::ROWS, t, lane);
            }
          }
          const uint32_t st = at_mine + 4 * S::ROWS + stage * S::STAGE;
          const float *side = reinterpret_cast<const float *>(mine + 4 * S::ROWS + stage * S::STAGE + 2 * S::COLS) + gc;
          const float *stat = side + DIM * AS_COLS;
          const int left = (int)(count - (int64_t)j * AS_COLS < AS_COLS ? count - (int64_t)j * AS_COLS : AS_COLS);
          float s[NT][4] = {}, dp[FORWARD ? 1 : NT][4] = {};
#pragma unroll
          for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int n = 0; n < NT; n += 2) {
              uint32_t f[4];
              aw_cols<CP>(f, st, n, t, lane);
              aw_mma<T>(s[n], r0[t], f[0], f[1]);
              aw_mma<T>(s[n + 1], r0[t], f[2], f[3]);
              if constexpr (!FORWARD) {
                aw_cols<CP>(f, st + S::COLS, n, t, lane);
                aw_mma<T>(dp[n], r1[t], f[0], f[1]);
                aw_mma<T>(dp[n + 1], r1[t], f[2], f[3]);
              }
            }
          // scores in units of log 2; backward: P (times 2^SHIFT) and dS in their place
#pragma unroll
          for (int n = 0; n < NT; ++n)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                float t, w = 0.f;
                if constexpr (CAP) {
                  w = fmaf(-2.f, t5_rcp(t5_ex2(s[n][2 * h + c] * pre) + 1.f), 1.f);
                  t = w * post;
                } else {
                  t = s[n][2 * h + c] * pre;
                }
                if constexpr (DIM > 0) {
                  float d2 = 0.f;
#pragma unroll
                  for (int d = 0; d < DIM; ++d) {
                    const float df = pos[h][d] - side[d * AS_COLS + n * 8 + c];
                    d2 = DIM == 1 ? fabsf(df) : fmaf(df, df, d2);
                  }
                  t = fmaf(-slope2, DIM == 1 ? d2 : t5_sqrt(d2), t);
                }
                const bool there = n * 8 + gc + c < left;
                if constexpr (FORWARD) {
                  s[n][2 * h + c] = there ? t : -pos_inf<float>();
                } else {
                  const float l = KV ? stat[n * 8 + c] - A::SHIFT : lse[h];
                  const float de = KV ? stat[AS_COLS + n * 8 + c] : delta[h];
                  const float pr = t5_ex2(t - l);
                  float ds = pr * (dp[n][2 * h + c] - de);
                  if constexpr (CAP) ds *= fmaf(-w, w, 1.f);
                  if constexpr (!A::BF16) ds *= sig;
                  s[n][2 * h + c] = there ? pr : 0.f;
                  dp[n][2 * h + c] = there ? ds : 0.f;
                }
              }
          if constexpr (FORWARD) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              float m = -pos_inf<float>();
#pragma unroll
              for (int n = 0; n < NT; ++n) m = fmaxf(m, fmaxf(s[n][2 * h], s[n][2 * h + 1]));
              m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, 1));
              m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, 2));
              m = fmaxf(top[h], m - A::TOP);  // what the weights are relative to
              const float sub = m == -pos_inf<float>() ? 0.f : m, shrink = t5_ex2(top[h] - sub);
              top[h] = m;
              float part = 0.f;
#pragma unroll
              for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                  s[n][2 * h + c] = t5_ex2(s[n][2 * h + c] - sub);
                  part += s[n][2 * h + c];
                }
              sum[h] = fmaf(sum[h], shrink, part);
#pragma unroll
              for (int n = 0; n < CT; ++n) {
                acc[n][2 * h] *= shrink;
                acc[n][2 * h + 1] *= shrink;
              }
            }
          }
          // products with the weights, 16 columns at a time
#pragma unroll
          for (int t = 0; t < NT / 2; ++t) {
            uint32_t w[4], w2[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const int n = 2 * t + (i >> 1), h = i & 1;
              if constexpr (FORWARD) {
                w[i] = aw_pack<T>(s[n][2 * h], s[n][2 * h + 1]);
              } else {
                w[i] = aw_pack<T>(dp[n][2 * h], dp[n][2 * h + 1]);
                const float2 back = aw_unpack<T>(w[i]);
                w2[i] = KV ? aw_pack<T>(s[n][2 * h], s[n][2 * h + 1])
                           : aw_pack<T>(dp[n][2 * h] - back.x, dp[n][2 * h + 1] - back.y);
              }
            }
#pragma unroll
            for (int n = 0; n < CT; n += 2) {
              uint32_t f[4];
              aw_sums<CP>(f, st + (FORWARD ? S::COLS : 0), t, n, lane);
              aw_mma<T>(acc[n], w, f[0], f[1]);
              aw_mma<T>(acc[n + 1], w, f[2], f[3]);
              if constexpr (ROLE == AS_DQ) {
                aw_mma<T>(acc[n], w2, f[0], f[1]);
                aw_mma<T>(acc[n + 1], w2, f[2], f[3]);
              }
              if constexpr (KV) {
                aw_sums<CP>(f, st + S::COLS, t, n, lane);
                aw_mma<T>(acc2[n], w2, f[0], f[1]);
                aw_mma<T>(acc2[n + 1], w2, f[2], f[3]);
              }
            }
          }
          __syncwarp();  // the stage has been read
        }
      }
      // the example's rows of this unit: over the rows' tiles, which have been read, and out in 16-byte pieces
      float times[2] = {p.scale / sigma, p.scale / sigma};
      if constexpr (FORWARD) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          sum[h] += __shfl_xor_sync(FULL_MASK, sum[h], 1);
          sum[h] += __shfl_xor_sync(FULL_MASK, sum[h], 2);
          times[h] = sum[h] == 0.f ? 0.f : 1.f / sum[h];
          const int64_t row = t0 + gr + 8 * h;
          if (a.lse && (lane & 3) == 0 && row >= at && row < to)
            a.lse[(int64_t)u * p.m + row] = sum[h] == 0.f ? pos_inf<float>() : top[h] + log2f(sum[h]);
        }
      }
      unsigned char *out0 = mine + (u & 1) * (2 * S::ROWS), *out1 = out0 + S::ROWS;
#pragma unroll
      for (int n = 0; n < CT; ++n)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint32_t off = aw_at<CP>(gr + 8 * h, n) + gc * 2;
          const bool none = FORWARD && sum[h] == 0.f;
          const float x = none ? 0.f : acc[n][2 * h] * times[h], y = none ? 0.f : acc[n][2 * h + 1] * times[h];
          const uint32_t w = aw_pack<T>(x, y);
          *reinterpret_cast<uint32_t *>(out0 + off) = w;
          if constexpr (FORWARD) {
            const float2 back = aw_unpack<T>(w);
            *reinterpret_cast<uint32_t *>(out1 + off) = aw_pack<T>(x - back.x, y - back.y);
          } else if constexpr (KV) {
            const float down = A::BF16 ? 1.f : 1.f / 4096.f;
            *reinterpret_cast<uint32_t *>(out1 + off) = aw_pack<T>(acc2[n][2 * h] * down, acc2[n][2 * h + 1] * down);
          }
        }
      __syncwarp();
      T *dst0 = (T *)(FORWARD ? a.out : KV ? a.dk : a.dq), *dst1 = (T *)(FORWARD ? a.rest : KV ? a.dv : nullptr);
      const int64_t stride = (int64_t)units * p.channels;
      for (int i = lane; i < AS_ROWS * CHUNKS; i += 32) {
        const int r = i / CHUNKS, c = i % CHUNKS;
        if (t0 + r < at || t0 + r >= to || c >= chunks) continue;
        const int64_t where = (t0 + r) * stride + u * p.channels + c * 8;
        *reinterpret_cast<uint4 *>(dst0 + where) = *reinterpret_cast<const uint4 *>(out0 + aw_at<CP>(r, c));
        if (dst1) *reinterpret_cast<uint4 *>(dst1 + where) = *reinterpret_cast<const uint4 *>(out1 + aw_at<CP>(r, c));
      }
      __syncwarp();  // the tiles take the rows of the unit after the next
    }
    cp_async_wait<0>();
    __syncwarp();
    at = to;
  }
}

template <typename T, int CP, int DIM, bool CAP, AsRole ROLE>
static int as_launch(const AttnArgs &a) {
  using S = AsTiles<CP, DIM, ROLE>;
  static unsigned long long configured = 0ull;
  B200C_CUDA(opt_in_shared_memory(attention_short_kernel<T, CP, DIM, CAP, ROLE>, S::SMEM, configured));
  const int64_t rows = ROLE == AS_DKV ? a.p.n : a.p.m;
  const int units = ROLE == AS_DKV ? a.p.groups : a.p.heads;
  constexpr int SHARE = AS_ROWS * AS_WARPS;
  const dim3 grid((unsigned)((rows + SHARE - 1) / SHARE), (unsigned)((units + AS_HEADS - 1) / AS_HEADS));
  attention_short_kernel<T, CP, DIM, CAP, ROLE><<<grid, 32 * AS_WARPS, S::SMEM, a.stream>>>(a);
  B200C_LAUNCH_CHECK("attention_short_kernel");
  return B200C_OK;
}
template <typename T, int CP, bool CAP, AsRole ROLE>
static int as_dims(const AttnArgs &a) {
  if (a.p.dims == 0) return as_launch<T, CP, 0, CAP, ROLE>(a);
  if (a.p.dims == 1) return as_launch<T, CP, 1, CAP, ROLE>(a);
  if (a.p.dims <= 3) return as_launch<T, CP, 3, CAP, ROLE>(a);
  return as_launch<T, CP, 8, CAP, ROLE>(a);
}
template <typename T, AsRole ROLE>
static int as_dispatch(const AttnArgs &a) {
  return a.p.cap > 0.f ? as_dims<T, 32, true, ROLE>(a) : as_dims<T, 32, false, ROLE>(a);
}

}  // namespace b200c
