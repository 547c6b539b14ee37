// Attention of a few queries per example over many keys (see attention.cuh for the formulas): pooling by a learned
// query, or one new token over a long memory.  Every key and value is read once for all query heads that share it,
// so memory bandwidth bounds it while a group serves few heads.
//
// A block owns one (example, key/value head, split of the example's keys) and takes up to QB rows (query, head of the
// group) at a time.  LPK lanes share a key, 16 bytes of its channels each; the lane groups of the block walk the
// split's keys in turn, U keys ahead of their use, each with a running maximum, sum and result of its own, which are
// joined by shuffles and through shared memory at the end.  The splits' parts go to the workspace in fp32 and a second
// kernel joins them, in ascending order of the splits.
#include "attention_tensor.cuh"
#include "attention_warp.cuh"

namespace b200c {

constexpr int AF_THREADS = 128;
constexpr int AF_WARPS = AF_THREADS / 32;

template <typename T>
struct AfVec {
  static constexpr int N = 16 / (int)sizeof(T);
};

template <typename T>
__device__ __forceinline__ void af_widen(const uint4 &raw, float (&f)[AfVec<T>::N]) {
  if constexpr (sizeof(T) == 4) {
    f[0] = __uint_as_float(raw.x);
    f[1] = __uint_as_float(raw.y);
    f[2] = __uint_as_float(raw.z);
    f[3] = __uint_as_float(raw.w);
  } else {
    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __nv_bfloat16>::value) {
        f[2 * i] = __uint_as_float(w[i] << 16);
        f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
      } else {
        const float2 t = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
        f[2 * i] = t.x;
        f[2 * i + 1] = t.y;
      }
    }
  }
}

// 16 bytes of channels from p; element by element, zeros past `left` channels, where rows are not 16-byte aligned
template <typename T>
__device__ __forceinline__ uint4 af_load(const T *p, bool vec, int left) {
  if (left <= 0) return make_uint4(0u, 0u, 0u, 0u);
  if (vec) return __ldg(reinterpret_cast<const uint4 *>(p));
  __align__(16) T tmp[AfVec<T>::N];
#pragma unroll
  for (int i = 0; i < AfVec<T>::N; ++i) tmp[i] = i < left ? p[i] : at_round<T>(0.f);
  return *reinterpret_cast<const uint4 *>(tmp);
}

template <typename T, int LPK, int QB>
__global__ void __launch_bounds__(AF_THREADS) attention_few_kernel(AttnArgs a, int splits, int vec,
                                                                   float *__restrict__ parts) {
  constexpr int VL = AfVec<T>::N, CP = LPK * VL, SLOTS = AF_THREADS / LPK, U = QB >= 8 ? 2 : 4;
  __shared__ float s_part[AF_WARPS][QB][CP + 2];
  const b200c_attention_t &p = a.p;
  const int per_group = p.heads / p.groups;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, slot = tid / LPK, part = tid % LPK;
  const int split = blockIdx.x % splits;
  const int group = (blockIdx.x / splits) % p.groups;
  const int64_t b = blockIdx.x / (splits * p.groups);
  int64_t q_lo, q_hi, k_lo, k_hi;
  at_segment(p.ptr_q, p.m, b, q_lo, q_hi);
  at_segment(p.ptr_k, p.n, b, k_lo, k_hi);
  const int64_t rows = (q_hi - q_lo) * per_group;
  const int64_t each = ((k_hi - k_lo + splits - 1) / splits + SLOTS - 1) / SLOTS * SLOTS;
  const int64_t lo = k_lo + split * each, hi = lo + each < k_hi ? lo + each : k_hi;
  const T *k = (const T *)p.k + group * p.k_head + part * VL;
  const T *v = (const T *)p.v + group * p.v_head + part * VL;
  const int left = p.channels - part * VL;
  const bool bend = p.cap > 0.f;
  const float pre = bend ? p.scale : p.scale * AT_LOG2E, post = p.cap * AT_LOG2E, inv_cap = bend ? 1.f / p.cap : 0.f;

  for (int64_t r0 = 0; r0 < rows; r0 += QB) {
    float q[QB][VL], pos[QB][AT_MAX_DIMS], slope[QB], top[QB], sum[QB], o[QB][VL];
#pragma unroll
    for (int i = 0; i < QB; ++i) {
      const int64_t r = r0 + i < rows ? r0 + i : rows - 1;  // the last row stands in for those past the end
      const int64_t row = q_lo + r / per_group;
      const int head = group * per_group + (int)(r % per_group);
      const T *src = (const T *)p.q + row * p.q_row + head * p.q_head + part * VL;
#pragma unroll
      for (int c = 0; c < VL; ++c) q[i][c] = c < left ? at_float(src[c]) * pre : 0.f;
      if (p.dims > 0) {
        slope[i] = p.slope[head] * AT_LOG2E;
#pragma unroll
        for (int d = 0; d < AT_MAX_DIMS; ++d) pos[i][d] = d < p.dims ? p.pos_q[row * p.dims + d] : 0.f;
      }
      top[i] = -pos_inf<float>();
      sum[i] = 0.f;
#pragma unroll
      for (int c = 0; c < VL; ++c) o[i][c] = 0.f;
    }
    // all lanes of a warp take the same number of steps: the sums over a key's lanes are warp-wide shuffles
    for (int64_t j0 = lo; j0 < hi; j0 += SLOTS * U) {
      uint4 kr[U], vr[U];
      float s[U][QB];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t j = j0 + u * SLOTS + slot;
        const int have = j < hi ? left : 0;
        kr[u] = af_load<T>(k + j * p.k_row, vec, have);
        vr[u] = af_load<T>(v + j * p.v_row, vec, have);
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int64_t j = j0 + u * SLOTS + slot;
        float f[VL], dist[QB];
        af_widen<T>(kr[u], f);
        if (p.dims > 0) {
#pragma unroll
          for (int i = 0; i < QB; ++i) dist[i] = 0.f;
#pragma unroll
          for (int d = 0; d < AT_MAX_DIMS; ++d)
            if (d < p.dims) {
              const float x = j < hi ? p.pos_k[j * p.dims + d] : 0.f;
#pragma unroll
              for (int i = 0; i < QB; ++i) dist[i] = fmaf(pos[i][d] - x, pos[i][d] - x, dist[i]);
            }
        }
#pragma unroll
        for (int i = 0; i < QB; ++i) {
          float t = 0.f;
#pragma unroll
          for (int c = 0; c < VL; ++c) t = fmaf(q[i][c], f[c], t);
#pragma unroll
          for (int w = LPK / 2; w > 0; w >>= 1) t += __shfl_xor_sync(FULL_MASK, t, w);
          if (bend) t = post * tanhf(t * inv_cap);
          if (p.dims > 0) t = fmaf(-slope[i], sqrtf(dist[i]), t);
          s[u][i] = j < hi ? t : -pos_inf<float>();
        }
      }
#pragma unroll
      for (int i = 0; i < QB; ++i) {
        float m = top[i];
#pragma unroll
        for (int u = 0; u < U; ++u) m = fmaxf(m, s[u][i]);
        const float base = m == -pos_inf<float>() ? 0.f : m;
        const float shrink = exp2f(top[i] - base);
        top[i] = m;
        sum[i] *= shrink;
#pragma unroll
        for (int c = 0; c < VL; ++c) o[i][c] *= shrink;
#pragma unroll
        for (int u = 0; u < U; ++u) {
          s[u][i] = exp2f(s[u][i] - base);
          sum[i] += s[u][i];
        }
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float f[VL];
        af_widen<T>(vr[u], f);
#pragma unroll
        for (int i = 0; i < QB; ++i)
#pragma unroll
          for (int c = 0; c < VL; ++c) o[i][c] = fmaf(s[u][i], f[c], o[i][c]);
      }
    }
    // join the lane groups of the warp, then the warps
#pragma unroll
    for (int i = 0; i < QB; ++i) {
#pragma unroll
      for (int w = LPK; w < 32; w <<= 1) {
        const float m2 = __shfl_xor_sync(FULL_MASK, top[i], w), l2 = __shfl_xor_sync(FULL_MASK, sum[i], w);
        const float m = fmaxf(top[i], m2), base = m == -pos_inf<float>() ? 0.f : m;
        const float mine = exp2f(top[i] - base), other = exp2f(m2 - base);
        top[i] = m;
        sum[i] = sum[i] * mine + l2 * other;
#pragma unroll
        for (int c = 0; c < VL; ++c)
          o[i][c] = o[i][c] * mine + __shfl_xor_sync(FULL_MASK, o[i][c], w) * other;
      }
      if (lane < LPK) {
#pragma unroll
        for (int c = 0; c < VL; ++c) s_part[warp][i][lane * VL + c] = o[i][c];
        if (lane == 0) {
          s_part[warp][i][CP] = top[i];
          s_part[warp][i][CP + 1] = sum[i];
        }
      }
    }
    __syncthreads();
    for (int t = tid; t < QB * CP; t += AF_THREADS) {
      const int i = t / CP, c = t % CP;
      if (r0 + i >= rows) continue;
      float m = -pos_inf<float>();
#pragma unroll
      for (int w = 0; w < AF_WARPS; ++w) m = fmaxf(m, s_part[w][i][CP]);
      const float base = m == -pos_inf<float>() ? 0.f : m;
      float acc = 0.f, l = 0.f;
#pragma unroll
      for (int w = 0; w < AF_WARPS; ++w) {
        const float f = exp2f(s_part[w][i][CP] - base);
        acc = fmaf(s_part[w][i][c], f, acc);
        l = fmaf(s_part[w][i][CP + 1], f, l);
      }
      const int64_t r = r0 + i;
      const int64_t at = ((q_lo + r / per_group) * p.heads + group * per_group + r % per_group) * splits + split;
      float *dst = parts + at * (p.channels + 2);
      if (c < p.channels) dst[2 + c] = acc;
      if (c == 0) {
        dst[0] = m;
        dst[1] = l;
      }
    }
    __syncthreads();
  }
}

// ---- 16-bit types ------------------------------------------------------------------------------------------------
// The same split over examples, key heads and keys, with the two products on the tensor cores.  Up to 16 rows are too
// few for a tcgen05 tile of 128; warp-wide products of 16 x 8 x 16 take them as they are, so a warp spends a few
// hundred instructions on 16 KB of keys and values and memory is the only bound.  Each of the block's warps has a ring
// of its own in shared memory, 32 keys and values to a stage, filled by asynchronous 16-byte copies two stages ahead:
// no barrier between warps until the end.  A row of 2 * CP bytes keeps its 16-byte chunk c at c ^ (row & 7), so that
// neither the copies nor the matrix loads meet bank conflicts.  Weights are rounded to the 16-bit type (fp16: times 2^15);
// maxima, sums and results are fp32. Shared memory of keys past the split's end is cleared: their weights are 0, and 0 times
// whatever stood there must be 0.
constexpr int AF_KEYS = 32;    // keys of a stage
constexpr int AF_STAGES = 3;
constexpr int AF_ROWS = 16;    // rows (query, head of the group) of a pass

template <int CP>
struct AfTensor {
  static constexpr int CHUNKS = CP / 8;  // 16-byte chunks of a row
  static constexpr int TILE = AF_KEYS * CP * 2, STAGE = 2 * TILE + AF_KEYS * AT_MAX_DIMS * 4;
  static constexpr int SMEM = AF_WARPS * AF_STAGES * STAGE;
  static constexpr int PART = AF_ROWS * (CP + 2);  // floats of a warp's part, over its ring at the end
  static_assert(PART * 4 <= AF_STAGES * STAGE, "a warp's part fits its ring");
};

template <typename T, int CP, int DIM, bool CAP>
__global__ void __launch_bounds__(AF_THREADS) attention_few_tensor_kernel(AttnArgs a, int splits,
                                                                          float *__restrict__ parts) {
  using F = AfTensor<CP>;
  constexpr int KT = CP / 16, NT = AF_KEYS / 8, CT = CP / 8;
  extern __shared__ __align__(128) unsigned char af_smem[];
  const b200c_attention_t &p = a.p;
  const int per_group = p.heads / p.groups;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int split = blockIdx.x % splits;
  const int group = (blockIdx.x / splits) % p.groups;
  const int64_t b = blockIdx.x / (splits * p.groups);
  int64_t q_lo, q_hi, k_lo, k_hi;
  at_segment(p.ptr_q, p.m, b, q_lo, q_hi);
  at_segment(p.ptr_k, p.n, b, k_lo, k_hi);
  const int64_t rows = (q_hi - q_lo) * per_group;
  const int64_t each = ((k_hi - k_lo + splits - 1) / splits + AF_KEYS - 1) / AF_KEYS * AF_KEYS;
  const int64_t lo = k_lo + split * each, hi = lo + each < k_hi ? lo + each : k_hi;
  const T *k = (const T *)p.k + group * p.k_head;
  const T *v = (const T *)p.v + group * p.v_head;
  unsigned char *ring = af_smem + warp * (AF_STAGES * F::STAGE);
  const uint32_t ring_at = (uint32_t)__cvta_generic_to_shared(ring);
  // tanh(y) = 1 - 2 / (e^2y + 1)
  const float pre = CAP ? 2.f * AT_LOG2E * p.scale / p.cap : p.scale * AT_LOG2E, post = p.cap * AT_LOG2E;
  const int chunks = p.channels / 8;
  // this warp's steps of 32 keys: lo + 32 (warp + 4 i)
  const int64_t all_steps = hi > lo ? (hi - lo + AF_KEYS - 1) / AF_KEYS : 0;
  const int64_t steps = all_steps > warp ? (all_steps - warp + AF_WARPS - 1) / AF_WARPS : 0;

  // a lane copies chunk my_c of rows my_r, my_r + 32 / CHUNKS, ...
  constexpr int PER = 32 / F::CHUNKS, COPIES = AF_KEYS / PER;
  const int my_r = lane / F::CHUNKS, my_c = lane % F::CHUNKS;
  const int64_t first = lo + warp * AF_KEYS + my_r;
  const T *k_at = k + first * p.k_row + my_c * 8, *v_at = v + first * p.v_row + my_c * 8;  // of the next step fetched
  int fetch_slot = 0;
  int64_t fetch_j = lo + warp * AF_KEYS;
  auto rewind = [&]() {
    k_at = k + first * p.k_row + my_c * 8;
    v_at = v + first * p.v_row + my_c * 8;
    fetch_slot = 0;
    fetch_j = lo + warp * AF_KEYS;
  };
  auto fetch = [&]() {
    if (fetch_j < hi) {
      const uint32_t st = ring_at + fetch_slot * F::STAGE;
      const bool whole = fetch_j + AF_KEYS <= hi;
#pragma unroll
      for (int n = 0; n < COPIES; ++n) {
        const int r = n * PER + my_r;
        const uint32_t dk = st + r * (CP * 2) + ((my_c ^ (r & 7)) << 4);
        if (my_c < chunks && (whole || fetch_j + r < hi)) {
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dk), "l"(k_at + n * PER * p.k_row) : "memory");
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(dk + F::TILE), "l"(v_at + n * PER * p.v_row)
                       : "memory");
        } else {
          unsigned char *z = ring + (dk - ring_at);
          *reinterpret_cast<uint4 *>(z) = *reinterpret_cast<uint4 *>(z + F::TILE) = make_uint4(0u, 0u, 0u, 0u);
        }
      }
      if constexpr (DIM > 0) {
        float *sp = reinterpret_cast<float *>(ring + fetch_slot * F::STAGE + 2 * F::TILE);
        const float *src = p.pos_k + fetch_j * p.dims;
#pragma unroll
        for (int n = 0; n < DIM; ++n) {  // [dims][32 keys]
          const int i = n * 32 + lane, j = i / DIM, d = i - j * DIM;
          if (d < p.dims && (whole || fetch_j + j < hi))
            cp_async_4(sp + d * AF_KEYS + j, src + j * p.dims + d);
          else
            sp[d * AF_KEYS + j] = 0.f;
        }
      }
    }
    cp_async_commit();
    fetch_slot = fetch_slot + 1 == AF_STAGES ? 0 : fetch_slot + 1;
    fetch_j += AF_WARPS * AF_KEYS;
    k_at += AF_WARPS * AF_KEYS * p.k_row;
    v_at += AF_WARPS * AF_KEYS * p.v_row;
  };

  for (int64_t r0 = 0; r0 < rows; r0 += AF_ROWS) {
    // the rows' queries as the first operand: lane holds rows lane / 4 and lane / 4 + 8, channels 2 (lane % 4) + {0, 1,
    // 8, 9}
    const int gr = lane >> 2, gc = (lane & 3) * 2;
    uint32_t qf[KT][4];
    float pos[2][DIM == 0 ? 1 : DIM], slope[2] = {}, top[2], sum[2] = {}, o[CT][4] = {};
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      const int64_t r = r0 + gr + 8 * e;
      const bool there = r < rows;
      const int64_t row = q_lo + (there ? r : 0) / per_group;
      const int head = group * per_group + (int)((there ? r : 0) % per_group);
      const T *src = (const T *)p.q + row * p.q_row + head * p.q_head;
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int c = t * 16 + h * 8 + gc;
          qf[t][e + 2 * h] = there && c < p.channels ? *reinterpret_cast<const uint32_t *>(src + c) : 0u;
        }
      top[e] = -pos_inf<float>();
      if constexpr (DIM > 0) {
        slope[e] = p.slope[head] * AT_LOG2E;
#pragma unroll
        for (int d = 0; d < DIM; ++d) pos[e][d] = there && d < p.dims ? p.pos_q[row * p.dims + d] : 0.f;
      }
    }
    const bool both = rows - r0 > 8;  // whether rows 8 .. 15 are taken at all
    rewind();
#pragma unroll
    for (int i = 0; i < AF_STAGES - 1; ++i) fetch();
    int slot = 0;
    for (int64_t i = 0; i < steps; ++i, slot = slot + 1 == AF_STAGES ? 0 : slot + 1) {
      cp_async_wait<AF_STAGES - 2>();
      __syncwarp();
      const int64_t j0 = lo + (warp + i * AF_WARPS) * AF_KEYS;
      const uint32_t st = ring_at + slot * F::STAGE;
      const float *sp = reinterpret_cast<const float *>(ring + slot * F::STAGE + 2 * F::TILE) + gc;
      float s[NT][4] = {};
      // scores: 8 keys a tile; one matrix load brings 16 keys of 16 channels
#pragma unroll
      for (int t = 0; t < KT; ++t)
#pragma unroll
        for (int n = 0; n < NT; n += 2) {
          const int r = n * 8 + (lane & 7) + ((lane & 16) >> 1), c = 2 * t + ((lane >> 3) & 1);
          uint32_t kf[4];
          aw_ldmatrix(kf, st + r * (CP * 2) + ((c ^ (r & 7)) << 4));
          aw_mma<T>(s[n], qf[t], kf[0], kf[1]);
          aw_mma<T>(s[n + 1], qf[t], kf[2], kf[3]);
        }
      const bool whole = j0 + AF_KEYS <= hi;
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if (e == 1 && !both) break;
        float m = -pos_inf<float>();
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const int j = n * 8 + gc + u;
            float t;
            if constexpr (CAP)
              t = post * fmaf(-2.f, t5_rcp(t5_ex2(s[n][2 * e + u] * pre) + 1.f), 1.f);
            else
              t = s[n][2 * e + u] * pre;
            if constexpr (DIM > 0) {
              float d2 = 0.f;
#pragma unroll
              for (int d = 0; d < DIM; ++d) {
                const float df = pos[e][d] - sp[d * AF_KEYS + n * 8 + u];
                d2 = DIM == 1 ? fabsf(df) : fmaf(df, df, d2);
              }
              t = fmaf(-slope[e], DIM == 1 ? d2 : t5_sqrt(d2), t);
            }
            if (!whole && j0 + j >= hi) t = -pos_inf<float>();
            s[n][2 * e + u] = t;
            m = fmaxf(m, t);
          }
        m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, 1));
        m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, 2));
        m = fmaxf(top[e], m - AtType<T>::TOP);  // what the weights are relative to
        const float base = m == -pos_inf<float>() ? 0.f : m;
        const float shrink = t5_ex2(top[e] - base);
        top[e] = m;
        float part = 0.f;
#pragma unroll
        for (int n = 0; n < NT; ++n)
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            const float w = t5_ex2(s[n][2 * e + u] - base);
            s[n][2 * e + u] = w;
            part += w;
          }
        sum[e] = fmaf(sum[e], shrink, part);
#pragma unroll
        for (int n = 0; n < CT; ++n) {
          o[n][2 * e] *= shrink;
          o[n][2 * e + 1] *= shrink;
        }
      }
      if (!both) {
#pragma unroll
        for (int n = 0; n < NT; ++n) s[n][2] = s[n][3] = 0.f;
      }
#pragma unroll
      for (int t = 0; t < NT / 2; ++t) {  // 16 keys of the weights against 16 channels a matrix load
        const uint32_t wf[4] = {aw_pack<T>(s[2 * t][0], s[2 * t][1]), aw_pack<T>(s[2 * t][2], s[2 * t][3]),
                                aw_pack<T>(s[2 * t + 1][0], s[2 * t + 1][1]), aw_pack<T>(s[2 * t + 1][2], s[2 * t + 1][3])};
#pragma unroll
        for (int n = 0; n < CT; n += 2) {
          const int r = t * 16 + (lane & 15), c = n + (lane >> 4);
          uint32_t vf[4];
          aw_ldmatrix_t(vf, st + F::TILE + r * (CP * 2) + ((c ^ (r & 7)) << 4));
          aw_mma<T>(o[n], wf, vf[0], vf[1]);
          aw_mma<T>(o[n + 1], wf, vf[2], vf[3]);
        }
      }
      __syncwarp();  // the stage is read: it takes the step two ahead
      fetch();
    }
    cp_async_wait<0>();
    __syncwarp();
    // a warp's part over its ring: rows of CP results, the maximum and the sum
    float *mine = reinterpret_cast<float *>(ring);
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      sum[e] += __shfl_xor_sync(FULL_MASK, sum[e], 1);
      sum[e] += __shfl_xor_sync(FULL_MASK, sum[e], 2);
      float *dst = mine + (gr + 8 * e) * (CP + 2);
#pragma unroll
      for (int n = 0; n < CT; ++n) {
        dst[n * 8 + gc] = o[n][2 * e];
        dst[n * 8 + gc + 1] = o[n][2 * e + 1];
      }
      if ((lane & 3) == 0) {
        dst[CP] = top[e];
        dst[CP + 1] = sum[e];
      }
    }
    __syncthreads();
    for (int t = tid; t < AF_ROWS * CP; t += AF_THREADS) {
      const int i = t / CP, c = t % CP;
      if (r0 + i >= rows) break;
      float m = -pos_inf<float>(), acc = 0.f, l = 0.f;
      const float *src[AF_WARPS];
#pragma unroll
      for (int w = 0; w < AF_WARPS; ++w) {
        src[w] = reinterpret_cast<const float *>(af_smem + w * (AF_STAGES * F::STAGE)) + i * (CP + 2);
        m = fmaxf(m, src[w][CP]);
      }
      const float base = m == -pos_inf<float>() ? 0.f : m;
#pragma unroll
      for (int w = 0; w < AF_WARPS; ++w) {
        const float f = exp2f(src[w][CP] - base);
        acc = fmaf(src[w][c], f, acc);
        l = fmaf(src[w][CP + 1], f, l);
      }
      const int64_t r = r0 + i;
      const int64_t at = ((q_lo + r / per_group) * p.heads + group * per_group + r % per_group) * splits + split;
      float *dst = parts + at * (p.channels + 2);
      if (c < p.channels) dst[2 + c] = acc;
      if (c == 0) {
        dst[0] = m;
        dst[1] = l;
      }
    }
    __syncthreads();
  }
}

// joins the splits of a (row, head), in ascending order, a warp each
template <typename T>
__global__ void __launch_bounds__(256) attention_join_kernel(const __grid_constant__ AttnArgs a) {
  const b200c_attention_t &p = a.p;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31, splits = a.splits;
  if (i >= p.m * p.heads) return;
  const int64_t row = i / p.heads;
  const int head = (int)(i % p.heads), width = p.channels + 2;
  const float *src = a.parts + i * splits * width;
  float top[4], sum[4], m = -pos_inf<float>();  // at most 128 splits: four per lane (attention_few_splits)
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int s = n * 32 + lane;
    top[n] = s < splits ? src[(int64_t)s * width] : -pos_inf<float>();
    sum[n] = s < splits ? src[(int64_t)s * width + 1] : 0.f;
  }
  int64_t lo, hi;
  at_segment(p.ptr_q, p.m, at_segment_of_warp(p.ptr_q, (int)p.num_segments, row, lane), lo, hi);
  const bool inside = row >= lo && row < hi;  // else nothing was written there
#pragma unroll
  for (int n = 0; n < 4; ++n) m = fmaxf(m, top[n]);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, o));
  const float sub = m == -pos_inf<float>() ? 0.f : m;
  float l = 0.f;
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    top[n] = t5_ex2(top[n] - sub);  // now the split's factor
    l = fmaf(sum[n], top[n], l);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(FULL_MASK, l, o);
  if (!inside) l = 0.f;
  const float inv = l == 0.f ? 0.f : 1.f / l;
  float acc[AT_MAX_CHANNELS / 32] = {};
#pragma unroll
  for (int n = 0; n < 4; ++n) {
    const int most = splits - n * 32 < 32 ? splits - n * 32 : 32;
#pragma unroll 4
    for (int s = 0; s < most; ++s) {
      const float f = __shfl_sync(FULL_MASK, top[n], s);
#pragma unroll
      for (int c = 0; c < AT_MAX_CHANNELS / 32; ++c)
        if (c * 32 + lane < p.channels) acc[c] = fmaf(src[(int64_t)(n * 32 + s) * width + 2 + c * 32 + lane], f, acc[c]);
    }
  }
#pragma unroll
  for (int c = 0; c < AT_MAX_CHANNELS / 32; ++c)
    if (c * 32 + lane < p.channels) {
      const float x = l == 0.f ? 0.f : acc[c] * inv;
      const T r = at_round<T>(x);
      ((T *)a.out)[i * p.channels + c * 32 + lane] = r;
      if (a.rest) ((T *)a.rest)[i * p.channels + c * 32 + lane] = at_round<T>(x - at_float(r));
    }
  if (a.lse && lane == 0) a.lse[(int64_t)head * p.m + row] = l == 0.f ? pos_inf<float>() : m + log2f(l);
}

int launch_attention_join(const AttnArgs &a) {
  const int64_t rows = a.p.m * a.p.heads;
  if (a.p.dtype == B200C_F32)
    attention_join_kernel<float><<<(unsigned)((rows + 7) / 8), 256, 0, a.stream>>>(a);
  else if (a.p.dtype == B200C_F16)
    attention_join_kernel<__half><<<(unsigned)((rows + 7) / 8), 256, 0, a.stream>>>(a);
  else
    attention_join_kernel<__nv_bfloat16><<<(unsigned)((rows + 7) / 8), 256, 0, a.stream>>>(a);
  B200C_LAUNCH_CHECK("attention_join_kernel");
  return B200C_OK;
}

// Rows (query, head of the group) per example, on average, up to which these kernels are taken.  They read the keys once for
// every 16 rows (16-bit types) or 8 (fp32); the tiled kernels read them once for 128 or 64.  A block takes all rows of its
// example one after the other: an example of many queries among many of few is right, and slow (1000 examples of one
// query over 100 keys and one of 10000 over 10000, 4 heads, bf16: 36 ms, where the two apart take 0.5).
constexpr int64_t AF_MAX_ROWS = 16;
constexpr int AF_MIN_KEYS = 256;  // keys of a split, on average: below that the join costs more than it gains

int attention_few_splits(const b200c_attention_t &p) {
  if (p.m == 0 || p.n == 0) return 0;
  const int64_t segs = p.num_segments, per_group = p.heads / p.groups;
  if (p.m * per_group > AF_MAX_ROWS * segs || p.n < 64 * segs) return 0;
  const int64_t blocks = segs * p.groups;
  if (blocks > (1ll << 24)) return 0;
  // about four blocks per SM, so that ragged examples even out; 128 at most (the join)
  int64_t splits = (148 * 4 + blocks - 1) / blocks;
  const int64_t most = p.n / segs / AF_MIN_KEYS;
  if (splits > most) splits = most;
  if (splits > 128) splits = 128;
  return (int)(splits < 1 ? 1 : splits);
}

size_t attention_few_workspace_bytes(const b200c_attention_t &p) {
  return (size_t)p.m * p.heads * attention_few_splits(p) * (p.channels + 2) * 4;
}

static int af_join(const AttnArgs &a, int splits, float *parts) {
  AttnArgs j = a;
  j.splits = splits;
  j.parts = parts;
  return launch_attention_join(j);
}

template <typename T, int LPK, int QB>
static int af_launch(const AttnArgs &a, int splits, int vec, float *parts) {
  const unsigned blocks = (unsigned)(a.p.num_segments * a.p.groups * splits);
  attention_few_kernel<T, LPK, QB><<<blocks, AF_THREADS, 0, a.stream>>>(a, splits, vec, parts);
  B200C_LAUNCH_CHECK("attention_few_kernel");
  return af_join(a, splits, parts);
}

template <typename T, int CP, int DIM, bool CAP>
static int af_launch_tensor(const AttnArgs &a, int splits, float *parts) {
  using F = AfTensor<CP>;
  static unsigned long long configured = 0ull;
  B200C_CUDA(opt_in_shared_memory(attention_few_tensor_kernel<T, CP, DIM, CAP>, F::SMEM, configured));
  const unsigned blocks = (unsigned)(a.p.num_segments * a.p.groups * splits);
  attention_few_tensor_kernel<T, CP, DIM, CAP><<<blocks, AF_THREADS, F::SMEM, a.stream>>>(a, splits, parts);
  B200C_LAUNCH_CHECK("attention_few_tensor_kernel");
  return af_join(a, splits, parts);
}
template <typename T, int CP, bool CAP>
static int af_tensor_dims(const AttnArgs &a, int splits, float *parts) {
  if (a.p.dims == 0) return af_launch_tensor<T, CP, 0, CAP>(a, splits, parts);
  if (a.p.dims == 1) return af_launch_tensor<T, CP, 1, CAP>(a, splits, parts);
  if (a.p.dims <= 3) return af_launch_tensor<T, CP, 3, CAP>(a, splits, parts);
  return af_launch_tensor<T, CP, 8, CAP>(a, splits, parts);
}
template <typename T>
static int af_tensor(const AttnArgs &a, int splits, float *parts) {
  if (a.p.channels <= 64)
    return a.p.cap > 0.f ? af_tensor_dims<T, 64, true>(a, splits, parts) : af_tensor_dims<T, 64, false>(a, splits, parts);
  return a.p.cap > 0.f ? af_tensor_dims<T, 128, true>(a, splits, parts) : af_tensor_dims<T, 128, false>(a, splits, parts);
}

template <typename T, int LPK>
static int af_rows(const AttnArgs &a, int splits, int vec, float *parts) {
  const int64_t rows = (a.p.m + a.p.num_segments - 1) / a.p.num_segments * (a.p.heads / a.p.groups);
  if (rows <= 1) return af_launch<T, LPK, 1>(a, splits, vec, parts);
  if (rows <= 4) return af_launch<T, LPK, 4>(a, splits, vec, parts);
  return af_launch<T, LPK, 8>(a, splits, vec, parts);
}

template <typename T>
static int af_channels(const AttnArgs &a, int splits, float *parts) {
  constexpr int VL = AfVec<T>::N;
  const b200c_attention_t &p = a.p;
  const int vec = ((uintptr_t)p.k & 15) == 0 && ((uintptr_t)p.v & 15) == 0 && p.channels % VL == 0 &&
                  p.k_row % VL == 0 && p.v_row % VL == 0 && p.k_head % VL == 0 && p.v_head % VL == 0;
  if constexpr (sizeof(T) == 2) {
    // queries are read as pairs of channels
    const bool pairs = ((uintptr_t)p.q & 3) == 0 && p.q_row % 2 == 0 && p.q_head % 2 == 0;
    if (vec && pairs && !(p.cap > AT_MAX_FAST_CAP)) return af_tensor<T>(a, splits, parts);
  }
  if (p.channels <= 32) return af_rows<T, 32 / VL>(a, splits, vec, parts);
  if (p.channels <= 64) return af_rows<T, 64 / VL>(a, splits, vec, parts);
  return af_rows<T, 128 / VL>(a, splits, vec, parts);
}

int launch_attention_few(const AttnArgs &a, int splits, void *workspace) {
  if (a.p.dtype == B200C_F32) return af_channels<float>(a, splits, (float *)workspace);
  if (a.p.dtype == B200C_F16) return af_channels<__half>(a, splits, (float *)workspace);
  return af_channels<__nv_bfloat16>(a, splits, (float *)workspace);
}

}  // namespace b200c
