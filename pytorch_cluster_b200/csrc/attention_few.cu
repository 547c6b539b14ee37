// Attention of a few queries per example over many keys (see attention.cuh for the formulas): pooling by a learned
// query, or one new token over a long memory.  Every key and value is read once for all query heads that share it,
// so memory bandwidth bounds it while a group serves few heads.
//
// A block owns one (example, key/value head, split of the example's keys) and takes up to QB rows (query, head of the
// group) at a time.  LPK lanes share a key, 16 bytes of its channels each; the lane groups of the block walk the
// split's keys in turn, U keys ahead of their use, each with a running maximum, sum and result of its own, which are
// joined by shuffles and through shared memory at the end.  The splits' parts go to the workspace in fp32 and a second kernel joins
// them, in ascending order of the splits.
#include <type_traits>

#include "attention.cuh"

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
  const float pre = bend ? p.scale / p.cap : p.scale * AT_LOG2E, post = p.cap * AT_LOG2E;

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
          if (bend) t = post * tanhf(t);
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

// joins the splits of a (row, head), one warp each
template <typename T>
__global__ void __launch_bounds__(256) attention_few_join_kernel(AttnArgs a, int splits,
                                                                 const float *__restrict__ parts) {
  const b200c_attention_t &p = a.p;
  const int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) >> 5;
  const int lane = threadIdx.x & 31;
  if (i >= p.m * p.heads) return;
  const int64_t row = i / p.heads;
  const int head = (int)(i % p.heads);
  int64_t lo, hi;
  at_segment(p.ptr_q, p.m, segment_of(p.ptr_q, p.num_segments, row), lo, hi);
  const bool inside = row >= lo && row < hi;
  const int width = p.channels + 2;
  const float *src = parts + i * splits * width;
  float m = -pos_inf<float>(), l = 0.f;
  if (inside) {
    for (int s = lane; s < splits; s += 32) m = fmaxf(m, src[(int64_t)s * width]);
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(FULL_MASK, m, o));
  }
  const float base = m == -pos_inf<float>() ? 0.f : m;
  if (inside)
    for (int s = 0; s < splits; ++s) l = fmaf(src[(int64_t)s * width + 1], exp2f(src[(int64_t)s * width] - base), l);
  const float inv = l == 0.f ? 0.f : 1.f / l;
  T *out = (T *)a.out + i * p.channels;
  for (int c = lane; c < p.channels; c += 32) {
    float acc = 0.f;
    if (inside)
      for (int s = 0; s < splits; ++s)
        acc = fmaf(src[(int64_t)s * width + 2 + c], exp2f(src[(int64_t)s * width] - base), acc);
    const T r = at_round<T>(acc * inv);
    out[c] = r;
    if (a.rest) ((T *)a.rest)[i * p.channels + c] = at_round<T>(acc * inv - at_float(r));
  }
  if (a.lse && lane == 0) a.lse[(int64_t)head * p.m + row] = l == 0.f ? pos_inf<float>() : m + log2f(l);
}

// Queries of a group per example, on average, up to which this kernel is taken.  It reads the keys once for every
// QB = 8 rows; the tiled kernels read them once for 64 or 128.
constexpr int64_t AF_MAX_ROWS = 16;
constexpr int AF_MIN_KEYS = 256;  // keys of a split, on average: below that the join costs more than it gains

int attention_few_splits(const b200c_attention_t &p) {
  if (p.m == 0 || p.n == 0) return 0;
  const int64_t segs = p.num_segments, per_group = p.heads / p.groups;
  if (p.m * per_group > AF_MAX_ROWS * segs || p.n < 64 * segs) return 0;
  const int64_t blocks = segs * p.groups;
  if (blocks > (1ll << 24)) return 0;
  // about eight blocks per SM, so that ragged examples even out
  int64_t splits = (148 * 8 + blocks - 1) / blocks;
  const int64_t most = p.n / segs / AF_MIN_KEYS;
  if (splits > most) splits = most;
  return (int)(splits < 1 ? 1 : splits);
}

size_t attention_few_workspace_bytes(const b200c_attention_t &p) {
  return (size_t)p.m * p.heads * attention_few_splits(p) * (p.channels + 2) * 4;
}

template <typename T, int LPK, int QB>
static int af_launch(const AttnArgs &a, int splits, int vec, float *parts) {
  const unsigned blocks = (unsigned)(a.p.num_segments * a.p.groups * splits);
  attention_few_kernel<T, LPK, QB><<<blocks, AF_THREADS, 0, a.stream>>>(a, splits, vec, parts);
  B200C_LAUNCH_CHECK("attention_few_kernel");
  const int64_t rows = a.p.m * a.p.heads;
  attention_few_join_kernel<T><<<(unsigned)((rows + 7) / 8), 256, 0, a.stream>>>(a, splits, parts);
  B200C_LAUNCH_CHECK("attention_few_join_kernel");
  return B200C_OK;
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
