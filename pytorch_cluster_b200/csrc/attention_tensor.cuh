// Attention on the 5th-generation tensor cores, 16-bit types (see attention.cuh for the formulas): what the forward
// and the backward kernel share.
//
// A block owns 128 rows of one side and walks the other side's rows of the same examples ("columns"), 64 to a stage:
//   forward: rows = queries of a head,  columns = keys;     S = Q K^T,  then O += P V
//   dq:      rows = queries of a head,  columns = keys;     S = Q K^T, dP = dO V^T,  then dQ += dS K
//   dk, dv:  rows = keys of a group,    columns = queries;  S' = K Q^T, dP' = V dO^T,  then dV += P' dO, dK += dS' Q
// One warp brings the operands to shared memory (TMA, 128-byte swizzle, a ring of stages, with the columns' coordinates
// and statistics beside them), one issues the products of the scores, one the products with the weights.  The other
// warps form G groups of four; a pair of groups takes a stage, 32 columns each: they read the scores from tensor
// memory, a row per thread, and put the 16-bit weights back there, where the second products take them as their first
// operand.  The first products have both operands K-major; the second take the column tile MN-major, as it stands.
// Exponentials and roots bound these kernels, not the products: everything is arranged so that the groups never wait
// for a product. They hand the scores' place back as soon as they have read them, so that the next scores are formed
// while they work on these, and the weights have a place of their own.
//
// A tile may hold rows of several (short) examples.  Its columns are then the union of their ranges, one pass over
// them, every row masked to its own range.  A masked weight is 0, and 0 times a NaN or an infinity of another example
// would be NaN: in such tiles the operand of the second product is looked through for them, and if there is one the
// pass is repeated example by example.  Column rows past the range's end are cleared in shared memory for the same
// reason.
#pragma once

#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200c {

constexpr int AT_ROWS = 128;  // rows of a block = lanes of tensor memory
constexpr int AT_COLS = 64;   // columns of a stage
constexpr int AT_SUB = 32;    // columns of a group's share of it

// tensor map of [rows, heads, channels] with boxes of 64 channels x box_rows rows of one head
int attention_tensor_map(CUtensorMap *map, const void *base, int dtype, int64_t rows, int heads, int channels,
                         int64_t row_stride, int64_t head_stride, int box_rows);

// segment_of for a whole warp: 32 probes at a time, a third of the dependent loads
__device__ __forceinline__ int at_segment_of_warp(const int64_t *__restrict__ ptr, int num_segments, int64_t row,
                                                  int lane) {
  if (ptr == nullptr) return 0;
  int lo = 0, hi = num_segments - 1;
  while (lo < hi) {
    const int step = (hi - lo + 32) / 32;
    const int64_t want = (int64_t)lo + (int64_t)(lane + 1) * step - 1;
    const int pos = want < hi ? (int)want : hi;
    const unsigned found = __ballot_sync(FULL_MASK, pos == hi || ptr[pos + 1] > row);
    const int k = __ffs(found) - 1;
    lo += k * step;
    hi = __shfl_sync(FULL_MASK, pos, k);
  }
  return lo;
}

// The tile of this block: the heads of a tile run side by side, tiles in the order given, so that what runs last is
// cheap (16 clouds of 1594 to 2555 points: forward 642 -> 613 us, dq 705 -> 637; 8 of 4000 points with 128 channels
// 1344 -> 1223).
__device__ __forceinline__ int64_t at_tile_of(const int *order, int per_tile) {
  const unsigned i = blockIdx.x / (unsigned)per_tile;
  return order ? order[i] : (int64_t)i;
}

// The columns of a pass over the tile.
struct AtPass {
  int64_t c_lo, c_hi;
  int segment;  // -1: all rows of the tile
};

// What the threads of a block find out together about its rows.
struct AtTileShared {
  int b_first, b_last;
  int64_t r[AT_ROWS + 1], c[AT_ROWS + 1];  // both sides' pointers from b_first on, as far as the tile's segments go
  int segment[AT_ROWS];                    // of each row
};

struct AtTile {
  int64_t t0, t1;  // rows of the tile
  const int64_t *ptr_r, *ptr_c;
  int64_t rows, cols;
  int segments, b_first, b_last;

  __device__ __forceinline__ void init(int64_t t0_, const int64_t *pr, const int64_t *pc, int64_t rows_, int64_t cols_,
                                       int64_t segs) {
    t0 = t0_;
    rows = rows_;
    cols = cols_;
    t1 = t0 + AT_ROWS < rows ? t0 + AT_ROWS : rows;
    ptr_r = pr;
    ptr_c = pc;
    segments = (int)segs;
  }
  // by warps 0 and 1, before a block-wide barrier; the rest after it
  __device__ __forceinline__ void search(AtTileShared &sh, int warp, int lane) const {
    if (warp < 2) {
      const int b = at_segment_of_warp(ptr_r, segments, warp == 0 ? t0 : t1 - 1, lane);
      if (lane == 0) (warp == 0 ? sh.b_first : sh.b_last) = b;
    }
  }
  __device__ __forceinline__ void found(const AtTileShared &sh) {
    b_first = sh.b_first;
    b_last = sh.b_last;
  }
  // whether the tile's segments are few enough to be listed; then all threads do so, and a barrier follows
  __device__ __forceinline__ bool listed() const { return ptr_r != nullptr && b_last - b_first < AT_ROWS - 1; }
  __device__ __forceinline__ void list(AtTileShared &sh, int tid) const {
    if (tid <= b_last - b_first + 1) {
      sh.r[tid] = ptr_r[b_first + tid];
      sh.c[tid] = ptr_c[b_first + tid];
    }
  }
  __device__ __forceinline__ int segment(const AtTileShared &sh, int64_t row) const {
    if (b_first == b_last) return b_first;
    if (!listed()) return segment_of(ptr_r, segments, row);
    int lo = 0, hi = b_last - b_first;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (sh.r[mid + 1] > row)
        hi = mid;
      else
        lo = mid + 1;
    }
    return b_first + lo;
  }
  // rows and columns of a segment of the tile, clipped as at_segment does
  __device__ __forceinline__ void rows_of(const AtTileShared &sh, int b, int64_t &lo, int64_t &hi) const {
    if (listed())
      at_clip(sh.r[b - b_first], sh.r[b - b_first + 1], rows, lo, hi);
    else
      at_segment(ptr_r, rows, b, lo, hi);
  }
  __device__ __forceinline__ void cols_of(const AtTileShared &sh, int b, int64_t &lo, int64_t &hi) const {
    if (listed())
      at_clip(sh.c[b - b_first], sh.c[b - b_first + 1], cols, lo, hi);
    else
      at_segment(ptr_c, cols, b, lo, hi);
  }
  __device__ __forceinline__ AtPass all(const AtTileShared &sh) const {
    AtPass p;
    int64_t unused;
    cols_of(sh, b_first, p.c_lo, unused);
    cols_of(sh, b_last, unused, p.c_hi);
    if (p.c_hi < p.c_lo) p.c_hi = p.c_lo;
    p.segment = -1;
    return p;
  }
  // the next pass of a tile taken example by example; `at` is the first row not yet taken
  __device__ __forceinline__ bool next(int64_t &at, AtPass &p) const {
    if (at >= t1) return false;
    p.segment = segment_of(ptr_r, segments, at);
    at_segment(ptr_c, cols, p.segment, p.c_lo, p.c_hi);
    int64_t lo, hi;
    at_segment(ptr_r, rows, p.segment, lo, hi);
    // rows that belong to no example go with the one that segment_of names
    at = p.segment == segments - 1 ? t1 : hi > at ? hi : at + 1;
    return true;
  }
};

template <typename T>
struct AtType;
template <>
struct AtType<__nv_bfloat16> {
  static constexpr bool BF16 = true;
  static constexpr uint32_t EXP = 0x7fff7fffu, ONE = 0x00800080u;  // |w| + one step of the exponent overflows for inf, NaN
  static constexpr float SHIFT = 0.f;  // weights of the backward pass are kept times 2^SHIFT
  // forward: weights are kept times 2^RAISED in tiles, where their sum over a step may grow to MOST, and times 2^TOP
  // where none is above 1
  static constexpr float RAISED = 0.f, MOST = 1024.f, TOP = 0.f;
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  __device__ __forceinline__ static float low(uint32_t v) { return __uint_as_float(v << 16); }
  __device__ __forceinline__ static float high(uint32_t v) { return __uint_as_float(v & 0xffff0000u); }
};
template <>
struct AtType<__half> {
  static constexpr bool BF16 = false;
  static constexpr uint32_t EXP = 0x7fff7fffu, ONE = 0x04000400u;
  // probabilities below 2^-14 would lose bits in fp16: times 2^12 they keep them down to 2^-26
  static constexpr float SHIFT = 12.f;
  // forward: below 2^-14 of a row's largest they would lose bits and vanish below 2^-25, however many they are
  static constexpr float RAISED = 9.f, MOST = 32768.f, TOP = 15.f;
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
  __device__ __forceinline__ static float low(uint32_t v) { return __low2float(*reinterpret_cast<const __half2 *>(&v)); }
  __device__ __forceinline__ static float high(uint32_t v) { return __high2float(*reinterpret_cast<const __half2 *>(&v)); }
};

// The power of two that fp16's dS is kept times: it brings the largest value that |do| and |v| of the row's example and
// key head allow to 2^14.  With one power for the whole call the examples would not be apart: one with output gradients
// of 6e4 took all bits from another's of 1e-4.  norms: the largest |do|^2 and |v|^2 of the finite rows, [segments, groups,
// 2]; b < 0: a row that is not there.
template <typename T>
__device__ __forceinline__ float at_sigma(const float *norms, int groups, int b, int group) {
  if constexpr (AtType<T>::BF16) {
    return 1.f;
  } else {
    if (b < 0) return 1.f;
    const float2 n = reinterpret_cast<const float2 *>(norms)[(int64_t)b * groups + group];
    const float most = 2.f * sqrtf(n.x) * sqrtf(n.y);
    return most > 1e-30f ? exp2f(14.f - ceilf(log2f(most))) : 1.f;
  }
}

template <typename T>
__device__ __forceinline__ uint32_t at_not_finite(const uint4 &w) {
  using A = AtType<T>;
  return (((w.x & A::EXP) + A::ONE) | ((w.y & A::EXP) + A::ONE) | ((w.z & A::EXP) + A::ONE) |
          ((w.w & A::EXP) + A::ONE)) & 0x80008000u;
}

// Looks through 32 rows of a column tile ([CP / 64][64 rows][128 bytes]) with 128 threads; non-zero if a value is not
// finite.
template <typename T, int CP>
__device__ __forceinline__ uint32_t at_scan(const unsigned char *tile, int tid) {
  uint32_t bad = 0u;
#pragma unroll
  for (int a = 0; a < CP / 64; ++a)
#pragma unroll
    for (int i = 0; i < 2; ++i)
      bad |= at_not_finite<T>(reinterpret_cast<const uint4 *>(tile + a * (AT_COLS * 128))[i * 128 + tid]);
  return bad;
}
// Clears rows [count, 32) of them.
template <int CP>
__device__ __forceinline__ void at_clear(unsigned char *tile, int count, int tid) {
#pragma unroll
  for (int a = 0; a < CP / 64; ++a)
    for (int i = tid; i < (AT_SUB - count) * 8; i += 128)
      reinterpret_cast<uint4 *>(tile + a * (AT_COLS * 128) + count * 128)[i] = make_uint4(0u, 0u, 0u, 0u);
}

// Stages of one walk over `count` columns.
__device__ __forceinline__ uint32_t at_stages(int64_t count) { return (uint32_t)((count + AT_COLS - 1) / AT_COLS); }

// The place in a ring of stages, with the parity of its current round.
template <int STAGES>
struct AtRing {
  uint32_t st, parity;
  __device__ __forceinline__ explicit AtRing(uint32_t g) : st(g % STAGES), parity((g / STAGES) & 1u) {}
  __device__ __forceinline__ void next() {
    if (++st == STAGES) {
      st = 0;
      parity ^= 1u;
    }
  }
};

// The columns [lo, hi) that the rows of a warp see, relative to the pass's first: a step can be skipped where no row
// sees any of its columns, and needs no mask where every row sees all of them.
struct AtSeen {
  int lo, hi, any_lo, any_hi, all_lo, all_hi;
  __device__ __forceinline__ AtSeen(int64_t row_lo, int64_t row_hi, const AtPass &pass, bool mine) {
    const int64_t count = pass.c_hi - pass.c_lo, l = mine ? row_lo - pass.c_lo : 0, h = mine ? row_hi - pass.c_lo : 0;
    lo = (int)(l < 0 ? 0 : l > count ? count : l);
    hi = (int)(h < 0 ? 0 : h > count ? count : h);
    const bool none = lo >= hi;
    any_lo = __reduce_min_sync(FULL_MASK, none ? 0x7fffffff : lo);
    any_hi = __reduce_max_sync(FULL_MASK, none ? 0 : hi);
    all_lo = __reduce_max_sync(FULL_MASK, none ? 0x7fffffff : lo);
    all_hi = __reduce_min_sync(FULL_MASK, none ? 0 : hi);
  }
  __device__ __forceinline__ bool any(int base) const { return base < any_hi && base + AT_SUB > any_lo; }
  __device__ __forceinline__ bool all(int base) const { return base >= all_lo && base + AT_SUB <= all_hi; }
};

// Coordinates of a stage's columns: a lane's share in registers, then [dims][64] in shared memory.
template <int DIM>
__device__ __forceinline__ void at_fetch_places(float *v, const float *__restrict__ src, int dims, int64_t c0,
                                                int64_t c_hi, int lane) {
#pragma unroll
  for (int n = 0; n < 2 * DIM; ++n) {
    const int i = n * 32 + lane, c = i / DIM, d = i - c * DIM;
    v[n] = c0 + c < c_hi && d < dims ? src[(c0 + c) * dims + d] : 0.f;
  }
}
template <int DIM>
__device__ __forceinline__ void at_put_places(float *dst, const float *v, int lane) {
#pragma unroll
  for (int n = 0; n < 2 * DIM; ++n) {
    const int i = n * 32 + lane, c = i / DIM, d = i - c * DIM;
    dst[d * AT_COLS + c] = v[n];
  }
}
template <>
__device__ __forceinline__ void at_fetch_places<0>(float *, const float *__restrict__, int, int64_t, int64_t, int) {}
template <>
__device__ __forceinline__ void at_put_places<0>(float *, const float *, int) {}

// The bias and the cap of 32 scores of a row: s[j] (dot products) become log2 e (t - slope |pos - pos_j|) - sub, with
// one `sub` of the row or, with COL, one per column.  col_pos: [dims][64] coordinates of the stage's columns, from the
// step's first.  u[j] = tanh of the capped score, where wanted.
template <int DIM, bool CAP, bool KEEP, bool COL>
__device__ __forceinline__ void at_logits(float *s, float *u, const float *col_pos, const float *pos, float slope2,
                                          float pre, float post, float sub, const float *col_sub) {
#pragma unroll
  for (int j4 = 0; j4 < AT_SUB; j4 += 4) {
    float d2[4] = {}, off[4] = {sub, sub, sub, sub};
    if constexpr (COL) {
      const float4 x = *reinterpret_cast<const float4 *>(col_sub + j4);
      off[0] = x.x, off[1] = x.y, off[2] = x.z, off[3] = x.w;
    }
    if constexpr (DIM > 0) {
#pragma unroll
      for (int d = 0; d < DIM; ++d) {
        const float4 x = *reinterpret_cast<const float4 *>(col_pos + d * AT_COLS + j4);
        const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float df = pos[d] - xs[j];
          d2[j] = DIM == 1 ? fabsf(df) : d == 0 ? df * df : fmaf(df, df, d2[j]);
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float t;
      if constexpr (CAP) {
        // tanh(y) = 1 - 2 / (e^2y + 1); pre = 2 log2 e scale / cap, post = cap log2 e
        const float w = fmaf(-2.f, t5_rcp(t5_ex2(s[j4 + j] * pre) + 1.f), 1.f);
        if constexpr (KEEP) u[j4 + j] = w;
        t = fmaf(w, post, -off[j]);
      } else {
        t = fmaf(s[j4 + j], pre, -off[j]);  // pre = scale log2 e
      }
      if constexpr (DIM == 1)
        t = fmaf(-slope2, d2[j], t);
      else if constexpr (DIM > 1)
        t = fmaf(-slope2, t5_sqrt(d2[j]), t);
      s[j4 + j] = t;
    }
  }
}

// A block's rows leave by way of shared memory (the ring, idle at the end of a pass): a thread has 16 bytes of its row
// in hand at a time, and 32 rows' worth of them would be 32 places for the memory to go to.  16-byte chunk c of row r
// is kept at c ^ (r & 7).
template <int CP>
__device__ __forceinline__ void at_put(unsigned char *tile, int r, int chunk, const uint4 &v) {
  *reinterpret_cast<uint4 *>(tile + r * (CP * 2) + ((chunk ^ (r & 7)) << 4)) = v;
}
// rows of the pass to dst + row * stride (elements)
template <typename T, int CP>
__device__ __forceinline__ void at_write_rows(const unsigned char *tile, const AtTileShared &sh, const AtTile &t,
                                              const AtPass &pass, T *dst, int64_t stride, int channels, int tid,
                                              int threads) {
  constexpr int CHUNKS = CP / 8;
  for (int i = tid; i < AT_ROWS * CHUNKS; i += threads) {
    const int r = i / CHUNKS, c = i % CHUNKS;
    if (t.t0 + r < t.t1 && (pass.segment < 0 || pass.segment == sh.segment[r]) && c * 8 < channels)
      *reinterpret_cast<uint4 *>(dst + (t.t0 + r) * stride + c * 8) =
          *reinterpret_cast<const uint4 *>(tile + r * (CP * 2) + ((c ^ (r & 7)) << 4));
  }
}

// After a wait ran out: the copies of the last steps that were issued must land before the block's memory goes.
__device__ __forceinline__ void at_drain(uint64_t *full, uint32_t stages, uint32_t issued) {
  for (uint32_t g = issued > stages ? issued - stages : 0; g < issued; ++g)
    for (int n = 0; n < T5_SPIN_LIMIT && !t5_mbar_try(&full[g % stages], (g / stages) & 1); ++n) {
    }
}

}  // namespace b200c
