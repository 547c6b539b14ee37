// Attention on the 5th-generation tensor cores, 16-bit types (see attention.cuh for the formulas): what the forward
// and the backward kernel share.
//
// A block owns 128 rows of one side and walks the other side's rows of the same examples ("columns") in tiles of 64:
//   forward: rows = queries of a head,  columns = keys;     S = Q K^T,  then O += P V
//   dq:      rows = queries of a head,  columns = keys;     S = Q K^T, dP = dO V^T,  then dQ += dS K
//   dk, dv:  rows = keys of a group,    columns = queries;  S' = K Q^T, dP' = V dO^T,  then dV += P' dO, dK += dS' Q
// One warp brings the operands to shared memory (TMA, 128-byte swizzle, a ring of stages, with the columns' coordinates
// and statistics beside them), one thread issues the products, and the other warps read the scores from tensor
// memory, a row per thread, and put the 16-bit weights back there, where the second products take them as their
// first operand.  The first products have both operands K-major; the second take the column tile MN-major, as it stands.
//
// A tile may hold rows of several (short) examples.  Its columns are then the union of their ranges, one pass over
// them, every row masked to its own range.  A masked weight is 0, and 0 times a NaN or an infinity of another example would be
// NaN: in such tiles the operand of the second product is looked through for them, and if there is one the pass is
// repeated example by example.  Column rows past the range's end are cleared in shared memory for the same reason.
#pragma once

#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200c {

constexpr int AT_ROWS = 128;  // rows of a block = lanes of tensor memory
constexpr int AT_COLS = 64;   // columns of a step

// tensor map of [rows, heads, channels] with boxes of 64 channels x box_rows rows of one head
int attention_tensor_map(CUtensorMap *map, const void *base, int dtype, int64_t rows, int heads, int channels,
                         int64_t row_stride, int64_t head_stride, int box_rows);

// Rows [r_lo, r_hi) of the block's tile and the columns they see.
struct AtPass {
  int64_t c_lo, c_hi;
  int segment;  // -1: all rows of the tile
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
    b_first = segment_of(pr, segments, t0);
    b_last = segment_of(pr, segments, t1 - 1);
  }
  __device__ __forceinline__ AtPass all() const {
    AtPass p;
    int64_t unused;
    at_segment(ptr_c, cols, b_first, p.c_lo, unused);
    at_segment(ptr_c, cols, b_last, unused, p.c_hi);
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
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};
template <>
struct AtType<__half> {
  static constexpr bool BF16 = false;
  static constexpr uint32_t EXP = 0x7fff7fffu, ONE = 0x04000400u;
  // probabilities below 2^-14 would lose bits in fp16: times 2^12 they keep them down to 2^-26
  static constexpr float SHIFT = 12.f;
  __device__ __forceinline__ static uint32_t pack(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
  }
};

template <typename T>
__device__ __forceinline__ uint32_t at_not_finite(const uint4 &w) {
  using A = AtType<T>;
  return (((w.x & A::EXP) + A::ONE) | ((w.y & A::EXP) + A::ONE) | ((w.z & A::EXP) + A::ONE) |
          ((w.w & A::EXP) + A::ONE)) & 0x80008000u;
}

// Looks through a column tile ([CP / 64][64 rows][128 bytes]); returns non-zero if a value is not finite.
template <typename T, int CP>
__device__ __forceinline__ uint32_t at_scan(const unsigned char *tile, int tid, int threads) {
  uint32_t bad = 0u;
  for (int i = tid; i < CP * 8; i += threads) bad |= at_not_finite<T>(reinterpret_cast<const uint4 *>(tile)[i]);
  return bad;
}
// Clears rows [count, 64) of a column tile.
template <int CP>
__device__ __forceinline__ void at_clear(unsigned char *tile, int count, int tid, int threads) {
  const int each = (AT_COLS - count) * 8;
#pragma unroll
  for (int a = 0; a < CP / 64; ++a)
    for (int i = tid; i < each; i += threads)
      reinterpret_cast<uint4 *>(tile + a * (AT_COLS * 128) + count * 128)[i] = make_uint4(0u, 0u, 0u, 0u);
}

// The bias and the cap of 32 scores of a row: s[j] (dot products) become log2 e (t - slope |pos - pos_j|).
// col_pos: [dims][64] coordinates of the step's columns.  u[j] = tanh of the capped score, where wanted.
template <int DIM, bool CAP, bool KEEP>
__device__ __forceinline__ void at_logits(float *s, float *u, const float *col_pos, const float *pos, float slope2,
                                          float pre, float post) {
#pragma unroll
  for (int j4 = 0; j4 < 32; j4 += 4) {
    float d2[4] = {};
    if constexpr (DIM > 0) {
#pragma unroll
      for (int d = 0; d < DIM; ++d) {
        const float4 x = *reinterpret_cast<const float4 *>(col_pos + d * AT_COLS + j4);
        const float xs[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          const float df = pos[d] - xs[j];
          d2[j] = DIM == 1 ? fabsf(df) : fmaf(df, df, d2[j]);
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
        t = w * post;
      } else {
        t = s[j4 + j] * pre;  // pre = scale log2 e
      }
      if constexpr (DIM == 1)
        t = fmaf(-slope2, d2[j], t);
      else if constexpr (DIM > 1)
        t = fmaf(-slope2, t5_sqrt(d2[j]), t);
      s[j4 + j] = t;
    }
  }
}

// After a wait ran out: the copies of the last steps that were issued must land before the block's memory goes.
__device__ __forceinline__ void at_drain(uint64_t *full, uint32_t stages, uint32_t issued) {
  for (uint32_t g = issued > stages ? issued - stages : 0; g < issued; ++g)
    for (int n = 0; n < T5_SPIN_LIMIT && !t5_mbar_try(&full[g % stages], (g / stages) & 1); ++n) {
    }
}

}  // namespace b200c
