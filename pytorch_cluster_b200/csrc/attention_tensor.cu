// Host side of the tensor-core attention: which calls it takes, tensor maps, dispatch over types.
#include "attention_tensor.cuh"
#include "attention_tensor_launch.h"

namespace b200c {

using EncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                 const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeTiled encode_tiled() {
  static EncodeTiled fn = [] {
    void *p = nullptr;
    cudaDriverEntryPointQueryResult found = cudaDriverEntryPointSymbolNotFound;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &p, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      p = nullptr;
    return (EncodeTiled)p;
  }();
  return fn;
}

int attention_tensor_map(CUtensorMap *map, const void *base, int dtype, int64_t rows, int heads, int channels,
                         int64_t row_stride, int64_t head_stride, int box_rows) {
  EncodeTiled encode = encode_tiled();
  if (encode == nullptr) {
    set_error("the driver has no cuTensorMapEncodeTiled");
    return B200C_ERR_CUDA;
  }
  const cuuint64_t dims[3] = {(cuuint64_t)channels, (cuuint64_t)heads, (cuuint64_t)rows};
  // a stride that no coordinate uses still has to be a valid one
  const cuuint64_t strides[2] = {(cuuint64_t)(heads > 1 ? head_stride : 128) * 2, (cuuint64_t)(rows > 1 ? row_stride : 128) * 2};
  const cuuint32_t box[3] = {64, 1, (cuuint32_t)box_rows}, step[3] = {1, 1, 1};
  const CUresult r = encode(map, dtype == B200C_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                            3, (void *)base, dims, strides, box, step, CU_TENSOR_MAP_INTERLEAVE_NONE,
                            CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) {
    set_error("cuTensorMapEncodeTiled failed: %d", (int)r);
    return B200C_ERR_CUDA;
  }
  return B200C_OK;
}

// 16-byte rows that a tensor map can describe
static bool at_side(const void *base, int64_t rows, int heads, int64_t row_stride, int64_t head_stride) {
  const auto fits = [](int64_t s) { return s > 0 && s % 8 == 0 && s < (1ll << 38); };
  return ((uintptr_t)base & 15) == 0 && (rows <= 1 || fits(row_stride)) && (heads <= 1 || fits(head_stride));
}

bool attention_tensor_applicable(const b200c_attention_t &p) {
  constexpr int64_t most = 0x7fffffffLL - 1024;  // column numbers of a step past the last stay in 32 bits
  return p.dtype != B200C_F32 && p.channels % 8 == 0 && !(p.cap > AT_MAX_FAST_CAP) && p.m > 0 && p.n > 0 && p.m < most && p.n < most &&
         at_side(p.q, p.m, p.heads, p.q_row, p.q_head) && at_side(p.k, p.n, p.groups, p.k_row, p.k_head) &&
         at_side(p.v, p.n, p.groups, p.v_row, p.v_head);
}

// Up to 32 channels and 128 rows per example on average (either side) the kernels of attention_short.cuh are taken.  Measured
// on 60000 rows, 8 heads, three coordinates, bfloat16, forward / gradient in us, 128-row tiles against 16-row ones:
//   32 channels: 16 rows 185 / 437, 125 / 254;  64 rows 220 / 488, 151 / 331;  128 rows 251 / 567, 208 / 463;
//                192 rows 277 / 633, 266 / 594
//   64 channels: 16 rows 188 / 465, 198 / 471;  64 rows 220 / 510, 250 / 602
constexpr int64_t AT_SHORT_ROWS = 128;
constexpr int AT_SHORT_CHANNELS = 32;
static bool is_short(const b200c_attention_t &p) {
  return p.channels <= AT_SHORT_CHANNELS && p.m <= AT_SHORT_ROWS * p.num_segments &&
         p.n <= AT_SHORT_ROWS * p.num_segments;
}

// A small call leaves most SMs without a block of 128 rows: the columns are dealt out to several, 128 and more to each, as long
// as that fills the SMs, and a second kernel joins them (one cloud of 1024 points, 4 heads: 33 -> 25 us).
int attention_tensor_splits(const b200c_attention_t &p) {
  if (!attention_tensor_applicable(p) || is_short(p)) return 1;
  const int64_t blocks = (p.m + AT_ROWS - 1) / AT_ROWS * p.heads;
  int64_t splits = 148 / blocks;
  const int64_t most = p.n / p.num_segments / 128;
  if (splits > most) splits = most;
  return (int)(splits < 1 ? 1 : splits > 16 ? 16 : splits);
}

int launch_attention_tensor_forward(const AttnArgs &a) {
  const bool bf16 = a.p.dtype == B200C_BF16;
  if (a.splits > 1) {
    const int st = bf16 ? attention_tensor_forward_bf16(a) : attention_tensor_forward_f16(a);
    return st != B200C_OK ? st : launch_attention_join(a);
  }
  if (is_short(a.p)) return bf16 ? attention_short_forward_bf16(a) : attention_short_forward_f16(a);
  return bf16 ? attention_tensor_forward_bf16(a) : attention_tensor_forward_f16(a);
}

int launch_attention_tensor_backward(const AttnArgs &a) {
  const bool bf16 = a.p.dtype == B200C_BF16, brief = is_short(a.p);
  if (a.dq) {
    const int st = brief ? bf16 ? attention_short_dq_bf16(a) : attention_short_dq_f16(a)
                         : bf16 ? attention_tensor_dq_bf16(a) : attention_tensor_dq_f16(a);
    if (st != B200C_OK) return st;
  }
  if (!a.dk) return B200C_OK;
  if (brief) return bf16 ? attention_short_dkv_bf16(a) : attention_short_dkv_f16(a);
  return bf16 ? attention_tensor_dkv_bf16(a) : attention_tensor_dkv_f16(a);
}

}  // namespace b200c
