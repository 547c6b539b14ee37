// Warp-wide matrix products (16 x 8 x 16, 16-bit operands, fp32 sums) and the shared-memory tiles they read, for the
// attention kernels whose rows are too few for a tcgen05 tile of 128.
#pragma once

#include <type_traits>

#include "attention.cuh"
#include "tcgen05.cuh"

namespace b200c {

template <typename T>
__device__ __forceinline__ void aw_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  else
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void aw_ldmatrix(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void aw_ldmatrix_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
template <typename T>
__device__ __forceinline__ uint32_t aw_pack(float lo, float hi) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  } else {
    const __half2 v = __floats2half2_rn(lo, hi);
    return *reinterpret_cast<const uint32_t *>(&v);
  }
}
template <typename T>
__device__ __forceinline__ float2 aw_unpack(uint32_t v) {
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
  else
    return __half22float2(*reinterpret_cast<const __half2 *>(&v));
}

// Byte offset of 16-byte chunk c of row r in a tile of rows of CP 16-bit values: eight rows of one chunk, which a
// matrix load takes, and eight chunks of one row, which a copy writes, lie in different banks.
template <int CP>
__device__ __forceinline__ uint32_t aw_at(int r, int c) {
  return (uint32_t)(r * (CP * 2) + ((CP == 32 ? c ^ ((r >> 1) & 3) : c ^ (r & 7)) << 4));
}

// 16 rows of 16 channels (tile t of 16) as the first operand
template <int CP>
__device__ __forceinline__ void aw_rows(uint32_t (&f)[4], uint32_t tile, int t, int lane) {
  aw_ldmatrix(f, tile + aw_at<CP>(lane & 15, 2 * t + (lane >> 4)));
}
// columns 8 n .. 8 n + 15 of 16 channels as two second operands: (f0, f1) and (f2, f3)
template <int CP>
__device__ __forceinline__ void aw_cols(uint32_t (&f)[4], uint32_t tile, int n, int t, int lane) {
  aw_ldmatrix(f, tile + aw_at<CP>(n * 8 + (lane & 7) + ((lane & 16) >> 1), 2 * t + ((lane >> 3) & 1)));
}
// rows 16 t .. 16 t + 15 of channels 8 n .. 8 n + 15, transposed, as two second operands
template <int CP>
__device__ __forceinline__ void aw_sums(uint32_t (&f)[4], uint32_t tile, int t, int n, int lane) {
  aw_ldmatrix_t(f, tile + aw_at<CP>(t * 16 + (lane & 15), n + (lane >> 4)));
}

}  // namespace b200c
