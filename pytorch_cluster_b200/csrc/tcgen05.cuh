// Small wrappers of the sm_100a instructions the tensor-core attention kernels use: mbarriers with bounded waits,
// bulk tensor copies (TMA), tensor memory and tcgen05.mma.
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace b200c {

__device__ __forceinline__ uint32_t t5_smem(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

// One lane of the warp, the same every time.  The descriptors of a product live in uniform registers: issued by an
// elected lane in code that the whole warp runs, they stay there; behind a test of the lane number each would be moved
// over first (measured: 85 cycles per product against about 20).
__device__ __forceinline__ bool t5_elect() {
  uint32_t one;
  asm volatile("{\n.reg .pred p;\nelect.sync _|p, 0xffffffff;\nselp.u32 %0, 1, 0, p;\n}" : "=r"(one));
  return one != 0;
}
// the warp's number as a value the compiler knows to be the same in all lanes
__device__ __forceinline__ int t5_warp() { return __shfl_sync(FULL_MASK, (int)(threadIdx.x >> 5), 0); }

__device__ __forceinline__ void t5_mbar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(t5_smem(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void t5_mbar_arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(t5_smem(bar)) : "memory");
}
// raises the bytes the current phase waits for, without arriving
__device__ __forceinline__ void t5_mbar_expect(uint64_t *bar, uint32_t bytes) {
  asm volatile("mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(t5_smem(bar)), "r"(bytes) : "memory");
}
__device__ __forceinline__ bool t5_mbar_try(uint64_t *bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}"
               : "=r"(done)
               : "r"(t5_smem(bar)), "r"(parity)
               : "memory");
  return done != 0;
}
// polls of a wait, of some ten nanoseconds each; a step takes a microsecond or two
constexpr int T5_SPIN_LIMIT = 1 << 22;
// Waits for the phase of the given parity.  A parity tells two neighbouring phases apart, no more: a caller must know
// that the phase before is over and that the one after cannot end before it has gone on.  Gives up after T5_SPIN_LIMIT
// polls, or when another thread of the block did (*failed), and says so.
__device__ __forceinline__ bool t5_mbar_wait(uint64_t *bar, uint32_t parity, volatile int *failed) {
  if (t5_mbar_try(bar, parity)) return true;
  for (int i = 0; i < T5_SPIN_LIMIT; ++i) {
    if (t5_mbar_try(bar, parity)) return true;
    if (*failed) return false;
  }
  *failed = 1;
  return false;
}

// The same for a warp that has nothing else to do and whose answer is not waited for at once: a loop of few
// instructions, asleep between its looks, which otherwise take issue slots from the warps that work (forward 692 -> 641
// us).
__device__ __forceinline__ bool t5_mbar_wait_idle(uint64_t *bar, uint32_t parity, volatile int *failed) {
  const uint32_t at = t5_smem(bar);
  uint32_t over = 0;
  for (int i = 0; i < T5_SPIN_LIMIT / 512; ++i) {
    // up to 64 looks
    asm volatile(
        "{\n.reg .pred p;\n.reg .u32 n;\nmov.u32 n, 64;\n"
        "LOOK_%=:\n"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n"
        "@p bra OVER_%=;\n"
        "nanosleep.u32 60;\n"
        "sub.u32 n, n, 1;\nsetp.ne.u32 p, n, 0;\n@p bra LOOK_%=;\n"
        "OVER_%=:\nselp.u32 %0, 1, 0, p;\n}"
        : "=r"(over)
        : "r"(at), "r"(parity)
        : "memory");
    if (over || *failed) break;
  }
  const bool all = __all_sync(FULL_MASK, over != 0);
  if (!all) *failed = 1;
  return all;
}
// the same by a whole warp, with one answer
__device__ __forceinline__ bool t5_mbar_wait_warp(uint64_t *bar, uint32_t parity, volatile int *failed) {
  return __all_sync(FULL_MASK, t5_mbar_wait(bar, parity, failed));
}

// tells the host that a wait of this block ran out
__device__ __forceinline__ void t5_report(int *word) {
  if (word == nullptr) return;
  *(volatile int *)word = 1;
  __threadfence_system();
}

// two barriers at once (the second only if `second`): where both are over already, one round trip instead of two
__device__ __forceinline__ bool t5_mbar_wait_both(uint64_t *a, uint32_t pa, uint64_t *b, uint32_t pb, bool second,
                                                  volatile int *failed) {
  const bool ta = t5_mbar_try(a, pa), tb = !second || t5_mbar_try(b, pb);
  if (__all_sync(FULL_MASK, ta && tb)) return true;
  return t5_mbar_wait_warp(a, pa, failed) && (!second || t5_mbar_wait_warp(b, pb, failed));
}

// a box of a 3-d tensor to shared memory, without multicast
__device__ __forceinline__ void t5_tma_3d(void *dst, const CUtensorMap *map, int c0, int c1, int c2, uint64_t *bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
      ::"r"(t5_smem(dst)), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(t5_smem(bar))
      : "memory");
}

__device__ __forceinline__ void t5_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void t5_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void t5_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void t5_commit(uint64_t *bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(t5_smem(bar))
               : "memory");
}

// Shared-memory operand descriptors, 128-byte swizzle (8 rows of 128 bytes are one 1024-byte block).
//   K-major: rows of 64 16-bit values along K; next 8 rows 1024 bytes on.
//   MN-major: rows of 64 values along M or N, one row per K; next 8 K 1024 bytes on, next 64 values `mn_block` on.
__device__ __forceinline__ uint64_t t5_desc(uint32_t saddr, uint32_t mn_block = 16) {
  uint64_t d = 0;
  d |= (uint64_t)((saddr >> 4) & 0x3fffu);
  d |= (uint64_t)(mn_block >> 4) << 16;
  d |= (uint64_t)(1024u >> 4) << 32;
  d |= (uint64_t)1 << 46;
  d |= (uint64_t)2 << 61;
  return d;
}
// kind::f16, D fp32, A and B of one 16-bit type, M = 128
__host__ __device__ constexpr uint32_t t5_idesc(bool bf16, int n, bool b_mn_major) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((b_mn_major ? 1u : 0u) << 16) |
         ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24);
}
__device__ __forceinline__ void t5_mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}
__device__ __forceinline__ void t5_mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate) {
  asm volatile(
      "{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"((uint32_t)accumulate)
      : "memory");
}

// Waits for the thread's loads from tensor memory.  The values pass through the instruction, so that no use of them can
// be moved ahead of it.
__device__ __forceinline__ void t5_wait_ld32(float *v) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]),"+f"(v[1]),"+f"(v[2]),"+f"(v[3]),"+f"(v[4]),"+f"(v[5]),"+f"(v[6]),"+f"(v[7]),
                 "+f"(v[8]),"+f"(v[9]),"+f"(v[10]),"+f"(v[11]),"+f"(v[12]),"+f"(v[13]),"+f"(v[14]),"+f"(v[15]),
                 "+f"(v[16]),"+f"(v[17]),"+f"(v[18]),"+f"(v[19]),"+f"(v[20]),"+f"(v[21]),"+f"(v[22]),"+f"(v[23]),
                 "+f"(v[24]),"+f"(v[25]),"+f"(v[26]),"+f"(v[27]),"+f"(v[28]),"+f"(v[29]),"+f"(v[30]),"+f"(v[31])
               ::"memory");
}

// 32 columns of the thread's lane; the caller waits (t5_wait_ld32) before it reads v
__device__ __forceinline__ void t5_ld32(uint32_t taddr, float *r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,"
      "%28,%29,%30,%31}, [%32];"
      : "=f"(r[0]), "=f"(r[1]), "=f"(r[2]), "=f"(r[3]), "=f"(r[4]), "=f"(r[5]), "=f"(r[6]), "=f"(r[7]), "=f"(r[8]),
        "=f"(r[9]), "=f"(r[10]), "=f"(r[11]), "=f"(r[12]), "=f"(r[13]), "=f"(r[14]), "=f"(r[15]), "=f"(r[16]),
        "=f"(r[17]), "=f"(r[18]), "=f"(r[19]), "=f"(r[20]), "=f"(r[21]), "=f"(r[22]), "=f"(r[23]), "=f"(r[24]),
        "=f"(r[25]), "=f"(r[26]), "=f"(r[27]), "=f"(r[28]), "=f"(r[29]), "=f"(r[30]), "=f"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void t5_st32(uint32_t taddr, const float *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,"
      "%29,%30,%31,%32};" ::"r"(taddr),
      "f"(r[0]), "f"(r[1]), "f"(r[2]), "f"(r[3]), "f"(r[4]), "f"(r[5]), "f"(r[6]), "f"(r[7]), "f"(r[8]), "f"(r[9]),
      "f"(r[10]), "f"(r[11]), "f"(r[12]), "f"(r[13]), "f"(r[14]), "f"(r[15]), "f"(r[16]), "f"(r[17]), "f"(r[18]),
      "f"(r[19]), "f"(r[20]), "f"(r[21]), "f"(r[22]), "f"(r[23]), "f"(r[24]), "f"(r[25]), "f"(r[26]), "f"(r[27]),
      "f"(r[28]), "f"(r[29]), "f"(r[30]), "f"(r[31])
      : "memory");
}
__device__ __forceinline__ void t5_st16(uint32_t taddr, const uint32_t *r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void t5_alloc(uint32_t *where, uint32_t columns) {  // one warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(t5_smem(where)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void t5_dealloc(uint32_t taddr, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(columns));
}

__device__ __forceinline__ float t5_ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float t5_sqrt(float x) {
  float y;
  asm("sqrt.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float t5_rcp(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

}  // namespace b200c
