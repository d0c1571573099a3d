// Thin wrappers of the sm_100a instructions that the matrix kernel uses:
// mbarriers with bounded waits, TMA tile loads, tensor memory and tcgen05.mma.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>

#include <cstdint>

namespace ftb {
namespace sm100 {

// The instructions that one lane of a warp issues take `lead`, true in that
// lane, as their predicate. The whole warp runs up to them in step, which leaves
// their operands in uniform registers; inside a branch that one lane takes,
// each operand is moved there first, 170 cycles for every product.
__device__ __forceinline__ uint32_t smem_addr(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(pred));
  return pred != 0;
}

__device__ __forceinline__ void mbar_init(uint64_t *bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_addr(bar)), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_init_fence() { asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory"); }
__device__ __forceinline__ void mbar_expect(uint64_t *bar, uint32_t bytes, bool lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t"
      "@q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}" ::"r"(smem_addr(bar)),
      "r"(bytes), "r"((uint32_t)lead)
      : "memory");
}
// More bytes for the phase under way, without an arrival.
__device__ __forceinline__ void mbar_expect_more(uint64_t *bar, uint32_t bytes, bool lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %2, 0;\n\t"
      "@q mbarrier.expect_tx.relaxed.cta.shared::cta.b64 [%0], %1;\n\t}" ::"r"(smem_addr(bar)),
      "r"(bytes), "r"((uint32_t)lead)
      : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint64_t *bar, bool lead = true) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "@q mbarrier.arrive.shared::cta.b64 _, [%0];\n\t}" ::"r"(smem_addr(bar)),
      "r"((uint32_t)lead)
      : "memory");
}
__device__ __forceinline__ bool mbar_try(uint64_t *bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(smem_addr(bar)), "r"(parity)
      : "memory");
  return ok != 0;
}

__device__ __forceinline__ uint64_t nanoseconds() {
  uint64_t t;
  asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
  return t;
}

// Waits for the phase, two seconds at most (no tile takes a thousandth of
// that). A wait that runs out sets `gave_up`, which ends every other wait of
// the block.
constexpr uint64_t kWaitLimit = 2000000000;
__device__ __forceinline__ bool mbar_wait(uint64_t *bar, uint32_t parity, volatile uint32_t *gave_up) {
  for (int i = 0; i < 16; ++i)
    if (mbar_try(bar, parity)) return true;
  const uint64_t begin = nanoseconds();
  do {
    if (mbar_try(bar, parity)) return true;
    if (*gave_up) return false;
  } while (nanoseconds() - begin < kWaitLimit);
  *gave_up = 1;
  return false;
}
// The same for copies in flight when the block has given up already.
__device__ __forceinline__ void mbar_settle(uint64_t *bar, uint32_t parity) {
  const uint64_t begin = nanoseconds();
  while (!mbar_try(bar, parity) && nanoseconds() - begin < kWaitLimit) {
  }
}

// A kernel launched to overlap the one before it: everything that reads what
// that one wrote comes after the wait. The one before allows it by `launch_next`.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void launch_next() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

__device__ __forceinline__ void prefetch_map(const CUtensorMap *map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}
// x is the innermost coordinate, in elements; x * element size is a multiple
// of 16 bytes at every call.
__device__ __forceinline__ void tma_load_2d(void *dst, const CUtensorMap *map, uint64_t *bar, int32_t x, int32_t y,
                                            bool lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];\n\t}" ::
          "r"(smem_addr(dst)),
      "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"((uint32_t)lead)
      : "memory");
}
__device__ __forceinline__ void tma_load_3d(void *dst, const CUtensorMap *map, uint64_t *bar, int32_t x, int32_t y,
                                            int32_t z, bool lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %6, 0;\n\t"
      "@q cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}" ::
          "r"(smem_addr(dst)),
      "l"(map), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"((uint32_t)lead)
      : "memory");
}

// A run of bytes: both addresses and the size are multiples of 16.
__device__ __forceinline__ void bulk_load(void *dst, const void *src, uint32_t bytes, uint64_t *bar, bool lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %4, 0;\n\t"
      "@q cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];\n\t}" ::"r"(
          smem_addr(dst)),
      "l"(src), "r"(bytes), "r"(smem_addr(bar)), "r"((uint32_t)lead)
      : "memory");
}

__device__ __forceinline__ void tmem_alloc(uint32_t *at, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(at)), "r"(columns)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// Shared-memory operand whose rows hold 128, 64 or 32 bytes along the inner
// dimension, swizzled over that width; groups of 8 rows are `apart` bytes apart.
__device__ __forceinline__ uint64_t operand(const void *smem, uint32_t row_bytes = 128, uint32_t apart = 1024) {
  const uint64_t layout = row_bytes == 128 ? 2 : row_bytes == 64 ? 4 : 6;
  return (uint64_t)((smem_addr(smem) & 0x3FFFF) >> 4) | ((uint64_t)1 << 16) | ((uint64_t)(apart >> 4) << 32) |
         ((uint64_t)1 << 46) | (layout << 61);
}
// The same swizzle for a byte offset from the start of a group of 8 rows: the
// 16-byte piece is exchanged by the number of its 128 bytes.
__device__ __forceinline__ uint32_t swizzled(uint32_t offset, uint32_t row_bytes) {
  return offset ^ ((offset >> 7 & (row_bytes / 16 - 1)) << 4);
}
// f32 accumulator, both operands bf16 (or both f16), inner dimension contiguous.
__host__ __device__ constexpr uint32_t mma_shape(bool bf16, uint32_t m, uint32_t n) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((n >> 3) << 17) | ((m >> 4) << 24);
}
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b, uint32_t shape, bool add, bool lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.u32 p, %4, 0;\n\tsetp.ne.u32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(shape), "r"((uint32_t)add), "r"((uint32_t)lead)
      : "memory");
}
// The barrier gets one arrival when all MMAs issued before have finished.
__device__ __forceinline__ void mma_commit(uint64_t *bar, bool lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.u32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_addr(bar)),
      "r"((uint32_t)lead)
      : "memory");
}

__device__ __forceinline__ void tmem_load16(uint32_t at, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, "
      "[%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(at));
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

}  // namespace sm100
}  // namespace ftb
