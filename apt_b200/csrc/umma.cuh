// The fifth-generation tensor cores from inside a kernel: barriers in shared memory with bounded waits, tiled copies, tensor memory
// and products of tiles (tcgen05).
#pragma once

#include <cuda.h>

#include "common.cuh"

namespace apt {

__device__ __forceinline__ uint32_t shared_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void barrier_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void barrier_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void barrier_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool barrier_over(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile("{ .reg .pred p; mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
               : "=r"(done)
               : "r"(bar), "r"(parity)
               : "memory");
  return done;
}
// Until the barrier's phase of this parity is over, or for that many polls, each of which may suspend for a while itself. False: somebody
// has given up (*gave_up); nothing may be used then but what ends the kernel. The first poll stands by itself: with the count in front of it, products of
// 65536 x 1024 -> 1024 fp32 take 820 us, not 807.
__device__ __forceinline__ bool barrier_wait(uint32_t bar, uint32_t parity, volatile int* gave_up, int polls) {
  if (polls && barrier_over(bar, parity)) return true;
  for (int i = 1; i < polls; ++i) {
    if (barrier_over(bar, parity)) return true;
    if ((i & 63) == 63 && *gave_up) return false;
  }
  *gave_up = 1;
  return false;
}
// For what is in flight and has to land before a block ends, whoever has given up.
constexpr int kLastPolls = 1 << 20;
__device__ __forceinline__ void barrier_settle(uint32_t bar, uint32_t parity) {
  int nobody = 0;
  barrier_wait(bar, parity, &nobody, kLastPolls);
}

// True for one lane of a converged warp, which the compiler knows to be one: products and copies, which take their operands in uniform
// registers, are issued as they are then. Under a condition on the lane's number a product took 140 cycles to issue.
__device__ __forceinline__ bool one_of_warp() {
  uint32_t is;
  asm volatile("{ .reg .pred p; elect.sync _|p, 0xffffffff; selp.u32 %0, 1, 0, p; }" : "=r"(is));
  return is;
}

// Boxes of a row-major matrix, or of a stack of them, on their way to shared memory; `bar` counts their bytes.
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int y, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(dst),
               "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y)
               : "memory");
}
__device__ __forceinline__ void copy_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t bar) {
  asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
               "l"((uint64_t)map), "r"(bar), "r"(x), "r"(y), "r"(z)
               : "memory");
}
// What ordinary stores of this thread wrote to shared memory, for the tensor cores.
__device__ __forceinline__ void fence_for_tensor_cores() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- tensor memory: 128 lanes of 512 columns of 32 bits ----------------------------
__device__ __forceinline__ void tmem_alloc(uint32_t slot, uint32_t columns) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(slot), "r"(columns) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t base, uint32_t columns) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(base), "r"(columns));
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// 32 columns of the calling warp's 32 lanes: a lane has a row.
__device__ __forceinline__ void tmem_load_32(uint32_t at, float (&v)[32]) {
  uint32_t* const r = (uint32_t*)v;
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
      "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]),
        "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
        "=r"(r[31])
      : "r"(at));
}
// Until the loads so far are done; what was loaded is used behind settled() of it only (the registers are written when the load is done, which the
// compiler does not know).
__device__ __forceinline__ void tmem_wait_loads() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void settled(float& v) { asm volatile("" : "+f"(v)); }
template <int N>
__device__ __forceinline__ void settled(float (&v)[N]) {
#pragma unroll
  for (int k = 0; k < N; ++k) settled(v[k]);
}

// ---- products ----------------------------------------------------------------------
// A tile in shared memory, its 16-byte slices swizzled within rows of 128 or 64 bytes as the copies leave them. Along the
// contraction (K): rows of the tile follow one another at the row's length, eight of them `stride` bytes apart. Across it (MN): a row
// has 64 elements of one k; eight k's are `stride` bytes apart, the next 64 elements `leading` bytes.
constexpr uint64_t kSwizzle128 = 2ull << 61, kSwizzle64 = 4ull << 61;
__device__ __forceinline__ uint64_t tile_descriptor(uint32_t at, uint32_t leading, uint32_t stride, uint64_t swizzle) {
  return (uint64_t)((at & 0x3ffff) >> 4) | (uint64_t)(leading >> 4) << 16 | (uint64_t)(stride >> 4) << 32 | 1ull << 46 | swizzle;
}
// Sums in fp32 of products of bf16 (or f16) tiles, m x n; a_mn, b_mn: rows of the operand run across the contraction.
__host__ __device__ inline uint32_t product_descriptor(bool bf16, bool a_mn, bool b_mn, int m, int n) {
  return 1u << 4 | (bf16 ? 1u << 7 | 1u << 10 : 0u) | (a_mn ? 1u << 15 : 0u) | (b_mn ? 1u << 16 : 0u) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24;
}
// By one thread: d (+)= a b over 16 elements of the contraction.
__device__ __forceinline__ void tile_product(uint32_t d, uint64_t a, uint64_t b, uint32_t what, bool add) {
  asm volatile(
      "{ .reg .pred p; setp.ne.u32 p, %4, 0; tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p; }" ::"r"(d), "l"(a), "l"(b), "r"(what),
      "r"((uint32_t)add)
      : "memory");
}
// By the same thread: the barrier is arrived at once when all products so far are done.
__device__ __forceinline__ void products_done(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

}  // namespace apt
