// rg_sm100_pair.cuh -- inline-PTX wrappers for tcgen05 on CTA pairs (cta_group::2): two SMs
// of a cluster work on one tile, each holding half of A, half of B and half of D.
#pragma once
#include "rg_sm100.cuh"

namespace rg {
namespace sm100 {

__device__ __forceinline__ uint32_t cluster_ctarank() {
  uint32_t r;
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// The shared::cluster address of `p` (an address of this CTA's shared memory) in CTA `rank`.
__device__ __forceinline__ uint32_t cluster_addr(const void* p, uint32_t rank) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(smem_addr(p)), "r"(rank));
  return r;
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(addr) : "memory");
}
// Both CTAs' allocating warps call these.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst_smem, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst_smem)),
               "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}
// 32 lanes x 32 bits, 32 consecutive columns per thread.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, "
      "%15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
        "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
        "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}

// ---- issued by one elected lane of a converged warp -----------------------------------
// Every lane of the warp calls these with the same arguments, and one lane issues (always the
// same one: tcgen05.commit covers the products of the thread that issued them).  The copies and
// products take their operands from uniform registers, which the compiler can fill ahead in
// converged code; inside `if (lane == 0)` each operand is moved there one by one: a product then
// took about 80 clocks of its thread and a copy about 250, more than their execution.
__device__ __forceinline__ void expect_tx_elect(uint64_t* bar, uint32_t bytes) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n}" ::"r"(smem_addr(bar)),
      "r"(bytes)
      : "memory");
}
__device__ __forceinline__ void arrive_elect(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n @q mbarrier.arrive.shared::cta.b64 _, [%0];\n}" ::"r"(
          smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void tma_load_2d_elect(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int32_t x,
                                                  int32_t y) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], "
      "[%2];\n}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void tma_load_4d_elect(uint32_t dst, const CUtensorMap* map, uint64_t* bar, int32_t x,
                                                  int32_t y, int32_t z, int32_t w) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%3, %4, %5, %6}], [%2];\n}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(smem_addr(bar)), "r"(x), "r"(y), "r"(z), "r"(w)
      : "memory");
}
// Completes on a barrier of either CTA of the pair (`bar`: its shared::cluster address).
__device__ __forceinline__ void tma_load_2d_pair_elect(uint32_t dst, const CUtensorMap* map, uint32_t bar, int32_t x,
                                                       int32_t y) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], "
      "[%1, {%3, %4}], [%2];\n}" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(x), "r"(y)
      : "memory");
}
// D[tmem] (+)= A[smem] B[smem]^T, i8: one CTA's product, and a pair's (256 rows over both CTAs,
// issued by the even one).
__device__ __forceinline__ void mma_i8_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_i8_pair_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                                  uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// 16-bit operands, A from shared memory or from TMEM.
__device__ __forceinline__ void mma_16_ss_elect(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ void mma_16_ts_elect(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc,
                                                uint32_t accumulate) {
  asm volatile(
      "{\n .reg .pred p, q;\n elect.sync _|q, 0xffffffff;\n setp.ne.b32 p, %4, 0;\n"
      " @q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Arrive on `bar` (of this CTA; of both CTAs of the pair) once every prior product of the
// issuing lane has completed.
__device__ __forceinline__ void commit_elect(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n}" ::"r"(smem_addr(bar))
      : "memory");
}
__device__ __forceinline__ void commit_pair_elect(uint64_t* bar) {
  asm volatile(
      "{\n .reg .pred q;\n elect.sync _|q, 0xffffffff;\n"
      " @q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n}" ::"r"(
          smem_addr(bar)),
      "h"((uint16_t)3)
      : "memory");
}
// mbar_wait_tight by a converged warp, which stays converged.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort, uint64_t limit_ns) {
  return __all_sync(0xffffffffu, mbar_wait_tight(bar, parity, abort, limit_ns));
}

}  // namespace sm100
}  // namespace rg
