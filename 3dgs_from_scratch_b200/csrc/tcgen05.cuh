// tcgen05.cuh -- the fifth-generation tensor core's instructions used by the
// matrix kernels: operands in shared memory behind 64-bit descriptors, fp32
// accumulators in tensor memory.
#pragma once

#include "cluster.cuh"

namespace gs {
namespace tc {

// CTAS = 1: a block by itself. CTAS = 2: the two blocks of a cluster work on
// one tile (cta_group::2): each holds its half of A's rows and of B's in its
// own shared memory and its half of the accumulator's rows in its own tensor
// memory; block 0 issues for both.

// One lane of a converged warp.
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
  return p != 0;
}

// Tensor memory: `columns` (a power of two from 32) of 128 lanes x 32 bits,
// address written to shared memory; one whole warp (of each block) allocates
// and frees.
template <int CTAS>
__device__ __forceinline__ void tmem_alloc(uint32_t *dst, uint32_t columns) {
  if (CTAS == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  } else {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(dst)),
                 "r"(columns)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
  }
}
template <int CTAS>
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t columns) {
  if (CTAS == 1)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
  else
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(columns));
}

__device__ __forceinline__ void fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// Shared-memory descriptor of an operand in 128-byte swizzled rows: start
// address, leading and stride byte offsets (all / 16), the fixed bits and the
// swizzle mode. For K-major operands `stride` leads from 8 rows to the next
// 8; for MN-major ones `lead` leads from 64 elements along MN to the next 64,
// `stride` from 8 K rows to the next 8.
__device__ __forceinline__ uint64_t descriptor(uint32_t addr, uint32_t lead, uint32_t stride) {
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)((lead >> 4) & 0x3FFF) << 16) |
         ((uint64_t)((stride >> 4) & 0x3FFF) << 32) | (1ull << 46) | (2ull << 61);
}

// Instruction descriptor: fp16 operands, fp32 accumulator, tile m x n, each
// operand K-major or (mn) MN-major.
__host__ __device__ constexpr uint32_t instruction_f16(int m, int n, bool a_mn, bool b_mn) {
  return (1u << 4) | ((a_mn ? 1u : 0u) << 15) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// D = A B (ADD: D += A B) over 16 elements of K; one lane issues it for the
// block or pair. What kind of instruction it is is known at compile time: with
// the instruction descriptor or the predicate in registers each issue took
// about 100 cycles, 48 (64, 128) otherwise for N = 64 (128, 256).
template <int CTAS, bool ADD, uint32_t INSTRUCTION>
__device__ __forceinline__ void mma_f16(uint32_t d, uint64_t a, uint64_t b) {
  if (CTAS == 1)
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "n"(INSTRUCTION), "n"(ADD ? 1 : 0)
        : "memory");
  else
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.u32 p, %4, 0;\n"
        " tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "n"(INSTRUCTION), "n"(ADD ? 1 : 0)
        : "memory");
}

__device__ __forceinline__ void arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_addr(bar)) : "memory");
}

// Registers handed between the warpgroups of a block: every warp of a group
// (four from a multiple of four on) calls one of these.
template <int N>
__device__ __forceinline__ void registers_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void registers_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}

// The same on the barrier at `bar`'s place in block `rank` of the cluster. With
// an explicit release at cluster scope every arrival took about 1 us; nothing
// that this orders is written by the arriving thread (bulk copies and MMAs
// complete on barriers of their own before it).
__device__ __forceinline__ void arrive_at(uint64_t *bar, uint32_t rank) {
  asm volatile(
      "{\n .reg .b32 a;\n mapa.shared::cluster.u32 a, %0, %1;\n"
      " mbarrier.arrive.shared::cluster.b64 _, [a];\n}\n" ::"r"(smem_addr(bar)),
      "r"(rank)
      : "memory");
}

// Bounded wait that also orders what the other block did before it arrived.
__device__ __forceinline__ bool wait_cluster(uint64_t *bar, uint32_t parity) {
  for (uint32_t i = 0; i < kSpinLimit; ++i) {
    uint32_t ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
        " selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(smem_addr(bar)), "r"(parity)
        : "memory");
    if (ok) return true;
  }
  return false;
}

// Arrives on the barrier (of both blocks of a pair) when the thread's MMAs so
// far are done.
template <int CTAS>
__device__ __forceinline__ void commit(uint64_t *bar) {
  if (CTAS == 1)
    asm volatile(
        "tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_addr(bar))
        : "memory");
  else
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_addr(bar)),
        "h"((uint16_t)3)
        : "memory");
}

// 32 columns of the warp's 32 lanes: thread l gets row l, columns addr... The
// wait belongs to the same statement, so that nothing is read before it.
__device__ __forceinline__ void load_columns(uint32_t addr, float (&v)[32]) {
  uint32_t r[32];
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
}

// The sum of 32 columns of two accumulators, both on their way at once.
__device__ __forceinline__ void load_sum(uint32_t addr, uint32_t other, float (&v)[32]) {
  uint32_t r[32], q[32];
#define GS_TC_LD(R, ADDR)                                                                                  \
  asm volatile(                                                                                            \
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "                                                            \
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "                            \
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"            \
      : "=r"(R[0]), "=r"(R[1]), "=r"(R[2]), "=r"(R[3]), "=r"(R[4]), "=r"(R[5]), "=r"(R[6]), "=r"(R[7]),    \
        "=r"(R[8]), "=r"(R[9]), "=r"(R[10]), "=r"(R[11]), "=r"(R[12]), "=r"(R[13]), "=r"(R[14]),           \
        "=r"(R[15]), "=r"(R[16]), "=r"(R[17]), "=r"(R[18]), "=r"(R[19]), "=r"(R[20]), "=r"(R[21]),         \
        "=r"(R[22]), "=r"(R[23]), "=r"(R[24]), "=r"(R[25]), "=r"(R[26]), "=r"(R[27]), "=r"(R[28]),         \
        "=r"(R[29]), "=r"(R[30]), "=r"(R[31])                                                              \
      : "r"(ADDR)                                                                                          \
      : "memory")
  GS_TC_LD(r, addr);
  GS_TC_LD(q, other);
#undef GS_TC_LD
  // The wait takes the registers along, so that nothing reads them before it.
#define GS_TC_PASS(R)                                                                                      \
  asm volatile(""                                                                                          \
               : "+r"(R[0]), "+r"(R[1]), "+r"(R[2]), "+r"(R[3]), "+r"(R[4]), "+r"(R[5]), "+r"(R[6]),       \
                 "+r"(R[7]), "+r"(R[8]), "+r"(R[9]), "+r"(R[10]), "+r"(R[11]), "+r"(R[12]), "+r"(R[13]),   \
                 "+r"(R[14]), "+r"(R[15]), "+r"(R[16]), "+r"(R[17]), "+r"(R[18]), "+r"(R[19]),             \
                 "+r"(R[20]), "+r"(R[21]), "+r"(R[22]), "+r"(R[23]), "+r"(R[24]), "+r"(R[25]),             \
                 "+r"(R[26]), "+r"(R[27]), "+r"(R[28]), "+r"(R[29])                                        \
               :                                                                                           \
               : "memory");                                                                                \
  asm volatile("" : "+r"(R[30]), "+r"(R[31])::"memory")
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
  GS_TC_PASS(r);
  GS_TC_PASS(q);
#undef GS_TC_PASS
#pragma unroll
  for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]) + __uint_as_float(q[i]);
}

}  // namespace tc
}  // namespace gs
