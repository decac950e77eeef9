// Thin wrappers around the fifth-generation tensor core instructions (sm_100a): tensor memory,
// tcgen05.mma with bf16 operands and fp32 accumulators, and their fences.
#pragma once

#include "common.cuh"

namespace asterq {
namespace tc {

// ---------------------------------------------------------------------------
// Tensor memory: 128 lanes x 512 columns of 32 bits.  An address has the lane in bits 16-31 and the
// column in bits 0-15; a warp reaches the 32 lanes from 32 (warp % 4) on.
// ---------------------------------------------------------------------------
ASTERQ_DEVICE void alloc512(uint32_t smem_slot) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_slot) : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
ASTERQ_DEVICE void dealloc512(uint32_t addr) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(addr) : "memory");
}
ASTERQ_DEVICE void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
ASTERQ_DEVICE void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
ASTERQ_DEVICE void wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
ASTERQ_DEVICE void wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// thread i of the warp <-> lane i, 32 or 16 consecutive columns
ASTERQ_DEVICE void ld32(uint32_t (&r)[32], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,"
      "%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr));
}
ASTERQ_DEVICE void st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
      "%31,%32};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
ASTERQ_DEVICE void ld16(uint32_t (&r)[16], uint32_t addr) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr));
}
ASTERQ_DEVICE void st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// 16 lanes from the address's on, four columns four times over: thread t <-> lanes t / 4 and t / 4 + 8,
// column t % 4 (r0, r1), then the next four columns (r2, r3), ..: the layout of ldmatrix's 8 x 8 matrices.
// A store takes a warp some 40 cycles whatever its width.
ASTERQ_DEVICE void st_16x128b_x4(uint32_t addr, uint32_t r0, uint32_t r1, uint32_t r2, uint32_t r3, uint32_t r4,
                                 uint32_t r5, uint32_t r6, uint32_t r7) {
  asm volatile("tcgen05.st.sync.aligned.16x128b.x4.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(addr), "r"(r0), "r"(r1),
               "r"(r2), "r"(r3), "r"(r4), "r"(r5), "r"(r6), "r"(r7)
               : "memory");
}

// ---------------------------------------------------------------------------
// Operand descriptors for tiles in shared memory with the 128-byte swizzle: rows of 128 bytes,
// 64 16-bit values, 1024-byte aligned groups of eight rows.
//   k_major   rows are M or N, the 64 values run along K; a tile wider than 64 is several boxes, each
//             with a descriptor of its own
//   mn_major  rows are K, the 64 values run along M or N; boxes of the next 64 are `box_bytes` on
// ---------------------------------------------------------------------------
// A descriptor here is its low word: the start address and the stride between boxes, in 16-byte units.
// The high word is the same for all of them: 1024 bytes between groups of eight rows, the swizzle.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
ASTERQ_DEVICE uint32_t desc_k_major(uint32_t smem) { return ((smem & 0x3ffff) >> 4) | (1u << 16); }
ASTERQ_DEVICE uint32_t desc_mn_major(uint32_t smem, uint32_t box_bytes) {
  return ((smem & 0x3ffff) >> 4) | ((box_bytes >> 4) << 16);
}
// packed bf16 arithmetic, rounded once
ASTERQ_DEVICE uint32_t mul_bf162(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}
ASTERQ_DEVICE uint32_t fma_bf162(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}
ASTERQ_DEVICE uint32_t neg_bf162(uint32_t a) { return a ^ 0x80008000u; }

// bf16 x bf16 -> fp32, A K-major, M = 128
constexpr uint32_t idesc_bf16(int n, bool b_mn_major) {
  return (1u << 4) | (1u << 7) | (1u << 10) | ((b_mn_major ? 1u : 0u) << 16) | ((uint32_t)(n / 8) << 17) |
         ((128u / 16) << 24);
}

// one lane of a converged warp; products are issued under it so that their operands stay in uniform
// registers (issued from a divergent thread in a rolled loop they took 110 cycles each instead of 64)
ASTERQ_DEVICE bool elect() {
  uint32_t p;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}" : "=r"(p));
  return p;
}

// D[tmem] (+)= A B, both operands in shared memory; issued by one thread
ASTERQ_DEVICE void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 a, b;\n setp.ne.u32 p, %4, 0;\n mov.b64 a, {%1, %5};\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(kDescHigh)
      : "memory");
}
// A in tensor memory: lane = row, 32-bit column = two consecutive k
ASTERQ_DEVICE void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 b;\n setp.ne.u32 p, %4, 0;\n mov.b64 b, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)add), "r"(kDescHigh)
      : "memory");
}
// the mbarrier gets one arrival when all MMAs issued so far by this thread are done
ASTERQ_DEVICE void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

}  // namespace tc
}  // namespace asterq
