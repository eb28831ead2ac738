// The fifth-generation tensor cores (tcgen05) as the tile kernels use them: products of an operand
// in tensor memory and one in shared memory, f32 sums in tensor memory, a thread per row of it;
// and packed f32 arithmetic, two values an instruction.
#pragma once

#include "hv_common.cuh"

namespace hv {

HV_DEV uint64_t smem_desc(uint32_t addr) {      // 128-byte swizzle, 1024 bytes per 8 rows
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}
// One lane of a whole warp issues: the warp stays together, so that the descriptors are uniform
// registers, which the instruction wants (in a branch of one lane it took 190 cycles to issue
// a product that runs for 64).
HV_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t desc, bool add, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :: "r"(d), "r"(a), "l"(b), "r"(desc), "r"((uint32_t)add), "r"(leader) : "memory");
}
HV_DEV void mma_commit(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      :: "r"(bar), "r"(leader) : "memory");
}
HV_DEV uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
HV_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
HV_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
HV_DEV void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define HV_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define HV_P4(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3])
#define HV_W4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
// Columns of this thread's row: begun here, in hand after tmem_wait. One load is under way
// while the columns before it are worked on.
HV_DEV void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : HV_R4(v, 0), HV_R4(v, 4), HV_R4(v, 8), HV_R4(v, 12), HV_R4(v, 16), HV_R4(v, 20),
        HV_R4(v, 24), HV_R4(v, 28)
      : "r"(at) : "memory");
}
HV_DEV void tmem_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : HV_P4(v, 0), HV_P4(v, 4), HV_P4(v, 8), HV_P4(v, 12), HV_P4(v, 16), HV_P4(v, 20),
                 HV_P4(v, 24), HV_P4(v, 28) :: "memory");
}
HV_DEV void tmem_ld16(uint32_t at, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : HV_R4(v, 0), HV_R4(v, 4), HV_R4(v, 8), HV_R4(v, 12) : "r"(at) : "memory");
}
HV_DEV void tmem_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : HV_P4(v, 0), HV_P4(v, 4), HV_P4(v, 8), HV_P4(v, 12) :: "memory");
}
HV_DEV void tmem_ld8(uint32_t at, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : HV_R4(v, 0), HV_R4(v, 4) : "r"(at) : "memory");
}
HV_DEV void tmem_wait(uint32_t (&v)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : HV_P4(v, 0), HV_P4(v, 4) :: "memory");
}
HV_DEV void tmem_st8(uint32_t at, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :: "r"(at), HV_W4(v, 0), HV_W4(v, 4) : "memory");
}
HV_DEV void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(at), HV_W4(v, 0), HV_W4(v, 4), HV_W4(v, 8), HV_W4(v, 12) : "memory");
}
HV_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

HV_DEV void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
}
HV_DEV uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
HV_DEV float2 unpair(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
HV_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
HV_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
HV_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

}  // namespace hv
