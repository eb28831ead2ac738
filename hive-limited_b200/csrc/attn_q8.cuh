// Tensor-pipe pieces of the attention over the 8-bit cache (kv_q8.cuh).
//
// A code is an integer of at most 127, exact in binary16, so K and V enter the f16 tensor
// pipe without rounding and the scale of a block multiplies its sums in f32. The f32 factors
// (queries and weights) enter as two binary16 terms, x = hi + lo with hi = f16(x) and
// lo = f16(x - hi), scaled by a power of two so that the largest is near 2^14: together 22
// bits, and the products accumulate in f32.
#pragma once

#include "hv_wait.cuh"
#include "kv_q8.cuh"

namespace hv {

constexpr float kLog2e = 1.4426950408889634f;

HV_DEV void mma_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, "
      "{%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Four biased codes as two pairs of exact halves: 0x6400 | byte is 1024 + byte, less 1152.
HV_DEV void q8_halves(uint32_t w, uint32_t* lo, uint32_t* hi) {
  const __half2 c = __floats2half2_rn(1152.f, 1152.f);
  uint32_t a = __byte_perm(w, 0x64646464u, 0x4140), b = __byte_perm(w, 0x64646464u, 0x4342);
  __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), c);
  __half2 y = __hsub2(*reinterpret_cast<__half2*>(&b), c);
  *lo = *reinterpret_cast<uint32_t*>(&x);
  *hi = *reinterpret_cast<uint32_t*>(&y);
}

HV_DEV uint32_t pack_half2(float x, float y) {
  const __half2 h = __floats2half2_rn(x, y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// hi and lo terms of (x, y) as packed pairs.
HV_DEV void split_half2(float x, float y, uint32_t* hi, uint32_t* lo) {
  const __half2 h = __floats2half2_rn(x, y);
  const float2 f = __half22float2(h);
  *hi = *reinterpret_cast<const uint32_t*>(&h);
  *lo = pack_half2(x - f.x, y - f.y);
}

// The 8x8 binary16 matrix whose row g the lanes 4 g + t hold, transposed.
HV_DEV uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}

// 2^x; below 2^-126 it is 0, which the weights of a softmax may be (without .ftz the compiler
// scales around the instruction: five instructions for one).
HV_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^e that brings a largest value of `amax` to [2^13, 2^14) (1 for zero and non-finite).
HV_DEV float q8_lift(float amax) {
  if (!(amax > 0.0f && amax < INFINITY)) return 1.0f;
  int e = 13 + 127 - (int)(__float_as_uint(amax) >> 23);        // 13 - floor(log2 amax)
  e = e > 126 ? 126 : (e < -126 ? -126 : e);
  return __uint_as_float((unsigned)(e + 127) << 23);
}

constexpr unsigned long long kQ8WaitNs = 2000000000ull;     // of a wait on a barrier of a CTA's own

HV_DEV void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
// False when the wait ran out here or elsewhere in the CTA.
HV_DEV bool bar_wait(uint32_t bar, uint32_t parity, volatile int* given_up) {
  unsigned long long t0 = 0;
  for (unsigned n = 1;; ++n) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, 1000;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    if (ok) return true;
    if ((n & 63) == 0) {
      if (*given_up) return false;
      const unsigned long long now = global_ns();
      if (t0 == 0) t0 = now;
      else if (now - t0 > kQ8WaitNs) { *given_up = 1; return false; }
    }
  }
}

// The same for a whole warp, whose lanes go on or leave together.
HV_DEV bool bar_wait_warp(uint32_t bar, uint32_t parity, volatile int* given_up) {
  const bool ok = bar_wait(bar, parity, given_up);
  return __all_sync(0xFFFFFFFFu, ok) != 0;
}

}  // namespace hv
