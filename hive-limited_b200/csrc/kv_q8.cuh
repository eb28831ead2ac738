// The 8-bit KV cache of one layer: its arrangement in memory and the rule that makes a code.
//
// For every kv head and every block of 32 positions the cache holds an int8 code per value
// and one f32 scale for the block's 32 x 128 K values, and the same for V:
//   s = f32(max|x| / 127), 1 where that is 0
//   c = trunc(f32(x / s) + (x < 0 ? -0.5 : 0.5)), clipped to +-127   (quant_a8s's rule)
// and a value reads back as f32(c s). A block with a NaN or an infinity in it has the scale
// NaN, so all of it reads NaN. The block that is still open stays in f32 (the tail) and is
// quantised when its 32nd row arrives: once, unless a write goes back into it later, which reopens
// it from its codes.
//
// One buffer per layer (every part starts on 256 bytes; nblk = ceil(cap / 32)):
//   codes  u8  [nkv][nblk][2][4096]   a block's K codes, then its V codes, each code + 128
//   scales f32 [nkv][nblk][2]         (K, V)
//   tail   f32 [nkv][2][32][128]      rows of block (held - 1) / 32
//   held   i32 [nkv][2]               positions written; a zeroed buffer is an empty cache
//
// Inside a block the codes stand as the tensor pipe's fragments want them, so that a lane
// (lane = 4 g + t) finds what it multiplies in eight 16-byte units at 512 u + 16 lane:
//   K, position 8 j + g, dim 64 h + 16 s + 4 t + e:  unit 2 j + h, byte 4 s + e
//   V, position 16 k + 8 j + 2 t + e, dim 16 u + 8 h + g:  unit u, byte 8 h + 4 k + 2 j + e
#pragma once

#include "attn_decode.cuh"

namespace hv {

constexpr int kQ8Blk = 32;                    // positions per scale
constexpr int kQ8Codes = kQ8Blk * kHd;        // code bytes of a block's K (or V)

struct KvQ8 {
  uint8_t* codes;
  float* scales;
  float* tail;
  int32_t* held;
  int nblk;
};

HV_HD size_t kv_q8_up(size_t n) { return (n + 255) & ~(size_t)255; }

HV_HD size_t kv_q8_view(void* base, int nkv, int cap, KvQ8* v) {
  const size_t nblk = ((size_t)cap + kQ8Blk - 1) / kQ8Blk;
  const size_t codes = (size_t)nkv * nblk * 2 * kQ8Codes;
  const size_t scales = kv_q8_up((size_t)nkv * nblk * 2 * sizeof(float));
  const size_t tail = (size_t)nkv * 2 * kQ8Codes * sizeof(float);
  uint8_t* p = static_cast<uint8_t*>(base);
  v->codes = p;
  v->scales = reinterpret_cast<float*>(p + codes);
  v->tail = reinterpret_cast<float*>(p + codes + scales);
  v->held = reinterpret_cast<int32_t*>(p + codes + scales + tail);
  v->nblk = (int)nblk;
  return codes + scales + tail + kv_q8_up((size_t)nkv * 2 * sizeof(int32_t));
}

// Byte of (position r of the block, dim d) among the block's 4096 K (V) codes.
HV_DEV int q8_k_at(int r, int d) {
  const int g = r & 7, j = r >> 3, h = d >> 6, s = (d >> 4) & 3, t = (d >> 2) & 3, e = d & 3;
  return (2 * j + h) * 512 + (4 * g + t) * 16 + 4 * s + e;
}
HV_DEV int q8_v_at(int r, int d) {
  const int k = r >> 4, j = (r >> 3) & 1, t = (r >> 1) & 3, e = r & 1;
  const int u = d >> 4, h = (d >> 3) & 1, g = d & 7;
  return u * 512 + (4 * g + t) * 16 + 8 * h + 4 * k + 2 * j + e;
}

HV_DEV int q8_code(float x, float s) {
  const int q = (int)truncf(__fadd_rn(__fdiv_rn(x, s), x < 0.0f ? -0.5f : 0.5f));
  return q > 127 ? 127 : (q < -127 ? -127 : q);
}

HV_DEV float q8_value(uint32_t biased, float s) {   // 2^23 + code + 128 as a float, less that
  return __fmul_rn(__fsub_rn(__uint_as_float(0x4B000000u | biased), 8388608.0f + 128.0f), s);
}

HV_DEV float q8_max(float a, float b) {          // the larger magnitude; NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(fabsf(a)), "f"(fabsf(b)));
  return r;
}

// Positions the cache holds for kv head g: those both K and V have.
HV_DEV int q8_held(const KvQ8& c, int g) {
  const int2 h = __ldg(reinterpret_cast<const int2*>(c.held) + g);
  return min(h.x, h.y);
}

}  // namespace hv
