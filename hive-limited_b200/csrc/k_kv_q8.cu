// Writing and reading the 8-bit KV cache (kv_q8.cuh has the arrangement and the rule).
//
// One CTA per (kv head, K or V, block of 32 positions): it gathers the block's rows -- those
// the tail already holds and those of this call -- finds their maximum and, if the block is
// complete, writes its 4096 codes and its scale. The CTA of a call's first block also moves
// the tail on to the call's last block and sets the number of positions held: the tail it
// reads and the tail it writes may be the same memory, and no other CTA touches either.
//
// Bound by HBM for long runs: 16377 positions of 8 heads written and read back (335 MB) take
// 63 us, 5.3 TB/s, 81% of a plain copy's rate; a row and its block read back take 5.5 us in a
// graph, two launches. A CTA holds a block's 16 KB in registers (four rows a warp), so that the
// maximum and the codes need one read; the codes pass through shared memory, padded by unit, and
// leave as 16-byte stores. Seven CTAs an SM at 32 registers: 57.6 us in a graph, 61.8 at 48.
#include <cfloat>

#include "hv_internal.h"
#include "kv_q8.cuh"

namespace hv {
namespace {

// Rows of K (which = 0) and V (which = 1) as the caller holds them.
struct Q8Src {
  const float* k;
  const float* v;
  size_t ld;                   // floats from one position's row to the next
  // with kNorm: K rows are raw and get the head norm and the rotation first
  const float* kn;
  const float* cos_t;
  const float* sin_t;
  float eps;
};

// Bytes between the 512-byte units of a block's codes in shared memory: such that the warps'
// 4-byte pieces of K and 2-byte pieces of V fall on different banks (two to a bank for V).
constexpr int kKUnit = 576, kVUnit = 528;

// Row `t` of the call for head g as a float4 per lane (dims 4 lane ..). One warp.
template <bool kNorm>
HV_DEV float4 q8_row(const Q8Src& s, int which, int g, int t, int pos, float* tmp) {
  const int lane = threadIdx.x & 31;
  const float* row = (which ? s.v : s.k) + (size_t)t * s.ld + (size_t)g * kHd;
  if constexpr (kNorm) {
    if (which == 0) {
      const size_t at = (size_t)pos * (kHd / 2);
      warp_norm_rope(row, s.kn, s.cos_t + at, s.sin_t + at, s.eps, tmp, tmp + kHd);
      const float4 r = reinterpret_cast<const float4*>(tmp + kHd)[lane];
      __syncwarp();
      return r;
    }
  }
  return __ldg(reinterpret_cast<const float4*>(row) + lane);
}

// blockIdx.x: (head, which) pairs; blockIdx.y: blocks of the call. With pos_p the call is one
// row at *pos_p.
template <bool kNorm>
HV_DEV void q8_write_block(const Q8Src& src, const KvQ8& c, int item, int nth, int pos0,
                           int ntok) {
  __shared__ float s_max[8];
  __shared__ int s_held;
  __shared__ __align__(16) uint8_t s_codes[8 * kKUnit];
  __shared__ __align__(16) float s_tmp[kNorm ? 8 : 1][kNorm ? 2 * kHd : 4];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = item >> 1, which = item & 1;
  const int b0 = pos0 / kQ8Blk, blk = b0 + nth, end = pos0 + ntok;
  const int blk_last = (end - 1) / kQ8Blk;
  const bool first = nth == 0;
  float* tail = c.tail + (size_t)item * kQ8Codes;
  uint8_t* codes = c.codes + (((size_t)g * c.nblk + blk) * 2 + which) * kQ8Codes;
  float* scale = c.scales + ((size_t)g * c.nblk + blk) * 2 + which;
  const int old = first ? pos0 % kQ8Blk : 0;          // rows of this block already held
  const int have = min(end - blk * kQ8Blk, kQ8Blk);
  bool in_tail = true;
  if (first) {
    if (threadIdx.x == 0) s_held = c.held[item];
    __syncthreads();
    // a gap before pos0: the head's length and what it holds stay (the codes that the call's other
    // CTAs write are past the length, where nothing reads them before they are written again)
    if (pos0 > s_held) return;
    in_tail = old == 0 || (s_held - 1) / kQ8Blk == blk;
  }

  // rows 4 warp .. 4 warp + 3 of the block
  float4 x[4];
  float mx = 0.0f;                     // NaN once a NaN has been seen
  if (old == 0 && have == kQ8Blk) {     // the usual block: four loads under way at once
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int p = blk * kQ8Blk + 4 * warp + i;
      x[i] = q8_row<kNorm>(src, which, g, p - pos0, p, s_tmp[kNorm ? warp : 0]);
    }
  } else {
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * warp + i;
      float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < old) {
        if (in_tail) {
          y = reinterpret_cast<const float4*>(tail + (size_t)r * kHd)[lane];
        } else {                         // the block was complete: reopen it from its codes
          const float s = *scale;
          float v[4];
          for (int e = 0; e < 4; ++e) {
            const int d = 4 * lane + e;
            v[e] = q8_value(codes[which ? q8_v_at(r, d) : q8_k_at(r, d)], s);
          }
          y = make_float4(v[0], v[1], v[2], v[3]);
        }
      } else if (r < have) {
        y = q8_row<kNorm>(src, which, g, blk * kQ8Blk + r - pos0, blk * kQ8Blk + r,
                             s_tmp[kNorm ? warp : 0]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (k == i) x[k] = y;
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    mx = q8_max(q8_max(mx, x[i].x), q8_max(x[i].y, x[i].z));
    mx = q8_max(mx, x[i].w);
  }
  if (have == kQ8Blk) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = q8_max(mx, __shfl_xor_sync(0xFFFFFFFFu, mx, o));
    if (lane == 0) s_max[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < 8; ++w) mx = q8_max(mx, s_max[w]);
    const bool any_bad = !(mx <= FLT_MAX);
    float s = __fdiv_rn(mx, 127.0f);
    if (s == 0.0f) s = 1.0f;
    // The code is the nearest integer to x / s. x times 1 / s is off by 2 parts in 2^24 of 127,
    // and the rule's own roundings are 2^-17 together: where that product is not within 5e-5 of
    // a half the nearest integer to it is the rule's, and else the rule itself is asked (so too
    // where s is so small that its rounding counts).
    const float inv = __frcp_rn(s);
    const bool slow = any_bad || s < 0x1p-100f;
    const int unit = which ? kVUnit : kKUnit;
    uint32_t y[4];                     // a row's four codes each, plus 128
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float v[4] = {x[i].x, x[i].y, x[i].z, x[i].w};
      uint32_t q[4];
      bool near = slow;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        constexpr float kMagic = 12582912.0f + 128.0f;      // 1.5 2^23: the sum's low bits count
        const float z = __fmul_rn(v[e], inv), n = __fadd_rn(z, kMagic);
        q[e] = __float_as_uint(n);
        near |= fabsf(__fsub_rn(z, __fsub_rn(n, kMagic))) > 0.49995f;
      }
      if (near) {
#pragma unroll
        for (int e = 0; e < 4; ++e) q[e] = any_bad ? 128u : (uint32_t)(q8_code(v[e], s) + 128);
      }
      y[i] = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    }
    if (which == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = q8_k_at(4 * warp + i, 4 * lane);
        *reinterpret_cast<uint32_t*>(s_codes + (at >> 9) * unit + (at & 511)) = y[i];
      }
    } else {
      // two rows' codes of a dim are neighbours
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = q8_v_at(4 * warp + i, 4 * lane + e);
          const uint32_t two = __byte_perm(y[i], y[i + 1], e | (4 + e) << 4);
          *reinterpret_cast<uint16_t*>(s_codes + (at >> 9) * unit + (at & 511)) = (uint16_t)two;
        }
      }
    }
    __syncthreads();
    reinterpret_cast<uint4*>(codes)[threadIdx.x] =
        *reinterpret_cast<const uint4*>(s_codes + (threadIdx.x >> 5) * unit + (threadIdx.x & 31) * 16);
    if (threadIdx.x == 0) *scale = any_bad ? __int_as_float(0x7fc00000) : s;
  }
  if (!first) return;

  __syncthreads();                     // every old tail row has been read
  if (blk_last == blk) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * warp + i;
      if (r < have && (r >= old || !in_tail))
        reinterpret_cast<float4*>(tail + (size_t)r * kHd)[lane] = x[i];
    }
  } else {
    const int n = end - blk_last * kQ8Blk;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = 4 * warp + i;
      if (r < n)
        reinterpret_cast<float4*>(tail + (size_t)r * kHd)[lane] =
            q8_row<kNorm>(src, which, g, blk_last * kQ8Blk + r - pos0, blk_last * kQ8Blk + r,
                          s_tmp[kNorm ? warp : 0]);
    }
  }
  if (threadIdx.x == 0) c.held[item] = end;
}

__global__ void __launch_bounds__(256, 7) k_kv_rows_q8(Q8Src src, KvQ8 c, int pos0, int ntok) {
  q8_write_block<false>(src, c, blockIdx.x, blockIdx.y, pos0, ntok);
}

// One row at *pos; a *pos outside [0, cap) writes nothing.
__global__ void __launch_bounds__(256) k_kvapp_q8(Q8Src src, KvQ8 c, const int32_t* pos,
                                                  int cap) {
  const int p = *pos;
  if (p < 0 || p >= cap) return;
  q8_write_block<false>(src, c, blockIdx.x, 0, p, 1);
}

// hv_qk_rows with an 8-bit cache: CTAs [0, 2 nkv nb) write K (normed and rotated) and V
// blocks, the others norm and rotate eight query rows each.
__global__ void __launch_bounds__(256) k_qk_rows_q8(Q8Src src, KvQ8 c,
                                                    const float* __restrict__ q,
                                                    const float* __restrict__ qn,
                                                    float* __restrict__ q_out, int nq, int nkv,
                                                    int nb, int pos0, int ntok) {
  const int kv_ctas = 2 * nkv * nb;
  if ((int)blockIdx.x < kv_ctas) {
    q8_write_block<true>(src, c, blockIdx.x % (2 * nkv), blockIdx.x / (2 * nkv), pos0, ntok);
    return;
  }
  __shared__ __align__(16) float tmp[8][kHd];
  const long long wi = (long long)(blockIdx.x - kv_ctas) * 8 + (threadIdx.x >> 5);
  if (wi >= (long long)ntok * nq) return;                     // whole warps
  const int t = (int)(wi / nq), h = (int)(wi % nq);
  const size_t at = (size_t)(pos0 + t) * (kHd / 2);
  warp_norm_rope(q + (size_t)t * src.ld + (size_t)h * kHd, qn, src.cos_t + at, src.sin_t + at,
                 src.eps, tmp[threadIdx.x >> 5], q_out + ((size_t)t * nq + h) * kHd);
}

// Positions pos0 .. pos0 + ntok - 1 as f32 rows [ntok][nkv][128]; NaN where nothing is held.
// One CTA per (head, K or V) and block; the codes pass through shared memory.
__global__ void __launch_bounds__(256) k_kv_read_q8(KvQ8 c, float* __restrict__ k_out,
                                                    float* __restrict__ v_out, int pos0, int ntok,
                                                    int nkv) {
  __shared__ __align__(16) uint8_t s_codes[8 * kKUnit];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int g = blockIdx.x >> 1, which = blockIdx.x & 1;
  const int blk = pos0 / kQ8Blk + blockIdx.y;
  const int held = q8_held(c, g), p0 = blk * kQ8Blk;
  const bool closed = p0 + kQ8Blk <= held;
  const int unit = which ? kVUnit : kKUnit;
  float s = 0.0f;
  if (closed) {
    const uint8_t* codes = c.codes + (((size_t)g * c.nblk + blk) * 2 + which) * kQ8Codes;
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(codes) + threadIdx.x);
    *reinterpret_cast<uint4*>(s_codes + (threadIdx.x >> 5) * unit + (threadIdx.x & 31) * 16) = w;
    s = __ldg(c.scales + ((size_t)g * c.nblk + blk) * 2 + which);
  }
  __syncthreads();
  const float* tail = c.tail + ((size_t)g * 2 + which) * kQ8Codes;
  float* out = which ? v_out : k_out;
  uint32_t y[4] = {0, 0, 0, 0};                  // a row's four codes each
  if (closed) {
    if (which == 0) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int at = q8_k_at(4 * warp + i, 4 * lane);
        y[i] = *reinterpret_cast<const uint32_t*>(s_codes + (at >> 9) * unit + (at & 511));
      }
    } else {
#pragma unroll
      for (int i = 0; i < 4; i += 2) {
        uint32_t two[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int at = q8_v_at(4 * warp + i, 4 * lane + e);
          two[e] = *reinterpret_cast<const uint16_t*>(s_codes + (at >> 9) * unit + (at & 511));
        }
        const uint32_t a = __byte_perm(two[0], two[1], 0x5140), b = __byte_perm(two[2], two[3], 0x5140);
        y[i] = __byte_perm(a, b, 0x5410);
        y[i + 1] = __byte_perm(a, b, 0x7632);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * warp + i, p = p0 + r;
    if (p < pos0 || p >= pos0 + ntok) continue;
    float4 x;
    if (closed) {
      const uint32_t w = y[i];
      x = make_float4(q8_value(w & 255, s), q8_value((w >> 8) & 255, s), q8_value((w >> 16) & 255, s),
                      q8_value(w >> 24, s));
    } else if (p < held) {
      x = __ldg(reinterpret_cast<const float4*>(tail + (size_t)r * kHd) + lane);
    } else {
      const float nan = __int_as_float(0x7fc00000);
      x = make_float4(nan, nan, nan, nan);
    }
    reinterpret_cast<float4*>(out + ((size_t)(p - pos0) * nkv + g) * kHd)[lane] = x;
  }
}

int q8_cache_check(const char* name, const void* kv, int nkv, int hd, int cap) {
  HV_REQUIRE(kv && nkv > 0 && cap > 0, HV_E_INVALID, "%s: bad arguments", name);
  HV_REQUIRE(hd == kHd, HV_E_UNSUPPORTED, "%s: head_dim %d (only 128)", name, hd);
  HV_REQUIRE(((uintptr_t)kv & 15) == 0, HV_E_INVALID, "%s: unaligned cache pointer", name);
  HV_REQUIRE(nkv <= 32768 && cap <= (1 << 30), HV_E_UNSUPPORTED,
             "%s: %d kv heads, %d positions", name, nkv, cap);
  return HV_OK;
}

int q8_rows_check(const char* name, int pos0, int ntok, int cap, int* nb) {
  HV_REQUIRE(ntok > 0 && pos0 >= 0, HV_E_INVALID, "%s: bad arguments", name);
  HV_REQUIRE((long long)pos0 + ntok <= cap, HV_E_INVALID,
             "%s: positions %d .. %lld outside the cache of %d", name, pos0,
             (long long)pos0 + ntok - 1, cap);
  *nb = (pos0 + ntok - 1) / kQ8Blk - pos0 / kQ8Blk + 1;
  HV_REQUIRE(*nb <= 65535, HV_E_UNSUPPORTED, "%s: %d rows at once", name, ntok);
  return HV_OK;
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_kv_q8_size(int nkv, int hd, int cap, size_t* bytes) {
  HV_REQUIRE(bytes, HV_E_INVALID, "hv_kv_q8_size: null pointer");
  static char nowhere[16] __attribute__((aligned(16)));
  const int rc = q8_cache_check("hv_kv_q8_size", nowhere, nkv, hd, cap);
  if (rc) return rc;
  KvQ8 v;
  *bytes = kv_q8_view(nowhere, nkv, cap, &v);
  return HV_OK;
}

extern "C" int hv_kv_append_q8(const float* k, const float* v, void* kv, const int32_t* pos,
                               int nkv, int hd, int cap, void* stream) {
  HV_REQUIRE(k && v && pos, HV_E_INVALID, "hv_kv_append_q8: bad arguments");
  const int rc = q8_cache_check("hv_kv_append_q8", kv, nkv, hd, cap);
  if (rc) return rc;
  HV_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0, HV_E_INVALID,
             "hv_kv_append_q8: unaligned pointer");
  Q8Src s{k, v, (size_t)nkv * kHd, nullptr, nullptr, nullptr, 0.0f};
  KvQ8 c;
  kv_q8_view(kv, nkv, cap, &c);
  k_kvapp_q8<<<2 * nkv, 256, 0, (cudaStream_t)stream>>>(s, c, pos, cap);
  HV_LAUNCHED("k_kvapp_q8");
}

extern "C" int hv_kv_rows_q8(const float* k, const float* v, int ld, void* kv, int pos0, int nkv,
                             int hd, int cap, int ntok, void* stream) {
  HV_REQUIRE(k && v, HV_E_INVALID, "hv_kv_rows_q8: bad arguments");
  int nb = 0;
  int rc = q8_cache_check("hv_kv_rows_q8", kv, nkv, hd, cap);
  if (!rc) rc = q8_rows_check("hv_kv_rows_q8", pos0, ntok, cap, &nb);
  if (rc) return rc;
  HV_REQUIRE(ld >= nkv * kHd && ld % 4 == 0, HV_E_INVALID,
             "hv_kv_rows_q8: row stride %d (at least %d, a multiple of 4)", ld, nkv * kHd);
  HV_REQUIRE(((uintptr_t)k & 15) == 0 && ((uintptr_t)v & 15) == 0, HV_E_INVALID,
             "hv_kv_rows_q8: unaligned pointer");
  Q8Src s{k, v, (size_t)ld, nullptr, nullptr, nullptr, 0.0f};
  KvQ8 c;
  kv_q8_view(kv, nkv, cap, &c);
  k_kv_rows_q8<<<dim3(2 * nkv, nb), 256, 0, (cudaStream_t)stream>>>(s, c, pos0, ntok);
  HV_LAUNCHED("k_kv_rows_q8");
}

extern "C" int hv_qk_rows_q8(const float* qkv, const float* qn, const float* kn,
                             const float* cos_t, const float* sin_t, int pos0, float* q_out,
                             void* kv, int nq, int nkv, int hd, int cap, float eps, int ntok,
                             void* stream) {
  HV_REQUIRE(qkv && qn && kn && cos_t && sin_t && q_out && nq > 0, HV_E_INVALID,
             "hv_qk_rows_q8: bad arguments");
  int nb = 0;
  int rc = q8_cache_check("hv_qk_rows_q8", kv, nkv, hd, cap);
  if (!rc) rc = q8_rows_check("hv_qk_rows_q8", pos0, ntok, cap, &nb);
  if (rc) return rc;
  HV_REQUIRE(((uintptr_t)qkv & 15) == 0, HV_E_INVALID, "hv_qk_rows_q8: unaligned pointer");
  const long long ctas = 2ll * nkv * nb + ((long long)ntok * nq + 7) / 8;
  HV_REQUIRE(nq <= 32768 && ctas <= 0x7FFFFFFFll, HV_E_UNSUPPORTED,
             "hv_qk_rows_q8: %d rows of %d heads at once", ntok, nq);
  const size_t ld = (size_t)(nq + 2 * nkv) * kHd;
  Q8Src s{qkv + (size_t)nq * kHd, qkv + (size_t)(nq + nkv) * kHd, ld, kn, cos_t, sin_t, eps};
  KvQ8 c;
  kv_q8_view(kv, nkv, cap, &c);
  k_qk_rows_q8<<<(unsigned)ctas, 256, 0, (cudaStream_t)stream>>>(s, c, qkv, qn, q_out, nq, nkv,
                                                                 nb, pos0, ntok);
  HV_LAUNCHED("k_qk_rows_q8");
}

extern "C" int hv_kv_read_q8(const void* kv, float* k_out, float* v_out, int pos0, int nkv,
                             int hd, int cap, int ntok, void* stream) {
  HV_REQUIRE(k_out && v_out, HV_E_INVALID, "hv_kv_read_q8: bad arguments");
  int nb = 0;
  int rc = q8_cache_check("hv_kv_read_q8", kv, nkv, hd, cap);
  if (!rc) rc = q8_rows_check("hv_kv_read_q8", pos0, ntok, cap, &nb);
  if (rc) return rc;
  HV_REQUIRE(((uintptr_t)k_out & 15) == 0 && ((uintptr_t)v_out & 15) == 0, HV_E_INVALID,
             "hv_kv_read_q8: unaligned pointer");
  KvQ8 c;
  kv_q8_view(const_cast<void*>(kv), nkv, cap, &c);
  k_kv_read_q8<<<dim3(2 * nkv, nb), 256, 0, (cudaStream_t)stream>>>(c, k_out, v_out, pos0, ntok,
                                                                    nkv);
  HV_LAUNCHED("k_kv_read_q8");
}
