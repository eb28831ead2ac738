// Attention over the 8-bit KV cache (kv_q8.cuh): one query token (hv_attn_decode_q8) or a run
// of them, each seeing the positions up to its own (hv_attn_rows_q8).
//
//   ctx_h = sum_t w_t v_t / sum_t w_t,   w_t = exp(scale q_h . k_t - max)
//
// in one pass with the running maximum and sum of the softmax. k_t and v_t are the values the
// cache reads back: f32(c s) in complete blocks, the f32 rows of the open one.
#include "hv_internal.h"
#include "kv_q8.cuh"

namespace hv {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

// One CTA per (query head, query row); its warps take positions in turn, a lane four dims.
__global__ void __launch_bounds__(128) k_attn_q8(const float* __restrict__ q, KvQ8 c,
                                                 float* __restrict__ ctx,
                                                 const float* __restrict__ scale,
                                                 const int32_t* __restrict__ pos_p, int pos0,
                                                 int nq, int group) {
  __shared__ float s_m[4], s_l[4];
  __shared__ float4 s_acc[4][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int h = blockIdx.x, g = h / group;
  const int pos = pos_p ? *pos_p : pos0 + (int)blockIdx.y;
  const size_t row = ((size_t)blockIdx.y * nq + h) * kHd;
  const int held = q8_held(c, g);
  if (pos < 0 || pos >= held) {
    ctx[row + threadIdx.x] = __int_as_float(0x7fc00000);
    return;
  }
  const float4 qv = __ldg(reinterpret_cast<const float4*>(q + row) + lane);
  const float sc = __ldg(scale) * kLog2e;
  float m = -INFINITY, l = 0.0f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int p = warp; p <= pos; p += 4) {
    const int blk = p / kQ8Blk, r = p % kQ8Blk;
    float4 k, v;
    if ((blk + 1) * kQ8Blk <= held) {
      const uint8_t* kc = c.codes + ((size_t)g * c.nblk + blk) * 2 * kQ8Codes;
      const float2 s = __ldg(reinterpret_cast<const float2*>(c.scales) + (size_t)g * c.nblk + blk);
      float kk[4], vv[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        kk[e] = q8_value(__ldg(kc + q8_k_at(r, 4 * lane + e)), s.x);
        vv[e] = q8_value(__ldg(kc + kQ8Codes + q8_v_at(r, 4 * lane + e)), s.y);
      }
      k = make_float4(kk[0], kk[1], kk[2], kk[3]);
      v = make_float4(vv[0], vv[1], vv[2], vv[3]);
    } else {
      const float4* t = reinterpret_cast<const float4*>(c.tail + (size_t)g * 2 * kQ8Codes);
      k = __ldg(t + r * (kHd / 4) + lane);
      v = __ldg(t + kQ8Codes / 4 + r * (kHd / 4) + lane);
    }
    float x = qv.x * k.x + qv.y * k.y + qv.z * k.z + qv.w * k.w;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xFFFFFFFFu, x, o);
    x *= sc;
    const float m1 = fmaxf(m, x);
    const float a = exp2f(m - m1), w = exp2f(x - m1);
    m = m1;
    l = l * a + w;
    acc.x = acc.x * a + w * v.x;
    acc.y = acc.y * a + w * v.y;
    acc.z = acc.z * a + w * v.z;
    acc.w = acc.w * a + w * v.w;
  }
  if (lane == 0) { s_m[warp] = m; s_l[warp] = l; }
  s_acc[warp][lane] = acc;
  __syncthreads();
  const float mx = fmaxf(fmaxf(s_m[0], s_m[1]), fmaxf(s_m[2], s_m[3]));
  float num = 0.0f, den = 0.0f;
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    const float a = s_l[w] == 0.0f ? 0.0f : exp2f(s_m[w] - mx);
    den += a * s_l[w];
    num += a * reinterpret_cast<const float*>(s_acc[w])[threadIdx.x];
  }
  ctx[row + threadIdx.x] = num / den;
}

int attn_q8_check(const char* name, const float* q, const void* kv, const float* ctx,
                  const float* scale, int nq, int hd, int group, int cap, const void* scratch) {
  HV_REQUIRE(q && kv && ctx && scale && scratch && nq > 0 && group > 0 && cap > 0, HV_E_INVALID,
             "%s: bad arguments", name);
  HV_REQUIRE(hd == kHd, HV_E_UNSUPPORTED, "%s: head_dim %d (only 128)", name, hd);
  HV_REQUIRE(nq % group == 0, HV_E_INVALID, "%s: nq %% group is not zero", name);
  HV_REQUIRE(group <= 8, HV_E_UNSUPPORTED, "%s: group size %d (1 to 8)", name, group);
  HV_REQUIRE(nq <= 32768 && cap <= (1 << 30), HV_E_UNSUPPORTED, "%s: %d heads, %d positions",
             name, nq, cap);
  HV_REQUIRE(((uintptr_t)q & 15) == 0 && ((uintptr_t)kv & 15) == 0 &&
                 ((uintptr_t)ctx & 15) == 0 && ((uintptr_t)scratch & 15) == 0,
             HV_E_INVALID, "%s: unaligned pointer", name);
  return HV_OK;
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_attn_q8_scratch(int nq, int group, int cap, int ntok, size_t* bytes) {
  HV_REQUIRE(nq > 0 && group > 0 && nq % group == 0 && cap > 0 && ntok > 0 && bytes,
             HV_E_INVALID, "hv_attn_q8_scratch: bad arguments");
  HV_REQUIRE(group <= 8, HV_E_UNSUPPORTED, "hv_attn_q8_scratch: group size %d (1 to 8)", group);
  *bytes = 256;
  return HV_OK;
}

extern "C" int hv_attn_decode_q8(const float* q, const void* kv, float* ctx, const float* scale,
                                 const int32_t* pos, int nq, int hd, int group, int cap,
                                 void* scratch, void* stream) {
  const int rc = attn_q8_check("hv_attn_decode_q8", q, kv, ctx, scale, nq, hd, group, cap,
                               scratch);
  if (rc) return rc;
  HV_REQUIRE(pos, HV_E_INVALID, "hv_attn_decode_q8: bad arguments");
  KvQ8 c;
  kv_q8_view(const_cast<void*>(kv), nq / group, cap, &c);
  k_attn_q8<<<nq, 128, 0, (cudaStream_t)stream>>>(q, c, ctx, scale, pos, 0, nq, group);
  HV_LAUNCHED("k_attn_q8");
}

extern "C" int hv_attn_rows_q8(const float* q, const void* kv, float* ctx, const float* scale,
                               int pos0, int nq, int hd, int group, int cap, int ntok,
                               void* scratch, void* stream) {
  const int rc = attn_q8_check("hv_attn_rows_q8", q, kv, ctx, scale, nq, hd, group, cap, scratch);
  if (rc) return rc;
  HV_REQUIRE(ntok > 0 && pos0 >= 0, HV_E_INVALID, "hv_attn_rows_q8: bad arguments");
  HV_REQUIRE((long long)pos0 + ntok <= cap, HV_E_INVALID,
             "hv_attn_rows_q8: positions %d .. %lld outside the cache of %d", pos0,
             (long long)pos0 + ntok - 1, cap);
  HV_REQUIRE(ntok <= 65535, HV_E_UNSUPPORTED, "hv_attn_rows_q8: %d rows at once", ntok);
  KvQ8 c;
  kv_q8_view(const_cast<void*>(kv), nq / group, cap, &c);
  k_attn_q8<<<dim3(nq, ntok), 128, 0, (cudaStream_t)stream>>>(q, c, ctx, scale, nullptr, pos0, nq,
                                                              group);
  HV_LAUNCHED("k_attn_q8");
}
