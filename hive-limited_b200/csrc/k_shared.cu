// One prompt with many continuations, over the binary16 cache: attention of a batch of rows that
// share a prefix (hv_attn_shared_f16), the write of such rows (hv_qk_shared_f16), and the lane's
// causal attention with the weights that every position gets added up (hv_attn_decode_mass_f16,
// hv_attn_rows_mass_f16).
//
//   ctx_h = sum_t w_t v_t / sum_t w_t,   w_t = exp(scale q_h . k_t - max)
//   mass[g][t] += sum over rows and the heads of kv head g of w_t / sum w
#include "attn_decode.cuh"
#include "attn_f16.cuh"

namespace hv {
namespace {

constexpr int kShWarps = 8;

// A CTA per (row, kv head), its warps taking positions in turn, a lane four dims.
__global__ void __launch_bounds__(32 * kShWarps) k_span_rows(SpanArgs a, float2* __restrict__ stat) {
  __shared__ float s_m[kShWarps][8], s_l[kShWarps][8];
  __shared__ __align__(16) float s_o[kShWarps][8][kHd];
  const int r = blockIdx.x, kvh = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  SpanSeq x;
  if (!span_find(a, r, &x)) return;
  const int np = span_prefix(a);
  float* out = a.ctx + ((size_t)r * a.nq + (size_t)kvh * a.group) * kHd;
  float2* st = stat + ((size_t)kvh * a.nrow + r) * a.group;
  if (np < 0 || x.len < 0) {
    for (int i = threadIdx.x; i < a.group * kHd; i += blockDim.x) out[i] = __int_as_float(0x7fc00000);
    if (threadIdx.x < a.group) st[threadIdx.x] = make_float2(0.f, __int_as_float(0x7fc00000));
    return;
  }
  const float f = __ldg(a.scale) * kLog2e;
  float4 q[8], o[8];
  float m[8], l[8];
#pragma unroll
  for (int h = 0; h < 8; ++h) {
    if (h < a.group)
      q[h] = __ldg(reinterpret_cast<const float4*>(a.q + ((size_t)r * a.nq + (size_t)kvh * a.group + h) * kHd) + lane);
    o[h] = make_float4(0.f, 0.f, 0.f, 0.f);
    m[h] = -INFINITY;
    l[h] = 0.f;
  }
  const int n = np + x.sees(r);
  for (int t = warp; t < n; t += kShWarps) {
    const bool tail = t >= np;
    const size_t at = tail ? (size_t)x.s * a.t_seq + kvh * a.t_head + (size_t)(t - np) * kHd
                           : kvh * a.p_head + (size_t)t * kHd;
    const uint2 kw = reinterpret_cast<const uint2*>((tail ? a.tk : a.pk) + at)[lane];
    const uint2 vw = reinterpret_cast<const uint2*>((tail ? a.tv : a.pv) + at)[lane];
    const float2 k0 = __half22float2(*reinterpret_cast<const __half2*>(&kw.x));
    const float2 k1 = __half22float2(*reinterpret_cast<const __half2*>(&kw.y));
    const float2 v0 = __half22float2(*reinterpret_cast<const __half2*>(&vw.x));
    const float2 v1 = __half22float2(*reinterpret_cast<const __half2*>(&vw.y));
#pragma unroll
    for (int h = 0; h < 8; ++h) {
      if (h >= a.group) break;
      float s = q[h].x * k0.x + q[h].y * k0.y + q[h].z * k1.x + q[h].w * k1.y;
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
      s *= f;
      const float up = fmaxf(m[h], s), c = m[h] == -INFINITY ? 0.f : ex2(m[h] - up), w = ex2(s - up);
      m[h] = up;
      l[h] = l[h] * c + w;
      o[h].x = o[h].x * c + w * v0.x;
      o[h].y = o[h].y * c + w * v0.y;
      o[h].z = o[h].z * c + w * v1.x;
      o[h].w = o[h].w * c + w * v1.y;
    }
  }
#pragma unroll
  for (int h = 0; h < 8; ++h) {
    if (h >= a.group) break;
    if (lane == 0) { s_m[warp][h] = m[h]; s_l[warp][h] = l[h]; }
    reinterpret_cast<float4*>(s_o[warp][h])[lane] = o[h];
  }
  __syncthreads();
  for (int i = threadIdx.x; i < a.group * kHd; i += blockDim.x) {
    const int h = i / kHd, d = i % kHd;
    float M = -INFINITY, L = 0.f, s = 0.f;
    for (int w = 0; w < kShWarps; ++w) M = fmaxf(M, s_m[w][h]);
    for (int w = 0; w < kShWarps; ++w) {
      const float c = s_l[w][h] == 0.f ? 0.f : ex2(s_m[w][h] - M);
      L += c * s_l[w][h];
      s += c * s_o[w][h][d];
    }
    out[i] = n == 0 ? 0.f : s / L;
    if (d == 0) st[h] = make_float2(M, 1.f / L);
  }
}

// A warp per (position, kv head): the weights that the rows give it.
__global__ void __launch_bounds__(256) k_mass_rows(SpanArgs a, const float2* __restrict__ stat,
                                                   const float* mass_in, float* mass_out, int cap) {
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), kvh = blockIdx.y, lane = threadIdx.x & 31;
  const int np = span_prefix(a);
  if (np < 0 || t >= np + max(a.tlen, 0)) return;
  const bool tail = t >= np;
  const size_t at = tail ? kvh * a.t_head + (size_t)(t - np) * kHd : kvh * a.p_head + (size_t)t * kHd;
  const uint2 kw = reinterpret_cast<const uint2*>((tail ? a.tk : a.pk) + at)[lane];
  const float2 k0 = __half22float2(*reinterpret_cast<const __half2*>(&kw.x));
  const float2 k1 = __half22float2(*reinterpret_cast<const __half2*>(&kw.y));
  const float f = __ldg(a.scale) * kLog2e;
  float sum = 0.f;
  for (int r = tail ? t - np : 0; r < a.nrow; ++r)
    for (int h = 0; h < a.group; ++h) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(a.q + ((size_t)r * a.nq + (size_t)kvh * a.group + h) * kHd) + lane);
      float s = q.x * k0.x + q.y * k0.y + q.z * k1.x + q.w * k1.y;
#pragma unroll
      for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, d);
      const float2 st = stat[((size_t)kvh * a.nrow + r) * a.group + h];
      sum += ex2(s * f - st.x) * st.y;
    }
  if (lane == 0) {
    const size_t i = (size_t)kvh * cap + t;
    mass_out[i] = (mass_in ? mass_in[i] : 0.f) + sum;
  }
}

// hv_qk_rows's arithmetic for the rows of a batch: a warp per (row, head).
__global__ void __launch_bounds__(256) k_qk_shared(const float* __restrict__ qkv, const float* __restrict__ qn,
                                                   const float* __restrict__ kn, const float* __restrict__ cos_t,
                                                   const float* __restrict__ sin_t, int cap,
                                                   const int32_t* __restrict__ base, SpanArgs a,
                                                   float* __restrict__ q_out, __half* tk, __half* tv,
                                                   int nkv, float eps) {
  __shared__ __align__(16) float tmp[8][kHd], row_s[8][kHd];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, heads = a.nq + nkv;
  const long long wi = (long long)blockIdx.x * 8 + warp;
  if (wi >= (long long)a.nrow * heads) return;            // whole warps
  const int r = (int)(wi / heads), h = (int)(wi % heads);
  SpanSeq x;
  if (!span_find(a, r, &x)) return;
  const int slot = x.len - (x.end - r);
  const long long pos = (long long)__ldg(base) + slot;
  const bool ok = x.len >= 0 && slot >= 0 && pos >= 0 && pos < cap;
  const float* row = qkv + (size_t)r * (a.nq + 2 * nkv) * kHd;
  if (!ok) {
    if (h < a.nq) {
      const float nan = __int_as_float(0x7fc00000);
      reinterpret_cast<float4*>(q_out + ((size_t)r * a.nq + h) * kHd)[lane] = make_float4(nan, nan, nan, nan);
    }
    return;
  }
  const float* cs = cos_t + (size_t)pos * (kHd / 2);
  const float* sn = sin_t + (size_t)pos * (kHd / 2);
  if (h < a.nq) {
    warp_norm_rope(row + (size_t)h * kHd, qn, cs, sn, eps, tmp[warp], q_out + ((size_t)r * a.nq + h) * kHd);
    return;
  }
  const int g = h - a.nq;
  warp_norm_rope(row + (size_t)h * kHd, kn, cs, sn, eps, tmp[warp], row_s[warp]);
  const float4 k4 = reinterpret_cast<const float4*>(row_s[warp])[lane];
  const float4 v4 = reinterpret_cast<const float4*>(row + (size_t)(h + nkv) * kHd)[lane];
  const size_t at = (size_t)x.s * a.t_seq + g * a.t_head + (size_t)slot * kHd + 4 * lane;
  reinterpret_cast<__half2*>(tk + at)[0] = __floats2half2_rn(k4.x, k4.y);
  reinterpret_cast<__half2*>(tk + at)[1] = __floats2half2_rn(k4.z, k4.w);
  reinterpret_cast<__half2*>(tv + at)[0] = __floats2half2_rn(v4.x, v4.y);
  reinterpret_cast<__half2*>(tv + at)[1] = __floats2half2_rn(v4.z, v4.w);
}

constexpr int kShMaxRows = 65535;      // rows and sequences of a call
constexpr long long kShMaxCap = 1 << 24;

int span_check(const char* name, int nq, int hd, int group, int nseq, int nrow) {
  HV_REQUIRE(nq > 0 && group > 0 && nseq > 0 && nrow > 0 && nq % group == 0, HV_E_INVALID, "%s: bad arguments", name);
  HV_REQUIRE(hd == kHd, HV_E_UNSUPPORTED, "%s: head_dim %d (only 128)", name, hd);
  HV_REQUIRE(group <= 8, HV_E_UNSUPPORTED, "%s: group size %d (1 to 8)", name, group);
  HV_REQUIRE(nrow <= kShMaxRows && nseq <= kShMaxRows && nq / group <= kShMaxRows, HV_E_UNSUPPORTED,
             "%s: %d rows of %d sequences at once", name, nrow, nseq);
  return HV_OK;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

int mass_any(const char* name, const SpanArgs& a, const float* mass_in, float* mass_out, int cap,
             void* scratch, cudaStream_t st) {
  HV_REQUIRE(a.q && a.pk && a.pv && a.ctx && a.scale && mass_out && scratch && cap > 0, HV_E_INVALID, "%s: bad arguments", name);
  HV_REQUIRE(cap <= kShMaxCap, HV_E_UNSUPPORTED, "%s: a cache of %d positions", name, cap);
  HV_REQUIRE(aligned16(a.q) && aligned16(a.pk) && aligned16(a.pv) && aligned16(a.ctx) && aligned16(scratch),
             HV_E_INVALID, "%s: unaligned pointer", name);
  const unsigned nkv = (unsigned)(a.nq / a.group);
  float2* stat = reinterpret_cast<float2*>(scratch);
  k_span_rows<<<dim3((unsigned)a.nrow, nkv), 32 * kShWarps, 0, st>>>(a, stat);
  k_mass_rows<<<dim3((unsigned)((cap + 7) / 8), nkv), 256, 0, st>>>(a, stat, mass_in, mass_out, cap);
  HV_LAUNCHED(name);
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_attn_shared_scratch(int nq, int group, int pcap, int tcap, int nseq, int nrow,
                                      size_t* bytes) {
  const int rc = span_check("hv_attn_shared_scratch", nq, kHd, group, nseq, nrow);
  if (rc) return rc;
  HV_REQUIRE(pcap >= 0 && tcap > 0 && bytes, HV_E_INVALID, "hv_attn_shared_scratch: bad arguments");
  HV_REQUIRE(pcap <= kShMaxCap && tcap <= kShMaxCap, HV_E_UNSUPPORTED,
             "hv_attn_shared_scratch: a prefix of %d, tails of %d positions", pcap, tcap);
  *bytes = (size_t)nq * nrow * sizeof(float2);
  return HV_OK;
}

extern "C" int hv_attn_shared_f16(const float* q, const uint16_t* pk, const uint16_t* pv, int pcap,
                                  const int32_t* plen, const uint16_t* tk, const uint16_t* tv, int tcap,
                                  const int32_t* row0, const int32_t* tlen, float* ctx,
                                  const float* scale, int nq, int hd, int group, int nseq, int nrow,
                                  void* scratch, void* stream) {
  const char* name = "hv_attn_shared_f16";
  const int rc = span_check(name, nq, hd, group, nseq, nrow);
  if (rc) return rc;
  HV_REQUIRE(q && tk && tv && tlen && ctx && scale && scratch && tcap > 0 && pcap >= 0 &&
                 (pcap == 0 || (pk && pv && plen)),
             HV_E_INVALID, "%s: bad arguments", name);
  HV_REQUIRE(row0 || nseq == nrow, HV_E_INVALID, "%s: %d sequences of one row each, %d rows", name, nseq, nrow);
  HV_REQUIRE(pcap <= kShMaxCap && tcap <= kShMaxCap, HV_E_UNSUPPORTED, "%s: a prefix of %d, tails of %d positions", name, pcap, tcap);
  HV_REQUIRE(aligned16(q) && aligned16(pk) && aligned16(pv) && aligned16(tk) && aligned16(tv) && aligned16(ctx) &&
                 aligned16(scratch),
             HV_E_INVALID, "%s: unaligned pointer", name);
  const size_t nkv = nq / group;
  SpanArgs a{};
  a.q = q; a.ctx = ctx; a.scale = scale;
  a.pk = reinterpret_cast<const __half*>(pk); a.pv = reinterpret_cast<const __half*>(pv);
  a.tk = reinterpret_cast<const __half*>(tk); a.tv = reinterpret_cast<const __half*>(tv);
  a.p_head = (size_t)pcap * kHd; a.t_head = (size_t)tcap * kHd; a.t_seq = nkv * a.t_head;
  a.plen_p = pcap ? plen : nullptr; a.row0 = row0; a.tlen_p = tlen;
  a.pcap = pcap; a.tcap = tcap;
  a.nq = nq; a.group = group; a.nseq = nseq; a.nrow = nrow;
  k_span_rows<<<dim3((unsigned)nrow, (unsigned)nkv), 32 * kShWarps, 0, (cudaStream_t)stream>>>(
      a, reinterpret_cast<float2*>(scratch));
  HV_LAUNCHED(name);
}

extern "C" int hv_attn_mass_scratch(int nq, int group, int cap, int ntok, size_t* bytes) {
  const int rc = span_check("hv_attn_mass_scratch", nq, kHd, group, 1, ntok);
  if (rc) return rc;
  HV_REQUIRE(cap > 0 && bytes, HV_E_INVALID, "hv_attn_mass_scratch: bad arguments");
  HV_REQUIRE(cap <= kShMaxCap, HV_E_UNSUPPORTED, "hv_attn_mass_scratch: a cache of %d positions", cap);
  *bytes = (size_t)nq * ntok * sizeof(float2);
  return HV_OK;
}

extern "C" int hv_attn_decode_mass_f16(const float* q, const uint16_t* kc, const uint16_t* vc, float* ctx,
                                       const float* mass_in, float* mass_out, const float* scale,
                                       const int32_t* pos, int nq, int hd, int group, int cap,
                                       void* scratch, void* stream) {
  const char* name = "hv_attn_decode_mass_f16";
  const int rc = span_check(name, nq, hd, group, 1, 1);
  if (rc) return rc;
  HV_REQUIRE(pos, HV_E_INVALID, "%s: bad arguments", name);
  SpanArgs a{};
  a.q = q; a.ctx = ctx; a.scale = scale;
  a.pk = reinterpret_cast<const __half*>(kc); a.pv = reinterpret_cast<const __half*>(vc);
  a.p_head = (size_t)cap * kHd;
  a.plen_p = pos; a.plen = a.pmin = 1; a.pcap = cap;
  a.nq = nq; a.group = group; a.nseq = a.nrow = 1;
  return mass_any(name, a, mass_in, mass_out, cap, scratch, (cudaStream_t)stream);
}

extern "C" int hv_attn_rows_mass_f16(const float* q, const uint16_t* kc, const uint16_t* vc, float* ctx,
                                     const float* mass_in, float* mass_out, const float* scale, int pos0,
                                     int nq, int hd, int group, int cap, int ntok, void* scratch,
                                     void* stream) {
  const char* name = "hv_attn_rows_mass_f16";
  const int rc = span_check(name, nq, hd, group, 1, ntok);
  if (rc) return rc;
  HV_REQUIRE(pos0 >= 0 && (long long)pos0 + ntok <= cap, HV_E_INVALID,
             "%s: positions %d .. %lld outside the cache of %d", name, pos0, (long long)pos0 + ntok - 1, cap);
  SpanArgs a{};
  a.q = q; a.ctx = ctx; a.scale = scale;
  a.pk = reinterpret_cast<const __half*>(kc); a.pv = reinterpret_cast<const __half*>(vc);
  a.p_head = a.t_head = (size_t)cap * kHd;
  if (kc && vc) { a.tk = a.pk + (size_t)pos0 * kHd; a.tv = a.pv + (size_t)pos0 * kHd; }
  a.plen = pos0; a.pcap = cap;
  a.tlen = a.tcap = ntok;
  a.nq = nq; a.group = group; a.nseq = 1; a.nrow = ntok;
  return mass_any(name, a, mass_in, mass_out, cap, scratch, (cudaStream_t)stream);
}

extern "C" int hv_qk_shared_f16(const float* qkv, const float* qn, const float* kn, const float* cos_t,
                                const float* sin_t, int cap, const int32_t* base, const int32_t* row0,
                                const int32_t* tlen, float* q_out, uint16_t* tk, uint16_t* tv, int nq,
                                int nkv, int hd, int tcap, float eps, int nseq, int nrow, void* stream) {
  const char* name = "hv_qk_shared_f16";
  HV_REQUIRE(qkv && qn && kn && cos_t && sin_t && cap > 0 && base && tlen && q_out && tk && tv && nq > 0 &&
                 nkv > 0 && tcap > 0 && nseq > 0 && nrow > 0 && nq <= (1 << 20) && nkv <= (1 << 20),
             HV_E_INVALID, "%s: bad arguments", name);
  HV_REQUIRE(hd == kHd, HV_E_UNSUPPORTED, "%s: head_dim %d (only 128)", name, hd);
  HV_REQUIRE(row0 || nseq == nrow, HV_E_INVALID, "%s: %d sequences of one row each, %d rows", name, nseq, nrow);
  HV_REQUIRE(nrow <= kShMaxRows && nseq <= kShMaxRows && tcap <= kShMaxCap, HV_E_UNSUPPORTED,
             "%s: %d rows of %d sequences, tails of %d positions", name, nrow, nseq, tcap);
  HV_REQUIRE(aligned16(qkv) && aligned16(q_out) && aligned16(tk) && aligned16(tv), HV_E_INVALID,
             "%s: unaligned pointer", name);
  SpanArgs a{};
  a.row0 = row0; a.tlen_p = tlen; a.tcap = tcap;
  a.t_head = (size_t)tcap * kHd; a.t_seq = (size_t)nkv * a.t_head;
  a.nq = nq; a.group = 1; a.nseq = nseq; a.nrow = nrow;
  const long long warps = (long long)(nq + nkv) * nrow;
  k_qk_shared<<<(unsigned)((warps + 7) / 8), 256, 0, (cudaStream_t)stream>>>(
      qkv, qn, kn, cos_t, sin_t, cap, base, a, q_out, reinterpret_cast<__half*>(tk),
      reinterpret_cast<__half*>(tv), nkv, eps);
  HV_LAUNCHED(name);
}
