// One prompt with many continuations, over the binary16 cache: attention of a batch of rows that
// share a prefix (hv_attn_shared_f16), the write of such rows (hv_qk_shared_f16), and the lane's
// causal attention with the weights that every position gets added up (hv_attn_decode_mass_f16,
// hv_attn_rows_mass_f16).
//
//   ctx_h = sum_t w_t v_t / sum_t w_t,   w_t = exp(scale q_h . k_t - max)
//   mass[g][t] += sum over rows and the heads of kv head g of w_t / sum w
#include <algorithm>
#include <type_traits>

#include "attn_decode.cuh"
#include "attn_f16.cuh"

namespace hv {
namespace {

// ---- long tails of many rows --------------------------------------------------------------
//
// A CTA has up to 64 (row, head) pairs of a kv head and a chunk of the prefix or of a sequence's
// tail, so that K and V come from the L2 cache once for 64 pairs. Rows stand by eights as the 16-row operand of the f16 tensor pipe, their first binary16
// terms above their second ones, so that one product serves both and a thread adds what belongs
// together (the same for the weights of the second product). Warps share the CTA's rows by eights
// and then its positions, 32 at a time. K and V come by 16-byte asynchronous copies, 64 positions
// to a stage, swizzled so that eight rows' 16 bytes meet no bank twice. Bound by the f16 pipe, of
// which a product takes 16 cycles of a quarter of an SM: 64 rows by 64 positions are 2.5 us of a
// CTA's time (16 runs of 100 to 120 rows with tails to 600, 32 q over 8 kv heads: 177 us).
constexpr int kPtWarps = 8;
constexpr int kPtTile = kSpanStage * kHd * 2;            // bytes of K or of V of a stage
constexpr int kPtQ = kSpanItem * 2 * kHd * 2;            // bytes of 64 rows' two terms
constexpr int kPtLine = kHd + 4;                         // floats between rows that are joined
constexpr float kPtLift = 14.0f;                         // log2 of what weights are multiplied by
constexpr float kPtDrop = 0x1p-14f;
constexpr int kPtStages = 2;
constexpr int kPtSmem = kPtQ + kPtStages * 2 * kPtTile;
static_assert(kPtWarps * 8 * kPtLine * 4 <= kPtStages * 2 * kPtTile, "rows to join");

HV_DEV uint32_t swz(int row, int unit) { return row * 256 + ((unit ^ (row & 7)) << 4); }
HV_DEV void ldsm(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
HV_DEV void ldsm_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// A product's sums to those of the products before it, both terms together. The tensor pipe cuts what
// it adds where this rounds: over 30000 positions the cuts come to 2e-5 of the sum, all one way.
HV_DEV void add_up(float (&sum)[2], const float (&c)[4]) {
  sum[0] += c[0] + c[2];
  sum[1] += c[1] + c[3];
}
HV_DEV float4 dropped(const float4& x) { return make_float4(x.x * kPtDrop, x.y * kPtDrop, x.z * kPtDrop, x.w * kPtDrop); }
HV_DEV void cp16(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;"
               :: "r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}

// A row of 128 values, four a lane, as two binary16 terms of itself times a power of two, which is
// returned.
HV_DEV float row_terms(const float4& x, uint2* hi, uint2* lo) {
  float m = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
  m = __uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m)));
  const float lift = q8_lift(m);
  split_half2(x.x * lift, x.y * lift, &hi->x, &lo->x);
  split_half2(x.z * lift, x.w * lift, &hi->y, &lo->y);
  return lift;
}

// The two terms of rows f0 .. f0 + nf - 1 of kv head kvh to shared memory, eight rows of first
// terms, then their second ones; what takes a row's sums of products to exponents to `fac`.
// A warp's rows are all loaded before the first is worked on.
template <int kRows, int kWarps>
HV_DEV void rows_load(const SpanArgs& a, int kvh, int f0, int nf, int warp, float4 (&x)[kRows / kWarps]) {
#pragma unroll
  for (int j = 0; j < kRows / kWarps; ++j) {
    const int i = warp + j * kWarps;
    x[j] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < nf) {
      const int r = span_row(a, f0 + i), h = f0 + i - r * a.group;
      x[j] = __ldg(reinterpret_cast<const float4*>(a.q + ((size_t)r * a.nq + (size_t)kvh * a.group + h) * kHd) + (threadIdx.x & 31));
    }
  }
}
template <int kRows, int kWarps>
HV_DEV void rows_put(const float4 (&x)[kRows / kWarps], float f, int nf, uint8_t* to, float* fac, int warp) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int j = 0; j < kRows / kWarps; ++j) {
    const int i = warp + j * kWarps;
    if (i >= (nf + 7) / 8 * 8) break;
    uint2 hi, lo;
    const float lift = row_terms(x[j], &hi, &lo);
    const int at = (i >> 3) * 16 + (i & 7);
    *reinterpret_cast<uint2*>(to + swz(at, lane >> 1) + 8 * (lane & 1)) = hi;
    *reinterpret_cast<uint2*>(to + swz(at + 8, lane >> 1) + 8 * (lane & 1)) = lo;
    if (lane == 0) fac[i] = f / lift;
  }
}
template <int kRows, int kWarps>
HV_DEV void rows_split(const SpanArgs& a, int kvh, int f0, int nf, uint8_t* to, float* fac, int warp) {
  float4 x[kRows / kWarps];
  const float f = __ldg(a.scale) * kLog2e;
  rows_load<kRows, kWarps>(a, kvh, f0, nf, warp, x);
  rows_put<kRows, kWarps>(x, f, nf, to, fac, warp);
}

HV_DEV void span_part(const SpanArgs& a, const SpanParts& p, int tiles) {
  extern __shared__ __align__(1024) uint8_t smem[];         // the rows, then stages of K and V
  __shared__ float s_fac[kSpanItem], s_m[kPtWarps][8], s_l[kPtWarps][8];
  __shared__ int s_bad[kSpanStage];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, F = a.nrow * a.group;
  // what this CTA has
  const __half *k, *v;
  int f0, nf, p0, p1, slot, lim_all;     // lim_all: positions that every row sees
  SpanSeq x;
  const bool prefix = blockIdx.x < (unsigned)(tiles * p.npc);
  if (prefix) {
    const int tile = blockIdx.x / p.npc, chunk = blockIdx.x % p.npc;
    f0 = tile * kSpanItem;
    nf = min(kSpanItem, F - f0);
    const int n = max(span_prefix(a), 0), len = span_chunk(n, p.npc);
    p0 = chunk * len;
    p1 = min(n, p0 + len);
    if (p0 >= p1) return;
    slot = p.nwt + chunk;
    k = a.pk + kvh * a.p_head;
    v = a.pv + kvh * a.p_head;
    lim_all = p1;
  } else {
    const int b = blockIdx.x - tiles * p.npc, chunk = b % p.ntc;
    const SpanItem it = span_item(a, b / p.ntc, kSpanItem);
    if (it.nf == 0 || it.x.len <= 0) return;
    x = it.x;
    f0 = it.f0;
    nf = it.nf;
    const int len = span_chunk(x.len, p.ntc);
    p0 = chunk * len;
    p1 = min(x.sees(span_row(a, f0 + nf - 1)), p0 + len);
    if (p0 >= p1) return;
    slot = p.nwt + p.npc + chunk;
    k = a.tk + (size_t)x.s * a.t_seq + kvh * a.t_head;
    v = a.tv + (size_t)x.s * a.t_seq + kvh * a.t_head;
    lim_all = min(p1, x.sees(span_row(a, f0)));
  }
  const int ns = (p1 - p0 + kSpanStage - 1) / kSpanStage;
  const uint32_t sm = (uint32_t)__cvta_generic_to_shared(smem), kv_s = sm + kPtQ;
  auto fetch = [&](int s) {
    if (s < ns) {
      const uint32_t to = kv_s + (s % kPtStages) * 2 * kPtTile;
#pragma unroll
      for (int i = 0; i < kSpanStage * 16 / (32 * kPtWarps); ++i) {
        const int u = threadIdx.x + i * 32 * kPtWarps, r = u >> 4, c = u & 15;
        const int pos = p0 + s * kSpanStage + r;
        const bool live = pos < p1;
        const size_t at = (size_t)(live ? pos : p0) * kHd + 8 * c;
        cp16(to + swz(r, c), k + at, live);
        cp16(to + kPtTile + swz(r, c), v + at, live);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kPtStages; ++s) fetch(s);
  rows_split<kSpanItem, kPtWarps>(a, kvh, f0, nf, smem, s_fac, warp);

  // warps by eights of rows, then by positions
  const int oct = (nf + 7) / 8;
  const int wo = oct > 4 ? 8 : oct > 2 ? 4 : oct, wp = kPtWarps / wo;
  const int o = warp & (wo - 1), pg = warp / wo;
  const bool mine = o < oct;
  const int fr = f0 + 8 * o + gl;                          // this thread's row
  const bool row_live = mine && fr < f0 + nf;
  const int lim = !row_live ? 0 : prefix ? p1 : min(p1, x.sees(span_row(a, fr)));
  float m = -INFINITY, l = 0.0f;
  float acc[16][2];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i][0] = acc[i][1] = 0.0f;
  __syncthreads();
  const float fac = row_live ? s_fac[8 * o + gl] : 0.0f;
  const int qr = 16 * o + (lane & 15);                     // ldmatrix rows of the 16-row operand
  const uint32_t q_at = sm + qr * 256;
  for (int s = 0; s < ns; ++s) {
    asm volatile("cp.async.wait_group %0;" :: "n"(kPtStages - 1) : "memory");
    __syncthreads();
    const uint32_t kt = kv_s + (s % kPtStages) * 2 * kPtTile, vt = kt + kPtTile;
    const int base = p0 + s * kSpanStage;
    const bool partial = lim_all < min(p1, base + kSpanStage);
    if (partial) {
      // V of positions that some row does not see must be finite, as 0 times it is added there:
      // what is not becomes 0 and takes the rows that see it with it
      if (threadIdx.x < kSpanStage) s_bad[threadIdx.x] = 0;
      __syncthreads();
      for (int u = threadIdx.x; u < kSpanStage * 16; u += 32 * kPtWarps) {
        uint4* w = reinterpret_cast<uint4*>(smem + kPtQ + (s % kPtStages) * 2 * kPtTile + kPtTile + swz(u >> 4, u & 15));
        const uint4 y = *w;
        if (not_finite(y)) {
          *w = make_uint4(0, 0, 0, 0);
          s_bad[u >> 4] = 1;
        }
      }
      __syncthreads();
    }
    // kN times 16 positions at a time, the warps that share rows in turn
    auto unit = [&](int at, auto n_form) {
      constexpr int kN = decltype(n_form)::value;
      const int b = base + at;
      float sc[2 * kN][4];
#pragma unroll
      for (int j = 0; j < 2 * kN; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[j][i] = 0.0f;
#pragma unroll
      for (int kk = 0; kk < 8; ++kk) {
        uint32_t qa[4];
        ldsm(qa, q_at + (((2 * kk + (lane >> 4)) ^ (qr & 7)) << 4));
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          uint32_t kb[4];
          ldsm(kb, kt + swz(at + 16 * j + (lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
          mma_f16(sc[2 * j], qa, kb[0], kb[1]);
          mma_f16(sc[2 * j + 1], qa, kb[2], kb[3]);
        }
      }
      float w[4 * kN];
      float up = m;
      const bool all = b + 16 * kN <= lim_all;
#pragma unroll
      for (int j = 0; j < 4 * kN; ++j) {
        const int pos = b + 8 * (j >> 1) + 2 * t + (j & 1);
        const float y = (sc[j >> 1][j & 1] + sc[j >> 1][2 + (j & 1)]) * fac;
        w[j] = all || pos < lim ? y : -INFINITY;
        up = fmaxf(up, w[j]);
      }
      up = fmaxf(up, __shfl_xor_sync(0xFFFFFFFFu, up, 1));
      up = fmaxf(up, __shfl_xor_sync(0xFFFFFFFFu, up, 2));
      if (__any_sync(0xFFFFFFFFu, up > m)) {
        const float c = m == -INFINITY ? 0.0f : ex2(m - up);
        l *= c;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          acc[i][0] *= c;
          acc[i][1] *= c;
        }
        m = up;
      }
      const float m0 = m == -INFINITY ? 0.0f : m;
      uint32_t wa[kN][4];
#pragma unroll
      for (int j = 0; j < 4 * kN; ++j) {
        w[j] = ex2((w[j] - m0) + kPtLift);       // (m - kPtLift may be m)
        l += w[j];
      }
#pragma unroll
      for (int j = 0; j < 2 * kN; ++j)
        split_half2(w[2 * j], w[2 * j + 1], &wa[j >> 1][2 * (j & 1)], &wa[j >> 1][2 * (j & 1) + 1]);
      if (partial) {
#pragma unroll
        for (int j = 0; j < 4 * kN; ++j) {
          const int pos = b + 8 * (j >> 1) + 2 * t + (j & 1);
          if (pos < lim && s_bad[pos - base]) l = __int_as_float(0x7fc00000);
        }
      }
#pragma unroll
      for (int d = 0; d < 8; ++d) {
        float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          uint32_t vb[4];
          ldsm_t(vb, vt + swz(at + 16 * j + (lane & 15), 2 * d + (lane >> 4)));
          mma_f16(c[0], wa[j], vb[0], vb[1]);
          mma_f16(c[1], wa[j], vb[2], vb[3]);
        }
        add_up(acc[2 * d], c[0]);
        add_up(acc[2 * d + 1], c[1]);
      }
    };
    if (mine) {
      if (wp >= 4) {
        // four warps with the same rows have 16 positions each, eight those of every second stage
        const int at = 16 * (pg & 3);
        if ((wp == 4 || (s & 1) == pg >> 2) && base + at < p1) unit(at, std::integral_constant<int, 1>{});
      } else {
#pragma unroll 1
        for (int u = 0; u < 2; ++u)
          if ((2 * s + u) % wp == pg && base + 32 * u < p1) unit(32 * u, std::integral_constant<int, 2>{});
      }
    }
    __syncthreads();
    fetch(s + kPtStages);
  }
  // the warps that share rows meet
  asm volatile("cp.async.wait_all;" ::: "memory");
  l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
  l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
  if (t == 0) { s_m[warp][gl] = m; s_l[warp][gl] = l; }
  float* line = reinterpret_cast<float*>(smem + kPtQ) + (size_t)warp * 8 * kPtLine;
#pragma unroll
  for (int i = 0; i < 16; ++i)
    *reinterpret_cast<float2*>(line + gl * kPtLine + 8 * i + 2 * t) =
        make_float2(acc[i][0], acc[i][1]);
  __syncthreads();
  const size_t row = ((size_t)slot * gridDim.y + kvh) * F + f0;
#pragma unroll 2
  for (int i = warp; i < nf; i += kPtWarps) {
    const int oo = i >> 3, g = i & 7;
    float M = -INFINITY, L = 0.0f;
    for (int j = 0; j < wp; ++j) M = fmaxf(M, s_m[oo + j * wo][g]);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int j = 0; j < wp; ++j) {
      const int w = oo + j * wo;
      const float c = s_l[w][g] == 0.0f ? 0.0f : ex2(s_m[w][g] - M);
      const float4 z = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem + kPtQ) + (size_t)w * 8 * kPtLine + g * kPtLine + 4 * lane);
      L += c * s_l[w][g];
      y.x += c * z.x; y.y += c * z.y; y.z += c * z.z; y.w += c * z.w;
    }
    reinterpret_cast<float4*>(p.part + (row + i) * kHd)[lane] = dropped(y);
    if (lane == 0) p.ml[row + i] = make_float2(M, L * kPtDrop);
  }
}

__global__ void __launch_bounds__(32 * kPtWarps, 2) k_span_part(SpanArgs a, SpanParts p, int tiles) {
  next_may_start();
  span_part(a, p, tiles);
  if ((blockIdx.x | blockIdx.y | threadIdx.x) == 0) prior_done();
}

// ---- attention of up to eight rows ---------------------------------------------------------
//
// One item of eight (row, head) pairs and a chunk of positions a CTA, as for k_span_part, but every
// warp has all rows, takes 16 positions in turn with the others and has a ring of its own for them,
// so that no warp waits for another before the end. With four warps two CTAs fit an SM, with two
// six and with one ten: short items want few warps, as they are over in a few steps, and few
// items many. One row over a long cache is bound by HBM (39999 positions of 8 heads: 164 MB in 33 us),
// most calls by the chain of an item: lengths, rows and first blocks, steps, the warps' meeting
// (4 us).
constexpr int kFwBlock = 16;
constexpr int kFwTile = kFwBlock * kHd * 2;              // bytes of K or of V of 16 positions
constexpr int kFwQ = 2 * kFewRows * kHd * 2;
constexpr int few_stages(int warps) { return warps == 4 ? 3 : 2; }
constexpr int few_smem(int warps) { return kFwQ + warps * few_stages(warps) * 2 * kFwTile; }

template <int kFwWarps>
HV_DEV void span_few(const SpanArgs& a, const SpanParts& p, int tiles) {
  constexpr int kFwStages = few_stages(kFwWarps);
  extern __shared__ __align__(1024) uint8_t smem[];         // the rows, then the warps' rings
  __shared__ float s_fac[kFewRows], s_m[kFwWarps][8], s_l[kFwWarps][8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, F = a.nrow * a.group;
  const __half *k, *v;
  int f0, nf, p0, p1, slot, lim_all;
  SpanSeq x;
  const bool prefix = blockIdx.x < (unsigned)(tiles * p.npc);
  if (prefix) {
    const int tile = blockIdx.x / p.npc, chunk = blockIdx.x % p.npc;
    f0 = tile * kFewRows;
    nf = min(kFewRows, F - f0);
    const int n = span_sees(a, span_prefix(a), f0 + nf - 1), len = span_chunk(n, p.npc);
    p0 = chunk * len;
    p1 = min(n, p0 + len);
    slot = p.nwt + chunk;
    k = a.pk + kvh * a.p_head;
    v = a.pv + kvh * a.p_head;
    lim_all = a.run ? min(p1, a.plen + span_row(a, f0) + 1) : p1;
  } else {
    const int b = blockIdx.x - tiles * p.npc, chunk = b % p.ntc;
    const SpanItem it = span_item(a, b / p.ntc, kFewRows);
    if (it.nf == 0 || it.x.len <= 0) return;
    x = it.x;
    f0 = it.f0;
    nf = it.nf;
    const int len = span_chunk(x.len, p.ntc);
    p0 = chunk * len;
    p1 = min(x.sees(span_row(a, f0 + nf - 1)), p0 + len);
    slot = p.nwt + p.npc + chunk;
    k = a.tk + (size_t)x.s * a.t_seq + kvh * a.t_head;
    v = a.tv + (size_t)x.s * a.t_seq + kvh * a.t_head;
    lim_all = min(p1, x.sees(span_row(a, f0)));
  }
  if (p0 >= p1) return;
  const int nb = (p1 - p0 + kFwBlock - 1) / kFwBlock;
  const uint32_t sm = (uint32_t)__cvta_generic_to_shared(smem);
  uint8_t* ring = smem + kFwQ + warp * kFwStages * 2 * kFwTile;
  const uint32_t ring_s = sm + kFwQ + warp * kFwStages * 2 * kFwTile;
  auto fetch = [&](int b, int stage) {
    if (b < nb) {
      const uint32_t to = ring_s + stage * 2 * kFwTile;
#pragma unroll
      for (int i = 0; i < kFwBlock * 16 / 32; ++i) {
        const int u = lane + 32 * i, r = u >> 4, c = u & 15, pos = p0 + b * kFwBlock + r;
        const bool live = pos < p1;
        const size_t at = (size_t)(live ? pos : p0) * kHd + 8 * c;
        cp16(to + swz(r, c), k + at, live);
        cp16(to + kFwTile + swz(r, c), v + at, live);
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kFwStages; ++s) fetch(warp + s * kFwWarps, s);
  rows_split<kFewRows, kFwWarps>(a, kvh, f0, nf, smem, s_fac, warp);
  __syncthreads();
  const int fr = f0 + gl;
  const bool row_live = gl < nf;
  const int lim = !row_live ? 0 : a.run ? min(p1, a.plen + span_row(a, fr) + 1) : prefix ? p1 : min(p1, x.sees(span_row(a, fr)));
  const float fac = row_live ? s_fac[gl] : 0.0f;
  uint32_t qa[8][4];
#pragma unroll
  for (int kk = 0; kk < 8; ++kk) ldsm(qa[kk], sm + swz(lane & 15, 2 * kk + (lane >> 4)));
  float m = -INFINITY, l = 0.0f;
  float acc[16][2];
#pragma unroll
  for (int i = 0; i < 16; ++i) acc[i][0] = acc[i][1] = 0.0f;
  int stage = 0;
#pragma unroll 1
  for (int b = warp; b < nb; b += kFwWarps) {
    asm volatile("cp.async.wait_group %0;" :: "n"(kFwStages - 1) : "memory");
    __syncwarp();
    const uint32_t kt = ring_s + stage * 2 * kFwTile, vt = kt + kFwTile;
    const int base = p0 + b * kFwBlock;
    const bool all = base + kFwBlock <= lim_all;
    unsigned bad = 0;
    if (lim_all < min(p1, base + kFwBlock)) {
      // V of positions that some row does not see: as in k_span_part
      uint8_t* vs = ring + stage * 2 * kFwTile + kFwTile;
#pragma unroll
      for (int i = 0; i < kFwBlock * 16 / 32; ++i) {
        const int u = lane + 32 * i;
        uint4* w = reinterpret_cast<uint4*>(vs + swz(u >> 4, u & 15));
        if (not_finite(*w)) {
          *w = make_uint4(0, 0, 0, 0);
          bad |= 1u << (u >> 4);
        }
      }
      bad = __reduce_or_sync(0xFFFFFFFFu, bad);
      __syncwarp();
    }
    float sc[2][4];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[j][i] = 0.0f;
#pragma unroll
    for (int kk = 0; kk < 8; ++kk) {
      uint32_t kb[4];
      ldsm(kb, kt + swz((lane & 7) + ((lane >> 4) << 3), 2 * kk + ((lane >> 3) & 1)));
      mma_f16(sc[0], qa[kk], kb[0], kb[1]);
      mma_f16(sc[1], qa[kk], kb[2], kb[3]);
    }
    float w[4];
    float up = m;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int pos = base + 8 * (j >> 1) + 2 * t + (j & 1);
      const float y = (sc[j >> 1][j & 1] + sc[j >> 1][2 + (j & 1)]) * fac;
      w[j] = all || pos < lim ? y : -INFINITY;
      up = fmaxf(up, w[j]);
    }
    if (p.scores && row_live) {
      float* to = p.scores + ((size_t)kvh * a.group + fr) * p.scores_ld;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int pos = base + 8 * (j >> 1) + 2 * t + (j & 1);
        if (pos < p1) to[pos] = w[j];
      }
    }
    up = fmaxf(up, __shfl_xor_sync(0xFFFFFFFFu, up, 1));
    up = fmaxf(up, __shfl_xor_sync(0xFFFFFFFFu, up, 2));
    if (__any_sync(0xFFFFFFFFu, up > m)) {
      const float c = m == -INFINITY ? 0.0f : ex2(m - up);
      l *= c;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        acc[i][0] *= c;
        acc[i][1] *= c;
      }
      m = up;
    }
    const float m0 = m == -INFINITY ? 0.0f : m;
    uint32_t wa[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      w[j] = ex2((w[j] - m0) + kPtLift);       // (m - kPtLift may be m)
      l += w[j];
    }
    if (bad) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int at = 8 * (j >> 1) + 2 * t + (j & 1);
        if (base + at < lim && (bad >> at & 1)) l = __int_as_float(0x7fc00000);
      }
    }
    split_half2(w[0], w[1], &wa[0], &wa[1]);
    split_half2(w[2], w[3], &wa[2], &wa[3]);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      uint32_t vb[4];
      float c[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      ldsm_t(vb, vt + swz(lane & 15, 2 * d + (lane >> 4)));
      mma_f16(c[0], wa, vb[0], vb[1]);
      mma_f16(c[1], wa, vb[2], vb[3]);
      add_up(acc[2 * d], c[0]);
      add_up(acc[2 * d + 1], c[1]);
    }
    __syncwarp();
    fetch(b + kFwStages * kFwWarps, stage);
    stage = stage + 1 == kFwStages ? 0 : stage + 1;
  }
  // the warps meet
  asm volatile("cp.async.wait_all;" ::: "memory");
  l += __shfl_xor_sync(0xFFFFFFFFu, l, 1);
  l += __shfl_xor_sync(0xFFFFFFFFu, l, 2);
  if (t == 0) { s_m[warp][gl] = m; s_l[warp][gl] = l; }
  __syncthreads();                                         // the rings are free
  float* lines = reinterpret_cast<float*>(smem + kFwQ);
#pragma unroll
  for (int i = 0; i < 16; ++i)
    *reinterpret_cast<float2*>(lines + (warp * 8 + gl) * kPtLine + 8 * i + 2 * t) =
        make_float2(acc[i][0], acc[i][1]);
  __syncthreads();
  const size_t row = ((size_t)slot * gridDim.y + kvh) * F + f0;
  for (int g = warp; g < nf; g += kFwWarps) {
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int j = 0; j < kFwWarps; ++j) M = fmaxf(M, s_m[j][g]);
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kFwWarps; ++j) {
      const float c = s_l[j][g] == 0.0f ? 0.0f : ex2(s_m[j][g] - M);
      const float4 z = *reinterpret_cast<const float4*>(lines + (j * 8 + g) * kPtLine + 4 * lane);
      L += c * s_l[j][g];
      y.x += c * z.x; y.y += c * z.y; y.z += c * z.z; y.w += c * z.w;
    }
    reinterpret_cast<float4*>(p.part + (row + g) * kHd)[lane] = dropped(y);
    if (lane == 0) p.ml[row + g] = make_float2(M, L * kPtDrop);
  }
}

template <int kFwWarps>
__global__ void __launch_bounds__(32 * kFwWarps, kFwWarps == 1 ? 11 : kFwWarps == 2 ? 6 : 2) k_span_few(SpanArgs a, SpanParts p, int tiles) {
  next_may_start();
  span_few<kFwWarps>(a, p, tiles);
  if ((blockIdx.x | blockIdx.y | threadIdx.x) == 0) prior_done();
}

// ---- a row's chunks added up -----------------------------------------------------------------
//
// kWarps warps share a row's slots, kPer rows a CTA (all of one tile of kStRows): one warp a row
// where slots are few, with several rows after each other where rows are many, so that the fixed
// part (which slots there are) is spread over them; four where a row's loads would follow each other
// (16 sequences over 4096 positions, 512 rows of up to 20 slots: 21.1 us for the call, 23.2 by one). A row's sequence is looked up
// before the wait for the parts: 1 us of the 3 that the join adds to a call.
template <int kWarps, int kPer>
HV_DEV void span_join(const SpanArgs& a, const SpanParts& p) {
  constexpr int kAt = kWarps == 1 ? 4 : 8;                 // slots' rows under way
  __shared__ float4 s_sum[8][32];
  __shared__ float2 s_ml[8];
  const int kvh = blockIdx.y, F = a.nrow * a.group, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int fb = blockIdx.x * kPer;             // the CTA's first row
  const int np = span_prefix(a);
  const size_t step = (size_t)gridDim.y * F;
  const float nan = __int_as_float(0x7fc00000);
  SpanSeq x;
  auto find = [&](int i) { return fb + i < F && span_find(a, span_row(a, fb + i), &x); };
  bool here = find(warp / kWarps);                         // the same for the row's warps
  prior_done();
  // its stretches of tiles
  int nw = 0;
  if (p.nwt && fb < F && span_tiles_of(a, np, fb / kStRows))
    nw = __ldcg(p.stretches + kvh * ((F + kStRows - 1) / kStRows) + fb / kStRows);
#pragma unroll 1
  for (int i = warp / kWarps; i < kPer; i += 8 / kWarps, here = kPer > 8 / kWarps && i < kPer && find(i)) {
    const int f = fb + i;
    if (f >= F) {
      const int Fp = (F + kStRows - 1) / kStRows * kStRows;
      if (p.terms && f < Fp && lane < 2) p.facs[((size_t)lane * gridDim.y + kvh) * Fp + f] = lane ? -INFINITY : 0.0f;
      if (kWarps == 1) continue;
    }
    const int r = span_row(a, f);
    if (kWarps == 1 && !here) continue;
    const size_t at = (size_t)kvh * F + f;
    const bool no = here && (np < 0 || x.len < 0);
    // its chunks of the prefix, its chunks of the tail
    int n0 = 0, n1 = 0;
    if (here && !no && p.npc) {
      const int n = span_sees(a, np, min(F, (f / p.size + 1) * p.size) - 1), len = span_chunk(n, p.npc);
      if (n > 0) n0 = (span_sees(a, np, f) + len - 1) / len;
    }
    if (here && !no && p.ntc) {
      const int see = x.sees(r);
      if (see) n1 = p.ntc == 1 ? 1 : (see + span_chunk(x.len, p.ntc) - 1) / span_chunk(x.len, p.ntc);
    }
    const int all = here && !no ? nw + n0 + n1 : 0;
    auto slot = [&](int k) {
      const int j = k * kWarps + warp % kWarps;            // this warp's k-th
      return at + (j < nw ? j : j < nw + n0 ? p.nwt + j - nw : p.nwt + p.npc + j - nw - n0) * step;
    };
    const int mine = (all - warp % kWarps + kWarps - 1) / kWarps;
    // a lane has a chunk's maximum and sum, 32 chunks at a time; the rows' sums are loaded before
    // those are known, kAt at a time
    float M = -INFINITY, L = 0.0f;
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 1
    for (int i0 = 0; i0 < mine; i0 += 32) {
      const int n = min(32, mine - i0);
      float4 y[kAt];
      auto load = [&](int j0) {
#pragma unroll
        for (int j = 0; j < kAt; ++j)
          if (j0 + j < n) y[j] = __ldcg(reinterpret_cast<const float4*>(p.part + slot(i0 + j0 + j) * kHd) + lane);
      };
      const float2 ml = lane < n ? __ldcg(p.ml + slot(i0 + lane)) : make_float2(-INFINITY, 0.0f);
      load(0);
      float up = fmaxf(M, ml.x);
#pragma unroll
      for (int d = 16; d; d >>= 1) up = fmaxf(up, __shfl_xor_sync(0xFFFFFFFFu, up, d));
      const float c = ml.y == 0.0f ? 0.0f : ex2(ml.x - up), old = M == -INFINITY ? 0.0f : ex2(M - up);
      float sum = c * ml.y;
#pragma unroll
      for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, d);
      M = up;
      L = L * old + sum;
      s.x *= old; s.y *= old; s.z *= old; s.w *= old;
#pragma unroll 1
      for (int j0 = 0; j0 < n; j0 += kAt) {
        if (j0) load(j0);
#pragma unroll
        for (int j = 0; j < kAt; ++j) {
          if (j0 + j >= n) continue;
          const float g = __shfl_sync(0xFFFFFFFFu, c, j0 + j);
          s.x += g * y[j].x; s.y += g * y[j].y; s.z += g * y[j].z; s.w += g * y[j].w;
        }
      }
    }
    if constexpr (kWarps > 1) {
      s_sum[warp][lane] = s;
      if (lane == 0) s_ml[warp] = make_float2(M, L);
      __syncthreads();                                     // (one round: kPer is 8 / kWarps)
      if (warp % kWarps != 0) continue;
      for (int j = 1; j < kWarps; ++j) M = fmaxf(M, s_ml[warp + j].x);
      L = 0.0f;
      s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
      for (int j = 0; j < kWarps; ++j) {
        const float2 ml = s_ml[warp + j];
        const float g = ml.y == 0.0f ? 0.0f : ex2(ml.x - M);
        const float4 z = s_sum[warp + j][lane];
        L += g * ml.y;
        s.x += g * z.x; s.y += g * z.y; s.z += g * z.z; s.w += g * z.w;
      }
      if (!here) continue;
    }
    const float inv = no ? nan : all ? 1.0f / L : 0.0f;
    if (no) L = nan;
    const size_t out = ((size_t)r * a.nq + (size_t)kvh * a.group + f - r * a.group) * kHd;
    reinterpret_cast<float4*>(a.ctx + out)[lane] = make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
    if (p.stat && lane == 0) p.stat[at] = make_float2(M, L);
    if (p.terms) {
      const float4 q = __ldg(reinterpret_cast<const float4*>(a.q + out) + lane);
      uint2 hi, lo;
      const float lift = row_terms(q, &hi, &lo);
      reinterpret_cast<uint2*>(p.terms + at * kHd)[lane] = hi;
      reinterpret_cast<uint2*>(p.terms + (at + step) * kHd)[lane] = lo;
      const int Fp = (F + kStRows - 1) / kStRows * kStRows;
      if (lane < 2)
        p.facs[((size_t)lane * gridDim.y + kvh) * Fp + f] = lane ? -(span_top(M) + log2f(L)) : __ldg(a.scale) * kLog2e / lift;
    }
  }
}

template <int kWarps, int kPer>
__global__ void __launch_bounds__(256, kWarps == 1 ? 4 : 3) k_span_join(SpanArgs a, SpanParts p) {
  next_may_start();
  span_join<kWarps, kPer>(a, p);
}

// A single row's end: its chunks added up by the first CTAs of a kv head, and by the others the
// weights of the scores that k_span_few has left, 1024 positions each (39999 positions, 64 q over 8
// kv heads: 51 us for the call with two launches in place of this one, 39 with it).
constexpr int kOnePos = 1024;
__global__ void __launch_bounds__(256) k_span_one(SpanArgs a, SpanParts p, const float* mass_in, float* mass_out, int joins) {
  if ((int)blockIdx.x < joins) return span_join<4, 2>(a, p);
  __shared__ float2 s_one[8];
  const int kvh = blockIdx.y, np = span_prefix(a), lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int t0 = (blockIdx.x - joins) * kOnePos + 4 * threadIdx.x;
  prior_done();
  if (np < 0 || t0 - 4 * (int)threadIdx.x >= np) return;
  const float* scores = p.scores + (size_t)kvh * a.group * p.scores_ld + t0;
  float4 x[8];
#pragma unroll
  for (int h = 0; h < 8; ++h)
    if (h < a.group && t0 < np) x[h] = __ldcg(reinterpret_cast<const float4*>(scores + (size_t)h * p.scores_ld));
  const size_t i = (size_t)kvh * a.pcap + t0;
  float in[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) in[k] = mass_in && t0 + k < np - 1 ? mass_in[i + k] : 0.0f;
  const int len = span_chunk(np, p.npc), n0 = (np + len - 1) / len;
  if (warp < a.group) {
    const size_t at = (size_t)kvh * a.group + warp, step = (size_t)gridDim.y * a.group;
    float M = -INFINITY, L = 0.0f;
    for (int c = lane; c < n0; c += 32) {
      const float2 ml = __ldcg(p.ml + at + c * step);
      const float up = fmaxf(M, ml.x);
      L = (M == -INFINITY ? 0.0f : L * ex2(M - up)) + (ml.y == 0.0f ? 0.0f : ex2(ml.x - up) * ml.y);
      M = up;
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) {
      const float m2 = __shfl_xor_sync(0xFFFFFFFFu, M, d), l2 = __shfl_xor_sync(0xFFFFFFFFu, L, d), up = fmaxf(M, m2);
      L = (L == 0.0f ? 0.0f : L * ex2(M - up)) + (l2 == 0.0f ? 0.0f : l2 * ex2(m2 - up));
      M = up;
    }
    if (lane == 0) s_one[warp] = make_float2(M, 1.0f / L);
  }
  __syncthreads();
  float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int h = 0; h < 8; ++h) {
    if (h >= a.group) break;
    const float2 s = s_one[h];
    sum[0] += ex2(x[h].x - s.x) * s.y;
    sum[1] += ex2(x[h].y - s.x) * s.y;
    sum[2] += ex2(x[h].z - s.x) * s.y;
    sum[3] += ex2(x[h].w - s.x) * s.y;
  }
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (t0 + k < np) mass_out[i + k] = in[k] + sum[k];
}

// ---- the weights that a run's rows give ------------------------------------------------------
//
// w = 2^(x - m) / l once every row's m and l are known, so the scores are formed again, this time
// with the positions as the 16-row operand: a thread then has two positions and adds up over
// the columns, the rows. wpos of a CTA's warps have 16 positions each, and wpos warps at a time
// take the rows in turn, 64 to a stage, split as k_span_part splits them. Bound by the f16 pipe where
// rows or positions are many, else by its chain of row stages (16 rows at 8176, 8 q over 8 kv heads:
// 22.7 us for the call, 30 by tiles; 256 at 704, 32 over 8: 30.6 and 22.6).
template <int kPos>                                        // warps with positions of their own
__global__ void __launch_bounds__(256) k_mass_rows(SpanArgs a, SpanParts p, const float* mass_in, float* mass_out, int cap) {
  extern __shared__ __align__(1024) uint8_t smem[];         // 64 rows' two terms, then K
  __shared__ float s_fac[kSpanItem], s_part[8][16];
  __shared__ float2 s_stat[kSpanItem];
  constexpr int kN = 16 * kPos;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, F = a.nrow * a.group, p0 = blockIdx.x * kN;
  const int n = a.plen + a.nrow;
  if (p0 >= n) return;                                      // (the others wait)
  uint8_t* ks = smem + kPtQ;
  for (int u = threadIdx.x; u < kN * 16; u += 256) {
    const int r = u >> 4, pos = p0 + r;
    uint4 x = make_uint4(0, 0, 0, 0);
    if (pos < n) x = __ldg(reinterpret_cast<const uint4*>(a.pk + kvh * a.p_head + (size_t)pos * kHd) + (u & 15));
    *reinterpret_cast<uint4*>(ks + swz(r, u & 15)) = x;
  }
  __syncthreads();
  const int wpos = warp % kPos, wrow = warp / kPos;
  uint32_t ka[8][4];
  {
    const int r = 16 * wpos + (lane & 15);
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(ks);
#pragma unroll
    for (int k = 0; k < 8; ++k) ldsm(ka[k], at + swz(r, 2 * k + (lane >> 4)));
  }
  // the first (row, head) pair that sees each of the thread's two positions
  const int pos_a = p0 + 16 * wpos + gl, pos_b = pos_a + 8;
  const int see_a = max(0, pos_a - a.plen) * a.group, see_b = max(0, pos_b - a.plen) * a.group;
  const uint32_t q_at = (uint32_t)__cvta_generic_to_shared(smem);
  float sum_a = 0.0f, sum_b = 0.0f;
  const int first = max(0, p0 - a.plen) * a.group / kSpanItem * kSpanItem;   // rows before see none of it
  const float scale = __ldg(a.scale) * kLog2e;
  float4 x[kSpanItem / 8];                                  // the next stage's rows
  rows_load<kSpanItem, 8>(a, kvh, first, min(kSpanItem, F - first), warp, x);
  prior_done();
  for (int f0 = first; f0 < F; f0 += kSpanItem) {
    const int nf = min(kSpanItem, F - f0);
    __syncthreads();
    rows_put<kSpanItem, 8>(x, scale, nf, smem, s_fac, warp);
    if (f0 + kSpanItem < F) rows_load<kSpanItem, 8>(a, kvh, f0 + kSpanItem, min(kSpanItem, F - f0 - kSpanItem), warp, x);
    if (threadIdx.x < nf) {
      const float2 s = __ldcg(p.stat + (size_t)kvh * F + f0 + threadIdx.x);
      s_stat[threadIdx.x] = make_float2(span_top(s.x), 1.0f / s.y);
    }
    __syncthreads();
    for (int o = wrow; o < (nf + 7) / 8; o += 8 / kPos) {
      float c[4] = {0.f, 0.f, 0.f, 0.f}, d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        uint32_t b[4];
        ldsm(b, q_at + swz(16 * o + (lane & 7) + ((lane >> 4) << 3), 2 * k + ((lane >> 3) & 1)));
        mma_f16(d, ka[k], b[2], b[3]);
        mma_f16(c, ka[k], b[0], b[1]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int j = 8 * o + 2 * t + i;
        if (j < nf) {
          const float fac = s_fac[j];
          const float2 s = s_stat[j];
          const float wa = ex2(fmaf(c[i] + d[i], fac, -s.x)), wb = ex2(fmaf(c[2 + i] + d[2 + i], fac, -s.x));
          if (f0 + j >= see_a) sum_a = fmaf(wa, s.y, sum_a);
          if (f0 + j >= see_b) sum_b = fmaf(wb, s.y, sum_b);
        }
      }
    }
  }
#pragma unroll
  for (int i = 1; i < 4; i <<= 1) {
    sum_a += __shfl_xor_sync(0xFFFFFFFFu, sum_a, i);
    sum_b += __shfl_xor_sync(0xFFFFFFFFu, sum_b, i);
  }
  if (t == 0) { s_part[warp][gl] = sum_a; s_part[warp][gl + 8] = sum_b; }
  __syncthreads();
  if (threadIdx.x < kN && p0 + threadIdx.x < n) {
    float s = 0.0f;
#pragma unroll
    for (int w = 0; w < 8 / kPos; ++w) s += s_part[(threadIdx.x >> 4) + w * kPos][threadIdx.x & 15];
    const size_t i = (size_t)kvh * cap + p0 + threadIdx.x;
    mass_out[i] = (mass_in && p0 + (int)threadIdx.x < a.plen ? mass_in[i] : 0.0f) + s;
  }
}

// hv_qk_rows's arithmetic for the rows of a batch. Eight lanes have a head, lane j its dims j, j + 8,
// ..: those are numpy's accumulator j of the sum of squares, and a dim's partner in the rotation is
// the same lane's, so that a head takes three shuffles and no shared memory (a warp a head, as
// k_qk_rows has it: 228 rows of 64 + 8 heads 10.5 us).
constexpr int kQkWarps = 2;             // of a CTA: few rows are to be spread over the SMs
__global__ void __launch_bounds__(32 * kQkWarps) k_qk_shared(const float* __restrict__ qkv, const float* __restrict__ qn,
                                                   const float* __restrict__ kn, const float* __restrict__ cos_t,
                                                   const float* __restrict__ sin_t, int cap,
                                                   const int32_t* __restrict__ base, SpanArgs a,
                                                   float* __restrict__ q_out, __half* tk, __half* tv,
                                                   int nkv, float eps) {
  const int heads = a.nq + nkv, per = (heads + 3) / 4;     // warps a row
  const long long wi = (long long)blockIdx.x * kQkWarps + (threadIdx.x >> 5);
  const int r = (int)(wi / per), h = 4 * (int)(wi - (long long)r * per) + ((threadIdx.x & 31) >> 3), j = threadIdx.x & 7;
  if (r >= a.nrow) return;                                 // whole warps
  const float* row = qkv + (size_t)r * (a.nq + 2 * nkv) * kHd + j;
  const bool here = h < heads, is_q = h < a.nq;
  float x[16], v[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    x[i] = here ? __ldg(row + (size_t)h * kHd + 8 * i) : 0.0f;
    v[i] = here && !is_q ? __ldg(row + (size_t)(h + nkv) * kHd + 8 * i) : 0.0f;
  }
  const int first = __ldg(base);
  SpanSeq s;
  if (!span_find(a, r, &s)) return;
  const int slot = s.len - (s.end - r);
  const long long pos = (long long)first + slot;
  const bool ok = s.len >= 0 && slot >= 0 && pos >= 0 && pos < cap;
  float* q = q_out + ((size_t)r * a.nq + h) * kHd + j;
  if (!ok) {
    if (is_q)
#pragma unroll
      for (int i = 0; i < 16; ++i) q[8 * i] = __int_as_float(0x7fc00000);
    return;
  }
  // the norm, as warp_norm_rope forms it
  float ss = __fmul_rn(x[0], x[0]);
#pragma unroll
  for (int i = 1; i < 16; ++i) ss = __fadd_rn(ss, __fmul_rn(x[i], x[i]));
#pragma unroll
  for (int d = 1; d < 8; d <<= 1) ss = __fadd_rn(ss, __shfl_xor_sync(0xFFFFFFFFu, ss, d));
  if (!here) return;
  const float d = __fsqrt_rn(__fadd_rn(__fdiv_rn(__fadd_rn(0.0f, ss), (float)kHd), eps));
  const float* gain = (is_q ? qn : kn) + j;
#pragma unroll
  for (int i = 0; i < 16; ++i) x[i] = __fmul_rn(__ldg(gain + 8 * i), __fdiv_rn(x[i], d));
  const float* cs = cos_t + (size_t)pos * (kHd / 2) + j;
  const float* sn = sin_t + (size_t)pos * (kHd / 2) + j;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = __ldg(cs + 8 * i), t = __ldg(sn + 8 * i), lo = x[i], hi = x[i + 8];
    x[i] = __fsub_rn(__fmul_rn(lo, c), __fmul_rn(hi, t));
    x[i + 8] = __fadd_rn(__fmul_rn(hi, c), __fmul_rn(lo, t));
  }
  if (is_q) {
#pragma unroll
    for (int i = 0; i < 16; ++i) q[8 * i] = x[i];
    return;
  }
  const size_t at = (size_t)s.s * a.t_seq + (h - a.nq) * a.t_head + (size_t)slot * kHd + j;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    tk[at + 8 * i] = __float2half_rn(x[i]);
    tv[at + 8 * i] = __float2half_rn(v[i]);
  }
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
void span_group(SpanArgs* a, int group) {
  a->group = group;
  a->inv = ((1ull << 32) + group - 1) / group;
}
bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// How a call's positions are cut, by its capacities (the lengths are on the device): as many
// chunks as give every SM two CTAs, of a stage at the least.
constexpr int kSms = 148, kPtCtas = 2 * kSms, kFwCtas2 = 6 * kSms;   // that run at once; k_span_few<2>
struct SpanPlan {
  int size, tiles, items, nwt, npc, ntc;   // tiles of the prefix's rows, items of the tails'
  int grid;                                // CTAs of k_span_tile
  size_t part, ml, stretches, stat, scores, terms, facs, bytes;
  bool mass_tiles;
  int few;                                 // warps of k_span_few, or 0: k_span_part
};
SpanPlan span_plan(int nkv, int F, int nseq, int pcap, int tcap, bool run, bool mass) {
  SpanPlan p{};
  auto stages = [](int n) { return (n + kSpanStage - 1) / kSpanStage; };
  // Many rows over many positions go by whole tiles, whose kernel takes 10 us for the first of them
  // (256 pairs a head, 8 heads: over 512 positions 18 us, and 25 by eights; over 256 14 and 11; a
  // run's 128 over 1280 26.5 and 24.6, over 2048 24.6 and 26.6)
  const long long work = (long long)nkv * F * pcap;
  if (F > 32 && work >= (run ? 3 : 2) << 19) {
    const long long rows = (long long)nkv * ((F + kStRows - 1) / kStRows);
    if (rows * ((pcap + kStRows - 1) / kStRows) < 1ll << 31)
      p.nwt = (int)std::min((long long)((pcap + kStRows - 1) / kStRows), kSms / rows + 2);
  }
  // Eights of rows, four warps to an item, as long as all items find room at once: an item is over
  // sooner then. Else two, or one where only short tails are left (256 sequences of one row, tails
  // up to 250, group 4: 97 us with four, 84 with two; tails up to 20: 65 and, with one, 50; a run of
  // 64 at 0, 64 q over 8 kv heads: 33, 28; of 16 at 1000: 21, 23, and 27 by k_span_part). k_span_part
  // has long tails of many rows (24 runs of 3 to 17 rows, tails of 1000: group 4 109 us, and 90 by
  // fours; group 8 145 and 153).
  const int eights = (F + kFewRows - 1) / kFewRows;
  const bool tails = !run && p.nwt;
  const long long items = (long long)nkv * (run ? eights : std::max(nseq, eights) + (p.nwt ? 0 : eights));
  if (F <= kFewRows || items <= kPtCtas) p.few = 4;
  else if (run || tcap <= 256) p.few = tails && tcap <= 32 ? 1 : 2;
  else if (F / nseq <= 2 * kFewRows || (F / nseq <= 64 && (long long)nkv * (eights + nseq) <= 8 * kSms)) p.few = !tails && F / nseq <= kFewRows ? 2 : 4;
  p.size = p.few ? kFewRows : kSpanItem;
  p.tiles = (F + p.size - 1) / p.size;
  p.items = run ? 0 : nseq + p.tiles;
  // Chunks: as many as run at once, the prefix's and the tails' by their shares of the work
  const int fit = p.few == 2 && !tails ? kFwCtas2 : kPtCtas, lines = std::max(nseq, p.tiles);
  const long long work_t = (long long)lines * stages(tcap), work_p = tails ? 0 : (long long)p.tiles * stages(pcap);
  if (!run) p.ntc = std::min(stages(tcap), (int)std::max(1ll, fit * work_t / (work_t + work_p) / ((long long)nkv * lines)));
  if (!p.nwt) p.npc = std::min(stages(pcap), std::max(1, (fit / nkv - (run ? 0 : lines * p.ntc)) / p.tiles));
  // Where few tiles are a CTA's, they go to fewer CTAs, so that the tails run on the SMs that leaves
  // (times in us: of a CTA's n tiles and of an item, as measured). 16 sequences over 4096
  // positions, tails up to 250, 32 q over 8 kv heads: 21.3 us with 128 CTAs for the tiles, 18.8 with 88;
  // 64 over 2000, 16 q: 29.5 and 21.8.
  p.grid = kSms;
  if (tails) {
    const int rows = nkv * ((F + kStRows - 1) / kStRows), whole = (pcap + kStRows - 1) / kStRows;
    const int warps = p.few ? p.few : 8, at_once = p.few == 1 ? 10 : p.few == 2 ? 6 : 2;
    const int chunk = span_chunk(tcap, p.ntc), steps = (chunk + 16 * warps - 1) / (16 * warps);
    const float item = p.few ? 2.3f + std::max(2, steps) : 4.0f + 2.5f * (chunk / kSpanStage);
    auto tiles_take = [](float n) { return 9.0f + 1.4f * std::min(n - 1, 6.0f) + 1.8f * std::max(n - 7, 0.0f); };
    const long long all_items = (long long)nkv * lines * p.ntc;
    auto behind = [&](long long n) { return item * ((n + at_once * kSms - 1) / (at_once * kSms)); };
    // evenly cut among all SMs, where most CTAs go from one tile of rows to the next
    float best = tiles_take((float)rows * whole / kSms + 3) + behind(all_items);
    for (int each = std::min(kSms / rows, whole), last = 0; each > 0; --each) {
      const int share = (whole + each - 1) / each;
      if (share == last) continue;
      last = share;
      const int ctas = rows * ((whole + share - 1) / share);
      const float time = tiles_take(share);
      const long long beside = (long long)(at_once * (kSms - ctas) * (time / item));
      const float all_time = time + behind(std::max(0ll, all_items - beside));
      if (all_time < best) {
        best = all_time;
        p.grid = ctas;
      }
      if (time > best) break;
    }
  }
  // room for this call and any smaller one, which may have more chunks of fewer rows: chunks times
  // tiles (or sequences) are at most what fits / nkv, or one each
  const size_t all = (size_t)nkv * F;
  auto room = [&](int n) {
    return std::min((size_t)stages(n) * all, (size_t)std::max(kPtCtas * std::min(F, kSpanItem), kFwCtas2 * std::min(F, kFewRows)) + all);
  };
  const size_t whole = std::min((size_t)((pcap + kStRows - 1) / kStRows) * all, (size_t)kSms * std::min(F, kStRows) + 2 * all);
  const size_t rows = whole + room(pcap) + (run ? 0 : room(tcap));
  auto up = [](size_t n) { return (n + 255) & ~(size_t)255; };
  p.part = up(rows * kHd * 4);
  p.ml = up(rows * 8);
  p.stretches = up((size_t)nkv * ((F + kStRows - 1) / kStRows) * 4);
  p.stat = up(mass ? (size_t)nkv * F * 8 : 0);
  p.scores = up(mass ? (size_t)nkv * 8 * (pcap + 4) * 4 : 0);
  p.terms = up(mass ? 2 * all * kHd * 2 : 0);
  p.facs = up(mass ? 2 * (size_t)nkv * (F + kStRows) * 4 : 0);
  p.bytes = p.part + p.ml + p.stretches + p.stat + p.scores + p.terms + p.facs + 256;
  return p;
}
SpanParts span_parts(const SpanPlan& p, void* scratch, int pcap, bool mass, bool scores) {
  uint8_t* at = reinterpret_cast<uint8_t*>(scratch);
  SpanParts s{};
  s.part = reinterpret_cast<float*>(at);
  s.ml = reinterpret_cast<float2*>(at + p.part);
  at += p.part + p.ml;
  s.stretches = reinterpret_cast<int32_t*>(at);
  at += p.stretches;
  s.stat = mass ? reinterpret_cast<float2*>(at) : nullptr;
  at += p.stat;
  s.scores = scores ? reinterpret_cast<float*>(at) : nullptr;
  at += p.scores;
  s.terms = p.mass_tiles ? reinterpret_cast<__half*>(at) : nullptr;
  s.facs = reinterpret_cast<float*>(at + p.terms);
  s.nwt = p.nwt;
  s.npc = p.npc;
  s.ntc = p.ntc;
  s.size = p.size;
  s.grid = p.grid;
  s.scores_ld = (size_t)(pcap + 3) / 4 * 4;
  return s;
}

int span_launch(const char* name, const SpanArgs& a, const SpanPlan& p, const SpanParts& s, cudaStream_t st) {
  if (s.nwt) {
    const int rc = span_tile_launch(a, s, st);
    if (rc) return rc;
  }
  const unsigned nkv = (unsigned)(a.nq / a.group), F = (unsigned)(a.nrow * a.group);
  const long long ctas = (long long)p.tiles * p.npc + (long long)p.items * p.ntc;
  if (ctas == 0) return HV_OK;                              // a run that k_span_tile has all of
  HV_REQUIRE(ctas < (1ll << 31), HV_E_UNSUPPORTED, "%s: too many rows", name);
  const void* fn = p.few == 4   ? (const void*)k_span_few<4>
                   : p.few == 2 ? (const void*)k_span_few<2>
                   : p.few == 1 ? (const void*)k_span_few<1>
                                : (const void*)k_span_part;
  const int smem = p.few ? few_smem(p.few) : kPtSmem;
  const int rc = smem_attr(fn, smem);
  if (rc) return rc;
  // the tails need nothing of k_span_tile's
  const dim3 grid((unsigned)ctas, nkv);
  if (p.few == 4) HV_CUDA(launch_beside(k_span_few<4>, grid, 128, smem, st, s.nwt > 0, a, s, p.tiles));
  else if (p.few == 2) HV_CUDA(launch_beside(k_span_few<2>, grid, 64, smem, st, s.nwt > 0, a, s, p.tiles));
  else if (p.few == 1) HV_CUDA(launch_beside(k_span_few<1>, grid, 32, smem, st, s.nwt > 0, a, s, p.tiles));
  else HV_CUDA(launch_beside(k_span_part, grid, 32 * kPtWarps, smem, st, s.nwt > 0, a, s, p.tiles));
  return HV_OK;
}
int join_launch(const SpanArgs& a, const SpanParts& s, cudaStream_t st) {
  const unsigned nkv = (unsigned)(a.nq / a.group), F = (unsigned)(a.nrow * a.group);
  const unsigned rows = s.terms ? (F + kStRows - 1) / kStRows * kStRows : F;
  const size_t all = (size_t)rows * nkv;
  if (s.nwt + s.npc + s.ntc > 8 && all <= 1024)
    HV_CUDA(launch_beside(k_span_join<4, 2>, dim3((rows + 1) / 2, nkv), 256, 0, st, true, a, s));
  else if (all <= 8192)
    HV_CUDA(launch_beside(k_span_join<1, 8>, dim3((rows + 7) / 8, nkv), 256, 0, st, true, a, s));
  else
    HV_CUDA(launch_beside(k_span_join<1, 32>, dim3((rows + 31) / 32, nkv), 256, 0, st, true, a, s));
  return HV_OK;
}

template <int kPos>
int mass_rows_launch(const SpanArgs& a, const SpanParts& s, const float* mass_in, float* mass_out,
                     int cap, cudaStream_t st) {
  constexpr int smem = kPtQ + 16 * kPos * kHd * 2;
  const int rc = smem_attr((const void*)k_mass_rows<kPos>, smem);
  if (rc) return rc;
  const unsigned n = (unsigned)(a.plen + a.nrow);
  HV_CUDA(launch_beside(k_mass_rows<kPos>, dim3((n + 16 * kPos - 1) / (16 * kPos), (unsigned)(a.nq / a.group)), 256, smem,
                        st, true, a, s, mass_in, mass_out, cap));
  return HV_OK;
}

int mass_any(const char* name, const SpanArgs& a, const float* mass_in, float* mass_out, int cap,
             void* scratch, cudaStream_t st) {
  HV_REQUIRE(a.q && a.pk && a.pv && a.ctx && a.scale && mass_out && scratch && cap > 0, HV_E_INVALID, "%s: bad arguments", name);
  HV_REQUIRE(cap <= kShMaxCap, HV_E_UNSUPPORTED, "%s: a cache of %d positions", name, cap);
  HV_REQUIRE(aligned16(a.q) && aligned16(a.pk) && aligned16(a.pv) && aligned16(a.ctx) && aligned16(scratch),
             HV_E_INVALID, "%s: unaligned pointer", name);
  const int nkv = a.nq / a.group;
  const bool one = a.plen_p != nullptr;                     // a single row at a device position
  SpanPlan p = span_plan(nkv, a.nrow * a.group, 1, cap, 0, true, true);
  const int n = a.plen + a.nrow;
  // k_mass_rows goes through the rows one stage after the other (8 heads: 128 pairs over 768
  // positions 19.7 us, and 18.0 by tiles; 512 over 128 32.7 and 20.4; 40 over 5000 28.5 and 31.8)
  const long long F = (long long)a.nrow * a.group, work = nkv * F * n;
  p.mass_tiles = !one && work >= (1ll << (F >= kStRows ? 26 : 27)) / F;
  SpanParts s = span_parts(p, scratch, cap, true, one);
  int rc = span_launch(name, a, p, s, st);
  if (rc) return rc;
  if (one) {
    const int joins = (a.group + 1) / 2;
    HV_CUDA(launch_beside(k_span_one, dim3((unsigned)(joins + (cap + kOnePos - 1) / kOnePos), (unsigned)nkv), 256, 0, st,
                          true, a, s, mass_in, mass_out, joins));
    return HV_OK;
  }
  rc = join_launch(a, s, st);
  if (rc) return rc;
  if (p.mass_tiles) return mass_tile_launch(a, s, mass_in, mass_out, cap, st);
  // a CTA an SM, as far as the positions go
  auto ctas = [&](int pos) { return (long long)nkv * ((n + 16 * pos - 1) / (16 * pos)); };
  if (ctas(8) >= 148) return mass_rows_launch<8>(a, s, mass_in, mass_out, cap, st);
  if (ctas(4) >= 148) return mass_rows_launch<4>(a, s, mass_in, mass_out, cap, st);
  if (ctas(2) >= 148) return mass_rows_launch<2>(a, s, mass_in, mass_out, cap, st);
  return mass_rows_launch<1>(a, s, mass_in, mass_out, cap, st);
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
  *bytes = span_plan(nq / group, nrow * group, nseq, pcap, tcap, false, false).bytes;
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
  a.nq = nq; a.nseq = nseq; a.nrow = nrow;
  span_group(&a, group);
  const SpanPlan p = span_plan((int)nkv, nrow * group, nseq, pcap, tcap, false, false);
  const SpanParts s = span_parts(p, scratch, pcap, false, false);
  const int rc2 = span_launch(name, a, p, s, (cudaStream_t)stream);
  return rc2 ? rc2 : join_launch(a, s, (cudaStream_t)stream);
}

extern "C" int hv_attn_mass_scratch(int nq, int group, int cap, int ntok, size_t* bytes) {
  const int rc = span_check("hv_attn_mass_scratch", nq, kHd, group, 1, ntok);
  if (rc) return rc;
  HV_REQUIRE(cap > 0 && bytes, HV_E_INVALID, "hv_attn_mass_scratch: bad arguments");
  HV_REQUIRE(cap <= kShMaxCap, HV_E_UNSUPPORTED, "hv_attn_mass_scratch: a cache of %d positions", cap);
  *bytes = span_plan(nq / group, ntok * group, 1, cap, 0, true, true).bytes;
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
  a.nq = nq; a.nseq = a.nrow = 1;
  span_group(&a, group);
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
  a.p_head = (size_t)cap * kHd;
  a.plen = pos0; a.pcap = cap;
  a.run = true;
  a.nq = nq; a.nseq = 1; a.nrow = ntok;
  span_group(&a, group);
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
  a.nq = nq; a.nseq = nseq; a.nrow = nrow;
  span_group(&a, 1);
  const long long warps = (long long)((nq + nkv + 3) / 4) * nrow;
  HV_REQUIRE(warps < (1ll << 31), HV_E_UNSUPPORTED, "%s: %d rows of %d heads", name, nrow, nq);
  k_qk_shared<<<(unsigned)((warps + kQkWarps - 1) / kQkWarps), 32 * kQkWarps, 0, (cudaStream_t)stream>>>(
      qkv, qn, kn, cos_t, sin_t, cap, base, a, q_out, reinterpret_cast<__half*>(tk),
      reinterpret_cast<__half*>(tv), nkv, eps);
  HV_LAUNCHED(name);
}
