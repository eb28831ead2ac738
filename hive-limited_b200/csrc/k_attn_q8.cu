// Attention over the 8-bit KV cache (kv_q8.cuh): one query token (hv_attn_decode_q8) or a run
// of them, each seeing the positions up to its own (hv_attn_rows_q8).
//
//   ctx_h = sum_t w_t v_t / sum_t w_t,   w_t = exp(scale q_h . k_t - max)
//
// in one pass with the running maximum and sum of the softmax. k_t and v_t are the values the
// cache reads back: f32(c s) in complete blocks, the f32 rows of the open one.
#include <algorithm>

#include "attn_q8.cuh"
#include "hv_internal.h"

namespace hv {
namespace {

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

// ---- one query token ------------------------------------------------------------------
//
// Bound by the bytes of the cache for long contexts and by latency for short ones: the
// positions of a kv head are cut into chunks of whole blocks, one CTA each, and a warp takes
// blocks in turn. A block's 8 KB of codes comes by asynchronous copies, kDecStages of them
// ahead; a lane copies exactly the bytes it will multiply, so nothing has to be synchronised.
// Both products keep the codes as the 16-row operand and the group's queries as the 8
// columns: S^T = K q^T, then ctx^T += V^T w^T. With up to four heads in the group the columns
// are the four hi and the four lo terms (kTwo = false); with five to eight, hi and lo are two
// products. Each warp keeps its own running maximum and sums; they meet in shared memory and,
// between a head's chunks, in the caller's scratch, where the last CTA to arrive adds them
// in chunk order.
constexpr int kDecWarps = 8;
constexpr int kDecStages = 3;
constexpr int kDecBlocksMin = 8;       // blocks a chunk holds before a head gets another CTA
constexpr int kDecStride = 132;        // floats between the columns of a warp's sums
constexpr int kDecTickets = 1024;      // kv heads with chunks to join: first in the scratch
constexpr int kDecPart = 8 * (kHd + 2);    // scratch floats of a chunk: sums, then (max, sum)
constexpr int kDecSmem = kDecWarps * kDecStages * 2 * kQ8Codes;

HV_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}

template <bool kTwo>
__global__ void __launch_bounds__(32 * kDecWarps, 1)
    k_attn_dec_q8(const float* __restrict__ q, KvQ8 c, float* __restrict__ ctx,
                  const float* __restrict__ scale, const int32_t* __restrict__ pos_p, int group,
                  float* __restrict__ part, unsigned* __restrict__ ticket) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_m[kDecWarps][8], s_l[kDecWarps][8], s_q[8][kHd];
  __shared__ unsigned s_last;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
  const int kvh = blockIdx.y, chunk = blockIdx.x;
  const int pos = *pos_p, held = q8_held(c, kvh);
  float* out = ctx + (size_t)kvh * group * kHd;
  if (pos < 0 || pos >= held) {
    if (chunk == 0)
      for (int i = threadIdx.x; i < group * kHd; i += blockDim.x)
        out[i] = __int_as_float(0x7fc00000);
    return;
  }
  const int closed = held / kQ8Blk;
  const int nb = min(closed, pos / kQ8Blk + 1);           // complete blocks to read
  const int ntail = max(0, pos + 1 - closed * kQ8Blk);
  int nact = (nb + kDecBlocksMin - 1) / kDecBlocksMin;
  nact = max(1, min(nact, (int)gridDim.x));
  if (chunk >= nact) return;
  const int b0 = (int)((long long)nb * chunk / nact), b1 = (int)((long long)nb * (chunk + 1) / nact);

  // this lane's units of a block: 16 bytes at 512 u + 16 lane of K, then of V
  const uint8_t* codes = c.codes + (size_t)kvh * c.nblk * 2 * kQ8Codes + 16 * lane;
  const float2* scales = reinterpret_cast<const float2*>(c.scales) + (size_t)kvh * c.nblk;
  const uint8_t* ring = smem + (size_t)warp * kDecStages * 2 * kQ8Codes + 16 * lane;
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
  auto fetch = [&](int b, int stage) {
    if (b < b1) {
      const uint8_t* src = codes + (size_t)b * 2 * kQ8Codes;
#pragma unroll
      for (int u = 0; u < 16; ++u) cp_async16(ring_s + stage * 2 * kQ8Codes + 512 * u, src + 512 * u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < kDecStages; ++i) fetch(b0 + warp + i * kDecWarps, i);
  float2 sc_next = make_float2(0.f, 0.f);
  if (b0 + warp < b1) sc_next = __ldg(scales + b0 + warp);

  // the queries as B fragments: column gl; k-step s holds dims 16 s + 4 t ..
  const float qscale = __ldg(scale) * kLog2e;
  const int col_head = kTwo ? gl : (gl & 3);
  const float* qrow = q + ((size_t)kvh * group + col_head) * kHd;
  uint32_t qb[kTwo ? 2 : 1][16];
  float lift;
  {
    float4 x[8];
    float amax = 0.0f;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      x[s] = col_head < group ? __ldg(reinterpret_cast<const float4*>(qrow + 16 * s + 4 * t))
                              : make_float4(0.f, 0.f, 0.f, 0.f);
      amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x[s].x), fabsf(x[s].y))),
                   fmaxf(fabsf(x[s].z), fabsf(x[s].w)));
      if (warp == 0 && (kTwo || gl < 4) && col_head < group)
        *reinterpret_cast<float4*>(&s_q[col_head][16 * s + 4 * t]) = x[s];
    }
    amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
    lift = q8_lift(amax);
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      uint32_t h0, h1, l0, l1;
      split_half2(x[s].x * lift, x[s].y * lift, &h0, &l0);
      split_half2(x[s].z * lift, x[s].w * lift, &h1, &l1);
      if (kTwo) {
        qb[0][2 * s] = h0; qb[0][2 * s + 1] = h1;
        qb[kTwo ? 1 : 0][2 * s] = l0; qb[kTwo ? 1 : 0][2 * s + 1] = l1;
      } else {
        qb[0][2 * s] = gl < 4 ? h0 : l0;
        qb[0][2 * s + 1] = gl < 4 ? h1 : l1;
      }
    }
  }
  // this lane's two heads among the columns, and what turns their sums into exponents of 2
  const int head0 = kTwo ? 2 * t : 2 * (t & 1);
  const float qs0 = qscale / __shfl_sync(0xFFFFFFFFu, lift, 4 * head0);
  const float qs1 = qscale / __shfl_sync(0xFFFFFFFFu, lift, 4 * head0 + 4);

  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  float acc[8][4];
#pragma unroll
  for (int u = 0; u < 8; ++u) acc[u][0] = acc[u][1] = acc[u][2] = acc[u][3] = 0.0f;
  // a larger maximum: what was summed so far counts less
  auto raise = [&](float x0, float x1) {
    const float n0 = fmaxf(m0, x0), n1 = fmaxf(m1, x1);
    if (__any_sync(0xFFFFFFFFu, n0 > m0 || n1 > m1)) {
      const float a0 = m0 == -INFINITY ? 0.0f : ex2(m0 - n0);
      const float a1 = m1 == -INFINITY ? 0.0f : ex2(m1 - n1);
      m0 = n0; m1 = n1;
      l0 *= a0; l1 *= a1;
#pragma unroll
      for (int u = 0; u < 8; ++u) { acc[u][0] *= a0; acc[u][1] *= a1; acc[u][2] *= a0; acc[u][3] *= a1; }
    }
  };

  int stage = 0;
  for (int b = b0 + warp; b < b1; b += kDecWarps) {
    asm volatile("cp.async.wait_group %0;" :: "n"(kDecStages - 1) : "memory");
    const float2 sc = sc_next;
    if (b + kDecWarps < b1) sc_next = __ldg(scales + b + kDecWarps);
    const uint8_t* blk = ring + stage * 2 * kQ8Codes;
    float s[2][4];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.0f;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint4 x = *reinterpret_cast<const uint4*>(blk + 512 * (4 * i + h));
        const uint4 y = *reinterpret_cast<const uint4*>(blk + 512 * (4 * i + 2 + h));
        const uint32_t xw[4] = {x.x, x.y, x.z, x.w}, yw[4] = {y.x, y.y, y.z, y.w};
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          uint32_t a[4];
          q8_halves(xw[k], &a[0], &a[2]);
          q8_halves(yw[k], &a[1], &a[3]);
          const int ks = 4 * h + k;
          mma_f16(s[i], a, qb[0][2 * ks], qb[0][2 * ks + 1]);
          if (kTwo) mma_f16(s[i], a, qb[kTwo ? 1 : 0][2 * ks], qb[kTwo ? 1 : 0][2 * ks + 1]);
        }
      }
    }
    // x[j]: scores of position 32 b + 8 j + gl for this lane's two heads
    const float f0 = sc.x * qs0, f1 = sc.x * qs1;
    float x0[4], x1[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float v0 = s[j >> 1][2 * (j & 1)], v1 = s[j >> 1][2 * (j & 1) + 1];
      if (!kTwo) {
        v0 += __shfl_xor_sync(0xFFFFFFFFu, v0, 2);
        v1 += __shfl_xor_sync(0xFFFFFFFFu, v1, 2);
      }
      x0[j] = v0 * f0;
      x1[j] = v1 * f1;
    }
    if ((b + 1) * kQ8Blk > pos + 1) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (b * kQ8Blk + 8 * j + gl > pos) x0[j] = x1[j] = -INFINITY;
    }
    float y0 = fmaxf(fmaxf(x0[0], x0[1]), fmaxf(x0[2], x0[3]));
    float y1 = fmaxf(fmaxf(x1[0], x1[1]), fmaxf(x1[2], x1[3]));
#pragma unroll
    for (int o = 4; o < 32; o <<= 1) {
      y0 = fmaxf(y0, __shfl_xor_sync(0xFFFFFFFFu, y0, o));
      y1 = fmaxf(y1, __shfl_xor_sync(0xFFFFFFFFu, y1, o));
    }
    raise(y0, y1);
    // weights as 2^15 times what they are to the maximum's, so that the lo terms of small
    // ones stay above binary16's smallest: a weight is exact to 2^-40 of the largest
    uint32_t wh[4], wl[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float p0 = ex2(x0[j] - m0) * 32768.0f, p1 = ex2(x1[j] - m1) * 32768.0f;
      l0 += p0;
      l1 += p1;
      uint32_t hi, lo;
      split_half2(p0, p1, &hi, &lo);
      if (kTwo) {
        wh[j] = transpose_8x8(hi);
        wl[j] = transpose_8x8(lo);
      } else {
        wh[j] = transpose_8x8(t < 2 ? hi : lo);
      }
    }
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const uint4 v = *reinterpret_cast<const uint4*>(blk + kQ8Codes + 512 * u);
      uint32_t a[4], e[4];
      q8_halves(v.x, &a[0], &a[2]);
      q8_halves(v.z, &a[1], &a[3]);
      q8_halves(v.y, &e[0], &e[2]);
      q8_halves(v.w, &e[1], &e[3]);
      float d[4] = {0.f, 0.f, 0.f, 0.f};
      mma_f16(d, a, wh[0], wh[1]);
      mma_f16(d, e, wh[2], wh[3]);
      if (kTwo) {
        mma_f16(d, a, wl[0], wl[1]);
        mma_f16(d, e, wl[2], wl[3]);
      }
#pragma unroll
      for (int k = 0; k < 4; ++k) acc[u][k] = fmaf(d[k], sc.y, acc[u][k]);
    }
    fetch(b + kDecStages * kDecWarps, stage);
    stage = stage + 1 == kDecStages ? 0 : stage + 1;
  }

  if (chunk == nact - 1 && ntail > 0) {          // the open block's rows, in f32
    __syncthreads();                             // s_q
    const float* tail = c.tail + (size_t)kvh * 2 * kQ8Codes;
    float x0[4], x1[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = warp + kDecWarps * i;
      x0[i] = x1[i] = -INFINITY;
      if (r < ntail) {
        const float4 k = __ldg(reinterpret_cast<const float4*>(tail + r * kHd) + lane);
        for (int h = 0; h < group; ++h) {
          const float4 w = *reinterpret_cast<const float4*>(&s_q[h][4 * lane]);
          float v = k.x * w.x + k.y * w.y + k.z * w.z + k.w * w.w;
#pragma unroll
          for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
          v *= qscale;
          if (h == head0) x0[i] = v;
          if (h == head0 + 1) x1[i] = v;
        }
      }
    }
    raise(fmaxf(fmaxf(x0[0], x0[1]), fmaxf(x0[2], x0[3])),
          fmaxf(fmaxf(x1[0], x1[1]), fmaxf(x1[2], x1[3])));
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = warp + kDecWarps * i;
      if (r >= ntail) continue;
      const float p0 = head0 < group ? ex2(x0[i] - m0) * 32768.0f : 0.0f;
      const float p1 = head0 + 1 < group ? ex2(x1[i] - m1) * 32768.0f : 0.0f;
      if (gl == 0) { l0 += p0; l1 += p1; }
      if (kTwo || t < 2) {
        const float* v = tail + kQ8Codes + r * kHd;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float va = __ldg(v + 16 * u + gl), vb = __ldg(v + 16 * u + 8 + gl);
          acc[u][0] = fmaf(p0, va, acc[u][0]);
          acc[u][1] = fmaf(p1, va, acc[u][1]);
          acc[u][2] = fmaf(p0, vb, acc[u][2]);
          acc[u][3] = fmaf(p1, vb, acc[u][3]);
        }
      }
    }
  }
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) {
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, o);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, o);
  }

  // the CTA's warps meet
  if (gl == 0 && (kTwo || t < 2)) {
    s_m[warp][head0] = m0; s_m[warp][head0 + 1] = m1;
    s_l[warp][head0] = l0; s_l[warp][head0 + 1] = l1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* red = reinterpret_cast<float*>(smem);           // [warp][column][kDecStride]
  float M0 = -INFINITY, M1 = -INFINITY;
#pragma unroll
  for (int w = 0; w < kDecWarps; ++w) {
    M0 = fmaxf(M0, s_m[w][head0]);
    M1 = fmaxf(M1, s_m[w][head0 + 1]);
  }
  {
    const float a0 = m0 == -INFINITY && l0 == 0.0f ? 0.0f : ex2(m0 - M0);
    const float a1 = m1 == -INFINITY && l1 == 0.0f ? 0.0f : ex2(m1 - M1);
    float* r = red + ((size_t)warp * 8 + 2 * t) * kDecStride + gl;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      r[16 * u] = acc[u][0] * a0;
      r[kDecStride + 16 * u] = acc[u][1] * a1;
      r[16 * u + 8] = acc[u][2] * a0;
      r[kDecStride + 16 * u + 8] = acc[u][3] * a1;
    }
  }
  __syncthreads();
  const int vals = group * kHd;
  const size_t slot = (size_t)kvh * gridDim.x + chunk;
  float* pacc = part + slot * kDecPart;
  float* pml = pacc + 8 * kHd;
  for (int i = threadIdx.x; i < vals; i += blockDim.x) {
    const int h = i / kHd, d = i % kHd;
    float M = -INFINITY, L = 0.0f, A = 0.0f;
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, s_m[w][h]);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      const float a = s_l[w][h] == 0.0f ? 0.0f : ex2(s_m[w][h] - M);
      L += a * s_l[w][h];
      A += red[((size_t)w * 8 + h) * kDecStride + d];
      if (!kTwo) A += red[((size_t)w * 8 + 4 + h) * kDecStride + d];
    }
    if (nact == 1) {
      out[i] = A / L;
    } else {
      pacc[i] = A;
      if (d == 0) { pml[2 * h] = M; pml[2 * h + 1] = L; }
    }
  }
  if (nact == 1) return;

  // the head's chunks meet: the last CTA adds them in order
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) {
    s_last = atomicAdd(ticket + kvh, 1u) == (unsigned)nact - 1;
    if (s_last) ticket[kvh] = 0;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();
  const float* base = part + (size_t)kvh * gridDim.x * kDecPart;
  for (int i = threadIdx.x; i < vals; i += blockDim.x) {
    const int h = i / kHd;
    float M = -INFINITY, L = 0.0f, A = 0.0f;
    for (int k = 0; k < nact; ++k) M = fmaxf(M, __ldcg(base + (size_t)k * kDecPart + 8 * kHd + 2 * h));
#pragma unroll 8
    for (int k = 0; k < nact; ++k) {
      const float* p = base + (size_t)k * kDecPart;
      const float a = ex2(__ldcg(p + 8 * kHd + 2 * h) - M);
      L += a * __ldcg(p + 8 * kHd + 2 * h + 1);
      A += a * __ldcg(p + i);
    }
    out[i] = A / L;
  }
}

// CTAs per kv head: every SM has one, unless the cache cannot fill them.
int dec_chunks(int nkv, int cap, int* out) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  const int most = (cap / kQ8Blk + kDecBlocksMin - 1) / kDecBlocksMin;
  *out = nkv > kDecTickets ? 1 : std::max(1, std::min(sms / nkv, most));
  return HV_OK;
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
  int nch = 0;
  const int rc = dec_chunks(nq / group, cap, &nch);
  if (rc) return rc;
  *bytes = kDecTickets * sizeof(unsigned) + (size_t)(nq / group) * nch * kDecPart * sizeof(float);
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
  const int nkv = nq / group;
  int nch = 0;
  const int rc2 = dec_chunks(nkv, cap, &nch);
  if (rc2) return rc2;
  unsigned* ticket = static_cast<unsigned*>(scratch);
  float* part = reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) + kDecTickets * sizeof(unsigned));
  const void* fn = group > 4 ? (const void*)k_attn_dec_q8<true> : (const void*)k_attn_dec_q8<false>;
  const int rc3 = smem_attr(fn, kDecSmem);
  if (rc3) return rc3;
  if (group > 4)
    k_attn_dec_q8<true><<<dim3(nch, nkv), 32 * kDecWarps, kDecSmem, (cudaStream_t)stream>>>(
        q, c, ctx, scale, pos, group, part, ticket);
  else
    k_attn_dec_q8<false><<<dim3(nch, nkv), 32 * kDecWarps, kDecSmem, (cudaStream_t)stream>>>(
        q, c, ctx, scale, pos, group, part, ticket);
  HV_LAUNCHED("k_attn_dec_q8");
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
