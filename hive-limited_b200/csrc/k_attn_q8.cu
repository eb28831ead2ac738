// Attention over the 8-bit KV cache (kv_q8.cuh): one query token (hv_attn_decode_q8) or a run
// of them, each seeing the positions up to its own (hv_attn_rows_q8).
//
//   ctx_h = sum_t w_t v_t / sum_t w_t,   w_t = exp(scale q_h . k_t - max)
//
// in one pass with the running maximum and sum of the softmax. k_t and v_t are the values the
// cache reads back: f32(c s) in complete blocks, the f32 rows of the open one.
#include <algorithm>
#include <mutex>
#include <type_traits>

#include "attn_q8.cuh"
#include "attn_q8_rows.h"
#include "hv_internal.h"
#include "q8_ring.h"

namespace hv {
namespace {

// ---- one query token ------------------------------------------------------------------
//
// Bound by the bytes of the cache for long contexts and by latency for short ones: the
// positions of a kv head are cut into chunks of whole blocks, one CTA each, and a warp takes
// blocks in turn, the 8 KB of codes of kDecStages blocks on their way. For short caches they come
// by 16-byte asynchronous copies, a lane copying exactly the bytes it will multiply, for long ones
// (kLong) by one bulk copy a block, with barriers of each warp's own (1000 positions 6.8 us and 7.1
// in a graph, 131072 positions 54.2 and 49.8). Their waits are bounded: one that runs out leaves NaN
// in every head's context, and what is under way is waited for (q8_ring.h).
// Both products keep the codes as the 16-row operand and the group's queries as the 8
// columns: S^T = K q^T, then ctx^T += V^T w^T. With up to four heads in the group the columns
// are the four hi and the four lo terms (kTwo = false); with five to eight, hi and lo are two
// products. Each warp keeps its own running maximum and sums; they meet in shared memory. The
// chunks of a head meet, added in chunk order, in a cluster's shared memory, or, where a head has
// more than a cluster's eight (kLong), in the caller's scratch by the last CTA to arrive.
// 131072 positions of 8 heads x 4 queries (269 MB) take 51 us among other calls, 5.3 TB/s, 80% of
// a plain copy's rate, and 47 in a graph: 16000 and 131072 positions differ by what their bytes
// take, and 7 us are there whatever the length, the launch, the first blocks' way and the two joins.
// 4225 take 8.6 us in a graph.
constexpr float kLowest = -3e38f;      // finite, so that scores of -infinity are that less it
constexpr int kDecWarps = 8;
constexpr int kDecStages = 2;
// Of a chunk, one a warp. In a graph, 4, 8, 12, 16: 300 positions 6.4, 6.5, 6.5, 6.5 us, 1000 6.3,
// 6.7, 7.5, 7.8, 2000 7.1, 7.1, 7.6, 8.2, the same from 4225 on: 4 would gain 0.4 us around 1000.
constexpr int kDecBlocksMin = 8;
constexpr int kDecStride = 132;        // floats between the columns of a warp's sums
constexpr int kDecTickets = 1024;      // kv heads with chunks to join: first in the scratch
constexpr int kDecPart = 8 * (kHd + 2);    // scratch floats of a chunk: sums, then (max, sum)
constexpr int kDecLine = kHd + 4;      // floats between rows that a warp reads four at a time
constexpr int kDecRing = kDecWarps * kDecStages * 2 * kQ8Codes;
constexpr int kDecSmem = kDecRing + kQ8Blk * (kDecLine + kHd) * 4;     // then the open rows

HV_DEV void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" :: "r"(dst), "l"(src) : "memory");
}

template <bool kTwo, bool kLong>
__global__ void __launch_bounds__(32 * kDecWarps, 1)
    k_attn_dec_q8(const float* __restrict__ q, KvQ8 c, float* __restrict__ ctx,
                  const float* __restrict__ scale, const int32_t* __restrict__ pos_p, int pos0, int group,
                  float* __restrict__ part, unsigned* __restrict__ ticket) {
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_m[kDecWarps][8], s_l[kDecWarps][8], s_x[kQ8Blk][8];
  __shared__ __align__(16) float s_q[8][kDecLine];
  __shared__ unsigned s_last;
  __shared__ unsigned long long s_full[kDecWarps][kDecStages];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
  constexpr bool kMeet = !kLong;
  const int kvh = blockIdx.y, chunk = blockIdx.x;
  const int pos = pos_p ? *pos_p : pos0, held = q8_held(c, kvh);
  float* out = ctx + (size_t)kvh * group * kHd;
  if (pos < 0 || pos >= held) {
    if (chunk == 0)
      for (int i = threadIdx.x; i < group * kHd; i += blockDim.x)
        out[i] = __int_as_float(0x7fc00000);
    if (kMeet) { cluster_sync(); cluster_sync(); }
    return;
  }
  const int closed = held / kQ8Blk;
  const int nb = min(closed, pos / kQ8Blk + 1);           // complete blocks to read
  const int ntail = max(0, pos + 1 - closed * kQ8Blk);
  int nact = (nb + kDecBlocksMin - 1) / kDecBlocksMin;
  nact = max(1, min(nact, (int)gridDim.x));
  if (chunk >= nact) {
    if (kMeet) { cluster_sync(); cluster_sync(); }
    return;
  }
  const int b0 = (int)((long long)nb * chunk / nact), b1 = (int)((long long)nb * (chunk + 1) / nact);

  // this lane's units of a block: 16 bytes at 512 u + 16 lane of K, then of V
  const uint8_t* codes = c.codes + (size_t)kvh * c.nblk * 2 * kQ8Codes;
  const float2* scales = reinterpret_cast<const float2*>(c.scales) + (size_t)kvh * c.nblk;
  const uint8_t* ring = smem + (size_t)warp * kDecStages * 2 * kQ8Codes + 16 * lane;
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring);
  const uint32_t full = (uint32_t)__cvta_generic_to_shared(&s_full[warp][0]);
  if constexpr (kLong) {
    if (lane == 0) {
#pragma unroll
      for (int i = 0; i < kDecStages; ++i) bar_init(full + 8 * i, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();                                // the other lanes wait on them, too
  }
  auto fetch = [&](int b, int stage) {
    const uint8_t* src = codes + (size_t)b * 2 * kQ8Codes;
    if constexpr (kLong) {
      if (b < b1 && lane == 0) {
        asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                     :: "r"(full + 8 * stage), "n"(2 * kQ8Codes) : "memory");
        asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                     :: "r"(ring_s + stage * 2 * kQ8Codes), "l"(src), "n"(2 * kQ8Codes),
                        "r"(full + 8 * stage) : "memory");
      }
    } else {
      if (b < b1) {
#pragma unroll
        for (int u = 0; u < 16; ++u)
          cp_async16(ring_s + stage * 2 * kQ8Codes + 512 * u, src + 16 * lane + 512 * u);
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
  };
  // the open block's rows go first, to the CTA with the last chunk
  const bool open = chunk == nact - 1 && ntail > 0;
  float* open_k = reinterpret_cast<float*>(smem + kDecRing);           // [row][kDecLine]
  float* open_v = open_k + kQ8Blk * kDecLine;                          // [row][kHd]
  if (open) {
    const float* src = c.tail + (size_t)kvh * 2 * kQ8Codes + 4 * lane;
    for (int r = warp; r < ntail; r += kDecWarps) {
      cp_async16((uint32_t)__cvta_generic_to_shared(open_k + r * kDecLine + 4 * lane), src + r * kHd);
      cp_async16((uint32_t)__cvta_generic_to_shared(open_v + r * kHd + 4 * lane), src + kQ8Codes + r * kHd);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
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

  if (open) {                                    // in f32, while the first blocks come in
    asm volatile("cp.async.wait_group %0;" :: "n"(kLong ? 0 : kDecStages) : "memory");
    __syncthreads();
    const int xr = threadIdx.x >> 3, xh = threadIdx.x & 7;     // a thread per row and head
    if (xr < ntail && xh < group) {
      float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
      for (int d = 0; d < kHd; d += 4) {
        const float4 k = *reinterpret_cast<const float4*>(open_k + xr * kDecLine + d);
        const float4 x = *reinterpret_cast<const float4*>(&s_q[xh][d]);
        v[0] = fmaf(k.x, x.x, v[0]);
        v[1] = fmaf(k.y, x.y, v[1]);
        v[2] = fmaf(k.z, x.z, v[2]);
        v[3] = fmaf(k.w, x.w, v[3]);
      }
      s_x[xr][xh] = ((v[0] + v[1]) + (v[2] + v[3])) * qscale;
    }
    __syncthreads();
    float x0[4], x1[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = warp + kDecWarps * i;
      x0[i] = r < ntail && head0 < group ? s_x[r][head0] : -INFINITY;
      x1[i] = r < ntail && head0 + 1 < group ? s_x[r][head0 + 1] : -INFINITY;
      // a row with a value that is not finite loses all of the context, as a complete block does
      const float4 k = *reinterpret_cast<const float4*>(open_k + r * kDecLine + 4 * lane);
      const float4 v = *reinterpret_cast<const float4*>(open_v + r * kHd + 4 * lane);
      const float most = q8_max(q8_max(q8_max(k.x, k.y), q8_max(k.z, k.w)),
                                q8_max(q8_max(v.x, v.y), q8_max(v.z, v.w)));
      if (__any_sync(0xFFFFFFFFu, r < ntail && !(most < INFINITY))) x0[i] = x1[i] = __int_as_float(0x7fc00000);
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
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float va = open_v[r * kHd + 16 * u + gl], vb = open_v[r * kHd + 16 * u + 8 + gl];
          acc[u][0] = fmaf(p0, va, acc[u][0]);
          acc[u][1] = fmaf(p1, va, acc[u][1]);
          acc[u][2] = fmaf(p0, vb, acc[u][2]);
          acc[u][3] = fmaf(p1, vb, acc[u][3]);
        }
      }
    }
  }

  auto wait = [&](int stage, int parity) {
    if constexpr (kLong) {
      int given_up = 0;                          // each wait has its whole limit
      return bar_wait_warp(full + 8 * stage, parity, &given_up);
    } else {
      asm volatile("cp.async.wait_group %0;" :: "n"(kDecStages - 1) : "memory");
      return true;
    }
  };
  auto use = [&](int b, int stage) {
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
    // (a block of scores of -infinity has weights of 0)
    y0 = fmaxf(y0, kLowest);
    y1 = fmaxf(y1, kLowest);
    // Weights as 2^15 times what they are to the block's largest, so that the lo terms of small
    // ones stay above binary16's smallest: a weight is exact to 2^-40 of its block's largest, and
    // a block that is hardly attended to counts in full where its values are large.
    float sum0 = 0.0f, sum1 = 0.0f;
    uint32_t wh[4], wl[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float p0 = ex2(x0[j] - y0) * 32768.0f, p1 = ex2(x1[j] - y1) * 32768.0f;
      sum0 += p0;
      sum1 += p1;
      uint32_t hi, lo;
      split_half2(p0, p1, &hi, &lo);
      if (kTwo) {
        wh[j] = transpose_8x8(hi);
        wl[j] = transpose_8x8(lo);
      } else {
        wh[j] = transpose_8x8(t < 2 ? hi : lo);
      }
    }
    raise(y0, y1);                               // here, so that the weights do not wait for it
    const float g0 = ex2(y0 - m0), g1 = ex2(y1 - m1);
    l0 = fmaf(sum0, g0, l0);
    l1 = fmaf(sum1, g1, l1);
    const float v0 = sc.y * g0, v1 = sc.y * g1;
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
      for (int k = 0; k < 4; ++k) acc[u][k] = fmaf(d[k], k & 1 ? v1 : v0, acc[u][k]);
    }
    if (kLong) __syncwarp();
  };
  if (!ring_walk<kDecStages>(b0 + warp, b1, kDecWarps, wait, fetch, use))
    l0 = l1 = __int_as_float(0x7fc00000);        // in every lane, so in every head

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
  const size_t slot = (size_t)kvh * gridDim.x + chunk;
  float* pacc = part + slot * kDecPart;
  float* pml = pacc + 8 * kHd;
  float* sums = reinterpret_cast<float*>(smem + kDecRing);   // where the open rows were
  float* sums_ml = sums + 8 * kHd;
  const int units = group * (kHd / 4);                   // of four outputs, one a thread
  static_assert(8 * (kHd / 4) <= 32 * kDecWarps, "a thread for each");
  if ((int)threadIdx.x < units) {
    const int i = threadIdx.x, h = i / (kHd / 4), d = 4 * (i % (kHd / 4));
    float M = -INFINITY, L = 0.0f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) M = fmaxf(M, s_m[w][h]);
    auto add = [&](const float* p) {
      const float4 x = *reinterpret_cast<const float4*>(p);
      A.x += x.x; A.y += x.y; A.z += x.z; A.w += x.w;
    };
#pragma unroll
    for (int w = 0; w < kDecWarps; ++w) {
      L += s_l[w][h] == 0.0f ? 0.0f : ex2(s_m[w][h] - M) * s_l[w][h];
      add(red + ((size_t)w * 8 + h) * kDecStride + d);
      if (!kTwo) add(red + ((size_t)w * 8 + 4 + h) * kDecStride + d);
    }
    if (nact == 1) {
      reinterpret_cast<float4*>(out)[i] = make_float4(A.x / L, A.y / L, A.z / L, A.w / L);
    } else if (kMeet) {
      reinterpret_cast<float4*>(sums)[i] = A;
      if (d == 0) { sums_ml[2 * h] = M; sums_ml[2 * h + 1] = L; }
    } else {
      reinterpret_cast<float4*>(pacc)[i] = A;
      if (d == 0) { pml[2 * h] = M; pml[2 * h + 1] = L; }
    }
  }
  if (kMeet) {
    cluster_sync();
    if (nact > 1) {
      const RowsArgs a{q, ctx, scale, pos, 1, 0, group, 0, true, nullptr};
      cluster_add_up(a, sums, kHd, sums_ml, nact, kvh, 0, group, chunk, warp, kDecWarps, held);
    }
    cluster_sync();
    return;
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
  float2* ml = reinterpret_cast<float2*>(smem);          // [chunk][head]: (max, sum), then factors
  for (int i = threadIdx.x; i < nact * 8; i += blockDim.x)
    if ((i & 7) < group)
      ml[i] = __ldcg(reinterpret_cast<const float2*>(base + (size_t)(i >> 3) * kDecPart + 8 * kHd) + (i & 7));
  __syncthreads();
  if (warp < group) {                                    // a warp per head
    float M = -INFINITY, L = 0.0f;
    for (int k = lane; k < nact; k += 32) M = fmaxf(M, ml[8 * k + warp].x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
    for (int k = lane; k < nact; k += 32) {
      const float f = ex2(ml[8 * k + warp].x - M);
      L += f * ml[8 * k + warp].y;
      ml[8 * k + warp].x = f;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, o);
    if (lane == 0) s_l[0][warp] = L;
  }
  __syncthreads();
  if ((int)threadIdx.x < units) {
    const int i = threadIdx.x, h = i / (kHd / 4);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int k = 0; k < nact; ++k) {
      const float4 x = __ldcg(reinterpret_cast<const float4*>(base + (size_t)k * kDecPart) + i);
      const float f = ml[8 * k + h].x;
      s.x += f * x.x; s.y += f * x.y; s.z += f * x.z; s.w += f * x.w;
    }
    const float L = s_l[0][h];
    reinterpret_cast<float4*>(out)[i] = make_float4(s.x / L, s.y / L, s.z / L, s.w / L);
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

// ---- a run of query tokens ------------------------------------------------------------
//
// The rows of a kv head are its (token, head of the group) pairs; a CTA takes 16 kWM of them
// and a chunk of the positions. Its eight warps stand as kWM groups of 16 rows by 8 / kWM
// shares of the chunk's blocks: few rows spread over the positions, many share each block.
// Here the rows are the 16-row operand: S = q K^T and ctx += w V, both terms of q (of w) into
// the same sums. The open block's f32 rows become two binary16 terms as well, so that it is
// a block like the others with a third product, hi x lo. Each of its rows has a power of two of
// its own, so that no row, least of all one that a query does not see, takes bits from another:
// a K row's is taken back from its scores, a V row's goes with its weights.
// Bound by latency: 44 tokens of 16 heads (8 kv heads) over 300 positions take 11.7 us in a
// graph, 38 tokens of 32 heads over 38 positions 10.3.
constexpr int kRowWarps = 8;

template <int kWM>
struct RowsCfg {
  static constexpr int kShares = kRowWarps / kWM;
  static constexpr int kRows = 16 * kWM;
  static constexpr int kStages = kShares == 8 ? 2 : 3;
  static constexpr int kRing = kShares * kStages * 2 * kQ8Codes;
  static constexpr int kLine = kHd + 8;                    // floats: a fragment's stores meet no bank twice
  static constexpr int kMerge = kRowWarps * 16 * kLine * 4;
  static constexpr int kTail = 4 * kQ8Codes * 2;          // K hi, K lo, V hi, V lo
  static constexpr int kOpen = 2 * kQ8Codes * 4;          // the open rows in f32
  static constexpr int kSmem = (kRing > kMerge ? kRing : kMerge) + kTail + kOpen;
};

template <int kWM, bool kMeet>
__global__ void __launch_bounds__(32 * kRowWarps, 1) k_attn_rows_q8(RowsArgs a, KvQ8 c) {
  using Cfg = RowsCfg<kWM>;
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ float s_m[kRowWarps][16], s_l[kRowWarps][16], s_amax[2][kQ8Blk], s_lift[2][kQ8Blk];
  // of the open rows: what a score takes after the largest row's power of two, what V lacks
  __shared__ __align__(8) float s_down[kQ8Blk], s_up[kQ8Blk];
  __shared__ float s_most;              // that power of two
  __shared__ int s_bad;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gl = lane >> 2, t = lane & 3;
  const int wm = warp % kWM, share = warp / kWM;
  const int kvh = blockIdx.y, tile = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const int nrows = a.ntok * a.group, row0 = tile * Cfg::kRows;
  // the queries first, both of a lane's rows: nothing else tells where they are
  const int r0 = row0 + 16 * wm + gl, r1 = r0 + 8;
  float4 x[2][8];
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int r = min(half ? r1 : r0, nrows - 1), tok = r / a.group;
    const float* src = a.q + ((size_t)tok * a.nq + (size_t)kvh * a.group + r - tok * a.group) * kHd;
#pragma unroll
    for (int s = 0; s < 8; ++s) x[half][s] = __ldg(reinterpret_cast<const float4*>(src + 4 * t) + 4 * s);
  }
  const RowsSpan sp = rows_span(a, c, kvh, row0, Cfg::kRows, Cfg::kShares);
  const int held = sp.held, closed = sp.closed, nb = sp.nb, items = sp.items, nact = sp.nact;
  if (chunk >= nact) {
    if (kMeet) { cluster_sync(); cluster_sync(); }
    return;
  }
  const int b0 = (int)((long long)items * chunk / nact);
  const int b1 = (int)((long long)items * (chunk + 1) / nact);
  const int c1 = min(b1, nb);                       // blocks b0 .. c1 from codes, then the tail

  // this warp's two rows per lane
  const int lim0 = r0 < nrows ? min(a.pos0 + r0 / a.group, held - 1) : -1;
  const int lim1 = r1 < nrows ? min(a.pos0 + r1 / a.group, held - 1) : -1;
  const int warp_last = min(row0 + 16 * wm + 15, nrows - 1);
  const int warp_first = row0 + 16 * wm;
  const int warp_top = warp_first < nrows ? a.pos0 + warp_last / a.group : -1;
  const int warp_low = warp_first < nrows ? min(a.pos0 + warp_first / a.group, held - 1) : -1;

  uint8_t* ring = smem + (size_t)share * Cfg::kStages * 2 * kQ8Codes;
  const uint32_t ring_s = (uint32_t)__cvta_generic_to_shared(ring) + 16 * lane;
  const uint8_t* codes = c.codes + (size_t)kvh * c.nblk * 2 * kQ8Codes + 16 * lane;
  const float2* scales = reinterpret_cast<const float2*>(c.scales) + (size_t)kvh * c.nblk;
  auto fetch = [&](int b, int stage) {
    if (b < c1) {
      const uint8_t* src = codes + (size_t)b * 2 * kQ8Codes;
#pragma unroll
      for (int u = wm; u < 16; u += kWM)
        cp_async16(ring_s + stage * 2 * kQ8Codes + 512 * u, src + 512 * u);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto share_sync = [&] {
    if constexpr (kWM == 1) __syncwarp();
    else asm volatile("bar.sync %0, %1;" :: "r"(1 + share), "n"(32 * kWM) : "memory");
  };
  // the open rows go first, to the CTA with the last chunk
  const bool has_open = items > nb && b1 == items;
  const int nopen = min(held - closed * kQ8Blk, kQ8Blk);
  float* open = reinterpret_cast<float*>(smem + Cfg::kSmem - Cfg::kOpen);
  if (has_open) {
    const float* src = c.tail + (size_t)kvh * 2 * kQ8Codes + 4 * lane;
    for (int r = warp; r < 2 * nopen; r += kRowWarps) {
      const int at = r < nopen ? r * kHd : kQ8Codes + (r - nopen) * kHd;
      cp_async16((uint32_t)__cvta_generic_to_shared(open + at + 4 * lane), src + at);
    }
  }
  asm volatile("cp.async.commit_group;" ::: "memory");
#pragma unroll
  for (int i = 0; i < Cfg::kStages; ++i) fetch(b0 + share + i * Cfg::kShares, i);

  uint32_t qh[8][4], ql[8][4];
  float qs0, qs1;
  {
    const float qscale = __ldg(a.scale) * kLog2e;
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      float amax = 0.0f;
#pragma unroll
      for (int s = 0; s < 8; ++s)
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x[half][s].x), fabsf(x[half][s].y))),
                     fmaxf(fabsf(x[half][s].z), fabsf(x[half][s].w)));
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, 2));
      const float lift = q8_lift(amax);
#pragma unroll
      for (int s = 0; s < 8; ++s) {
        split_half2(x[half][s].x * lift, x[half][s].y * lift, &qh[s][half], &ql[s][half]);
        split_half2(x[half][s].z * lift, x[half][s].w * lift, &qh[s][2 + half], &ql[s][2 + half]);
      }
      (half ? qs1 : qs0) = qscale / lift;
    }
  }

  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  float acc[16][4];
#pragma unroll
  for (int d = 0; d < 16; ++d) acc[d][0] = acc[d][1] = acc[d][2] = acc[d][3] = 0.0f;

  // scores of block b in s (position 32 b + 8 j + 2 t + e: s[j][e] of row r0, s[j][2 + e] of
  // r1), already sums of products; f0, f1 make them exponents of 2. Leaves the weights as A
  // fragments of the second product: 2^15 times what they are to the block's largest, which is
  // g0 (g1) of the row's.
  uint32_t wh[2][4], wl[2][4];
  float g0, g1;
  auto raise = [&](float y0, float y1) {         // a larger maximum: what was summed so far counts less
    if (__any_sync(0xFFFFFFFFu, y0 > m0 || y1 > m1)) {
      const float n0 = fmaxf(m0, y0), n1 = fmaxf(m1, y1);
      const float a0 = m0 == -INFINITY ? 0.0f : ex2(m0 - n0);
      const float a1 = m1 == -INFINITY ? 0.0f : ex2(m1 - n1);
      m0 = n0; m1 = n1;
      l0 *= a0; l1 *= a1;
#pragma unroll
      for (int d = 0; d < 16; ++d) { acc[d][0] *= a0; acc[d][1] *= a0; acc[d][2] *= a1; acc[d][3] *= a1; }
    }
  };
  auto weights = [&](int b, float (&s)[4][4], float f0, float f1, auto is_open) {
    const bool cut = 32 * b + 31 > warp_low;
    float y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        s[j][e] *= f0;
        s[j][2 + e] *= f1;
        if (cut) {
          const int p = 32 * b + 8 * j + 2 * t + e;
          if (p > lim0) s[j][e] = -INFINITY;
          if (p > lim1) s[j][2 + e] = -INFINITY;
        }
        y0 = fmaxf(y0, s[j][e]);
        y1 = fmaxf(y1, s[j][2 + e]);
      }
    }
    y0 = fmaxf(y0, __shfl_xor_sync(0xFFFFFFFFu, y0, 1));
    y1 = fmaxf(y1, __shfl_xor_sync(0xFFFFFFFFu, y1, 1));
    y0 = fmaxf(y0, __shfl_xor_sync(0xFFFFFFFFu, y0, 2));
    y1 = fmaxf(y1, __shfl_xor_sync(0xFFFFFFFFu, y1, 2));
    if constexpr (decltype(is_open)::value) {
      raise(y0, y1);
      // The sum of the weights by the scores, the weights by w v. A V row's exponent is a whole
      // number, of which a whole number near the largest w v is taken before a score is added, so
      // that the score keeps its bits.
      const float n0 = m0 == -INFINITY ? 0.0f : m0, n1 = m1 == -INFINITY ? 0.0f : m1;
      y0 = y1 = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          l0 += ex2(s[j][e] - n0) * 32768.0f;
          l1 += ex2(s[j][2 + e] - n1) * 32768.0f;
          const float up = s_up[8 * j + 2 * t + e];
          y0 = fmaxf(y0, s[j][e] + up);
          y1 = fmaxf(y1, s[j][2 + e] + up);
        }
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        y0 = fmaxf(y0, __shfl_xor_sync(0xFFFFFFFFu, y0, o));
        y1 = fmaxf(y1, __shfl_xor_sync(0xFFFFFFFFu, y1, o));
      }
      const float e0 = y0 == -INFINITY ? 0.0f : ceilf(y0), e1 = y1 == -INFINITY ? 0.0f : ceilf(y1);
      const float c0 = ceilf(n0), c1 = ceilf(n1);
      // 2^16 times what they are, which the sums (up to 2^35) lack
      g0 = y0 == -INFINITY ? 0.0f : ex2(e0 - c0 + 16.0f) * ex2(c0 - n0);
      g1 = y1 == -INFINITY ? 0.0f : ex2(e1 - c1 + 16.0f) * ex2(c1 - n1);
      y0 = y1 = 0.0f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float up = s_up[8 * j + 2 * t + e];
          s[j][e] += up - e0;
          s[j][2 + e] += up - e1;
        }
      }
    } else {
      y0 = fmaxf(y0, kLowest);                   // a row that sees nothing of the block has weights of 0
      y1 = fmaxf(y1, kLowest);
    }
    float sum0 = 0.0f, sum1 = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      float p[4];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        p[e] = ex2(s[j][e] - y0) * 32768.0f;
        p[2 + e] = ex2(s[j][2 + e] - y1) * 32768.0f;
        sum0 += p[e];
        sum1 += p[2 + e];
      }
      // A fragment: (row g, k 2t), (row g + 8, k 2t), (row g, k 2t + 8), (row g + 8, k 2t + 8)
      split_half2(p[0], p[1], &wh[j >> 1][2 * (j & 1)], &wl[j >> 1][2 * (j & 1)]);
      split_half2(p[2], p[3], &wh[j >> 1][2 * (j & 1) + 1], &wl[j >> 1][2 * (j & 1) + 1]);
    }
    if constexpr (!decltype(is_open)::value) {
      raise(y0, y1);
      g0 = ex2(y0 - m0);
      g1 = ex2(y1 - m1);
      l0 = fmaf(sum0, g0, l0);
      l1 = fmaf(sum1, g1, l1);
    }
  };

  if (has_open) {                                // while the first blocks come in
    // the open rows as fragments in two terms; rows past the last one held are zero, and so
    // are values that are not finite, whose weight of 0 for the rows that do not see them
    // would not be nothing: the rows that see one get a sum of NaN instead
    __half* frag = reinterpret_cast<__half*>(smem + Cfg::kSmem - Cfg::kOpen - Cfg::kTail);
    if (threadIdx.x < 2 * kQ8Blk) s_amax[threadIdx.x / kQ8Blk][threadIdx.x % kQ8Blk] = 0.0f;
    if (threadIdx.x == 0) s_bad = kQ8Blk;
    asm volatile("cp.async.wait_group %0;" :: "n"(Cfg::kStages) : "memory");
    __syncthreads();
    for (int r = warp; r < 2 * nopen; r += kRowWarps) {        // a row a warp, K's before V's
      const int which = r >= nopen, at = which ? r - nopen : r;
      const float4 x = reinterpret_cast<const float4*>(open + which * kQ8Codes + at * kHd)[lane];
      const float v[4] = {fabsf(x.x), fabsf(x.y), fabsf(x.z), fabsf(x.w)};
      float amax = 0.0f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        if (v[e] < INFINITY) amax = fmaxf(amax, v[e]);
        else atomicMin(&s_bad, at);
      }
      const unsigned top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(amax));
      if (lane == 0) {
        s_amax[which][at] = __uint_as_float(top);
        s_lift[which][at] = q8_lift(__uint_as_float(top));
      }
    }
    __syncthreads();
    if (warp == kRowWarps - 1) {
      // the scores by the largest row's power of two: the others' sums fall, and none overflows
      const float k = s_amax[0][lane], v = s_amax[1][lane];
      const float most = q8_lift(__uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(k))));
      s_down[lane] = k > 0.0f ? most / q8_lift(k) : 0.0f;
      s_up[lane] = v > 0.0f ? (float)(127 - (int)(__float_as_uint(q8_lift(v)) >> 23)) : -INFINITY;
      if (lane == 0) s_most = most;
    }
    auto term = [&](float x, float lift) { return fabsf(x) < INFINITY ? x * lift : 0.0f; };
    // four dims of a K row are neighbours in a fragment, two rows of a V dim
    for (int i = threadIdx.x; i < kQ8Codes / 4; i += blockDim.x) {
      const int r = i / (kHd / 4), d = 4 * (i % (kHd / 4));
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < nopen) x = *reinterpret_cast<const float4*>(open + r * kHd + d);
      const float lk = r < nopen ? s_lift[0][r] : 0.0f;
      uint2 hi, lo;
      split_half2(term(x.x, lk), term(x.y, lk), &hi.x, &lo.x);
      split_half2(term(x.z, lk), term(x.w, lk), &hi.y, &lo.y);
      *reinterpret_cast<uint2*>(frag + q8_k_at(r, d)) = hi;
      *reinterpret_cast<uint2*>(frag + kQ8Codes + q8_k_at(r, d)) = lo;
    }
    for (int i = threadIdx.x; i < kQ8Codes / 2; i += blockDim.x) {
      const int r = 2 * (i / kHd), d = i % kHd;
      const float* v = open + kQ8Codes + r * kHd + d;
      uint32_t hi, lo;
      split_half2(r < nopen ? term(v[0], s_lift[1][r]) : 0.0f,
                  r + 1 < nopen ? term(v[kHd], s_lift[1][r + 1]) : 0.0f, &hi, &lo);
      *reinterpret_cast<uint32_t*>(frag + 2 * kQ8Codes + q8_v_at(r, d)) = hi;
      *reinterpret_cast<uint32_t*>(frag + 3 * kQ8Codes + q8_v_at(r, d)) = lo;
    }
    __syncthreads();
    if (share == 0 && 32 * closed <= warp_top) {
      // 16 halves of a unit: the 16 bytes of a coded one
      auto word2 = [&](int part, int u, int w) {
        return *reinterpret_cast<const uint2*>(frag + part * kQ8Codes + 512 * u + 16 * lane + 4 * w);
      };
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const uint2 kh = word2(0, 2 * j + (k >> 2), k & 3), kl = word2(1, 2 * j + (k >> 2), k & 3);
          mma_f16(s[j], qh[k], kh.x, kh.y);
          mma_f16(s[j], ql[k], kh.x, kh.y);
          mma_f16(s[j], qh[k], kl.x, kl.y);
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float f = s_down[8 * j + 2 * t + e];
          s[j][e] *= f;
          s[j][2 + e] *= f;
        }
      weights(closed, s, qs0 / s_most, qs1 / s_most, std::true_type{});
#pragma unroll
      for (int u = 0; u < 8; ++u) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            const uint2 vh = word2(2, u, 2 * h + k), vl = word2(3, u, 2 * h + k);
            mma_f16(d, wh[k], vh.x, vh.y);
            mma_f16(d, wl[k], vh.x, vh.y);
            mma_f16(d, wh[k], vl.x, vl.y);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[2 * u + h][i] = fmaf(d[i] * 0x1p-16f, i < 2 ? g0 : g1, acc[2 * u + h][i]);
        }
      }
      if (lim0 >= closed * kQ8Blk + s_bad) l0 = __int_as_float(0x7fc00000);
      if (lim1 >= closed * kQ8Blk + s_bad) l1 = __int_as_float(0x7fc00000);
    }
  }

  int stage = 0;
  for (int b = b0 + share; b < c1; b += Cfg::kShares) {
    asm volatile("cp.async.wait_group %0;" :: "n"(Cfg::kStages - 1) : "memory");
    share_sync();
    if (32 * b <= warp_top) {
      const float2 sc = __ldg(scales + b);
      const uint8_t* blk = ring + stage * 2 * kQ8Codes + 16 * lane;
      float s[4][4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j][0] = s[j][1] = s[j][2] = s[j][3] = 0.0f;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const uint4 x = *reinterpret_cast<const uint4*>(blk + 512 * (2 * j + h));
          const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t k0, k1;
            q8_halves(w[k], &k0, &k1);
            mma_f16(s[j], qh[4 * h + k], k0, k1);
            mma_f16(s[j], ql[4 * h + k], k0, k1);
          }
        }
      }
      weights(b, s, sc.x * qs0, sc.x * qs1, std::false_type{});
      // a row that sees nothing of the block takes nothing from it, whatever its scale
      const float f0 = 32 * b <= lim0 ? sc.y * g0 : 0.0f, f1 = 32 * b <= lim1 ? sc.y * g1 : 0.0f;
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint4 x = *reinterpret_cast<const uint4*>(blk + kQ8Codes + 512 * u);
        const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int k = 0; k < 2; ++k) {
            uint32_t v0, v1;
            q8_halves(w[2 * h + k], &v0, &v1);
            mma_f16(d, wh[k], v0, v1);
            mma_f16(d, wl[k], v0, v1);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i)
            acc[2 * u + h][i] = fmaf(d[i], i < 2 ? f0 : f1, acc[2 * u + h][i]);
        }
      }
    }
    share_sync();
    fetch(b + Cfg::kStages * Cfg::kShares, stage);
    stage = stage + 1 == Cfg::kStages ? 0 : stage + 1;
  }

#pragma unroll
  for (int o = 1; o < 4; o <<= 1) {
    l0 += __shfl_xor_sync(0xFFFFFFFFu, l0, o);
    l1 += __shfl_xor_sync(0xFFFFFFFFu, l1, o);
  }

  // the shares meet: all of a row's sums in shared memory, then four outputs a thread
  static_assert(Cfg::kShares > 1, "a row group has two warps at the least");
  if (t == 0) {
    s_m[warp][gl] = m0; s_m[warp][gl + 8] = m1;
    s_l[warp][gl] = l0; s_l[warp][gl + 8] = l1;
  }
  asm volatile("cp.async.wait_group 0;" ::: "memory");
  __syncthreads();
  float* sums = reinterpret_cast<float*>(smem + Cfg::kSmem - Cfg::kOpen - Cfg::kTail);
  float* sums_ml = sums + Cfg::kRows * kHd;
  static_assert(Cfg::kRows * (kHd + 2) * 4 <= Cfg::kOpen + Cfg::kTail, "room for the rows' sums");
  {
    float M0 = -INFINITY, M1 = -INFINITY;
#pragma unroll
    for (int w = 0; w < Cfg::kShares; ++w) {
      M0 = fmaxf(M0, s_m[w * kWM + wm][gl]);
      M1 = fmaxf(M1, s_m[w * kWM + wm][gl + 8]);
    }
    const float a0 = l0 == 0.0f ? 0.0f : ex2(m0 - M0), a1 = l1 == 0.0f ? 0.0f : ex2(m1 - M1);
    float* red = reinterpret_cast<float*>(smem) + (size_t)warp * 16 * Cfg::kLine;
#pragma unroll
    for (int d = 0; d < 16; ++d) {
      *reinterpret_cast<float2*>(red + gl * Cfg::kLine + 8 * d + 2 * t) =
          make_float2(acc[d][0] * a0, acc[d][1] * a0);
      *reinterpret_cast<float2*>(red + (gl + 8) * Cfg::kLine + 8 * d + 2 * t) =
          make_float2(acc[d][2] * a1, acc[d][3] * a1);
    }
  }
  const int ntile = gridDim.x / a.chunks;
  const size_t slot = ((size_t)kvh * ntile + tile) * a.chunks;
  float* mine = a.part + (slot + chunk) * rows_part(Cfg::kRows);
  __syncthreads();
#pragma unroll
  for (int k = 0; k < Cfg::kRows / kRowWarps; ++k) {
    const int r = warp + kRowWarps * k, d4 = lane, i = r * (kHd / 4) + d4, gr = row0 + r;
    if (gr >= nrows) continue;
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int w = 0; w < Cfg::kShares; ++w) M = fmaxf(M, s_m[w * kWM + (r >> 4)][r & 15]);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int w = 0; w < Cfg::kShares; ++w) {
      const int at = w * kWM + (r >> 4);
      const float4 x = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) +
                                                        ((size_t)at * 16 + (r & 15)) * Cfg::kLine + 4 * d4);
      const float lw = s_l[at][r & 15];
      L += lw == 0.0f ? 0.0f : lw * ex2(s_m[at][r & 15] - M);
      s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
    }
    if (nact == 1) {
      const float inv = a.pos0 + gr / a.group >= held ? __int_as_float(0x7fc00000) : 1.0f / L;
      float* o = a.ctx + ((size_t)(gr / a.group) * a.nq + (size_t)kvh * a.group + gr % a.group) * kHd;
      reinterpret_cast<float4*>(o)[d4] = make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
    } else if (kMeet) {
      reinterpret_cast<float4*>(sums)[i] = s;
      if (d4 == 0) *reinterpret_cast<float2*>(sums_ml + 2 * r) = make_float2(M, L);
    } else {
      reinterpret_cast<float4*>(mine)[i] = s;
      if (d4 == 0) *reinterpret_cast<float2*>(mine + (size_t)Cfg::kRows * kHd + 2 * r) = make_float2(M, L);
    }
  }
  if (kMeet) {
    cluster_sync();
    if (nact > 1)
      cluster_add_up(a, sums, kHd, sums_ml, nact, kvh, row0, Cfg::kRows, chunk, warp, kRowWarps, held);
    cluster_sync();
  }
}

// Adds the chunks of every row that are no cluster, in order: a warp per row, a lane per four
// dims. (The last CTA of a row tile, behind a ticket, took 8 us for 16 rows of 18 chunks.)
__global__ void __launch_bounds__(256) k_rows_join_q8(RowsArgs a, KvQ8 c, int rows, int least) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, kvh = blockIdx.y;
  const int row = blockIdx.x * 8 + warp, nrows = a.ntok * a.group;
  if (row >= nrows) return;
  const int tile = row / rows, r = row % rows;
  const RowsSpan sp = rows_span(a, c, kvh, tile * rows, rows, least);
  if (sp.nact == 1) return;                    // the rows are in ctx already
  const int ntile = (nrows + rows - 1) / rows;
  const size_t step = rows_part(rows);
  const float* base = a.part + ((size_t)kvh * ntile + tile) * a.chunks * step;
  const float2* ml = reinterpret_cast<const float2*>(base + (size_t)rows * kHd) + r;
  float M = -INFINITY, L = 0.0f;
  for (int k = lane; k < sp.nact; k += 32) M = fmaxf(M, __ldcg(ml + k * (step / 2)).x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xFFFFFFFFu, M, o));
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int k0 = 0; k0 < sp.nact; k0 += 32) {
    const int k = k0 + lane;
    float w = 0.0f;                            // a row that sees nothing of a chunk has no sum there
    if (k < sp.nact) {
      const float2 x = __ldcg(ml + k * (step / 2));
      w = x.y == 0.0f ? 0.0f : ex2(x.x - M);
      L += w * x.y;
    }
    const int n = min(32, sp.nact - k0);
#pragma unroll 8
    for (int j = 0; j < n; ++j) {
      const float f = __shfl_sync(0xFFFFFFFFu, w, j);
      const float4 x = __ldcg(reinterpret_cast<const float4*>(base + (k0 + j) * step + (size_t)r * kHd) + lane);
      s.x += f * x.x; s.y += f * x.y; s.z += f * x.z; s.w += f * x.w;
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) L += __shfl_xor_sync(0xFFFFFFFFu, L, o);
  const int tok = row / a.group;
  const float inv = a.pos0 + tok >= sp.held ? __int_as_float(0x7fc00000) : 1.0f / L;
  float* o = a.ctx + ((size_t)tok * a.nq + (size_t)kvh * a.group + row - tok * a.group) * kHd;
  reinterpret_cast<float4*>(o)[lane] = make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
}

// Rows per CTA and chunks per row tile of a run. The tile kernel (k_attn_q8_tile.cu) pays for
// filling its tensor memory, its shared memory and a pipeline of five roles, so it takes runs of
// more than 64 rows a head that have 2^21 (row, position) pairs or more. Tiles of 64 rows here
// against it, in microseconds of a graph, on either side of that: 0.5 M pairs (8 heads x 256 rows
// over 264 positions) 13.7 : 21.7, 1.0 M 12.4 : 14.1, 1.8 M 18.6 : 18.4, 2.2 M (with an open block)
// 21.8 : 23.9, 4.2 M 23.6 : 19.8, 6.3 M 32.0 : 19.4, 8.4 M 40.3 : 20.8, 17 M 73.7 : 28.6.
// Up to 64 rows fill at most half of the 128 that a product of the tile kernel has; they take the
// fewest of 16, 32 or 64 that hold them, whose warps then share the positions: 16 rows in tiles of
// 16, 32 and 64 over 104 positions 9.8, 10.2, 11.0, over 500 13.0, 12.4, 12.2, over 2000 13.3, 14.5,
// 18.0, over 16000 20.2, 26.4, 40.4; 32 rows in 32 and 64 over 108 11.4, 12.1, over 500 13.2, 12.9,
// over 2000 15.7, 18.5, over 16000 27.0, 40.5. What that loses around 500 positions (up to 0.8) it
// gains many times over elsewhere.
struct RowsPlan {
  int rows, tiles, chunks;
  bool cluster;
};
constexpr long long kTilePairs = 1ll << 21;
// Blocks that a CTA works on at once, and of a chunk at the least: one for each share.
int rows_step(int rows) { return rows == 128 ? kTileLeast / 2 : 16 * kRowWarps / rows; }
int rows_least(int rows) { return rows == 128 ? kTileLeast : rows_step(rows); }
// As many chunks as leave no SM without a CTA.
int rows_chunks(int nkv, int npos, int rows, int tiles, int sms) {
  const int most = (npos + kQ8Blk - 1) / kQ8Blk / rows_least(rows);
  return (int)std::max(1ll, std::min((long long)most, sms / ((long long)tiles * nkv)));
}
// Clusters of n CTAs that the GPU holds at once, a CTA having an SM to itself.
int cluster_room(int n, int* room) {
  static std::mutex mu;
  static int known[64][kRowsCluster + 1];
  int dev = 0;
  HV_CUDA(cudaGetDevice(&dev));
  std::lock_guard<std::mutex> lk(mu);
  int (&of)[kRowsCluster + 1] = known[dev & 63];
  for (int k = 2; k <= kRowsCluster && !of[kRowsCluster]; ++k) {
    const int rc = attn_tile_q8_room(k, &of[k]);
    if (rc) return rc;
  }
  *room = of[n];
  return HV_OK;
}
int rows_plan(int nkv, int group, int pos0, int ntok, RowsPlan* p) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  const long long n = (long long)ntok * group;
  const int npos = pos0 + ntok, blocks = (npos + kQ8Blk - 1) / kQ8Blk;
  const bool tile = n * nkv * npos >= kTilePairs;
  p->rows = n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 || !tile ? 64 : 128;
  p->tiles = (int)((n + p->rows - 1) / p->rows);
  p->chunks = rows_chunks(nkv, npos, p->rows, p->tiles, sms);
  p->cluster = false;
  // Chunks that are a cluster need no second launch, which costs as much as one step here or two
  // of the tile kernel's; they are eight at most, and as many as let all clusters run at once. In
  // microseconds of a graph, as a cluster and not: 44 x 2 rows, 300 positions (2 steps, 2)
  // 11.6 : 13.7; 4 x 4 rows, 4000 positions (2, 1) 11.4 : 14.3; 32 x 4 rows, 1032 positions (3, 2)
  // 17.0 : 16.5, half a microsecond lost; 8 x 4 rows, 4000 positions (4, 2) 16.1 : 15.8; tile
  // kernel, 32 x 4 rows, 4000 positions (4, 2) 20.8 : 22.0 and 256 x 4, 4096 positions (16, 16)
  // 43.4 : 47.1; 16 clusters of 8, where 15 run at once, 26.1 : 16.9.
  const int step = rows_step(p->rows);
  auto steps = [&](int chunks) { return ((blocks + chunks - 1) / chunks + step - 1) / step; };
  for (int c = std::min(p->chunks, kRowsCluster); c > 1; --c) {
    int room = 0;
    const int rc2 = cluster_room(c, &room);
    if (rc2) return rc2;
    if ((long long)p->tiles * nkv > room) continue;
    p->cluster = steps(c) <= steps(p->chunks) + (p->rows == 128 ? 2 : 1);
    if (p->cluster) p->chunks = c;
    break;
  }
  return HV_OK;
}
// Floats of scratch that any run of up to ntok rows needs: a shorter run can have more chunks.
int rows_floats(int nkv, int group, int cap, int ntok, size_t* floats) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  const long long n = (long long)ntok * group;
  *floats = 0;
  for (int rows = 16; rows <= 128; rows *= 2) {
    const long long tiles = rows < 64 ? 1 : (n + rows - 1) / rows;
    for (int t = 1; t <= tiles && 2ll * t * nkv <= sms; ++t) {
      const int chunks = rows_chunks(nkv, cap, rows, t, sms);
      if (chunks > 1) *floats = std::max(*floats, (size_t)nkv * t * chunks * rows_part(rows));
    }
  }
  return HV_OK;
}

template <int kWM, bool kMeet>
int rows_go(const RowsArgs& a, const KvQ8& c, dim3 grid, cudaStream_t st) {
  const int rc = smem_attr((const void*)k_attn_rows_q8<kWM, kMeet>, RowsCfg<kWM>::kSmem);
  return rc ? rc : rows_launch(k_attn_rows_q8<kWM, kMeet>, grid, 32 * kRowWarps, RowsCfg<kWM>::kSmem, a, c, st);
}
template <int kWM>
int rows_go(const RowsArgs& a, const KvQ8& c, dim3 grid, cudaStream_t st) {
  return a.cluster ? rows_go<kWM, true>(a, c, grid, st) : rows_go<kWM, false>(a, c, grid, st);
}

// One query token at *pos (at pos0 without one).
int dec_launch(const float* q, const KvQ8& c, float* ctx, const float* scale, const int32_t* pos,
               int pos0, int nkv, int group, int cap, void* scratch, void* stream) {
  int nch = 0;
  int rc = dec_chunks(nkv, cap, &nch);
  if (rc) return rc;
  const bool two = group > 4;
  // As a cluster the chunks are joined through shared memory, for which the two trips to the
  // scratch and the ticket take 2 us. It has eight at most, and as many as let all heads run at
  // once, so that a full cache takes more steps of a block a warp. In microseconds of a graph, as a
  // cluster and not, 8 heads x 4 queries: 300 positions (steps 1, 1) 6.5 : 8.5, 2000 (1, 1)
  // 7.1 : 9.1, 4225 (3, 1) 8.6 : 9.6, 8000 (4, 2) 8.9 : 10.0, 12000 (6, 3) 11.2 : 11.1, 16000 (8, 4)
  // 13.1 : 11.8. Only the cache's size is known here: a cache that is too long for clusters when it
  // is full takes the second figures from its first position on.
  const int blocks = (cap + kQ8Blk - 1) / kQ8Blk;
  auto steps = [&](int chunks) { return ((blocks + chunks - 1) / chunks + kDecWarps - 1) / kDecWarps; };
  bool meet = false;
  for (int k = std::min(nch, kRowsCluster); k > 1 && !meet; --k) {
    int room = 0;
    rc = cluster_room(k, &room);
    if (rc) return rc;
    if (nkv > room) continue;
    meet = steps(k) <= steps(nch) + 3;
    if (!meet) break;
    nch = k;
  }
  const bool few = meet || nch == 1;
  unsigned* ticket = static_cast<unsigned*>(scratch);
  float* part = reinterpret_cast<float*>(ticket + kDecTickets);
  auto* fn = two ? (few ? k_attn_dec_q8<true, false> : k_attn_dec_q8<true, true>)
                 : (few ? k_attn_dec_q8<false, false> : k_attn_dec_q8<false, true>);
  rc = smem_attr((const void*)fn, kDecSmem);
  if (rc) return rc;
  cudaLaunchAttribute at{};
  const cudaLaunchConfig_t cfg = rows_config(dim3(nch, nkv), 32 * kDecWarps, kDecSmem,
                                             meet ? nch : 1, &at, (cudaStream_t)stream);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, q, c, ctx, scale, pos, pos0, group, part, ticket);
  return e == cudaSuccess ? HV_OK : cuda_fail("k_attn_dec_q8", e);
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
  HV_REQUIRE(nq <= 32768 && cap <= (1 << 30) && ntok <= 65535, HV_E_UNSUPPORTED,
             "hv_attn_q8_scratch: %d heads, %d positions, %d rows", nq, cap, ntok);
  int nch = 0;
  const int rc = dec_chunks(nq / group, cap, &nch);
  if (rc) return rc;
  size_t rows = 0;
  const int rc2 = ntok > 1 ? rows_floats(nq / group, group, cap, ntok, &rows) : HV_OK;
  if (rc2) return rc2;
  const size_t dec = (size_t)(nq / group) * nch * kDecPart;
  *bytes = kDecTickets * sizeof(unsigned) + std::max(dec, rows) * sizeof(float);
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
  return dec_launch(q, c, ctx, scale, pos, 0, nq / group, group, cap, scratch, stream);
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
  if (ntok == 1)
    return dec_launch(q, c, ctx, scale, nullptr, pos0, nq / group, group, cap, scratch, stream);
  RowsPlan p;
  const int rc2 = rows_plan(nq / group, group, pos0, ntok, &p);
  if (rc2) return rc2;
  RowsArgs a{q, ctx, scale, pos0, ntok, nq, group, p.chunks,
p.cluster,
             reinterpret_cast<float*>(static_cast<uint8_t*>(scratch) +
                                      kDecTickets * sizeof(unsigned))};
  const dim3 grid((unsigned)(p.tiles * p.chunks), (unsigned)(nq / group));
  const cudaStream_t st = (cudaStream_t)stream;
  const int rc3 = p.rows == 16 ? rows_go<1>(a, c, grid, st) : p.rows == 32 ? rows_go<2>(a, c, grid, st)
                : p.rows == 64 ? rows_go<4>(a, c, grid, st)
                : attn_tile_q8_launch(a, c, (unsigned)p.tiles, (unsigned)(nq / group), st);
  if (rc3) return rc3;
  if (p.chunks == 1 || a.cluster) return HV_OK;
  k_rows_join_q8<<<dim3((unsigned)((ntok * group + 7) / 8), (unsigned)(nq / group)), 256, 0,
                   st>>>(a, c, p.rows, rows_least(p.rows));
  HV_LAUNCHED("k_rows_join_q8");
}
