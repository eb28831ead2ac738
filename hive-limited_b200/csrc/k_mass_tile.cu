// The weights that the rows of a long run give to the positions of a binary16 cache, on the
// fifth-generation tensor cores: mass[t] += sum over rows of 2^(x - m - log2 l), once k_span_join
// knows every row's m and l. The scores are formed again, this time with the positions as the operand
// in tensor memory and the rows in shared memory, so that a thread has one position and adds up
// along its columns, and nothing is added across threads.
//
// A CTA takes tiles of 128 positions two at a time (K rows in tensor memory, 64 columns each) and
// goes through the rows that see them, 128 to a tile, whose two binary16 terms k_span_join has left
// in the scratch:
//   warps 0-15       by fours: one adds up the first 64 rows' scores of the first tile of positions,
//                    one of the second tile, the others the last 64 rows'
//   warp 16          issues D = K ql^T + K qh^T, D one of three
//   warp 17          one thread: the copies of the rows' terms, three tiles of rows under way, and
//                    of what their exponents take
// Tiles of positions are cut evenly among the CTAs, one an SM; an odd one goes alone, its tiles of
// rows to the first and the second tile's warps in turn.
//
// 256 rows of 64 heads over 16384 positions: 127 us for 137 GFLOP with two terms, 84 us of them at
// the rate of a library's product; tensor pipe and exponentials are both active 54% of the time, and
// every score's factor and offset come from shared memory. Eight warps in place of sixteen: 152 us.
//
// Every wait is bounded, from the end of the kernel before on, beside which this one starts: one
// that runs out leaves NaN in the positions' mass.
#include <type_traits>

#include "attn_f16.cuh"
#include "hv_internal.h"
#include "tcgen05.cuh"

namespace hv {
namespace {

constexpr int kMtSumThreads = 512, kMtThreads = kMtSumThreads + 64;
constexpr int kMtHalf = kStRows * 128;          // bytes of 128 rows of 64 halves
constexpr int kMtTerm = 2 * kMtHalf;
constexpr int kMtStages = 3, kMtSums = 3;
constexpr int kMtStage = 2 * kMtTerm + 2 * kStRows * 4;   // both terms, then what takes them to exponents
constexpr int kMtStageStep = (kMtStage + 1023) / 1024 * 1024;
constexpr uint32_t kMtColK = 128 * kMtSums;     // tensor memory: D, then K of two tiles
constexpr uint32_t kMtDesc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);

struct MtShared {
  unsigned long long q_full[kMtStages], q_free[kMtStages], d_full[2][2], d_free[kMtSums], drain;
  float sum[4][kStRows];
  uint32_t tmem;
  int given_up;
};
constexpr int kMtSmem = kMtStages * kMtStageStep + (int)sizeof(MtShared);

__global__ void __launch_bounds__(kMtThreads, 1)
    k_mass_tile(SpanArgs a, SpanParts p, const float* mass_in, float* mass_out, int cap,
                const __grid_constant__ CUtensorMap map_q) {
  extern __shared__ __align__(1024) uint8_t smem[];
  MtShared& sh = *reinterpret_cast<MtShared*>(smem + kMtStages * kMtStageStep);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int F = a.nrow * a.group, nkv = a.nq / a.group, n = a.plen + a.nrow;
  const int tiles = (n + kStRows - 1) / kStRows, rtiles = (F + kStRows - 1) / kStRows;
  const long long units = (long long)nkv * tiles;
  const long long u0 = units * blockIdx.x / gridDim.x, u1 = units * (blockIdx.x + 1) / gridDim.x;
  if (u0 >= u1) return;
  const uint32_t sm = (uint32_t)__cvta_generic_to_shared(smem);
  auto bar = [](const unsigned long long& b) { return (uint32_t)__cvta_generic_to_shared(&b); };
  if (threadIdx.x == 0) {
    for (int i = 0; i < kMtStages; ++i) {
      bar_init(bar(sh.q_full[i]), 1);
      bar_init(bar(sh.q_free[i]), 1 + kMtSumThreads);
    }
    for (int i = 0; i < kMtSums; ++i) bar_init(bar(sh.d_free[i]), 256);
    for (int i = 0; i < 4; ++i) bar_init(bar(sh.d_full[i >> 1][i & 1]), 1);
    bar_init(bar(sh.drain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.given_up = (sm & 1023) != 0;               // the swizzle goes by addresses
  }
  if (warp == 16) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                 :: "r"((uint32_t)__cvta_generic_to_shared(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* given_up = &sh.given_up;
  // the next one or two tiles of positions: head, first position, how many, first tile of rows
  struct Unit {
    long long u;
    int kvh, p0, two, r0;
  };
  auto next = [&](Unit& x) {
    if (x.u >= u1) return false;
    x.kvh = (int)(x.u / tiles);
    const int t = (int)(x.u - (long long)x.kvh * tiles);
    x.p0 = t * kStRows;
    x.two = x.u + 1 < u1 && t + 1 < tiles;
    x.u += 1 + x.two;
    x.r0 = max(0, x.p0 - a.plen) * a.group / kStRows;     // rows before see none of it
    return true;
  };
  Unit x;
  x.u = u0;
  int qi = 0, di = 0;                             // tiles of rows, sums, so far
  // Sum di goes to group `two ? k : di & 1` of the warps that add up, which has d_full barriers of
  // its own, two in turn: a barrier's phases can only be told apart by who follows each of them. Two
  // are enough: no three sums in a row are one group's, so that before the next but one of it is
  // issued, the present one has been left (there are kMtSums places).
  if (warp < 16) {
    const int g = (warp >> 2) & 1, half = warp >> 3, row = threadIdx.x & 127;
    const uint32_t to_lane = (uint32_t)(32 * (warp & 3)) << 16;
    int di_own = 0;                               // the group's sums so far
    while (next(x)) {
      const int pos = x.p0 + (x.two ? g * kStRows : 0) + row;
      if (g <= x.two) {                           // half of this position's K: 32 of a lane's 64 columns
        const uint4* src = reinterpret_cast<const uint4*>(a.pk + x.kvh * a.p_head + (size_t)pos * kHd) + 8 * half;
#pragma unroll
        for (int c = 0; c < 32; c += 16) {
          uint32_t v[16];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint4 y = pos < n ? __ldg(src + c / 4 + k) : make_uint4(0, 0, 0, 0);
            v[4 * k] = y.x; v[4 * k + 1] = y.y; v[4 * k + 2] = y.z; v[4 * k + 3] = y.w;
          }
          tmem_st16(tmem + to_lane + kMtColK + 64 * g + 32 * half + c, v);
        }
        tmem_st_wait();
      }
      fence_before();
      prior_done();                                        // waits are for this kernel's work alone
      asm volatile("bar.sync 1, 544;" ::: "memory");       // with the warp that issues
      uint64_t acc[2] = {0, 0};
      const int first = max(0, pos - a.plen) * a.group;    // the first row that sees the position
      bool ok = true;
      // 64 columns; `see`: those from there on count (most tiles of rows see every position)
      auto add_up = [&](int stage, int b, int see, auto whole_form) {
        constexpr bool whole = decltype(whole_form)::value;
        const float4* fac = reinterpret_cast<const float4*>(smem + stage * kMtStageStep + 2 * kMtTerm) + 16 * half;
        const float4* off = fac + kStRows / 4;
        const uint32_t at = tmem + to_lane + 128 * b + 64 * half;
        uint32_t v[2][16];
        tmem_ld16(at, v[0]);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
          uint32_t (&c)[16] = v[h & 1];
          tmem_wait(c);
          if (h < 3) {
            tmem_ld16(at + 16 * (h + 1), v[(h + 1) & 1]);
          } else {
            fence_before();
            bar_arrive(bar(sh.d_free[b]));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float4 f = fac[4 * h + i], o = off[4 * h + i];
            const float2 e0 = unpair(fma2(pair(__uint_as_float(c[4 * i]), __uint_as_float(c[4 * i + 1])), pair(f.x, f.y), pair(o.x, o.y)));
            const float2 e1 = unpair(fma2(pair(__uint_as_float(c[4 * i + 2]), __uint_as_float(c[4 * i + 3])), pair(f.z, f.w), pair(o.z, o.w)));
            float w0 = ex2(e0.x), w1 = ex2(e0.y), w2 = ex2(e1.x), w3 = ex2(e1.y);
            if (!whole) {
              const int col = 16 * h + 4 * i;
              w0 = col < see ? 0.0f : w0;
              w1 = col + 1 < see ? 0.0f : w1;
              w2 = col + 2 < see ? 0.0f : w2;
              w3 = col + 3 < see ? 0.0f : w3;
            }
            acc[0] = add2(acc[0], pair(w0, w1));
            acc[1] = add2(acc[1], pair(w2, w3));
          }
        }
      };
      for (int r = x.r0; r < rtiles; ++r, ++qi) {
        const int stage = qi % kMtStages;
        ok = ok && bar_wait_warp(bar(sh.q_full[stage]), (qi / kMtStages) & 1, given_up);
        for (int k = 0; k <= x.two; ++k, ++di) {
          if (x.two ? k != g : (di & 1) != g) continue;
          const int b = di % kMtSums;
          ok = ok && bar_wait_warp(bar(sh.d_full[g][di_own & 1]), (di_own >> 1) & 1, given_up);
          ++di_own;
          if (!ok) continue;
          fence_after();
          const int see = first - r * kStRows - 64 * half;
          if (__any_sync(0xFFFFFFFFu, see > 0)) add_up(stage, b, see, std::false_type{});
          else add_up(stage, b, see, std::true_type{});
        }
        if (ok) bar_arrive(bar(sh.q_free[stage]));
      }
      const float2 s0 = unpair(acc[0]), s1 = unpair(acc[1]);
      sh.sum[warp >> 2][row] = ok ? (s0.x + s0.y) + (s1.x + s1.y) : __int_as_float(0x7fc00000);
      asm volatile("bar.sync 2, 512;" ::: "memory");
      if (half == 0 && g <= x.two && pos < n) {
        const size_t i = (size_t)x.kvh * cap + pos;
        float s = sh.sum[g][row] + sh.sum[g + 2][row];
        if (!x.two) s += sh.sum[1][row] + sh.sum[3][row];
        mass_out[i] = (mass_in && pos < a.plen ? mass_in[i] : 0.0f) + s;
      }
      asm volatile("bar.sync 2, 512;" ::: "memory");
    }
  } else if (warp == 16) {
    const uint32_t leader = elect_one();
    bool ok = true;
    int di_of[2] = {0, 0};                        // each group's sums so far
    prior_done();
    while (next(x)) {
      asm volatile("bar.sync 1, 544;" ::: "memory");
      fence_after();
      for (int r = x.r0; r < rtiles; ++r, ++qi) {
        const int stage = qi % kMtStages;
        ok = ok && bar_wait_warp(bar(sh.q_full[stage]), (qi / kMtStages) & 1, given_up);
        for (int k = 0; k <= x.two; ++k, ++di) {
          const int b = di % kMtSums;
          if (di >= kMtSums) ok = ok && bar_wait_warp(bar(sh.d_free[b]), (di / kMtSums - 1) & 1, given_up);
          if (!ok) continue;
          fence_after();
          const uint64_t qd = smem_desc(sm + stage * kMtStageStep);
#pragma unroll 1
          for (int pass = 1; pass >= 0; --pass)            // the small terms first
#pragma unroll
            for (int s = 0; s < 8; ++s)
              mma_ts(tmem + 128 * b, tmem + kMtColK + 64 * k + 8 * s,
                     qd + (uint64_t)((pass * kMtTerm + (s >> 2) * kMtHalf + (s & 3) * 32) >> 4), kMtDesc,
                     pass == 0 || s > 0, leader);
          const int g = x.two ? k : di & 1;
          mma_commit(bar(sh.d_full[g][(g ? di_of[1] : di_of[0]) & 1]), leader);
          di_of[0] += g == 0;
          di_of[1] += g;
        }
        mma_commit(bar(sh.q_free[stage]), leader);
      }
    }
    int no = 0;                                   // what was issued ends before the memory goes
    mma_commit(bar(sh.drain), leader);
    bar_wait_warp(bar(sh.drain), 0, &no);
  } else if (lane == 0) {
    int issued = 0;
    bool ok = true;
    prior_done();                                 // the rows' terms
    while (next(x))
      for (int r = x.r0; r < rtiles && ok; ++r, ++qi) {
        const int stage = qi % kMtStages;
        if (qi >= kMtStages) ok = bar_wait(bar(sh.q_free[stage]), (qi / kMtStages - 1) & 1, given_up);
        ok = ok && !*given_up;
        if (!ok) break;
        const uint32_t full = bar(sh.q_full[stage]), to = sm + stage * kMtStageStep;
        bar_expect(full, kMtStage);
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            tile_copy(to + t * kMtTerm + h * kMtHalf, &map_q, 64 * h, r * kStRows, t * nkv + x.kvh, full);
        const int Fp = rtiles * kStRows;
#pragma unroll
        for (int t = 0; t < 2; ++t)
          asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                       :: "r"(to + 2 * kMtTerm + t * kStRows * 4),
                          "l"(p.facs + ((size_t)t * nkv + x.kvh) * Fp + r * kStRows), "n"(kStRows * 4), "r"(full) : "memory");
        issued = qi + 1;
      }
    int no = 0;                                   // no copy outlives the CTA
    for (int i = max(0, issued - kMtStages); i < issued; ++i)
      bar_wait(bar(sh.q_full[i % kMtStages]), (i / kMtStages) & 1, &no);
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == 16) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem));
  }
}

}  // namespace

int mass_tile_launch(const SpanArgs& a, const SpanParts& p, const float* mass_in, float* mass_out, int cap,
                     cudaStream_t st) {
  int rc = smem_attr((const void*)k_mass_tile, kMtSmem);
  if (rc) return rc;
  CUtensorMap mq;
  rc = f16_rows_map(p.terms, a.nrow * a.group, 2 * (a.nq / a.group), &mq);
  if (rc) return rc;
  HV_CUDA(launch_beside(k_mass_tile, dim3((unsigned)p.grid), kMtThreads, kMtSmem, st, true, a, p, mass_in, mass_out, cap, mq));
  return HV_OK;
}

}  // namespace hv
