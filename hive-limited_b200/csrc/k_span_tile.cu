// Attention of many rows a head over a binary16 cache, on the fifth-generation tensor cores: a shared
// prefix, or all that a run's rows see, for tiles of 128 (row, head) pairs by 128 positions. Tails
// are k_span_few's or k_span_part's, and k_span_join adds up. Four products of 128 x 128 x 128 a tile
// (two terms of queries, two of weights), 1.4 us at the rate that a library's product has; 256 rows of
// 64 heads over 16384 positions take 208 us, 81% of that rate, with the tensor pipe active two thirds of
// the time and the clock held down by power. A CTA's first tile has left it after 9 us (queries in
// tensor memory 3.2, products 1.8, weights 2, sums 1), every further one 1.8 us later.
//
// The rows' first and second binary16 terms are the operand in tensor memory, K and V tiles come
// by tensor copies into swizzled shared memory as they stand in the cache: K with the dims
// contiguous, V with its dims contiguous too, which for the second product is the other operand's
// outer dimension. Tiles go in turn to two lanes of work w = tile mod 2:
//   warps 0-3    (lane of work 0) and 4-7 (1): a thread has one row of S_w; it writes the row's
//                weights over S_w, two binary16 terms in place of 16 sums; then warp 0 (4),
//                which has nothing to do until S_w is there again, issues O = wl V + wh V and
//                the next S_w = ql K^T + qh K^T
//   warps 8-11   a thread adds its row of O to 128 sums in registers (tensor memory's sums are cut,
//                not rounded, so O is of one tile, and the small terms go first)
//   warps 12, 13 the copies of K and of V, issued by one thread
//   warps 13-15  look over V of tiles that some row does not see whole: what lies behind the rows'
//                positions becomes zeros, and so does a position that is not finite, as 0 times it
//                would be added to rows that do not see it; those that do end as NaN
// A row's weights are 2^(x - m + 8) with m a whole number that a tile's largest exponent may pass:
// as long as no 16 of them add up to more than 2^15 they fit binary16 and are exact to 2^-33 of
// the largest, so that the scores are read once, without a pass for their maximum. The first tile
// has that pass, and a tile that passes the bound makes up for it on the spot: m rises, and what
// has been written of the tile is multiplied by a power of two.
//
// The work is (kv head, tile of rows, tile of positions) in that order, cut evenly among the CTAs,
// one an SM: a CTA has one to three stretches, each of one (kv head, tile of rows), whose sums go
// to the scratch.
//
// Every wait is bounded: one that runs out ends the CTA's work, whose rows are then NaN.
#include "attn_f16.cuh"
#include "hv_internal.h"
#include "tcgen05.cuh"

namespace hv {
namespace {

constexpr int kStThreads = 512;
constexpr int kStHalf = kStRows * 128;          // bytes of 128 positions of 64 halves
constexpr int kStTile = 2 * kStHalf;
constexpr int kStLine = kHd + 4;                // floats from row to row on their way in and out
constexpr int kStLift = 8;                      // log2 of what weights are multiplied by
constexpr float kStDrop = 1.0f / (1 << kStLift);
constexpr uint32_t kStColO = 256, kStColQ = 384;   // tensor memory: S twice, O, qh, ql
// registers per thread: 128 at launch, then dealt out anew
constexpr int kStRegs = 128, kStRegsRow = 144, kStRegsSum = 184, kStRegsCopy = 40;
static_assert(2 * kStRegsRow + kStRegsSum + kStRegsCopy <= 4 * kStRegs, "registers");

// kind::f16 with f32 sums, 128 x 128; V has its outer dimension contiguous
constexpr uint32_t kStDescK = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
constexpr uint32_t kStDescV = kStDescK | (1u << 16);

HV_DEV uint64_t smem_desc_mn(uint32_t addr) {   // 128-byte swizzle, 64 halves outward to a row:
  // 8 rows (of the inner dimension) every 1024 bytes, the next 64 of the outer one after kStHalf
  return (uint64_t)((addr >> 4) & 0x3FFF) | ((uint64_t)(kStHalf >> 4) << 16) | (64ull << 32) |
         (1ull << 46) | (2ull << 61);
}

struct StShared {
  unsigned long long full_k[2], full_v[2], s_ready[2], w_ready[2], o_done[2];
  unsigned long long o_free[2], v_clean[2], drain[2];
  float top[4][kStRows];         // of the last four tiles: what their weights are relative to
  float m[2][kStRows], l[2][kStRows];
  uint32_t tmem;
  int bad;                       // first position of the stretch that is not finite
  int given_up;
};
constexpr int kStSmem = 4 * kStTile + kStRows * kStLine * 4 + (int)sizeof(StShared);   // K, V twice

__global__ void __launch_bounds__(kStThreads, 1)
    k_span_tile(SpanArgs a, SpanParts p, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v) {
  extern __shared__ __align__(1024) uint8_t smem[];
  StShared& sh = *reinterpret_cast<StShared*>(smem + 4 * kStTile + kStRows * kStLine * 4);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int F = a.nrow * a.group, nkv = a.nq / a.group;
  next_may_start();
  const int np = span_prefix(a);
  const uint32_t sm = (uint32_t)__cvta_generic_to_shared(smem);
  auto bar = [](const unsigned long long& b) { return (uint32_t)__cvta_generic_to_shared(&b); };
  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(bar(sh.full_k[i]), 1);
      bar_init(bar(sh.full_v[i]), 1);
      bar_init(bar(sh.s_ready[i]), 1);
      bar_init(bar(sh.w_ready[i]), 128);
      bar_init(bar(sh.o_done[i]), 1);
      bar_init(bar(sh.drain[i]), 1);
      bar_init(bar(sh.v_clean[i]), 96);
      bar_init(bar(sh.o_free[i]), 128);
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.given_up = (sm & 1023) != 0;               // the swizzle goes by addresses
  }
  if (warp == 15) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                 :: "r"((uint32_t)__cvta_generic_to_shared(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  const SpanWhole wh = span_whole(a, np, gridDim.x);         // (its loads take as long as what is above)
  const bool some = (int)blockIdx.x < wh.ctas;
  const unsigned u0 = some ? span_first(wh, blockIdx.x) : 0, u1 = some ? span_first(wh, blockIdx.x + 1) : 0;
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* given_up = &sh.given_up;
  const int w = warp >> 2, row = threadIdx.x & 127;
  float* lines = reinterpret_cast<float*>(smem + 4 * kStTile);    // [row][kStLine]
  auto rows_sync = [] { asm volatile("bar.sync 3, 256;" ::: "memory"); };
  // the next stretch with work: its place, tiles j0 .. j0 + nt - 1 of positions, and its rows' slot
  struct Stretch {
    unsigned u;
    int kvh, row0, j0, nt;
    int full, end;                                // its tiles that all rows see whole, positions
    int last;                                     // with the last of its rows' tiles: their slots
    size_t part_row;
  };
  auto next = [&](Stretch& s) {
    while (s.u < u1) {
      const unsigned R = s.u / wh.tiles;
      s.kvh = (int)(R / wh.rows);
      const int tile = (int)(R - s.kvh * wh.rows);
      s.j0 = (int)(s.u - R * wh.tiles);
      const int some = min(wh.tiles - s.j0, (int)(u1 - s.u));
      s.u += some;
      const int tiles = span_tiles_of(a, np, tile);
      s.nt = min(tiles - s.j0, some);
      if (s.nt <= 0) continue;
      s.row0 = tile * kStRows;
      s.full = min(max(span_sees(a, np, s.row0) / kStRows - s.j0, 0), s.nt);
      s.end = span_sees(a, np, min(F, s.row0 + kStRows) - 1) - s.j0 * kStRows;
      const int slot = blockIdx.x - span_cta(wh, R * wh.tiles);
      s.last = s.j0 + s.nt == tiles ? slot + 1 : 0;
      s.part_row = ((size_t)slot * nkv + s.kvh) * F + s.row0;
      return true;
    }
    return false;
  };
  auto stretch_end = [] {                         // every role, before the next one's rows
    __syncwarp();
    fence_before();
    asm volatile("bar.sync 0, 512;" ::: "memory");
    fence_after();
  };
  Stretch st;
  st.u = u0;
  int g0 = 0, parts = 0;                          // tiles before this stretch's; bit i mod 2: was the
                                                  // number of those with a part odd?
  auto step_on = [&] {                            // (at most two tiles of a stretch are parts)
    for (int i = g0 + st.full; i < g0 + st.nt; ++i) parts ^= 1 << (i & 1);
    g0 += st.nt;
  };
  auto rows_out = [&] {
    asm volatile("bar.sync 2, 384;" ::: "memory");
    float4* to = reinterpret_cast<float4*>(p.part + st.part_row * kHd);
#pragma unroll 4
    for (int r = warp; r < kStRows; r += 12)
      if (st.row0 + r < F)
        to[r * (kHd / 4) + lane] = *reinterpret_cast<const float4*>(lines + (size_t)r * kStLine + 4 * lane);
  };
  if (warp < 8) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kStRegsRow));
    int drains = 0;
#pragma unroll 1
    for (; next(st); step_on(), stretch_end()) {
      // The queries in two terms. A warp loads whole rows (a thread its own row's half: 32 rows an
      // instruction, 4 us), and through shared memory a row's two threads get half of its dims
      // each. They take the scale's sign.
      float qs;
      {
        float4 x[kStRows / 8];
#pragma unroll
        for (int j = 0; j < kStRows / 8; ++j) {
          const int gr = min(st.row0 + warp + 8 * j, F - 1), tok = span_row(a, gr);
          x[j] = __ldg(reinterpret_cast<const float4*>(
              a.q + ((size_t)tok * a.nq + (size_t)st.kvh * a.group + gr - tok * a.group) * kHd) + lane);
        }
        const float qscale = __ldg(a.scale) * kLog2e;
#pragma unroll
        for (int j = 0; j < kStRows / 8; ++j) {
          const float big = fmaxf(fmaxf(fabsf(x[j].x), fabsf(x[j].y)), fmaxf(fabsf(x[j].z), fabsf(x[j].w)));
          const unsigned u = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(big));
          if (lane == 0) sh.m[0][warp + 8 * j] = __uint_as_float(u);
          *reinterpret_cast<float4*>(lines + (size_t)(warp + 8 * j) * kStLine + 4 * lane) = x[j];
        }
        asm volatile("bar.sync 5, 288;" ::: "memory");     // with the warp that copies V
        static_assert(kStRows == kHd, "x");
#pragma unroll
        for (int d = 0; d < kHd / 8; ++d)
          x[d] = *reinterpret_cast<const float4*>(lines + (size_t)row * kStLine + 64 * w + 4 * d);
        const float lift = copysignf(q8_lift(sh.m[0][row]), qscale);
        qs = qscale / lift;
        qs = qs == 0.0f ? 2e-38f : qs;             // -infinity times it is to stay that
        const uint32_t to = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + kStColQ + 32 * w;
#pragma unroll
        for (int d = 0; d < kHd / 8; d += 8) {
          uint32_t hi[16], lo[16];
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            split_half2(x[d + k].x * lift, x[d + k].y * lift, &hi[2 * k], &lo[2 * k]);
            split_half2(x[d + k].z * lift, x[d + k].w * lift, &hi[2 * k + 1], &lo[2 * k + 1]);
          }
          tmem_st16(to + 2 * d, hi);
          tmem_st16(to + 64 + 2 * d, lo);
        }
        tmem_st_wait();
      }
      fence_before();
      rows_sync();
      fence_after();
      float m = -INFINITY, l = 0.0f;              // of this thread's row, m in units of `unit`
      float unit = 1.0f;
      const int sees = span_sees(a, np, min(st.row0 + row, F - 1)) - st.j0 * kStRows;
      const uint32_t s_at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 128 * w;
      const uint32_t leader = elect_one();
      const uint32_t qh = tmem + kStColQ, ql = qh + 64;
      bool ok = true;
      auto product_s = [&](int i) {
        const int s = i & 1;
        const uint64_t kd = smem_desc(sm + s * kStTile);
        const uint32_t d = tmem + 128 * s;
        ok = ok && bar_wait_warp(bar(sh.full_k[s]), (i >> 1) & 1, given_up);
        fence_after();
#pragma unroll 1
        for (int pass = 0; pass < 2 && ok; ++pass) {
          const uint32_t q = pass ? qh : ql;
          // a step of 16 dims: the half it is in, then 32 bytes each
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_ts(d, q + 8 * k, kd + (uint64_t)(((k >> 2) * kStHalf + (k & 3) * 32) >> 4), kStDescK,
                   pass > 0 || k > 0, leader);
        }
        mma_commit(bar(sh.s_ready[s]), leader);
      };
      auto product_o = [&](int i) {
        const int s = i & 1;
        const uint64_t vd = smem_desc_mn(sm + (2 + s) * kStTile);
        const uint32_t d = tmem + kStColO;
        ok = ok && bar_wait_warp(bar(sh.full_v[s]), (i >> 1) & 1, given_up);
        ok = ok && bar_wait_warp(bar(sh.w_ready[s]), (i >> 1) & 1, given_up);
        // (O of the tile before, on a barrier of which this lane follows every phase)
        if (i > 0) ok = ok && bar_wait_warp(bar(sh.o_free[1 - s]), ((i - 1) >> 1) & 1, given_up);
        if (i - g0 >= st.full) ok = ok && bar_wait_warp(bar(sh.v_clean[s]), parts >> s & 1, given_up);
        fence_after();
#pragma unroll 1
        for (int pass = 0; pass < 2 && ok; ++pass) {
          // the weights of 16 positions are 8 columns of first terms, then 8 of second ones; 16
          // positions of V are 16 rows of 128 bytes
          const uint32_t wt = tmem + 128 * s + (pass ? 0 : 8);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            mma_ts(d, wt + 16 * k, vd + (uint64_t)(k * 2048 >> 4), kStDescV, pass > 0 || k > 0, leader);
        }
        mma_commit(bar(sh.o_done[s]), leader);
      };
      const bool issues = (warp & 3) == 0;
      // the row's largest exponent from column c0 on, as a whole number
      auto largest = [&](int c0) {
        float big = -INFINITY;
#pragma unroll 1
        for (int c = c0; c < kStRows; c += 16) {
          uint32_t x[16];
          tmem_ld16(s_at + c, x);
          tmem_wait(x);
#pragma unroll
          for (int k = 0; k < 16; ++k) big = fmaxf(big, __uint_as_float(x[k]));
        }
        return ceilf(big * qs);
      };
      auto weights = [&](int i, bool first) {
        if (i - g0 >= st.full) {                  // what the row does not see of the tile
          const int see = sees - (i - g0) * kStRows;
#pragma unroll 1
          for (int c = 0; c < kStRows; c += 16) {
            uint32_t x[16];
            tmem_ld16(s_at + c, x);
            tmem_wait(x);
#pragma unroll
            for (int k = 0; k < 16; ++k) x[k] = c + k < see ? x[k] : 0xFF800000u;
            tmem_st16(s_at + c, x);
          }
          tmem_st_wait();
        }
        // An exponent is a product's, rounded once with m taken off, so it may pass m by half of what
        // m is rounded by: beyond 2^26 too much for a weight. Exponents of such rows count in units
        // of a power of two that keeps them under it. Weights are then not 0 within 150 such units, which
        // is 2^-17.8 of the score: no more than what errors of 44 u on two scores come to.
        uint64_t f2, off, sum = 0;
        auto base = [&](float top) {
          if (fabsf(top) > 67108864.0f && fabsf(top) < INFINITY) {
            const float s = __uint_as_float((127u + 25u + 127u) * 0x800000u - (__float_as_uint(top) & 0x7F800000u));
            top = ceilf(top * s);
            qs *= s;
            unit /= s;
          }
          m = top;
          f2 = pair(qs, qs);
          const float o = m == -INFINITY ? 0.0f : (float)kStLift - m;
          off = pair(o, o);
        };
        base(first ? largest(0) : m);
        uint32_t z[2][16];
        tmem_ld16(s_at, z[0]);
#pragma unroll 1
        for (int h = 0; h < 8; h += 2) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t (&x)[16] = z[g];
            tmem_wait(x);
            if (g == 0 || h < 6) tmem_ld16(s_at + 16 * (h + g) + 16, z[1 - g]);
            uint64_t pr[8], cs;
            auto exps = [&] {
              cs = 0;
#pragma unroll
              for (int k = 0; k < 8; ++k) {
                const float2 e = unpair(fma2(pair(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), f2, off));
                pr[k] = pair(ex2(e.x), ex2(e.y));
                cs = add2(cs, pr[k]);
              }
            };
            exps();
            const float2 both = unpair(cs);
            if (__builtin_expect(__any_sync(0xFFFFFFFFu, !(both.x + both.y <= 32768.0f)), 0)) {
              m *= unit;                           // (units are chosen anew)
              qs *= unit;
              unit = 1.0f;
              const float up = fmaxf(m, largest(16 * (h + g)));
              const float fall = m == -INFINITY ? 0.0f : fmaxf(m - up, -60.0f);   // 2^-60 of it is as good as 0
              const float f0 = ex2(fall);
              l *= f0;
              const float2 s2 = unpair(sum);
              sum = pair(s2.x * f0, s2.y * f0);
              const float fa = ex2(floorf(0.5f * fall)), fb = ex2(fall - floorf(0.5f * fall));
              const __half2 ha = __floats2half2_rn(fa, fa), hb = __floats2half2_rn(fb, fb);
              base(up);
              tmem_st_wait();
#pragma unroll 1
              for (int c = 0; c < h + g; ++c) {             // what has been written of the tile
                uint32_t y[16];
                tmem_ld16(s_at + 16 * c, y);
                tmem_wait(y);
#pragma unroll
                for (int k = 0; k < 16; ++k) {
                  const __half2 t2 = __hmul2(__hmul2(*reinterpret_cast<const __half2*>(&y[k]), ha), hb);
                  y[k] = *reinterpret_cast<const uint32_t*>(&t2);
                }
                tmem_st16(s_at + 16 * c, y);
              }
              exps();
            }
            sum = add2(sum, cs);
            // the first term is cut to binary16's 11 bits, so that the rest is exact
            uint32_t wt[16];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const float2 q = unpair(pr[k]);
              const float2 c1 = make_float2(__uint_as_float(__float_as_uint(q.x) & 0xFFFFE000u),
                                            __uint_as_float(__float_as_uint(q.y) & 0xFFFFE000u));
              const float2 r = unpair(fma2(pair(c1.x, c1.y), pair(-1.0f, -1.0f), pr[k]));
              wt[k] = pack_half2(c1.x, c1.y);
              wt[8 + k] = pack_half2(r.x, r.y);
            }
            tmem_st16(s_at + 16 * (h + g), wt);
          }
        }
        const float2 s2 = unpair(sum);
        l += s2.x + s2.y;
        sh.top[i & 3][row] = m * unit;
        tmem_st_wait();
        fence_before();
        bar_arrive(bar(sh.w_ready[w]));
      };
      const int end = g0 + st.nt;
      int i = g0 + ((g0 ^ w) & 1);                // this lane's tiles: those of its parity
      bool first = true;
#pragma unroll 1
      for (;; i += 2) {
        if (issues) {
          if (i - 2 >= g0) product_o(i - 2);
          if (i < end) product_s(i);
        }
        if (i >= end) break;
        if (!bar_wait_warp(bar(sh.s_ready[w]), (i >> 1) & 1, given_up)) break;
        fence_after();
        weights(i, first);
        first = false;
      }
      if (issues && !ok) {                        // what was issued ends before the memory goes
        int no = 0;
        mma_commit(bar(sh.drain[w]), leader);
        bar_wait_warp(bar(sh.drain[w]), drains++ & 1, &no);
      }
      sh.m[w][row] = m * unit;
      sh.l[w][row] = l;
      asm volatile("bar.sync 1, 384;" ::: "memory");       // with the warps that have the sums
      rows_out();
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kStRegsSum));
#pragma unroll 1
    for (; next(st); step_on(), stretch_end()) {
      uint64_t acc[kHd / 2];
#pragma unroll
      for (int d = 0; d < kHd / 2; ++d) acc[d] = 0;
      float M = -INFINITY;                        // what the sums are relative to
      const uint32_t o_at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + kStColO;
      for (int i = g0; i < g0 + st.nt; ++i) {
        if (!bar_wait_warp(bar(sh.o_done[i & 1]), (i >> 1) & 1, given_up)) break;
        fence_after();
        const float m = sh.top[i & 3][row], up = fmaxf(M, m);
        const float fa = M == -INFINITY ? 0.0f : ex2(M - up), fo = m == -INFINITY ? 0.0f : ex2(m - up);
        const uint64_t fa2 = pair(fa, fa), fo2 = pair(fo, fo);
        M = up;
        uint32_t v[2][16];
        tmem_ld16(o_at, v[0]);
#pragma unroll
        for (int h = 0; h < 8; ++h) {
          uint32_t (&x)[16] = v[h & 1];
          tmem_wait(x);
          if (h < 7) {
            tmem_ld16(o_at + 16 * (h + 1), v[(h + 1) & 1]);
          } else {
            fence_before();
            bar_arrive(bar(sh.o_free[i & 1]));
          }
#pragma unroll
          for (int k = 0; k < 8; ++k)
            acc[8 * h + k] = fma2(acc[8 * h + k], fa2,
                                  mul2(pair(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), fo2));
        }
      }
      asm volatile("bar.sync 1, 384;" ::: "memory");
      float L = 0.0f;
#pragma unroll
      for (int k = 0; k < 2; ++k)
        L += sh.l[k][row] == 0.0f ? 0.0f : sh.l[k][row] * ex2(sh.m[k][row] - M);
      // (V has been looked over once the last sums are there)
      if (*given_up || span_sees(a, np, min(st.row0 + row, F - 1)) - st.j0 * kStRows > sh.bad)
        L = __int_as_float(0x7fc00000);
      float* line = lines + (size_t)row * kStLine;
#pragma unroll
      for (int d = 0; d < kHd / 2; d += 2) {
        const float2 x = unpair(mul2(acc[d], pair(kStDrop, kStDrop))), y = unpair(mul2(acc[d + 1], pair(kStDrop, kStDrop)));
        *reinterpret_cast<float4*>(line + 2 * d) = make_float4(x.x, x.y, y.x, y.y);
      }
      if (st.last && row == 0) p.stretches[st.kvh * wh.rows + st.row0 / kStRows] = st.last;
      if (st.row0 + row < F) p.ml[st.part_row + row] = make_float2(M, L * kStDrop);
      rows_out();
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kStRegsCopy));
    // a tile of K or V; a buffer is free once its last product is done
    auto tile_load = [&](int to, const CUtensorMap* map, int pos, int head, uint32_t full) {
      if (lane != 0) return;
      bar_expect(full, kStTile);
      tile_copy(sm + to, map, 0, pos, head, full);
      tile_copy(sm + to + kStHalf, map, 64, pos, head, full);
    };
#pragma unroll 1
    for (; next(st); step_on(), stretch_end()) {
      if (warp == 13 && lane == 0) sh.bad = 1 << 30;
      // Warps 13 to 15 meet at every part once its V has come, which warp 13 has seen: a barrier's
      // phases can only be told apart by who follows each of them.
      auto clean = [&](int i, bool live) {
        asm volatile("bar.sync 4, 96;" ::: "memory");
        if (live) {
          // a thread has 16 bytes of every twelfth row
          uint8_t* v = smem + (2 + (i & 1)) * kStTile + 16 * (lane & 7);
          const int at = (i - g0) * kStRows;
          for (int r = (lane >> 3) + 4 * (warp - 13); r < kStRows; r += 12)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              uint4* y = reinterpret_cast<uint4*>(v + h * kStHalf + r * 128);
              const bool behind = at + r >= st.end;
              if (behind || not_finite(*y)) {
                *y = make_uint4(0, 0, 0, 0);
                if (!behind) atomicMin(&sh.bad, at + r);
              }
            }
        }
        fence_async();
        bar_arrive(bar(sh.v_clean[i & 1]));
      };
      if (warp >= 14) {
#pragma unroll 1
        for (int i = g0 + st.full; i < g0 + st.nt; ++i) clean(i, true);
        continue;
      }
      if (warp == 13) {
        asm volatile("bar.sync 5, 288;" ::: "memory");     // the queries come before V
        bool live = true;
        int issued = g0;
#pragma unroll 1
        for (int i = g0; i < g0 + st.nt; ++i) {
          const int s = i & 1;
          live = live && (i < 2 || bar_wait_warp(bar(sh.o_done[s]), ((i - 2) >> 1) & 1, given_up));
          live = live && !__any_sync(0xFFFFFFFFu, *given_up);
          if (live) {
            tile_load(2 * kStTile + s * kStTile, &map_v, (st.j0 + i - g0) * kStRows, st.kvh, bar(sh.full_v[s]));
            issued = i + 1;
          }
          if (i - g0 >= st.full) {
            if (live) bar_wait_warp(bar(sh.full_v[s]), (i >> 1) & 1, given_up);
            clean(i, live);
          }
        }
        int no = 0;                               // no copy outlives the CTA
        for (int i = max(g0, issued - 2); i < issued; ++i)
          bar_wait_warp(bar(sh.full_v[i & 1]), (i >> 1) & 1, &no);
        continue;
      }
      if (lane != 0) continue;
      int issued = g0;
      for (int i = g0; i < g0 + st.nt; ++i, ++issued) {
        const int s = i & 1;
        if (i >= 2 && !bar_wait(bar(sh.s_ready[s]), ((i - 2) >> 1) & 1, given_up)) break;
        if (*given_up) break;
        tile_load(s * kStTile, &map_k, (st.j0 + i - g0) * kStRows, st.kvh, bar(sh.full_k[s]));
      }
      int no = 0;
      for (int i = max(g0, issued - 2); i < issued; ++i)
        bar_wait(bar(sh.full_k[i & 1]), (i >> 1) & 1, &no);
    }
  }
  if (warp == 15)
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem));
}

typedef CUresult (*MapFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                          const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                          CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
}  // namespace

int f16_rows_map(const __half* base, int rows, int outer, CUtensorMap* out) {
  static MapFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult r;
    return cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &r) == cudaSuccess &&
                   r == cudaDriverEntryPointSuccess
               ? (MapFn)f
               : (MapFn) nullptr;
  }();
  HV_REQUIRE(fn != nullptr, HV_E_UNSUPPORTED, "the driver has no cuTensorMapEncodeTiled");
  const cuuint64_t dims[3] = {(cuuint64_t)kHd, (cuuint64_t)rows, (cuuint64_t)outer};
  const cuuint64_t strides[2] = {(cuuint64_t)kHd * 2, (cuuint64_t)rows * kHd * 2};
  const cuuint32_t box[3] = {64u, (cuuint32_t)kStRows, 1u}, step[3] = {1u, 1u, 1u};
  const CUresult r = fn(out, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, const_cast<__half*>(base), dims, strides, box, step,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                        CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  HV_REQUIRE(r == CUDA_SUCCESS, HV_E_INVALID, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return HV_OK;
}


int span_tile_launch(const SpanArgs& a, const SpanParts& p, cudaStream_t st) {
  int rc = smem_attr((const void*)k_span_tile, kStSmem);
  if (rc) return rc;
  // registers are dealt out of what the kernel starts with: a share too large would wait for good
  static const int regs = [] {
    cudaFuncAttributes f{};
    return cudaFuncGetAttributes(&f, k_span_tile) == cudaSuccess ? f.numRegs : 0;
  }();
  HV_REQUIRE(regs == kStRegs, HV_E_UNSUPPORTED, "k_span_tile: built with %d registers", regs);
  CUtensorMap mk, mv;
  rc = f16_rows_map(a.pk, a.pcap, a.nq / a.group, &mk);
  if (!rc) rc = f16_rows_map(a.pv, a.pcap, a.nq / a.group, &mv);
  if (rc) return rc;
  k_span_tile<<<(unsigned)p.grid, kStThreads, kStSmem, st>>>(a, p, mk, mv);
  HV_LAUNCHED("k_span_tile");
}

}  // namespace hv
