// Attention of a long run of query rows over the 8-bit cache, on the fifth-generation tensor
// cores. The mathematics is k_attn_q8.cu's: f32 factors as two binary16 terms, codes exact.
//
// A CTA has 128 (token, head) rows of a kv head and a chunk of its positions, 128 positions
// (four blocks) to a tile, tiles in turn to two lanes of work w = tile mod 2:
//   warps 8-11  turn the codes of a tile into binary16 in shared memory: K [position][dim] and
//               V transposed [dim][position], 128-byte swizzled rows; the codes of the next
//               tile come by asynchronous copies meanwhile
//   warp 12     issues S_w = ql K^T + qh K^T and O_w = wl V + wh V (wh, wl in tensor memory)
//   warps 0-3   (lane of work 0) and 4-7 (1): a thread has one row of S_w; it writes the row's
//               weights over S_w, two binary16 terms in place of 32 sums, and adds O_w to the
//               row's 128 sums in registers
// so while one lane of work is at its weights the tensor cores run the other's products. Each
// lane has its own maximum and sums, and the two meet at the end.
//
// The tensor cores cut their f32 sums instead of rounding them, once for every 16 positions:
// kept in tensor memory over 64 tiles, O was 1.8e-5 too small. So O_w is of one tile, and the
// small terms go first, while the sums are small.
//
// The scale of a V block has to multiply its weights here, as a tile's sum stays in tensor
// memory: a weight enters as w s_v, that is 2^(x + log2 s_v), and the maximum that the row
// keeps is that of these products, so that a block with a large scale that the row hardly
// attends to does not cost the others precision; the sum of the weights adds w s_v / s_v.
// Weights stand as 2^15 times themselves, exact to 2^-40 of the row's largest.
// The open block's f32 rows are two binary16 terms: after the tile's products with the first
// term, the same buffer holds the second one (zero elsewhere) for one product more.
//
// Every wait is bounded: one that runs out ends the CTA, whose rows are then NaN.
#include "attn_q8.cuh"
#include "attn_q8_rows.h"
#include "hv_internal.h"
#include "hv_wait.cuh"

namespace hv {
namespace {

constexpr int kTlRows = 128;                    // rows of a CTA and positions of a tile
constexpr int kTlThreads = 512;
constexpr int kTlHalf = 128 * 128;              // bytes of 128 rows of 64 halves
constexpr int kTlTile = 2 * kTlHalf;            // bytes of a 128 x 128 binary16 tile
constexpr int kTlStage = 4 * 2 * kQ8Codes;      // codes of a tile's four blocks
constexpr float kTlLift = 32768.0f;             // 2^15
// registers per thread: 128 at launch, given from the converting and issuing warps to the rows
constexpr int kTlRegsRow = 192, kTlRegsConv = 80, kTlRegsIssue = 48;
constexpr int kTlRegsSum = 256 * kTlRegsRow + 128 * kTlRegsConv + 128 * kTlRegsIssue;
static_assert(kTlRegsSum <= 512 * 128, "registers");
constexpr unsigned long long kTlWaitNs = 2000000000ull;

// kind::f16 with f32 sums, 128 x 128, both operands with the inner dimension contiguous
constexpr uint32_t kTlDesc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);

HV_DEV uint64_t smem_desc(uint32_t addr) {      // 128-byte swizzle, 1024 bytes per 8 rows
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}
// One lane of a whole warp issues: the warp stays together, so that the descriptors are uniform
// registers, which the instruction wants (in a branch of one lane it took 190 cycles to issue
// a product that runs for 64).
HV_DEV void mma_ss(uint32_t d, uint64_t a, uint64_t b, bool add, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :: "r"(d), "l"(a), "l"(b), "r"(kTlDesc), "r"((uint32_t)add), "r"(leader) : "memory");
}
HV_DEV void mma_ts(uint32_t d, uint32_t a, uint64_t b, bool add, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      :: "r"(d), "r"(a), "l"(b), "r"(kTlDesc), "r"((uint32_t)add), "r"(leader) : "memory");
}
HV_DEV void mma_commit(uint32_t bar, uint32_t leader) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}"
      :: "r"(bar), "r"(leader) : "memory");
}
HV_DEV uint32_t elect_one() {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
  return r;
}
HV_DEV void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
HV_DEV void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
HV_DEV void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

#define HV_R4(v, i) "=r"(v[i]), "=r"(v[i + 1]), "=r"(v[i + 2]), "=r"(v[i + 3])
#define HV_P4(v, i) "+r"(v[i]), "+r"(v[i + 1]), "+r"(v[i + 2]), "+r"(v[i + 3])
#define HV_W4(v, i) "r"(v[i]), "r"(v[i + 1]), "r"(v[i + 2]), "r"(v[i + 3])
// 16 columns of this thread's row: begun here, in hand after tmem_wait. One load is under way
// while the columns before it are worked on.
HV_DEV void tmem_ld16(uint32_t at, uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : HV_R4(v, 0), HV_R4(v, 4), HV_R4(v, 8), HV_R4(v, 12) : "r"(at) : "memory");
}
HV_DEV void tmem_wait(uint32_t (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : HV_P4(v, 0), HV_P4(v, 4), HV_P4(v, 8), HV_P4(v, 12) :: "memory");
}
// Columns past `see` become -infinity.
HV_DEV void hide(uint32_t (&v)[16], int see) {
  asm volatile("" ::: "memory");                // a branch, not 16 selections every time
#pragma unroll
  for (int k = 0; k < 16; ++k) v[k] = k <= see ? v[k] : 0xFF800000u;
}
HV_DEV void tmem_st8(uint32_t at, const uint32_t (&v)[8]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
      :: "r"(at), HV_W4(v, 0), HV_W4(v, 4) : "memory");
}
HV_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

HV_DEV void bar_init(uint32_t bar, int count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" :: "r"(bar), "r"(count) : "memory");
}
HV_DEV void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
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
      else if (now - t0 > kTlWaitNs) { *given_up = 1; return false; }
    }
  }
}

// The same for a whole warp, whose lanes go on or leave together.
HV_DEV bool bar_wait_warp(uint32_t bar, uint32_t parity, volatile int* given_up) {
  const bool ok = bar_wait(bar, parity, given_up);
  return __all_sync(0xFFFFFFFFu, ok) != 0;
}

HV_DEV uint64_t pair(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
HV_DEV float2 unpair(uint64_t x) {
  float2 r;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(r.x), "=f"(r.y) : "l"(x));
  return r;
}
HV_DEV uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
HV_DEV uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
HV_DEV uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

struct TlShared {
  unsigned long long full_k[2], full_v[2], s_ready[2], w_ready[2], o_done[2], k_free, v_free, drain;
  float sc[4][4][4];             // of the last four tiles' blocks: s_k, log2 s_v, 1 / s_v
  float lift[kTlRows];
  float m[2][kTlRows], l[2][kTlRows];
  uint32_t tmem;
  int bad;                       // first open row with a value that is not finite
  int given_up;
  unsigned last;
};
constexpr int kTlSmem = 6 * kTlTile + kTlStage + (int)sizeof(TlShared);   // qh, ql, K, V twice
static_assert(kTlSmem <= 232448, "shared memory of an SM");

__global__ void __launch_bounds__(kTlThreads, 1) k_attn_tile_q8(RowsArgs a, KvQ8 c) {
  extern __shared__ __align__(1024) uint8_t smem[];
  TlShared& sh = *reinterpret_cast<TlShared*>(smem + 6 * kTlTile + kTlStage);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, tile = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const int nrows = a.ntok * a.group, row0 = tile * kTlRows;
  const int last_row = min(nrows, row0 + kTlRows) - 1;
  const int held = q8_held(c, kvh), closed = held / kQ8Blk;
  const int top = min(a.pos0 + last_row / a.group, held - 1);     // the last position to read
  const int nb = min(closed, top < 0 ? 0 : top / kQ8Blk + 1);
  const bool tail = top >= closed * kQ8Blk;
  const int items = nb + (tail ? 1 : 0);                          // blocks, the open one last
  const int nact = max(1, min(a.chunks, items / 8));
  if (chunk >= nact) return;
  const int b0 = (int)((long long)items * chunk / nact);
  const int b1 = (int)((long long)items * (chunk + 1) / nact);
  const int nt = (b1 - b0 + 3) / 4;
  const bool has_tail = tail && b1 == items;

  const uint32_t sm = (uint32_t)__cvta_generic_to_shared(smem);
  uint8_t* k_buf = smem + 2 * kTlTile;            // two tiles, then V's two
  uint8_t* v_buf = smem + 4 * kTlTile;
  auto bar = [](const unsigned long long& b) { return (uint32_t)__cvta_generic_to_shared(&b); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(bar(sh.full_k[i]), 128);
      bar_init(bar(sh.full_v[i]), 128);
      bar_init(bar(sh.s_ready[i]), 1);
      bar_init(bar(sh.w_ready[i]), 128);
      bar_init(bar(sh.o_done[i]), 1);
    }
    bar_init(bar(sh.k_free), 1);
    bar_init(bar(sh.v_free), 1);
    bar_init(bar(sh.drain), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.bad = kQ8Blk;
    sh.given_up = 0;
  }
  if (warp == 12) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                 :: "r"((uint32_t)__cvta_generic_to_shared(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  // the queries in two terms, a row per warp at a time; they take the scale's sign, so that the
  // largest sum of products is the largest exponent
  const float qscale = __ldg(a.scale) * kLog2e;
  for (int r = warp; r < kTlRows; r += kTlThreads / 32) {
    const int gr = row0 + r;
    float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
    if (gr < nrows)
      x = __ldg(reinterpret_cast<const float4*>(
                    a.q + ((size_t)(gr / a.group) * a.nq + (size_t)kvh * a.group + gr % a.group) * kHd) +
                lane);
    float amax = fmaxf(fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xFFFFFFFFu, amax, o));
    const float lift = copysignf(q8_lift(amax), qscale);
    uint32_t h0, h1, l0, l1;
    split_half2(x.x * lift, x.y * lift, &h0, &l0);
    split_half2(x.z * lift, x.w * lift, &h1, &l1);
    const int at = (lane >> 4) * kTlHalf + r * 128 + ((((lane & 15) >> 1) ^ (r & 7)) << 4) +
                   (lane & 1) * 8;
    *reinterpret_cast<uint2*>(smem + at) = make_uint2(h0, h1);
    *reinterpret_cast<uint2*>(smem + kTlTile + at) = make_uint2(l0, l1);
    if (lane == 0) sh.lift[r] = lift;
  }
  fence_async();
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* given_up = &sh.given_up;

  const int ntile = gridDim.x / a.chunks;
  const size_t slot = ((size_t)kvh * ntile + tile) * a.chunks;
  if (warp < 8) {
    float m = -INFINITY, l = 0.0f;                // of this thread's row
    uint64_t acc[kHd / 2];
    const int w = warp >> 2, row = threadIdx.x & 127, grow = row0 + row;
    auto rows_sync = [] { asm volatile("bar.sync 1, 256;" ::: "memory"); };
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kTlRegsRow));
#pragma unroll
    for (int d = 0; d < kHd / 2; ++d) acc[d] = 0;
    const uint32_t s_at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 128 * w;
    const uint32_t o_at = s_at + 256;
    const int lim = grow < nrows ? min(min(a.pos0 + grow / a.group, held - 1), 32 * b1 - 1) : -1;
    const float qs = qscale / sh.lift[row];
    for (int i = w; i < nt; i += 2) {
      if (!bar_wait_warp(bar(sh.s_ready[w]), (i >> 1) & 1, given_up)) break;
      fence_after();
      const int see0 = lim - 32 * (b0 + 4 * i);            // columns 0 .. see0 are seen
      const bool all = __all_sync(0xFFFFFFFFu, see0 >= kTlRows - 1);
      uint32_t v[2][16];
      // the largest exponent of the row in this tile
      float up = m, mx = -INFINITY;
      // (loops over blocks stay rolled: three roles' code has to fit the instruction cache)
      tmem_ld16(s_at, v[0]);
#pragma unroll 1
      for (int b = 0; b < 4; ++b) {
        const int see = see0 - 32 * b;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t (&x)[16] = v[h];
          tmem_wait(x);
          tmem_ld16(s_at + (32 * b + 16 * (h + 1)) % 128, v[1 - h]);
          if (!all) hide(x, see - 16 * h);
#pragma unroll
          for (int k = 0; k < 16; ++k) mx = fmaxf(mx, __uint_as_float(x[k]));
        }
        if (see >= 0) up = fmaxf(up, fmaf(mx, sh.sc[i & 3][b][0] * qs, sh.sc[i & 3][b][1]));
        mx = -INFINITY;
      }
      const float shrink = m == -INFINITY ? 0.0f : ex2(m - up);
      l *= shrink;
      m = up;
      const float m0 = m == -INFINITY ? 0.0f : m;
      // the first columns are under way again
#pragma unroll 1
      for (int b = 0; b < 4; ++b) {
        const int see = see0 - 32 * b;
        float f = sh.sc[i & 3][b][0] * qs;
        f = f == 0.0f ? 1e-38f : f;                         // -inf f has to stay -inf
        const float lv = sh.sc[i & 3][b][1] - m0;
        const uint64_t f2 = pair(f, f), lv2 = pair(lv, lv);
        uint64_t sum = 0;
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t (&x)[16] = v[h];
          tmem_wait(x);
          if (h == 0 || b < 3) tmem_ld16(s_at + 32 * b + 16 * (h + 1), v[1 - h]);
          if (!all) hide(x, see - 16 * h);
          uint32_t hi[8], lo[8];
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const float2 e = unpair(fma2(pair(__uint_as_float(x[k]), __uint_as_float(x[k + 1])), f2, lv2));
            float2 p = make_float2(ex2(e.x), ex2(e.y));
            const uint64_t p2 = mul2(pair(p.x, p.y), pair(kTlLift, kTlLift));
            sum = add2(sum, p2);
            // the first term is cut to binary16's 11 bits, so that the rest is exact
            p = unpair(p2);
            const float2 c1 = make_float2(__uint_as_float(__float_as_uint(p.x) & 0xFFFFE000u),
                                          __uint_as_float(__float_as_uint(p.y) & 0xFFFFE000u));
            const float2 r = unpair(fma2(pair(c1.x, c1.y), pair(-1.0f, -1.0f), p2));
            hi[k >> 1] = pack_half2(c1.x, c1.y);
            lo[k >> 1] = pack_half2(r.x, r.y);
          }
          tmem_st8(s_at + 32 * b + 16 * h, hi);
          tmem_st8(s_at + 32 * b + 16 * h + 8, lo);
        }
        const float2 s = unpair(sum);
        l = fmaf(s.x + s.y, sh.sc[i & 3][b][2], l);
      }
      if (has_tail && i == nt - 1 && lim >= 32 * closed + sh.bad) l = __int_as_float(0x7fc00000);
      tmem_st_wait();
      fence_before();
      bar_arrive(bar(sh.w_ready[w]));
      // this tile's O, while the tensor cores go on
      if (!bar_wait_warp(bar(sh.o_done[w]), (i >> 1) & 1, given_up)) break;
      fence_after();
      const uint64_t shrink2 = pair(shrink, shrink);
      tmem_ld16(o_at, v[0]);
#pragma unroll
      for (int h = 0; h < 8; ++h) {
        uint32_t (&x)[16] = v[h & 1];
        tmem_wait(x);
        if (h < 7) tmem_ld16(o_at + 16 * (h + 1), v[(h + 1) & 1]);
#pragma unroll
        for (int k = 0; k < 16; k += 2)
          acc[8 * h + (k >> 1)] = fma2(acc[8 * h + (k >> 1)], shrink2,
                                       pair(__uint_as_float(x[k]), __uint_as_float(x[k + 1])));
      }
    }
    // the two lanes of work meet in what was K's (and, for the last rows, V's) memory
    float* red = reinterpret_cast<float*>(k_buf) + (size_t)row * (kHd + 4);
    sh.m[w][row] = m;
    sh.l[w][row] = l;
    rows_sync();
    const float l0 = sh.l[0][row], l1 = sh.l[1][row];
    const float M = fmaxf(sh.m[0][row], sh.m[1][row]);
    const float a0 = l0 == 0.0f ? 0.0f : ex2(sh.m[0][row] - M);
    const float a1 = l1 == 0.0f ? 0.0f : ex2(sh.m[1][row] - M);
    if (w == 1) {
#pragma unroll
      for (int d = 0; d < kHd / 2; d += 2) {
        const float2 x = unpair(acc[d]), y = unpair(acc[d + 1]);
        *reinterpret_cast<float4*>(red + 2 * d) = make_float4(x.x * a1, x.y * a1, y.x * a1, y.y * a1);
      }
    }
    rows_sync();
    if (w == 0) {
      const float nan = __int_as_float(0x7fc00000);
      const float L = *given_up ? nan : l0 * a0 + l1 * a1;
      float* part = a.part + (slot + chunk) * rows_part(kTlRows);
      float* out = part + (size_t)row * kHd;
      float f = 1.0f;
      if (nact == 1) {
        const int r = min(grow, nrows - 1);
        out = a.ctx + ((size_t)(r / a.group) * a.nq + (size_t)kvh * a.group + r % a.group) * kHd;
        f = a.pos0 + grow / a.group >= held ? nan : 1.0f / L;
      }
#pragma unroll
      for (int d = 0; d < kHd / 2; d += 2) {
        const float2 x = unpair(acc[d]), y = unpair(acc[d + 1]);
        const float4 o = *reinterpret_cast<const float4*>(red + 2 * d);
        if (nact > 1 || grow < nrows)
          *reinterpret_cast<float4*>(out + 2 * d) =
              make_float4((x.x * a0 + o.x) * f, (x.y * a0 + o.y) * f, (y.x * a0 + o.z) * f,
                          (y.y * a0 + o.w) * f);
      }
      if (nact > 1) {
        *reinterpret_cast<float2*>(part + kTlRows * kHd + 2 * row) = make_float2(M, L);
        __threadfence();
      }
    }
  } else if (warp < 12) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kTlRegsConv));
    // a warp per block of the tile
    const int cw = warp - 8, g = lane >> 2, t = lane & 3;
    const uint8_t* codes = c.codes + (size_t)kvh * c.nblk * 2 * kQ8Codes + 16 * lane;
    const float2* scales = reinterpret_cast<const float2*>(c.scales) + (size_t)kvh * c.nblk;
    const float* open = c.tail + (size_t)kvh * 2 * kQ8Codes;
    const int nopen = held - closed * kQ8Blk;
    // a lane's 16-byte units of a block pass through its own bytes of the staging area
    uint8_t* stage = smem + 6 * kTlTile + cw * 2 * kQ8Codes + 16 * lane;
    const uint32_t stage_s = (uint32_t)__cvta_generic_to_shared(stage);
    float2 sc = make_float2(1.f, 1.f), sc_next;
    auto live = [&](int i) { return i < nt && b0 + 4 * i + cw < min(b1, nb); };
    auto fetch = [&](int i, int which) {
      if (live(i)) {
        const uint8_t* src = codes + ((size_t)(b0 + 4 * i + cw) * 2 + which) * kQ8Codes;
#pragma unroll
        for (int u = 0; u < 8; ++u)
          asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                       :: "r"(stage_s + which * kQ8Codes + 512 * u), "l"(src + 512 * u) : "memory");
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto put_k = [&](uint8_t* to, int j, int h, int s, uint32_t x, uint32_t y) {
      // position 32 cw + 8 j + g, dims 64 h + 16 s + 4 t ..
      *reinterpret_cast<uint2*>(to + h * kTlHalf + (32 * cw + 8 * j + g) * 128 +
                                (((2 * s + (t >> 1)) ^ g) << 4) + (t & 1) * 8) = make_uint2(x, y);
    };
    auto put_v = [&](uint8_t* to, int u, int h, int k, int j, uint32_t x) {
      // dim 16 u + 8 h + g, positions 32 cw + 16 k + 8 j + 2 t ..
      *reinterpret_cast<uint32_t*>(to + (cw >> 1) * kTlHalf + (16 * u + 8 * h + g) * 128 +
                                   (((4 * (cw & 1) + 2 * k + j) ^ g) << 4) + 4 * t) = x;
    };
    // the open rows' values in one of their two terms (second: 1)
    float lk = 1.0f, lv = 1.0f;
    auto term = [&](float x0, float x1, float lift, int second) {
      x0 = fabsf(x0) < INFINITY ? x0 * lift : 0.0f;
      x1 = fabsf(x1) < INFINITY ? x1 * lift : 0.0f;
      uint32_t hi, lo;
      split_half2(x0, x1, &hi, &lo);
      return second ? lo : hi;
    };
    auto open_k = [&](uint8_t* to, int second) {
#pragma unroll 1
      for (int j = 0; j < 4; ++j)
#pragma unroll 1
        for (int hs = 0; hs < 8; ++hs) {
          const int r = 8 * j + g;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (r < nopen) x = __ldg(reinterpret_cast<const float4*>(open + r * kHd + 16 * hs + 4 * t));
          put_k(to, j, hs >> 2, hs & 3, term(x.x, x.y, lk, second), term(x.z, x.w, lk, second));
        }
    };
    auto open_v = [&](uint8_t* to, int second) {
#pragma unroll 1
      for (int uh = 0; uh < 16; ++uh)
#pragma unroll
        for (int kj = 0; kj < 4; ++kj) {
          const int r = 8 * kj + 2 * t, d = 8 * uh + g;
          const float x0 = r < nopen ? __ldg(open + kQ8Codes + r * kHd + d) : 0.0f;
          const float x1 = r + 1 < nopen ? __ldg(open + kQ8Codes + (r + 1) * kHd + d) : 0.0f;
          put_v(to, uh >> 1, uh & 1, kj >> 1, kj & 1, term(x0, x1, lv, second));
        }
    };
    auto none_k = [&](uint8_t* to) {
#pragma unroll 1
      for (int u = 0; u < 32; ++u) put_k(to, u >> 3, (u >> 2) & 1, u & 3, 0u, 0u);
    };
    auto none_v = [&](uint8_t* to) {
#pragma unroll 1
      for (int u = 0; u < 64; ++u) put_v(to, u >> 3, (u >> 2) & 1, (u >> 1) & 1, u & 1, 0u);
    };
    fetch(0, 0);
    fetch(0, 1);
    sc_next = live(0) ? __ldg(scales + b0 + cw) : sc;
    for (int i = 0; i < nt; ++i) {
      const int s = i & 1;
      uint8_t* kt = k_buf + s * kTlTile;
      uint8_t* vt = v_buf + s * kTlTile;
      const bool two = has_tail && i == nt - 1;             // this tile ends with the open block
      const bool mine = two && b0 + 4 * i + cw == closed;   // and this warp has it
      sc = sc_next;
      sc_next = live(i + 1) ? __ldg(scales + b0 + 4 * (i + 1) + cw) : make_float2(1.f, 1.f);
      if (i >= 2 && !bar_wait_warp(bar(sh.s_ready[s]), ((i - 2) >> 1) & 1, given_up)) break;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      if (mine) {
        float mk = 0.0f, mv = 0.0f;
        for (int r = 0; r < nopen; ++r) {
          const float4 x = __ldg(reinterpret_cast<const float4*>(open + r * kHd) + lane);
          const float4 y = __ldg(reinterpret_cast<const float4*>(open + kQ8Codes + r * kHd) + lane);
          const float e[8] = {fabsf(x.x), fabsf(x.y), fabsf(x.z), fabsf(x.w),
                              fabsf(y.x), fabsf(y.y), fabsf(y.z), fabsf(y.w)};
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            if (!(e[k] < INFINITY)) atomicMin(&sh.bad, r);
            else if (k < 4) mk = fmaxf(mk, e[k]);
            else mv = fmaxf(mv, e[k]);
          }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          mk = fmaxf(mk, __shfl_xor_sync(0xFFFFFFFFu, mk, o));
          mv = fmaxf(mv, __shfl_xor_sync(0xFFFFFFFFu, mv, o));
        }
        lk = q8_lift(mk);
        // values up to 2^10: their scale is then near that of coded values, which is what a
        // weight's precision goes by
        lv = q8_lift(mv) * 0.0625f;
        sc = make_float2(1.0f / lk, 1.0f / lv);
        open_k(kt, 0);
      } else if (!live(i)) {                    // past the chunk's last block
        none_k(kt);
      } else {
#pragma unroll 2
        for (int u = 0; u < 8; ++u) {
          const uint4 y4 = *reinterpret_cast<const uint4*>(stage + 512 * u);
          const uint32_t x[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            uint32_t y0, y1;
            q8_halves(x[k], &y0, &y1);
            put_k(kt, u >> 1, u & 1, k, y0, y1);
          }
        }
      }
      if (lane == 0) {
        // a scale under 2^-120 counts as that, so that its reciprocal is a number; a NaN stays
        const float sv = sc.y < 0x1p-120f ? 0x1p-120f : sc.y;
        sh.sc[i & 3][cw][0] = sc.x;
        sh.sc[i & 3][cw][1] = log2f(sv);
        sh.sc[i & 3][cw][2] = sv == sv ? 1.0f / sv : 0.0f;
      }
      fence_async();
      bar_arrive(bar(sh.full_k[s]));
      fetch(i + 1, 0);
      if (two) {
        if (!bar_wait_warp(bar(sh.k_free), 0, given_up)) break;
        if (mine) open_k(kt, 1);
        else none_k(kt);
        fence_async();
        bar_arrive(bar(sh.full_k[s]));
      }
      if (i >= 2 && !bar_wait_warp(bar(sh.o_done[s]), ((i - 2) >> 1) & 1, given_up)) break;
      asm volatile("cp.async.wait_group 1;" ::: "memory");
      if (mine) {
        open_v(vt, 0);
      } else if (!live(i)) {
        none_v(vt);
      } else {
#pragma unroll 2
        for (int u = 0; u < 8; ++u) {
          const uint4 y4 = *reinterpret_cast<const uint4*>(stage + kQ8Codes + 512 * u);
          const uint32_t x[4] = {y4.x, y4.y, y4.z, y4.w};
#pragma unroll
          for (int k = 0; k < 4; ++k) {                     // word 2 h + k
            uint32_t y0, y1;
            q8_halves(x[k], &y0, &y1);
            put_v(vt, u, k >> 1, k & 1, 0, y0);
            put_v(vt, u, k >> 1, k & 1, 1, y1);
          }
        }
      }
      fence_async();
      bar_arrive(bar(sh.full_v[s]));
      fetch(i + 1, 1);
      if (two) {
        if (!bar_wait_warp(bar(sh.v_free), 0, given_up)) break;
        if (mine) open_v(vt, 1);
        else none_v(vt);
        fence_async();
        bar_arrive(bar(sh.full_v[s]));
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kTlRegsIssue));
  }
  if (warp == 12) {
    const uint32_t leader = elect_one();
    const uint64_t qh = smem_desc(sm), ql = smem_desc(sm + kTlTile);
    // step k of 16 along the inner dimension: the half it is in, then 32 bytes each
    auto step = [](int k) { return (uint64_t)(((k >> 2) * kTlHalf + (k & 3) * 32) >> 4); };
    bool ok = true;
    auto product_s = [&](int i) {
      const int s = i & 1;
      const uint64_t kd = smem_desc(sm + (2 + s) * kTlTile);
      const uint32_t d = tmem + 128 * s;
      ok = ok && bar_wait_warp(bar(sh.full_k[s]), (i >> 1) & 1, given_up);
      if (!ok) return;
      fence_after();
#pragma unroll
      for (int k = 0; k < 8; ++k) mma_ss(d, ql + step(k), kd + step(k), k > 0, leader);
#pragma unroll
      for (int k = 0; k < 8; ++k) mma_ss(d, qh + step(k), kd + step(k), true, leader);
      if (has_tail && i == nt - 1) {
        mma_commit(bar(sh.k_free), leader);
        ok = bar_wait_warp(bar(sh.full_k[s]), ((i >> 1) + 1) & 1, given_up);
        if (!ok) return;
        fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k) mma_ss(d, qh + step(k), kd + step(k), true, leader);
      }
      mma_commit(bar(sh.s_ready[s]), leader);
    };
    auto product_o = [&](int i) {
      const int s = i & 1;
      const uint64_t vd = smem_desc(sm + (4 + s) * kTlTile);
      const uint32_t p = tmem + 128 * s, d = tmem + 256 + 128 * s;
      ok = ok && bar_wait_warp(bar(sh.full_v[s]), (i >> 1) & 1, given_up);
      ok = ok && bar_wait_warp(bar(sh.w_ready[s]), (i >> 1) & 1, given_up);
      if (!ok) return;
      fence_after();
      // the weights of 16 positions are 8 columns of first terms, then 8 of second ones
#pragma unroll
      for (int k = 0; k < 8; ++k) mma_ts(d, p + 16 * k + 8, vd + step(k), k > 0, leader);
#pragma unroll
      for (int k = 0; k < 8; ++k) mma_ts(d, p + 16 * k, vd + step(k), true, leader);
      if (has_tail && i == nt - 1) {
        mma_commit(bar(sh.v_free), leader);
        ok = bar_wait_warp(bar(sh.full_v[s]), ((i >> 1) + 1) & 1, given_up);
        if (!ok) return;
        fence_after();
#pragma unroll
        for (int k = 0; k < 8; ++k) mma_ts(d, p + 16 * k, vd + step(k), true, leader);
      }
      mma_commit(bar(sh.o_done[s]), leader);
    };
    if (nt > 0) product_s(0);
    if (nt > 1) product_s(1);
    for (int i = 0; i < nt && ok; ++i) {
      product_o(i);
      if (i + 2 < nt) product_s(i + 2);
    }
    if (!ok) {                                    // what was issued ends before the memory goes
      int no = 0;
      mma_commit(bar(sh.drain), leader);
      bar_wait_warp(bar(sh.drain), 0, &no);
    }
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == 12) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem));
  }
  if (nact == 1) return;
  if (threadIdx.x == 0) {
    unsigned* tk = a.ticket + (size_t)kvh * ntile + tile;
    sh.last = atomicAdd(tk, 1u) == (unsigned)nact - 1;
    if (sh.last) *tk = 0;
  }
  __syncthreads();
  if (!sh.last) return;
  __threadfence();
  rows_join<kTlRows>(a, kvh, slot, nact, row0, nrows, held);
}

}  // namespace

int attn_tile_q8_launch(const RowsArgs& a, const KvQ8& c, unsigned tiles, unsigned nkv,
                        cudaStream_t st) {
  const int rc = smem_attr((const void*)k_attn_tile_q8, kTlSmem);
  if (rc) return rc;
  // a split of more registers than the kernel starts with would wait for good
  static const int regs = [] {
    cudaFuncAttributes f{};
    return cudaFuncGetAttributes(&f, k_attn_tile_q8) == cudaSuccess ? f.numRegs : 0;
  }();
  HV_REQUIRE(regs * kTlThreads >= kTlRegsSum, HV_E_UNSUPPORTED,
             "k_attn_tile_q8: built with %d registers", regs);
  k_attn_tile_q8<<<dim3(tiles * a.chunks, nkv), kTlThreads, kTlSmem, st>>>(a, c);
  HV_LAUNCHED("k_attn_tile_q8");
}

}  // namespace hv
