// Attention of a long run of query rows over the 8-bit cache, on the fifth-generation tensor
// cores. The mathematics is k_attn_q8.cu's: f32 factors as two binary16 terms, codes exact.
//
// A CTA has 128 (token, head) rows of a kv head and a chunk of its positions, 128 positions
// (four blocks) to a tile, tiles in turn to two lanes of work w = tile mod 2:
//   warps 12-15  turn the codes of a tile into binary16 in shared memory: K [position][dim] and
//                V transposed [dim][position], 128-byte swizzled rows
//   warps 0-3    (lane of work 0) and 4-7 (1): a thread has one row of S_w; it writes the row's
//                weights over S_w, two binary16 terms in place of 16 sums; then warp 0 (4),
//                which has nothing to do until S_w is there again, issues O = wl V + wh V and
//                the next S_w = ql K^T + qh K^T
//   warps 8-11   a thread adds its row of O to 128 sums in registers
// so while one lane of work is at its weights the tensor cores run the other's products. Each
// lane has its own maximum; the sums go by the larger of the two. The queries and the weights
// are the operand in tensor memory (S twice, O, and the queries fill its 512 columns), so that
// shared memory, which would bound the products if it held both operands, is left to K and V.
//
// The order of dims in a K row (and of the queries) and that of positions in a tile are free as
// long as both operands agree. They are such that a lane's codes of one 16-byte unit become 16
// or 32 adjacent bytes, and that eight lanes' 16-byte stores meet no bank twice: dim
// 64 h + 16 s + 4 t + e stands at 64 h + 16 t + 4 s + e, position 8 j + 2 t + e of block c of
// the tile at 64 (c / 2) + 16 t + 8 (c mod 2) + 2 j + e.
//
// The tensor cores cut their f32 sums instead of rounding them, once for every 16 positions:
// kept in tensor memory over 64 tiles, O was 1.8e-5 too small. So O is of one tile, and the
// small terms go first, while the sums are small.
//
// The scale of a V block has to multiply its weights here, as a tile's sum stays in tensor
// memory: a weight enters as w s_v, that is 2^(x + log2 s_v), and the maximum that the row
// keeps is that of these products, so that a block with a large scale that the row hardly
// attends to does not cost the others precision; the sum of the weights adds w s_v / s_v.
// Weights stand as 2^15 times themselves, exact to 2^-40 of the row's largest w s_v.
// Where a block's largest is under 2^-64 of that, its weights would be lost to the sum too: they
// are added up apart, without the scale, by a maximum of their own, and leave the tile's scores. So
// do those of a block of which the row sees no V but zeros, whose w s_v stands for nothing. Only
// chunks whose scales are 2^30 apart, or 1 as those of zeros are, and tiles where a row sees part of
// a block look for them. At a chunk's end all goes by one power of two of the sum of the weights.
// The open block's f32 rows are two binary16 terms: after the tile's products with the first
// term, the same buffer holds the second one (zero elsewhere) for one product more. Each of its
// rows has a power of two of its own, so that no row, least of all one that a query does not see,
// takes bits from another: the scores become exponents of w with a K row's taken back, which are
// added up with the weights apart, and then those of w v with what a V row's lacks.
//
// Every wait is bounded: one that runs out ends the CTA, whose rows are then NaN.
//
// Bound by the tensor cores and by what feeds them: with two terms on one side of each product,
// 256 tokens of 64 heads over 16384 positions take 265 us and 256 of 32 heads over 4096 45 us (239
// and 43 in a graph), 1.03 and 0.74 PFLOP/s of issued products, 62% and 45% of a large library
// product's rate. A tile's weights (a pass for the maximum and one for the exponents over 128
// columns a thread) stand between two of its lane's products; two lanes of work hide the one behind
// the other, but not the ends of a chunk.
#include <type_traits>

#include "attn_q8.cuh"
#include "attn_q8_rows.h"
#include "hv_internal.h"

namespace hv {
namespace {

constexpr int kTlRows = 128;                    // rows of a CTA and positions of a tile
constexpr int kTlThreads = 512;
constexpr int kTlHalf = 128 * 128;              // bytes of 128 rows of 64 halves
constexpr int kTlTile = 2 * kTlHalf;            // bytes of a 128 x 128 binary16 tile
constexpr int kTlLine = kHd + 4;               // floats from row to row on their way in and out
constexpr float kTlLift = 32768.0f;             // 2^15
constexpr float kTlDrop = 0x1p-20f;             // of the sum of weights: room for 2^20 of them over
                                                // a scale of 2^-110
constexpr int kTlNone = 1 << 29;
constexpr float kTlApart = -64.0f;              // log2 of a block's largest w s_v over the row's
constexpr float kTlFar = 30.0f;                 // exponents between scales: so that without `far` all
                                                // weights of note are within kTlApart
constexpr uint32_t kTlColO = 256, kTlColQ = 384;   // tensor memory: S twice, O, qh, ql
// registers per thread: 128 at launch, then dealt out anew
constexpr int kTlRegs = 128, kTlRegsRow = 112, kTlRegsSum = 184, kTlRegsConv = 104;
static_assert(2 * kTlRegsRow + kTlRegsSum + kTlRegsConv <= 4 * kTlRegs, "registers");

// kind::f16 with f32 sums, 128 x 128, both operands with the inner dimension contiguous
constexpr uint32_t kTlDesc = (1u << 4) | ((128u >> 3) << 17) | ((128u >> 4) << 24);

HV_DEV uint64_t smem_desc(uint32_t addr) {      // 128-byte swizzle, 1024 bytes per 8 rows
  return (uint64_t)((addr >> 4) & 0x3FFF) | (1ull << 16) | (64ull << 32) | (1ull << 46) |
         (2ull << 61);
}
// One lane of a whole warp issues: the warp stays together, so that the descriptors are uniform
// registers, which the instruction wants (in a branch of one lane it took 190 cycles to issue
// a product that runs for 64).
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
// Columns of this thread's row: begun here, in hand after tmem_wait. One load is under way
// while the columns before it are worked on.
HV_DEV void tmem_ld32(uint32_t at, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : HV_R4(v, 0), HV_R4(v, 4), HV_R4(v, 8), HV_R4(v, 12), HV_R4(v, 16), HV_R4(v, 20),
        HV_R4(v, 24), HV_R4(v, 28)
      : "r"(at) : "memory");
}
HV_DEV void tmem_wait(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : HV_P4(v, 0), HV_P4(v, 4), HV_P4(v, 8), HV_P4(v, 12), HV_P4(v, 16), HV_P4(v, 20),
                 HV_P4(v, 24), HV_P4(v, 28) :: "memory");
}
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
HV_DEV void tmem_ld8(uint32_t at, uint32_t (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : HV_R4(v, 0), HV_R4(v, 4) : "r"(at) : "memory");
}
HV_DEV void tmem_wait(uint32_t (&v)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : HV_P4(v, 0), HV_P4(v, 4) :: "memory");
}
HV_DEV void tmem_st8(uint32_t at, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};"
               :: "r"(at), HV_W4(v, 0), HV_W4(v, 4) : "memory");
}
HV_DEV void tmem_st16(uint32_t at, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      :: "r"(at), HV_W4(v, 0), HV_W4(v, 4), HV_W4(v, 8), HV_W4(v, 12) : "memory");
}
HV_DEV void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

HV_DEV void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" :: "r"(bar) : "memory");
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
  unsigned long long full_k[2], full_v[2], s_ready[2], w_ready[2], o_done[2];
  unsigned long long o_free, k_free, v_free, drain[2];
  float sc[4][4][4];             // of the last four tiles' blocks: s_k, log2 s_v, 1 / s_v
  int first[4][4];               // first position with a V that is not zero, where that is looked for
  float top[4][kTlRows];         // of the last four tiles: what their weights are relative to
  float m[2][kTlRows], l[2][kTlRows];
  float n[2][kTlRows], k[2][kTlRows];     // of the weights apart: maximum, sum
  float ml[kTlRows][2];          // of the rows' sums, where another CTA of the cluster adds them up
  uint32_t tmem;
  float open_max[2][kQ8Blk];     // of the open rows: largest |K|, |V|; what takes K's power of two
  float open_k[kQ8Blk], open_v[kQ8Blk];   // back but for the block's, the exponent that V lacks
  int bad;                       // first open row with a value that is not finite
  int given_up;
  int far;                       // scales of V too far apart for one sum of weights
};
constexpr int kTlSmem = 4 * kTlTile + kTlRows * kTlLine * 4 + (int)sizeof(TlShared);   // K, V twice

template <bool kMeet>
__global__ void __launch_bounds__(kTlThreads, 1) k_attn_tile_q8(RowsArgs a, KvQ8 c) {
  extern __shared__ __align__(1024) uint8_t smem[];
  TlShared& sh = *reinterpret_cast<TlShared*>(smem + 4 * kTlTile + kTlRows * kTlLine * 4);
  const int warp = __shfl_sync(0xFFFFFFFFu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  const int kvh = blockIdx.y, tile = blockIdx.x / a.chunks, chunk = blockIdx.x % a.chunks;
  const int nrows = a.ntok * a.group, row0 = tile * kTlRows;
  const RowsSpan sp = rows_span(a, c, kvh, row0, kTlRows, kTileLeast);
  const int held = sp.held, closed = sp.closed, nb = sp.nb, items = sp.items, nact = sp.nact;
  if (chunk >= nact) {
    if (kMeet) { cluster_sync(); cluster_sync(); }
    return;
  }
  const int b0 = (int)((long long)items * chunk / nact);
  const int b1 = (int)((long long)items * (chunk + 1) / nact);
  const int nt = (b1 - b0 + 3) / 4;
  const bool has_tail = items > nb && b1 == items;

  const uint32_t sm = (uint32_t)__cvta_generic_to_shared(smem);
  uint8_t* k_buf = smem;                          // two tiles, then V's two
  uint8_t* v_buf = smem + 2 * kTlTile;
  auto bar = [](const unsigned long long& b) { return (uint32_t)__cvta_generic_to_shared(&b); };

  if (threadIdx.x == 0) {
    for (int i = 0; i < 2; ++i) {
      bar_init(bar(sh.full_k[i]), 128);
      bar_init(bar(sh.full_v[i]), 128);
      bar_init(bar(sh.s_ready[i]), 1);
      bar_init(bar(sh.w_ready[i]), 128);
      bar_init(bar(sh.o_done[i]), 1);
    }
    bar_init(bar(sh.o_free), 128);
    bar_init(bar(sh.k_free), 1);
    bar_init(bar(sh.v_free), 1);
    bar_init(bar(sh.drain[0]), 1);
    bar_init(bar(sh.drain[1]), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    sh.bad = kQ8Blk;
    sh.far = 0;
    sh.given_up = (sm & 1023) != 0;               // the swizzle goes by addresses
  }
  if (warp == 15) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;"
                 :: "r"((uint32_t)__cvta_generic_to_shared(&sh.tmem)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = sh.tmem;
  volatile int* given_up = &sh.given_up;
  const int w = warp >> 2, row = threadIdx.x & 127, grow = row0 + row;
  const int ntile = gridDim.x / a.chunks;
  const size_t slot = ((size_t)kvh * ntile + tile) * a.chunks;
  float* lines = reinterpret_cast<float*>(smem + 4 * kTlTile);    // [row][kTlLine]
  auto rows_sync = [] { asm volatile("bar.sync 3, 256;" ::: "memory"); };
  // the rows' sums, once they stand in `lines`: to ctx, or to this chunk's part of the scratch (a
  // cluster's stay where they are)
  auto rows_out = [&] {
    if (kMeet && nact > 1) return;
    asm volatile("bar.sync 2, 384;" ::: "memory");
    float4* part = reinterpret_cast<float4*>(a.part + (slot + chunk) * rows_part(kTlRows));
#pragma unroll 4
    for (int r = warp; r < kTlRows; r += 12) {
      const float4 x = *reinterpret_cast<const float4*>(lines + (size_t)r * kTlLine + 4 * lane);
      const int gr = row0 + r, tok = gr / a.group;
      if (nact > 1)
        part[r * (kHd / 4) + lane] = x;
      else if (gr < nrows)
        reinterpret_cast<float4*>(a.ctx + ((size_t)tok * a.nq + (size_t)kvh * a.group + gr - tok * a.group) * kHd)[lane] = x;
    }
  };
  if (warp < 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kTlRegsRow));
    auto exponent = [](float x) { return (int)(__float_as_uint(x) >> 23) - 127; };
    int first_e = 0;
    // The queries in two terms, a row per thread (whole lines at a time through shared memory):
    // the first ones from warps 0-3, the second from 4-7. They take the scale's sign, so that
    // the largest sum of products is the largest exponent.
    {
      // a warp takes rows warp, warp + 8, ..., all of them under way at once
      const uint32_t to = sm + 4 * kTlTile + 16 * lane;
#pragma unroll 4
      for (int r = warp; r < kTlRows; r += 8) {
        const int gr = min(row0 + r, nrows - 1), tok = gr / a.group;
        const float* src = a.q + ((size_t)tok * a.nq + (size_t)kvh * a.group + gr - tok * a.group) * kHd + 4 * lane;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                     :: "r"(to + r * kTlLine * 4), "l"(src) : "memory");
      }
      // meanwhile: are there scales of V far from the chunk's first, or one that may be of zeros?
      const float2* scales = reinterpret_cast<const float2*>(c.scales) + (size_t)kvh * c.nblk;
      const int end = min(b1, nb);
      if (b0 < end) first_e = exponent(__ldg(scales + b0).y);
      for (int b = b0 + threadIdx.x; b < end; b += 256) {
        const float s = __ldg(scales + b).y;
        if (s == 1.0f || abs(exponent(s) - first_e) > (int)kTlFar) sh.far = 1;
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
    }
    const float qscale = __ldg(a.scale) * kLog2e;
    rows_sync();
    const bool far = sh.far;
    float qs;
    {
      // each of a row's two threads looks over half of it
      const float4* q = reinterpret_cast<const float4*>(lines + (size_t)row * kTlLine);
      float amax = 0.0f;
#pragma unroll 4
      for (int d = 0; d < kHd / 8; ++d) {
        const float4 x = q[(kHd / 8) * w + d];
        amax = fmaxf(fmaxf(amax, fmaxf(fabsf(x.x), fabsf(x.y))), fmaxf(fabsf(x.z), fabsf(x.w)));
      }
      sh.m[w][row] = amax;
      rows_sync();
      amax = fmaxf(amax, sh.m[1 - w][row]);
      const float lift = copysignf(q8_lift(amax), qscale);
      qs = qscale / lift;
      const uint32_t to = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + kTlColQ + 64 * w;
      // dims in the order of K's tiles: 64 h + 16 s + 4 t + e stands at 64 h + 16 t + 4 s + e
#pragma unroll 1
      for (int d = 0; d < kHd / 4; d += 8) {
        uint32_t v[16];
#pragma unroll
        for (int k = 0; k < 8; ++k) {
          const float4 x = q[(d & 16) + 4 * (k & 3) + ((d >> 2) & 2) + (k >> 2)];
          uint32_t h0, h1, l0, l1;
          split_half2(x.x * lift, x.y * lift, &h0, &l0);
          split_half2(x.z * lift, x.w * lift, &h1, &l1);
          v[2 * k] = w ? l0 : h0;
          v[2 * k + 1] = w ? l1 : h1;
        }
        tmem_st16(to + 2 * d, v);
      }
      tmem_st_wait();
    }
    fence_before();
    rows_sync();
    fence_after();
    float m = -INFINITY, l = 0.0f;                // of this thread's row
    float n = -INFINITY, apart = 0.0f;            // maximum and sum of the weights apart
    const uint32_t s_at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + 128 * w;
    const int lim = grow < nrows ? min(min(a.pos0 + grow / a.group, held - 1), 32 * b1 - 1) : -1;
    const uint32_t leader = elect_one();
    const uint32_t qh = tmem + kTlColQ, ql = qh + 64;
    // step k of 16 along the inner dimension: the half it is in, then 32 bytes each
    auto step = [](int k) { return (uint64_t)(((k >> 2) * kTlHalf + (k & 3) * 32) >> 4); };
    bool ok = true;
    // the small terms first; with the open block, its values' second terms last
    auto product_s = [&](int i) {
      const int s = i & 1, passes = has_tail && i == nt - 1 ? 3 : 2;
      const uint64_t kd = smem_desc(sm + s * kTlTile);
      const uint32_t d = tmem + 128 * s;
      ok = ok && bar_wait_warp(bar(sh.full_k[s]), (i >> 1) & 1, given_up);
      fence_after();
#pragma unroll 1
      for (int pass = 0; pass < passes && ok; ++pass) {
        if (pass == 2) {
          mma_commit(bar(sh.k_free), leader);
          ok = bar_wait_warp(bar(sh.full_k[s]), ((i >> 1) + 1) & 1, given_up);
          if (!ok) break;
          fence_after();
        }
        const uint32_t q = pass ? qh : ql;
#pragma unroll
        for (int k = 0; k < 8; ++k) mma_ts(d, q + 8 * k, kd + step(k), pass > 0 || k > 0, leader);
      }
      mma_commit(bar(sh.s_ready[s]), leader);
    };
    auto product_o = [&](int i) {
      const int s = i & 1, passes = has_tail && i == nt - 1 ? 3 : 2;
      const uint64_t vd = smem_desc(sm + (2 + s) * kTlTile);
      const uint32_t d = tmem + kTlColO;
      ok = ok && bar_wait_warp(bar(sh.full_v[s]), (i >> 1) & 1, given_up);
      ok = ok && bar_wait_warp(bar(sh.w_ready[s]), (i >> 1) & 1, given_up);
      if (i > 0) ok = ok && bar_wait_warp(bar(sh.o_free), (i - 1) & 1, given_up);
      fence_after();
#pragma unroll 1
      for (int pass = 0; pass < passes && ok; ++pass) {
        if (pass == 2) {
          mma_commit(bar(sh.v_free), leader);
          ok = bar_wait_warp(bar(sh.full_v[s]), ((i >> 1) + 1) & 1, given_up);
          if (!ok) break;
          fence_after();
        }
        // the weights of 16 positions are 8 columns of first terms, then 8 of second ones
        const uint32_t wt = tmem + 128 * s + (pass ? 0 : 8);
#pragma unroll
        for (int k = 0; k < 8; ++k) mma_ts(d, wt + 16 * k, vd + step(k), pass > 0 || k > 0, leader);
      }
      mma_commit(bar(sh.o_done[s]), leader);
    };
    const bool issues = (warp & 3) == 0;
    // block b of the tile: its columns by eights, its largest sum of products
    auto block_at = [&](int b, int h) { return s_at + 64 * (b >> 1) + 16 * h + 8 * (b & 1); };
    auto block_max = [&](int b) {
      float big = -INFINITY;
#pragma unroll 1
      for (int h = 0; h < 4; ++h) {
        uint32_t x[8];
        tmem_ld8(block_at(b, h), x);
        tmem_wait(x);
#pragma unroll
        for (int k = 0; k < 8; ++k) big = fmaxf(big, __uint_as_float(x[k]));
      }
      return big;
    };
    // The weights of tile i. Most tiles are seen whole by every row and have nothing to look for:
    // those have a form of their own (`whole`), which the rest would slow by their code alone
    // (256 rows at 16128 in a graph 239 us with it, 250 without).
    auto weights = [&](int i, auto whole_form) {
      constexpr bool whole = decltype(whole_form)::value;
      const int see0 = lim - 32 * (b0 + 4 * i);            // positions 0 .. see0 are seen
      const bool all = whole || __all_sync(0xFFFFFFFFu, see0 >= kTlRows - 1);
      const float (&sc)[4][4] = sh.sc[i & 3];
      const int (&first)[4] = sh.first[i & 3];
      bool look = !whole && far;
      if (!all) {
        // columns of positions that the row does not see become -infinity
#pragma unroll 1
        for (int h = 0; h < 8; ++h) {
          uint32_t x[16];
          tmem_ld16(s_at + 16 * h, x);
          tmem_wait(x);
          const int see = see0 - 64 * (h >> 2) - 2 * (h & 3);
#pragma unroll
          for (int k = 0; k < 16; ++k) {
            const int r = 32 * (k >> 3) + 8 * ((k & 7) >> 1) + (k & 1);
            x[k] = r <= see ? x[k] : 0xFF800000u;
          }
          tmem_st16(s_at + 16 * h, x);
        }
        tmem_st_wait();
        bool zeros = false;                                 // are they all that the row sees of a block?
#pragma unroll
        for (int b = 0; b < 4; ++b) zeros |= see0 >= 32 * b && see0 < 32 * b + first[b];
        look |= __any_sync(0xFFFFFFFFu, zeros) != 0;
      }
      // The largest exponent of the row in this tile. Here and below loops stay as rolled as
      // the two buffers allow: the code of all roles has to fit the instruction cache.
      uint32_t v[2][32];
      const bool tail = !whole && has_tail && i == nt - 1;
      const int ob = tail ? (nb - b0) & 3 : -1;             // the open block
      if (tail) {
        const float f = sc[ob][3] * qs;
        float most = -INFINITY;
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
          uint32_t x[8];
          float big = n;
          tmem_ld8(block_at(ob, h), x);
          tmem_wait(x);
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = 8 * (k >> 1) + 2 * h + (k & 1);
            const float y = r <= see0 - 32 * ob ? __uint_as_float(x[k]) * sh.open_k[r] * f : -INFINITY;
            x[k] = __float_as_uint(y);
            big = fmaxf(big, y);
          }
          const float n0 = big == -INFINITY ? 0.0f : big;
          apart *= n == -INFINITY ? 0.0f : ex2(n - n0);
          n = big;
#pragma unroll
          for (int k = 0; k < 8; ++k) {
            const int r = 8 * (k >> 1) + 2 * h + (k & 1);
            const float y = __uint_as_float(x[k]), v = sh.open_v[r];
            apart += ex2(y - n0);
            x[k] = __float_as_uint(y + v);
            most = fmaxf(most, v);
          }
          tmem_st8(block_at(ob, h), x);
        }
        tmem_st_wait();
        look |= most - (float)first_e > kTlFar;
      }
      float up = m;
      tmem_ld32(s_at, v[0]);
#pragma unroll 1
      for (int b = 0; b < 4; b += 2) {
        const int see = see0 - 32 * b;
        float mx[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t (&x)[32] = v[h];
          tmem_wait(x);
          if (h == 0 || b == 0) tmem_ld32(s_at + 32 * (b + h + 1), v[1 - h]);
#pragma unroll
          for (int k = 0; k < 32; ++k) {
            float& y = mx[((k >> 3) & 1) + 2 * (k & 1)];
            y = fmaxf(y, __uint_as_float(x[k]));
          }
        }
        const float qs0 = b == ob ? 1.0f : qs, qs1 = b + 1 == ob ? 1.0f : qs;
        if (whole || see >= 0) up = fmaxf(up, fmaf(fmaxf(mx[0], mx[2]), sc[b][0] * qs0, sc[b][1]));
        if (whole || see >= 32) up = fmaxf(up, fmaf(fmaxf(mx[1], mx[3]), sc[b + 1][0] * qs1, sc[b + 1][1]));
      }
      if (__builtin_expect(look, 0)) {                      // the largest again, without zeros
        up = m;
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          const float x = block_max(b);
          if (see0 >= 32 * b + first[b]) up = fmaxf(up, fmaf(x, sc[b][0] * (b == ob ? 1.0f : qs), sc[b][1]));
        }
      }
      const float fl = m == -INFINITY ? 0.0f : ex2(0.5f * (m - up));   // twice: 2^(m - up) may be 0
      l = l * fl * fl;
      m = up;
      sh.top[i & 3][row] = m;
      const float m0 = m == -INFINITY ? 0.0f : m;
      if (__builtin_expect(look, 0)) {
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          const float f = sc[b][0] * qs, x = block_max(b) * f;
          const int at = see0 - 32 * b;
          const bool go = b != ob && at >= 0 && (at < first[b] || x + sc[b][1] - m0 < kTlApart) && x > -INFINITY;
          if (go && x > n) {
            apart *= n == -INFINITY ? 0.0f : ex2(n - x);
            n = x;
          }
#pragma unroll 1
          for (int h = 0; h < 4; ++h) {
            uint32_t y[8];
            tmem_ld8(block_at(b, h), y);
            tmem_wait(y);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const bool out = go && y[k] != 0xFF800000u;
              apart += out ? ex2(fmaf(__uint_as_float(y[k]), f, -n)) : 0.0f;
              y[k] = out ? 0xFF800000u : y[k];
            }
            tmem_st8(block_at(b, h), y);
          }
        }
        tmem_st_wait();
      }
      uint32_t z[2][16];
      tmem_ld16(s_at, z[0]);
#pragma unroll 1
      for (int b = 0; b < 4; b += 2) {
        uint64_t f2[2], lv2[2], sum[2] = {0, 0};
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          // -inf f has to stay -inf: not with a scale of 0, nor with the scales (which may be
          // NaN) of a block that the row sees nothing of
          const bool seen = whole || see0 >= 32 * (b + e);
          float f = seen ? sc[b + e][0] * (b + e == ob ? 1.0f : qs) : 1.0f;
          f = f == 0.0f ? 1e-38f : f;
          const float add = seen ? sc[b + e][1] - m0 : 0.0f;
          f2[e] = pair(f, f);
          lv2[e] = pair(add, add);
        }
#pragma unroll 1
        for (int h = 0; h < 4; h += 2) {
#pragma unroll
          for (int g = 0; g < 2; ++g) {
            uint32_t (&x)[16] = z[g];
            tmem_wait(x);
            if (g == 0 || b + h < 4) tmem_ld16(s_at + 32 * b + 16 * (h + g) + 16, z[1 - g]);
            // 16 positions: 8 columns of first terms, 8 of second ones
            uint32_t wt[16];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
              const uint64_t s2 = pair(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1]));
              const float2 e = unpair(fma2(s2, f2[k >> 2], lv2[k >> 2]));
              const uint64_t p2 = mul2(pair(ex2(e.x), ex2(e.y)), pair(kTlLift, kTlLift));
              sum[k >> 2] = add2(sum[k >> 2], p2);
              // the first term is cut to binary16's 11 bits, so that the rest is exact
              const float2 p = unpair(p2);
              const float2 c1 = make_float2(__uint_as_float(__float_as_uint(p.x) & 0xFFFFE000u),
                                            __uint_as_float(__float_as_uint(p.y) & 0xFFFFE000u));
              const float2 r = unpair(fma2(pair(c1.x, c1.y), pair(-1.0f, -1.0f), p2));
              wt[k] = pack_half2(c1.x, c1.y);
              wt[8 + k] = pack_half2(r.x, r.y);
            }
            tmem_st16(s_at + 32 * b + 16 * (h + g), wt);
          }
        }
        const float2 s0 = unpair(sum[0]), s1 = unpair(sum[1]);
        l = fmaf(s0.x + s0.y, sc[b][2], l);
        l = fmaf(s1.x + s1.y, sc[b + 1][2], l);
      }
      if (tail && lim >= 32 * closed + sh.bad) l = __int_as_float(0x7fc00000);
      tmem_st_wait();
      fence_before();
      bar_arrive(bar(sh.w_ready[w]));
    };
    const int whole_end = far ? 0 : min((b1 - b0) / 4 - (has_tail ? 1 : 0), (a.pos0 + row0 / a.group + 1 - 32 * b0) / kTlRows);
#pragma unroll 1
    for (int i = w;; i += 2) {
      if (issues) {
        if (i >= 2) product_o(i - 2);
        if (i < nt) product_s(i);
      }
      if (i >= nt) break;
      if (!bar_wait_warp(bar(sh.s_ready[w]), (i >> 1) & 1, given_up)) break;
      fence_after();
      if (i < whole_end) weights(i, std::true_type{});
      else weights(i, std::false_type{});
    }
    if (issues && !ok) {                          // what was issued ends before the memory goes
      int no = 0;
      mma_commit(bar(sh.drain[w]), leader);
      bar_wait_warp(bar(sh.drain[w]), 0, &no);
    }
    sh.m[w][row] = m;
    sh.l[w][row] = l;
    sh.n[w][row] = n;
    sh.k[w][row] = apart;
    asm volatile("bar.sync 1, 384;" ::: "memory");         // with the warps that have the sums
    rows_out();
    if (kMeet) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kTlRegs));
  } else if (warp < 12) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kTlRegsSum));
    uint64_t acc[kHd / 2];
#pragma unroll
    for (int d = 0; d < kHd / 2; ++d) acc[d] = 0;
    float M = -INFINITY;                          // what the sums are relative to
    const uint32_t o_at = tmem + ((uint32_t)(32 * (warp & 3)) << 16) + kTlColO;
    for (int i = 0; i < nt; ++i) {
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
          bar_arrive(bar(sh.o_free));
        }
#pragma unroll
        for (int k = 0; k < 8; ++k)
          acc[8 * h + k] = fma2(acc[8 * h + k], fa2,
                                mul2(pair(__uint_as_float(x[2 * k]), __uint_as_float(x[2 * k + 1])), fo2));
      }
    }
    asm volatile("bar.sync 1, 384;" ::: "memory");
    const float nan = __int_as_float(0x7fc00000);
    // The sums go by M, and so does l, which lacks 2^-5 of the lift; the weights apart by n. From
    // here on all goes by N, M and a whole number e that brings the sum of the weights near 1; 2^-e
    // in two factors, as it may pass the range of one.
    float l = 0.0f, n = -INFINITY, apart = 0.0f;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      const float f = ex2(0.5f * (sh.m[k][row] - M)), x = sh.n[k][row], up = fmaxf(n, x);
      l += sh.l[k][row] == 0.0f ? 0.0f : sh.l[k][row] * f * f;
      if (up == -INFINITY) continue;
      apart = apart * ex2(n - up) + sh.k[k][row] * ex2(x - up);
      n = up;
    }
    int e = l == 0.0f ? -250 : (int)(__float_as_uint(l) >> 23 & 255) - 127 + 5;
    if (apart > 0.0f) e = max(e, (int)fmaxf(fminf(ceilf(n - M), 250.0f), -250.0f));
    auto two_to = [](int x) { return __int_as_float((127 + x) << 23); };
    const float p0 = two_to(-(e >> 1)), p1 = two_to((e >> 1) - e);
    float N = M + (float)e, L = l * p0 * p1 * 32.0f + (apart > 0.0f ? apart * ex2(n - N) : 0.0f);
    if (M == -INFINITY && l == 0.0f) { N = n; L = apart; }        // no V but zeros
    if (*given_up) L = nan;
    if (nact == 1) {
      L = 1.0f / L;
      if (a.pos0 + grow / a.group >= held) L = nan;
    }
    const float f0 = p0 * (1.0f / kTlLift), f1 = nact > 1 ? p1 : p1 * L;
    float* line = lines + (size_t)row * kTlLine;
#pragma unroll
    for (int d = 0; d < kHd / 2; d += 2) {
      const float2 x = unpair(acc[d]), y = unpair(acc[d + 1]);
      *reinterpret_cast<float4*>(line + 2 * d) =
          make_float4(x.x * f0 * f1, x.y * f0 * f1, y.x * f0 * f1, y.y * f0 * f1);
    }
    float* part = a.part + (slot + chunk) * rows_part(kTlRows);
    if (nact > 1)
      *reinterpret_cast<float2*>(kMeet ? sh.ml[row] : part + kTlRows * kHd + 2 * row) = make_float2(N, L);
    rows_out();
    if (kMeet) asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kTlRegs));
  } else if (warp < 16) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" :: "n"(kTlRegsConv));
    // a warp per block of the tile
    const int cw = warp - 12, g = lane >> 2, t = lane & 3;
    const uint8_t* codes = c.codes + (size_t)kvh * c.nblk * 2 * kQ8Codes + 16 * lane;
    const float2* scales = reinterpret_cast<const float2*>(c.scales) + (size_t)kvh * c.nblk;
    const float* open = c.tail + (size_t)kvh * 2 * kQ8Codes;
    const int nopen = held - closed * kQ8Blk;
    // the codes of the next tile are loaded while this one's are worked on
    uint4 kx[8], vx[8];
    auto live = [&](int i) { return i < nt && b0 + 4 * i + cw < min(b1, nb); };
    auto fetch = [&](int i, int which, uint4 (&x)[8]) {
      if (live(i)) {
        const uint8_t* src = codes + ((size_t)(b0 + 4 * i + cw) * 2 + which) * kQ8Codes;
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = __ldg(reinterpret_cast<const uint4*>(src + 512 * u));
      }
    };
    auto put_k = [&](uint8_t* to, int c, int j, int h, const uint32_t (&x)[8]) {
      // position 8 j + g of block c, dims 64 h + 16 s + 4 t .. for s = 0 .. 3
      const int n = 64 * (c >> 1) + 16 * (g >> 1) + 8 * (c & 1) + 2 * j + (g & 1);
#pragma unroll
      for (int e = 0; e < 2; ++e)
        *reinterpret_cast<uint4*>(to + h * kTlHalf + n * 128 + (((2 * t + e) ^ (n & 7)) << 4)) =
            make_uint4(x[4 * e], x[4 * e + 1], x[4 * e + 2], x[4 * e + 3]);
    };
    auto put_v = [&](uint8_t* to, int c, int u, int h, const uint32_t (&x)[4]) {
      // dim 16 u + 8 h + g, positions 8 j + 2 t .. of block c for j = 0 .. 3
      *reinterpret_cast<uint4*>(to + (c >> 1) * kTlHalf + (16 * u + 8 * h + g) * 128 +
                                (((2 * t + (c & 1)) ^ g) << 4)) = make_uint4(x[0], x[1], x[2], x[3]);
    };
    // the open rows' values in one of their two terms (second: 1); V's up to 2^10: a weight's
    // precision then goes by w v much as with coded values
    float lk = 1.0f;
    auto lift_k = [&](int r) { return q8_lift(sh.open_max[0][r]); };
    auto lift_v = [&](int r) { return q8_lift(sh.open_max[1][r]) * 0.0625f; };
    auto term = [&](float x0, float x1, float lift0, float lift1, int second) {
      x0 = fabsf(x0) < INFINITY ? x0 * lift0 : 0.0f;
      x1 = fabsf(x1) < INFINITY ? x1 * lift1 : 0.0f;
      uint32_t hi, lo;
      split_half2(x0, x1, &hi, &lo);
      return second ? lo : hi;
    };
    // all four warps share the open block, block `oc` of its tile: two units of K and four of V
    // each, several loads under way at a time
    const int oc = (nb - b0) & 3;
    auto open_k = [&](uint8_t* to, int second) {
      const float lift = lift_k(8 * cw + g);
      float4 x[2][4];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          const int r = 8 * cw + g;
          x[i][s] = r < nopen ? __ldg(reinterpret_cast<const float4*>(open + r * kHd + 64 * i + 16 * s + 4 * t))
                              : make_float4(0.f, 0.f, 0.f, 0.f);
        }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t y[8];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
          y[2 * s] = term(x[i][s].x, x[i][s].y, lift, lift, second);
          y[2 * s + 1] = term(x[i][s].z, x[i][s].w, lift, lift, second);
        }
        put_k(to, oc, cw, i, y);
      }
    };
    auto open_v = [&](uint8_t* to, int second) {
#pragma unroll 1
      for (int i0 = 0; i0 < 4; i0 += 2) {
        float x[2][8];
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            const int r = 8 * (j >> 1) + 2 * t + (j & 1), d = 8 * (4 * cw + i0 + i) + g;
            x[i][j] = r < nopen ? __ldg(open + kQ8Codes + r * kHd + d) : 0.0f;
          }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t y[4];
#pragma unroll
          for (int j = 0; j < 4; ++j)
            y[j] = term(x[i][2 * j], x[i][2 * j + 1], lift_v(8 * j + 2 * t), lift_v(8 * j + 2 * t + 1), second);
          put_v(to, oc, 2 * cw + (i0 >> 1), i, y);
        }
      }
    };
    // the largest of each open row's values, eight rows a warp
    auto open_scan = [&] {
#pragma unroll 1
      for (int i0 = 0; i0 < 8; i0 += 4) {
        float4 x[4][2];
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int r = 8 * cw + i0 + i;
            x[i][e] = r < nopen ? __ldg(reinterpret_cast<const float4*>(open + e * kQ8Codes + r * kHd) + lane)
                                : make_float4(0.f, 0.f, 0.f, 0.f);
          }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float m = 0.0f;
            const float v[4] = {fabsf(x[i][e].x), fabsf(x[i][e].y), fabsf(x[i][e].z), fabsf(x[i][e].w)};
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              if (v[k] < INFINITY) m = fmaxf(m, v[k]);
              else atomicMin(&sh.bad, 8 * cw + i0 + i);
            }
            const unsigned top = __reduce_max_sync(0xFFFFFFFFu, __float_as_uint(m));
            if (lane == 0) sh.open_max[e][8 * cw + i0 + i] = __uint_as_float(top);
          }
      }
      asm volatile("bar.sync 4, 128;" ::: "memory");
      const float k_max = sh.open_max[0][lane], v_max = sh.open_max[1][lane];
      lk = q8_lift(__uint_as_float(__reduce_max_sync(0xFFFFFFFFu, __float_as_uint(k_max))));
      if (cw == 0) {
        sh.open_k[lane] = k_max > 0.0f ? lk / q8_lift(k_max) : 0.0f;
        sh.open_v[lane] = v_max > 0.0f ? (float)(127 - (int)(__float_as_uint(lift_v(lane)) >> 23)) : -INFINITY;
      }
    };
    auto none_k = [&](uint8_t* to) {
      const uint32_t y[8] = {0, 0, 0, 0, 0, 0, 0, 0};
#pragma unroll 1
      for (int u = 0; u < 8; ++u) put_k(to, cw, u >> 1, u & 1, y);
    };
    auto none_v = [&](uint8_t* to) {
      const uint32_t y[4] = {0, 0, 0, 0};
#pragma unroll 1
      for (int uh = 0; uh < 16; ++uh) put_v(to, cw, uh >> 1, uh & 1, y);
    };
    auto coded_k = [&](int i, uint8_t* to) {
      if (!live(i)) return none_k(to);          // past the chunk's last block
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint32_t x[4] = {kx[u].x, kx[u].y, kx[u].z, kx[u].w};
        uint32_t y[8];
#pragma unroll
        for (int k = 0; k < 4; ++k) q8_halves(x[k], &y[2 * k], &y[2 * k + 1]);
        put_k(to, cw, u >> 1, u & 1, y);
      }
    };
    auto coded_v = [&](int i, uint8_t* to) {
      if (!live(i)) return none_v(to);
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        const uint32_t x[4] = {vx[u].x, vx[u].y, vx[u].z, vx[u].w};
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t y[4];
          q8_halves(x[2 * h], &y[0], &y[1]);
          q8_halves(x[2 * h + 1], &y[2], &y[3]);
          put_v(to, cw, u, h, y);
        }
      }
    };
    // the block's first position with a V code that is not 0 (kTlNone without one): a lane's bytes
    // are those of positions 16 k + 8 j + 2 t + e
    auto first_of = [&] {
      constexpr uint32_t kZeros = 0x80808080u;
      uint32_t any[2] = {0, 0};
#pragma unroll
      for (int u = 0; u < 8; ++u) {
        any[0] |= (vx[u].x ^ kZeros) | (vx[u].z ^ kZeros);
        any[1] |= (vx[u].y ^ kZeros) | (vx[u].w ^ kZeros);
      }
      int at = kTlNone;
#pragma unroll
      for (int k = 0; k < 8; ++k)
        if (any[k >> 2] >> 8 * (k & 3) & 255) at = min(at, 16 * (k >> 2) + 8 * (k >> 1 & 1) + 2 * t + (k & 1));
      return __reduce_min_sync(0xFFFFFFFFu, at);
    };
    auto put_scales = [&](int i, float sk, float sv, int first) {
      if (lane == 0) {
        // a scale under 2^-110 counts as that (values up to 10^-31), so that a chunk of such
        // blocks alone, whose sum of weights goes by its reciprocal, stays in range; a NaN stays
        sv = sv < 0x1p-110f ? 0x1p-110f : sv;
        sh.sc[i & 3][cw][0] = sk;
        sh.sc[i & 3][cw][1] = log2f(sv);
        sh.sc[i & 3][cw][2] = sv == sv ? kTlDrop / sv : 0.0f;
        sh.first[i & 3][cw] = first;
      }
    };
    // only a scale of 1 can be that of a block of zeros, and only a block that some row does not
    // see whole can have no others to a row
    auto put_coded = [&](int i, float2 s) {
      const bool find = live(i) && (s.y == 1.0f || 32 * (b0 + 4 * i + cw) + 31 > a.pos0 + row0 / a.group);
      put_scales(i, s.x, s.y, find ? first_of() : 0);
    };
    auto scales_of = [&](int i) { return live(i) ? __ldg(scales + b0 + 4 * i + cw) : make_float2(1.f, 1.f); };
    fetch(0, 0, kx);
    fetch(0, 1, vx);
    float2 sc = scales_of(0);
    const int coded = nt - (has_tail ? 1 : 0);  // tiles without the open block
    bool ok = true;
#pragma unroll 1
    for (int i = 0; i < coded && ok; ++i) {
      const int s = i & 1;
      ok = i < 2 || bar_wait_warp(bar(sh.s_ready[s]), ((i - 2) >> 1) & 1, given_up);
      if (!ok) break;
      put_coded(i, sc);                         // before the codes (after them 13 us of 278 more)
      coded_k(i, k_buf + s * kTlTile);
      fence_async();
      bar_arrive(bar(sh.full_k[s]));
      fetch(i + 1, 0, kx);
      sc = scales_of(i + 1);
      ok = i < 2 || bar_wait_warp(bar(sh.o_done[s]), ((i - 2) >> 1) & 1, given_up);
      if (!ok) break;
      coded_v(i, v_buf + s * kTlTile);
      fence_async();
      bar_arrive(bar(sh.full_v[s]));
      fetch(i + 1, 1, vx);
    }
    if (has_tail && ok) {
      // the last tile, twice: with the open block's first terms and what comes before it, then
      // with its second terms alone
      const int i = nt - 1, s = i & 1;
      uint8_t* kt = k_buf + s * kTlTile;
      uint8_t* vt = v_buf + s * kTlTile;
      const bool mine = b0 + 4 * i + cw == closed;          // the open block is this warp's
      ok = i < 2 || bar_wait_warp(bar(sh.s_ready[s]), ((i - 2) >> 1) & 1, given_up);
      if (ok && !mine) coded_k(i, kt);
      if (ok) open_scan();
      if (!mine) put_coded(i, sc);
      else if (lane == 0) {            // the scores come as exponents; their weights are added up already
        sh.sc[i & 3][cw][0] = 1.0f;
        sh.sc[i & 3][cw][1] = sh.sc[i & 3][cw][2] = 0.0f;
        sh.sc[i & 3][cw][3] = 1.0f / lk;
        sh.first[i & 3][cw] = 0;
      }
#pragma unroll 1
      for (int pass = 0; pass < 2 && ok; ++pass) {
        if (pass) {
          ok = bar_wait_warp(bar(sh.k_free), 0, given_up);
          if (!mine) none_k(kt);
        }
        open_k(kt, pass);
        fence_async();
        bar_arrive(bar(sh.full_k[s]));
      }
      ok = ok && (i < 2 || bar_wait_warp(bar(sh.o_done[s]), ((i - 2) >> 1) & 1, given_up));
      if (ok && !mine) coded_v(i, vt);
#pragma unroll 1
      for (int pass = 0; pass < 2 && ok; ++pass) {
        if (pass) {
          ok = bar_wait_warp(bar(sh.v_free), 0, given_up);
          if (!mine) none_v(vt);
        }
        open_v(vt, pass);
        fence_async();
        bar_arrive(bar(sh.full_v[s]));
      }
    }
    if (kMeet) asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" :: "n"(kTlRegs));
  }
  if (kMeet) {                                    // all roles have the launch's registers again
    cluster_sync();
    if (nact > 1)
      cluster_add_up(a, lines, kTlLine, sh.ml[0], nact, kvh, row0, kTlRows, chunk, warp, kTlThreads / 32, held);
    cluster_sync();
  }
  __syncwarp();
  fence_before();
  __syncthreads();
  if (warp == 15) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" :: "r"(tmem));
  }
}

}  // namespace

template <bool kMeet>
static int tile_launch(const RowsArgs& a, const KvQ8& c, unsigned tiles, unsigned nkv, cudaStream_t st) {
  const int rc = smem_attr((const void*)k_attn_tile_q8<kMeet>, kTlSmem);
  if (rc) return rc;
  // registers are dealt out of what the kernel starts with: a share too large would wait for good
  static const int regs = [] {
    cudaFuncAttributes f{};
    return cudaFuncGetAttributes(&f, k_attn_tile_q8<kMeet>) == cudaSuccess ? f.numRegs : 0;
  }();
  HV_REQUIRE(regs == kTlRegs, HV_E_UNSUPPORTED, "k_attn_tile_q8: built with %d registers", regs);
  return rows_launch(k_attn_tile_q8<kMeet>, dim3(tiles * a.chunks, nkv), kTlThreads, kTlSmem, a, c, st);
}

int attn_tile_q8_room(int n, int* room) {
  const int rc = smem_attr((const void*)k_attn_tile_q8<true>, kTlSmem);
  if (rc) return rc;
  cudaLaunchAttribute at{};
  cudaLaunchConfig_t cfg = rows_config(dim3(n), kTlThreads, kTlSmem, n, &at, nullptr);
  HV_CUDA(cudaOccupancyMaxActiveClusters(room, k_attn_tile_q8<true>, &cfg));
  return HV_OK;
}

int attn_tile_q8_launch(const RowsArgs& a, const KvQ8& c, unsigned tiles, unsigned nkv,
                        cudaStream_t st) {
  return a.cluster ? tile_launch<true>(a, c, tiles, nkv, st) : tile_launch<false>(a, c, tiles, nkv, st);
}

}  // namespace hv
