// A cache thinned to the positions that attention goes to (hv_kv_evict_f16): of every cache and
// kv head the latest positions stay, and of the others those with the most accumulated weight.
// What stays keeps its order and moves down.
//
// One launch. A (cache, kv head) has one CTA or several, each of which finds the edge for itself (the
// largest key that the wanted number reach, eight bits at a time, by counts in shared memory) and
// then goes through the positions, some thousands at a time: which of them stay and where to, by a
// scan over the CTA, and their rows on their way there through a ring in shared memory. In place a
// row goes to where it is or below, in order, so that whoever writes a batch of rows needs to know
// only that the CTA has read it: what a batch overwrites lies below what later ones read. Several
// CTAs of a head in place have some of every row's dims each and are a cluster, because none may
// move the masses before all have read them; apart they have some of the rows each.
//
// Bound by HBM when caches are many (36 caches of 8 heads, 4352 positions to 4096: 1.21 GB read and
// written in 228 us, 82% of a copy's rate; 271 with rows through registers and one bit of the border a
// pass), by latency when they are few (300 positions of 2 heads to 256: 8.4 us for 19).
#include <cuda_fp16.h>

#include <algorithm>
#include <cstdlib>

#include "attn_decode.cuh"
#include "hv_internal.h"

namespace hv {
namespace {

struct EvictArgs {
  const __half *kc, *vc;
  __half *kd, *vd;
  const float* mass;
  float* mass_d;
  int32_t* kept;
  const int32_t* len;
  int32_t* len_out;
  size_t set, set_d;
  int cap, dcap, added, limit, keep, recent, nkv;
  unsigned* ticket;
};

// The order of masses as an unsigned number: NaN above all, -0 equal to +0.
HV_DEV unsigned mass_key(float x) {
  if (x != x) return 0xFFFFFFFFu;
  const unsigned u = __float_as_uint(x + 0.0f);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kEvThreads = 512, kEvWarps = kEvThreads / 32;
constexpr int kEvStage = 2 * kEvThreads * 16, kEvStages = 5;    // bytes; two 16-byte units a thread
constexpr int kEvChunk = 4 * kEvThreads, kEvSegment = 4 * kEvChunk;
constexpr int kEvMost = 8;                                      // CTAs of a head in place
constexpr int kEvSmem = kEvStages * kEvStage + kEvSegment * 2;

struct EvShared {
  unsigned hist[256];
  unsigned sum[2][kEvWarps];
  unsigned edge, left;
};

// The largest key that `want` of mass[0, n) reach, and how many of those equal to it are among
// them: the count above it is less than want.
HV_DEV void find_edge(const float* mass, int n, int want, EvShared& sh, unsigned* edge, int* ties) {
  unsigned top = 0;
  int left = want;                               // wanted among the keys that begin as top does
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < 256; i += kEvThreads) sh.hist[i] = 0;
    __syncthreads();
    const unsigned mask = shift == 24 ? 0 : ~0u << (shift + 8);
    for (int i = threadIdx.x; i < n; i += kEvThreads) {
      const unsigned k = mass_key(mass[i]);
      if ((k & mask) == top) atomicAdd(&sh.hist[k >> shift & 255], 1u);
    }
    __syncthreads();
    if (threadIdx.x < 32) {
      // lane l has the counts of 8 l .. 8 l + 7; from the top down until they are `left`
      unsigned c[8], s = 0;
#pragma unroll
      for (int j = 0; j < 8; ++j) s += c[j] = sh.hist[8 * threadIdx.x + j];
      unsigned above = s;                        // of this lane's and all higher ones
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) {
        const unsigned y = __shfl_down_sync(0xFFFFFFFFu, above, d);
        if (threadIdx.x + d < 32) above += y;
      }
      above -= s;
      const bool mine = (int)above < left && (int)(above + s) >= left;
      if (mine) {
        int j = 7;
        while ((int)(above + c[j]) < left) above += c[j--];
        sh.edge = top | (8 * threadIdx.x + j) << shift;
        sh.left = left - above;
      }
    }
    __syncthreads();
    top = sh.edge;
    left = (int)sh.left;
    __syncthreads();
  }
  *edge = top;
  *ties = left;
}

// kApart: the destination is other memory than the source.
template <bool kApart>
__global__ void __launch_bounds__(kEvThreads, 2) k_evict(EvictArgs a) {
  extern __shared__ __align__(16) uint8_t smem[];           // the ring, then a segment's rows
  __shared__ EvShared sh;
  uint16_t* list = reinterpret_cast<uint16_t*>(smem + kEvStages * kEvStage);
  const int parts = gridDim.x, part = blockIdx.x, head = blockIdx.y, set = blockIdx.z;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long n_ = (long long)*a.len + a.added;
  const bool bad = n_ < 0 || n_ > a.cap;
  const int n = bad ? 0 : (int)n_;
  const bool thin = n > a.limit;
  const size_t hi = (size_t)set * a.nkv + head;
  const float* mass = a.mass + hi * a.cap;
  float* mass_d = a.mass_d + hi * a.dcap;
  const size_t src0 = set * a.set + (size_t)head * a.cap * kHd, dst0 = set * a.set_d + (size_t)head * a.dcap * kHd;
  const int old = thin ? max(0, n - a.recent) : n;         // the others start at 0
  const int want = thin ? a.keep - (n - old) : old;        // of [0, old)
  unsigned edge = 0;                                       // keys above it stay, `ties` of those at it
  int ties = 0;
  if (thin && want > 0 && want < old) find_edge(mass, old, want, sh, &edge, &ties);
  const bool all = want == old;                            // (want = 0 and ties = 0: none)
  if (want == 0) edge = 0xFFFFFFFFu;
  // this CTA's part of a row: `units` 16-byte units; or, apart, every parts-th batch of whole rows
  const int units = kApart ? 32 : 32 / parts;
  const int per = 2 * kEvThreads / units;                  // rows of a batch
  const uint32_t ring = (uint32_t)__cvta_generic_to_shared(smem);

  // Which of positions i0 + 4 tid .. + 3 stay, and where to (bits 0-3 of `stay`); `above`, `tied`:
  // those before the chunk, which it adds its own to.
  int above = 0, tied = 0;
  auto scan = [&](int i0, int turn, int (&to)[4], float (&m)[4]) {
    unsigned up = 0, at = 0;                               // of this thread: above (or late), at the edge
    unsigned is_up = 0, is_at = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const int i = i0 + 4 * tid + j;
      m[j] = i < n ? mass[i] : 0.0f;
      const unsigned k = mass_key(m[j]);
      const bool u = i < n && (i >= old || all || k > edge), e = i < old && !all && k == edge;
      is_up |= (unsigned)u << j;
      is_at |= (unsigned)e << j;
    }
    up = __popc(is_up);
    at = __popc(is_at);
    unsigned mine = up | at << 16, s = mine;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
      const unsigned y = __shfl_up_sync(0xFFFFFFFFu, s, d);
      if (lane >= d) s += y;
    }
    if (lane == 31) sh.sum[turn & 1][warp] = s;
    __syncthreads();
    unsigned before = 0, total = 0;
#pragma unroll
    for (int w = 0; w < kEvWarps; ++w) {
      const unsigned y = sh.sum[turn & 1][w];
      before += w < warp ? y : 0;
      total += y;
    }
    s += before - mine;
    int u = above + (int)(s & 0xFFFF), e = tied + (int)(s >> 16);
    unsigned stay = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      to[j] = u + min(e, ties);
      const bool x = is_up >> j & 1, y = is_at >> j & 1;
      stay |= (unsigned)(x || (y && e < ties)) << j;
      u += x;
      e += y;
    }
    above += (int)(total & 0xFFFF);
    tied += (int)(total >> 16);
    return stay;
  };
  const bool work = thin || kApart;
  // masses move as they are scanned, unless other CTAs of the head still read them here
  const bool masses = part == 0 && (kApart || parts == 1);
  int turn = 0;
  for (int s0 = 0; work && s0 < n; s0 += kEvSegment) {
    const int done = above + min(tied, ties);              // rows out before this segment
    for (int i0 = s0; i0 < min(n, s0 + kEvSegment); i0 += kEvChunk, ++turn) {
      int to[4];
      float m[4];
      const unsigned stay = scan(i0, turn, to, m);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (!(stay >> j & 1)) continue;
        list[to[j] - done] = (uint16_t)(i0 + 4 * tid + j - s0);
        if (masses) mass_d[to[j]] = m[j];                  // (read by all before the scan's barrier)
        if (a.kept && part == 0) a.kept[hi * a.dcap + to[j]] = i0 + 4 * tid + j;
      }
    }
    __syncthreads();
    const int rows = above + min(tied, ties) - done;
    const int step = kApart ? parts : 1;
    const int nb = (rows + per - 1) / per;
    const int mine = kApart ? (nb - part + parts - 1) / parts : nb;
    // unit u of a thread: row u / units of the batch, unit u % units of this CTA's part of it
    auto place = [&](int b, int u, int* row, int* unit) {
      *row = ((kApart ? part : 0) + b * step) * per + u / units;
      *unit = (kApart ? 0 : part * units) + u % units;     // of 16 of K, then 16 of V
    };
    auto fetch = [&](int b) {
      if (b < mine) {
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          int row, unit;
          place(b, tid + e * kEvThreads, &row, &unit);
          if (row < rows) {
            const size_t at = src0 + (size_t)(s0 + list[row]) * kHd + 8 * (unit & 15);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;"
                         :: "r"(ring + (b % kEvStages) * kEvStage + (tid + e * kEvThreads) * 16),
                            "l"((unit < 16 ? a.kc : a.vc) + at) : "memory");
          }
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
    };
#pragma unroll
    for (int b = 0; b < kEvStages - 1; ++b) fetch(b);
    for (int b = 0; b < mine; ++b) {
      asm volatile("cp.async.wait_group %0;" :: "n"(kEvStages - 2) : "memory");
      if (!kApart) __syncthreads();                        // the CTA has read the batch
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        int row, unit;
        place(b, tid + e * kEvThreads, &row, &unit);
        if (row < rows) {
          const uint4 x = *reinterpret_cast<const uint4*>(smem + (b % kEvStages) * kEvStage + (tid + e * kEvThreads) * 16);
          *reinterpret_cast<uint4*>((unit < 16 ? a.kd : a.vd) + dst0 + (size_t)(done + row) * kHd + 8 * (unit & 15)) = x;
        }
      }
      fetch(b + kEvStages - 1);                            // a unit's place in the ring is its thread's own
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    __syncthreads();                                       // the list is free
  }
  if (!kApart && parts > 1) {
    // no CTA of the head has a use for the masses any more: the first moves them
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    if (part == 0 && thin) {
      above = tied = 0;
      for (int i0 = 0; i0 < n; i0 += kEvChunk, ++turn) {
        int to[4];
        float m[4];
        const unsigned stay = scan(i0, turn, to, m);
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (stay >> j & 1) mass_d[to[j]] = m[j];
      }
    }
  }
  __syncthreads();                                         // all have read the length
  if (tid == 0) {                                          // the last CTA to come by writes the length
    __threadfence();
    const unsigned total = gridDim.x * gridDim.y * gridDim.z;
    if (atomicAdd(a.ticket, 1) == total - 1) {
      *a.ticket = 0;
      if (!bad) *a.len_out = thin ? a.keep : n;
    }
  }
}

template <bool kApart>
int evict_launch(const EvictArgs& a, int parts, int nkv, int nset, cudaStream_t st) {
  const int rc = smem_attr((const void*)k_evict<kApart>, kEvSmem);
  if (rc) return rc;
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = (unsigned)parts;
  at.val.clusterDim.y = at.val.clusterDim.z = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3((unsigned)parts, (unsigned)nkv, (unsigned)nset);
  cfg.blockDim = dim3(kEvThreads);
  cfg.dynamicSmemBytes = kEvSmem;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = !kApart && parts > 1 ? 1 : 0;
  const cudaError_t e = cudaLaunchKernelEx(&cfg, k_evict<kApart>, a);
  return e == cudaSuccess ? HV_OK : cuda_fail("hv_kv_evict_f16", e);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

// Do n pieces of `bytes` from x on and n from y on, each `step` after the one before it, share
// nothing? Pieces i and j are |y - x + (j - i) step| apart, the least at one of two j - i.
bool pieces_apart(const void* x, const void* y, long long bytes, long long step, int n) {
  const long long d = (long long)((uintptr_t)y - (uintptr_t)x);
  if (n == 1) return std::llabs(d) >= bytes;
  const long long near = std::max<long long>(1 - n, std::min<long long>(n - 1, -(d / step)));
  for (long long m = std::max<long long>(1 - n, near - 1); m <= std::min<long long>(n - 1, near + 1); ++m)
    if (std::llabs(d + m * step) < bytes) return false;
  return true;
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_kv_evict_scratch(int nkv, int cap, int nset, size_t* bytes) {
  HV_REQUIRE(nkv > 0 && cap > 0 && nset > 0 && bytes, HV_E_INVALID, "hv_kv_evict_scratch: bad arguments");
  HV_REQUIRE(nkv <= 65535 && nset <= 65535 && cap <= (1 << 24), HV_E_UNSUPPORTED,
             "hv_kv_evict_scratch: %d caches of %d heads, %d positions", nset, nkv, cap);
  *bytes = 256;
  return HV_OK;
}

extern "C" int hv_kv_evict_f16(const uint16_t* kc, const uint16_t* vc, long long set, const float* mass,
                               int cap, const int32_t* len, int added, uint16_t* kd, uint16_t* vd,
                               long long set_d, float* mass_d, int dcap, int32_t* len_out, int32_t* kept,
                               int limit, int keep, int recent, int nkv, int hd, int nset, void* scratch,
                               void* stream) {
  const char* name = "hv_kv_evict_f16";
  HV_REQUIRE(kc && vc && mass && len && kd && vd && mass_d && len_out && scratch && cap > 0 && dcap > 0 &&
                 added >= 0 && nkv > 0 && nset > 0,
             HV_E_INVALID, "%s: bad arguments", name);
  HV_REQUIRE(hd == kHd, HV_E_UNSUPPORTED, "%s: head_dim %d (only 128)", name, hd);
  HV_REQUIRE(keep > 0 && recent >= 0 && recent <= keep && keep <= limit && limit <= dcap, HV_E_INVALID,
             "%s: recent %d, keep %d, limit %d, room for %d: each at most the next", name, recent, keep, limit, dcap);
  HV_REQUIRE(nkv <= 65535 && nset <= 65535 && cap <= (1 << 24) && dcap <= (1 << 24), HV_E_UNSUPPORTED,
             "%s: %d caches of %d heads, %d positions", name, nset, nkv, cap);
  const long long one = (long long)nkv * cap * kHd, one_d = (long long)nkv * dcap * kHd;
  HV_REQUIRE(nset == 1 || (set >= one && set_d >= one_d && set % 8 == 0 && set_d % 8 == 0 && set < (1ll << 40) &&
                           set_d < (1ll << 40)),
             HV_E_INVALID, "%s: caches %lld and %lld elements apart", name, set, set_d);
  HV_REQUIRE(aligned16(kc) && aligned16(vc) && aligned16(kd) && aligned16(vd) && aligned16(scratch), HV_E_INVALID,
             "%s: unaligned pointer", name);
  const bool in_place = kd == kc && vd == vc;
  if (in_place) {
    HV_REQUIRE(mass_d == mass && dcap == cap && (nset == 1 || set == set_d), HV_E_INVALID,
               "%s: in place with another arrangement", name);
  } else {
    auto apart = [](const void* x, long long nx, const void* y, long long ny) {
      const uintptr_t a = (uintptr_t)x, b = (uintptr_t)y;
      return a + (uintptr_t)nx <= b || b + (uintptr_t)ny <= a;
    };
    const long long from = 2 * ((nset - 1) * set * (nset > 1) + one), to = 2 * ((nset - 1) * set_d * (nset > 1) + one_d);
    HV_REQUIRE(apart(kc, from, kd, to) && apart(kc, from, vd, to) && apart(vc, from, kd, to) &&
                   apart(vc, from, vd, to) &&
                   apart(mass, 4ll * nset * nkv * cap, mass_d, 4ll * nset * nkv * dcap),
               HV_E_INVALID, "%s: source and destination overlap", name);
  }
  HV_REQUIRE(pieces_apart(kd, vd, 2 * one_d, 2 * set_d, nset), HV_E_INVALID, "%s: K and V of the destination overlap", name);
  EvictArgs a{};
  a.kc = reinterpret_cast<const __half*>(kc); a.vc = reinterpret_cast<const __half*>(vc);
  a.kd = reinterpret_cast<__half*>(kd); a.vd = reinterpret_cast<__half*>(vd);
  a.mass = mass; a.mass_d = mass_d; a.kept = kept; a.len = len; a.len_out = len_out;
  a.set = nset > 1 ? (size_t)set : 0; a.set_d = nset > 1 ? (size_t)set_d : 0;
  a.cap = cap; a.dcap = dcap; a.added = added; a.limit = limit; a.keep = keep; a.recent = recent; a.nkv = nkv;
  a.ticket = reinterpret_cast<unsigned*>(scratch);
  // two CTAs an SM; a head's share in a segment of some thousands of rows is hundreds of batches
  const long long heads = (long long)nkv * nset;
  int parts = (int)std::max(1ll, std::min<long long>(in_place ? kEvMost : 64, 296 / heads));
  parts = std::min(parts, std::max(1, cap / 64));
  if (!in_place) return evict_launch<true>(a, parts, nkv, nset, (cudaStream_t)stream);
  while (parts & (parts - 1)) parts &= parts - 1;           // of a row's 32 units
  return evict_launch<false>(a, parts, nkv, nset, (cudaStream_t)stream);
}
