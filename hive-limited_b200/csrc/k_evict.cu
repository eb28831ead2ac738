// A cache thinned to the positions that attention goes to (hv_kv_evict_f16): of every cache and
// kv head the latest positions stay, and of the others those with the most accumulated weight.
// What stays keeps its order and moves down.
#include <cuda_fp16.h>

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

constexpr int kEvThreads = 1024;

HV_DEV int block_sum(int x, int* s) {
  x = __reduce_add_sync(0xFFFFFFFFu, x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = x;
  __syncthreads();
  return __reduce_add_sync(0xFFFFFFFFu, s[threadIdx.x & 31]);
}

// A CTA per (cache, kv head).
__global__ void __launch_bounds__(kEvThreads) k_evict(EvictArgs a) {
  __shared__ int s_sum[32], s_list[kEvThreads];
  const int head = blockIdx.x, set = blockIdx.y, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const long long n_ = (long long)*a.len + a.added;
  const bool bad = n_ < 0 || n_ > a.cap;
  const int n = bad ? 0 : (int)n_;
  const bool thin = n > a.limit;
  const bool copy = a.kd != a.kc;
  const size_t hi = (size_t)set * a.nkv + head;
  const float* mass = a.mass + hi * a.cap;
  float* mass_d = a.mass_d + hi * a.dcap;
  const size_t src0 = set * a.set + (size_t)head * a.cap * kHd, dst0 = set * a.set_d + (size_t)head * a.dcap * kHd;
  const int old = thin ? max(0, n - a.recent) : n;         // the others start at 0
  const int want = thin ? a.keep - (n - old) : old;        // of [0, old)
  unsigned edge = 0;                                       // keys above it stay, `ties` of those at it
  int ties = old;
  if (want < old) {
    for (int b = 31; b >= 0; --b) {                        // the largest edge that `want` keys reach
      const unsigned e = edge | 1u << b;
      int c = 0;
      for (int i = tid; i < old; i += kEvThreads) c += mass_key(mass[i]) >= e;
      if (block_sum(c, s_sum) >= want) edge = e;
    }
    int c = 0;
    for (int i = tid; i < old; i += kEvThreads) c += mass_key(mass[i]) > edge;
    ties = want - block_sum(c, s_sum);
  }
  int done = 0, seen = 0;                                  // rows out, ties met
  for (int i0 = 0; (thin || copy) && i0 < n; i0 += kEvThreads) {
    const int i = i0 + tid;
    const unsigned k = i < old ? mass_key(mass[i]) : 0;
    const float m = i < n ? mass[i] : 0.0f;
    const bool tie = i < old && k == edge;
    // where this one stands among the chunk's ties, then among its rows that stay
    unsigned w = __ballot_sync(0xFFFFFFFFu, tie);
    int at = __popc(w & ((1u << lane) - 1));
    __syncthreads();
    if (lane == 0) s_sum[warp] = __popc(w);
    __syncthreads();
    int all = 0;
    for (int j = 0; j < 32; ++j) {
      at += j < warp ? s_sum[j] : 0;
      all += s_sum[j];
    }
    const bool stay = i < n && (i >= old || want == old || k > edge || (tie && seen + at < ties));
    seen += all;
    w = __ballot_sync(0xFFFFFFFFu, stay);
    at = __popc(w & ((1u << lane) - 1));
    __syncthreads();
    if (lane == 0) s_sum[warp] = __popc(w);
    __syncthreads();
    all = 0;
    for (int j = 0; j < 32; ++j) {
      at += j < warp ? s_sum[j] : 0;
      all += s_sum[j];
    }
    if (stay) {
      s_list[at] = i;
      mass_d[done + at] = m;
      if (a.kept) a.kept[hi * a.dcap + done + at] = i;
    }
    __syncthreads();
    // rows go to their place or below it, in order: a batch is read before it is written, and
    // no later one reads what it wrote
    for (int r0 = 0; r0 < all; r0 += 64) {
      const int r = r0 + (tid >> 4), u = tid & 15;
      uint4 x, y;
      if (r < all) {
        x = reinterpret_cast<const uint4*>(a.kc + src0 + (size_t)s_list[r] * kHd)[u];
        y = reinterpret_cast<const uint4*>(a.vc + src0 + (size_t)s_list[r] * kHd)[u];
      }
      __syncthreads();
      if (r < all) {
        reinterpret_cast<uint4*>(a.kd + dst0 + (size_t)(done + r) * kHd)[u] = x;
        reinterpret_cast<uint4*>(a.vd + dst0 + (size_t)(done + r) * kHd)[u] = y;
      }
      __syncthreads();
    }
    done += all;
  }
  __syncthreads();                                         // all have read the length
  if (tid == 0) {                                          // the last CTA to come by writes the length
    __threadfence();
    const unsigned total = gridDim.x * gridDim.y;
    if (atomicAdd(a.ticket, 1) == total - 1) {
      *a.ticket = 0;
      if (!bad) *a.len_out = thin ? a.keep : n;
    }
  }
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

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
                   apart(vc, from, vd, to) && apart(kd, one_d * 2, vd, one_d * 2) &&
                   apart(mass, 4ll * nset * nkv * cap, mass_d, 4ll * nset * nkv * dcap),
               HV_E_INVALID, "%s: source and destination overlap", name);
  }
  EvictArgs a{};
  a.kc = reinterpret_cast<const __half*>(kc); a.vc = reinterpret_cast<const __half*>(vc);
  a.kd = reinterpret_cast<__half*>(kd); a.vd = reinterpret_cast<__half*>(vd);
  a.mass = mass; a.mass_d = mass_d; a.kept = kept; a.len = len; a.len_out = len_out;
  a.set = nset > 1 ? (size_t)set : 0; a.set_d = nset > 1 ? (size_t)set_d : 0;
  a.cap = cap; a.dcap = dcap; a.added = added; a.limit = limit; a.keep = keep; a.recent = recent; a.nkv = nkv;
  a.ticket = reinterpret_cast<unsigned*>(scratch);
  k_evict<<<dim3((unsigned)nkv, (unsigned)nset), kEvThreads, 0, (cudaStream_t)stream>>>(a);
  HV_LAUNCHED(name);
}
