// Log probabilities of given tokens, the entropy of each row's distribution and its most
// likely tokens, from rows of logits.
//
// With m the row's maximum and z_i = x_i - m (z = 0 at the maximum's first place, a), the
// kernel sums what the other tokens add:
//   S = sum_{i != a} exp(z_i)      T = sum_{i != a} -z_i exp(z_i)
//   log p_i = z_i - log1p(S)       entropy = log1p(S) + T / (1 + S)
// All terms are positive and the large one is left out of the sums, so a distribution that
// is nearly certain (S near 0) keeps its relative precision.
// A row with a NaN, a +infinity or nothing above -infinity has no distribution: its log
// probabilities and entropy are NaN. Tokens order as np.argmax orders them: by value, -0
// equal to +0, a NaN above all, ties to the lower id.
//
// One pass over the logits. 256 rows of 151936 (155 MB) take 40 us, 3.9 TB/s, 59% of a plain
// copy's rate, with half of the issue slots used: an exponential, four packed operations and two
// comparisons for each logit in a chain that a warp waits on, and 256 CTAs where 296 fit, so that 40
// of 148 SMs have one row and the others two. One row takes 12 us (6 without alternatives), all
// of it latency: the first batches' list, the trip through the scratch, the merge of 38 lists.
//
// Alternatives: a warp keeps its 32 largest, and what is under a bound costs one comparison. The
// CTA's first logits give the bound (block_first; a list per warp that met afterwards took 14 us
// for one row and 42 for 256), which the lists' meetings raise while what has been seen grows
// fourfold.
#include <cfloat>

#include "hv_common.cuh"
#include "hv_internal.h"

namespace hv {
namespace {

constexpr int kMaxTop = 32;
constexpr int kLpThreads = 512, kLpWarps = kLpThreads / 32;
constexpr int kLpEach = 8;                        // logits a thread holds at a time
constexpr int kLpBatch = 32 * kLpEach;            // a warp's
constexpr int kLpTile = kLpWarps * kLpBatch;      // a CTA's
constexpr int kLpPieces = 64;                     // CTAs that may share a row
constexpr int kLpTickets = 1024;                  // rows that may be shared; their tickets stand
                                                  // first in the scratch whatever the call

constexpr float kLog2e = 1.4426950408889634f;

using u64 = unsigned long long;

// 64-bit key in np.argmax's order: the f32 bits mapped to an unsigned order, then ~id. A key
// is never 0.
HV_DEV u64 lp_key(float v, int id) {
  unsigned u = __float_as_uint(v);
  if (v != v) u = 0x7FC00000u;
  else if (v == 0.f) u = 0u;
  const unsigned ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((u64)ord << 32) | (u64)(~(unsigned)id);
}
HV_DEV float lp_key_value(u64 k) {
  const unsigned ord = (unsigned)(k >> 32);
  return __uint_as_float((ord & 0x80000000u) ? (ord & 0x7FFFFFFFu) : ~ord);
}
HV_DEV u64 max64(u64 a, u64 b) { return a > b ? a : b; }
HV_DEV u64 min64(u64 a, u64 b) { return a < b ? a : b; }

HV_DEV float max_nan(float a, float b) {          // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
HV_DEV float ex2f(float x) {                       // 0 below 2^-126
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// A warp's 32 keys in falling order over the lanes.
HV_DEV u64 warp_sort(u64 v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int k = 2; k <= 32; k <<= 1) {
#pragma unroll
    for (int j = k >> 1; j > 0; j >>= 1) {
      const u64 w = __shfl_xor_sync(0xFFFFFFFFu, v, j);
      const bool high = ((lane & j) == 0) == ((lane & k) == 0 || k == 32);
      v = high ? max64(v, w) : min64(v, w);
    }
  }
  return v;
}
// The 32 largest of two falling lists, falling.
HV_DEV u64 warp_merge(u64 a, u64 b) {
  const int lane = threadIdx.x & 31;
  a = max64(a, __shfl_sync(0xFFFFFFFFu, b, 31 - lane));
#pragma unroll
  for (int j = 16; j > 0; j >>= 1) {
    const u64 w = __shfl_xor_sync(0xFFFFFFFFu, a, j);
    a = (lane & j) == 0 ? max64(a, w) : min64(a, w);
  }
  return a;
}

// What a set of logits adds to a row: its maximum m, and over all its elements but one at the
// maximum S = sum exp(x - m), T = sum (m - x) exp(x - m). m = -inf: nothing (yet).
struct LpSum {
  float m, s, t;
};
HV_DEV LpSum lp_join(LpSum a, LpSum b) {
  if (b.m == -INFINITY) return a;
  if (a.m == -INFINITY) return b;
  if (a.m < b.m) { const LpSum c = a; a = b; b = c; }
  const float d = fmaxf(b.m - a.m, -200.0f), f = ex2f(d * kLog2e);
  a.t += f * (b.t - d * (1.0f + b.s));
  a.s += f * (1.0f + b.s);
  if (!(b.m <= a.m)) a.m = b.m - b.m + a.m;         // a NaN on either side stays one
  return a;
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

constexpr int kLpCand = 512;                      // keys that are put in order side by side

struct LpShared {
  u64 lists[kLpWarps][32];
  u64 cand[kLpCand];
  u64 best[32];
  LpSum sums[kLpWarps];
  u64 least;
  unsigned lead[32];             // the first batches' two largest lanes of each warp
  unsigned count, last;
};
static_assert(2 * kLpWarps == 32, "two leading lanes a warp are a warp's lanes");

// The 32 largest of every warp's falling list `v`, falling, in warp 0 (all warps call).
HV_DEV u64 block_merge(u64 v, LpShared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
#pragma unroll
  for (int half = kLpWarps / 2; half > 0; half >>= 1) {
    if (warp >= half && warp < 2 * half) sh.lists[warp][lane] = v;
    __syncthreads();
    if (warp < half) v = warp_merge(v, sh.lists[warp + half][lane]);
  }
  return v;
}

// The 32 largest of the `n` keys in sh.cand, falling, in warp 0: a key's place is how many are
// above it. All warps call, after a barrier.
HV_DEV u64 block_order(int n, LpShared& sh) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < n; i += kLpThreads) {
    const u64 k = sh.cand[i];
    int above = 0;
#pragma unroll 8
    for (int j = 0; j < n; ++j) above += sh.cand[j] > k;
    if (above < 32) sh.best[above] = k;
  }
  __syncthreads();
  return warp == 0 && lane < n ? sh.best[lane] : 0;
}

// The first batches of all warps, v of ids as in warp_take, those below n. The lanes' two largest
// of each warp, 32 in all, give a bound that at least `top` logits reach, and
// few more do: those are put side by side and in order. The list, in warp 0; false where too many
// reach the bound (equal logits) or there is none.
HV_DEV bool block_first(const float (&v)[kLpEach], int id, int n, int top, LpShared& sh, u64* list) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float mine = -INFINITY;                               // the lane's largest, if it has any
  bool any = false;
#pragma unroll
  for (int k = 0; k < kLpEach; ++k) {
    const int i = id + (k & 3) + 128 * (k >> 2);
    if (i >= 0 && i < n) {
      mine = any ? max_nan(mine, v[k]) : v[k];
      any = true;
    }
  }
  const unsigned ord = any ? (unsigned)(lp_key(mine, 0) >> 32) : 0u;
  const unsigned o0 = __reduce_max_sync(0xFFFFFFFFu, ord);
  const int l0 = __ffs(__ballot_sync(0xFFFFFFFFu, ord == o0)) - 1;
  const unsigned o1 = __reduce_max_sync(0xFFFFFFFFu, lane == l0 ? 0u : ord);
  if (lane < 2) sh.lead[2 * warp + lane] = lane ? o1 : o0;
  if (threadIdx.x == 0) sh.count = 0;
  __syncthreads();
  const unsigned lead = sh.lead[lane];
  int above = 0;
#pragma unroll
  for (int j = 0; j < 32; ++j) above += sh.lead[j] > lead || (sh.lead[j] == lead && j < lane);
  const unsigned bound =
      __shfl_sync(0xFFFFFFFFu, lead, __ffs(__ballot_sync(0xFFFFFFFFu, above == top - 1)) - 1);
  if (bound && o0 >= bound) {
#pragma unroll
    for (int k = 0; k < kLpEach; ++k) {
      const int i = id + (k & 3) + 128 * (k >> 2);
      const u64 key = i >= 0 && i < n ? lp_key(v[k], i) : 0;
      const unsigned who = __ballot_sync(0xFFFFFFFFu, (unsigned)(key >> 32) >= bound);
      if (!who) continue;
      unsigned at = 0;
      if (lane == 0) at = atomicAdd(&sh.count, (unsigned)__popc(who));
      at = __shfl_sync(0xFFFFFFFFu, at, 0) + __popc(who & ((1u << lane) - 1));
      if ((who >> lane & 1) && at < kLpCand) sh.cand[at] = key;
    }
  }
  __syncthreads();
  const unsigned count = sh.count;
  if (!bound || count > kLpCand) return false;
  *list = block_order(count, sh);
  return true;
}

HV_DEV u64 shfl64(u64 v, int src) { return __shfl_sync(0xFFFFFFFFu, v, src); }

// Takes a batch's logits (of ids id + (k & 3) + 128 (k >> 2)) that are above `least` into the
// warp's falling list of 32; without a bound it starts from the lanes' largest.
// Returns the list; the `top`th of it raises `least`.
HV_DEV u64 warp_take(u64 list, const float (&v)[kLpEach], int id, int n, int top, u64* least) {
  const int lane = threadIdx.x & 31;
  if (*least == 0) {                                      // nothing to go by yet
    u64 best = 0;
#pragma unroll
    for (int k = 0; k < kLpEach; ++k) {
      const int i = id + (k & 3) + 128 * (k >> 2);
      if (i >= 0 && i < n) best = max64(best, lp_key(v[k], i));
    }
    list = warp_sort(best);
    *least = max64(*least, shfl64(list, top - 1));
  }
  float bar = lp_key_value(*least);                       // NaN while there is no bound
#pragma unroll
  for (int k = 0; k < kLpEach; ++k) {
    const int i = id + (k & 3) + 128 * (k >> 2);
    unsigned who = __ballot_sync(0xFFFFFFFFu, i >= 0 && i < n && !(v[k] < bar));
    while (who) {
      const int src = __ffs(who) - 1;
      who &= who - 1;
      const u64 key = lp_key(__shfl_sync(0xFFFFFFFFu, v[k], src), __shfl_sync(0xFFFFFFFFu, i, src));
      if (key <= *least || __any_sync(0xFFFFFFFFu, list == key)) continue;
      const int pos = __popc(__ballot_sync(0xFFFFFFFFu, list > key));
      const u64 up = __shfl_up_sync(0xFFFFFFFFu, list, 1);
      list = lane < pos ? list : lane == pos ? key : up;
      *least = max64(*least, shfl64(list, top - 1));
      bar = lp_key_value(*least);
    }
  }
  return list;
}

// One CTA per (row, piece of the row); a warp takes batches of 256 logits. Four logits of a row
// stand on 16 bytes: `off` floats before the row's first one make it so, and units at the edges
// are read one by one. kTop: alternatives are wanted.
template <bool kTop>
__global__ void __launch_bounds__(kLpThreads, 2)
    k_logprob(const float* __restrict__ logits, size_t ld, int n, const int32_t* __restrict__ tok,
              int top, float* __restrict__ lp, float* __restrict__ ent,
              int32_t* __restrict__ top_id, float* __restrict__ top_lp, int pieces,
              LpSum* __restrict__ psum, u64* __restrict__ plist, unsigned* __restrict__ ticket) {
  __shared__ LpShared sh;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int r = blockIdx.x / pieces, piece = blockIdx.x % pieces;
  const float* x = logits + (size_t)r * ld;
  const int off = (int)(((uintptr_t)x >> 2) & 3);
  const int batches = (int)(((long long)off + n + kLpBatch - 1) / kLpBatch);
  const int b0 = (int)((long long)batches * piece / pieces);
  const int b1 = (int)((long long)batches * (piece + 1) / pieces);

  // a lane holds ids 256 b + 4 lane - off .. + 3 of batch b, and the same 128 later
  auto load = [&](int b, float (&v)[kLpEach]) {
#pragma unroll
    for (int i = 0; i < kLpEach / 4; ++i) {
      const int e = b * kLpBatch + 128 * i + 4 * lane - off;
      if (e >= 0 && e + 4 <= n) {
        const float4 f = __ldcs(reinterpret_cast<const float4*>(x + e));
        v[4 * i] = f.x; v[4 * i + 1] = f.y; v[4 * i + 2] = f.z; v[4 * i + 3] = f.w;
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j) v[4 * i + j] = e + j >= 0 && e + j < n ? x[e + j] : -INFINITY;
      }
    }
  };

  float m = -INFINITY, ties = 0.0f;                      // m is the warp's
  uint64_t s2 = 0, t2 = 0;                               // two sums each of exp(z) and z exp(z)
  u64 list = 0, least = 0;                               // the warp's 32 largest, falling
  float bar = -INFINITY;                                 // a lower logit is not among the `top`
  float v[kLpEach], next[kLpEach];
  auto add = [&](const float (&y)[kLpEach]) {
#pragma unroll
    for (int k = 0; k < kLpEach; k += 2) {
      float2 z = unpair(add2(pair(y[k], y[k + 1]), pair(-m, -m)));
      z = make_float2(fmaxf(z.x, -200.0f), fmaxf(z.y, -200.0f));
      const float2 g = unpair(mul2(pair(z.x, z.y), pair(kLog2e, kLog2e)));
      const uint64_t e = pair(ex2f(g.x), ex2f(g.y));
      s2 = add2(s2, e);
      t2 = fma2(pair(z.x, z.y), e, t2);
    }
  };
  const int rounds = (b1 - b0 + kLpWarps - 1) / kLpWarps;
  const int given = threadIdx.x == 0 ? tok[r] : -1;
  const float given_x = given >= 0 && given < n ? x[given] : 0.0f;
  int meet = 1;                                          // the round after which lists meet
  if (b0 + warp < b1) load(b0 + warp, next);
  bool listed = false;                                   // the CTA's list is there already
  if constexpr (kTop) {
    const int id = (b0 + warp) * kLpBatch + 4 * lane - off, end = b0 + warp < b1 ? n : 0;
    if (block_first(next, id, end, top, sh, &list)) {
      if (rounds == 1) {
        listed = true;
        least = ~(u64)0;
        bar = INFINITY;
      } else {
        // the first batches are gone over again, now by a bound that `top` of the CTA's reach
        if (warp == 0 && lane == top - 1) sh.least = list - 1;
        __syncthreads();
        list = 0;
        least = sh.least;
        bar = lp_key_value(least);
        meet = 4;
      }
    }
  }
  for (int i = 0; i < rounds; ++i) {
    const int b = b0 + i * kLpWarps + warp;
    if (b < b1) {
#pragma unroll
      for (int k = 0; k < kLpEach; ++k) v[k] = next[k];
      if (b + kLpWarps < b1) load(b + kLpWarps, next);
      float mine = v[0];
#pragma unroll
      for (int k = 1; k < kLpEach; ++k) mine = max_nan(mine, v[k]);
      const bool usual = __all_sync(0xFFFFFFFFu, mine < m);
      if (kTop && __any_sync(0xFFFFFFFFu, !(mine < bar))) {
        list = warp_take(list, v, b * kLpBatch + 4 * lane - off, n, top, &least);
        bar = least ? lp_key_value(least) : -INFINITY;
      }
      if (usual) {                                       // nothing at the warp's maximum
        add(v);
      } else {
        float lm = mine;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) lm = max_nan(lm, __shfl_xor_sync(0xFFFFFFFFu, lm, o));
        if (lm != -INFINITY) {
          if (!(lm <= m)) {
            // what was summed counts less: S' = f (S + ties), T' = f (T + (m' - m)(S + ties))
            const float d = fmaxf(m - lm, -200.0f);
            const float f = m == -INFINITY ? 0.0f : ex2f(d * kLog2e);
            float2 s = unpair(s2), u = unpair(t2);
            s.x += ties;
            ties = 0.0f;
            u.x = f * fmaf(d, s.x, u.x);
            u.y = f * fmaf(d, s.y, u.y);
            s2 = pair(f * s.x, f * s.y);
            t2 = pair(u.x, u.y);
            m = max_nan(m, lm);
          }
#pragma unroll
          for (int k = 0; k < kLpEach; ++k)
            if (v[k] == m) {
              ties += 1.0f;
              v[k] = -INFINITY;                          // adds nothing below
            }
          add(v);
        }
      }
    }
    if (kTop && i + 1 == meet && meet < rounds) {
      // The warps' lists become one, warp 0's, whose `top`th bounds all of them from below.
      // While what has been seen grows fourfold, a few times `top` logits pass the bound.
      meet *= 4;
      list = block_merge(list, sh);
      if (warp == 0 && lane == top - 1) sh.least = list;
      if (warp > 0) list = 0;
      __syncthreads();
      least = max64(least, sh.least);
      bar = least ? lp_key_value(least) : -INFINITY;
    }
  }

  // the warp's sums, then the CTA's
  float s = unpair(s2).x + unpair(s2).y, t = -(unpair(t2).x + unpair(t2).y);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
    t += __shfl_xor_sync(0xFFFFFFFFu, t, o);
    ties += __shfl_xor_sync(0xFFFFFFFFu, ties, o);
  }
  if (lane == 0) sh.sums[warp] = LpSum{m, s + (ties - 1.0f), t};
  if (kTop && !listed) list = block_merge(list, sh);
  __syncthreads();
  if (warp > 0 && pieces == 1) return;
  LpSum sum = lane < kLpWarps ? sh.sums[lane] : LpSum{-INFINITY, 0.f, 0.f};
  auto warp_join = [&](LpSum a) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const LpSum b{__shfl_xor_sync(0xFFFFFFFFu, a.m, o), __shfl_xor_sync(0xFFFFFFFFu, a.s, o),
                    __shfl_xor_sync(0xFFFFFFFFu, a.t, o)};
      a = lane & o ? lp_join(b, a) : lp_join(a, b);      // the same bits in every lane
    }
    return a;
  };
  if (warp == 0) sum = warp_join(sum);

  if (pieces > 1) {
    if (warp == 0) {
      if (lane == 0) psum[(size_t)r * pieces + piece] = sum;
      if (kTop && lane < top) plist[((size_t)r * pieces + piece) * kMaxTop + lane] = list;
      __threadfence();
    }
    __syncthreads();
    if (threadIdx.x == 0) {
      sh.last = atomicAdd(ticket + r, 1u) == (unsigned)pieces - 1;
      if (sh.last) ticket[r] = 0;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    sum = LpSum{-INFINITY, 0.f, 0.f};
    if (warp == 0)
      for (int i = lane; i < pieces; i += 32) {
        const float* p = reinterpret_cast<const float*>(psum + (size_t)r * pieces + i);
        sum = lp_join(sum, LpSum{__ldcg(p), __ldcg(p + 1), __ldcg(p + 2)});
      }
    if constexpr (kTop) {
      list = 0;
#pragma unroll 4
      for (int i = warp; i < pieces; i += kLpWarps) {
        const u64 k = lane < top ? __ldcg(plist + ((size_t)r * pieces + i) * kMaxTop + lane) : 0;
        list = warp_merge(list, k);
      }
      list = block_merge(list, sh);
    }
    if (warp > 0) return;
    sum = warp_join(sum);
  }
  const float nan = __int_as_float(0x7fc00000), ls = log1pf(sum.s);
  const bool fine = fabsf(sum.m) <= FLT_MAX;             // not NaN, +inf, or all -inf
  if (lane == 0) {
    lp[r] = fine && given >= 0 && given < n ? (given_x - sum.m) - ls : nan;
    ent[r] = fine ? ls + sum.t / (1.0f + sum.s) : nan;
  }
  if (kTop && lane < top) {
    top_id[(size_t)r * top + lane] = (int)~(unsigned)list;
    top_lp[(size_t)r * top + lane] = fine ? (lp_key_value(list) - sum.m) - ls : nan;
  }
}

// CTAs per row: enough rows fill the SMs with one each; few rows are cut into pieces of whole
// tiles, as many as run at once. Without tiles to cut (or tickets) a row is one piece. Rows of
// 151936, in microseconds, whole and cut so: 16 rows 23.5 : 14.9, 37 24.6 : 18.3, 64 24.5 : 21.7,
// 100 25.0 : 27.6 (from 75 to about 110 rows the cut loses up to 10%), 128 29.2 : 27.7, 148
// 31.9 : 28.1; 200 whole 35.9, in two pieces 51.5.
int lp_pieces(int rows, int n, int* out, long long* most = nullptr) {
  int sms = 0;
  const int rc = sm_count(&sms);
  if (rc) return rc;
  const int tiles = (int)(((long long)n + 3 + kLpTile - 1) / kLpTile);
  const int cut = tiles < kLpPieces ? tiles : kLpPieces;
  int p = 2 * sms / rows;
  p = p < cut ? p : cut;
  *out = p < 1 || rows > kLpTickets ? 1 : p;
  // pieces of all rows together, for any number of rows up to `rows`
  if (most) {
    const long long all = (long long)rows * cut < 2ll * sms ? (long long)rows * cut : 2ll * sms;
    *most = all > rows ? all : rows;
  }
  return HV_OK;
}

size_t lp_up(size_t b) { return (b + 255) & ~(size_t)255; }

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_logprob_scratch(int rows, int n, int top, size_t* bytes) {
  HV_REQUIRE(rows > 0 && n > 0 && top >= 0 && bytes, HV_E_INVALID,
             "hv_logprob_scratch: bad arguments");
  HV_REQUIRE(top <= kMaxTop, HV_E_UNSUPPORTED, "hv_logprob_scratch: %d alternatives (at most %d)",
             top, kMaxTop);
  HV_REQUIRE(n <= 1 << 30, HV_E_UNSUPPORTED, "hv_logprob_scratch: %d tokens", n);
  int pieces = 0;
  long long most = 0;
  const int rc = lp_pieces(rows, n, &pieces, &most);
  if (rc) return rc;
  *bytes = kLpTickets * sizeof(unsigned) + lp_up((size_t)most * sizeof(LpSum)) +
           (size_t)most * (top ? kMaxTop : 0) * sizeof(u64);
  return HV_OK;
}

extern "C" int hv_logprob_rows(const float* logits, long long ld, int rows, int n,
                               const int32_t* tok, int top, float* lp, float* ent,
                               int32_t* top_id, float* top_lp, void* scratch, void* stream) {
  HV_REQUIRE(logits && tok && lp && ent && scratch && rows > 0 && n > 0 && top >= 0 &&
                 (top == 0 || (top_id && top_lp)),
             HV_E_INVALID, "hv_logprob_rows: bad arguments");
  HV_REQUIRE(ld >= n, HV_E_INVALID, "hv_logprob_rows: row stride %lld under %d", ld, n);
  HV_REQUIRE(n <= 1 << 30, HV_E_UNSUPPORTED, "hv_logprob_rows: %d tokens", n);
  HV_REQUIRE(top <= n, HV_E_INVALID, "hv_logprob_rows: %d alternatives of %d tokens", top, n);
  HV_REQUIRE(top <= kMaxTop, HV_E_UNSUPPORTED, "hv_logprob_rows: %d alternatives (at most %d)",
             top, kMaxTop);
  HV_REQUIRE(((uintptr_t)logits & 3) == 0 && ((uintptr_t)scratch & 15) == 0, HV_E_INVALID,
             "hv_logprob_rows: unaligned pointer");
  int pieces = 0;
  const int rc = lp_pieces(rows, n, &pieces);
  if (rc) return rc;
  HV_REQUIRE((long long)rows * pieces <= 0x7FFFFFFFll, HV_E_UNSUPPORTED,
             "hv_logprob_rows: %d rows at once", rows);
  uint8_t* p = static_cast<uint8_t*>(scratch);
  unsigned* ticket = reinterpret_cast<unsigned*>(p);
  p += kLpTickets * sizeof(unsigned);
  LpSum* psum = reinterpret_cast<LpSum*>(p);
  p += lp_up((size_t)rows * pieces * sizeof(LpSum));
  u64* plist = reinterpret_cast<u64*>(p);
  if (top)
    k_logprob<true><<<rows * pieces, kLpThreads, 0, (cudaStream_t)stream>>>(
        logits, (size_t)ld, n, tok, top, lp, ent, top_id, top_lp, pieces, psum, plist, ticket);
  else
    k_logprob<false><<<rows * pieces, kLpThreads, 0, (cudaStream_t)stream>>>(
        logits, (size_t)ld, n, tok, top, lp, ent, top_id, top_lp, pieces, psum, plist, ticket);
  HV_LAUNCHED("k_logprob");
}
