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
#include <cfloat>

#include "hv_common.cuh"
#include "hv_internal.h"

namespace hv {
namespace {

constexpr int kMaxTop = 32;

// 64-bit key in np.argmax's order: the f32 bits mapped to an unsigned order, then ~id.
HV_DEV unsigned long long lp_key(float v, int id) {
  unsigned u = __float_as_uint(v);
  if (v != v) u = 0x7FC00000u;
  else if (v == 0.f) u = 0u;
  const unsigned ord = (u & 0x80000000u) ? ~u : (u | 0x80000000u);
  return ((unsigned long long)ord << 32) | (unsigned long long)(~(unsigned)id);
}

HV_DEV unsigned long long block_max64(unsigned long long v, unsigned long long* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long w = __shfl_xor_sync(0xFFFFFFFFu, v, o);
    v = w > v ? w : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  for (int i = 0; i < (int)blockDim.x / 32; ++i) v = s[i] > v ? s[i] : v;
  return v;
}

HV_DEV float block_sum(float v, float* s) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xFFFFFFFFu, v, o);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = 0.0f;
  for (int i = 0; i < (int)blockDim.x / 32; ++i) v += s[i];
  return v;
}

__global__ void __launch_bounds__(512) k_logprob(const float* __restrict__ logits, size_t ld,
                                                 int n, const int32_t* __restrict__ tok, int top,
                                                 float* __restrict__ lp, float* __restrict__ ent,
                                                 int32_t* __restrict__ top_id,
                                                 float* __restrict__ top_lp) {
  __shared__ unsigned long long s_k[16];
  __shared__ float s_f[16];
  const int r = blockIdx.x;
  const float* x = logits + (size_t)r * ld;
  unsigned long long best = 0;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const unsigned long long k = lp_key(x[i], i);
    best = k > best ? k : best;
  }
  best = block_max64(best, s_k);
  const int a = (int)~(unsigned)best;
  const float m = x[a];
  const bool fine = fabsf(m) <= FLT_MAX;       // not NaN, +inf, or all -inf
  float S = 0.0f, T = 0.0f;
  for (int i = threadIdx.x; i < n; i += blockDim.x) {
    const float z = x[i] - m, e = expf(z);
    if (i != a && e > 0.0f) { S += e; T -= z * e; }
  }
  S = block_sum(S, s_f);
  T = block_sum(T, s_f);
  const float nan = __int_as_float(0x7fc00000), ls = log1pf(S);
  if (threadIdx.x == 0) {
    const int t = tok[r];
    lp[r] = fine && t >= 0 && t < n ? (x[t] - m) - ls : nan;
    ent[r] = fine ? ls + T / (1.0f + S) : nan;
  }
  unsigned long long last = ~0ull;
  for (int j = 0; j < top; ++j) {
    unsigned long long b = 0;
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
      const unsigned long long k = lp_key(x[i], i);
      if (k < last && k > b) b = k;
    }
    last = block_max64(b, s_k);
    if (threadIdx.x == 0) {
      const int id = (int)~(unsigned)last;
      top_id[(size_t)r * top + j] = id;
      top_lp[(size_t)r * top + j] = fine ? (x[id] - m) - ls : nan;
    }
  }
}

}  // namespace
}  // namespace hv

using namespace hv;

extern "C" int hv_logprob_scratch(int rows, int n, int top, size_t* bytes) {
  HV_REQUIRE(rows > 0 && n > 0 && top >= 0 && bytes, HV_E_INVALID,
             "hv_logprob_scratch: bad arguments");
  HV_REQUIRE(top <= kMaxTop, HV_E_UNSUPPORTED, "hv_logprob_scratch: %d alternatives (at most %d)",
             top, kMaxTop);
  *bytes = 256;
  return HV_OK;
}

extern "C" int hv_logprob_rows(const float* logits, long long ld, int rows, int n,
                               const int32_t* tok, int top, float* lp, float* ent,
                               int32_t* top_id, float* top_lp, void* scratch, void* stream) {
  HV_REQUIRE(logits && tok && lp && ent && scratch && rows > 0 && n > 0 && top >= 0 &&
                 (top == 0 || (top_id && top_lp)),
             HV_E_INVALID, "hv_logprob_rows: bad arguments");
  HV_REQUIRE(ld >= n, HV_E_INVALID, "hv_logprob_rows: row stride %lld under %d", ld, n);
  HV_REQUIRE(top <= n, HV_E_INVALID, "hv_logprob_rows: %d alternatives of %d tokens", top, n);
  HV_REQUIRE(top <= kMaxTop, HV_E_UNSUPPORTED, "hv_logprob_rows: %d alternatives (at most %d)",
             top, kMaxTop);
  k_logprob<<<rows, 512, 0, (cudaStream_t)stream>>>(logits, (size_t)ld, n, tok, top, lp, ent,
                                                    top_id, top_lp);
  HV_LAUNCHED("k_logprob");
}
