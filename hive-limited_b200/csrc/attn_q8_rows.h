// What the two kernels of hv_attn_rows_q8 share: their arguments, the scratch of a row tile's
// chunks, and how the last CTA of a row tile adds them.
#pragma once

#include "attn_q8.cuh"

namespace hv {

struct RowsArgs {
  const float* q;
  float* ctx;
  const float* scale;
  int pos0, ntok, nq, group, chunks;
  float* part;
  unsigned* ticket;
};

// Floats of the scratch per (tile of n rows, chunk): their sums, then (max, sum of weights).
HV_HD size_t rows_part(int n) { return (size_t)n * (kHd + 2); }

template <int kRows>
HV_DEV void rows_join(const RowsArgs& a, int kvh, size_t slot, int nact, int row0, int nrows,
                      int held) {
  const float* base = a.part + slot * rows_part(kRows);
  for (int i = threadIdx.x; i < kRows * (kHd / 4); i += blockDim.x) {
    const int r = i / (kHd / 4), d4 = i % (kHd / 4), gr = row0 + r;
    if (gr >= nrows) break;
    float M = -INFINITY, L = 0.0f;
    float4 A = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < nact; ++k)
      M = fmaxf(M, __ldcg(base + k * rows_part(kRows) + kRows * kHd + 2 * r));
    for (int k = 0; k < nact; ++k) {
      const float* p = base + k * rows_part(kRows);
      const float2 ml = __ldcg(reinterpret_cast<const float2*>(p + kRows * kHd + 2 * r));
      if (ml.y == 0.0f) continue;                 // this row sees nothing of the chunk
      const float w = ex2(ml.x - M);
      const float4 x = __ldcg(reinterpret_cast<const float4*>(p + (size_t)r * kHd) + d4);
      L += w * ml.y;
      A.x += w * x.x; A.y += w * x.y; A.z += w * x.z; A.w += w * x.w;
    }
    const float inv = a.pos0 + gr / a.group >= held ? __int_as_float(0x7fc00000) : 1.0f / L;
    float* o = a.ctx + ((size_t)(gr / a.group) * a.nq + (size_t)kvh * a.group + gr % a.group) * kHd;
    reinterpret_cast<float4*>(o)[d4] = make_float4(A.x * inv, A.y * inv, A.z * inv, A.w * inv);
  }
}

int attn_tile_q8_launch(const RowsArgs& a, const KvQ8& c, unsigned tiles, unsigned nkv,
                        cudaStream_t st);

}  // namespace hv
