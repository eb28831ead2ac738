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

// `fac` is shared memory for 2 nact kRows floats.
template <int kRows>
HV_DEV void rows_join(const RowsArgs& a, int kvh, size_t slot, int nact, int row0, int nrows,
                      int held, float* fac) {
  constexpr int kQuads = kHd / 4, kAhead = 4;
  const float* base = a.part + slot * rows_part(kRows);
  float2* ml = reinterpret_cast<float2*>(fac);             // [chunk][row]
  for (int i = threadIdx.x; i < nact * kRows; i += blockDim.x)
    ml[i] = __ldcg(reinterpret_cast<const float2*>(base + (i / kRows) * rows_part(kRows) + kRows * kHd) +
                   i % kRows);
  __syncthreads();
  // what a chunk's sums of a row are multiplied by; 0 where the row sees nothing of the chunk
  for (int r = threadIdx.x; r < kRows; r += blockDim.x) {
    float M = -INFINITY, L = 0.0f;
    for (int k = 0; k < nact; ++k) M = fmaxf(M, ml[k * kRows + r].x);
    for (int k = 0; k < nact; ++k) {
      const float2 x = ml[k * kRows + r];
      const float w = x.y == 0.0f ? 0.0f : ex2(x.x - M);
      L += w * x.y;
      ml[k * kRows + r].x = w;
    }
    ml[r].y = a.pos0 + (row0 + r) / a.group >= held ? __int_as_float(0x7fc00000) : 1.0f / L;
  }
  __syncthreads();
  const int n = min(kRows, nrows - row0) * kQuads;
  for (int i0 = threadIdx.x; i0 < n; i0 += kAhead * blockDim.x) {
    float4 s[kAhead];
#pragma unroll
    for (int u = 0; u < kAhead; ++u) s[u] = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 2
    for (int k = 0; k < nact; ++k) {
      const float4* p = reinterpret_cast<const float4*>(base + k * rows_part(kRows));
      float4 x[kAhead];
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * blockDim.x;
        x[u] = i < n ? __ldcg(p + i) : make_float4(0.f, 0.f, 0.f, 0.f);
      }
#pragma unroll
      for (int u = 0; u < kAhead; ++u) {
        const int i = i0 + u * blockDim.x;
        const float w = i < n ? ml[k * kRows + i / kQuads].x : 0.0f;
        s[u].x += w * x[u].x; s[u].y += w * x[u].y; s[u].z += w * x[u].z; s[u].w += w * x[u].w;
      }
    }
#pragma unroll
    for (int u = 0; u < kAhead; ++u) {
      const int i = i0 + u * blockDim.x, gr = row0 + i / kQuads;
      if (i >= n) break;
      const float f = ml[i / kQuads].y;
      float* o = a.ctx + ((size_t)(gr / a.group) * a.nq + (size_t)kvh * a.group + gr % a.group) * kHd;
      reinterpret_cast<float4*>(o)[i % kQuads] = make_float4(s[u].x * f, s[u].y * f, s[u].z * f, s[u].w * f);
    }
  }
}

int attn_tile_q8_launch(const RowsArgs& a, const KvQ8& c, unsigned tiles, unsigned nkv,
                        cudaStream_t st);

}  // namespace hv
