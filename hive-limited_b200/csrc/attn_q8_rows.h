// What the kernels of hv_attn_rows_q8 share: their arguments, the scratch of a row tile's
// chunks, and which chunks there are.
#pragma once

#include "attn_q8.cuh"
#include "hv_internal.h"

namespace hv {

struct RowsArgs {
  const float* q;
  float* ctx;
  const float* scale;
  int pos0, ntok, nq, group, chunks;
  bool cluster;                           // a row tile's chunks are a cluster
  float* part;
};

// Floats of the scratch per (tile of n rows, chunk): their sums, then (max, sum of weights).
HV_HD size_t rows_part(int n) { return (size_t)n * (kHd + 2); }

// The chunks of a row tile that a launch has work for: `least` blocks each, at most a.chunks.
struct RowsSpan {
  int held, closed, nb, items, nact;      // nb coded blocks; items: with the open one
};
HV_DEV RowsSpan rows_span(const RowsArgs& a, const KvQ8& c, int kvh, int row0, int rows, int least) {
  RowsSpan s;
  const int last = min(a.ntok * a.group, row0 + rows) - 1;
  s.held = q8_held(c, kvh);
  s.closed = s.held / kQ8Blk;
  const int top = min(a.pos0 + last / a.group, s.held - 1);       // the last position to read
  s.nb = min(s.closed, top < 0 ? 0 : top / kQ8Blk + 1);
  s.items = s.nb + (top >= s.closed * kQ8Blk ? 1 : 0);
  s.nact = max(1, min(a.chunks, s.items / least));
  return s;
}

// The chunks of a row tile meet in shared memory when they are a cluster (at most eight CTAs):
// every CTA leaves its rows' sums, 128 floats each, and (max, sum of weights) in its own, and row
// r is added up by CTA r mod nact, which reads them all. Two cluster barriers: the first says that
// the sums are there, the second that they have been read. Every CTA of a cluster takes part in
// both, whatever it has to do, so that none is gone while another reads from it. (Sending the
// sums to where they are added up, in microseconds against this: decode over 8000 positions
// 9.6 : 9.3, 256 x 4 rows over 4096 44.2 : 43.0, 44 x 2 rows over 300 11.3 : 11.6.)
constexpr int kRowsCluster = 8;
HV_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
HV_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
HV_DEV void cluster_sync() { cluster_arrive(); cluster_wait(); }

HV_DEV uint32_t cluster_at(const void* x, int cta) {
  uint32_t r;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(x)), "r"(cta));
  return r;
}
// Rows at `sums`, `line` floats apart, with (max, sum) pairs at `ml`, the same places in every
// CTA; this one's to ctx, in chunk order: a warp per row, a lane per four dims.
HV_DEV void cluster_add_up(const RowsArgs& a, const float* sums, int line, const float* ml, int nact,
                           int kvh, int row0, int rows, int cta, int warp, int warps, int held) {
  const int lane = threadIdx.x & 31;
  for (int r = cta + nact * warp; r < rows; r += nact * warps) {
    const int gr = row0 + r;
    if (gr >= a.ntok * a.group) break;
    float m[kRowsCluster], l[kRowsCluster];
    float4 x[kRowsCluster];
#pragma unroll
    for (int j = 0; j < kRowsCluster; ++j) {
      if (j >= nact) continue;
      asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];"
                   : "=f"(m[j]), "=f"(l[j]) : "r"(cluster_at(ml + 2 * r, j)) : "memory");
      asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(x[j].x), "=f"(x[j].y), "=f"(x[j].z), "=f"(x[j].w)
                   : "r"(cluster_at(sums + (size_t)r * line + 4 * lane, j)) : "memory");
    }
    float M = -INFINITY, L = 0.0f;
#pragma unroll
    for (int j = 0; j < kRowsCluster; ++j)
      if (j < nact) M = fmaxf(M, m[j]);
    float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
    for (int j = 0; j < kRowsCluster; ++j) {
      if (j >= nact) continue;
      const float f = l[j] == 0.0f ? 0.0f : ex2(m[j] - M);   // 0: the row sees nothing of the chunk
      L += f * l[j];
      s.x += f * x[j].x; s.y += f * x[j].y; s.z += f * x[j].z; s.w += f * x[j].w;
    }
    const int tok = gr / a.group;
    const float inv = a.pos0 + tok >= held ? __int_as_float(0x7fc00000) : 1.0f / L;
    float* o = a.ctx + ((size_t)tok * a.nq + (size_t)kvh * a.group + gr - tok * a.group) * kHd;
    reinterpret_cast<float4*>(o)[lane] = make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
  }
}

constexpr int kTileLeast = 8;            // blocks of a chunk of the tile kernel at the least: two steps

inline cudaLaunchConfig_t rows_config(dim3 grid, int threads, int smem, int cluster,
                                      cudaLaunchAttribute* at, cudaStream_t st) {
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  at->id = cudaLaunchAttributeClusterDimension;
  at->val.clusterDim.x = cluster;
  at->val.clusterDim.y = at->val.clusterDim.z = 1;
  cfg.attrs = at;
  cfg.numAttrs = cluster > 1 ? 1 : 0;
  return cfg;
}
inline int rows_launch(void (*fn)(RowsArgs, KvQ8), dim3 grid, int threads, int smem, const RowsArgs& a,
                       const KvQ8& c, cudaStream_t st) {
  cudaLaunchAttribute at{};
  const cudaLaunchConfig_t cfg = rows_config(grid, threads, smem, a.cluster ? a.chunks : 1, &at, st);
  const cudaError_t e = cudaLaunchKernelEx(&cfg, fn, a, c);
  return e == cudaSuccess ? HV_OK : cuda_fail("hv_attn_rows_q8", e);
}

// Clusters of n CTAs of the tile kernel that run at once.
int attn_tile_q8_room(int n, int* room);
int attn_tile_q8_launch(const RowsArgs& a, const KvQ8& c, unsigned tiles, unsigned nkv,
                        cudaStream_t st);

}  // namespace hv
