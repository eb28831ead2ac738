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
// row r is added up by CTA r mod nact, and every chunk sends its sums there, 128 floats and
// (max, sum of weights) of row r to slot [chunk][r / nact] of a buffer that has no other use by
// then. Two cluster barriers: the first says that the buffers are free (a CTA arrives when it has
// done with its own), the second that all sums are in them. Every CTA of a cluster takes part in
// both, whatever it has to do, so that none is gone while another writes to it.
constexpr int kRowsCluster = 8;
HV_HD constexpr int rows_land_bytes(int rows) { return (rows + kRowsCluster - 1) * (kHd + 2) * 4; }
HV_DEV void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
HV_DEV void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }
HV_DEV void cluster_stay() { cluster_arrive(); cluster_wait(); cluster_arrive(); cluster_wait(); }

struct RowsLand {
  uint8_t* at;
  int nact, per;
  HV_DEV RowsLand(uint8_t* buf, int rows, int n) : at(buf), nact(n), per((rows + n - 1) / n) {}
  HV_DEV float* sums(int chunk, int k) const {
    return reinterpret_cast<float*>(at) + (size_t)(chunk * per + k) * kHd;
  }
  HV_DEV float* ml(int chunk, int k) const {
    return reinterpret_cast<float*>(at) + (size_t)nact * per * kHd + 2 * (chunk * per + k);
  }
  HV_DEV static uint32_t peer(const float* x, int cta) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;"
        : "=r"(r) : "r"((uint32_t)__cvta_generic_to_shared(x)), "r"(cta));
    return r;
  }
  HV_DEV void send_sums(int chunk, int r, int d4, float4 x) const {
    asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};"
                 :: "r"(peer(sums(chunk, r / nact) + 4 * d4, r % nact)), "f"(x.x), "f"(x.y),
                    "f"(x.z), "f"(x.w) : "memory");
  }
  HV_DEV void send_ml(int chunk, int r, float m, float l) const {
    asm volatile("st.shared::cluster.v2.f32 [%0], {%1, %2};"
                 :: "r"(peer(ml(chunk, r / nact), r % nact)), "f"(m), "f"(l) : "memory");
  }
  // This CTA's rows to ctx, in chunk order: a warp per row, a lane per four dims.
  HV_DEV void add_up(const RowsArgs& a, int kvh, int row0, int rows, int cta, int warp, int warps,
                     int lane, int held) const {
    for (int k = warp; k < per; k += warps) {
      const int r = k * nact + cta, gr = row0 + r;
      if (r >= rows || gr >= a.ntok * a.group) break;
      float M = -INFINITY, L = 0.0f;
      for (int j = 0; j < nact; ++j) M = fmaxf(M, ml(j, k)[0]);
      float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
      for (int j = 0; j < nact; ++j) {
        const float l = ml(j, k)[1];           // 0: the row sees nothing of the chunk
        const float f = l == 0.0f ? 0.0f : ex2(ml(j, k)[0] - M);
        const float4 x = reinterpret_cast<const float4*>(sums(j, k))[lane];
        L += f * l;
        s.x += f * x.x; s.y += f * x.y; s.z += f * x.z; s.w += f * x.w;
      }
      const int tok = gr / a.group;
      const float inv = a.pos0 + tok >= held ? __int_as_float(0x7fc00000) : 1.0f / L;
      float* o = a.ctx + ((size_t)tok * a.nq + (size_t)kvh * a.group + gr - tok * a.group) * kHd;
      reinterpret_cast<float4*>(o)[lane] = make_float4(s.x * inv, s.y * inv, s.z * inv, s.w * inv);
    }
  }
};

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
