// What the kernels of hv_attn_rows_q8 share: their arguments, the scratch of a row tile's
// chunks, and which chunks there are.
#pragma once

#include "attn_q8.cuh"

namespace hv {

struct RowsArgs {
  const float* q;
  float* ctx;
  const float* scale;
  int pos0, ntok, nq, group, chunks;
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

constexpr int kTileLeast = 8;            // blocks of a chunk of the tile kernel at the least

int attn_tile_q8_launch(const RowsArgs& a, const KvQ8& c, unsigned tiles, unsigned nkv,
                        cudaStream_t st);

}  // namespace hv
