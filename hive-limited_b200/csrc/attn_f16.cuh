// What the attention kernels over a binary16 cache in an order of their own share: which
// positions a query row sees.
//
// A row sees a prefix, which every row of the call sees whole, and then part of a tail: the
// sequence's own positions, up to the row's. hv_attn_shared_f16 has a tail a sequence;
// hv_attn_decode_mass_f16 is one row and a prefix; hv_attn_rows_mass_f16 (`run`) is one cache
// without tails, of which row t sees plen + t + 1 positions.
#pragma once

#include <cuda.h>
#include <cuda_fp16.h>

#include "attn_q8.cuh"
#include "hv_internal.h"

namespace hv {

struct SpanArgs {
  const float* q;                      // [nrow][nq][128]
  float* ctx;
  const float* scale;
  const __half *pk, *pv;               // prefix: head after head, p_head elements apart
  const __half *tk, *tv;               // tails: sequences t_seq, heads t_head elements apart
  size_t p_head, t_seq, t_head;
  const int32_t* plen_p;               // prefix positions: *plen_p + plen, or plen
  const int32_t *row0, *tlen_p;        // rows row0[s] .. row0[s + 1] - 1 are sequence s's
  int plen, pmin, pcap, tlen, tcap;    // a prefix of pmin to pcap positions
  int nq, group, nseq, nrow;
  unsigned long long inv;              // 2^32 / group, rounded up: see span_row
  bool run;
};
// The row of pair f: f / group, exact for f under 2^29 (a division takes some thirty instructions,
// several of them in every kernel before its first load).
HV_DEV int span_row(const SpanArgs& a, int f) { return (int)(((unsigned long long)(unsigned)f * a.inv) >> 32); }

// Positions of the prefix; -1 if it cannot have that many.
HV_DEV int span_prefix(const SpanArgs& a) {
  const int n = a.plen + (a.plen_p ? __ldg(a.plen_p) : 0);
  return n < a.pmin || n > a.pcap ? -1 : n;
}

// Rows [row, end) of sequence s, whose first row sees `first` positions of its tail and every
// later one a position more. Without row0 a single sequence has all rows, several one each.
struct SpanSeq {
  int s, row, end, len;                // len: the tail's positions, -1 if it cannot hold them
  HV_DEV int sees(int r) const { return max(0, len - (end - 1 - r)); }
};
HV_DEV int span_row0(const SpanArgs& a, int s) {
  if (a.row0) return min(max(__ldg(a.row0 + s), 0), a.nrow);
  return a.nseq == 1 ? s * a.nrow : s;
}
HV_DEV SpanSeq span_seq(const SpanArgs& a, int s) {
  SpanSeq x;
  x.s = s;
  x.row = span_row0(a, s);
  x.end = span_row0(a, s + 1);
  x.len = a.tlen_p ? __ldg(a.tlen_p + s) : a.tlen;
  if (x.len < 0 || x.len > a.tcap) x.len = -1;
  return x;
}
// The sequence that row r belongs to; false if it lies behind the last one's rows. By a whole warp
// with the same r, 32 sequences looked at together: one after the other their loads would take
// longer than most of what follows.
HV_DEV bool span_find(const SpanArgs& a, int r, SpanSeq* x) {
  int s = a.nseq == 1 ? 0 : r;
  if (a.row0) {
    const int lane = threadIdx.x & 31;
    int lo = 0, n = a.nseq;            // the last sequence that starts at or before r is in [lo, lo + n)
    while (n > 1) {
      const int step = (n + 31) / 32, at = lo + lane * step;
      const bool before = lane * step < n && (lane == 0 || span_row0(a, at) <= r);
      const int k = 31 - __clz(__ballot_sync(0xFFFFFFFFu, before));
      lo += k * step;
      n = min(step, n - k * step);
    }
    s = lo;
  }
  if (s >= a.nseq) return false;
  *x = span_seq(a, s);
  return r >= x->row && r < x->end;
}

// The sequences' rows of a call in items of up to `size` (row, head) pairs each, as blocks of a grid:
// nseq + F / size of them, F = nrow * group. The first nseq have each sequence's first pairs; what a
// sequence has more starts, `size` further every time, in windows of `size` pairs of all, at most
// one start a window, and that of the sequence that has the window's first. Pairs [f0, f0 + nf) of
// sequence x; nf 0: nothing for this block.
constexpr int kSpanItem = 64, kFewRows = 8;
struct SpanItem {
  SpanSeq x;
  int f0, nf;
};
HV_DEV SpanItem span_item(const SpanArgs& a, int b, int size) {
  SpanItem it;
  it.nf = 0;
  if (b < a.nseq) {
    it.x = span_seq(a, b);
    it.f0 = it.x.row * a.group;
  } else {
    const int w = (b - a.nseq) * size;
    if (!span_find(a, span_row(a, w), &it.x)) return it;
    const int start = it.x.row * a.group;
    const int k = (w - start + size - 1) / size;
    it.f0 = start + k * size;
    if (k == 0) return it;
  }
  it.nf = min(size, it.x.end * a.group - it.f0);
  it.nf = max(it.nf, 0);
  return it;
}

// Positions of a chunk when n are cut into at most `most` chunks of whole stages.
constexpr int kSpanStage = 64;
HV_HD int span_chunk(int n, int most) {
  const int c = most == 1 ? n : (n + most - 1) / most;
  return (c + kSpanStage - 1) / kSpanStage * kSpanStage;
}

// What k_span_tile takes: a shared prefix, or all that a run's rows see, in tiles of kStRows
// positions. Units of work are (kv head, tile of kStRows (row, head) pairs, tile of positions),
// `tiles` of the last for every tile of rows (a run's first ones have fewer), cut evenly among `ctas`
// CTAs.
constexpr int kStRows = 128;
struct SpanWhole {
  unsigned units;
  int tiles, rows, ctas;
};
// Positions of the prefix (or cache) that pair f sees.
HV_DEV int span_sees(const SpanArgs& a, int np, int f) {
  return np < 0 ? 0 : a.run ? np + span_row(a, f) + 1 : np;
}
HV_DEV int span_tiles_of(const SpanArgs& a, int np, int tile) {
  const int last = min(a.nrow * a.group, (tile + 1) * kStRows) - 1;
  return (span_sees(a, np, last) + kStRows - 1) / kStRows;
}
// Where the tiles of rows are few enough, as many CTAs take each as there are SMs for: a CTA that
// ends one tile of rows and begins another pays for it about what three tiles of positions take.
HV_DEV SpanWhole span_whole(const SpanArgs& a, int np, int grid) {
  SpanWhole w;
  w.rows = (a.nrow * a.group + kStRows - 1) / kStRows;
  w.tiles = span_tiles_of(a, np, w.rows - 1);
  const unsigned all = (unsigned)(a.nq / a.group) * w.rows;
  w.units = all * w.tiles;                       // under 2^31: see span_plan
  w.ctas = (int)min((unsigned)grid, w.units);
  unsigned each = min((unsigned)grid / all, (unsigned)w.tiles);
  if (each > 0) {                                // no more than make the longest share shorter
    const unsigned most = (w.tiles + each - 1) / each;
    each = (w.tiles + most - 1) / most;
  }
  if (each > 0 && (w.tiles + each - 1) / each <= w.units / grid + 3) w.ctas = (int)(all * each);
  return w;
}
// CTA c's first unit, units * c / ctas, and the CTA that has unit u.
HV_DEV unsigned span_first(const SpanWhole& w, unsigned c) {
  const unsigned q = w.units / w.ctas, r = w.units - q * w.ctas;
  return q * c + r * c / w.ctas;
}
HV_DEV int span_cta(const SpanWhole& w, unsigned u) {
  int c = (int)((float)u * ((float)w.ctas / (float)w.units));      // one off at the most
  if (span_first(w, c) > u) --c;
  if (span_first(w, c + 1) <= u) ++c;
  return c;
}

// What the exponents of a row's weights are taken relative to where its scores are formed a second
// time, for a first time's m. From 2^26 on the two times differ by enough to be seen in any weight;
// what is added there keeps weights from passing 1, so that sums of them stay finite.
HV_DEV float span_top(float m) { return fabsf(m) > 67108864.0f ? m + fabsf(m) * 0x1p-20f : m; }

// Is one of eight halves an infinity or a NaN?
HV_DEV bool not_finite(const uint4& y) {
  auto odd = [](uint32_t z) { return (z & 0x7C00u) == 0x7C00u || (z & 0x7C000000u) == 0x7C000000u; };
  return odd(y.x) || odd(y.y) || odd(y.z) || odd(y.w);
}

// Kernels of a call may start before the one before them has ended: what they read of it, or write
// over, comes after prior_done. Each of them calls it, at its end at the latest, so that the end of
// one is the end of all before it. What an earlier kernel of the call writes is read by __ldcg, never
// by __ldg: that one is for what nobody writes as long as the kernel lives, and it began before.
HV_DEV void next_may_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
HV_DEV void prior_done() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
template <class... P, class... A>
cudaError_t launch_beside(void (*fn)(P...), dim3 grid, int threads, int smem, cudaStream_t st, bool beside, A... args) {
  cudaLaunchAttribute at{};
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = &at;
  cfg.numAttrs = beside ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, fn, (P)args...);
}

// Partial results in the caller's scratch, in slots: nwt for the stretches of k_span_tile (at most
// that many a tile of rows) or npc for the prefix's chunks, ntc for the tails'. part [slot][nkv][F][128], ml [slot][nkv][F]: sums and the sum of the weights 2^(x - m),
// relative to m.
struct SpanParts {
  float* part;
  float2* ml;
  int32_t* stretches;                  // [nkv][tiles of rows]: the slots that k_span_tile has used
  float2* stat;                        // [nkv][F]: m and the sum of all, for the weights' sake
  float* scores;                       // [nq][scores_ld], of a single row
  size_t scores_ld;
  // what k_mass_tile reads of the rows: their two binary16 terms [2][nkv][F][128]; and, F rounded
  // up to whole tiles, the factor and the term [2][nkv][..] that take their sums of products to
  // exponents of weights (-m - log2 l; -infinity behind F)
  __half* terms;
  float* facs;
  int nwt, npc, ntc, grid;             // grid: CTAs of k_span_tile
  int size;                            // pairs of a tile of the prefix's chunks and of an item
};

// Tensor copies of boxes of kStRows rows by 64 values of [outer][rows][128], rows of 128 bytes in
// shared memory, swizzled; rows past the end are zeros.
int f16_rows_map(const __half* base, int rows, int outer, CUtensorMap* out);
HV_DEV void tile_copy(uint32_t to, const CUtensorMap* map, int dim, int pos, int head, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4}], [%5];"
      :: "r"(to), "l"(map), "r"(dim), "r"(pos), "r"(head), "r"(bar) : "memory");
}
HV_DEV void bar_expect(uint32_t bar, int bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" :: "r"(bar), "r"(bytes) : "memory");
}

int span_tile_launch(const SpanArgs& a, const SpanParts& p, cudaStream_t st);
int mass_tile_launch(const SpanArgs& a, const SpanParts& p, const float* mass_in, float* mass_out, int cap,
                     cudaStream_t st);

}  // namespace hv
