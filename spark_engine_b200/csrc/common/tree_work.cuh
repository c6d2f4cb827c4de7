// What the kernels of tree attention share: arguments, the division of the work, visibility, the merge of split rows.
//
// The (row, head) pairs of a request and a key / value head are numbered node by node and cut into tiles of `bm`; a tile's keys are the pages
// from the first one that any of its rows can see to the request's last node.  All (request, head, tile) items together are `total` pages,
// and CTA c of the grid takes the same number of consecutive ones as every other: lengths may differ as they like, the host needs to know
// none of them, and a captured launch may be replayed with others.  To begin an item costs as much as `extra` pages (queries in, results out):
// it counts as that many more, in front of its own, so that a CTA which ends one item and begins another is not the last to finish.  An item
// that ends in another CTA than it began leaves partial results (sums, maxima) that a second launch joins in ascending order.
#pragma once
#include "rows.cuh"
#include "tree_args.h"

namespace spark {

constexpr int TA_PAGE = TREE_PAGE;
constexpr float TA_LOG2E = 1.4426950408889634f, TA_LN2 = 0.6931471805599453f;

__device__ __forceinline__ int ta_first_visible(const TreeAttn& a, int p) {
  return a.chunk > 0 ? p / a.chunk * a.chunk : (a.window > 0 ? max(p - a.window + 1, 0) : 0);
}

struct TreeSeg {                         // a request's share of the work
  int r0, n, len, j0, nt, rts;           // first row, rows, committed tokens, first page, pages, row tiles
};
__device__ __forceinline__ TreeSeg ta_segment(const TreeAttn& a, int s) {
  TreeSeg t;
  t.r0 = a.starts[s];
  t.n = a.starts[s + 1] - t.r0;
  t.len = max(a.lengths[s], 0);
  t.j0 = ta_first_visible(a, t.len) / TA_PAGE;
  t.nt = (t.len + t.n + TA_PAGE - 1) / TA_PAGE - t.j0;
  t.rts = t.n > 0 ? (t.n * (a.H / a.G) + a.bm - 1) / a.bm : 0;
  return t;
}
__device__ __forceinline__ long long ta_tiles(const TreeAttn& a, const TreeSeg& t) { return static_cast<long long>(a.G) * t.rts * (t.nt + a.extra); }

// Exclusive prefix over the block; every thread calls it.  sh: [NT / 32].
template <int NT>
__device__ __forceinline__ long long ta_prefix(long long v, long long* sh, long long& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const long long y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[w] = x;
  __syncthreads();
  long long before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    const long long y = sh[i];
    if (i < w) before += y;
    total += y;
  }
  __syncthreads();
  return before + x - v;
}

struct TreeRange { long long rem, count, per; int s; };       // pages into request s, pages of this CTA, pages of every CTA
template <int NT>
__device__ __forceinline__ TreeRange ta_range(const TreeAttn& a, long long* sh) {      // sh: [NT / 32 + 2]
  const int each = (a.S + NT - 1) / NT, s0 = threadIdx.x * each;                       // a thread's requests
  long long mine = 0, total;
  for (int s = s0; s < min(s0 + each, a.S); ++s) mine += ta_tiles(a, ta_segment(a, s));
  long long before = ta_prefix<NT>(mine, sh, total);
  TreeRange r;
  r.per = (total + a.ctas - 1) / a.ctas;
  if (r.per < a.min_tiles) r.per = a.min_tiles;
  const long long begin = r.per * blockIdx.x;
  r.count = begin < total ? (total - begin < r.per ? total - begin : r.per) : 0;
  long long* found = sh + NT / 32;
  if (r.count > 0 && before <= begin && begin < before + mine) {
    for (int s = s0;; ++s) {
      const long long n = ta_tiles(a, ta_segment(a, s));
      if (begin < before + n) { found[0] = s; found[1] = begin - before; break; }
      before += n;
    }
  }
  __syncthreads();
  r.s = r.count > 0 ? static_cast<int>(found[0]) : 0;
  r.rem = r.count > 0 ? found[1] : 0;
  return r;
}

struct TreeItem {                        // a row tile of one key / value head and this CTA's pages of it
  TreeSeg seg;
  int s, g, rt, j, nj;                   // request, head, tile, first page, pages
  bool first, last;                      // it begins / ends in this CTA
  int parts;                             // CTAs that share it (known to the one it begins in)
};
// The next item of the range; false at its end.
__device__ __forceinline__ bool ta_next(const TreeAttn& a, TreeRange& r, TreeItem& it) {
  while (r.count > 0) {
    it.seg = ta_segment(a, r.s);
    while (r.rem >= ta_tiles(a, it.seg)) {                   // (the range ends with the last request's tiles)
      r.rem -= ta_tiles(a, it.seg);
      it.seg = ta_segment(a, ++r.s);
    }
    const int nt = it.seg.nt, all = nt + a.extra, i = static_cast<int>(r.rem / all), at = static_cast<int>(r.rem - static_cast<long long>(i) * all);
    const int take = r.count < all - at ? static_cast<int>(r.count) : all - at;
    const int off = at > a.extra ? at - a.extra : 0, end = at + take - a.extra;
    r.count -= take;
    r.rem += take;
    if (end <= off) continue;                                // the range ends in front of the item's first page
    it.s = r.s;
    it.g = i / it.seg.rts;
    it.rt = i - it.g * it.seg.rts;
    it.j = it.seg.j0 + off;
    it.nj = end - off;
    it.first = off == 0;
    it.last = end == nt;
    it.parts = 1 + static_cast<int>((nt - end + r.per - 1) / r.per);
    return true;
  }
  return false;
}
// What the second launch needs of an item: (parts, first row of the request, head, first pair and pairs of the tile).
__device__ __forceinline__ int4 ta_split(const TreeAttn& a, const TreeItem& it) {
  const int pairs = it.seg.n * (a.H / a.G) - it.rt * a.bm;
  return make_int4(it.parts | (pairs < a.bm ? pairs : a.bm) << 16, it.seg.r0, it.g, it.rt * a.bm);
}

__device__ __forceinline__ void ta_set_split(const TreeAttn& a, int4 v) { reinterpret_cast<int4*>(a.split)[blockIdx.x] = v; }
__device__ __forceinline__ int4 ta_get_split(const TreeAttn& a, int c) { return __ldcg(reinterpret_cast<const int4*>(a.split) + c); }

template <typename T>
__device__ __forceinline__ float ta_head_factor(const TreeAttn& a, int row, int h) {
  return a.gate ? a.out_scale * sigmoid_f(ldf(static_cast<const T*>(a.gate) + static_cast<size_t>(row) * a.ldg + h)) : a.out_scale;
}
// Cache page of a request's page j (-1: the table does not lead anywhere).
__device__ __forceinline__ int ta_page(const TreeAttn& a, int slot, int j) {
  const int p = slot >= 0 && slot < a.n_slots && j < a.page_ld ? a.pages[static_cast<size_t>(slot) * a.page_ld + j] : -1;
  return p < a.n_pages ? p : -1;
}

}  // namespace spark
