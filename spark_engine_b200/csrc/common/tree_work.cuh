// What the kernels of tree attention share: arguments, the division of the work, visibility, the merge of split rows.
//
// The (row, head) pairs of a request and a key / value head are numbered node by node and cut into tiles of bm = 2^bm_log; a tile's keys are the pages
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

// two fp32 at a time
__device__ __forceinline__ uint64_t ta_two(float x, float y) { return static_cast<uint64_t>(__float_as_uint(y)) << 32 | __float_as_uint(x); }
__device__ __forceinline__ float ta_lo(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v)); }
__device__ __forceinline__ float ta_hi(uint64_t v) { return __uint_as_float(static_cast<uint32_t>(v >> 32)); }
__device__ __forceinline__ uint64_t ta_fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t ta_add2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t ta_mul2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ int ta_first_visible(const TreeAttn& a, int p) {
  // (p / chunk as a product: chunk_mul = ceil(2^chunk_shift / chunk) is exact for all p below 2^31)
  return a.chunk > 0 ? static_cast<int>(static_cast<unsigned long long>(p) * a.chunk_mul >> a.chunk_shift) * a.chunk : (a.window > 0 ? max(p - a.window + 1, 0) : 0);
}

struct TreeSeg {                         // a request's share of the work
  int r0, n, len, j0, nt, rts;           // first row, rows, committed tokens, first page, pages, row tiles
};
// (not inlined, like all that is done once per item: the first run of every instruction waits for memory)
static __device__ __noinline__ TreeSeg ta_segment(const TreeAttn& a, int s) {
  TreeSeg t;
  t.r0 = a.starts[s];
  t.n = a.starts[s + 1] - t.r0;
  const int most = a.page_ld * TA_PAGE;                      // (what lies behind the table's last page is not there)
  t.len = min(max(a.lengths[s], 0), most);
  if (t.n > 0 && t.len + t.n > most) set_status(a.status, ST_BOUNDS, t.r0, t.len + t.n, most);
  t.j0 = min(ta_first_visible(a, t.len) / TA_PAGE, a.page_ld - 1);
  t.nt = max(min((t.len + t.n + TA_PAGE - 1) / TA_PAGE, a.page_ld) - t.j0, 1);
  t.rts = t.n > 0 ? (t.n * (a.H / a.G) + (1 << a.bm_log) - 1) >> a.bm_log : 0;
  return t;
}
// (the caller of the kernel sees to it that all of them together are below 2^31)
__device__ __forceinline__ int ta_tiles(const TreeAttn& a, const TreeSeg& t) { return a.G * t.rts * (t.nt + a.extra); }

// Exclusive prefix over the block; every thread calls it.  sh: [NT / 32].
template <int NT>
__device__ __forceinline__ int ta_prefix(int v, int* sh, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[w] = x;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int i = 0; i < NT / 32; ++i) {
    const int y = sh[i];
    if (i < w) before += y;
    total += y;
  }
  return before + x - v;
}

struct TreeRange { TreeSeg seg; int s, rem, count, per; };    // request, pages into it, pages of this CTA, pages of every CTA
// Called by one whole warp.
__device__ __forceinline__ TreeRange ta_range(const TreeAttn& a) {
  const int lane = threadIdx.x & 31, each = (a.S + 31) >> 5, s0 = lane * each;         // a lane's requests
  int mine = 0;
  TreeSeg seg = {};
#pragma unroll 1
  for (int s = s0; s < min(s0 + each, a.S); ++s) { seg = ta_segment(a, s); mine += ta_tiles(a, seg); }
  int x = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  const int total = __shfl_sync(0xffffffffu, x, 31);
  TreeRange r;
  r.per = max(static_cast<int>((static_cast<unsigned>(total) + a.ctas - 1) / a.ctas), 1);
  const long long begin = static_cast<long long>(r.per) * blockIdx.x;
  r.count = begin < total ? min(total - static_cast<int>(begin), r.per) : 0;
  if (r.count == 0) return r;
  const int owner = __ffs(__ballot_sync(0xffffffffu, x > static_cast<int>(begin))) - 1;
  int s = s0, rem = static_cast<int>(begin) - (x - mine);
  if (lane == owner && each > 1) {
#pragma unroll 1
    for (;; ++s) {
      seg = ta_segment(a, s);
      const int n = ta_tiles(a, seg);
      if (rem < n) break;
      rem -= n;
    }
  }
  const auto from = [&](int v) { return __shfl_sync(0xffffffffu, v, owner); };
  r.s = from(s);
  r.rem = from(rem);
  r.seg = {from(seg.r0), from(seg.n), from(seg.len), from(seg.j0), from(seg.nt), from(seg.rts)};
  return r;
}

struct __align__(16) TreeItem {          // a row tile of one key / value head and this CTA's pages of it
  int r0, n, len, slot;                  // request: first row, rows, committed tokens, row of the tables
  int g, rt, j, nj;                      // head, tile, first page, pages (0: there is no further item)
  int edge, first, last, parts;          // from this token on every row sees committed tokens; the item begins / ends in this CTA; CTAs that
};                                       // share it (known to the one it begins in)
// The next item of the range; false at its end.
__device__ __forceinline__ bool ta_next(const TreeAttn& a, TreeRange& r, TreeItem& it) {
#pragma unroll 1
  while (r.count > 0) {
#pragma unroll 1
    while (r.rem >= ta_tiles(a, r.seg)) {                    // (the range ends with the last request's tiles)
      r.rem -= ta_tiles(a, r.seg);
      r.seg = ta_segment(a, ++r.s);
    }
    const int nt = r.seg.nt, all = nt + a.extra, i = static_cast<int>(static_cast<unsigned>(r.rem) / static_cast<unsigned>(all)), at = r.rem - i * all;
    const int take = min(r.count, all - at), off = max(at - a.extra, 0), end = at + take - a.extra;
    r.count -= take;
    r.rem += take;
    if (end <= off) continue;                                // the range ends in front of the item's first page
    it.r0 = r.seg.r0;
    it.n = r.seg.n;
    it.len = r.seg.len;
    it.slot = a.slots ? a.slots[r.s] : r.s;
    it.edge = ta_first_visible(a, r.seg.len + r.seg.n - 1);
    it.g = static_cast<int>(static_cast<unsigned>(i) / static_cast<unsigned>(r.seg.rts));
    it.rt = i - it.g * r.seg.rts;
    it.j = r.seg.j0 + off;
    it.nj = end - off;
    it.first = off == 0;
    it.last = end == nt;
    it.parts = 1 + static_cast<int>(static_cast<unsigned>(nt - end + r.per - 1) / static_cast<unsigned>(r.per));
    return true;
  }
  it.nj = 0;
  return false;
}
// What the second launch needs of an item: (parts, first row of the request, head, first pair and pairs of the tile).
__device__ __forceinline__ int4 ta_split(const TreeAttn& a, const TreeItem& it) {
  const int bm = 1 << a.bm_log, pairs = it.n * (a.H / a.G) - it.rt * bm;
  return make_int4(it.parts | min(pairs, bm) << 16, it.r0, it.g, it.rt * bm);
}

// Columns 8 c8 .. + 8 of a row of part p: the rows of a part lie side by side, 32 bytes each, so that threads that have a row each write whole
// lines (with rows one behind the other 64 requests of 64 nodes took 14 us more, windows of 1024 4.5 more).
__device__ __forceinline__ float* ta_part(const TreeAttn& a, size_t p, int row, int c8) {
  return a.part_o + (p << a.bm_log) * a.V + ((static_cast<size_t>(c8) << a.bm_log) + row) * 8;
}

__device__ __forceinline__ void ta_set_split(const TreeAttn& a, int4 v) { reinterpret_cast<int4*>(a.split)[blockIdx.x] = v; }
__device__ __forceinline__ int4 ta_get_split(const TreeAttn& a, int c) { return __ldcg(reinterpret_cast<const int4*>(a.split) + c); }

// exponential of the outputs' accuracy
template <typename T> __device__ __forceinline__ float ta_exp(float x) { return sizeof(T) == 2 ? __expf(x) : expf(x); }
// The sum of a row (against its maximum m) with a sink; what its outputs shrink by.
template <typename T>
__device__ __forceinline__ float ta_sink(float sink, float m, float& l) {
  const float top = fmaxf(m, sink), ref = top == -INFINITY ? 0.f : top, k = ta_exp<T>(m - ref);
  l = l * k + ta_exp<T>(sink - ref);
  return k;
}
template <typename T>
__device__ __forceinline__ float ta_head_factor(const TreeAttn& a, int row, int h) {
  return a.gate ? a.out_scale * sigmoid_f(ldf(static_cast<const T*>(a.gate) + static_cast<size_t>(row) * a.ldg + h)) : a.out_scale;
}
// Cache page of a request's page j (-1: the table does not lead anywhere).
__device__ __forceinline__ int ta_page(const TreeAttn& a, int slot, int j) {
  const int p = slot >= 0 && slot < a.n_slots && j < a.page_ld ? a.pages[static_cast<size_t>(slot) * a.page_ld + j] : -1;
  return p < a.n_pages ? p : -1;
}

// Bits b .. b + 63 of a row's ancestors.
__device__ __forceinline__ uint64_t ta_ancestors(const TreeAttn& a, const TreeItem& sg, int node, int b) {
  if (a.anc) {
    const uint32_t* w = a.anc + static_cast<size_t>(sg.r0 + node) * a.words;
    const int k = b >> 5, sh = b & 31;
    const uint64_t w0 = k < a.words ? w[k] : 0u, w1 = k + 1 < a.words ? w[k + 1] : 0u, w2 = k + 2 < a.words ? w[k + 2] : 0u;
    const uint64_t t = (w0 | w1 << 32) >> sh;
    return sh ? t | w2 << (64 - sh) : t;
  }
  const int n = node - b + 1;
  return n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
}
// Which of the 64 tokens from tok0 on row `node` (position p) sees; near: its ancestors 0 .. 63.
__device__ __forceinline__ uint64_t ta_mask(const TreeAttn& a, const TreeItem& sg, int tok0, int node, int p, uint64_t near) {
  const int first = ta_first_visible(a, p), i0 = tok0 - sg.len;        // the page's token 0 is node i0
  const int lo = min(max(first - tok0, 0), 64), hi = min(max(-i0, 0), 64);
  uint64_t m = hi > lo ? (hi == 64 ? ~0ull : (1ull << hi) - 1) & ~(lo == 0 ? 0ull : (1ull << lo) - 1) : 0ull;
  if (hi == 64) return m;
  const int b0 = max(i0, 0);                                 // bit b of t: node b0 + b
  uint64_t t = b0 == 0 ? near : sg.n <= 64 ? (b0 < 64 ? near >> b0 : 0ull) : ta_ancestors(a, sg, node, b0);
  const int left = sg.n - b0;                                // nodes there are
  if (left < 64) t &= left <= 0 ? 0ull : (1ull << left) - 1;
  if (first > sg.len)                                        // ancestors outside the window or chunk
    for (uint64_t x = t; x; x &= x - 1) {
      const int b = __ffsll(x) - 1;
      if (a.pos[sg.r0 + b0 + b] < first) t &= ~(1ull << b);
    }
  return m | t << hi;
}

}  // namespace spark
