// Tree attention on tcgen05 (bf16 caches): the tiles of tree_attn.cu with 128 (node, head) rows per accumulator, a page of keys per step.
//   warp 0      finds this CTA's items and announces them; TMA: pages of keys and values into a ring of slots in the order the products use
//               them (K0 K1 V0 K2 V1 ..)
//   warp 1      issues S = Q K^T one page ahead of O += P V (P in tensor memory), into the place whose weights the product has read
//   the others  softmax, one row per thread: 64 scores are one tensor-memory load, statistics stay in the thread
// NQ = 2: two tiles of 128 rows with their own issuing and softmax warps share the keys in shared memory (large trees: a page is read once for
// 256 rows); each tile's products wait for its own softmax alone.
//
// Weights are exponentials against a reference that may lag far behind the maximum: the maximum of the first page that a row sees, renewed
// (and the accumulator rescaled) only when a page's weights add up to more than 2^40; fp32 sums and bf16 weights lose nothing by a common
// factor.  So most pages need no maximum.  Weights enter the product as two bf16 terms (2^-17 of a weight is lost), as in all paged attention
// here: what a round of drafts is verified with does not depend on how large their trees are.  (One term, half a step of bf16 per weight,
// makes the error of 64 requests of 64 nodes over 4k tokens 1.4 times that of the rounded outputs, and the call 321 us instead of 378.)
// A page's weights take the place of its scores, and two such places alternate, so that they need not wait for the product of the page
// before (398 us with weights in one place beside the scores).  (A visible value of infinity times two terms, of either sign or 0, may be NaN where
// the definition has infinity.)
//
// A page that not every row sees whole (the tree itself, the edge of a window or chunk) is masked by 64 bits per row.  Warp 1 looks its values
// over first: rows that hold no token of the request are zeroed, and where a value is not finite, 0 * value would spoil the rows that do not
// see it, so the softmax warps add it by hand for the rows that do and zero it in front of the product.
//
// What bounds it (kernel time, inputs from HBM): few rows over long caches stream at 6.1 TB/s between the first page and the last, about 8 us
// after the launch (four requests of 16 nodes over 16k tokens, two heads of 256 of 8 each: 132 MB in 41 us); 256 rows are bound by the products of
// a page, 1536 clocks, and its exponentials, 1024, which overlap in part (64 requests of 64 nodes over 4k tokens, 8 heads of 128 of 4 each: 272 GFLOP
// in 369 us, 450 at the clock that 1000 W leave after seconds; the tensor pipe is active in 53 % of the clocks, issue slots in 39 %).  Short calls
// are the latency of what is done once: 10 us for 8 nodes over 900 tokens.  What did not pay (measured with weights of one term): the two tiles'
// softmax in turn (412 us instead of 363), results through shared memory (no change), an earlier start of the second launch (no change).
#include "../common/tree_work.cuh"

namespace spark {

int make_tmap_page(CUtensorMap* m, const void* base, uint64_t pages, uint64_t G, uint64_t D, uint64_t tok, uint64_t page);

constexpr float TC_MOST = 1099511627776.f;                   // 2^40
constexpr int TC_ITEMS = 16;                                 // items announced at a time

template <int DC, int NQ> struct Tc {
  static constexpr bool QT = DC == 256;                      // queries in tensor memory: shared memory has no room for them beside the ring
  static constexpr int SLOT = TA_PAGE * DC * 2, Q_BYTES = QT ? 0 : 128 * DC * 2;
  static constexpr int SLOTS = DC == 256 ? 6 : DC == 128 ? (NQ == 2 ? 9 : 4) : (NQ == 2 ? 16 : 8);
  static constexpr int BARS = 2 * SLOTS + 11 * NQ + 2 * TC_ITEMS;
  static constexpr int SMEM = 1024 + NQ * Q_BYTES + SLOTS * SLOT + BARS * 8 + 16 + TC_ITEMS * static_cast<int>(sizeof(TreeItem)) + 4 + SLOTS * 8;
  // per tile: two places of 64 columns, a page's scores and then its weights (high and low terms, 32 columns each), and the accumulator
  static constexpr int TILE_COLS = 128 + DC, Q_COL = 128 + DC;
  static constexpr int COLS = QT || NQ == 2 ? 512 : 256;
  static constexpr int SOFTMAX = 1 + NQ, WARPS = SOFTMAX + 4 * NQ, THREADS = WARPS * 32, PER_SM = QT || NQ == 2 ? 1 : 2;
  static_assert(NQ * TILE_COLS + (QT ? DC / 2 : 0) <= COLS && SMEM <= 232448, "tensor memory, shared memory");
};

__device__ __forceinline__ uint32_t tc_ld1(uint32_t taddr) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(r) : "r"(taddr) : "memory");
  tmem_ld_wait();
  return r;
}
__device__ __forceinline__ void tc_st1(uint32_t taddr, uint32_t v) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(taddr), "r"(v) : "memory");
  tmem_st_wait();
}
__device__ __forceinline__ void tc_load_page(void* dst, const CUtensorMap* m, uint64_t* bar, int c, int head, int page) {
  asm volatile("cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
               ::"r"(smem_u32(dst)), "l"(reinterpret_cast<uint64_t>(m)), "r"(smem_u32(bar)), "r"(c), "r"(head), "r"(0), "r"(page) : "memory");
}
__device__ __forceinline__ uint32_t tc_pack(float a, float b) {
  const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// N-major operand, 128-byte swizzle: 64 n are a 128-byte row per k; chunks of 64 n `chunk` bytes apart, groups of 8 k 1024 bytes
__device__ __forceinline__ uint64_t tc_desc_nmajor(uint32_t addr, uint32_t chunk) {
  return static_cast<uint64_t>((addr & 0x3FFFF) >> 4) | static_cast<uint64_t>(chunk >> 4) << 16 | static_cast<uint64_t>(1024 >> 4) << 32 |
         static_cast<uint64_t>(1) << 46 | static_cast<uint64_t>(2) << 61;
}
__device__ __forceinline__ float tc_ex2(float x) {          // relative error 2^-22, results below 2^-126 are 0
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ void tc_set(float (&s)[64], int i, uint64_t v) { s[i] = ta_lo(v); s[i + 1] = ta_hi(v); }
__device__ __forceinline__ float tc_rcp(float x) {          // relative error 2^-23
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// A wait that ends: each try may suspend the thread for 20 us, a hundred thousand of them are two seconds.
__device__ __forceinline__ bool tc_wait(uint64_t* bar, uint32_t parity) {
  uint32_t ok = 0;
#pragma unroll 1
  for (int i = 0; i < 100000 && !ok; ++i)
    asm volatile(
        "{\n"
        ".reg .pred P;\n"
        "mbarrier.try_wait.parity.shared::cta.b64 P, [%1], %2, 20000;\n"
        "selp.u32 %0, 1, 0, P;\n"
        "}\n" : "=r"(ok) : "r"(smem_u32(bar)), "r"(parity) : "memory");
  return __all_sync(0xffffffffu, ok);
}
// All softmax warps of the item (4 or 8): a barrier whose wait ends.
__device__ __forceinline__ bool tc_sync(uint64_t* bar, uint32_t& phase) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
  const bool ok = tc_wait(bar, phase);
  phase ^= 1u;
  return ok;
}

struct TcCount { int slot = 0; uint32_t ph = 0; };
template <int N> __device__ __forceinline__ void tc_step(TcCount& c) { if (++c.slot == N) { c.slot = 0; c.ph ^= 1; } }

// grid: a.ctas.  FEAT: soft cap, distance bias or slopes, or a scale that is not positive (the scaled scores are then masked, not the products).
template <int DC, int NQ, bool FEAT>
__global__ void __launch_bounds__(Tc<DC, NQ>::THREADS, Tc<DC, NQ>::PER_SM)
tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TreeAttn a) {
  using L = Tc<DC, NQ>;
  constexpr int SLOT = L::SLOT, SLOTS = L::SLOTS, KV_CHUNK = TA_PAGE * 128, Q_CHUNK = 128 * 128;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + NQ * L::Q_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + SLOTS * SLOT);
  uint64_t* empty = full + SLOTS;
  uint64_t* q_full = empty + SLOTS;                          // [NQ]
  uint64_t* s_full = q_full + NQ;                            // [NQ][2], like the next two: of the place
  uint64_t* p_full = s_full + 2 * NQ;
  uint64_t* o_full = p_full + 2 * NQ;
  uint64_t* v_seen = o_full + 2 * NQ;                        // warp 1 has looked over a masked page's values
  uint64_t* v_read = v_seen + NQ;                            // the tile's softmax warps know of it (tile 1 may be masked pages behind tile 0)
  uint64_t* v_sync = v_read + NQ;                            // [NQ]: of 4 and of 8 softmax warps
  uint64_t* drained = v_sync + NQ;                           // [NQ]: the tile's products have all ended
  uint64_t* item_full = drained + NQ;                        // [TC_ITEMS]
  uint64_t* item_read = item_full + TC_ITEMS;                // [TC_ITEMS]: by every warp but the producer
  TreeItem* items = reinterpret_cast<TreeItem*>((reinterpret_cast<uintptr_t>(ring + SLOTS * SLOT + L::BARS * 8) + 15) & ~uintptr_t(15));      // [TC_ITEMS]
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(items + TC_ITEMS);
  uint32_t* odd_rows = tmem_ptr + 1;                         // [SLOTS][2]: tokens of a masked page with a value that is not finite
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    for (int s = 0; s < SLOTS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], NQ); }
    for (int s = 0; s < NQ; ++s) {
      mbar_init(&q_full[s], 4);
      mbar_init(&v_seen[s], 1); mbar_init(&v_read[s], 4); mbar_init(&v_sync[s], 4 * (s + 1)); mbar_init(&drained[s], 1);
    }
    for (int s = 0; s < 2 * NQ; ++s) { mbar_init(&s_full[s], 1); mbar_init(&p_full[s], 4); mbar_init(&o_full[s], 1); }
    for (int s = 0; s < TC_ITEMS; ++s) { mbar_init(&item_full[s], 1); mbar_init(&item_read[s], L::WARPS - 1); }
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc<L::COLS>(tmem_ptr); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  pdl_wait();
  pdl_trigger();
  if (threadIdx.x == L::SOFTMAX * 32) ta_set_split(a, make_int4(0, 0, 0, 0));
  const int rep = a.H / a.G;
  bool ok = true;
  int why = ST_OK;                                           // what a wait that ran out waited for
  const auto place = [](int n) { return n & 1; };                       // of page n, and the phase of its barriers
  const auto announced = [&](int k, TreeItem& it) {                     // item k of this CTA; nj = 0: there is none, or the wait for it ran out
    const bool there = tc_wait(&item_full[k % TC_ITEMS], (k / TC_ITEMS) & 1);
    it = items[k % TC_ITEMS];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_read[k % TC_ITEMS]);
    if (!there) { why = ST_TIMEOUT_MBAR_FULL; it.nj = 0; }
    return it.nj > 0;
  };
  const auto phase = [](int n) { return static_cast<uint32_t>(n >> 1 & 1); };

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    TcCount c;
    int loads = 0;                                           // slots filled so far
    const int kch = (a.D + 63) / 64, vch = (a.V + 63) / 64;
    TreeRange range = ta_range(a);
#pragma unroll 1
    for (int k = 0; ok; ++k) {
      TreeItem it;
      ta_next(a, range, it);
      if (k >= TC_ITEMS) ok = tc_wait(&item_read[k % TC_ITEMS], (k / TC_ITEMS - 1) & 1);
      if (!ok) { why = ST_TIMEOUT_MBAR_EMPTY; break; }
      if (lane == 0) {
        items[k % TC_ITEMS] = it;
        mbar_arrive(&item_full[k % TC_ITEMS]);
      }
      if (it.nj == 0) break;
      const int slot = it.slot;
      int page = 0, page_v = 0;                              // of tile (lane) of the current 32: keys run one tile ahead of values
#pragma unroll 1
      for (int i = 0; i < 2 * it.nj; ++i) {
        const bool is_v = i == 2 * it.nj - 1 || (i >= 2 && !(i & 1));
        const int j = i == 0 ? 0 : i == 2 * it.nj - 1 ? it.nj - 1 : is_v ? i / 2 - 1 : (i + 1) / 2;
        if ((j & 31) == 0) {
          int p = j + lane < it.nj ? ta_page(a, slot, it.j + j + lane) : 0;
          if (p < 0) {
            if (!is_v) set_status(a.status, ST_BOUNDS, it.r0, (it.j + j + lane) * TA_PAGE, slot);
            p = 0;                                           // some page: its tokens are masked
          }
          if (is_v) page_v = p; else page = p;
        }
        ok = tc_wait(&empty[c.slot], c.ph ^ 1);
        if (!ok) { why = ST_TIMEOUT_MBAR_EMPTY; break; }
        const int pg = __shfl_sync(0xffffffffu, is_v ? page_v : page, j & 31), ch = is_v ? vch : kch;
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[c.slot], ch * KV_CHUNK);
#pragma unroll 1
          for (int x = 0; x < ch; ++x) tc_load_page(ring + c.slot * SLOT + x * KV_CHUNK, is_v ? &tmV : &tmK, &full[c.slot], x * 64, it.g, pg);
        }
        __syncwarp();
        tc_step<SLOTS>(c);
        ++loads;
      }
    }
    // no copy is on its way to shared memory when the CTA ends, whatever ended the loop
    bool come = true;
#pragma unroll 1
    for (int s = 0; s < SLOTS && come; ++s)
      if (s < c.slot || loads >= SLOTS) come = tc_wait(&full[s], s < c.slot ? c.ph : c.ph ^ 1);
    if (!come) why = ST_TIMEOUT_MBAR_FULL;
  } else if (warp <= NQ) {
    // ------------------------------------------------------------ MMA issuer of tile q (the whole warp walks, one elected lane issues)
    const int q = warp - 1, ksteps = (a.D + 15) / 16, vn = (a.V + 15) / 16 * 16, vunits = (a.V + 63) / 64 * 8;
    const uint32_t id_s = make_idesc(1, 1, 128, TA_PAGE), id_o = make_idesc(1, 1, 128, vn) | (1u << 16);
    const uint32_t qs = __shfl_sync(0xffffffffu, smem_u32(smem), 0) + q * L::Q_BYTES, rs = __shfl_sync(0xffffffffu, smem_u32(ring), 0);
    const uint32_t tm = __shfl_sync(0xffffffffu, tmem, 0) + q * L::TILE_COLS;
    TcCount c;
    int n = 0, own = 0;                                      // pages and items of the tile so far
    int shown[NQ] = {};                                      // masked pages announced to the tiles
    TreeItem it;
#pragma unroll 1
    for (int k = 0; ok && announced(k, it); ++k) {
      const int pairs = it.n * rep - (it.rt << a.bm_log), act = NQ == 2 && pairs > 128 ? 2 : 1;
      if (q >= act) {                                        // no rows here: the slots are passed on
#pragma unroll 1
        for (int i = 0; i < 2 * it.nj; ++i) {
          ok = tc_wait(&full[c.slot], c.ph);
          if (!ok) { why = ST_TIMEOUT_MBAR_FULL; break; }
          if (lane == 0) mbar_arrive(&empty[c.slot]);
          tc_step<SLOTS>(c);
        }
        continue;
      }
      uint32_t there = 0u;                                   // pages of the current 32 that the table leads to
      ok = tc_wait(&q_full[q], own & 1);
      if (!ok) { why = ST_TIMEOUT_MBAR_FULL; break; }
      ++own;
#pragma unroll 1
      for (int j = -1; j < it.nj; ++j) {
        if (j + 1 < it.nj) {
          const int t = n + j + 1;
          // (the weights of two pages back lie where the scores go: their product has read them, and all softmax warps these scores)
          ok = tc_wait(&full[c.slot], c.ph) && (t < 2 || tc_wait(&o_full[q * 2 + place(t)], phase(t - 2)));
          if (!ok) { why = ST_TIMEOUT_MBAR_FULL; break; }
          tc_fence_after();
          if (elect_one()) {
            const uint64_t kd = make_smem_desc_sw128(rs + c.slot * SLOT), qd = make_smem_desc_sw128(qs);
#pragma unroll
            for (int k = 0; k < DC / 16; ++k) {
              if (k >= ksteps) break;
              const uint64_t kk = kd + (k >> 2) * (KV_CHUNK >> 4) + 2 * (k & 3);
              if (L::QT) umma_f16_ts(tm + place(t) * 64, tm + L::Q_COL + k * 8, kk, id_s, k != 0);
              else umma_f16(tm + place(t) * 64, qd + (k >> 2) * (Q_CHUNK >> 4) + 2 * (k & 3), kk, id_s, k != 0);
            }
            umma_commit(&s_full[q * 2 + place(t)]);
            umma_commit(&empty[c.slot]);
          }
          __syncwarp();
          tc_step<SLOTS>(c);
        }
        if (j < 0) continue;
        const int tok0 = (it.j + j) * TA_PAGE;
        if ((j & 31) == 0) there = __ballot_sync(0xffffffffu, j + lane < it.nj && ta_page(a, it.slot, it.j + j + lane) >= 0);
        ok = tc_wait(&full[c.slot], c.ph);
        if (q == 0 && ok && (tok0 + TA_PAGE > it.len || tok0 < it.edge || !((there >> (j & 31)) & 1u))) {
          // ---- a masked page's values: tokens that are not the request's are zeroed, the others with a value that is not finite noted
          const int valid = (there >> (j & 31)) & 1u ? min(TA_PAGE, it.len + it.n - tok0) : 0;
          uint32_t odd[2];
#pragma unroll
          for (int half = 0; half < 2; ++half) {
            const int tok = half * 32 + lane;
            uint8_t* vrow = ring + c.slot * SLOT + tok * 128;
            uint32_t most = 0u;                              // largest exponents of the row's even and odd columns
#pragma unroll 4
            for (int u = 0; u < vunits; ++u) {
              uint4* x = reinterpret_cast<uint4*>(vrow + (u >> 3) * KV_CHUNK + (((u & 7) ^ (tok & 7)) * 16));
              if (tok >= valid) *x = make_uint4(0u, 0u, 0u, 0u);
              else {
                const uint4 v = *x;
                most = __vmaxu2(__vmaxu2(most, v.x & 0x7f807f80u), __vmaxu2(v.y & 0x7f807f80u, __vmaxu2(v.z & 0x7f807f80u, v.w & 0x7f807f80u)));
              }
            }
            odd[half] = __ballot_sync(0xffffffffu, (most & 0xffffu) == 0x7f80u || (most >> 16) == 0x7f80u);
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) { odd_rows[2 * c.slot] = odd[0]; odd_rows[2 * c.slot + 1] = odd[1]; }
#pragma unroll
          for (int i = 0; i < NQ; ++i)
            if (i < act) {
              if (shown[i] > 0) ok = ok && tc_wait(&v_read[i], (shown[i] - 1) & 1);
              if (lane == 0) mbar_arrive(&v_seen[i]);
              ++shown[i];
            }
        }
        ok = ok && tc_wait(&p_full[q * 2 + place(n + j)], phase(n + j));
        if (!ok) { why = ST_TIMEOUT_MBAR_FULL; break; }
        tc_fence_after();
        if (elect_one()) {
          const uint64_t vd = tc_desc_nmajor(rs + c.slot * SLOT, KV_CHUNK);
          const uint32_t w = tm + place(n + j) * 64;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            umma_f16_ts(tm + 128, w + k * 8, vd + k * 128, id_o, 1);
            umma_f16_ts(tm + 128, w + 32 + k * 8, vd + k * 128, id_o, 1);
          }
          umma_commit(&o_full[q * 2 + place(n + j)]);
          umma_commit(&empty[c.slot]);
        }
        __syncwarp();
        tc_step<SLOTS>(c);
      }
      n += it.nj;
    }
    // nor does a product read it, or write tensor memory
    if (elect_one()) umma_commit(&drained[q]);
    __syncwarp();
    if (!tc_wait(&drained[q], 0)) why = ST_TIMEOUT_TMEM_FULL;
  } else {
    // ------------------------------------------------------------ softmax, one row per thread
    const int q = (warp - L::SOFTMAX) >> 2, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16) + q * L::TILE_COLS;
    const int vn = (a.V + 15) / 16 * 16, vn_units = (a.V + 63) / 64 * 8;
    uint32_t sync_phase[NQ] = {}, seen_phase = 0u;
    int n = 0, seq = 0;                                      // pages of this tile so far; position of the item in the ring's sequence
    TreeItem sg;
#pragma unroll 1
    for (int i = 0; ok && announced(i, sg); ++i) {
      const TreeItem& it = sg;
      const int all = sg.n * rep - (it.rt << a.bm_log), pairs = min(128, all - q * 128);        // rows of this tile
      const int seq0 = seq;
      seq += 2 * it.nj;
      if (it.first && !it.last && threadIdx.x == L::SOFTMAX * 32) ta_set_split(a, ta_split(a, it));
      if (pairs <= 0) continue;
      const bool both = NQ == 2 && all > 128;
      uint64_t* sync = &v_sync[both ? NQ - 1 : 0];
      uint32_t& sync_ph = sync_phase[both ? NQ - 1 : 0];
      const int f = (it.rt << a.bm_log) + q * 128 + min(row, pairs - 1), node = f / rep, h = it.g * rep + f - node * rep, pr = sg.r0 + node;
      const bool idle = quad * 32 >= pairs;                  // a warp without rows keeps the pace and computes nothing
      const int p = a.pos[pr];
      const uint64_t near = ta_ancestors(a, sg, node, 0);    // (asked for long before the tree's page)
      {                                                      // the row's query; columns from D on are zero
        const uint4* src = reinterpret_cast<const uint4*>(static_cast<const __nv_bfloat16*>(a.q) + static_cast<size_t>(pr) * a.ldq + static_cast<size_t>(h) * a.hq);
        const int units = row < pairs ? a.D / 8 : 0;
        if (L::QT) {
          for (int c = 0; c < DC / 2; c += 32) {
            uint32_t w[32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              const uint4 v = c / 4 + i < units ? __ldg(src + c / 4 + i) : make_uint4(0u, 0u, 0u, 0u);
              w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
            }
            tmem_st_32x32(t_lane + L::Q_COL + c, w);
          }
        } else {
#pragma unroll 8
          for (int u = 0; u < DC / 8; ++u) {
            const uint4 v = u < units ? __ldg(src + u) : make_uint4(0u, 0u, 0u, 0u);
            *reinterpret_cast<uint4*>(smem + q * L::Q_BYTES + (u >> 3) * Q_CHUNK + row * 128 + (((u & 7) ^ (row & 7)) * 16)) = v;
          }
        }
        uint32_t z[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) z[i] = 0u;
        for (int c = 0; c < vn; c += 32) tmem_st_32x32(t_lane + 128 + c, z);
        tmem_st_wait();
        fence_proxy_async();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&q_full[q]);
      }
      bool fresh = true;                                     // some row of the warp has no reference yet
      float ref = -INFINITY, l = 0.f;                        // of the exponentials (FEAT: natural, else log2), and their sum
      const float c1 = FEAT ? 1.f : a.scale * TA_LOG2E;
      uint32_t there = 0u;                                   // pages of the current 32 that the table leads to
#pragma unroll 1
      for (int j = 0; j < it.nj; ++j, ++n) {
        const int tok0 = (it.j + j) * TA_PAGE;
        if ((j & 31) == 0) there = __ballot_sync(0xffffffffu, j + lane < it.nj && ta_page(a, it.slot, it.j + j + lane) >= 0);
        const bool page = (there >> (j & 31)) & 1u, whole = tok0 + TA_PAGE <= sg.len && tok0 >= it.edge && page;
        uint64_t seen = ~0ull;
        int at_lo = tok0 + lane, at_hi = at_lo + 32;           // FEAT: positions of the page's tokens `lane` and 32 + lane
        if (!whole && !idle) {
          seen = page ? ta_mask(a, sg, tok0, node, p, near) : 0ull;
          if (FEAT && tok0 + TA_PAGE > sg.len) {
            const int n0 = tok0 + lane - sg.len, n1 = n0 + 32;
            if (n0 >= 0) at_lo = n0 < sg.n ? a.pos[sg.r0 + n0] : p;
            if (n1 >= 0) at_hi = n1 < sg.n ? a.pos[sg.r0 + n1] : p;
          }
        }
        ok = tc_wait(&s_full[q * 2 + place(n)], phase(n));
        if (!ok) { why = ST_TIMEOUT_TMEM_FULL; break; }
        tc_fence_after();
        float s[64];
        const uint32_t t_page = t_lane + place(n) * 64;
        if (!idle) {
          {
            uint32_t raw[2][32];
            tmem_ld_32x32(t_page, raw[0]);
            tmem_ld_32x32(t_page + 32, raw[1]);
            tmem_ld_wait();
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] = __uint_as_float(raw[i >> 5][i & 31]);
          }
          if (FEAT) {
            if (a.cap > 0.f) {
              const float to_z = a.scale / a.cap;
              float big[4] = {};                             // scores far below the cap need no exponential
#pragma unroll
              for (int i = 0; i < 64; ++i) big[i & 3] = fmaxf(big[i & 3], fabsf(s[i]));
              if (__any_sync(0xffffffffu, fmaxf(fmaxf(big[0], big[1]), fmaxf(big[2], big[3])) * fabsf(to_z) >= CAP_NEAR)) {
#pragma unroll
                for (int i = 0; i < 64; ++i) {               // (cap_tanh with the approximate instructions; NaN stays NaN)
                  const float z = s[i] * to_z, e = tc_ex2(min_or_nan(z, 40.f) * (2.f * TA_LOG2E));
                  s[i] = a.cap * (fabsf(z) < CAP_NEAR ? z * tanh_over_z(z) : fmaf(-2.f, tc_rcp(1.f + e), 1.f));
                }
              } else {
                const uint64_t to_z2 = ta_two(to_z, to_z);
#pragma unroll
                for (int i = 0; i < 64; i += 2) {            // (scale * tanh_over_z, two at a time)
                  const uint64_t x = ta_two(s[i], s[i + 1]), z = ta_mul2(x, to_z2), zz = ta_mul2(z, z);
                  uint64_t y = ta_two(62.f / 2835.f * a.scale, 62.f / 2835.f * a.scale);
                  for (const float c : {-17.f / 315.f, 2.f / 15.f, -1.f / 3.f, 1.f}) y = ta_fma2(zz, y, ta_two(c * a.scale, c * a.scale));
                  tc_set(s, i, ta_mul2(x, y));
                }
              }
            } else {
              const uint64_t scale2 = ta_two(a.scale, a.scale);
#pragma unroll
              for (int i = 0; i < 64; i += 2) tc_set(s, i, ta_mul2(ta_two(s[i], s[i + 1]), scale2));
            }
            const int d0 = p - tok0;                         // distance of the page's token 0, were it committed
            const bool nodes = tok0 + TA_PAGE > sg.len;
            if (a.bias) {
              const float* bh = a.bias + static_cast<size_t>(h) * a.bias_n;
              if (!nodes && __all_sync(0xffffffffu, d0 - 63 >= a.bias_n - 1)) {
                const float far = __ldg(bh + a.bias_n - 1);
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] += far;
              } else if (!nodes && __all_sync(0xffffffffu, d0 >= 63 && d0 < a.bias_n)) {           // (within the table: 31.5 -> 29.4 us of a ragged round)
                const float* near_to = bh + d0;
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] += __ldg(near_to - i);
              } else {
#pragma unroll
                for (int i0 = 0; i0 < 64; i0 += 16) {        // sixteen in flight
                  float x[16];
#pragma unroll
                  for (int i = 0; i < 16; ++i) {
                    const int d = p - __shfl_sync(0xffffffffu, i0 < 32 ? at_lo : at_hi, (i0 & 31) + i);
                    x[i] = __ldg(bh + min(max(d, 0), a.bias_n - 1));
                  }
#pragma unroll
                  for (int i = 0; i < 16; ++i) s[i0 + i] += x[i];
                }
              }
            }
            if (a.slopes) {
              const float sl = __ldg(a.slopes + h);
              if (nodes) {
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] -= sl * static_cast<float>(p - __shfl_sync(0xffffffffu, i < 32 ? at_lo : at_hi, i & 31));
              } else {
                // (near tokens, the ones that weigh, have a small d0: nothing is lost by taking the products apart)
                const float s0 = -sl * static_cast<float>(d0);
                const uint64_t s2 = ta_two(s0, s0), sl2 = ta_two(sl, sl);
#pragma unroll
                for (int i = 0; i < 64; i += 2)
                  tc_set(s, i, ta_fma2(sl2, ta_two(static_cast<float>(i), static_cast<float>(i + 1)), ta_add2(ta_two(s[i], s[i + 1]), s2)));
              }
            }
          }
          if (!whole) {
            const uint32_t m0 = static_cast<uint32_t>(seen), m1 = static_cast<uint32_t>(seen >> 32);
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] = ((i < 32 ? m0 : m1) >> (i & 31)) & 1u ? s[i] : -INFINITY;
          }
          // ---- weights
          const uint64_t c2 = FEAT ? ta_two(TA_LOG2E, TA_LOG2E) : ta_two(c1, c1);
          bool renew = fresh, rescale = false;
          float c = 1.f, page_sum;
#pragma unroll 1
          while (true) {
            if (renew) {
              float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
              for (int i = 4; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
              float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c1;
              if (FEAT && a.slopes)                          // nearer pages weigh more by as much as is known: room for 2^86 of it
                top += fminf(fmaxf(__ldg(a.slopes + h) * static_cast<float>(p - tok0 - 63), 0.f), 60.f);
              if (ref == -INFINITY) ref = top;
              else if (top > ref) {
                rescale = true;
                c = exp2f(FEAT ? (ref - top) * TA_LOG2E : ref - top);
                l *= c;
                ref = top;
              }
              fresh = __any_sync(0xffffffffu, ref == -INFINITY);       // rows that have seen nothing yet
            }
            const float r = ref == -INFINITY ? 0.f : ref;
            const uint64_t r2 = ta_two(-r, -r), one = ta_two(-1.f, -1.f);
            uint64_t sum[2] = {0ull, 0ull};
#pragma unroll
            for (int part = 0; part < 2; ++part) {
              uint32_t hi[16], lo[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) {
                const uint64_t x = ta_two(s[part * 32 + 2 * i], s[part * 32 + 2 * i + 1]);
                const uint64_t z = FEAT ? ta_mul2(ta_add2(x, r2), c2) : ta_fma2(x, c2, r2);
                const uint64_t e = ta_two(tc_ex2(ta_lo(z)), tc_ex2(ta_hi(z)));
                sum[i & 1] = ta_add2(sum[i & 1], e);
                hi[i] = tc_pack(ta_lo(e), ta_hi(e));
                const uint64_t d = ta_fma2(ta_two(__uint_as_float(hi[i] << 16), __uint_as_float(hi[i] & 0xffff0000u)), one, e);
                lo[i] = tc_pack(ta_lo(d), ta_hi(d));
              }
              tmem_st_32x16(t_page + part * 16, hi);         // (over the scores, which are in registers)
              tmem_st_32x16(t_page + 32 + part * 16, lo);
            }
            sum[0] = ta_add2(sum[0], sum[1]);
            page_sum = ta_lo(sum[0]) + ta_hi(sum[0]);
            if (renew || !__any_sync(0xffffffffu, !(page_sum < TC_MOST))) break;
            renew = true;
          }
          l += page_sum;
          if (renew && __any_sync(0xffffffffu, rescale)) {
            ok = tc_wait(&o_full[q * 2 + place(n - 1)], phase(n - 1));
            if (!ok) { why = ST_TIMEOUT_TMEM_FULL; break; }
            tc_fence_after();
            const uint64_t k2 = ta_two(c, c);
#pragma unroll 1
            for (int cc = 0; cc < vn; cc += 32) {
              uint32_t o[32];
              tmem_ld_32x32(t_lane + 128 + cc, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const uint64_t v = ta_mul2(static_cast<uint64_t>(o[i + 1]) << 32 | o[i], k2);
                o[i] = static_cast<uint32_t>(v); o[i + 1] = static_cast<uint32_t>(v >> 32);
              }
              tmem_st_32x32(t_lane + 128 + cc, o);
            }
          }
        }
        if (!whole) {
          ok = tc_wait(&v_seen[q], seen_phase);
          seen_phase ^= 1u;
          if (!ok) { why = ST_TIMEOUT_MBAR_FULL; break; }
          __syncwarp();
          if (lane == 0) mbar_arrive(&v_read[q]);
          const int vs = (seq0 + (j < it.nj - 1 ? 2 * j + 2 : 2 * j + 1)) % SLOTS;       // the values' place in the ring's sequence
          const uint64_t bad = odd_rows[2 * vs] | static_cast<uint64_t>(odd_rows[2 * vs + 1]) << 32;
          if (bad) {                                         // (rare)
            uint8_t* vals = ring + vs * SLOT;
            if (n > 0) {
              ok = tc_wait(&o_full[q * 2 + place(n - 1)], phase(n - 1));
              if (!ok) { why = ST_TIMEOUT_TMEM_FULL; break; }
              tc_fence_after();
            }
            if (!idle) {                                     // (the weights are there already; their high terms are enough)
              tmem_st_wait();
#pragma unroll 1
              for (uint64_t left = bad; left; left &= left - 1) {
                const int k = __ffsll(left) - 1;
                const uint32_t pair = tc_ld1(t_page + k / 2);
                const float w = __uint_as_float(k & 1 ? pair & 0xffff0000u : pair << 16);
#pragma unroll 1
                for (int col = 0; col < vn; ++col) {
                  const uint32_t v = *reinterpret_cast<const uint16_t*>(vals + (col >> 6) * KV_CHUNK + k * 128 + (((col >> 3 & 7) ^ (k & 7)) * 16) + (col & 7) * 2);
                  if ((v & 0x7f80u) != 0x7f80u) continue;    // (the same for the whole warp)
                  const float o = __uint_as_float(tc_ld1(t_lane + 128 + col));
                  tc_st1(t_lane + 128 + col, __float_as_uint(seen >> k & 1ull ? fmaf(w, __uint_as_float(v << 16), o) : o));
                }
              }
            }
            ok = tc_sync(sync, sync_ph);                     // everyone has read them
            if (!ok) { why = ST_TIMEOUT_MBAR_FULL; break; }
            const int tok = row & 63, parts = both ? 4 : 2;
            for (int u = q * 2 * both + (row >> 6); u < vn_units; u += parts) {
              uint16_t* x = reinterpret_cast<uint16_t*>(vals + (u >> 3) * KV_CHUNK + tok * 128 + (((u & 7) ^ (tok & 7)) * 16));
              for (int e = 0; e < 8; ++e)
                if ((x[e] & 0x7f80u) == 0x7f80u) x[e] = 0;
            }
            fence_proxy_async();
            ok = tc_sync(sync, sync_ph);
            if (!ok) { why = ST_TIMEOUT_MBAR_FULL; break; }
          }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[q * 2 + place(n)]);
      }
      if (!ok) break;
      // ---- the rows' outputs, or this CTA's part of them
      ok = tc_wait(&o_full[q * 2 + place(n - 1)], phase(n - 1));
      if (!ok) { why = ST_TIMEOUT_TMEM_FULL; break; }
      tc_fence_after();
      if (idle) { tc_fence_before(); continue; }
      const bool done = it.first && it.last;
      float m = ref;
      if (!FEAT && m != -INFINITY) m *= TA_LN2;
      const size_t pb = ((static_cast<size_t>(blockIdx.x) * 2 + (it.first ? 1 : 0)) << a.bm_log) + q * 128 + row;
      float k = 1.f;
      if (done) {
        if (a.sink) k = ta_sink<__nv_bfloat16>(a.sink[h], m, l);
        k = l > 0.f ? ta_head_factor<__nv_bfloat16>(a, pr, h) * k / l : 0.f;
        if (l != l) k = l;
      } else if (row < pairs) {
        *reinterpret_cast<float2*>(a.part_ml + pb * 2) = make_float2(m, l);
      }
      __nv_bfloat16* out = static_cast<__nv_bfloat16*>(a.out) + static_cast<size_t>(pr) * a.ldo + static_cast<size_t>(h) * a.ho;
#pragma unroll 1
      for (int cc = 0; cc < vn; cc += 32) {
        uint32_t o[32];
        tmem_ld_32x32(t_lane + 128 + cc, o);
        tmem_ld_wait();
        if (row < pairs) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            if (cc + i * 8 >= a.V) break;
            if (done) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = tc_pack(__uint_as_float(o[i * 8 + 2 * e]) * k, __uint_as_float(o[i * 8 + 2 * e + 1]) * k);
              *reinterpret_cast<uint4*>(out + cc + i * 8) = make_uint4(w[0], w[1], w[2], w[3]);
            } else {
              uint4* part = reinterpret_cast<uint4*>(ta_part(a, static_cast<size_t>(blockIdx.x) * 2 + (it.first ? 1 : 0), q * 128 + row, (cc >> 3) + i));
              part[0] = make_uint4(o[i * 8], o[i * 8 + 1], o[i * 8 + 2], o[i * 8 + 3]);
              part[1] = make_uint4(o[i * 8 + 4], o[i * 8 + 5], o[i * 8 + 6], o[i * 8 + 7]);
            }
          }
        }
        __syncwarp();
      }
      tc_fence_before();
    }
  }
  if (why != ST_OK && lane == 0) set_status(a.status, why, blockIdx.x, warp);
  tc_fence_before();
  __syncthreads();
  if (warp == 1) { tc_fence_after(); tmem_dealloc<L::COLS>(tmem); }
}

template <int DC, int NQ, bool FEAT>
static int launch_tc(const CUtensorMap& tk, const CUtensorMap& tv, const TreeAttn& a, cudaStream_t s) {
  using L = Tc<DC, NQ>;
  auto kern = tree_attn_tc_kernel<DC, NQ, FEAT>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, L::SMEM) != cudaSuccess) return -4;
  spark_launch_pdl(kern, dim3(a.ctas), dim3(L::THREADS), L::SMEM, s, dim3(1, 1, 1), tk, tv, a);
  return spark_launch_rc("spark_tree_attn");
}
template <int DC, int NQ>
static int launch_tc_feat(const CUtensorMap& tk, const CUtensorMap& tv, const TreeAttn& a, cudaStream_t s) {
  return a.cap > 0.f || a.bias || a.slopes || !(a.scale > 0.f) ? launch_tc<DC, NQ, true>(tk, tv, a, s) : launch_tc<DC, NQ, false>(tk, tv, a, s);
}

int launch_tree_tc(const TreeAttn& a, cudaStream_t s) {
  const int w = a.D > a.V ? a.D : a.V;
  if (w > 256 || ((a.ldq | a.hq | a.ldo | a.ho) & 7) || (a.bm_log == 8 && w > 128)) return -5;
  CUtensorMap tk, tv;
  if (const int r = make_tmap_page(&tk, a.k, a.n_pages, a.G, a.D, a.k_tok, a.k_page)) return r;
  if (const int r = make_tmap_page(&tv, a.v, a.n_pages, a.G, a.V, a.v_tok, a.v_page)) return r;
  if (w > 128) return launch_tc_feat<256, 1>(tk, tv, a, s);
  if (w > 64) return a.bm_log == 8 ? launch_tc_feat<128, 2>(tk, tv, a, s) : launch_tc_feat<128, 1>(tk, tv, a, s);
  return a.bm_log == 8 ? launch_tc_feat<64, 2>(tk, tv, a, s) : launch_tc_feat<64, 1>(tk, tv, a, s);
}

}  // namespace spark
