// Tree attention on tcgen05 (bf16 caches): the tiles of tree_attn.cu with 128 (node, head) rows per accumulator, a page of keys per step.
//   warp 0      TMA: pages of keys and values into a ring of slots in the order the products use them (K0 K1 V0 K2 V1 ..)
//   warp 1      issues S = Q K^T one page ahead of O += P V (P in tensor memory, over the scores that it was made from)
//   warps 2 ..  softmax, one row per thread: 64 scores are one tensor-memory load, statistics stay in the thread
// NQ = 2: two tiles of 128 rows with their own softmax warps share the keys in shared memory (large trees: a page is read once for 256 rows).
//
// Weights enter the product as two bf16 terms (2^-17 of a weight is lost), so that the reference of the exponentials may lag behind the
// maximum: the accumulator is rescaled only when a row's maximum outgrew its reference by 2^8.
//
// A page that not every row sees whole (the tree itself, the edge of a window or chunk) is masked by 64 bits per row.  Its values are looked
// over first: rows that hold no token of the request are zeroed, and where a value is not finite, 0 * value would spoil the rows that do not
// see it, so it is added by hand for the rows that do and zeroed in front of the product.
#include "../common/tree_work.cuh"

namespace spark {

int make_tmap_page(CUtensorMap* m, const void* base, uint64_t pages, uint64_t G, uint64_t D, uint64_t tok, uint64_t page);

constexpr float TC_LAG = 8.f;                                // log2

template <int DC, int NQ> struct Tc {
  static constexpr bool QT = DC == 256;                      // queries in tensor memory: shared memory has no room for them beside the ring
  static constexpr int SLOT = TA_PAGE * DC * 2, Q_BYTES = QT ? 0 : 128 * DC * 2;
  static constexpr int SLOTS = DC == 256 ? 6 : DC == 128 ? (NQ == 2 ? 9 : 4) : (NQ == 2 ? 16 : 8);
  static constexpr int SMEM = NQ * Q_BYTES + SLOTS * SLOT + 1024 + 1024;
  // per tile: two buffers of scores / weights of 64 columns, the accumulator
  static constexpr int TILE_COLS = 128 + DC, Q_COL = 128 + DC;
  static constexpr int COLS = QT || NQ == 2 ? 512 : 256;
  static constexpr int WARPS = 2 + 4 * NQ, THREADS = WARPS * 32, PER_SM = QT || NQ == 2 ? 1 : 2;
  static_assert(NQ * TILE_COLS + (QT ? DC / 2 : 0) <= COLS && SMEM <= 232448, "tensor memory, shared memory");
};

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
__device__ __forceinline__ bool tc_odd(uint32_t w) {         // one of two bf16 is not finite
  return (w & 0x7f80u) == 0x7f80u || (w & 0x7f800000u) == 0x7f800000u;
}
// All softmax warps of the item (4 or 8): a barrier whose wait ends.
__device__ __forceinline__ bool tc_sync(uint64_t* bar, uint32_t& phase) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
  const bool ok = __all_sync(0xffffffffu, mbar_wait(bar, phase));
  phase ^= 1u;
  return ok;
}

struct TcCount { int slot = 0; uint32_t ph = 0; };
template <int N> __device__ __forceinline__ void tc_step(TcCount& c) { if (++c.slot == N) { c.slot = 0; c.ph ^= 1; } }

// Which of the 64 tokens of page j row `node` (position p) sees.
__device__ __forceinline__ uint64_t tc_mask(const TreeAttn& a, const TreeSeg& sg, int tok0, int node, int p) {
  const int first = ta_first_visible(a, p), i0 = tok0 - sg.len;        // the page's token 0 is node i0
  const int lo = min(max(first - tok0, 0), 64), hi = min(max(-i0, 0), 64);
  uint64_t m = hi > lo ? (hi == 64 ? ~0ull : (1ull << hi) - 1) & ~(lo == 0 ? 0ull : (1ull << lo) - 1) : 0ull;
  if (hi == 64) return m;
  uint64_t t = 0;                                            // bit b: node max(i0, 0) + b
  const int b0 = max(i0, 0);
  if (a.anc) {
    const uint32_t* w = a.anc + static_cast<size_t>(sg.r0 + node) * a.words;
    const int k = b0 >> 5, sh = b0 & 31;
    const uint64_t w0 = k < a.words ? w[k] : 0u, w1 = k + 1 < a.words ? w[k + 1] : 0u, w2 = k + 2 < a.words ? w[k + 2] : 0u;
    t = (w0 | w1 << 32) >> sh;
    if (sh) t |= w2 << (64 - sh);
  } else {
    const int n = node - b0 + 1;
    t = n <= 0 ? 0ull : n >= 64 ? ~0ull : (1ull << n) - 1;
  }
  const int left = sg.n - b0;                                // nodes there are
  if (left < 64) t &= left <= 0 ? 0ull : (1ull << left) - 1;
  if (first > sg.len)                                        // ancestors outside the window or chunk
    for (uint64_t x = t; x; x &= x - 1) {
      const int b = __ffsll(x) - 1;
      if (a.pos[sg.r0 + b0 + b] < first) t &= ~(1ull << b);
    }
  return m | t << hi;
}

// grid: a.ctas.  FEAT: soft cap, distance bias or slopes, or a scale that is not positive (the scaled scores are then masked, not the products).
template <int DC, int NQ, bool FEAT>
__global__ void __launch_bounds__(Tc<DC, NQ>::THREADS, Tc<DC, NQ>::PER_SM)
tree_attn_tc_kernel(const __grid_constant__ CUtensorMap tmK, const __grid_constant__ CUtensorMap tmV, const __grid_constant__ TreeAttn a) {
  using L = Tc<DC, NQ>;
  constexpr int CH = DC / 64, SLOT = L::SLOT, SLOTS = L::SLOTS, KV_CHUNK = TA_PAGE * 128, Q_CHUNK = 128 * 128, NT = L::THREADS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + NQ * L::Q_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(ring + SLOTS * SLOT);
  uint64_t* empty = full + SLOTS;
  uint64_t* q_full = empty + SLOTS;                          // [NQ]
  uint64_t* s_full = q_full + NQ;                            // [NQ][2] from here on
  uint64_t* p_full = s_full + 2 * NQ;
  uint64_t* o_full = p_full + 2 * NQ;
  uint64_t* v_sync = o_full + 2 * NQ;                        // [NQ]: of 4 and of 8 softmax warps
  long long* sh = reinterpret_cast<long long*>(v_sync + NQ); // [NT / 32 + 2]
  uint32_t* tmem_ptr = reinterpret_cast<uint32_t*>(sh + NT / 32 + 2);
  uint32_t* odd_rows = tmem_ptr + 1;                         // [2]: tokens of a masked page with a value that is not finite
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    tma_prefetch_desc(&tmK); tma_prefetch_desc(&tmV);
    for (int s = 0; s < SLOTS; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int s = 0; s < NQ; ++s) { mbar_init(&q_full[s], 4); mbar_init(&v_sync[s], 4 * (s + 1)); }
    for (int s = 0; s < 2 * NQ; ++s) { mbar_init(&s_full[s], 1); mbar_init(&p_full[s], 4); mbar_init(&o_full[s], 1); }
    odd_rows[0] = odd_rows[1] = 0u;
    fence_barrier_init();
  }
  if (warp == 1) { tmem_alloc<L::COLS>(tmem_ptr); tmem_relinquish(); }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_ptr;
  pdl_wait();
  pdl_trigger();
  TreeRange range = ta_range<NT>(a, sh);
  if (threadIdx.x == 64) a.split[blockIdx.x] = make_int4(0, 0, 0, 0);
  const int rep = a.H / a.G;
  TreeItem it;
  bool ok = true;

  if (warp == 0) {
    // ------------------------------------------------------------ producer
    TcCount c;
    const int kch = (a.D + 63) / 64, vch = (a.V + 63) / 64;
    while (ok && ta_next(a, range, it)) {
      const int slot = a.slots ? a.slots[it.s] : it.s;
      int page = 0, page_v = 0;                              // of tile (lane) of the current 32: keys run one tile ahead of values
      for (int i = 0; i < 2 * it.nj; ++i) {
        const bool is_v = i == 2 * it.nj - 1 || (i >= 2 && !(i & 1));
        const int j = i == 0 ? 0 : i == 2 * it.nj - 1 ? it.nj - 1 : is_v ? i / 2 - 1 : (i + 1) / 2;
        if ((j & 31) == 0) {
          int p = j + lane < it.nj ? ta_page(a, slot, it.j + j + lane) : 0;
          if (p < 0) {
            if (!is_v) set_status(a.status, ST_BOUNDS, it.seg.r0, (it.j + j + lane) * TA_PAGE, slot);
            p = 0;                                           // some page: its tokens are masked
          }
          if (is_v) page_v = p; else page = p;
        }
        ok = __all_sync(0xffffffffu, mbar_wait(&empty[c.slot], c.ph ^ 1));
        if (!ok) { set_status(a.status, ST_TIMEOUT_MBAR_EMPTY, blockIdx.x, it.s, i); break; }
        const int pg = __shfl_sync(0xffffffffu, is_v ? page_v : page, j & 31), ch = is_v ? vch : kch;
        if (lane == 0) {
          mbar_arrive_expect_tx(&full[c.slot], ch * KV_CHUNK);
          for (int x = 0; x < ch; ++x) tc_load_page(ring + c.slot * SLOT + x * KV_CHUNK, is_v ? &tmV : &tmK, &full[c.slot], x * 64, it.g, pg);
        }
        __syncwarp();
        tc_step<SLOTS>(c);
      }
    }
  } else if (warp == 1) {
    // ------------------------------------------------------------ MMA issuer (the whole warp walks, one elected lane issues)
    const int ksteps = (a.D + 15) / 16, vn = (a.V + 15) / 16 * 16;
    const uint32_t id_s = make_idesc(1, 1, 128, TA_PAGE), id_o = make_idesc(1, 1, 128, vn) | (1u << 16);
    const uint32_t qs = __shfl_sync(0xffffffffu, smem_u32(smem), 0), rs = qs + NQ * L::Q_BYTES, tm = __shfl_sync(0xffffffffu, tmem, 0);
    TcCount c;
    int n[NQ] = {}, items[NQ] = {};                          // pages and items of each tile so far
    while (ok && ta_next(a, range, it)) {
      const int pairs = it.seg.n * rep - it.rt * a.bm, act = NQ == 2 && pairs > 128 ? 2 : 1;
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        if (q < act && ok) {
          ok = __all_sync(0xffffffffu, mbar_wait(&q_full[q], items[q] & 1));
          ++items[q];
        }
      if (!ok) { set_status(a.status, ST_TIMEOUT_MBAR_FULL, blockIdx.x, it.s, -2); break; }
      for (int j = -1; j < it.nj && ok; ++j) {
        if (j + 1 < it.nj) {
          ok = __all_sync(0xffffffffu, mbar_wait(&full[c.slot], c.ph));
#pragma unroll
          for (int q = 0; q < NQ; ++q) {
            if (q >= act) continue;
            // the scores go where the weights of two pages back were: their product has to be done
            const int b = (n[q] + j + 1) & 1;
            if (ok && n[q] + j + 1 >= 2) ok = __all_sync(0xffffffffu, mbar_wait(&o_full[q * 2 + b], ((n[q] + j - 1) >> 1) & 1));
            if (!ok) break;
            tc_fence_after();
            if (elect_one()) {
              const uint32_t d = tm + q * L::TILE_COLS + b * 64;
              for (int k = 0; k < ksteps; ++k) {
                const uint64_t kd = make_smem_desc_sw128(rs + c.slot * SLOT + (k >> 2) * KV_CHUNK) + 2 * (k & 3);
                if (L::QT) umma_f16_ts(d, tm + L::Q_COL + k * 8, kd, id_s, k != 0);
                else umma_f16(d, make_smem_desc_sw128(qs + q * L::Q_BYTES + (k >> 2) * Q_CHUNK) + 2 * (k & 3), kd, id_s, k != 0);
              }
              umma_commit(&s_full[q * 2 + b]);
            }
            __syncwarp();
          }
          if (!ok) { set_status(a.status, ST_TIMEOUT_MBAR_FULL, blockIdx.x, it.s, j); break; }
          if (elect_one()) umma_commit(&empty[c.slot]);
          __syncwarp();
          tc_step<SLOTS>(c);
        }
        if (j < 0) continue;
        ok = __all_sync(0xffffffffu, mbar_wait(&full[c.slot], c.ph));
#pragma unroll
        for (int q = 0; q < NQ; ++q) {
          if (q >= act) continue;
          const int b = (n[q] + j) & 1;
          ok = ok && __all_sync(0xffffffffu, mbar_wait(&p_full[q * 2 + b], ((n[q] + j) >> 1) & 1));
          if (!ok) break;
          tc_fence_after();
          if (elect_one()) {
            const uint32_t base = tm + q * L::TILE_COLS;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const uint64_t vd = tc_desc_nmajor(rs + c.slot * SLOT + k * 2048, KV_CHUNK);
              umma_f16_ts(base + 128, base + b * 64 + k * 8, vd, id_o, 1);
              umma_f16_ts(base + 128, base + b * 64 + 32 + k * 8, vd, id_o, 1);
            }
            umma_commit(&o_full[q * 2 + b]);
          }
          __syncwarp();
        }
        if (!ok) { set_status(a.status, ST_TIMEOUT_MBAR_FULL, blockIdx.x, it.s, j); break; }
        if (elect_one()) umma_commit(&empty[c.slot]);
        __syncwarp();
        tc_step<SLOTS>(c);
      }
#pragma unroll
      for (int q = 0; q < NQ; ++q)
        if (q < act) n[q] += it.nj;
    }
  } else {
    // ------------------------------------------------------------ softmax, one row per thread
    const int q = NQ == 2 ? (warp - 2) >> 2 : 0, quad = warp & 3, row = quad * 32 + lane;
    const uint32_t t_lane = tmem + (static_cast<uint32_t>(quad * 32) << 16) + q * L::TILE_COLS;
    const int vn = (a.V + 15) / 16 * 16, vn_units = (a.V + 63) / 64 * 8;
    uint32_t sync_phase[NQ] = {};
    int n = 0, seq = 0;                                      // pages of this tile so far; position of the item in the ring's sequence
    while (ok && ta_next(a, range, it)) {
      const TreeSeg& sg = it.seg;
      const int all = sg.n * rep - it.rt * a.bm, pairs = min(128, all - q * 128);      // rows of this tile
      const int seq0 = seq;
      seq += 2 * it.nj;
      if (it.first && !it.last && threadIdx.x == 64) a.split[blockIdx.x] = make_int4(it.parts, it.s, it.g, it.rt);
      if (pairs <= 0) continue;
      const bool both = NQ == 2 && all > 128;
      uint64_t* sync = &v_sync[both ? NQ - 1 : 0];
      uint32_t& sync_ph = sync_phase[both ? NQ - 1 : 0];
      const int f = it.rt * a.bm + q * 128 + min(row, pairs - 1), node = f / rep, h = it.g * rep + f - node * rep, pr = sg.r0 + node;
      const bool idle = quad * 32 >= pairs;                  // a warp without rows keeps the pace and computes nothing
      const int p = a.pos[pr], slot = a.slots ? a.slots[it.s] : it.s;
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
      float ref = -INFINITY, l = 0.f;                        // of the exponentials (FEAT: natural, else log2), and their sum
      const float c1 = FEAT ? 1.f : a.scale * TA_LOG2E;
      const int edge = ta_first_visible(a, sg.len + sg.n - 1);         // from here on every row sees committed tokens
      for (int j = 0; j < it.nj; ++j, ++n) {
        const int b = n & 1, tok0 = (it.j + j) * TA_PAGE;
        const bool page = ta_page(a, slot, it.j + j) >= 0, whole = tok0 + TA_PAGE <= sg.len && tok0 >= edge && page;
        ok = __all_sync(0xffffffffu, mbar_wait(&s_full[q * 2 + b], (n >> 1) & 1));
        if (!ok) { set_status(a.status, ST_TIMEOUT_TMEM_FULL, blockIdx.x, it.s, j); break; }
        tc_fence_after();
        uint64_t seen = ~0ull;
        float s[64];
        if (!idle) {
          uint32_t raw[2][32];
          tmem_ld_32x32(t_lane + b * 64, raw[0]);
          tmem_ld_32x32(t_lane + b * 64 + 32, raw[1]);
          tmem_ld_wait();
#pragma unroll
          for (int i = 0; i < 64; ++i) s[i] = __uint_as_float(raw[i >> 5][i & 31]);
          if (!whole) seen = page ? tc_mask(a, sg, tok0, node, p) : 0ull;
          if (FEAT) {
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] *= a.scale;
            if (a.cap > 0.f) {
              const float icap = 1.f / a.cap;
#pragma unroll
              for (int i = 0; i < 64; ++i) s[i] = a.cap * cap_tanh(s[i] * icap);
            }
            const int d0 = p - tok0;                         // distance of the page's token 0, were it committed
            if (a.bias) {
              const float* bh = a.bias + static_cast<size_t>(h) * a.bias_n;
              if (tok0 + TA_PAGE <= sg.len && __all_sync(0xffffffffu, d0 - 63 >= a.bias_n - 1)) {
                const float far = __ldg(bh + a.bias_n - 1);
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] += far;
              } else {
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                  const int nd = tok0 + i - sg.len, d = nd < 0 ? d0 - i : (nd < sg.n ? p - __ldg(a.pos + sg.r0 + nd) : 0);
                  s[i] += __ldg(bh + min(max(d, 0), a.bias_n - 1));
                }
              }
            }
            if (a.slopes) {
              const float sl = __ldg(a.slopes + h);
              if (tok0 + TA_PAGE <= sg.len) {
#pragma unroll
                for (int i = 0; i < 64; ++i) s[i] -= sl * static_cast<float>(d0 - i);
              } else {
#pragma unroll
                for (int i = 0; i < 64; ++i) {
                  const int nd = tok0 + i - sg.len, d = nd < 0 ? d0 - i : (nd < sg.n ? p - __ldg(a.pos + sg.r0 + nd) : 0);
                  s[i] -= sl * static_cast<float>(d);
                }
              }
            }
          }
          if (!whole) {
#pragma unroll
            for (int i = 0; i < 64; ++i) s[i] = (seen >> i) & 1ull ? s[i] : -INFINITY;
          }
          // ---- weights
          float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
          for (int i = 4; i < 64; ++i) mx[i & 3] = fmaxf(mx[i & 3], s[i]);
          const float top = fmaxf(fmaxf(mx[0], mx[1]), fmaxf(mx[2], mx[3])) * c1;
          const float lag = FEAT ? TC_LAG * TA_LN2 : TC_LAG;
          const bool grow = ref == -INFINITY ? top > -INFINITY : top > ref + lag;
          const float c = ref == -INFINITY ? 1.f : exp2f(FEAT ? (ref - top) * TA_LOG2E : ref - top);
          const bool rescale = grow && ref != -INFINITY;
          if (grow) { if (rescale) l *= c; ref = top; }
          const float r = ref == -INFINITY ? 0.f : ref;
          float sum[4] = {0.f, 0.f, 0.f, 0.f};
          uint32_t hi[32], lo[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const float e0 = exp2f(FEAT ? (s[2 * i] - r) * TA_LOG2E : fmaf(s[2 * i], c1, -r));
            const float e1 = exp2f(FEAT ? (s[2 * i + 1] - r) * TA_LOG2E : fmaf(s[2 * i + 1], c1, -r));
            sum[i & 1] += e0; sum[2 + (i & 1)] += e1;
            hi[i] = tc_pack(e0, e1);
            lo[i] = tc_pack(e0 - __uint_as_float(hi[i] << 16), e1 - __uint_as_float(hi[i] & 0xffff0000u));
          }
          l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
          tmem_st_32x32(t_lane + b * 64, hi);
          tmem_st_32x32(t_lane + b * 64 + 32, lo);
          if (__any_sync(0xffffffffu, rescale)) {            // the product before has to be done
            ok = __all_sync(0xffffffffu, mbar_wait(&o_full[q * 2 + (b ^ 1)], ((n - 1) >> 1) & 1));
            if (!ok) { set_status(a.status, ST_TIMEOUT_TMEM_FULL, blockIdx.x, it.s, j); break; }
            tc_fence_after();
            const float k = rescale ? c : 1.f;
#pragma unroll 1
            for (int cc = 0; cc < vn; cc += 32) {
              uint32_t o[32];
              tmem_ld_32x32(t_lane + 128 + cc, o);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * k);
              tmem_st_32x32(t_lane + 128 + cc, o);
            }
          }
        }
        if (!whole) {
          // ---- the page's values: tokens that are not the request's are zeroed, values that are not finite taken out
          const int i = seq0 + (j < it.nj - 1 ? 2 * j + 2 : 2 * j + 1), vs = i % SLOTS;
          ok = __all_sync(0xffffffffu, mbar_wait(&full[vs], (i / SLOTS) & 1));
          if (!ok) { set_status(a.status, ST_TIMEOUT_MBAR_FULL, blockIdx.x, it.s, j); break; }
          const int tok = row & 63, half = both ? q * 2 + (row >> 6) : row >> 6, parts = both ? 4 : 2;
          const bool there = tok0 + tok < sg.len + sg.n && page;
          uint8_t* vrow = ring + vs * SLOT + tok * 128;
          bool odd = false;
          for (int u = half; u < vn_units; u += parts) {
            uint4* x = reinterpret_cast<uint4*>(vrow + (u >> 3) * KV_CHUNK + (((u & 7) ^ (tok & 7)) * 16));
            if (!there) *x = make_uint4(0u, 0u, 0u, 0u);
            else { const uint4 v = *x; odd |= tc_odd(v.x) | tc_odd(v.y) | tc_odd(v.z) | tc_odd(v.w); }
          }
          if (odd) atomicOr(&odd_rows[tok >> 5], 1u << (tok & 31));
          ok = tc_sync(sync, sync_ph);
          if (!ok) { set_status(a.status, ST_TIMEOUT_MBAR_FULL, blockIdx.x, it.s, j); break; }
          const uint64_t bad = odd_rows[0] | static_cast<uint64_t>(odd_rows[1]) << 32;
          if (bad) {                                         // (rare)
            if (j > 0) {
              ok = __all_sync(0xffffffffu, mbar_wait(&o_full[q * 2 + (b ^ 1)], ((n - 1) >> 1) & 1));
              if (!ok) { set_status(a.status, ST_TIMEOUT_TMEM_FULL, blockIdx.x, it.s, j); break; }
            }
            tc_fence_after();
            const float r = ref == -INFINITY ? 0.f : ref;
#pragma unroll 1
            for (int cc = 0; cc < vn && !idle; cc += 32) {
              uint32_t o[32];
              tmem_ld_32x32(t_lane + 128 + cc, o);
              tmem_ld_wait();
#pragma unroll 1
              for (int k = 0; k < 64; ++k) {
                if (!((bad >> k) & 1ull)) continue;
                float x = -INFINITY;
#pragma unroll
                for (int e = 0; e < 64; ++e) x = e == k ? s[e] : x;
                const float w = (seen >> k) & 1ull ? exp2f(FEAT ? (x - r) * TA_LOG2E : fmaf(x, c1, -r)) : 0.f;
#pragma unroll
                for (int e = 0; e < 32; ++e) {
                  const int col = cc + e, u = col >> 3;
                  const uint16_t v = *reinterpret_cast<const uint16_t*>(ring + vs * SLOT + (u >> 3) * KV_CHUNK + k * 128 + (((u & 7) ^ (k & 7)) * 16) + (col & 7) * 2);
                  if ((v & 0x7f80u) == 0x7f80u && w != 0.f) o[e] = __float_as_uint(fmaf(w, __uint_as_float(static_cast<uint32_t>(v) << 16), __uint_as_float(o[e])));
                }
              }
              tmem_st_32x32(t_lane + 128 + cc, o);
            }
            ok = tc_sync(sync, sync_ph);                     // everyone has read them
            if (!ok) { set_status(a.status, ST_TIMEOUT_MBAR_FULL, blockIdx.x, it.s, j); break; }
            if (row + q * 128 == 0) { odd_rows[0] = 0u; odd_rows[1] = 0u; }
            for (int u = half; u < vn_units; u += parts) {
              uint16_t* x = reinterpret_cast<uint16_t*>(vrow + (u >> 3) * KV_CHUNK + (((u & 7) ^ (tok & 7)) * 16));
              for (int e = 0; e < 8; ++e)
                if ((x[e] & 0x7f80u) == 0x7f80u) x[e] = 0;
            }
          }
          fence_proxy_async();
          ok = tc_sync(sync, sync_ph);                       // the values are clean, and the marks are read
          if (!ok) { set_status(a.status, ST_TIMEOUT_MBAR_FULL, blockIdx.x, it.s, j); break; }
        }
        tmem_st_wait();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&p_full[q * 2 + b]);
      }
      if (!ok) break;
      // ---- the rows' outputs, or this CTA's part of them
      ok = __all_sync(0xffffffffu, mbar_wait(&o_full[q * 2 + ((n - 1) & 1)], ((n - 1) >> 1) & 1));
      if (!ok) { set_status(a.status, ST_TIMEOUT_TMEM_FULL, blockIdx.x, it.s, it.nj); break; }
      tc_fence_after();
      if (idle) { tc_fence_before(); continue; }
      const bool done = it.first && it.last;
      float m = ref;
      if (!FEAT && m != -INFINITY) m *= TA_LN2;
      const size_t pb = (static_cast<size_t>(blockIdx.x) * 2 + (it.first ? 1 : 0)) * a.bm + q * 128 + row;
      float k = 1.f;
      if (done) {
        if (a.sink) {
          const float M = fmaxf(m, a.sink[h]);
          k = expf(m - M);
          l = l * k + expf(a.sink[h] - M);
        }
        k = l > 0.f ? ta_head_factor<__nv_bfloat16>(a, pr, h) * k / l : 0.f;
        if (l != l) k = l;
      } else if (row < pairs) {
        a.part_ml[pb * 2] = m;
        a.part_ml[pb * 2 + 1] = l;
      }
#pragma unroll 1
      for (int cc = 0; cc < vn; cc += 32) {
        uint32_t o[32];
        tmem_ld_32x32(t_lane + 128 + cc, o);
        tmem_ld_wait();
        if (row < pairs) {
          if (done) {
            uint4* dst = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(a.out) + static_cast<size_t>(pr) * a.ldo + static_cast<size_t>(h) * a.ho + cc);
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              if (cc + i * 8 >= a.V) break;
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = tc_pack(__uint_as_float(o[i * 8 + 2 * e]) * k, __uint_as_float(o[i * 8 + 2 * e + 1]) * k);
              dst[i] = make_uint4(w[0], w[1], w[2], w[3]);
            }
          } else {
            uint4* dst = reinterpret_cast<uint4*>(a.part_o + pb * a.V + cc);
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (cc + i * 4 < a.V) dst[i] = make_uint4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
          }
        }
        __syncwarp();
      }
      tc_fence_before();
    }
  }
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
  if (w > 256 || ((a.ldq | a.hq | a.ldo | a.ho) & 7) || (a.bm == 256 && w > 128)) return -5;
  CUtensorMap tk, tv;
  if (const int r = make_tmap_page(&tk, a.k, a.n_pages, a.G, a.D, a.k_tok, a.k_page)) return r;
  if (const int r = make_tmap_page(&tv, a.v, a.n_pages, a.G, a.V, a.v_tok, a.v_page)) return r;
  if (w > 128) return launch_tc_feat<256, 1>(tk, tv, a, s);
  if (w > 64) return a.bm == 256 ? launch_tc_feat<128, 2>(tk, tv, a, s) : launch_tc_feat<128, 1>(tk, tv, a, s);
  return a.bm == 256 ? launch_tc_feat<64, 2>(tk, tv, a, s) : launch_tc_feat<64, 1>(tk, tv, a, s);
}

}  // namespace spark
