// Rows of a verification round over paged caches (64-token pages), from request lengths that live on the device:
//
//   block_tables  a request's pages follow its length: pages go back on a stack and come off it
//   slot_maps     request, index, position, cache row and ancestors of every row of the round
//   path_conv     short causal convolution along a drafted tree's paths, keys and values into their pages
//   commit_paths  the accepted path's cache rows of all layers together, the convolutions' states along it
//
// Row r of request s has index j = r - starts[s].  It is written to the cache at the request's token len_s + j, whatever its depth in the
// tree; its position is len_s + depth.  What a table or a path gives is checked before it is used as an address: a bad entry sets the status
// word and the row is skipped.
#include "../common/rows.cuh"
#include "../common/tree_args.h"

namespace spark {

// Exclusive prefix of v over the block's 1024 threads, and the sum; `sh`: 33 ints.  Every thread calls it.
__device__ __forceinline__ int block_prefix(int v, int* sh, int& total) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  int x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) sh[w] = x;
  __syncthreads();
  if (w == 0) {
    int s = lane < nw ? sh[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += y;
    }
    sh[lane] = s;
  }
  __syncthreads();
  const int before = w ? sh[w - 1] : 0;
  total = sh[nw - 1];
  __syncthreads();
  return before + x - v;
}

// ------------------------------------------------------------------------------------------------ block tables

// One CTA, a warp per request in turn.  Pages go back first, the last request's last page first, then requests take theirs in order, each
// from the top of the stack: giving back what was just taken restores the stack.  A request whose pages are not all there gets none, nor
// does one behind it that needs any.  4 us (8 for 256 requests that take 18 pages each): one launch and three trips to memory; a thread for every
// page instead took 4.5 and 7.8.
__global__ void __launch_bounds__(1024)
block_tables_kernel(const __grid_constant__ BlockTables a) {
  __shared__ int sh[33], s_have[1024], s_need[1024], s_off[1024];
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31;
  const int nf = min(max(*a.n_free, 0), a.cap);
  auto load = [&](int s, int& have, int& need) {
    have = need = 0;
    if (s >= a.S) return;
    const int len = a.lengths[s];
    have = min(max(a.held[s], 0), a.ld);
    need = len < 0 ? have : len / TREE_PAGE + (len % TREE_PAGE != 0);
    if (need > a.ld) { set_status(a.status, ST_BOUNDS, s, len, a.ld); need = a.ld; }
  };
  int total = 0;                                             // pages given back
  for (int s0 = 0; s0 < a.S; s0 += 1024) {
    int have, need, n;
    load(s0 + t, have, need);
    block_prefix(max(have - need, 0), sh, n);
    total += n;
  }
  int done = 0;
  for (int s0 = 0; s0 < a.S && total > 0; s0 += 1024) {
    int n;
    load(s0 + t, s_have[t], s_need[t]);
    s_off[t] = done + block_prefix(max(s_have[t] - s_need[t], 0), sh, n);
    done += n;
    __syncthreads();
    for (int i = warp; i < min(1024, a.S - s0); i += 32) {
      int* row = a.tables + static_cast<size_t>(s0 + i) * a.ld;
      for (int p = s_need[i] + lane; p < s_have[i]; p += 32) {
        const int to = nf + total - 1 - (s_off[i] + p - s_need[i]);
        if (to < a.cap) a.free[to] = row[p];
        else set_status(a.status, ST_BOUNDS, s0 + i, to, a.cap);
        row[p] = -1;
      }
    }
    __syncthreads();
  }
  const int top = min(nf + total, a.cap);
  int asked = 0, used = 0;
  for (int s0 = 0; s0 < a.S; s0 += 1024) {
    int n, m;
    load(s0 + t, s_have[t], s_need[t]);
    const int want = max(s_need[t] - s_have[t], 0), off = asked + block_prefix(want, sh, n);
    const bool ok = off + want <= top;
    block_prefix(ok ? want : 0, sh, m);
    asked = min(asked + n, 1 << 30);
    used += m;
    s_off[t] = off;
    if (!ok) s_need[t] = min(s_need[t], s_have[t]);
    if (s0 + t < a.S) { a.held[s0 + t] = s_need[t]; a.room[s0 + t] = s_need[t] * TREE_PAGE; }
    __syncthreads();
    for (int i = warp; i < min(1024, a.S - s0); i += 32) {
      int* row = a.tables + static_cast<size_t>(s0 + i) * a.ld;
      for (int p = s_have[i] + lane; p < s_need[i]; p += 32) row[p] = a.free[top - 1 - (s_off[i] + p - s_have[i])];
    }
    __syncthreads();
  }
  if (t == 0) *a.n_free = top - used;
}

// ------------------------------------------------------------------------------------------------ row maps

constexpr int MAP_THREADS = 256;

// grid: rows.  Every CTA forms the prefix of all counts (a few hundred numbers) instead of waiting for another launch that does.  4 us for 64 rows
// of trees, 6 for 300 thousand of prompts: the latency of lengths, parents and tables in turn.
__global__ void __launch_bounds__(MAP_THREADS)
slot_maps_kernel(const __grid_constant__ SlotMaps a) {
  extern __shared__ int s_start[];                           // [S + 1]
  __shared__ int sh[33];
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x;
  int base = 0;
  for (int s0 = 0; s0 < a.S; s0 += MAP_THREADS) {
    int n;
    const int c = s0 + t < a.S ? min(max(a.counts[s0 + t], 0), a.R) : 0;
    const int b = min(base + block_prefix(c, sh, n), a.R);
    if (s0 + t < a.S) s_start[s0 + t] = b;
    if (base + n > a.R && t == 0 && blockIdx.x == 0) set_status(a.status, ST_BOUNDS, s0, base + n, a.R);
    base = min(base + n, a.R);
  }
  if (t == 0) s_start[a.S] = base;
  __syncthreads();
  if (blockIdx.x == 0)
    for (int s = t; s <= a.S; s += MAP_THREADS) a.starts[s] = s_start[s];
  for (int r = blockIdx.x * MAP_THREADS + t; r < a.R; r += gridDim.x * MAP_THREADS) {
    int slot = -1, j = -1, pos = -1;
    long long row = -1;
    if (r < base) {
      int lo = 0, hi = a.S;                                  // the last request that starts at or before r (and is not empty)
      while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (s_start[m] <= r) lo = m; else hi = m; }
      const int r0 = s_start[lo], len = max(a.lengths[lo], 0);
      slot = a.slots ? a.slots[lo] : lo;
      j = r - r0;
      int depth = j;
      if (a.words) {
        if (j >= a.nodes) set_status(a.status, ST_BOUNDS, r, j, a.nodes);
        depth = -1;
        int* out = a.anc + static_cast<size_t>(r) * a.words;
        uint32_t bits = 0;
        int word = j >> 5;
        for (int w = word + 1; w < a.words; ++w) out[w] = 0;
        for (int at = j; at >= 0;) {                         // every step goes to a lower index
          for (; word > (at >> 5); --word) { if (word < a.words) out[word] = bits; bits = 0; }
          bits |= 1u << (at & 31);
          ++depth;
          int p = a.parents ? a.parents[r0 + at] : at - 1;
          if (p >= at || p < -1) { set_status(a.status, ST_BAD_ARGUMENT, r0 + at, p, at); p = -1; }
          at = p;
        }
        for (; word >= 0; --word) { if (word < a.words) out[word] = bits; bits = 0; }
      }
      pos = len + depth;
      const long long tok = static_cast<long long>(len) + j;
      const bool ok = slot >= 0 && slot < a.n_slots && tok / TREE_PAGE < a.ld;
      const int page = ok ? a.tables[static_cast<size_t>(slot) * a.ld + tok / TREE_PAGE] : -1;
      if (page >= 0) row = static_cast<long long>(page) * TREE_PAGE + tok % TREE_PAGE;
      else set_status(a.status, ST_BOUNDS, r, static_cast<int>(tok), slot);
    } else if (a.words) {
      for (int w = 0; w < a.words; ++w) a.anc[static_cast<size_t>(r) * a.words + w] = 0;
    }
    a.slot[r] = slot; a.index[r] = j; a.pos[r] = pos; a.cache_row[r] = row;
  }
}

// ------------------------------------------------------------------------------------------------ convolution along paths

constexpr int PC_ROWS = 64, PC_FAR = 64, PC_THREADS = 256, PC_UNITS = 16;     // rows of a tile and brought in beside them; 16-byte pieces of its channels
constexpr int PC_STAGES = 2, PC_PER_SM = 3;                    // (three stages leave room for two CTAs: 38.2 us instead of 35.6)

__device__ __forceinline__ void pc_copy(void* d, const void* s) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(d)), "l"(s) : "memory");
}

// channels of a 16-byte piece
__device__ __forceinline__ void pc_split(const uint4& u, float (&f)[8], __nv_bfloat16) {
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) { f[2 * i] = __uint_as_float(w[i] << 16); f[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
__device__ __forceinline__ void pc_split(const uint4& u, float (&f)[4], float) {
  f[0] = __uint_as_float(u.x); f[1] = __uint_as_float(u.y); f[2] = __uint_as_float(u.z); f[3] = __uint_as_float(u.w);
}
__device__ __forceinline__ uint4 pc_join(const float (&f)[8], __nv_bfloat16) {
  uint32_t w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 b = __floats2bfloat162_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t*>(&b);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}
__device__ __forceinline__ uint4 pc_join(const float (&f)[4], float) {
  return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
}

// grid (groups of `per` channel tiles, row tiles).  A tile's rows are brought to shared memory once and every row takes its taps from there;
// so are up to PC_FAR rows that lie elsewhere (ancestors in front of the tile, the sequences' past).  The paths are
// followed once for all channel tiles of a CTA, and the next tile's rows are on their way while one is computed.  The bytes do not bound it (a
// quarter of DRAM's rate under the profiler): the shared-memory pipe is busy half of the time, issue slots 56 %, and the barrier per channel tile
// holds up as many warps as the shared memory does.  So what depends on the row alone is formed once, and the common loop has no branches
// (nobody's rows take a row of zeros).
// 5.2 us for 50 rows of 2560 channels, 36 us for 5000 rows of 6144 (126 MB, 3.5 TB/s; 52 with the taps' places looked up per tile, 87 with every
// tap loaded from memory; two products per instruction: no change).  Where more than PC_FAR rows lie elsewhere (four taps: the pasts of 22 requests
// that begin in a tile), its taps are looked up one by one and some come from memory: 96 requests of one row take 16 us, of eight rows 14.
template <typename T, int TAPS>
__global__ void __launch_bounds__(PC_THREADS, PC_PER_SM)
path_conv_kernel(const __grid_constant__ PathConv a, int per) {
  constexpr int VEC = 16 / sizeof(T), STEP = PC_THREADS / PC_UNITS, ZERO = (PC_ROWS + PC_FAR) * PC_UNITS;
  extern __shared__ __align__(16) uint4 s_x[];               // [PC_STAGES][PC_ROWS + PC_FAR + 1][PC_UNITS]
  constexpr int BUF = ZERO + PC_UNITS, LAST = PC_STAGES - 1;
  __shared__ const T* s_far[PC_FAR];                         // channel 0 of the rows brought in
  __shared__ int s_fars, s_left, s_rest;                     // rows that lie elsewhere; some tap found no place; some row is nobody's
  __shared__ int s_before[PC_ROWS], s_past[PC_ROWS];         // places: of the rows in front of the tile; of the past of the request that begins here
  __shared__ long long s_k[PC_ROWS], s_v[PC_ROWS];           // places of the results in the caches (-1: none)
  __shared__ int s_slot[PC_ROWS], s_parent[PC_ROWS];
  int* s_src = reinterpret_cast<int*>(s_x + PC_STAGES * BUF);        // [PC_ROWS][taps, 3 padded to 4]: a tap's place in s_x; else as `elsewhere` takes it
  pdl_wait();
  pdl_trigger();
  const int taps = TAPS > 0 ? TAPS : a.taps, ld = taps == 3 ? 4 : taps, t = threadIdx.x, unit = t % PC_UNITS, b0 = blockIdx.y * PC_ROWS;
  const int n = min(PC_ROWS, a.R - b0), tile0 = blockIdx.x * per;
  // -1 - a flat row, or -2^30 - e: the e-th newest entry of the slot's tail
  auto elsewhere = [&](int s, int slot) {
    return s < -(1 << 30) ? static_cast<const T*>(a.tail) + ((static_cast<size_t>(slot) + 1) * (taps - 1) + (s + (1 << 30))) * a.C
                          : static_cast<const T*>(a.x) + static_cast<size_t>(-1 - s) * a.ldx;
  };
  auto load = [&](int i) {                                   // rows of channel tile tile0 + i
    const int c = ((tile0 + i) * PC_UNITS + unit) * VEC;
    if (i < per && c < a.C)
#pragma unroll
      for (int r = t / PC_UNITS; r < PC_ROWS; r += STEP)
        if (r < n) pc_copy(s_x + (i % PC_STAGES) * BUF + r * PC_UNITS + unit, static_cast<const T*>(a.x) + static_cast<size_t>(b0 + r) * a.ldx + c);
  };
  auto load_far = [&](int i) {
    const int c = ((tile0 + i) * PC_UNITS + unit) * VEC;
    if (i < per && c < a.C)
      for (int r = t / PC_UNITS; r < min(s_fars, PC_FAR); r += STEP) pc_copy(s_x + (i % PC_STAGES) * BUF + (PC_ROWS + r) * PC_UNITS + unit, s_far[r] + c);
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int i = 0; i < LAST; ++i) load(i);
  if (t < PC_STAGES * PC_UNITS) s_x[t / PC_UNITS * BUF + ZERO + unit] = make_uint4(0u, 0u, 0u, 0u);
  for (int r = t; r < PC_ROWS * ld; r += PC_THREADS) s_src[r] = ZERO;
  int j = 0;
  if (t == 0) s_fars = s_left = s_rest = 0;
  if (t < PC_ROWS) s_before[t] = -1;
  if (t < n) {
    j = a.index[b0 + t];
    s_parent[t] = a.parents ? a.parents[b0 + t] : j - 1;
    const int slot = a.slot[b0 + t];
    s_slot[t] = slot < a.n_slots ? slot : -1;
    const long long row = a.cache_row[b0 + t];
    const bool ok = slot >= 0 && slot < a.n_slots && row >= 0 && row < a.cache_rows;
    if (slot >= 0 && !ok) set_status(a.status, ST_BOUNDS, b0 + t, static_cast<int>(row), slot);
    s_k[t] = ok ? row / TREE_PAGE * a.k_page + row % TREE_PAGE * a.k_tok : -1;
    s_v[t] = ok ? row / TREE_PAGE * a.v_page + row % TREE_PAGE * a.v_tok : -1;
  }
  __syncthreads();
  const bool live = t < n && s_slot[t] >= 0;
  if (t < n && !live) s_rest = 1;
  const int r0 = b0 + t - j, head = max(r0 - b0, 0);         // the request's first row, and its first one in the tile
  if (live) {                                                // the row, its ancestors, then the sequence's past
    if (t == head) {
      const int f = s_past[t] = atomicAdd(&s_fars, taps - 1);
      for (int e = 1; e < taps; ++e)
        if (f + e - 1 < PC_FAR) s_far[f + e - 1] = elsewhere(-(1 << 30) - e, s_slot[t]);
    }
    int at = j, back = 0;
    for (int tp = taps - 1; tp >= 0; --tp) {
      const int x = at >= 0 ? (r0 + at >= b0 ? (r0 + at - b0) * PC_UNITS : -1 - (r0 + at)) : -(1 << 30) - ++back;
      s_src[t * ld + tp] = x;
      if (x < 0 && x >= -(1 << 30) && -1 - x >= b0 - PC_ROWS && atomicCAS(&s_before[-1 - x - (b0 - PC_ROWS)], -1, -2) == -1) {
        const int f = atomicAdd(&s_fars, 1);
        if (f < PC_FAR) s_far[f] = elsewhere(x, 0);
        s_before[-1 - x - (b0 - PC_ROWS)] = f;
      }
      if (tp && at >= 0) {
        const int p = r0 + at >= b0 ? s_parent[r0 + at - b0] : a.parents ? a.parents[r0 + at] : at - 1;
        at = p < at ? p : -1;
      }
    }
  }
  __syncthreads();
  if (live)
    for (int tp = 0; tp < taps; ++tp) {
      const int x = s_src[t * ld + tp];
      if (x >= 0) continue;
      const int f = x < -(1 << 30) ? s_past[head] - x - (1 << 30) - 1 : -1 - x >= b0 - PC_ROWS ? s_before[-1 - x - (b0 - PC_ROWS)] : PC_FAR;
      if (f < PC_FAR) s_src[t * ld + tp] = (PC_ROWS + f) * PC_UNITS;
      else s_left = 1;
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < LAST; ++i) load_far(i);                // (the first group has the rows of both)
  const bool near = !s_left, rest = s_rest;                  // every tap is in shared memory
  for (int i = 0; i < per; ++i) {
    const int c0 = ((tile0 + i) * PC_UNITS + unit) * VEC;
    float w[TAPS > 0 ? TAPS : 1][VEC];
    if (TAPS > 0 && c0 < a.C)
#pragma unroll
      for (int tp = 0; tp < TAPS; ++tp)
#pragma unroll
        for (int e = 0; e < VEC; e += 4) *reinterpret_cast<float4*>(&w[tp][e]) = *reinterpret_cast<const float4*>(a.w + static_cast<size_t>(tp) * a.C + c0 + e);
    asm volatile("cp.async.wait_group %0;" ::"n"(LAST - 1) : "memory");
    __syncthreads();                                         // tile i is there, and tile i - 1 is used up
    load(i + LAST);
    load_far(i + LAST);
    const uint4* xs = s_x + (i % PC_STAGES) * BUF + unit;
    const bool isq = c0 < a.nq, isk = c0 < a.nq + a.nk;
    T* base = isq ? static_cast<T*>(a.q) + static_cast<size_t>(b0) * a.nq + c0 : isk ? static_cast<T*>(a.k) + (c0 - a.nq) : static_cast<T*>(a.v) + (c0 - a.nq - a.nk);
    auto store = [&](int r, const float (&y)[VEC]) {
      const long long to = isq ? static_cast<long long>(r) * a.nq : isk ? s_k[r] : s_v[r];
      if (to >= 0) *reinterpret_cast<uint4*>(base + to) = pc_join(y, T());
    };
    if (c0 >= a.C) continue;
    if (TAPS > 0 && near) {
#pragma unroll
      for (int k = 0; k < PC_ROWS / STEP; ++k) {
        const int r = t / PC_UNITS + k * STEP;
        float y[VEC] = {};
#pragma unroll
        for (int tp = 0; tp < TAPS; ++tp) {
          float f[VEC];
          pc_split(xs[s_src[r * (TAPS == 3 ? 4 : TAPS) + tp]], f, T());
#pragma unroll
          for (int e = 0; e < VEC; ++e) y[e] = fmaf(w[tp][e], f[e], y[e]);
        }
        if (r < n) store(r, y);
      }
    } else {
      for (int r = t / PC_UNITS; r < n; r += STEP) {
        float y[VEC] = {};
        for (int tp = 0; tp < taps; ++tp) {
          const int s = s_src[r * ld + tp];
          float f[VEC];
          pc_split(s >= 0 ? xs[s] : *reinterpret_cast<const uint4*>(elsewhere(s, s_slot[r]) + c0), f, T());
#pragma unroll
          for (int e = 0; e < VEC; ++e) y[e] = fmaf(a.w[static_cast<size_t>(tp) * a.C + c0 + e], f[e], y[e]);
        }
        store(r, y);
      }
    }
    if (rest && isq)                                         // (a weight that is not finite times their zeros is not 0; the same thread's stores)
      for (int r = t / PC_UNITS; r < n; r += STEP)
        if (s_slot[r] < 0) *reinterpret_cast<uint4*>(base + static_cast<long long>(r) * a.nq) = make_uint4(0u, 0u, 0u, 0u);
  }
}

// ------------------------------------------------------------------------------------------------ commit

// grid (requests, column blocks, jobs); 128 threads x 16 bytes.  A path is ascending, so row i is written after row path[i] >= i was read,
// and no later row of the path lies at or below i: every thread moves its columns in order and in place.  One launch for all layers: 6 us for 12,
// 31 to 35 us for 24 of 64 requests (142 MB in rows of 2 KB, 4.0 to 4.7 TB/s; with 4 or 8 rows read before any is written the same,
// with two or four layers per CTA 34 and 37).
__global__ void __launch_bounds__(128)
commit_paths_kernel(const __grid_constant__ CommitPaths a) {
  extern __shared__ int s_path[];                            // [P], then [P] source and [P] target rows of the cache
  pdl_wait();
  pdl_trigger();
  const CommitJob& jb = a.job[blockIdx.z];
  const int s = blockIdx.x, t = threadIdx.x, n = min(a.n_path[s], a.P), count = a.starts[s + 1] - a.starts[s];
  if (n <= 0) return;
  const int slot = a.slots ? a.slots[s] : s, len = max(a.lengths[s], 0);
  bool ok = slot >= 0 && slot < a.n_slots;
  int* src = s_path + a.P;
  int* dst = src + a.P;
  for (int i = t; i < n; i += 128) {
    const int p = a.path[static_cast<size_t>(s) * a.P + i];
    if (p < i || p >= count || (i > 0 && p <= a.path[static_cast<size_t>(s) * a.P + i - 1])) ok = false;
    s_path[i] = p;
  }
  ok = __syncthreads_and(ok);
  // (the caches' rows are looked up for tails as well: all jobs of a request go ahead, or none does)
  if (ok && a.pages >= 0)
    for (int i = t; i < n; i += 128) {
      const long long from = static_cast<long long>(len) + s_path[i], to = static_cast<long long>(len) + i;
      const int pf = from / TREE_PAGE < a.ld ? a.tables[static_cast<size_t>(slot) * a.ld + from / TREE_PAGE] : -1;
      const int pt = to / TREE_PAGE < a.ld ? a.tables[static_cast<size_t>(slot) * a.ld + to / TREE_PAGE] : -1;
      if (pf < 0 || pt < 0 || pf >= a.pages || pt >= a.pages) ok = false;
      src[i] = pf * TREE_PAGE + static_cast<int>(from % TREE_PAGE);
      dst[i] = pt * TREE_PAGE + static_cast<int>(to % TREE_PAGE);
    }
  ok = __syncthreads_and(ok);
  if (!ok) {
    if (t == 0) set_status(a.status, ST_BOUNDS, s, slot, n);
    return;
  }
  const int col = (blockIdx.y * 128 + t) * 16;
  if (col >= jb.bytes) return;
  if (jb.x) {
    char* tail = jb.base + static_cast<long long>(slot) * jb.kept * jb.tok + col;
    for (int e = 0; e < jb.kept; ++e) {                       // ascending: an entry is read before any later one is written
      const int at = n - jb.kept + e;
      const char* p = at >= 0 ? jb.x + static_cast<long long>(a.starts[s] + s_path[at]) * jb.page + col : tail + (jb.kept + at) * jb.tok;
      *reinterpret_cast<uint4*>(tail + e * jb.tok) = *reinterpret_cast<const uint4*>(p);
    }
    return;
  }
  for (int i = 0; i < n; ++i) {
    if (src[i] == dst[i]) continue;
    const uint4 v = *reinterpret_cast<const uint4*>(jb.base + (src[i] / TREE_PAGE) * jb.page + (src[i] % TREE_PAGE) * jb.tok + col);
    *reinterpret_cast<uint4*>(jb.base + (dst[i] / TREE_PAGE) * jb.page + (dst[i] % TREE_PAGE) * jb.tok + col) = v;
  }
}

}  // namespace spark

using namespace spark;

extern "C" unsigned spark_tree_layout() { return SPARK_TREE_LAYOUT; }

extern "C" int spark_block_tables(const BlockTables* a, cudaStream_t s) {
  if (a->S <= 0) return 0;
  if (a->ld <= 0 || a->cap < 0 || static_cast<long long>(a->S) * a->ld > (1 << 24)) return -5;
  spark_launch_pdl(block_tables_kernel, dim3(1), dim3(1024), 0, s, dim3(1, 1, 1), *a);
  return spark_launch_rc(__func__);
}

extern "C" int spark_slot_maps(const SlotMaps* a, cudaStream_t s) {
  if (a->S <= 0 || a->S > 8192 || a->R < 0 || a->R > (1 << 22) || a->ld <= 0 || a->words < 0 || a->nodes > a->words * 32) return -5;
  const int blocks = (a->R + MAP_THREADS - 1) / MAP_THREADS;
  spark_launch_pdl(slot_maps_kernel, dim3(blocks < 1 ? 1 : (blocks > 1184 ? 1184 : blocks)), dim3(MAP_THREADS), (a->S + 1) * 4, s, dim3(1, 1, 1), *a);
  return spark_launch_rc(__func__);
}

extern "C" int spark_path_conv(const PathConv* a, int f32, cudaStream_t s) {
  if (a->R <= 0) return 0;
  if (a->taps < 1 || ((a->C | a->nq | a->nk | a->ldx) & 7) || a->nq + a->nk > a->C || a->n_slots <= 0) return -5;
  const int cols = PC_UNITS * (f32 ? 4 : 8), smem = PC_STAGES * (PC_ROWS + PC_FAR + 1) * PC_UNITS * 16 + PC_ROWS * (a->taps == 3 ? 4 : a->taps) * 4;
  const int tiles = (a->C + cols - 1) / cols, rows = (a->R + PC_ROWS - 1) / PC_ROWS;
  int dev = 0, sms = 148;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -4;
  // channel tiles per CTA: the least of rounds x (tiles + 2 for the start)
  int per = 1;
  long long best = 1ll << 60;
  for (int p = 1; p <= 16 && p <= tiles; ++p) {
    const long long ctas = static_cast<long long>((tiles + p - 1) / p) * rows, cost = (ctas + PC_PER_SM * sms - 1) / (PC_PER_SM * sms) * (p + 2);
    if (cost < best) { best = cost; per = p; }
  }
  const dim3 grid((tiles + per - 1) / per, rows);
  if (rows > 65535 || a->taps > 32) return -5;
#define SPARK_PATH(T, TAPS)                                                                                                     \
  {                                                                                                                             \
    if (cudaFuncSetAttribute(path_conv_kernel<T, TAPS>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) return -4; \
    spark_launch_pdl(path_conv_kernel<T, TAPS>, grid, dim3(PC_THREADS), smem, s, dim3(1, 1, 1), *a, per);                        \
  }
#define SPARK_PATH_T(T)               \
  switch (a->taps) {                  \
    case 1: SPARK_PATH(T, 1) break;   \
    case 2: SPARK_PATH(T, 2) break;   \
    case 3: SPARK_PATH(T, 3) break;   \
    case 4: SPARK_PATH(T, 4) break;   \
    default: SPARK_PATH(T, 0)         \
  }
  if (f32) { SPARK_PATH_T(float) } else { SPARK_PATH_T(__nv_bfloat16) }
#undef SPARK_PATH_T
#undef SPARK_PATH
  return spark_launch_rc(__func__);
}

// `most`: bytes of the widest job's row.
extern "C" int spark_commit_paths(const CommitPaths* a, int jobs, int most, cudaStream_t s) {
  if (a->S <= 0 || jobs <= 0 || a->P <= 0) return 0;
  if (jobs > COMMIT_JOBS || a->P > 4096 || a->ld <= 0 || (most & 15) || most <= 0 || a->pages > (1 << 24)) return -5;
  for (int i = 0; i < jobs; ++i)
    if ((a->job[i].bytes & 15) || a->job[i].bytes > most || (!a->job[i].x && a->pages < 0)) return -5;
  spark_launch_pdl(commit_paths_kernel, dim3(a->S, (most / 16 + 127) / 128, jobs), dim3(128), a->P * 12, s, dim3(1, 1, 1), *a);
  return spark_launch_rc(__func__);
}
