// Attention of drafted trees over a paged cache (64-token pages): every node of a tree sees the request's committed tokens, inside a chunk
// or a window, its ancestors and itself.
//
//   o[j][h] = sum_i p_i v_i / (sum_i p_i + e^(sink_h)),  p_i = e^(cap tanh(scale q.k_i / cap) + bias[h][d] - slope_h d),  d: distance of the
//   positions; a row that sees nothing is 0.  Statistics and sums are fp32 and kept against the running maximum.
//
//   tree_tile    FP32 units: the 32-bit mode and head sizes the tensor-core kernel does not take
//   tree_merge   joins the parts of items that several CTAs share, and zeroes the rows behind the last request
#include "../common/tree_work.cuh"

#include <type_traits>

namespace spark {

// ------------------------------------------------------------------------------------------------ FP32 units
constexpr int TT_BM = 64, TT_THREADS = 256, TT_WARPS = TT_THREADS / 32, TT_STAGES = 3, TT_LD = 68, TT_PIECE = TA_PAGE * TT_LD;

template <int N>                                             // bytes
__device__ __forceinline__ void tt_copy(void* d, const void* s) {
  if (N == 16) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(d)), "l"(s) : "memory");
  else asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(smem_u32(d)), "l"(s) : "memory");
}

// 2 or 4 columns
template <typename T>
__device__ __forceinline__ void tt_load(float (&x)[4], const T* p) {
  const float4 v = ldf4(p);
  x[0] = v.x; x[1] = v.y; x[2] = v.z; x[3] = v.w;
}
__device__ __forceinline__ void tt_load(float (&x)[2], const float* p) {
  const float2 v = *reinterpret_cast<const float2*>(p);
  x[0] = v.x; x[1] = v.y;
}
__device__ __forceinline__ void tt_load(float (&x)[2], const __nv_bfloat16* p) {
  const float2 v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(p));
  x[0] = v.x; x[1] = v.y;
}
template <typename T>
__device__ __forceinline__ void tt_store(T* p, const float (&x)[4], float k) { stf4(p, make_float4(x[0] * k, x[1] * k, x[2] * k, x[3] * k)); }
__device__ __forceinline__ void tt_store(float* p, const float (&x)[2], float k) { *reinterpret_cast<float2*>(p) = make_float2(x[0] * k, x[1] * k); }
__device__ __forceinline__ void tt_store(__nv_bfloat16* p, const float (&x)[2], float k) {
  *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x[0] * k, x[1] * k);
}

struct TtRows { uint64_t seen[TT_BM]; int pos[TT_BM], head[TT_BM], at[TA_PAGE]; };    // of a row: tokens of the page it sees, position, head

// One item, 8 * MR rows: a warp has rows warp + 8 i, so that what is read of a row is the same for all lanes (one shared-memory cycle instead
// of four); a lane has keys lane + 32 e of a page's scores and CW neighbouring columns in every 32 CW of the outputs.  Keys pass in pieces of
// 64 tokens x 64 channels, values in pieces of 4096 (128 channels, or 64 where there are no more), two of them on their way while one is worked
// on.  The FP32 units and the instructions that feed them bound it: one request of 64 nodes, 12 heads of 128 over 39k tokens runs at 27 TFLOP/s
// (with 4 x 4 scores and outputs per thread 23, with copies waited for where they are needed 14), a single row over 30k tokens, 4 heads, at 1.5 TB/s; 5 to
// 11 nodes over 2k tokens are 24 us of latency (35 with the rows' softmax unrolled: every instruction's first run waits for memory).
template <typename T, int VP, int CW, int MR>
__device__ __forceinline__ void tt_item(const TreeAttn& a, const TreeItem& it, T* ring, float* Qs, float* Ss, TtRows& rows) {
  constexpr int VW = 32 * CW, VT = 4096 / VW;                // channels and tokens of a piece of values
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, D = a.D, V = a.V, LDQ = (D + 63) / 64 * 64, rep = a.H / a.G;
  const int f0 = it.rt * TT_BM, pairs = min(TT_WARPS * MR, it.n * rep - f0), kc = (D + 63) >> 6, vc = (V + VW - 1) / VW;
  int lj = 0, lc = 0, stage = 0;                             // the piece to be asked for next
  int lpage = ta_page(a, it.slot, it.j), npage = it.nj > 1 ? ta_page(a, it.slot, it.j + 1) : -1;
  auto load = [&](int to) {
    if (lj < it.nj) {
      const int valid = lpage < 0 ? 0 : min(TA_PAGE, it.len + it.n - (it.j + lj) * TA_PAGE);
      T* dst = ring + to * TT_PIECE;
      if (lc < kc) {
        const int c = lc * 64 + (t & 15) * 4;
        const T* src = static_cast<const T*>(a.k) + max(lpage, 0) * a.k_page + static_cast<size_t>(it.g) * D + c;
        if (c < D)
#pragma unroll
          for (int row = t >> 4; row < TA_PAGE; row += 16)
            if (row < valid) tt_copy<4 * sizeof(T)>(dst + row * TT_LD + (t & 15) * 4, src + row * a.k_tok);
      } else {
        constexpr int UNITS = VW / 4;                        // per token
        const int x = lc - kc, u = t % UNITS, c = x / (TA_PAGE / VT) * VW + u * 4, tok0 = x % (TA_PAGE / VT) * VT;
        const T* src = static_cast<const T*>(a.v) + max(lpage, 0) * a.v_page + static_cast<size_t>(it.g) * V + c;
        if (c < V)
#pragma unroll
          for (int row = t / UNITS; row < VT; row += TT_THREADS / UNITS)
            if (tok0 + row < valid) tt_copy<4 * sizeof(T)>(dst + row * VW + u * 4, src + (tok0 + row) * a.v_tok);
      }
      if (++lc == kc + vc * (TA_PAGE / VT)) {
        lc = 0;
        ++lj;
        lpage = npage;
        npage = lj + 1 < it.nj ? ta_page(a, it.slot, it.j + lj + 1) : -1;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  auto next = [&]() {                                        // the piece that has come; everyone is done with the one before
    asm volatile("cp.async.wait_group %0;" ::"n"(TT_STAGES - 2) : "memory");
    __syncthreads();
    const int now = stage;
    stage = stage == TT_STAGES - 1 ? 0 : stage + 1;
    load(now == 0 ? TT_STAGES - 1 : now - 1);
    return ring + now * TT_PIECE;
  };
  int node = 0, pos = 0;                                     // of row t
  uint64_t near = 0ull;
  if (t < TT_WARPS * MR) {
    const int f = f0 + min(t, pairs - 1);
    node = f / rep;
    pos = rows.pos[t] = a.pos[it.r0 + node];
    rows.head[t] = it.g * rep + f - node * rep;
    near = ta_ancestors(a, it, node, 0);
  }
#pragma unroll 1
  for (int row = t >> 4; row < pairs; row += 16) {
    const T* src = static_cast<const T*>(a.q) + static_cast<size_t>(it.r0 + (f0 + row) / rep) * a.ldq + static_cast<size_t>(it.g * rep + (f0 + row) % rep) * a.hq;
#pragma unroll 1
    for (int c = (t & 15) * 4; c < D; c += 64)
      if (sizeof(T) == 4) tt_copy<16>(Qs + row * LDQ + c, src + c);
      else *reinterpret_cast<float4*>(Qs + row * LDQ + c) = ldf4(src + c);
  }
#pragma unroll 1
  for (int i = 0; i < TT_STAGES - 1; ++i) load(i);
  float o[VP][MR][CW] = {};
  float m = -INFINITY, l = 0.f;                              // of the row warp + 8 lane: maximum and sum
#pragma unroll 1
  for (int j = it.j; j < it.j + it.nj; ++j) {
    const int page = ta_page(a, it.slot, j), tok0 = j * TA_PAGE;
    const bool whole = page >= 0 && tok0 >= it.edge && tok0 + TA_PAGE <= it.len;
    if (page < 0 && t == 0) set_status(a.status, ST_BOUNDS, it.r0, tok0, it.slot);
    if (!whole && t < TT_WARPS * MR) rows.seen[t] = page >= 0 ? ta_mask(a, it, tok0, node, pos, near) : 0ull;
    if ((a.bias || a.slopes) && t >= TT_THREADS - TA_PAGE) {
      const int x = t - (TT_THREADS - TA_PAGE), n = tok0 + x - it.len;
      rows.at[x] = n < 0 ? tok0 + x : n < it.n ? a.pos[it.r0 + n] : 0;
    }
    // ---- scores: even and odd channels apart
    uint64_t s2[MR][2] = {};
#pragma unroll 1
    for (int d0 = 0; d0 < D; d0 += 64) {
      const T* kp = next() + lane * TT_LD;
      const float* qp = Qs + warp * LDQ + d0;
      const int width = min(64, D - d0);
#pragma unroll 2
      for (int c = 0; c < width; c += 4) {
        ulonglong2 q[MR];
#pragma unroll
        for (int i = 0; i < MR; ++i) q[i] = *reinterpret_cast<const ulonglong2*>(qp + TT_WARPS * i * LDQ + c);
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float4 k = ldf4(kp + 32 * e * TT_LD + c);
          const uint64_t k0 = ta_two(k.x, k.y), k1 = ta_two(k.z, k.w);
#pragma unroll
          for (int i = 0; i < MR; ++i) s2[i][e] = ta_fma2(q[i].y, k1, ta_fma2(q[i].x, k0, s2[i][e]));
        }
      }
    }
    float* sw = Ss + warp * TA_PAGE;
#pragma unroll
    for (int i = 0; i < MR; ++i)
#pragma unroll
      for (int e = 0; e < 2; ++e) sw[i * TT_WARPS * TA_PAGE + lane + 32 * e] = (ta_lo(s2[i][e]) + ta_hi(s2[i][e])) * a.scale;
    // ---- weights, row by row (little code: in short calls the first run of every instruction is what takes time)
    float k = 1.f;                                           // of the row warp + 8 lane: what its outputs shrink by
#pragma unroll 1
    for (int i = 0, row = warp; row < pairs; ++i, row += TT_WARPS) {
      float* sr = Ss + row * TA_PAGE + lane;
      float x[2];
      const int h = rows.head[row], p = rows.pos[row];
      const uint64_t seen = whole ? ~0ull : rows.seen[row];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        x[e] = sr[32 * e];
        if (a.cap > 0.f) x[e] = a.cap * tanhf(x[e] / a.cap);
        if (a.bias || a.slopes) {
          const int dist = p - rows.at[lane + 32 * e];
          if (a.bias) x[e] += a.bias[static_cast<size_t>(h) * a.bias_n + min(max(dist, 0), a.bias_n - 1)];
          if (a.slopes) x[e] -= a.slopes[h] * static_cast<float>(dist);
        }
        if (!(seen >> (lane + 32 * e) & 1ull)) x[e] = -INFINITY;
      }
      const float m0 = __shfl_sync(0xffffffffu, m, i);
      float top = fmaxf(fmaxf(x[0], x[1]), m0);
#pragma unroll
      for (int z = 1; z < 32; z <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, z));
      const float ref = top == -INFINITY ? 0.f : top;
      x[0] = expf(x[0] - ref);
      x[1] = expf(x[1] - ref);
      sr[0] = seen >> lane & 1ull ? x[0] : -0.f;             // (a weight of 0 counts: times infinity it is NaN)
      sr[32] = seen >> (lane + 32) & 1ull ? x[1] : -0.f;
      float sum = x[0] + x[1];
#pragma unroll
      for (int z = 1; z < 32; z <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, z);
      if (lane == i) {
        k = expf(m0 - ref);
        l = l * k + sum;
        m = top;
      }
    }
    if (__any_sync(0xffffffffu, k != 1.f))
#pragma unroll
      for (int i = 0; i < MR; ++i) {
        const float ki = __shfl_sync(0xffffffffu, k, i);
#pragma unroll
        for (int v = 0; v < VP; ++v)
#pragma unroll
          for (int x = 0; x < CW; ++x) o[v][i][x] *= ki;
      }
    __syncwarp();                                            // (a row's weights stay in its warp)
#pragma unroll
    for (int v = 0; v < VP; ++v) {
      if (v >= vc) break;
#pragma unroll 1
      for (int tk = 0; tk < TA_PAGE; tk += VT) {
        const T* vp = next() + lane * CW;
        const float* wp = Ss + warp * TA_PAGE + tk;
        auto add = [&](int k0, auto seen) {                  // four tokens
          float4 w[MR];
#pragma unroll
          for (int i = 0; i < MR; ++i) w[i] = *reinterpret_cast<const float4*>(wp + TT_WARPS * i * TA_PAGE + k0);
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float x[CW];
            tt_load(x, vp + (k0 + k) * VW);
#pragma unroll
            for (int i = 0; i < MR; ++i) {
              const float y = k == 0 ? w[i].x : k == 1 ? w[i].y : k == 2 ? w[i].z : w[i].w;
              if (decltype(seen)::value || __float_as_uint(y) != 0x80000000u) {        // what a row does not see stays out of it, whatever it holds
#pragma unroll
                for (int z = 0; z < CW; ++z) o[v][i][z] = fmaf(y, x[z], o[v][i][z]);
              }
            }
          }
        };
        if (whole) {
#pragma unroll 2
          for (int k0 = 0; k0 < VT; k0 += 4) add(k0, std::true_type());
        } else {
#pragma unroll 1
          for (int k0 = 0; k0 < VT; k0 += 4) add(k0, std::false_type());
        }
      }
    }
  }
  // ---- whole: the rows' outputs; else this CTA's part of them
  const bool done = it.first && it.last;
  if (it.first && !it.last && t == 0) ta_set_split(a, ta_split(a, it));
  const size_t pb = (static_cast<size_t>(blockIdx.x) * 2 + (it.first ? 1 : 0)) * TT_BM;
  float scale = 1.f;                                         // of the row warp + 8 lane
  const int mine = warp + TT_WARPS * lane;
  if (lane < MR && mine < pairs) {
    if (done) {
      const int h = rows.head[mine];
      const float c = a.sink ? ta_sink<T>(a.sink[h], m, l) : 1.f;
      scale = l > 0.f ? ta_head_factor<T>(a, it.r0 + (f0 + mine) / rep, h) * c / l : 0.f;
      if (l != l) scale = l;
    } else {
      *reinterpret_cast<float2*>(a.part_ml + (pb + mine) * 2) = make_float2(m, l);
    }
  }
#pragma unroll
  for (int i = 0; i < MR; ++i) {
    const int row = warp + TT_WARPS * i;
    if (row >= pairs) break;
    const int h = rows.head[row], r = it.r0 + (f0 + row) / rep;
    const float by = __shfl_sync(0xffffffffu, scale, i);
#pragma unroll
    for (int v = 0; v < VP; ++v) {
      const int col = v * VW + lane * CW;
      if (col >= V) continue;
      T* out = static_cast<T*>(a.out) + static_cast<size_t>(r) * a.ldo + static_cast<size_t>(h) * a.ho + col;
      float* part = ta_part(a, static_cast<size_t>(blockIdx.x) * 2 + (it.first ? 1 : 0), row, col >> 3) + (col & 7);
      if (done) tt_store(out, o[v][i], by);
      else tt_store(part, o[v][i], 1.f);
    }
  }
}

template <typename T, int VP, int CW>
__global__ void __launch_bounds__(TT_THREADS, VP == 1 ? 2 : 1)
tree_tile_kernel(const __grid_constant__ TreeAttn a) {
  extern __shared__ __align__(16) float smem_tt[];
  __shared__ TreeItem s_item;
  __shared__ TtRows rows;
  float* Qs = smem_tt;                                       // [64][D, in 64s]
  float* Ss = Qs + TT_BM * ((a.D + 63) / 64 * 64);           // [64][64]
  T* ring = reinterpret_cast<T*>(Ss + TT_BM * TA_PAGE);      // [3][64][68]
  const int t = threadIdx.x;
  pdl_wait();
  pdl_trigger();
  TreeRange range;
  if (t < 32) range = ta_range(a);
  if (t == 0) ta_set_split(a, make_int4(0, 0, 0, 0));
#pragma unroll 1
  while (true) {
    if (t < 32) {
      TreeItem next;
      ta_next(a, range, next);
      if (t == 0) s_item = next;
    }
    __syncthreads();                                         // (everyone is done with the item before)
    const TreeItem it = s_item;
    if (it.nj == 0) break;
    const int pairs = it.n * (a.H / a.G) - it.rt * TT_BM;
    if (pairs <= 8) tt_item<T, VP, CW, 1>(a, it, ring, Qs, Ss, rows);
    else if (pairs <= 16) tt_item<T, VP, CW, 2>(a, it, ring, Qs, Ss, rows);
    else if (pairs <= 32) tt_item<T, VP, CW, 4>(a, it, ring, Qs, Ss, rows);
    else tt_item<T, VP, CW, 8>(a, it, ring, Qs, Ss, rows);
  }
}

// ------------------------------------------------------------------------------------------------ merge
constexpr int TM_MAX_CTAS = 512;

// Every CTA makes the list of the split items' rows (four of an item that begins in one CTA of the first launch and ends in another are a task)
// and takes its share of them; the fewer there are, the more warps join one task.  Parts are added in ascending order within a warp, warps in
// ascending order.  A lane has 4 columns in every 32 of one of the four rows, so that loads are whole lines of the parts' layout (ta_part).
// 5 to 6 us behind the first launch, most of it the way to the first part (8 for rows of 256); 12 us for the 39 MB that 148 CTAs with tiles of
// 256 rows leave (a row per warp: 20).
template <typename T, int VC, int THREADS>                   // VC: 32-column pieces of a row
__global__ void __launch_bounds__(THREADS)
tree_merge_kernel(const __grid_constant__ TreeAttn a) {
  constexpr int WARPS = THREADS / 32, EACH = TM_MAX_CTAS / THREADS, FLIGHT = VC <= 4 ? 4 : VC <= 8 ? 2 : 1;        // parts in flight
  __shared__ int sh[WARPS];
  __shared__ int s_first[TM_MAX_CTAS + 1];                   // tasks of the items in front of CTA c's
  __shared__ float4 s_o[WARPS][32 * VC];
  __shared__ float2 s_ml[WARPS][32];
  __shared__ int4 s_split[TM_MAX_CTAS];
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, V8 = a.V >> 3, V4 = a.V >> 2, rep = a.H / a.G;
  const int half = lane & 1, of4 = lane >> 1 & 3, c8 = lane >> 3;
  const int end = a.zero_rest ? a.starts[a.S] : a.R;         // rows of the requests
  const int each = (a.ctas + THREADS - 1) / THREADS;
  int n[EACH], mine = 0;
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    const int c = t * each + i;
    n[i] = 0;
    if (i < each && c < a.ctas) {
      const int4 sp = ta_get_split(a, c);
      s_split[c] = sp;
      n[i] = ((sp.x >> 16) + 3) >> 2;
    }
    mine += n[i];
  }
  int tasks;
  int before = ta_prefix<THREADS>(mine, sh, tasks);
#pragma unroll
  for (int i = 0; i < EACH; ++i) {
    if (i < each && t * each + i < a.ctas) s_first[t * each + i] = before;
    before += n[i];
  }
  __syncthreads();
  int lw = 31 - __clz(WARPS);                                // log2 of the warps that join one task
  while (lw > 0 && tasks << lw > static_cast<int>(gridDim.x) * WARPS) --lw;
  const int wpt = 1 << lw, tpb = WARPS >> lw, sub = warp & (wpt - 1);
#pragma unroll 1
  for (int task0 = blockIdx.x * tpb; task0 < tasks; task0 += gridDim.x * tpb) {
    const int task = task0 + (warp >> lw);
    int lo = 0, hi = a.ctas;                                 // the last CTA whose tasks begin at or before this one
#pragma unroll 1
    while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (s_first[m] <= task) lo = m; else hi = m; }
    const int4 sp = s_split[lo];
    const int row = (task - s_first[lo]) * 4 + of4;
    const bool on = task < tasks && row < sp.x >> 16;
    const int parts = on ? sp.x & 0xffff : 0;
    // part 0 lies behind the others' in its CTA's pair, see TreeAttn
    auto part = [&](int i) { return static_cast<size_t>(lo + i) * 2 + (i == 0 ? 1 : 0); };
    float m = -INFINITY, l = 0.f;
    float4 o[VC] = {};
#pragma unroll 1
    for (int i0 = sub; i0 < parts; i0 += FLIGHT * wpt) {
      float4 x[FLIGHT][VC];
      float2 ml[FLIGHT];
      float top = m;
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) {
        const int i = i0 + u * wpt;
        ml[u] = i < parts ? __ldcg(reinterpret_cast<const float2*>(a.part_ml) + (part(i) << a.bm_log) + row) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int v = 0; v < VC; ++v)
          if (i < parts && v * 4 + c8 < V8) x[u][v] = __ldcg(reinterpret_cast<const float4*>(ta_part(a, part(i), row, v * 4 + c8)) + half);
      }
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) top = fmaxf(top, ml[u].x);
      const float ref = top == -INFINITY ? 0.f : top, k = ta_exp<T>(m - ref);
      m = top;
      l *= k;
#pragma unroll
      for (int v = 0; v < VC; ++v) { o[v].x *= k; o[v].y *= k; o[v].z *= k; o[v].w *= k; }
#pragma unroll
      for (int u = 0; u < FLIGHT; ++u) {
        if (i0 + u * wpt >= parts) break;
        const float w = ta_exp<T>(ml[u].x - ref);            // (a part counts where it is 0 too: it may hold what is not finite)
        l = fmaf(w, ml[u].y, l);
#pragma unroll
        for (int v = 0; v < VC; ++v)
          if (v * 4 + c8 < V8) {
            o[v].x = fmaf(w, x[u][v].x, o[v].x); o[v].y = fmaf(w, x[u][v].y, o[v].y);
            o[v].z = fmaf(w, x[u][v].z, o[v].z); o[v].w = fmaf(w, x[u][v].w, o[v].w);
          }
      }
    }
    if (wpt > 1) {
      __syncthreads();                                       // (the task before has been read)
      s_ml[warp][lane] = make_float2(m, l);
#pragma unroll
      for (int v = 0; v < VC; ++v)
        if (v * 4 + c8 < V8) s_o[warp][v * 32 + lane] = o[v];
      __syncthreads();
      if (sub == 0) {
        const float m0 = m;
#pragma unroll 1
        for (int i = 1; i < wpt; ++i) m = fmaxf(m, s_ml[warp + i][lane].x);
        const float ref = m == -INFINITY ? 0.f : m, k = ta_exp<T>(m0 - ref);
        l *= k;
#pragma unroll
        for (int v = 0; v < VC; ++v) { o[v].x *= k; o[v].y *= k; o[v].z *= k; o[v].w *= k; }
#pragma unroll 1
        for (int i = 1; i < wpt; ++i) {
          const float2 ml = s_ml[warp + i][lane];
          const float w = ta_exp<T>(ml.x - ref);
          l = fmaf(w, ml.y, l);
#pragma unroll
          for (int v = 0; v < VC; ++v)
            if (v * 4 + c8 < V8) {
              const float4 y = s_o[warp + i][v * 32 + lane];
              o[v].x = fmaf(w, y.x, o[v].x); o[v].y = fmaf(w, y.y, o[v].y); o[v].z = fmaf(w, y.z, o[v].z); o[v].w = fmaf(w, y.w, o[v].w);
            }
        }
      }
    }
    if (!on || sub) continue;
    const int f = sp.w + row, h = sp.z * rep + f % rep, r = sp.y + f / rep;
    const float k = a.sink ? ta_sink<T>(a.sink[h], m, l) : 1.f;
    float scale = l > 0.f ? ta_head_factor<T>(a, r, h) * k / l : 0.f;
    if (l != l) scale = l;
    T* out = static_cast<T*>(a.out) + static_cast<size_t>(r) * a.ldo + static_cast<size_t>(h) * a.ho + c8 * 8 + half * 4;
#pragma unroll
    for (int v = 0; v < VC; ++v)
      if (v * 4 + c8 < V8) stf4(out + v * 32, make_float4(o[v].x * scale, o[v].y * scale, o[v].z * scale, o[v].w * scale));
  }
#pragma unroll 1
  for (int r = end + blockIdx.x; r < a.R; r += gridDim.x)
#pragma unroll 1
    for (int i = t; i < a.H * V4; i += THREADS) {
      const int h = i / V4;
      stf4(static_cast<T*>(a.out) + static_cast<size_t>(r) * a.ldo + static_cast<size_t>(h) * a.ho + (i - h * V4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    }
}
template <typename T, int VC, int THREADS>
static void launch_merge(const TreeAttn& a, cudaStream_t s) {
  // (narrow rows: more CTAs to an SM)
  spark_launch_pdl(tree_merge_kernel<T, VC, THREADS>, dim3((VC <= 4 ? 2 : 1) * a.sms), dim3(THREADS), 0, s, dim3(1, 1, 1), a);
}
template <typename T>
static void launch_merges(const TreeAttn& a, cudaStream_t s) {
  if (a.V <= 128) launch_merge<T, 4, 256>(a, s);
  else if (a.V <= 256) launch_merge<T, 8, 256>(a, s);
  else launch_merge<T, 16, 128>(a, s);
}

constexpr int TA_SMEM = 220 * 1024;

template <typename T, int VP, int CW>
static int launch_tile(const TreeAttn& a, cudaStream_t s) {
  auto kern = tree_tile_kernel<T, VP, CW>;
  const int smem = (TT_BM * ((a.D + 63) / 64 * 64) + TT_BM * TA_PAGE) * 4 + TT_STAGES * TT_PIECE * static_cast<int>(sizeof(T));
  if (smem > TA_SMEM) return -6;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TA_SMEM) != cudaSuccess) return -4;
  spark_launch_pdl(kern, dim3(a.ctas), dim3(TT_THREADS), smem, s, dim3(1, 1, 1), a);
  return spark_launch_rc("spark_tree_attn");
}
template <typename T>
static int launch_tiles(const TreeAttn& a, cudaStream_t s) {
  return a.V <= 64 ? launch_tile<T, 1, 2>(a, s) : a.V <= 128 ? launch_tile<T, 1, 4>(a, s) : a.V <= 256 ? launch_tile<T, 2, 4>(a, s) : launch_tile<T, 4, 4>(a, s);
}

int launch_tree_tc(const TreeAttn& a, cudaStream_t s);       // tree_attn_tc.cu

}  // namespace spark

using namespace spark;

// tc: the tensor-core kernel (bf16, head widths of up to 256; tiles of 128 or 256 rows), else the FP32 units (tiles of 64).
extern "C" int spark_tree_attn(const TreeAttn* a, int f32, int tc, cudaStream_t s) {
  if (a->S <= 0 || a->R <= 0) return 0;
  if (a->H <= 0 || a->G <= 0 || a->H % a->G || a->D <= 0 || a->V <= 0 || ((a->D | a->V) & 7) || a->D > 512 || a->V > 512 || a->ctas <= 0 || a->ctas > TM_MAX_CTAS || a->sms <= 0 ||
      (a->bias && a->bias_n <= 0) || a->page_ld <= 0 || ((a->ldq | a->hq | a->ldo | a->ho) & 3)) return -5;
  if (tc ? f32 || (a->bm_log != 7 && a->bm_log != 8) : 1 << a->bm_log != TT_BM) return -5;
  if (const int rc = tc ? launch_tree_tc(*a, s) : f32 ? launch_tiles<float>(*a, s) : launch_tiles<__nv_bfloat16>(*a, s)) return rc;
  if (f32) launch_merges<float>(*a, s);
  else launch_merges<__nv_bfloat16>(*a, s);
  return spark_launch_rc("spark_tree_attn");
}
