// Attention of drafted trees over a paged cache (64-token pages): every node of a tree sees the request's committed tokens, inside a chunk
// or a window, its ancestors and itself.
//
//   o[j][h] = sum_i p_i v_i / (sum_i p_i + e^(sink_h)),  p_i = e^(cap tanh(scale q.k_i / cap) + bias[h][d] - slope_h d),  d: distance of the
//   positions; a row that sees nothing is 0.  Statistics and sums are fp32 and kept against the running maximum.
//
//   tree_tile    FP32 units: the 32-bit mode and head sizes the tensor-core kernel does not take
//   tree_merge   joins the parts of items that several CTAs share, and zeroes the rows behind the last request
#include "../common/tree_work.cuh"

namespace spark {

// ------------------------------------------------------------------------------------------------ FP32 units
constexpr int TT_BM = 32, TT_THREADS = 128, TT_LDK = 68, TT_LDV = 132, TT_LDS = 68;

// Scores: four rows x four keys per thread over 64-wide pieces of the head; outputs: four rows x eight columns per 128-wide piece of V.
template <typename T, int VC>
__global__ void __launch_bounds__(TT_THREADS)
tree_tile_kernel(const __grid_constant__ TreeAttn a) {
  extern __shared__ __align__(16) float smem_tt[];
  __shared__ TreeItem s_item;
  __shared__ float s_m[TT_BM], s_l[TT_BM], s_f[TT_BM];
  __shared__ int s_pos[TT_BM], s_first[TT_BM], s_at[TA_PAGE];
  const int D = a.D, V = a.V, LDQ = (D + 63) / 64 * 64 + 4, rep = a.H / a.G;
  float* Qs = smem_tt;                                       // [32][LDQ]
  float* Ks = Qs + TT_BM * LDQ;                              // [64][68]
  float* Vs = Ks + TA_PAGE * TT_LDK;                         // [64][132]
  float* Ss = Vs + TA_PAGE * TT_LDV;                         // [32][68]
  const int t = threadIdx.x, ty = t >> 4, tx = t & 15;
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
    __syncthreads();
    const TreeItem it = s_item;
    if (it.nj == 0) break;
    const TreeItem& sg = it;
    const int slot = it.slot, pairs = min(TT_BM, sg.n * rep - it.rt * TT_BM);
    __syncthreads();
    for (int i = t; i < TT_BM * (LDQ / 4); i += TT_THREADS) {
      const int row = i / (LDQ / 4), c = (i - row * (LDQ / 4)) * 4, f = it.rt * TT_BM + row;
      float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
      if (row < pairs && c < D) x = ldf4(static_cast<const T*>(a.q) + static_cast<size_t>(sg.r0 + f / rep) * a.ldq + static_cast<size_t>(it.g * rep + f % rep) * a.hq + c);
      *reinterpret_cast<float4*>(Qs + row * LDQ + c) = x;
    }
    if (t < TT_BM) {
      const int p = t < pairs ? a.pos[sg.r0 + (it.rt * TT_BM + t) / rep] : 0;
      s_pos[t] = p;
      s_first[t] = ta_first_visible(a, p);
      s_m[t] = -INFINITY;
      s_l[t] = 0.f;
    }
    float o[VC][4][8] = {};
    for (int j = it.j; j < it.j + it.nj; ++j) {
      const int page = ta_page(a, slot, j), tok0 = j * TA_PAGE;
      if (page < 0 && t == 0) set_status(a.status, ST_BOUNDS, sg.r0, tok0, slot);
      const int valid = page < 0 ? 0 : min(TA_PAGE, sg.len + sg.n - tok0);
      const T* kp = static_cast<const T*>(a.k) + max(page, 0) * a.k_page + static_cast<size_t>(it.g) * D;
      const T* vp = static_cast<const T*>(a.v) + max(page, 0) * a.v_page + static_cast<size_t>(it.g) * V;
      if (t < TA_PAGE) {
        const int node = tok0 + t - sg.len;
        s_at[t] = node < 0 ? tok0 + t : (node < sg.n ? a.pos[sg.r0 + node] : 0);
      }
      float s[4][4] = {};
      for (int d0 = 0; d0 < D; d0 += 64) {
        __syncthreads();
        for (int i = t; i < TA_PAGE * 16; i += TT_THREADS) {
          const int row = i >> 4, c = (i & 15) * 4;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (row < valid && d0 + c < D) x = ldf4(kp + row * a.k_tok + d0 + c);
          *reinterpret_cast<float4*>(Ks + row * TT_LDK + c) = x;
        }
        __syncthreads();
#pragma unroll 4
        for (int c = 0; c < 64; c += 4) {
          float4 q[4], k[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) q[i] = *reinterpret_cast<const float4*>(Qs + (ty * 4 + i) * LDQ + d0 + c);
#pragma unroll
          for (int i = 0; i < 4; ++i) k[i] = *reinterpret_cast<const float4*>(Ks + (tx + 16 * i) * TT_LDK + c);
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[i][e] = fmaf(q[i].x, k[e].x, fmaf(q[i].y, k[e].y, fmaf(q[i].z, k[e].z, fmaf(q[i].w, k[e].w, s[i][e]))));
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int row = ty * 4 + i, f = it.rt * TT_BM + row, h = it.g * rep + f % rep, node = f / rep;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int key = tx + 16 * e, kn = tok0 + key - sg.len;
          bool on = row < pairs && key < valid && s_at[key] >= s_first[row];
          if (on && kn >= 0) on = a.anc ? (kn >> 5) < a.words && (a.anc[static_cast<size_t>(sg.r0 + node) * a.words + (kn >> 5)] >> (kn & 31)) & 1u : kn <= node;
          float x = -INFINITY;
          if (on) {
            const int dist = s_pos[row] - s_at[key];
            x = s[i][e] * a.scale;
            if (a.cap > 0.f) x = a.cap * tanhf(x / a.cap);
            if (a.bias) x += a.bias[static_cast<size_t>(h) * a.bias_n + min(max(dist, 0), a.bias_n - 1)];
            if (a.slopes) x -= a.slopes[h] * static_cast<float>(dist);
          }
          Ss[row * TT_LDS + key] = x;
        }
      }
      __syncthreads();
      {                                                      // statistics: four threads per row
        const int row = t >> 2, c = t & 3;
        float* sr = Ss + row * TT_LDS + c;
        float mx = -INFINITY;
#pragma unroll
        for (int i = 0; i < 16; ++i) mx = fmaxf(mx, sr[4 * i]);
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 1));
        mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 2));
        const float m0 = s_m[row], m = fmaxf(m0, mx), ref = m == -INFINITY ? 0.f : m;
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const float e = expf(sr[4 * i] - ref);
          sr[4 * i] = e;
          sum += e;
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        __syncwarp();
        if (c == 0) {
          const float f = expf(m0 - ref);
          s_f[row] = f;
          s_m[row] = m;
          s_l[row] = s_l[row] * f + sum;
        }
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float f = s_f[ty * 4 + i];
#pragma unroll
        for (int v = 0; v < VC; ++v)
#pragma unroll
          for (int e = 0; e < 8; ++e) o[v][i][e] *= f;
      }
#pragma unroll
      for (int v = 0; v < VC; ++v) {
        if (v) __syncthreads();
        for (int i = t; i < TA_PAGE * 32; i += TT_THREADS) {
          const int row = i >> 5, c = (i & 31) * 4;
          float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
          if (row < valid && v * 128 + c < V) x = ldf4(vp + row * a.v_tok + v * 128 + c);
          *reinterpret_cast<float4*>(Vs + row * TT_LDV + c) = x;
        }
        __syncthreads();
        for (int k = 0; k < TA_PAGE; ++k) {
          const float4 x = *reinterpret_cast<const float4*>(Vs + k * TT_LDV + tx * 4), y = *reinterpret_cast<const float4*>(Vs + k * TT_LDV + 64 + tx * 4);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float p = Ss[(ty * 4 + i) * TT_LDS + k];
            if (p != 0.f) {                                  // what a row does not see stays out of it, whatever it holds
              o[v][i][0] = fmaf(p, x.x, o[v][i][0]); o[v][i][1] = fmaf(p, x.y, o[v][i][1]);
              o[v][i][2] = fmaf(p, x.z, o[v][i][2]); o[v][i][3] = fmaf(p, x.w, o[v][i][3]);
              o[v][i][4] = fmaf(p, y.x, o[v][i][4]); o[v][i][5] = fmaf(p, y.y, o[v][i][5]);
              o[v][i][6] = fmaf(p, y.z, o[v][i][6]); o[v][i][7] = fmaf(p, y.w, o[v][i][7]);
            }
          }
        }
      }
    }
    // ---- whole: the rows' outputs; else this CTA's part of them
    const bool whole = it.first && it.last;
    if (it.first && !it.last && t == 0) ta_set_split(a, ta_split(a, it));
    const size_t pb = (static_cast<size_t>(blockIdx.x) * 2 + (it.first ? 1 : 0)) * TT_BM;
    if (!whole && t < pairs) { a.part_ml[(pb + t) * 2] = s_m[t]; a.part_ml[(pb + t) * 2 + 1] = s_l[t]; }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = ty * 4 + i, f = it.rt * TT_BM + row, h = it.g * rep + f % rep, r = sg.r0 + f / rep;
      if (row >= pairs) continue;
      float scale = 1.f;
      if (whole) {
        float l = s_l[row], c = 1.f;
        if (a.sink) {
          const float m = fmaxf(s_m[row], a.sink[h]);
          c = expf(s_m[row] - m);
          l = l * c + expf(a.sink[h] - m);
        }
        scale = l > 0.f ? ta_head_factor<T>(a, r, h) * c / l : 0.f;
        if (l != l) scale = l;
      }
#pragma unroll
      for (int v = 0; v < VC; ++v)
#pragma unroll
        for (int half = 0; half < 2; ++half) {
          const int col = v * 128 + half * 64 + tx * 4;
          if (col >= V) continue;
          const float4 x = make_float4(o[v][i][half * 4] * scale, o[v][i][half * 4 + 1] * scale, o[v][i][half * 4 + 2] * scale, o[v][i][half * 4 + 3] * scale);
          if (whole) stf4(static_cast<T*>(a.out) + static_cast<size_t>(r) * a.ldo + static_cast<size_t>(h) * a.ho + col, x);
          else *reinterpret_cast<float4*>(a.part_o + (pb + row) * V + col) = x;
        }
    }
  }
}

// ------------------------------------------------------------------------------------------------ merge
// exponential of the outputs' accuracy
template <typename T> __device__ __forceinline__ float tm_exp(float x) { return sizeof(T) == 2 ? __expf(x) : expf(x); }

constexpr int TM_THREADS = 256, TM_WARPS = TM_THREADS / 32, TM_MAX_CTAS = 1024;

// Every CTA makes the list of the split items' rows (a row per item that begins in one CTA of the first launch and ends in another) and
// takes its share of them; the fewer there are, the more warps join one row.  Parts are added in ascending order within a warp, warps in
// ascending order.
template <typename T, int VC>                                // VC: 128-column pieces of a row
__global__ void __launch_bounds__(TM_THREADS)
tree_merge_kernel(const __grid_constant__ TreeAttn a) {
  __shared__ int sh[TM_WARPS];
  __shared__ int s_first[TM_MAX_CTAS + 1];                   // rows of the items in front of CTA c's
  __shared__ float4 s_o[TM_WARPS][32 * VC];
  __shared__ float s_ml[TM_WARPS][2];
  __shared__ int4 s_split[TM_MAX_CTAS];
  pdl_wait();
  pdl_trigger();
  const int t = threadIdx.x, warp = t >> 5, lane = t & 31, V4 = a.V >> 2, rep = a.H / a.G;
  const int end = a.zero_rest ? a.starts[a.S] : a.R;         // rows of the requests
  const int each = (a.ctas + TM_THREADS - 1) / TM_THREADS;   // up to four
  int n[4], mine = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = t * each + i;
    n[i] = 0;
    if (i < each && c < a.ctas) {
      const int4 sp = ta_get_split(a, c);
      s_split[c] = sp;
      n[i] = sp.x >> 16;
    }
    mine += n[i];
  }
  int rows;
  int before = ta_prefix<TM_THREADS>(mine, sh, rows);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (i < each && t * each + i < a.ctas) s_first[t * each + i] = before;
    before += n[i];
  }
  if (t == 0) s_first[a.ctas] = rows;
  __syncthreads();
  int lw = 3;                                                // log2 of the warps that join one row
  while (lw > 0 && rows << lw > static_cast<int>(gridDim.x) * TM_WARPS) --lw;
  const int wpr = 1 << lw, rpb = TM_WARPS >> lw, sub = warp & (wpr - 1);
#pragma unroll 1
  for (int task0 = blockIdx.x * rpb; task0 < rows; task0 += gridDim.x * rpb) {
    const int task = task0 + (warp >> lw);
    const bool on = task < rows;
    int lo = 0, hi = a.ctas;                                 // the last CTA whose rows begin at or before the task
#pragma unroll 1
    while (hi - lo > 1) { const int m = (lo + hi) >> 1; if (s_first[m] <= task) lo = m; else hi = m; }
    const int c = lo, row = on ? task - s_first[lo] : 0;
    const int4 sp = s_split[c];
    const int parts = on ? sp.x & 0xffff : 0;
    // part 0 lies behind the others' in its CTA's pair, see TreeAttn
    auto part = [&](int i) { return ((static_cast<size_t>(c + i) * 2 + (i == 0 ? 1 : 0)) << a.bm_log) + row; };
    float m = -INFINITY, l = 0.f;
    float4 o[VC] = {};
#pragma unroll 1
    for (int i0 = sub; i0 < parts; i0 += 4 * wpr) {          // four parts in flight
      float4 x[4][VC];
      float2 ml[4];
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const int i = i0 + u * wpr;
        ml[u] = i < parts ? __ldcg(reinterpret_cast<const float2*>(a.part_ml + part(i) * 2)) : make_float2(-INFINITY, 0.f);
#pragma unroll
        for (int v = 0; v < VC; ++v)
          if (i < parts && lane + v * 32 < V4) x[u][v] = __ldcg(reinterpret_cast<const float4*>(a.part_o + part(i) * a.V) + lane + v * 32);
      }
      const float top = fmaxf(m, fmaxf(fmaxf(ml[0].x, ml[1].x), fmaxf(ml[2].x, ml[3].x))), ref = top == -INFINITY ? 0.f : top;
      const float k = tm_exp<T>(m - ref);
      m = top;
      l *= k;
#pragma unroll
      for (int v = 0; v < VC; ++v) { o[v].x *= k; o[v].y *= k; o[v].z *= k; o[v].w *= k; }
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const float w = tm_exp<T>(ml[u].x - ref);
        if (w == 0.f && ml[u].y == ml[u].y) continue;        // (a part of NaN scores alone stays)
        l = fmaf(w, ml[u].y, l);
#pragma unroll
        for (int v = 0; v < VC; ++v)
          if (lane + v * 32 < V4) {
            o[v].x = fmaf(w, x[u][v].x, o[v].x); o[v].y = fmaf(w, x[u][v].y, o[v].y);
            o[v].z = fmaf(w, x[u][v].z, o[v].z); o[v].w = fmaf(w, x[u][v].w, o[v].w);
          }
      }
    }
    if (wpr > 1) {
      __syncthreads();                                       // (the task before has been read)
      if (lane == 0) { s_ml[warp][0] = m; s_ml[warp][1] = l; }
#pragma unroll
      for (int v = 0; v < VC; ++v)
        if (lane + v * 32 < V4) s_o[warp][lane + v * 32] = o[v];
      __syncthreads();
      if (sub == 0) {
        for (int i = 1; i < wpr; ++i) m = fmaxf(m, s_ml[warp + i][0]);
        const float ref = m == -INFINITY ? 0.f : m, c0 = tm_exp<T>(s_ml[warp][0] - ref);
        l *= c0;
#pragma unroll
        for (int v = 0; v < VC; ++v) { o[v].x *= c0; o[v].y *= c0; o[v].z *= c0; o[v].w *= c0; }
#pragma unroll 1
        for (int i = 1; i < wpr; ++i) {
          const float w = tm_exp<T>(s_ml[warp + i][0] - ref);
          if (w == 0.f && s_ml[warp + i][1] == s_ml[warp + i][1]) continue;
          l = fmaf(w, s_ml[warp + i][1], l);
#pragma unroll
          for (int v = 0; v < VC; ++v)
            if (lane + v * 32 < V4) {
              const float4 y = s_o[warp + i][lane + v * 32];
              o[v].x = fmaf(w, y.x, o[v].x); o[v].y = fmaf(w, y.y, o[v].y); o[v].z = fmaf(w, y.z, o[v].z); o[v].w = fmaf(w, y.w, o[v].w);
            }
        }
      }
    }
    if (!on || sub) continue;
    const int f = sp.w + row, h = sp.z * rep + f % rep, r = sp.y + f / rep;
    float k = 1.f;
    if (a.sink) {
      const float M = fmaxf(m, a.sink[h]);
      k = tm_exp<T>(m - M);
      l = l * k + tm_exp<T>(a.sink[h] - M);
    }
    float scale = l > 0.f ? ta_head_factor<T>(a, r, h) * k / l : 0.f;
    if (l != l) scale = l;
#pragma unroll
    for (int v = 0; v < VC; ++v)
      if (lane + v * 32 < V4)
        stf4(static_cast<T*>(a.out) + static_cast<size_t>(r) * a.ldo + static_cast<size_t>(h) * a.ho + (lane + v * 32) * 4,
             make_float4(o[v].x * scale, o[v].y * scale, o[v].z * scale, o[v].w * scale));
  }
#pragma unroll 1
  for (int r = end + blockIdx.x; r < a.R; r += gridDim.x)
#pragma unroll 1
    for (int i = t; i < a.H * V4; i += TM_THREADS) {
      const int h = i / V4;
      stf4(static_cast<T*>(a.out) + static_cast<size_t>(r) * a.ldo + static_cast<size_t>(h) * a.ho + (i - h * V4) * 4, make_float4(0.f, 0.f, 0.f, 0.f));
    }
}

constexpr int TA_SMEM = 220 * 1024;

template <typename T, int VC>
static int launch_tile(const TreeAttn& a, cudaStream_t s) {
  auto kern = tree_tile_kernel<T, VC>;
  const int smem = (TT_BM * ((a.D + 63) / 64 * 64 + 4) + TA_PAGE * (TT_LDK + TT_LDV) + TT_BM * TT_LDS) * 4;
  if (smem > TA_SMEM) return -6;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TA_SMEM) != cudaSuccess) return -4;
  spark_launch_pdl(kern, dim3(a.ctas), dim3(TT_THREADS), smem, s, dim3(1, 1, 1), a);
  return spark_launch_rc("spark_tree_attn");
}
template <typename T>
static int launch_tiles(const TreeAttn& a, cudaStream_t s) {
  return a.V <= 128 ? launch_tile<T, 1>(a, s) : a.V <= 256 ? launch_tile<T, 2>(a, s) : launch_tile<T, 4>(a, s);
}

int launch_tree_tc(const TreeAttn& a, cudaStream_t s);       // tree_attn_tc.cu

}  // namespace spark

using namespace spark;

// tc: the tensor-core kernel (bf16, head widths of up to 256; tiles of 128 or 256 rows), else the FP32 units (tiles of 32).
extern "C" int spark_tree_attn(const TreeAttn* a, int f32, int tc, cudaStream_t s) {
  if (a->S <= 0 || a->R <= 0) return 0;
  if (a->H <= 0 || a->G <= 0 || a->H % a->G || a->D <= 0 || a->V <= 0 || ((a->D | a->V) & 7) || a->D > 512 || a->V > 512 || a->ctas <= 0 || a->ctas > TM_MAX_CTAS || a->sms <= 0 ||
      a->min_tiles <= 0 || (a->bias && a->bias_n <= 0) || a->page_ld <= 0 || ((a->ldq | a->hq | a->ldo | a->ho) & 3)) return -5;
  if (tc ? f32 || (a->bm_log != 7 && a->bm_log != 8) : 1 << a->bm_log != TT_BM) return -5;
  if (const int rc = tc ? launch_tree_tc(*a, s) : f32 ? launch_tiles<float>(*a, s) : launch_tiles<__nv_bfloat16>(*a, s)) return rc;
  // (narrow rows: more CTAs to an SM)
  const dim3 grid((a->V <= 128 ? 4 : 2) * a->sms);
  auto merge = f32 ? (a->V <= 128 ? tree_merge_kernel<float, 1> : a->V <= 256 ? tree_merge_kernel<float, 2> : tree_merge_kernel<float, 4>)
                   : (a->V <= 128 ? tree_merge_kernel<__nv_bfloat16, 1> : a->V <= 256 ? tree_merge_kernel<__nv_bfloat16, 2> : tree_merge_kernel<__nv_bfloat16, 4>);
  spark_launch_pdl(merge, grid, dim3(TM_THREADS), 0, s, dim3(1, 1, 1), *a);
  return spark_launch_rc("spark_tree_attn");
}
