// Counts of a request's tokens, and what the penalties, biases and masks make of logits.
//
//   count_tokens   counts[slot][t] = 2 * times generated + (1 if in the prompt), grown by a round's tokens or written anew for a request
//   adjust_rows    z / rep or z * rep of tokens that are in the counts, - freq * generated - pres, + biases, -inf where not allowed
//
// Bound by memory where rows are many: 64 new rows of 152k counts in 13.0 us (39 MB written: 3 TB/s; every CTA looks through all of its request's tokens,
// 32000 at most here), 256 bf16 rows of 129k with counts, masks and 103 entries each in 69 us (236 MB: 3.4 TB/s; the lists' trips to memory come before
// and after the columns'), four rows in 6.3 us.
#include "../common/token_rows.cuh"

namespace spark {

// ------------------------------------------------------------------------------------------------ counts

// Integer additions and the prompt's bit: the order of the atomics changes nothing.
__global__ void __launch_bounds__(256)
count_more_kernel(const __grid_constant__ CountTokens a) {
  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.y, i = blockIdx.x * 256 + threadIdx.x;
  const int n = min(a.n[s], a.P);
  const int slot = a.slots ? a.slots[s] : s;
  if (slot < 0 || i >= n) return;
  if (slot >= a.n_slots) { set_status(a.status, ST_BOUNDS, s, slot, a.n_slots); return; }
  const int t = a.tokens[s * a.ld_tokens + i];
  if (t < 0 || t >= a.V) return;
  int* c = a.counts + slot * a.ld_counts + t;
  if (a.prompt) atomicOr(c, 1);
  else atomicAdd(c, 2);
}

// A request's row is written whole: a CTA has a slice of the vocabulary in shared memory, marks it by the tokens that fall into it and writes it out.
constexpr int COUNT_SLICE = 24576, COUNT_THREADS = 1024;
__global__ void __launch_bounds__(COUNT_THREADS)
count_anew_kernel(const __grid_constant__ CountTokens a) {
  extern __shared__ __align__(16) int slice[];
  pdl_wait();
  pdl_trigger();
  const int s = blockIdx.y, b = blockIdx.x * COUNT_SLICE, len = min(COUNT_SLICE, a.V - b), t0 = threadIdx.x;
  const int slot = a.slots ? a.slots[s] : s;
  if (slot < 0) return;
  if (slot >= a.n_slots) { set_status(a.status, ST_BOUNDS, s, slot, a.n_slots); return; }
  for (int i = t0; i < (len + 3) / 4; i += COUNT_THREADS) reinterpret_cast<int4*>(slice)[i] = make_int4(0, 0, 0, 0);
  __syncthreads();
  const int n = min(a.n[s], a.P);
  const int* tok = a.tokens + s * a.ld_tokens;
  const auto mark = [&](int t) {
    t -= b;
    if (t < 0 || t >= len) return;
    if (a.prompt) slice[t] = 1;                    // (whoever writes it)
    else atomicAdd(&slice[t], 2);
  };
  int done = 0;
  if ((reinterpret_cast<uintptr_t>(tok) & 15) == 0) {
    constexpr int U = 4;
    const int whole = n / 4;
    for (int i = t0; i < whole; i += U * COUNT_THREADS) {
      int4 q[U];
#pragma unroll
      for (int u = 0; u < U; ++u) q[u] = i + u * COUNT_THREADS < whole ? __ldg(reinterpret_cast<const int4*>(tok) + i + u * COUNT_THREADS) : make_int4(-1, -1, -1, -1);
#pragma unroll
      for (int u = 0; u < U; ++u) { mark(q[u].x); mark(q[u].y); mark(q[u].z); mark(q[u].w); }
    }
    done = max(whole, 0) * 4;
  }
  for (int i = done + t0; i < n; i += COUNT_THREADS) mark(__ldg(tok + i));
  __syncthreads();
  int* out = a.counts + slot * a.ld_counts + b;
  done = 0;
  if ((reinterpret_cast<uintptr_t>(out) & 15) == 0) {
    for (int i = t0; i < len / 4; i += COUNT_THREADS) reinterpret_cast<int4*>(out)[i] = reinterpret_cast<const int4*>(slice)[i];
    done = len / 4 * 4;
  }
  for (int i = done + t0; i < len; i += COUNT_THREADS) out[i] = slice[i];
}

// ------------------------------------------------------------------------------------------------ adjustments

// Four columns of 16 or 8 bytes.
__device__ __forceinline__ float4 four(const float* p) { return *reinterpret_cast<const float4*>(p); }
template <class H>
__device__ __forceinline__ float4 four(const H* p) {
  const uint2 q = *reinterpret_cast<const uint2*>(p);
  const H* a = reinterpret_cast<const H*>(&q.x);
  const H* b = reinterpret_cast<const H*>(&q.y);
  return make_float4(logit(a), logit(a + 1), logit(b), logit(b + 1));
}

// A CTA has some tiles of ADJUST_COLS columns of a row: first all of them as if nothing were drafted and no bias given, then those in the lists again,
// by what they were.
constexpr int ADJUST_THREADS = 256, ADJUST_COLS = ADJUST_THREADS * 16;
template <class T>
__global__ void __launch_bounds__(ADJUST_THREADS, 5)
adjust_rows_kernel(const __grid_constant__ AdjustRows a, int tiles) {
  extern __shared__ int ids[];                     // the lists' entries, and of those in this CTA's columns what belongs to them
  pdl_wait();
  pdl_trigger();
  const int r = blockIdx.y, b = blockIdx.x * tiles * ADJUST_COLS, e = min(b + tiles * ADJUST_COLS, a.V), t = threadIdx.x;
  const T* x = static_cast<const T*>(a.x) + r * a.ldx;
  float* out = a.out + r * a.ldo;
  const RowAdjust adj(a.a, r, a.status);
  const int n = adj.entries();
  float *was = reinterpret_cast<float*>(ids + n), *more = was + n;
  int* count = ids + 3 * n;
  bool any = false;                                // whether any entry is of these columns
  if (n) {
    for (int i = t; i < n; i += ADJUST_THREADS) {  // (read before they are written: `out` may be the logits)
      const int id = adj.entry(i), col = id < 0 ? -1 : id - a.offset;
      ids[i] = id;
      if (i >= adj.nd) more[i] = adj.bias[i - adj.nd];
      if (col < b || col >= e) continue;
      was[i] = logit(x + col);
      count[i] = adj.allows(col) ? (adj.counts ? max(adj.counts[col], 0) : 0) : -1;
      any = true;
    }
    any = __syncthreads_or(any);
  }
  const uintptr_t places = reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(adj.counts) | reinterpret_cast<uintptr_t>(x) * (4 / sizeof(T));
  if ((places & 15) == 0) {
    constexpr int U = ADJUST_COLS / ADJUST_THREADS / 4;
#pragma unroll 1
    for (int at = b; at < e; at += ADJUST_COLS) {
      float4 z[U];
      int4 c[U];
      uint32_t bits[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = at + (u * ADJUST_THREADS + t) * 4;
        if (col + 4 > e) continue;
        z[u] = four(x + col);
        c[u] = adj.counts ? __ldg(reinterpret_cast<const int4*>(adj.counts + col)) : make_int4(0, 0, 0, 0);
        bits[u] = adj.allowed ? __ldg(adj.allowed + (col >> 5)) >> (col & 31) : 15u;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int col = at + (u * ADJUST_THREADS + t) * 4;
        if (col + 4 > e) {
          for (int i = col; i < e; ++i) out[i] = adj.common(logit(x + i), i);
          continue;
        }
        float4 y = z[u];
        if (c[u].x | c[u].y | c[u].z | c[u].w)
          y = make_float4(adj.penalised(y.x, c[u].x, 0), adj.penalised(y.y, c[u].y, 0), adj.penalised(y.z, c[u].z, 0), adj.penalised(y.w, c[u].w, 0));
        if (!(bits[u] & 1)) y.x = -INFINITY;
        if (!(bits[u] & 2)) y.y = -INFINITY;
        if (!(bits[u] & 4)) y.z = -INFINITY;
        if (!(bits[u] & 8)) y.w = -INFINITY;
        *reinterpret_cast<float4*>(out + col) = y;
      }
    }
  } else {
    constexpr int U = 8;
    for (int col = b + t; col < e; col += U * ADJUST_THREADS) {
      float z[U];
      int c[U];
      uint32_t words[U];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = min(col + u * ADJUST_THREADS, e - 1);
        z[u] = logit(x + at);
        c[u] = adj.counts ? __ldg(adj.counts + at) : 0;
        words[u] = adj.allowed ? __ldg(adj.allowed + (at >> 5)) : ~0u;
      }
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const int at = col + u * ADJUST_THREADS;
        if (at < e) out[at] = words[u] >> (at & 31) & 1 ? adj.penalised(z[u], c[u], 0) : -INFINITY;
      }
    }
  }
  if (!any) return;
  __syncthreads();
  for (int i = t; i < n; i += ADJUST_THREADS) {
    const int col = ids[i] < 0 ? -1 : ids[i] - a.offset;
    if (col < b || col >= e) continue;
    // all entries of its id together; where one in front of it is of the same id, that one does it
    int first = i, times = 0;
    for (int j = 0; j < adj.nd; ++j)
      if (ids[j] == ids[i]) { first = min(first, j); ++times; }
    float y = adj.penalised(was[i], max(count[i], 0), times);
    for (int j = adj.nd; j < n; ++j)
      if (ids[j] == ids[i]) { first = min(first, j); y = __fadd_rn(y, more[j]); }
    if (first == i) out[col] = count[i] < 0 ? -INFINITY : y;
  }
}

}  // namespace spark

using namespace spark;

extern "C" unsigned spark_sampling_layout() { return SPARK_SAMPLING_LAYOUT; }

extern "C" int spark_count_tokens(const CountTokens* a, cudaStream_t s) {
  if (a->S <= 0 || a->V <= 0) return 0;
  if (a->reset) {
    constexpr int bytes = COUNT_SLICE * 4;
    if (cudaFuncSetAttribute(count_anew_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return spark_launch_rc("spark_count_tokens");
    spark_launch_pdl(count_anew_kernel, dim3((a->V + COUNT_SLICE - 1) / COUNT_SLICE, a->S), dim3(COUNT_THREADS), bytes, s, dim3(1, 1, 1), *a);
  } else if (a->P > 0) {
    spark_launch_pdl(count_more_kernel, dim3((a->P + 255) / 256, a->S), dim3(256), 0, s, dim3(1, 1, 1), *a);
  }
  return spark_launch_rc("spark_count_tokens");
}

extern "C" int spark_adjust_rows(const AdjustRows* a, cudaStream_t s) {
  if (a->R <= 0 || a->V <= 0) return 0;
  // Tiles per CTA: one where that fills the GPU no more than once, else four (their lists are read once for all of them).
  const int all = (a->V + ADJUST_COLS - 1) / ADJUST_COLS, tiles = static_cast<long long>(all) * a->R <= 4ll * a->sms ? 1 : all < 4 ? all : 4;
  const dim3 grid((all + tiles - 1) / tiles, a->R), block(ADJUST_THREADS), one(1, 1, 1);
  const int sm = (a->a.n_drafted + a->a.n_bias) * 16;
  if (a->type == LT_F32) spark_launch_pdl(adjust_rows_kernel<float>, grid, block, sm, s, one, *a, tiles);
  else if (a->type == LT_BF16) spark_launch_pdl(adjust_rows_kernel<__nv_bfloat16>, grid, block, sm, s, one, *a, tiles);
  else spark_launch_pdl(adjust_rows_kernel<__half>, grid, block, sm, s, one, *a, tiles);
  return spark_launch_rc("spark_adjust_rows");
}
