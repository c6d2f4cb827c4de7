// Counts of a request's tokens, and what the penalties, biases and masks make of logits.
//
//   count_tokens   counts[slot][t] = 2 * times generated + (1 if in the prompt), grown by a round's tokens or written anew for a request
//   adjust_rows    z / rep or z * rep of tokens that are in the counts, - freq * generated - pres, + biases, -inf where not allowed
#include "../common/token_rows.cuh"

namespace spark {

// ------------------------------------------------------------------------------------------------ counts

// Integer additions and the prompt's bit: the order of the atomics changes nothing.
__global__ void __launch_bounds__(256)
count_more_kernel(const __grid_constant__ CountTokens a) {
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
constexpr int COUNT_SLICE = 24576;
__global__ void __launch_bounds__(512)
count_anew_kernel(const __grid_constant__ CountTokens a) {
  extern __shared__ __align__(16) int slice[];
  const int s = blockIdx.y, b = blockIdx.x * COUNT_SLICE, len = min(COUNT_SLICE, a.V - b);
  const int slot = a.slots ? a.slots[s] : s;
  if (slot < 0) return;
  if (slot >= a.n_slots) { set_status(a.status, ST_BOUNDS, s, slot, a.n_slots); return; }
  for (int i = threadIdx.x; i < len; i += 512) slice[i] = 0;
  __syncthreads();
  const int n = min(a.n[s], a.P);
  const int* tok = a.tokens + s * a.ld_tokens;
  for (int i = threadIdx.x; i < n; i += 512) {
    const int t = tok[i] - b;
    if (t < 0 || t >= len) continue;
    if (a.prompt) slice[t] = 1;
    else atomicAdd(&slice[t], 2);
  }
  __syncthreads();
  int* out = a.counts + slot * a.ld_counts + b;
  for (int i = threadIdx.x; i < len; i += 512) out[i] = slice[i];
}

// ------------------------------------------------------------------------------------------------ adjustments

constexpr int ADJUST_COLS = 4096;
template <class T>
__global__ void __launch_bounds__(256)
adjust_rows_kernel(const __grid_constant__ AdjustRows a) {
  extern __shared__ int ids[];                     // the lists' entries, then the logits of those in this CTA's columns
  const int r = blockIdx.y, b = blockIdx.x * ADJUST_COLS, e = min(b + ADJUST_COLS, a.V);
  const RowAdjust adj(a.a, r, a.status);
  const T* x = static_cast<const T*>(a.x) + r * a.ldx;
  float* out = a.out + r * a.ldo;
  const int n = adj.entries();
  float* was = reinterpret_cast<float*>(ids + n);
  for (int i = threadIdx.x; i < n; i += 256) {     // (read before they are written: `out` may be the logits)
    const int id = adj.entry(i), col = id < 0 ? -1 : id - a.offset;
    ids[i] = id;
    if (col >= b && col < e) was[i] = logit(x + col);
  }
  __syncthreads();
  for (int col = b + threadIdx.x; col < e; col += 256) out[col] = adj.common(logit(x + col), col);
  if (!n) return;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += 256) {
    const int col = ids[i] < 0 ? -1 : ids[i] - a.offset;
    float y;
    if (col >= b && col < e && adj.listed(i, ids, col, was[i], y)) out[col] = y;
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
    count_anew_kernel<<<dim3((a->V + COUNT_SLICE - 1) / COUNT_SLICE, a->S), 512, bytes, s>>>(*a);
  } else if (a->P > 0) {
    count_more_kernel<<<dim3((a->P + 255) / 256, a->S), 256, 0, s>>>(*a);
  }
  return spark_launch_rc("spark_count_tokens");
}

extern "C" int spark_adjust_rows(const AdjustRows* a, cudaStream_t s) {
  if (a->R <= 0 || a->V <= 0) return 0;
  const dim3 grid((a->V + ADJUST_COLS - 1) / ADJUST_COLS, a->R);
  const int sm = (a->a.n_drafted + a->a.n_bias) * 8;
  if (a->type == LT_F32) adjust_rows_kernel<float><<<grid, 256, sm, s>>>(*a);
  else if (a->type == LT_BF16) adjust_rows_kernel<__nv_bfloat16><<<grid, 256, sm, s>>>(*a);
  else adjust_rows_kernel<__half><<<grid, 256, sm, s>>>(*a);
  return spark_launch_rc("spark_adjust_rows");
}
