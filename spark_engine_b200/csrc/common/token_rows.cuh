// Logits of a row as the token kernels see them: their order, the adjustments that clients ask for, reductions over a cluster's CTAs.
#pragma once
#include <cooperative_groups.h>

#include "rows.cuh"
#include "sampling_args.h"

namespace spark {

namespace cg = cooperative_groups;

__device__ __forceinline__ float logit(const float* p) { return *p; }
__device__ __forceinline__ float logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float logit(const __half* p) { return __half2float(*p); }

// What is not a number is no token, as -inf.
__device__ __forceinline__ float plain_logit(float z) { return fmaxf(z, -INFINITY); }

template <class T> constexpr int LOGITS_16B = 16 / sizeof(T);
__device__ __forceinline__ void unpack(const uint4& q, float (&f)[4]) {
  f[0] = __uint_as_float(q.x); f[1] = __uint_as_float(q.y); f[2] = __uint_as_float(q.z); f[3] = __uint_as_float(q.w);
}
template <class H>
__device__ __forceinline__ void unpack_halves(const uint4& q, float (&f)[8]) {
  const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const H* h = reinterpret_cast<const H*>(&w[i]);
    f[2 * i] = logit(h);
    f[2 * i + 1] = logit(h + 1);
  }
}
template <class T>
__device__ __forceinline__ void unpack_logits(const uint4& q, float (&f)[LOGITS_16B<T>]) {
  if constexpr (sizeof(T) == 4) unpack(q, f);
  else unpack_halves<T>(q, f);
}

// ------------------------------------------------------------------------------------------------ adjustments

// A row's adjustments, for the columns that belong to ids offset .. offset + V.
struct RowAdjust {
  const int* counts = nullptr;                     // the row's, or null
  const int *drafted = nullptr, *bias_ids = nullptr;
  const float* bias = nullptr;
  const uint32_t* allowed = nullptr;
  float rep = 1.f, pres = 0.f, freq = 0.f;
  int nd = 0, nb = 0;

  __device__ __forceinline__ RowAdjust(const Adjustments& a, int r, int* status) {
    const int slot = a.slots ? a.slots[r] : r;
    if (slot >= 0) {
      if (a.repetition) rep = a.repetition[r];
      if (a.presence) pres = a.presence[r];
      if (a.frequency) freq = a.frequency[r];
      if (a.drafted) { nd = a.n_drafted; drafted = a.drafted + static_cast<long long>(r) * nd; }
      if (a.counts) {
        if (slot < a.n_slots) {
          counts = a.counts + slot * a.ld_counts;
        } else {                                   // (what the row has said is not known: it has no penalties)
          set_status(status, ST_BOUNDS, r, slot, a.n_slots);
          rep = 1.f; pres = freq = 0.f; nd = 0;
        }
      }
    }
    if (a.bias_ids) { nb = a.n_bias; bias_ids = a.bias_ids + static_cast<long long>(r) * nb; bias = a.bias + static_cast<long long>(r) * nb; }
    if (a.allowed) allowed = a.allowed + static_cast<long long>(r) * a.words;
  }
  // Rounded after every step, as the definition is: products and differences are not contracted.
  __device__ __forceinline__ float penalised(float z, int count, int more) const {
    const int c = (count >> 1) + more;
    if (count > 0 || more > 0) z = z > 0.f ? __fdiv_rn(z, rep) : __fmul_rn(z, rep);
    z = __fsub_rn(z, __fmul_rn(freq, static_cast<float>(c)));
    return __fsub_rn(z, c > 0 ? pres : 0.f);
  }
  __device__ __forceinline__ bool allows(int col) const { return !allowed || (allowed[col >> 5] >> (col & 31) & 1); }
  // Column `col` with nothing drafted and no bias.
  __device__ __forceinline__ float common(float z, int col) const {
    z = penalised(z, counts ? counts[col] : 0, 0);
    return allows(col) ? z : -INFINITY;
  }
  // Entries of the lists: drafted tokens, then biases.
  __device__ __forceinline__ int entries() const { return nd + nb; }
  __device__ __forceinline__ int entry(int i) const { return i < nd ? drafted[i] : bias_ids[i - nd]; }
};

// ------------------------------------------------------------------------------------------------ reductions

struct Best {                                      // the first of an order: value descending, id ascending
  float v;
  int id;
};
__device__ __forceinline__ Best first_of(Best a, Best b) { return b.v > a.v || (b.v == a.v && b.id < a.id) ? b : a; }
constexpr int NO_ID = 0x7fffffff;

template <class V>
__device__ __forceinline__ V shfl_words(V v, int o) {
  static_assert(sizeof(V) % 4 == 0, "words");
  union { V v; int w[sizeof(V) / 4]; } a, b;
  a.v = v;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(V) / 4); ++i) b.w[i] = __shfl_xor_sync(0xffffffffu, a.w[i], o);
  return b.v;
}

template <class V>
__device__ __forceinline__ V bcast_words(V v) {    // lane 0's
  union { V v; int w[sizeof(V) / 4]; } a, b;
  a.v = v;
#pragma unroll
  for (int i = 0; i < static_cast<int>(sizeof(V) / 4); ++i) b.w[i] = __shfl_sync(0xffffffffu, a.w[i], 0);
  return b.v;
}

// Values of a row's cluster.  A CTA writes its value to every CTA's boxes and all meet at a barrier: what is read then is near.  Two sets in turn, so that
// one barrier per reduction is enough.
struct alignas(16) Mail { unsigned long long w[4]; };
struct Mailboxes {
  Mail box[2][8], warp[16];
};
struct Cluster {
  cg::cluster_group g;
  Mailboxes* mine;
  int phase = 0, rank, size;
  __device__ __forceinline__ explicit Cluster(Mailboxes* m) : g(cg::this_cluster()), mine(m), rank(static_cast<int>(g.block_rank())), size(static_cast<int>(g.num_blocks())) {
    if (size > 1) asm volatile("barrier.cluster.arrive.relaxed.aligned;" ::: "memory");
  }
  // Once, before anything is written to another CTA: all of them run.
  __device__ __forceinline__ void ready() {
    if (size > 1) asm volatile("barrier.cluster.wait.aligned;" ::: "memory");
  }
  __device__ __forceinline__ void sync() {
    if (size > 1) g.sync();
    else __syncthreads();
  }
  template <class V>
  __device__ __forceinline__ V* of(V* p, int r) { return size > 1 ? g.map_shared_rank(p, r) : p; }

  // Warp 0's value, which every CTA finds at its rank in `box` afterwards.
  template <class V>
  __device__ __forceinline__ const Mail* tell(V v) {
    static_assert(sizeof(V) <= sizeof(Mail), "mailboxes");
    if (threadIdx.x < size) *reinterpret_cast<V*>(of(&mine->box[phase][rank], threadIdx.x)) = v;
    sync();
    const Mail* b = mine->box[phase];
    phase ^= 1;
    return b;
  }
  // op over the block's threads; warp 0 gets it.
  template <class V, class Op>
  __device__ __forceinline__ V block(V v, V none, Op op) {
    static_assert(sizeof(V) <= sizeof(Mail), "mailboxes");
    const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
#pragma unroll
    for (int o = 16; o; o >>= 1) v = op(v, shfl_words(v, o));
    if (lane == 0) *reinterpret_cast<V*>(&mine->warp[w]) = v;
    __syncthreads();
    if (w == 0) {
      v = lane < nw ? *reinterpret_cast<V*>(&mine->warp[lane]) : none;
#pragma unroll
      for (int o = 8; o; o >>= 1) v = op(v, shfl_words(v, o));     // (at most 16 warps)
    }
    return v;
  }
  // op over all threads of the cluster, in an order that is the same in every run; every thread gets it.
  template <class V, class Op>
  __device__ __forceinline__ V reduce(V v, V none, Op op) {
    const Mail* b = tell(bcast_words(block(v, none, op)));
    v = *reinterpret_cast<const V*>(b);
    for (int r = 1; r < size; ++r) v = op(v, *reinterpret_cast<const V*>(b + r));
    return v;
  }
};

}  // namespace spark
