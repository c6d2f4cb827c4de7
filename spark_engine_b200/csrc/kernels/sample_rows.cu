// Tokens and log-probabilities from rows of logits.
//
// A row's tokens are ordered by (logit descending, id ascending); NaN and -inf are no tokens.  With w_v = e^{(z_v - max) / T}:
//
//   sample     kept are the first k tokens; of them those with (z - max) / T >= log(min_p); of those the shortest prefix whose weight is >= top_p of theirs.
//              The token is the arg-max over kept of fl(fl(z / T) + fl(g)), g = -log(-log u(seed, position, id)).
//   logprobs   z_t - max - log sum e^{z - max}, the rank of t, the first tokens of the order
//
// What is kept is always a prefix of the order, given by its last token.
//
// A row lies in the shared memory of a cluster's CTAs: it is read once, whatever the passes over it.  The prefix is found among a few candidates where
// there are few: the largest of every eight logits go to a histogram, whose first bins with k tokens (or top_p of the weight) in them hold what is kept,
// since the other seven only add to it; what lies in these bins goes to a list, which one CTA sorts.  Where more are kept than the list takes, the k-th
// token comes from a histogram of all, and for top_p a token is drawn first and its weight in front looked at then: a prefix of the order that ends in
// front of a token drawn in vain holds all that is kept, and holds half as much on average.
#include "../common/token_rows.cuh"

namespace spark {

constexpr int ROW_THREADS = 512, ROW_WARPS = ROW_THREADS / 32;
constexpr int ROW_BLOCK = 256;                     // logits that a warp takes at once, 8 per lane
constexpr int ROW_SLICE_MAX = SAMPLE_MAX_V / 16;
constexpr int ROW_PAD = ROW_BLOCK + 8;
constexpr int BINS = 1024;                         // of a sixteenth of a bit of weight; what weighs less than 2^-64 shares the last one
constexpr float BINS_PER_BIT = 16.f;
constexpr int LIST = 2048;

using u64 = unsigned long long;

__device__ __forceinline__ uint32_t order_key(float z) {       // larger logits have larger keys
  const uint32_t b = __float_as_uint(z + 0.f);                 // (zeros are equal whatever their sign)
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_order(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ u64 list_key(float z, int id) { return static_cast<u64>(order_key(z)) << 32 | static_cast<uint32_t>(~id); }
__device__ __forceinline__ float list_z(u64 k) { return key_order(static_cast<uint32_t>(k >> 32)); }
__device__ __forceinline__ int list_id(u64 k) { return static_cast<int>(~static_cast<uint32_t>(k)); }

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max4(const float4& a) { return fmaxf(fmaxf(a.x, a.y), fmaxf(a.z, a.w)); }

// A prefix of the order: its last token.
struct Prefix { float z; int id; };
__device__ __forceinline__ bool within(const Prefix& p, float z, int id) { return z > p.z || (z == p.z && id <= p.id); }
constexpr float LOWEST = -3.402823466e38f;

struct RowShared {
  Mailboxes mail;
  unsigned count[BINS], mass[BINS];
  u64 list[LIST];
  u64 warp[ROW_WARPS];
  double dwarp[ROW_WARPS];
  unsigned n_list, before, kept;
  int bin;
  float z;
  Prefix cut;
  u64 total;
};

// ------------------------------------------------------------------------------------------------ a CTA's part of a row

// This CTA's logits as fp32 in shared memory: z[j] is id first + j; -inf in front of them, behind them and up to whole blocks.
struct Slice {
  float* z;
  int first, blocks;

  template <class F>
  __device__ __forceinline__ void quads(F f) const {          // f(four logits, id of the first)
    const int lane = threadIdx.x & 31;
    for (int k = threadIdx.x >> 5; k < blocks; k += ROW_WARPS) {
      const int j = k * ROW_BLOCK + lane * 4;
      const float4 a = *reinterpret_cast<const float4*>(z + j), b = *reinterpret_cast<const float4*>(z + j + 128);
      f(a, first + j);
      f(b, first + j + 128);
    }
  }
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    quads([&](const float4& a, int id) { f(a.x, id); f(a.y, id + 1); f(a.z, id + 2); f(a.w, id + 3); });
  }
};

// Columns [b, e) of a row, its best token seen on the way.  Whole 16 bytes are read as such wherever the row starts; their place in shared memory is
// shifted as theirs in memory is.
template <class T, bool ADJUSTED>
__device__ __forceinline__ Slice load_slice(float* z, const T* x, int b, int e, const RowAdjust* adj, int* ids, Best& best) {
  constexpr int N = LOGITS_16B<T>;
  const int t = threadIdx.x, n = e - b;
  const int shift = n ? static_cast<int>(reinterpret_cast<uintptr_t>(x + b) / sizeof(T) % N) : 0, end = shift + n;
  const Slice s{z, b - shift, (end + ROW_BLOCK - 1) / ROW_BLOCK};
  int entries = 0;
  if constexpr (ADJUSTED) {
    entries = adj->entries();
    for (int i = t; i < entries; i += ROW_THREADS) ids[i] = adj->entry(i);
  }
  const auto one = [&](int j) {
    float v = logit(x + b - shift + j);
    if constexpr (ADJUSTED) v = adj->common(v, s.first + j);
    z[j] = v = plain_logit(v);
    best = first_of(best, Best{v, s.first + j});
  };
  const int v0 = shift ? 1 : 0, v1 = end / N;                  // whole vectors
  if (t < N && t >= shift && shift && t < end) one(t);
  if (t < N && v1 >= v0 && v1 * N + t < end) one(v1 * N + t);
  if (t < shift) z[t] = -INFINITY;
  for (int j = end + t; j < s.blocks * ROW_BLOCK; j += ROW_THREADS) z[j] = -INFINITY;
  float top = -INFINITY;
  int at = -1;
  const uint4* src = reinterpret_cast<const uint4*>(x + b - shift);
  const int* cnt = ADJUSTED && adj->counts ? adj->counts + s.first : nullptr;
  const bool counts16 = (reinterpret_cast<uintptr_t>(cnt) & 15) == 0;
  constexpr int U = 4;
  for (int v = v0 + t; v < v1; v += U * ROW_THREADS) {
    uint4 q[U];
#pragma unroll
    for (int u = 0; u < U; ++u)
      if (v + u * ROW_THREADS < v1) q[u] = __ldg(src + v + u * ROW_THREADS);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = (v + u * ROW_THREADS) * N;
      if (v + u * ROW_THREADS >= v1) break;
      float f[N];
      unpack_logits<T>(q[u], f);
      if constexpr (ADJUSTED) {
        int c[N] = {};
        if (cnt && counts16) {
#pragma unroll
          for (int i = 0; i < N; i += 4) *reinterpret_cast<int4*>(c + i) = __ldg(reinterpret_cast<const int4*>(cnt + j + i));
        } else if (cnt) {
#pragma unroll
          for (int i = 0; i < N; ++i) c[i] = __ldg(cnt + j + i);
        }
        uint32_t bits = 0xffffffffu;
        if (adj->allowed) {
          const int col = s.first + j;
          bits = __funnelshift_r(adj->allowed[col >> 5], adj->allowed[(col + N - 1) >> 5], col & 31);
        }
#pragma unroll
        for (int i = 0; i < N; ++i) {
          f[i] = adj->penalised(f[i], c[i], 0);
          if (!(bits >> i & 1)) f[i] = -INFINITY;
        }
      }
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < N; ++i) m = fmaxf(m, f[i] = plain_logit(f[i]));
      if (m > top) { top = m; at = j; }
#pragma unroll
      for (int i = 0; i < N; i += 4) *reinterpret_cast<float4*>(z + j + i) = make_float4(f[i], f[i + 1], f[i + 2], f[i + 3]);
    }
  }
  if (at >= 0) {
    int i = 0;
    while (i < N - 1 && z[at + i] != top) ++i;
    best = first_of(best, Best{top, s.first + at + i});
  }
  if (entries) {                                               // drafted tokens and biases: their columns again
    __syncthreads();
    for (int i = t; i < entries; i += ROW_THREADS) {
      const int col = ids[i];
      float y;
      if (col >= b && col < e && adj->listed(i, ids, col, logit(x + col), y)) z[col - s.first] = plain_logit(y);
    }
    __syncthreads();
    best = Best{-INFINITY, NO_ID};
    s.each([&](float v, int id) { best = first_of(best, Best{v, id}); });
  }
  return s;
}

template <class F>
__device__ __forceinline__ u64 row_count(const Slice& s, Cluster& c, F f) {
  u64 n = 0;
  s.each([&](float z, int id) { n += f(z, id); });
  return c.reduce(n, u64{0}, [](u64 a, u64 b) { return a + b; });
}
__device__ __forceinline__ double row_total(Cluster& c, double v) { return c.reduce(v, 0.0, [](double a, double b) { return a + b; }); }

// Weights relative to the best token's.  The difference comes first: it is exact or rounded by half a step, whatever the logits' size.
struct Weights {
  float top, c;                                    // c = log2(e) / T
  __device__ __forceinline__ float bits(float z) const { return (z - top) * c; }
  __device__ __forceinline__ float operator()(float z) const { return exp2_fast(bits(z)); }
  __device__ __forceinline__ int bin(float z) const { return min(static_cast<int>(bits(z) * -BINS_PER_BIT), BINS - 1); }
};

// Weight of what `f` lets through; four at a time in fp32, 64 bits beyond.
template <class F>
__device__ __forceinline__ double row_mass(const Slice& s, Cluster& c, const Weights& w, F f) {
  double sum = 0;
  s.quads([&](const float4& a, int id) {
    const float p = f(a.x, id) ? w(a.x) : 0.f, q = f(a.y, id + 1) ? w(a.y) : 0.f, r = f(a.z, id + 2) ? w(a.z) : 0.f, t = f(a.w, id + 3) ? w(a.w) : 0.f;
    sum += (p + q) + (r + t);
  });
  return row_total(c, sum);
}

// ------------------------------------------------------------------------------------------------ histograms and lists

__device__ __forceinline__ void clear_bins(RowShared& sh) {
  for (int i = threadIdx.x; i < BINS; i += ROW_THREADS) sh.count[i] = sh.mass[i] = 0;
}

// The leader's: the first bin with which the cluster's bins hold `k` tokens, or `target` of weight (2^16 of a bin's best token's each); the last one
// where they do not; with it the tokens in front of it.
__device__ __forceinline__ void find_bin(RowShared& sh, Cluster& c, bool by_count, unsigned k, double target) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  constexpr int PER = BINS / ROW_THREADS;
  double v[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const int b = t * PER + i;
    unsigned n = 0;
    double m = 0;
    for (int r = 0; r < c.size; ++r) {
      const RowShared* p = c.size > 1 ? c.of(&sh, r) : &sh;
      if (by_count) n += p->count[b];
      else m += p->mass[b];
    }
    v[i] = by_count ? static_cast<double>(n) : m * exp2f(b * (-1.f / BINS_PER_BIT));
    sum += v[i];
  }
  double incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const double y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) sh.dwarp[w] = incl;
  if (t == 0) { sh.bin = BINS - 1; sh.before = 0; }
  __syncthreads();
  double at = incl - sum;
  for (int i = 0; i < w; ++i) at += sh.dwarp[i];
  if (by_count) target = k;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (at < target && at + v[i] >= target) { sh.bin = t * PER + i; sh.before = by_count ? static_cast<unsigned>(at) : 0; }
    at += v[i];
  }
}

// Tokens of the row that `f` lets through, into the leader's list; their number, which may be more than it takes.  Everyone has it.
template <class F>
__device__ __forceinline__ unsigned gather(RowShared& sh, const Slice& s, Cluster& c, float least, F f) {
  s.quads([&](const float4& a, int id) {
    if (!(max4(a) >= least)) return;
    const float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (v[i] >= least && f(v[i], id + i)) {
        const unsigned at = atomicAdd(&sh.n_list, 1u);
        if (at < LIST) sh.list[at] = list_key(v[i], id + i);
      }
  });
  c.sync();
  unsigned n = 0;
  for (int r = 0; r < c.size; ++r) n += c.size > 1 ? *c.of(&sh.n_list, r) : sh.n_list;
  return n;
}
__device__ __forceinline__ void collect(RowShared& sh, Cluster& c) {           // the leader's copy of the others' lists
  unsigned at = sh.n_list;
  for (int r = 1; r < c.size; ++r) {
    const unsigned n = *c.of(&sh.n_list, r);
    const u64* from = c.of(sh.list, r);
    for (unsigned i = threadIdx.x; i < n; i += ROW_THREADS) sh.list[at + i] = from[i];
    at += n;
  }
}

// list[0, n) in the row's order (descending keys; all differ).
__device__ __forceinline__ void sort_list(RowShared& sh, unsigned n) {
  unsigned m = 32;
  while (m < n) m *= 2;
  for (unsigned i = n + threadIdx.x; i < m; i += ROW_THREADS) sh.list[i] = 0;
  __syncthreads();
  for (unsigned k = 2; k <= m; k *= 2)
    for (unsigned j = k / 2; j; j /= 2) {
      for (unsigned p = threadIdx.x; p < m / 2; p += ROW_THREADS) {
        const unsigned a = 2 * p - (p & (j - 1)), b = a + j;
        const u64 x = sh.list[a], y = sh.list[b];
        if ((x < y) == ((a & k) == 0)) { sh.list[a] = y; sh.list[b] = x; }
      }
      __syncthreads();
    }
}

// ------------------------------------------------------------------------------------------------ draws

__device__ __forceinline__ u64 mix64(u64 x) {
  x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
  x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}

struct Top2 { float a1; int id; float a2; int none; };         // the best score, its token, the second best score
__device__ __forceinline__ Top2 best2(Top2 x, Top2 y) {
  const bool first = x.a1 >= y.a1;
  return first ? Top2{x.a1, x.id, fmaxf(x.a2, y.a1), 0} : Top2{y.a1, y.id, fmaxf(y.a2, x.a1), 0};
}

// A token's score is known from below and above at the price of a few fp32 operations: `margin` is more than twice what the rough one may be off.
// Where the two best are further apart than that, the best is the best; else both are computed as the definition says.
struct Race {
  float temp, c, margin;
  u64 key;
  __device__ __forceinline__ Race(float T, float c_, float top, long long seed, long long pos)
      : temp(T), c(c_), margin(1.f / 512 + (fabsf(top / T) + 64.f) * (1.f / 524288)),
        key((static_cast<u64>(seed) * 0x9E3779B97F4A7C15ull) ^ (static_cast<u64>(pos + 1) * 0xBF58476D1CE4E5B9ull)) {}
  __device__ __forceinline__ u64 hash(int id) const { return mix64(static_cast<u64>(id) * 0x9E3779B97F4A7C15ull + key); }
  __device__ __forceinline__ float exact(float z, int id) const {
    const double u = (static_cast<double>(hash(id) >> 11) + 0.5) * (1.0 / 9007199254740992.0);
    return __fadd_rn(__fdiv_rn(z, temp), static_cast<float>(-log(-log(u))));
  }
  // -log u from q = 1 - u where u is near 1 (to q^3 of it), from u where it is near 0; each to 2^-13 of itself.
  __device__ __forceinline__ float rough(float z, u64 h) const {
    const float q = (__ull2float_rn(~h >> 11) + 0.5f) * (1.f / 9007199254740992.f);
    const float L = q < 1.f / 256 ? q * (1.f + q * (0.5f + q * (1.f / 3))) : -__logf(q < 0.5f ? 1.f - q : (__ull2float_rn(h >> 11) + 0.5f) * (1.f / 9007199254740992.f));
    return __fdiv_rn(z, temp) - __logf(L);
  }
};

__device__ __forceinline__ float warp_highest(float v) {
  const int b = __float_as_int(v);
  const int m = __reduce_max_sync(0xffffffffu, b ^ (b >> 31 & 0x7fffffff));
  return __int_as_float(m ^ (m >> 31 & 0x7fffffff));
}

// The token that wins among those within `kept`.  -log u >= 1 - u, so that a score is at most z / T - log(1 - u): most tokens are out of the race by the
// 32 upper bits of their hash, without a logarithm.
__device__ __forceinline__ int draw_row(const Slice& s, Cluster& c, const Race& race, const Prefix& kept, const Best& top) {
  Top2 m{-INFINITY, NO_ID, -INFINITY, 0};
  float bound = race.rough(top.v, race.hash(top.id));          // (the best token is always kept)
  float off = (race.margin - bound) * 1.4426950408889634f + 32.f;
  s.quads([&](const float4& a, int id0) {
    if (__all_sync(0xffffffffu, !(max4(a) >= kept.z))) return;
    const float v[4] = {a.x, a.y, a.z, a.w};
    bool more = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if (!within(kept, v[i], id0 + i)) continue;
      const u64 h = race.hash(id0 + i);
      if (static_cast<float>(static_cast<uint32_t>(~h >> 32)) > exp2_fast(fmaf(v[i], race.c, off))) continue;
      const float y = race.rough(v[i], h);
      m = best2(m, Top2{y, id0 + i, -INFINITY, 0});
      more |= y > bound;
    }
    if (__any_sync(0xffffffffu, more)) {
      bound = fmaxf(bound, warp_highest(m.a1));
      off = (race.margin - bound) * 1.4426950408889634f + 32.f;
    }
  });
  m = c.reduce(m, Top2{-INFINITY, NO_ID, -INFINITY, 0}, best2);
  if (m.a2 < m.a1 - race.margin) return m.id;
  Best b{-INFINITY, NO_ID};
  s.each([&](float v, int id) {
    if (!within(kept, v, id)) return;
    const u64 h = race.hash(id);
    if (race.rough(v, h) < m.a1 - race.margin) return;
    b = first_of(b, Best{race.exact(v, id), id});
  });
  return c.reduce(b, Best{-INFINITY, NO_ID}, first_of).id;
}

// The leader's: the token that wins among the first n of its list.  Thread 0 has it.
__device__ __forceinline__ int draw_list(RowShared& sh, Cluster& c, const Race& race, unsigned n) {
  Top2 m{-INFINITY, NO_ID, -INFINITY, 0};
  for (unsigned i = threadIdx.x; i < n; i += ROW_THREADS) {
    const u64 k = sh.list[i];
    m = best2(m, Top2{race.rough(list_z(k), race.hash(list_id(k))), list_id(k), -INFINITY, 0});
  }
  m = c.block(m, Top2{-INFINITY, NO_ID, -INFINITY, 0}, best2);
  if (threadIdx.x == 0) sh.kept = m.a2 < m.a1 - race.margin;
  __syncthreads();
  if (sh.kept) return m.id;
  Best b{-INFINITY, NO_ID};
  for (unsigned i = threadIdx.x; i < n; i += ROW_THREADS) {
    const u64 k = sh.list[i];
    b = first_of(b, Best{race.exact(list_z(k), list_id(k)), list_id(k)});
  }
  return c.block(b, Best{-INFINITY, NO_ID}, first_of).id;
}

// ------------------------------------------------------------------------------------------------ the k-th token

// By the bits of keys and ids, for the rare row in which more tokens than a list takes share a bin.
__device__ __forceinline__ Prefix kth_by_bits(const Slice& s, Cluster& c, const Prefix& of, u64 k) {
  if (row_count(s, c, [&](float z, int id) { return u64{within(of, z, id)}; }) <= k) return of;
  uint32_t key = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = key | 1u << bit;
    if (row_count(s, c, [&](float z, int id) { return u64{order_key(z) >= t && within(of, z, id)}; }) >= k) key = t;
  }
  const float v = key_order(key);
  k -= row_count(s, c, [&](float z, int) { return u64{z > v}; });
  int id = 0;
  for (int bit = 20; bit >= 0; --bit) {            // the largest id with less than k of these in front of it
    const int t = id | 1 << bit;
    if (row_count(s, c, [&](float z, int i) { return u64{z == v && i < t && within(of, z, i)}; }) < k) id = t;
  }
  return Prefix{v, id};
}

__device__ __forceinline__ Prefix kth_token(RowShared& sh, const Slice& s, Cluster& c, const Weights& w, const Prefix& of, unsigned k) {
  c.sync();                                        // (nobody reads the bins and lists of before any more)
  clear_bins(sh);
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  s.quads([&](const float4& a, int) {
    const float v[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (v[i] >= of.z) atomicAdd(&sh.count[w.bin(v[i])], 1u);
  });
  c.sync();
  if (c.rank == 0) {
    find_bin(sh, c, true, k, 0);
    __syncthreads();
  }
  c.sync();
  const RowShared* lead = c.size > 1 ? c.of(&sh, 0) : &sh;
  const int bin = lead->bin;
  const unsigned before = lead->before;
  // (the last bin's `before` is 0 where the row has fewer than k tokens)
  const unsigned n = gather(sh, s, c, of.z, [&](float z, int) { return w.bin(z) == bin; });
  if (n > LIST) return kth_by_bits(s, c, of, k);
  if (c.rank == 0) {
    collect(sh, c);
    sort_list(sh, n);
    if (threadIdx.x == 0) {
      const u64 last = k - before <= n ? sh.list[k - before - 1] : 0;
      sh.cut = last ? Prefix{list_z(last), list_id(last)} : of;
    }
  }
  c.sync();
  return lead->cut;
}

// ------------------------------------------------------------------------------------------------ kernels

template <class T, bool ADJUSTED>
__global__ void __launch_bounds__(ROW_THREADS)
sample_kernel(const __grid_constant__ SampleRows a, int slice) {
  extern __shared__ __align__(16) float z[];
  __shared__ RowShared sh;
  Cluster c(&sh.mail);
  const int t = threadIdx.x, r = blockIdx.x / c.size, b = min(c.rank * slice, a.V), e = min(b + slice, a.V);
  const T* x = static_cast<const T*>(a.x) + r * a.ldx;
  Best top{-INFINITY, NO_ID};
  Slice s;
  if constexpr (ADJUSTED) {
    const RowAdjust adj(a.a, r, a.status);
    s = load_slice<T, true>(z, x, b, e, &adj, reinterpret_cast<int*>(sh.list), top);
  } else {
    s = load_slice<T, false>(z, x, b, e, nullptr, nullptr, top);
  }
  clear_bins(sh);
  if (t == 0) sh.n_list = 0;
  const float temp = a.temps[r];
  float p = a.top_p ? a.top_p[r] : 1.f;
  const float mp = a.min_p ? a.min_p[r] : 0.f;
  int k = a.top_k ? a.top_k[r] : 0;
  if (k >= a.V) k = 0;
  top = c.reduce(top, Best{-INFINITY, NO_ID}, first_of);
  const bool lead = c.rank == 0 && t == 0;
  // Greedy too: a best score that is not finite, beside which noise is nothing.
  if (top.v == -INFINITY || !(temp > 0.f) || !isfinite(__fdiv_rn(top.v, temp)) || k == 1 || p <= 0.f || mp > 1.f) {
    if (lead) a.out[r] = top.v == -INFINITY ? -1 : top.id;
    c.sync();                                      // (a CTA's mailbox stays until all have read it)
    return;
  }
  const Weights weight{top.v, fmaxf(fminf(__fdiv_rn(1.4426950408889634f, temp), -LOWEST), 1e-44f)};       // (products of it with 0 and infinity are 0 and infinity)
  const Race race(temp, weight.c, top.v, a.seeds[r], a.positions[r]);
  Prefix kept{LOWEST, NO_ID};
  if (mp > 0.f && isfinite(temp)) {                // the smallest logit that is not too improbable, decided in 64 bits
    if (t == 0) {
      const double top64 = top.v, T64 = temp, least = log(static_cast<double>(mp));
      const auto scaled = [&](float v) { return (static_cast<double>(v) - top64) / T64; };
      float v = fminf(static_cast<float>(top64 + T64 * least), top.v);
      for (int i = 0; i < 8 && scaled(v) >= least; ++i) v = nextafterf(v, -INFINITY);
      for (int i = 0; i < 16 && scaled(v) < least; ++i) v = nextafterf(v, INFINITY);
      sh.z = v;
    }
    __syncthreads();
    kept.z = fmaxf(kept.z, sh.z);
  }
  if (k > 0 || p < 1.f) {
    double all = 0;
    unsigned n = LIST + 1;
    if (k <= LIST) {
      // weight of the row, and the best of every eight in bins
      const bool by_count = k > 0;
      double sum = 0;
      const int lane = t & 31;
      for (int i = t >> 5; i < s.blocks; i += ROW_WARPS) {
        const float4 u = *reinterpret_cast<const float4*>(z + i * ROW_BLOCK + lane * 4), v = *reinterpret_cast<const float4*>(z + i * ROW_BLOCK + 128 + lane * 4);
        if (!by_count) {
          const auto w = [&](float y) { return y >= kept.z ? weight(y) : 0.f; };
          sum += (w(u.x) + w(u.y)) + (w(u.z) + w(u.w));
          sum += (w(v.x) + w(v.y)) + (w(v.z) + w(v.w));
        }
        const float m = fmaxf(max4(u), max4(v));
        if (m >= kept.z) {
          const int bin = weight.bin(m);
          if (by_count) atomicAdd(&sh.count[bin], 1u);
          else atomicAdd(&sh.mass[bin], static_cast<unsigned>(fminf(exp2_fast(weight.bits(m) + bin * (1.f / BINS_PER_BIT)) * 65536.f, 65536.f)));
        }
      }
      all = row_total(c, sum);
      if (c.rank == 0) find_bin(sh, c, by_count, k, p * all * 65536.0 * (1 + 1.0 / 262144));
      c.sync();
      const int bin = c.size > 1 ? *c.of(&sh.bin, 0) : sh.bin;
      float least = kept.z;                        // (a little below the bin's edge)
      if (bin < BINS - 1) {
        const float d = (bin + 1) / (BINS_PER_BIT * weight.c) * (1 + 1.f / 1048576);
        least = fmaxf(least, top.v - d - fabsf(top.v) * (1.f / 4194304));
      }
      n = gather(sh, s, c, least, [](float, int) { return true; });
    }
    if (n <= LIST) {
      if (c.rank == 0) collect(sh, c);
      c.sync();
      if (c.rank) return;
      sort_list(sh, n);
      // weights in the row's order, in whole numbers of 2^-40: every token before the one that reaches top_p is kept
      constexpr int PER = LIST / ROW_THREADS;
      u64 w[PER], sum = 0;
#pragma unroll
      for (int i = 0; i < PER; ++i) {
        const unsigned at = t * PER + i;
        w[i] = at < n && p < 1.f ? __float2ull_rn(weight(list_z(sh.list[at])) * 1099511627776.f) : 0;
        sum += w[i];
      }
      const unsigned n1 = k > 0 ? min(n, static_cast<unsigned>(k)) : n;
      unsigned m = n1;
      if (p < 1.f) {
        u64 incl = sum;
        const int lane = t & 31;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const u64 y = __shfl_up_sync(0xffffffffu, incl, o);
          if (lane >= o) incl += y;
        }
        if (lane == 31) sh.warp[t >> 5] = incl;
        if (t == 0) sh.kept = 0;
        __syncthreads();
        u64 before = incl - sum;
        for (int i = 0; i < t >> 5; ++i) before += sh.warp[i];
        u64 at = before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          at += w[i];
          if (t * PER + i + 1 == n1) sh.total = at;
        }
        __syncthreads();
        const double target = static_cast<double>(p) * (k > 0 ? static_cast<double>(sh.total) : all * 1099511627776.0);
        unsigned mine = 0;
        at = before;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
          const unsigned j = t * PER + i;
          mine += j < n1 && (j == 0 || static_cast<double>(at) < target);
          at += w[i];
        }
        if (mine) atomicAdd(&sh.kept, mine);
        __syncthreads();
        m = sh.kept;
        __syncthreads();
      }
      const int token = draw_list(sh, c, race, m);
      if (t == 0) a.out[r] = token;
      return;
    }
    if (k > 0) {
      kept = kth_token(sh, s, c, weight, kept, k);
      if (p < 1.f) all = row_mass(s, c, weight, [&](float v, int id) { return within(kept, v, id); });
    }
    const double target = p < 1.f ? p * all : 0;
    int token;
    for (;;) {
      token = draw_row(s, c, race, kept, top);
      if (p >= 1.f || token == top.id) break;
      __syncthreads();
      if (t == 0 && token >= b && token < e) sh.z = z[token - s.first];
      c.sync();
      const int owner = token / slice;
      const float v = c.size > 1 ? *c.of(&sh.z, owner) : sh.z;
      const Prefix front{v, token - 1};
      if (row_mass(s, c, weight, [&](float y, int id) { return within(front, y, id); }) < target) break;
      kept = front;
    }
    if (lead) a.out[r] = token;
    c.sync();
    return;
  }
  const int token = draw_row(s, c, race, kept, top);
  if (lead) a.out[r] = token;
  c.sync();
}

template <class T>
__global__ void __launch_bounds__(ROW_THREADS)
logprob_kernel(const __grid_constant__ LogprobRows a, int slice) {
  extern __shared__ __align__(16) float z[];
  __shared__ RowShared sh;
  Cluster c(&sh.mail);
  const int tid = threadIdx.x, r = blockIdx.x / c.size, b = min(c.rank * slice, a.V), e = min(b + slice, a.V);
  const T* x = static_cast<const T*>(a.x) + r * a.ldx;
  const int t = a.tokens[r];
  const bool there = t >= 0 && t < a.V;
  const float zt = there ? plain_logit(logit(x + t)) : -INFINITY;
  Best top{-INFINITY, NO_ID};
  const Slice s = load_slice<T, false>(z, x, b, e, nullptr, nullptr, top);
  clear_bins(sh);
  if (tid == 0) sh.n_list = 0;
  top = c.reduce(top, Best{-INFINITY, NO_ID}, first_of);
  const bool listed = a.top > 1 && top.v > -INFINITY && top.v < INFINITY;
  const Weights weight{top.v, 1.4426950408889634f};
  const auto below = [&](float v) { return v == top.v ? 0.f : v - top.v; };       // (infinite logits: a limit)
  struct Sums { double w; u64 before; };
  Sums m{0, 0};
  unsigned before = 0;
  const int lane = tid & 31;
  const float c2 = 1.4426950408889634f;
  for (int i = tid >> 5; i < s.blocks; i += ROW_WARPS) {
    const int j = i * ROW_BLOCK + lane * 4;
    const float4 u = *reinterpret_cast<const float4*>(z + j), v = *reinterpret_cast<const float4*>(z + j + 128);
    const float y[8] = {u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w};
    float w[8];
#pragma unroll
    for (int q = 0; q < 8; ++q) {
      const int id = s.first + j + (q & 3) + (q >> 2) * 128;
      w[q] = exp2_fast(below(y[q]) * c2);
      before += y[q] > zt || (y[q] == zt && id < t && id >= b && id < e);
    }
    m.w += (w[0] + w[1]) + (w[2] + w[3]);
    m.w += (w[4] + w[5]) + (w[6] + w[7]);
    if (listed) {
      const float g = fmaxf(max4(u), max4(v));
      if (g > -INFINITY) atomicAdd(&sh.count[weight.bin(g)], 1u);
    }
  }
  m.before = before;
  m = c.reduce(m, Sums{0, 0}, [](Sums p, Sums q) { return Sums{p.w + q.w, p.before + q.before}; });
  const double lse = log(m.w);
  const bool lead = c.rank == 0 && tid == 0;
  const auto lp = [&](float v) { return v == -INFINITY ? -INFINITY : static_cast<float>(static_cast<double>(below(v)) - lse); };
  int* ids = a.ids + static_cast<long long>(r) * a.top;
  float* lps = a.logprobs + static_cast<long long>(r) * a.top;
  if (lead) {
    a.logprob[r] = lp(zt);
    a.rank[r] = there ? static_cast<int>(m.before) + 1 : 0;
    if (a.top == 1) {
      ids[0] = top.v == -INFINITY ? -1 : top.id;
      lps[0] = lp(top.v);
    }
  }
  if (a.top < 2) { c.sync(); return; }
  if (listed) {
    if (c.rank == 0) find_bin(sh, c, true, a.top, 0);
    c.sync();
    const int bin = c.size > 1 ? *c.of(&sh.bin, 0) : sh.bin;
    float least = LOWEST;
    if (bin < BINS - 1) least = top.v - (bin + 1) / (BINS_PER_BIT * weight.c) * (1 + 1.f / 1048576) - fabsf(top.v) * (1.f / 4194304);
    const unsigned n = gather(sh, s, c, least, [](float, int) { return true; });
    if (n <= LIST) {
      if (c.rank == 0) collect(sh, c);
      c.sync();
      if (c.rank) return;
      sort_list(sh, n);
      for (unsigned i = tid; i < static_cast<unsigned>(a.top); i += ROW_THREADS) {
        const float v = i < n ? list_z(sh.list[i]) : -INFINITY;
        ids[i] = i < n ? list_id(sh.list[i]) : -1;
        lps[i] = lp(v);
      }
      return;
    }
  }
  Best last{INFINITY, -1};                         // one after the other: rows of nothing, of infinities, of very many equal logits
  for (int i = 0; i < a.top; ++i) {
    Best g{-INFINITY, NO_ID};
    s.each([&](float v, int id) { if (v < last.v || (v == last.v && id > last.id)) g = first_of(g, Best{v, id}); });
    last = c.reduce(g, Best{-INFINITY, NO_ID}, first_of);
    if (lead) {
      ids[i] = last.v == -INFINITY ? -1 : last.id;
      lps[i] = lp(last.v);
    }
  }
  c.sync();
}

// CTAs of a row's cluster: enough to hold it, more where there are few rows.
static int row_cluster(int R, int V, int sms) {
  int c = 1;
  while (c < 16 && (static_cast<long long>(c) * 20480 < V || (static_cast<long long>(R) * c * 2 <= sms && V / c > 4096))) c *= 2;
  return c;
}

template <class A, class K>
static int launch_rows(const char* name, K kern, const A& a, cudaStream_t s) {
  const int c = row_cluster(a.R, a.V, a.sms), slice = ((a.V + c - 1) / c + ROW_BLOCK - 1) / ROW_BLOCK * ROW_BLOCK, bytes = (slice + ROW_PAD) * 4;
  if (slice > ROW_SLICE_MAX) return -5;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
      cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return spark_launch_rc(name);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.R * c); cfg.blockDim = dim3(ROW_THREADS); cfg.dynamicSmemBytes = bytes; cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, a, slice) != cudaSuccess) return spark_launch_rc(name);
  return spark_launch_rc(name);
}

template <bool ADJUSTED>
static int sample_rows(const SampleRows& a, cudaStream_t s) {
  if (a.type == LT_F32) return launch_rows("spark_sample_rows", sample_kernel<float, ADJUSTED>, a, s);
  if (a.type == LT_BF16) return launch_rows("spark_sample_rows", sample_kernel<__nv_bfloat16, ADJUSTED>, a, s);
  return launch_rows("spark_sample_rows", sample_kernel<__half, ADJUSTED>, a, s);
}

}  // namespace spark

using namespace spark;

extern "C" int spark_sample_rows(const SampleRows* a, int adjusted, cudaStream_t s) {
  if (a->R <= 0 || a->V <= 0) return 0;
  return adjusted ? sample_rows<true>(*a, s) : sample_rows<false>(*a, s);
}

extern "C" int spark_logprob_rows(const LogprobRows* a, cudaStream_t s) {
  if (a->R <= 0 || a->V <= 0) return 0;
  if (a->type == LT_F32) return launch_rows("spark_logprob_rows", logprob_kernel<float>, *a, s);
  if (a->type == LT_BF16) return launch_rows("spark_logprob_rows", logprob_kernel<__nv_bfloat16>, *a, s);
  return launch_rows("spark_logprob_rows", logprob_kernel<__half>, *a, s);
}
