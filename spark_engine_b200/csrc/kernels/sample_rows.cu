// Tokens and log-probabilities from rows of logits.
//
// A row's tokens are ordered by (logit descending, id ascending); NaN and -inf are no tokens.  With w_v = e^{(z_v - max) / T}:
//
//   sample     kept are the first k tokens; of them those with (z - max) / T >= log(min_p); of those the shortest prefix whose weight is >= top_p of theirs.
//              The token is the arg-max over kept of fl(fl(z / T) + fl(g)), g = -log(-log u(seed, position, id)).
//   logprobs   z_t - log sum e^z, the rank of t, the first tokens of the order
//
// What is kept is always a prefix of the order, given by its last token.
//
// A row is read once, by one CTA or, where there are few rows, by a cluster's; what stays of it in shared memory is the largest of every eight logits
// (76 KB of 152k logits, where the row itself is 608).  The largest that each thread has seen go to a histogram, whose first bins with k tokens (or top_p of
// the weight) in them hold what is kept, since all others can only add to it; where they do not reach that far, the largest of every eight do.  The
// groups that come into these bins are read again, and what of them lies there goes to a list, in which one CTA finds the prefix.  Where more are kept than
// the list takes, the row is read again: the k-th token comes from a histogram of all (what is kept then fits the
// CTAs' lists together), and for top_p a token is drawn first and the weight in front of it looked at then: what lies in front of a token drawn in vain
// holds all that is kept, and half as much as before on average.
//
// Sums of weights that decide what is kept are whole numbers of 2^-40, which no order changes: a row draws the same whatever CTAs it has and wherever in
// memory it begins.  The weight of a row that top_p alone filters is streamed: a chunk's in fp32 in units 2^E of its own, E whole, chunks' in 64 bits.
// Where the weight in front of the token drawn is within 2^-18 of top_p of that sum, the row is drawn again by a sum in whole numbers.  Log-probabilities go by the streamed sum:
// they are the same however chunks are dealt to CTAs (to 2^-53); rows that begin elsewhere between two 16-byte boundaries have other chunks, and may have
// another last bit.
//
// What bounds it (one B200, fp32 logits).  One row: ten trips to memory and barriers of a cluster one after the other, 12.7 us for 152k logits, of which
// 2.5 are the row's own, 1.4 sums and best over eight CTAs, 1.4 bins, 4 the groups read again and lists joined, 2 the prefix and the draw.  Many rows whose
// distributions have few likely tokens: memory latency of what is read again, 62 us for 256 rows (24 at the copy rate).  Rows without filters: issue slots,
// 40 instructions per logit and lane, two thirds of them the hash: 79 us for 256.  Rows that keep most of 152k tokens: one such race and one look at
// the weights, 229 us for 256 of them.  Scored rows: 1024 of 152k in 100 us, 6.2 TB/s.
#include "../common/token_rows.cuh"

namespace spark {

constexpr int CHUNK = 1024;                        // logits that a warp takes at once, 32 per lane
constexpr int BINS = 1024;                         // of a sixteenth of a bit of weight; what weighs less than 2^-64 shares the last one
constexpr float BINS_PER_BIT = 16.f;
constexpr int LIST = 2048;
constexpr int HITS = 512;
template <int NT> constexpr int FEW_OF = NT < 256 ? NT : 256;       // of the list: ordered by counting
constexpr int CLUSTER_MAX = 8;

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
__device__ __forceinline__ float warp_highest(float v) {
  const int b = __float_as_int(v);
  const int m = __reduce_max_sync(0xffffffffu, b ^ (b >> 31 & 0x7fffffff));
  return __int_as_float(m ^ (m >> 31 & 0x7fffffff));
}
__device__ __forceinline__ double warp_total(double v) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ double pow2(float n) {  // 2^n for a whole n <= 0
  return n < -1022.f ? 0.0 : __hiloint2double((1023 + static_cast<int>(n)) << 20, 0);
}

// A prefix of the order: its last token.
struct Prefix { float z; int id; };
__device__ __forceinline__ bool within(const Prefix& p, float z, int id) { return z > p.z || (z == p.z && id <= p.id); }
constexpr float LOWEST = -3.402823466e38f;
__device__ __forceinline__ Prefix whole_row() { return Prefix{LOWEST, NO_ID}; }
__device__ __forceinline__ float at_least(float z) { return fmaxf(z, LOWEST); }

template <int NT>
struct RowShared {
  Mailboxes mail;
  unsigned hist[BINS], hits[HITS];
  u64 list[LIST], weight[FEW_OF<NT>];
  float fsum[NT / 32];
  unsigned n_list, n_hits, before, kept;
  int bin, score;
  float z;
  double log;
  Prefix cut;
  u64 total, unsure;
};

// ------------------------------------------------------------------------------------------------ a CTA's part of a row

template <class T> __device__ __forceinline__ T no_logit();
template <> __device__ __forceinline__ float no_logit<float>() { return -INFINITY; }
template <> __device__ __forceinline__ __nv_bfloat16 no_logit<__nv_bfloat16>() { return __ushort_as_bfloat16(0xff80); }
template <> __device__ __forceinline__ __half no_logit<__half>() { return __ushort_as_half(0xfc00); }

// 16 bytes at the row's ends: -inf where they are not the row's.
template <class T>
__device__ __noinline__ uint4 edge_vector(const T* base, int j, int lo, int hi) {
  alignas(16) T v[LOGITS_16B<T>];
  for (int e = 0; e < LOGITS_16B<T>; ++e) v[e] = j + e >= lo && j + e < hi ? base[j + e] : no_logit<T>();
  return *reinterpret_cast<const uint4*>(v);
}

// Places j of a row from a 16-byte boundary on: id j - lo; those in [lo, hi) are the row's.  Lane l of a warp has N = 16 bytes' logits of every
// 32 * N: value i of its 32 in chunk k is place k * CHUNK + (i / N) * 32 N + l * N + i % N.
template <class T, int NT>
struct Row {
  static constexpr int N = LOGITS_16B<T>, WARPS = NT / 32;
  const T* base;
  int lo, hi, chunk0, chunks;                      // this CTA's chunks

  __device__ __forceinline__ Row(const T* x, int V, int rank, int per) {
    lo = static_cast<int>(reinterpret_cast<uintptr_t>(x) / sizeof(T) % N);
    hi = lo + V;
    base = x - lo;
    chunk0 = rank * per;
    chunks = max(0, min(per, (hi + CHUNK - 1) / CHUNK - chunk0));
  }
  __device__ __forceinline__ int id(int j) const { return j - lo; }
  __device__ __forceinline__ float one(int j) const { return j >= lo && j < hi ? plain_logit(logit(base + j)) : -INFINITY; }
  static __device__ __forceinline__ int place(int chunk, int i, int lane) { return chunk * CHUNK + (i / N) * (32 * N) + lane * N + i % N; }

  // A lane's values from value `from` on, M of them.
  template <int M>
  __device__ __forceinline__ void load(int chunk, int from, int lane, float (&v)[M]) const {
    const int j0 = place(chunk, from, lane);
    uint4 q[M / N];
    if (chunk * CHUNK >= lo && chunk * CHUNK + CHUNK <= hi) {
#pragma unroll
      for (int i = 0; i < M / N; ++i) q[i] = __ldg(reinterpret_cast<const uint4*>(base + j0 + i * 32 * N));
    } else {
#pragma unroll
      for (int i = 0; i < M / N; ++i) {
        const int j = j0 + i * 32 * N;
        if (j >= lo && j + N <= hi) q[i] = __ldg(reinterpret_cast<const uint4*>(base + j));
        else q[i] = edge_vector(base, j, lo, hi);
      }
    }
#pragma unroll
    for (int i = 0; i < M / N; ++i) {
      float f[N];
      unpack_logits<T>(q[i], f);
#pragma unroll
      for (int e = 0; e < N; ++e) v[i * N + e] = plain_logit(f[e]);
    }
  }
  // f(32 logits, chunk's number in the CTA) for each of a warp's chunks; what it reads AHEAD chunks later is asked for (0: nothing).
  template <int AHEAD, class F>
  __device__ __forceinline__ void stream(F f) const {
    for (int k = threadIdx.x >> 5; k < chunks; k += WARPS) {
      float v[32];
      const int j = (chunk0 + k + AHEAD * WARPS) * CHUNK + (threadIdx.x & 31) * 32;          // (a lane: 128 bytes of fp32)
      if (AHEAD && k + AHEAD * WARPS < chunks && j < hi) asm volatile("prefetch.global.L2 [%0];" ::"l"(base + j));
      load(chunk0 + k, 0, threadIdx.x & 31, v);
      f(v, k);
    }
  }
  // f(8 logits, chunk's number, value of the first) for each of a warp's chunks that is `wanted`.
  template <class W, class F>
  __device__ __forceinline__ void again(W wanted, F f) const {
    for (int k = threadIdx.x >> 5; k < chunks; k += WARPS) {
      if (!wanted(k)) continue;
      float v[32];
      load(chunk0 + k, 0, threadIdx.x & 31, v);
#pragma unroll
      for (int q = 0; q < 32; q += 8) f(v + q, k, q);
    }
  }
  // The same in less code, for what hardly ever happens: it waits for memory four times a chunk.
  template <class W, class F>
  __device__ __forceinline__ void eights(W wanted, F f) const {
    for (int k = threadIdx.x >> 5; k < chunks; k += WARPS) {
      if (!wanted(k)) continue;
#pragma unroll 1
      for (int q = 0; q < 32; q += 8) {
        float v[8];
        load(chunk0 + k, q, threadIdx.x & 31, v);
        f(v, k, q);
      }
    }
  }
};

// The largest logits of groups of 1 << lg values of a lane (8 to 32); group (k, q, lane) at (k * (32 >> lg) + q) * 32 + lane.
struct Groups {
  float* g;
  int lg;
  __device__ __forceinline__ void put(const float (&m)[4], int k) const {
    const int lane = threadIdx.x & 31;
    if (lg == 3) {
#pragma unroll
      for (int q = 0; q < 4; ++q) g[(k * 4 + q) * 32 + lane] = m[q];
    } else if (lg == 4) {
      g[k * 64 + lane] = fmaxf(m[0], m[1]);
      g[k * 64 + 32 + lane] = fmaxf(m[2], m[3]);
    } else {
      g[k * 32 + lane] = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
    }
  }
  __device__ __forceinline__ int number(int chunks) const { return chunks * CHUNK >> lg; }
  // Whether the chunk has a logit of `least` or more.
  __device__ __forceinline__ bool reaches(int k, float least) const {
    const int lane = threadIdx.x & 31;
    float m = -INFINITY;
    for (int q = 0; q < 32 >> lg; ++q) m = fmaxf(m, g[(k * (32 >> lg) + q) * 32 + lane]);
    return __any_sync(0xffffffffu, m >= least);
  }
};

// Behind a CTA's groups: of a cluster, the largest logits of all its threads, and the leader's inbox.
template <int NT>
struct Parts {
  Groups groups;
  float* maxima;
  u64* inbox;
  // (Two CTAs of an SM have to fit: 300 rows of 170k logits with top_k 40 76 us, by groups of eight 93; of 400k 132, by groups of sixteen 147.)
  static constexpr __host__ __device__ __forceinline__ int lg_of(int per) { return per <= 160 ? 3 : per <= 320 ? 4 : 5; }
  static constexpr __host__ int bytes(int per, int size) { return (per * CHUNK >> lg_of(per)) * 4 + (size > 1 ? size * NT * 4 + LIST * 8 : 0); }
  __device__ __forceinline__ Parts(float* smem, int per, int size) {
    groups = Groups{smem, lg_of(per)};
    maxima = smem + (per * CHUNK >> groups.lg);
    inbox = reinterpret_cast<u64*>(maxima + size * NT);
  }
};

// What the longest row needs: shared memory of the CTA that has it alone, or of those that share one of the widest clusters; bins whose sums of weights, 2^16
// a group at most, and numbers, which become fp32, do not leave 32 and 24 bits; ids that kth_by_bits looks for by 21 of them.
constexpr int MAX_CHUNKS = (SAMPLE_MAX_V + 8 + CHUNK - 1) / CHUNK, MAX_SMEM = 227 * 1024;
static_assert(Parts<512>::bytes(MAX_CHUNKS, 1) + sizeof(RowShared<512>) <= MAX_SMEM && Parts<512>::bytes(320, CLUSTER_MAX) + sizeof(RowShared<512>) <= MAX_SMEM, "shared memory");
static_assert((MAX_CHUNKS * CHUNK >> Parts<512>::lg_of(MAX_CHUNKS)) < 65536 && (320 * CHUNK >> Parts<512>::lg_of(320)) < 65536 && SAMPLE_MAX_V < 1 << 24, "bins");
static_assert(SAMPLE_MAX_V <= 1 << 21, "ids");

__device__ __forceinline__ float max8(const float* v) {
  float m = v[0];
#pragma unroll
  for (int e = 1; e < 8; ++e) m = fmaxf(m, v[e]);
  return m;
}

// What a thread has seen of the row: the best token and the units (its warp's), its own share of the sums of 2^(z c - E), E whole: a change of units changes
// no bit, and in which batch a row is makes no difference.  s: of all logits, g: of the largest of every eight; n: a number.
struct Seen {
  Best top{-INFINITY, NO_ID};
  float E = LOWEST;
  unsigned n = 0;
  double s = 0, g = 0;
  __device__ __forceinline__ void add(double a, double b, float units) {
    if (units > E) {
      const double f = s ? pow2(E - units) : 0;    // (warps alike)
      s *= f;
      g *= f;
      E = units;
    }
    const double f = pow2(units - E);
    s += a * f;
    g += b * f;
  }
};
// The largest of a lane's eights, of the lane, of the chunk; the warp's best token kept: chunks come in the order of their ids, so that only larger logits
// replace it.
template <class R>
__device__ __forceinline__ float look(const R& row, const float (&v)[32], int k, float (&m)[4], float& mine, Best& best) {
#pragma unroll
  for (int q = 0; q < 4; ++q) m[q] = max8(v + 8 * q);
  mine = fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
  const float highest = warp_highest(mine);
  if (highest > best.v) {
    int j = NO_ID;
    if (mine == highest) {
#pragma unroll
      for (int i = 31; i >= 0; --i)
        if (v[i] == highest) j = R::place(row.chunk0 + k, i, threadIdx.x & 31);
    }
    best = Best{highest, row.id(__reduce_min_sync(0xffffffffu, j))};
  }
  return highest;
}
// Of the whole row.
__device__ __forceinline__ Seen row_seen(Cluster& c, Seen m, bool sums, bool numbers) {
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5, nw = blockDim.x >> 5;
  if (sums) { m.s = warp_total(m.s); m.g = warp_total(m.g); }
  if (numbers) m.n = __reduce_add_sync(0xffffffffu, m.n);
  if (lane == 0) *reinterpret_cast<Seen*>(&c.mine->warp[w]) = m;
  __syncthreads();
  const auto join = [&](const Mail* from, int n) {
    const Seen x = lane < n ? *reinterpret_cast<const Seen*>(from + lane) : Seen{};
    Seen y;
    y.top.v = warp_highest(x.top.v);
    y.top.id = __reduce_min_sync(0xffffffffu, x.top.v == y.top.v ? x.top.id : NO_ID);
    if (sums) {
      y.E = warp_highest(x.E);
      const double f = x.s ? pow2(x.E - y.E) : 0;
      y.s = x.s * f;
      y.g = x.g * f;
#pragma unroll
      for (int o = 8; o; o >>= 1) {                // (at most 16 of them)
        y.s += __shfl_xor_sync(0xffffffffu, y.s, o);
        y.g += __shfl_xor_sync(0xffffffffu, y.g, o);
      }
      y.s = __shfl_sync(0xffffffffu, y.s, 0);
      y.g = __shfl_sync(0xffffffffu, y.g, 0);
    }
    if (numbers) y.n = __reduce_add_sync(0xffffffffu, x.n);
    return y;
  };
  if (w == 0) m = join(c.mine->warp, nw);
  const Mail* b = c.tell(m);
  return join(b, c.size);
}

// ------------------------------------------------------------------------------------------------ histograms and lists

// Weights 2^((z - from) c - E).  `from` is 0, and the product exact and the difference rounded once, but for scores of 2^20 and more, in which that
// would leave too few bits of the difference: they are seen from the best.
struct Weights {
  float c, E, from;
  __device__ __forceinline__ float bits(float z) const { return fmaf(z - from, c, -E); }
  __device__ __forceinline__ float operator()(float z) const { return exp2_fast(bits(z)); }
  __device__ __forceinline__ int bin(float z) const { return max(0, min(static_cast<int>(bits(z) * -BINS_PER_BIT), BINS - 1)); }
  // A logit a little below the bin's edge.
  __device__ __forceinline__ float edge(int b) const {
    if (b >= BINS - 1) return LOWEST;
    const float y = E - (b + 1) * (1.f / BINS_PER_BIT), z = y / c;
    return at_least(from + z - (fabsf(z) + fabsf(from)) * (1.f / 1048576) - (fabsf(E) + (b + 1)) * (1.f / 4194304) / c);
  }
};

// Weights (less than 2) in whole numbers of 2^-40, rounded to nearest: sums of them are the same in every order, so that what is kept does not depend on how
// a row is dealt out.  Of w + 2 the last bit is 2^-22, and what it leaves of w is exact: both parts are read from the bits of a sum (a conversion to 64 bits
// would take the unit that exponentials wait for: 256 rows that keep most 233 us with it, 230 without, 228 with fp32 sums of eight; two by two in packed
// additions 232).
struct Whole {
  static constexpr uint32_t TWO = 0x40000000u, SMALL = 0x37400000u;    // 2 and 1.5 * 2^-17
  uint32_t hi = 0, lo = 0;                         // of 2^-22, and of 2^-40 (with a sign): up to 512 weights
  __device__ __forceinline__ void add(float w) {
    const float a = w + 2.f;
    hi += __float_as_uint(a) - TWO;
    lo += __float_as_uint(w - (a - 2.f) + __uint_as_float(SMALL)) - SMALL;
  }
  __device__ __forceinline__ u64 sum() const { return (static_cast<u64>(hi) << 18) + static_cast<u64>(static_cast<long long>(static_cast<int>(lo))); }
};
__device__ __forceinline__ u64 whole(float w) {
  Whole s;
  s.add(w);
  return s.sum();
}
__device__ __forceinline__ double weight_of(u64 n) { return static_cast<double>(n) * (1.0 / 1099511627776.0); }

template <int NT>
__device__ __forceinline__ void clear_bins(RowShared<NT>& sh) {
  for (int i = threadIdx.x; i < BINS; i += NT) sh.hist[i] = 0;
}
// A logit into its bin: as one, or as its weight in 2^-16 of the bin's highest (a little less at most).
template <int NT>
__device__ __forceinline__ void to_bin(RowShared<NT>& sh, const Weights& w, float z, bool by_count) {
  const int bin = w.bin(z);
  atomicAdd(&sh.hist[bin], by_count ? 1u : static_cast<unsigned>(fminf(exp2_fast(w.bits(z) + bin * (1.f / BINS_PER_BIT)) * 65536.f, 65536.f)));
}
// The first bin with which the bins (of the cluster's CTAs together, or this one's) hold `target`, tokens or weight: the last one where they do not.
// Into sh.bin, with the tokens in front of it in sh.before.  (fp32: numbers of tokens are exact, weights are asked for with some to spare.)
template <int NT>
__device__ __forceinline__ void find_bin(RowShared<NT>& sh, Cluster& c, bool together, bool by_count, float target) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  constexpr int PER = BINS / NT;
  float v[PER], sum = 0;
#pragma unroll
  for (int i = 0; i < PER; ++i) v[i] = 0;
  if (!together || c.size == 1) {
#pragma unroll
    for (int i = 0; i < PER; ++i) v[i] = sh.hist[PER * t + i];
  } else {
#pragma unroll
    for (int i = 0; i < PER; i += 2) {
      uint2 n[CLUSTER_MAX];
#pragma unroll
      for (int r = 0; r < CLUSTER_MAX; ++r)
        if (r < c.size) n[r] = *reinterpret_cast<const uint2*>(c.of(sh.hist, r) + PER * t + i);
#pragma unroll
      for (int r = 0; r < CLUSTER_MAX; ++r)
        if (r < c.size) { v[i] += n[r].x; v[i + 1] += n[r].y; }
    }
  }
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    if (!by_count) v[i] *= exp2_fast((PER * t + i) * (-1.f / BINS_PER_BIT)) * (1.f / 65536);
    sum += v[i];
  }
  float incl = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const float y = __shfl_up_sync(0xffffffffu, incl, o);
    if (lane >= o) incl += y;
  }
  if (lane == 31) sh.fsum[w] = incl;
  if (t == 0) { sh.bin = BINS - 1; sh.before = 0; }
  __syncthreads();
  float at = incl - sum;
  for (int i = 0; i < w; ++i) at += sh.fsum[i];
#pragma unroll
  for (int i = 0; i < PER; ++i) {                  // (rounding may find two: the first counts)
    if (at < target && at + v[i] >= target) { atomicMin(&sh.bin, PER * t + i); if (by_count) sh.before = static_cast<unsigned>(at); }
    at += v[i];
  }
  __syncthreads();
}

template <int NT>
__device__ __forceinline__ void to_list(RowShared<NT>& sh, float z, int id) {
  const unsigned at = atomicAdd(&sh.n_list, 1u);
  if (at < LIST) sh.list[at] = list_key(z, id);
}
// The CTAs' lists behind the leader's own; how many they hold together, which everyone gets and which may be more than a list takes (nothing is moved then).
// A CTA has a part of the leader's `inbox` to itself, so that entries and numbers travel together; only longer lists wait for the others' numbers.
template <int NT>
__device__ __forceinline__ unsigned join_lists(RowShared<NT>& sh, Cluster& c, u64* inbox) {
  __syncthreads();
  const unsigned mine = sh.n_list;
  if (c.size == 1) return mine;
  const unsigned part = LIST / c.size, t = threadIdx.x;
  if (c.rank && mine <= part) {
    u64* to = c.of(inbox, 0) + c.rank * part;
    for (unsigned i = t; i < mine; i += NT) to[i] = sh.list[i];
  }
  const Mail* box = c.tell(mine);
  unsigned n = 0, before = 0, most = 0;
  for (int r = 0; r < c.size; ++r) {
    const unsigned m = *reinterpret_cast<const unsigned*>(box + r);
    before += r < c.rank ? m : 0;
    most = max(most, r ? m : 0);
    n += m;
  }
  if (n > LIST) return n;
  if (most > part) {
    if (c.rank && mine > part) {
      u64* to = c.of(sh.list, 0) + before;
      for (unsigned i = t; i < mine; i += NT) to[i] = sh.list[i];
    }
    c.sync();
  }
  if (c.rank == 0) {
    unsigned at = mine;
    for (int r = 1; r < c.size; ++r) {
      const unsigned m = *reinterpret_cast<const unsigned*>(box + r);
      if (m <= part)
        for (unsigned i = t; i < m; i += NT) sh.list[at + i] = inbox[r * part + i];
      at += m;
    }
    __syncthreads();
  }
  return n;
}

// list[0, n) in the row's order (descending keys; all differ), for the tokens that log-probabilities list.  Bitonic: 2000 entries take 12 us, which is why
// few entries are counted and draws look for what they need in the list as it is.
template <int NT>
__device__ __noinline__ void sort_list(u64* list, unsigned n) {
  unsigned m = 32;
  while (m < n) m *= 2;
  for (unsigned i = n + threadIdx.x; i < m; i += NT) list[i] = 0;
  __syncthreads();
  for (unsigned k = 2; k <= m; k *= 2)
    for (unsigned j = k / 2; j; j /= 2) {
      for (unsigned p = threadIdx.x; p < m / 2; p += NT) {
        const unsigned a = 2 * p - (p & (j - 1)), b = a + j;
        const u64 x = list[a], y = list[b];
        if ((x < y) == ((a & k) == 0)) { list[a] = y; list[b] = x; }
      }
      __syncthreads();
    }
}

// The m-th largest of list[0, n), from 1: by the bits in which its keys differ, until one is left (2000 entries: 5 us).
template <int NT>
__device__ __forceinline__ u64 nth_key(RowShared<NT>& sh, unsigned n, unsigned m) {
  const int t = threadIdx.x, lane = t & 31, w = t >> 5;
  constexpr int WARPS = NT / 32;
  unsigned* part = sh.hits;                        // of each warp, two sets in turn
  const u64 one = sh.list[0];
  u64 d = 0;
  for (unsigned i = t; i < n; i += NT) d |= sh.list[i] ^ one;
  const auto joined = [&](unsigned x, int set, auto op) {
    if (lane == 0) part[set * WARPS + w] = x;
    __syncthreads();
    return op(lane < WARPS ? part[set * WARPS + lane] : 0u);
  };
  const auto any = [](unsigned x) { return __reduce_or_sync(0xffffffffu, x); };
  const auto sum = [](unsigned x) { return __reduce_add_sync(0xffffffffu, x); };
  const uint32_t lo = joined(any(static_cast<uint32_t>(d)), 0, any), hi = joined(any(static_cast<uint32_t>(d >> 32)), 1, any);
  u64 differ = static_cast<u64>(hi) << 32 | lo, key = one & ~differ, upper = 0;
  unsigned front = 0, left = n;                    // keys above those that begin like `key`, and those
  for (int set = 0; left > 1; set ^= 1) {
    const u64 bit = 1ull << (63 - __clzll(differ)), with = key | bit;
    differ ^= bit;
    upper = ~(bit - 1);
    unsigned c = 0;
#pragma unroll 4
    for (unsigned i = t; i < n; i += NT) c += (sh.list[i] & upper) == (with & upper);
    c = joined(sum(c), set, sum);
    if (front + c >= m) { key = with; left = c; }
    else { front += c; left -= c; }
  }
  for (unsigned i = t; i < n; i += NT)
    if ((sh.list[i] & upper) == (key & upper)) sh.total = sh.list[i];
  __syncthreads();
  return sh.total;
}

// Up to FEW entries: how many of the list are in front of an entry, and their weight.  Threads share an entry; the first of them has it.
struct Counted { u64 key, weight, before; unsigned rank; bool mine; };
template <int NT>
__device__ __forceinline__ Counted count_list(RowShared<NT>& sh, unsigned n, bool weights) {
  int per = 16;
  while (per * n > NT) per /= 2;
  const unsigned at = threadIdx.x / per, part = threadIdx.x % per;
  Counted e{0, 0, 0, 0, part == 0 && at < n};
  if (at < n) {
    e.key = sh.list[at];
    for (unsigned j = part; j < n; j += per) {
      const bool front = sh.list[j] > e.key;
      e.rank += front;
      if (weights && front) e.before += sh.weight[j];
    }
  }
  for (int o = per / 2; o; o /= 2) {
    e.rank += __shfl_xor_sync(0xffffffffu, e.rank, o);
    e.before += __shfl_xor_sync(0xffffffffu, e.before, o);
  }
  if (at < n && weights) e.weight = sh.weight[at];
  return e;
}

// The bins below which the row's first tokens lie, from the largest logit of every thread.
template <int NT>
__device__ __forceinline__ void bins_of_threads(RowShared<NT>& sh, Cluster& c, const float* maxima, float mine, const Weights& w, float least, bool by_count, float target) {
  for (int r = 0; r < c.size; ++r) {
    const float z = c.size > 1 ? maxima[r * NT + threadIdx.x] : mine;
    if (z >= least) to_bin(sh, w, z, by_count);
  }
  __syncthreads();
  find_bin(sh, c, false, by_count, target);
}
// The same from the groups' (the bins are of no use any more).
template <int NT>
__device__ __noinline__ void bins_of_groups(RowShared<NT>& sh, Cluster& c, const Groups groups, int chunks, const Weights w, float least, bool by_count, float target) {
  clear_bins(sh);
  __syncthreads();
  for (int i = threadIdx.x; i < groups.number(chunks); i += NT)
    if (groups.g[i] >= least) to_bin(sh, w, groups.g[i], by_count);
  c.sync();
  find_bin(sh, c, true, by_count, target);
}
// The same from all logits, of short rows: their few groups may hide much.
template <class T, int NT>
__device__ __noinline__ void bins_of_all(RowShared<NT>& sh, Cluster& c, const Row<T, NT> row, const Weights w, float least, bool by_count, float target) {
  c.sync();                                        // (nobody reads the bins any more)
  clear_bins(sh);
  __syncthreads();
  row.again([](int) { return true; }, [&](const float* v, int, int) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v[i] >= least) to_bin(sh, w, v[i], by_count);
  });
  c.sync();
  find_bin(sh, c, true, by_count, target);
}
// What lies at `least` and above, in the leader's list.  First which groups of eight have any, then a thread for each of them.
template <class T, int NT>
__device__ __forceinline__ unsigned gather(RowShared<NT>& sh, Cluster& c, const Row<T, NT>& row, const Parts<NT>& parts, float mine, float least) {
  const int lane = threadIdx.x & 31, lg = parts.groups.lg, per = 32 >> lg;
  const auto read = [&](int i) {                   // group i
    const int g = i >> 5, chunk = row.chunk0 + g / per, from = g % per << lg;
    for (int q = 0; q < 1 << lg; q += 8) {
      float v[8];
      row.load(chunk, from + q, i & 31, v);
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (v[e] >= least) to_list(sh, v[e], row.id(Row<T, NT>::place(chunk, from + q + e, i & 31)));
    }
  };
  if (__any_sync(0xffffffffu, mine >= least))
    for (int k = threadIdx.x >> 5; k < row.chunks; k += NT / 32)
      for (int q = 0; q < per; ++q) {
        const int i = (k * per + q) * 32 + lane;
        const bool hit = parts.groups.g[i] >= least;
        const unsigned who = __ballot_sync(0xffffffffu, hit);
        if (!who) continue;
        unsigned at = 0;
        if (lane == 0) at = atomicAdd(&sh.n_hits, __popc(who));
        at = __shfl_sync(0xffffffffu, at, 0) + __popc(who & ((1u << lane) - 1));
        if (hit && at < HITS) sh.hits[at] = i;
        else if (hit) read(i);
      }
  __syncthreads();
  for (unsigned h = threadIdx.x; h < min(sh.n_hits, static_cast<unsigned>(HITS)); h += NT) read(sh.hits[h]);
  return join_lists(sh, c, parts.inbox);
}

// Whether so few groups of the row reach `least` that the list takes all they may hold.
template <int NT>
__device__ __noinline__ bool few_reach(Cluster& c, const Groups groups, int chunks, float least) {
  unsigned n = 0;
  for (int i = threadIdx.x; i < groups.number(chunks); i += NT) n += groups.g[i] >= least;
  return (c.reduce(n, 0u, [](unsigned a, unsigned b) { return a + b; }) << groups.lg) <= LIST;
}

// ------------------------------------------------------------------------------------------------ draws

__device__ __forceinline__ u64 mix64(u64 x) {
  x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
  x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}

struct Top2 { float a1; int id; float a2, z; };                // the best score, its token, the second best score, the token's logit
__device__ __forceinline__ Top2 no_top() { return Top2{-INFINITY, NO_ID, -INFINITY, -INFINITY}; }
__device__ __forceinline__ Top2 best2(Top2 x, Top2 y) {
  return x.a1 >= y.a1 ? Top2{x.a1, x.id, fmaxf(x.a2, y.a1), x.z} : Top2{y.a1, y.id, fmaxf(y.a2, x.a1), y.z};
}
struct Win { float v; int id; float z; int none; };
__device__ __forceinline__ Win first_win(Win a, Win b) { return b.v > a.v || (b.v == a.v && b.id < a.id) ? b : a; }

// A token's score is known from below and above at the price of a few fp32 operations: `margin` is more than twice what the rough one may be off.
// Where the two best are further apart than that, the best is the best; else both are computed as the definition says.
struct Race {
  float temp, c;
  u64 key;
  static constexpr u64 STEP = 0x9E3779B97F4A7C15ull;
  __device__ __forceinline__ Race(float T, float c_, long long seed, long long pos)
      : temp(T), c(c_), key((static_cast<u64>(seed) * STEP) ^ (static_cast<u64>(pos + 1) * 0xBF58476D1CE4E5B9ull)) {}
  __device__ __forceinline__ u64 hash(int id) const { return mix64(static_cast<u64>(id) * STEP + key); }
  __device__ __forceinline__ float exact(float z, int id) const {
    const double u = (static_cast<double>(hash(id) >> 11) + 0.5) * (1.0 / 9007199254740992.0);
    return __fadd_rn(__fdiv_rn(z, temp), static_cast<float>(-log(-log(u))));
  }
  // -log u from q = 1 - u where u is near 1 (to q^3 of it), from u where it is near 0; each to 2^-13 of itself.
  __device__ __forceinline__ float rough(float z, int id) const {
    const u64 h = hash(id);
    const float q = (__ull2float_rn(~h >> 11) + 0.5f) * (1.f / 9007199254740992.f);
    const float L = q < 1.f / 256 ? q * (1.f + q * (0.5f + q * (1.f / 3))) : -__logf(q < 0.5f ? 1.f - q : (__ull2float_rn(h >> 11) + 0.5f) * (1.f / 9007199254740992.f));
    return __fdiv_rn(z, temp) - __logf(L);
  }
  // (noise lies between -3.7 and 37.5: what comes near a score is z / T from not much further than that)
  static __device__ __forceinline__ float margin(float score) { return 1.f / 512 + (fabsf(score) + 128.f) * (1.f / 524288); }
};

// Scores as whole numbers of the same order.
__device__ __forceinline__ int score_key(float v) { const int b = __float_as_int(v); return b ^ (b >> 31 & 0x7fffffff); }
__device__ __forceinline__ float key_score(int k) { return __int_as_float(k ^ (k >> 31 & 0x7fffffff)); }

// The values from place j0 on that `near` names: their scores among the best two.
template <class R>
__device__ __noinline__ Top2 look_at(const Race race, const R row, unsigned near, int j0, const Prefix kept, Top2 m) {
  while (near) {
    const int i = __ffs(near) - 1, j = j0 + i / R::N * (32 * R::N) + i % R::N;
    near &= near - 1;
    const float z = row.one(j);
    if (within(kept, z, row.id(j))) m = best2(m, Top2{race.rough(z, row.id(j)), row.id(j), -INFINITY, z});
  }
  return m;
}

// A warp's race over the logits that come by.  -log u >= 1 - u, so that a score is at most z / T - log(1 - u): most tokens are out of it by the 32
// upper bits of their hash, without a logarithm.  `shared`: the best score that any warp of the CTA knows of, which spares the others the look at tokens
// that do not come near it; who wins does not depend on when they see it.
struct Racer {
  Top2 m = no_top();
  float bound = -INFINITY, off = 0.f;              // the best score so far, and what it takes to come near it
  __device__ __forceinline__ void raise(float b) {
    bound = b;
    off = (Race::margin(b) - b) * 1.4426950408889634f + 32.f;
  }
  __device__ __forceinline__ void tell(int* shared) const {
    if ((threadIdx.x & 31) == 0) atomicMax(shared, score_key(bound));
  }
  __device__ __forceinline__ void hear(const int* shared) {
    const float b = key_score(*static_cast<const volatile int*>(shared));
    if (b > bound) raise(b);                       // (each lane for itself)
  }
  // The lanes' largest logits raise the bound before all others come; false where none of them is within `kept`, and no other then.
  template <int M, class R>
  __device__ __forceinline__ bool begin(const Race& race, const R& row, const float* v, float mine, int chunk, int from, const Prefix& kept, int* shared) {
    int j = 0;
#pragma unroll
    for (int i = M - 1; i >= 0; --i)
      if (v[i] == mine) j = R::place(chunk, from + i, threadIdx.x & 31);
    const float b = warp_highest(within(kept, mine, row.id(j)) ? race.rough(mine, row.id(j)) : -INFINITY);
    if (b == -INFINITY) return false;
    raise(b);
    tell(shared);
    return true;
  }
  // Eight values of the lane, from value `from` of the chunk on.  The hash's last step changes the lowest of its 32 upper bits at most: one is added to
  // what may come near instead.
  template <bool ALL, class R>
  __device__ __forceinline__ void run(const Race& race, const R& row, const float* v, int chunk, int from, const Prefix& kept, int* shared) {
    const int j0 = R::place(chunk, from, threadIdx.x & 31), id0 = row.id(j0);
    const u64 first = static_cast<u64>(static_cast<long long>(id0)) * Race::STEP + race.key;
    unsigned near = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      u64 x = first + static_cast<u64>(i / R::N * (32 * R::N) + i % R::N) * Race::STEP;
      x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
      x ^= x >> 27;
      const uint32_t lo = static_cast<uint32_t>(x), hi = static_cast<uint32_t>(x >> 32);
      const uint32_t rest = ~(__umulhi(lo, 0x133111EBu) + lo * 0x94D049BBu + hi * 0x133111EBu);
      const bool in = ALL || v[i] >= kept.z;
      if (static_cast<float>(rest) <= exp2_fast(fmaf(v[i], race.c, off)) + 1.f && in) near |= 1u << i;
    }
    bool more = false;
    if (near) {
      m = look_at(race, row, near, j0, kept, m);
      more = m.a1 > bound;
    }
    if (__any_sync(0xffffffffu, more)) {
      raise(fmaxf(bound, warp_highest(m.a1)));
      tell(shared);
    }
    hear(shared);
  }
};

// A race over what lies within `front`, and the weight of that.
struct Lap { Top2 m; u64 s; };
template <bool RACE, bool MASS, class T, int NT>
__device__ __noinline__ Lap lap(const Row<T, NT> row, const Groups groups, const Race race, const Weights w, const Prefix front, int* shared) {
  Racer racer;
  u64 s = 0;
  row.again([&](int k) { return groups.reaches(k, front.z); }, [&](const float* v, int k, int q) {
    const int chunk = row.chunk0 + k;
    const float mine = max8(v);
    if (__all_sync(0xffffffffu, !(mine >= front.z))) return;
    if (MASS) {
      bool last = false;
      Whole eight;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        eight.add(v[i] > front.z ? w(v[i]) : 0.f);
        last |= v[i] == front.z;
      }
      if (last) {                                  // as the last token of it: by their ids
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (v[i] == front.z && row.id(Row<T, NT>::place(chunk, q + i, threadIdx.x & 31)) <= front.id) eight.add(w(v[i]));
      }
      s += eight.sum();
    }
    if (RACE && (__any_sync(0xffffffffu, racer.bound > -INFINITY) || racer.template begin<8>(race, row, v, mine, chunk, q, front, shared)))
      racer.template run<false>(race, row, v, chunk, q, front, shared);
  });
  return Lap{racer.m, s};
}
template <class S>
__device__ __forceinline__ S row_total(Cluster& c, S s) {
  return c.reduce(s, S{0}, [](S a, S b) { return a + b; });
}
// The streamed sum of a row is off from that in whole numbers by less than this of itself: 2^-20 for ten fp32 additions in a row at most (half a step
// each), as much for the arguments of weights that count, seen from the chunk's best here and from the row's there.
constexpr double SUM_OFF = 1.0 / 262144;
__device__ __forceinline__ bool close_to(double in_front, double target) { return fabs(in_front - target) <= target * SUM_OFF; }

// The winner among the tokens within `kept`, from the two best of a race.
template <class T, int NT>
__device__ __noinline__ Win photo_finish(const Row<T, NT> row, Cluster& c, const Race race, const Prefix kept, float best) {
  Win b{-INFINITY, NO_ID, -INFINITY, 0};
  row.eights([](int) { return true; }, [&](const float (&)[8], int k, int q) {
#pragma unroll 1
    for (int i = 0; i < 8; ++i) {
      const int j = Row<T, NT>::place(row.chunk0 + k, q + i, threadIdx.x & 31), id = row.id(j);
      const float z = row.one(j);
      if (within(kept, z, id) && race.rough(z, id) >= best - Race::margin(best)) b = first_win(b, Win{race.exact(z, id), id, z, 0});
    }
  });
  return c.reduce(b, Win{-INFINITY, NO_ID, -INFINITY, 0}, first_win);
}
template <class T, int NT>
__device__ __forceinline__ Win settle(const Row<T, NT>& row, Cluster& c, const Race& race, const Prefix& kept, Top2 m) {
  m = c.reduce(m, no_top(), best2);
  if (m.a2 < m.a1 - Race::margin(m.a1)) return Win{m.a1, m.id, m.z, 0};
  return photo_finish(row, c, race, kept, m.a1);
}

// The leader's: the winner among what `each` gives (f(key) for the thread's candidates).  All of its threads have it.
template <int NT, class E>
__device__ __forceinline__ Prefix draw_listed(RowShared<NT>& sh, Cluster& c, const Race& race, E each) {
  Top2 m = no_top();
  each([&](u64 k) { m = best2(m, Top2{race.rough(list_z(k), list_id(k)), list_id(k), -INFINITY, list_z(k)}); });
  m = c.block(m, no_top(), best2);
  if (threadIdx.x == 0) {
    sh.kept = m.a2 < m.a1 - Race::margin(m.a1);
    sh.cut = Prefix{m.z, m.id};
  }
  __syncthreads();
  if (!sh.kept) {
    Win b{-INFINITY, NO_ID, -INFINITY, 0};
    each([&](u64 k) { b = first_win(b, Win{race.exact(list_z(k), list_id(k)), list_id(k), list_z(k), 0}); });
    b = c.block(b, Win{-INFINITY, NO_ID, -INFINITY, 0}, first_win);
    if (threadIdx.x == 0) sh.cut = Prefix{b.z, b.id};
    __syncthreads();
  }
  return sh.cut;
}

// ------------------------------------------------------------------------------------------------ the k-th token

template <class T, int NT, class F>
__device__ __forceinline__ u64 row_count(const Row<T, NT>& row, Cluster& c, F f) {
  u64 n = 0;
  row.eights([](int) { return true; }, [&](const float (&v)[8], int k, int q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) n += f(v[i], row.id(Row<T, NT>::place(row.chunk0 + k, q + i, threadIdx.x & 31))) ? 1 : 0;
  });
  return c.reduce(n, u64{0}, [](u64 a, u64 b) { return a + b; });
}

// By the bits of keys and ids, where more tokens than a list takes share the k-th one's bin: many equal logits, or a k-th one in the last bin, below 2^-64 of
// the first (top_k 40 at temperature 0.1, or beside a bias of 100).  Up to 55 readings of the row: 0.29 ms for 152k logits, 1.8 ms for 256 such rows.
template <class T, int NT>
__device__ __noinline__ Prefix kth_by_bits(const Row<T, NT> row, Cluster& c, const Prefix of, u64 k) {
  if (row_count(row, c, [&](float z, int id) { return within(of, z, id); }) <= k) return of;
  uint32_t key = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = key | 1u << bit;
    if (row_count(row, c, [&](float z, int id) { return order_key(z) >= t && within(of, z, id); }) >= k) key = t;
  }
  const float v = key_order(key);
  k -= row_count(row, c, [&](float z, int) { return z > v; });
  int id = 0;
  for (int bit = 20; bit >= 0; --bit) {            // the largest id with less than k of these in front of it
    const int t = id | 1 << bit;
    if (row_count(row, c, [&](float z, int i) { return z == v && i < t && within(of, z, i); }) < k) id = t;
  }
  return Prefix{v, id};
}

// The prefix of the first k tokens of `of` = (least logit, any id).
template <class T, int NT>
__device__ __noinline__ Prefix kth_token(RowShared<NT>& sh, const Row<T, NT> row, const Groups groups, Cluster& c, const Weights w, const Prefix of, unsigned k, u64* inbox) {
  c.sync();                                        // (nobody reads the bins and lists of before any more)
  // four sets of bins where the list will be, each for a fourth of the lanes: most tokens of a flat row fall into few bins
  unsigned* sets = reinterpret_cast<unsigned*>(sh.list);
  static_assert(4 * BINS * sizeof(unsigned) <= LIST * sizeof(u64), "sets of bins");
  for (int i = threadIdx.x; i < 4 * BINS; i += NT) sets[i] = 0;
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  unsigned* mine = sets + (threadIdx.x & 3) * BINS;
  row.again([&](int i) { return groups.reaches(i, of.z); }, [&](const float* v, int, int) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v[i] >= of.z) atomicAdd(&mine[w.bin(v[i])], 1u);
  });
  __syncthreads();
  for (int i = threadIdx.x; i < BINS; i += NT) sh.hist[i] = (sets[i] + sets[BINS + i]) + (sets[2 * BINS + i] + sets[3 * BINS + i]);
  c.sync();
  find_bin(sh, c, true, true, k);
  const int bin = sh.bin;
  const unsigned before = sh.before;               // (0 with the last bin where the row has fewer than k tokens)
  row.again([&](int i) { return groups.reaches(i, fmaxf(of.z, w.edge(bin))); }, [&](const float* v, int n, int q) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (v[i] >= of.z && w.bin(v[i]) == bin) to_list(sh, v[i], row.id(Row<T, NT>::place(row.chunk0 + n, q + i, threadIdx.x & 31)));
  });
  const unsigned n = join_lists(sh, c, inbox);
  if (n > LIST) return kth_by_bits(row, c, of, k);
  if (c.rank == 0) {
    const u64 last = k - before <= n ? nth_key(sh, n, k - before) : 0;
    const Prefix cut = last ? Prefix{list_z(last), list_id(last)} : of;
    if (threadIdx.x < c.size) c.of(&sh, threadIdx.x)->cut = cut;
  }
  c.sync();
  return sh.cut;
}

// What lies within `kept` in its CTA's own list; false (and of no use) where one of them is too short.
template <class T, int NT>
__device__ __noinline__ bool list_kept(RowShared<NT>& sh, Cluster& c, const Row<T, NT> row, const Groups groups, const Prefix kept) {
  if (threadIdx.x == 0) sh.n_list = 0;
  __syncthreads();
  row.again([&](int i) { return groups.reaches(i, kept.z); }, [&](const float* v, int n, int q) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int id = row.id(Row<T, NT>::place(row.chunk0 + n, q + i, threadIdx.x & 31));
      if (v[i] >= kept.z && within(kept, v[i], id)) to_list(sh, v[i], id);
    }
  });
  __syncthreads();
  return c.reduce(sh.n_list, 0u, [](unsigned a, unsigned b) { return max(a, b); }) <= LIST;
}
// A race over the list's entries within `front`, and their weight.
template <int NT>
__device__ __noinline__ Lap list_lap(const RowShared<NT>& sh, const Race race, const Weights w, const Prefix front, bool race_too, bool mass_too) {
  Top2 m = no_top();
  Whole s;
  const unsigned n = sh.n_list;
  for (unsigned i = threadIdx.x; i < n; i += NT) {
    const u64 key = sh.list[i];
    const float z = list_z(key);
    const int id = list_id(key);
    if (!within(front, z, id)) continue;
    if (mass_too) s.add(w(z));
    if (race_too) m = best2(m, Top2{race.rough(z, id), id, -INFINITY, z});
  }
  return Lap{m, s.sum()};
}

// Whether the row's sum is the streamed one.
__device__ __forceinline__ bool streamed(const SampleRows& a, int r, const Weights& w) {
  return !(a.top_k && a.top_k[r] > 0 && a.top_k[r] < a.V) && !(a.min_p && a.min_p[r] > 0.f && isfinite(a.temps[r])) && w.from == 0.f;
}
// Whether a listed token that is as near to the border as the streamed sum is off may be drawn: it may, and if it or one behind it is, the draw is made again.
template <int NT>
__device__ __noinline__ bool perhaps(RowShared<NT>& sh, const SampleRows& a, int r, const Weights w, u64 key, bool otherwise) {
  if (!streamed(a, r, w)) return otherwise;
  atomicMax(&sh.unsure, key);
  return true;
}
// A draw by top_p alone, of a row whose tokens begin with `first`: by a sum in whole numbers and the scores as they are defined, by one CTA that reads
// the row again and again (it is for what comes so near to the border that the streamed sum does not tell: 0.3 ms for 152k logits).  Other rows' sums are
// in whole numbers from the start: `otherwise`.
template <class T, int NT>
__device__ __noinline__ int draw_in_whole(RowShared<NT>& sh, Cluster& c, const SampleRows& a, int r, const Weights w, int first, int otherwise) {
  if (!streamed(a, r, w)) return otherwise;
  const Row<T, NT> row(static_cast<const T*>(a.x) + r * a.ldx, a.V, 0, a.V);
  const Race race(a.temps[r], w.c, a.seeds[r], a.positions[r]);
  const auto every = [&](auto f) {
    row.eights([](int) { return true; }, [&](const float (&v)[8], int k, int q) {
#pragma unroll 1
      for (int i = 0; i < 8; ++i) f(row.one(Row<T, NT>::place(k, q + i, threadIdx.x & 31)), row.id(Row<T, NT>::place(k, q + i, threadIdx.x & 31)));
    });
  };
  const auto mass = [&](const Prefix& front) {
    u64 s = 0;
    every([&](float z, int id) { s += within(front, z, id) ? whole(w(z)) : 0; });
    s = c.block(s, u64{0}, [](u64 x, u64 y) { return x + y; });
    if (threadIdx.x == 0) sh.total = s;
    __syncthreads();
    return weight_of(sh.total);
  };
  Prefix front = whole_row();
  const double target = a.top_p[r] * mass(front);
  for (;;) {
    Win b{-INFINITY, NO_ID, -INFINITY, 0};
    every([&](float z, int id) { if (within(front, z, id)) b = first_win(b, Win{race.exact(z, id), id, z, 0}); });
    b = c.block(b, Win{-INFINITY, NO_ID, -INFINITY, 0}, first_win);
    if (threadIdx.x == 0) sh.cut = Prefix{b.z, b.id};
    __syncthreads();
    const Prefix win = sh.cut;
    front = Prefix{win.z, win.id - 1};
    if (win.id == first || mass(front) < target) return win.id;
  }
}

// ------------------------------------------------------------------------------------------------ kernels

// The smallest logit that is not too improbable, decided in 64 bits.
__device__ __noinline__ float min_p_logit(float top, float temp, float mp) {
  const double top64 = top, T64 = temp, least = log(static_cast<double>(mp));
  const auto scaled = [&](float v) { return (static_cast<double>(v) - top64) / T64; };
  float v = fminf(static_cast<float>(top64 + T64 * least), top);
  for (int i = 0; i < 8 && scaled(v) >= least; ++i) v = nextafterf(v, -INFINITY);
  for (int i = 0; i < 16 && scaled(v) < least; ++i) v = nextafterf(v, INFINITY);
  return at_least(v);
}

template <class T, int NT>
__global__ void __launch_bounds__(NT, 1024 / NT)
sample_kernel(const __grid_constant__ SampleRows a, int per) {
  extern __shared__ __align__(16) float smem[];
  __shared__ RowShared<NT> sh;
  pdl_wait();
  pdl_trigger();
  Cluster c(&sh.mail);
  const int t = threadIdx.x, r = blockIdx.x / c.size;
  const float temp = a.temps[r], mp = a.min_p ? a.min_p[r] : 0.f, p = a.top_p ? a.top_p[r] : 1.f;
  const int asked = a.top_k ? a.top_k[r] : 0, k = asked < a.V ? asked : 0;
  const Row<T, NT> row(static_cast<const T*>(a.x) + r * a.ldx, a.V, c.rank, per);
  const Parts<NT> parts(smem, per, c.size);
  const Groups groups = parts.groups;
  const bool greedy = !(temp > 0.f) || k == 1 || p <= 0.f || mp > 1.f, by_p = p < 1.f, by_k = k > 0, by_min = mp > 0.f && isfinite(temp);
  const bool all = !greedy && !by_p && !by_k && !by_min, sums = !greedy && by_p && !by_k && !by_min;
  // (products of it with 0 and infinity are 0 and infinity)
  const float scale = greedy ? 0.f : fmaxf(fminf(__fdiv_rn(1.4426950408889634f, temp), -LOWEST), 1e-44f);
  const Race race(temp, scale, a.seeds[r], a.positions[r]);
  clear_bins(sh);
  if (t == 0) { sh.n_list = sh.n_hits = 0; sh.unsure = 0; sh.score = score_key(-INFINITY); }
  if (all) __syncthreads();

  Seen seen;
  Racer racer;
  float largest = -INFINITY;                       // of the thread
  if (all) {
    row.template stream<0>([&](const float (&v)[32], int i) {
      float m[4], mine;
      const float highest = look(row, v, i, m, mine, seen.top);
      if (!(highest > -INFINITY && highest < INFINITY)) return;
      if (racer.bound == -INFINITY) racer.template begin<32>(race, row, v, mine, row.chunk0 + i, 0, whole_row(), &sh.score);
#pragma unroll
      for (int q = 0; q < 32; q += 8) racer.template run<true>(race, row, v + q, row.chunk0 + i, q, whole_row(), &sh.score);
    });
  } else if (sums) {
    row.template stream<0>([&](const float (&v)[32], int i) {
      float m[4], mine;
      const float highest = look(row, v, i, m, mine, seen.top);
      largest = fmaxf(largest, mine);
      groups.put(m, i);
      if (!(highest > -INFINITY)) return;
      const float E = fmaxf(ceilf(highest * scale), -1e30f);     // the chunk's weight in units of its own
      float s = 0.f, g = 0.f;
#pragma unroll
      for (int q = 0; q < 32; q += 4)
        s += (exp2_fast(fmaf(v[q], scale, -E)) + exp2_fast(fmaf(v[q + 1], scale, -E))) + (exp2_fast(fmaf(v[q + 2], scale, -E)) + exp2_fast(fmaf(v[q + 3], scale, -E)));
#pragma unroll
      for (int q = 0; q < 4; ++q) g += exp2_fast(fmaf(m[q], scale, -E));
      seen.add(s, g, E);
    });
  } else {
    row.template stream<0>([&](const float (&v)[32], int i) {
      float m[4], mine;
      look(row, v, i, m, mine, seen.top);
      largest = fmaxf(largest, mine);
      if (!greedy) groups.put(m, i);
    });
  }
  c.ready();
  if (c.size > 1 && !greedy && !all)
    for (int i = 0; i < c.size; ++i) c.of(parts.maxima, i)[c.rank * NT + t] = largest;
  seen = row_seen(c, seen, sums, false);
  const Best top = seen.top;
  const bool lead = c.rank == 0 && t == 0;
  // Greedy too: a best score beside which noise is nothing.
  if (greedy || top.v == -INFINITY || !(fabsf(__fdiv_rn(top.v, temp)) < 1073741824.f)) {
    if (lead) a.out[r] = top.v == -INFINITY ? -1 : top.id;
    c.sync();                                      // (what a CTA's shared memory holds stays until all have read it)
    return;
  }
  if (all) {
    const Win win = settle(row, c, race, whole_row(), racer.m);
    if (lead) a.out[r] = win.id;
    c.sync();
    return;
  }
  const bool far = !(fabsf(top.v * scale) < 1048576.f);
  const Weights weight = far ? Weights{scale, 0.f, top.v} : Weights{scale, ceilf(top.v * scale), 0.f};
  Prefix kept = whole_row();
  if (by_min) {
    if (t == 0) sh.z = min_p_logit(top.v, temp, mp);
    __syncthreads();
    kept.z = sh.z;
  }
  double total = 0;
  if (sums && !far) total = seen.s * pow2(seen.E - weight.E);
  else if (by_p && !by_k) total = weight_of(row_total(c, lap<false, true>(row, groups, race, weight, kept, &sh.score).s));
  unsigned n = LIST + 1;
  if (k <= LIST && !far) {
    float least = kept.z;
    bool found = false;
    if (by_k || by_p) {
      const float need = by_k ? k : static_cast<float>(p * total * (1 + SUM_OFF));
      bins_of_threads(sh, c, parts.maxima, largest, weight, kept.z, by_k, need);
      // (the groups' largest may have the weight that the threads' have not, and they are more than these)
      if (sh.bin == BINS - 1 && (by_k || by_min || seen.g * pow2(seen.E - weight.E) >= need)) bins_of_groups(sh, c, groups, row.chunks, weight, kept.z, by_k, need);
      if (NT == 128 && sh.bin == BINS - 1) bins_of_all(sh, c, row, weight, kept.z, by_k, need);
      found = sh.bin < BINS - 1;
      if (found) least = fmaxf(least, weight.edge(sh.bin));
    }
    if (found || few_reach<NT>(c, groups, row.chunks, least)) n = gather(sh, c, row, parts, largest, least);
  }
  if (n <= LIST) {
    if (c.rank) return;
    const unsigned n1 = by_k ? min(n, static_cast<unsigned>(k)) : n;
    int token;
    if (n <= FEW_OF<NT>) {
      if (by_p) {
        if (t < n) sh.weight[t] = whole(weight(list_z(sh.list[t])));
        __syncthreads();
      }
      const Counted e = count_list(sh, n, by_p);
      bool in = e.mine && e.rank < n1;
      if (by_p) {                                  // every token before the one that reaches top_p
        if (e.mine && e.rank + 1 == n1) sh.total = e.before + e.weight;
        __syncthreads();
        const double before = weight_of(e.before), target = p * (by_k ? weight_of(sh.total) : total);
        if (in && e.rank) in = close_to(before, target) ? perhaps(sh, a, r, weight, e.key, before < target) : before < target;
      }
      const Prefix win = draw_listed(sh, c, race, [&](auto f) { if (in) f(e.key); });
      token = list_key(win.z, win.id) > sh.unsure ? win.id : draw_in_whole<T, NT>(sh, c, a, r, weight, top.id, win.id);
    } else {                                       // longer ones as rows are that keep very many: drawn first, looked at then
      Prefix in = whole_row();
      if (n1 < n) {
        const u64 last = nth_key(sh, n, n1);
        in = Prefix{list_z(last), list_id(last)};
      }
      const auto in_front = [&](const Prefix& f) {
        Whole mine;
        for (unsigned i = t; i < n; i += NT) {
          const u64 key = sh.list[i];
          mine.add(within(f, list_z(key), list_id(key)) ? weight(list_z(key)) : 0.f);
        }
        const u64 w = c.block(mine.sum(), u64{0}, [](u64 x, u64 y) { return x + y; });
        if (t == 0) sh.total = w;
        __syncthreads();
        return weight_of(sh.total);
      };
      const auto draw = [&](const Prefix& f) {
        return draw_listed(sh, c, race, [&](auto g) {
          for (unsigned i = t; i < n; i += NT)
            if (within(f, list_z(sh.list[i]), list_id(sh.list[i]))) g(sh.list[i]);
        });
      };
      const double target = by_p ? p * (by_k ? in_front(in) : total) : 0;
      Prefix win = draw(in);
      while (by_p && win.id != top.id) {
        const Prefix front{win.z, win.id - 1};
        const double w = in_front(front);
        if (close_to(w, target)) {
          const int exact = draw_in_whole<T, NT>(sh, c, a, r, weight, top.id, -1);
          if (exact >= 0) { win.id = exact; break; }
        }
        if (w < target) break;
        win = draw(front);
      }
      token = win.id;
    }
    if (t == 0) a.out[r] = token;
    return;
  }
  bool listed = false;                             // what is kept is in the CTAs' own lists
  if (by_k) {
    kept = kth_token(sh, row, groups, c, weight, kept, k, parts.inbox);
    if (k <= LIST * c.size) listed = list_kept(sh, c, row, groups, kept);
  }
  // A race among what lies within `front`, its weight, or both.
  const auto go = [&](const Prefix& front, bool race_too, bool mass_too) {
    if (listed) return list_lap(sh, race, weight, front, race_too, mass_too);
    if (!race_too) return lap<false, true>(row, groups, race, weight, front, &sh.score);
    return mass_too ? lap<true, true>(row, groups, race, weight, front, &sh.score) : lap<true, false>(row, groups, race, weight, front, &sh.score);
  };
  const Lap l = go(kept, true, by_k && by_p);
  if (by_k && by_p) total = weight_of(row_total(c, l.s));
  Win win = settle(row, c, race, kept, l.m);
  const double target = p * total;
  while (by_p && win.id != top.id) {               // what lies in front of it; who wins there, should that be too much
    const Prefix front{win.z, win.id - 1};
    const double w = weight_of(row_total(c, go(front, false, true).s));
    if (close_to(w, target)) {
      const int exact = draw_in_whole<T, NT>(sh, c, a, r, weight, top.id, -1);
      if (exact >= 0) { win.id = exact; break; }
    }
    if (w < target) break;
    if (t == 0) sh.score = score_key(-INFINITY);   // (all warps are past the last race, and none begins the next before the barrier)
    __syncthreads();
    win = settle(row, c, race, front, go(front, true, false).m);
  }
  if (lead) a.out[r] = win.id;
  c.sync();
}

template <class T, int NT, int AHEAD, bool LISTING>
__global__ void __launch_bounds__(NT, 1024 / NT)
logprob_kernel(const __grid_constant__ LogprobRows a, int per) {
  extern __shared__ __align__(16) float smem[];
  __shared__ RowShared<NT> sh;
  pdl_wait();
  pdl_trigger();
  Cluster c(&sh.mail);
  const int tid = threadIdx.x, r = blockIdx.x / c.size;
  const T* x = static_cast<const T*>(a.x) + r * a.ldx;
  const int t = a.tokens[r];
  const bool there = t >= 0 && t < a.V;
  const float zt = there ? plain_logit(logit(x + t)) : -INFINITY;
  const Row<T, NT> row(x, a.V, c.rank, per);
  const Parts<NT> parts(smem, per, c.size);
  if (LISTING) {
    clear_bins(sh);
    if (tid == 0) sh.n_list = sh.n_hits = 0;
  }
  // log2(e) in two parts: z log2(e) - E as exact as its own size in fp32
  constexpr float HI = 1.4426950408889634f, LO = static_cast<float>(1.4426950408889634 - static_cast<double>(HI));
  Seen seen;
  float largest = -INFINITY;                       // of the thread
  const int tj = t + row.lo;
  row.template stream<AHEAD>([&](const float (&v)[32], int i) {
    const int chunk = row.chunk0 + i;
    float m[4], mine;
    const float highest = look(row, v, i, m, mine, seen.top);
    if (LISTING) {
      largest = fmaxf(largest, mine);
      parts.groups.put(m, i);
    }
    if (highest > -INFINITY && highest < INFINITY) {           // the chunk's sum in units of its own
      const float E = fmaxf(ceilf(highest * HI), -1e30f);
      float s = 0.f;
#pragma unroll
      for (int q = 0; q < 32; q += 4) {
        float w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) w[e] = exp2_fast(fmaf(v[q + e], LO, fmaf(v[q + e], HI, -E)));
        s += (w[0] + w[1]) + (w[2] + w[3]);
      }
      seen.add(s, 0.0, E);
    }
    if (isinf(zt) || (chunk * CHUNK <= tj && tj < (chunk + 1) * CHUNK)) {
#pragma unroll
      for (int q = 0; q < 32; ++q) {
        const int j = Row<T, NT>::place(chunk, q, tid & 31);
        seen.n += v[q] > zt || (v[q] == zt && j < tj && j >= row.lo);
      }
    } else {                                                   // (equal ones are in front of it in the chunks in front of its own; of a finite logit there is a next one)
      const float least = (chunk + 1) * CHUNK <= tj ? zt : nextafterf(zt, INFINITY);
#pragma unroll
      for (int q = 0; q < 32; ++q) seen.n += v[q] >= least;
    }
  });
  c.ready();
  if (c.size > 1 && LISTING)
    for (int i = 0; i < c.size; ++i) c.of(parts.maxima, i)[c.rank * NT + tid] = largest;
  seen = row_seen(c, seen, true, true);
  const Best top = seen.top;
  const bool lead = c.rank == 0 && tid == 0;
  // log-probabilities: z - (E log 2 + log(sum)); seen from the best where logits are so large that this would leave too few bits of it, or infinite
  const bool far = !(fabsf(top.v) < 1e6f);
  double sum = seen.s;
  if (far) {
    sum = 0;
    row.eights([](int) { return true; }, [&](const float (&v)[8], int, int) {
      float f = 0.f;
#pragma unroll
      for (int q = 0; q < 8; ++q) f += v[q] == top.v ? 1.f : exp2_fast((v[q] - top.v) * HI);
      sum += f;
    });
    sum = row_total(c, sum);
  }
  if (lead) sh.log = (far ? 0.0 : static_cast<double>(seen.E) * 0.69314718055994530942) + log(sum);
  const auto lp = [&](float z) {
    if (z == -INFINITY) return -INFINITY;
    return static_cast<float>((far ? (z == top.v ? 0.0 : static_cast<double>(z) - top.v) : static_cast<double>(z)) - sh.log);
  };
  int* ids = a.ids + static_cast<long long>(r) * a.top;
  float* lps = a.logprobs + static_cast<long long>(r) * a.top;
  if (lead) {
    a.logprob[r] = lp(zt);
    a.rank[r] = there ? static_cast<int>(seen.n) + 1 : 0;
    if (a.top == 1) {
      ids[0] = top.v == -INFINITY ? -1 : top.id;
      lps[0] = lp(top.v);
    }
  }
  if (!LISTING) { c.sync(); return; }
  if (!far) {
    const Weights w{HI, ceilf(top.v * HI), 0.f};
    bins_of_threads(sh, c, parts.maxima, largest, w, LOWEST, true, a.top);
    if (sh.bin == BINS - 1) bins_of_groups(sh, c, parts.groups, row.chunks, w, LOWEST, true, a.top);
    const bool found = sh.bin < BINS - 1;
    const float least = found ? w.edge(sh.bin) : LOWEST;
    unsigned n = LIST + 1;
    if (found || few_reach<NT>(c, parts.groups, row.chunks, least)) n = gather(sh, c, row, parts, largest, least);
    if (n <= LIST) {
      if (c.rank) return;
      const auto put = [&](unsigned i, u64 key) { ids[i] = list_id(key); lps[i] = lp(list_z(key)); };
      if (n <= FEW_OF<NT>) {
        const Counted e = count_list(sh, n, false);
        if (e.mine && e.rank < static_cast<unsigned>(a.top)) put(e.rank, e.key);
      } else {
        sort_list<NT>(sh.list, n);
        for (unsigned i = tid; i < min(n, static_cast<unsigned>(a.top)); i += NT) put(i, sh.list[i]);
      }
      for (unsigned i = n + tid; i < static_cast<unsigned>(a.top); i += NT) { ids[i] = -1; lps[i] = -INFINITY; }
      return;
    }
  }
  Best last{INFINITY, -1};                         // one after the other: rows of nothing, of infinities, of very many equal logits
  for (int i = 0; i < a.top; ++i) {
    Best g{-INFINITY, NO_ID};
    row.eights([](int) { return true; }, [&](const float (&v)[8], int n, int q) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int id = row.id(Row<T, NT>::place(row.chunk0 + n, q + e, tid & 31));
        if (v[e] < last.v || (v[e] == last.v && id > last.id)) g = first_of(g, Best{v[e], id});
      }
    });
    last = c.reduce(g, Best{-INFINITY, NO_ID}, first_of);
    if (lead) {
      ids[i] = last.v == -INFINITY ? -1 : last.id;
      lps[i] = lp(last.v);
    }
  }
  c.sync();
}

// CTAs of a row's cluster: as many as run at once, of four chunks each at least.  Clusters of four and eight do not fill every SM (36 rows by eight CTAs take
// 26.5 us, by four 17.3; 74 by four 28.4, by two 18.0).  Draws take two also while that is up to twice as many as run at once, since a row that keeps
// very many tokens holds the others up (256 draws of eight kinds from 152k logits 105 us, with one CTA each 148; without such rows 62 and 49.  1024
// draws from 66k: 189 and 173).
static int row_cluster(int R, int chunks, int sms, bool draws) {
  int c = 1;
  while (c < CLUSTER_MAX && R * c * 2 <= (c == 1 ? 2 * sms : sms * 7 / 4) && c * 4 < chunks) c *= 2;
  return c == 1 && draws && R <= 2 * sms && chunks > 16 ? 2 : c;
}

template <int NT, class A, class K>
static int launch_rows(const char* name, K kern, const A& a, int chunks, int c, cudaStream_t s) {
  const int per = (chunks + c - 1) / c, bytes = Parts<NT>::bytes(per, c);
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) return spark_launch_rc(name);
  spark_launch_pdl(kern, dim3(a.R * c), dim3(NT), bytes, s, dim3(c, 1, 1), a, per);
  return spark_launch_rc(name);
}
// Rows of up to eight chunks take CTAs of four warps: with sixteen most of a short row's would wait at barriers.  500 rows, top_k 40 and top_p 0.9: of 2040
// logits 14.9 us (sixteen warps 22.9), of 4088 12.8 (21.9), of 8184 14.8 (22.6), of 16376 18.6 (24.3).  Rows that keep most of their tokens (top_p 0.98 at
// temperature 1.4) turn at eight chunks: 4088 24 (48), 8184 69 (53), 16376 113 (61).  Log-probabilities with 20 listed: 4088 10.3 (18.6), 16376 15.7 (22.3).
template <class T>
static int sample_rows(const SampleRows& a, cudaStream_t s) {
  const char* name = "spark_sample_rows";
  const int chunks = (a.V + 8 + CHUNK - 1) / CHUNK, c = row_cluster(a.R, chunks, a.sms, true);
  return chunks <= 8 ? launch_rows<128>(name, sample_kernel<T, 128>, a, chunks, c, s) : launch_rows<512>(name, sample_kernel<T, 512>, a, chunks, c, s);
}
// Log-probabilities without lists of the best have a kernel of their own: without the code for lists the loads of a chunk stay together (1024 rows of 152k
// logits 110 us, with it 118), and asking for what comes two chunks later helps (100 us; the other kernels, which read some of a row again, lose by
// it: 256 draws 62 us without and 64 with it, 1024 rows of 66k with their first five 73 and 77).
template <class T>
static int logprob_rows(const LogprobRows& a, cudaStream_t s) {
  const char* name = "spark_logprob_rows";
  const int chunks = (a.V + 8 + CHUNK - 1) / CHUNK, c = row_cluster(a.R, chunks, a.sms, false);
  if (a.top > 1)
    return chunks <= 8 ? launch_rows<128>(name, logprob_kernel<T, 128, 0, true>, a, chunks, c, s) : launch_rows<512>(name, logprob_kernel<T, 512, 0, true>, a, chunks, c, s);
  if (chunks <= 8) return launch_rows<128>(name, logprob_kernel<T, 128, 0, false>, a, chunks, c, s);
  return launch_rows<512>(name, logprob_kernel<T, 512, 2, false>, a, chunks, c, s);
}

}  // namespace spark

using namespace spark;

extern "C" int spark_sample_rows(const SampleRows* a, cudaStream_t s) {
  if (a->R <= 0 || a->V <= 0) return 0;
  return a->type == LT_F32 ? sample_rows<float>(*a, s) : a->type == LT_BF16 ? sample_rows<__nv_bfloat16>(*a, s) : sample_rows<__half>(*a, s);
}

extern "C" int spark_logprob_rows(const LogprobRows* a, cudaStream_t s) {
  if (a->R <= 0 || a->V <= 0) return 0;
  return a->type == LT_F32 ? logprob_rows<float>(*a, s) : a->type == LT_BF16 ? logprob_rows<__nv_bfloat16>(*a, s) : logprob_rows<__half>(*a, s);
}
