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
// A row lies in the shared memory of a cluster's CTAs: it is read once, whatever the passes over it.
#include "../common/token_rows.cuh"

namespace spark {

constexpr int ROW_THREADS = 512;
constexpr int ROW_SLICE_MAX = SAMPLE_MAX_V / 16;

__device__ __forceinline__ uint32_t order_key(float z) {       // larger logits have larger keys
  const uint32_t b = __float_as_uint(z);
  return b & 0x80000000u ? ~b : b | 0x80000000u;
}
__device__ __forceinline__ float key_order(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ unsigned long long mix64(unsigned long long x) {
  x = (x ^ (x >> 30)) * 0xBF58476D1CE4E5B9ull;
  x = (x ^ (x >> 27)) * 0x94D049BB133111EBull;
  return x ^ (x >> 31);
}

// This CTA's columns [b, e) of a row, as fp32 in shared memory.
template <class T>
__device__ __forceinline__ void load_slice(float* z, const T* x, int b, int e) {
  for (int i = threadIdx.x; i < e - b; i += ROW_THREADS) z[i] = plain_logit(logit(x + b + i));
}
template <class T>
__device__ __forceinline__ void load_adjusted(float* z, const T* x, int b, int e, const RowAdjust& adj, int* ids) {
  const int n = adj.entries();
  for (int i = threadIdx.x; i < n; i += ROW_THREADS) ids[i] = adj.entry(i);
  for (int i = threadIdx.x; i < e - b; i += ROW_THREADS) z[i] = plain_logit(adj.common(logit(x + b + i), b + i));
  if (!n) return;
  __syncthreads();
  for (int i = threadIdx.x; i < n; i += ROW_THREADS) {
    const int col = ids[i];
    float y;
    if (col >= b && col < e && adj.listed(i, ids, col, logit(x + col), y)) z[col - b] = plain_logit(y);
  }
}

struct Slice {
  const float* z;
  int b, n;
  template <class F>
  __device__ __forceinline__ void each(F f) const {
    for (int i = threadIdx.x; i < n; i += ROW_THREADS) f(z[i], b + i);
  }
};

__device__ __forceinline__ Best row_best(const Slice& s, Cluster& c) {
  Best m{-INFINITY, NO_ID};
  s.each([&](float z, int id) { m = first_of(m, Best{z, id}); });
  return c.reduce(m, Best{-INFINITY, NO_ID}, first_of);
}

using u64 = unsigned long long;
template <class F>
__device__ __forceinline__ u64 row_sum(const Slice& s, Cluster& c, F f) {
  u64 n = 0;
  s.each([&](float z, int id) { n += f(z, id); });
  return c.reduce(n, u64{0}, [](u64 a, u64 b) { return a + b; });
}

// Weights as whole numbers of 2^-40 of the best token's: sums that no order changes.
struct Weights {
  float top, c;                                    // c = log2(e) / T
  __device__ __forceinline__ u64 operator()(float z) const { return __float2ull_rn(exp2f((z - top) * c) * 1099511627776.f); }
};

// A prefix of the order: its last token.
struct Prefix { float z; int id; };
__device__ __forceinline__ bool within(const Prefix& p, float z, int id) { return z > p.z || (z == p.z && id <= p.id); }

// The largest key for which enough(sum over keys at or above it) holds.
template <class F, class E>
__device__ __forceinline__ uint32_t last_key(const Slice& s, Cluster& c, F f, E enough) {
  uint32_t k = 0;
  for (int bit = 31; bit >= 0; --bit) {
    const uint32_t t = k | 1u << bit;
    if (enough(row_sum(s, c, [&](float z, int id) { return order_key(z) >= t ? f(z, id) : u64{0}; }))) k = t;
  }
  return k;
}
// The prefix that ends with the n-th (from 1) of the tokens equal to z within `of`.
__device__ __forceinline__ Prefix nth_equal(const Slice& s, Cluster& c, float v, u64 n, const Prefix& of) {
  int id = 0;
  for (int bit = 20; bit >= 0; --bit) {            // the largest id with less than n of them in front of it
    const int t = id | 1 << bit;
    if (row_sum(s, c, [&](float z, int i) { return u64{z == v && i < t && within(of, z, i)}; }) < n) id = t;
  }
  return Prefix{v, id};
}

template <class T>
__global__ void __launch_bounds__(ROW_THREADS)
sample_kernel(const __grid_constant__ SampleRows a, int slice, int adjusted) {
  extern __shared__ __align__(16) float z[];
  __shared__ Mailboxes mail;
  Cluster c(&mail);
  const int r = blockIdx.x / c.size, b = min(c.rank * slice, a.V), e = min(b + slice, a.V);
  const T* x = static_cast<const T*>(a.x) + r * a.ldx;
  if (adjusted) load_adjusted(z, x, b, e, RowAdjust(a.a, r, a.status), reinterpret_cast<int*>(z + slice));
  else load_slice(z, x, b, e);
  __syncthreads();
  const Slice s{z, b, e - b};
  const Best top = row_best(s, c);
  const float temp = a.temps[r];
  int token = top.v == -INFINITY ? -1 : top.id;
  // (greedy too: a best score that is not finite, beside which noise is nothing)
  if (top.v != -INFINITY && temp > 0.f && isfinite(__fdiv_rn(top.v, temp))) {
    const double T64 = temp, top64 = top.v;
    const auto scaled = [&](float v) { return (static_cast<double>(v) - top64) / T64; };
    const Weights weight{top.v, 1.4426950408889634f / temp};
    const float p = a.top_p ? a.top_p[r] : 1.f, mp = a.min_p ? a.min_p[r] : 0.f;
    int k = a.top_k ? a.top_k[r] : 0;
    if (p <= 0.f || mp > 1.f) k = 1;
    Prefix kept{-3.402823466e38f, NO_ID};
    if (k == 1) {
      kept = Prefix{top.v, top.id};
    } else {
      if (mp > 0.f) {                              // the smallest logit that is not too improbable
        const double least = log(static_cast<double>(mp));
        float v = fminf(static_cast<float>(top64 + T64 * least), top.v);
        for (int i = 0; i < 8 && scaled(v) >= least; ++i) v = nextafterf(v, -INFINITY);
        for (int i = 0; i < 16 && scaled(v) < least; ++i) v = nextafterf(v, INFINITY);
        kept.z = fmaxf(kept.z, v);
      }
      const auto count = [&](float v, int id) { return u64{within(kept, v, id)}; };
      if (k > 0 && k < a.V && row_sum(s, c, count) > static_cast<u64>(k)) {
        const uint32_t key = last_key(s, c, count, [&](u64 n) { return n >= static_cast<u64>(k); });
        const float v = key_order(key);
        const u64 before = row_sum(s, c, [&](float y, int) { return u64{y > v}; });
        kept = nth_equal(s, c, v, k - before, kept);
      }
      if (p < 1.f) {
        const auto mass = [&](float v, int id) { return within(kept, v, id) ? weight(v) : u64{0}; };
        const double target = static_cast<double>(p) * static_cast<double>(row_sum(s, c, mass));
        const float v = key_order(last_key(s, c, mass, [&](u64 m) { return static_cast<double>(m) >= target; }));
        const u64 before = row_sum(s, c, [&](float y, int) { return y > v ? weight(y) : u64{0}; });
        const u64 same = row_sum(s, c, [&](float y, int id) { return u64{y == v && within(kept, y, id)}; }), w = weight(v);
        const double more = w ? ceil((target - static_cast<double>(before)) / static_cast<double>(w)) : static_cast<double>(same);
        if (more < static_cast<double>(same)) kept = nth_equal(s, c, v, static_cast<u64>(fmax(more, 1.0)), kept);
        else if (v > kept.z) kept = Prefix{v, NO_ID};
      }
    }
    const u64 key = (static_cast<u64>(a.seeds[r]) * 0x9E3779B97F4A7C15ull) ^ (static_cast<u64>(a.positions[r] + 1) * 0xBF58476D1CE4E5B9ull);
    Best m{-INFINITY, NO_ID};
    s.each([&](float v, int id) {
      if (!within(kept, v, id)) return;
      const u64 h = mix64(static_cast<u64>(id) * 0x9E3779B97F4A7C15ull + key);
      const double u = (static_cast<double>(h >> 11) + 0.5) * (1.0 / 9007199254740992.0);
      m = first_of(m, Best{__fadd_rn(__fdiv_rn(v, temp), static_cast<float>(-log(-log(u)))), id});
    });
    token = c.reduce(m, Best{-INFINITY, NO_ID}, first_of).id;
  }
  if (c.rank == 0 && threadIdx.x == 0) a.out[r] = token;
  c.g.sync();                                      // (a CTA's mailbox stays until all have read it)
}

template <class T>
__global__ void __launch_bounds__(ROW_THREADS)
logprob_kernel(const __grid_constant__ LogprobRows a, int slice) {
  extern __shared__ __align__(16) float z[];
  __shared__ Mailboxes mail;
  Cluster c(&mail);
  const int r = blockIdx.x / c.size, b = min(c.rank * slice, a.V), e = min(b + slice, a.V);
  const T* x = static_cast<const T*>(a.x) + r * a.ldx;
  load_slice(z, x, b, e);
  __syncthreads();
  const Slice s{z, b, e - b};
  const Best top = row_best(s, c);
  const int t = a.tokens[r];
  const bool there = t >= 0 && t < a.V;
  const float zt = there ? plain_logit(logit(x + t)) : -INFINITY;
  const auto below = [&](float v) { return v == top.v ? 0.f : v - top.v; };       // (infinite logits: a limit)
  double sum = 0;
  s.each([&](float v, int) { sum += expf(below(v)); });
  sum = c.reduce(sum, 0.0, [](double p, double q) { return p + q; });
  const double lse = log(sum);
  const u64 before = row_sum(s, c, [&](float v, int id) { return u64{v > zt || (v == zt && id < t)}; });
  const bool lead = c.rank == 0 && threadIdx.x == 0;
  if (lead) {
    a.logprob[r] = zt == -INFINITY ? -INFINITY : static_cast<float>(static_cast<double>(below(zt)) - lse);
    a.rank[r] = there ? static_cast<int>(before) + 1 : 0;
  }
  Best last{INFINITY, -1};
  for (int i = 0; i < a.top; ++i) {
    Best m{-INFINITY, NO_ID};
    s.each([&](float v, int id) { if (v < last.v || (v == last.v && id > last.id)) m = first_of(m, Best{v, id}); });
    last = c.reduce(m, Best{-INFINITY, NO_ID}, first_of);
    if (lead) {
      a.ids[static_cast<long long>(r) * a.top + i] = last.v == -INFINITY ? -1 : last.id;
      a.logprobs[static_cast<long long>(r) * a.top + i] = last.v == -INFINITY ? -INFINITY : static_cast<float>(static_cast<double>(below(last.v)) - lse);
    }
  }
  c.g.sync();
}

// CTAs of a row's cluster: enough to hold it, more where there are few rows.
static int row_cluster(int R, int V, int sms) {
  int c = 1;
  while (c < 16 && (static_cast<long long>(c) * 24576 < V || (static_cast<long long>(R) * c * 2 <= sms && V / c > 4096))) c *= 2;
  return c;
}

template <class A, class K, class... X>
static int launch_rows(const char* name, K kern, const A& a, int extra_bytes, cudaStream_t s, X... x) {
  const int c = row_cluster(a.R, a.V, a.sms), slice = ((a.V + c - 1) / c + 63) / 64 * 64, bytes = slice * 4 + extra_bytes;
  if (slice > ROW_SLICE_MAX) return -5;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess ||
      cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return spark_launch_rc(name);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(a.R * c); cfg.blockDim = dim3(ROW_THREADS); cfg.dynamicSmemBytes = bytes; cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = c; attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, kern, a, slice, x...) != cudaSuccess) return spark_launch_rc(name);
  return spark_launch_rc(name);
}

}  // namespace spark

using namespace spark;

extern "C" int spark_sample_rows(const SampleRows* a, int adjusted, cudaStream_t s) {
  if (a->R <= 0 || a->V <= 0) return 0;
  const int extra = adjusted ? (a->a.n_drafted + a->a.n_bias) * 4 : 0;
  if (a->type == LT_F32) return launch_rows("spark_sample_rows", sample_kernel<float>, *a, extra, s, adjusted);
  if (a->type == LT_BF16) return launch_rows("spark_sample_rows", sample_kernel<__nv_bfloat16>, *a, extra, s, adjusted);
  return launch_rows("spark_sample_rows", sample_kernel<__half>, *a, extra, s, adjusted);
}

extern "C" int spark_logprob_rows(const LogprobRows* a, cudaStream_t s) {
  if (a->R <= 0 || a->V <= 0) return 0;
  if (a->type == LT_F32) return launch_rows("spark_logprob_rows", logprob_kernel<float>, *a, 0, s);
  if (a->type == LT_BF16) return launch_rows("spark_logprob_rows", logprob_kernel<__nv_bfloat16>, *a, 0, s);
  return launch_rows("spark_logprob_rows", logprob_kernel<__half>, *a, 0, s);
}
