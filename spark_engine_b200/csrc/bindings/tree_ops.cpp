// Device side of ops/tree.py: arguments checked, outputs and workspaces taken from torch's allocator, kernels launched on the tensors' device
// and its current stream.  In C++ because a round makes these calls for every layer and the kernels take a few microseconds.
#include <algorithm>
#include <cmath>
#include <cstdlib>

#include "plumbing.h"
#include "tree_args.h"

namespace {

// ------------------------------------------------------------------------------------------------ plumbing
Entry e_tables{"spark_block_tables"}, e_maps{"spark_slot_maps"}, e_conv{"spark_path_conv"}, e_commit{"spark_commit_paths"}, e_attn{"spark_tree_attn", 2};

void bind_entry(const std::string& name, uintptr_t fn) {
  for (Entry* e : {&e_tables, &e_maps, &e_conv, &e_commit, &e_attn})
    if (name == e->name) { e->fn = reinterpret_cast<void*>(fn); return; }
  throw py::value_error("no entry " + name);
}
void need_tables(const Tensor& t) {
  NEED(t.scalar_type() == at::kInt && t.dim() == 2 && t.is_contiguous() && t.size(1) > 0, "tables must be a contiguous int32 tensor [slots, pages]");
  NEED(t.numel() <= 1 << 24, "tables of more than 2^24 entries");
}
int64_t quantum(const Tensor& t) { return 16 / t.element_size(); }
// Stride of dimension i; 0 where it has one entry, whose stride may be anything and means nothing.
int64_t step(const Tensor& t, int64_t i) { return t.size(i) < 2 ? 0 : t.stride(i); }
bool strides_fit(const Tensor& t) {               // the kernels take strides of rows and heads in 32 bits
  for (int64_t i = 0; i < t.dim(); ++i)
    if (step(t, i) >= 1ll << 31) return false;
  return true;
}
bool aligned(const Tensor& t) { return (reinterpret_cast<uintptr_t>(t.data_ptr()) & 15) == 0; }
// Whether kernels can read t in pieces of 16 bytes: channels side by side, the others on multiples of `quantum` elements.
bool in_pieces(const Tensor& t, int64_t quantum) {
  bool ok = aligned(t) && strides_fit(t) && (t.size(-1) < 2 || t.stride(-1) == 1);
  for (int64_t i = 0; i + 1 < t.dim(); ++i) ok = ok && step(t, i) % quantum == 0;
  return ok;
}
// t, or a copy of it that they can.  (A new one: `contiguous` gives a contiguous tensor back wherever it starts.)
Tensor pieces(const Tensor& t, int64_t quantum) {
  if (in_pieces(t, quantum)) return t;
  const Tensor c = t.clone(at::MemoryFormat::Contiguous);
  NEED(in_pieces(c, quantum), "rows must be multiples of 16 bytes");
  return c;
}

// Whether n0 x n1 pieces of `width` elements, s0 and s1 apart, share no memory.
bool apart(int64_t n0, int64_t s0, int64_t n1, int64_t s1, int64_t width) {
  if ((n0 > 1 && s0 < width) || (n1 > 1 && s1 < width)) return false;
  if (n0 < 2 || n1 < 2 || s0 >= (n1 - 1) * s1 + width || s1 >= (n0 - 1) * s0 + width) return true;
  for (int64_t d = 1; d < n1; ++d)               // piece (0, d) and its neighbours (r, 0), (r + 1, 0): any two that meet are that far apart
    for (int64_t r = d * s1 / s0; r <= std::min(d * s1 / s0 + 1, n0 - 1); ++r)
      if (std::abs(d * s1 - r * s0) < width) return false;
  return true;
}

struct Cache { int64_t page, tok, width; };      // strides and a token's channels, in elements
Cache need_cache(const char* name, const Tensor& t, at::ScalarType dtype, const at::Device& dev) {
  NEED(t.dim() >= 3 && t.size(1) == spark::TREE_PAGE && t.scalar_type() == dtype && t.device() == dev, name, " must be a cache [pages, ", spark::TREE_PAGE,
       ", heads, channels] of ", toString(dtype), " on ", dev);
  int64_t want = 1;
  for (int64_t i = t.dim() - 1; i >= 2; --i) {
    NEED(t.size(i) == 1 || t.stride(i) == want, name, ": a token's channels must be contiguous");
    want *= t.size(i);
  }
  const int64_t e = quantum(t);
  NEED(want > 0 && want % e == 0 && (t.size(0) < 2 || t.stride(0) % e == 0) && t.stride(1) % e == 0 && t.stride(1) >= want && aligned(t), name, ": tokens must start on 16 bytes");
  NEED(t.size(0) <= 1 << 24, name, " has more than 2^24 pages");
  NEED(apart(t.size(0), t.stride(0), t.size(1), t.stride(1), want), name, ": pages must not overlap");
  return {t.size(0) < 2 ? spark::TREE_PAGE * t.stride(1) : t.stride(0), t.stride(1), want};
}
bool is_act(at::ScalarType t) { return t == at::kBFloat16 || t == at::kFloat; }

// ------------------------------------------------------------------------------------------------ block tables
Tensor block_tables(const Tensor& lengths, const Tensor& tables, const Tensor& held, const Tensor& free, const Tensor& n_free, bool run) {
  need_tables(tables);
  const at::Device dev = tables.device();
  const int64_t S = tables.size(0);
  need_ints("lengths", lengths, S, dev);
  need_ints("held", held, S, dev);
  need_ints("free", free, -1, dev);
  need_ints("n_free", n_free, 1, dev);
  NEED(free.numel() <= 1 << 24, "more than 2^24 pages");
  Tensor room = at::empty({S}, tables.options());
  if (!run || S == 0) return room;
  const On on(tables);
  spark::BlockTables a{ip(lengths), ip(tables), ip(held), ip(free), ip(n_free), ip(room), on.dev.status, static_cast<int>(S), static_cast<int>(tables.size(1)),
                       static_cast<int>(free.size(0))};
  on.launch(e_tables, &a);
  return room;
}

// ------------------------------------------------------------------------------------------------ row maps
struct RowMaps {
  Tensor starts, slot, index, pos, cache_row, lengths, counts, tables;
  Opt anc, slots, parents;
  int64_t nodes = 0;
  int64_t rows() const { return slot.size(0); }
};

constexpr int64_t MAX_ROWS = 1 << 22, MAX_NODES = 1024, MAX_REQUESTS = 8192, MAX_PATH = 1024, MAX_HEAD = 512;

std::shared_ptr<RowMaps> slot_maps(const Tensor& lengths, const Tensor& counts, const Tensor& tables, int64_t rows, const Opt& slots, const Opt& parents,
                                   int64_t nodes, bool run) {
  need_tables(tables);
  const at::Device dev = tables.device();
  need_ints("lengths", lengths, -1, dev);
  const int64_t S = lengths.size(0);
  need_ints("counts", counts, S, dev);
  if (slots) need_ints("slots", *slots, S, dev);
  else NEED(S <= tables.size(0), "more requests than rows of the tables");
  NEED(rows >= 0 && rows <= MAX_ROWS && S <= MAX_REQUESTS, "at most ", MAX_ROWS, " rows of ", MAX_REQUESTS, " requests");
  if (parents) {
    need_ints("parents", *parents, rows, dev);
    NEED(nodes > 0 && nodes <= MAX_NODES, "a request's tree has 1 to ", MAX_NODES, " nodes (`nodes`)");
  } else {
    NEED(nodes == 0, "`nodes` belongs to `parents`");
  }
  const int64_t words = (nodes + 31) / 32;
  const auto opt = tables.options();
  auto m = std::make_shared<RowMaps>();
  m->lengths = lengths; m->counts = counts; m->tables = tables; m->slots = slots; m->parents = parents; m->nodes = nodes;
  // one allocation for what is int32: [anc | slot | index | pos | starts]
  const at::AutoDispatchBelowADInplaceOrView plain;      // (integers: nobody differentiates them)
  const int64_t na = rows * words;
  Tensor all = at::empty({na + 3 * rows + S + 1}, opt);
  if (words) m->anc = all.as_strided({rows, words}, {words, 1}, 0);
  m->slot = all.as_strided({rows}, {1}, na);
  m->index = all.as_strided({rows}, {1}, na + rows);
  m->pos = all.as_strided({rows}, {1}, na + 2 * rows);
  m->starts = all.as_strided({S + 1}, {1}, na + 3 * rows);
  m->cache_row = at::empty({rows}, opt.dtype(at::kLong));
  if (!run) return m;
  if (S == 0) {
    m->starts.zero_();
    for (Tensor* t : {&m->slot, &m->index, &m->pos, &m->cache_row}) t->fill_(-1);
    if (words) m->anc->zero_();
    return m;
  }
  const On on(tables);
  spark::SlotMaps a{ip(lengths), ip(counts), ip(tables), ip(slots), ip(parents), ip(m->starts), ip(m->slot), ip(m->index), ip(m->pos), ip(m->anc),
                    rows ? static_cast<long long*>(m->cache_row.data_ptr()) : nullptr, on.dev.status, static_cast<int>(S), static_cast<int>(rows),
                    static_cast<int>(tables.size(1)), static_cast<int>(tables.size(0)), static_cast<int>(nodes), static_cast<int>(words)};
  on.launch(e_maps, &a);
  return m;
}

// ------------------------------------------------------------------------------------------------ convolution along paths
Tensor path_conv(Tensor x, const Tensor& w, const Tensor& tail, const RowMaps& m, int64_t nq, const Tensor& k, const Tensor& v, bool run) {
  const auto dt = x.scalar_type();
  const at::Device dev = x.device();
  NEED(x.dim() == 2 && is_act(dt), "rows must be bf16 or fp32 [rows, channels]");
  const int64_t R = x.size(0), C = x.size(1);
  NEED(R == m.rows() && m.slot.device() == dev, "the maps are another round's");
  NEED(w.dim() == 2 && w.size(0) > 0 && w.size(1) == C && w.scalar_type() == at::kFloat && w.device() == dev && w.is_contiguous() && aligned(w),
       "w must be fp32 [taps, channels]");
  const int64_t taps = w.size(0);
  NEED(taps <= 32, "at most 32 taps");
  NEED(tail.dim() == 3 && tail.size(1) == taps - 1 && tail.size(2) == C && tail.scalar_type() == dt && tail.device() == dev && tail.is_contiguous() && aligned(tail),
       "tail must be [slots, taps - 1, channels] in the rows' type");
  NEED(tail.size(0) == m.tables.size(0), "tail and tables must have the same slots");
  const Cache kc = need_cache("k", k, dt, dev), vc = need_cache("v", v, dt, dev);
  NEED(k.size(0) == v.size(0), "k and v must have the same pages");
  NEED(nq >= 0 && nq + kc.width + vc.width == C, "a row's ", C, " channels are not ", nq, " of queries, ", kc.width, " of keys and ", vc.width, " of values");
  NEED(nq % 8 == 0 && kc.width % 8 == 0 && C % 8 == 0, "channels must be multiples of 8");
  NEED(R <= 65535 * 64, "at most 65535 tiles of 64 rows");
  Tensor q = at::empty({R, nq}, x.options());
  if (!run || R == 0) return q;
  NEED(k.size(0) > 0, "caches without pages");
  x = pieces(x, 8);
  const On on(x);
  spark::PathConv a{x.data_ptr(), static_cast<float*>(w.data_ptr()), tail.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), ip(m.slot), ip(m.index),
                    ip(m.parents), static_cast<long long*>(m.cache_row.data_ptr()), on.dev.status, kc.page, kc.tok, vc.page, vc.tok,
                    k.size(0) * spark::TREE_PAGE, static_cast<int>(step(x, 0)), static_cast<int>(R), static_cast<int>(C), static_cast<int>(taps),
                    static_cast<int>(nq), static_cast<int>(kc.width), static_cast<int>(tail.size(0))};
  on.launch(e_conv, &a, static_cast<int>(dt == at::kFloat));
  return q;
}

// ------------------------------------------------------------------------------------------------ attention
void need_heads(const char* name, const Opt& t, int64_t dim, int64_t H, const at::Device& dev) {
  NEED(!t || (t->scalar_type() == at::kFloat && t->device() == dev && t->is_contiguous() && t->dim() == dim && t->size(0) == H && t->numel() > 0), name,
       " must be a contiguous fp32 tensor of ", H, " heads on ", dev);
}
float* fp(const Opt& t) { return t ? static_cast<float*>(t->data_ptr()) : nullptr; }

// Rows of a tile on the tensor cores, for heads of up to 128 (wider ones leave room for one tile of 128 and one CTA per SM): 128 (node, head) rows, two
// CTAs per SM; or, where requests have more of them, two such tiles per CTA that share the keys, one CTA per SM.  A request's rows are known by
// `nodes`; of chains, which may be of any lengths, by the average.  One tile / two (us of a call, 32 query heads on 8 of 128 over 4k tokens): 64 requests
// of trees of 8 nodes (32 rows) 200 / 265, 32 nodes (128 rows) 224 / 299, 33 nodes 384 / 339, 64 nodes (256 rows) 423 / 376; 8 requests of 32 nodes
// 54 / 60, of 33 71 / 65; 64 chains of one row 196 / 253, of 64 rows 421 / 374, one of 500 beside 63 of one 244 / 395.
int64_t tile_rows(int64_t R, int64_t S, int64_t nodes, int64_t rep) {
  const int64_t rows = nodes ? std::min(nodes, R) : (R + S - 1) / S;
  return rows * rep > 128 ? 256 : 128;
}

Tensor tree_attention(Tensor q, const Tensor& k, const Tensor& v, const RowMaps& m, double scale, double softcap, const Opt& bias, const Opt& slopes,
                      const Opt& sink, int64_t window, int64_t chunk, const Opt& gate, double out_scale, const Opt& given, bool run) {
  const auto dt = q.scalar_type();
  const at::Device dev = q.device();
  NEED(q.dim() == 3 && is_act(dt), "queries must be bf16 or fp32 [rows, heads, channels]");
  const int64_t R = q.size(0), H = q.size(1), D = q.size(2);
  const Cache kc = need_cache("k", k, dt, dev), vc = need_cache("v", v, dt, dev);
  NEED(k.dim() == 4 && v.dim() == 4 && k.size(0) == v.size(0) && k.size(2) == v.size(2) && k.size(3) == D,
       "caches must be [pages, ", spark::TREE_PAGE, ", heads, channels], keys as wide as queries");
  const int64_t G = k.size(2), V = v.size(3);
  NEED(H > 0 && H % G == 0, "query heads must be a multiple of the key / value heads");
  NEED(R * H < 1ll << 31, "at most 2^31 rows of heads");
  NEED(D % 8 == 0 && V % 8 == 0 && D <= MAX_HEAD && V <= MAX_HEAD, "head widths must be multiples of 8 up to ", MAX_HEAD);
  NEED(R == m.rows() && m.slot.device() == dev, "the maps are another round's");
  NEED(window >= 0 && chunk >= 0 && !(window && chunk) && window < 1ll << 31 && chunk < 1ll << 31, "either a window or a chunk");
  NEED(softcap >= 0 && std::isfinite(softcap) && std::isfinite(scale) && std::isfinite(out_scale), "scales and soft cap must be finite, the cap not negative");
  need_heads("bias", bias, 2, H, dev);
  need_heads("slopes", slopes, 1, H, dev);
  need_heads("sink", sink, 1, H, dev);
  NEED(!gate || (gate->dim() == 2 && gate->size(0) == R && gate->size(1) == H && gate->scalar_type() == dt && gate->device() == dev && (H < 2 || gate->stride(1) == 1) && strides_fit(*gate)),
       "gate must be [rows, heads] in the queries' type");
  const int64_t e = quantum(q);
  if (given)
    NEED(given->dim() == 3 && given->size(0) == R && given->size(1) == H && given->size(2) == V && given->scalar_type() == dt && given->device() == dev &&
             in_pieces(*given, e) && apart(R, given->stride(0), H, given->stride(1), V),
         "out must be [rows, heads, value channels] in the queries' type, heads apart and on 16 bytes");
  Tensor out = given ? *given : at::empty({R, H, V}, q.options());
  if (!run || R == 0) return out;
  const int64_t S = m.lengths.size(0);
  if (S == 0) return given ? out : out.zero_();
  NEED(k.size(0) > 0, "caches without pages");
  q = pieces(q, e);
  const On on(q);
  const bool tc = dt == at::kBFloat16 && D <= 256 && V <= 256, wide = D > 128 || V > 128;
  const int bm = !tc ? 64 : wide ? 128 : static_cast<int>(tile_rows(R, S, m.nodes, H / G));
  const int ctas = std::min(512, on.dev.sms * (bm == 256 || wide ? 1 : 2));
  // What beginning an item costs, in pages (us of a call: four requests of 16k tokens, heads of 256, with 5 / 8 / 10 / 14 / 20: 51.1 / 48.0 / 47.1 /
  // 47.2 / 47.1; a ragged round with soft cap and bias, whose pages take longer, with 2 / 3 / 4 / 6 / 8: 30.6 / 30.3 / 30.1 / 32.4 / 32.4; windows of 1024
  // and 64 requests of 64 nodes: 3 to 12 make no difference; the FP32 units' pages are long)
  const int extra = !tc ? 0 : wide ? 10 : softcap > 0 || bias || slopes ? 4 : 6;
  const int64_t work = G * (R * (H / G) / bm + S) * (m.tables.size(1) + extra);
  NEED(work < 1ll << 31, "a round of ", R, " rows over tables of ", m.tables.size(1), " pages is more than one call takes");
  // (places for two parts per CTA, whatever the lengths turn out to be: 39 MB for values of 128, in bf16 calls of any size)
  const int64_t no = static_cast<int64_t>(ctas) * 2 * bm * V, nm = static_cast<int64_t>(ctas) * 2 * bm * 2;
  Tensor ws = at::empty({no + nm + ctas * 4}, q.options().dtype(at::kFloat));
  float* part = static_cast<float*>(ws.data_ptr());
  spark::TreeAttn a{q.data_ptr(), k.data_ptr(), v.data_ptr(), out.data_ptr(), ip(m.starts), ip(m.lengths), ip(m.slots), ip(m.pos), ip(m.tables),
                    reinterpret_cast<uint32_t*>(ip(m.anc)), fp(bias), fp(slopes), fp(sink), gate ? gate->data_ptr() : nullptr, part, part + no,
                    reinterpret_cast<int*>(part + no + nm), on.dev.status, kc.page, kc.tok, vc.page, vc.tok};
  const auto i = [](int64_t x) { return static_cast<int>(x); };
  a.S = i(S); a.R = i(R); a.words = m.anc ? i(m.anc->size(1)) : 0; a.page_ld = i(m.tables.size(1)); a.n_slots = i(m.tables.size(0)); a.n_pages = i(k.size(0));
  a.H = i(H); a.G = i(G); a.D = i(D); a.V = i(V); a.ldq = i(step(q, 0)); a.hq = i(step(q, 1)); a.ldo = i(step(out, 0)); a.ho = i(step(out, 1));
  a.ldg = gate ? i(step(*gate, 0)) : 0; a.bias_n = bias ? i(bias->size(1)) : 0; a.window = i(window); a.chunk = i(chunk);
  if (chunk) {
    a.chunk_shift = 31;
    while (1ll << (a.chunk_shift - 31) < chunk) ++a.chunk_shift;
    a.chunk_mul = static_cast<unsigned>(((static_cast<unsigned __int128>(1) << a.chunk_shift) + chunk - 1) / chunk);
  }
  a.bm_log = bm == 64 ? 6 : bm == 128 ? 7 : 8; a.sms = on.dev.sms; a.ctas = ctas; a.extra = extra; a.zero_rest = !given;
  a.scale = static_cast<float>(scale); a.cap = static_cast<float>(softcap); a.out_scale = static_cast<float>(out_scale);
  on.launch(e_attn, &a, static_cast<int>(dt == at::kFloat), static_cast<int>(tc));
  return out;
}

// ------------------------------------------------------------------------------------------------ commit
void commit_paths(const RowMaps& m, const Tensor& path, const Tensor& n_path, const std::vector<Tensor>& caches,
                  const std::vector<std::pair<Tensor, Tensor>>& tails, bool run) {
  const at::Device dev = m.tables.device();
  const int64_t S = m.lengths.size(0);
  NEED(path.scalar_type() == at::kInt && path.device() == dev && path.dim() == 2 && path.size(0) == S && path.is_contiguous(),
       "path must be a contiguous int32 tensor [", S, ", rows] on ", dev);
  need_ints("n_path", n_path, S, dev);
  const int64_t P = path.size(1);
  NEED(P <= MAX_PATH, "paths of at most ", MAX_PATH, " rows");
  std::vector<spark::CommitJob> jobs;
  int64_t pages = -1;
  jobs.reserve(caches.size() + tails.size());
  for (const Tensor& c : caches) {
    NEED(is_act(c.scalar_type()), "caches must be bf16 or fp32");
    const Cache x = need_cache("a cache", c, c.scalar_type(), dev);
    const int64_t e = c.element_size();
    pages = pages < 0 ? c.size(0) : std::min(pages, c.size(0));
    if (c.numel()) jobs.push_back({static_cast<char*>(c.data_ptr()), nullptr, x.page * e, x.tok * e, static_cast<int>(x.width * e), 0});
  }
  for (const auto& [x, t] : tails) {
    NEED(t.dim() == 3 && t.is_contiguous() && t.size(0) == m.tables.size(0) && t.device() == dev && is_act(t.scalar_type()),
         "tails must be contiguous bf16 or fp32 tensors [slots, kept, channels] on ", dev);
    NEED(x.dim() == 2 && x.size(0) == m.rows() && x.size(1) == t.size(2) && x.scalar_type() == t.scalar_type() && x.device() == dev && (x.size(1) < 2 || x.stride(1) == 1),
         "the rows behind a tail must be [rows, channels] in its type");
    const int64_t e = t.element_size();
    NEED(t.size(2) * e % 16 == 0 && step(x, 0) * e % 16 == 0 && aligned(x) && aligned(t), "rows and tails must start on 16 bytes");
    if (t.numel() && x.numel())
      jobs.push_back({static_cast<char*>(t.data_ptr()), static_cast<char*>(x.data_ptr()), step(x, 0) * e, t.size(2) * e, static_cast<int>(t.size(2) * e),
                      static_cast<int>(t.size(1))});
  }
  std::vector<char*> seen;
  for (const auto& j : jobs) seen.push_back(j.base);
  std::sort(seen.begin(), seen.end());
  NEED(std::adjacent_find(seen.begin(), seen.end()) == seen.end(), "a cache or tail is given twice");
  if (!run || jobs.empty() || S == 0 || P == 0 || m.rows() == 0) return;
  const On on(m.tables);
  for (size_t at = 0; at < jobs.size(); at += spark::COMMIT_JOBS) {
    spark::CommitPaths a{{}, ip(path), ip(n_path), ip(m.starts), ip(m.lengths), ip(m.slots), ip(m.tables), on.dev.status, static_cast<int>(S),
                         static_cast<int>(P), static_cast<int>(m.tables.size(1)), static_cast<int>(m.tables.size(0)), static_cast<int>(pages)};
    const int n = static_cast<int>(std::min<size_t>(spark::COMMIT_JOBS, jobs.size() - at));
    int most = 0;
    for (int i = 0; i < n; ++i) { a.job[i] = jobs[at + i]; most = std::max(most, a.job[i].bytes); }
    on.launch(e_commit, &a, n, most);
  }
}

}  // namespace

PYBIND11_MODULE(_tree, mod) {
  mod.doc() = "spark_engine_b200: verification of drafted trees over paged caches (checks and launches)";
  mod.def("bind_entry", &bind_entry).def("bind_device", &bind_device).def("take_launched", &take_launched).def("pieces", &pieces).def("apart", &apart).def("tile_rows", &tile_rows);
  mod.def("layout", [] { return SPARK_TREE_LAYOUT; });
  py::class_<RowMaps, std::shared_ptr<RowMaps>>(mod, "RowMaps",
      "Where a round's rows belong (int32 unless said otherwise; -1 for rows behind the last request): slot [R] row of the tables, index [R]\n"
      "within the request, pos [R], cache_row [R] int64 (page * 64 + token; -1 too where the table has no page), starts [S + 1] first row of\n"
      "every request, anc [R, words] ancestors-or-self as bits over the request's rows (trees; else None).")
      .def_readonly("starts", &RowMaps::starts).def_readonly("slot", &RowMaps::slot).def_readonly("index", &RowMaps::index)
      .def_readonly("pos", &RowMaps::pos).def_readonly("cache_row", &RowMaps::cache_row).def_readonly("anc", &RowMaps::anc)
      .def_readonly("lengths", &RowMaps::lengths).def_readonly("counts", &RowMaps::counts).def_readonly("tables", &RowMaps::tables)
      .def_readonly("slots", &RowMaps::slots).def_readonly("parents", &RowMaps::parents).def_readonly("nodes", &RowMaps::nodes)
      .def_property_readonly("rows", &RowMaps::rows);
  mod.def("block_tables", &block_tables).def("slot_maps", &slot_maps).def("path_conv", &path_conv).def("tree_attention", &tree_attention)
      .def("commit_paths", &commit_paths);
}
