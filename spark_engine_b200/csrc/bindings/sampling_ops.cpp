// Device side of ops/sampling.py: arguments checked, outputs taken from torch's allocator, kernels launched on the tensors' device and its current
// stream.  In C++ because a round makes these calls between two forwards and the kernels take a few microseconds.
#include <torch/csrc/autograd/python_variable.h>

#include "plumbing.h"
#include "sampling_args.h"

namespace {

Entry e_count{"spark_count_tokens"}, e_adjust{"spark_adjust_rows"}, e_sample{"spark_sample_rows"}, e_logprob{"spark_logprob_rows"};

void bind_entry(const std::string& name, uintptr_t fn) {
  for (Entry* e : {&e_count, &e_adjust, &e_sample, &e_logprob})
    if (name == e->name) { e->fn = reinterpret_cast<void*>(fn); return; }
  throw py::value_error("no entry " + name);
}

constexpr int64_t MAX_ROWS = 65535;

int64_t row_step(const Tensor& t) { return t.size(0) < 2 ? 0 : t.stride(0); }
template <class T> T* ptr(const Tensor& t) { return t.numel() ? static_cast<T*>(t.data_ptr()) : nullptr; }
template <class T> T* ptr(const Opt& t) { return t ? ptr<T>(*t) : nullptr; }

void need_vec(const char* name, const Tensor& t, at::ScalarType type, int64_t n, const at::Device& dev) {
  NEED(t.scalar_type() == type && t.device() == dev && t.dim() == 1 && t.size(0) == n && t.is_contiguous(), name, " must be a contiguous tensor of ", n, " ",
       toString(type), " on ", dev, ", not ", t.toString(), " ", t.sizes(), " on ", t.device());
}
void need_vec(const char* name, const Opt& t, at::ScalarType type, int64_t n, const at::Device& dev) { if (t) need_vec(name, *t, type, n, dev); }
void need_table(const char* name, const Tensor& t, at::ScalarType type, int64_t rows, const at::Device& dev) {
  NEED(t.scalar_type() == type && t.device() == dev && t.dim() == 2 && (rows < 0 || t.size(0) == rows) && t.is_contiguous(), name, " must be a contiguous tensor [",
       rows < 0 ? "slots" : std::to_string(rows), ", ...] of ", toString(type), " on ", dev, ", not ", t.toString(), " ", t.sizes(), " on ", t.device());
}
// A table of counts: rows side by side or apart, of whole lines.
void need_counts(const Tensor& t, int64_t V, const at::Device& dev) {
  NEED(t.scalar_type() == at::kInt && t.device() == dev && t.dim() == 2 && (V < 0 || t.size(1) == V) && (t.size(1) < 2 || t.stride(1) == 1) &&
           (t.size(0) < 2 || t.stride(0) >= t.size(1)), "counts must be an int32 tensor [slots, ", V < 0 ? "vocabulary" : std::to_string(V), "] on ", dev,
       ", its rows contiguous and apart, not ", t.toString(), " ", t.sizes(), " on ", t.device());
}

int type_of(const Tensor& t) {
  const auto s = t.scalar_type();
  NEED(s == at::kFloat || s == at::kBFloat16 || s == at::kHalf, "logits must be fp32, bf16 or fp16, not ", toString(s));
  return s == at::kFloat ? spark::LT_F32 : s == at::kBFloat16 ? spark::LT_BF16 : spark::LT_F16;
}
// Rows of logits whose columns lie side by side (copied where they do not).
Tensor rows_of(const Tensor& t) {
  NEED(t.dim() == 2, "logits must be [rows, vocabulary], not ", t.sizes());
  NEED(t.size(0) <= MAX_ROWS && t.size(1) >= 1 && t.size(1) <= spark::SAMPLE_MAX_V, "logits must have at most ", MAX_ROWS, " rows of 1 to ", spark::SAMPLE_MAX_V,
       " columns, not ", t.sizes());
  return t.size(1) < 2 || t.stride(1) == 1 ? t : t.contiguous();
}

// ------------------------------------------------------------------------------------------------ adjustments
struct Adjust {                                  // `Adjust` of ops/sampling.py
  Opt counts, slots, drafted, repetition, presence, frequency, bias_ids, bias, allowed;
  explicit Adjust(const py::object& from) {
    if (from.is_none()) return;
    Opt* to[] = {&counts, &slots, &drafted, &repetition, &presence, &frequency, &bias_ids, &bias, &allowed};
    NEED(py::isinstance<py::tuple>(from) && py::len(from) == 9, "adjustments are given as an `Adjust`");
    for (int i = 0; i < 9; ++i) {
      PyObject* o = PyTuple_GET_ITEM(from.ptr(), i);
      if (o == Py_None) continue;
      NEED(THPVariable_Check(o), "an `Adjust` holds tensors");
      *to[i] = THPVariable_Unpack(o);
    }
  }
  bool any() const { return counts || drafted || repetition || presence || frequency || bias_ids || allowed; }
};

spark::Adjustments adjustments(const Adjust& a, int64_t R, int64_t V, const at::Device& dev) {
  spark::Adjustments k{};
  if (a.counts) {
    need_counts(*a.counts, V, dev);
    NEED(a.slots || R <= a.counts->size(0), "more rows than slots of the counts, and no `slots`");
    k.counts = ptr<int>(*a.counts); k.ld_counts = row_step(*a.counts); k.n_slots = static_cast<int>(a.counts->size(0));
  }
  need_vec("slots", a.slots, at::kInt, R, dev);
  need_vec("repetition", a.repetition, at::kFloat, R, dev);
  need_vec("presence", a.presence, at::kFloat, R, dev);
  need_vec("frequency", a.frequency, at::kFloat, R, dev);
  NEED(a.bias_ids.has_value() == a.bias.has_value(), "bias and bias_ids belong together");
  if (a.drafted) need_table("drafted", *a.drafted, at::kInt, R, dev);
  if (a.bias) {
    need_table("bias_ids", *a.bias_ids, at::kInt, R, dev);
    need_table("bias", *a.bias, at::kFloat, R, dev);
    NEED(a.bias->size(1) == a.bias_ids->size(1), "bias and bias_ids must have the same shape");
  }
  if (a.allowed) {
    need_table("allowed", *a.allowed, at::kInt, R, dev);
    NEED(a.allowed->size(1) == (V + 31) / 32, "allowed must be [", R, ", ", (V + 31) / 32, "] words of 32 columns, not ", a.allowed->sizes());
    k.words = static_cast<int>(a.allowed->size(1));
  }
  const int64_t nd = a.drafted ? a.drafted->size(1) : 0, nb = a.bias ? a.bias->size(1) : 0;
  NEED(nd <= spark::SAMPLE_MAX_LIST && nb <= spark::SAMPLE_MAX_LIST, "at most ", spark::SAMPLE_MAX_LIST, " drafted tokens and biases of a row");
  k.slots = ptr<int>(a.slots); k.drafted = ptr<int>(a.drafted); k.n_drafted = static_cast<int>(nd);
  k.repetition = ptr<float>(a.repetition); k.presence = ptr<float>(a.presence); k.frequency = ptr<float>(a.frequency);
  k.bias_ids = ptr<int>(a.bias_ids); k.bias = ptr<float>(a.bias); k.n_bias = static_cast<int>(nb);
  k.allowed = ptr<uint32_t>(a.allowed);
  return k;
}

// [first, last) byte of a tensor's elements.
std::pair<const char*, const char*> span(const Tensor& t) {
  const char* p = static_cast<const char*>(t.data_ptr());
  int64_t last = 0;
  for (int64_t i = 0; i < t.dim(); ++i) last += (t.size(i) - 1) * t.stride(i);
  return {p, p + (last + 1) * t.element_size()};
}

Tensor adjust_logits(const Tensor& given, const py::object& adjust, int64_t offset, const Opt& out, bool run) {
  const Adjust a(adjust);
  const int type = type_of(given);
  const Tensor x = rows_of(given);
  const at::Device dev = x.device();
  const int64_t R = x.size(0), V = x.size(1);
  NEED(offset >= 0 && offset + V < 1ll << 31, "ids from ", offset, " do not fit 31 bits");
  const spark::Adjustments k = adjustments(a, R, V, dev);
  if (out) {
    NEED(out->scalar_type() == at::kFloat && out->device() == dev && out->sizes() == x.sizes() && (V < 2 || out->stride(1) == 1) && (R < 2 || out->stride(0) >= V),
         "out must be fp32 [", R, ", ", V, "] on ", dev, ", its rows contiguous and apart");
    const bool same = type == spark::LT_F32 && out->data_ptr() == given.data_ptr() && row_step(*out) == row_step(given) && (V < 2 || given.stride(1) == 1);
    if (!same && x.numel()) {
      const auto p = span(*out), q = span(given);
      NEED(p.second <= q.first || q.second <= p.first, "out must be the logits themselves or share no memory with them");
    }
  }
  Tensor y = out ? *out : at::empty({R, V}, x.options().dtype(at::kFloat));
  if (!run || R == 0) return y;
  const On on(x);
  spark::AdjustRows arg{x.data_ptr(), ptr<float>(y), row_step(x), row_step(y), on.dev.status, static_cast<int>(R), static_cast<int>(V), type, static_cast<int>(offset), on.dev.sms, k};
  on.launch(e_adjust, &arg);
  return y;
}

// ------------------------------------------------------------------------------------------------ counts
void count_tokens(const Tensor& counts, const Tensor& tokens, const Tensor& n, const Opt& slots, bool prompt, bool reset, bool run) {
  const at::Device dev = counts.device();
  need_counts(counts, -1, dev);
  NEED(counts.size(1) >= 1 && counts.size(1) <= 1ll << 30, "counts must have 1 to 2^30 columns");
  NEED(tokens.scalar_type() == at::kInt && tokens.device() == dev && tokens.dim() == 2 && (tokens.size(1) < 2 || tokens.stride(1) == 1), "tokens must be an int32 tensor [requests, tokens] on ",
       dev, ", its rows contiguous");
  const int64_t S = tokens.size(0), P = tokens.size(1);
  NEED(S <= MAX_ROWS && P <= 1ll << 30, "at most ", MAX_ROWS, " requests of 2^30 tokens");     // (CTAs step beyond both by some thousands)
  need_vec("n", n, at::kInt, S, dev);
  need_vec("slots", slots, at::kInt, S, dev);
  NEED(slots || S <= counts.size(0), "more requests than slots of the counts, and no `slots`");
  if (!run || S == 0 || (P == 0 && !reset)) return;
  const On on(counts);
  spark::CountTokens arg{ptr<int>(counts), ptr<int>(tokens), ptr<int>(n), ptr<int>(slots), on.dev.status, row_step(counts), row_step(tokens), static_cast<int>(S),
                         static_cast<int>(P), static_cast<int>(counts.size(1)), static_cast<int>(counts.size(0)), prompt, reset};
  on.launch(e_count, &arg);
}

// ------------------------------------------------------------------------------------------------ tokens
Tensor sample_tokens(const Tensor& logits, const Tensor& temps, const Tensor& seeds, const Tensor& positions, const Opt& top_k, const Opt& top_p, const Opt& min_p,
                     const py::object& adjust, bool run) {
  const Adjust a(adjust);
  const int type = type_of(logits);
  const Tensor x = rows_of(logits);
  const at::Device dev = x.device();
  const int64_t R = x.size(0), V = x.size(1);
  need_vec("temps", temps, at::kFloat, R, dev);
  need_vec("seeds", seeds, at::kLong, R, dev);
  need_vec("positions", positions, at::kLong, R, dev);
  need_vec("top_k", top_k, at::kInt, R, dev);
  need_vec("top_p", top_p, at::kFloat, R, dev);
  need_vec("min_p", min_p, at::kFloat, R, dev);
  const spark::Adjustments k = adjustments(a, R, V, dev);
  Tensor out = at::empty({R}, temps.options().dtype(at::kInt));
  if (!run || R == 0) return out;
  const On on(x);
  spark::SampleRows arg{x.data_ptr(), row_step(x), ptr<float>(temps), ptr<long long>(seeds), ptr<long long>(positions), ptr<int>(top_k), ptr<float>(top_p),
                        ptr<float>(min_p), ptr<int>(out), on.dev.status, static_cast<int>(R), static_cast<int>(V), type, on.dev.sms};
  Tensor z;
  if (a.any()) {                                 // (rows of whole 16 bytes)
    const int64_t ld = (V + 3) / 4 * 4;
    z = at::empty({R, ld}, temps.options());
    spark::AdjustRows first{x.data_ptr(), ptr<float>(z), row_step(x), ld, on.dev.status, static_cast<int>(R), static_cast<int>(V), type, 0, on.dev.sms, k};
    on.launch(e_adjust, &first);
    arg.x = z.data_ptr(); arg.ldx = ld; arg.type = spark::LT_F32;
  }
  on.launch(e_sample, &arg);
  return out;
}

py::tuple token_logprobs(const Tensor& logits, const Tensor& tokens, int64_t top, bool run) {
  const int type = type_of(logits);
  const Tensor x = rows_of(logits);
  const at::Device dev = x.device();
  const int64_t R = x.size(0), V = x.size(1);
  need_vec("tokens", tokens, at::kInt, R, dev);
  NEED(top >= 0 && top <= spark::SAMPLE_MAX_TOP, "top must be 0 to ", spark::SAMPLE_MAX_TOP);
  const auto opt = tokens.options();
  Tensor f = at::empty({R * (1 + top)}, opt.dtype(at::kFloat)), i = at::empty({R * (1 + top)}, opt);
  const at::AutoDispatchBelowADInplaceOrView plain;
  Tensor lp = f.as_strided({R}, {1}, 0), lps = f.as_strided({R, top}, {top, 1}, R), rank = i.as_strided({R}, {1}, 0), ids = i.as_strided({R, top}, {top, 1}, R);
  if (run && R) {
    const On on(x);
    spark::LogprobRows arg{x.data_ptr(), row_step(x), ptr<int>(tokens), ptr<float>(lp), ptr<int>(rank), ptr<int>(ids), ptr<float>(lps), on.dev.status,
                           static_cast<int>(R), static_cast<int>(V), type, on.dev.sms, static_cast<int>(top)};
    on.launch(e_logprob, &arg);
  }
  return py::make_tuple(lp, rank, ids, lps);
}

}  // namespace

PYBIND11_MODULE(_sampling, mod) {
  mod.doc() = "spark_engine_b200: from logits to tokens (checks and launches)";
  mod.def("bind_entry", &bind_entry).def("bind_device", &bind_device).def("take_launched", &take_launched);
  mod.def("layout", [] { return SPARK_SAMPLING_LAYOUT; });
  mod.def("count_tokens", &count_tokens).def("adjust_logits", &adjust_logits).def("sample_tokens", &sample_tokens).def("token_logprobs", &token_logprobs);
}
