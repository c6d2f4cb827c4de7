// What the bindings share: entries of the kernel library, devices and their streams, refusals.  Each module has its own.
#pragma once
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/extension.h>

#include <sstream>
#include <utility>
#include <vector>

namespace py = pybind11;
using at::Tensor;
using Opt = std::optional<Tensor>;

namespace {

struct Entry {                                   // an entry point of the kernel library
  const char* name;
  int kernels = 1;                               // of a call
  void* fn = nullptr;
};
int64_t launched = 0;                            // kernels since it was last asked for
int64_t take_launched() { return std::exchange(launched, 0); }
struct Device { int* status = nullptr; int sms = 0; };
std::vector<Device> devices;

void bind_device(int index, uintptr_t status, int sms) {
  if (static_cast<int>(devices.size()) <= index) devices.resize(index + 1);
  devices[index] = {reinterpret_cast<int*>(status), sms};
}
bool knows_device(int index) { return index >= 0 && index < static_cast<int>(devices.size()) && devices[index].sms > 0; }

template <class... A>
[[noreturn]] void refuse(const A&... a) {
  std::ostringstream s;
  (s << ... << a);
  throw py::value_error(s.str());
}
#define NEED(c, ...) do { if (!(c)) refuse(__VA_ARGS__); } while (0)

struct On {                                      // the tensors' device and its current stream
  c10::cuda::OptionalCUDAGuard guard;
  Device dev;
  cudaStream_t stream;
  explicit On(const Tensor& t) {
    NEED(t.is_cuda() && knows_device(t.get_device()), "no such device: ", t.device());
    if (c10::cuda::current_device() != t.get_device()) guard.set_device(t.device());
    dev = devices[t.get_device()];
    stream = c10::cuda::getCurrentCUDAStream(t.get_device()).stream();
  }
  template <class... A>
  void launch(const Entry& e, A... args) const {
    const int rc = reinterpret_cast<int (*)(A..., cudaStream_t)>(e.fn)(args..., stream);
    if (rc) throw std::runtime_error(std::string(e.name) + " failed with code " + std::to_string(rc));
    launched += e.kernels;
  }
};

void need_ints(const char* name, const Tensor& t, int64_t n, const at::Device& dev) {
  NEED(t.scalar_type() == at::kInt && t.device() == dev && t.dim() == 1 && t.is_contiguous() && (n < 0 || t.size(0) == n), name,
       " must be a contiguous int32 tensor", n < 0 ? "" : " of ", n < 0 ? "" : std::to_string(n), " on ", dev, ", not ", t.toString(), " ", t.sizes());
}
int* ip(const Tensor& t) { return t.numel() ? static_cast<int*>(t.data_ptr()) : nullptr; }
int* ip(const Opt& t) { return t ? ip(*t) : nullptr; }

}  // namespace
