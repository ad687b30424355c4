// Python bindings of the 8-bit integer kernels (module `_int8`).
#include <torch/extension.h>
#include <torch/library.h>

#include <tuple>
#include <vector>

namespace pd {
namespace i8 {
std::vector<at::Tensor> save8(at::Tensor);
at::Tensor load8(at::Tensor, at::Tensor, int64_t);
std::vector<at::Tensor> quantize_rows(at::Tensor);
at::Tensor linear(at::Tensor, at::Tensor, at::Tensor, int64_t, bool, c10::optional<at::Tensor>, int64_t,
                  c10::optional<at::Tensor>);
int64_t error_code(int64_t);
}  // namespace i8
long long launches();
}  // namespace pd

namespace {
using OptTensor = c10::optional<at::Tensor>;

// Forward-mode derivatives do not pass through the kernels: refused, not dropped.
void no_tangent(const OptTensor& t, const char* who) {
  TORCH_CHECK(!t.has_value() || !t->_fw_grad(0).defined(), who, " has no forward-mode derivative");
}

at::Tensor linear(at::Tensor x, at::Tensor codes, at::Tensor scale, int64_t K, bool grouped, OptTensor bias, int64_t act,
                  OptTensor residual) {
  for (const OptTensor& t : {OptTensor(x), bias, residual}) no_tangent(t, "int8_linear");
  const at::NoGradGuard none;                     // the conversions inside make no graph
  return pd::i8::linear(x, codes, scale, K, grouped, bias, act, residual);
}
}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "primus_dlrm_b200 sm_100a kernels: activations in 8 bits, products of 8-bit integers";
  m.def("save8", &pd::i8::save8, "x [rows, K] -> int8 codes [rows, K], scale bytes [blocks of 32, rows]");
  m.def("load8", [](at::Tensor c, at::Tensor e, at::ScalarType t) { return pd::i8::load8(c, e, int64_t(t)); },
        "values of save8's codes and scale bytes in a type");
  m.def("quantize_rows", &pd::i8::quantize_rows, "x [outer, inner, K] -> int8 codes, fp32 scales [outer, inner]");
  m.def("linear", &linear, "act(x W^T + bias) + residual by 8-bit integers");
  m.def("error_code", &pd::i8::error_code, "the device's error word (2: a bounded wait ran out)");
  m.def("launch_count", &pd::launches);
}

// For the layers of the _gemm module, which keep their activations in 8 bits.
namespace {
std::tuple<at::Tensor, at::Tensor> save_rows(const at::Tensor& x) {
  auto v = pd::i8::save8(x);
  return {v[0], v[1]};
}
at::Tensor load_rows(const at::Tensor& codes, const at::Tensor& scale_bytes, at::ScalarType type) {
  return pd::i8::load8(codes, scale_bytes, int64_t(type));
}
}  // namespace
TORCH_LIBRARY(primus_int8, m) {
  m.def("save8(Tensor x) -> (Tensor, Tensor)", save_rows);
  m.def("load8(Tensor codes, Tensor scale_bytes, ScalarType type) -> Tensor", load_rows);
}
