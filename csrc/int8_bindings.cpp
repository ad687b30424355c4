// Python bindings of the 8-bit integer kernels (module `_int8`).
#include <torch/extension.h>
#include <torch/library.h>

#include <cstdlib>
#include <cstring>
#include <tuple>
#include <vector>

namespace pd {
namespace i8 {
std::vector<at::Tensor> save8(at::Tensor);
at::Tensor load8(at::Tensor, at::Tensor, int64_t);
std::vector<at::Tensor> quantize_rows(at::Tensor);
at::Tensor linear(at::Tensor, at::Tensor, at::Tensor, int64_t, bool, c10::optional<at::Tensor>, int64_t,
                  c10::optional<at::Tensor>);
at::Tensor error_tensor(int64_t);
}  // namespace i8
long long launches();
}  // namespace pd

namespace {
using OptTensor = c10::optional<at::Tensor>;

// Forward-mode derivatives do not pass through the kernels: refused, not dropped.
void no_tangent(const OptTensor& t, const char* who) {
  TORCH_CHECK(!t.has_value() || !t->_fw_grad(0).defined(), who, " has no forward-mode derivative");
}

at::Tensor product(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale, int64_t K, bool grouped,
                   const OptTensor& bias, int64_t act, const OptTensor& residual) {
  const at::NoGradGuard none;                     // the conversions inside make no graph
  return pd::i8::linear(x, codes, scale, K, grouped, bias, act, residual);
}
// A product of integers has no gradient: an output of inputs that require one says so where it is asked for.
struct NoGradient : public torch::autograd::Function<NoGradient> {
  static at::Tensor forward(torch::autograd::AutogradContext*, at::Tensor x, at::Tensor codes, at::Tensor scale, int64_t K,
                            bool grouped, OptTensor bias, int64_t act, OptTensor residual) {
    return product(x, codes, scale, K, grouped, bias, act, residual);
  }
  static torch::autograd::variable_list backward(torch::autograd::AutogradContext*, torch::autograd::variable_list) {
    TORCH_CHECK(false, "int8_linear has no gradient: call it under no_grad, or with detached inputs");
  }
};
// None where the eager form is asked for.
OptTensor linear(const at::Tensor& x, const at::Tensor& codes, const at::Tensor& scale, int64_t K, bool grouped,
                 const OptTensor& bias, int64_t act, const OptTensor& residual) {
  const char* kernels = std::getenv("PD_KERNELS");
  if (kernels != nullptr && std::strcmp(kernels, "eager") == 0) return c10::nullopt;
  no_tangent(x, "int8_linear");
  no_tangent(bias, "int8_linear");
  no_tangent(residual, "int8_linear");
  auto asks = [](const OptTensor& t) { return t.has_value() && t->requires_grad(); };
  if (at::GradMode::is_enabled() && (x.requires_grad() || asks(bias) || asks(residual)))
    return NoGradient::apply(x, codes, scale, K, grouped, bias, act, residual);
  return product(x, codes, scale, K, grouped, bias, act, residual);
}
}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "primus_dlrm_b200 sm_100a kernels: activations in 8 bits, products of 8-bit integers";
  m.def("save8", [](const at::Tensor& x) { no_tangent(x, "save8"); const at::NoGradGuard none; return pd::i8::save8(x); },
        "x [..., K] -> int8 codes [rows, K], scale bytes [blocks of 32, rows]");
  m.def("load8", [](at::Tensor c, at::Tensor e, at::ScalarType t) { return pd::i8::load8(c, e, int64_t(t)); },
        "values of save8's codes and scale bytes in a type");
  m.def("quantize_rows", &pd::i8::quantize_rows, "x [outer, inner, K] -> int8 codes, fp32 scales [outer, inner]");
  m.def("linear", &linear, "act(x W^T + bias) + residual by 8-bit integers");
  m.def("error_word", &pd::i8::error_tensor, "the device's int32 error word (2: a bounded wait ran out)");
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
