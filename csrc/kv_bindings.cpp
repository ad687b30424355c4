// Python bindings of the rotary and key/value-cache kernels (module `_kv`).
#include <torch/extension.h>

namespace pd {
namespace kv {
std::vector<at::Tensor> qk_norm_rope(at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>,
                                     c10::optional<at::Tensor>, at::Tensor, c10::optional<at::Tensor>, double, bool,
                                     at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>);
void kv_append(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
               at::Tensor, c10::optional<at::Tensor>, int64_t, c10::optional<at::Tensor>, c10::optional<double>,
               c10::optional<at::Tensor>, bool);
std::vector<at::Tensor> kv_read(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                                c10::optional<at::Tensor>, int64_t);
std::vector<at::Tensor> paged_attention(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                                        at::Tensor, at::Tensor, c10::optional<at::Tensor>, int64_t, int64_t, double,
                                        bool, bool);
}  // namespace kv
long long launches();
}  // namespace pd

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "primus_dlrm_b200 sm_100a kernels: query/key norm with rotation, paged 8-bit key/value cache, attention";
  m.def("qk_norm_rope", &pd::kv::qk_norm_rope, py::arg("q"), py::arg("k"), py::arg("w_q"), py::arg("w_k"),
        py::arg("table"), py::arg("positions"), py::arg("eps"), py::arg("interleaved"), py::arg("err"),
        py::arg("dy_q") = py::none(), py::arg("dy_k") = py::none(),
        "[y_q, y_k]; with the outputs' gradients [dq, dk, dw_q, dw_k] (without k: its entries are left out)");
  m.def("append", &pd::kv::kv_append, "new tokens' keys and values into the pages of a cache");
  m.def("read", &pd::kv::kv_read, "tokens [first, first + n) of each sequence as bf16 [B, n, H, d]");
  m.def("paged_attention", &pd::kv::paged_attention, "attention of the last tokens over a cache -> [o(, lse)]");
  m.def("launch_count", &pd::launches);
}
