// Python bindings of the rotary and key/value-cache kernels (module `_kv`).
#include <torch/extension.h>

#include <tuple>
#include <vector>

namespace pd {
namespace kv {
std::vector<at::Tensor> qk_norm_rope(at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>,
                                     c10::optional<at::Tensor>, at::Tensor, c10::optional<at::Tensor>, double, bool,
                                     at::Tensor, c10::optional<at::Tensor>, c10::optional<at::Tensor>);
void kv_append(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
               at::Tensor, c10::optional<at::Tensor>, c10::optional<int64_t>, c10::optional<at::Tensor>, c10::optional<double>,
               c10::optional<at::Tensor>, bool);
void kv_copy_pages(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor);
std::vector<at::Tensor> kv_read(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                                c10::optional<at::Tensor>, c10::optional<int64_t>);
std::vector<at::Tensor> paged_attention(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
                                        at::Tensor, at::Tensor, c10::optional<at::Tensor>, c10::optional<int64_t>,
                                        c10::optional<int64_t>, c10::optional<double>, bool, bool);
}  // namespace kv
long long launches();
}  // namespace pd

// Gradient through qk_norm_rope. In C++ so that a small call is not bound by
// the interpreter: a backward in Python takes the interpreter's lock on the
// autograd thread.
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;
namespace {
using OptTensor = c10::optional<at::Tensor>;

OptTensor fp32(const OptTensor& w) {
  return !w.has_value() || (w->scalar_type() == at::kFloat && w->is_contiguous()) ? w
                                                                                  : OptTensor(w->to(at::kFloat).contiguous());
}

struct QkNormRope : public torch::autograd::Function<QkNormRope> {
  static variable_list forward(AutogradContext* ctx, at::Tensor q, OptTensor k, OptTensor wq, OptTensor wk,
                               at::Tensor table, OptTensor pos, double eps, bool interleaved, at::Tensor err) {
    const OptTensor fq = fp32(wq), fk = fp32(wk);
    auto y = pd::kv::qk_norm_rope(q, k, fq, fk, table, pos, eps, interleaved, err, c10::nullopt, c10::nullopt);
    auto or_none = [](const OptTensor& t) { return t.has_value() ? *t : at::Tensor(); };
    ctx->save_for_backward({q, or_none(k), or_none(fq), or_none(fk), table, or_none(pos), err});
    ctx->saved_data["eps"] = eps;
    ctx->saved_data["interleaved"] = interleaved;
    ctx->saved_data["wq"] = wq.has_value() ? int64_t(wq->scalar_type()) : int64_t(-1);
    ctx->saved_data["wk"] = wk.has_value() ? int64_t(wk->scalar_type()) : int64_t(-1);
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list dy) {
    // the kernel's outputs carry no graph: a gradient of this gradient would be wrong without a word
    TORCH_CHECK(!at::GradMode::is_enabled(), "qk_norm_rope is differentiable once (no create_graph)");
    const auto v = ctx->get_saved_variables();
    auto opt = [&](int i) { return v[i].defined() ? OptTensor(v[i]) : OptTensor(); };
    const OptTensor k = opt(1);
    auto grad = [&](size_t i, const at::Tensor& x) {
      return i < dy.size() && dy[i].defined() ? dy[i].to(x.scalar_type()).contiguous()
                                              : at::zeros(x.sizes(), x.options());
    };
    auto g = pd::kv::qk_norm_rope(v[0], k, opt(2), opt(3), v[4], opt(5), ctx->saved_data["eps"].toDouble(),
                                  ctx->saved_data["interleaved"].toBool(), v[6], grad(0, v[0]),
                                  k.has_value() ? OptTensor(grad(1, *k)) : OptTensor());
    auto weight = [&](const char* name, size_t i) {
      const int64_t t = ctx->saved_data[name].toInt();
      return t < 0 || i >= g.size() ? at::Tensor() : g[i].to(at::ScalarType(t));
    };
    const bool two = k.has_value();
    return {g[0], two ? g[1] : at::Tensor(), weight("wq", two ? 2 : 1), two ? weight("wk", 3) : at::Tensor(),
            at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

// Forward-mode derivatives do not pass through the kernels: refused, not dropped.
void no_tangent(const OptTensor& t, const char* who) {
  TORCH_CHECK(!t.has_value() || !t->_fw_grad(0).defined(), who, " has no forward-mode derivative");
}

// Attention over a cache has no gradient: its output of a query that requires one says so where it is asked for.
using Attended = std::vector<at::Tensor>;
struct PagedAttention : public torch::autograd::Function<PagedAttention> {
  static variable_list forward(AutogradContext*, at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor ks, at::Tensor vs,
                               at::Tensor err, at::Tensor table, at::Tensor lens, OptTensor cu,
                               c10::optional<int64_t> max_q, c10::optional<int64_t> max_len, c10::optional<double> scale,
                               bool causal, bool want_lse) {
    return pd::kv::paged_attention(q, k, v, ks, vs, err, table, lens, cu, max_q, max_len, scale, causal, want_lse);
  }
  static variable_list backward(AutogradContext*, variable_list) {
    TORCH_CHECK(false, "paged_attention has no gradient: call it under no_grad, or with a detached query");
  }
};
Attended attend(at::Tensor q, at::Tensor k, at::Tensor v, at::Tensor ks, at::Tensor vs, at::Tensor err, at::Tensor table,
                at::Tensor lens, OptTensor cu, c10::optional<int64_t> max_q, c10::optional<int64_t> max_len,
                c10::optional<double> scale, bool causal, bool want_lse) {
  no_tangent(q, "paged_attention");
  if (at::GradMode::is_enabled() && q.requires_grad())
    return PagedAttention::apply(q, k, v, ks, vs, err, table, lens, cu, max_q, max_len, scale, causal, want_lse);
  return pd::kv::paged_attention(q, k, v, ks, vs, err, table, lens, cu, max_q, max_len, scale, causal, want_lse);
}

OptTensor unit_stride(const OptTensor& x) {
  return !x.has_value() || x->dim() == 0 || x->stride(-1) == 1 ? x : OptTensor(x->contiguous());
}

// One error word a device for the calls that have no object to keep one in.
at::Tensor rotary_err(int64_t device) {
  static auto* words = new std::vector<at::Tensor>(64);      // never freed: the driver may be gone at exit
  TORCH_CHECK(device >= 0 && device < 64, "no such device");
  at::Tensor& w = (*words)[size_t(device)];
  if (!w.defined()) {
    const c10::InferenceMode normal(false);                  // a later training step saves it for its backward
    w = at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, c10::DeviceIndex(device)));
  }
  return w;
}

std::tuple<at::Tensor, OptTensor> rotary(at::Tensor q, OptTensor k, OptTensor wq, OptTensor wk, at::Tensor table,
                                         OptTensor pos, double eps, bool interleaved) {
  TORCH_CHECK(q.is_cuda() && q.dim() == 4, "q must be a CUDA tensor [B, T, H, d]");
  for (const OptTensor& t : {OptTensor(q), k, wq, wk, OptTensor(table)}) no_tangent(t, "qk_norm_rope");
  TORCH_CHECK(!(at::GradMode::is_enabled() && table.requires_grad()),
              "qk_norm_rope gives the angle table no gradient: detach it");
  const at::Tensor err = rotary_err(q.get_device());
  q = *unit_stride(q);
  k = unit_stride(k);
  if (pos.has_value() && !pos->is_contiguous()) pos = pos->contiguous();
  auto needs = [](const OptTensor& t) { return t.has_value() && t->requires_grad(); };
  const bool grad = at::GradMode::is_enabled() && (q.requires_grad() || needs(k) || needs(wq) || needs(wk));
  std::vector<at::Tensor> y =
      grad ? QkNormRope::apply(q, k, wq, wk, table, pos, eps, interleaved, err)
           : pd::kv::qk_norm_rope(q, k, fp32(wq), fp32(wk), table, pos, eps, interleaved, err, c10::nullopt, c10::nullopt);
  return {y[0], k.has_value() ? OptTensor(y[1]) : OptTensor()};
}
}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "primus_dlrm_b200 sm_100a kernels: query/key norm with rotation, paged 8-bit key/value cache, attention";
  m.def("rotary", &rotary, "(q', k') of qk_norm_rope, with gradients where asked for");
  m.def("rotary_err", &rotary_err, "the device's int32 error word of `rotary`");
  m.def("append", &pd::kv::kv_append, "new tokens' keys and values into the pages of a cache");
  m.def("copy_pages", &pd::kv::kv_copy_pages, "pages dst become copies of pages src");
  m.def("read", &pd::kv::kv_read, "tokens [first, first + n) of each sequence as bf16 [B, n, H, d]");
  m.def("paged_attention", &attend, "attention of the last tokens over a cache -> [o(, lse)]");
  m.def("launch_count", &pd::launches);
}
