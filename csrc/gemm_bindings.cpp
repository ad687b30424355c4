// Python bindings of the primus_dlrm_b200 tensor-core kernels (module `_gemm`):
// pyramid attention (attn_fmha.cu) and the tcgen05 GEMMs (gemm_*.cu).
#include <torch/extension.h>

#include "gemm_mat.h"

#include <ATen/core/dispatch/Dispatcher.h>
#include <c10/core/DeviceGuard.h>

#include <tuple>

namespace pd {
std::vector<at::Tensor> fmha_fwd(at::Tensor, at::Tensor, at::Tensor, double, int64_t);
void fmha_bwd(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor,
              at::Tensor, double);
long long launches();
std::vector<at::Tensor> fmha_fwd_tc(at::Tensor, int64_t, double, at::Tensor);
void fmha_bwd_tc(at::Tensor, at::Tensor, at::Tensor, at::Tensor, at::Tensor, int64_t, double, at::Tensor,
                 c10::optional<at::Tensor>);
int64_t fmha_bwd_tc_max_q();
void tc_gemm(at::Tensor, at::Tensor, at::Tensor, int64_t, c10::optional<at::Tensor>, c10::optional<at::Tensor>,
             at::Tensor, bool, c10::optional<at::Tensor>);
void gemm_lines(const Mat&, const Mat&, const Mat&, const Mat*, int*, bool);
void gemm_saved8(const Mat&, const Mat&, const Mat&, const MatCodes&, const Mat*, int*, bool);
at::Tensor wgrad_as(const Mat&, const Mat&, const at::Device&, int*, bool, int64_t);
void tc_wgrad(at::Tensor, at::Tensor, at::Tensor, at::Tensor, bool);
at::Tensor gemm_error_word(int64_t, int64_t);
at::Tensor tc_mma_rate(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, at::Tensor);
at::Tensor tc_mma_burst(int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, int64_t, at::Tensor);
}  // namespace pd

// Layers that keep their activations in 8 bits. Their nodes are in C++: a step calls a dozen kernels, and a backward in
// Python would hold the interpreter's lock on the autograd thread between them.
namespace {
using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

std::tuple<at::Tensor, at::Tensor> save8(const at::Tensor& x) {
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("primus_int8::save8", "")
                       .typed<std::tuple<at::Tensor, at::Tensor>(const at::Tensor&)>();
  return op.call(x);
}
at::Tensor load8(const at::Tensor& codes, const at::Tensor& scale_bytes) {          // exact in bf16
  static auto op = c10::Dispatcher::singleton()
                       .findSchemaOrThrow("primus_int8::load8", "")
                       .typed<at::Tensor(const at::Tensor&, const at::Tensor&, at::ScalarType)>();
  return op.call(codes, scale_bytes, at::kBFloat16);
}

// bf16, in one piece, on 16 bytes: what the products read (a copy only where t is not).
at::Tensor whole(const at::Tensor& t) {
  const at::Tensor c = t.to(at::kBFloat16).contiguous();
  return reinterpret_cast<uintptr_t>(c.data_ptr()) % 16 == 0 ? c : c.clone();
}
// Rows of a whole [B, T, N] tensor: all of them; those of every sample before n_s, one batch for each sample; those from n_s
// on, one batch for each of them. Taken from the sizes: a whole tensor's stride over an axis of length 1 may be anything.
pd::Mat flat(const at::Tensor& t) {
  return {t.data_ptr(), 1, t.size(0) * t.size(1), t.size(2), 0, t.size(2)};
}
pd::Mat head(const at::Tensor& t, int64_t n_s) {
  return {t.data_ptr(), t.size(0), n_s, t.size(2), t.size(1) * t.size(2), t.size(2)};
}
pd::Mat tail(const at::Tensor& t, int64_t n_s) {
  return {static_cast<char*>(t.data_ptr()) + n_s * t.size(2) * t.element_size(), t.size(1) - n_s, t.size(0), t.size(2),
          t.size(2), t.size(1) * t.size(2)};
}
// A whole weight [N, K] or [L, N, K].
pd::Mat weight(const at::Tensor& w) {
  const int64_t n = w.size(-2), k = w.size(-1);
  return {w.data_ptr(), w.dim() == 3 ? w.size(0) : 1, n, k, n * k, k};
}
pd::Mat* ref(pd::Mat&& m) { return &m; }                  // for the length of a call

// out = x by the shared weight, the rows from n_s on by their own; b_kn: by the weights transposed.
void mixed(const at::Tensor& x, int64_t n_s, const at::Tensor& ws, const at::Tensor& wn, const at::Tensor& out, int* err,
           bool b_kn, const at::Tensor& residual = at::Tensor()) {
  const bool r = residual.defined();
  pd::gemm_lines(flat(x), weight(ws), flat(out), r ? ref(flat(residual)) : nullptr, err, b_kn);
  if (x.size(1) > n_s)
    pd::gemm_lines(tail(x, n_s), weight(wn), tail(out, n_s), r ? ref(tail(residual, n_s)) : nullptr, err, b_kn);
}
// The same around pre-activations in 8 bits (codes [B T, N], bytes [N / 32, B T]): without aux out = gelu(..) and the codes
// are written, with it out = .. * gelu'(p), aux = gelu(p).
void mixed_saved(const at::Tensor& x, int64_t n_s, const at::Tensor& ws, const at::Tensor& wn, const at::Tensor& out,
                 const at::Tensor& codes, const at::Tensor& bytes, const at::Tensor& aux, int* err, bool b_kn) {
  const int64_t T = x.size(1), N = codes.size(1), rows = codes.size(0);
  int8_t* c = codes.data_ptr<int8_t>();
  uint8_t* e = bytes.data_ptr<uint8_t>();
  const bool use = aux.defined();
  pd::gemm_saved8(flat(x), weight(ws), flat(out), pd::MatCodes{c, 0, N, e, 0, 1, rows}, use ? ref(flat(aux)) : nullptr, err,
                  b_kn);
  if (T > n_s)
    pd::gemm_saved8(tail(x, n_s), weight(wn), tail(out, n_s), pd::MatCodes{c + n_s * N, N, T * N, e + n_s, 1, T, rows},
                    use ? ref(tail(aux, n_s)) : nullptr, err, b_kn);
}
// Gradients of the shared weight (one sum over the samples' rows, read in place) and of the others.
at::Tensor shared_grad(const at::Tensor& dy, const at::Tensor& x, int64_t n_s, int* err, int64_t type) {
  if (x.size(1) == n_s) return pd::wgrad_as(flat(dy), flat(x), dy.device(), err, true, type);
  return pd::wgrad_as(head(dy, n_s), head(x, n_s), dy.device(), err, true, type);
}
at::Tensor own_grad(const at::Tensor& dy, const at::Tensor& x, int64_t n_s, int* err, int64_t type) {
  return pd::wgrad_as(tail(dy, n_s), tail(x, n_s), dy.device(), err, false, type);
}

at::Tensor rows_of(const at::Tensor& t) { return t.view({t.size(0) * t.size(1), t.size(2)}); }
at::Tensor like(const at::Tensor& x, int64_t N) { return at::empty({x.size(0), x.size(1), N}, x.options()); }
std::tuple<at::Tensor, at::Tensor> room(const at::Tensor& x, int64_t N) {            // codes and scale bytes of [B, T, N]
  const int64_t rows = x.size(0) * x.size(1);
  return {at::empty({rows, N}, x.options().dtype(at::kChar)), at::empty({N / 32, rows}, x.options().dtype(at::kByte))};
}
void once() {
  TORCH_CHECK(!at::GradMode::is_enabled(), "a layer with activations in 8 bits is differentiable once (no create_graph)");
}

struct MixedLinearSaved8 : public torch::autograd::Function<MixedLinearSaved8> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor x, at::Tensor w_s, at::Tensor w_ns, int64_t n_s, bool gelu,
                            at::Tensor err) {
    const at::Tensor xb = whole(x), ws = whole(w_s), wn = whole(w_ns);
    const at::Tensor y = like(xb, ws.size(0));
    at::Tensor pc, pb;
    if (gelu) {
      std::tie(pc, pb) = room(xb, ws.size(0));
      mixed_saved(xb, n_s, ws, wn, y, pc, pb, at::Tensor(), err.data_ptr<int>(), false);
    } else {
      mixed(xb, n_s, ws, wn, y, err.data_ptr<int>(), false);
    }
    auto [xc, xs] = save8(rows_of(xb));
    ctx->save_for_backward({ws, wn, xc, xs, pc, pb});
    ctx->saved_data["err"] = err;
    ctx->saved_data["n_s"] = n_s;
    ctx->saved_data["ws"] = int64_t(w_s.scalar_type());
    ctx->saved_data["wn"] = int64_t(w_ns.scalar_type());
    return y;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once();
    const c10::DeviceGuard guard(g[0].device());
    const auto v = ctx->get_saved_variables();
    const at::Tensor &ws = v[0], &wn = v[1], word = ctx->saved_data["err"].toTensor();
    int* err = word.data_ptr<int>();
    const int64_t n_s = ctx->saved_data["n_s"].toInt();
    at::Tensor dy = whole(g[0]), dx, dws, dwn;
    if (v[4].defined()) dy = at::gelu_backward(dy, load8(v[4], v[5]).view(dy.sizes()));
    if (ctx->needs_input_grad(0)) {
      dx = like(dy, ws.size(1));
      mixed(dy, n_s, ws, wn, dx, err, true);
    }
    if (ctx->needs_input_grad(1) || ctx->needs_input_grad(2)) {
      const at::Tensor x = load8(v[2], v[3]).view({dy.size(0), dy.size(1), ws.size(1)});
      if (ctx->needs_input_grad(1)) dws = shared_grad(dy, x, n_s, err, ctx->saved_data["ws"].toInt());
      if (ctx->needs_input_grad(2)) dwn = own_grad(dy, x, n_s, err, ctx->saved_data["wn"].toInt());
    }
    return {dx, dws, dwn, at::Tensor(), at::Tensor(), at::Tensor()};
  }
};

struct MixedFFNSaved8 : public torch::autograd::Function<MixedFFNSaved8> {
  static at::Tensor forward(AutogradContext* ctx, at::Tensor x, at::Tensor z, at::Tensor w1, at::Tensor w2, at::Tensor wn1,
                            at::Tensor wn2, int64_t n_s, at::Tensor err) {
    const at::Tensor xb = whole(x), w[4] = {whole(w1), whole(w2), whole(wn1), whole(wn2)};
    const at::Tensor h = like(xb, w[0].size(0)), out = like(xb, w[1].size(0));
    auto [pc, pb] = room(xb, w[0].size(0));
    mixed_saved(xb, n_s, w[0], w[2], h, pc, pb, at::Tensor(), err.data_ptr<int>(), false);
    mixed(h, n_s, w[1], w[3], out, err.data_ptr<int>(), false, whole(z));
    auto [xc, xs] = save8(rows_of(xb));
    ctx->save_for_backward({xc, xs, pc, pb, w[0], w[1], w[2], w[3]});
    ctx->saved_data["err"] = err;
    ctx->saved_data["n_s"] = n_s;
    ctx->saved_data["types"] = std::vector<int64_t>{int64_t(w1.scalar_type()), int64_t(w2.scalar_type()),
                                                    int64_t(wn1.scalar_type()), int64_t(wn2.scalar_type())};
    return out;
  }
  static variable_list backward(AutogradContext* ctx, variable_list g) {
    once();
    const c10::DeviceGuard guard(g[0].device());
    const auto v = ctx->get_saved_variables();
    const at::Tensor &w1 = v[4], &w2 = v[5], &wn1 = v[6], &wn2 = v[7], word = ctx->saved_data["err"].toTensor();
    int* err = word.data_ptr<int>();
    const int64_t n_s = ctx->saved_data["n_s"].toInt();
    const auto types = ctx->saved_data["types"].toIntVector();
    const at::Tensor dy = whole(g[0]);
    at::Tensor grads[6];
    if (ctx->needs_input_grad(1)) grads[1] = g[0];
    const at::Tensor dp = like(dy, w1.size(0));
    {
      const at::Tensor h = like(dy, w1.size(0));
      mixed_saved(dy, n_s, w2, wn2, dp, v[2], v[3], h, err, true);
      if (ctx->needs_input_grad(3)) grads[3] = shared_grad(dy, h, n_s, err, types[1]);
      if (ctx->needs_input_grad(5)) grads[5] = own_grad(dy, h, n_s, err, types[3]);
    }
    if (ctx->needs_input_grad(0)) {
      grads[0] = like(dy, w1.size(1));
      mixed(dp, n_s, w1, wn1, grads[0], err, true);
    }
    if (ctx->needs_input_grad(2) || ctx->needs_input_grad(4)) {
      const at::Tensor x = load8(v[0], v[1]).view({dy.size(0), dy.size(1), w1.size(1)});
      if (ctx->needs_input_grad(2)) grads[2] = shared_grad(dp, x, n_s, err, types[0]);
      if (ctx->needs_input_grad(4)) grads[4] = own_grad(dp, x, n_s, err, types[2]);
    }
    return {grads[0], grads[1], grads[2], grads[3], grads[4], grads[5], at::Tensor(), at::Tensor()};
  }
};

// Forward-mode derivatives do not pass through the kernels: refused, not dropped.
void no_tangents(std::initializer_list<at::Tensor> ts) {
  for (const at::Tensor& t : ts)
    TORCH_CHECK(!t._fw_grad(0).defined(), "a layer with activations in 8 bits has no forward-mode derivative");
}
void fits(const at::Tensor& x, int64_t n_s, const at::Tensor& ws, const at::Tensor& wn) {
  TORCH_CHECK(x.dim() == 3 && x.scalar_type() == at::kBFloat16 && ws.dim() == 2 && wn.dim() == 3 && n_s >= 0 &&
                  wn.size(0) == x.size(1) - n_s && wn.size(1) == ws.size(0) && wn.size(2) == ws.size(1) &&
                  ws.size(1) == x.size(2) && ws.device() == x.device() && wn.device() == x.device(),
              "x [B, T, K] must be bf16, the weights [N, K] and [T - n_s, N, K], on one device");
}

at::Tensor mixed_linear_saved8(at::Tensor x, at::Tensor w_s, at::Tensor w_ns, int64_t n_s, bool gelu, at::Tensor err) {
  no_tangents({x, w_s, w_ns});
  fits(x, n_s, w_s, w_ns);
  const c10::DeviceGuard guard(x.device());
  return MixedLinearSaved8::apply(x, w_s, w_ns, n_s, gelu, err);
}
at::Tensor mixed_ffn_saved8(at::Tensor x, at::Tensor z, at::Tensor w1, at::Tensor w2, at::Tensor wn1, at::Tensor wn2, int64_t n_s,
                            at::Tensor err) {
  no_tangents({x, z, w1, w2, wn1, wn2});
  fits(x, n_s, w1, wn1);
  TORCH_CHECK(z.sizes() == x.sizes() && z.scalar_type() == at::kBFloat16 && z.device() == x.device() && w2.dim() == 2 &&
                  w2.size(0) == w1.size(1) && w2.size(1) == w1.size(0) && wn2.dim() == 3 && wn2.size(0) == wn1.size(0) &&
                  wn2.size(1) == w2.size(0) && wn2.size(2) == w2.size(1) && w2.device() == x.device() &&
                  wn2.device() == x.device(),
              "z must be bf16 of x's shape, the second weights [K, F] and [T - n_s, K, F], on one device");
  const c10::DeviceGuard guard(x.device());
  return MixedFFNSaved8::apply(x, z, w1, w2, wn1, wn2, n_s, err);
}
}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.doc() = "primus_dlrm_b200 sm_100a tensor-core kernels";
  m.def("fmha_fwd", &pd::fmha_fwd, py::arg("q"), py::arg("k"), py::arg("v"), py::arg("scale"), py::arg("warps") = 0,
        "pyramid causal attention forward -> (o, lse); warps (d = 32): 4 (64-query CTAs), 8 (128), 0 = default");
  m.def("fmha_fwd_tc", &pd::fmha_fwd_tc, "tcgen05 pyramid causal attention forward from qkv [B,T,3,H,d] -> (o, lse)");
  m.def("fmha_bwd_tc", &pd::fmha_bwd_tc, py::arg("qkv"), py::arg("o"), py::arg("lse"), py::arg("dout"),
        py::arg("dqkv"), py::arg("q_len"), py::arg("scale"), py::arg("err"), py::arg("dbg") = py::none(),
        "tcgen05 attention backward (d=32) into dqkv [B,T,3,H,d]; dbg: optional int64 stage stamps of CTA 0");
  m.def("fmha_bwd_tc_max_q", &pd::fmha_bwd_tc_max_q, "largest q_len the tcgen05 backward supports");
  m.def("fmha_bwd", &pd::fmha_bwd, "pyramid causal attention backward into dq/dk/dv views");
  m.def("tc_gemm", &pd::tc_gemm, py::arg("A"), py::arg("B"), py::arg("C"), py::arg("epi") = 0,
        py::arg("R") = py::none(), py::arg("AUX") = py::none(), py::arg("err"), py::arg("b_kn") = false,
        py::arg("R2") = py::none(),
        "C[l] = epi(A[l] @ B[l]^T) on tcgen05 (A [L,M,K], B [L|1,N,K] or with b_kn [L|1,K,N], C [L,M,N] bf16 views); "
        "epi 0 none, 1 gelu, 2 +R, 3 dgelu(R), 4 gelu+gelu' to AUX, 5 *R, 6 relu(+R), 7 acc where R>0, 8 R*acc+R2");
  m.def("error_word", &pd::gemm_error_word, py::arg("device"), py::arg("which") = 0,
        "the device's int32 error word for the calls that take one: 0 the GEMMs', 1 the attention's");
  m.def("mixed_linear_saved8", &mixed_linear_saved8, "a mixed projection whose input waits for the backward in 8 bits");
  m.def("mixed_ffn_saved8", &mixed_ffn_saved8, "a mixed FFN whose input and pre-activation wait for the backward in 8 bits");
  m.def("tc_wgrad", &pd::tc_wgrad, py::arg("A"), py::arg("B"), py::arg("C"), py::arg("err"), py::arg("l_sum") = false,
        "C[l] (fp32, zeroed) += A[l]^T B[l] over rows on tcgen05, split over rows (A [L,K,M], B [L,K,N] bf16 views); "
        "l_sum: one C summed over the batches too");
  m.def("tc_mma_rate", &pd::tc_mma_rate, py::arg("mode"), py::arg("n"), py::arg("iters"), py::arg("nacc"),
        py::arg("swz"), py::arg("issue"), py::arg("err"),
        "tcgen05.mma probe: int64 [SMs, 2] (issue cycles, issue + execution cycles) for `iters` M=128 x n x 16 "
        "MMAs; mode 0 SS K/K, 1 SS K/MN, 2 SS MN/MN, 3 TS B K-major, 4 TS B MN-major; swz 2 = 128 B, 4 = 64 B; "
        "issue 0 = lone lane, 1 = converged warp + elect.sync, 2 = as 1 with the lane-mask operand form");
  m.def("tc_mma_burst", &pd::tc_mma_burst, py::arg("n"), py::arg("iters"), py::arg("issuers"), py::arg("per_sm"),
        py::arg("ts"), py::arg("wstride"), py::arg("lanes"), py::arg("var"), py::arg("err"),
        "unrolled tcgen05.mma probe: int64 [CTAs, 8] (issue, total cycles per issuing warp) for iters x 16 MMAs; "
        "issuers are warps 0, wstride, 2 wstride, ...; var: 0 fixed operands, 1 B advances, 2 A advances, "
        "3 run-time accumulate flag, 4 not unrolled, 5 = 1 + 2 + 3");
  m.def("launch_count", &pd::launches);
}
