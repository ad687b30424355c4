// Host side of the 8-bit integer products (int8_gemm.cuh).
#include "int8_few.cuh"
#include "int8_gemm.cuh"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/util/SmallVector.h>

namespace pd {
namespace i8 {

void quantize_into(const void* x, int dtype, int64_t outer, int64_t inner, int64_t K, int64_t so, int64_t si, int8_t* codes,
                   int64_t pitch, float* scale);
extern template void product<__nv_bfloat16>(const CUtensorMap&, const void*, int64_t, int64_t, const CUtensorMap&, Params&, at::Device);
extern template void product<__half>(const CUtensorMap&, const void*, int64_t, int64_t, const CUtensorMap&, Params&, at::Device);
extern template void product<float>(const CUtensorMap&, const void*, int64_t, int64_t, const CUtensorMap&, Params&, at::Device);

// The kernels' error word on each device: 2 a bounded wait ran out, 4 shared memory not aligned.
__device__ int g_err;

static int* error_word() {
  static std::atomic<int*> words[64];
  int dev = 0;
  PD_CHECK_CUDA(cudaGetDevice(&dev));
  int* w = words[dev & 63].load(std::memory_order_relaxed);
  if (w == nullptr) {
    PD_CHECK_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&w), g_err));
    words[dev & 63].store(w, std::memory_order_relaxed);
  }
  return w;
}

at::Tensor error_tensor(int64_t device) {
  const c10::cuda::CUDAGuard guard{c10::DeviceIndex(device)};
  return word_tensor(error_word(), device);
}

// Rows of a [..., K] tensor (or [..., L, K]) as they lie: row m of position l at `at` + m * outer + l * inner elements.
struct Rows {
  const void* at;
  int64_t outer, inner;
  at::Tensor held;                                        // where they had to be laid out anew
};
static Rows rows_of(at::Tensor t, int64_t M, int64_t L, int64_t K, bool grouped) {
  if (K > 1 && t.stride(-1) != 1) t = t.contiguous();
  const int64_t lead = t.dim() - (grouped ? 2 : 1);       // dims over rows
  if (lead > 1 && !t.is_contiguous()) t = t.reshape({M, L, K});
  const bool plain = lead > 1 && t.is_contiguous();       // the rows follow one another
  Rows r{t.data_ptr(), 0, 0, t};
  if (M > 1) r.outer = plain ? L * K : t.stride(0);
  if (L > 1) r.inner = plain ? K : t.stride(-2);
  return r;
}

// x [..., K] or, with a matrix for each of L positions, [..., L, K], by codes [L, N, Kp] (contiguous, zeros from K on)
// with scales [L, N] -> y [..., N] of x's type.
at::Tensor linear(at::Tensor x, at::Tensor codes, at::Tensor scale, int64_t K, bool grouped, c10::optional<at::Tensor> bias,
                  int64_t act, c10::optional<at::Tensor> residual) {
  PD_CHECK(x.is_cuda(), "int8_linear: x must be a CUDA tensor");
  const int dtype = kv::dtype_of(x, "int8_linear");
  PD_CHECK(codes.dim() == 3 && codes.scalar_type() == at::kChar && codes.is_contiguous() && scale.dim() == 2 &&
               scale.scalar_type() == at::kFloat && scale.is_contiguous() && scale.size(0) == codes.size(0) &&
               scale.size(1) == codes.size(1) && (grouped || codes.size(0) == 1) && act >= kIdentity && act <= kRelu,
           "int8_linear: a weight laid out by Int8Weight is expected");
  PD_CHECK(reinterpret_cast<uintptr_t>(codes.data_ptr()) % 16 == 0, "int8_linear: a weight's codes must lie on 16 bytes");
  PD_CHECK(codes.device() == x.device() && scale.device() == x.device(), "int8_linear: x and the weight lie on two devices");
  const int64_t L = codes.size(0), N = codes.size(1), Kp = codes.size(2);
  PD_CHECK(Kp % 16 == 0 && K <= Kp && K >= 1 && N >= 1 && N < (int64_t(1) << 31) && K <= 131072,
           "int8_linear: 1 to 131072 input features are expected");
  PD_CHECK(x.dim() >= (grouped ? 2 : 1) && x.size(-1) == K && (!grouped || x.size(-2) == L),
           "int8_linear: x does not fit the weight (its last dim is %lld, the weight takes %lld%s)",
           x.dim() ? (long long)x.size(-1) : -1, (long long)K, grouped ? " for each of its positions" : "");
  const c10::cuda::CUDAGuard guard(x.device());
  c10::SmallVector<int64_t, 5> shape(x.sizes().begin(), x.sizes().end());
  shape.back() = N;
  at::Tensor y = at::detail::empty_cuda(shape, x.scalar_type(), x.device(), c10::nullopt);
  const int64_t M = x.numel() / (L * K);
  PD_CHECK(M < (int64_t(1) << 31) && M * L < (int64_t(1) << 40), "int8_linear: too many rows");
  const Rows xr = rows_of(x, M, L, K, grouped);
  Params p{};
  Rows rr{};
  if (bias) {
    PD_CHECK(bias->device() == x.device() && bias->is_floating_point() && bias->dim() == 1 && bias->size(0) == N,
             "int8_linear: bias must be [N] of a floating type on x's device");
    if (bias->scalar_type() != at::kFloat || !bias->is_contiguous()) bias = bias->to(at::kFloat).contiguous();
    p.bias = bias->data_ptr<float>();
  }
  if (residual) {
    PD_CHECK(residual->device() == x.device() && residual->scalar_type() == x.scalar_type() && residual->sizes() == y.sizes(),
             "int8_linear: residual must have the result's shape and x's type, on x's device");
    rr = rows_of(*residual, M, L, N, grouped);
  }
  if (M == 0) return y;

  const int64_t size = y.element_size();
  if (M <= kFewRows && few_bytes(M, Kp) <= kFewBytes && L <= 65535) {
    FewParams f{};
    f.M = int(M); f.N = int(N); f.L = int(L); f.K = int(K); f.Kp = int(Kp);
    f.x = xr.at; f.x_outer = xr.outer; f.x_inner = xr.inner;
    f.W = codes.data_ptr<int8_t>();
    f.t = scale.data_ptr<float>();
    f.bias = p.bias;
    f.R_ = rr.at; f.r_ls = rr.inner; f.r_ms = rr.outer;
    f.C = y.data_ptr(); f.c_ls = N; f.c_ms = N * L;
    f.act = int(act);
    few(f, dtype, K % 8 == 0 && reinterpret_cast<uintptr_t>(f.x) % 16 == 0 && f.x_outer * size % 16 == 0 &&
                      f.x_inner * size % 16 == 0);
    return y;
  }

  at::Tensor a = at::detail::empty_cuda({M * L, Kp}, at::kChar, x.device(), c10::nullopt);
  at::Tensor s = at::detail::empty_cuda({M * L}, at::kFloat, x.device(), c10::nullopt);
  quantize_into(xr.at, dtype, M, L, K, xr.outer, xr.inner, a.data_ptr<int8_t>(), Kp, s.data_ptr<float>());

  p.M = int(M); p.N = int(N); p.L = int(L);
  p.m_blocks = int((M + BM - 1) / BM);
  p.k_blocks = int((K + BK - 1) / BK);
  p.s = s.data_ptr<float>(); p.s_ls = 1; p.s_ms = L;
  p.t = scale.data_ptr<float>(); p.t_ls = N;
  p.C = y.data_ptr(); p.c_ls = N; p.c_ms = N * L;
  p.R = rr.at; p.r_ls = rr.inner; p.r_ms = rr.outer;
  p.r_vec = reinterpret_cast<uintptr_t>(p.R) % 16 == 0 && p.r_ls * size % 16 == 0 && p.r_ms * size % 16 == 0;
  p.act = int(act);
  p.err = error_word();
  const CUtensorMap ta = map_of(CU_TENSOR_MAP_DATA_TYPE_UINT8, a.data_ptr(), Kp, M, L, Kp * L, Kp, BK, BM,
                                CU_TENSOR_MAP_SWIZZLE_128B, p.a_mode);
  p.c_tma = N * size % 16 == 0;
  CUtensorMap tc = ta;
  if (p.c_tma)
    tc = map_of(dtype == kv::kF32 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : dtype == kv::kF16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                                       : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
                p.C, N, M, L, N * L * size, N * size, 32, 32,
                size == 2 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, p.c_mode);
  p.b_shared = L == 1;
  if (dtype == kv::kBf16) product<__nv_bfloat16>(ta, codes.data_ptr(), Kp, L, tc, p, x.device());
  else if (dtype == kv::kF16) product<__half>(ta, codes.data_ptr(), Kp, L, tc, p, x.device());
  else product<float>(ta, codes.data_ptr(), Kp, L, tc, p, x.device());
  return y;
}

}  // namespace i8
}  // namespace pd
