// Host side of the 8-bit integer products (int8_gemm.cuh).
#include "int8_few.cuh"
#include "int8_gemm.cuh"

#include <c10/cuda/CUDAGuard.h>

namespace pd {
namespace i8 {

void quantize_into(const at::Tensor& x, int8_t* codes, int64_t pitch, float* scale);
extern template void product<__nv_bfloat16>(const CUtensorMap&, const void*, int64_t, int64_t, const CUtensorMap&, Params&);
extern template void product<__half>(const CUtensorMap&, const void*, int64_t, int64_t, const CUtensorMap&, Params&);
extern template void product<float>(const CUtensorMap&, const void*, int64_t, int64_t, const CUtensorMap&, Params&);

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

int64_t error_code(int64_t device) {
  const c10::cuda::CUDAGuard guard{c10::DeviceIndex(device)};
  int v = 0;
  PD_CHECK_CUDA(cudaMemcpyFromSymbol(&v, g_err, sizeof(int)));
  return v;
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
  std::vector<int64_t> shape = x.sizes().vec();
  shape.back() = N;
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor y = at::empty(shape, x.options());
  if (K > 1 && x.stride(-1) != 1) x = x.contiguous();
  const int64_t M = x.numel() / (L * K);
  x = x.reshape({M, L, K});
  PD_CHECK(M < (int64_t(1) << 31) && M * L < (int64_t(1) << 40), "int8_linear: too many rows");
  Params p{};
  if (bias) {
    PD_CHECK(bias->device() == x.device() && bias->is_floating_point() && bias->dim() == 1 && bias->size(0) == N,
             "int8_linear: bias must be [N] of a floating type on x's device");
    bias = bias->to(at::kFloat).contiguous();
    p.bias = bias->data_ptr<float>();
  }
  if (residual) {
    PD_CHECK(residual->device() == x.device() && residual->scalar_type() == x.scalar_type() && residual->sizes() == y.sizes(),
             "int8_linear: residual must have the result's shape and x's type, on x's device");
    if (N > 1 && residual->stride(-1) != 1) residual = residual->contiguous();
    residual = residual->reshape({M, L, N});
  }
  if (M == 0) return y;

  const int64_t size = y.element_size();
  const int64_t r_ls = residual && L > 1 ? residual->stride(1) : 0, r_ms = residual && M > 1 ? residual->stride(0) : 0;
  if (M <= kFewRows && few_bytes(M, Kp) <= kFewBytes && L <= 65535) {
    FewParams f{};
    f.M = int(M); f.N = int(N); f.L = int(L); f.K = int(K); f.Kp = int(Kp);
    f.x = x.data_ptr();
    f.x_outer = M > 1 ? x.stride(0) : 0; f.x_inner = L > 1 ? x.stride(1) : 0;
    f.W = codes.data_ptr<int8_t>();
    f.t = scale.data_ptr<float>();
    f.bias = p.bias;
    f.R_ = residual ? residual->data_ptr() : nullptr; f.r_ls = r_ls; f.r_ms = r_ms;
    f.C = y.data_ptr(); f.c_ls = N; f.c_ms = N * L;
    f.act = int(act);
    few(f, dtype, K % 8 == 0 && reinterpret_cast<uintptr_t>(f.x) % 16 == 0 && f.x_outer * size % 16 == 0 &&
                      f.x_inner * size % 16 == 0);
    return y;
  }

  at::Tensor a = at::empty({M * L, Kp}, codes.options());
  at::Tensor s = at::empty({M * L}, scale.options());
  quantize_into(x, a.data_ptr<int8_t>(), Kp, s.data_ptr<float>());

  p.M = int(M); p.N = int(N); p.L = int(L);
  p.m_blocks = int((M + BM - 1) / BM);
  p.k_blocks = int((K + BK - 1) / BK);
  p.s = s.data_ptr<float>(); p.s_ls = 1; p.s_ms = L;
  p.t = scale.data_ptr<float>(); p.t_ls = N;
  p.C = y.data_ptr(); p.c_ls = N; p.c_ms = N * L;
  if (residual) {
    p.R = residual->data_ptr();
    p.r_ls = r_ls; p.r_ms = r_ms;
    p.r_vec = reinterpret_cast<uintptr_t>(p.R) % 16 == 0 && p.r_ls * size % 16 == 0 && p.r_ms * size % 16 == 0;
  }
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
  if (dtype == kv::kBf16) product<__nv_bfloat16>(ta, codes.data_ptr(), Kp, L, tc, p);
  else if (dtype == kv::kF16) product<__half>(ta, codes.data_ptr(), Kp, L, tc, p);
  else product<float>(ta, codes.data_ptr(), Kp, L, tc, p);
  return y;
}

}  // namespace i8
}  // namespace pd
