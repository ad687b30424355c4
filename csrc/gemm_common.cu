// Launch counter and error word of the _gemm extension.
#include "common.cuh"

#include <c10/cuda/CUDAGuard.h>

namespace pd {

// 2: a bounded wait ran out, 3: a shape or an alignment that a kernel cannot run (ErrorCode).
__device__ int g_gemm_err;

at::Tensor gemm_error_word(int64_t device) {
  const c10::cuda::CUDAGuard guard{c10::DeviceIndex(device)};
  int* word = nullptr;
  PD_CHECK_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&word), g_gemm_err));
  return word_tensor(word, device);
}

long long launches() { return launch_counter().load(); }

}  // namespace pd
