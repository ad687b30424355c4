// Launch counter and error words of the _gemm extension.
#include "common.cuh"

#include <c10/cuda/CUDAGuard.h>

namespace pd {

// 2: a bounded wait ran out, 3: a shape or an alignment that a kernel cannot run (ErrorCode). [0] the GEMMs', [1] the
// attention's.
__device__ int g_gemm_err[2];

at::Tensor gemm_error_word(int64_t device, int64_t which) {
  PD_CHECK(which == 0 || which == 1, "no such error word");
  const c10::cuda::CUDAGuard guard{c10::DeviceIndex(device)};
  int* word = nullptr;
  PD_CHECK_CUDA(cudaGetSymbolAddress(reinterpret_cast<void**>(&word), g_gemm_err));
  return word_tensor(word + which, device);
}

long long launches() { return launch_counter().load(); }

}  // namespace pd
