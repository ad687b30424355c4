// The 8-bit integer products with results of this type.
#include "int8_gemm.cuh"

namespace pd {
namespace i8 {
template void product<float>(const CUtensorMap&, const void*, int64_t, int64_t, const CUtensorMap&, Params&, at::Device);
}  // namespace i8
}  // namespace pd
