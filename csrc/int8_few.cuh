// The integer product of up to 16 rows in one launch (int8_few.cu).
#pragma once

#include <atomic>
#include <type_traits>

#include "int8_common.cuh"

namespace pd {
namespace i8 {

struct FewParams {
  int M, N, L, K, Kp;
  const void* x; int64_t x_outer, x_inner;               // row m of position l: x + m * x_outer + l * x_inner
  const int8_t* W;                                        // [L, N, Kp], rows on 16 bytes
  const float* t;                                         // [L, N]
  const float* bias;
  const void* R_; int64_t r_ls, r_ms;
  void* C; int64_t c_ls, c_ms;
  int act;
  int R, pitch;                                           // rows of codes (a power of two) and their pitch, set by few()
};

constexpr int kFewRows = 16;
constexpr int kFewBytes = 192 * 1024;                     // of codes in shared memory at most

// Whole steps of 64 bytes; 64 over a multiple of 128, so that two rows of 64 bytes fall on different banks.
inline int64_t few_pitch(int64_t Kp) { return (Kp + 127) / 128 * 128 + 64; }
int64_t few_bytes(int64_t M, int64_t Kp);
void few(FewParams p, int dtype, bool vec);

}  // namespace i8
}  // namespace pd
