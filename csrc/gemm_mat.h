// Operands of the layers that keep their activations in 8 bits, as the kernels
// take them (no tensor is made for a view: a step has some thirty of them).
#pragma once

#include <cstdint>

namespace pd {

// A [L, rows, cols] matrix: unit stride over cols, `ms` elements from row to row, `ls` from batch to batch.
struct Mat {
  void* p;
  int64_t L, rows, cols, ls, ms;
};

// Codes of a [L, rows, cols] matrix and their scale bytes [L, rows, cols / 32].
struct MatCodes {
  int8_t* codes;
  int64_t ls, ms;
  uint8_t* bytes;
  int64_t e_ls, e_ms, e_bs;
};

}  // namespace pd
