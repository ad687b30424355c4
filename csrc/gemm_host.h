// Checks and tensor maps of the GEMMs' operands (host side).
#pragma once

#include "common.cuh"
#include "driver_api.h"

namespace pd {

// 3-D tensor map over bf16 rows of length K (strides in elements).  mode 0:
// dims {K, rows, L}; mode 1 (batch stride smaller than the row stride, e.g.
// one batch per NS token): dims {K, L, rows} so the strides stay ascending.
// Preconditions of cuTensorMapEncodeTiled checked on the host, so a bad view
// fails with a message instead of reaching the driver: 16-byte aligned base,
// extents in [1, 2^32), strides multiples of 16 bytes below 2^40, boxes of
// 1..256 elements.
inline void check_encode(const void* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box,
                  int rank, const char* what) {
  PD_CHECK(reinterpret_cast<uintptr_t>(base) % 16 == 0, "%s: base address not 16-byte aligned", what);
  for (int i = 0; i < rank; ++i) {
    PD_CHECK(dims[i] >= 1 && dims[i] < (cuuint64_t(1) << 32), "%s: extent %d out of range (%llu)", what, i,
             (unsigned long long)dims[i]);
    PD_CHECK(box[i] >= 1 && box[i] <= 256, "%s: box %d out of range (%u)", what, i, (unsigned)box[i]);
  }
  for (int i = 0; i + 1 < rank; ++i)
    PD_CHECK(strides[i] % 16 == 0 && strides[i] > 0 && strides[i] < (cuuint64_t(1) << 40),
             "%s: stride %d (%llu bytes) must be a positive multiple of 16 below 2^40", what, i,
             (unsigned long long)strides[i]);
}

// Every element a [L, rows, K] view addresses lies inside its storage (a TMA
// map of a view reaching past its allocation would read or write memory that
// is not the tensor's).
inline void check_extent(const at::Tensor& t, const char* name) {
  if (t.numel() == 0) return;
  int64_t last = t.storage_offset();
  for (int64_t d = 0; d < t.dim(); ++d) {
    PD_CHECK(t.stride(d) >= 0, "%s: negative strides are not supported", name);
    last += (t.size(d) - 1) * t.stride(d);
  }
  PD_CHECK(int64_t((last + 1) * t.element_size()) <= int64_t(t.storage().nbytes()),
           "%s: the view reaches past the end of its storage", name);
}

inline CUtensorMap make_map(const void* base, int64_t K, int64_t rows, int64_t L, int64_t row_stride, int64_t l_stride,
                     int box_rows, int& mode) {
  CUtensorMap m;
  if (L <= 1) l_stride = row_stride * rows;
  mode = (L > 1 && l_stride < row_stride) ? 1 : 0;
  cuuint64_t dims[3], strides[2];
  cuuint32_t box[3];
  if (mode == 0) {
    dims[0] = K; dims[1] = rows; dims[2] = L;
    strides[0] = row_stride * 2; strides[1] = l_stride * 2;
    box[0] = 64; box[1] = box_rows; box[2] = 1;
  } else {
    dims[0] = K; dims[1] = L; dims[2] = rows;
    strides[0] = l_stride * 2; strides[1] = row_stride * 2;
    box[0] = 64; box[1] = 1; box[2] = box_rows;
  }
  cuuint32_t estr[3] = {1, 1, 1};
  check_encode(base, dims, strides, box, 3, "operand map");
  CUresult r = tensor_map_encode_tiled(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides,
                                      box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  PD_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d): K=%lld rows=%lld L=%lld row_stride=%lld l_stride=%lld",
           int(r), (long long)K, (long long)rows, (long long)L, (long long)row_stride, (long long)l_stride);
  return m;
}

// Map of a [L, rows, N] bf16 epilogue operand (C / AUX stores, R loads):
// 32 x 32 boxes, 64-byte swizzle (the epilogue's staging layout); dim order
// as in make_map.
inline CUtensorMap make_store_map(const void* base, int64_t N, int64_t rows, int64_t L, int64_t row_stride,
                           int64_t l_stride, int& mode) {
  CUtensorMap m;
  if (L <= 1) l_stride = row_stride * rows;
  mode = (L > 1 && l_stride < row_stride) ? 1 : 0;
  cuuint64_t dims[3], strides[2];
  cuuint32_t box[3];
  if (mode == 0) {
    dims[0] = N; dims[1] = rows; dims[2] = L;
    strides[0] = row_stride * 2; strides[1] = l_stride * 2;
    box[0] = 32; box[1] = 32; box[2] = 1;
  } else {
    dims[0] = N; dims[1] = L; dims[2] = rows;
    strides[0] = l_stride * 2; strides[1] = row_stride * 2;
    box[0] = 32; box[1] = 1; box[2] = 32;
  }
  cuuint32_t estr[3] = {1, 1, 1};
  check_encode(base, dims, strides, box, 3, "epilogue map");
  CUresult r = tensor_map_encode_tiled(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides,
                                      box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_64B,
                                      CU_TENSOR_MAP_L2_PROMOTION_NONE, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  PD_CHECK(r == CUDA_SUCCESS,
           "cuTensorMapEncodeTiled (store) failed (%d): N=%lld rows=%lld L=%lld row_stride=%lld l_stride=%lld",
           int(r), (long long)N, (long long)rows, (long long)L, (long long)row_stride, (long long)l_stride);
  return m;
}

// [L, rows, K] view (L may be 1): unit stride on K, 16-byte aligned rows.
inline void check_operand(const at::Tensor& t, const char* name) {
  PD_CHECK(t.is_cuda() && t.scalar_type() == at::kBFloat16, "%s: bf16 CUDA tensor required", name);
  PD_CHECK(t.dim() == 3 && t.stride(2) == 1, "%s: [L, rows, K] with unit stride on K required", name);
  PD_CHECK(t.stride(1) % 8 == 0 && (t.size(0) == 1 || t.stride(0) % 8 == 0) &&
              reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0, "%s: rows must be 16-byte aligned", name);
  PD_CHECK(t.size(2) % 8 == 0, "%s: K must be a multiple of 8", name);
  check_extent(t, name);
}

}  // namespace pd
