// Activations to 8-bit integers and back: blocks of 32 values with a
// power-of-two scale (save8 / load8, for training), and whole rows with a
// 32-bit scale (quantize_rows, for integer products).
//
// All are bound by memory. 233,472 x 256 bf16: save8 35 us for 181 MB (5.2 TB/s),
// load8 28 us (6.4 TB/s); 7919 x 1001 fp32, off 16 bytes: 13 and 15 us for 40 MB
// each (byte stores and loads of 32 lanes). quantize_rows: 16,417 x 1024 bf16 12
// us for 50 MB, 16,384 x 256 4 us for 12.6 MB.
#include "int8_common.cuh"
#include "kv_common.cuh"
#include "tc_common.cuh"

#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>

#include <algorithm>
#include <type_traits>

namespace pd {
namespace i8 {

using kv::Raw;

// Eight consecutive values of a row from element k on, zeros behind its end.
template <bool VEC, typename T>
struct Eight {
  Raw<VEC ? 8 : 1, T> r[VEC ? 1 : 8];
  __device__ __forceinline__ void load(const T* row, int64_t k, int64_t K) {
    if constexpr (VEC) {
      if (k < K) r[0].load(row + k); else r[0].zero();
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        if (k + i < K) r[i].load(row + k + i); else r[i].zero();
      }
    }
  }
  __device__ __forceinline__ void floats(float* f) const {
    if constexpr (VEC) {
      r[0].floats(f);
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) r[i].floats(f + i);
    }
  }
};
template <bool VEC>
__device__ __forceinline__ void store_codes(int8_t* row, int64_t k, int64_t K, uint2 c) {
  if constexpr (VEC) {
    if (k < K) *reinterpret_cast<uint2*>(row + k) = c;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (k + i < K) row[k + i] = int8_t(__byte_perm(c.x, c.y, i));
  }
}
__device__ __forceinline__ uint32_t most_bits(const float* f) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) m = max(m, abs_bits(f[i]));
  return m;
}

// save8 and load8. Scale bytes lie block-major ([blocks, rows]): that is how the
// GEMM epilogues, whose threads own rows, write and read them in whole sectors.
// Rows on 16 bytes (VEC): a warp takes 8 rows x 4 blocks at a time; four lanes
// hold a block, so its maximum takes two shuffles, a row's 64 to 128 bytes of a
// load are whole sectors and four loads of a lane are on their way.
// Other rows: a lane is an element, so loads and stores of any alignment are
// whole runs of 32 and the maximum is one warp reduction; 8 blocks on their way.
// Blocks of the grid go over row groups (x) and groups of blocks (y).
constexpr int kRows = 8, kBlocks = 4, kLong = 8;

template <typename T>
__global__ void __launch_bounds__(256) save_kernel(const T* __restrict__ x, int64_t x_stride, int8_t* __restrict__ codes,
                                                   uint8_t* __restrict__ exps, int64_t rows, int K, int blocks,
                                                   uint32_t top) {
  tc::wait_for_launch_before();
  tc::let_next_launch();
  const int lane = threadIdx.x & 31, q = lane & 3;
  for (int64_t r0 = (int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5)) * kRows; r0 < rows; r0 += int64_t(gridDim.x) * 8 * kRows) {
    const int64_t row = r0 + (lane >> 2);
    const bool there = row < rows;
    const T* src = x + (there ? row : 0) * x_stride;
    for (int b0 = blockIdx.y * kBlocks; b0 < blocks; b0 += gridDim.y * kBlocks) {
      Eight<true, T> raw[kBlocks];
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) raw[j].load(src, (b0 + j) * kBlock + q * 8, there ? K : 0);
      uint32_t mine = 0;
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const int k = (b0 + j) * kBlock + q * 8;
        float f[8];
        raw[j].floats(f);
        uint32_t m = most_bits(f);
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 1));
        m = max(m, __shfl_xor_sync(0xffffffffu, m, 2));
        const uint32_t b = scale_byte(m);
        if (q == j) mine = b;
        const float inv = inv_scale(b);
        uint2 c = make_uint2(block_codes4(f, inv), block_codes4(f + 4, inv));
        if (b >= top) {                                   // no numbers, or codes held to 63: rare
          const float most = most_code(b, top);
          c = make_uint2(codes4(f[0], f[1], f[2], f[3], inv, most), codes4(f[4], f[5], f[6], f[7], inv, most));
        }
        if (there && k < K) *reinterpret_cast<uint2*>(codes + row * K + k) = c;
      }
      if (there && b0 + q < blocks) exps[(b0 + q) * rows + row] = uint8_t(mine);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) save_any_kernel(const T* __restrict__ x, int64_t x_stride, int8_t* __restrict__ codes,
                                                       uint8_t* __restrict__ exps, int64_t rows, int K, int blocks,
                                                       uint32_t top) {
  tc::wait_for_launch_before();
  tc::let_next_launch();
  const int lane = threadIdx.x & 31;
  for (int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); row < rows; row += int64_t(gridDim.x) * 8) {
    const T* src = x + row * x_stride;
    for (int b0 = blockIdx.y * kLong; b0 < blocks; b0 += gridDim.y * kLong) {
      float f[kLong];
#pragma unroll
      for (int j = 0; j < kLong; ++j) {
        const int k = (b0 + j) * kBlock + lane;
        f[j] = k < K ? kv::to_f(src[k]) : 0.0f;
      }
      uint32_t mine = 0;
#pragma unroll
      for (int j = 0; j < kLong; ++j) {
        const int k = (b0 + j) * kBlock + lane;
        const uint32_t b = scale_byte(__reduce_max_sync(0xffffffffu, abs_bits(f[j])));
        if (lane == j) mine = b;
        uint32_t c = __float_as_uint(fmaf(f[j], inv_scale(b), 12582912.0f));       // the low byte, as in block_codes4
        if (b >= top) c = codes4(f[j], 0.0f, 0.0f, 0.0f, inv_scale(b), most_code(b, top));
        if (k < K) codes[row * K + k] = int8_t(c);
      }
      if (lane < kLong && b0 + lane < blocks) exps[(b0 + lane) * rows + row] = uint8_t(mine);
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) load_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                   T* __restrict__ y, int64_t rows, int K, int blocks) {
  tc::wait_for_launch_before();
  tc::let_next_launch();
  const int lane = threadIdx.x & 31, q = lane & 3;
  for (int64_t r0 = (int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5)) * kRows; r0 < rows; r0 += int64_t(gridDim.x) * 8 * kRows) {
    const int64_t row = r0 + (lane >> 2);
    if (row >= rows) continue;
    for (int b0 = blockIdx.y * kBlocks; b0 < blocks; b0 += gridDim.y * kBlocks) {
      uint2 c[kBlocks];
      uint32_t e[kBlocks];
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const int k = (b0 + j) * kBlock + q * 8;
        c[j] = k < K ? *reinterpret_cast<const uint2*>(codes + row * K + k) : make_uint2(0, 0);
        e[j] = b0 + j < blocks ? exps[(b0 + j) * rows + row] : 1;
      }
#pragma unroll
      for (int j = 0; j < kBlocks; ++j) {
        const int k = (b0 + j) * kBlock + q * 8;
        float f[8];
        const float s = scale_of(e[j]);
        values4(c[j].x, s, f);
        values4(c[j].y, s, f + 4);
        if (k < K) kv::store_v<8, T>(y + row * K + k, f);
      }
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(256) load_any_kernel(const int8_t* __restrict__ codes, const uint8_t* __restrict__ exps,
                                                       T* __restrict__ y, int64_t rows, int K, int blocks) {
  tc::wait_for_launch_before();
  tc::let_next_launch();
  const int lane = threadIdx.x & 31;
  for (int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); row < rows; row += int64_t(gridDim.x) * 8) {
    for (int b0 = blockIdx.y * kLong; b0 < blocks; b0 += gridDim.y * kLong) {
      int c[kLong];
      uint32_t e[kLong];
#pragma unroll
      for (int j = 0; j < kLong; ++j) {
        const int k = (b0 + j) * kBlock + lane;
        c[j] = k < K ? codes[row * K + k] : 0;
        e[j] = b0 + j < blocks ? exps[(b0 + j) * rows + row] : 1;
      }
#pragma unroll
      for (int j = 0; j < kLong; ++j) {
        const int k = (b0 + j) * kBlock + lane;
        if (k < K) y[row * K + k] = kv::from_f<T>(float(c[j]) * scale_of(e[j]));
      }
    }
  }
}

// quantize_rows: TPR threads share a row and keep it in registers between the
// maximum and the codes (NV vectors of 8 a thread, so that a row's loads are all
// on their way at once); longer rows are read again. Codes lie in rows of `pitch`
// bytes, zeros behind a row's end.
template <bool VEC, int TPR, int NV, typename T>
__global__ void __launch_bounds__(256) rows_kernel(const T* __restrict__ x, int64_t x_outer, int64_t x_inner, int inner,
                                                   int8_t* __restrict__ codes, int64_t pitch, float* __restrict__ scale,
                                                   int64_t rows, int K) {
  constexpr int kPer = 256 / TPR;
  __shared__ uint32_t s_most[8];
  tc::let_next_launch();                                   // the product may set itself up while this runs
  const int part = threadIdx.x % TPR;
  for (int64_t r0 = int64_t(blockIdx.x) * kPer; r0 < rows; r0 += int64_t(gridDim.x) * kPer) {
    const int64_t row = r0 + threadIdx.x / TPR;
    const bool there = row < rows;
    const T* src = x;
    if (there) src += inner == 1 ? row * x_outer : row / inner * x_outer + row % inner * x_inner;
    Eight<VEC, T> raw[NV];
    uint32_t m = 0;
    const int len = there ? K : 0;
#pragma unroll
    for (int i = 0; i < NV; ++i) raw[i].load(src, (i * TPR + part) * 8, len);
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8];
      raw[i].floats(f);
      m = max(m, most_bits(f));
    }
    for (int k = NV * TPR * 8 + part * 8; k < len; k += TPR * 8) {
      Eight<VEC, T> e;
      float f[8];
      e.load(src, k, len);
      e.floats(f);
      m = max(m, most_bits(f));
    }
    if constexpr (TPR < 32) {
#pragma unroll
      for (int o = TPR / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
    } else {
      m = __reduce_max_sync(0xffffffffu, m);
    }
    if constexpr (TPR > 32) {
      __syncthreads();                                     // the row before has been read out of s_most
      if ((threadIdx.x & 31) == 0) s_most[threadIdx.x >> 5] = m;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < TPR / 32; ++w) m = max(m, s_most[threadIdx.x / TPR * (TPR / 32) + w]);
    }
    const RowScale sc = row_scale(m);
    if (!there) continue;
    if (part == 0) scale[row] = sc.scale;
    int8_t* dst = codes + row * pitch;
    auto put = [&](const float* f, int k) {
      store_codes<VEC>(dst, k, pitch, make_uint2(codes4(f[0], f[1], f[2], f[3], sc.inv, sc.most),
                                                 codes4(f[4], f[5], f[6], f[7], sc.inv, sc.most)));
    };
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float f[8];
      raw[i].floats(f);
      put(f, (i * TPR + part) * 8);
    }
    for (int k = NV * TPR * 8 + part * 8; k < pitch; k += TPR * 8) {
      Eight<VEC, T> e;
      float f[8];
      e.load(src, k, len);
      e.floats(f);
      put(f, k);
    }
  }
}

// A lane an element, for rows of any alignment: whole runs of 32 values a load, 8 of them on their way.
template <typename T>
__global__ void __launch_bounds__(256) rows_any_kernel(const T* __restrict__ x, int64_t x_outer, int64_t x_inner, int inner,
                                                       int8_t* __restrict__ codes, int64_t pitch, float* __restrict__ scale,
                                                       int64_t rows, int K) {
  constexpr int kAhead = 16;
  const int lane = threadIdx.x & 31;
  tc::let_next_launch();
  for (int64_t row = int64_t(blockIdx.x) * 8 + (threadIdx.x >> 5); row < rows; row += int64_t(gridDim.x) * 8) {
    const T* src = x + (inner == 1 ? row * x_outer : row / inner * x_outer + row % inner * x_inner);
    float f[kAhead];
    float m = 0.0f;
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = j * 32 + lane;
      f[j] = k < K ? kv::to_f(src[k]) : 0.0f;
    }
#pragma unroll
    for (int j = 0; j < kAhead; j += 2) m = max_abs3(m, f[j], f[j + 1]);
    for (int k = kAhead * 32 + lane; k < K; k += 32) m = max_abs3(m, kv::to_f(src[k]), 0.0f);
    const RowScale sc = row_scale(__reduce_max_sync(0xffffffffu, abs_bits(m)));
    if (lane == 0) scale[row] = sc.scale;
    int8_t* dst = codes + row * pitch;
    auto code = [&](float v) { return int8_t(codes4(v, 0.0f, 0.0f, 0.0f, sc.inv, sc.most)); };
#pragma unroll
    for (int j = 0; j < kAhead; ++j) {
      const int k = j * 32 + lane;
      if (k < pitch) dst[k] = code(f[j]);
    }
    for (int64_t k = kAhead * 32 + lane; k < pitch; k += 32) dst[k] = k < K ? code(kv::to_f(src[k])) : int8_t(0);
  }
}

// ---------------------------------------------------------------------------
namespace {

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

int grid_for(int64_t work, int per_sm) {
  return int(std::max<int64_t>(1, std::min<int64_t>(work, int64_t(num_sms()) * per_sm)));
}

// Blocks of 256 threads for row groups and, where those are few, for groups of blocks along a row too.
dim3 pack_grid(int64_t row_groups, int64_t block_groups) {
  const int64_t x = std::min<int64_t>(std::max<int64_t>(row_groups, 1), int64_t(num_sms()) * 8);
  const int64_t y = std::min<int64_t>(block_groups, std::max<int64_t>(1, int64_t(num_sms()) * 8 / x));
  return dim3(unsigned(x), unsigned(std::min<int64_t>(y, 65535)));
}

template <typename F>
void by_type(int dtype, F&& f) {
  if (dtype == kv::kBf16) f(static_cast<__nv_bfloat16*>(nullptr));
  else if (dtype == kv::kF16) f(static_cast<__half*>(nullptr));
  else f(static_cast<float*>(nullptr));
}

}  // namespace

// x [..., K] -> codes [rows, K], scale bytes [blocks, rows]
std::vector<at::Tensor> save8(at::Tensor x) {
  PD_CHECK(x.is_cuda() && x.dim() >= 1, "save8: a CUDA tensor with a last dim is expected");
  const int dtype = kv::dtype_of(x, "save8");
  const c10::cuda::CUDAGuard guard(x.device());
  const int64_t K = x.size(-1);
  int64_t rows = 1;
  for (int64_t d = 0; d + 1 < x.dim(); ++d) rows *= x.size(d);
  const int64_t blocks = (K + kBlock - 1) / kBlock;
  at::Tensor codes = at::detail::empty_cuda({rows, K}, at::kChar, x.device(), c10::nullopt);
  at::Tensor exps = at::detail::empty_cuda({blocks, rows}, at::kByte, x.device(), c10::nullopt);
  if (rows == 0 || K == 0) return {codes, exps};
  if (K > 1 && x.stride(-1) != 1) x = x.contiguous();
  if (x.dim() > 2 && !x.is_contiguous()) x = x.reshape({rows, K});
  const int64_t row_stride = x.dim() == 2 ? x.stride(0) : K;
  PD_CHECK(K < (int64_t(1) << 30), "save8: rows of fewer than 2^30 values are expected");
  by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const T* p = static_cast<const T*>(x.data_ptr());
    const int64_t stride = rows == 1 ? K : row_stride;
    const uint32_t top = dtype == kv::kF16 ? kTopHalf : kTopWide;
    const bool vec = K % 8 == 0 && aligned16(p) && stride * int64_t(sizeof(T)) % 16 == 0;
    if (vec)
      tc::launch_behind(save_kernel<T>, pack_grid((rows + 8 * kRows - 1) / (8 * kRows), (blocks + kBlocks - 1) / kBlocks), 256, 0,
                        p, stride, codes.data_ptr<int8_t>(), exps.data_ptr<uint8_t>(), rows, int(K), int(blocks), top);
    else
      tc::launch_behind(save_any_kernel<T>, pack_grid((rows + 7) / 8, (blocks + kLong - 1) / kLong), 256, 0,
                        p, stride, codes.data_ptr<int8_t>(), exps.data_ptr<uint8_t>(), rows, int(K), int(blocks), top);
  });
  return {codes, exps};
}

at::Tensor load8(at::Tensor codes, at::Tensor exps, int64_t dtype) {
  PD_CHECK(codes.is_cuda() && codes.dim() == 2 && codes.scalar_type() == at::kChar && codes.is_contiguous(),
           "load8: contiguous int8 codes [rows, K] are expected");
  const int64_t rows = codes.size(0), K = codes.size(1), blocks = (K + kBlock - 1) / kBlock;
  PD_CHECK(exps.is_cuda() && exps.device() == codes.device() && exps.scalar_type() == at::kByte && exps.is_contiguous() &&
               exps.dim() == 2 && exps.size(0) == blocks && exps.size(1) == rows,
           "load8: contiguous uint8 scale bytes [blocks, rows] are expected");
  const c10::cuda::CUDAGuard guard(codes.device());
  at::Tensor y = at::detail::empty_cuda({rows, K}, at::ScalarType(dtype), codes.device(), c10::nullopt);
  const int t = kv::dtype_of(y, "load8");
  if (rows == 0 || K == 0) return y;
  PD_CHECK(K < (int64_t(1) << 30), "load8: rows of fewer than 2^30 values are expected");
  by_type(t, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    T* out = static_cast<T*>(y.data_ptr());
    if (K % 8 == 0 && aligned16(codes.data_ptr()))
      tc::launch_behind(load_kernel<T>, pack_grid((rows + 8 * kRows - 1) / (8 * kRows), (blocks + kBlocks - 1) / kBlocks), 256, 0,
                        codes.data_ptr<int8_t>(), exps.data_ptr<uint8_t>(), out, rows, int(K), int(blocks));
    else
      tc::launch_behind(load_any_kernel<T>, pack_grid((rows + 7) / 8, (blocks + kLong - 1) / kLong), 256, 0,
                        codes.data_ptr<int8_t>(), exps.data_ptr<uint8_t>(), out, rows, int(K), int(blocks));
  });
  return y;
}

// Rows of x (row `i` of position `l` at x + i * so + l * si elements) into codes (rows of `pitch` bytes) and scales, both in
// the order [outer, inner].
void quantize_into(const void* x, int dtype, int64_t outer, int64_t inner, int64_t K, int64_t so, int64_t si, int8_t* codes,
                   int64_t pitch, float* scale) {
  const int64_t rows = outer * inner;
  if (rows == 0) return;
  by_type(dtype, [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    const T* p = static_cast<const T*>(x);
    const bool vec = K % 8 == 0 && pitch % 8 == 0 && aligned16(p) && so * int64_t(sizeof(T)) % 16 == 0 &&
                     si * int64_t(sizeof(T)) % 16 == 0;
    auto go = [&](auto* kern, int per_block) {
      kern<<<grid_for((rows + per_block - 1) / per_block, 8), 256, 0, stream()>>>(p, so, si, int(inner), codes, pitch, scale,
                                                                                rows, int(K));
      PD_CHECK_LAUNCH();
    };
    // few rows: a block for each, so that a row's reads are spread over threads (rows of 1024: 64 1.8 us against 2.2 by
    // warps, 300 2.0 and 2.2, 1000 2.8 and 2.2)
    const bool few = rows < 512;
    if (!vec) {
      if (few && K > 512) go(rows_kernel<false, 256, 1, T>, 1);
      else go(rows_any_kernel<T>, 8);
    } else if (few && K > 256) {
      if (K <= 2048) go(rows_kernel<true, 256, 1, T>, 1);
      else go(rows_kernel<true, 256, 2, T>, 1);
    } else if (K <= 256) {
      go(rows_kernel<true, 8, 4, T>, 32);
    } else if (K <= 512) {
      go(rows_kernel<true, 16, 4, T>, 16);
    } else if (K <= 1024) {
      go(rows_kernel<true, 32, 4, T>, 8);
    } else {
      go(rows_kernel<true, 256, 2, T>, 1);
    }
  });
}

std::vector<at::Tensor> quantize_rows(at::Tensor x) {
  PD_CHECK(x.is_cuda() && x.dim() == 3, "quantize_rows: a CUDA tensor [outer, inner, K] is expected");
  kv::dtype_of(x, "quantize_rows");
  PD_CHECK(x.size(2) <= 1 || x.stride(2) == 1, "quantize_rows: unit stride over the last dim is expected");
  PD_CHECK(x.size(1) < (int64_t(1) << 31) && x.size(2) < (int64_t(1) << 30), "quantize_rows: rows of fewer than 2^30 values are expected");
  const c10::cuda::CUDAGuard guard(x.device());
  at::Tensor codes = at::empty(x.sizes(), x.options().dtype(at::kChar));
  at::Tensor scale = at::empty({x.size(0), x.size(1)}, x.options().dtype(at::kFloat));
  quantize_into(x.data_ptr(), kv::dtype_of(x, "quantize_rows"), x.size(0), x.size(1), x.size(2),
                x.size(0) > 1 ? x.stride(0) : 0, x.size(1) > 1 ? x.stride(1) : 0, codes.data_ptr<int8_t>(), x.size(2),
                scale.data_ptr<float>());
  return {codes, scale};
}

}  // namespace i8

long long launches() { return launch_counter().load(); }

}  // namespace pd
