// Products of 8-bit integers for up to 16 rows (a token of a few users): one
// launch that turns the rows into codes and multiplies.
//
// Such a call reads the weight once and is bound by latency: a launch less, the
// weight's loads on their way while the rows are still being turned into codes,
// and the long axis split over a block's eight warps. A block owns 8 T output
// columns; every block makes the rows' codes for itself (up to 16 x K values out
// of L2), in shared memory. Products by mma.m16n8k32 on 8-bit integers: tcgen05
// would multiply 128 rows, 112 of them empty, behind a TMEM allocation and three
// barriers. The instruction's k index is permuted alike in both operands, so that
// a lane's 16 bytes of a weight row are one load.
//
// Measured (1 B200): 1 x 1024 -> 4096 3.5 us on the device (4.2 MB; 0.65 us at the
// memory's rate), 16 x 256 -> 768 3.4; a call takes 5.6, its host time (12.3 and
// 12.1 as codes and a tcgen05 product).
#include "int8_common.cuh"
#include "int8_few.cuh"
#include "kv_common.cuh"

namespace pd {
namespace i8 {

constexpr int kWarps = 8;

template <typename T, bool VEC>
__device__ __forceinline__ void eight(const T* row, int k, int K, float* f) {
  if constexpr (VEC) {
    kv::Raw<8, T> r;
    if (k < K) r.load(row + k); else r.zero();
    r.floats(f);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = k + i < K ? kv::to_f(row[k + i]) : 0.0f;
  }
}

__device__ __forceinline__ void mma_s8(int (&c)[4], const uint32_t a0, const uint32_t a1, const uint32_t a2, const uint32_t a3,
                                       const uint32_t b0, const uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
               : "+r"(c[0]), "+r"(c[1]), "+r"(c[2]), "+r"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// T8: tiles of 8 columns a block; kAhead steps of 64 bytes of K are loaded at a time
template <typename T, bool VEC, int T8>
__global__ void __launch_bounds__(32 * kWarps) few_kernel(const FewParams p) {
  constexpr int kAhead = 8 / T8, kCols = 8 * T8;
  extern __shared__ __align__(16) uint8_t codes[];        // [16 rows][pitch]
  __shared__ int s_sum[kWarps][16][kCols + 2];
  __shared__ uint32_t s_most[16];
  __shared__ float s_scale[16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int l = blockIdx.y, n0 = blockIdx.x * kCols;
  const int8_t* wl = p.W + int64_t(l) * p.N * p.Kp;
  const int steps = (p.Kp + 63) / 64;

  uint4 w[T8][kAhead];
  auto load = [&](int s0) {                               // this warp's steps s0, s0 + 8, ...
#pragma unroll
    for (int j = 0; j < T8; ++j) {
      const int n = n0 + 8 * j + g;
#pragma unroll
      for (int i = 0; i < kAhead; ++i) {
        const int k = (s0 + i * kWarps) * 64 + t * 16;
        w[j][i] = n < p.N && k < p.Kp ? __ldg(reinterpret_cast<const uint4*>(wl + int64_t(n) * p.Kp + k)) : make_uint4(0, 0, 0, 0);
      }
    }
  };
  load(warp);

  // ---- the rows as codes: 256 / R threads share a row ----
  const T* x = static_cast<const T*>(p.x) + l * p.x_inner;
  if (threadIdx.x < 16) s_most[threadIdx.x] = 0;
  __syncthreads();
  const int per = 32 * kWarps / p.R, r = threadIdx.x / per, part = threadIdx.x % per;
  const T* row = x + (r < p.M ? r : 0) * p.x_outer;
  const int len = r < p.M ? p.K : 0;
  uint32_t m = 0;
  for (int k = part * 8; k < len; k += per * 8) {
    float f[8];
    eight<T, VEC>(row, k, len, f);
#pragma unroll
    for (int i = 0; i < 8; ++i) m = max(m, abs_bits(f[i]));
  }
  for (int o = min(per, 32) / 2; o > 0; o >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
  if (part % 32 == 0) atomicMax(&s_most[r], m);
  __syncthreads();
  const RowScale sc = row_scale(s_most[r]);
  if (part == 0) s_scale[r] = sc.scale;
  for (int k = part * 8; k < steps * 64; k += per * 8) {
    float f[8];
    eight<T, VEC>(row, k, len, f);
    *reinterpret_cast<uint2*>(codes + r * p.pitch + k) = make_uint2(codes4(f[0], f[1], f[2], f[3], sc.inv, sc.most),
                                                                    codes4(f[4], f[5], f[6], f[7], sc.inv, sc.most));
  }
  __syncthreads();

  // ---- products ----
  int c[T8][4] = {};
  for (int s0 = warp; s0 < steps; s0 += kWarps * kAhead) {
    if (s0 != warp) load(s0);
#pragma unroll
    for (int i = 0; i < kAhead; ++i) {
      const int s = s0 + i * kWarps;
      if (s >= steps) break;
      const uint4 lo = *reinterpret_cast<const uint4*>(codes + (g < p.R ? g : 0) * p.pitch + s * 64 + t * 16);
      uint4 hi = make_uint4(0, 0, 0, 0);
      if (p.R > 8) hi = *reinterpret_cast<const uint4*>(codes + (g + 8) * p.pitch + s * 64 + t * 16);
#pragma unroll
      for (int j = 0; j < T8; ++j) {
        mma_s8(c[j], lo.x, hi.x, lo.y, hi.y, w[j][i].x, w[j][i].y);
        mma_s8(c[j], lo.z, hi.z, lo.w, hi.w, w[j][i].z, w[j][i].w);
      }
    }
  }
#pragma unroll
  for (int j = 0; j < T8; ++j) {
    *reinterpret_cast<int2*>(&s_sum[warp][g][8 * j + 2 * t]) = make_int2(c[j][0], c[j][1]);
    *reinterpret_cast<int2*>(&s_sum[warp][g + 8][8 * j + 2 * t]) = make_int2(c[j][2], c[j][3]);
  }
  __syncthreads();

  // ---- the warps' sums, scales, bias, activation, residual ----
  for (int i = threadIdx.x; i < p.M * kCols; i += 32 * kWarps) {
    const int mrow = i / kCols, col = i % kCols, n = n0 + col;
    if (n >= p.N) continue;
    int sum = 0;
#pragma unroll
    for (int k = 0; k < kWarps; ++k) sum += s_sum[k][mrow][col];
    float v = fmaf(float(sum), s_scale[mrow] * p.t[int64_t(l) * p.N + n], p.bias != nullptr ? p.bias[n] : 0.0f);
    if (p.act == kGelu) {
      v = from_below(v);
      if constexpr (sizeof(T) == 4) v *= fmaf(0.5f, erff(v * 0.70710678f), 0.5f);
      else v = gelu_f(v);
    } else if (p.act == kRelu) {
      v = v < 0.0f ? 0.0f : v;
    }
    if (p.R_ != nullptr) v += kv::to_f(static_cast<const T*>(p.R_)[l * p.r_ls + mrow * p.r_ms + n]);
    static_cast<T*>(p.C)[l * p.c_ls + mrow * p.c_ms + n] = kv::from_f<T>(v);
  }
}

namespace {
template <typename T, bool VEC, int T8>
void launch(const FewParams& p, size_t smem) {
  auto* kern = few_kernel<T, VEC, T8>;
  if (smem > 24 * 1024) {                                 // with the static arrays past the default limit
    static std::atomic<uint64_t> allowed{0};
    int dev = 0;
    PD_CHECK_CUDA(cudaGetDevice(&dev));
    const uint64_t bit = uint64_t(1) << (dev & 63);
    if (!(allowed.load(std::memory_order_relaxed) & bit)) {
      PD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kFewBytes));
      allowed.fetch_or(bit, std::memory_order_relaxed);
    }
  }
  kern<<<dim3((p.N + 8 * T8 - 1) / (8 * T8), p.L), 32 * kWarps, smem, stream()>>>(p);
  PD_CHECK_LAUNCH();
}
}  // namespace

int64_t few_bytes(int64_t M, int64_t Kp) {
  const int64_t R = M <= 1 ? 1 : M <= 2 ? 2 : M <= 4 ? 4 : M <= 8 ? 8 : 16;
  return R * few_pitch(Kp);
}

void few(FewParams p, int dtype, bool vec) {
  p.R = p.M <= 1 ? 1 : p.M <= 2 ? 2 : p.M <= 4 ? 4 : p.M <= 8 ? 8 : 16;
  p.pitch = int(few_pitch(p.Kp));
  const size_t smem = size_t(few_bytes(p.M, p.Kp));
  // the widest block that still leaves most SMs one
  const int64_t want = num_sms() * 4 / 5;
  const int t8 = int64_t(p.L) * ((p.N + 31) / 32) >= want ? 4 : int64_t(p.L) * ((p.N + 15) / 16) >= want ? 2 : 1;
  auto go = [&](auto* tag) {
    using T = std::remove_pointer_t<decltype(tag)>;
    auto wide = [&](auto v) {
      constexpr bool V = decltype(v)::value;
      if (t8 == 4) launch<T, V, 4>(p, smem);
      else if (t8 == 2) launch<T, V, 2>(p, smem);
      else launch<T, V, 1>(p, smem);
    };
    if (vec) wide(std::true_type()); else wide(std::false_type());
  };
  if (dtype == kv::kBf16) go(static_cast<__nv_bfloat16*>(nullptr));
  else if (dtype == kv::kF16) go(static_cast<__half*>(nullptr));
  else go(static_cast<float*>(nullptr));
}

}  // namespace i8
}  // namespace pd
