// Products of 8-bit integers on tcgen05, sums in 32-bit integers:
//
//   C[l, m, n] = act( (sum_k A[l, m, k] B[l, n, k]) * (s[l, m] t[l, n]) + bias[n] ) + R[l, m, n]
//
// A: a token's codes with its scale s, B: a weight's codes with the scale t of
// each output channel. Persistent, one block an SM, 14 warps, the roles of the
// bf16 GEMM (gemm_tc.cu):
//   warp 0       TMA producer: 128 x 128 and BN x 128 byte tiles (128-byte
//                swizzle) into a ring of STAGES; rows and columns past the
//                operands' ends arrive as zeros
//   warp 1       TMEM (2 x BN columns of s32) and the tcgen05.mma of one lane:
//                kind::i8, M = 128, N = BN, K = 32
//   warps 2..13  epilogue: a thread owns a row of 32 columns at a time; scales,
//                bias and activation in 32-bit floats, one rounding to the
//                output type, out through a swizzled 32 x 32 block in shared
//                memory and a TMA store (or row by row, where C's rows do not
//                lie on 16 bytes)
// Sums stay below 2^31 for K up to 133,000 (codes within +-127).
#pragma once

#include "int8_common.cuh"
#include "kv_common.cuh"
#include "tc_common.cuh"

#include <atomic>
#include <type_traits>

namespace pd {
namespace i8 {

namespace tcx = pd::tc;

constexpr int BM = 128;
constexpr int BK = 128;                 // bytes, four instructions of 32
constexpr int kEpiWarps = 12;
constexpr int kParts = kEpiWarps / 4;   // warps that share 32 rows, by 32-column chunks
constexpr int kThreads = 64 + 32 * kEpiWarps;

struct Params {
  int M, N, L;
  int m_blocks, n_blocks, k_blocks, tiles;
  const float* s; int64_t s_ls, s_ms;
  const float* t; int64_t t_ls;
  const float* bias;
  const void* R; int64_t r_ls, r_ms; int r_vec;     // r_vec: rows of R on 16 bytes, whole chunks
  void* C; int64_t c_ls, c_ms;
  int act;
  int a_mode, c_mode, c_tma;
  int b_shared;
  int* err;
};

template <typename T> struct Out { static constexpr int kStage = 32 * 32 * int(sizeof(T)); };

// Byte offset of 16-byte chunk c of row r in a staged 32 x 32 block: the TMA
// swizzle of 64-byte (2-byte types) or 128-byte rows.
template <typename T>
__device__ __forceinline__ int staged(int r, int c) {
  return sizeof(T) == 2 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : r * 128 + ((c ^ (r & 7)) << 4);
}

template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  uint4 u;
  T* e = reinterpret_cast<T*>(&u);
#pragma unroll
  for (int i = 0; i < 16 / int(sizeof(T)); ++i) e[i] = kv::from_f<T>(v[i]);
  return u;
}

__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
// kind::i8: s32 accumulators, signed A and B, both K-major
constexpr uint32_t instr_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

__device__ __forceinline__ void tile_at(const Params& p, int w, int& l, int& mb, int& nb) {
  nb = w % p.n_blocks;
  const int r = w / p.n_blocks;
  mb = r % p.m_blocks;
  l = r / p.m_blocks;
}

template <int BN, int STAGES, typename T>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ CUtensorMap tmA,
                                                              const __grid_constant__ CUtensorMap tmB,
                                                              const __grid_constant__ CUtensorMap tmC, const Params p) {
  constexpr uint32_t kA = BM * BK, kB = BN * BK, kCols = 2 * BN;
  extern __shared__ __align__(1024) uint8_t ring[];       // A and B tiles, then a staged block for each epilogue warp
  __shared__ uint64_t full[STAGES], empty[STAGES], tfull[2], tempty[2], mma_done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  uint8_t* sA = ring;
  uint8_t* sB = ring + STAGES * kA;

  if (tcx::smem_u32(ring) % 1024 != 0) {                  // the swizzled tiles need it
    set_error(p.err, 4);
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { tcx::mbar_init(&full[s], 1); tcx::mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { tcx::mbar_init(&tfull[a], 1); tcx::mbar_init(&tempty[a], kEpiWarps * 32); }
    tcx::mbar_init(&mma_done, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(tcx::smem_u32(&tmem_slot)), "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcx::tc_fence_before();
  __syncthreads();
  tcx::tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 1;
      int issued_on[STAGES];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) issued_on[s] = 0;
      for (int w = blockIdx.x; w < p.tiles && !abort_flag; w += gridDim.x) {
        int l, mb, nb;
        tile_at(p, w, l, mb, nb);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!tcx::mbar_wait(&empty[stage], phase, p.err)) { abort_flag = 1; break; }
          tcx::mbar_expect_tx(&full[stage], kA + kB);
          tcx::tma_load_rows(sA + stage * kA, &tmA, &full[stage], p.a_mode, kb * BK, mb * BM, l);
          tcx::tma_load_rows(sB + stage * kB, &tmB, &full[stage], 0, kb * BK, nb * BN, p.b_shared ? 0 : l);
          ++issued_on[stage];
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (abort_flag) {                                   // every issued load lands before the block may exit
#pragma unroll
        for (int s = 0; s < STAGES; ++s)
          if (issued_on[s] > 0) (void)tcx::mbar_wait(&full[s], uint32_t(issued_on[s] - 1) & 1u, p.err);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      for (int w = blockIdx.x; w < p.tiles && !abort_flag; w += gridDim.x, ++local) {
        const int a = local & 1;
        if (!tcx::mbar_wait(&tempty[a], ((local >> 1) & 1) ^ 1, p.err)) { abort_flag = 1; break; }
        tcx::tc_fence_after();
        const uint32_t d = tmem + uint32_t(a * BN);
        bool ok = true;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!tcx::mbar_wait(&full[stage], phase, p.err)) { abort_flag = 1; ok = false; break; }
          tcx::tc_fence_after();
          const uint32_t a_addr = tcx::smem_u32(sA + stage * kA), b_addr = tcx::smem_u32(sB + stage * kB);
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)
            mma_i8(d, tcx::smem_desc(a_addr + k * 32), tcx::smem_desc(b_addr + k * 32), instr_i8(BM, BN),
                   (kb | k) ? 1u : 0u);
          tcx::tc_commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tcx::tc_commit(&tfull[a]);
      }
      tcx::tc_commit(&mma_done);                          // all issued products have finished before TMEM is freed
      (void)tcx::mbar_wait(&mma_done, 0, p.err);
    }
  } else {
    // ---------------- epilogue ----------------
    const int ew = warp - 2, q = warp & 3, part = ew >> 2;
    uint8_t* stage_c = ring + STAGES * (kA + kB) + ew * Out<T>::kStage;
    int local = 0;
    for (int w = blockIdx.x; w < p.tiles; w += gridDim.x, ++local) {
      const int a = local & 1;
      int l, mb, nb;
      tile_at(p, w, l, mb, nb);
      const int m0 = mb * BM + q * 32, n0 = nb * BN, row = m0 + lane;
      const bool there = row < p.M;
      const float s = there ? p.s[l * p.s_ls + row * p.s_ms] : 0.0f;
      if (!tcx::mbar_wait(&tfull[a], (local >> 1) & 1, p.err)) { abort_flag = 1; break; }
      tcx::tc_fence_after();
      const uint32_t tbase = tmem + (uint32_t(q * 32) << 16) + uint32_t(a * BN);
#pragma unroll 1
      for (int c = part * 32; c < BN && n0 + c < p.N; c += kParts * 32) {
        const int n = n0 + c, cols = min(32, p.N - n);
        uint32_t r[32];
        tcx::tc_ld32_issue(tbase + c, r);
        const float tl = lane < cols ? p.t[l * p.t_ls + n + lane] : 0.0f;
        const float bl = p.bias != nullptr && lane < cols ? p.bias[n + lane] : 0.0f;
        tcx::tc_ld_wait(r);
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i)
          v[i] = fmaf(float(int(r[i])), s * __shfl_sync(0xffffffffu, tl, i), __shfl_sync(0xffffffffu, bl, i));
        if (p.act == kGelu) {
#pragma unroll
          for (int i = 0; i < 32; i += 2) {
            v[i] = from_below(v[i]);
            v[i + 1] = from_below(v[i + 1]);
            if constexpr (sizeof(T) == 4) {               // the polynomial of the 16-bit types is 5.5e-6 off
              v[i] *= fmaf(0.5f, erff(v[i] * 0.70710678f), 0.5f);
              v[i + 1] *= fmaf(0.5f, erff(v[i + 1] * 0.70710678f), 0.5f);
            } else {
              gelu2(v[i], v[i + 1]);
            }
          }
        } else if (p.act == kRelu) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];     // NaN stays
        }
        if (p.R != nullptr && there) {
          const T* res = static_cast<const T*>(p.R) + l * p.r_ls + row * p.r_ms + n;
          if (p.r_vec && cols == 32) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              kv::Raw<8, T> x;
              float f[8];
              x.load(res + i);
              x.floats(f);
#pragma unroll
              for (int e = 0; e < 8; ++e) v[i + e] += f[e];
            }
          } else {
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (i < cols) v[i] += kv::to_f(res[i]);
          }
        }
        if (lane == 0) tcx::bulk_wait_read_all();         // the staged block's last store has read it
        __syncwarp();
        constexpr int kPer = 16 / int(sizeof(T));
#pragma unroll
        for (int j = 0; j < 32 / kPer; ++j)
          *reinterpret_cast<uint4*>(stage_c + staged<T>(lane, j)) = pack16<T>(v + j * kPer);
        if (p.c_tma) {
          tcx::fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tcx::tma_store_rows(&tmC, stage_c, p.c_mode, n, m0, l);
            tcx::bulk_commit();
          }
        } else {
          __syncwarp();
          T* out = static_cast<T*>(p.C) + l * p.c_ls + n;
          for (int i = 0; i < 32 && m0 + i < p.M; ++i)
            if (lane < cols)
              out[(m0 + i) * p.c_ms + lane] =
                  *reinterpret_cast<const T*>(stage_c + staged<T>(i, lane / kPer) + lane % kPer * int(sizeof(T)));
          __syncwarp();
        }
      }
      tcx::tc_fence_before();
      tcx::mbar_arrive(&tempty[a]);
    }
    if (lane == 0) tcx::bulk_wait_all();
    __syncwarp();
  }
  tcx::tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tcx::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

// ---------------------------------------------------------------------------
// 3-D map {inner, rows, L} of a [L, rows, inner] view; dims in the order {inner, L, rows} (mode 1) where the batches lie
// inside the rows, so that strides ascend. Strides in bytes.
inline CUtensorMap map_of(CUtensorMapDataType type, const void* base, int64_t inner, int64_t rows, int64_t L, int64_t row_bytes,
                   int64_t l_bytes, int box_inner, int box_rows, CUtensorMapSwizzle swizzle, int& mode) {
  CUtensorMap m;
  if (L <= 1) l_bytes = row_bytes * rows;
  mode = L > 1 && l_bytes < row_bytes ? 1 : 0;
  cuuint64_t dims[3] = {cuuint64_t(inner), cuuint64_t(mode ? L : rows), cuuint64_t(mode ? rows : L)};
  cuuint64_t strides[2] = {cuuint64_t(mode ? l_bytes : row_bytes), cuuint64_t(mode ? row_bytes : l_bytes)};
  cuuint32_t box[3] = {cuuint32_t(box_inner), cuuint32_t(mode ? 1 : box_rows), cuuint32_t(mode ? box_rows : 1)};
  cuuint32_t one[3] = {1, 1, 1};
  PD_CHECK(reinterpret_cast<uintptr_t>(base) % 16 == 0 && strides[0] % 16 == 0 && strides[1] % 16 == 0 && strides[0] > 0 &&
               strides[1] > 0 && strides[0] < (cuuint64_t(1) << 40) && strides[1] < (cuuint64_t(1) << 40),
           "int8 product: an operand's rows do not lie on 16 bytes");
  const CUresult r = tensor_map_encode_tiled(&m, type, 3, const_cast<void*>(base), dims, strides, box, one,
                                             CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  PD_CHECK(r == CUDA_SUCCESS, "int8 product: cuTensorMapEncodeTiled failed (%d)", int(r));
  return m;
}

template <int BN, int STAGES, typename T>
void launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tc, const Params& p) {
  constexpr size_t smem = STAGES * size_t(BM + BN) * BK + kEpiWarps * size_t(Out<T>::kStage);
  static_assert(smem + 1024 <= 232448, "shared memory of a block");
  auto* kern = product_kernel<BN, STAGES, T>;
  static std::atomic<uint64_t> allowed{0};               // by device: the call costs a small launch's time
  int dev = 0;
  PD_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {
    PD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  kern<<<std::min(p.tiles, num_sms()), kThreads, smem, stream()>>>(ta, tb, tc, p);
  PD_CHECK_LAUNCH();
}

template <typename T>
void product(const CUtensorMap& ta, const void* B, int64_t Kp, int64_t B_l, const CUtensorMap& tc, Params& p) {
  auto go = [&](auto bn, auto stages) {
    constexpr int BN = decltype(bn)::value;
    p.n_blocks = (p.N + BN - 1) / BN;
    const int64_t tiles = int64_t(p.L) * p.m_blocks * p.n_blocks;
    PD_CHECK(tiles < (int64_t(1) << 31), "int8_linear: too many rows");
    p.tiles = int(tiles);
    int mode;
    const CUtensorMap tb = map_of(CU_TENSOR_MAP_DATA_TYPE_UINT8, B, Kp, p.N, B_l, Kp, Kp * p.N, BK, BN,
                                  CU_TENSOR_MAP_SWIZZLE_128B, mode);
    launch<BN, decltype(stages)::value, T>(ta, tb, tc, p);
  };
  // The widest tile that still gives every SM one.
  const int64_t rows = int64_t(p.L) * p.m_blocks, sms = num_sms();
  constexpr bool two = sizeof(T) == 2;
  if (rows * ((p.N + 255) / 256) >= sms) go(std::integral_constant<int, 256>(), std::integral_constant<int, two ? 4 : 3>());
  else if (rows * ((p.N + 127) / 128) >= sms) go(std::integral_constant<int, 128>(), std::integral_constant<int, two ? 6 : 5>());
  else go(std::integral_constant<int, 64>(), std::integral_constant<int, two ? 8 : 7>());
}

}  // namespace i8
}  // namespace pd
