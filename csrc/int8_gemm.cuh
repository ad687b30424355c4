// Products of 8-bit integers on tcgen05, sums in 32-bit integers:
//
//   C[l, m, n] = act( (sum_k A[l, m, k] B[l, n, k]) * (s[l, m] t[l, n]) + bias[n] ) + R[l, m, n]
//
// A: a token's codes with its scale s, B: a weight's codes with the scale t of
// each output channel; kind::i8, M = 128, K = 32 an instruction. Sums stay below
// 2^31 for K up to 131072 (codes down to -128).
//
// product_kernel is persistent, one block an SM, 14 warps, the roles of the bf16
// GEMM (gemm_tc.cu):
//   warp 0       TMA producer: 128 x 128 and BN x 128 byte tiles (128-byte
//                swizzle) into a ring; rows and columns past the operands' ends
//                arrive as zeros
//   warp 1       TMEM (2 x BN columns of s32) and the tcgen05.mma of one lane
//   warps 2..13  epilogue: a thread owns a row of 32 columns at a time; scales,
//                bias and activation in 32-bit floats, one rounding to the
//                output type, out through a swizzled 32 x 32 block in shared
//                memory and a TMA store (or row by row, where C's rows do not
//                lie on 16 bytes)
// Measured (1 B200, with the rows' codes): 16,417 x 1024 -> 4096 with GELU 100 us (1.4 PFLOP/s), 16 x 1024 rows by 256 ->
// 1024 with GELU 27, 2069 x 333 -> 1001 fp32 12. What bounds it: the epilogue's instructions (17 an element with GELU,
// 14 of them its polynomial; a tile of 256 columns takes 8.5 thousand cycles of twelve warps) and, less, shared memory: a
// k-block is written (48 KB) and read for 512 cycles of products, and takes 650 to 750.
//
// split_kernel is for calls whose tiles leave most SMs idle (few rows, a long
// axis): a cluster shares a tile and splits K. Every block writes its sums to a
// workspace, which stays in L2, and behind the cluster's barrier takes a part of
// the rows from all of them (out of the others' shared memory the same 32 KB took
// 3600 cycles a block, and a second barrier).
#pragma once

#include "int8_common.cuh"
#include "kv_common.cuh"
#include "tc_common.cuh"

#include <ATen/cuda/EmptyTensor.h>
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
constexpr int kMaxStages = 8;
constexpr int kSplitN = 64;             // columns of a tile whose K is split
constexpr int kSplitStages = 4;
constexpr int kSplitThreads = 192;      // TMA, MMA, four warps of 32 rows

struct Params {
  int M, N, L;
  int m_blocks, n_blocks, k_blocks, tiles;
  int bn, stages;
  int splits, kb_per_split;
  int* work;                                              // sums of a split tile [tiles][splits][128][64]
  const float* s; int64_t s_ls, s_ms;
  const float* t; int64_t t_ls;
  const float* bias;
  const void* R; int64_t r_ls, r_ms; int r_vec;           // r_vec: rows of R on 16 bytes
  void* C; int64_t c_ls, c_ms;
  int act;
  int a_mode, c_mode, c_tma;
  int b_shared;
  int* err;
};

template <typename T> constexpr int kStageBytes = 32 * 32 * int(sizeof(T));

// Byte offset of 16-byte chunk c of row r in a staged 32 x 32 block: the TMA
// swizzle of 64-byte (2-byte types) or 128-byte rows.
template <typename T>
__device__ __forceinline__ int staged(int r, int c) {
  return sizeof(T) == 2 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : r * 128 + ((c ^ (r & 7)) << 4);
}

template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if constexpr (std::is_same_v<T, __nv_bfloat16>) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
}
template <typename T>
__device__ __forceinline__ uint4 pack16(const float* v) {
  if constexpr (sizeof(T) == 4) {
    return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
  } else {
    return make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
  }
}

template <typename T>
__device__ __forceinline__ void gelu_pair(float& a, float& b) {
  if constexpr (sizeof(T) == 4) {                         // the polynomial of the 16-bit types is 5.5e-6 off
    a *= fmaf(0.5f, erff(a * 0.70710678f), 0.5f);
    b *= fmaf(0.5f, erff(b * 0.70710678f), 0.5f);
  } else {
    gelu2(a, b);
  }
}

__device__ __forceinline__ void mma_i8(uint32_t d, uint64_t da, uint64_t db, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(da), "l"(db), "r"(idesc), "r"(acc) : "memory");
}
// kind::i8: s32 accumulators, signed A and B, both K-major
__host__ __device__ constexpr uint32_t instr_i8(int m, int n) {
  return (2u << 4) | (1u << 7) | (1u << 10) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

__device__ __forceinline__ void tile_at(const Params& p, int w, int& l, int& mb, int& nb) {
  nb = w % p.n_blocks;
  const int r = w / p.n_blocks;
  mb = r % p.m_blocks;
  l = r / p.m_blocks;
}

using tcx::wait_for_launch_before;

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) product_kernel(const __grid_constant__ CUtensorMap tmA,
                                                              const __grid_constant__ CUtensorMap tmB,
                                                              const __grid_constant__ CUtensorMap tmC, const Params p) {
  extern __shared__ __align__(1024) uint8_t ring[];       // A tiles, B tiles, then a staged block for each epilogue warp
  __shared__ uint64_t full[kMaxStages], empty[kMaxStages], tfull[2], tempty[2], mma_done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  __shared__ __align__(16) float s_cols[kEpiWarps][64];   // a chunk's channel scales and biases, as t0 t1 b0 b1, ...
  const uint32_t kA = BM * BK, kB = p.bn * BK;
  uint8_t* sA = ring;
  uint8_t* sB = ring + p.stages * kA;
  if (tcx::smem_u32(ring) % 1024 != 0) {                  // the swizzled tiles need it
    set_error(p.err, 4);
    wait_for_launch_before();                             // kernels behind this one count on it
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < p.stages; ++s) { tcx::mbar_init(&full[s], 1); tcx::mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { tcx::mbar_init(&tfull[a], 1); tcx::mbar_init(&tempty[a], kEpiWarps * 32); }
    tcx::mbar_init(&mma_done, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(tcx::smem_u32(&tmem_slot)), "r"(2 * p.bn) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcx::tc_fence_before();
  __syncthreads();
  tcx::tc_fence_after();
  const uint32_t tmem = tmem_slot;
  wait_for_launch_before();

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 1;
      for (int w = blockIdx.x; w < p.tiles && !abort_flag; w += gridDim.x) {
        int l, mb, nb;
        tile_at(p, w, l, mb, nb);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!tcx::mbar_wait(&empty[stage], phase, p.err)) { abort_flag = 1; break; }
          tcx::mbar_expect_tx(&full[stage], kA + kB);
          tcx::tma_load_rows(sA + stage * kA, &tmA, &full[stage], p.a_mode, kb * BK, mb * BM, l);
          tcx::tma_load_rows(sB + stage * kB, &tmB, &full[stage], 0, kb * BK, nb * p.bn, p.b_shared ? 0 : l);
          ++issued;
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
        }
      }
      if (abort_flag) {                                   // every issued load lands before the block may exit
        for (int s = 0; s < p.stages; ++s) {
          const int n = (issued - s + p.stages - 1) / p.stages;     // loads issued on this stage
          if (n > 0) (void)tcx::mbar_wait(&full[s], uint32_t(n - 1) & 1u, p.err);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t idesc = instr_i8(BM, p.bn);
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      for (int w = blockIdx.x; w < p.tiles && !abort_flag; w += gridDim.x, ++local) {
        const int a = local & 1;
        if (!tcx::mbar_wait(&tempty[a], ((local >> 1) & 1) ^ 1, p.err)) { abort_flag = 1; break; }
        tcx::tc_fence_after();
        const uint32_t d = tmem + uint32_t(a * p.bn);
        bool ok = true;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!tcx::mbar_wait(&full[stage], phase, p.err)) { abort_flag = 1; ok = false; break; }
          tcx::tc_fence_after();
          const uint64_t da = tcx::smem_desc(tcx::smem_u32(sA + stage * kA)), db = tcx::smem_desc(tcx::smem_u32(sB + stage * kB));
#pragma unroll
          for (int k = 0; k < BK / 32; ++k)               // 32 bytes further: 2 in the descriptors' units of 16
            mma_i8(d, da + 2 * k, db + 2 * k, idesc, (kb | k) ? 1u : 0u);
          tcx::tc_commit(&empty[stage]);
          if (++stage == p.stages) { stage = 0; phase ^= 1; }
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
    uint8_t* stage_c = ring + p.stages * (kA + kB) + ew * kStageBytes<T>;
    float* cols = s_cols[ew];
    const int slot = (lane >> 1) * 4 + (lane & 1);        // t of column `lane`; its bias two further
    int local = 0;
    for (int w = blockIdx.x; w < p.tiles; w += gridDim.x, ++local) {
      const int a = local & 1;
      int l, mb, nb;
      tile_at(p, w, l, mb, nb);
      const int m0 = mb * BM + q * 32, n0 = nb * p.bn, row = m0 + lane;
      const bool there = row < p.M;
      const float s = there ? p.s[l * p.s_ls + row * p.s_ms] : 0.0f;
      const float s_most = __uint_as_float(p.act == kGelu ? __reduce_max_sync(0xffffffffu, abs_bits(s)) : 0u);
      const int c_end = min(p.bn, p.N - n0);
      auto column = [&](int c) {                          // (t, bias) of this lane's column of chunk c
        const int n = n0 + c + lane;
        const bool in = c < c_end && n < p.N;
        return make_float2(in ? __ldg(p.t + l * p.t_ls + n) : 0.0f, in && p.bias != nullptr ? __ldg(p.bias + n) : 0.0f);
      };
      float2 tb = column(part * 32);
      if (!tcx::mbar_wait(&tfull[a], (local >> 1) & 1, p.err)) { abort_flag = 1; break; }
      tcx::tc_fence_after();
      const uint32_t tbase = tmem + (uint32_t(q * 32) << 16) + uint32_t(a * p.bn);
#pragma unroll 1
      for (int c = part * 32; c < c_end; c += kParts * 32) {
        const int n = n0 + c, width = min(32, p.N - n);
        uint32_t r[32];
        tcx::tc_ld32_issue(tbase + c, r);
        cols[slot] = tb.x;
        cols[slot + 2] = tb.y;
        // GELU's guard is needed where minus infinity may come out: |sum * s * t + bias| < 2^31 * s * t + |bias|, in range where
        // neither passes 1e28. Each lane asks for its own column, so that a channel without a number hides no other; NaN asks.
        const bool guard = p.act == kGelu &&
                           __any_sync(0xffffffffu, !(s_most * fabsf(tb.x) <= 1e28f && fabsf(tb.y) <= 1e28f));
        __syncwarp();
        tb = column(c + kParts * 32);                             // the next chunk's, on its way
        tcx::tc_ld_wait(r);
        float v[32];
        const uint64_t s2 = pk2s(s);
#pragma unroll
        for (int i = 0; i < 32; i += 2) {
          const ulonglong2 tb2 = *reinterpret_cast<const ulonglong2*>(cols + 2 * i);
          pk2_split(pk2_fma(pk2(float(int(r[i])), float(int(r[i + 1]))), pk2_mul(s2, tb2.x), tb2.y), v[i], v[i + 1]);
        }
        if (p.act == kGelu) {
          if (guard) {
#pragma unroll
            for (int i = 0; i < 32; ++i) v[i] = from_below(v[i]);
          }
#pragma unroll
          for (int i = 0; i < 32; i += 2) gelu_pair<T>(v[i], v[i + 1]);
        } else if (p.act == kRelu) {
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];     // NaN stays
        }
        if (p.R != nullptr && there) {
          const T* res = static_cast<const T*>(p.R) + l * p.r_ls + row * p.r_ms + n;
          if (p.r_vec && width == 32) {
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
              if (i < width) v[i] += kv::to_f(res[i]);
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
          if (lane < width) {
            T* out = static_cast<T*>(p.C) + l * p.c_ls + m0 * p.c_ms + n + lane;
            const int rows = min(32, p.M - m0);
#pragma unroll 8
            for (int i = 0; i < rows; ++i, out += p.c_ms)
              *out = *reinterpret_cast<const T*>(stage_c + staged<T>(i, lane / kPer) + lane % kPer * int(sizeof(T)));
          }
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
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(2 * p.bn) : "memory");
  }
}

// ---------------------------------------------------------------------------
__device__ __forceinline__ void cluster_barrier() {
  asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
  asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ void store_sector(int* dst, const uint32_t* w) {          // 32 bytes
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
               ::"l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7]) : "memory");
}

template <typename T>
__global__ void __launch_bounds__(kSplitThreads, 1) split_kernel(const __grid_constant__ CUtensorMap tmA,
                                                                 const __grid_constant__ CUtensorMap tmB, const Params p) {
  constexpr uint32_t kA = BM * BK, kB = kSplitN * BK;
  extern __shared__ __align__(1024) uint8_t ring[];       // A and B tiles
  __shared__ uint64_t full[kSplitStages], empty[kSplitStages], done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  uint8_t* sA = ring;
  uint8_t* sB = ring + kSplitStages * kA;
  if (tcx::smem_u32(ring) % 1024 != 0) {                  // alike in every block of the cluster
    set_error(p.err, 4);
    wait_for_launch_before();                             // kernels behind this one count on it
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int rank = blockIdx.x % p.splits;
  int l, mb, nb;
  tile_at(p, blockIdx.x / p.splits, l, mb, nb);
  int* tile_sums = p.work + int64_t(blockIdx.x / p.splits) * p.splits * (BM * kSplitN);
  const int kb0 = rank * p.kb_per_split, kb1 = min(kb0 + p.kb_per_split, p.k_blocks);
  if (threadIdx.x == 0) {
    for (int s = 0; s < kSplitStages; ++s) { tcx::mbar_init(&full[s], 1); tcx::mbar_init(&empty[s], 1); }
    tcx::mbar_init(&done, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(tcx::smem_u32(&tmem_slot)), "r"(kSplitN) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tcx::tc_fence_before();
  __syncthreads();
  tcx::tc_fence_after();
  const uint32_t tmem = tmem_slot;

  if (warp == 0) {
    if (lane == 0) {
      int issued = 0;
      // the weight's first tiles do not wait for the rows' codes
      for (int kb = kb0; kb < min(kb1, kb0 + kSplitStages); ++kb) {
        const int stage = kb - kb0;
        tcx::mbar_expect_tx(&full[stage], kA + kB);
        tcx::tma_load_rows(sB + stage * kB, &tmB, &full[stage], 0, kb * BK, nb * kSplitN, p.b_shared ? 0 : l);
      }
      wait_for_launch_before();
      for (int kb = kb0; kb < kb1; ++kb, ++issued) {
        const int stage = issued % kSplitStages;
        if (issued >= kSplitStages) {
          if (!tcx::mbar_wait(&empty[stage], uint32_t(issued / kSplitStages - 1) & 1u, p.err)) { abort_flag = 1; break; }
          tcx::mbar_expect_tx(&full[stage], kA + kB);
          tcx::tma_load_rows(sB + stage * kB, &tmB, &full[stage], 0, kb * BK, nb * kSplitN, p.b_shared ? 0 : l);
        }
        tcx::tma_load_rows(sA + stage * kA, &tmA, &full[stage], p.a_mode, kb * BK, mb * BM, l);
      }
      if (abort_flag) {                                   // every issued load lands before the block may exit
        for (int s = 0; s < kSplitStages; ++s) {
          const int n = (issued - s + kSplitStages - 1) / kSplitStages;
          if (n > 0) (void)tcx::mbar_wait(&full[s], uint32_t(n - 1) & 1u, p.err);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      bool ok = true;
      for (int kb = kb0; kb < kb1 && ok; ++kb) {
        const int i = kb - kb0, stage = i % kSplitStages;
        ok = tcx::mbar_wait(&full[stage], uint32_t(i / kSplitStages) & 1u, p.err);
        if (!ok) { abort_flag = 1; break; }
        tcx::tc_fence_after();
        const uint64_t da = tcx::smem_desc(tcx::smem_u32(sA + stage * kA)), db = tcx::smem_desc(tcx::smem_u32(sB + stage * kB));
#pragma unroll
        for (int k = 0; k < BK / 32; ++k) mma_i8(tmem, da + 2 * k, db + 2 * k, instr_i8(BM, kSplitN), (i | k) ? 1u : 0u);
        tcx::tc_commit(&empty[stage]);
      }
      tcx::tc_commit(&done);
      (void)tcx::mbar_wait(&done, 0, p.err);              // finished before TMEM is freed
    }
  } else {
    // sums of this block's part of K, 32 rows a warp (TMEM lanes by the warp's place in its group of four)
    const int q = warp & 3, r_tile = q * 32 + lane;
    const bool there = mb * BM + r_tile < p.M;
    int* mine = tile_sums + (rank * BM + r_tile) * kSplitN;
    if (kb1 > kb0) {
      (void)tcx::mbar_wait(&done, 0, p.err);
      tcx::tc_fence_after();
      wait_for_launch_before();                           // the workspace may be the last call's too
#pragma unroll
      for (int c = 0; c < kSplitN; c += 32) {
        uint32_t r[32];
        tcx::tc_ld32_issue(tmem + (uint32_t(q * 32) << 16) + c, r);
        tcx::tc_ld_wait(r);
        if (there) {
#pragma unroll
          for (int i = 0; i < 32; i += 8) store_sector(mine + c + i, r + i);
        }
      }
      tcx::tc_fence_before();
    } else if (there) {
      wait_for_launch_before();
      const uint32_t none[8] = {};
#pragma unroll
      for (int i = 0; i < kSplitN; i += 8) store_sector(mine + i, none);
    }
  }
  __syncwarp();

  // this block's share of the rows, eight columns a thread; what else they need is on its way during the barrier
  constexpr int kWide = 8, kUnits = kSplitN / kWide;
  const int rows = BM / p.splits, base = rank * rows;
  float s = 0.0f, t[kWide], add[kWide], res[kWide];
  int row, n, width;
  auto operands = [&](int i) {
    row = mb * BM + base + i / kUnits;
    n = nb * kSplitN + i % kUnits * kWide;
    width = i < rows * kUnits && row < p.M ? min(kWide, p.N - n) : 0;
    if (width > 0) s = p.s[l * p.s_ls + row * p.s_ms];
#pragma unroll
    for (int e = 0; e < kWide; ++e) {
      t[e] = e < width ? __ldg(p.t + l * p.t_ls + n + e) : 0.0f;
      add[e] = e < width && p.bias != nullptr ? __ldg(p.bias + n + e) : 0.0f;
      res[e] = e < width && p.R != nullptr ? kv::to_f(static_cast<const T*>(p.R)[l * p.r_ls + row * p.r_ms + n + e]) : 0.0f;
    }
  };
  wait_for_launch_before();
  operands(threadIdx.x);
  cluster_barrier();                                      // every block's sums are in place
  for (int i = threadIdx.x; i < rows * kUnits; i += kSplitThreads) {
    if (i != threadIdx.x) operands(i);
    if (width <= 0) continue;
    const int4* at = reinterpret_cast<const int4*>(tile_sums + (base + i / kUnits) * kSplitN + i % kUnits * kWide);
    int4 part[2][8];
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (k < p.splits) {
        part[0][k] = __ldcg(at + k * (BM * kSplitN / 4));
        part[1][k] = __ldcg(at + k * (BM * kSplitN / 4) + 1);
      }
    }
    float v[kWide];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      int4 sum = part[h][0];
#pragma unroll
      for (int k = 1; k < 8; ++k)
        if (k < p.splits) { sum.x += part[h][k].x; sum.y += part[h][k].y; sum.z += part[h][k].z; sum.w += part[h][k].w; }
      v[4 * h] = float(sum.x); v[4 * h + 1] = float(sum.y); v[4 * h + 2] = float(sum.z); v[4 * h + 3] = float(sum.w);
    }
#pragma unroll
    for (int e = 0; e < kWide; ++e) {
      v[e] = fmaf(v[e], s * t[e], add[e]);
      if (p.act == kGelu) v[e] = from_below(v[e]);
      if (p.act == kRelu) v[e] = v[e] < 0.0f ? 0.0f : v[e];
    }
    if (p.act == kGelu) {
#pragma unroll
      for (int e = 0; e < kWide; e += 2) gelu_pair<T>(v[e], v[e + 1]);
    }
    if (p.R != nullptr) {
#pragma unroll
      for (int e = 0; e < kWide; ++e) v[e] += res[e];
    }
    T* out = static_cast<T*>(p.C) + l * p.c_ls + row * p.c_ms + n;
    if (p.c_tma && width == kWide) {                      // rows of C on 16 bytes
      constexpr int kPer = 16 / int(sizeof(T));
#pragma unroll
      for (int e = 0; e < kWide; e += kPer) *reinterpret_cast<uint4*>(out + e) = pack16<T>(v + e);
    } else {
#pragma unroll
      for (int e = 0; e < kWide; ++e)
        if (e < width) out[e] = kv::from_f<T>(v[e]);
    }
  }
  if (warp == 1) {
    tcx::tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kSplitN) : "memory");
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

// Launch right behind the rows' codes (before they are done: the kernel waits for them itself), as clusters if asked. The
// codes' kernel is launched in full order, so that the weight, read before that wait, is complete.
template <typename... Args>
void launch_behind(void (*kern)(Args...), std::atomic<uint64_t>& allowed, int most_smem, int grid, int threads, size_t smem,
                   int cluster, Args... args) {
  int dev = 0;
  PD_CHECK_CUDA(cudaGetDevice(&dev));
  const uint64_t bit = uint64_t(1) << (dev & 63);
  if (!(allowed.load(std::memory_order_relaxed) & bit)) {  // once a device: the call costs a small launch's time
    PD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, most_smem));
    allowed.fetch_or(bit, std::memory_order_relaxed);
  }
  cudaLaunchConfig_t cfg{};
  cfg.gridDim = dim3(unsigned(grid));
  cfg.blockDim = dim3(unsigned(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream();
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = unsigned(cluster);
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = cluster > 1 ? 2 : 1;
  PD_CHECK_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
  note_launch();
}

template <typename T>
void product(const CUtensorMap& ta, const void* B, int64_t Kp, int64_t B_l, const CUtensorMap& tc, Params& p, at::Device device) {
  at::Tensor work;                                        // freed behind the launch, on its stream
  constexpr int kMost = 226 * 1024;
  const int64_t blocks = int64_t(p.L) * p.m_blocks, sms = num_sms();
  auto weight = [&](int bn) {
    int mode;
    return map_of(CU_TENSOR_MAP_DATA_TYPE_UINT8, B, Kp, p.N, B_l, Kp, Kp * p.N, BK, bn, CU_TENSOR_MAP_SWIZZLE_128B, mode);
  };
  auto count = [&](int bn) {
    p.n_blocks = (p.N + bn - 1) / bn;
    const int64_t tiles = blocks * p.n_blocks;
    PD_CHECK(tiles < (int64_t(1) << 28), "int8_linear: too many rows");
    p.tiles = int(tiles);
  };
  const int64_t narrow = blocks * ((p.N + kSplitN - 1) / kSplitN);
  if (narrow * 2 <= sms && p.k_blocks >= 2) {             // tiles of 64 columns leave half of the SMs idle: split K
    count(kSplitN);
    p.splits = 2;
    while (p.splits < 8 && narrow * p.splits * 2 <= sms && p.splits * 2 <= p.k_blocks) p.splits *= 2;
    p.kb_per_split = (p.k_blocks + p.splits - 1) / p.splits;
    work = at::detail::empty_cuda({int64_t(p.tiles) * p.splits * BM * kSplitN}, at::kInt, device, c10::nullopt);
    p.work = work.data_ptr<int>();
    constexpr size_t smem = kSplitStages * size_t(BM + kSplitN) * BK;    // two blocks an SM: clusters of 8 fit everywhere
    static std::atomic<uint64_t> allowed{0};
    launch_behind(split_kernel<T>, allowed, int(smem), p.tiles * p.splits, kSplitThreads, smem, p.splits, ta, weight(kSplitN), p);
    return;
  }
  // Waves of tiles, each taking its columns and about 64 more (its start and end). us by tiles of 64 / 128 / 256 columns:
  // 2069 x 333 -> 1001 12.1 / 11.8 / 15.6; 16 x 1024 rows by 256 -> 1024 29.5 / 23.7 / 22.9; 1024 x 1024 -> 1024
  // 8.5 / 9.2 / 11.0; 16,417 x 1024 -> 4096 154 / 95 / 82.
  int64_t best = -1;
  for (int bn : {256, 128, 64}) {
    const int64_t waves = (blocks * ((p.N + bn - 1) / bn) + sms - 1) / sms, cost = waves * (bn + 64);
    if (best < 0 || cost < best) { best = cost; p.bn = bn; }
  }
  count(p.bn);
  const int stage = (BM + p.bn) * BK, staging = kEpiWarps * kStageBytes<T>;
  p.stages = std::min(kMaxStages, (kMost - 5 * 1024 - staging) / stage);
  static std::atomic<uint64_t> allowed{0};
  launch_behind(product_kernel<T>, allowed, kMost - 5 * 1024, std::min(p.tiles, int(sms)), kThreads,
                size_t(p.stages) * stage + staging, 1, ta, weight(p.bn), tc, p);
}

}  // namespace i8
}  // namespace pd
