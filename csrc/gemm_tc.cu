// Persistent tcgen05 GEMM for sm_100a with fused epilogues.
//
//   C[l, m, n] = epi( sum_k A[l, m, k] * B[l, n, k] )        (A, B K-major, bf16)
//
// Structure (one CTA per SM, 6 warps):
//   warp 0      TMA producer: A/B tiles (128 x 64 and BN x 64, 128-byte
//               swizzle) into a STAGES-deep shared-memory ring, one mbarrier
//               per stage with expected-transaction bytes; each CTA loads
//               its own tiles.
//   warp 1      allocates TMEM (2 x BN fp32 columns: a double-buffered
//               accumulator) and one elected lane issues tcgen05.mma
//               (M=128, N=BN, K=16 per instruction) for every k-step,
//               releasing each smem stage with tcgen05.commit.
//   warps 2..5  epilogue: tcgen05.ld 32 columns at a time (each thread owns
//               one accumulator row = one TMEM lane), apply the fused op,
//               convert to bf16 and store; then hand the accumulator buffer
//               back to the MMA warp.  The MMA of tile i+1 overlaps the
//               epilogue of tile i.
// Fused epilogues: none | GELU (optionally also storing the pre-activation) |
// GELU storing its derivative | residual add | GELU backward from the
// pre-activation (acc * gelu'(pre)) | product with a stored derivative. An addend R (residual, or
// a bias / positional table broadcast through zero strides) is added before
// the activation in every mode but the GELU backward, where R is the
// pre-activation.
//
// A and B are described by 3-D TMA maps {K, rows, L} with arbitrary row and
// batch strides, so strided views (e.g. the NS rows of every sample, one
// batch per NS token) are consumed in place; C / R / AUX take element strides.
//
// Every mbarrier wait is bounded (2 s on %globaltimer); on timeout the warp
// records kWaitTimeout in the error word, stops issuing work, drains its own
// in-flight operations (bounded) and the CTA frees its TMEM and exits.
#include "common.cuh"
#include "driver_api.h"
#include "gemm_host.h"
#include "gemm_mat.h"
#include "tc_common.cuh"

#include <cuda.h>

#include <type_traits>

namespace pd {
namespace tc {

constexpr int BM = 128;
constexpr int BK = 64;
constexpr int kEpiWarps = 12;  // three warps per TMEM lane quarter, splitting the columns
constexpr int kThreads = 64 + 32 * kEpiWarps;

// kGeluD: C = GELU(x), AUX = GELU'(x) for x = acc + R in fp32 -- the derivative
// stored in the forward makes the backward's epilogue a plain product (kMul:
// C = acc * R), with no transcendental per element.
// kRelu: C = max(acc + R, 0) (R: a bias through a zero row stride);
// kMaskPos: C = acc where R > 0, else 0 (R: the ReLU layer's stored output,
// so the data gradient of the next layer leaves as the pre-activation
// gradient of this one); kMulAdd: C = R * (acc + b) + R2, with b added via
// the operands (an extra K row), AUX optionally storing acc (the DCNv2 cross
// layer: x_{l+1} = x0 * (t V + b) + x_l with R = x0, R2 = x_l).
enum Epi : int { kNone = 0, kGelu = 1, kResidual = 2, kDGelu = 3, kGeluD = 4, kMul = 5, kRelu = 6, kMaskPos = 7,
                 kMulAdd = 8 };

struct Params {
  int M, N, K, L;
  int m_blocks, n_blocks, k_blocks, tiles;
  __nv_bfloat16* C; int64_t c_ls, c_ms;
  const __nv_bfloat16* R; int64_t r_ls, r_ms;      // addend, pre-activation (kDGelu) or factor (kMul)
  __nv_bfloat16* AUX; int64_t aux_ls, aux_ms;       // pre-activation (kGelu, optional) or GELU' (kGeluD)
  const __nv_bfloat16* R2; int64_t r2_ls, r2_ms;    // second addend (kMulAdd)
  int epi;
  int a_mode, b_mode;   // TMA map dim order: 0 = {K, rows, L}, 1 = {K, L, rows}
  int c_mode, x_mode;   // store maps of C / AUX: 0 = {N, rows, L}, 1 = {N, L, rows}
  int r_tma, r_mode;    // R read by TMA (a full [L, M, N] view) and its map's dim order
  int b_shared;         // B has one batch shared by every l
  int b_kn;             // B stored [L, K, N] (N contiguous: a weight used transposed), loaded MN-major
  int* err;
};

__device__ __forceinline__ void tile_coords(const Params& p, int t, int& l, int& mb, int& nb) {
  nb = t % p.n_blocks;
  const int r = t / p.n_blocks;
  mb = r % p.m_blocks;
  l = r / p.m_blocks;
}

template <int BN, int STAGES>
__global__ void __launch_bounds__(kThreads, 1) gemm_kernel(const __grid_constant__ CUtensorMap tmA,
                                                           const __grid_constant__ CUtensorMap tmB,
                                                           const __grid_constant__ CUtensorMap tmC,
                                                           const __grid_constant__ CUtensorMap tmX,
                                                           const __grid_constant__ CUtensorMap tmR,
                                                           const Params p) {
  constexpr uint32_t kABytes = BM * BK * 2;
  constexpr uint32_t kBBytes = BN * BK * 2;
  constexpr uint32_t kTmemCols = 2 * BN;  // power of two for BN in {64, 128, 256}
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * kABytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + STAGES * kBBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;     // [2]
  uint64_t* tempty = tfull + 2;         // [2]
  uint64_t* mma_done = tempty + 2;      // [1]
  uint64_t* rbar_all = mma_done + 1;    // [kEpiWarps][2]: R blocks landed (TMA)
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(rbar_all + 2 * kEpiWarps);
  // per epilogue warp: 32 x 32 bf16 staging blocks for C and R / AUX (64-byte
  // rows, 16-byte chunks XOR-swizzled by (row >> 1) & 3: conflict-free both
  // when a thread writes its own row and when 4 lanes cover one row)
  // (the 64-byte swizzle of the TMA stores: buffers 512-byte aligned)
  uint8_t* stage_base = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(tmem_slot) + 64 + 1023) & ~uintptr_t(1023));
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull[a], 1); mbar_init(&tempty[a], kEpiWarps * 32); }
    mbar_init(mma_done, 1);
    for (int i = 0; i < 2 * kEpiWarps; ++i) mbar_init(&rbar_all[i], 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmC) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_launch_before();
  let_next_launch();

  if (warp == 0) {
    // ---------------- TMA producer ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 1;
      int issued = 0;
      int issued_on[STAGES];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) issued_on[s] = 0;
      for (int t = blockIdx.x; t < p.tiles && !*abort_flag; t += gridDim.x) {
        int l, mb, nb;
        tile_coords(p, t, l, mb, nb);
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(&empty[stage], phase, p.err)) { *abort_flag = 1; break; }
          mbar_expect_tx(&full[stage], kABytes + kBBytes);
          tma_load_rows(sA + stage * kABytes, &tmA, &full[stage], p.a_mode, kb * BK, mb * BM, l);
          if (p.b_kn) {
#pragma unroll
            for (int g = 0; g < BN / 64; ++g)   // [64 k-rows][64 n] boxes
              tma_load_rows(sB + stage * kBBytes + g * 8192, &tmB, &full[stage], p.b_mode, nb * BN + 64 * g, kb * BK,
                            p.b_shared ? 0 : l);
          } else {
            tma_load_rows(sB + stage * kBBytes, &tmB, &full[stage], p.b_mode, kb * BK, nb * BN, p.b_shared ? 0 : l);
          }
          ++issued_on[stage];
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      // drain: every issued load must have landed before the CTA can exit
      if (*abort_flag) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s)
          if (issued_on[s] > 0) (void)mbar_wait(&full[s], uint32_t(issued_on[s] - 1) & 1u, p.err);
      }
      (void)issued;
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(BM, BN);
      const uint32_t idesc_run = idesc | (p.b_kn ? (1u << 16) : 0u);   // B MN-major
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      for (int t = blockIdx.x; t < p.tiles && !*abort_flag; t += gridDim.x, ++local) {
        const int a = local & 1;
        const uint32_t ephase = ((local >> 1) & 1) ^ 1;
        if (!mbar_wait(&tempty[a], ephase, p.err)) { *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(a * BN);
        bool ok = true;
        for (int kb = 0; kb < p.k_blocks; ++kb) {
          if (!mbar_wait(&full[stage], phase, p.err)) { *abort_flag = 1; ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + stage * kABytes);
          const uint32_t b_addr = smem_u32(sB + stage * kBBytes);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t db = p.b_kn ? smem_desc_mn(b_addr + k * 2048) : smem_desc(b_addr + k * 32);
            tc_mma(d, smem_desc(a_addr + k * 32), db, idesc_run, (kb | k) ? 1u : 0u);
          }
          tc_commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit(&tfull[a]);
      }
      // all MMAs issued by this thread have finished before TMEM is freed
      tc_commit(mma_done);
      (void)mbar_wait(mma_done, 0, p.err);
    }
  } else {
    // ---------------- epilogue ----------------
    // Warp ew owns TMEM lane quarter q (rows q*32..q*32+31 of the tile) and the
    // 32-column chunks c with (c / 32) % 3 == part.  Per chunk: the R block
    // (residual, GELU' factor or pre-activation) arrives by TMA into a
    // two-deep ring, issued one chunk ahead (a broadcast addend -- bias or
    // positional table, zero strides -- is prefetched into registers
    // instead); tcgen05.ld the accumulator, apply the epilogue, stage the
    // bf16 block in swizzled smem and hand it to a TMA store (C, and AUX),
    // which runs while the next chunk is computed.
    const int ew = warp - 2;
    const int q = warp & 3;
    const int part = ew >> 2;
    constexpr int kParts = kEpiWarps / 4;
    uint8_t* stC = stage_base + ew * 3 * 2048;
    uint8_t* stR0 = stC + 2048;   // R ring: buffers stR0 and stR0 + 2048
    uint64_t* rbar = rbar_all + 2 * ew;
    const bool r_tma = p.r_tma != 0;
    int kc = 0;          // chunks processed by this warp (R ring position)
    int r_pending = 0;   // R blocks issued and not yet waited for
    const int cr = lane >> 2, cc = lane & 3;
    auto sw = [](int r, int c) { return r * 64 + ((c ^ ((r >> 1) & 3)) << 4); };
    const bool has_r = (p.R != nullptr);   // addend (bias / residual), or GELU's pre-activation for kDGelu
    // work items: (tile, chunk) in this warp's order
    auto first_chunk = [&]() { return part * 32; };
    auto next_work = [&](int& t, int& c) {
      c += kParts * 32;
      if (c >= BN) { c = first_chunk(); t += gridDim.x; }
    };
    auto load_r = [&](int t, int c, uint4* dst) {
      int l, mb, nb;
      tile_coords(p, t, l, mb, nb);
      const int m0 = mb * BM + q * 32;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = cr + 8 * i;
        dst[i] = (m0 + r < p.M)
                     ? __ldcs(reinterpret_cast<const uint4*>(p.R + l * p.r_ls + int64_t(m0 + r) * p.r_ms + nb * BN + c +
                                                             cc * 8))
                     : make_uint4(0, 0, 0, 0);
      }
    };
    auto issue_r = [&](int t, int c, int buf) {   // lane 0 only
      int l, mb, nb;
      tile_coords(p, t, l, mb, nb);
      mbar_expect_tx(&rbar[buf], 32 * 32 * 2);
      tma_load_rows(stR0 + (buf << 11), &tmR, &rbar[buf], p.r_mode, nb * BN + c, mb * BM + q * 32, l);
    };
    uint4 pref[4];
    if (has_r && first_chunk() < BN && blockIdx.x < p.tiles) {
      if (r_tma) {
        if (lane == 0) issue_r(blockIdx.x, first_chunk(), 0);
        r_pending = 1;
      } else {
        load_r(blockIdx.x, first_chunk(), pref);
      }
    }
    int local = 0;
    for (int t = blockIdx.x; t < p.tiles; t += gridDim.x, ++local) {
      const int a = local & 1;
      if (!mbar_wait(&tfull[a], (local >> 1) & 1, p.err)) { *abort_flag = 1; break; }
      tc_fence_after();
      int l, mb, nb;
      tile_coords(p, t, l, mb, nb);
      const int m0 = mb * BM + q * 32;
      const int n0 = nb * BN;
      const uint32_t tbase = tmem + (uint32_t(q * 32) << 16) + uint32_t(a * BN);
      // one chunk: 32 accumulator columns of this warp's 32 rows, already in r
      auto process = [&](uint32_t (&r)[32], int c) -> bool {
        // the previous chunk's TMA stores have read the staging blocks: waited
        // for here when an R block is about to land in one of them, else only
        // just before the first staging write (the math of this chunk overlaps
        // the stores' shared-memory reads)
        bool waited = false;
        auto wait_staging = [&]() {
          if (waited) return;
          if (lane == 0) bulk_wait_read_all();
          __syncwarp();
          waited = true;
        };
        if (has_r) wait_staging();
        uint8_t* stR = stR0 + (r_tma ? ((kc & 1) << 11) : 0);
        uint8_t* stX = stR;   // AUX staging reuses the R block once it has been consumed
        if (has_r) {
          int tn = t, cn = c;
          next_work(tn, cn);
          if (r_tma) {
            if (tn < p.tiles) {   // the next block lands in the other buffer while this chunk runs
              if (lane == 0) issue_r(tn, cn, (kc + 1) & 1);
              ++r_pending;
            }
            const bool ok = mbar_wait(&rbar[kc & 1], uint32_t(kc >> 1) & 1u, p.err);
            --r_pending;
            if (!ok) { *abort_flag = 1; return false; }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) *reinterpret_cast<uint4*>(stR + sw(cr + 8 * i, cc)) = pref[i];
            __syncwarp();
            if (tn < p.tiles) load_r(tn, cn, pref);   // in flight during this chunk
          }
        }
        float v[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
        if (has_r && p.epi != kDGelu && p.epi != kMul && p.epi != kMaskPos && p.epi != kMulAdd) {
          // addend before the activation: residual, or a bias broadcast through a zero row stride
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 pk = *reinterpret_cast<const uint4*>(stR + sw(lane, j));
            const __nv_bfloat162* hh = reinterpret_cast<const __nv_bfloat162*>(&pk);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = __bfloat1622float2(hh[e]);
              v[8 * j + 2 * e] += f.x;
              v[8 * j + 2 * e + 1] += f.y;
            }
          }
        }
        if (p.epi == kGelu && p.AUX) {
          wait_staging();
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4 pk;
            __nv_bfloat162 h0 = __floats2bfloat162_rn(v[8 * j], v[8 * j + 1]);
            __nv_bfloat162 h1 = __floats2bfloat162_rn(v[8 * j + 2], v[8 * j + 3]);
            __nv_bfloat162 h2 = __floats2bfloat162_rn(v[8 * j + 4], v[8 * j + 5]);
            __nv_bfloat162 h3 = __floats2bfloat162_rn(v[8 * j + 6], v[8 * j + 7]);
            pk.x = *reinterpret_cast<uint32_t*>(&h0); pk.y = *reinterpret_cast<uint32_t*>(&h1);
            pk.z = *reinterpret_cast<uint32_t*>(&h2); pk.w = *reinterpret_cast<uint32_t*>(&h3);
            *reinterpret_cast<uint4*>(stX + sw(lane, j)) = pk;
          }
        }
        if (p.epi == kGelu) {
          // GELU of the bf16-rounded pre-activation (the value AUX stores)
#pragma unroll
          for (int j = 0; j < 32; j += 2) {
            float x0 = __bfloat162float(__float2bfloat16_rn(v[j]));
            float x1 = __bfloat162float(__float2bfloat16_rn(v[j + 1]));
            gelu2(x0, x1);
            v[j] = x0;
            v[j + 1] = x1;
          }
        } else if (p.epi == kGeluD) {
          uint4 dpk[4];
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            float d[8];
#pragma unroll
            for (int e = 0; e < 8; e += 2)       // the fp32 pre-activation (no bf16 round trip)
              gelu_grad2<true>(v[8 * j + e], v[8 * j + e + 1], d[e], d[e + 1]);
            __nv_bfloat162 h0 = __floats2bfloat162_rn(d[0], d[1]);
            __nv_bfloat162 h1 = __floats2bfloat162_rn(d[2], d[3]);
            __nv_bfloat162 h2 = __floats2bfloat162_rn(d[4], d[5]);
            __nv_bfloat162 h3 = __floats2bfloat162_rn(d[6], d[7]);
            dpk[j].x = *reinterpret_cast<uint32_t*>(&h0); dpk[j].y = *reinterpret_cast<uint32_t*>(&h1);
            dpk[j].z = *reinterpret_cast<uint32_t*>(&h2); dpk[j].w = *reinterpret_cast<uint32_t*>(&h3);
            // half of the math runs before the staging wait (register budget:
            // four warps per SMSP leave 128 registers a thread)
            if (j == 1) {
              wait_staging();
              *reinterpret_cast<uint4*>(stX + sw(lane, 0)) = dpk[0];
              *reinterpret_cast<uint4*>(stX + sw(lane, 1)) = dpk[1];
            } else if (j > 1) {
              *reinterpret_cast<uint4*>(stX + sw(lane, j)) = dpk[j];
            }
          }
        } else if (p.epi == kMul) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 pk = *reinterpret_cast<const uint4*>(stR + sw(lane, j));
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&pk);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = __bfloat1622float2(h[e]);
              v[8 * j + 2 * e] *= f.x;
              v[8 * j + 2 * e + 1] *= f.y;
            }
          }
        } else if (p.epi == kRelu) {
#pragma unroll
          for (int j = 0; j < 32; ++j) v[j] = fmaxf(v[j], 0.f);
        } else if (p.epi == kMaskPos) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 pk = *reinterpret_cast<const uint4*>(stR + sw(lane, j));
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&pk);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = __bfloat1622float2(h[e]);
              v[8 * j + 2 * e] = f.x > 0.f ? v[8 * j + 2 * e] : 0.f;
              v[8 * j + 2 * e + 1] = f.y > 0.f ? v[8 * j + 2 * e + 1] : 0.f;
            }
          }
        } else if (p.epi == kMulAdd) {
          // R2 row of this thread: 32 columns straight from global memory
          const int row = m0 + lane;
          uint4 q4[4] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0),
                         make_uint4(0, 0, 0, 0)};
          if (row < p.M) {
            const uint4* src = reinterpret_cast<const uint4*>(p.R2 + l * p.r2_ls + int64_t(row) * p.r2_ms + n0 + c);
#pragma unroll
            for (int j = 0; j < 4; ++j) q4[j] = __ldcs(src + j);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 pk = *reinterpret_cast<const uint4*>(stR + sw(lane, j));
            if (p.AUX) {   // acc to AUX, in the 16 bytes of R this thread has just read
              uint4 ax;
              __nv_bfloat162 a0 = __floats2bfloat162_rn(v[8 * j], v[8 * j + 1]);
              __nv_bfloat162 a1 = __floats2bfloat162_rn(v[8 * j + 2], v[8 * j + 3]);
              __nv_bfloat162 a2 = __floats2bfloat162_rn(v[8 * j + 4], v[8 * j + 5]);
              __nv_bfloat162 a3 = __floats2bfloat162_rn(v[8 * j + 6], v[8 * j + 7]);
              ax.x = *reinterpret_cast<uint32_t*>(&a0); ax.y = *reinterpret_cast<uint32_t*>(&a1);
              ax.z = *reinterpret_cast<uint32_t*>(&a2); ax.w = *reinterpret_cast<uint32_t*>(&a3);
              *reinterpret_cast<uint4*>(stX + sw(lane, j)) = ax;
            }
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&pk);
            const __nv_bfloat162* h2 = reinterpret_cast<const __nv_bfloat162*>(&q4[j]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = __bfloat1622float2(h[e]), g = __bfloat1622float2(h2[e]);
              v[8 * j + 2 * e] = fmaf(f.x, v[8 * j + 2 * e], g.x);
              v[8 * j + 2 * e + 1] = fmaf(f.y, v[8 * j + 2 * e + 1], g.y);
            }
          }
        } else if (p.epi == kDGelu) {
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const uint4 pk = *reinterpret_cast<const uint4*>(stR + sw(lane, j));
            const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&pk);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const float2 f = __bfloat1622float2(h[e]);
              float x0 = f.x, x1 = f.y, d0, d1;
              gelu_grad2<false>(x0, x1, d0, d1);
              v[8 * j + 2 * e] *= d0;
              v[8 * j + 2 * e + 1] *= d1;
            }
          }
        }
        wait_staging();
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          uint4 pk;
          __nv_bfloat162 h0 = __floats2bfloat162_rn(v[8 * j], v[8 * j + 1]);
          __nv_bfloat162 h1 = __floats2bfloat162_rn(v[8 * j + 2], v[8 * j + 3]);
          __nv_bfloat162 h2 = __floats2bfloat162_rn(v[8 * j + 4], v[8 * j + 5]);
          __nv_bfloat162 h3 = __floats2bfloat162_rn(v[8 * j + 6], v[8 * j + 7]);
          pk.x = *reinterpret_cast<uint32_t*>(&h0); pk.y = *reinterpret_cast<uint32_t*>(&h1);
          pk.z = *reinterpret_cast<uint32_t*>(&h2); pk.w = *reinterpret_cast<uint32_t*>(&h3);
          *reinterpret_cast<uint4*>(stC + sw(lane, j)) = pk;
        }
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          tma_store_rows(&tmC, stC, p.c_mode, n0 + c, m0, l);
          if ((p.epi == kGelu || p.epi == kGeluD || p.epi == kMulAdd) && p.AUX)
            tma_store_rows(&tmX, stX, p.x_mode, n0 + c, m0, l);
          bulk_commit();
        }
        ++kc;
        return true;
      };
      constexpr int kStep = kParts * 32;
      const int c0 = first_chunk();
      {
        bool ok = true;
#pragma unroll 1
        for (int c = c0; c < BN && ok; c += kStep) {
          uint32_t r0[32];
          tc_ld32_issue(tbase + c, r0);
          tc_ld_wait(r0);
          ok = process(r0, c);
        }
        if (!ok) break;
      }
      tc_fence_before();
      mbar_arrive(&tempty[a]);
    }
    // an R block still in flight (the loop ended early) lands before the CTA exits
    if (r_pending > 0) (void)mbar_wait(&rbar[kc & 1], uint32_t(kc >> 1) & 1u, p.err);
    if (lane == 0) bulk_wait_all();   // every store of this warp has completed
    __syncwarp();
  }
  // teardown: all roles are out of their loops (every wait above is bounded)
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}


// ---------------------------------------------------------------------------
// Weight gradient: C[l] (fp32, [M, N]) += sum over rows k of A[l][k, m] B[l][k, n]
// with A = dY [rows, M] and B = X [rows, N] both stored row-major, i.e. both
// operands MN-major (no transposes). The row dimension is long (every token of
// the batch) and the output small, so the work is split over K: a work item
// is (tile, k-range); items cycle over tiles first so concurrent CTAs hit
// different outputs. The epilogue adds its fp32 partial tile into C with
// vector reductions (red.global.add.v4.f32); C must be zeroed by the caller.
// Warp roles, TMEM double buffering and the bounded waits are those of
// gemm_kernel.
// ---------------------------------------------------------------------------
struct WgParams {
  int M, N, K, L;
  int m_blocks, n_blocks, k_blocks, tiles, splits, kb_per_split, items;
  int l_sum;        // 1: the L batches are part of the reduction (one output); k-blocks run over (l, k)
  int kb_per_l;     // k-blocks of one batch when l_sum
  void* C; int64_t c_ls, c_ms;
  int a_mode, b_mode;
  int* err;
};

__device__ __forceinline__ void wg_item(const WgParams& p, int w, int& l, int& mb, int& nb, int& kb0, int& kb1) {
  const int t = w % p.tiles;
  const int sp = w / p.tiles;
  nb = t % p.n_blocks;
  const int r = t / p.n_blocks;
  mb = r % p.m_blocks;
  l = p.l_sum ? 0 : r / p.m_blocks;
  kb0 = sp * p.kb_per_split;
  kb1 = min(kb0 + p.kb_per_split, p.k_blocks);
}

__device__ __forceinline__ void red_add_v4(float* addr, float a, float b, float c, float d) {
  asm volatile("red.global.add.v4.f32 [%0], {%1, %2, %3, %4};" ::"l"(addr), "f"(a), "f"(b), "f"(c), "f"(d)
               : "memory");
}

// Out = void: partial tiles are added into fp32 C. Out = float or __nv_bfloat16 (one split): a tile is the whole sum, so
// it is stored in the gradient's type at once, with no zeroing, no reductions in memory and no conversion afterwards: eight
// warps stage 32 rows of 128 bytes each for a TMA store, so that whole lines are written.
template <int BN, int STAGES, typename Out = void>
__global__ void __launch_bounds__(kThreads, 1) wgrad_kernel(const __grid_constant__ CUtensorMap tmA,
                                                            const __grid_constant__ CUtensorMap tmB,
                                                            const __grid_constant__ CUtensorMap tmC,
                                                            const WgParams p) {
  constexpr uint32_t kABytes = BM * BK * 2;
  constexpr uint32_t kBBytes = BN * BK * 2;
  constexpr uint32_t kTmemCols = 2 * BN;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* sA = smem;
  uint8_t* sB = smem + STAGES * kABytes;
  uint64_t* full = reinterpret_cast<uint64_t*>(sB + STAGES * kBBytes);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;     // [2]
  uint64_t* tempty = tfull + 2;         // [2]
  uint64_t* mma_done = tempty + 2;      // [1]
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(mma_done + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
  // (direct) a staged block of 4 KB for each of eight warps
  [[maybe_unused]] uint8_t* stage_base = reinterpret_cast<uint8_t*>(
      (reinterpret_cast<uintptr_t>(tmem_slot) + 64 + 1023) & ~uintptr_t(1023));

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { mbar_init(&tfull[a], 1); mbar_init(&tempty[a], kEpiWarps * 32); }
    mbar_init(mma_done, 1);
    *abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(tmem_slot)), "r"(kTmemCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  wait_for_launch_before();
  let_next_launch();

  if (warp == 0) {
    // ---------------- TMA producer: [64 k-rows][64 cols] boxes ----------------
    if (lane == 0) {
      int stage = 0;
      uint32_t phase = 1;
      int issued_on[STAGES];
#pragma unroll
      for (int s = 0; s < STAGES; ++s) issued_on[s] = 0;
      for (int w = blockIdx.x; w < p.items && !*abort_flag; w += gridDim.x) {
        int l, mb, nb, kb0, kb1;
        wg_item(p, w, l, mb, nb, kb0, kb1);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase, p.err)) { *abort_flag = 1; break; }
          mbar_expect_tx(&full[stage], kABytes + kBBytes);
          // with l_sum a k-block is (batch, block within the batch); rows past a batch's end load as zeros
          const int lb = p.l_sum ? kb / p.kb_per_l : l;
          const int kr = (p.l_sum ? kb % p.kb_per_l : kb) * BK;
#pragma unroll
          for (int g = 0; g < BM / 64; ++g)
            tma_load_rows(sA + stage * kABytes + g * 8192, &tmA, &full[stage], p.a_mode, mb * BM + 64 * g, kr, lb);
#pragma unroll
          for (int g = 0; g < BN / 64; ++g)
            tma_load_rows(sB + stage * kBBytes + g * 8192, &tmB, &full[stage], p.b_mode, nb * BN + 64 * g, kr, lb);
          ++issued_on[stage];
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (*abort_flag) {
#pragma unroll
        for (int s = 0; s < STAGES; ++s)
          if (issued_on[s] > 0) (void)mbar_wait(&full[s], uint32_t(issued_on[s] - 1) & 1u, p.err);
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer (A and B MN-major) ----------------
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(BM, BN) | (1u << 15) | (1u << 16);
      int stage = 0;
      uint32_t phase = 0;
      int local = 0;
      for (int w = blockIdx.x; w < p.items && !*abort_flag; w += gridDim.x, ++local) {
        int l, mb, nb, kb0, kb1;
        wg_item(p, w, l, mb, nb, kb0, kb1);
        const int a = local & 1;
        const uint32_t ephase = ((local >> 1) & 1) ^ 1;
        if (!mbar_wait(&tempty[a], ephase, p.err)) { *abort_flag = 1; break; }
        tc_fence_after();
        const uint32_t d = tmem + uint32_t(a * BN);
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full[stage], phase, p.err)) { *abort_flag = 1; ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + stage * kABytes);
          const uint32_t b_addr = smem_u32(sB + stage * kBBytes);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k)
            tc_mma(d, smem_desc_mn(a_addr + k * 2048), smem_desc_mn(b_addr + k * 2048), idesc,
                   (kb > kb0 || k > 0) ? 1u : 0u);
          tc_commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit(&tfull[a]);
      }
      tc_commit(mma_done);
      (void)mbar_wait(mma_done, 0, p.err);
    }
  } else {
    // ---------------- epilogue: fp32 partial tile added into C ----------------
    const int ew = warp - 2;
    const int q = warp & 3;
    const int part = ew >> 2;
    constexpr int kParts = kEpiWarps / 4;
    int local = 0;
    for (int w = blockIdx.x; w < p.items; w += gridDim.x, ++local) {
      const int a = local & 1;
      if (!mbar_wait(&tfull[a], (local >> 1) & 1, p.err)) { *abort_flag = 1; break; }
      tc_fence_after();
      int l, mb, nb, kb0, kb1;
      wg_item(p, w, l, mb, nb, kb0, kb1);
      const int row = mb * BM + q * 32 + lane;
      const uint32_t tbase = tmem + (uint32_t(q * 32) << 16) + uint32_t(a * BN);
      if constexpr (!std::is_void_v<Out>) {
        constexpr int kWide = 128 / int(sizeof(Out));
        uint8_t* st = stage_base + ew * 4096;
#pragma unroll 1
        for (int c = part * kWide; c < BN && part < 2; c += 2 * kWide) {
          if (lane == 0) bulk_wait_read_all();            // the staged block's last store has read it
          __syncwarp();
#pragma unroll
          for (int h = 0; h < kWide; h += 32) {
            uint32_t r[32];
            tc_ld32_issue(tbase + c + h, r);
            tc_ld_wait(r);
            constexpr int kChunks = sizeof(Out) == 4 ? 8 : 4;                       // of 16 bytes
#pragma unroll
            for (int j = 0; j < kChunks; ++j) {
              uint32_t w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                if constexpr (sizeof(Out) == 4) {
                  w[e] = r[4 * j + e];
                } else {
                  const __nv_bfloat162 b = __floats2bfloat162_rn(__uint_as_float(r[8 * j + 2 * e]), __uint_as_float(r[8 * j + 2 * e + 1]));
                  w[e] = *reinterpret_cast<const uint32_t*>(&b);
                }
              }
              *reinterpret_cast<uint4*>(st + lane * 128 + (((h / 32 * kChunks + j) ^ (lane & 7)) << 4)) =
                  make_uint4(w[0], w[1], w[2], w[3]);
            }
          }
          fence_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&tmC, st, nb * BN + c, mb * BM + q * 32, l);
            bulk_commit();
          }
        }
      } else {
#pragma unroll 1
        for (int c = part * 32; c < BN; c += kParts * 32) {
          uint32_t r[32];
          tc_ld32_issue(tbase + c, r);
          tc_ld_wait(r);
          if (row < p.M && kb1 > kb0) {
            float* dst = static_cast<float*>(p.C) + l * p.c_ls + int64_t(row) * p.c_ms + nb * BN + c;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              red_add_v4(dst + j, __uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]),
                         __uint_as_float(r[j + 3]));
          }
        }
      }
      tc_fence_before();
      mbar_arrive(&tempty[a]);
    }
    if (!std::is_void_v<Out> && lane == 0) bulk_wait_all();
    __syncwarp();
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols) : "memory");
  }
}

// The same sum with tiles of 256 x 256: two accumulators share B. wgrad_kernel writes 48 KB of operands to shared memory and
// reads them back for 512 cycles of products, more than its bandwidth; here it is 64 KB for 1024. The accumulators fill
// TMEM, so a block works on one long item (or few) and its epilogue overlaps nothing. 8,960 x 4096 x 1024: 88 -> 66 us;
// 98,560 x 256 x 1024: 69 -> 63; 114,688 x 768 x 256: 60 -> 57.
constexpr int kWideStages = 3;
__global__ void __launch_bounds__(kThreads, 1) wgrad_wide_kernel(const __grid_constant__ CUtensorMap tmA,
                                                                 const __grid_constant__ CUtensorMap tmB, const WgParams p) {
  constexpr uint32_t kOp = 256 * BK * 2;                  // bytes of A or B in a stage
  extern __shared__ __align__(1024) uint8_t wide_ring[];
  __shared__ uint64_t full[kWideStages], empty[kWideStages], tfull, tempty, mma_done;
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  if (smem_u32(wide_ring) % 1024 != 0) {                  // the swizzled tiles need it
    set_error(p.err, kBadShape);
    wait_for_launch_before();                             // kernels behind this one count on it
    return;
  }
  uint8_t* sA = wide_ring;
  uint8_t* sB = wide_ring + kWideStages * kOp;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < kWideStages; ++s) { mbar_init(&full[s], 1); mbar_init(&empty[s], 1); }
    mbar_init(&tfull, 1);
    mbar_init(&tempty, kEpiWarps * 32);
    mbar_init(&mma_done, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&tmem_slot)) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_slot;
  wait_for_launch_before();
  let_next_launch();

  if (warp == 0) {
    if (lane == 0) {
      int stage = 0, issued = 0;
      uint32_t phase = 1;
      for (int w = blockIdx.x; w < p.items && !abort_flag; w += gridDim.x) {
        int l, mb, nb, kb0, kb1;
        wg_item(p, w, l, mb, nb, kb0, kb1);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&empty[stage], phase, p.err)) { abort_flag = 1; break; }
          mbar_expect_tx(&full[stage], 2 * kOp);
          const int lb = p.l_sum ? kb / p.kb_per_l : l;
          const int kr = (p.l_sum ? kb % p.kb_per_l : kb) * BK;
#pragma unroll
          for (int g = 0; g < 4; ++g) {
            tma_load_rows(sA + stage * kOp + g * 8192, &tmA, &full[stage], p.a_mode, mb * 256 + 64 * g, kr, lb);
            tma_load_rows(sB + stage * kOp + g * 8192, &tmB, &full[stage], p.b_mode, nb * 256 + 64 * g, kr, lb);
          }
          ++issued;
          if (++stage == kWideStages) { stage = 0; phase ^= 1; }
        }
      }
      if (abort_flag) {                                   // every issued load lands before the block may exit
        for (int s = 0; s < kWideStages; ++s) {
          const int n = (issued - s + kWideStages - 1) / kWideStages;
          if (n > 0) (void)mbar_wait(&full[s], uint32_t(n - 1) & 1u, p.err);
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0) {
      constexpr uint32_t idesc = instr_desc(BM, 256) | (1u << 15) | (1u << 16);     // A and B MN-major
      int stage = 0, local = 0;
      uint32_t phase = 0;
      for (int w = blockIdx.x; w < p.items && !abort_flag; w += gridDim.x, ++local) {
        int l, mb, nb, kb0, kb1;
        wg_item(p, w, l, mb, nb, kb0, kb1);
        if (!mbar_wait(&tempty, uint32_t(local & 1) ^ 1u, p.err)) { abort_flag = 1; break; }
        tc_fence_after();
        bool ok = true;
        for (int kb = kb0; kb < kb1; ++kb) {
          if (!mbar_wait(&full[stage], phase, p.err)) { abort_flag = 1; ok = false; break; }
          tc_fence_after();
          const uint32_t a_addr = smem_u32(sA + stage * kOp), b_addr = smem_u32(sB + stage * kOp);
#pragma unroll
          for (int k = 0; k < BK / 16; ++k) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
              tc_mma(tmem + h * 256, smem_desc_mn(a_addr + h * 16384 + k * 2048), smem_desc_mn(b_addr + k * 2048), idesc,
                     (kb > kb0 || k > 0) ? 1u : 0u);
          }
          tc_commit(&empty[stage]);
          if (++stage == kWideStages) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tc_commit(&tfull);
      }
      tc_commit(&mma_done);
      (void)mbar_wait(&mma_done, 0, p.err);
    }
  } else {
    const int ew = warp - 2, q = warp & 3, part = ew >> 2;
    constexpr int kParts = kEpiWarps / 4;
    int local = 0;
    for (int w = blockIdx.x; w < p.items; w += gridDim.x, ++local) {
      if (!mbar_wait(&tfull, uint32_t(local) & 1u, p.err)) { abort_flag = 1; break; }
      tc_fence_after();
      int l, mb, nb, kb0, kb1;
      wg_item(p, w, l, mb, nb, kb0, kb1);
#pragma unroll 1
      for (int c = part * 32; c < 512; c += kParts * 32) {
        uint32_t r[32];
        tc_ld32_issue(tmem + (uint32_t(q * 32) << 16) + c, r);
        tc_ld_wait(r);
        const int row = mb * 256 + (c >> 8) * 128 + q * 32 + lane;
        float* dst = static_cast<float*>(p.C) + l * p.c_ls + int64_t(row) * p.c_ms + nb * 256 + (c & 255);
        if (kb1 > kb0) {
#pragma unroll
          for (int j = 0; j < 32; j += 4)
            red_add_v4(dst + j, __uint_as_float(r[j]), __uint_as_float(r[j + 1]), __uint_as_float(r[j + 2]),
                       __uint_as_float(r[j + 3]));
        }
      }
      tc_fence_before();
      mbar_arrive(&tempty);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 1) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
  }
}

}  // namespace tc

// ---------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------
namespace {

template <int BN, int STAGES>
void launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tcm, const CUtensorMap& txm,
            const CUtensorMap& trm, const tc::Params& p) {
  constexpr size_t smem = STAGES * (tc::BM * tc::BK * 2 + BN * tc::BK * 2) + 1024 + 1024 + tc::kEpiWarps * 3 * 2048;
  static_assert(smem <= 232448, "GEMM shared memory over the 227 KB per-block limit");
  static tc::SharedLimit limit;
  limit.allow(tc::gemm_kernel<BN, STAGES>, smem);
  const int grid = p.tiles < num_sms() ? p.tiles : num_sms();
  tc::launch_behind(tc::gemm_kernel<BN, STAGES>, dim3(unsigned(grid)), tc::kThreads, smem, ta, tb, tcm, txm, trm, p);
}

}  // namespace

// C[l, m, :N] = epi(A[l] @ B[l]^T).  A: [L, M, K], B: [L or 1, N, K] -- or, with b_kn,
// [L or 1, K, N] (a weight used transposed, read MN-major) -- C/R/AUX: [L, M, N] views
// (unit column stride).  epi: 0 none, 1 gelu (aux = pre-activation, optional), 2 residual (R),
// 3 dgelu (R = pre-activation), 4 gelu storing gelu' in AUX, 5 product with R, 6 relu (R = bias
// addend), 7 acc where R > 0, 8 R * acc + R2 (AUX: acc, optional).
void tc_gemm(at::Tensor A, at::Tensor B, at::Tensor C, int64_t epi, c10::optional<at::Tensor> R,
             c10::optional<at::Tensor> AUX, at::Tensor err, bool b_kn, c10::optional<at::Tensor> R2) {
  check_operand(A, "A");
  check_operand(B, "B");
  const int64_t L = A.size(0), M = A.size(1), K = A.size(2), N = b_kn ? B.size(2) : B.size(1);
  TORCH_CHECK((b_kn ? B.size(1) : B.size(2)) == K && (B.size(0) == L || B.size(0) == 1),
              b_kn ? "B must be [L or 1, K, N]" : "B must be [L or 1, N, K]");
  TORCH_CHECK(N % 64 == 0, "N must be a multiple of 64");
  TORCH_CHECK(C.dim() == 3 && C.size(0) == L && C.size(1) == M && C.size(2) == N && C.stride(2) == 1 &&
              C.scalar_type() == at::kBFloat16 && C.stride(1) % 8 == 0 && (C.size(0) == 1 || C.stride(0) % 8 == 0) &&
              reinterpret_cast<uintptr_t>(C.data_ptr()) % 16 == 0, "C must be a [L, M, N] bf16 view with aligned rows");
  check_extent(C, "C");
  if (R && R->defined()) check_extent(*R, "R");
  if (AUX && AUX->defined()) check_extent(*AUX, "AUX");
  tc::Params p{};
  p.M = int(M); p.N = int(N); p.K = int(K); p.L = int(L);
  p.m_blocks = int((M + tc::BM - 1) / tc::BM);
  p.k_blocks = int((K + tc::BK - 1) / tc::BK);
  p.C = reinterpret_cast<__nv_bfloat16*>(C.data_ptr()); p.c_ls = C.stride(0); p.c_ms = C.stride(1);
  p.epi = int(epi);
  p.err = err.data_ptr<int>();
  PD_CHECK(epi >= tc::kNone && epi <= tc::kMulAdd, "unknown epilogue %lld", (long long)epi);
  TORCH_CHECK(!(epi == tc::kResidual || epi == tc::kDGelu || epi == tc::kMul || epi == tc::kMaskPos ||
                epi == tc::kMulAdd) || (R && R->defined()),
              "this epilogue needs R");
  TORCH_CHECK(epi != tc::kMulAdd || (R2 && R2->defined()), "the multiply-add epilogue needs R2");
  if (epi == tc::kMulAdd) {
    TORCH_CHECK(R2->dim() == 3 && R2->sizes() == C.sizes() && R2->stride(2) == 1 && R2->stride(1) % 8 == 0 &&
                (R2->size(0) == 1 || R2->stride(0) % 8 == 0) && reinterpret_cast<uintptr_t>(R2->data_ptr()) % 16 == 0 &&
                R2->scalar_type() == at::kBFloat16, "R2 must match C (bf16, 16-byte aligned rows)");
    check_extent(*R2, "R2");
    p.R2 = reinterpret_cast<const __nv_bfloat16*>(R2->data_ptr()); p.r2_ls = R2->stride(0); p.r2_ms = R2->stride(1);
    TORCH_CHECK(R->stride(1) != 0 && (L == 1 || R->stride(0) != 0), "the multiply-add factor R must be a full matrix");
  }
  TORCH_CHECK(epi != tc::kGeluD || (AUX && AUX->defined()), "the GELU-derivative epilogue needs AUX");
  if (R && R->defined()) {
    // R: [L, M, N] view (stride 0 allowed on L and M: a bias or per-row-block addend)
    TORCH_CHECK(R->dim() == 3 && R->sizes() == C.sizes() && R->stride(2) == 1 && R->stride(1) % 8 == 0 &&
                (R->size(0) == 1 || R->stride(0) % 8 == 0) && reinterpret_cast<uintptr_t>(R->data_ptr()) % 16 == 0 &&
                R->scalar_type() == at::kBFloat16, "R must match C (bf16, 16-byte aligned rows)");
    p.R = reinterpret_cast<const __nv_bfloat16*>(R->data_ptr()); p.r_ls = R->stride(0); p.r_ms = R->stride(1);
  }
  if (AUX && AUX->defined()) {
    TORCH_CHECK(AUX->dim() == 3 && AUX->sizes() == C.sizes() && AUX->stride(2) == 1 && AUX->stride(1) % 8 == 0 &&
                (AUX->size(0) == 1 || AUX->stride(0) % 8 == 0) && reinterpret_cast<uintptr_t>(AUX->data_ptr()) % 16 == 0,
                "AUX must match C (16-byte aligned rows)");
    p.AUX = reinterpret_cast<__nv_bfloat16*>(AUX->data_ptr()); p.aux_ls = AUX->stride(0); p.aux_ms = AUX->stride(1);
  }
  if (M == 0 || L == 0) return;
  const int BN = (N % 256 == 0) ? 256 : (N % 128 == 0 ? 128 : 64);
  p.n_blocks = int(N / BN);
  p.tiles = int(L) * p.m_blocks * p.n_blocks;
  const CUtensorMap ta = make_map(A.data_ptr(), K, M, L, A.stride(1), A.stride(0), tc::BM, p.a_mode);
  p.b_kn = b_kn ? 1 : 0;
  // MN-major B: boxes of 64 n x 64 k-rows over dims {N, K, L}
  const CUtensorMap tb = b_kn ? make_map(B.data_ptr(), N, K, B.size(0), B.stride(1), B.stride(0), tc::BK, p.b_mode)
                              : make_map(B.data_ptr(), K, N, B.size(0), B.stride(1), B.stride(0), BN, p.b_mode);
  p.b_shared = (B.size(0) == 1) ? 1 : 0;
  const CUtensorMap tcm = make_store_map(C.data_ptr(), N, M, L, C.stride(1), C.stride(0), p.c_mode);
  p.x_mode = p.c_mode;
  const CUtensorMap txm = p.AUX ? make_store_map(AUX->data_ptr(), N, M, L, AUX->stride(1), AUX->stride(0), p.x_mode)
                                : tcm;
  // R by TMA unless it broadcasts through a zero stride (bias / positional addend)
  p.r_tma = (p.R && p.r_ms != 0 && (L == 1 || p.r_ls != 0)) ? 1 : 0;
  p.r_mode = 0;
  const CUtensorMap trm = p.r_tma ? make_store_map(R->data_ptr(), N, M, L, R->stride(1), R->stride(0), p.r_mode) : tcm;
  if (BN == 256) launch<256, 3>(ta, tb, tcm, txm, trm, p);
  else if (BN == 128) launch<128, 4>(ta, tb, tcm, txm, trm, p);
  else launch<64, 6>(ta, tb, tcm, txm, trm, p);
}

namespace {

// Map of a contiguous [L, M, N] gradient for stores of 32 rows of 128 bytes (128-byte swizzle).
CUtensorMap make_line_map(const at::Tensor& C, int64_t M, int64_t N) {
  CUtensorMap m;
  const int64_t size = C.element_size();
  const cuuint64_t dims[3] = {cuuint64_t(N), cuuint64_t(M), cuuint64_t(C.size(0))};
  const cuuint64_t strides[2] = {cuuint64_t(N * size), cuuint64_t(M * N * size)};
  const cuuint32_t box[3] = {cuuint32_t(128 / size), 32, 1}, one[3] = {1, 1, 1};
  check_encode(C.data_ptr(), dims, strides, box, 3, "gradient map");
  const CUresult r = tensor_map_encode_tiled(
      &m, size == 4 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, C.data_ptr(), dims, strides, box,
      one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_NONE,
      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  PD_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled (gradient) failed (%d)", int(r));
  return m;
}

// Blocks, tiles and splits of a weight gradient [M, N] over L batches of K rows.
tc::WgParams wgrad_plan(int64_t L, int64_t K, int64_t M, int64_t N, bool l_sum) {
  tc::WgParams p{};
  p.M = int(M); p.N = int(N); p.K = int(K); p.L = int(L);
  p.m_blocks = int((M + tc::BM - 1) / tc::BM);
  const int BN = (N % 256 == 0) ? 256 : (N % 128 == 0 ? 128 : 64);
  p.n_blocks = int(N / BN);
  p.l_sum = l_sum ? 1 : 0;
  p.kb_per_l = int((K + tc::BK - 1) / tc::BK);
  p.k_blocks = l_sum ? int(L) * p.kb_per_l : p.kb_per_l;
  p.tiles = int(l_sum ? 1 : L) * p.m_blocks * p.n_blocks;
  // about two items per SM without a ragged last wave, each at least 8 k-blocks long
  int splits = std::max(1, (2 * num_sms()) / p.tiles);
  splits = std::min(splits, std::max(1, p.k_blocks / 8));
  p.kb_per_split = (p.k_blocks + splits - 1) / splits;
  p.splits = (p.k_blocks + p.kb_per_split - 1) / p.kb_per_split;
  p.items = p.tiles * p.splits;
  return p;
}

// The same for tiles of 256 x 256, M and N multiples of it: the split that takes the fewest waves of k-blocks, some four of
// which an item's epilogue costs.
tc::WgParams wgrad_wide_plan(int64_t L, int64_t K, int64_t M, int64_t N, bool l_sum) {
  tc::WgParams p = wgrad_plan(L, K, M, N, l_sum);
  p.m_blocks = int(M / 256);
  p.n_blocks = int(N / 256);
  p.tiles = int(l_sum ? 1 : L) * p.m_blocks * p.n_blocks;
  int64_t best = -1;
  for (int splits = 1; splits <= std::max(1, p.k_blocks / 4) && splits <= 2 * num_sms(); ++splits) {
    const int per = (p.k_blocks + splits - 1) / splits, n = (p.k_blocks + per - 1) / per;
    const int64_t cost = (int64_t(p.tiles) * n + num_sms() - 1) / num_sms() * (per + 4);
    if (best < 0 || cost < best) { best = cost; p.kb_per_split = per; p.splits = n; }
  }
  p.items = p.tiles * p.splits;
  return p;
}

void run_wgrad_wide(const Mat& A, const Mat& B, const at::Tensor& C, tc::WgParams p, int* err) {
  p.C = C.data_ptr(); p.c_ls = C.stride(0); p.c_ms = C.stride(1);
  p.err = err;
  const CUtensorMap ta = make_map(A.p, p.M, p.K, p.L, A.ms, A.ls, tc::BK, p.a_mode);
  const CUtensorMap tb = make_map(B.p, p.N, p.K, p.L, B.ms, B.ls, tc::BK, p.b_mode);
  constexpr int smem = tc::kWideStages * 2 * 256 * tc::BK * 2;
  PD_CHECK_CUDA(cudaFuncSetAttribute(tc::wgrad_wide_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  tc::launch_behind(tc::wgrad_wide_kernel, dim3(unsigned(std::min(p.items, num_sms()))), tc::kThreads, size_t(smem), ta, tb, p);
}

// direct: C in its own type, stored by the one split.
void run_wgrad(const Mat& A, const Mat& B, const at::Tensor& C, tc::WgParams p, int* err, bool direct) {
  p.C = C.data_ptr(); p.c_ls = C.stride(0); p.c_ms = C.stride(1);
  p.err = err;
  // MN-major operands: [64 k-rows][64 cols] boxes over dims {cols, rows, L}
  const CUtensorMap ta = make_map(A.p, p.M, p.K, p.L, A.ms, A.ls, tc::BK, p.a_mode);
  const CUtensorMap tb = make_map(B.p, p.N, p.K, p.L, B.ms, B.ls, tc::BK, p.b_mode);
  const CUtensorMap tcm = direct ? make_line_map(C, p.M, p.N) : ta;
  auto go = [&](auto kern, int bn, int stages) {
    const size_t smem = size_t(stages) * (tc::BM * tc::BK * 2 + bn * tc::BK * 2) + 1024 + 1024 + (direct ? 8 * 4096 + 1024 : 0);
    PD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    const int grid = p.items < num_sms() ? p.items : num_sms();
    tc::launch_behind(kern, dim3(unsigned(grid)), tc::kThreads, smem, ta, tb, tcm, p);
  };
  auto by_width = [&](auto* tag) {
    using Out = std::remove_pointer_t<decltype(tag)>;
    constexpr int kLess = std::is_void_v<Out> ? 0 : 1;   // stages that make room for the staged blocks
    if (p.N % 256 == 0) go(tc::wgrad_kernel<256, 4 - kLess, Out>, 256, 4 - kLess);
    else if (p.N % 128 == 0) go(tc::wgrad_kernel<128, 6 - kLess, Out>, 128, 6 - kLess);
    else go(tc::wgrad_kernel<64, 8 - kLess, Out>, 64, 8 - kLess);
  };
  if (!direct) by_width(static_cast<void*>(nullptr));
  else if (C.scalar_type() == at::kFloat) by_width(static_cast<float*>(nullptr));
  else by_width(static_cast<__nv_bfloat16*>(nullptr));
}

}  // namespace

// C[l] (fp32 [M, N], zeroed by the caller) += A[l]^T B[l] over the rows:
// A [L, K, M], B [L, K, N] bf16 views with unit stride on the last dim.
// With l_sum, C is [1, M, N] and the sum runs over the batches as well.
void tc_wgrad(at::Tensor A, at::Tensor B, at::Tensor C, at::Tensor err, bool l_sum) {
  check_operand(A, "A");
  check_operand(B, "B");
  const int64_t L = A.size(0), K = A.size(1), M = A.size(2), N = B.size(2);
  TORCH_CHECK(B.size(0) == L && B.size(1) == K, "B must be [L, K, N] over the same rows as A");
  TORCH_CHECK(M % 64 == 0 && N % 64 == 0, "wgrad: M and N must be multiples of 64");
  const int64_t LC = l_sum ? 1 : L;
  TORCH_CHECK(C.scalar_type() == at::kFloat && C.dim() == 3 && C.size(0) == LC && C.size(1) == M && C.size(2) == N &&
                  C.stride(2) == 1 && C.stride(1) % 4 == 0 && (LC == 1 || C.stride(0) % 4 == 0) &&
                  reinterpret_cast<uintptr_t>(C.data_ptr()) % 16 == 0,
              "wgrad: C must be an fp32 [L, M, N] view with 16-byte aligned rows");
  if (K == 0 || L == 0) return;
  auto mat = [](const at::Tensor& t) { return Mat{t.data_ptr(), t.size(0), t.size(1), t.size(2), t.stride(0), t.stride(1)}; };
  run_wgrad(mat(A), mat(B), C, wgrad_plan(L, K, M, N, l_sum), err.data_ptr<int>(), false);
}

// The weight gradient of tc_wgrad (A [L, K, M], B [L, K, N], bf16) as a new tensor [L, M, N] (l_sum: [M, N]) of a type, on the
// current device and stream. Where one split covers the rows a tile leaves in that type at once (fp32 or bf16); else it is
// added up in fp32 and converted.
at::Tensor wgrad_as(const Mat& A, const Mat& B, const at::Device& device, int* err, bool l_sum, int64_t dtype) {
  const int64_t L = A.L, K = A.rows, M = A.cols, N = B.cols, LC = l_sum ? 1 : L;
  const auto type = at::ScalarType(dtype);
  PD_CHECK(B.L == L && B.rows == K, "B must be [L, K, N] over the same rows as A");
  PD_CHECK(M % 64 == 0 && N % 64 == 0, "wgrad: M and N must be multiples of 64");
  PD_CHECK(K < (int64_t(1) << 31) && L * ((K + 63) / 64) < (int64_t(1) << 30), "wgrad: too many rows");
  auto out = [&](bool zeros, at::ScalarType t) {
    const auto options = at::TensorOptions().dtype(t).device(device);
    const std::vector<int64_t> shape = {LC, M, N};
    return zeros ? at::zeros(shape, options) : at::empty(shape, options);
  };
  at::Tensor C;
  if (K == 0 || L == 0) {
    C = out(true, type);
  } else if (const tc::WgParams wide = wgrad_wide_plan(L, K, M, N, l_sum); M % 256 == 0 && N % 256 == 0 && wide.splits > 1) {
    C = out(true, at::kFloat);
    run_wgrad_wide(A, B, C, wide, err);
    C = C.to(type);
  } else {
    const tc::WgParams p = wgrad_plan(L, K, M, N, l_sum);
    const bool direct = p.splits == 1 && (type == at::kFloat || type == at::kBFloat16);
    C = out(!direct, direct ? type : at::kFloat);
    run_wgrad(A, B, C, p, err, direct);
    C = C.to(type);
  }
  return l_sum ? C.squeeze(0) : C;
}

}  // namespace pd
