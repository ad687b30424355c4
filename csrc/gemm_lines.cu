// The GEMMs of the layers that keep their activations in 8 bits (ops/dense.py,
// save8): C[l] = f(A[l] @ B[l]^T), bf16 operands, fp32 sums.
//
//   kPlain  C = acc (+ R)
//   kSave   C = GELU(acc), the pre-activation acc leaves as 8-bit codes
//           (int8_common.cuh): a thread holds 32 columns of its row, one block
//           of codes, so maximum and scale take no exchange
//   kUse    p = the values of such codes; C = acc * GELU'(p), X = GELU(p)
//
// Roles as in gemm_tc.cu: TMA producer, one MMA lane, epilogue warps; sums
// double-buffered in TMEM. The difference is the way out: an epilogue unit is 64
// columns of 32 rows, so that a TMA store writes whole lines of 128 bytes, and the
// ring takes what 8 or 16 staged blocks of 4 KB leave (four stages of 48 KB for
// kPlain: of a stage only A comes from DRAM, and three in flight do not cover its
// latency). kUse has two results and room for one block a warp: two warps share a
// unit, 32 columns each, and its two blocks.
//
// Measured (1 B200, 100,608 rows): kSave 256 -> 1024 85 us for 361 MB (98 by
// half lines), kUse 128 us for 566 MB (146), both bound by their epilogues'
// instructions (17 and 26 an element); kPlain 1024 -> 256 with R 67 us for 308 MB,
// without 50 for 257 (gemm_tc.cu's kernel 70 and 60), bound by the operands' way
// into shared memory: about 1000 cycles a k-block of 48 KB. Two blocks on one tile
// of 256 rows (cta_group::2, 32 KB) took 45 us without R, but 95 and 143 in the
// forms with codes.
#include "gemm_host.h"
#include "gemm_mat.h"
#include "int8_common.cuh"
#include "tc_common.cuh"

#include <type_traits>

namespace pd {
namespace lines {

namespace tcx = pd::tc;

constexpr int BM = 128;
constexpr int BK = 64;
constexpr int kBlockBytes = 4096;       // a staged block: 32 rows of 128 bytes
enum Mode : int { kPlain = 0, kSave = 1, kUse = 2 };

// GELU's arithmetic wants more warps (an FFN 256 -> 1024 over 100,608 rows, both launches: kSave 118 us with 16, 128 with 8;
// kUse, with more arithmetic, has pairs of warps for 16 alone), the plain products want the room in shared memory.
constexpr int epi_warps(int mode) { return mode == kPlain ? 8 : 16; }
constexpr int threads_of(int mode) { return 64 + 32 * epi_warps(mode); }

struct Params {
  int M, N, L;
  int m_blocks, n_blocks, k_blocks, tiles;
  int a_mode, b_mode, c_mode, x_mode, r_mode;      // tensor maps' dim order: 0 = {inner, rows, L}, 1 = {inner, L, rows}
  int b_shared;                                     // B has one batch shared by every l
  int b_kn;                                         // B stored [L, K, N] (a weight used transposed), loaded MN-major
  int has_r;                                        // (kPlain) R is added
  int8_t* X8; int64_t x8_ls, x8_ms;                 // codes [L, M, N]
  uint8_t* E; int64_t e_ls, e_ms, e_bs;             // scale bytes [L, M, N / 32]
  int* err;
};

__device__ __forceinline__ void tile_at(const Params& p, int w, int& l, int& mb, int& nb) {
  nb = w % p.n_blocks;
  const int r = w / p.n_blocks;
  mb = r % p.m_blocks;
  l = r / p.m_blocks;
}

// 16-byte chunk c (0..7) of row r of a staged block, in the TMA's 128-byte swizzle
__device__ __forceinline__ int staged(int r, int c) { return r * 128 + ((c ^ (r & 7)) << 4); }

__device__ __forceinline__ uint4 pack8(const float* v) {
  uint32_t w[4];
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(v[2 * e], v[2 * e + 1]);
    w[e] = *reinterpret_cast<const uint32_t*>(&h);
  }
  return make_uint4(w[0], w[1], w[2], w[3]);
}

template <int BN, int STAGES, int MODE>
__global__ void __launch_bounds__(threads_of(MODE), 1) lines_kernel(const __grid_constant__ CUtensorMap tmA,
                                                                    const __grid_constant__ CUtensorMap tmB,
                                                                    const __grid_constant__ CUtensorMap tmC,
                                                                    const __grid_constant__ CUtensorMap tmX,
                                                                    const __grid_constant__ CUtensorMap tmR, const Params p) {
  constexpr int kEw = epi_warps(MODE), kParts = kEw / 4;
  constexpr uint32_t kA = BM * BK * 2, kB = BN * BK * 2, kCols = 2 * BN;
  extern __shared__ __align__(1024) uint8_t line_ring[];  // A tiles, B tiles, staged blocks
  __shared__ uint64_t full[STAGES], empty[STAGES], tfull[2], tempty[2], mma_done;
  __shared__ uint64_t rbar[8];                            // (kPlain) a warp's R block has landed
  __shared__ uint64_t pair_filled[8], pair_free[8];       // (kUse) a pair's blocks are written, and may be written again
  __shared__ uint32_t tmem_slot;
  __shared__ volatile int abort_flag;
  if (tcx::smem_u32(line_ring) % 1024 != 0) {             // the swizzled tiles need it
    set_error(p.err, kBadShape);
    tcx::wait_for_launch_before();                        // kernels behind this one count on it
    return;
  }
  uint8_t* sA = line_ring;
  uint8_t* sB = line_ring + STAGES * kA;
  uint8_t* blocks = line_ring + STAGES * (kA + kB);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) { tcx::mbar_init(&full[s], 1); tcx::mbar_init(&empty[s], 1); }
    for (int a = 0; a < 2; ++a) { tcx::mbar_init(&tfull[a], 1); tcx::mbar_init(&tempty[a], kEw * 32); }
    for (int i = 0; i < 8; ++i) {
      tcx::mbar_init(&rbar[i], 1);
      tcx::mbar_init(&pair_filled[i], 2);
      tcx::mbar_init(&pair_free[i], 1);
    }
    tcx::mbar_init(&mma_done, 1);
    abort_flag = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmA) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmB) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tmC) : "memory");
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
  tcx::wait_for_launch_before();
  tcx::let_next_launch();

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
          if (p.b_kn) {
#pragma unroll
            for (int g = 0; g < BN / 64; ++g)             // [64 k-rows][64 n] boxes
              tcx::tma_load_rows(sB + stage * kB + g * 8192, &tmB, &full[stage], p.b_mode, nb * BN + 64 * g, kb * BK,
                                 p.b_shared ? 0 : l);
          } else {
            tcx::tma_load_rows(sB + stage * kB, &tmB, &full[stage], p.b_mode, kb * BK, nb * BN, p.b_shared ? 0 : l);
          }
          ++issued;
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
      if (abort_flag) {                                   // every issued load lands before the block may exit
        for (int s = 0; s < STAGES; ++s) {
          const int n = (issued - s + STAGES - 1) / STAGES;
          if (n > 0) (void)tcx::mbar_wait(&full[s], uint32_t(n - 1) & 1u, p.err);
        }
      }
    }
  } else if (warp == 1) {
    // ---------------- MMA issuer ----------------
    if (lane == 0) {
      const uint32_t idesc = tcx::instr_desc(BM, BN) | (p.b_kn ? (1u << 16) : 0u);          // B MN-major
      int stage = 0, local = 0;
      uint32_t phase = 0;
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
          for (int k = 0; k < BK / 16; ++k) {
            const uint64_t db = p.b_kn ? tcx::smem_desc_mn(b_addr + k * 2048) : tcx::smem_desc(b_addr + k * 32);
            tcx::tc_mma(d, tcx::smem_desc(a_addr + k * 32), db, idesc, (kb | k) ? 1u : 0u);
          }
          tcx::tc_commit(&empty[stage]);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
        if (!ok) break;
        tcx::tc_commit(&tfull[a]);
      }
      tcx::tc_commit(&mma_done);                          // all issued products have finished before TMEM is freed
      (void)tcx::mbar_wait(&mma_done, 0, p.err);
    }
  } else if constexpr (MODE != kUse) {
    // ---------------- epilogue: a warp's units are 64 columns of its 32 rows ----------------
    const int ew = warp - 2, q = warp & 3, part = ew >> 2;
    uint8_t* st = blocks + ew * kBlockBytes;
    const bool has_r = MODE == kPlain && p.has_r;
    int unit = 0;                                         // of this warp, counted: the phase of its R barrier
    bool r_pending = false, ok = true;
    auto request_r = [&](int l, int m0, int n) {          // R lands in the staged block itself: C overwrites it in place
      if (lane == 0) {
        tcx::bulk_wait_read_all();                        // the block's last store has read it
        tcx::mbar_expect_tx(&rbar[ew & 7], kBlockBytes);
        tcx::tma_load_rows(st, &tmR, &rbar[ew & 7], p.r_mode, n, m0, l);
      }
      r_pending = true;
    };
    int local = 0;
    for (int w = blockIdx.x; w < p.tiles && ok; w += gridDim.x, ++local) {
      const int a = local & 1;
      int l, mb, nb;
      tile_at(p, w, l, mb, nb);
      const int m0 = mb * BM + q * 32, n0 = nb * BN, row = m0 + lane;
      if (has_r && part * 64 < BN) request_r(l, m0, n0 + part * 64);
      if (!tcx::mbar_wait(&tfull[a], (local >> 1) & 1, p.err)) { abort_flag = 1; break; }
      tcx::tc_fence_after();
      const uint32_t tbase = tmem + (uint32_t(q * 32) << 16) + uint32_t(a * BN);
#pragma unroll 1
      for (int c = part * 64; c < BN; c += kParts * 64, ++unit) {
        if (has_r) {
          if (c != part * 64) request_r(l, m0, n0 + c);
          ok = tcx::mbar_wait(&rbar[ew & 7], uint32_t(unit) & 1u, p.err);
          if (!ok) { abort_flag = 1; break; }
          r_pending = false;
        } else {
          if (lane == 0) tcx::bulk_wait_read_all();
          __syncwarp();
        }
#pragma unroll 1
        for (int h = 0; h < 64; h += 32) {
          uint32_t r[32];
          tcx::tc_ld32_issue(tbase + c + h, r);
          tcx::tc_ld_wait(r);
          float v[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) v[i] = __uint_as_float(r[i]);
          if constexpr (MODE == kSave) {
            uint32_t code[8];
            const uint32_t byte = i8::save_block(v, i8::kTopWide, code);
            if (row < p.M) {
              uint4* dst = reinterpret_cast<uint4*>(p.X8 + l * p.x8_ls + int64_t(row) * p.x8_ms + n0 + c + h);
              dst[0] = make_uint4(code[0], code[1], code[2], code[3]);
              dst[1] = make_uint4(code[4], code[5], code[6], code[7]);
              p.E[l * p.e_ls + row * p.e_ms + ((n0 + c + h) >> 5) * p.e_bs] = uint8_t(byte);
            }
#pragma unroll
            for (int i = 0; i < 32; i += 2) gelu2(v[i], v[i + 1]);
          }
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            uint4* at = reinterpret_cast<uint4*>(st + staged(lane, h / 8 + j));
            if (has_r) {
              const uint4 x = *at;
              const __nv_bfloat162* e = reinterpret_cast<const __nv_bfloat162*>(&x);
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                const float2 f = __bfloat1622float2(e[i]);
                v[8 * j + 2 * i] += f.x;
                v[8 * j + 2 * i + 1] += f.y;
              }
            }
            *at = pack8(v + 8 * j);
          }
        }
        tcx::fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          tcx::tma_store_rows(&tmC, st, p.c_mode, n0 + c, m0, l);
          tcx::bulk_commit();
        }
      }
      tcx::tc_fence_before();
      tcx::mbar_arrive(&tempty[a]);
    }
    if (r_pending) (void)tcx::mbar_wait(&rbar[ew & 7], uint32_t(unit) & 1u, p.err);         // lands before the block exits
    if (lane == 0) tcx::bulk_wait_all();
    __syncwarp();
  } else {
    // ---------------- epilogue (kUse): two warps share a unit, 32 columns each, and its blocks of C and X ----------------
    const int ew = warp - 2, q = warp & 3, part = ew >> 2, half = part & 1;
    const int pair = (part >> 1) * 4 + q;
    uint8_t* stC = blocks + pair * 2 * kBlockBytes;
    uint8_t* stX = stC + kBlockBytes;
    // the codes and scale byte of this thread's next row and columns, on their way
    uint4 code0 = make_uint4(0, 0, 0, 0), code1 = code0;
    uint32_t code_scale = 1;
    auto load_codes = [&](int w, int u) {
      int l, mb, nb;
      tile_at(p, w, l, mb, nb);
      const int m = mb * BM + q * 32 + lane, n = nb * BN + u * 64 + half * 32;
      if (m < p.M) {
        const uint4* src = reinterpret_cast<const uint4*>(p.X8 + l * p.x8_ls + int64_t(m) * p.x8_ms + n);
        code0 = __ldcs(src);
        code1 = __ldcs(src + 1);
        code_scale = p.E[l * p.e_ls + m * p.e_ms + (n >> 5) * p.e_bs];
      }
    };
    constexpr int kUnits = BN / 64;
    const int first = part >> 1;                          // this pair's units: first, first + 2, ...
    if (first < kUnits && blockIdx.x < p.tiles) load_codes(blockIdx.x, first);
    int unit = 0;                                         // of this pair, counted: the phase of its barriers
    bool ok = true;
    int local = 0;
    for (int w = blockIdx.x; w < p.tiles && ok; w += gridDim.x, ++local) {
      const int a = local & 1;
      if (!tcx::mbar_wait(&tfull[a], (local >> 1) & 1, p.err)) { abort_flag = 1; break; }
      tcx::tc_fence_after();
      int l, mb, nb;
      tile_at(p, w, l, mb, nb);
      const int m0 = mb * BM + q * 32, n0 = nb * BN;
      const uint32_t tbase = tmem + (uint32_t(q * 32) << 16) + uint32_t(a * BN) + uint32_t(half * 32);
#pragma unroll 1
      for (int u = first; u < kUnits; u += 2, ++unit) {
        uint32_t r[32];
        tcx::tc_ld32_issue(tbase + u * 64, r);
        const uint32_t code[8] = {code0.x, code0.y, code0.z, code0.w, code1.x, code1.y, code1.z, code1.w};
        const float scale = i8::scale_of(code_scale);
        if (u + 2 < kUnits) load_codes(w, u + 2);
        else if (w + gridDim.x < p.tiles) load_codes(w + gridDim.x, first);
        // the pair's last stores have read its blocks
        if (unit > 0) {
          if (half == 0 && lane == 0) {
            tcx::bulk_wait_read_all();
            tcx::mbar_arrive(&pair_free[pair]);
          }
          ok = tcx::mbar_wait(&pair_free[pair], uint32_t(unit - 1) & 1u, p.err);
          if (!ok) { abort_flag = 1; break; }
        }
        tcx::tc_ld_wait(r);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          float g[8], v[8];
          i8::values4(code[2 * j], scale, g);
          i8::values4(code[2 * j + 1], scale, g + 4);
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float d0, d1;
            gelu_grad2<true>(g[e], g[e + 1], d0, d1);
            v[e] = __uint_as_float(r[8 * j + e]) * d0;
            v[e + 1] = __uint_as_float(r[8 * j + e + 1]) * d1;
          }
          *reinterpret_cast<uint4*>(stX + staged(lane, half * 4 + j)) = pack8(g);
          *reinterpret_cast<uint4*>(stC + staged(lane, half * 4 + j)) = pack8(v);
        }
        tcx::fence_async_smem();
        __syncwarp();
        if (lane == 0) tcx::mbar_arrive(&pair_filled[pair]);
        if (half == 0) {
          ok = tcx::mbar_wait(&pair_filled[pair], uint32_t(unit) & 1u, p.err);
          if (!ok) { abort_flag = 1; break; }
          if (lane == 0) {
            tcx::tma_store_rows(&tmC, stC, p.c_mode, n0 + u * 64, m0, l);
            tcx::tma_store_rows(&tmX, stX, p.x_mode, n0 + u * 64, m0, l);
            tcx::bulk_commit();
          }
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

}  // namespace lines

// ---------------------------------------------------------------------------
namespace {

template <int BN, int STAGES, int MODE>
void launch(const CUtensorMap& ta, const CUtensorMap& tb, const CUtensorMap& tcm, const CUtensorMap& tx, const CUtensorMap& tr,
            const lines::Params& p) {
  constexpr size_t smem = STAGES * size_t(lines::BM + BN) * lines::BK * 2 + lines::epi_warps(MODE) * size_t(lines::kBlockBytes);
  static_assert(smem + 2048 <= 232448, "shared memory of a block");
  static tc::SharedLimit limit;
  limit.allow(lines::lines_kernel<BN, STAGES, MODE>, smem);
  tc::launch_behind(lines::lines_kernel<BN, STAGES, MODE>, dim3(unsigned(std::min(p.tiles, num_sms()))),
                    lines::threads_of(MODE), smem, ta, tb, tcm, tx, tr, p);
}

void aligned(const Mat& t, const char* what) {            // bf16 rows on 16 bytes
  PD_CHECK(reinterpret_cast<uintptr_t>(t.p) % 16 == 0 && t.ms % 8 == 0 && (t.L == 1 || t.ls % 8 == 0),
           "%s: rows must lie on 16 bytes", what);
}

// The common part: operands checked, maps made; X or R where a mode has them.
void run(const Mat& A, const Mat& B, const Mat& C, const Mat* X, const Mat* R, const MatCodes* codes, int* err, bool b_kn,
         int mode) {
  const int64_t L = A.L, M = A.rows, K = A.cols, N = b_kn ? B.cols : B.rows;
  PD_CHECK((b_kn ? B.rows : B.cols) == K && (B.L == L || B.L == 1), "B must fit A");
  PD_CHECK(K % 8 == 0 && N % 64 == 0, "K must be a multiple of 8, N of 64");
  for (const Mat* t : {&C, X, R})
    PD_CHECK(t == nullptr || (t->L == L && t->rows == M && t->cols == N), "a result or addend does not fit the product");
  PD_CHECK(M < (int64_t(1) << 31) && L < (int64_t(1) << 31), "too many rows");
  if (M == 0 || L == 0) return;
  aligned(A, "A");
  aligned(B, "B");
  aligned(C, "C");
  if (X) aligned(*X, "X");
  if (R) aligned(*R, "R");
  if (codes)
    PD_CHECK(reinterpret_cast<uintptr_t>(codes->codes) % 16 == 0 && codes->ms % 16 == 0 && (L == 1 || codes->ls % 16 == 0),
             "codes: rows must lie on 16 bytes");
  lines::Params p{};
  p.M = int(M); p.N = int(N); p.L = int(L);
  p.m_blocks = int((M + lines::BM - 1) / lines::BM);
  p.k_blocks = int((K + lines::BK - 1) / lines::BK);
  const int BN = (N % 256 == 0) ? 256 : (N % 128 == 0 ? 128 : 64);
  p.n_blocks = int(N / BN);
  PD_CHECK(L * p.m_blocks * p.n_blocks < (int64_t(1) << 30), "too many rows");
  p.tiles = int(L) * p.m_blocks * p.n_blocks;
  p.b_kn = b_kn ? 1 : 0;
  p.b_shared = B.L == 1 ? 1 : 0;
  p.has_r = R ? 1 : 0;
  p.err = err;
  if (codes) {
    p.X8 = codes->codes; p.x8_ls = codes->ls; p.x8_ms = codes->ms;
    p.E = codes->bytes; p.e_ls = codes->e_ls; p.e_ms = codes->e_ms; p.e_bs = codes->e_bs;
  }
  auto map = [](const Mat& t, int box_rows, int& order) {
    return make_map(t.p, t.cols, t.rows, t.L, t.ms, t.ls, box_rows, order);
  };
  const CUtensorMap ta = map(A, lines::BM, p.a_mode), tb = map(B, b_kn ? lines::BK : BN, p.b_mode);
  // blocks of 64 columns (128 bytes) x 32 rows: an operand's map with another number of rows
  const CUtensorMap tcm = map(C, 32, p.c_mode);
  const CUtensorMap tx = X ? map(*X, 32, p.x_mode) : tcm, tr = R ? map(*R, 32, p.r_mode) : tcm;
  // rings: three stages of 48 KB beside 16 staged blocks, four beside 8
  auto go = [&](auto m) {
    constexpr int kMode = decltype(m)::value, kMore = kMode == lines::kPlain ? 1 : 0;
    if (BN == 256) launch<256, 3 + kMore, kMode>(ta, tb, tcm, tx, tr, p);
    else if (BN == 128) launch<128, 5 + kMore, kMode>(ta, tb, tcm, tx, tr, p);
    else launch<64, 6 + 2 * kMore, kMode>(ta, tb, tcm, tx, tr, p);
  };
  if (mode == lines::kPlain) go(std::integral_constant<int, lines::kPlain>());
  else if (mode == lines::kSave) go(std::integral_constant<int, lines::kSave>());
  else go(std::integral_constant<int, lines::kUse>());
}

}  // namespace

// All run on the current device and stream.
// C[l] = A[l] @ B[l]^T (+ R[l]): bf16, A [L, M, K], B [L or 1, N, K] -- or, with b_kn, [L or 1, K, N] -- C and R [L, M, N].
void gemm_lines(const Mat& A, const Mat& B, const Mat& C, const Mat* R, int* err, bool b_kn) {
  run(A, B, C, nullptr, R, nullptr, err, b_kn, lines::kPlain);
}
// The two GEMMs around pre-activations kept in 8 bits. Without X (the up projection): C = GELU(A @ B^T), the codes are
// written. With X (the down projection's data gradient): p = the codes' values, C = (A @ B^T) * GELU'(p), X = GELU(p).
void gemm_saved8(const Mat& A, const Mat& B, const Mat& C, const MatCodes& codes, const Mat* X, int* err, bool b_kn) {
  run(A, B, C, X, nullptr, &codes, err, b_kn, X ? lines::kUse : lines::kSave);
}

}  // namespace pd
