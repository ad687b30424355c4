// Attention over the paged 8-bit cache for many rows (prompts, pieces of
// prompts) on the 5th-generation tensor cores, heads of 32 or 64.
//
// Same sums as kv_attn.cu. A block takes 128 rows (query, head of the group)
// of one sequence and key head and walks over the keys they see, 64 at a time:
//
//   warp 0      copies: TMA loads of codes (four tiles), and the scales of their pages
//   warps 2, 3  conversion: e4m3 codes -> fp16 operand tiles in the swizzled layout that the products read
//   warp 1      products, issued by one lane: S = Q K^T two tiles ahead of the softmax, O += P V (P from TMEM)
//   warps 4-7   softmax, a thread a row: 64 scores from TMEM to registers, P (fp16) back over them
//
// With heads this small the exponentials and the softmax's instructions bound
// the kernel, not the products: 128 x 64 scores cost 512 cycles of the
// exponential unit and 128 (d = 32) or 256 (d = 64) of the tensor pipe. So the
// conversion (once a tile for all rows) and the products run beside the
// softmax, and two blocks an SM fill each other's gaps.
//
// A page's key scale multiplies its 16 to 64 columns of scores; its value
// scale goes into the exponent, relative to a reference of the row, and out of
// the sum again. Products of probability and relative scale are held as 2^7
// times themselves. A row's maximum, and its reference (the largest product that
// it has seen), are raised only when they grow by more than 2^8, so the output
// in TMEM is seldom scaled. Pages of 64 (one pair of scales a tile) have a
// variant of their own: 153 us below, 164 with the general one. TMEM (256 columns): S / P of tile t at 64 (t % 3), O at 192.
//
// B200: 12 prompts of 911 to 1824 tokens, 16 x 64: 153 us, 298 TFLOP/s of the
// products that the mask leaves (floor 27 us by the products, 45 by the
// exponentials); the same on mma.sync took 254 us. Of the 2890 cycles that a block
// spent on a tile (at 154 us, before rows had references), the softmax warps worked 2400 (two warps a sub-partition, each
// waiting on its own chain) and the issuing lane 1800 (100 to 200 a product).
// The exponential unit is 37% and issue slots 41% busy. Four more softmax warps, each
// pair of warps sharing a quarter of the rows, took 160 us, and 164 to 186 with the
// two products issued by different warps.
//
// Waits are bounded; where one runs out the error word is set, every role
// leaves its loop and the block drains what it has issued.
#include <c10/cuda/CUDAGuard.h>

#include "kv_attn.cuh"

namespace pd {
namespace kv {

constexpr int kTcRows = 128;
constexpr int kTcThreads = 256;
constexpr int kRaw = 4;                 // tiles of codes in flight
constexpr int kOps = 3;                 // operand tiles, and S / P buffers
constexpr int kSc = 8;                  // tiles whose scales are kept (writer and reader are at most kRaw + kOps apart)

__device__ __forceinline__ void mbar_init(uint64_t* b, int n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(n));
}
__device__ __forceinline__ void mbar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory");
}
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_commit(uint64_t* b) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(b)) : "memory");
}
// D (TMEM) (+)= A (shared memory) * B (shared memory)
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      ::"r"(d), "l"(a), "l"(b), "r"(id), "r"(uint32_t(add)) : "memory");
}
// D (TMEM) (+)= A (TMEM, fp16 pairs) * B (shared memory)
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(d), "r"(a), "l"(b), "r"(id), "r"(uint32_t(add)) : "memory");
}
#define PD_R8(r, i) "=r"(r[i]), "=r"(r[i + 1]), "=r"(r[i + 2]), "=r"(r[i + 3]), "=r"(r[i + 4]), "=r"(r[i + 5]), "=r"(r[i + 6]), "=r"(r[i + 7])
#define PD_W8(r, i) "r"(r[i]), "r"(r[i + 1]), "r"(r[i + 2]), "r"(r[i + 3]), "r"(r[i + 4]), "r"(r[i + 5]), "r"(r[i + 6]), "r"(r[i + 7])
// 32 columns of this thread's TMEM lane
__device__ __forceinline__ void tm_ld32(uint32_t at, uint32_t* r) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : PD_R8(r, 0), PD_R8(r, 8), PD_R8(r, 16), PD_R8(r, 24) : "r"(at));
}
__device__ __forceinline__ void tm_st32(uint32_t at, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(at), PD_W8(r, 0), PD_W8(r, 8), PD_W8(r, 16), PD_W8(r, 24) : "memory");
}
// waits for loads, and names their registers so that no use moves in front of it
#define PD_RW8(r, i) "+r"(r[i]), "+r"(r[i + 1]), "+r"(r[i + 2]), "+r"(r[i + 3]), "+r"(r[i + 4]), "+r"(r[i + 5]), "+r"(r[i + 6]), "+r"(r[i + 7])
__device__ __forceinline__ void tm_ld_wait(uint32_t* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" : PD_RW8(r, 0), PD_RW8(r, 8), PD_RW8(r, 16), PD_RW8(r, 24)::"memory");
}
__device__ __forceinline__ void tm_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
#undef PD_R8
#undef PD_W8
#undef PD_RW8

// Operand tiles of fp16 rows of D elements: rows of 2 D bytes, 8-row atoms,
// chunks of 16 bytes exchanged within a row (64- or 128-byte swizzle).
template <int D>
struct Op {
  static constexpr uint32_t kRow = 2 * D, kAtom = 8 * kRow;
  static constexpr uint64_t kSwizzle = D == 32 ? 4 : 2;
  __device__ static __forceinline__ uint32_t chunk(int row, int c) {          // byte offset of chunk c of a row
    return row * kRow + uint32_t(c ^ (D == 32 ? (row >> 1) & 3 : row & 7)) * 16;
  }
  __device__ static __forceinline__ uint64_t desc(uint32_t at, uint32_t lead) {
    return uint64_t((at >> 4) & 0x3FFF) | (uint64_t((lead >> 4) & 0x3FFF) << 16) |
           (uint64_t((kAtom >> 4) & 0x3FFF) << 32) | (uint64_t(1) << 46) | (kSwizzle << 61);
  }
  // Descriptors of step 0 of 16 dims (rows = M or N) and of 16 rows (rows = K, dims = N) of a tile; those of another
  // step or tile differ by the distance in 16-byte units, whose sum stays within the 14 bits of an address.
  __device__ static __forceinline__ uint64_t dims(uint32_t tile) { return desc(tile, 16); }
  __device__ static __forceinline__ uint64_t rows(uint32_t tile) { return desc(tile, kUnit * kRow); }
  static constexpr uint32_t kDims = 32 / 16, kRows = 2 * kAtom / 16, kTile = kUnit * kRow / 16;
};
// fp16 operands, 32-bit sums; b_mn: B's rows are its K
constexpr uint32_t tc_id(int m, int n, int b_mn) {
  return (1u << 4) | (uint32_t(b_mn) << 16) | (uint32_t(n >> 3) << 17) | (uint32_t(m >> 4) << 24);
}

template <int D, bool ONE>               // ONE: a page holds a whole tile of keys, so a tile has one pair of scales
__global__ void __launch_bounds__(kTcThreads, 2)
paged_attn_tc_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap tm_k,
                     const __grid_constant__ CUtensorMap tm_v) {
  constexpr int kOpBytes = kUnit * Op<D>::kRow, kRawBytes = kUnit * D;
  constexpr uint32_t kCols = 256, cO = kOps * kUnit;
  extern __shared__ __align__(1024) uint8_t s_tiles[];      // Q, kOps x K, kOps x V (fp16), kRaw x (codes of K, of V)
  __shared__ uint64_t raw_full[kRaw], raw_empty[kRaw], sc_full[kSc], kv_full[kOps], kv_empty[kOps];
  __shared__ uint64_t s_full[kOps], p_full[kOps], pv_done[kOps], q_full, o_full, mma_done;
  __shared__ float s_ks[kSc][4], s_lv[kSc][4];              // scales of a tile's pages: keys, log2 of values'
  __shared__ uint32_t s_gone[kSc];
  __shared__ uint32_t s_tmem;
  __shared__ volatile int s_abort;

  if (!tiles_aligned(s_tiles, A.err)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / A.H, h = blockIdx.x % A.H, mt = gridDim.y - 1 - blockIdx.y;
  Seq<kTcRows> S;
  S.load(A, b);
  if (S.gaps(A, b))
    clear_gaps<D>(A, b, b + 1, h * A.G, A.G, mt * kTcThreads + threadIdx.x, gridDim.y * kTcThreads);
  if (mt >= S.tiles_m) return;
  const int rows = S.n * A.G, r0 = mt * kTcRows;
  const int last = min(r0 + kTcRows, rows) - 1;
  const int lim = A.causal ? max(0, S.len - S.n + last / A.G + 1) : S.len;    // keys that the last row sees
  const int units = (lim + kUnit - 1) / kUnit;
  const int* table = A.table + b * A.table_stride;
  const uint32_t sQ = smem_u32(s_tiles), sK = sQ + kTcRows * Op<D>::kRow, sV = sK + kOps * kOpBytes;
  const uint32_t sRaw = sV + kOps * kOpBytes;

  if (threadIdx.x == 0) {
    for (int i = 0; i < kRaw; ++i) { mbar_init(&raw_full[i], 1); mbar_init(&raw_empty[i], 64); }
    for (int i = 0; i < kSc; ++i) mbar_init(&sc_full[i], 1);
    for (int i = 0; i < kOps; ++i) {
      mbar_init(&kv_full[i], 64);
      mbar_init(&kv_empty[i], 1);
      mbar_init(&s_full[i], 1);
      mbar_init(&p_full[i], kTcRows);
      mbar_init(&pv_done[i], 1);
    }
    mbar_init(&q_full, kTcRows);
    mbar_init(&o_full, 1);
    mbar_init(&mma_done, 1);
    s_abort = 0;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                 ::"r"(smem_u32(&s_tmem)), "r"(kCols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = s_tmem;
  auto aborted = [&]() { return __any_sync(0xffffffffu, s_abort != 0); };    // one answer for a whole warp
  auto wait = [&](uint64_t* bar, int turn) { return mbar_wait(smem_u32(bar), uint32_t(turn) & 1u, A.err); };

  // the softmax warps take the registers that the others do not need: (64 + 192) x 128 = 128 x 256
  if (warp < 4) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == 0) {
      // ---------------- copies ----------------
      const int boxes = kUnit >> A.logP;
      int page = -1, pending = -1, issued = 0;
      float new_ks = 0.f, new_vs = 0.f;
      uint32_t new_gone = 0;
      auto fetch = [&](int v) {
        const int key = v * kUnit + lane * A.P;
        page = lane < boxes && key < lim ? __ldg(table + (key >> A.logP)) : -1;
      };
      auto settle = [&]() {                   // the scales of the tile before have arrived
        if (pending < 0) return;
        const int e = pending % kSc;
        if (lane < boxes) {
          s_ks[e][lane] = new_ks;
          s_lv[e][lane] = scale_log2_of(new_vs);
        }
        if (lane == 0) s_gone[e] = new_gone;
        __syncwarp();
        if (lane == 0) mbar_arrive(&sc_full[e]);
        pending = -1;
      };
      fetch(0);
      bool ok = true;
      for (int v = 0; v < units && !aborted(); ++v) {
        const int sl = v % kRaw;
        const bool want = lane < boxes && v * kUnit + lane * A.P < lim;
        const bool have = want && page >= 0 && page < A.n_pages;
        if (want && !have) set_error(A.err, kIdOutOfRange);
        const int block = have ? page * A.H + h : 0;
        const uint32_t mask = __ballot_sync(0xffffffffu, have);
        settle();
        if (v >= kRaw) ok = wait(&raw_empty[sl], v / kRaw - 1);
        if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
        const uint32_t full = smem_u32(&raw_full[sl]), dst = sRaw + sl * 2 * kRawBytes;
        if (lane == 0)
          asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                       ::"r"(full), "r"(uint32_t(__popc(mask) * 2 * A.P * D)) : "memory");
#pragma unroll 1
        for (int i = 0; i < boxes; ++i) {
          const int row = __shfl_sync(0xffffffffu, block, i) * A.P;
          if (lane == 0 && (mask >> i & 1)) {
            tma_rows(dst + i * A.P * D, &tm_k, full, row);
            tma_rows(dst + kRawBytes + i * A.P * D, &tm_v, full, row);
          }
        }
        new_ks = have ? __ldg(A.ks + block) : 0.f;
        new_vs = have ? __ldg(A.vs + block) : 0.f;
        new_gone = ~mask;
        pending = v;
        issued = v + 1;
        fetch(v + 1);
      }
      settle();
      if (!ok) s_abort = 1;
      // Every copy lands before the block may end, whichever role gives up, and when; else the last ones are all that
      // this waits for.
      for (int v = max(0, issued - kRaw); v < issued; ++v) (void)wait(&raw_full[v % kRaw], v / kRaw);
    } else if (warp == 1) {
      // ---------------- products ----------------
      if (lane == 0 && units > 0) {
        constexpr uint32_t id_s = tc_id(kTcRows, kUnit, 0), id_pv = tc_id(kTcRows, D, 1);
        const uint64_t dq = Op<D>::dims(sQ), dk = Op<D>::dims(sK), dv = Op<D>::rows(sV);
        bool ok = wait(&q_full, 0);
        auto scores = [&](int t) {
          const int sl = t % kOps;
          if (!wait(&kv_full[sl], t / kOps)) return false;
          if (t >= kOps && !wait(&pv_done[sl], t / kOps - 1)) return false;
          tc_after();
#pragma unroll
          for (int k = 0; k < D / 16; ++k)
            mma_ss(tmem + kUnit * sl, dq + k * Op<D>::kDims, dk + sl * Op<D>::kTile + k * Op<D>::kDims, id_s, k > 0);
          tc_commit(&s_full[sl]);
          return true;
        };
        for (int t = 0; t < 2 && t < units && ok; ++t) ok = scores(t);
        for (int t = 0; t < units && ok && !s_abort; ++t) {
          const int sl = t % kOps;
          ok = wait(&p_full[sl], t / kOps);
          if (!ok) break;
          tc_after();
#pragma unroll
          for (int k = 0; k < kUnit / 16; ++k)
            mma_ts(tmem + cO, tmem + kUnit * sl + 8 * k, dv + sl * Op<D>::kTile + k * Op<D>::kRows, id_pv, t > 0 || k > 0);
          tc_commit(&kv_empty[sl]);
          tc_commit(&pv_done[sl]);
          if (t + 1 == units) tc_commit(&o_full);
          if (t + 2 < units) ok = scores(t + 2);
        }
        if (!ok) s_abort = 1;
        tc_commit(&mma_done);
        (void)wait(&mma_done, 0);
      }
    } else {
      // ---------------- conversion ----------------
      const int ct = threadIdx.x - 64;
      constexpr int C = D / 16;               // chunks of 16 codes of a row
      const int row0 = ct / C;                // this thread converts chunk ct % C of rows row0, row0 + 64 / C, ...
      const uint32_t to0 = Op<D>::chunk(row0, 2 * (ct % C)), to1 = Op<D>::chunk(row0, 2 * (ct % C) + 1);
      bool ok = true;
      for (int v = 0; v < units && ok && !s_abort; ++v) {
        const int sl = v % kRaw, op = v % kOps, e = v % kSc;
        ok = wait(&raw_full[sl], v / kRaw) && wait(&sc_full[e], v / kSc);
        if (ok && v >= kOps) ok = wait(&kv_empty[op], v / kOps - 1);
        if (!ok) break;
        const uint32_t gone = s_gone[e];
        const int keys = min(kUnit, lim - v * kUnit);         // of the tile that some row sees
        const bool whole = keys == kUnit && !(gone & ((2u << ((kUnit - 1) >> A.logP)) - 1));
        const uint32_t src = sRaw + sl * 2 * kRawBytes + ct * 16;
#pragma unroll
        for (int half = 0; half < 2; ++half) {                // keys, values
          uint4 u[C];
#pragma unroll
          for (int i = 0; i < C; ++i) u[i] = lds128(src + half * kRawBytes + i * 1024);
          if (half == 1 && !whole) {
            // values behind the keys may be anything, NaN too; scores of such keys are masked
#pragma unroll
            for (int i = 0; i < C; ++i) {
              const int row = row0 + i * (64 / C);
              if (row >= keys || (gone >> (row >> A.logP) & 1)) u[i] = make_uint4(0, 0, 0, 0);
            }
          }
          const uint32_t dst = (half ? sV : sK) + op * kOpBytes;
#pragma unroll
          for (int i = 0; i < C; ++i) {
            uint32_t w[8];
            cvt4(u[i].x, w[0], w[1]);
            cvt4(u[i].y, w[2], w[3]);
            cvt4(u[i].z, w[4], w[5]);
            cvt4(u[i].w, w[6], w[7]);
            const uint32_t at = dst + i * (64 / C) * Op<D>::kRow;       // the exchange of chunks repeats every 8 rows
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + to0), "r"(w[0]), "r"(w[1]), "r"(w[2]),
                         "r"(w[3]) : "memory");
            asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at + to1), "r"(w[4]), "r"(w[5]), "r"(w[6]),
                         "r"(w[7]) : "memory");
          }
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        mbar_arrive(&kv_full[op]);
        mbar_arrive(&raw_empty[sl]);
      }
      if (!ok) s_abort = 1;
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
    // ---------------- softmax, a thread a row ----------------
    const int quarter = warp & 3, r = quarter * 32 + lane, row = r0 + r;
    const uint32_t lane_base = tmem + (uint32_t(quarter * 32) << 16);
    const bool live = row < rows;
    const int qi = live ? row / A.G : 0;
    const int my_lim = !live ? 0 : A.causal ? max(0, S.len - S.n + qi + 1) : S.len;
    float rs;                               // softmax scale of the row, in the log2 domain
    {
      const uint16_t* src = static_cast<const uint16_t*>(A.q) +
                            (A.cu ? int64_t(S.tok0 + qi) * A.q_ts : int64_t(b) * A.q_bs + int64_t(qi) * A.q_ts) +
                            int64_t(h * A.G + (live ? row - qi * A.G : 0)) * A.q_hs;
      float x[D];
#pragma unroll
      for (int e = 0; e < D; ++e) x[e] = 0.f;
      if (live) load_row<D>(src, A.bf16, x);
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < D; ++e) amax = fmaxf(amax, fabsf(x[e]));
      const float up = row_scale(amax, A.scale_log2, rs);
#pragma unroll
      for (int c = 0; c < D / 8; ++c)
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(sQ + Op<D>::chunk(r, c)),
                     "r"(pack_f16(x[8 * c] * up, x[8 * c + 1] * up)), "r"(pack_f16(x[8 * c + 2] * up, x[8 * c + 3] * up)),
                     "r"(pack_f16(x[8 * c + 4] * up, x[8 * c + 5] * up)),
                     "r"(pack_f16(x[8 * c + 6] * up, x[8 * c + 7] * up)) : "memory");
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      mbar_arrive(&q_full);
    }
    float m = -INFINITY, w = 0.f;           // running maximum; log2 of the value reference, relative to it
    uint64_t l2 = pk2(0.f, 0.f);
    bool ok = true;
    for (int t = 0; t < units && ok && !aborted(); ++t) {
      const int sl = t % kOps, e = t % kSc, k0 = t * kUnit;
      ok = wait(&sc_full[e], t / kSc) && wait(&s_full[sl], t / kOps);
      if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
      tc_after();
      float f[4], lv[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int pg = ONE ? 0 : (16 * i) >> A.logP;
        f[i] = ONE && i > 0 ? f[0] : fmaxf(s_ks[e][pg] * rs, kTiny);
        lv[i] = ONE && i > 0 ? lv[0] : s_lv[e][pg];
      }
      const bool large = __any_sync(0xffffffffu, fmaxf(fmaxf(f[0], f[1]), fmaxf(f[2], f[3])) >= kLargeFactor);
      uint32_t sr[64];
      tm_ld32(lane_base + kUnit * sl, sr);
      tm_ld32(lane_base + kUnit * sl + 32, sr + 32);
      tm_ld_wait(sr);
      tm_ld_wait(sr + 32);
      const uint32_t gone = s_gone[e];
      if (large) {
        // the products of scores and factors are rounded by themselves, as those of the maximum are; 7 - m is then at most
        // 8 - m in 32 bits, and no score passes m
#pragma unroll
        for (int c = 0; c < 64; ++c) sr[c] = __float_as_uint(__fmul_rn(__uint_as_float(sr[c]), f[c / 16]));
        f[0] = f[1] = f[2] = f[3] = 1.f;
      }
      const int see = my_lim - k0;                          // columns c < see are visible
      if (__any_sync(0xffffffffu, see < kUnit)) {
#pragma unroll
        for (int c = 0; c < 64; ++c) sr[c] = c < see ? sr[c] : __float_as_uint(-INFINITY);
      }
      const uint32_t seen = (2u << ((min(kUnit, lim - k0) - 1) >> A.logP)) - 1;
      if (gone & seen) {                                    // seldom: a page in front of the end is missing
#pragma unroll
        for (int c = 0; c < 64; ++c)
          if (gone >> (c >> A.logP) & 1) sr[c] = __float_as_uint(-INFINITY);
      }
      float y[4], mx = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
        for (int c = 16 * i; c < 16 * i + 16; c += 4) {
          y0 = fmaxf(y0, fmaxf(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])));
          y1 = fmaxf(y1, fmaxf(__uint_as_float(sr[c + 2]), __uint_as_float(sr[c + 3])));
        }
        y[i] = fmaxf(y0, y1) * f[i];
        mx = fmaxf(mx, y[i]);
      }
      if (ONE) y[0] = mx;
      // the running maximum and the value reference (relative to it) lag by up to 2^8
      const float lag = large ? 0.f : 8.f;
      const float top_m = mx > m + lag ? mx : m, base = top_m == -INFINITY ? 0.f : top_m;
      float v = -INFINITY;
#pragma unroll
      for (int i = 0; i < (ONE ? 1 : 4); ++i) v = fmaxf(v, (y[i] - base) + lv[i]);
      const float x = top_m == m ? w : w + (m - top_m);     // the reference as it is, relative to the new maximum
      if (__any_sync(0xffffffffu, mx > m + lag || v > x + lag)) {
        const float top_w = v > x + lag ? v : x, al = exp2f_approx(x - top_w);
        if (t > 0) {
          // the output is scaled once the products of the tile before, its last writers, are done
          ok = wait(&pv_done[(t - 1) % kOps], (t - 1) / kOps);
          if (!__all_sync(0xffffffffu, ok)) { ok = false; break; }
          tc_after();
#pragma unroll
          for (int c0 = 0; c0 < D; c0 += 32) {
            uint32_t o[32];
            tm_ld32(lane_base + cO + c0, o);
            tm_ld_wait(o);
#pragma unroll
            for (int c = 0; c < 32; ++c) o[c] = __float_as_uint(__uint_as_float(o[c]) * al);
            tm_st32(lane_base + cO + c0, o);
          }
          tm_st_wait();
        }
        if (top_m != m) l2 = pk2_mul(l2, pk2s(exp2f_approx(m - top_m)));
        m = top_m;
        w = top_w;
      }
      const float z = 7.f - base;
      float rel;                              // log2 of the page's factor
      uint32_t pk[32];
      uint64_t s0 = pk2(0.f, 0.f), s1 = s0;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (!ONE || i == 0) rel = fmaxf(lv[i] - w, kLeastRel);
        const uint64_t ff = pk2s(f[i]), zz = pk2s(z + rel);
        if (!ONE) s0 = s1 = pk2(0.f, 0.f);
#pragma unroll
        for (int c = 16 * i; c < 16 * i + 16; c += 2) {
          float p0, p1;
          pk2_split(pk2_fma(pk2(__uint_as_float(sr[c]), __uint_as_float(sr[c + 1])), ff, zz), p0, p1);
          p0 = exp2f_approx(p0);
          p1 = exp2f_approx(p1);
          if (c & 2) s1 = pk2_add(s1, pk2(p0, p1));
          else s0 = pk2_add(s0, pk2(p0, p1));
          pk[c / 2] = pack_f16(p0, p1);
        }
        if (!ONE || i == 3) l2 = pk2_fma(pk2_add(s0, s1), pk2s(exp2f_approx(-rel)), l2);
      }
      tm_st32(lane_base + kUnit * sl, pk);
      tm_st_wait();
      tc_before();
      mbar_arrive(&p_full[sl]);
    }
    if (ok && units > 0 && !aborted()) ok = wait(&o_full, 0);
    ok = __all_sync(0xffffffffu, ok);
    tc_after();
    float l, l1;
    pk2_split(l2, l, l1);
    l += l1;
    // a sum of 0: no keys. A NaN stays one. The reference may be near the largest number: half of it at a time
    const float half = exp2f_approx(0.5f * w), inv = l == 0.f ? 0.f : half / l;
    const int64_t at = int64_t(S.tok0 + qi) * A.Hq + h * A.G + (live ? row - qi * A.G : 0);
    uint16_t* dst = static_cast<uint16_t*>(A.o) + at * D;
    const auto out = [&](uint32_t v) { return __uint_as_float(v) * inv * half; };
#pragma unroll
    for (int c0 = 0; c0 < D; c0 += 32) {
      uint32_t o[32];
      if (units > 0) {
        tm_ld32(lane_base + cO + c0, o);
        tm_ld_wait(o);
      } else {
#pragma unroll
        for (int c = 0; c < 32; ++c) o[c] = 0;
      }
      if (live) {
#pragma unroll
        for (int c = 0; c < 32; c += 8)
          *reinterpret_cast<uint4*>(dst + c0 + c) =
              make_uint4(pack_16(out(o[c]), out(o[c + 1]), A.bf16), pack_16(out(o[c + 2]), out(o[c + 3]), A.bf16),
                         pack_16(out(o[c + 4]), out(o[c + 5]), A.bf16), pack_16(out(o[c + 6]), out(o[c + 7]), A.bf16));
      }
    }
    if (live && A.lse) A.lse[at] = l == 0.f ? -INFINITY : (m - 7.f + log2f(l)) * 0.6931471805599453f;
    if (!ok) s_abort = 1;
  }
  tc_before();
  __syncthreads();
  if (warp == 1) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kCols) : "memory");
  }
}

template <int D, bool ONE>
static void tc_launch(AttnArgs& A, const at::Tensor& ck, const at::Tensor& cv, const Bounds& U) {
  constexpr int kSmem = kTcRows * Op<D>::kRow + 2 * kOps * kUnit * Op<D>::kRow + kRaw * 2 * kUnit * D;
  static int known[64] = {};
  auto kern = paged_attn_tc_kernel<D, ONE>;
  blocks_per_sm(kern, kTcThreads, kSmem, known);
  const dim3 grid(unsigned(U.B * A.H), unsigned((U.rows + kTcRows - 1) / kTcRows));
  kern<<<grid, kTcThreads, kSmem, stream()>>>(A, code_map(ck, A.P, false), code_map(cv, A.P, false));
  PD_CHECK_LAUNCH();
}

void attn_tc_launch(AttnArgs& A, const at::Tensor& ck, const at::Tensor& cv, int d, const Bounds& U) {
  if (A.P == kUnit) d == 32 ? tc_launch<32, true>(A, ck, cv, U) : tc_launch<64, true>(A, ck, cv, U);
  else d == 32 ? tc_launch<32, false>(A, ck, cv, U) : tc_launch<64, false>(A, ck, cv, U);
}

}  // namespace kv
}  // namespace pd
