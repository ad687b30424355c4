// Attention over the paged 8-bit key/value cache.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,   k_j = code * key scale of j's page, v_j likewise
//
// The n new queries of a sequence are its last n tokens: query i of a sequence
// of len tokens sees the keys j <= len - n + i (all keys without the causal
// mask). A query without keys gives 0 (and -inf as its log-sum-exp).
//
// Arithmetic. Codes of e4m3 are exact in fp16, so both products run on fp16
// operands with 32-bit sums and no rounding of the cache's values: a query row
// is scaled by the power of two that brings its largest magnitude to
// [2^14, 2^15) (elements down to 2^-29 of it keep all bits of bf16) and the
// softmax scale undoes it. A page's key scale multiplies its scores in 32 bits,
// its value scale t = log2 its probabilities, in the exponent: a row's operand
// of the second product is 2^15 2^(s + t - w) with w the largest s + t of the
// tile's keys that it sees, 11 bits down to 2^-29 of the largest product and
// some down to 2^-39. Running maximum, sum (without t) and output stay in 32 bits.
#include "kv_attn.cuh"

namespace pd {
namespace kv {

template <int D> struct Cfg;
// TK keys of products and softmax at a time, SUB such tiles (8 KB of keys and values) to a copy, ST copies in flight
template <> struct Cfg<32> { static constexpr int TK = 64, SUB = 2, ST = 2; };
template <> struct Cfg<64> { static constexpr int TK = 64, SUB = 1, ST = 2; };
template <> struct Cfg<128> { static constexpr int TK = 32, SUB = 1, ST = 2; };

// A wait has run out: the n copies on their way, from slot st on, land before the block may end.
__device__ __noinline__ void drain(uint32_t bars, uint32_t slots, uint32_t st, uint32_t phase, int n, int* err) {
  for (int i = 0; i < n; ++i) {
    (void)mbar_wait(bars + st * 8, phase, err);
    if (++st == slots) {
      st = 0;
      phase ^= 1;
    }
  }
}

// Sums of 2^15 p v are held in this unit (few rows): 65536 of the largest 32-bit numbers fit, and the smallest page scale
// times it still has 18 bits.
constexpr float kSumUnit = 0x1p-31f, kSumLog2 = -31.f;

// Few rows to a segment (one or some query tokens of one sequence, the heads
// that share a key head): bound by reading the cache.
//
// W warps take a segment's keys in turn, a tile of TK keys each, from rings of
// their own that TMA fills (one copy a page, 32 to 128 bytes a row, swizzled by
// the hardware so that fragments load without bank conflicts); W = 1 where
// there are segments enough for every warp. Blocks (W = 4) take equal shares
// of all tiles of all segments where segments are few, their pieces are joined
// by a second launch.
//
// R = 16: a warp's rows are the A operand of S = Q K^T, R = 8 (up to 8 rows):
// keys and values are, S^T = K Q^T and O^T = V^T P^T, with half the products
// and registers; P^T turns from accumulator into operand by movmatrix. Dims
// are dealt to lanes so that a lane's four codes of a step of 16 dims are
// neighbours: lane % 4 owns a quarter of a key's dims, lane / 4 an eighth of a
// value's, and keys go to registers in the order of memory.
//
// ONE: pages hold whole tiles, which then have one pair of scales each (the
// single tokens below 111 us, the candidates 133; the general form 126 and 152).
//
// B200: 64 single tokens over 300 to 8191 keys, 32 heads over 8 x 128 (R = 8):
// 111 us, 5.0 TB/s of the cache (floor 85 us); three over 65537 to 131071 keys, 16
// heads over 4 x 64, pages of 16: 45 us, 3.4 TB/s (floor 23 us). Neither pipe is full (issue
// slots 38%, DRAM 75%): 12 warps an SM, bound by registers and the ring (by the ring
// alone at d = 64), wait on their own chains. 1024 x 16 candidate tokens behind 896 shared keys, 8 x 32 (R = 16, W =
// 1): 133 us; the keys come from L2 and the instructions around 16-row products
// bound it (issue 50% of active cycles; a copy's bookkeeping is 30% of them: 64
// keys a copy instead of 128 cost 179 us).
template <int D, int R, int W, bool ONE>
__global__ void __launch_bounds__(kWarps * 32, D == 128 && R == 16 ? 2 : 3)
paged_attn_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  constexpr int TK = Cfg<D>::TK, SUB = Cfg<D>::SUB, ST = Cfg<D>::ST;
  constexpr int WK = TK * SUB;          // keys of a warp's copy
  constexpr int SUP = WK * W;           // keys of a unit
  constexpr int KS = D / 16;            // steps of 16 dims
  constexpr int TS = TK / 16;           // steps of 16 keys
  constexpr int SF = R == 16 ? 2 * TS : TS;   // score fragments of a tile
  constexpr int NO = R * D / 128;       // output fragments
  constexpr int NP = WK / 16;           // most pages of a copy
  constexpr int kHalf = WK * D;         // bytes of its keys
  extern __shared__ __align__(1024) uint8_t s_ring[];       // [kWarps][ST] copies: WK rows of keys, WK rows of values
  __shared__ float s_merge[W > 1 ? 2 : 1][W > 1 ? R * D : 1];
  __shared__ float s_ml[2][R][2];
  __shared__ uint64_t s_bar[kWarps][ST];
  __shared__ int64_t s_scan[kWarps], s_start[kWarps / W][2];

  if (!tiles_aligned(s_ring, A.err)) {
    if (A.split && threadIdx.x < 2) A.part_head[(blockIdx.x * 2 + threadIdx.x) * 4] = -1;      // no pieces
    return;
  }
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int part = W == 1 ? 0 : warp;                       // of the segment's warps
  const int g = lane >> 2, qd = lane & 3;
  const uint32_t ring = smem_u32(s_ring) + warp * ST * 2 * kHalf;
  const uint32_t bars = smem_u32(s_bar[warp]);
  if (lane < ST) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(bars + lane * 8));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_k) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_v) : "memory");
  }
  if (threadIdx.x < kWarps / W) s_start[threadIdx.x][1] = -1;
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

  // ---- this worker's range of units: each thread counts a run of sequences ----
  Cursor<R> c;
  c.left = 0;
  int64_t share;
  {
    constexpr int kWorkers = kWarps / W;                    // of a block
    const int per = (A.B + kWarps * 32 - 1) / (kWarps * 32);
    const int lo = min(int(threadIdx.x) * per, A.B), hi = min(lo + per, A.B);
    int64_t mine = 0;
    bool gaps = false;                                      // rows of q that no sequence computes
    for (int b = lo; b < hi; ++b) {
      Seq<R> s;
      s.load(A, b);
      gaps |= s.gaps(A, b);
      mine += A.split ? s.all(A.H, SUP) : int64_t(A.H) * s.tiles_m;
    }
    int64_t incl = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int64_t v = __shfl_up_sync(0xffffffffu, incl, o);
      if (lane >= o) incl += v;
    }
    if (lane == 31) s_scan[warp] = incl;
    if (__syncthreads_or(gaps))
      clear_gaps<D>(A, 0, A.B, 0, A.Hq, int64_t(blockIdx.x) * kWarps * 32 + threadIdx.x, int64_t(gridDim.x) * kWarps * 32);
    int64_t before = incl - mine, total = 0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      if (w < warp) before += s_scan[w];
      total += s_scan[w];
    }
    // split: equal shares of the units; else equal shares of the segments
    const int64_t workers = int64_t(gridDim.x) * kWorkers;
    share = max(int64_t(A.split ? A.min_units : 1), (total + workers - 1) / workers);
#pragma unroll 1
    for (int w = 0; w < kWorkers; ++w) {
      const int64_t u0 = share * (int64_t(blockIdx.x) * kWorkers + w);
      if (u0 < total && before <= u0 && u0 < before + mine) {
        int64_t at = before;
        for (int b = lo; b < hi; ++b) {
          Seq<R> s;
          s.load(A, b);
          const int64_t k = A.split ? s.all(A.H, SUP) : int64_t(A.H) * s.tiles_m;
          if (u0 < at + k) {
            s_start[w][0] = u0 - at;
            s_start[w][1] = b;
            break;
          }
          at += k;
        }
      }
    }
    __syncthreads();
    const int me = W == 1 ? warp : 0;
    const int64_t u0 = share * (int64_t(blockIdx.x) * kWorkers + me), u1 = min(total, u0 + share);
    c.b = int(s_start[me][1]);
    if (c.b >= 0) {
      c.s.load(A, c.b);
      c.units = c.s.units(SUP);
      int64_t r = s_start[me][0];
      c.unit = A.split ? int(r % c.units) : 0;
      if (A.split) r /= c.units;
      c.mt = int(r % c.s.tiles_m);
      c.h = int(r / c.s.tiles_m);
      c.left = int(u1 - u0);
      if (!A.split) {
        // whole segments: count their units
        Cursor<R> t = c;
        int64_t units = 0, segs = u1 - u0;
        while (segs > 0) {
          const int64_t here = min(segs, int64_t(A.H - t.h) * t.s.tiles_m - t.mt);
          units += here * t.units;
          segs -= here;
          t.mt = t.h = 0;
          t.left = 1;
          if (segs > 0) t.next_seq(A, SUP);
        }
        c.left = int(units);
      }
      c.limits(A);
    }
  }
  if (A.split && threadIdx.x < 2) A.part_head[(blockIdx.x * 2 + threadIdx.x) * 4] = -1;
  if (c.left <= 0) return;                  // a whole block for W > 1, a warp for W = 1

  // ---- producer: this warp's tile of each unit ----
  // Lane i < NP loads key scales, lane NP + i value scales, of page i of a tile, into a register for each tile in
  // flight; `gone` has a bit for each of its pages that is not loaded (behind the keys, or no such page).
  Cursor<R> p = c;
  int page = -1;                            // lane i: id of page i of the tile at p
  const int box = ONE ? TK : A.P, boxes = WK / box, box_log = ONE ? (TK == 64 ? 6 : 5) : A.logP;
  float scl[ST];
  uint32_t gone[ST];
#pragma unroll
  for (int i = 0; i < ST; ++i) scl[i] = 0.f, gone[i] = 0;
  auto fetch_page = [&]() {
    page = -1;
    const int key = p.unit * SUP + part * WK + lane * box;
    if (p.left > 0 && lane < boxes && key < p.lim) page = __ldg(A.table + p.b * A.table_stride + (key >> A.logP));
  };
  auto issue = [&](int st, float& sc, uint32_t& gn) {
    if (p.left <= 0) return;
    const uint32_t bar = bars + st * 8, dst = ring + st * 2 * kHalf;
    const int key = p.unit * SUP + part * WK + lane * box;
    const bool want = lane < boxes && key < p.lim;
    const bool have = want && page >= 0 && page < A.n_pages;
    if (want && !have) set_error(A.err, kIdOutOfRange);
    const int block = have ? page * A.H + p.h : -1;
    const uint32_t mask = __ballot_sync(0xffffffffu, have);
    gn = ~mask;
    const int bk = __shfl_sync(0xffffffffu, block, lane % NP);
    const int row = have ? block * A.P + (key & (A.P - 1)) : 0;
    if (lane == 0)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                   ::"r"(bar), "r"(uint32_t(__popc(mask) * 2 * box * D)) : "memory");
#pragma unroll 1
    for (int i = 0; i < boxes; ++i) {
      const int row_i = __shfl_sync(0xffffffffu, row, i);
      if (lane == 0 && (mask >> i & 1)) {
        tma_rows(dst + i * box * D, &tm_k, bar, row_i);
        tma_rows(dst + kHalf + i * box * D, &tm_v, bar, row_i);
      }
    }
    sc = lane < 2 * NP && bk >= 0 ? __ldg((lane < NP ? A.ks : A.vs) + bk) : 0.f;
    __syncwarp();
    p.next(A, SUP);
    fetch_page();
  };
  fetch_page();
#pragma unroll
  for (int i = 0; i < ST - 1; ++i) issue(i, scl[i], gone[i]);

  // ---- consumer ----
  uint32_t k_off, v_off[2];
  lane_offsets<D>(g, qd, k_off, v_off);
  // the two rows of this lane's accumulators
  const int row_a = R == 16 ? g : 2 * qd, row_b = R == 16 ? g + 8 : 2 * qd + 1;
  bool alive = true;                        // no wait of this warp has run out
  uint32_t st = 0, phase = 0;               // slot of the ring and its turn
  bool first = true;                        // of this worker's segments
  while (c.left > 0) {
    // ---- a segment: this warp's share of its keys ----
    const int seg_b = c.b, seg_h = c.h, r0 = c.mt * R;
    const Seq<R> S = c.s;
    const bool begins = c.unit == 0;
    const int seg_lim = c.lim, rows = S.n * A.G;
    const int seg_mt = c.mt;
    uint32_t qf[KS][R / 4];
    float rs0, rs1;                         // softmax scale of the two rows, in the log2 domain
    {
      constexpr int E = D / 4;              // dims of a lane
      float x[R / 8][E], back[R / 8];
#pragma unroll
      for (int i = 0; i < R / 8; ++i) {
        const int r = r0 + g + 8 * i;
        const bool live = r < rows;
        const int qi = live ? r / A.G : 0;
        const uint16_t* src = static_cast<const uint16_t*>(A.q) +
                              (A.cu ? int64_t(S.tok0 + qi) * A.q_ts
                                    : int64_t(seg_b) * A.q_bs + int64_t(qi) * A.q_ts) +
                              int64_t(seg_h * A.G + (live ? r - qi * A.G : 0)) * A.q_hs + qd * E;
#pragma unroll
        for (int e = 0; e < E; ++e) x[i][e] = 0.f;
        if (live) load_row<E>(src, A.bf16, x[i]);
        float amax = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e) amax = fmaxf(amax, fabsf(x[i][e]));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        const float up = row_scale(amax, A.scale_log2, back[i]);
#pragma unroll
        for (int e = 0; e < E; ++e) x[i][e] *= up;
      }
      if constexpr (R == 16) {
        rs0 = back[0];
        rs1 = back[R / 8 - 1];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          qf[k][0] = pack_f16(x[0][4 * k], x[0][4 * k + 1]);
          qf[k][1] = pack_f16(x[R / 8 - 1][4 * k], x[R / 8 - 1][4 * k + 1]);
          qf[k][R / 4 - 2] = pack_f16(x[0][4 * k + 2], x[0][4 * k + 3]);
          qf[k][R / 4 - 1] = pack_f16(x[R / 8 - 1][4 * k + 2], x[R / 8 - 1][4 * k + 3]);
        }
      } else {
        rs0 = __shfl_sync(0xffffffffu, back[0], row_a * 4);
        rs1 = __shfl_sync(0xffffffffu, back[0], row_b * 4);
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          qf[k][0] = pack_f16(x[0][4 * k], x[0][4 * k + 1]);
          qf[k][1] = pack_f16(x[0][4 * k + 2], x[0][4 * k + 3]);
        }
      }
    }
    // keys that each of the two rows sees, and the fewest of any row
    auto limit = [&](int r) { return r >= rows ? 0 : A.causal ? max(0, S.len - S.n + r / A.G + 1) : S.len; };
    const int lim0 = limit(r0 + row_a), lim1 = limit(r0 + row_b);
    const int min_lim = A.causal ? S.len - S.n + r0 / A.G + 1 : S.len;
    float o[NO][4];
#pragma unroll
    for (int u = 0; u < NO; ++u) o[u][0] = o[u][1] = o[u][2] = o[u][3] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;

    bool ends = false;
    int used = 0;                           // units of the segment so far, for a segment that begins here
    do {
      issue(st == 0 ? ST - 1 : st - 1, scl[ST - 1], gone[ST - 1]);    // refills the slot of the tile before
      const float my_scl = scl[0], my_lv = scale_log2_of(my_scl);
      const uint32_t my_gone = gone[0];
      if (alive) {
        alive = __all_sync(0xffffffffu, mbar_wait(bars + st * 8, phase, A.err));
        if (!alive) {
          // nothing more is copied; what the ring holds is computed on, for the block's barriers (the error word says so)
          drain(bars, ST, st, phase, c.left - max(p.left, 0), A.err);
          p.left = 0;
        }
      }
      __syncwarp();
#pragma unroll 1
      for (int sub = 0; sub < SUB; ++sub) {
        const int k0 = c.unit * SUP + part * WK + sub * TK;
        if (k0 >= seg_lim) break;
        const uint32_t kt = ring + st * 2 * kHalf + sub * TK * D, vt = kt + kHalf;
        const int pg0 = (sub * TK) >> box_log;                        // the tile's first page in the copy
        const uint32_t missing = my_gone >> pg0;                      // its pages that were not loaded
        // ---- scores: fragment j holds keys 8 j.. (R = 16) or 16 j.. (R = 8) ----
        float s[SF][4];
#pragma unroll
        for (int j = 0; j < SF; ++j) {
          if constexpr (R == 16) {
            uint32_t w[KS];
            load_key<D>(kt + k_off + 8 * j * D, w);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              uint32_t b0, b1;
              cvt4(w[k], b0, b1);
              if (k == 0) mma_f16_0(s[j], qf[k], b0, b1);
              else mma_f16(s[j], qf[k], b0, b1);
            }
          } else {
            uint32_t w[KS], x[KS];
            load_key<D>(kt + k_off + 16 * j * D, w);
            load_key<D>(kt + k_off + (16 * j + 8) * D, x);
#pragma unroll
            for (int k = 0; k < KS; ++k) {
              uint32_t a[4];
              cvt4(w[k], a[0], a[2]);
              cvt4(x[k], a[1], a[3]);
              if (k == 0) mma_f16_0(s[j], a, qf[k][0], qf[k][1]);
              else mma_f16(s[j], a, qf[k][0], qf[k][1]);
            }
          }
        }
        uint32_t vw[TS][4][D / 32];
        auto load_values = [&]() {
#pragma unroll
          for (int i = 0; i < TS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) load_value<D>(vt + v_off[r & 1] + (16 * i + 8 * (r >> 1)) * D, vw[i][r]);
        };
        if constexpr (R == 8) load_values();  // on their way while the softmax runs; R = 16 has no registers for that
        // ---- masks: behind a row's keys, and pages that were not loaded ----
        const int end = min(TK, seg_lim - k0);                        // keys of the tile that some row sees
        // a page in front of `end` is missing
        const bool hole = missing & ((1u << ((end + box - 1) >> box_log)) - 1);
        if (k0 + TK > min_lim || hole) {
#pragma unroll
          for (int j = 0; j < SF; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const int at = R == 16 ? 8 * j + 2 * qd + (e & 1) : 16 * j + g + 8 * (e >> 1);
              const bool second = R == 16 ? e >> 1 : e & 1;
              if (k0 + at >= (second ? lim1 : lim0)) s[j][e] = -INFINITY;
              if (missing >> (at >> box_log) & 1) s[j][e] = -INFINITY;
            }
        }
        // ---- running maximum, and the largest product of probability and value scale of the tile ----
        float f0[TS], f1[TS], lv[TS];                                 // by step of 16 keys (ONE: all alike)
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          if (ONE && i > 0) {
            f0[i] = f0[0], f1[i] = f1[0], lv[i] = lv[0];
            continue;
          }
          const int pg = pg0 + (ONE ? 0 : (i * 16) >> box_log);
          const float ks = __shfl_sync(0xffffffffu, my_scl, pg);
          f0[i] = fmaxf(ks * rs0, kTiny);
          f1[i] = fmaxf(ks * rs1, kTiny);
          lv[i] = __shfl_sync(0xffffffffu, my_lv, pg + NP);
        }
        float f_top = 0.f;
#pragma unroll
        for (int i = 0; i < TS; ++i) f_top = fmaxf(f_top, fmaxf(f0[i], f1[i]));
        const bool large = __any_sync(0xffffffffu, f_top >= kLargeFactor);
        constexpr int PS = SF / TS;                                   // fragments of a step of 16 keys
        float x0 = -INFINITY, x1 = -INFINITY, v0 = -INFINITY, v1 = -INFINITY;
        auto reduce = [&](float& a, float& b) {                       // over the lanes of a row
#pragma unroll
          for (int t = R == 16 ? 1 : 4; t < (R == 16 ? 4 : 32); t *= 2) {
            a = fmaxf(a, __shfl_xor_sync(0xffffffffu, a, t));
            b = fmaxf(b, __shfl_xor_sync(0xffffffffu, b, t));
          }
        };
        auto maxima = [&]() {
#pragma unroll
          for (int i = 0; i < TS; ++i) {
            float y0 = -INFINITY, y1 = -INFINITY;
#pragma unroll
            for (int j = PS * i; j < PS * i + PS; ++j) {
              y0 = fmaxf(y0, fmaxf(s[j][0], s[j][R == 16 ? 1 : 2]));
              y1 = fmaxf(y1, fmaxf(s[j][R == 16 ? 2 : 1], s[j][3]));
            }
            x0 = fmaxf(x0, y0 * f0[i]);
            x1 = fmaxf(x1, y1 * f1[i]);
            if (!ONE) {
              v0 = fmaxf(v0, fmaf(y0, f0[i], lv[i]));
              v1 = fmaxf(v1, fmaf(y1, f1[i], lv[i]));
            }
          }
          reduce(x0, x1);
          if (!ONE) reduce(v0, v1);
        };
        maxima();
        const float n0 = fmaxf(x0, m0), n1 = fmaxf(x1, m1);
        const float b0 = n0 == -INFINITY ? 0.f : n0, b1 = n1 == -INFINITY ? 0.f : n1;
        const float al0 = exp2f_approx(m0 - b0), al1 = exp2f_approx(m1 - b1);
        m0 = n0;
        m1 = n1;
        float z0 = 15.f - b0, z1 = 15.f - b1;
        float w0 = ONE ? (x0 - b0) + lv[0] : v0 - b0, w1 = ONE ? (x1 - b1) + lv[0] : v1 - b1;
        if (large) {
#pragma unroll
          for (int i = 0; i < TS; ++i) {
#pragma unroll
            for (int j = PS * i; j < PS * i + PS; ++j)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool second = R == 16 ? e >> 1 : e & 1;
                s[j][e] = score_diff(s[j][e], second ? f1[i] : f0[i], second ? b1 : b0);
              }
            f0[i] = f1[i] = 1.f;
          }
          z0 = z1 = 15.f;
          if (!ONE) {
            v0 = v1 = -INFINITY;
            maxima();
            w0 = v0;
            w1 = v1;
          }
        }
        // log2 of the row's reference for this tile, relative to its running maximum; no key in sight: any
        w0 = fmaxf(w0, kLeastScale - 100.f);
        w1 = fmaxf(w1, kLeastScale - 100.f);
        // ---- probabilities (times 2^15 and the page's relative value scale) and their sum ----
        uint64_t sum = pk2(0.f, 0.f), sum2 = pk2(0.f, 0.f);          // R = 16: row a and row b apart; R = 8: (a, b)
        uint32_t pf[TS][4];
        float c0, c1, i0, i1;                                         // log2 of the page's factor, and what takes it out
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          if (!ONE || i == 0) {
            c0 = fmaxf(lv[i] - w0, kLeastRel);
            c1 = fmaxf(lv[i] - w1, kLeastRel);
            i0 = exp2f_approx(-c0);
            i1 = exp2f_approx(-c1);
            c0 += z0;
            c1 += z1;
          }
          const uint64_t fa = R == 16 ? pk2s(f0[i]) : pk2(f0[i], f1[i]), za = R == 16 ? pk2s(c0) : pk2(c0, c1);
          const uint64_t fb = R == 16 ? pk2s(f1[i]) : fa, zb = R == 16 ? pk2s(c1) : za;
          uint64_t part_a, part_b;
#pragma unroll
          for (int t = 0; t < PS; ++t) {
            const float* sj = s[PS * i + t];
            float p0, p1, p2, p3;
            pk2_split(pk2_fma(pk2(sj[0], sj[1]), fa, za), p0, p1);
            pk2_split(pk2_fma(pk2(sj[2], sj[3]), fb, zb), p2, p3);
            p0 = exp2f_approx(p0);
            p1 = exp2f_approx(p1);
            p2 = exp2f_approx(p2);
            p3 = exp2f_approx(p3);
            part_a = t == 0 ? pk2(p0, p1) : pk2_add(part_a, pk2(p0, p1));
            part_b = t == 0 ? pk2(p2, p3) : pk2_add(part_b, pk2(p2, p3));
            pf[i][2 * t] = pack_f16(p0, p1);
            pf[i][2 * t + 1] = pack_f16(p2, p3);
          }
          const uint64_t ia = R == 16 ? pk2s(i0) : pk2(i0, i1), ib = R == 16 ? pk2s(i1) : ia;
          sum = pk2_fma(part_a, ia, sum);
          sum2 = pk2_fma(part_b, ib, sum2);
          if constexpr (R == 8) {
            pf[i][0] = transpose8(pf[i][0]);
            pf[i][1] = transpose8(pf[i][1]);
          }
        }
        float t0, t1, t2, t3;
        pk2_split(sum, t0, t1);
        pk2_split(sum2, t2, t3);
        l0 = l0 * al0 + (R == 16 ? t0 + t1 : t0 + t2);
        l1 = l1 * al1 + (R == 16 ? t2 + t3 : t1 + t3);
        // ---- values: what lies behind the keys may be anything, NaN too ----
        if constexpr (R == 16) load_values();
        if (hole || end < TK) {
#pragma unroll
          for (int i = 0; i < TS; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              const int at = 16 * i + 2 * qd + (r & 1) + 8 * (r >> 1);
              const bool drop = at >= end || (missing >> (at >> box_log) & 1);
#pragma unroll
              for (int w = 0; w < D / 32; ++w) vw[i][r][w] = drop ? 0u : vw[i][r][w];
            }
        }
        const uint64_t alx = R == 16 ? pk2s(al0) : pk2(al0, al1), aly = R == 16 ? pk2s(al1) : alx;
        const float ref0 = exp2f_small(w0 + kSumLog2), ref1 = exp2f_small(w1 + kSumLog2);
        const uint64_t vrx = R == 16 ? pk2s(ref0) : pk2(ref0, ref1), vry = R == 16 ? pk2s(ref1) : vrx;
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          constexpr int F = R / 4;                                    // output fragments of four of the lane's dims
          float acc[F][4];
#pragma unroll
          for (int i = 0; i < TS; ++i) {
            // pairs of keys for four dims: bytes of two rows side by side
            uint32_t b0[4], b1[4];
            cvt4(__byte_perm(vw[i][0][w], vw[i][1][w], 0x5140), b0[0], b0[1]);
            cvt4(__byte_perm(vw[i][0][w], vw[i][1][w], 0x7362), b0[2], b0[3]);
            cvt4(__byte_perm(vw[i][2][w], vw[i][3][w], 0x5140), b1[0], b1[1]);
            cvt4(__byte_perm(vw[i][2][w], vw[i][3][w], 0x7362), b1[2], b1[3]);
            if constexpr (R == 16) {
#pragma unroll
              for (int e = 0; e < 4; ++e)
                if (i == 0) mma_f16_0(acc[e % F], pf[i], b0[e], b1[e]);
                else mma_f16(acc[e % F], pf[i], b0[e], b1[e]);
            } else {
#pragma unroll
              for (int e = 0; e < 2; ++e) {
                const uint32_t a[4] = {b0[2 * e], b0[2 * e + 1], b1[2 * e], b1[2 * e + 1]};
                if (i == 0) mma_f16_0(acc[e], a, pf[i][0], pf[i][1]);
                else mma_f16(acc[e], a, pf[i][0], pf[i][1]);
              }
            }
          }
#pragma unroll
          for (int e = 0; e < F; ++e) {
            float* ou = o[F * w + e];
            pk2_split(pk2_fma(pk2(acc[e][0], acc[e][1]), vrx, pk2_mul(pk2(ou[0], ou[1]), alx)), ou[0], ou[1]);
            pk2_split(pk2_fma(pk2(acc[e][2], acc[e][3]), vry, pk2_mul(pk2(ou[2], ou[3]), aly)), ou[2], ou[3]);
          }
        }
      }
      __syncwarp();                         // the slot has been read
#pragma unroll
      for (int i = 0; i + 1 < ST; ++i) scl[i] = scl[i + 1], gone[i] = gone[i + 1];
      if (++st == ST) {
        st = 0;
        phase ^= 1;
      }
      const int was = c.unit, left = c.left;
      used = was + 1;
      c.next(A, SUP);
      ends = was == S.units(SUP) - 1;
      if (left == 1) break;
    } while (!ends);

    // ---- the segment's warps become one ----
#pragma unroll
    for (int t = R == 16 ? 1 : 4; t < (R == 16 ? 4 : 32); t *= 2) {
      l0 += __shfl_xor_sync(0xffffffffu, l0, t);
      l1 += __shfl_xor_sync(0xffffffffu, l1, t);
    }
    const bool writes_ml = R == 16 ? qd == 0 : g == 0;      // one lane for each pair of rows
    if constexpr (W > 1) {
      if (S.len > WK) {                     // else warp 0 has it all
#pragma unroll
        for (int n = W / 2; n > 0; n /= 2) {                // warps n .. 2 n - 1 go to warps 0 .. n - 1
          __syncthreads();
          if (warp >= n && warp < 2 * n) {
#pragma unroll
            for (int u = 0; u < NO; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) s_merge[warp - n][(u * 4 + e) * 32 + lane] = o[u][e];
            if (writes_ml) {
              s_ml[warp - n][row_a][0] = m0;
              s_ml[warp - n][row_a][1] = l0;
              s_ml[warp - n][row_b][0] = m1;
              s_ml[warp - n][row_b][1] = l1;
            }
          }
          __syncthreads();
          if (warp < n) {
            const float n0 = s_ml[warp][row_a][0], n1 = s_ml[warp][row_b][0];
            const float x0 = fmaxf(m0, n0), x1 = fmaxf(m1, n1);
            const float c0 = x0 == -INFINITY ? 0.f : x0, c1 = x1 == -INFINITY ? 0.f : x1;
            const float a0 = exp2f_approx(m0 - c0), a1 = exp2f_approx(m1 - c1);
            const float d0 = exp2f_approx(n0 - c0), d1 = exp2f_approx(n1 - c1);
            l0 = l0 * a0 + s_ml[warp][row_a][1] * d0;
            l1 = l1 * a1 + s_ml[warp][row_b][1] * d1;
            m0 = x0;
            m1 = x1;
#pragma unroll
            for (int u = 0; u < NO; ++u)
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const bool second = R == 16 ? e >> 1 : e & 1;
                o[u][e] = o[u][e] * (second ? a1 : a0) + s_merge[warp][(u * 4 + e) * 32 + lane] * (second ? d1 : d0);
              }
          }
        }
      }
    }
    if (part == 0) {
      if (begins && ends) {
        // a sum of 0: no keys. A NaN stays one
        const float i0 = l0 == 0.f ? 0.f : 1.f / kSumUnit / l0, i1 = l1 == 0.f ? 0.f : 1.f / kSumUnit / l1;
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const int r = r0 + (i ? row_b : row_a);
          if (r >= rows) continue;
          const int qi = r / A.G;
          const int64_t at = int64_t(S.tok0 + qi) * A.Hq + seg_h * A.G + (r - qi * A.G);
          const float inv = i ? i1 : i0;
          if constexpr (R == 16) {
            uint16_t* dst = static_cast<uint16_t*>(A.o) + at * D + qd * (D / 4);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
              for (int u = 0; u < NO; u += 4)
                *reinterpret_cast<uint2*>(dst + t * NO + u) =
                    make_uint2(pack_16(o[u][2 * i + t] * inv, o[u + 1][2 * i + t] * inv, A.bf16),
                               pack_16(o[u + 2][2 * i + t] * inv, o[u + 3][2 * i + t] * inv, A.bf16));
          } else {
            uint16_t* dst = static_cast<uint16_t*>(A.o) + at * D + g * (D / 8);
#pragma unroll
            for (int u = 0; u < NO; ++u)
              *reinterpret_cast<uint32_t*>(dst + 2 * u) = pack_16(o[u][i] * inv, o[u][i + 2] * inv, A.bf16);
          }
          const float l = i ? l1 : l0, m = i ? m1 : m0;
          if (A.lse && writes_ml) A.lse[at] = l == 0.f ? -INFINITY : (m - 15.f + log2f(l)) * 0.6931471805599453f;
        }
      } else {
        const int slot = blockIdx.x * 2 + (first ? 0 : 1);
        float* dst = A.part_o + int64_t(slot) * R * D;
#pragma unroll
        for (int u = 0; u < NO; ++u)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if constexpr (R == 16) dst[(e >> 1 ? row_b : row_a) * D + (2 * qd + (e & 1)) * (D / 8) + u] = o[u][e];
            else dst[(e & 1 ? row_b : row_a) * D + g * (D / 8) + 2 * u + (e >> 1)] = o[u][e];
        if (writes_ml) {
          float* ml = A.part_ml + int64_t(slot) * R * 2;
          ml[row_a * 2] = m0;
          ml[row_a * 2 + 1] = l0;
          ml[row_b * 2] = m1;
          ml[row_b * 2 + 1] = l1;
        }
        if (lane == 0) {
          int* hd = A.part_head + slot * 4;
          hd[0] = seg_b;
          hd[1] = seg_h;
          hd[2] = seg_mt;
          // a piece that begins a segment: how many blocks hold the rest of it
          hd[3] = begins ? int((S.units(SUP) - used + share - 1) / share) : 0;
        }
      }
    }
    first = false;
  }
}

// Pieces of the segments that blocks share: one block for each row of each
// piece that begins a segment takes those that follow in the next blocks, a
// group of D / 4 threads a piece at a time, and adds the groups in order.
template <int D, int R>
__global__ void __launch_bounds__(256) paged_attn_join_kernel(const AttnArgs A) {
  constexpr int L = D / 4, GR = 256 / L;
  __shared__ float4 s_o[GR][L];
  __shared__ float s_m[GR], s_l[GR];
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int here = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, gr = tid / L, ln = tid % L;
  // a block's last piece is the only one that can begin a segment without ending it
  const int4 h0 = reinterpret_cast<const int4*>(A.part_head)[here * 2];
  const int4 h1 = reinterpret_cast<const int4*>(A.part_head)[here * 2 + 1];
  const bool second = h1.x >= 0 && h1.w > 0;
  const int4 hd = second ? h1 : h0;
  if (hd.x < 0 || hd.w <= 0) return;
  Seq<R> S;
  S.load(A, hd.x);
  const int r = hd.z * R + row;
  if (r >= S.n * A.G) return;
  float m = -INFINITY, l = 0.f;
  float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
  auto take = [&](float n, float k, float4 x) {
    const float top = fmaxf(m, n), base = top == -INFINITY ? 0.f : top;
    const float a = exp2f_approx(m - base), c = exp2f_approx(n - base);
    m = top;
    l = l * a + k * c;
    o.x = o.x * a + x.x * c;
    o.y = o.y * a + x.y * c;
    o.z = o.z * a + x.z * c;
    o.w = o.w * a + x.w * c;
  };
#pragma unroll 4
  for (int i = gr; i <= hd.w; i += GR) {
    const int64_t at = (i == 0 ? here * 2 + int(second) : 2 * (here + i)) * int64_t(R) + row;
    const float2 ml = *reinterpret_cast<const float2*>(A.part_ml + at * 2);
    take(ml.x, ml.y, *reinterpret_cast<const float4*>(A.part_o + at * D + ln * 4));
  }
  s_o[gr][ln] = o;
  if (ln == 0) {
    s_m[gr] = m;
    s_l[gr] = l;
  }
  __syncthreads();
  if (gr > 0) return;
  for (int i = 1; i < min(GR, hd.w + 1); ++i) take(s_m[i], s_l[i], s_o[i][ln]);
  const float inv = l == 0.f ? 0.f : 1.f / kSumUnit / l;
  const int qi = r / A.G;
  const int64_t at = int64_t(S.tok0 + qi) * A.Hq + hd.y * A.G + (r - qi * A.G);
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(A.o) + at * D + ln * 4) =
      make_uint2(pack_16(o.x * inv, o.y * inv, A.bf16), pack_16(o.z * inv, o.w * inv, A.bf16));
  if (A.lse && ln == 0) A.lse[at] = l == 0.f ? -INFINITY : (m - 15.f + log2f(l)) * 0.6931471805599453f;
}

// Many rows to a key head (prompts, pieces of prompts): bound by the products.
//
// A block takes 64 rows, 16 a warp, of one sequence and key head; its warps
// share copies of 64 keys that warp 0 has TMA load a copy ahead. Queries wait
// in shared memory in the order of their fragments, which leaves registers for
// three blocks an SM. Value scales are taken relative to a reference of each
// row, so that products go straight into the output; the output is scaled only
// when some row's maximum, or its reference (the largest product of probability
// and scale that it has seen), has grown by more than 2^8 (products are held
// times 2^7 and reach 2^15). Blocks with many keys come first. With 16 rows a warp every code is converted for 16 rows' products; 32
// rows a warp need more registers than two blocks an SM leave at d = 128.
// B200: 40 sequences x 8 heads x 256 rows over 1000 keys, pages of 64: 176 us
// (16-row form: 274); of 16, whose tiles have two pairs of scales: 202 us.
constexpr int kManyRows = 16 * kWarps, kManyCopies = 3;

template <bool ONE>                       // a page holds a whole tile of 32 keys
__global__ void __launch_bounds__(kWarps * 32, 3)
paged_attn_many_kernel(const __grid_constant__ AttnArgs A, const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v) {
  constexpr int D = 128, TK = 32, ST = kManyCopies, R = kManyRows;
  constexpr int KS = D / 16, NT = TK / 8, TS = TK / 16, NO = D / 8;
  constexpr int kHalf = kUnit * D;
  extern __shared__ __align__(1024) uint8_t s_ring[];       // [ST] copies: 64 rows of keys, 64 rows of values
  __shared__ uint4 s_q[kWarps][KS][32];
  __shared__ uint64_t s_full[ST], s_empty[ST];
  __shared__ float s_ks[ST][4], s_lv[ST][4];                // scales of a copy's pages: keys, log2 of values'
  __shared__ uint32_t s_gone[ST];
  __shared__ volatile int s_abort;          // a wait has run out: every warp leaves its loop

  if (!tiles_aligned(s_ring, A.err)) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.x / A.H, h = blockIdx.x % A.H, mt = gridDim.y - 1 - blockIdx.y;
  Seq<R> S;
  S.load(A, b);
  if (S.gaps(A, b))
    clear_gaps<D>(A, b, b + 1, h * A.G, A.G, mt * kWarps * 32 + threadIdx.x, gridDim.y * kWarps * 32);
  if (mt >= S.tiles_m) return;
  const int rows = S.n * A.G, r0 = mt * R;
  const int last = min(r0 + R, rows) - 1;
  const int lim = A.causal ? max(0, S.len - S.n + last / A.G + 1) : S.len;    // keys that the last row sees
  const int units = (lim + kUnit - 1) / kUnit;
  const int* table = A.table + b * A.table_stride;
  if (threadIdx.x == 0) s_abort = 0;
  if (threadIdx.x < ST) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], 2;" ::"r"(smem_u32(&s_full[threadIdx.x])));
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(smem_u32(&s_empty[threadIdx.x])), "r"(kWarps));
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();

  // ---- copies (warp 0): those of unit v, then, a step later, its pages' scales ----
  const uint32_t ring = smem_u32(s_ring);
  int issued = 0;                           // units
  int page = -1, pending = -1;              // lane i: page i of the next unit; slot whose scales are on their way
  float new_ks = 0.f, new_vs = 0.f;
  uint32_t new_gone = 0;
  const int boxes = kUnit >> A.logP;
  auto fetch = [&](int v) {
    const int key = v * kUnit + lane * A.P;
    page = lane < boxes && key < lim ? __ldg(table + (key >> A.logP)) : -1;
  };
  auto settle = [&]() {
    if (pending < 0) return;
    if (lane < boxes) {
      s_ks[pending][lane] = new_ks;
      s_lv[pending][lane] = scale_log2_of(new_vs);
    }
    if (lane == 0) s_gone[pending] = new_gone;
    __syncwarp();
    if (lane == 0)
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&s_full[pending])) : "memory");
    pending = -1;
  };
  auto copy = [&](int v) {
    if (v >= units) return;
    const int sl = v % ST, turn = v / ST;
    const uint32_t full = smem_u32(&s_full[sl]), dst = ring + sl * 2 * kHalf;
    const bool want = lane < boxes && v * kUnit + lane * A.P < lim;
    const bool have = want && page >= 0 && page < A.n_pages;
    if (want && !have) set_error(A.err, kIdOutOfRange);
    const int block = have ? page * A.H + h : 0;
    const uint32_t mask = __ballot_sync(0xffffffffu, have);
    if (turn > 0 && !__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_empty[sl]), (turn - 1) & 1, A.err))) {
      s_abort = 1;
      return;
    }
    if (lane == 0)
      asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;"
                   ::"r"(full), "r"(uint32_t(__popc(mask) * 2 * A.P * D)) : "memory");
#pragma unroll 1
    for (int i = 0; i < boxes; ++i) {
      const int row = __shfl_sync(0xffffffffu, block, i) * A.P;
      if (lane == 0 && (mask >> i & 1)) {
        tma_rows(dst + i * A.P * D, &tm_k, full, row);
        tma_rows(dst + kHalf + i * A.P * D, &tm_v, full, row);
      }
    }
    new_ks = have ? __ldg(A.ks + block) : 0.f;
    new_vs = have ? __ldg(A.vs + block) : 0.f;
    new_gone = ~mask;
    pending = sl;
    issued = v + 1;
    fetch(v + 1);
  };
  if (warp == 0) {
    fetch(0);
#pragma unroll 1
    for (int v = 0; v < ST - 2; ++v) {
      settle();
      copy(v);
    }
  }

  // ---- rows ----
  const int g = lane >> 2, qd = lane & 3;
  const int w0 = r0 + warp * 16;            // this warp's first row
  float rs[2];                              // softmax scale of rows g and g + 8, in the log2 domain
  int lims[2];
  int min_lim, max_lim;
  {
    constexpr int E = D / 4;
    float x[2][E];
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int r = w0 + 8 * i + g;
      const bool live = r < rows;
      const int qi = live ? r / A.G : 0;
      const uint16_t* src = static_cast<const uint16_t*>(A.q) +
                            (A.cu ? int64_t(S.tok0 + qi) * A.q_ts : int64_t(b) * A.q_bs + int64_t(qi) * A.q_ts) +
                            int64_t(h * A.G + (live ? r - qi * A.G : 0)) * A.q_hs + qd * E;
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] = 0.f;
      if (live) load_row<E>(src, A.bf16, x[i]);
      float amax = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) amax = fmaxf(amax, fabsf(x[i][e]));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
      amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
      const float up = row_scale(amax, A.scale_log2, rs[i]);
      lims[i] = !live ? 0 : A.causal ? max(0, S.len - S.n + qi + 1) : S.len;
#pragma unroll
      for (int e = 0; e < E; ++e) x[i][e] *= up;
    }
#pragma unroll
    for (int k = 0; k < KS; ++k)
      s_q[warp][k][lane] = make_uint4(pack_f16(x[0][4 * k], x[0][4 * k + 1]), pack_f16(x[1][4 * k], x[1][4 * k + 1]),
                                      pack_f16(x[0][4 * k + 2], x[0][4 * k + 3]),
                                      pack_f16(x[1][4 * k + 2], x[1][4 * k + 3]));
    min_lim = A.causal ? S.len - S.n + w0 / A.G + 1 : S.len;
    const int wl = min(w0 + 16, rows) - 1;                  // this warp's last row
    max_lim = wl < w0 ? 0 : A.causal ? max(0, S.len - S.n + wl / A.G + 1) : S.len;
  }
  uint32_t k_off, v_off[2];
  lane_offsets<D>(g, qd, k_off, v_off);
  // running maxima and sums; log2 of the rows' value references, relative to the maxima
  float o[NO][4], m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, w[2] = {0.f, 0.f};
#pragma unroll
  for (int u = 0; u < NO; ++u) o[u][0] = o[u][1] = o[u][2] = o[u][3] = 0.f;
  uint32_t st = 0, phase = 0;
#pragma unroll 1
  for (int u = 0; u < units && !__any_sync(0xffffffffu, s_abort); ++u) {
    if (warp == 0) {
      settle();
      copy(u + ST - 2);
    }
    if (!__all_sync(0xffffffffu, mbar_wait(smem_u32(&s_full[st]), phase, A.err))) {
      s_abort = 1;
      break;
    }
    const uint32_t all_gone = s_gone[st];
#pragma unroll 1
    for (int sub = 0; sub < kUnit / TK; ++sub) {
      const int k0 = u * kUnit + sub * TK;
      if (k0 >= max_lim) break;
      const uint32_t kt = ring + st * 2 * kHalf + sub * TK * D, vt = kt + kHalf;
      // ---- scores ----
      float s[NT][4];
      {
        uint32_t qf[KS][4];
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          const uint4 v = lds128(smem_u32(&s_q[warp][k][lane]));
          qf[k][0] = v.x; qf[k][1] = v.y; qf[k][2] = v.z; qf[k][3] = v.w;
        }
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          uint32_t w[KS];
          load_key<D>(kt + k_off + 8 * j * D, w);
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            uint32_t b0, b1;
            cvt4(w[k], b0, b1);
            if (k == 0) mma_f16_0(s[j], qf[k], b0, b1);
            else mma_f16(s[j], qf[k], b0, b1);
          }
        }
      }
      // ---- masks ----
      const int end = min(TK, max_lim - k0);                // keys of the tile that some row of the warp sees
      const uint32_t seen = (2u << ((sub * TK + end - 1) >> A.logP)) - 1;     // pages of the copy up to there
      const bool hole = all_gone & seen;
      if (k0 + TK > min_lim || hole) {
#pragma unroll
        for (int j = 0; j < NT; ++j)
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            const int at = sub * TK + 8 * j + 2 * qd + e, key = u * kUnit + at;
            const bool drop = all_gone >> (at >> A.logP) & 1;
            if (drop || key >= lims[0]) s[j][e] = -INFINITY;
            if (drop || key >= lims[1]) s[j][2 + e] = -INFINITY;
          }
      }
      // ---- maxima in the log2 domain: scores, and scores times value scales ----
      float ks[TS], lv[TS];
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        const int pg = (sub * TK + (ONE ? 0 : 16 * i)) >> A.logP;
        ks[i] = ONE && i > 0 ? ks[0] : s_ks[st][pg];
        lv[i] = ONE && i > 0 ? lv[0] : s_lv[st][pg];
      }
      const bool large = __any_sync(0xffffffffu, fmaxf(ks[0], ks[1]) * fmaxf(rs[0], rs[1]) >= kLargeFactor);
      bool grows = false;
      float n[2], x[2], seen_w[2];          // running maximum to come; log2 of the reference, and what it would have to be
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float y[TS], top = -INFINITY, v = -INFINITY;
#pragma unroll
        for (int k = 0; k < TS; ++k) {
          y[k] = fmaxf(fmaxf(s[2 * k][2 * i], s[2 * k][2 * i + 1]), fmaxf(s[2 * k + 1][2 * i], s[2 * k + 1][2 * i + 1])) *
                 fmaxf(ks[k] * rs[i], kTiny);
          top = fmaxf(top, y[k]);
          v = fmaxf(v, y[k] + lv[k]);
        }
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        if (!ONE) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (!ONE) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
        n[i] = top > m[i] + 8.f ? top : m[i];
        const float base = n[i] == -INFINITY ? 0.f : n[i];
        v = ONE ? (top - base) + lv[0] : v - base;
        if (!ONE && large) {                        // differences first: the sum above has lost the scales
          v = -INFINITY;
#pragma unroll
          for (int k = 0; k < TS; ++k) v = fmaxf(v, (y[k] - base) + lv[k]);
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 1));
          v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, 2));
        }
        x[i] = n[i] == m[i] ? w[i] : w[i] + (m[i] - n[i]);
        seen_w[i] = v;
        grows |= top > m[i] + 8.f || v > x[i] + 8.f;
      }
      if (__any_sync(0xffffffffu, grows)) {
        float al[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          if (m[i] != n[i]) l[i] *= exp2f_approx(m[i] - n[i]);
          m[i] = n[i];
          w[i] = seen_w[i] > x[i] + 8.f ? seen_w[i] : x[i];
          al[i] = exp2f_approx(x[i] - w[i]);
        }
#pragma unroll
        for (int v = 0; v < NO; ++v) {
          o[v][0] *= al[0];
          o[v][1] *= al[0];
          o[v][2] *= al[1];
          o[v][3] *= al[1];
        }
      }
      // ---- probabilities (times 2^7 and the page's relative value scale) and their sum ----
      uint32_t pf[TS][4];
      {
        const float b0 = m[0] == -INFINITY ? 0.f : m[0], b1 = m[1] == -INFINITY ? 0.f : m[1];
        float z0 = 7.f - b0, z1 = 7.f - b1;
        if (large) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e)
              s[j][e] = score_diff(s[j][e], fmaxf(ks[j / 2] * rs[e >> 1], kTiny), e >> 1 ? b1 : b0);
          z0 = z1 = 7.f;
        }
        uint64_t sum0 = pk2(0.f, 0.f), sum1 = pk2(0.f, 0.f);
        float c0, c1, i0, i1;               // log2 of the page's factor, and what takes it out
#pragma unroll
        for (int i = 0; i < TS; ++i) {
          if (!ONE || i == 0) {
            c0 = fmaxf(lv[i] - w[0], kLeastRel);
            c1 = fmaxf(lv[i] - w[1], kLeastRel);
            i0 = exp2f_approx(-c0);
            i1 = exp2f_approx(-c1);
          }
          const uint64_t fa = pk2s(large ? 1.f : fmaxf(ks[i] * rs[0], kTiny)), za = pk2s(z0 + c0);
          const uint64_t fb = pk2s(large ? 1.f : fmaxf(ks[i] * rs[1], kTiny)), zb = pk2s(z1 + c1);
          uint64_t pa, pb;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const float* sj = s[2 * i + c];
            float p0, p1, p2, p3;
            pk2_split(pk2_fma(pk2(sj[0], sj[1]), fa, za), p0, p1);
            pk2_split(pk2_fma(pk2(sj[2], sj[3]), fb, zb), p2, p3);
            p0 = exp2f_approx(p0);
            p1 = exp2f_approx(p1);
            p2 = exp2f_approx(p2);
            p3 = exp2f_approx(p3);
            pa = c == 0 ? pk2(p0, p1) : pk2_add(pa, pk2(p0, p1));
            pb = c == 0 ? pk2(p2, p3) : pk2_add(pb, pk2(p2, p3));
            pf[i][2 * c] = pack_f16(p0, p1);
            pf[i][2 * c + 1] = pack_f16(p2, p3);
          }
          sum0 = pk2_fma(pa, pk2s(i0), sum0);
          sum1 = pk2_fma(pb, pk2s(i1), sum1);
        }
        float a0, a1;
        pk2_split(sum0, a0, a1);
        l[0] += a0 + a1;
        pk2_split(sum1, a0, a1);
        l[1] += a0 + a1;
      }
      // ---- values: what lies behind the keys may be anything, NaN too ----
#pragma unroll
      for (int i = 0; i < TS; ++i) {
        uint32_t vw[4][D / 32];
#pragma unroll
        for (int r = 0; r < 4; ++r) load_value<D>(vt + v_off[r & 1] + (16 * i + 8 * (r >> 1)) * D, vw[r]);
        if (hole || end < TK) {
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const int at = 16 * i + 2 * qd + (r & 1) + 8 * (r >> 1);
            const bool drop = at >= end || (all_gone >> ((sub * TK + at) >> A.logP) & 1);
#pragma unroll
            for (int w = 0; w < D / 32; ++w) vw[r][w] = drop ? 0u : vw[r][w];
          }
        }
#pragma unroll
        for (int w = 0; w < D / 32; ++w) {
          uint32_t b0[4], b1[4];
          cvt4(__byte_perm(vw[0][w], vw[1][w], 0x5140), b0[0], b0[1]);
          cvt4(__byte_perm(vw[0][w], vw[1][w], 0x7362), b0[2], b0[3]);
          cvt4(__byte_perm(vw[2][w], vw[3][w], 0x5140), b1[0], b1[1]);
          cvt4(__byte_perm(vw[2][w], vw[3][w], 0x7362), b1[2], b1[3]);
#pragma unroll
          for (int e = 0; e < 4; ++e) mma_f16(o[4 * w + e], pf[i], b0[e], b1[e]);
        }
      }
    }
    __syncwarp();                           // the copy has been read
    if (lane == 0)
      asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(&s_empty[st])) : "memory");
    if (++st == ST) {
      st = 0;
      phase ^= 1;
    }
  }
  if (warp == 0 && __any_sync(0xffffffffu, s_abort)) {
    // every copy lands before the block may end
    settle();
    for (int v = max(0, issued - ST); v < issued; ++v) (void)mbar_wait(smem_u32(&s_full[v % ST]), v / ST & 1, A.err);
  }
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float sum = l[i];
    sum += __shfl_xor_sync(0xffffffffu, sum, 1);
    sum += __shfl_xor_sync(0xffffffffu, sum, 2);
    const int r = w0 + 8 * i + g;
    if (r >= rows) continue;
    const int qi = r / A.G;
    const int64_t at = int64_t(S.tok0 + qi) * A.Hq + h * A.G + (r - qi * A.G);
    // a sum of 0: no keys. A NaN stays one. The reference may be near the largest number: half of it at a time
    const float half = exp2f_approx(0.5f * w[i]), inv = sum == 0.f ? 0.f : half / sum;
    uint16_t* dst = static_cast<uint16_t*>(A.o) + at * D + qd * (D / 4);
#pragma unroll
    for (int c = 0; c < 2; ++c)
#pragma unroll
      for (int u = 0; u < NO; u += 4)
        *reinterpret_cast<uint2*>(dst + c * NO + u) =
            make_uint2(pack_16(o[u][2 * i + c] * inv * half, o[u + 1][2 * i + c] * inv * half, A.bf16),
                       pack_16(o[u + 2][2 * i + c] * inv * half, o[u + 3][2 * i + c] * inv * half, A.bf16));
    if (A.lse && qd == 0) A.lse[at] = sum == 0.f ? -INFINITY : (m[i] - 7.f + log2f(sum)) * 0.6931471805599453f;
  }
}

template <int D, int R, int W, bool ONE>
static void few_launch(AttnArgs& A, const at::Tensor& ck, const at::Tensor& cv, const Bounds& U) {
  constexpr int TK = Cfg<D>::TK, WK = TK * Cfg<D>::SUB, SUP = WK * W;
  constexpr int kSmem = kWarps * Cfg<D>::ST * 2 * WK * D;
  static int known[64] = {};
  auto kern = paged_attn_kernel<D, R, W, ONE>;
  const int64_t slots = int64_t(num_sms()) * blocks_per_sm(kern, kWarps * 32, kSmem, known);
  const int64_t segments = U.B * A.H * ((U.rows + R - 1) / R);
  const int64_t units = std::max<int64_t>(1, (U.len + SUP - 1) / SUP);        // of the longest segment
  // Shares of units instead of whole segments: the second launch and the pieces cost about 4 us, a unit about 1.2 us
  // of its block. d = 64, 8 key heads, us without / with: one sequence of 500 keys 10.5 / 11.4, of 1000 12.4 / 12.4, of
  // 2000 18.0 / 12.3; 64 of 2000 41.1 / 35.0; 512 ragged up to 2000 160 / 145. Pieces of 2 units (4: 2 us more).
  A.min_units = 2;
  A.split = W > 1 && units > 4;
  const int64_t most = A.split ? (segments * units + A.min_units - 1) / A.min_units : (segments * W + kWarps - 1) / kWarps;
  const int grid = int(std::min<int64_t>(slots, most));
  at::Tensor part;
  if (A.split) {
    const int64_t n = 2 * int64_t(grid);
    part = at::empty({n * (R * D + R * 2 + 4)}, ck.options().dtype(at::kFloat));
    A.part_o = part.data_ptr<float>();
    A.part_ml = A.part_o + n * R * D;
    A.part_head = reinterpret_cast<int*>(A.part_ml + n * R * 2);
  }
  const int box = std::min(A.P, TK);
  kern<<<grid, kWarps * 32, kSmem, stream()>>>(A, code_map(ck, box), code_map(cv, box));
  PD_CHECK_LAUNCH();
  if (A.split) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid, R);
    cfg.blockDim = 256;
    cfg.stream = stream();
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    PD_CHECK_CUDA(cudaLaunchKernelEx(&cfg, paged_attn_join_kernel<D, R>, (const AttnArgs)A));
    PD_CHECK_LAUNCH();
  }
}

template <int D, int R>
static void few_dispatch(AttnArgs& A, const at::Tensor& ck, const at::Tensor& cv, const Bounds& U) {
  // A warp a segment needs no merge, but pays where warps stay without one or sequences differ. R = 8, us with 4 warps
  // a segment / with one: 1000 keys, d = 64: 2368 segments 74 / 82, 4736 130 / 121, 18944 489 / 429; d = 32: 101 / 91 and
  // 375 / 313 (4736, 18944); d = 128 level. Keys of one unit, d = 32 (200): 592 14.4 / 12.4, 2368 33 / 25, 9472 113 / 66.
  constexpr int SUP = Cfg<D>::TK * Cfg<D>::SUB * kWarps;
  const int64_t segments = U.B * A.H * ((U.rows + R - 1) / R), warps = int64_t(num_sms()) * 12;
  const int64_t rounds = (segments + warps - 1) / warps;
  const bool one = U.len <= SUP ? segments >= int64_t(num_sms()) * 8 : rounds >= 3 && segments * 20 >= rounds * warps * 17;
  // pages that hold whole tiles of keys have one pair of scales a tile
  if (A.P >= Cfg<D>::TK) one ? few_launch<D, R, 1, true>(A, ck, cv, U) : few_launch<D, R, 4, true>(A, ck, cv, U);
  else one ? few_launch<D, R, 1, false>(A, ck, cv, U) : few_launch<D, R, 4, false>(A, ck, cv, U);
}

template <bool ONE>
static void many_launch(AttnArgs& A, const at::Tensor& ck, const at::Tensor& cv, const Bounds& U) {
  constexpr int kSmem = kManyCopies * 2 * kUnit * 128;
  static int known[64] = {};
  auto kern = paged_attn_many_kernel<ONE>;
  blocks_per_sm(kern, kWarps * 32, kSmem, known);
  const dim3 grid(unsigned(U.B * A.H), unsigned((U.rows + kManyRows - 1) / kManyRows));
  kern<<<grid, kWarps * 32, kSmem, stream()>>>(A, code_map(ck, A.P), code_map(cv, A.P));
  PD_CHECK_LAUNCH();
}

// The forms for many rows (tcgen05 for d = 32 and 64, shared copies for d = 128) do not split the keys, the form for
// few rows reads them again for every 16 rows. Which is faster is estimated in us from what they measured:
//   few   15 + (16-row tiles x keys) / 63e3, 40e3, 21e3 (d = 32, 64, 128)
//   many  waves of blocks x (5 + 64-key units x time of one), a unit 0.85 (tcgen05) or 2.4 with an SM to itself, 1.5 or
//         3.7 where two or three blocks share one
// d = 64, us few / tcgen05: 40 sequences x 8 heads over 1000 keys: 64 rows 43 / 47, 96 rows 70 / 47, 256 rows 122 / 64;
// one of 1824 x 16 heads 95 / 38; four of 128 rows over 4000 45 / 62; one of 512 over 16000 63 / 215.
// d = 128, few / many: 40 x 8 x 64 rows over 1000 92 / 64, 2 x 8 x 512 over 8000 204 / 287.
template <int D>
static bool use_many(const AttnArgs& A, const Bounds& U) {
  if (U.rows <= 16) return false;
  constexpr int rows = D <= 64 ? 128 : kManyRows, per_sm = D <= 64 ? 2 : 3;
  const int64_t tiles = (U.rows + rows - 1) / rows;
  if (tiles > 65535 || U.B * A.H >= (int64_t(1) << 31)) return false;
  const double blocks = double(U.B * A.H) * double(tiles), units = double((U.len + kUnit - 1) / kUnit);
  const double few = 15. + double(U.B * A.H) * double((U.rows + 15) / 16) * double(U.len) /
                               (D == 32 ? 63e3 : D == 64 ? 40e3 : 21e3);
  const double unit = D <= 64 ? (blocks <= num_sms() ? 0.85 : 1.5) : (blocks <= num_sms() ? 2.4 : 3.7);
  return std::ceil(blocks / (num_sms() * per_sm)) * (5. + units * unit) < few;
}

template <int D>
static void attn_dispatch(AttnArgs& A, const at::Tensor& ck, const at::Tensor& cv, const Bounds& U) {
  if (use_many<D>(A, U)) {
    if constexpr (D <= 64) attn_tc_launch(A, ck, cv, D, U);
    else A.P >= 32 ? many_launch<true>(A, ck, cv, U) : many_launch<false>(A, ck, cv, U);
  } else if (U.rows <= 8) {
    few_dispatch<D, 8>(A, ck, cv, U);
  } else {
    few_dispatch<D, 16>(A, ck, cv, U);
  }
}

// (o, lse): lse is an undefined tensor unless asked for.
std::vector<at::Tensor> paged_attention(at::Tensor q, at::Tensor ck, at::Tensor cv, at::Tensor ks, at::Tensor vs,
                                        at::Tensor err, at::Tensor table, at::Tensor lens,
                                        c10::optional<at::Tensor> cu, c10::optional<int64_t> max_q,
                                        c10::optional<int64_t> max_len, c10::optional<double> scale, bool causal,
                                        bool want_lse) {
  const CacheDims C = check_cache(ck, cv, ks, vs, err);
  check_table(table, ck);
  const int64_t B = table.size(0);
  check_ints(lens, ck, B, "kv_lens");
  const int qd = cu.has_value() ? 3 : 4;
  if (q.dim() > 0 && q.stride(-1) != 1) q = q.contiguous();
  PD_CHECK(q.device() == ck.device() && (q.scalar_type() == at::kBFloat16 || q.scalar_type() == at::kHalf),
           "q must be bf16 or fp16 on the cache's device");
  PD_CHECK(q.dim() == qd && q.size(qd - 1) == C.d && (q.stride(qd - 1) == 1 || q.numel() == 0),
           "q must be %s with the cache's head dim and unit stride on d",
           cu.has_value() ? "[tokens, heads, d]" : "[sequences, tokens, heads, d]");
  const int64_t Hq = q.size(qd - 2);
  PD_CHECK(Hq > 0 && Hq % C.H == 0, "%d query heads are no multiple of the cache's %d", int(Hq), C.H);
  if (cu.has_value()) check_ints(*cu, ck, B + 1, "cu_q");
  else PD_CHECK(q.size(0) == B, "q has %d sequences and the page table %d", int(q.size(0)), int(B));
  const c10::cuda::CUDAGuard guard(ck.device());
  AttnArgs A{};
  A.q = q.data_ptr();
  A.q_bs = qd == 4 ? q.stride(0) : 0;
  A.q_ts = q.stride(qd - 3);
  A.q_hs = q.stride(qd - 2);
  A.ks = ks.data_ptr<float>();
  A.vs = vs.data_ptr<float>();
  A.table = table.data_ptr<int>();
  A.table_stride = table.stride(0);
  A.lens = lens.data_ptr<int>();
  A.cu = cu.has_value() ? cu->data_ptr<int>() : nullptr;
  A.total = int(qd == 3 ? q.size(0) : 0);
  A.B = int(B); A.Hq = int(Hq); A.H = C.H; A.G = int(Hq / C.H); A.P = C.P; A.n_pages = C.n_pages;
  A.logP = C.P == 16 ? 4 : C.P == 32 ? 5 : 6;
  A.max_pages = int(table.size(1));
  A.causal = causal;
  A.bf16 = q.scalar_type() == at::kBFloat16;
  A.scale_log2 = float(scale.value_or(1. / std::sqrt(double(C.d))) * 1.4426950408889634);
  A.err = err.data_ptr<int>();
  at::Tensor o = at::empty(q.sizes(), q.options());
  at::Tensor lse;
  A.o = o.data_ptr();
  if (want_lse) {
    lse = at::empty(q.sizes().slice(0, qd - 1), q.options().dtype(at::kFloat));
    A.lse = lse.data_ptr<float>();
  }
  const int64_t most = qd == 4 ? q.size(1) : std::min<int64_t>(std::max<int64_t>(max_q.value_or(q.size(0)), 0), q.size(0));
  PD_CHECK((qd == 3 ? q.size(0) : B * q.size(1)) * A.G < (int64_t(1) << 31) - 128 && B < (int64_t(1) << 31),
           "too many queries");
  A.n = int(most);
  if (B > 0 && q.numel() > 0) {
    // a stated most of 0 launches too: queries that there are all the same are reported
    const Bounds U{B, std::max<int64_t>(most, 1) * A.G, std::min<int64_t>(table.size(1) * C.P, std::max<int64_t>(max_len.value_or(INT64_MAX), 0))};
    if (C.d == 32) attn_dispatch<32>(A, ck, cv, U);
    else if (C.d == 64) attn_dispatch<64>(A, ck, cv, U);
    else attn_dispatch<128>(A, ck, cv, U);
  } else {
    o.zero_();
    if (want_lse) lse.fill_(-INFINITY);
  }
  return want_lse ? std::vector<at::Tensor>{o, lse} : std::vector<at::Tensor>{o};
}

}  // namespace kv

long long launches() { return launch_counter().load(); }
}  // namespace pd
