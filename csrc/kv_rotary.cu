// RMS norm of queries and keys for each head, with the position rotation in
// the same pass; forward and backward.
//
//   r = (mean_d x^2 + eps)^-1/2,  xh = x r,  y = R(pos) (w * xh)
//   u = R(pos)^T dy,  dw = sum_rows u * xh,  g = u * w,  dx = r (g - xh mean_d(g * xh))
//
// R turns the pairs (i, i + rot / 2), or (2i, 2i + 1), of the first rot
// elements by the angle whose cos and sin the table holds for the row's
// position. Everything between the load and the store is 32-bit.
//
// Both directions are bound by memory: forward 2, backward 3 passes over the
// rows. A row (one head of one token) belongs to a group of 1 to 16 lanes, a
// lane holding the two 8-element vectors that turn against each other, so the
// rotation needs no exchange and the sums a few shuffles in the group. Heads
// of a token are neighbouring groups: they share the angles in L1, and the
// loads of a warp are contiguous where the heads are. Rows that no 16-byte
// access fits (odd strides, dims that are no multiple of 16) go through the
// same code with single elements and a warp a row. A block walks over rows. Of
// 16-bit types each lane has three (backward two) rows to come on their way into
// slots of shared memory that it alone writes and reads, so that they cost no
// registers and no barrier; of 32-bit ones, whose vectors are two accesses, the
// next row comes straight to registers (46 us below; 66 with slots). The row's
// angles are loaded before its sum of squares.
//
// B200, 912 x 8 x 32 queries and keys (786 x 8 x 32) of a projection, batch 256,
// bf16, forward and backward: 252 us, 4.4 TB/s over the 1.11 GB that both cannot
// do without (floor 170 us at the copy rate of 6.5 TB/s; 260 us with the next row
// in registers). The forward runs 22 and the backward 15 warps an SM; issue slots
// are 52 to 60% full and the ALU pipe 50%, mostly conversions and addresses, and
// neither more rows on their way nor a fourth forward block changes the time.
// 2049 x 40 x 128 in 32 bits, half turned: 46 us, 5.5 TB/s.
//
// dw: each lane keeps its 16 columns' sums over all rows of its block, blocks
// write theirs to a workspace and a second launch adds them in a fixed order,
// so that the same inputs give the same bits.
#include <c10/cuda/CUDAGuard.h>

#include "kv_common.cuh"

namespace pd {
namespace kv {

constexpr int kThreads = 256;

struct Part {                 // queries or keys
  const void* x;              // [B, T, H, d], unit stride on d
  const void* dy;             // backward: the gradient of y, strided like y (contiguous)
  void* y;                    // forward: y; backward: dx; contiguous
  const float* w;             // [d] or null
  int64_t bs, ts, hs;         // strides of x
  int rows, T, H, t_off;      // t_off: index of its first token in the positions
  uint32_t mul_h, sh_h, mul_t, sh_t;   // division by H and by T
};

struct Args {
  Part p[2];
  int blocks0;                // the first blocks0 blocks work on p[0]
  const float* table;         // [n_pos, rot]
  const void* pos;            // int32 / int64 [T] or [B, T], or null: the token's index
  int64_t pos_bs;
  bool pos64, interleaved;
  int n_pos, rot, d;
  float eps;
  float* dw_part;             // [grid, d]
  int* err;
};

// n / div for n < 2^31 by a multiplication (round-up method: the multiplier
// ceil(2^(31 + s) / div) with s = ceil(log2 div) fits 32 bits and is exact).
inline void set_div(uint32_t div, uint32_t& mul, uint32_t& sh) {
  uint32_t s = 0;
  while ((uint64_t(1) << s) < div) ++s;
  mul = uint32_t(((uint64_t(1) << (31 + s)) + div - 1) / div);
  sh = s;
}
__device__ __forceinline__ uint32_t fast_div(uint32_t n, uint32_t mul, uint32_t sh) {
  return uint32_t((uint64_t(n) * mul) >> (31 + sh));
}

// 16-byte copies to shared memory that a thread issues and reads itself, in groups a row
__device__ __forceinline__ void copy16(uint32_t to, const void* from) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
}
__device__ __forceinline__ void copy_group() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// rows that a lane holds in shared memory at once (1: none, the next one is in registers)
template <typename T, int V> constexpr bool kRinged = V == 8 && sizeof(T) == 2;
template <typename T, int V, bool BWD> constexpr int kStages = !kRinged<T, V> ? 1 : BWD ? 3 : 4;
template <typename T, int V, bool BWD>
constexpr int kRingBytes = !kRinged<T, V> ? 0 : kStages<T, V, BWD> * (BWD ? 4 : 2) * Raw<V, T>::N * 16 * kThreads;

template <typename T, int V, int L, int NP, bool BWD>
__global__ void __launch_bounds__(kThreads, BWD ? 2 : 3) qk_norm_rope_kernel(const __grid_constant__ Args A) {
  constexpr int G = kThreads / L;                       // rows of a block at a time
  const bool second = int(blockIdx.x) >= A.blocks0;
  const Part& P = A.p[second ? 1 : 0];
  const int block = second ? blockIdx.x - A.blocks0 : blockIdx.x;
  const int blocks = second ? gridDim.x - A.blocks0 : A.blocks0;
  const int lane = threadIdx.x % L, d = A.d, pairs = d / (2 * V);
  const T* x = static_cast<const T*>(P.x);
  const T* dy = static_cast<const T*>(P.dy);
  T* y = static_cast<T*>(P.y);
  const float inv_d = 1.f / float(d);

  __shared__ __align__(16) float s_w[256];
  for (int c = threadIdx.x; c < d; c += kThreads) s_w[c] = P.w ? P.w[c] : 1.f;
  __syncthreads();
  int off0[NP], off1[NP];
  bool on[NP], turned[NP];
  float acc0[NP][V], acc1[NP][V];
#pragma unroll
  for (int i = 0; i < NP; ++i) {
    const int j = lane + i * L;
    on[i] = j < pairs;
    off0[i] = off1[i] = 0;
    turned[i] = false;
    if (on[i]) pair_offsets<V>(j, d, A.rot, A.interleaved, off0[i], off1[i], turned[i]);
#pragma unroll
    for (int e = 0; e < V; ++e) acc0[i][e] = acc1[i][e] = 0.f;
  }
  auto weights = [&](int off, float* w) {
    if constexpr (V == 1) {
      w[0] = s_w[off];
    } else {
      const float4 a = *reinterpret_cast<const float4*>(s_w + off), c = *reinterpret_cast<const float4*>(s_w + off + 4);
      w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w; w[4] = c.x; w[5] = c.y; w[6] = c.z; w[7] = c.w;
    }
  };
  // a row on its way: its place in the output (or -1), its position, its elements where no 16-byte copy takes them
  constexpr bool RING = kRinged<T, V>;
  constexpr int S = kStages<T, V, BWD>, N = Raw<V, T>::N;
  extern __shared__ uint4 s_ring[];                     // [S][x, then dy: 2 N vectors each][thread]
  const auto slot = [&](int st, int k) { return s_ring + (st * (BWD ? 4 : 2) * N + k) * kThreads + threadIdx.x; };
  struct Row {
    Raw<V, T> xa[RING ? 1 : NP], xb[RING ? 1 : NP], ya[RING ? 1 : NP], yb[RING ? 1 : NP];
    int row_of = -1;
    int64_t pos = -1;
  };
  Row next[S];
  auto fetch = [&](int it, int st, Row& F) {
    const uint32_t row = uint32_t(it * blocks + block) * G + threadIdx.x / L;
    F.row_of = row < uint32_t(P.rows) ? int(row) : -1;
    if (F.row_of >= 0) {
      const uint32_t tok = fast_div(row, P.mul_h, P.sh_h), h = row - tok * P.H;
      const uint32_t bb = fast_div(tok, P.mul_t, P.sh_t), t = tok - bb * P.T;
      const T* xr = x + int64_t(bb) * P.bs + int64_t(t) * P.ts + int64_t(h) * P.hs;
      const T* dr = dy + int64_t(row) * d;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
        if (!on[i]) continue;
        if constexpr (RING) {
#pragma unroll
          for (int k = 0; k < N; ++k) {
            copy16(smem_u32(slot(st, k)), reinterpret_cast<const uint4*>(xr + off0[i]) + k);
            copy16(smem_u32(slot(st, N + k)), reinterpret_cast<const uint4*>(xr + off1[i]) + k);
            if (BWD) {
              copy16(smem_u32(slot(st, 2 * N + k)), reinterpret_cast<const uint4*>(dr + off0[i]) + k);
              copy16(smem_u32(slot(st, 3 * N + k)), reinterpret_cast<const uint4*>(dr + off1[i]) + k);
            }
          }
        } else {
          F.xa[i].load(xr + off0[i]);
          F.xb[i].load(xr + off1[i]);
          if (BWD) {
            F.ya[i].load(dr + off0[i]);
            F.yb[i].load(dr + off1[i]);
          }
        }
      }
      const int64_t pi = int64_t(bb) * A.pos_bs + t + P.t_off;
      F.pos = A.pos == nullptr ? int64_t(t) + P.t_off
              : A.pos64        ? __ldg(static_cast<const long long*>(A.pos) + pi)
                               : int64_t(__ldg(static_cast<const int*>(A.pos) + pi));
    }
    if (RING) copy_group();
  };
  // every lane of a warp takes part in the group sums of each turn
  const int turns = int((int64_t(P.rows) + blocks * G - 1) / (blocks * G));
  constexpr int AHEAD = RING ? S - 1 : 1;
#pragma unroll
  for (int i = 0; i < AHEAD; ++i) fetch(i, i, next[i]);
  int st = 0;
  for (int it = 0; it < turns; ++it) {
    Raw<V, T> xa[NP], xb[NP], ya[NP], yb[NP];
    const int row = next[0].row_of;
    const bool live = row >= 0, known = live && next[0].pos >= 0 && next[0].pos < A.n_pos;
    if (live && !known) set_error(A.err, kIdOutOfRange);
    const float* at = A.table + (known ? next[0].pos : 0) * A.rot;
    if (RING) copy_wait<AHEAD - 1>();
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      if (known && on[i]) {
        if constexpr (RING) {
#pragma unroll
          for (int k = 0; k < N; ++k) {
            xa[i].v[k] = *slot(st, k);
            xb[i].v[k] = *slot(st, N + k);
            if (BWD) {
              ya[i].v[k] = *slot(st, 2 * N + k);
              yb[i].v[k] = *slot(st, 3 * N + k);
            }
          }
        } else {
          xa[i] = next[0].xa[i];
          xb[i] = next[0].xb[i];
          if (BWD) {
            ya[i] = next[0].ya[i];
            yb[i] = next[0].yb[i];
          }
        }
      } else {                                          // behind the rows, or a position outside: zeros
        xa[i].zero();
        xb[i].zero();
        if (BWD) {
          ya[i].zero();
          yb[i].zero();
        }
      }
    }
#pragma unroll
    for (int i = 0; i + 1 < AHEAD; ++i) next[i] = next[i + 1];
    float c[NP][V], s[NP][V];
#pragma unroll
    for (int i = 0; i < NP; ++i)
      if (turned[i]) load_angles<V>(at, lane + i * L, A.rot, A.interleaved, off0[i], off1[i], c[i], s[i]);
    float a[NP][V], b[NP][V], ga[NP][V], gb[NP][V];
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      xa[i].floats(a[i]);
      xb[i].floats(b[i]);
      if (BWD) {
        ya[i].floats(ga[i]);
        yb[i].floats(gb[i]);
      }
      ss += dot_v<V>(a[i], a[i], b[i], b[i]);
    }
    // groups without a row hold zeros: with eps = 0 their root would be infinite, and NaN in the sums of dw
    const float rt = __frsqrt_rn(group_sum<L>(ss) * inv_d + A.eps), r = known ? rt : 0.f;
    // the stage read in the last turn is free
    fetch(it + AHEAD, st == 0 ? S - 1 : st - 1, next[AHEAD - 1]);
    st = st + 1 == S ? 0 : st + 1;
    T* out = y + int64_t(row) * d;
    float dot = 0.f;
#pragma unroll
    for (int i = 0; i < NP; ++i) {
      scale_v<V>(a[i], r);                              // xh
      scale_v<V>(b[i], r);
      float w0[V], w1[V];
      weights(off0[i], w0);
      weights(off1[i], w1);
      if (!BWD) {
        mul_v<V>(a[i], w0);
        mul_v<V>(b[i], w1);
      }
      if (turned[i]) {
        if (BWD) turn<V>(ga[i], gb[i], c[i], s[i], A.interleaved, -1.f);
        else turn<V>(a[i], b[i], c[i], s[i], A.interleaved, 1.f);
      }
      if (BWD) {
        add_mul_v<V>(acc0[i], ga[i], a[i]);
        add_mul_v<V>(acc1[i], gb[i], b[i]);
        mul_v<V>(ga[i], w0);
        mul_v<V>(gb[i], w1);
        dot += dot_v<V>(ga[i], a[i], gb[i], b[i]);
      }
    }
    if (BWD) {
      dot = -group_sum<L>(dot) * inv_d;
#pragma unroll
      for (int i = 0; i < NP; ++i) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          a[i][e] = r * fmaf(a[i][e], dot, ga[i][e]);
          b[i][e] = r * fmaf(b[i][e], dot, gb[i][e]);
        }
      }
    }
    if (live) {
#pragma unroll
      for (int i = 0; i < NP; ++i)
        if (on[i]) {
          store_v<V>(out + off0[i], a[i]);
          store_v<V>(out + off1[i], b[i]);
        }
    }
  }
  if (BWD) {
    // groups of a warp by shuffles, warps through shared memory, both in a fixed order
    __shared__ float part[kThreads / 32][256];
    const int warp = threadIdx.x >> 5;
#pragma unroll
    for (int i = 0; i < NP; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
#pragma unroll
        for (int o = 16; o >= L; o >>= 1) {
          acc0[i][e] += __shfl_xor_sync(0xffffffffu, acc0[i][e], o);
          acc1[i][e] += __shfl_xor_sync(0xffffffffu, acc1[i][e], o);
        }
        if ((threadIdx.x & 31) < L && on[i]) {
          part[warp][off0[i] + e] = acc0[i][e];
          part[warp][off1[i] + e] = acc1[i][e];
        }
      }
    __syncthreads();
    for (int c = threadIdx.x; c < d; c += kThreads) {
      float t = 0.f;
#pragma unroll
      for (int k = 0; k < kThreads / 32; ++k) t += part[k][c];
      A.dw_part[int64_t(blockIdx.x) * d + c] = t;
    }
  }
}

// dw[part] = the sum of its blocks' rows of the workspace; one block a part and
// 32 columns, 32 rows at a time.
__global__ void __launch_bounds__(1024) dw_sum_kernel(const float* part, int blocks0, int blocks, int d, float* dw0,
                                                      float* dw1) {
  __shared__ float t[32][33];
  const int c = blockIdx.x * 32 + threadIdx.x;
  const int lo = blockIdx.y == 0 ? 0 : blocks0, hi = blockIdx.y == 0 ? blocks0 : blocks;
  float s = 0.f;
  if (c < d) {
#pragma unroll 8
    for (int r = lo + threadIdx.y; r < hi; r += 32) s += part[int64_t(r) * d + c];
  }
  t[threadIdx.y][threadIdx.x] = s;
  __syncthreads();
  s = warp_sum(t[threadIdx.x][threadIdx.y]);
  const int col = blockIdx.x * 32 + threadIdx.y;
  float* dw = blockIdx.y == 0 ? dw0 : dw1;
  if (threadIdx.x == 0 && col < d && dw != nullptr) dw[col] = s;
}

template <typename T, int V, int L, int NP, bool BWD>
static void launch(const Args& A, int grid) {
  constexpr int kRing = kRingBytes<T, V, BWD>;
  const auto kern = qk_norm_rope_kernel<T, V, L, NP, BWD>;
  static bool known[64] = {};
  int dev = 0;
  PD_CHECK_CUDA(cudaGetDevice(&dev));
  if (kRing > 32 * 1024 && (dev >= 64 || !known[dev])) {
    PD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kRing));
    if (dev < 64) known[dev] = true;
  }
  kern<<<grid, kThreads, kRing, stream()>>>(A);
  PD_CHECK_LAUNCH();
}
template <typename T, int V, int L, int NP>
static void launch(const Args& A, int grid, bool bwd) {
  if (bwd) launch<T, V, L, NP, true>(A, grid);
  else launch<T, V, L, NP, false>(A, grid);
}

template <typename T>
static void dispatch(const Args& A, int grid, bool bwd, int lanes) {
  switch (lanes) {
    case 1: return launch<T, 8, 1, 1>(A, grid, bwd);
    case 2: return launch<T, 8, 2, 1>(A, grid, bwd);
    case 4: return launch<T, 8, 4, 1>(A, grid, bwd);
    case 8: return launch<T, 8, 8, 1>(A, grid, bwd);
    case 16: return launch<T, 8, 16, 1>(A, grid, bwd);
    default: return launch<T, 1, 32, 4>(A, grid, bwd);
  }
}

static bool aligned16(const at::Tensor& x) {
  const int64_t n = 16 / x.element_size();
  if (reinterpret_cast<uintptr_t>(x.data_ptr()) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (x.size(i) > 1 && x.stride(i) % n) return false;
  return true;
}

static void fill(Part& P, const at::Tensor& x, const c10::optional<at::Tensor>& w, int t_all, const char* what) {
  PD_CHECK(x.dim() == 4 && (x.stride(3) == 1 || x.numel() == 0), "%s must be [B, T, H, d] with unit stride on d", what);
  const int64_t rows = x.size(0) * x.size(1) * x.size(2);
  PD_CHECK(rows < (int64_t(1) << 31), "%s has 2^31 or more heads of tokens", what);
  P.x = x.data_ptr();
  P.bs = x.stride(0); P.ts = x.stride(1); P.hs = x.stride(2);
  P.rows = int(rows); P.T = int(x.size(1)); P.H = int(x.size(2));
  P.t_off = t_all - P.T;
  P.w = nullptr;
  if (w.has_value()) {
    PD_CHECK(w->device() == x.device() && w->scalar_type() == at::kFloat && w->is_contiguous() && w->dim() == 1 &&
             w->size(0) == x.size(3), "the weight of %s must be a contiguous fp32 [d] on its device", what);
    P.w = w->data_ptr<float>();
  }
  set_div(uint32_t(std::max<int64_t>(P.H, 1)), P.mul_h, P.sh_h);
  set_div(uint32_t(std::max<int64_t>(P.T, 1)), P.mul_t, P.sh_t);
}

// Forward (dq, dk absent): y of q and k. Backward: dq, dk, dw_q, dw_k.
std::vector<at::Tensor> qk_norm_rope(at::Tensor q, c10::optional<at::Tensor> k, c10::optional<at::Tensor> wq,
                                     c10::optional<at::Tensor> wk, at::Tensor table, c10::optional<at::Tensor> pos,
                                     double eps, bool interleaved, at::Tensor err, c10::optional<at::Tensor> dyq,
                                     c10::optional<at::Tensor> dyk) {
  const bool bwd = dyq.has_value();
  const int n_parts = k.has_value() ? 2 : 1;
  PD_CHECK(q.is_cuda() && q.dim() == 4, "q must be a CUDA tensor [B, T, H, d]");
  const int dt = dtype_of(q, "q");
  Args A{};
  A.d = int(q.size(3));
  const int t_all = int(k.has_value() ? k->size(1) : q.size(1));
  const int64_t B = q.size(0);
  PD_CHECK(q.size(3) >= 2 && q.size(3) <= 256 && q.size(3) % 2 == 0, "head dim %d: expected even, 2 to 256", A.d);
  if (k.has_value()) {
    PD_CHECK(k->is_cuda() && k->device() == q.device() && k->dim() == 4 && k->scalar_type() == q.scalar_type(),
             "k must be [B, T, H, d] of q's type on q's device");
    PD_CHECK(k->size(0) == B && k->size(3) == A.d, "q and k differ in their batch or head dim");
    PD_CHECK(q.size(1) <= k->size(1), "more query tokens (%d) than key tokens (%d)", int(q.size(1)), t_all);
  }
  PD_CHECK(table.device() == q.device() && table.scalar_type() == at::kFloat && table.dim() == 2 &&
           table.is_contiguous() && reinterpret_cast<uintptr_t>(table.data_ptr()) % 16 == 0,
           "the angle table must be a contiguous fp32 [positions, rotary_dim] on q's device");
  A.rot = int(table.size(1));
  PD_CHECK(A.rot % 2 == 0 && A.rot <= A.d, "rotary_dim %d: expected even and at most the head dim %d", A.rot, A.d);
  PD_CHECK(table.size(0) < (int64_t(1) << 31), "the angle table has 2^31 or more positions");
  A.n_pos = int(table.size(0));
  A.table = table.data_ptr<float>();
  PD_CHECK(err.device() == q.device() && err.scalar_type() == at::kInt && err.numel() == 1, "err must be one int32");
  A.err = err.data_ptr<int>();
  A.eps = float(eps);
  A.interleaved = interleaved;
  if (pos.has_value()) {
    const auto st = pos->scalar_type();
    PD_CHECK(pos->device() == q.device() && (st == at::kInt || st == at::kLong) && pos->is_contiguous(),
             "positions must be contiguous int32 or int64 on q's device");
    PD_CHECK((pos->dim() == 1 && pos->size(0) == t_all) ||
             (pos->dim() == 2 && pos->size(0) == B && pos->size(1) == t_all),
             "positions must be [T] or [B, T] for %d tokens", t_all);
    A.pos = pos->data_ptr();
    A.pos64 = st == at::kLong;
    A.pos_bs = pos->dim() == 2 ? t_all : 0;
  }
  const c10::cuda::CUDAGuard guard(q.device());
  fill(A.p[0], q, wq, t_all, "q");
  if (n_parts == 2) fill(A.p[1], *k, wk, t_all, "k");
  // rows outside the table take the angles of its first row, times zeros: there has to be one
  TORCH_CHECK_INDEX(A.n_pos > 0 || A.rot == 0 || (A.p[0].rows == 0 && A.p[1].rows == 0),
                    "every position lies outside an angle table of 0 rows");

  std::vector<at::Tensor> out;
  bool vec = A.d % 16 == 0 && A.rot % 16 == 0;
  for (int i = 0; i < n_parts; ++i) {
    const at::Tensor& x = i == 0 ? q : *k;
    vec = vec && aligned16(x);
    at::Tensor y = at::empty(x.sizes(), x.options());
    A.p[i].y = y.data_ptr();
    out.push_back(y);
    if (bwd) {
      const c10::optional<at::Tensor>& dy = i == 0 ? dyq : dyk;
      PD_CHECK(dy.has_value() && dy->is_contiguous() && dy->sizes() == x.sizes() && dy->device() == x.device() &&
               dy->scalar_type() == x.scalar_type(), "a gradient must be contiguous and like its output");
      A.p[i].dy = dy->data_ptr();
      vec = vec && reinterpret_cast<uintptr_t>(dy->data_ptr()) % 16 == 0;
    }
  }
  // lanes of a row: the power of two that covers its pairs of 8 + 8 elements; 32 for single elements
  int lanes = 32;
  if (vec) for (lanes = 1; lanes * 16 < A.d; lanes *= 2) {}
  const int64_t G = kThreads / lanes;
  // blocks that the device holds at once, shared out by rows
  int64_t nb[2] = {0, 0};
  const int64_t rows_all = int64_t(A.p[0].rows) + (n_parts == 2 ? A.p[1].rows : 0);
  const int64_t slots = int64_t(num_sms()) * (bwd ? 2 : 3);
  for (int i = 0; i < n_parts; ++i)
    if (A.p[i].rows > 0)
      nb[i] = std::min<int64_t>((A.p[i].rows + G - 1) / G,
                                std::max<int64_t>(1, (slots * A.p[i].rows + rows_all / 2) / rows_all));
  const int64_t grid = nb[0] + nb[1];
  A.blocks0 = int(nb[0]);
  at::Tensor part;
  if (bwd) {
    for (int i = 0; i < n_parts; ++i) out.push_back(at::empty({A.d}, q.options().dtype(at::kFloat)));
    part = at::empty({std::max<int64_t>(grid, 1), A.d}, q.options().dtype(at::kFloat));
    A.dw_part = part.data_ptr<float>();
  }
  if (grid > 0) {
    if (dt == kBf16) dispatch<__nv_bfloat16>(A, int(grid), bwd, lanes);
    else if (dt == kF16) dispatch<__half>(A, int(grid), bwd, lanes);
    else dispatch<float>(A, int(grid), bwd, lanes);
  }
  if (bwd) {
    const dim3 g((A.d + 31) / 32, n_parts);
    dw_sum_kernel<<<g, dim3(32, 32), 0, stream()>>>(part.data_ptr<float>(), A.blocks0, int(grid), A.d,
                                                    out[n_parts].data_ptr<float>(),
                                                    n_parts == 2 ? out[3].data_ptr<float>() : nullptr);
    PD_CHECK_LAUNCH();
  }
  return out;
}

}  // namespace kv
}  // namespace pd
