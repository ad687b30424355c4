// Attention over the paged 8-bit key/value cache.
//
//   o_i = sum_j softmax_j(scale * q_i . k_j) v_j,   k_j = code * key scale of j's page, v_j likewise
//
// The n new queries of a sequence are its last n tokens: query i of a sequence
// of len tokens sees the keys j <= len - n + i (all keys without the causal
// mask). A query without keys gives 0 (and -inf as its log-sum-exp).
//
// One warp a (query, head): a lane scores one key of 32, then the lanes own
// the head's dims for the weighted sum of values; one pass with a running
// maximum and sum, everything in 32 bits.
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>

#include "kv_common.cuh"

namespace pd {
namespace kv {

struct CacheDims { int n_pages, H, P, d; };
CacheDims check_cache(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&);
void check_ints(const at::Tensor&, const at::Tensor&, int64_t, const char*);
void check_table(const at::Tensor&, const at::Tensor&);

struct AttnArgs {
  const void* q;                // token, head (and batch) strides below
  int64_t q_bs, q_ts, q_hs;
  const uint8_t* kc; const uint8_t* vc;      // [pages, H, P, d]
  const float* ks; const float* vs;          // [pages, H]
  const int* table; int64_t table_stride;
  const int* lens;
  const int* cu;                // [B + 1] or null
  void* o;                      // [tokens, Hq, d]
  float* lse;                   // [tokens, Hq] or null
  int n, total, Hq, H, G, P, max_pages, n_pages;
  bool causal;
  float scale_log2;
  int* err;
};

__device__ __forceinline__ float fp8_at(const uint8_t* p) {
  return float(*reinterpret_cast<const __nv_fp8_e4m3*>(p));
}

template <typename T, int D>
__global__ void __launch_bounds__(128) paged_attn_simple_kernel(const AttnArgs A) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int b = blockIdx.y, hq = blockIdx.z, i = blockIdx.x * 4 + warp;
  const int n = A.cu ? A.cu[b + 1] - A.cu[b] : A.n;
  if (i >= n) return;
  const int64_t tok = A.cu ? int64_t(A.cu[b]) + i : int64_t(b) * A.n + i;
  if (A.cu && (tok < 0 || tok >= A.total)) return;
  const int h = hq / A.G;
  int len = A.lens[b];
  if (len > A.max_pages * int64_t(A.P)) {
    set_error(A.err, kBadShape);
    len = A.max_pages * A.P;
  }
  const int keys = A.causal ? len - n + i + 1 : len;
  const T* q = static_cast<const T*>(A.q) + (A.cu ? tok * A.q_ts : b * A.q_bs + i * A.q_ts) + hq * A.q_hs;
  __shared__ float sq[4][D];
  for (int c = lane; c < D; c += 32) sq[warp][c] = to_f(q[c]);
  __syncwarp();
  constexpr int E = D / 32;
  float m = -INFINITY, l = 0.f, o[E];
#pragma unroll
  for (int e = 0; e < E; ++e) o[e] = 0.f;
  for (int k0 = 0; k0 < keys; k0 += 32) {
    const int j = k0 + lane;
    float s = -INFINITY;
    int64_t row = 0;
    float vscale = 0.f;
    if (j < keys) {
      const int page = A.table[b * A.table_stride + j / A.P];
      if (page >= 0 && page < A.n_pages) {
        const int64_t block = int64_t(page) * A.H + h;
        row = block * A.P + j % A.P;
        s = 0.f;
        for (int c = 0; c < D; ++c) s += sq[warp][c] * fp8_at(A.kc + row * D + c);
        s *= A.ks[block] * A.scale_log2;
        vscale = A.vs[block];
      } else {
        set_error(A.err, kIdOutOfRange);
      }
    }
    const float mx = fmaxf(m, warp_max(s));
    if (mx == -INFINITY) continue;
    const float alpha = exp2f(m - mx), p = exp2f(s - mx);
    m = mx;
    l = l * alpha + warp_sum(p);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= alpha;
    for (int t = 0; t < 32; ++t) {
      const float pt = __shfl_sync(0xffffffffu, p * vscale, t);
      const int64_t rt = __shfl_sync(0xffffffffu, (long long)row, t);
      const bool on = __shfl_sync(0xffffffffu, s, t) != -INFINITY;
      if (!on) continue;
#pragma unroll
      for (int e = 0; e < E; ++e) o[e] += pt * fp8_at(A.vc + rt * D + lane + 32 * e);
    }
  }
  const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
  T* out = static_cast<T*>(A.o) + (tok * A.Hq + hq) * D;
#pragma unroll
  for (int e = 0; e < E; ++e) out[lane + 32 * e] = from_f<T>(o[e] * inv);
  if (A.lse && lane == 0) A.lse[tok * A.Hq + hq] = l > 0.f ? (m + log2f(l)) * 0.69314718056f : (l == 0.f ? -INFINITY : l);
}

template <typename T>
static void attn_launch(const AttnArgs& A, dim3 grid, int d) {
  if (d == 32) paged_attn_simple_kernel<T, 32><<<grid, 128, 0, stream()>>>(A);
  else if (d == 64) paged_attn_simple_kernel<T, 64><<<grid, 128, 0, stream()>>>(A);
  else paged_attn_simple_kernel<T, 128><<<grid, 128, 0, stream()>>>(A);
}

// (o, lse): lse is an undefined tensor unless asked for.
std::vector<at::Tensor> paged_attention(at::Tensor q, at::Tensor ck, at::Tensor cv, at::Tensor ks, at::Tensor vs,
                                        at::Tensor err, at::Tensor table, at::Tensor lens,
                                        c10::optional<at::Tensor> cu, int64_t max_q, int64_t max_len, double scale,
                                        bool causal, bool want_lse) {
  const CacheDims C = check_cache(ck, cv, ks, vs, err);
  check_table(table, ck);
  const int64_t B = table.size(0);
  check_ints(lens, ck, B, "kv_lens");
  const int qd = cu.has_value() ? 3 : 4;
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
  A.kc = static_cast<const uint8_t*>(ck.data_ptr());
  A.vc = static_cast<const uint8_t*>(cv.data_ptr());
  A.ks = ks.data_ptr<float>();
  A.vs = vs.data_ptr<float>();
  A.table = table.data_ptr<int>();
  A.table_stride = table.stride(0);
  A.lens = lens.data_ptr<int>();
  A.cu = cu.has_value() ? cu->data_ptr<int>() : nullptr;
  A.n = int(qd == 4 ? q.size(1) : 0);
  A.total = int(qd == 3 ? q.size(0) : 0);
  A.Hq = int(Hq); A.H = C.H; A.G = int(Hq / C.H); A.P = C.P; A.n_pages = C.n_pages;
  A.max_pages = int(table.size(1));
  A.causal = causal;
  A.scale_log2 = float(scale * 1.4426950408889634);
  A.err = err.data_ptr<int>();
  at::Tensor o = at::empty(q.sizes(), q.options());
  at::Tensor lse;
  A.o = o.data_ptr();
  if (want_lse) {
    lse = at::empty(q.sizes().slice(0, qd - 1), q.options().dtype(at::kFloat));
    A.lse = lse.data_ptr<float>();
  }
  const int64_t most = qd == 4 ? q.size(1) : std::min<int64_t>(max_q, q.size(0));
  if (B > 0 && most > 0 && q.numel() > 0) {
    const dim3 grid(unsigned((most + 3) / 4), unsigned(B), unsigned(Hq));
    if (q.scalar_type() == at::kBFloat16) attn_launch<__nv_bfloat16>(A, grid, C.d);
    else attn_launch<__half>(A, grid, C.d);
    PD_CHECK_LAUNCH();
  }
  return want_lse ? std::vector<at::Tensor>{o, lse} : std::vector<at::Tensor>{o};
}

}  // namespace kv

long long launches() { return launch_counter().load(); }
}  // namespace pd
