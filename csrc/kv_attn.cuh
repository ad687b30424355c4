// What the kernels of attention over the paged cache share (kv_attn*.cu):
// arguments, copies and waits, fp16 products, and which rows and keys a
// sequence has.
#pragma once

#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>

#include <cmath>

#include "kv_common.cuh"

namespace pd {
namespace kv {

struct CacheDims { int n_pages, H, P, d; };
CacheDims check_cache(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&);
void check_ints(const at::Tensor&, const at::Tensor&, int64_t, const char*);
void check_table(const at::Tensor&, const at::Tensor&);

constexpr int kMisaligned = 4;           // error word: behind the codes of all kernels

constexpr uint64_t kWaitLimitNs = 2000000000ull;
constexpr int kWarps = 4;               // warps of a block
constexpr int kUnit = 64;               // keys of a copy that a block shares

struct AttnArgs {
  const void* q;                // token, head (and batch) strides below
  int64_t q_bs, q_ts, q_hs;
  const float* ks; const float* vs;          // [pages, H]
  const int* table; int64_t table_stride;
  const int* lens;
  const int* cu;                // [B + 1] or null
  void* o;                      // [tokens, Hq, d]
  float* lse;                   // [tokens, Hq] or null
  int B, n, total;              // n: queries of each sequence, with `cu` the most of one; total: rows of q
  int Hq, H, G, P, logP, max_pages, n_pages;
  bool causal, split, bf16;
  int min_units;
  float scale_log2;
  float* part_o;                // split: [2 grid, R, d] sums, [2 grid, R, 2] (max, sum), [2 grid, 4] heads
  float* part_ml;
  int* part_head;
  int* err;
};

// The hardware's exchange of 16-byte chunks goes by address bits up to 2^10, and so does the code that reads the tiles:
// tiles off that boundary would be read wrongly without a word. The address goes through asm so that the check is not
// taken for granted.
__device__ __forceinline__ bool tiles_aligned(const void* tiles, int* err) {
  uint32_t at;
  asm volatile("mov.u32 %0, %1;" : "=r"(at) : "r"(smem_u32(tiles)));
  if (!(at & 1023)) return true;
  set_error(err, kMisaligned);
  return false;
}
__device__ __forceinline__ bool mbar_try(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
      "selp.b32 %0, 1, 0, p;\n\t}"
      : "=r"(ok) : "r"(bar), "r"(parity), "r"(200000u) : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int* err) {
  if (mbar_try(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  while (!mbar_try(bar, parity)) {
    if (globaltimer_ns() - t0 > kWaitLimitNs) {
      set_error(err, kWaitTimeout);
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, uint32_t bar, int row) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(row) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
  uint2 v;
  asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
// two pairs of e4m3 codes -> two f16x2
__device__ __forceinline__ void cvt4(uint32_t w, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 l, h;\n\t"
      "mov.b32 {l, h}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, l;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, h;\n\t}" : "=r"(lo), "=r"(hi) : "r"(w));
}
// D = A * B
__device__ __forceinline__ void mma_f16_0(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};\n"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
// queries and outputs are bf16 or fp16 by a flag of the call
__device__ __forceinline__ float to_f_16(uint16_t v, bool bf16) {
  return bf16 ? __bfloat162float(__ushort_as_bfloat16(v)) : __half2float(__ushort_as_half(v));
}
__device__ __forceinline__ void load8_16(const uint16_t* p, bool bf16, float* f) {
  const uint4 u = *reinterpret_cast<const uint4*>(p);
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    f[2 * i] = to_f_16(uint16_t(w[i] & 0xffffu), bf16);
    f[2 * i + 1] = to_f_16(uint16_t(w[i] >> 16), bf16);
  }
}
// n elements of a query row, at any alignment
template <int N>
__device__ __forceinline__ void load_row(const uint16_t* p, bool bf16, float* f) {
  if (reinterpret_cast<uintptr_t>(p) % 16 == 0) {
#pragma unroll
    for (int e = 0; e < N; e += 8) load8_16(p + e, bf16, f + e);
  } else {
#pragma unroll
    for (int e = 0; e < N; ++e) f[e] = to_f_16(p[e], bf16);
  }
}
// The power of two that brings a row's largest magnitude to [2^14, 2^15), negative for a negative softmax scale, and in
// `back` what undoes it times the softmax scale. A row of zeros, an infinity or NaN stays as it is.
__device__ __forceinline__ float row_scale(float amax, float scale_log2, float& back) {
  const int ex = amax > 0.f && amax < INFINITY ? max(-100, (__float_as_int(amax) >> 23) - 127) : 14;
  back = __int_as_float((ex - 14 + 127) << 23) * fabsf(scale_log2);
  return copysignf(__int_as_float((14 - ex + 127) << 23), scale_log2);
}
// Scores (log2 domain) beyond some 2^18 are multiplied by their factor before the maximum is subtracted, in a rounding of
// its own: the one fused operation that serves below leaves what the maximum's own rounding cut off, 2^-24 of it, which
// passes the range of fp16 at 2^24. A product of a scaled query and codes is below 2^15 * 448 * d <= 2^31, so a factor
// below this cannot get there; the check so stands off the chain from products to exponentials. Usual factors are some
// 2^-20.
constexpr float kLargeFactor = 1.220703125e-4f;             // 2^-13
__device__ __forceinline__ float score_diff(float s, float f, float base) { return __fsub_rn(__fmul_rn(s, f), base); }
// Value scales act in the exponent of the probabilities, relative to a reference of each row, and out of the sum again: a
// page's factor 2^z, z = log2 of its scale - reference, is cut at 2^-60, where probabilities are zeros in fp16 whatever
// they are. The reference comes from products of probability and scale that the row has seen, so that neither pages that
// it does not see nor those that hardly count cost its values bits. A scale of 0, or below 2^-200, counts as 2^-200.
constexpr float kLeastScale = -200.f, kLeastRel = -60.f;
__device__ __forceinline__ float scale_log2_of(float vs) { return fmaxf(__log2f(vs), kLeastScale); }
// 2^x, with results below 2^-126 too
__device__ __forceinline__ float exp2f_small(float x) {
  float y;
  asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// the least factor of scores: 0 would turn a masked score's -inf into NaN
constexpr float kTiny = 1.17549435e-38f;

// Where a lane (g = lane / 4, qd = lane % 4) finds its codes in a tile of rows of D bytes that TMA has swizzled: its
// quarter of key row g, and its eighth of value rows 2 qd and 2 qd + 1.
template <int D>
__device__ __forceinline__ void lane_offsets(int g, int qd, uint32_t& k_off, uint32_t* v_off) {
  if constexpr (D == 128) {
    k_off = g * 128 + ((2 * qd) ^ g) * 16;
    v_off[0] = (2 * qd) * 128 + (g ^ (2 * qd)) * 16;
    v_off[1] = (2 * qd + 1) * 128 + (g ^ (2 * qd + 1)) * 16;
  } else if constexpr (D == 64) {
    k_off = g * 64 + (qd ^ (g >> 1)) * 16;
    v_off[0] = (2 * qd) * 64 + ((g >> 1) ^ qd) * 16 + (g & 1) * 8;
    v_off[1] = v_off[0] + 64;
  } else {
    k_off = g * 32 + ((qd >> 1) ^ (g >> 2)) * 16 + (qd & 1) * 8;
    v_off[0] = (2 * qd) * 32 + ((g >> 2) ^ (qd >> 1)) * 16 + (g & 3) * 4;
    v_off[1] = v_off[0] + 32;
  }
}
// the lane's D / 4 codes of a key, a word for each step of 16 dims
template <int D>
__device__ __forceinline__ void load_key(uint32_t a, uint32_t* w) {
  if constexpr (D == 128) {
    const uint4 x = lds128(a), y = lds128(a ^ 16);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
    w[4] = y.x; w[5] = y.y; w[6] = y.z; w[7] = y.w;
  } else if constexpr (D == 64) {
    const uint4 x = lds128(a);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else {
    const uint2 x = lds64(a);
    w[0] = x.x; w[1] = x.y;
  }
}
// the lane's D / 8 codes of a value
template <int D>
__device__ __forceinline__ void load_value(uint32_t a, uint32_t* w) {
  if constexpr (D == 128) {
    const uint4 x = lds128(a);
    w[0] = x.x; w[1] = x.y; w[2] = x.z; w[3] = x.w;
  } else if constexpr (D == 64) {
    const uint2 x = lds64(a);
    w[0] = x.x; w[1] = x.y;
  } else {
    w[0] = lds32(a);
  }
}
__device__ __forceinline__ uint32_t pack_16(float lo, float hi, bool bf16) {
  if (bf16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
  }
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
  const __half2 v = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&v);
}
// the transpose of an 8 x 8 tile of 16-bit values (lane: row lane / 4, columns 2 (lane % 4) and the next)
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// D(16x8 f32) += A(16x16 f16, row) * B(16x8 f16, col)
__device__ __forceinline__ void mma_f16(float* d, const uint32_t* a, uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// Offsets of queries that are not served: they do not ascend or lie outside q, or are more than the call states.
__device__ __forceinline__ bool impossible(const AttnArgs& A, int tok0, int n) {
  return n < 0 || n > A.n || tok0 < 0 || tok0 > A.total - n;
}
// Zeros, and -inf for the sums, in rows [lo, hi) of packed outputs, query heads [h0, h0 + nh): thread `first` of `step`.
template <int D>
__device__ __forceinline__ void clear_rows(const AttnArgs& A, int lo, int hi, int h0, int nh, int64_t first, int64_t step) {
  lo = min(max(lo, 0), A.total);
  hi = min(max(hi, 0), A.total);
  constexpr int V = D / 8;                  // vectors of a row
  for (int64_t i = first; i < int64_t(hi - lo) * nh * V; i += step) {
    const int64_t r = i / V, at = (lo + r / nh) * A.Hq + h0 + r % nh;
    *(reinterpret_cast<uint4*>(static_cast<uint16_t*>(A.o) + at * D) + i % V) = make_uint4(0, 0, 0, 0);
    if (A.lse && i % V == 0) A.lse[at] = -INFINITY;
  }
}
// The same for what no sequence computes: rows in front of the first and behind the last one, and those of sequences
// that are not served, among sequences [b0, b1).
template <int D>
__device__ __noinline__ void clear_gaps(const AttnArgs& A, int b0, int b1, int h0, int nh, int64_t first, int64_t step) {
  if (b0 == 0) clear_rows<D>(A, 0, A.cu[0], h0, nh, first, step);
  if (b1 == A.B) clear_rows<D>(A, A.cu[A.B], A.total, h0, nh, first, step);
  for (int b = b0; b < b1; ++b) {
    const int lo = A.cu[b], hi = A.cu[b + 1];
    if (impossible(A, lo, hi - lo)) clear_rows<D>(A, lo, hi, h0, nh, first, step);
  }
}

// The queries and keys of one sequence, with impossible lengths cut (and reported).
template <int R>
struct Seq {
  int len, n, tok0, tiles_m;                // tiles_m: segments of R rows (query, head of the group) for a key head
  bool refused;                             // its offsets are impossible, or it is longer than stated
  __device__ __forceinline__ void load(const AttnArgs& A, int b) {
    len = __ldg(A.lens + b);
    if (A.cu) {
      tok0 = __ldg(A.cu + b);
      n = __ldg(A.cu + b + 1) - tok0;
      refused = impossible(A, tok0, n);
      if (refused) {
        set_error(A.err, kBadShape);
        n = 0;
      }
    } else {
      refused = false;
      n = A.n;
      tok0 = b * A.n;
    }
    if (int64_t(len) > int64_t(A.max_pages) << A.logP) {
      set_error(A.err, kBadShape);
      len = A.max_pages << A.logP;
    }
    if (len < 0) {
      set_error(A.err, kBadShape);
      len = 0;
    }
    tiles_m = int((int64_t(n) * A.G + R - 1) / R);
  }
  // rows of q in front of the first sequence, behind the last one, or this one's that nobody computes
  __device__ __forceinline__ bool gaps(const AttnArgs& A, int b) const {
    return A.cu && (refused || (b == 0 && tok0 != 0) || (b == A.B - 1 && tok0 + n != A.total));
  }
  // units of `sup` keys in each of its segments; a sequence without keys has one (it writes zeros)
  __device__ __forceinline__ int units(int sup) const { return max(1, (len + sup - 1) / sup); }
  __device__ __forceinline__ int64_t all(int H, int sup) const { return int64_t(units(sup)) * H * tiles_m; }
};

// A place in the list of units: sequence b, segment (head, row tile) in it, unit of its keys.
template <int R>
struct Cursor {
  int b, h, mt, unit, units;
  Seq<R> s;
  int lim;                        // keys that the row tile's last row sees
  int left;                       // units from here to the end of this worker's range
  __device__ __forceinline__ void limits(const AttnArgs& A) {
    const int last = min(mt * R + R, s.n * A.G) - 1;
    lim = A.causal ? max(0, s.len - s.n + last / A.G + 1) : s.len;
  }
  __device__ __forceinline__ void next_seq(const AttnArgs& A, int sup) {
    do {
      if (++b >= A.B) { left = 0; return; }
      s.load(A, b);
    } while (s.tiles_m == 0);
    units = s.units(sup);
  }
  __device__ __forceinline__ void next(const AttnArgs& A, int sup) {
    if (--left <= 0) return;
    if (++unit < units) return;
    unit = 0;
    if (++mt == s.tiles_m) {
      mt = 0;
      if (++h == A.H) {
        h = 0;
        next_seq(A, sup);
        if (left <= 0) return;
      }
    }
    limits(A);
  }
};

// cuTensorMapEncodeTiled through the runtime: the extension does not link
// libcuda, so it imports on machines without a driver.
inline CUresult encode_tiled(CUtensorMap* m, void* base, const cuuint64_t* dims, const cuuint64_t* strides,
                             const cuuint32_t* box, CUtensorMapSwizzle swizzle) {
  using Fn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                          const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                          CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
  static const Fn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
    const cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q);
    PD_CHECK(e == cudaSuccess && q == cudaDriverEntryPointSuccess && p != nullptr,
             "cuTensorMapEncodeTiled is unavailable (%d, %d)", int(e), int(q));
    return reinterpret_cast<Fn>(p);
  }();
  const cuuint32_t es[2] = {1, 1};
  return fn(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, base, dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
}

// The cache's codes as rows of d bytes, copied box_rows at a time; swizzled so that fragments load without bank
// conflicts, or as they are.
inline CUtensorMap code_map(const at::Tensor& x, int box_rows, bool swizzled = true) {
  CUtensorMap m;
  const int64_t d = x.size(3), rows = x.numel() / d;
  const cuuint64_t dims[2] = {cuuint64_t(d), cuuint64_t(rows)}, strides[1] = {cuuint64_t(d)};
  const cuuint32_t box[2] = {cuuint32_t(d), cuuint32_t(box_rows)};
  const CUresult r = encode_tiled(&m, x.data_ptr(), dims, strides, box,
                                  !swizzled ? CU_TENSOR_MAP_SWIZZLE_NONE
                                  : d == 128 ? CU_TENSOR_MAP_SWIZZLE_128B
                                  : d == 64 ? CU_TENSOR_MAP_SWIZZLE_64B
                                            : CU_TENSOR_MAP_SWIZZLE_32B);
  PD_CHECK(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed for the cache (%d)", int(r));
  return m;
}

// Blocks of a kernel that an SM of this device holds.
template <typename K>
int blocks_per_sm(K kern, int threads, int smem, int (&known)[64]) {
  int dev = 0;
  PD_CHECK_CUDA(cudaGetDevice(&dev));
  if (dev < 64 && known[dev] > 0) return known[dev];
  PD_CHECK_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  int n = 0;
  PD_CHECK_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, kern, threads, smem));
  PD_CHECK(n > 0, "an attention kernel does not fit an SM");
  if (dev < 64) known[dev] = n;
  return n;
}

struct Bounds {                 // of what the lengths on the device can ask for; they only decide how the work is split
  int64_t B, rows, len;         // rows: most (query, head of the group) of a sequence and key head
};

// Many rows, heads of 32 or 64, on the 5th-generation tensor cores (kv_attn_tc.cu).
void attn_tc_launch(AttnArgs& A, const at::Tensor& ck, const at::Tensor& cv, int d, const Bounds& U);

}  // namespace kv
}  // namespace pd
