// The paged key/value cache in 8 bits: append (with the norm and the position
// rotation of the keys on the way) and read.
//
// A page holds P tokens; one (page, head) is P x d codes of e4m3 in a row and
// one scale for keys, one for values: value = code * scale. The scale is a
// power of two, the smallest (2^-100 at least) that brings the page's largest
// finite magnitude to 448 or less:
//   amax = m 2^e, 1 <= m < 2;  448 = 1.75 * 2^8  =>  scale = 2^(e - 8), or 2^(e - 7) where m > 1.75
// A power of two costs no precision (e4m3 keeps 3 bits below the leading one
// at any scale) and makes it cheap and nearly exact to raise the scale of a
// page that is already partly filled: old codes move by whole binades, so only
// those that become subnormal are rounded again. A page's scale never falls
// while it fills; a page whose first row is written starts anew. Non-finite
// inputs do not enter the scale and are stored as NaN.
//
// append is bound by memory for long pieces (it reads k and v once and writes
// one byte a value) and by latency for single tokens, read by its writes.
// B200, append and read together: 128 histories of 896 x 8 x 32 (bf16, keys
// normed and rotated, pages of 64) 86 us for 361 MB (floor 55 us), of which the
// append takes about 52: its rows are 64 bytes, 16 an access, and the maximum of
// a page stands between its loads and its stores (24 warps an SM, issue slots 56%
// full). 48 ragged pieces of 8 x 128 (pages of 16) 72 us for 280 MB (floor 43 us).
// One token each of 64 sequences: 13 us, the two launches' host time.
#include <c10/cuda/CUDAGuard.h>
#include <cuda_fp8.h>

#include "kv_common.cuh"

namespace pd {
namespace kv {

constexpr int kMinExp = -100;

// exponent of the scale of a page whose largest finite magnitude has these bits
__device__ __forceinline__ int scale_exp(float amax) {
  if (amax == 0.f) return kMinExp;
  int e = 0;
  const float m = frexpf(amax, &e);               // amax = m 2^e, 0.5 <= m < 1
  return max(kMinExp, m > 0.875f ? e - 8 : e - 9);
}
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }   // -126 <= e <= 127
__device__ __forceinline__ int exp_of(float pow2_scale) { return (__float_as_int(pow2_scale) >> 23) - 127; }

// finite values or NaN (an infinity would come out as 448)
__device__ __forceinline__ uint32_t encode2(float a, float b) {
  return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
}
__device__ __forceinline__ uint2 encode8(const float* f, float inv) {
  uint2 u;
  u.x = encode2(f[0] * inv, f[1] * inv) | (encode2(f[2] * inv, f[3] * inv) << 16);
  u.y = encode2(f[4] * inv, f[5] * inv) | (encode2(f[6] * inv, f[7] * inv) << 16);
  return u;
}
__device__ __forceinline__ void decode8(uint2 u, float* f) {
  const uint32_t w[4] = {u.x & 0xffffu, u.x >> 16, u.y & 0xffffu, u.y >> 16};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2(__nv_fp8x2_storage_t(w[i]), __NV_E4M3);
    const float2 t = __half22float2(*reinterpret_cast<const __half2*>(&h));
    f[2 * i] = t.x;
    f[2 * i + 1] = t.y;
  }
}

__device__ __forceinline__ void load_w(const float* p, float* f) {
  const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
  f[0] = a.x; f[1] = a.y; f[2] = a.z; f[3] = a.w; f[4] = b.x; f[5] = b.y; f[6] = b.z; f[7] = b.w;
}

struct AppendArgs {
  const void* x[2];            // k, v: token strides ts, head strides hs, batch stride bs (uniform form)
  int64_t bs[2], ts[2], hs[2];
  uint8_t* code[2];            // [pages, H, P, d]
  float* scale[2];             // [pages, H]
  const int* table;            // [B, max_pages]
  int64_t table_stride;
  const int* lens;             // tokens before the call
  const int* cu;               // [B + 1] or null
  int n, total;                // new tokens of each sequence, with `cu` the most of one; of all
  int J, H, P, logP, max_pages, n_pages, n_pos;
  const float* kw;             // [d] or null
  const float* rope;           // [n_pos, d] or null
  bool norm, interleaved, vec;
  float eps;
  int* err;
};

constexpr int kAppendThreads = 128;

// One block: the new tokens of one sequence that fall into one page, for a run
// of units (keys, then values, of one head each). Blocks for 16 an SM: with 8 the
// histories above take 90, with 48 88 us instead of 86. A unit's rows stay in
// registers between the maximum and the encoding; the next unit's are on their
// way meanwhile. A row belongs to D / 16 lanes of 8 + 8 elements that turn against
// each other; PASSES times 128 / (D / 16) rows make a page.
template <typename T, int D, int PASSES>
__global__ void __launch_bounds__(kAppendThreads) append_kernel(const __grid_constant__ AppendArgs A) {
  constexpr int L = D / 16;                          // lanes of a row
  constexpr int R = kAppendThreads / L;              // rows at a time
  const int b = blockIdx.x / A.J, j = blockIdx.x - b * A.J;
  const int len = A.lens[b];
  const int tok0 = A.cu ? A.cu[b] : 0;
  const int n = A.cu ? A.cu[b + 1] - tok0 : A.n;
  if (n <= 0) return;
  if (len < 0 || len > INT32_MAX - 64 - n || n > A.n || (A.cu && (tok0 < 0 || tok0 > A.total - n))) {
    if (threadIdx.x == 0) set_error(A.err, kBadShape);
    return;
  }
  const int pi = (len >> A.logP) + j;                // page of the sequence
  const int64_t p0 = int64_t(pi) << A.logP;          // position of its first row
  const int lo = int(max(int64_t(len) - p0, int64_t(0)));
  const int hi = int(min(int64_t(len) + n - p0, int64_t(A.P)));
  if (hi <= lo) return;
  const int page = pi < A.max_pages ? A.table[b * A.table_stride + pi] : -1;
  if (page < 0 || page >= A.n_pages) {
    if (threadIdx.x == 0) set_error(A.err, kIdOutOfRange);
    return;
  }
  const int first = tok0 + int(p0 - len);            // token of the page's row 0 among the new ones (may be < tok0)
  const int lane = threadIdx.x % L, row0 = threadIdx.x / L;
  int off0, off1;
  bool turned;
  pair_offsets<8>(lane, D, A.rope ? D : 0, A.interleaved, off0, off1, turned);
  __shared__ float s_max[2][kAppendThreads / 32];

  Raw<8, T> xa[PASSES], xc[PASSES];
  auto fetch = [&](int u) {
    const int part = u >= A.H, h = part ? u - A.H : u;
    const T* x = static_cast<const T*>(part ? A.x[1] : A.x[0]) + h * (part ? A.hs[1] : A.hs[0]) +
                 (A.cu ? 0 : b * (part ? A.bs[1] : A.bs[0]));
    const int64_t ts = part ? A.ts[1] : A.ts[0];
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int r = ps * R + row0;
      if (r >= lo && r < hi) {
        const T* xr = x + (first + r) * ts;
        if (A.vec) {
          xa[ps].load(xr + off0);
          xc[ps].load(xr + off1);
        } else {
          T* ea = reinterpret_cast<T*>(xa[ps].v);
          T* ec = reinterpret_cast<T*>(xc[ps].v);
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            ea[e] = xr[off0 + e];
            ec[e] = xr[off1 + e];
          }
        }
      } else {
        xa[ps].zero();
        xc[ps].zero();
      }
    }
  };
  const int per = (2 * A.H + gridDim.y - 1) / gridDim.y, u0 = blockIdx.y * per, u1 = min(2 * A.H, u0 + per);
  if (u0 >= u1) return;
  fetch(u0);
  // where a thread has one row, its angles serve every head
  constexpr bool kHold = PASSES == 1;
  float held_c[8], held_s[8];
  if (kHold && A.rope && u0 < A.H && row0 >= lo && row0 < hi && p0 + row0 < A.n_pos)
    load_angles<8>(A.rope + (p0 + row0) * D, lane, D, A.interleaved, off0, off1, held_c, held_s);
  int buf = 0;
#pragma unroll 1
  for (int u = u0; u < u1; ++u, buf ^= 1) {
    const bool keys = u < A.H;
    const int64_t block = int64_t(page) * A.H + (keys ? u : u - A.H);
    uint8_t* code = (keys ? A.code[0] : A.code[1]) + (block << A.logP) * D;
    float* scale = (keys ? A.scale[0] : A.scale[1]) + block;
    const float old = lo > 0 ? *scale : 0.f;
    float a[PASSES][8], c[PASSES][8];
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      xa[ps].floats(a[ps]);
      xc[ps].floats(c[ps]);
    }
    if (u + 1 < u1) fetch(u + 1);
    float amax = 0.f;                                    // infinities count, NaN does not
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int r = ps * R + row0;
      if (keys && A.norm) {
        const float rs = __frsqrt_rn(group_sum<L>(dot_v<8>(a[ps], a[ps], c[ps], c[ps])) * (1.f / D) + A.eps);
        scale_v<8>(a[ps], rs);
        scale_v<8>(c[ps], rs);
        if (A.kw) {
          float w0[8], w1[8];
          load_w(A.kw + off0, w0);
          load_w(A.kw + off1, w1);
          mul_v<8>(a[ps], w0);
          mul_v<8>(c[ps], w1);
        }
      }
      if (keys && A.rope && r >= lo && r < hi) {
        if (p0 + r < A.n_pos) {
          if constexpr (kHold) {
            turn<8>(a[ps], c[ps], held_c, held_s, A.interleaved, 1.f);
          } else {
            float cs[8], sn[8];
            load_angles<8>(A.rope + (p0 + r) * D, lane, D, A.interleaved, off0, off1, cs, sn);
            turn<8>(a[ps], c[ps], cs, sn, A.interleaved, 1.f);
          }
        } else {
          set_error(A.err, kIdOutOfRange);
#pragma unroll
          for (int e = 0; e < 8; ++e) a[ps][e] = c[ps][e] = 0.f;
        }
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fmaxf(fabsf(a[ps][e]), fabsf(c[ps][e])));
    }
    amax = warp_max(amax);
    if ((threadIdx.x & 31) == 0) s_max[buf][threadIdx.x >> 5] = amax;
    __syncthreads();                                     // also: everyone has read the old scale
#pragma unroll
    for (int w = 0; w < kAppendThreads / 32; ++w) amax = fmaxf(amax, s_max[buf][w]);
    if (amax == INFINITY) {
      // seldom: infinities become NaN and leave the maximum
      amax = 0.f;
#pragma unroll
      for (int ps = 0; ps < PASSES; ++ps) {
  #pragma unroll
        for (int e = 0; e < 8; ++e) {
          if (fabsf(a[ps][e]) == INFINITY) a[ps][e] = NAN;
          if (fabsf(c[ps][e]) == INFINITY) c[ps][e] = NAN;
          amax = fmaxf(amax, fmaxf(fabsf(a[ps][e]), fabsf(c[ps][e])));
        }
      }
      __syncthreads();
      amax = warp_max(amax);
      if ((threadIdx.x & 31) == 0) s_max[buf][threadIdx.x >> 5] = amax;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < kAppendThreads / 32; ++w) amax = fmaxf(amax, s_max[buf][w]);
    }
    int e = scale_exp(amax);
    if (lo > 0) {
      // a scale from elsewhere that is no power of two counts as the next one
      e = max(e, max(kMinExp, min(exp_of(old) + ((__float_as_int(old) & 0x7fffff) != 0), 120)));
      const float ratio = old * pow2(-e);
      if (ratio != 1.f) {
        // the page's scale grows: its old rows move to the new one
#pragma unroll 1
        for (int r = row0; r < lo; r += R) {
          uint2* q0 = reinterpret_cast<uint2*>(code + r * D + lane * 16);
          float f[8];
          decode8(q0[0], f);
          q0[0] = encode8(f, ratio);
          decode8(q0[1], f);
          q0[1] = encode8(f, ratio);
        }
      }
    }
    const float inv = pow2(-e);
#pragma unroll
    for (int ps = 0; ps < PASSES; ++ps) {
      const int r = ps * R + row0;
      if (r >= lo && r < hi) {
        *reinterpret_cast<uint2*>(code + r * D + off0) = encode8(a[ps], inv);
        *reinterpret_cast<uint2*>(code + r * D + off1) = encode8(c[ps], inv);
      }
    }
    if (threadIdx.x == 0) *scale = pow2(e);
  }
}

struct ReadArgs {
  const uint8_t* code[2];
  const float* scale[2];
  const int* table;
  int64_t table_stride;
  const int* lens;
  const int* first;             // [B] or null (0)
  __nv_bfloat16* out[2];        // [B, n, H, d]
  int n, H, P, logP, max_pages, n_pages;
  int chunks;                   // blocks of a sequence
  int* err;
};

// One block: up to 64 tokens of one sequence, all heads. A thread takes 8
// codes of one head's row at a time (16 bytes out, side by side), four times on their way; the pages of the
// block's tokens are looked up once. Bound by the writes (2 bytes a value, 1 read): 34 us for 128 histories, 41 with
// one vector on its way and a division each; eight cost registers and gain nothing.
constexpr int kReadTokens = 64;
constexpr int U = 4;                                 // vectors of a thread on their way

template <int D>
__global__ void __launch_bounds__(256) read_kernel(const ReadArgs A) {
  constexpr int TOK = kReadTokens, L = D / 8;        // threads of a row
  __shared__ int s_row[TOK], s_page[TOK];             // row in its page, its page (or -1)
  const int part = blockIdx.y, b = blockIdx.x / A.chunks, t0 = (blockIdx.x - b * A.chunks) * TOK;
  const int tokens = min(TOK, A.n - t0);
  if (threadIdx.x < tokens) {
    const int64_t pos = int64_t(A.first ? A.first[b] : 0) + t0 + threadIdx.x;
    int page = -1;
    if (pos >= 0 && pos < A.lens[b]) {
      const int64_t pi = pos >> A.logP;
      page = pi < A.max_pages ? A.table[b * A.table_stride + pi] : -1;
      if (page < 0 || page >= A.n_pages) {
        page = -1;
        set_error(A.err, kIdOutOfRange);
      }
    }
    s_page[threadIdx.x] = page;
    s_row[threadIdx.x] = int(pos & (A.P - 1));
  }
  __syncthreads();
  const uint8_t* code = part ? A.code[1] : A.code[0];
  const float* scale = part ? A.scale[1] : A.scale[0];
  __nv_bfloat16* out = (part ? A.out[1] : A.out[0]) + (int64_t(b) * A.n + t0) * A.H * D;
  const int per_token = A.H * L, all = tokens * per_token;
  const int dt = 256 / per_token, dj = 256 - dt * per_token;              // from a thread's vector to its next
  int t = threadIdx.x / per_token, j = threadIdx.x - t * per_token;
#pragma unroll 1
  for (int i0 = threadIdx.x; i0 < all; i0 += 256 * U) {
    uint2 u[U];
    float sc[U];
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int page = i0 + 256 * k < all ? s_page[t] : -1;
      u[k] = make_uint2(0, 0);
      sc[k] = 0.f;
      if (page >= 0) {
        const int block = page * A.H + j / L;
        u[k] = __ldg(reinterpret_cast<const uint2*>(code + (int64_t(block) * A.P + s_row[t]) * D + j % L * 8));
        sc[k] = __ldg(scale + block);
      }
      t += dt;
      j += dj;
      if (j >= per_token) {
        j -= per_token;
        ++t;
      }
    }
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const int i = i0 + 256 * k;
      if (i >= all) break;
      float f[8];
      decode8(u[k], f);
      scale_v<8>(f, sc[k]);
      store_v<8>(out + int64_t(i) * 8, f);
    }
  }
}

// Pages to or from a copy of them, keys or values: block x takes pair x, blocks y share its 16-byte vectors. A pair with
// an id outside the pool is reported and left alone. All sources are read before the first page is written, so a page
// may be another pair's source and destination. Moves each byte four times; not a path whose time matters.
template <bool OUT>
__global__ void __launch_bounds__(256) copy_pages_kernel(const long long* src, const long long* dst, uint4* code,
                                                         float* scale, uint4* tmp, float* tmp_scale, int vecs, int H,
                                                         int n_pages, int* err) {
  const int i = blockIdx.x;
  const long long from = src[i], to = dst[i];
  if (from < 0 || from >= n_pages || to < 0 || to >= n_pages) {
    if (threadIdx.x == 0) set_error(err, kIdOutOfRange);
    return;
  }
  uint4* page = code + (OUT ? from : to) * vecs;
  uint4* copy = tmp + int64_t(i) * vecs;
  for (int v = blockIdx.y * 256 + threadIdx.x; v < vecs; v += gridDim.y * 256) {
    if (OUT) copy[v] = page[v];
    else page[v] = copy[v];
  }
  if (blockIdx.y > 0) return;
  for (int h = threadIdx.x; h < H; h += 256) {
    if (OUT) tmp_scale[int64_t(i) * H + h] = scale[from * H + h];
    else scale[to * H + h] = tmp_scale[int64_t(i) * H + h];
  }
}

// ---------------------------------------------------------------- entry points
// The cache's tensors; returns their sizes.
struct CacheDims { int n_pages, H, P, d; };
CacheDims check_cache(const at::Tensor& k, const at::Tensor& v, const at::Tensor& ks, const at::Tensor& vs,
                      const at::Tensor& err) {
  PD_CHECK(k.is_cuda() && k.dim() == 4 && k.is_contiguous() && k.scalar_type() == at::kFloat8_e4m3fn &&
           v.is_contiguous() && v.sizes() == k.sizes() && v.scalar_type() == k.scalar_type() && v.device() == k.device(),
           "the cache's codes must be contiguous float8_e4m3fn [pages, heads, page_size, d] on one CUDA device");
  PD_CHECK(reinterpret_cast<uintptr_t>(k.data_ptr()) % 16 == 0 && reinterpret_cast<uintptr_t>(v.data_ptr()) % 16 == 0,
           "the cache's codes must lie on 16-byte boundaries");
  const int64_t H = k.size(1), P = k.size(2), d = k.size(3);
  PD_CHECK(P == 16 || P == 32 || P == 64, "page size %d: expected 16, 32 or 64", int(P));
  PD_CHECK(d == 32 || d == 64 || d == 128, "head dim %d of a cache: expected 32, 64 or 128", int(d));
  PD_CHECK(k.size(0) > 0 && H > 0 && H < 32768 && k.size(0) * H * P < (int64_t(1) << 31),
           "a cache has at least one page and head, and fewer than 2^31 rows");
  for (const at::Tensor* s : {&ks, &vs})
    PD_CHECK(s->device() == k.device() && s->scalar_type() == at::kFloat && s->is_contiguous() && s->dim() == 2 &&
             s->size(0) == k.size(0) && s->size(1) == H, "the scales must be contiguous fp32 [pages, heads]");
  PD_CHECK(err.device() == k.device() && err.scalar_type() == at::kInt && err.numel() == 1, "err must be one int32");
  return {int(k.size(0)), int(H), int(P), int(d)};
}

void check_ints(const at::Tensor& t, const at::Tensor& like, int64_t n, const char* what) {
  PD_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous() &&
           t.size(0) == n, "%s must be contiguous int32 [%d] on the cache's device", what, int(n));
}

void check_table(const at::Tensor& t, const at::Tensor& like) {
  PD_CHECK(t.device() == like.device() && t.scalar_type() == at::kInt && t.dim() == 2 &&
           (t.size(1) <= 1 || t.stride(1) == 1), "the page table must be int32 [sequences, pages] on the cache's device");
  // kernels count a sequence's keys in 32 bits, rounded up to their tiles
  PD_CHECK(t.size(1) * like.size(2) <= INT32_MAX - 4096, "a page table has room for 2^31 - 4096 tokens of a sequence at most");
}

template <typename T>
static void append_launch(const AppendArgs& A, dim3 grid, int d) {
#define PD_GO(D, PASSES) append_kernel<T, D, PASSES><<<grid, kAppendThreads, 0, stream()>>>(A)
  if (d == 32) PD_GO(32, 1);
  else if (d == 64 && A.P <= 32) PD_GO(64, 1);
  else if (d == 64) PD_GO(64, 2);
  else if (A.P == 16) PD_GO(128, 1);
  else if (A.P == 32) PD_GO(128, 2);
  else PD_GO(128, 4);
#undef PD_GO
}

void kv_append(at::Tensor ck, at::Tensor cv, at::Tensor ks, at::Tensor vs, at::Tensor err, at::Tensor k, at::Tensor v,
               at::Tensor table, at::Tensor lens, c10::optional<at::Tensor> cu, c10::optional<int64_t> max,
               c10::optional<at::Tensor> k_weight, c10::optional<double> norm_eps, c10::optional<at::Tensor> rope,
               bool interleaved) {
  const CacheDims C = check_cache(ck, cv, ks, vs, err);
  check_table(table, ck);
  const int64_t B = table.size(0);
  check_ints(lens, ck, B, "kv_lens");
  const int dt = dtype_of(k, "k");
  if (k.dim() > 0 && k.stride(-1) != 1) k = k.contiguous();
  if (v.dim() > 0 && v.stride(-1) != 1) v = v.contiguous();
  const int td = cu.has_value() ? 3 : 4;
  AppendArgs A{};
  A.vec = true;
  for (int i = 0; i < 2; ++i) {
    const at::Tensor& x = i == 0 ? k : v;
    PD_CHECK(x.device() == ck.device() && x.scalar_type() == k.scalar_type() && x.dim() == td &&
             x.size(td - 2) == C.H && x.size(td - 1) == C.d && (x.stride(td - 1) == 1 || x.numel() == 0),
             "k and v must be %s of one type on the cache's device, with the cache's heads and head dim and unit "
             "stride on d", cu.has_value() ? "[tokens, heads, d]" : "[sequences, tokens, heads, d]");
    PD_CHECK(x.size(0) == k.size(0) && x.size(td - 3) == k.size(td - 3), "k and v differ in their tokens");
    A.x[i] = x.data_ptr();
    A.bs[i] = td == 4 ? x.stride(0) : 0;
    A.ts[i] = x.stride(td - 3);
    A.hs[i] = x.stride(td - 2);
    const int64_t q = 16 / x.element_size();
    A.vec = A.vec && reinterpret_cast<uintptr_t>(x.data_ptr()) % 16 == 0 && A.bs[i] % q == 0 && A.ts[i] % q == 0 &&
            A.hs[i] % q == 0;
    A.code[i] = static_cast<uint8_t*>((i == 0 ? ck : cv).data_ptr());
    A.scale[i] = (i == 0 ? ks : vs).data_ptr<float>();
  }
  if (cu.has_value()) check_ints(*cu, ck, B + 1, "cu_new");
  else PD_CHECK(k.size(0) == B, "k has %d sequences and the page table %d", int(k.size(0)), int(B));
  const int64_t max_new = max.value_or(k.size(td - 3));
  PD_CHECK(k.size(td - 3) < (int64_t(1) << 31) && max_new >= 0 && max_new < (int64_t(1) << 31), "too many new tokens");
  A.total = int(cu.has_value() ? k.size(0) : 0);
  A.n = int(cu.has_value() ? max_new : k.size(1));
  A.table = table.data_ptr<int>();
  A.table_stride = table.stride(0);
  A.max_pages = int(table.size(1));
  A.lens = lens.data_ptr<int>();
  A.cu = cu.has_value() ? cu->data_ptr<int>() : nullptr;
  A.H = C.H; A.P = C.P; A.n_pages = C.n_pages;
  A.logP = C.P == 16 ? 4 : C.P == 32 ? 5 : 6;
  A.err = err.data_ptr<int>();
  A.interleaved = interleaved;
  A.norm = norm_eps.has_value();
  A.eps = float(norm_eps.value_or(0.));
  if (k_weight.has_value() && !(k_weight->scalar_type() == at::kFloat && k_weight->is_contiguous()))
    k_weight = k_weight->to(at::kFloat).contiguous();
  if (k_weight.has_value()) {
    PD_CHECK(A.norm, "k_weight needs norm_eps");
    PD_CHECK(k_weight->device() == ck.device() && k_weight->scalar_type() == at::kFloat && k_weight->dim() == 1 &&
             k_weight->is_contiguous() && k_weight->size(0) == C.d && reinterpret_cast<uintptr_t>(k_weight->data_ptr()) % 16 == 0,
             "k_weight must be contiguous fp32 [d] on a 16-byte boundary");
    A.kw = k_weight->data_ptr<float>();
  }
  if (rope.has_value()) {
    PD_CHECK(rope->device() == ck.device() && rope->scalar_type() == at::kFloat && rope->dim() == 2 &&
             rope->is_contiguous() && rope->size(1) == C.d && reinterpret_cast<uintptr_t>(rope->data_ptr()) % 16 == 0,
             "rope must be a contiguous fp32 angle table [positions, d] (the cache rotates whole heads)");
    A.rope = rope->data_ptr<float>();
    A.n_pos = int(std::min<int64_t>(rope->size(0), INT32_MAX));
  }
  if (B == 0 || k.size(td - 3) == 0) return;
  // a stated most of 0 launches too: tokens that there are all the same are reported
  const int64_t most = cu.has_value() ? std::max<int64_t>(std::min(max_new, k.size(0)), 1) : k.size(1);
  A.J = int((most + C.P - 2) / C.P + 1);                 // pages that `most` tokens can touch
  PD_CHECK(B * A.J < (int64_t(1) << 31), "too many sequences and pages for one call");
  const c10::cuda::CUDAGuard guard(ck.device());
  // units that a block takes in turn: fewer blocks where there are many pages (16 blocks an SM are enough)
  const int64_t want = (int64_t(num_sms()) * 16 + B * A.J - 1) / (B * A.J);
  const dim3 grid(unsigned(B * A.J), unsigned(std::min<int64_t>(std::max<int64_t>(want, 1), 2 * C.H)));
  if (dt == kBf16) append_launch<__nv_bfloat16>(A, grid, C.d);
  else if (dt == kF16) append_launch<__half>(A, grid, C.d);
  else append_launch<float>(A, grid, C.d);
  PD_CHECK_LAUNCH();
}

void kv_copy_pages(at::Tensor ck, at::Tensor cv, at::Tensor ks, at::Tensor vs, at::Tensor err, at::Tensor src,
                   at::Tensor dst) {
  const CacheDims C = check_cache(ck, cv, ks, vs, err);
  for (const at::Tensor* t : {&src, &dst})
    PD_CHECK(t->device() == ck.device() && t->scalar_type() == at::kLong && t->dim() == 1 && t->is_contiguous() &&
             t->size(0) == src.size(0), "src and dst must be contiguous int64 [n] on the cache's device");
  const int64_t n = src.size(0), vecs = int64_t(C.H) * C.P * C.d / 16;
  PD_CHECK(n < (int64_t(1) << 31) && vecs < (int64_t(1) << 31) - (1 << 24), "too many pages, or too large ones");
  if (n == 0) return;
  const c10::cuda::CUDAGuard guard(ck.device());
  const at::Tensor tmp = at::empty({n, vecs * 16}, ck.options().dtype(at::kByte));
  const at::Tensor tmp_scale = at::empty({n, C.H}, ks.options());
  const dim3 grid(unsigned(n), unsigned(std::min<int64_t>((vecs + 1023) / 1024, 64)));
  for (int i = 0; i < 2; ++i) {
    uint4* code = static_cast<uint4*>((i == 0 ? ck : cv).data_ptr());
    float* scale = (i == 0 ? ks : vs).data_ptr<float>();
    const auto go = [&](auto kern) {
      kern<<<grid, 256, 0, stream()>>>(reinterpret_cast<const long long*>(src.data_ptr<int64_t>()),
                                       reinterpret_cast<const long long*>(dst.data_ptr<int64_t>()), code, scale,
                                       static_cast<uint4*>(tmp.data_ptr()), tmp_scale.data_ptr<float>(), int(vecs), C.H,
                                       C.n_pages, err.data_ptr<int>());
      PD_CHECK_LAUNCH();
    };
    go(copy_pages_kernel<true>);
    go(copy_pages_kernel<false>);
  }
}

std::vector<at::Tensor> kv_read(at::Tensor ck, at::Tensor cv, at::Tensor ks, at::Tensor vs, at::Tensor err,
                                at::Tensor table, at::Tensor lens, c10::optional<at::Tensor> first,
                                c10::optional<int64_t> most) {
  const CacheDims C = check_cache(ck, cv, ks, vs, err);
  check_table(table, ck);
  const int64_t B = table.size(0);
  check_ints(lens, ck, B, "kv_lens");
  if (first.has_value()) check_ints(*first, ck, B, "first");
  const int64_t n = most.value_or(table.size(1) * C.P);
  PD_CHECK(n >= 0 && n < (int64_t(1) << 31), "n must be from 0 to 2^31 - 1");
  const c10::cuda::CUDAGuard guard(ck.device());
  ReadArgs A{};
  std::vector<at::Tensor> out;
  for (int i = 0; i < 2; ++i) {
    A.code[i] = static_cast<const uint8_t*>((i == 0 ? ck : cv).data_ptr());
    A.scale[i] = (i == 0 ? ks : vs).data_ptr<float>();
    out.push_back(at::empty({B, n, C.H, C.d}, ck.options().dtype(at::kBFloat16)));
    A.out[i] = static_cast<__nv_bfloat16*>(out[i].data_ptr());
  }
  A.table = table.data_ptr<int>();
  A.table_stride = table.stride(0);
  A.max_pages = int(table.size(1));
  A.lens = lens.data_ptr<int>();
  A.first = first.has_value() ? first->data_ptr<int>() : nullptr;
  A.n = int(n); A.H = C.H; A.P = C.P; A.n_pages = C.n_pages;
  A.logP = C.P == 16 ? 4 : C.P == 32 ? 5 : 6;
  A.err = err.data_ptr<int>();
  A.chunks = int((n + kReadTokens - 1) / kReadTokens);
  PD_CHECK(B * A.chunks < (int64_t(1) << 31), "too many tokens for one call");
  if (B > 0 && n > 0) {
    const dim3 grid(unsigned(B * A.chunks), 2);
    if (C.d == 32) read_kernel<32><<<grid, 256, 0, stream()>>>(A);
    else if (C.d == 64) read_kernel<64><<<grid, 256, 0, stream()>>>(A);
    else read_kernel<128><<<grid, 256, 0, stream()>>>(A);
    PD_CHECK_LAUNCH();
  }
  return out;
}

}  // namespace kv
}  // namespace pd
