// Element access and rotation helpers shared by the rotary and key/value-cache
// kernels (kv_*.cu).
#pragma once

#include <cuda_fp16.h>

#include "common.cuh"

namespace pd {
namespace kv {

enum Dtype : int { kBf16 = 0, kF16 = 1, kF32 = 2 };

inline int dtype_of(const at::Tensor& t, const char* what) {
  const auto s = t.scalar_type();
  PD_CHECK(s == at::kBFloat16 || s == at::kHalf || s == at::kFloat, "%s: expected bf16, fp16 or fp32", what);
  return s == at::kBFloat16 ? kBf16 : s == at::kHalf ? kF16 : kF32;
}

template <typename T> __device__ __forceinline__ float to_f(T v);
template <> __device__ __forceinline__ float to_f(float v) { return v; }
template <> __device__ __forceinline__ float to_f(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_f(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_f(float v);
template <> __device__ __forceinline__ float from_f(float v) { return v; }
template <> __device__ __forceinline__ __half from_f(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_f(float v) { return __float2bfloat16_rn(v); }

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

// V consecutive elements as they lie in memory; V = 8 moves 16 bytes an access
// and needs 16-byte aligned addresses, V = 1 takes any element.
template <int V, typename T>
struct Raw {
  static constexpr int N = V == 1 ? 1 : int(sizeof(T)) / 2;      // uint4s of 8 elements
  T one;
  uint4 v[N];
  __device__ __forceinline__ void load(const T* p) {
    if constexpr (V == 1) {
      one = *p;
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = *(reinterpret_cast<const uint4*>(p) + i);
    }
  }
  __device__ __forceinline__ void zero() {
    one = T(0.f);
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = make_uint4(0, 0, 0, 0);
  }
  __device__ __forceinline__ void floats(float* f) const {
    if constexpr (V == 1) {
      f[0] = to_f(one);
    } else {
      const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) f[i] = to_f(e[i]);
    }
  }
};
template <int V, typename T>
__device__ __forceinline__ void store_v(T* p, const float* f) {
  if constexpr (V == 1) {
    *p = from_f<T>(f[0]);
  } else if constexpr (sizeof(T) == 4) {
    *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]);
    *(reinterpret_cast<float4*>(p) + 1) = make_float4(f[4], f[5], f[6], f[7]);
  } else {
    uint4 u;
    T* e = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 8; ++i) e[i] = from_f<T>(f[i]);
    *reinterpret_cast<uint4*>(p) = u;
  }
}

// Where a row's elements lie that one lane holds together: pair j of V + V
// elements starts at off0 and off1. In the rotated part [0, rot) the halves
// turn against each other (pair j covers elements j V.. of both halves); with
// interleaved pairs any V (even) neighbours close on themselves. The rest
// [rot, d) is split into halves the same way and not turned.
template <int V>
__device__ __forceinline__ void pair_offsets(int j, int d, int rot, bool interleaved, int& off0, int& off1,
                                             bool& turned) {
  turned = j * V < rot / 2;
  if (V == 1 && interleaved) {
    off0 = 2 * j;
    off1 = off0 + 1;
  } else if (turned) {
    off0 = j * V;
    off1 = rot / 2 + j * V;
  } else {
    off0 = rot + (j * V - rot / 2);
    off1 = off0 + (d - rot) / 2;
  }
}

// cos and sin of the elements of one pair, at[...] = a row of the angle table
// (cos of rot / 2 frequencies, then sin). For interleaved vectors the V angles
// are those of off0's V / 2 pairs, then off1's.
template <int V>
__device__ __forceinline__ void load_angles(const float* at, int j, int rot, bool interleaved, int off0, int off1,
                                            float* c, float* s) {
  const int h = rot / 2;
  if constexpr (V == 1) {
    c[0] = __ldg(at + j);
    s[0] = __ldg(at + h + j);
  } else {
    const int i0 = interleaved ? off0 / 2 : off0, i1 = interleaved ? off1 / 2 : off0 + 4;
    const float4 c0 = __ldg(reinterpret_cast<const float4*>(at + i0)), c1 = __ldg(reinterpret_cast<const float4*>(at + i1));
    const float4 s0 = __ldg(reinterpret_cast<const float4*>(at + h + i0));
    const float4 s1 = __ldg(reinterpret_cast<const float4*>(at + h + i1));
    c[0] = c0.x; c[1] = c0.y; c[2] = c0.z; c[3] = c0.w; c[4] = c1.x; c[5] = c1.y; c[6] = c1.z; c[7] = c1.w;
    s[0] = s0.x; s[1] = s0.y; s[2] = s0.z; s[3] = s0.w; s[4] = s1.x; s[5] = s1.y; s[6] = s1.z; s[7] = s1.w;
  }
}

__device__ __forceinline__ uint64_t pk2_add(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

// Vectors of V values as packed pairs (one instruction for two values).
template <int V>
__device__ __forceinline__ void scale_v(float* a, float r) {               // a *= r
  if constexpr (V == 1) {
    a[0] *= r;
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) pk2_split(pk2_mul(pk2(a[i], a[i + 1]), pk2s(r)), a[i], a[i + 1]);
  }
}
template <int V>
__device__ __forceinline__ void mul_v(float* a, const float* w) {          // a *= w
  if constexpr (V == 1) {
    a[0] *= w[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) pk2_split(pk2_mul(pk2(a[i], a[i + 1]), pk2(w[i], w[i + 1])), a[i], a[i + 1]);
  }
}
template <int V>
__device__ __forceinline__ void add_mul_v(float* s, const float* a, const float* b) {     // s += a b
  if constexpr (V == 1) {
    s[0] = fmaf(a[0], b[0], s[0]);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2)
      pk2_split(pk2_fma(pk2(a[i], a[i + 1]), pk2(b[i], b[i + 1]), pk2(s[i], s[i + 1])), s[i], s[i + 1]);
  }
}
// sum of a0 b0 + a1 b1 over the vectors
template <int V>
__device__ __forceinline__ float dot_v(const float* a0, const float* b0, const float* a1, const float* b1) {
  if constexpr (V == 1) {
    return a0[0] * b0[0] + a1[0] * b1[0];
  } else {
    uint64_t s = pk2_mul(pk2(a0[0], a0[1]), pk2(b0[0], b0[1])), t = pk2_mul(pk2(a1[0], a1[1]), pk2(b1[0], b1[1]));
#pragma unroll
    for (int i = 2; i < V; i += 2) {
      s = pk2_fma(pk2(a0[i], a0[i + 1]), pk2(b0[i], b0[i + 1]), s);
      t = pk2_fma(pk2(a1[i], a1[i + 1]), pk2(b1[i], b1[i + 1]), t);
    }
    float x, y;
    pk2_split(pk2_add(s, t), x, y);
    return x + y;
  }
}

// Turns a pair in place by the angles of load_angles (sgn = 1) or back (sgn = -1).
template <int V>
__device__ __forceinline__ void turn(float* a, float* b, const float* c, const float* s, bool interleaved, float sgn) {
  if (V > 1 && interleaved) {
#pragma unroll
    for (int i = 0; i < V / 2; ++i) {
      const float s0 = s[i] * sgn, s1 = s[V / 2 + i] * sgn;
      const float x = a[2 * i], y = a[2 * i + 1], z = b[2 * i], w = b[2 * i + 1];
      a[2 * i] = x * c[i] - y * s0;
      a[2 * i + 1] = x * s0 + y * c[i];
      b[2 * i] = z * c[V / 2 + i] - w * s1;
      b[2 * i + 1] = z * s1 + w * c[V / 2 + i];
    }
  } else if constexpr (V == 1) {
    const float x = a[0], y = b[0], si = s[0] * sgn;
    a[0] = x * c[0] - y * si;
    b[0] = x * si + y * c[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const uint64_t x = pk2(a[i], a[i + 1]), y = pk2(b[i], b[i + 1]), cc = pk2(c[i], c[i + 1]);
      const uint64_t ps = pk2(s[i], s[i + 1]), ns = pk2(-s[i], -s[i + 1]);
      pk2_split(pk2_fma(y, sgn > 0.f ? ns : ps, pk2_mul(x, cc)), a[i], a[i + 1]);
      pk2_split(pk2_fma(x, sgn > 0.f ? ps : ns, pk2_mul(y, cc)), b[i], b[i + 1]);
    }
  }
}

template <int L>
__device__ __forceinline__ float group_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}

}  // namespace kv
}  // namespace pd
