// Shared by the 8-bit integer kernels (int8_*.cu and the GEMM epilogues that
// save activations): codes with power-of-two scales for blocks of 32 values.
//
// A block's scale byte b stands for 2^(b - 127), the smallest power with
// max |x| <= 127 * 2^(b - 127), at least 2^-126 (scale and reciprocal stay
// normal numbers). Codes are rint(x 2^(127 - b)); code * scale has at most 7
// significant bits, so the loaded value is exact in bf16 (and in fp16 within
// its normal range) and enters a tensor-core product unrounded.
#pragma once

#include "common.cuh"

namespace pd {
namespace i8 {

constexpr int kBlock = 32;              // values that share a scale
constexpr uint32_t kNanByte = 255;      // a block with a NaN or an infinity: loads as NaN
// The one scale byte at which code 64 would pass the type's largest value; codes are held to 63 there.
constexpr uint32_t kTopWide = 249;      // bf16, fp32: 64 * 2^122
constexpr uint32_t kTopHalf = 137;      // fp16: 64 * 2^10

// |x| as an integer: orders like the value, NaN above infinity above numbers.
__device__ __forceinline__ uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// amax = m 2^k, 1 <= m < 2; 127 = 1.984375 * 2^6, whose mantissa field is 0x7e0000: adding 0x1ffff carries into the
// exponent exactly where m > 1.984375.
__device__ __forceinline__ uint32_t scale_byte(uint32_t amax_bits) {
  const int b = int((amax_bits + 0x1ffffu) >> 23) - 6;
  return amax_bits >= 0x7f800000u ? kNanByte : uint32_t(max(b, 1));
}
__device__ __forceinline__ float scale_of(uint32_t byte) {
  return __uint_as_float(byte == kNanByte ? 0x7fc00000u : byte << 23);
}
__device__ __forceinline__ float inv_scale(uint32_t byte) {
  return __uint_as_float(byte == kNanByte ? 0u : (254u - byte) << 23);
}

// The largest code of a block: 0 where the block holds no numbers.
__device__ __forceinline__ float most_code(uint32_t byte, uint32_t top) {
  return byte == kNanByte ? 0.0f : byte == top ? 63.0f : 127.0f;
}

// Four codes as bytes. x * inv is at most 127 by the choice of the scale; 12582912 = 1.5 * 2^23 rounds the sum to the
// nearest integer (ties to even) into the low mantissa bits, whose low byte is the code in two's complement.
__device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, float inv, float most) {
  auto one = [&](float v) {
    return __float_as_uint(__fadd_rn(fminf(fmaxf(__fmul_rn(v, inv), -most), most), 12582912.0f));
  };
  const uint32_t lo = __byte_perm(one(a), one(b), 0x0040), hi = __byte_perm(one(c), one(d), 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// Four codes of a block by its power-of-two scale: x * inv is exact, so one fused multiply-add rounds it to the integer.
__device__ __forceinline__ uint32_t block_codes4(const float* x, float inv) {
  uint32_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) c[i] = __float_as_uint(fmaf(x[i], inv, 12582912.0f));
  return __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
}
// max(|a|, |b|, |c|); NaN where one of them is.
__device__ __forceinline__ float max_abs3(float a, float b, float c) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
// The 32 values of a block in one thread's registers: its codes, and its scale byte.
__device__ __forceinline__ uint32_t save_block(const float* v, uint32_t top, uint32_t (&w)[8]) {
  float m0 = 0.0f, m1 = 0.0f;
#pragma unroll
  for (int i = 0; i < 32; i += 4) {
    m0 = max_abs3(m0, v[i], v[i + 1]);
    m1 = max_abs3(m1, v[i + 2], v[i + 3]);
  }
  const uint32_t byte = scale_byte(__float_as_uint(max_abs3(m0, m1, 0.0f)));
  const float inv = inv_scale(byte);
#pragma unroll
  for (int i = 0; i < 8; ++i) w[i] = block_codes4(v + 4 * i, inv);
  if (byte >= top) {                                      // no numbers, or codes held to 63: rare
    const float most = most_code(byte, top);
#pragma unroll
    for (int i = 0; i < 8; ++i) w[i] = codes4(v[4 * i], v[4 * i + 1], v[4 * i + 2], v[4 * i + 3], inv, most);
  }
  return byte;
}

// The values of four codes: byte + 128 below 2^23's mantissa, less 2^23 + 128, times the block's scale.
__device__ __forceinline__ void values4(uint32_t codes, float scale, float* f) {
  const uint32_t u = codes ^ 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f[i] = __fmul_rn(__fsub_rn(__uint_as_float(__byte_perm(u, 0x4b000000u, 0x7540 + i)), 8388736.0f), scale);
}

// Whole rows with a 32-bit scale: max(amax / 127, 2^-126) and its reciprocal; a row without numbers has codes of 0 and a
// scale of NaN.
struct RowScale { float scale, inv, most; };
__device__ __forceinline__ RowScale row_scale(uint32_t amax_bits) {
  const bool fine = amax_bits < 0x7f800000u;
  RowScale r;
  r.scale = fine ? fmaxf(__fmul_rn(__uint_as_float(amax_bits), 1.0f / 127.0f), 1.17549435e-38f) : __uint_as_float(0x7fc00000u);
  r.inv = fine ? __frcp_rn(r.scale) : 0.0f;
  r.most = fine ? 127.0f : 0.0f;
  return r;
}

enum Act : int { kIdentity = 0, kGelu = 1, kRelu = 2 };

// GELU of what lies below -1e30 is 0, of a sum that overflowed to -infinity too (-infinity * 0 would be NaN); NaN stays.
__device__ __forceinline__ float from_below(float v) {
  float r;
  asm("max.NaN.f32 %0, %1, 0fF149F2CA;" : "=f"(r) : "f"(v));          // -1e30
  return r;
}

}  // namespace i8
}  // namespace pd
