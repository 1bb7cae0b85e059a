// The 8-bit form of a KV cache. A vector (the D values of one token and one kv head, of K or of V) is D e4m3 codes and one power of
// two, 2^e, kept as the byte e + 127: the smallest with max|x| <= 448 * 2^e, and e >= -116. A vector that holds an infinity or a NaN
// has byte 255 and reads as NaN.
//
// Why a power of two: dividing by it and multiplying with it round nothing, so a value is rounded once, to the 3 mantissa bits of its
// code, and what a code stands for is exact in bf16. Attention over an 8-bit cache is then attention over the bf16 values that
// kv_cache_read gives. A scale max|x| / 448 would use up to one binade more of e4m3's 15 for small values, at the price of a second rounding.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp8.h>
#include <stdint.h>

namespace agrpo {

constexpr int kKv8MinByte = 11;   // e = -116: everything below is within half a step of zero
constexpr int kKv8NanByte = 255;
constexpr int kKv8TopByte = 247;  // e = 120: its codes above 240 would stand for 2^128

// Scale byte of a vector whose largest magnitude has these bf16 bits (sign cleared; 448 = 1.75 * 2^8: mantissa 96 of 128).
__device__ __forceinline__ int kv8_scale_byte(uint32_t top) {
  if (top >= 0x7f80u) return kKv8NanByte;
  return max(static_cast<int>(top >> 7) - 8 + ((top & 127u) > 96u ? 1 : 0), kKv8MinByte);
}

// Largest of the magnitudes of 8 bf16 values, as bits.
__device__ __forceinline__ uint32_t kv8_top(const uint4& v) {
  const uint32_t a = __vmaxu2(__vmaxu2(v.x & 0x7fff7fffu, v.y & 0x7fff7fffu), __vmaxu2(v.z & 0x7fff7fffu, v.w & 0x7fff7fffu));
  return max(a & 0xffffu, a >> 16);
}

// Codes of 8 bf16 values under a scale byte.
__device__ __forceinline__ uint2 kv8_encode(const uint4& v, int byte) {
  if (byte == kKv8NanByte) return make_uint2(0u, 0u);
  const float inv = __uint_as_float(static_cast<uint32_t>(254 - byte) << 23);
  const uint32_t w[4] = {v.x, v.y, v.z, v.w};
  float2 f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) f[i] = make_float2(__uint_as_float(w[i] << 16) * inv, __uint_as_float(w[i] & 0xffff0000u) * inv);  // at most 448
  if (byte >= kKv8TopByte) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = make_float2(fminf(fmaxf(f[i].x, -240.f), 240.f), fminf(fmaxf(f[i].y, -240.f), 240.f));
  }
  uint32_t half[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) half[i] = __nv_cvt_float2_to_fp8x2(f[i], __NV_SATFINITE, __NV_E4M3);
  return make_uint2(half[0] | (half[1] << 16), half[2] | (half[3] << 16));
}

__device__ __forceinline__ uint32_t mul_bf16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

// a * 0 + b, for both halves: a NaN where a is infinite or none, for b = 0 and for b that came of this.
__device__ __forceinline__ uint32_t times_zero(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("fma.rn.bf16x2 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(0u), "r"(b));
  return d;
}

__device__ __forceinline__ bool is_finite(uint32_t half) { return (half & 0x7f80u) != 0x7f80u; }  // of a bf16 value in the lower half
__device__ __forceinline__ uint32_t only_finite(uint32_t x) { return (is_finite(x) ? x & 0xffffu : 0u) | (is_finite(x >> 16) ? x & 0xffff0000u : 0u); }

// Factors (both halves of a word) that turn codes moved into bf16's exponent field into what they stand for. An e4m3 code moved there is
// 2^-120 of its value, subnormals included (bias 127 against 7); 2^120 * 2^e is a bf16 number up to e = 7, beyond that a second
// factor follows.
struct Kv8Scale {
  uint32_t first, second;
  bool twice;
};
__device__ __forceinline__ Kv8Scale kv8_scale(int byte) {
  Kv8Scale s;
  const uint32_t a = byte == kKv8NanByte ? 0x7fc0u : static_cast<uint32_t>(min(120 + byte, 254)) << 7;
  s.first = a | (a << 16);
  s.twice = byte > 134 && byte != kKv8NanByte;
  const uint32_t b = static_cast<uint32_t>(byte - 7) << 7;
  s.second = b | (b << 16);
  return s;
}
// Four codes -> four bf16 values. The move of a code by 4 bits and of its sign by 4 more are multiplications: shifts and logic run on a pipe of half the
// rate.
__device__ __forceinline__ uint2 kv8_decode4(uint32_t codes, const Kv8Scale& s) {
  uint32_t lo = __byte_perm(codes, 0u, 0x4140), hi = __byte_perm(codes, 0u, 0x4342);  // a code in the lower byte of each half
  lo = lo * 16u + (lo & 0x00800080u) * 240u;
  hi = hi * 16u + (hi & 0x00800080u) * 240u;
  lo = mul_bf16x2(lo, s.first);
  hi = mul_bf16x2(hi, s.first);
  if (s.twice) {
    lo = mul_bf16x2(lo, s.second);
    hi = mul_bf16x2(hi, s.second);
  }
  return make_uint2(lo, hi);
}

// ---- fp16, for the products over an 8-bit cache
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
// Two e4m3 codes (the lower or the upper half of a word) as fp16.
__device__ __forceinline__ uint32_t codes_f16x2(uint32_t w, bool upper) {
  uint32_t d;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(d) : "r"(upper ? w >> 16 : w));
  return d;
}
__device__ __forceinline__ uint32_t mul_f16x2(uint32_t a, uint32_t b) {
  uint32_t d;
  asm("mul.rn.f16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
  return d;
}

}  // namespace agrpo
