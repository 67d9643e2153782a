// Keys and values in 8 bits: 16 consecutive values of a head have one scale byte and a code byte each.
//
//   scale byte s: the f16 number d with the bits s << 7 - five bits of exponent, four significant bits - up to 0xBF (480); 0xC0 and above stand
//                 for 16 values that are not numbers (some value was not finite, or past 127 * 480 = 60960)
//   code byte c:  the value (c - 128) d
//
// d is the least such number with 127 d >= the largest magnitude, so a value is off by d / 2 at most.  Four significant bits make every value an f16
// number ((c - 128) has seven bits and a sign: eleven together), so that all kernels work on the same values, from the codes or from an f16 copy of them,
// and cost at most an eighth of a step against a scale of full precision (4.5% on average), which the blocks of 16 instead of 32 more than give back:
// 17 bytes for 16 values, as many as Q8_0 has.
#pragma once
#include <cuda_fp16.h>

#include "common.cuh"

namespace infr {

constexpr uint32_t Q8_ODD = 0xC0;  // scale bytes from here on: not numbers

#ifdef __CUDACC__

// Scale byte of 16 values whose largest magnitude is `big` (NaN where one is).
__device__ __forceinline__ uint32_t q8_scale_byte(float big) {
  const float t = __fdiv_rn(big, 127.f);
  if (!(t <= 480.f)) return 0xFFu;
  // (below 2^-14 f16 numbers are multiples of 2^-24; the byte's of 2^-17)
  if (t < 0x1p-14f) return (uint32_t)max((int)ceilf(t * 0x1p17f), big > 0.f ? 1 : 0);  // (the quotient may have underflowed)
  return ((__float_as_uint(t) + 0xFFFFFu) >> 20) - (112u << 3);
}

__device__ __forceinline__ float q8_scale(uint32_t s) {
  return __half2float(__ushort_as_half((unsigned short)(s < Q8_ODD ? s << 7 : 0x7FFFu)));
}

// Four values as codes, low byte first; r = 1 / d (0 where d is 0, or not a number).
__device__ __forceinline__ uint32_t q8_codes4(const float4& v, float r) {
  auto code = [r](float x) { return (uint32_t)(__float2int_rn(fminf(fmaxf(x * r, -127.f), 127.f)) + 128); };
  return code(v.x) | code(v.y) << 8 | code(v.z) << 16 | code(v.w) << 24;
}
__device__ __forceinline__ float q8_inverse(uint32_t s) { return s == 0 || s >= Q8_ODD ? 0.f : __frcp_rn(q8_scale(s)); }

// Codes as f16 pairs: the byte b behind 0x64 is 1024 + b.
__device__ __forceinline__ uint32_t q8_pair(uint32_t bytes_behind, uint32_t d2) {
  const __half2 u = *reinterpret_cast<const __half2*>(&bytes_behind), d = *reinterpret_cast<const __half2*>(&d2);
  const __half2 x = __hmul2(__hsub2(u, __half2half2(__ushort_as_half(0x6480))), d);  // - 1152: exact, and so is the product
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t q8_lo(uint32_t codes, uint32_t d2) { return q8_pair(__byte_perm(codes, 0x64646464u, 0x4140), d2); }
__device__ __forceinline__ uint32_t q8_hi(uint32_t codes, uint32_t d2) { return q8_pair(__byte_perm(codes, 0x64646464u, 0x4342), d2); }
// The same times 2^-5, in one operation where several pairs share their scales: (1024 + b) d / 32 - 36 d.  Exact too: 36 d, unlike 1152 d, is an f16 number.
__device__ __forceinline__ void q8_32nds(uint32_t d2, uint32_t& d32, uint32_t& off) {
  const __half2 d = *reinterpret_cast<const __half2*>(&d2), a = __hmul2(d, __half2half2(__ushort_as_half(0x2800))), b = __hmul2(d, __half2half2(__ushort_as_half(0xD080)));
  d32 = *reinterpret_cast<const uint32_t*>(&a), off = *reinterpret_cast<const uint32_t*>(&b);
}
__device__ __forceinline__ uint32_t q8_pair32(uint32_t bytes_behind, uint32_t d32, uint32_t off) {
  const __half2 x = __hfma2(*reinterpret_cast<const __half2*>(&bytes_behind), *reinterpret_cast<const __half2*>(&d32), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<const uint32_t*>(&x);
}
__device__ __forceinline__ uint32_t q8_lo32(uint32_t codes, uint32_t d32, uint32_t off) { return q8_pair32(__byte_perm(codes, 0x64646464u, 0x4140), d32, off); }
__device__ __forceinline__ uint32_t q8_hi32(uint32_t codes, uint32_t d32, uint32_t off) { return q8_pair32(__byte_perm(codes, 0x64646464u, 0x4342), d32, off); }
// A scale byte as a pair of the same f16 number.
__device__ __forceinline__ uint32_t q8_scale_pair(uint32_t s) { return (s < Q8_ODD ? s << 7 : 0x7FFFu) * 0x10001u; }

#endif

}  // namespace infr
