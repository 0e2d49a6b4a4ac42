// 8-bit cache codes: conversions shared by the kernels that write the cache and the one that reads it.
#pragma once

#include "fa_common.cuh"

namespace fa {

// A result rounded towards zero and what it lacks of the exact one: rounded to odd. The last bit of a result that is not
// exact is 1 then, so that rounding it again to a code is rounding the exact one once.
__device__ __forceinline__ float to_odd(float towards_zero, float rest) {
  return __uint_as_float(__float_as_uint(towards_zero) | (fabsf(rest) > 0.f ? 1u : 0u));
}

__device__ __forceinline__ float odd_product(float x, float y) {
  const float p = __fmul_rz(x, y);
  return to_odd(p, fmaf(x, y, -p));
}

// e4m3: 1 sign, 4 exponent (bias 7), 3 mantissa bits; largest finite value 448 = 1.75 * 2^8, code 0x7f is NaN.
// int8: -127 .. 127. Every e4m3 and every int8 value is an fp16 value, so codes become fp16 without rounding.
struct CodeE4M3 {
  // biased fp32 exponent of 448 (minus the bias), and the fp32 mantissa field above which 2^e * 448 is too small
  static constexpr int kTopExp = 8;
  static constexpr uint32_t kTopMant = 0x600000u;
  // bytes 0, 1 (lo) or 2, 3 (hi) of x as two fp16 values
  __device__ static __forceinline__ uint32_t lo(uint32_t x) {
    uint32_t r;
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, l;}" : "=r"(r) : "r"(x));
    return r;
  }
  __device__ static __forceinline__ uint32_t hi(uint32_t x) {
    uint32_t r;
    asm("{.reg .b16 l, h; mov.b32 {l, h}, %1; cvt.rn.f16x2.e4m3x2 %0, h;}" : "=r"(r) : "r"(x));
    return r;
  }
  // four values in units of the scale -> four codes, round to nearest even; infinities saturate, NaN stays NaN
  __device__ static __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    uint32_t r;
    asm("{.reg .b16 l, h; cvt.rn.satfinite.e4m3x2.f32 l, %2, %1; cvt.rn.satfinite.e4m3x2.f32 h, %4, %3; "
        "mov.b32 %0, {l, h};}"
        : "=r"(r)
        : "f"(a), "f"(b), "f"(c), "f"(d));
    return r;
  }
  __device__ static __forceinline__ uint32_t pack4_times(float a, float b, float c, float d, float f) {
    const uint64_t ff = pack_f32x2(f, f), x = mul_f32x2(pack_f32x2(a, b), ff), y = mul_f32x2(pack_f32x2(c, d), ff);
    unpack_f32x2(x, &a, &b);
    unpack_f32x2(y, &c, &d);
    return pack4(a, b, c, d);
  }
  // older codes under a new scale: times the ratio of the two
  __device__ static __forceinline__ uint32_t pack4_codes(float2 lo, float2 hi, float ratio) {
    return pack4(odd_product(lo.x, ratio), odd_product(lo.y, ratio), odd_product(hi.x, ratio), odd_product(hi.y, ratio));
  }
  // fp16 pairs times a power of two: exact, or below fp16's normal range, where every code is 0 (half of the smallest is 2^-10)
  __device__ static __forceinline__ uint32_t pack4_half(__half2 lo, __half2 hi, __half2 f) {
    const __half2 x = __hmul2(lo, f), y = __hmul2(hi, f);
    uint32_t r;
    asm("{.reg .b16 l, h; cvt.rn.satfinite.e4m3x2.f16x2 l, %1; cvt.rn.satfinite.e4m3x2.f16x2 h, %2; mov.b32 %0, {l, h};}"
        : "=r"(r)
        : "r"(*reinterpret_cast<const uint32_t*>(&x)), "r"(*reinterpret_cast<const uint32_t*>(&y)));
    return r;
  }
};

struct CodeInt8 {
  static constexpr int kTopExp = 6;  // 127 = 1.984375 * 2^6
  static constexpr uint32_t kTopMant = 0x7e0000u;
  // byte b ^ 0x80 = b + 128 under the exponent of 1024 is the fp16 value 1024 + 128 + b; 1152 is taken off exactly
  __device__ static __forceinline__ uint32_t unbias(uint32_t u) {
    const __half2 h = __hsub2(*reinterpret_cast<__half2*>(&u), __half2half2(__ushort_as_half(0x6480)));
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  __device__ static __forceinline__ uint32_t lo(uint32_t x) {
    return unbias(__byte_perm(x ^ 0x80808080u, 0x64646464u, 0x4140));
  }
  __device__ static __forceinline__ uint32_t hi(uint32_t x) {
    return unbias(__byte_perm(x ^ 0x80808080u, 0x64646464u, 0x4342));
  }
  __device__ static __forceinline__ int code(float v) { return max(-127, min(127, __float2int_rn(v))); }  // NaN: 0
  __device__ static __forceinline__ uint32_t pack4(float a, float b, float c, float d) {
    return __byte_perm(__byte_perm(code(a), code(b), 0x0040), __byte_perm(code(c), code(d), 0x0040), 0x5410);
  }
  // Finite values times a power of two that takes them into the range: in 1.5 * 2^23 + x the sum's last bit is 1, so
  // the addition rounds x to nearest even and leaves its two's complement in the low bits (four cvt would run at a
  // quarter of the rate)
  __device__ static __forceinline__ uint32_t pack4_times(float a, float b, float c, float d, float f) {
    const uint64_t ff = pack_f32x2(f, f), magic = pack_f32x2(12582912.f, 12582912.f);
    const uint64_t x = fma_f32x2(pack_f32x2(a, b), ff, magic), y = fma_f32x2(pack_f32x2(c, d), ff, magic);
    unpack_f32x2(x, &a, &b);
    unpack_f32x2(y, &c, &d);
    return __byte_perm(__byte_perm(__float_as_uint(a), __float_as_uint(b), 0x0040),
                       __byte_perm(__float_as_uint(c), __float_as_uint(d), 0x0040), 0x5410);
  }
  // Older codes under a new scale: the product is exact inside the fused addition. (A code of -128, which only the caller
  // can have written, becomes -127 at least; ratios above 1 only come from a scale that was no positive number.)
  __device__ static __forceinline__ uint32_t pack4_codes(float2 lo, float2 hi, float ratio) {
    if (!(fabsf(ratio) <= 1.f))
      return pack4(odd_product(lo.x, ratio), odd_product(lo.y, ratio), odd_product(hi.x, ratio), odd_product(hi.y, ratio));
    return __vmaxs4(pack4_times(lo.x, lo.y, hi.x, hi.y, ratio), 0x81818181u);
  }
  // The same in fp16, whose 1.5 * 2^10 + x has a last bit of 1 too: the product is exact inside the fused addition
  __device__ static __forceinline__ uint32_t pack4_half(__half2 lo, __half2 hi, __half2 f) {
    const __half2 magic = __half2half2(__ushort_as_half(0x6600));
    const __half2 x = __hfma2(lo, f, magic), y = __hfma2(hi, f, magic);
    return __byte_perm(*reinterpret_cast<const uint32_t*>(&x), *reinterpret_cast<const uint32_t*>(&y), 0x6420);
  }
};

}  // namespace fa
