// The 4-bit K/V pool's row format, shared by the kernels that write it and those that read it (gfx950).
//
// A row is one token of one KV head: 128 e2m1 codes (sign, 2 exponent bits, 1 mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6), two a
// byte with the even dim in the low half, and one exponent byte s for each block of 32 dims, value = code * 2^(s - 127).  The
// writer takes the smallest power of two that brings the block's largest magnitude a to at most 7:
//   a = f * 2^x with 1 <= f < 2;  7 = 1.75 * 2^2;  e = x - 2 (+ 1 if f > 1.75), in [-125, 125];  s = e + 127.
// Up to 7 and not to 6, the largest code: 6 is the nearest code to all up to 7 (the next one would be 8), and the block's other
// elements gain a bit.  Over normal and Laplace distributed rows the squared error is 6 to 12 % lower than with 6, and 5 % lower
// than with 8 (which clips); it is within 2 % of taking the better of both scales block by block.
// Rounding to the code (nearest, ties to the even one) is the only rounding: the value read back is a bf16 number as it is, and
// attention over the pool equals attention over the bf16 rows read back from it.  At e = -125 the smallest code, 0.5, is 2^-126,
// still a normal number; at 125 the largest is 1.5 * 2^127, and magnitudes over 7 * 2^125 become that.
// A code has no NaN.  A block with an element that is not finite is held as NaN, whole: s = 255 and codes 0.  The exponent byte
// with this meaning, and the conversions that take it along, are the chip's own (v_cvt_scalef32_pk_*_fp4).
#pragma once

#include "fp8_common.h"

namespace q3a {

constexpr int kFp4Row = kRowDims / 2;      // bytes of codes
constexpr int kFp4Blocks = kRowDims / 32;  // exponent bytes
constexpr int kFp4MinByte = 2, kFp4MaxByte = 252, kFp4NanByte = 255;

// bf16 magnitude bits of the block's largest element (0..0x7fff) -> exponent byte.
__device__ __forceinline__ uint32_t fp4_scale_byte(uint32_t amax_bf16) {
  const int s = (int)(amax_bf16 >> 7) - 2 + ((amax_bf16 & 0x7f) > 0x60 ? 1 : 0);
  return amax_bf16 >= 0x7f80u ? (uint32_t)kFp4NanByte : (uint32_t)max(kFp4MinByte, min(s, kFp4MaxByte));
}

// Four dwords of bf16 (8 elements) -> one dword of codes at the exponent byte s.  (The conversion rounds to nearest even and
// saturates at 6.)
__device__ __forceinline__ uint32_t fp4_codes8(uint32_t w0, uint32_t w1, uint32_t w2, uint32_t w3, uint32_t s) {
  const float f = fp8_scale(s);
  uint32_t r = 0;
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, w0), f, 0);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, w1), f, 1);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, w2), f, 2);
  r = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(r, __builtin_bit_cast(bf16x2_t, w3), f, 3);
  return s == kFp4NanByte ? 0u : r;
}

// Byte kByte (two codes) of a dword of codes -> a pair of bf16, times 2^(s - 127) with `scale` = fp8_scale(s): exact for the
// bytes that the writer makes, NaN for 255.
template <int kByte>
__device__ __forceinline__ uint32_t fp4_pair(uint32_t w, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, kByte));
}

// A pool's pointers, strides (in bytes) and sizes as every entry point over it needs them (kv_fp4.hip): Q3A_OK, or the error for
// the caller.
int check_fp4_pool(const char* who, const void* kc, const void* vc, int64_t sp, int64_t st, int64_t sh, const void* ks,
                   const void* vs, int64_t ss_p, int64_t ss_h, int num_pages, int page_size, int hkv);

}  // namespace q3a
